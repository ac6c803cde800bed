"""Rotary positions, the e4m3 paged cache and attention over it in float64
numpy — TEST INFRASTRUCTURE ONLY (see the package docstring).

Not in the reference; these functions restate the definitions of the calls
around a KV cache so that the kernels can be checked against them:

* ``rotate`` — y1 = s (x1 cos a - x2 sin a), y2 = s (x2 cos a + x1 sin a), a =
  position * inv_freq, pairs (i, i + n) or (2 i, 2 i + 1), the rest copied.  Pinned by
  closed forms (position 0, a quarter turn, norms, composition of positions).
* ``append`` — tokens into pages; in 8 bits the runs' scales and codes.  Pinned by the
  invariants that define them.
* ``decode`` — attention of a row's newest queries over its dequantised keys.
  Pinned against ``attention.forward``.
"""
import numpy as np

from . import fp8

RUN = 32


def rotate(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False) -> np.ndarray:
    """(B, H, T, D) float64 rotated to positions (B, T)."""
    x = np.asarray(x, np.float64)
    f = np.asarray(inv_freq, np.float64)
    n = f.size
    a = np.asarray(positions, np.float64)[:, None, :, None] * f
    c, s = scale * np.cos(a), scale * np.sin(a) * (-1.0 if inverse else 1.0)
    y = x.copy()
    i0, i1 = (np.arange(n) * 2, np.arange(n) * 2 + 1) if interleaved else (np.arange(n), np.arange(n) + n)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def run_scale(amax: float) -> float:
    """The smallest 2^e, -126 <= e <= 127, with 448 2^e >= amax."""
    if not amax > 0:
        return 2.0 ** -126
    m, e = np.frexp(amax / 448.0)
    return float(2.0 ** min(max(int(e) - (m == 0.5), -126), 127))


def append(cache, scales, x, kv_lens, page_table, new_lens=None):
    """Copies of ``cache`` (num_pages, H, page, D) and ``scales`` (num_pages, H,
    page / 32) with tokens x (B, H, T, D) float64 appended.  With ``scales`` the cache holds
    e4m3 codes (uint8); without, the unrounded values."""
    cache = np.array(cache)
    scales = None if scales is None else np.array(scales)
    B, H, T, _ = x.shape
    P, _, page, _ = cache.shape
    for b in range(B):
        n = T if new_lens is None else min(max(int(new_lens[b]), 0), T)
        t, base = 0, int(kv_lens[b])
        while t < n and base >= 0:
            pos = base + t
            upto = min(n, t + RUN - pos % RUN)
            pg, row, kept = pos // page, pos % page, pos % RUN
            run = x[b, :, t:upto]
            t0, t = t, upto
            if pg >= page_table.shape[1]:
                break
            pid = int(page_table[b, pg])
            if not 0 <= pid < P:
                continue
            kept = min(kept, base % RUN) if pos // RUN == base // RUN else 0
            for h in range(H):
                v = run[h]
                if scales is not None:
                    g = row // RUN
                    fin = np.abs(v[np.isfinite(v)])
                    s = run_scale(float(fin.max()) if fin.size else 0.0)
                    if kept:
                        had = float(scales[pid, h, g])
                        s = max(s, had)
                        old = cache[pid, h, row - kept:row]
                        if s > had:
                            val = fp8.decode_e4m3(old).astype(np.float64) * (had / s)
                            cache[pid, h, row - kept:row] = fp8.encode_e4m3(val)
                    scales[pid, h, g] = s
                    with np.errstate(invalid="ignore"):
                        v = fp8.encode_e4m3(v / s)
                cache[pid, h, row:row + upto - t0] = v
    return cache, scales


def decode(q, keys, values, kv_lens, q_lens=None, left=-1, right=-1, scale=None, slopes=None, softcap=0.0):
    """(o, lse, weight) of q (B, Hq, Sq, D) over keys / values (B, Hkv, S, D), float64: query i of
    row b at position kv_lens[b] - q_lens[b] + i; weight = sum p |v|, the size of O's terms."""
    q = np.asarray(q, np.float64)
    B, Hq, Sq, D = q.shape
    g = Hq // keys.shape[1]
    sc = D ** -0.5 if scale is None else scale
    o, w = np.zeros((B, Hq, Sq, D)), np.zeros((B, Hq, Sq, D))
    lse = np.full((B, Hq, Sq), -np.inf)
    for b in range(B):
        have = int(kv_lens[b])
        ql = Sq if q_lens is None else min(max(int(q_lens[b]), 0), Sq)
        for i in range(ql):
            at = have - ql + i
            lo = 0 if left < 0 else max(0, at - left)
            hi = have if right < 0 else min(have, at + right + 1)
            if hi <= lo:
                continue
            for h in range(Hq):
                k = np.asarray(keys[b, h // g, lo:hi], np.float64)
                v = np.asarray(values[b, h // g, lo:hi], np.float64)
                s = sc * (k @ q[b, h, i])
                if slopes is not None:
                    s = s + float(slopes[h]) * (np.arange(lo, hi) - at)
                if softcap > 0:
                    s = softcap * np.tanh(s / softcap)
                m = s.max()
                p = np.exp(s - m)
                l = p.sum()
                lse[b, h, i] = m + np.log(l)
                o[b, h, i] = (p / l) @ v
                w[b, h, i] = (p / l) @ np.abs(v)
    return o, lse, w
