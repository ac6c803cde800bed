"""append_latent_cache and flex_decode_latent on the GPU against float64 (oracle/kv_cache.py: a latent vector and its rotary
part are one key, the vector alone its value).

Tolerance of the attention: as in tests/test_gpu_prefill.py (weights rounded to bf16 once), with sums of
L + R products in the scores. Appends: latent vectors bit for bit; rotated parts half a bf16 step plus the
rotation's fp32 arithmetic (8 2^-24 (|x1| + |x2|), as for apply_rotary)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import kv_cache  # noqa: E402
from tests.test_gpu_rotary import _np, _partner  # noqa: E402


class Latent:
    """Random rows of the given lengths in pages of random order; all that no row uses is NaN."""

    def __init__(self, lens, L, R, page, seed, per_row=None, spread=1.0):
        import torch
        import pallas_flexattn as pf
        B = len(lens)
        per_row = per_row or max(1, -(-max(lens) // page))
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = B * per_row + 2
        self.table = torch.randperm(n, generator=g, device="cuda")[:B * per_row].reshape(B, per_row).to(torch.int32)
        self.lens = torch.tensor(lens, device="cuda", dtype=torch.int32)
        used = (torch.arange(per_row * page, device="cuda") < self.lens[:, None])[..., None]
        x = (torch.randn(B, per_row * page, L + R, device="cuda", generator=g) * spread).bfloat16()
        self.rows = torch.where(used, x.float(), 0.0)
        data = torch.full((n, page, L + R), float("nan"), device="cuda", dtype=torch.bfloat16)
        data[self.table.long().reshape(-1)] = torch.where(used, x, float("nan")).reshape(B * per_row, page, L + R)
        self.cache = pf.LatentKVCache(data, L)


def _q(B, H, T, L, R, seed, spread=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.randn(H, B, T, L, device="cuda", generator=g) * spread).bfloat16().transpose(0, 1),
            (torch.randn(B, T, H, R, device="cuda", generator=g) * spread).bfloat16().transpose(1, 2))


def _check(o, lse, q, qr, c, lens, scale, ql=None, left=-1, right=-1):
    L = q.shape[3]
    qq, keys = np.concatenate([_np(q), _np(qr)], -1), _np(c.rows)[:, None]
    values = keys.copy()
    values[..., L:] = 0
    wo, wl, w = kv_cache.decode(qq, keys, values, lens, ql, left, right, scale)
    wo, w = wo[..., :L], w[..., :L]
    D = qq.shape[3]
    smax = np.abs(qq).sum(-1).max() * np.abs(keys[np.isfinite(keys)]).max() * scale  # an upper bound of sum |q||k| scale
    ds = (D + 2) * 2.0 ** -24 * smax + 4 * 2.0 ** -24 * smax
    n = keys.shape[2]
    c1 = (2 * ds + 2.0 ** -8 + 2.0 ** -20 + 2 * n * 2.0 ** -24) * (1 + 2.0 ** -8)
    go, gl = _np(o), _np(lse)
    for got, want in ((go, wo), (gl, wl)):
        assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isneginf(gl), np.isneginf(wl)) and np.all(go[np.isneginf(wl)] == 0)
    fin = np.isfinite(wo)
    err, tol = np.abs(go - wo)[fin], (np.abs(wo) * 2.0 ** -8 + c1 * w + 1e-30)[fin]
    assert np.all(err <= tol), f"O off by {np.max(err / tol):.3g} times the tolerance"
    fin = np.isfinite(wl)
    el = np.abs(np.where(fin, gl, 0) - np.where(fin, wl, 0))
    assert np.all(el <= ds + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(fin, wl, 0))), f"LSE off by {el.max():.3g}"


CASES = [
    # keys (the queries' included), H, T, L, R, page, mask
    ([1], 1, 1, 512, 64, 32, None), ([0, 5, 33, 64], 16, 1, 512, 64, 64, None), ([700, 3, 129], 8, 3, 512, 64, 96, (-1, 0)),
    ([1000, 31], 32, 1, 512, 64, 128, None), ([400, 90], 17, 1, 256, 32, 32, (-1, 0)), ([300], 5, 7, 256, 64, 64, (-1, 0)),
    ([513, 64], 128, 1, 512, 64, 64, None), ([260, 7], 64, 3, 512, 32, 32, (-1, 0)), ([2000, 40, 900], 16, 4, 128, 64, 256, (100, 0)),
    ([333, 0, 90], 20, 5, 128, 32, 64, (50, 0)), ([64, 65, 63], 33, 2, 256, 64, 32, (-1, 2)), ([50] * 70, 3, 2, 128, 32, 32, (-1, 0)),
    ([90, 6000], 16, 1, 512, 64, 32, (1000, -1)), ([500, 20], 4, 100, 256, 32, 64, (-1, 0)), ([17, 450] * 140, 2, 1, 128, 64, 32, None),
    ([3000, 10], 40, 1, 512, 64, 512, None), ([5000, 4200, 100], 100, 2, 512, 64, 64, (-1, 0)), ([128] * 300, 16, 1, 128, 32, 128, None),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_decode(case):
    import pallas_flexattn as pf
    lens, H, T, L, R, page, win = case
    c = Latent(lens, L, R, page, 21)
    q, qr = _q(len(lens), H, T, L, R, 22)
    left, right = win or (-1, -1)
    mask = None if win is None else pf.MaskSpec(left=left, right=right)
    o, lse = pf.flex_decode_latent(q, qr, c.cache, 0.05, c.lens, c.table, mask_mod=mask, return_lse=True)
    assert o.is_contiguous()
    _check(o, lse, q, qr, c, lens, 0.05, None, left, right)
    assert (pf.flex_decode_latent(q, qr, c.cache, 0.05, c.lens, c.table, mask_mod=mask) == o).all()


@pytest.mark.parametrize("case", [([700, 90, 64], 32, 3, 512, 64, 64, (-1, 0)), ([400, 33], 24, 2, 256, 32, 32, (-1, 0)),
                                  ([1500, 7, 0], 45, 2, 128, 64, 96, (300, 0)), ([5000], 72, 1, 512, 32, 128, None),
                                  ([96, 95, 1], 37, 1, 256, 64, 32, (31, 3))], ids=range(5))
def test_blocks_of_48_rows(case):
    test_decode(case)


@pytest.mark.parametrize("H", [4, 10, 40])  # one, two and four 16-row blocks
def test_query_lens_and_what_is_not_there(H):
    """Padded rows to none, lengths past the table and below zero, page ids outside the cache (zero keys), kv_len, no table, 64-bit numbers."""
    import torch
    import pallas_flexattn as pf
    L, R = 128, 64
    c = Latent([192, 192, 192], L, R, 64, 7)
    q, qr = _q(3, H, 3, L, R, 8)
    nan = q.clone()
    nan[1, :, 1:], nan[2] = float("nan"), float("nan")

    def run(q, lens, table, **kw):
        return pf.flex_decode_latent(q, qr, c.cache, 0.1, lens, table, mask_mod=pf.causal_mask, return_lse=True, **kw)

    o, lse = run(nan, c.lens, c.table, query_lens=[3, 1, -2])
    _check(o, lse, q, qr, c, [192] * 3, 0.1, [3, 1, 0], -1, 0)
    o, lse = run(q, [10 ** 6, -3, 2 ** 40], c.table.long(), query_lens=torch.tensor([2 ** 35, 3, 3], device="cuda"))
    _check(o, lse, q, qr, c, [192, 0, 192], 0.1, None, -1, 0)
    o, lse = run(q, None, c.table, kv_len=100)
    _check(o, lse, q, qr, c, [100] * 3, 0.1, None, -1, 0)
    bad = c.table.clone()
    bad[0, 1], bad[1, 0], bad[2, 2] = -1, 10 ** 6, 2 ** 31 - 1
    c.rows[0, 64:128], c.rows[1, :64], c.rows[2, 128:] = 0, 0, 0
    o, lse = run(q, c.lens, bad)
    _check(o, lse, q, qr, c, [192] * 3, 0.1, None, -1, 0)
    one = Latent([50, 64], L, R, 64, 11)
    cache = pf.LatentKVCache(one.cache.data[one.table[:, 0].long()].clone(), L)
    o, lse = pf.flex_decode_latent(q[:2], qr[:2], cache, 0.1, one.lens, return_lse=True)
    _check(o, lse, q[:2], qr[:2], one, [50, 64], 0.1)


@pytest.mark.parametrize("H", [2, 9, 30])
def test_values_that_are_not_finite(H):
    """NaN and infinities reach the queries that see them, and no others; behind a window nobody sees them."""
    import pallas_flexattn as pf
    L, R, lens = 128, 32, [400, 260]
    c = Latent(lens, L, R, 32, 13)
    q, qr = _q(2, H, 3, L, R, 14)

    def put(b, key, d, x):
        c.cache.data[int(c.table[b, key // 32]), key % 32, d] = x
        c.rows[b, key, d] = x

    put(0, 399, 3, float("nan"))      # the last key: the last query alone
    put(1, 258, 9, float("nan"))      # the last two
    put(0, 398, L + 5, float("nan"))  # a rotary part
    put(0, 20, 0, float("nan"))       # long before: behind the window
    put(1, 10, 2, float("inf"))
    o, lse = pf.flex_decode_latent(q, qr, c.cache, 0.1, c.lens, c.table, mask_mod=pf.MaskSpec(left=60, right=0), return_lse=True)
    _check(o, lse, q, qr, c, lens, 0.1, None, 60, 0)


def test_large_scores_and_strides():
    """Scores that change by hundreds from key to key; queries that are slices, that start off a 16-byte line, that are expanded."""
    import torch
    import pallas_flexattn as pf
    c = Latent([900, 450], 256, 64, 64, 31, spread=3.0)
    q, qr = _q(2, 24, 2, 256, 64, 32, spread=5.0)
    o, lse = pf.flex_decode_latent(q, qr, c.cache, 0.3, c.lens, c.table, return_lse=True)
    _check(o, lse, q, qr, c, [900, 450], 0.3)
    wide = torch.randn(2, 3, 8, 320, device="cuda").bfloat16()
    raw = torch.randn(2 * 8 * 3 * 256 + 1, device="cuda").bfloat16()
    for a in (wide[..., :256].transpose(1, 2), raw[1:].reshape(2, 8, 3, 256), wide[:1, :, :1, :256].transpose(1, 2).expand(2, 8, 3, 256)):
        b = wide[..., 256:].transpose(1, 2)
        o, lse = pf.flex_decode_latent(a, b, c.cache, 0.05, c.lens, c.table, return_lse=True)
        _check(o, lse, a, b, c, [900, 450], 0.05)
    for z in (0, 2):
        o, lse = pf.flex_decode_latent(q[:z, :, :2 - z], qr[:z, :, :2 - z], c.cache, 0.1, c.lens[:z], c.table[:z], return_lse=True)
        assert o.shape == (z, 24, 2 - z, 256) and lse.shape == (z, 24, 2 - z)


APPENDS = [
    # B, H, T, L, R, page, lens, new, rotary_dim, interleaved
    (1, 4, 1, 512, 64, 64, [0], None, 64, False), (3, 0, 2, 256, 32, 32, [1, 63, 64], None, 32, True),
    (2, 6, 33, 128, 64, 96, [5, 31], [33, 2], 32, False), (4, 3, 7, 128, 32, 32, [0, 29, 3, 500], [7, 0, 3, 9], 16, True),
    (2, 0, 70, 512, 32, 64, [9, 64], None, 0, False), (40, 16, 3, 128, 64, 64, list(range(40)), None, 64, False),
]


@pytest.mark.parametrize("case", APPENDS, ids=[str(i) for i in range(len(APPENDS))])
def test_append(case):
    """Tokens past the table, on bad pages and past new_lens are dropped; everything else stays as it was."""
    import torch
    import pallas_flexattn as pf
    B, H, T, L, R, page, lens, new, rd, inter = case
    g = torch.Generator(device="cuda").manual_seed(3)
    per_row = 4
    P = B * per_row + 1
    data = torch.randn(P, page, L + R, device="cuda", generator=g).bfloat16()
    table = torch.randperm(P, device="cuda", generator=g)[:B * per_row].reshape(B, per_row).to(torch.int32)
    if B == 3:
        table[1, 1], table[2, 2] = -1, P + 3
    x = torch.randn(B, T, L + R, device="cuda", generator=g).bfloat16()
    q = torch.randn(B, T, H, R, device="cuda", generator=g).bfloat16().transpose(1, 2) if H else None
    rot = pf.rotary_embedding(rd, interleaved=inter, scaling="yarn", factor=4.0) if rd else None
    cache = pf.LatentKVCache(data.clone(), L)
    version = cache.data._version
    out = pf.append_latent_cache(cache, x[..., :L], x[..., L:], lens, table, new_lens=new, rotary=rot, query_rope=q)
    assert cache.data._version > version
    pos = np.array(lens)[:, None] + np.arange(T)
    f = _np(rot.inv_freq) if rd else np.zeros(0)
    turn = (lambda v: kv_cache.rotate(v, pos, f, inter, rot.scale)) if rd else (lambda v: v)
    wide = lambda v: _partner(v, len(f), inter) if rd else np.abs(v)  # noqa: E731
    want, tol = _np(data).copy(), np.zeros(data.shape)
    k = _np(x[..., L:])[:, None]
    turned, around = turn(k)[:, 0], wide(k)[:, 0]
    for b in range(B):
        for t in range(T if new is None else min(new[b], T)):
            pg = (lens[b] + t) // page
            pid = int(table[b, pg]) if pg < per_row else -1
            if 0 <= pid < P:
                at = pid, (lens[b] + t) % page
                want[at] = np.concatenate([_np(x[b, t, :L]), turned[b, t]])
                if rd:
                    tol[at][L:] = np.abs(turned[b, t]) * 2.0 ** -8 + 8 * 2.0 ** -24 * rot.scale * around[b, t] + 1e-38
    assert np.all(np.abs(_np(cache.data) - want) <= tol)
    if q is None:
        assert out is None
    else:
        w = turn(_np(q))
        assert out.is_contiguous()
        assert np.all(np.abs(_np(out) - w) <= np.abs(w) * 2.0 ** -8 + 8 * 2.0 ** -24 * rot.scale * wide(_np(q)) + 1e-38)


def test_replays_of_a_graph():
    """A captured step (append, then attend) takes lengths, tables and tokens as they are at each replay."""
    import torch
    import pallas_flexattn as pf
    L, R, B, H = 256, 64, 3, 20
    c = Latent([200, 90, 300], L, R, 64, 61, per_row=6)
    rot = pf.rotary_embedding(R)
    lens, tok = torch.tensor([200, 90, 300], device="cuda", dtype=torch.int32), torch.randn(B, 2, L + R, device="cuda").bfloat16()
    q, qr = (t.clone() for t in _q(B, H, 2, L, R, 62))

    def run(cache):
        rr = pf.append_latent_cache(cache, tok[..., :L], tok[..., L:], lens, c.table, rotary=rot, query_rope=qr)
        return pf.flex_decode_latent(q, rr, cache, 0.1, lens + 2, c.table, mask_mod=pf.causal_mask, return_lse=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(pf.LatentKVCache(c.cache.data.clone(), L))
    torch.cuda.current_stream().wait_stream(s)
    cache = pf.LatentKVCache(c.cache.data.clone(), L)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = run(cache)
    for ln in ([200, 90, 300], [0, 90, 1], [200, 60, 299]):
        lens.copy_(torch.tensor(ln)), tok.copy_(torch.randn_like(tok.float())), q.copy_(torch.randn_like(q.float()))
        cache.data.copy_(c.cache.data)
        g.replay()
        twin = pf.LatentKVCache(c.cache.data.clone(), L)
        eo, el = run(twin)
        assert torch.equal(o, eo) and torch.equal(lse, el)
        assert torch.equal(cache.data.view(torch.int16), twin.data.view(torch.int16))


def test_expanded_heads():
    """The absorbed form is the attention of the heads written out: keys W_k c with the rotary part behind, values W_v c."""
    import torch
    import pallas_flexattn as pf
    L, R, H, N, V, n, T = 128, 32, 6, 48, 40, 150, 2
    g = torch.Generator(device="cuda").manual_seed(5)
    c = Latent([n], L, R, 32, 71)
    wk = torch.randn(H, N, L, device="cuda", generator=g, dtype=torch.float64) / L ** 0.5
    wv = torch.randn(H, V, L, device="cuda", generator=g, dtype=torch.float64) / L ** 0.5
    qn = torch.randn(H, T, N, device="cuda", generator=g, dtype=torch.float64)
    qr = torch.randn(1, H, T, R, device="cuda", generator=g).bfloat16()
    scale = (N + R) ** -0.5
    q = torch.matmul(qn, wk).bfloat16()
    o = pf.flex_decode_latent(q[None], qr, c.cache, scale, c.lens, c.table, mask_mod=pf.causal_mask)
    got = torch.matmul(o[0].double(), wv.transpose(1, 2))
    x = c.rows[0, :n].double()
    keys, values = torch.matmul(x[None, :, :L], wk.transpose(1, 2)), torch.matmul(x[None, :, :L], wv.transpose(1, 2))
    s = (torch.matmul(qn, keys.transpose(1, 2)) + torch.matmul(qr[0].double(), x[:, L:].T.contiguous())) * scale
    s = s.masked_fill(torch.arange(n, device="cuda")[None] > (n - T + torch.arange(T, device="cuda"))[:, None], -float("inf"))
    p = torch.softmax(s, -1)
    want = torch.matmul(p, values)
    # q, the weights and o are rounded to bf16 on the way (half a step, 2^-8, each): scores are off by ds at most, weights by
    # 2 ds + 2^-8 relative (to first order; half as much again covers the rest), o by that of its terms and by 2^-8
    ds = (scale * 2.0 ** -8 * torch.matmul(torch.matmul(qn, wk).abs(), x[:, :L].abs().T.contiguous())).amax(-1, keepdim=True)
    mean = torch.matmul(p, x[:, :L].expand(H, n, L).contiguous())
    off = (2 * ds + 2.0 ** -8) * 1.5 * torch.matmul(p, x[:, :L].abs().expand(H, n, L).contiguous()) + 2.0 ** -8 * mean.abs()
    assert ((got - want).abs() <= 1.5 * torch.matmul(off, wv.abs().transpose(1, 2).contiguous())).all()
