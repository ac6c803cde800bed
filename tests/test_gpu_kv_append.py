"""append_kv_cache on the GPU against the float64 restatement (oracle/kv_cache.py).

Scales are equal; codes that only move to another scale are equal. New tokens in e4m3: half a step of the stored value
(2^-4 relative, or 2^-10 of the scale below 2^-6 of it) plus the rotation's fp32 arithmetic (8 2^-24 (|x1| + |x2|),
as for apply_rotary); in bf16 2^-8 relative plus the same. Values are bf16 to begin with: V's codes are equal, and
V in bf16 bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import fp8, kv_cache  # noqa: E402
from tests.test_gpu_rotary import _np, _partner  # noqa: E402


def _nan(c):
    """Codes with both NaN codes (S.1111.111) as one: a NaN's sign says nothing."""
    return np.where((c & 0x7f) == 0x7f, 0x7f, c).astype(np.uint8)


def _bytes(t):
    import torch
    return _nan(t.view(torch.uint8).cpu().numpy())


class Pages:
    """A cache of random content with a page table in random order (one spare page, in nobody's table)."""

    def __init__(self, B, H, page, D, per_row, fp8, seed):
        import torch
        import pallas_flexattn as pf
        g = np.random.default_rng(seed)
        n = B * per_row + 1
        self.table = g.permutation(n)[:B * per_row].reshape(B, per_row)
        self.t_table = torch.from_numpy(self.table.astype(np.int32)).cuda()
        if fp8:
            codes = [_nan(g.integers(0, 256, (n, H, page, D), dtype=np.uint8)) for _ in range(2)]
            scales = [np.exp2(g.integers(-9, -5, (n, H, page // 32))).astype(np.float32) for _ in range(2)]
            self.host = codes + scales
            self.cache = pf.Fp8KVCache(*[torch.from_numpy(c).cuda().view(torch.float8_e4m3fn) for c in codes],
                                       *[torch.from_numpy(s).cuda() for s in scales])
        else:
            self.cache = tuple(torch.randn(n, H, page, D, device="cuda").bfloat16() for _ in range(2))
            self.host = [_np(c) for c in self.cache]


def _tokens(B, Hq, H, T, D, seed, spread=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda h: (torch.randn(B, T, h, D, device="cuda", generator=g) * spread).bfloat16().transpose(1, 2)  # noqa: E731
    return mk(Hq), mk(H), mk(H)


CASES = [
    # B, Hq, H, T, D, page, lens, new, rotary_dim, interleaved
    (1, 4, 1, 1, 128, 64, [0], None, 128, False), (3, 8, 2, 1, 128, 128, [0, 31, 32], None, 128, False),
    (3, 4, 4, 1, 64, 32, [1, 63, 64], None, 64, True), (2, 4, 2, 33, 128, 64, [5, 31], None, 64, False),
    (2, 6, 3, 100, 64, 96, [0, 77], [100, 41], 32, True), (4, 4, 2, 7, 32, 32, [0, 29, 3, 64], [7, 0, 3, 9], 32, False),
    (2, 4, 2, 64, 32, 64, [32, 1], None, 16, True), (1, 7, 1, 600, 128, 256, [300], None, 128, False),
    (40, 4, 4, 3, 64, 64, list(range(40)), None, 64, False), (2, 0, 2, 40, 128, 64, [9, 64], [40, 1], 0, False),
]


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_append(case, kind):
    import torch
    import pallas_flexattn as pf
    B, Hq, H, T, D, page, lens, new, rd, inter = case
    is8 = kind == "fp8"
    per_row = (max(lens) + T + page - 1) // page
    P = Pages(B, H, page, D, per_row, is8, 11)
    q, k, v = _tokens(B, max(Hq, 1), H, T, D, 12)
    rot = pf.rotary_embedding(rd, interleaved=inter, scaling="linear", factor=2.0) if rd else None
    q0, ins = q.clone(), [t.clone() for t in (k, v)]
    tl = torch.tensor(lens, device="cuda", dtype=torch.int32)
    tn = None if new is None else torch.tensor(new, device="cuda", dtype=torch.int32)
    out = pf.append_kv_cache(P.cache, k, v, tl, P.t_table, new_lens=tn, rotary=rot, query=q if rd else None)
    assert torch.equal(q, q0) and torch.equal(k, ins[0]) and torch.equal(v, ins[1]) and tl.tolist() == lens
    pos = np.array(lens)[:, None] + np.arange(T)
    f = rot.inv_freq.cpu().numpy() if rd else np.zeros(0)
    kr = kv_cache.rotate(_np(k), pos, f, inter) if rd else _np(k)
    slack = 8 * 2.0 ** -24 * _partner(_np(k), len(f), inter)
    if rd:
        assert out.is_contiguous() and torch.equal(out, pf.apply_rotary(q, None, rot, positions=torch.from_numpy(pos).cuda()))
    else:
        assert out is None
    # values: exactly
    wv, wvs = kv_cache.append(P.host[1], P.host[3] if is8 else None, _np(v), lens, P.table, new)
    if is8:
        same = _bytes(P.cache.value) == wv
        assert same.all(), f"{(~same).sum()} value codes differ"
        assert np.array_equal(P.cache.value_scale.cpu().numpy(), wvs)
    else:
        assert np.array_equal(_np(P.cache[1]), wv)
    # keys
    wk, wks = kv_cache.append(P.host[0], P.host[2] if is8 else None, kr, lens, P.table, new)
    exact = kv_cache.append(np.zeros(wk.shape), None, kr, lens, P.table, new)[0]
    slk = kv_cache.append(np.zeros(wk.shape), None, slack, lens, P.table, new)[0]
    fresh = kv_cache.append(np.zeros(wk.shape), None, np.ones_like(kr), lens, P.table, new)[0] > 0
    if is8:
        got = _bytes(P.cache.key)
        assert np.array_equal(P.cache.key_scale.cpu().numpy(), wks)
        assert np.array_equal(got[~fresh], wk[~fresh]), "rows that are not new"
        s = np.repeat(wks, 32, axis=2)[..., None]
        val = fp8.decode_e4m3(got).astype(np.float64) * s
        tol = np.maximum(np.abs(exact) * 2.0 ** -4, s * 2.0 ** -10) + slk * 1.07
    else:
        val = _np(P.cache[0])
        assert np.array_equal(val[~fresh], wk[~fresh])
        tol = np.abs(exact) * 2.0 ** -8 + slk * 1.01
    err = np.abs(val - exact)[fresh]
    assert np.all(err <= tol[fresh] + 1e-30)


def test_token_by_token_equals_the_definition():
    """A row that grows over three runs, its tokens growing too: every call moves the run's older codes."""
    import torch
    import pallas_flexattn as pf
    H, D, page, n = 2, 64, 32, 70
    P = Pages(1, H, page, D, 3, True, 3)
    _, k, v = _tokens(1, 1, H, n, D, 4)
    grow = torch.exp2((torch.arange(n, device="cuda") % 32) * 0.5)[:, None].bfloat16()
    k, v = (k * grow).contiguous(), (v * grow).contiguous()
    host = [x.copy() for x in P.host]
    for t in range(n):
        lens = torch.tensor([t], device="cuda", dtype=torch.int32)
        pf.append_kv_cache(P.cache, k[:, :, t:t + 1], v[:, :, t:t + 1], lens, P.t_table)
        for i, x in ((0, k), (1, v)):
            host[i], host[2 + i] = kv_cache.append(host[i], host[2 + i], _np(x[:, :, t:t + 1]), [t], P.table)
    for i, got in enumerate(P.cache):
        assert np.array_equal(_bytes(got) if i < 2 else got.cpu().numpy(), host[i])


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_dropped_tokens(kind):
    """Page ids outside the cache, positions past the table, negative lengths, no new tokens: nothing else changes."""
    import torch
    import pallas_flexattn as pf
    B, H, page, D, T = 5, 2, 32, 64, 40
    P = Pages(B, H, page, D, 2, kind == "fp8", 5)
    table = P.table.copy()
    table[0, 1], table[1, 0] = -1, 10 ** 6
    lens, new = [10, 0, 50, -7, 3], [40, 40, 40, 40, 0]
    _, k, v = _tokens(B, 1, H, T, D, 6)
    pf.append_kv_cache(P.cache, k, v, torch.tensor(lens, device="cuda"), torch.from_numpy(table).cuda(),
                       new_lens=torch.tensor(new, device="cuda"))
    for i, x in ((0, k), (1, v)):
        if kind == "fp8":
            c, s = kv_cache.append(P.host[i], P.host[2 + i], _np(x), lens, table, new)
            assert np.array_equal(_bytes(P.cache[i]), c) and np.array_equal(P.cache[2 + i].cpu().numpy(), s)
        else:
            assert np.array_equal(_np(P.cache[i]), kv_cache.append(P.host[i], None, _np(x), lens, table, new)[0])


def test_without_a_page_table_and_with_lists():
    import torch
    import pallas_flexattn as pf
    P = Pages(3, 2, 96, 32, 1, True, 7)
    own = np.arange(3)[:, None]
    _, k, v = _tokens(3, 1, 2, 50, 32, 8)
    pf.append_kv_cache(P.cache, k, v, [0, 20, 46])
    for i, x in ((0, k), (1, v)):
        c, s = kv_cache.append(P.host[i], P.host[2 + i], _np(x), [0, 20, 46], own)
        assert np.array_equal(_bytes(P.cache[i]), c) and np.array_equal(P.cache[2 + i].cpu().numpy(), s)


def test_values_at_the_edges():
    """Zero runs, the smallest and largest numbers, a run's maximum on a scale's border, NaN and infinities."""
    import torch
    import pallas_flexattn as pf
    H, D, T = 1, 32, 32
    x = torch.zeros(6, H, T, D)
    x[1, 0, 3, 5] = 448.0 * 2.0 ** -3
    x[2, 0, 3, 5] = 450.0  # just past a border
    x[2, 0, 4, :] = 2.0 ** -40
    x[3, 0, 0, 0], x[3, 0, 0, 1], x[3, 0, 0, 2], x[3, 0, 0, 3] = float("nan"), float("inf"), -float("inf"), 3.0
    x[4] = torch.full((H, T, D), 3.3e38)
    x[5, 0, 0, 0] = 2.0 ** -133
    x = x.bfloat16()
    P = Pages(6, H, 32, D, 1, True, 9)
    pf.append_kv_cache(P.cache, x.cuda(), x.cuda(), [0] * 6, P.t_table)
    c, s = kv_cache.append(P.host[0], P.host[2], x.double().numpy(), [0] * 6, P.table)
    for i in range(2):
        got = _bytes(P.cache[i])[P.table[:, 0]]
        want = _nan(c)[P.table[:, 0]]
        nan = (want & 0x7f) == 0x7f
        assert np.array_equal((got & 0x7f) == 0x7f, nan)
        assert np.array_equal(got[~nan], want[~nan])
        assert np.array_equal(P.cache[2 + i].cpu().numpy()[P.table[:, 0]], s[P.table[:, 0]])


def test_strides_and_alignment_change_nothing():
    import torch
    import pallas_flexattn as pf
    B, H, T, D = 2, 2, 37, 64
    rot = pf.rotary_embedding(64)
    base = torch.randn(B, T, 3 * H * D + 8, device="cuda").bfloat16()
    cuts = [(0, H * D), (H * D, 2 * H * D), (1, H * D + 1)]
    views = [base[..., a:b].unflatten(-1, (H, D)).transpose(1, 2) for a, b in cuts] + [base[:, :, :D][:, None].expand(B, H, T, D)]
    for i, a in enumerate(views):
        b = views[(i + 1) % len(views)]
        P, R = (Pages(B, H, 32, D, 3, True, 10) for _ in range(2))
        o1 = pf.append_kv_cache(P.cache, a, b, [3, 40], P.t_table, rotary=rot, query=b)
        o2 = pf.append_kv_cache(R.cache, a.contiguous(), b.contiguous(), [3, 40], R.t_table, rotary=rot, query=b.contiguous())
        assert torch.equal(o1, o2)
        for x, y in zip(P.cache, R.cache):
            assert np.array_equal(_bytes(x), _bytes(y))


def test_empty_batch_and_no_tokens():
    import torch
    import pallas_flexattn as pf
    P = Pages(2, 2, 32, 64, 1, True, 1)
    k = torch.empty(2, 2, 0, 64, device="cuda", dtype=torch.bfloat16)
    assert pf.append_kv_cache(P.cache, k, k, [0, 0], P.t_table) is None
    k = torch.empty(0, 2, 3, 64, device="cuda", dtype=torch.bfloat16)
    pf.append_kv_cache(P.cache, k, k, torch.empty(0, device="cuda", dtype=torch.int32), P.t_table[:0])
    for i in range(4):
        assert np.array_equal(_bytes(P.cache[i]) if i < 2 else P.cache[i].cpu().numpy(), P.host[i])
