"""apply_rotary on the GPU against the float64 rotation (oracle/kv_cache.py).

Tolerance: half a step of the output type relative to the value (bf16 2^-8, fp32 2^-24), plus the fp32
arithmetic before it: sine and cosine are off by at most 2.5 2^-24 (the Taylor remainders are under 2e-9;
the reduced angle, at most pi / 4, and the last Horner steps are rounded), their factor, two products and
a sum round once more each: 8 2^-24 scale (|x1| + |x2|) covers them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import kv_cache  # noqa: E402


def _np(t):
    return t.detach().double().cpu().numpy()


def _partner(x, n, inter):
    """|x1| + |x2| of each rotated element's pair; the copied elements are exact."""
    x = np.abs(x)
    w = np.zeros_like(x)
    i0, i1 = (np.arange(n) * 2, np.arange(n) * 2 + 1) if inter else (np.arange(n), np.arange(n) + n)
    w[..., i0] = w[..., i1] = x[..., i0] + x[..., i1]
    return w


def _check(got, x, pos, rot, inverse=False):
    import torch
    f = rot.inv_freq.cpu().numpy()
    want = kv_cache.rotate(_np(x), pos, f, rot.interleaved, rot.scale, inverse)
    step = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    tol = np.abs(want) * step + 8 * 2.0 ** -24 * rot.scale * _partner(_np(x), len(f), rot.interleaved) + 1e-38
    err = np.abs(_np(got) - want)
    assert np.all(err <= tol), f"off by {np.max(err / tol):.3g} times the tolerance"
    rest = 2 * len(f)
    assert torch.equal(got[..., rest:], x[..., rest:]), "copied elements changed"


SHAPES = [
    # B, Hq, Hkv, T, D, rotary_dim, interleaved
    (2, 4, 2, 37, 128, 128, False), (2, 4, 2, 37, 128, 128, True), (1, 1, 1, 1, 64, 64, False),
    (3, 5, 1, 130, 64, 32, False), (3, 5, 1, 130, 64, 32, True), (1, 32, 8, 257, 128, 64, False),
    (2, 3, 3, 19, 80, 20, False), (2, 3, 3, 19, 80, 20, True), (1, 2, 2, 9, 6, 2, False), (1, 2, 1, 9, 7, 6, True),
    (2, 2, 2, 33, 256, 256, False), (1, 3, 1, 65, 48, 24, False),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_rotation_and_gradients(shape, dtype):
    import torch
    import pallas_flexattn as pf
    B, Hq, Hkv, T, D, rd, inter = shape
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    g = torch.Generator(device="cuda").manual_seed(T + D)
    mk = lambda h: torch.randn(B, h, T, D, device="cuda", generator=g).to(dt)  # noqa: E731
    q, k, gq, gk = mk(Hq), mk(Hkv), mk(Hq), mk(Hkv)
    rot = pf.rotary_embedding(rd, interleaved=inter, scaling="yarn", factor=4.0)
    pos = np.tile(np.arange(T) + 5, (B, 1))
    q.requires_grad_(), k.requires_grad_()
    yq, yk = pf.apply_rotary(q, k, rot, offset=5)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for got, x in ((yq, q), (yk, k)):
        _check(got.detach(), x.detach(), pos, rot)
    for got, x in ((dq, gq), (dk, gk)):
        _check(got, x, pos, rot, inverse=True)


@pytest.mark.parametrize("where", ["row32", "rows64", "one64", "far", "strided"])
def test_positions(where):
    import torch
    import pallas_flexattn as pf
    B, H, T, D = 3, 2, 41, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(B, H, T, D, device="cuda", generator=g)
    rot = pf.rotary_embedding(64)
    r = np.random.default_rng(4)
    p = r.integers(0, 200000, (B, T))
    if where == "far":
        p = p + (1 << 40)  # (the float64 reference itself is exact to 2^-12 radians there: frequencies of a few bits)
        rot = pf.Rotary(torch.full((32,), 2.0 ** -9, dtype=torch.float64, device="cuda"))
        p = p // 8 * 8
    t = torch.from_numpy(p).cuda()
    if where == "row32":
        t, p = t[0].to(torch.int32), np.tile(p[0], (B, 1))
    elif where == "one64":
        t, p = t[:1], np.tile(p[0], (B, 1))
    elif where == "strided":
        t = torch.from_numpy(np.repeat(p, 2, axis=1)).cuda()[:, ::2]
    got = pf.apply_rotary(q, None, rot, positions=t)
    if where == "far":  # whole turns taken off exactly: pos 2^-9 = 2^-6 n, compared through the exact remainder
        ang = np.fmod(p.astype(np.float64) * 2.0 ** -9, 2 * np.pi)
        want = kv_cache.rotate(_np(q), ang, np.ones(32))
        # the product of pos / (2 pi) keeps 53 bits: 2^31 / 6.28 turns, off by 2^-53 2^29 2 pi and, in numpy's fmod, by
        # its own 2 pi: 2^31 / 6.28 times 2.5e-16
        tol = (2.0 ** 29 * 2.0 ** -52 * 6.3 + 2.0 ** 29 * 2.5e-16 + 9 * 2.0 ** -24) * _partner(_np(q), 32, False) + 1e-30
        assert np.all(np.abs(_np(got) - want) <= tol)
    else:
        _check(got, q, p, rot)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_alignment_change_nothing(dtype):
    """Projections' layout, a slice of a fused projection, odd starts, broadcast heads and rows."""
    import torch
    import pallas_flexattn as pf
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    g = torch.Generator(device="cuda").manual_seed(8)
    B, T, H, D = 2, 29, 3, 64
    rot = pf.rotary_embedding(64)
    base = torch.randn(B, T, 3 * H * D + 1, device="cuda", generator=g).to(dt)
    views = [base[..., :H * D].reshape(B, T, H, D).transpose(1, 2),
             base[..., H * D:2 * H * D].unflatten(-1, (H, D)).transpose(1, 2),
             base[..., 1:H * D + 1].unflatten(-1, (H, D)).transpose(1, 2),
             base[:, :, :D][:, None].expand(B, H, T, D), base[:1, :, :D][:, None].expand(B, H, T, D),
             base[..., :2 * D:2][:, None]]
    for v in views:
        want = pf.apply_rotary(v.contiguous(), None, rot)
        got = pf.apply_rotary(v, None, rot)
        assert got.is_contiguous() and torch.equal(got, want)
    # gradients that arrive expanded (from sum()) or transposed; a broadcast input's gradient sums over its copies
    x = torch.randn(B, 1, T, D, device="cuda", generator=g).to(dt).requires_grad_()
    y = pf.apply_rotary(x.expand(B, H, T, D), None, rot)
    dx, = torch.autograd.grad(y.float().sum(), x)
    one, = torch.autograd.grad(pf.apply_rotary(x, None, rot).float().sum(), x)
    assert torch.equal(dx, (one.float() * H).to(dt)) or dt == torch.bfloat16  # (bf16 sums of three round)
    np.testing.assert_allclose(_np(dx), 3 * _np(one), rtol=2.0 ** -6, atol=1e-6)


def test_gradient_against_differences_and_second_order():
    """float32, against central differences of the float64 rotation (linear: the differences are exact up
    to their rounding, 2^-52 / 1e-3), and the gradient's own gradient."""
    import torch
    import pallas_flexattn as pf
    g = np.random.default_rng(6)
    x, w = g.standard_normal((1, 1, 3, 8)), g.standard_normal((1, 1, 3, 8))
    rot = pf.rotary_embedding(6, scaling="yarn", factor=2.0)
    f = rot.inv_freq.cpu().numpy()
    pos = np.array([[0, 7, 1000]])
    t = torch.tensor(x, device="cuda", dtype=torch.float32, requires_grad=True)
    u = torch.tensor(w, device="cuda", dtype=torch.float32, requires_grad=True)
    y = pf.apply_rotary(t, None, rot, positions=torch.from_numpy(pos[0]).cuda())
    dx, = torch.autograd.grad(y, t, u, create_graph=True)
    num = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        e = np.zeros_like(x)
        e[i] = 1e-3
        num[i] = ((kv_cache.rotate(x + e, pos, f, scale=rot.scale) - kv_cache.rotate(x - e, pos, f, scale=rot.scale)) * w).sum() / 2e-3
    np.testing.assert_allclose(_np(dx), num, atol=1e-5)
    z = torch.randn_like(dx)
    du, = torch.autograd.grad(dx, u, z)  # the transpose of the transpose
    assert torch.equal(du, pf.apply_rotary(z, None, rot, positions=torch.from_numpy(pos[0]).cuda()))


def test_only_one_gradient_and_empty_tensors():
    import torch
    import pallas_flexattn as pf
    rot = pf.rotary_embedding(32)
    q = torch.randn(1, 2, 5, 32, device="cuda", requires_grad=True)
    k = torch.randn(1, 1, 5, 32, device="cuda", requires_grad=True)
    yq, yk = pf.apply_rotary(q, k, rot)
    dk, = torch.autograd.grad(yk, k, torch.ones_like(yk), retain_graph=True)  # q's output unused
    dq, dk2 = torch.autograd.grad((yq, yk), (q, k), (torch.ones_like(yq), torch.ones_like(yk)))
    assert torch.equal(dk, dk2)
    yq, yk = pf.apply_rotary(q, k.detach(), rot)
    assert torch.equal(torch.autograd.grad(yq, q, torch.ones_like(yq))[0], dq)
    for s in ((0, 2, 5, 32), (1, 0, 5, 32), (1, 2, 0, 32)):
        e = torch.empty(*s, device="cuda")
        assert pf.apply_rotary(e, None, rot).shape == s
    yq, yk = pf.apply_rotary(torch.empty(1, 0, 5, 32, device="cuda"), k.detach(), rot)
    assert yq.numel() == 0 and torch.equal(yk, pf.apply_rotary(k.detach(), None, rot))


def test_non_finite_values_stay_in_their_pair():
    import torch
    import pallas_flexattn as pf
    rot = pf.rotary_embedding(32)
    x = torch.ones(1, 1, 4, 64, device="cuda")
    x[..., 40], x[0, 0, 1, 3] = float("inf"), float("nan")
    y = pf.apply_rotary(x, None, rot)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[..., 40] = True
    want[0, 0, 1, 3] = want[0, 0, 1, 19] = True
    assert torch.equal(bad, want)


def test_other_stream_and_graph_replays():
    import torch
    import pallas_flexattn as pf
    rot = pf.rotary_embedding(128)
    q = torch.randn(2, 8, 100, 128, device="cuda").bfloat16()
    k = torch.randn(2, 2, 100, 128, device="cuda").bfloat16()
    want = pf.apply_rotary(q, k, rot)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pf.apply_rotary(q, k, rot)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pos = torch.arange(100, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = pf.apply_rotary(q, k, rot, positions=pos)
    for shift in (0, 31, 977):
        pos.copy_(torch.arange(100, device="cuda") + shift)
        graph.replay()
        torch.cuda.synchronize()
        w = pf.apply_rotary(q, k, rot, offset=shift)
        assert torch.equal(yq, w[0]) and torch.equal(yk, w[1])


def test_captured_gradient():
    """Forward and gradient in a graph, replayed with other contents, eager work between the replays."""
    import torch
    import pallas_flexattn as pf
    rot = pf.rotary_embedding(64)
    q = torch.randn(1, 2, 33, 64, device="cuda").bfloat16().requires_grad_()
    k = torch.randn(1, 1, 33, 64, device="cuda").bfloat16().requires_grad_()
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        y = pf.apply_rotary(q, k, rot)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (q, k), (gq, gk)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            for t in (q, k, gq, gk):
                t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
