"""The float64 restatement of rotary positions, cache appends and decode (oracle/kv_cache.py), and
rotary_embedding's frequencies, against closed forms and independent formulas (CPU)."""
import math

import numpy as np
import pytest

import pallas_flexattn as pf
from oracle import attention, fp8, kv_cache


@pytest.mark.parametrize("inter", [False, True])
def test_rotation_closed_forms(inter):
    g = np.random.default_rng(0)
    x = g.standard_normal((2, 3, 5, 12))
    f = np.array([0.5, 0.25, 0.125])
    pos = g.integers(0, 1000, (2, 5))
    assert np.array_equal(kv_cache.rotate(x, np.zeros((2, 5)), f, inter), x)
    y = kv_cache.rotate(x, pos, f, inter)
    assert np.array_equal(y[..., 6:], x[..., 6:])
    np.testing.assert_allclose(np.linalg.norm(y, axis=-1), np.linalg.norm(x, axis=-1), rtol=1e-13)
    np.testing.assert_allclose(kv_cache.rotate(y, pos, f, inter, inverse=True), x, atol=1e-13)
    np.testing.assert_allclose(kv_cache.rotate(y, pos, f, inter), kv_cache.rotate(x, 2 * pos, f, inter), atol=1e-11)
    e = np.zeros((1, 1, 1, 4))
    e[..., 0] = 1.0
    y = kv_cache.rotate(e, np.array([[1]]), np.array([math.pi / 2, 0.0]), inter, scale=3.0)
    want = [0, 3, 0, 0] if inter else [0, 0, 3, 0]
    np.testing.assert_allclose(y[0, 0, 0], want, atol=1e-15)


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.5, 1), (449.0, 1), (224.0, -1), (1.0, -8), (0.0, -126), (1e-45, -126),
                                    (3.4e38, 120)])
def test_run_scale(amax, e):
    s = kv_cache.run_scale(amax)
    assert s == 2.0 ** e and 448.0 * s >= amax and (e == -126 or 224.0 * s < amax)


def test_append_keeps_everything_else_and_its_invariants():
    g = np.random.default_rng(1)
    P, H, page, D, B, T = 9, 2, 64, 32, 2, 40
    table = np.array([[3, 1, 7], [0, 8, 2]])
    codes = g.integers(0, 256, (P, H, page, D), dtype=np.uint8)
    scales = np.ones((P, H, page // 32), np.float32)
    x = g.standard_normal((B, H, T, D)) * 3
    lens, new = [50, 0], [40, 7]
    c2, s2 = kv_cache.append(codes, scales, x, lens, table, new)
    touched = np.zeros((P, H, page), bool)
    for b in range(B):
        for t in range(new[b]):
            pos = lens[b] + t
            pid, row = table[b, pos // page], pos % page
            touched[pid, :, row] = True
            val = fp8.decode_e4m3(c2[pid, :, row]) * s2[pid, :, row // 32][:, None]
            assert np.all(np.abs(val - x[b, :, t]) <= np.abs(x[b, :, t]) / 16 + s2[pid, :, row // 32][:, None] * 2.0 ** -10)
    begun = np.zeros_like(touched)
    begun[table[0, 0], :, 32:50] = True  # (may move to a larger scale)
    assert np.array_equal(c2[~touched & ~begun], codes[~touched & ~begun])
    u, _ = kv_cache.append(np.zeros((P, H, page, D)), None, x, lens, table, new)
    assert np.array_equal(u[3, :, 50], x[0, :, 0]) and np.array_equal(u[1, :, 25], x[0, :, 39])


def test_append_moves_a_begun_run_to_a_larger_scale():
    codes = np.zeros((1, 1, 32, 32), np.uint8)
    scales = np.ones((1, 1, 1), np.float32)
    table = np.zeros((1, 1), int)
    a = np.full((1, 1, 1, 32), 448.0)
    codes, scales = kv_cache.append(codes, scales, a, [0], table)
    codes, scales = kv_cache.append(codes, scales, 4 * a, [1], table)
    assert scales[0, 0, 0] == 4.0
    assert fp8.decode_e4m3(codes[0, 0, 0, 0]) == 112.0 and fp8.decode_e4m3(codes[0, 0, 1, 0]) == 448.0
    codes, scales = kv_cache.append(codes, scales, a / 1000, [2], table)  # a smaller token keeps the scale
    assert scales[0, 0, 0] == 4.0


def test_decode_is_attention_of_the_newest_queries():
    g = np.random.default_rng(2)
    B, Hq, Hkv, S, D, Sq = 1, 4, 2, 37, 32, 5
    q, k, v = (g.standard_normal(s) for s in ((B, Hq, S, D), (B, Hkv, S, D), (B, Hkv, S, D)))
    mask = lambda b, h, i, j: (j <= i) & (i - j <= 9)  # noqa: E731
    slopes = pf.alibi_slopes(Hq)
    ro, rlse = attention.forward(q, k, v, mask=mask, alibi_slopes=slopes, softcap=20.0)
    o, lse, w = kv_cache.decode(q[:, :, -Sq:], k, v, [S], left=9, right=0, slopes=slopes, softcap=20.0)
    np.testing.assert_allclose(o, ro[:, :, -Sq:], atol=2e-6)
    np.testing.assert_allclose(lse, rlse[:, :, -Sq:], atol=2e-6)
    assert np.all(w >= np.abs(o) - 1e-12)
    o, lse, _ = kv_cache.decode(q[:, :, :3], k, v, [S], q_lens=[1])
    assert np.all(o[:, :, 1:] == 0) and np.all(np.isneginf(lse[:, :, 1:])) and np.isfinite(lse[:, :, 0]).all()


def test_rotary_embedding_frequencies():
    r = pf.rotary_embedding(64, base=500.0, device="cpu")
    np.testing.assert_allclose(r.inv_freq.numpy(), 500.0 ** (-np.arange(32) / 32.0), rtol=1e-14)
    assert r.rotary_dim == 64 and r.scale == 1.0 and not r.interleaved
    lin = pf.rotary_embedding(64, base=500.0, scaling="linear", factor=4.0, device="cpu")
    np.testing.assert_allclose(lin.inv_freq.numpy(), r.inv_freq.numpy() / 4, rtol=1e-14)
    ntk = pf.rotary_embedding(64, base=500.0, scaling="ntk", factor=4.0, device="cpu").inv_freq.numpy()
    assert ntk[0] == 1.0
    np.testing.assert_allclose(ntk[-1], r.inv_freq.numpy()[-1] / 4, rtol=1e-12)
    yarn = pf.rotary_embedding(64, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    plain = pf.rotary_embedding(64, device="cpu").inv_freq.numpy()
    turns = 4096 * plain / (2 * math.pi)
    f = yarn.inv_freq.numpy()
    assert np.allclose(f[turns > 33], plain[turns > 33]) and np.allclose(f[turns < 0.7], plain[turns < 0.7] / 8)
    assert np.all(f <= plain * (1 + 1e-12)) and np.all(f >= plain / 8 * (1 - 1e-12))
    assert yarn.scale == pytest.approx(0.1 * math.log(8.0) + 1.0)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=8, base=1.0)):
        with pytest.raises(ValueError):
            pf.rotary_embedding(device="cpu", **bad)
