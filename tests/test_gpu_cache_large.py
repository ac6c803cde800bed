"""Tensors of more than 2^31 elements through the calls around a KV cache: the last rows as a small call gives them."""
import pytest

pytestmark = pytest.mark.gpu

LATE = 3000  # rows that are compared


@pytest.mark.parametrize("D,n", [(256, 256), (256, 20)])  # 16-byte accesses, single elements
def test_rotary(D, n):
    import torch
    import pallas_flexattn as pf
    T = (1 << 31) // D + 77
    q = torch.empty(1, 1, T, D, device="cuda", dtype=torch.bfloat16)
    q[:, :, -LATE:] = torch.randn(1, 1, LATE, D, device="cuda").bfloat16()
    rot = pf.rotary_embedding(n)
    y = pf.apply_rotary(q, None, rot)
    assert torch.equal(y[:, :, -LATE:], pf.apply_rotary(q[:, :, -LATE:], None, rot, offset=T - LATE))


def test_append():
    """The batch's last row, its keys, values and queries behind 2^31 elements of each."""
    import torch
    import pallas_flexattn as pf
    B, H, D, T = 3, 64, 128, 1 << 17  # 2^30 elements a row
    k = torch.empty(B, H, T, D, device="cuda", dtype=torch.bfloat16)
    last = torch.randn(1, H, LATE, D, device="cuda").bfloat16()
    k[2:, :, -LATE:] = last
    rot = pf.rotary_embedding(D)
    caches, outs = [], []
    # only the last row's last tokens have pages
    runs = -(-LATE // 32)
    for x, start, table in ((k, 0, [[-1] * (T // 32)] * 2 + [[-1] * (T // 32 - runs) + list(range(runs))]),
                            (last, T - LATE, [[-1] * (T // 32 - runs) + list(range(runs))])):
        c = pf.create_fp8_kv_cache(runs, H, 32, D)
        for t in c[:2]:
            t.view(torch.uint8).zero_()
        outs.append(pf.append_kv_cache(c, x, x, [start] * x.shape[0], torch.tensor(table, device="cuda"), rotary=rot, query=x))
        caches.append(c)
    assert torch.equal(outs[0][2:, :, -LATE:], outs[1])
    first = -LATE % 32  # (the first run holds other tokens in the large call)
    for a, b in zip(*caches):
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
        assert torch.equal(a[1 if first else 0:], b[1 if first else 0:])


def test_decode():
    import torch
    import pallas_flexattn as pf
    D, page = 128, 64
    Sq = (1 << 31) // D + 77
    c = pf.Fp8KVCache(*[torch.randn(1, 1, page, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)],
                      *[torch.ones(1, 1, 2, device="cuda") for _ in range(2)])
    q = torch.zeros(1, 1, Sq, D, device="cuda", dtype=torch.bfloat16)
    q[:, :, -48:] = torch.randn(1, 1, 48, D, device="cuda").bfloat16()
    o, lse = pf.flex_decode_fp8(q, c, [page], mask_mod=pf.causal_mask, return_lse=True)
    want, wl = pf.flex_decode_fp8(q[:, :, -48:], c, [page], mask_mod=pf.causal_mask, return_lse=True)
    # (each row's sums run over the same tiles in the same order, in other items)
    assert torch.allclose(o[:, :, -48:].float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -12)
    assert torch.allclose(lse[:, :, -48:], wl, rtol=1e-6, atol=1e-6)
    assert (o[:, :, :Sq - page] == 0).all() and (lse[:, :, :Sq - page] == float("-inf")).all()
