"""64-bit page ids and lengths past 32 bits mean what they say: a page outside the cache, a row longer than any."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FAR = [2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 40 + 1, 2 ** 63 - 1, -2 ** 32, -2 ** 63, -2 ** 63 + 1]


@pytest.mark.parametrize("far", FAR)
def test_append(far):
    import torch
    import pallas_flexattn as pf
    mk = lambda: pf.Fp8KVCache(*[torch.zeros(3, 1, 32, 32, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)],  # noqa: E731
                               *[torch.ones(3, 1, 1, device="cuda") for _ in range(2)])
    x = torch.ones(2, 1, 3, 32, device="cuda").bfloat16()
    untouched = [t.view(torch.uint8).clone() for t in mk()]
    same = lambda a, rows=slice(None): all(torch.equal(t.view(torch.uint8)[rows], u[rows]) for t, u in zip(a, untouched))  # noqa: E731
    i64 = lambda *v: torch.tensor(v, device="cuda", dtype=torch.int64)  # noqa: E731
    c = mk()
    pf.append_kv_cache(c, x, x, i64(0, 0), i64(far, 2)[:, None])  # a page id
    assert same(c, slice(0, 2)) and not same(c)
    c = mk()
    pf.append_kv_cache(c, x, x, i64(far, 0), i64(0, 2)[:, None])  # a length before the call: past the table, or negative
    assert same(c, slice(0, 2)) and not same(c)
    c = mk()
    pf.append_kv_cache(c, x, x, i64(0, 0), i64(1, 2)[:, None], new_lens=i64(far, 1))
    n = 3 if far > 0 else 0
    got = c.key.float()
    assert got[1].count_nonzero() == n * 32 and got[2].count_nonzero() == 32 and got[0].count_nonzero() == 0


@pytest.mark.parametrize("far", FAR)
def test_decode(far):
    import torch
    import pallas_flexattn as pf
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    c = pf.Fp8KVCache(*[rnd(3, 1, 32, 32).to(torch.float8_e4m3fn) for _ in range(2)],
                      *[torch.ones(3, 1, 1, device="cuda") for _ in range(2)])
    q = rnd(2, 2, 2, 32).bfloat16()
    i64 = lambda *v: torch.tensor(v, device="cuda", dtype=torch.int64)  # noqa: E731
    run = lambda *a, **k: pf.flex_decode_fp8(q, c, *a, enable_gqa=True, return_lse=True, **k)  # noqa: E731
    eq = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    table = i64(1, 2)[:, None]
    assert eq(run(i64(32, 32), i64(far, 2)[:, None]), run(i64(32, 32), i64(-1, 2)[:, None]))
    assert eq(run(i64(far, 20), table), run(i64(32 if far > 0 else 0, 20), table))
    assert eq(run(i64(32, 20), table, query_lens=i64(far, 1)), run(i64(32, 20), table, query_lens=i64(2 if far > 0 else 0, 1)))


def test_ordinary_64_bit_tables_are_read_as_they_are():
    import torch
    import pallas_flexattn as pf
    c = pf.Fp8KVCache(*[torch.randn(7, 2, 32, 64, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)],
                      *[torch.ones(7, 2, 1, device="cuda") for _ in range(2)])
    q = torch.randn(3, 4, 1, 64, device="cuda").bfloat16()
    table = torch.tensor([[6, 0], [3, 1], [5, -1]], device="cuda", dtype=torch.int64)
    wide = torch.stack((table, table + 1), dim=-1)[..., 0]  # (strided)
    lens = torch.tensor([64, 40, 3], device="cuda", dtype=torch.int64)
    want = pf.flex_decode_fp8(q, c, lens.int(), table.int(), enable_gqa=True)
    for t, n in ((table, lens), (wide, lens), (table.cpu(), lens.cpu()), (table, lens.int())):
        assert torch.equal(pf.flex_decode_fp8(q, c, n, t, enable_gqa=True), want)
    assert np.isfinite(want.float().cpu().numpy()).all()
