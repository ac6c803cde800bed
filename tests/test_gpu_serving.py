"""Prompts in chunks, forks, single tokens, compaction and further chunks over one set of pages, two layers that share the
tables; after each step attention against float64 over the rows' own tokens, which are kept apart (one row behind another, cloned by
torch at each fork).  Tolerances: those of tests/test_gpu_prefill.py and tests/test_gpu_latent.py.

Behind it: caches and queries of more than 2^32 and 2^31 elements, as small calls give them."""
import types

import pytest

pytestmark = pytest.mark.gpu

from tests import test_gpu_latent as latent, test_gpu_prefill as prefill  # noqa: E402

PAGE, WIDTH, PAGES, LAYERS = 32, 9, 60, 2
H, HQ, D, L, R = 2, 6, 64, 128, 32


class Run:
    def __init__(self, kind, rows):
        import torch
        import pallas_flexattn as pf
        self.kind, self.g = kind, torch.Generator(device="cuda").manual_seed(31)
        self.caches = [self._cache(PAGES) for _ in range(LAYERS)]
        self.own = [self._cache(rows * WIDTH) for _ in range(LAYERS)]  # (row b: pages b WIDTH ..)
        self.table = torch.full((rows, WIDTH), -1, device="cuda", dtype=torch.int32)
        self.lens = torch.zeros(rows, device="cuda", dtype=torch.int32)
        self.pf, self.n = pf, [0] * rows

    def _cache(self, n):
        import torch
        import pallas_flexattn as pf
        if self.kind == "latent":
            return pf.LatentKVCache(torch.full((n, PAGE, L + R), float("nan"), device="cuda", dtype=torch.bfloat16), L)
        if self.kind == "bf16":
            return tuple(torch.full((n, H, PAGE, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        return pf.Fp8KVCache(*[torch.full((n, H, PAGE, D), 0x7f, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
                               for _ in range(2)], *[torch.full((n, H, PAGE // 32), float("nan"), device="cuda") for _ in range(2)])

    def fork(self, parents, room, keep=None):
        import torch
        old, self.n = self.n, [self.n[p] if 0 <= p < len(self.n) else 0 for p in parents]
        self.table, self.lens, free = self.pf.fork_kv_rows(self.caches, self.table, self.lens, parents, room, keep)
        assert int(free) >= 0 and self.lens.tolist() == self.n
        p = torch.tensor([x if 0 <= x < len(old) else 0 for x in parents], device="cuda")
        ids = (p[:, None] * WIDTH + torch.arange(WIDTH, device="cuda")).reshape(-1)
        self.own = [c._replace(data=c.data[ids]) if self.kind == "latent" else type(c)(*[x[ids] for x in c]) if self.kind == "fp8"
                    else tuple(x[ids] for x in c) for c in self.own]

    def compact(self, spare):
        """The pages in use and `spare` free ones are all that is kept of the caches."""
        self.table, used = self.pf.compact_kv_pages(self.caches, self.table, self.lens)
        n = int(used) + spare
        assert n <= PAGES and int(self.table.max()) < int(used)
        self.caches = [c._replace(data=c.data[:n].clone()) if self.kind == "latent" else type(c)(*[x[:n].clone() for x in c])
                       if self.kind == "fp8" else tuple(x[:n].clone() for x in c) for c in self.caches]

    def _plain(self, c, i=0):
        """Rows of the i-th tensor, zero behind a row's tokens."""
        import torch
        B = len(self.n)
        used = torch.arange(WIDTH * PAGE, device="cuda") < self.lens[:, None]
        if self.kind == "latent":
            return torch.where(used[..., None], c.data.reshape(B, WIDTH * PAGE, L + R).float(), 0.0)
        x = c[i].float()
        if self.kind == "fp8":
            x = x * c[2 + i].repeat_interleave(32, 2)[..., None]
        x = x.reshape(B, WIDTH, H, PAGE, D).transpose(1, 2).reshape(B, H, WIDTH * PAGE, D)
        return torch.where(used[:, None, :, None], x, 0.0)

    def step(self, new, window=None):
        """Every row's next tokens (new[b] of them) are appended and attend."""
        import torch
        pf, B, T = self.pf, len(self.n), max(new)
        count = torch.tensor(new, device="cuda", dtype=torch.int32)
        before, self.lens = self.lens, self.lens + count
        self.n = [a + b for a, b in zip(self.n, new)]
        left = -1 if window is None else window
        mask = pf.MaskSpec(left=left, right=0)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=self.g).bfloat16()  # noqa: E731
        home = torch.arange(B * WIDTH, device="cuda", dtype=torch.int32).reshape(B, WIDTH)
        for c, o in zip(self.caches, self.own):
            if self.kind == "latent":
                x, r, q, qr = rnd(B, T, L), rnd(B, T, R), rnd(B, HQ, T, L), rnd(B, HQ, T, R)
                pf.append_latent_cache(c, x, r, before, self.table, count)
                pf.append_latent_cache(o, x, r, before, home, count)
                out, lse = pf.flex_decode_latent(q, qr, c, 0.08, self.lens, self.table, mask, True, count)
                latent._check(out, lse, q, qr, types.SimpleNamespace(rows=self._plain(o)), self.n, 0.08, new, left, 0)
                continue
            k, v, q = rnd(B, H, T, D), rnd(B, H, T, D), rnd(B, HQ, T, D)
            pf.append_kv_cache(c, k, v, before, self.table, count)
            pf.append_kv_cache(o, k, v, before, home, count)
            rows = types.SimpleNamespace(rows=[self._plain(o, 0), self._plain(o, 1)])
            out, lse = pf.flex_prefill(q, c, self.lens, self.table, mask, enable_gqa=True, return_lse=True, query_lens=count)
            prefill._check(out, lse, q, rows, self.n, new, left, 0)
            if self.kind == "fp8":
                out, lse = pf.flex_decode_fp8(q, c, self.lens, self.table, mask, enable_gqa=True, return_lse=True, query_lens=count)
                prefill._check(out, lse, q, rows, self.n, new, left, 0)
            packed = torch.cat([q[b, :, :n] for b, n in enumerate(new)], 1)[None]
            starts = torch.nn.functional.pad(count.cumsum(0), (1, 0)).int()
            po, pl = pf.flex_prefill(packed, c, self.lens, self.table, mask, enable_gqa=True, return_lse=True, query_starts=starts)
            at = [0, *count.cumsum(0).tolist()]
            full, flse = torch.zeros_like(q), torch.full((B, HQ, T), -float("inf"), device="cuda")
            for b, n in enumerate(new):
                full[b, :, :n], flse[b, :, :n] = po[0, :, at[b]:at[b + 1]], pl[0, :, at[b]:at[b + 1]]
            prefill._check(full, flse, q, rows, self.n, new, left, 0)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "latent"])
def test_a_batch_served(kind):
    r = Run(kind, 3)
    r.fork([0, 1, 2], [100, 40, 1])
    r.step([70, 33, 1])
    r.step([30, 0, 0])            # the rest of a longer prompt, while the others wait
    r.step([0, 7, 0], window=9)
    r.fork([0, 0, 1, 2, 2, 0], 40)
    for _ in range(3):
        r.step([1] * 6)
    r.step([5, 1, 0, 32, 2, 3], window=40)
    r.fork([5, 3, -1, 0, 0], 0)   # rows end, one begins
    r.compact(spare=8)
    r.fork(range(5), [1, 1, 40, 20, 1])
    r.step([0, 1, 40, 20, 1])
    r.compact(spare=6)
    r.fork([2, 1, 2, 0], 2)
    for _ in range(2):
        r.step([1] * 4)


def _high(kind):
    """A cache of more than 2^32 elements in each tensor, four pages of which matter -> (cache, their ids, a cache of them)."""
    import torch
    import pallas_flexattn as pf
    torch.manual_seed(7)
    if kind == "latent":
        n = (1 << 32) // (64 * 576) + 100
        c = pf.LatentKVCache(torch.empty(n, 64, 576, device="cuda", dtype=torch.bfloat16), 512)
        small = pf.LatentKVCache(torch.randn(4, 64, 576, device="cuda").bfloat16(), 512)
        pairs = [(c.data, small.data)]
    else:
        n = (1 << 32) // (8 * 64 * 128) + 100
        dt = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
        c = [torch.empty(n, 8, 64, 128, device="cuda", dtype=dt) for _ in range(2)]
        small = [torch.randn(4, 8, 64, 128, device="cuda").to(dt) for _ in range(2)]
        if kind == "fp8":
            c += [torch.empty(n, 8, 2, device="cuda") for _ in range(2)]
            small += [torch.rand(4, 8, 2, device="cuda") + 0.5 for _ in range(2)]
        pairs = list(zip(c, small))
        c, small = (tuple(c), tuple(small)) if kind == "bf16" else (pf.Fp8KVCache(*c), pf.Fp8KVCache(*small))
    ids = torch.tensor([n - 1, n - 77, 3, n - 2], device="cuda")
    for a, b in pairs:
        a[ids] = b
    return c, ids.int(), small, [a for a, _ in pairs]


@pytest.mark.parametrize("kind", ["bf16", "fp8", "latent"])
def test_caches_past_32_bits(kind):
    import torch
    import pallas_flexattn as pf
    c, ids, small, tensors = _high(kind)
    near = torch.arange(4, device="cuda", dtype=torch.int32)[None]

    def attend(cache, table, n):
        g = torch.Generator(device="cuda").manual_seed(8)
        if kind == "latent":
            q, qr = (torch.randn(1, 4, 3, x, device="cuda", generator=g).bfloat16() for x in (512, 64))
            return pf.flex_decode_latent(q, qr, cache, 0.05, [n], table, pf.causal_mask, True)
        q = torch.randn(1, 16, 70, 128, device="cuda", generator=g).bfloat16()
        return pf.flex_prefill(q, cache, [n], table, pf.causal_mask, enable_gqa=True, return_lse=True)

    for a, b in zip(attend(c, ids[None], 240), attend(small, near, 240)):
        assert torch.equal(a, b)
    # an append to the row's last page, then a fork whose copy, and a compaction whose moves, lie on both sides
    for cache, table in ((c, ids[None]), (small, near)):
        g = torch.Generator(device="cuda").manual_seed(9)
        if kind == "latent":
            x, r = (torch.randn(1, 7, m, device="cuda", generator=g).bfloat16() for m in (512, 64))
            pf.append_latent_cache(cache, x, r, [240], table)
        else:
            x = torch.randn(1, 8, 7, 128, device="cuda", generator=g).bfloat16()
            pf.append_kv_cache(cache, x, x, [240], table)
    want = attend(small, near, 247)
    table, lens, free = pf.fork_kv_rows(c, ids[None], [247], [0, 0])
    assert int(free) == tensors[0].shape[0] - 5 and int(table[1, 3]) == 0 and torch.equal(table[0], ids)
    for row in table:
        assert all(torch.equal(a, b) for a, b in zip(attend(c, row[None].contiguous(), 247), want))
    table, used = pf.compact_kv_pages(c, table, lens)
    assert int(used) == 5 and sorted(set(table.reshape(-1).tolist())) == [0, 1, 2, 3, 4]
    for row in table:
        assert all(torch.equal(a, b) for a, b in zip(attend(c, row[None].contiguous(), 247), want))
    last = tensors[0].shape[0] - 5
    pf.copy_kv_pages(c, table[0], [last, last + 1, last + 2, last + 3])
    row = torch.arange(last, last + 4, device="cuda", dtype=torch.int32)[None]
    assert all(torch.equal(a, b) for a, b in zip(attend(c, row, 247), want))


def test_queries_past_32_bits():
    """(Each row's sums run over the same keys in the same order.)"""
    import torch
    import pallas_flexattn as pf
    T = (1 << 31) // 128 + 77
    cache = tuple(torch.randn(1, 1, 64, 128, device="cuda").bfloat16() for _ in range(2))
    q = torch.zeros(1, 1, T, 128, device="cuda", dtype=torch.bfloat16)
    q[:, :, -48:] = torch.randn(1, 1, 48, 128, device="cuda").bfloat16()
    table = torch.zeros(1, 1, device="cuda", dtype=torch.int32)
    want, wl = pf.flex_prefill(q[:, :, -48:], cache, [64], table, pf.causal_mask, return_lse=True)
    for packed in (None, torch.tensor([0, T], device="cuda", dtype=torch.int32)):
        o, lse = pf.flex_prefill(q, cache, [64], table, pf.causal_mask, return_lse=True, query_starts=packed)
        # (order of a row's sums: the same; its place among the lanes may differ)
        assert torch.allclose(o[:, :, -48:].float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -12)
        assert torch.allclose(lse[:, :, -48:], wl, rtol=1e-6, atol=1e-6)
        assert (o[:, :, :T - 64] == 0).all() and (lse[:, :, :T - 64] == float("-inf")).all()
    del q, o
    T = (1 << 31) // 128 + 77
    c = pf.LatentKVCache(torch.randn(1, 64, 160, device="cuda").bfloat16(), 128)
    q, qr = (torch.zeros(1, 1, T, n, device="cuda", dtype=torch.bfloat16) for n in (128, 32))
    q[:, :, -48:] = torch.randn(1, 1, 48, 128, device="cuda").bfloat16()
    want, wl = pf.flex_decode_latent(q[:, :, -48:], qr[:, :, -48:], c, 0.1, [64], table, pf.causal_mask, True)
    o, lse = pf.flex_decode_latent(q, qr, c, 0.1, [64], table, pf.causal_mask, True)
    assert torch.allclose(o[:, :, -48:].float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -12)
    assert torch.allclose(lse[:, :, -48:], wl, rtol=1e-6, atol=1e-6)
    assert (o[:, :, :T - 64] == 0).all() and (lse[:, :, :T - 64] == float("-inf")).all()
