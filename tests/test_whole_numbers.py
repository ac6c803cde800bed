"""Empty lists and arrays where the calls on caches take whole numbers (CPU: what comes last is the refusal of CPU tensors)."""
import numpy as np
import pytest
import torch

import pallas_flexattn as pf


def _cache(pages=4):
    return tuple(torch.zeros(pages, 2, 64, 64, dtype=torch.bfloat16) for _ in range(2))


TABLE = torch.zeros(2, 3, dtype=torch.int32)


@pytest.mark.parametrize("empty", [[], (), np.array([]), np.array([], dtype=np.int64), torch.zeros(0, dtype=torch.int32)], ids=range(5))
def test_nothing_to_copy(empty):
    with pytest.raises(ValueError, match="on the GPU"):
        pf.copy_kv_pages(_cache(), empty, empty)


def test_an_empty_tensor_keeps_its_type():
    with pytest.raises(TypeError, match="int32 or int64"):
        pf.copy_kv_pages(_cache(), torch.zeros(0), torch.zeros(0))


def test_no_rows():
    """A batch without rows: its lengths, as a list, are an empty one."""
    q, latent = torch.zeros(0, 4, 3, 64, dtype=torch.bfloat16), pf.create_latent_cache(4, 64, 128, 32, device="cpu")
    none = TABLE[:0]
    with pytest.raises(ValueError, match="on the GPU"):
        pf.flex_prefill(q, _cache(), [], none, enable_gqa=True, query_lens=[])
    with pytest.raises(ValueError, match="on the GPU"):
        pf.flex_decode_fp8(q, pf.create_fp8_kv_cache(4, 2, 64, 64, device="cpu"), [], none, enable_gqa=True, query_lens=[])
    with pytest.raises(ValueError, match="on the GPU"):
        pf.flex_decode_latent(q.new_zeros(0, 4, 3, 128), q.new_zeros(0, 4, 3, 32), latent, 0.1, [], none, query_lens=[])
    with pytest.raises(ValueError, match="on the GPU"):
        pf.append_latent_cache(latent, q.new_zeros(0, 3, 128), q.new_zeros(0, 3, 32), [], none, new_lens=[])


@pytest.mark.gpu
def test_on_the_gpu():
    cache = tuple(torch.randn(6, 2, 32, 64, device="cuda").bfloat16() for _ in range(2))
    before = [x.clone() for x in cache]
    pf.copy_kv_pages(cache, [], [])
    assert all(torch.equal(x, y) for x, y in zip(cache, before))
    table = torch.tensor([[3, 1, -1]], device="cuda", dtype=torch.int32)
    q = torch.randn(0, 4, 3, 64, device="cuda").bfloat16()
    assert pf.flex_prefill(q, cache, [], table[:0], enable_gqa=True, query_lens=[]).shape == q.shape
