"""append_kv_cache writes its cache in place: autograd has to see that, as it does of torch's own in-place calls."""
import pytest

pytestmark = pytest.mark.gpu


def _append(cache, T=1):
    import torch
    import pallas_flexattn as pf
    k = torch.randn(1, 2, T, 64, device="cuda").bfloat16()
    pf.append_kv_cache(cache, k, k, [0])


def test_versions_rise():
    import torch
    import pallas_flexattn as pf
    for cache in (tuple(torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)),
                  pf.create_fp8_kv_cache(1, 2, 64, 64)):
        before = [t._version for t in cache]
        _append(cache, 0)
        assert [t._version for t in cache] == before  # (nothing written)
        _append(cache)
        assert all(t._version > b for t, b in zip(cache, before))


def test_a_saved_cache_is_noticed():
    import torch
    cache = tuple(torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w = torch.ones_like(cache[0], requires_grad=True)
    y = (w * cache[0][:, :, :8].repeat(1, 1, 8, 1)).sum() + (w * cache[0]).sum()  # (the second product saves the cache)
    _append(cache)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors_are_written_in_and_outside_inference_mode():
    """Tensors made in inference mode have no version."""
    import torch
    import pallas_flexattn as pf
    with torch.inference_mode():
        cache = pf.create_fp8_kv_cache(1, 2, 64, 64)
        _append(cache)
    with torch.no_grad():
        _append(cache)
    plain = pf.create_fp8_kv_cache(1, 2, 64, 64)
    with torch.inference_mode():
        _append(plain)
