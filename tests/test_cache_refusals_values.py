"""Arguments of the calls around a KV cache whose values, not shapes, are refused (CPU, before any GPU call)."""
import ctypes

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib
from tests.test_cache_refusals import _cache, _decode_cache, _decode_params, _rot, _t


def _append(cache):
    pf.append_kv_cache(cache, _t(2, 2, 5, 64), _t(2, 2, 5, 64), torch.zeros(2, dtype=torch.int32),
                       torch.zeros(2, 2, dtype=torch.int32), rotary=_rot(), query=_t(2, 4, 5, 64))


@pytest.mark.parametrize("field", pf.Fp8KVCache._fields)
def test_a_cache_without_one_of_its_tensors(field):
    cache = _cache()._replace(**{field: None})
    with pytest.raises((TypeError, ValueError)):
        _append(cache)
    with pytest.raises((TypeError, ValueError)):
        pf.flex_decode_fp8(_t(2, 4, 1, 64), cache, torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32),
                           enable_gqa=True)


def _decode(**kw):
    return pf.flex_decode_fp8(_t(2, 4, 1, 64), _cache(pages=1), torch.zeros(2, dtype=torch.int32),
                              torch.zeros(2, 2, dtype=torch.int32), enable_gqa=True, **kw)


@pytest.mark.parametrize("x", [1e-50, 1e-39, 1e39, float("inf"), float("nan")])
def test_numbers_that_float32_does_not_hold(x):
    """A scale that is zero in float32 would mean the default, a soft-cap none; infinite ones give NaN."""
    with pytest.raises(ValueError, match="float32" if x == x else "positive"):
        _decode(scale=x)
    if x == x:
        with pytest.raises(ValueError, match="float32"):
            _decode(score_mod=pf.softcap_score_mod(x))


@pytest.mark.parametrize("x", [2.0 ** -126, 1.0, 3e38])
def test_numbers_that_it_holds(x):
    for kw in (dict(scale=x), dict(score_mod=pf.softcap_score_mod(x))):
        with pytest.raises(ValueError, match="GPU"):  # (the device is looked at last)
            _decode(**kw)


@pytest.mark.parametrize("field", ["scale", "softcap"])
@pytest.mark.parametrize("x", [1e-39, float("inf"), float("nan"), -1.0])
def test_c_decode_numbers(field, x):
    lib = _lib.load()
    p, c = _decode_params(Skv=1 << 20, **{field: x}), _decode_cache(max_pages=1 << 14)
    assert lib.fa_fwd_kvcache_fp8(ctypes.byref(p), ctypes.byref(c), None, 16, 16, 16, 1 << 40, None) == -2
    assert lib.fa_fwd_kvcache_fp8_workspace_bytes(ctypes.byref(p), ctypes.byref(c)) == 0


@pytest.mark.parametrize("a,code", [((None, 16, 1), -1), ((16, None, 1), -1), ((16, 16, 0), -2), ((16, 16, -1), -2),
                                    ((16, 16, 2 ** 31), -2), ((12, 16, 1), -2), ((16, 18, 1), -2)])
def test_c_int64_to_int32_refuses(a, code):
    assert _lib.load().fa_int64_to_int32(*a, None) == code
