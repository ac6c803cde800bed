"""Arguments of the calls around a KV cache whose values, not shapes, are refused (CPU, before any GPU call)."""
import ctypes

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib
from tests.test_cache_refusals import _append_call, _cache, _decode_cache, _decode_params, _decode_q, _rot, _t


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
