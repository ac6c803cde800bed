"""What flex_prefill, the calls on caches of latent vectors and those on pages refuse, before any GPU call (CPU): the Python
entry points on CPU tensors (the device is the last thing they look at), and the C ABI."""
import ctypes

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib
from tests.test_capi import test_struct_layouts_match_header as _layouts

BF, I32 = torch.bfloat16, torch.int32


def _t(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def _fp8(pages=4, H=2, page=64, D=64):
    return pf.create_fp8_kv_cache(pages, H, page, D, device="cpu")


def _bf16(pages=4, H=2, page=64, D=64):
    return _t(pages, H, page, D), _t(pages, H, page, D)


PREFILL = [
    (dict(cache=_t(4, 2, 64, 64)), TypeError), (dict(cache=[_t(4, 2, 64, 64)]), TypeError), (dict(cache=3), TypeError),
    (dict(cache=(_t(4, 2, 64, 64), _t(4, 2, 64, 32))), ValueError), (dict(cache=(_t(4, 2, 48, 64),) * 2), ValueError),
    (dict(cache=(_t(4, 2, 64, 64, dtype=torch.float32),) * 2), TypeError), (dict(cache=_fp8(D=32)), ValueError),
    (dict(cache=(_t(4, 2, 64, 128)[..., :64],) * 2), ValueError), (dict(cache=_fp8()._replace(key_scale=torch.ones(4, 2, 3))), ValueError),
    (dict(cache=_fp8()._replace(value_scale=None)), TypeError),
    (dict(query=_t(2, 4, 9, 64, dtype=torch.float32)), TypeError), (dict(query=_t(2, 4, 64)), ValueError),
    (dict(query=_t(2, 3, 9, 64)), ValueError), (dict(enable_gqa=False), ValueError), (dict(query=_t(2, 4, 9, 96)), ValueError),
    (dict(kv_lens=_t(1, dtype=I32)), ValueError), (dict(kv_lens=_t(2)), TypeError), (dict(kv_lens=[1, 2, 3]), ValueError),
    (dict(query_lens=_t(2, 1, dtype=I32)), ValueError), (dict(page_table=_t(3, 2, dtype=I32)), ValueError),
    (dict(page_table=_t(2, 2)), TypeError), (dict(page_table=None, cache=_bf16(pages=1)), ValueError),
    (dict(kv_len=0), ValueError), (dict(kv_len=129), ValueError), (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError),
    (dict(scale=1e-50), ValueError), (dict(scale=float("inf")), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(mask_mod=pf.document_ids_mask([0, 0, 1, 1])), NotImplementedError),
    (dict(mask_mod=lambda q, k: q >= k + (k % 2)), NotImplementedError),
    (dict(score_mod=lambda s, b, h, q, k: s * 2), NotImplementedError), (dict(score_mod=pf.alibi_score_mod(8)), ValueError),
    # packed
    (dict(query_starts=_t(3, dtype=I32)), ValueError), (dict(query=_t(1, 4, 9, 64), query_starts=_t(3)), TypeError),
    (dict(query=_t(1, 4, 9, 64), query_starts=_t(3, dtype=I32), query_lens=[1, 1]), ValueError),
    (dict(query=_t(1, 4, 9, 64), query_starts=_t(1, dtype=I32)), ValueError),
    (dict(query=_t(1, 4, 9, 64), query_starts=_t(4, dtype=I32)), ValueError), (dict(query=_t(1, 4, 9, 64), query_starts=_t(2, 2, dtype=I32)), ValueError),
    (dict(query=_t(1, 4, 9, 64), query_starts=_t(3, dtype=I32)), ValueError),  # (CPU tensors)
    ({}, ValueError), (dict(cache=_bf16()), ValueError),
]


@pytest.mark.parametrize("kw,err", PREFILL, ids=range(len(PREFILL)))
def test_prefill_refuses(kw, err):
    a = dict(query=_t(2, 4, 9, 64), cache=_fp8(), kv_lens=_t(2, dtype=I32), page_table=_t(2, 2, dtype=I32), enable_gqa=True)
    a.update(kw)
    with pytest.raises(err):
        pf.flex_prefill(**a)


def _latent(pages=4, page=64, L=128, R=32):
    return pf.create_latent_cache(pages, page, L, R, device="cpu")


LATENT = [
    (dict(cache=_t(4, 64, 160)), TypeError), (dict(cache=_latent()._replace(latent_dim=96)), ValueError),
    (dict(cache=_latent()._replace(data=_t(4, 48, 160))), ValueError), (dict(cache=_latent()._replace(data=_t(4, 64, 160, dtype=torch.float32))), TypeError),
    (dict(cache=_latent()._replace(data=_t(4, 64, 320)[..., ::2])), ValueError), (dict(cache=_latent()._replace(data=_t(64, 160))), ValueError),
    (dict(query=_t(2, 4, 1, 160)), ValueError), (dict(query=_t(2, 4, 128)), ValueError), (dict(query=_t(2, 4, 1, 128, dtype=torch.float32)), TypeError),
    (dict(query_rope=_t(2, 4, 1, 64)), ValueError), (dict(query_rope=_t(2, 3, 1, 32)), ValueError), (dict(query_rope=_t(2, 4, 2, 32)), ValueError),
    (dict(kv_lens=_t(3, dtype=I32)), ValueError), (dict(query_lens=_t(2)), TypeError), (dict(page_table=_t(2, dtype=I32)), ValueError),
    (dict(page_table=None, cache=_latent(pages=1)), ValueError), (dict(kv_len=10 ** 6), ValueError), (dict(scale=0.0), ValueError),
    (dict(scale=-0.1), ValueError), (dict(scale=1e-60), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(mask_mod=pf.document_ids_mask([0, 1])), NotImplementedError), (dict(mask_mod=lambda q, k: q >= k + (k % 2)), NotImplementedError),
    ({}, ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("kw,err", LATENT, ids=range(len(LATENT)))
def test_latent_decode_refuses(kw, err):
    a = dict(query=_t(2, 4, 1, 128), query_rope=_t(2, 4, 1, 32), cache=_latent(), scale=0.1, kv_lens=_t(2, dtype=I32),
             page_table=_t(2, 2, dtype=I32))
    a.update(kw)
    with pytest.raises(err):
        pf.flex_decode_latent(**a)


def _rot(n=32):
    return pf.rotary_embedding(n, device="cpu")


LAPPEND = [
    (dict(cache=(_t(4, 64, 160),)), TypeError), (dict(latent=_t(2, 3, 256)), ValueError), (dict(latent=_t(2, 1, 3, 128)), ValueError),
    (dict(latent=_t(2, 3, 128, dtype=torch.float32)), TypeError), (dict(key_rope=_t(2, 4, 32)), ValueError), (dict(key_rope=_t(2, 3, 64)), ValueError),
    (dict(query_rope=_t(2, 4, 3, 64)), ValueError), (dict(query_rope=_t(2, 3, 32)), ValueError), (dict(rotary=None), ValueError),
    (dict(rotary=_rot(64)), ValueError), (dict(rotary=_rot(24)), ValueError), (dict(rotary=3), TypeError), (dict(kv_lens=_t(3, dtype=I32)), ValueError),
    (dict(new_lens=_t(2)), TypeError), (dict(page_table=_t(1, 2, dtype=I32)), ValueError), (dict(page_table=None, cache=_latent(pages=1)), ValueError),
    ({}, ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("kw,err", LAPPEND, ids=range(len(LAPPEND)))
def test_latent_append_refuses(kw, err):
    a = dict(cache=_latent(), latent=_t(2, 3, 128), key_rope=_t(2, 3, 32), kv_lens=_t(2, dtype=I32), page_table=_t(2, 2, dtype=I32),
             rotary=_rot(), query_rope=_t(2, 4, 3, 32))
    a.update(kw)
    with pytest.raises(err):
        pf.append_latent_cache(**a)


@pytest.mark.parametrize("kw", [dict(page_size=48), dict(page_size=0), dict(latent_dim=500), dict(rope_dim=16), dict(num_pages=0)])
def test_create_latent_refuses(kw):
    a = dict(num_pages=1, page_size=32, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError):
        pf.create_latent_cache(**a)


def _ids(*x, dtype=I32):
    return torch.tensor(x, dtype=dtype)


CACHES = [
    (3, TypeError), ([], TypeError), ([3], TypeError), ((_t(4, 2, 64, 64),), TypeError), ([(_t(4, 2, 64, 64),) * 3], TypeError),
    ((_t(4, 2, 64, 64), "x"), TypeError), ((_t(4, 2, 64), _t(4, 2, 64)), ValueError), (_fp8()._replace(key_scale=_t(4, 2, 1, 2)), ValueError),
    ((_t(4, 2, 64, 64), _t(3, 2, 64, 64)), ValueError), ([_bf16(), _bf16(page=32)], ValueError), ([_bf16(), _latent(page=32)], ValueError),
    ((_t(4, 2, 64, 128)[..., ::2],) * 2, ValueError), ((_t(0, 2, 64, 64),) * 2, ValueError),
    (_bf16(), ValueError), ([_fp8(), _fp8()], ValueError), (_latent(), ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("caches,err", CACHES, ids=range(len(CACHES)))
def test_pages_refuse_caches(caches, err):
    with pytest.raises(err):
        pf.copy_kv_pages(caches, _ids(0), _ids(1))
    with pytest.raises(err):
        pf.fork_kv_rows(caches, _t(1, 2, dtype=I32), _ids(0))
    with pytest.raises(err):
        pf.compact_kv_pages(caches, _t(1, 2, dtype=I32), _ids(0))


@pytest.mark.parametrize("src,dst,err", [(_ids(0.5, dtype=torch.float32), _ids(0), TypeError), (_ids(0, 1), _ids(0), ValueError),
                                         (_t(1, 1, dtype=I32), _t(1, 1, dtype=I32), ValueError)])
def test_copy_refuses(src, dst, err):
    with pytest.raises(err):
        pf.copy_kv_pages(_bf16(), src, dst)


PLANS = [
    (dict(page_table=_t(2, 3)), TypeError), (dict(page_table=_ids(0, 1)), ValueError), (dict(page_table=_t(0, 3, dtype=I32)), ValueError),
    (dict(kv_lens=_ids(1)), ValueError), (dict(kv_lens=_t(2)), TypeError), (dict(parents=_t(2)), TypeError),
    (dict(parents=_t(0, dtype=I32)), ValueError), (dict(parents=_t(1, 1, dtype=I32)), ValueError), (dict(room=-1), ValueError),
    (dict(room=_ids(1, 2, 3)), ValueError), (dict(room=_t(2)), TypeError), (dict(room=2 ** 31), ValueError), (dict(room=1.5), (TypeError, ValueError)),
    (dict(keep=_t(4, dtype=I32)), TypeError), (dict(keep=_t(3, dtype=torch.bool)), ValueError), ({}, ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("kw,err", PLANS, ids=range(len(PLANS)))
def test_fork_refuses(kw, err):
    a = dict(caches=_bf16(), page_table=_t(2, 3, dtype=I32), kv_lens=_ids(0, 1))
    a.update(kw)
    with pytest.raises(err):
        pf.fork_kv_rows(**a)


@pytest.mark.parametrize("kw,err", [p for p in PLANS if not {"parents"} & set(p[0])], ids=str)
def test_compact_refuses(kw, err):
    a = dict(caches=_bf16(), page_table=_t(2, 3, dtype=I32), kv_lens=_ids(0, 1))
    a.update(kw)
    with pytest.raises(TypeError if torch.is_tensor(kw.get("room")) else err):  # (one number for all rows)
        pf.compact_kv_pages(**a)


# ---- the C ABI (pointers that are never read) ----
@pytest.mark.parametrize("cname,pyname", [("fa_prefill_call", "FaPrefillCall"), ("fa_latent_append_call", "FaLatentAppendCall"),
                                          ("fa_latent_call", "FaLatentCall"), ("fa_paged_tensor", "FaPagedTensor"),
                                          ("fa_page_plan_call", "FaPagePlanCall")])
def test_struct_layouts(cname, pyname, tmp_path):
    _layouts(cname, pyname, tmp_path)


def _fill(c, base, kw):
    for k, v in {**base, **kw}.items():
        setattr(c, k, v)
    return c


def _strided(heads, data=16):
    return _lib.FaStrided(data, 4096, 64, 1024, heads)


def _prefill(**kw):
    return _fill(_lib.FaPrefillCall(), dict(
        abi_version=_lib.ABI_VERSION, cache_dtype=_lib.DTYPE_BF16, B=2, Hkv=2, T=100, D=64, page_size=64, max_pages=8, num_pages=16,
        kv_len=512, window_left=-1, window_right=0, query=_strided(4), out=_strided(4), lse=16, k_cache=16, v_cache=16,
        page_table=16, kv_lens=16), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=9), -8), (dict(cache_dtype=1), -3), (dict(D=96), -4), (dict(B=0), -2), (dict(T=0), -2), (dict(Hkv=3), -2),
    (dict(query=_strided(0)), -2), (dict(out=_strided(2)), -2), (dict(page_size=48), -2), (dict(num_pages=0), -2), (dict(max_pages=0), -2),
    (dict(page_table=None), -2), (dict(kv_len=513), -2), (dict(kv_len=0), -2), (dict(scale=float("nan")), -2), (dict(scale=-1.0), -2),
    (dict(softcap=1e-45), -2), (dict(q_lens=16, q_starts=16), -4), (dict(query=_strided(4, None)), -1), (dict(lse=None), -1),
    (dict(v_cache=None), -1), (dict(cache_dtype=_lib.DTYPE_FP8_E4M3), -1), (dict(k_cache=8), -2), (dict(query=_strided(4, 8)), -2),
    (dict(out=_lib.FaStrided(16, 4096, 64, 1028, 4)), -2), (dict(T=2 ** 30), -2), (dict(num_pages=2 ** 30), -2)])
def test_prefill_codes(kw, code):
    lib, c = _lib.load(), _prefill(**kw)
    assert lib.fa_prefill_workspace_bytes(ctypes.byref(c)) == 0
    assert lib.fa_prefill(ctypes.byref(c), None, 0, None) == code
    assert lib.fa_prefill(None, None, 0, None) == -1


def test_prefill_workspace():
    """Few items over long keys are split: their partial results want room, aligned."""
    lib, c = _lib.load(), _prefill(kv_len=512, T=8)
    need = lib.fa_prefill_workspace_bytes(ctypes.byref(c))
    assert need > 0 and need % (2 * 4 * 8 * 66 * 4) == 0
    assert lib.fa_prefill(ctypes.byref(c), None, need, None) == -6
    assert lib.fa_prefill(ctypes.byref(c), 16, need - 1, None) == -6
    assert lib.fa_prefill(ctypes.byref(c), 24, need, None) == -6
    many = _prefill(B=64, num_pages=64, T=512, Hkv=4)
    assert lib.fa_prefill_workspace_bytes(ctypes.byref(many)) == 0


def _lat(**kw):
    return _fill(_lib.FaLatentCall(), dict(
        abi_version=_lib.ABI_VERSION, B=2, T=1, latent_dim=512, rope_dim=64, page_size=64, max_pages=8, num_pages=16, kv_len=512,
        window_left=-1, window_right=-1, scale=0.1, query=_strided(16), query_rope=_strided(16), o=16, lse=16, cache=16, page_table=16,
        kv_lens=16), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -8), (dict(latent_dim=384), -4), (dict(rope_dim=48), -4), (dict(B=0), -2), (dict(T=0), -2), (dict(page_size=16), -2),
    (dict(page_table=None), -2), (dict(kv_len=1000), -2), (dict(scale=0.0), -2), (dict(scale=float("inf")), -2), (dict(query_rope=_strided(8)), -2),
    (dict(cache=None), -1), (dict(o=None), -1), (dict(query=_strided(16, 8)), -2), (dict(o=8), -2), (dict(query=_strided(2 ** 30), query_rope=_strided(2 ** 30), T=9), -2)])
def test_latent_codes(kw, code):
    lib, c = _lib.load(), _lat(**kw)
    assert lib.fa_latent_decode_workspace_bytes(ctypes.byref(c)) == 0
    assert lib.fa_latent_decode(ctypes.byref(c), None, 0, None) == code


def test_latent_workspace():
    lib, c = _lib.load(), _lat()
    need = lib.fa_latent_decode_workspace_bytes(ctypes.byref(c))
    assert need > 0 and lib.fa_latent_decode(ctypes.byref(c), None, need, None) == -6
    assert lib.fa_latent_decode(ctypes.byref(c), 16, need - 1, None) == -6
    short = _lat(kv_len=200)
    assert lib.fa_latent_decode_workspace_bytes(ctypes.byref(short)) == 0


def _lapp(**kw):
    return _fill(_lib.FaLatentAppendCall(), dict(
        abi_version=_lib.ABI_VERSION, B=2, T=3, latent_dim=128, rope_dim=32, page_size=64, max_pages=8, num_pages=16, latent=_strided(1),
        rope=_strided(1), query=_strided(4), query_out=16, cache=16, page_table=16, kv_lens=16, rotary=_lib.FaRotary(16, 16, 0, 1.0)), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -8), (dict(latent_dim=64), -4), (dict(rope_dim=0), -4), (dict(T=0), -2), (dict(latent=_strided(2)), -2),
    (dict(kv_lens=None), -1), (dict(cache=None), -1), (dict(cache=8), -2), (dict(rope=_strided(1, None)), -1), (dict(rotary=_lib.FaRotary(16, 24, 0, 1.0)), -2),
    (dict(rotary=_lib.FaRotary(16, 12, 0, 1.0)), -4), (dict(rotary=_lib.FaRotary(None, 16, 0, 1.0)), -1), (dict(rotary=_lib.FaRotary()), -2),
    (dict(query_out=None), -1), (dict(page_table=None), -2), (dict(B=2 ** 30, T=2 ** 20), -2)])
def test_latent_append_codes(kw, code):
    c = _lapp(**kw)
    assert _lib.load().fa_latent_append(ctypes.byref(c), None) == code


def _plan(**kw):
    t = (_lib.FaPagedTensor * 1)(_lib.FaPagedTensor(16, 4096))
    c = _fill(_lib.FaPagePlanCall(), dict(
        abi_version=_lib.ABI_VERSION, B=2, N=3, max_pages=4, page_size=64, num_pages=16, page_table=16, kv_lens=16, parents=16, out_table=16,
        out_lens=16, out_count=16, tensors=t, tensor_count=1), kw)
    return c, t


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -8), (dict(B=0), -2), (dict(N=0), -2), (dict(parents=None), -2), (dict(page_size=0), -2), (dict(num_pages=0), -2),
    (dict(room_all=-1), -2), (dict(max_pages=2 ** 30), -2), (dict(page_table=None), -1), (dict(out_lens=None), -1), (dict(tensor_count=-1), -2),
    (dict(tensors=(_lib.FaPagedTensor * 1)(_lib.FaPagedTensor(None, 64))), -1), (dict(tensors=(_lib.FaPagedTensor * 1)(_lib.FaPagedTensor(16, 6))), -2),
    (dict(tensors=(_lib.FaPagedTensor * 1)(_lib.FaPagedTensor(18, 64))), -2), ({}, -6)])
def test_plan_codes(kw, code):
    lib = _lib.load()
    c, _ = _plan(**kw)
    assert lib.fa_fork_rows(ctypes.byref(c), None, 0, None) == code
    c, _ = _plan(**{"parents": None, "N": 2, **{k: v for k, v in kw.items() if k != "out_lens"}})
    want = {(-1 if "out_lens" in kw else code)} | ({-6} if "out_lens" in kw or "parents" in kw else set())
    assert lib.fa_compact_pages(ctypes.byref(c), None, 0, None) in want
    assert (lib.fa_fork_rows_workspace_bytes(ctypes.byref(_plan()[0])) > 0)


def test_copy_codes():
    lib = _lib.load()
    t = (_lib.FaPagedTensor * 1)(_lib.FaPagedTensor(16, 64))
    for args, code in (((t, 1, 0, 16, 16, 1), -2), ((t, 1, 4, 16, 16, -1), -2), ((t, -1, 4, 16, 16, 1), -2), ((None, 1, 4, 16, 16, 1), -1),
                       ((t, 1, 4, None, 16, 1), -1), ((t, 1, 4, 16, 16, 0), 0), ((t, 0, 4, 16, 16, 1), 0)):
        assert lib.fa_copy_pages(*args, None) == code
