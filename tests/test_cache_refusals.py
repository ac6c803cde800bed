"""What the calls around a KV cache refuse, before any GPU call (CPU): the Python entry points on CPU
tensors (the device is the last thing they look at), and the C ABI."""
import ctypes

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib

BF = torch.bfloat16


def _t(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def _rot(n=32, **kw):
    return pf.rotary_embedding(n, device="cpu", **kw)


def _cache(pages=4, H=2, page=64, D=64):
    return pf.create_fp8_kv_cache(pages, H, page, D, device="cpu")


ROTARY = [
    (dict(q=_t(2, 4, 3, 64).float().half()), TypeError), (dict(k=_t(2, 2, 3, 64, dtype=torch.float32)), TypeError),
    (dict(q=_t(2, 4, 64)), ValueError), (dict(k=_t(2, 2, 4, 64)), ValueError), (dict(k=_t(1, 2, 3, 64)), ValueError),
    (dict(k=_t(2, 2, 3, 32)), ValueError), (dict(rotary=_rot(128)), ValueError),
    (dict(rotary=pf.Rotary(torch.ones(8))), ValueError), (dict(rotary=torch.ones(8)), TypeError),
    (dict(rotary=pf.Rotary(torch.ones(16, dtype=torch.float64)[::2])), ValueError),
    (dict(positions=torch.zeros(3)), TypeError), (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int64), offset=1), ValueError), ({}, ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("kw,err", ROTARY, ids=range(len(ROTARY)))
def test_apply_rotary_refuses(kw, err):
    a = dict(q=_t(2, 4, 3, 64), k=_t(2, 2, 3, 64), rotary=_rot(), positions=None, offset=0)
    a.update(kw)
    with pytest.raises(err):
        pf.apply_rotary(a["q"], a["k"], a["rotary"], a["positions"], a["offset"])


APPEND = [
    (dict(cache=_t(4, 2, 64, 64)), TypeError), (dict(cache=(_t(4, 2, 64, 64), _t(4, 2, 64, 32))), ValueError),
    (dict(cache=(_t(4, 2, 64, 64, dtype=torch.float32),) * 2), TypeError),
    (dict(cache=(_t(4, 2, 48, 64), _t(4, 2, 48, 64))), ValueError), (dict(cache=_cache(H=3)), ValueError),
    (dict(cache=_cache(D=32)), ValueError), (dict(cache=(_t(4, 2, 64, 128)[..., :64],) * 2), ValueError),
    (dict(cache=_cache()._replace(key_scale=torch.ones(4, 2, 3))), ValueError),
    (dict(cache=_cache()._replace(value_scale=torch.ones(4, 2, 2, dtype=torch.float64))), TypeError),
    (dict(cache=_cache()._replace(value=_t(4, 2, 64, 64))), TypeError),
    (dict(key=_t(2, 2, 5, 64, dtype=torch.float32)), TypeError), (dict(value=_t(2, 2, 4, 64)), ValueError),
    (dict(key=_t(2, 5, 64), value=_t(2, 5, 64)), ValueError),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(kv_lens=torch.zeros(2)), TypeError),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError), (dict(page_table=torch.zeros(2, 2)), TypeError),
    (dict(page_table=None, cache=_cache(pages=1)), ValueError), (dict(new_lens=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(rotary=_rot(24)), ValueError), (dict(rotary=_rot(128)), ValueError), (dict(rotary=None), ValueError),
    (dict(query=_t(2, 4, 4, 64)), ValueError), (dict(query=_t(2, 4, 5, 64, dtype=torch.float32)), TypeError),
    ({}, ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("kw,err", APPEND, ids=range(len(APPEND)))
def test_append_refuses(kw, err):
    a = dict(cache=_cache(), key=_t(2, 2, 5, 64), value=_t(2, 2, 5, 64), kv_lens=torch.zeros(2, dtype=torch.int32),
             page_table=torch.zeros(2, 2, dtype=torch.int32), new_lens=None, rotary=_rot(), query=_t(2, 4, 5, 64))
    a.update(kw)
    with pytest.raises(err):
        pf.append_kv_cache(**a)


def _labels():
    return pf.document_ids_mask([0, 0, 1, 1])


DECODE = [
    (dict(cache=(_t(4, 2, 64, 64),) * 2), TypeError), (dict(query=_t(2, 4, 1, 64, dtype=torch.float32)), TypeError),
    (dict(query=_t(2, 4, 64)), ValueError), (dict(query=_t(2, 3, 1, 64)), ValueError), (dict(enable_gqa=False), ValueError),
    (dict(query=_t(2, 4, 1, 128)), ValueError), (dict(kv_lens=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(query_lens=torch.zeros(2, 1, dtype=torch.int32)), ValueError), (dict(page_table=None), ValueError),
    (dict(mask_mod=_labels()), NotImplementedError), (dict(mask_mod=lambda q, k: q >= k + (k % 2)), NotImplementedError),
    (dict(score_mod=pf.alibi_score_mod(8)), ValueError), (dict(score_mod=lambda s, b, h, q, k: s * 2), NotImplementedError),
    (dict(scale=-1.0), ValueError), (dict(scale=0.0), ValueError), ({}, ValueError),  # (CPU tensors)
]


@pytest.mark.parametrize("kw,err", DECODE, ids=range(len(DECODE)))
def test_decode_refuses(kw, err):
    a = dict(query=_t(2, 4, 1, 64), cache=_cache(pages=1), kv_lens=torch.zeros(2, dtype=torch.int32),
             page_table=torch.zeros(2, 2, dtype=torch.int32), enable_gqa=True)
    a.update(kw)
    with pytest.raises(err):
        pf.flex_decode_fp8(**a)


@pytest.mark.parametrize("kw", [dict(page_size=48), dict(page_size=0), dict(head_dim=96), dict(num_pages=0)])
def test_create_refuses(kw):
    a = dict(num_pages=1, kv_heads=1, page_size=32, head_dim=64, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError):
        pf.create_fp8_kv_cache(**a)


# ---- the C ABI ----
def _rotary_call(**kw):
    c = _lib.FaRotaryCall()
    c.abi_version, c.dtype, c.B, c.T, c.D, c.count = _lib.ABI_VERSION, _lib.DTYPE_BF16, 1, 4, 64, 1
    c.rotary = _lib.FaRotary(16, 16, 0, 1.0)
    c.in_[0] = _lib.FaStrided(16, 256, 64, 64, 1)
    c.out[0] = 16
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=9), -8), (dict(dtype=2), -3), (dict(B=0), -2), (dict(T=0), -2), (dict(D=2000), -2), (dict(count=3), -2),
    (dict(rotary=_lib.FaRotary(16, 40, 0, 1.0)), -2), (dict(rotary=_lib.FaRotary(16, 0, 0, 1.0)), -2),
    (dict(rotary=_lib.FaRotary(None, 16, 0, 1.0)), -1), (dict(rotary=_lib.FaRotary(12, 16, 0, 1.0)), -2),
    (dict(count=2), -1), (dict(positions=18), -2), (dict(B=1 << 20, T=1 << 20), -2)])
def test_c_rotary_refuses(kw, code):
    assert _lib.load().fa_apply_rotary(ctypes.byref(_rotary_call(**kw)), None) == code
    assert _lib.load().fa_apply_rotary(None, None) == -1


@pytest.mark.parametrize("kv_len,err", [(0, ValueError), (-1, ValueError), (129, ValueError), (2 ** 40, ValueError), (1.5, TypeError)])
def test_decode_refuses_kv_len(kv_len, err):
    with pytest.raises(err):
        pf.flex_decode_fp8(_t(2, 4, 1, 64), _cache(pages=1), torch.zeros(2, dtype=torch.int32),
                           torch.zeros(2, 2, dtype=torch.int32), enable_gqa=True, kv_len=kv_len)


def test_c_calls_refuse_sizes_past_64_bits():
    """Products of sizes that would pass 2^63 are refused as well, and head counts that add up past 2^31."""
    lib, big = _lib.load(), 2 ** 31 - 1
    c = _rotary_call(B=big, T=big, D=1024)
    assert lib.fa_apply_rotary(ctypes.byref(c), None) == -2
    c = _rotary_call(count=2, T=1)
    for i in range(2):
        c.in_[i], c.out[i] = _lib.FaStrided(16, 0, 64, 64, 1 << 30), 16
    assert lib.fa_apply_rotary(ctypes.byref(c), None) == -2
    assert lib.fa_kv_append(ctypes.byref(_append_call(B=big, T=big)), None) == -2
    p, kv = _decode_params(B=1 << 30, Hq=1 << 30, Hkv=1 << 30, Sq=16), _decode_cache(num_pages=1)
    assert lib.fa_fwd_kvcache_fp8(ctypes.byref(p), ctypes.byref(kv), _decode_q(heads=1 << 30), 16, 16, 16, 1 << 40, None) == -2


def _append_call(**kw):
    c = _lib.FaKvAppendCall()
    c.abi_version, c.cache_dtype, c.B, c.T, c.D = _lib.ABI_VERSION, _lib.DTYPE_FP8_E4M3, 2, 4, 64
    c.page_size, c.max_pages, c.num_pages = 64, 2, 8
    for n in ("key", "value", "query"):
        setattr(c, n, _lib.FaStrided(16, 1024, 256, 64, 4))
    for n in ("query_out", "k_cache", "v_cache", "k_scale", "v_scale", "page_table", "kv_lens"):
        setattr(c, n, 16)
    c.rotary = _lib.FaRotary(16, 16, 0, 1.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=9), -8), (dict(cache_dtype=1), -3), (dict(D=48), -4), (dict(page_size=48), -2), (dict(page_size=0), -2),
    (dict(num_pages=0), -2), (dict(page_table=None), -2), (dict(kv_lens=None), -1), (dict(k_scale=None), -1),
    (dict(k_cache=24), -2), (dict(key=_lib.FaStrided(16, 1024, 260, 64, 4)), -2), (dict(T=0), -2),
    (dict(value=_lib.FaStrided(16, 1024, 256, 64, 2)), -2), (dict(rotary=_lib.FaRotary(16, 12, 0, 1.0)), -4),
    (dict(rotary=_lib.FaRotary(None, 16, 0, 1.0)), -1), (dict(rotary=_lib.FaRotary(None, 0, 0, 1.0)), -2),
    (dict(query_out=None), -1), (dict(rotary=_lib.FaRotary(16, 48, 0, 1.0)), -2)])
def test_c_append_refuses(kw, code):
    assert _lib.load().fa_kv_append(ctypes.byref(_append_call(**kw)), None) == code
    assert _lib.load().fa_kv_append(None, None) == -1


def _decode_params(**kw):
    p = _lib.FaParams()
    p.abi_version, p.dtype = _lib.ABI_VERSION, _lib.DTYPE_FP8_E4M3
    p.B, p.Hq, p.Hkv, p.Sq, p.Skv, p.D = 2, 4, 2, 1, 128, 64
    p.window_left = p.window_right = -1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _decode_cache(**kw):
    c = _lib.FaFp8Cache(16, 16, 16, 16, 16, 64, 2, 8, 16, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _decode_q(data=16, **kw):
    q = _lib.FaStrided(data, 256, 64, 64, 4)
    for k, v in kw.items():
        setattr(q, k, v)
    return ctypes.byref(q)


@pytest.mark.parametrize("pkw,ckw,code", [
    (dict(abi_version=9), {}, -8), (dict(dtype=0), {}, -3), (dict(D=96), {}, -4), (dict(Hq=3), {}, -2), (dict(Sq=0), {}, -2),
    (dict(Skv=129), {}, -2), (dict(Skv=2 ** 31 - 1), dict(max_pages=1 << 25), -2), (dict(softcap=-1.0), {}, -2), (dict(q_doc_ids=16), {}, -4), (dict(kv_num_blocks=16), {}, -4),
    ({}, dict(page_size=40), -2), ({}, dict(page_table=None), -2), ({}, dict(v_scale=None), -1), ({}, dict(k=24), -2),
    ({}, dict(num_pages=1 << 30, page_size=1 << 20), -2), (dict(B=1 << 14, Sq=1 << 14), {}, -2)])
def test_c_decode_refuses(pkw, ckw, code):
    lib = _lib.load()
    p, c = _decode_params(**pkw), _decode_cache(**ckw)
    assert lib.fa_fwd_kvcache_fp8(ctypes.byref(p), ctypes.byref(c), _decode_q(), 16, 16, 16, 1 << 40, None) == code
    assert lib.fa_fwd_kvcache_fp8_workspace_bytes(ctypes.byref(p), ctypes.byref(c)) == 0


def test_c_decode_workspace():
    lib = _lib.load()
    p, c = _decode_params(Skv=1 << 20), _decode_cache(max_pages=1 << 14)
    need = lib.fa_fwd_kvcache_fp8_workspace_bytes(ctypes.byref(p), ctypes.byref(c))
    assert need > 0
    call = lambda q, ws, n: lib.fa_fwd_kvcache_fp8(ctypes.byref(p), ctypes.byref(c), q, 16, 16, ws, n, None)  # noqa: E731
    ok = _decode_q()
    assert call(ok, 16, need - 1) == -6 and call(ok, None, need) == -6 and call(ok, 24, need) == -6
    assert call(None, 16, need) == -1 and call(_decode_q(None), 16, need) == -1 and call(_decode_q(24), 16, need) == -2
    assert call(_decode_q(heads=2), 16, need) == -2 and call(_decode_q(stride_h=36), 16, need) == -2
    # a walk short enough for one workgroup per item needs none
    p1, c1 = _decode_params(), _decode_cache()
    assert lib.fa_fwd_kvcache_fp8_workspace_bytes(ctypes.byref(p1), ctypes.byref(c1)) == 0
    assert lib.fa_fwd_kvcache_fp8(None, ctypes.byref(c), ok, 16, 16, 16, need, None) == -1
    assert lib.fa_fwd_kvcache_fp8(ctypes.byref(p), None, ok, 16, 16, 16, need, None) == -1


@pytest.mark.parametrize("cname,pyname", [("fa_rotary", "FaRotary"), ("fa_strided", "FaStrided"),
                                          ("fa_rotary_call", "FaRotaryCall"), ("fa_kv_append_call", "FaKvAppendCall"),
                                          ("fa_fp8_cache", "FaFp8Cache")])
def test_struct_layouts_match_header(cname, pyname, tmp_path):
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    st = getattr(_lib, pyname)
    fields = [f[0] for f in st._fields_]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flexattn.h"\nint main(void) {\n' +
                   "".join(f'  printf("%zu\\n", offsetof(struct {cname}, {f.rstrip("_")}));\n' for f in fields) +
                   f'  printf("%zu\\n", sizeof(struct {cname}));\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(st, f).offset for f in fields] + [ctypes.sizeof(st)]
