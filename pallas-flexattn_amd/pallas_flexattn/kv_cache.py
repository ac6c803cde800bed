"""Paged KV caches: appending tokens, and decode over a cache in 8 bits (not in the
reference, whose roadmap lists decode).

A cache is pages of ``page_size`` tokens, (num_pages, Hkv, page_size, D); token t of
batch row b sits in row t % page_size of page ``page_table[b, t // page_size]``.  In bf16 it is
a (key, value) pair of tensors, read by ``flex_decode``; in 8 bits an :class:`Fp8KVCache`
(OCP e4m3 with one power-of-two scale for each 32 tokens of a head), half the
bytes, read by :func:`flex_decode_fp8`.  :func:`append_kv_cache` fills either.

Lengths and page tables are int32 (read as they are) or int64, on the GPU; int64 ones cost a
small launch each, in which numbers past 32 bits become the nearest that 32 bits hold.
"""
from typing import NamedTuple, Optional

from . import _lib
from .flash_attn import _resolve, _torch
from .rotary import Rotary, _check_rotary

RUN_TOKENS = 32  # tokens of a head that share a scale


class Fp8KVCache(NamedTuple):
    """A paged cache in e4m3: ``key`` / ``value`` float8_e4m3fn (num_pages, Hkv,
    page_size, D), ``key_scale`` / ``value_scale`` float32 (num_pages, Hkv,
    page_size / 32), powers of two; a value is code * scale."""
    key: object
    value: object
    key_scale: object
    value_scale: object

    def dequantize(self):
        """float32 (key, value) of the whole cache (rows never written: anything)."""
        return tuple(c.float() * s.repeat_interleave(RUN_TOKENS, dim=2)[..., None]
                     for c, s in ((self.key, self.key_scale), (self.value, self.value_scale)))


def create_fp8_kv_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> Fp8KVCache:
    """An empty :class:`Fp8KVCache` (uninitialised codes: no call reads a row
    before a token was appended there).  ``page_size``: a multiple of 32;
    ``head_dim``: 32, 64 or 128."""
    torch = _torch()
    if page_size < RUN_TOKENS or page_size % RUN_TOKENS:
        raise ValueError("page_size must be a multiple of 32")
    if head_dim not in (32, 64, 128):
        raise ValueError("the 8-bit cache takes head dims 32, 64 and 128")
    if num_pages < 1 or kv_heads < 1:
        raise ValueError("a cache has at least one page and head")
    shape = (num_pages, kv_heads, page_size, head_dim)
    codes = [torch.empty(shape, device=device, dtype=torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones((num_pages, kv_heads, page_size // RUN_TOKENS), device=device) for _ in range(2)]
    return Fp8KVCache(*codes, *scales)


def _whole(x, device):
    """Whole numbers as a tensor (a list or array is copied to ``device``; an empty one has no type of its own)."""
    if x is None or hasattr(x, "data_ptr"):
        return x
    t = _torch().as_tensor(x, device=device)
    return t if t.numel() else t.int()


def _rows(x, like):
    """Per-row integers as a tensor (a list or array is copied to ``like``'s device)."""
    return _whole(x, like.device)


def append_kv_cache(cache, key, value, kv_lens, page_table=None, new_lens=None, rotary: Optional[Rotary] = None,
                    query=None):
    """Appends new tokens, in place: ``key`` / ``value`` (B, Hkv, T, D) bf16 go to
    positions ``kv_lens[b]`` .. of every row of ``cache`` (an :class:`Fp8KVCache`, or the bf16
    (key, value) tensors that ``flex_decode`` reads), through ``page_table`` (B, max_pages)
    (None: page b belongs to row b).  ``kv_lens`` (B,) are the keys each row has before
    the call; it is not changed.  ``new_lens`` (B,): only the first so many of a row's T
    tokens (a padded batch).

    With ``rotary`` the keys are rotated to their positions on the way, and ``query``
    (B, Hq, T, D), if given, to the same ones: the call returns it rotated, dense (padded
    tokens too); without a query it returns None.  ``rotary_dim`` must be a multiple of 16.

    8 bits: a run of 32 tokens (positions 32 i .. 32 i + 31 of a row) shares a
    scale, the smallest power of two that holds its largest value in +-448; a run begun
    by an earlier call keeps its scale unless the new tokens need a larger one, to
    which the older codes are then moved.  Keys are rounded once, from the rotated
    float32 values; NaN and infinities are stored as NaN.

    Tokens past the page table's last page, or on a page id outside the cache, are
    dropped.  The pages that one call writes must be distinct, each at one place of one row's
    table (shared prefix pages are read, never appended to).  ``page_size`` must be a multiple of 32; tokens of
    any strides whose rows are 16-byte aligned are read in place.  No gradient; the versions of the
    cache's tensors rise, so that autograd notices a cache that it had saved."""
    fp8 = isinstance(cache, Fp8KVCache)
    if not fp8 and not (isinstance(cache, (tuple, list)) and len(cache) == 2):
        raise TypeError("cache must be an Fp8KVCache or a (key, value) pair of tensors")
    inv_freq, inter, scale = None, False, 1.0
    if rotary is not None:
        _check_rotary(rotary)
        inv_freq, inter, scale = rotary
    rc, out = _lib.launcher().append(cache[0], cache[1], cache[2] if fp8 else None, cache[3] if fp8 else None, key, value,
                                     _rows(kv_lens, key), page_table, _rows(new_lens, key), inv_freq, inter, scale, query)
    if rc:
        _lib.check(rc)
    return out


def flex_decode_fp8(query, cache: Fp8KVCache, kv_lens=None, page_table=None, mask_mod=None, score_mod=None,
                    scale: Optional[float] = None, enable_gqa: bool = False, return_lse: bool = False,
                    query_lens=None, kv_len: Optional[int] = None):
    """Attention of each row's newest queries over an 8-bit paged cache (no
    gradient): ``query`` (B, Hq, Sq, D) bf16, ``cache`` an :class:`Fp8KVCache`, ``kv_lens`` (B,) the
    keys of each row, the queries' own included (None: ``kv_len`` of them).  ``kv_len``: the most keys
    that a row can have (None: the whole page table); longer rows are cut to it.  The work is
    divided by it: a bound near the longest row is faster than a table made for far longer ones.  Made for
    short query blocks (decoding, speculative decoding, short chunks): the cache is read once for
    every 16 to 32 rows of Sq * Hq / Hkv, and each row's keys are split over as many workgroups as
    the batch needs.  Chunks of hundreds of queries are right but not fast: every block of rows
    walks all keys that any query of the batch row sees (a causal prompt of 2000 tokens with 32
    heads 170 us, where ``flex_attention`` on bf16 keys takes 56).

    Query i sits at position ``kv_lens[b] - Sq + i`` (bottom-right aligned, as
    ``flex_attention_varlen``); with ``query_lens`` (B,) a row has only that many queries, at
    ``kv_lens[b] - query_lens[b] + i``, and the padded ones return O = 0 and LSE = -inf, as do
    queries that see no key.  ``mask_mod``: ``causal_mask``, ``sliding_window_mask`` or another window
    :class:`MaskSpec` without documents, over these positions; ``score_mod``: the built-in ALiBi
    and soft-cap descriptors.  What no query of a row sees may be anything, and a NaN stored for a
    key reaches the queries that see it alone.  Page ids outside the cache read as zero keys.  Scales must be powers of
    two (:func:`append_kv_cache` writes no others): the kernel reads their exponents only."""
    if not isinstance(cache, Fp8KVCache):
        raise TypeError("cache must be an Fp8KVCache")
    mask, score, mods = _resolve(mask_mod, score_mod)
    if mods is not None or (mask is not None and mask.doc_ids is not None):
        raise NotImplementedError("flex_decode_fp8 takes window masks and the built-in score descriptors")
    left, right = (-1, -1) if mask is None else (mask.left, mask.right)
    slopes, cap = None, 0.0
    if score is not None:
        cap = score.softcap
        if score.alibi is not None:
            slopes = score.device_slopes(query.device)
    if scale is not None and not scale > 0:
        raise ValueError("scale must be positive")
    rc, o, lse = _lib.launcher().decode(query, *cache, _rows(kv_lens, query), page_table, _rows(query_lens, query), left,
                                        right, slopes, cap, 0.0 if scale is None else scale, enable_gqa, kv_len)
    if rc:
        _lib.check(rc)
    return (o, lse) if return_lse else o
