"""Attention of chunks of new tokens over a paged KV cache (not in the reference, whose roadmap lists
decode): prompts, parts of prompts, and the mixed batches of a scheduler."""
from typing import Optional

from . import _lib
from .flash_attn import _resolve
from .kv_cache import Fp8KVCache, _rows


def _window(mask_mod, score_mod, what):
    """(left, right, ScoreSpec or None) of a call that takes windows without documents and the built-in modifiers."""
    mask, score, mods = _resolve(mask_mod, score_mod)
    if mods is not None or (mask is not None and mask.doc_ids is not None):
        raise NotImplementedError(f"{what} takes window masks and the built-in score descriptors")
    return (-1, -1, score) if mask is None else (mask.left, mask.right, score)


def flex_prefill(query, cache, kv_lens=None, page_table=None, mask_mod=None, score_mod=None, scale: Optional[float] = None,
                 enable_gqa: bool = False, return_lse: bool = False, query_lens=None, query_starts=None,
                 kv_len: Optional[int] = None):
    """Attention of each row's newest tokens over a paged cache that holds them already (see
    :func:`append_kv_cache`), forward only: ``cache`` an :class:`Fp8KVCache` or the bf16 (key, value) tensors that
    ``flex_decode`` reads, ``kv_lens`` (B,) the keys of each row, the new tokens' own included (None: ``kv_len``
    of them), ``page_table`` (B, max_pages) (None: page b belongs to row b).

    The new tokens, bf16, are padded or packed. Padded: ``query`` (B, Hq, T, D), of which row b has
    ``query_lens[b]`` (None: T). Packed: ``query`` (1, Hq, tokens, D) and ``query_starts`` (B + 1,): row b has tokens
    ``query_starts[b]`` .. ``query_starts[b + 1] - 1``; it starts with 0 and does not fall (a start below an earlier one counts
    as the highest before it).  Query i of a row's n sits at
    position ``kv_lens[b] - n + i``; ``mask_mod`` (``causal_mask``, ``sliding_window_mask`` or another
    window :class:`MaskSpec` without documents; None: every key) and ``score_mod`` (the built-in ALiBi and soft-cap descriptors)
    refer to it.  Padded tokens, packed ones behind the last row's, and queries that see no key return O = 0 and
    LSE = -inf.  The result has the query's memory layout where that is dense (a projection's (tokens, heads, D) output,
    transposed), LSE is (B, Hq, T) float32.

    Made for rows of from a few to thousands of new tokens: a group of query heads reads each key once per 128 / (Hq / Hkv)
    of a row's queries, and only those that they see.  Where that gives few workgroups the keys are split over several
    (in ranges that ``kv_len``, the most keys that a row can have, decides: longer rows are cut to it; None: the whole page
    table).  Rows of one token go well in a mixed batch; for nothing but those :func:`flex_decode_fp8` is faster.

    ``page_size`` must be a multiple of 32, D 32, 64 or 128.  What no query sees may be anything; a value that is not
    finite reaches the queries that see its key alone.  Page ids outside the cache read as zero keys.  An 8-bit
    cache's scales must be powers of two.  Lengths, starts and page tables are int32 (read as they are) or int64 on the GPU."""
    fp8 = isinstance(cache, Fp8KVCache)
    if not fp8 and not (isinstance(cache, (tuple, list)) and len(cache) == 2):
        raise TypeError("cache must be an Fp8KVCache or a (key, value) pair of tensors")
    left, right, score = _window(mask_mod, score_mod, "flex_prefill")
    slopes, cap = None, 0.0
    if score is not None:
        cap = score.softcap
        if score.alibi is not None:
            slopes = score.device_slopes(query.device)
    if scale is not None and not scale > 0:
        raise ValueError("scale must be positive")
    rc, o, lse = _lib.launcher().prefill(query, cache[0], cache[1], cache[2] if fp8 else None, cache[3] if fp8 else None,
                                         _rows(kv_lens, query), page_table, _rows(query_lens, query),
                                         _rows(query_starts, query), left, right, slopes, cap,
                                         0.0 if scale is None else scale, enable_gqa, kv_len)
    if rc:
        _lib.check(rc)
    return (o, lse) if return_lse else o
