"""Latent attention over a paged cache (not in the reference): every token keeps one latent vector, from which all
heads' keys and values are products, and a rotary part that is key only.

In the absorbed form a head's up-projections are taken into its query (before) and its output (after),
so that the attention itself reads the latent vectors: for heads with key W_k c and value W_v c,

    query = q_nope W_k,  score = scale (query . c + q_rope . k_rope),  o = softmax(score) c,  head's output = W_v o.

A cache is pages of ``page_size`` tokens, (num_pages, page_size, latent_dim + rope_dim) bf16, the latent
vector first; page tables and lengths as for :mod:`pallas_flexattn.kv_cache`.
"""
from typing import NamedTuple, Optional

from . import _lib
from .flash_attn import _torch
from .kv_cache import RUN_TOKENS, _rows
from .prefill import _window
from .rotary import Rotary, _check_rotary


class LatentKVCache(NamedTuple):
    """A paged cache of latent vectors: ``data`` bf16 (num_pages, page_size, latent_dim + rope_dim)."""
    data: object
    latent_dim: int

    @property
    def rope_dim(self) -> int:
        return self.data.shape[2] - self.latent_dim


def _check_cache(cache):
    if not isinstance(cache, LatentKVCache):
        raise TypeError("cache must be a LatentKVCache (see create_latent_cache)")


def create_latent_cache(num_pages: int, page_size: int, latent_dim: int = 512, rope_dim: int = 64, device="cuda") -> LatentKVCache:
    """An empty :class:`LatentKVCache` (uninitialised: no call reads a row before a token was appended there).
    ``page_size``: a multiple of 32; ``latent_dim``: 128, 256 or 512; ``rope_dim``: 32 or 64."""
    torch = _torch()
    if page_size < RUN_TOKENS or page_size % RUN_TOKENS:
        raise ValueError("page_size must be a multiple of 32")
    if latent_dim not in (128, 256, 512) or rope_dim not in (32, 64):
        raise ValueError("latent_dim must be 128, 256 or 512, rope_dim 32 or 64")
    if num_pages < 1:
        raise ValueError("a cache has at least one page")
    return LatentKVCache(torch.empty((num_pages, page_size, latent_dim + rope_dim), device=device, dtype=torch.bfloat16), latent_dim)


def append_latent_cache(cache: LatentKVCache, latent, key_rope, kv_lens, page_table=None, new_lens=None,
                        rotary: Optional[Rotary] = None, query_rope=None):
    """Appends new tokens, in place: ``latent`` (B, T, latent_dim) and ``key_rope`` (B, T, rope_dim), bf16, go to positions
    ``kv_lens[b]`` .. of every row, through ``page_table`` (B, max_pages) (None: page b belongs to row b).
    ``kv_lens`` (B,) are the keys each row has before the call; it is not changed.  ``new_lens`` (B,): only the
    first so many of a row's T tokens (a padded batch).

    With ``rotary`` the rotary parts are rotated to their positions on the way, and ``query_rope`` (B, H, T, rope_dim), if
    given, to the same ones: the call returns it rotated, dense (padded tokens too); without it, None.
    ``rotary_dim`` must be a multiple of 16.

    Tokens past the page table's last page, or on a page id outside the cache, are dropped.  The rows that one call writes must
    be distinct (shared prefix pages are read, never appended to).  Tokens of any strides whose rows are 16-byte aligned
    are read in place.  No gradient; the cache's version rises, so that autograd notices a cache that it had saved."""
    _check_cache(cache)
    inv_freq, inter, scale = None, False, 1.0
    if rotary is not None:
        _check_rotary(rotary)
        inv_freq, inter, scale = rotary
    rc, out = _lib.launcher().latent_append(cache.data, cache.latent_dim, latent, key_rope, _rows(kv_lens, latent), page_table,
                                            _rows(new_lens, latent), inv_freq, inter, scale, query_rope)
    if rc:
        _lib.check(rc)
    return out


def flex_decode_latent(query, query_rope, cache: LatentKVCache, scale: float, kv_lens=None, page_table=None, mask_mod=None,
                       return_lse: bool = False, query_lens=None, kv_len: Optional[int] = None):
    """Attention of each row's newest queries over a cache of latent vectors, absorbed form (no gradient):
    ``query`` (B, H, T, latent_dim), the heads' queries times their key up-projections, ``query_rope`` (B, H, T,
    rope_dim), rotated, both bf16 -> (B, H, T, latent_dim), the weighted latent vectors of each head.  ``scale`` is that of the
    heads as they were before (one over the root of their key's whole length): it has no default here.

    ``kv_lens`` (B,): the keys of each row, the queries' own included (None: ``kv_len`` of them).  Query i of ``query_lens[b]``
    (None: T) sits at position ``kv_lens[b] - query_lens[b] + i``, which ``mask_mod`` refers to (``causal_mask``,
    ``sliding_window_mask`` or another window :class:`MaskSpec` without documents); padded queries, and those that see no
    key, return O = 0 and LSE = -inf.  ``kv_len``: the most keys that a row can have (None: the whole page table); longer rows
    are cut to it, and the work is divided by it.

    Made for decoding and short chunks: each key is read once for up to 64 rows (heads x queries), and long rows' keys
    are split over as many workgroups as the batch needs.  (A prompt takes three times the operations that it
    would take with its heads' keys and values written out, which are of two lengths, so that no other call here takes them; and
    its blocks of rows walk all tiles that the batch row sees.)  Page ids outside the cache read as zero keys; what no query of a row sees
    may be anything."""
    _check_cache(cache)
    left, right, _ = _window(mask_mod, None, "flex_decode_latent")
    rc, o, lse = _lib.launcher().latent_decode(query, query_rope, cache.data, cache.latent_dim, scale, _rows(kv_lens, query),
                                               page_table, _rows(query_lens, query), left, right, kv_len)
    if rc:
        _lib.check(rc)
    return (o, lse) if return_lse else o
