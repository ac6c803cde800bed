"""The pages of paged KV caches (not in the reference): copying, forking, compacting and freeing them, on the
GPU and without synchronisation.

Every function takes one cache or a list of caches (the layers of a model) that share page tables: an
:class:`Fp8KVCache`, the bf16 (key, value) tensors, or a :class:`LatentKVCache`, of equal page
counts and sizes.  Nothing but the tables and lengths says which pages are in use: those that a row's tokens
fill, and those that the caller holds for something else (``keep``, (num_pages,) bool: a prefix cache).  All others are
free, so a row that is not taken over is freed by that.

Page ids, tables and lengths are int32 (read as they are) or int64; what comes back is int32.
"""
from numbers import Integral

from . import _lib
from .kv_cache import _whole


def _ints(x, caches):
    """Whole numbers as a tensor (a list or array is copied to the caches' device)."""
    c = caches
    while isinstance(c, (list, tuple)) and c:
        c = c[0]
    return _whole(x, getattr(c, "device", None))


def copy_kv_pages(caches, src, dst) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` in every cache, in place (``src``, ``dst``: vectors of page ids on the
    GPU).  Pairs with an id outside the cache are left out, so a vector may be padded with -1.  The pages ``dst``
    must be distinct, and none of them among ``src``."""
    rc = _lib.launcher().copy_pages(caches, _ints(src, caches), _ints(dst, caches))
    if rc:
        _lib.check(rc)


def fork_kv_rows(caches, page_table, kv_lens, parents=None, room=0, keep=None):
    """Rows that go on from other rows -> (page_table, kv_lens, free): the beams of a search after a step, samples of one
    prompt, a batch some of whose rows ended, or (``parents`` None: each row from itself) just room for the next tokens.

    Row b of the result has the tokens of row ``parents[b]`` of ``page_table`` (B, max_pages) and ``kv_lens`` (B,); a
    parent outside [0, B) gives an empty row.  Pages that a row's tokens fill are shared by all that have them.  A last page that they fill in
    part becomes the row's own, to be appended to: the first row that ends in it keeps it, unless another one has the whole of it or it
    is in ``keep``; the others get a copy, in every cache.  Behind its tokens a row gets pages for ``room`` (a
    number, or one per row) more, as far as the table goes; the entries behind those are -1.

    Copies and room come from the free pages, lowest first, row by row: pages that neither the result's rows nor ``keep``
    hold.  ``free`` (int32, on the GPU) is how many are left; where it is negative so many were lacking, and
    the entries that lack one are -1 (tokens of a copy that could not be made are lost: look before going on).
    Page ids outside the cache stay as they are."""
    per_row, number = (None, int(room)) if isinstance(room, Integral) else (_ints(room, caches), 0)
    rc, table, lens, free = _lib.launcher().page_plan(True, caches, page_table, _ints(kv_lens, caches), _ints(parents, caches),
                                                      per_row, number, keep)
    if rc:
        _lib.check(rc)
    return table, lens, free


def compact_kv_pages(caches, page_table, kv_lens, room: int = 0, keep=None):
    """Moves the pages in use to the front -> (page_table, used): with n pages in use (that a row's tokens and ``room`` more
    fill, or ``keep`` holds), those with ids from n on that ``keep`` does not hold move, in every cache, to the
    free ids below n, both in ascending order.  ``used`` (int32, on the GPU) is n; pages that ``keep`` holds stay where they
    are.  Entries past a row's tokens and room are -1, page ids outside the cache stay as they are."""
    rc, table, _, used = _lib.launcher().page_plan(False, caches, page_table, _ints(kv_lens, caches), None, None, room, keep)
    if rc:
        _lib.check(rc)
    return table, used
