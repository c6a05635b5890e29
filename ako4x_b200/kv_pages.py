"""The pages of a paged cache: rows that grow, share, copy and give back pages, on the device and without
a look from the host, so that a serving step can be captured.

The state is the caller's and is changed in place: ``block_table`` int32 [rows, max_pages] (a row's pages in the
order of its tokens, -1 behind them), ``seq_lens`` int32 [rows], ``ref_counts`` int32 [pages] (how many table
entries name a page; 0 is free). Start with -1, 0 and 0. Fresh pages are the lowest free ones, in the order of the
request. Requests are int32 tensors on the device; one that cannot be met changes nothing and is
False in the bool tensor that is returned. ``caches`` is the list of tensors with the pages along their first
dimension: keys and values of every layer, and their scales. Calls on one state belong on one stream.
"""
from . import _cabi


def extend(block_table, seq_lens, ref_counts, rows, add, page_size):
    """Row ``rows[i]`` grows by ``add[i]`` tokens. False for a row out of range or listed before, where ``add`` is
    negative, the table too narrow, or where the pages asked for up to here, met or not, are more than are free."""
    return _cabi.native().kv_pages_extend(block_table, seq_lens, ref_counts, rows, add, page_size)


def free(block_table, seq_lens, ref_counts, rows, page_size):
    """The rows are emptied, their pages given back. Rows out of range, empty or listed twice are fine."""
    _cabi.native().kv_pages_free(block_table, seq_lens, ref_counts, rows, page_size)


def fork(caches, block_table, seq_lens, ref_counts, parents, children, page_size):
    """The empty row ``children[i]`` becomes a copy of row ``parents[i]`` as it was before the call: full pages are
    shared, a last page that is not full is copied to a fresh one. False for rows out of range, a child that
    is not empty or was listed before, or where no page is left."""
    return _cabi.native().kv_pages_fork(caches, block_table, seq_lens, ref_counts, parents, children, page_size)


def copy(caches, src, dst):
    """Page ``src[i]`` to page ``dst[i]`` in every cache; pairs out of range are passed over. Returns a bool tensor [1]:
    False, and nothing is copied, where a page is a destination twice, or a destination and a source."""
    return _cabi.native().kv_pages_copy(caches, src, dst)


def compact(caches, block_table, ref_counts):
    """The pages in use move into the lowest places: the highest one into the lowest free place, and so on until
    there is none below it. ``block_table`` and ``ref_counts`` follow. Returns int32 [pages]: the new place of every
    page, -1 for the free ones."""
    return _cabi.native().kv_pages_compact(caches, block_table, ref_counts)
