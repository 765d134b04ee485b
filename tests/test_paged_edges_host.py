"""Edges of the paged cache entry points that need no GPU: workspaces, refusals, layouts."""

import ctypes as C

import pytest

P = 4096                                 # a well-aligned address that nothing reads: no call here reaches a launch


@pytest.fixture(scope="module")
def hip():
    from lcm import _hip
    return _hip


def _pages(hip, **kw):
    return hip.KVPages(**{**dict(k=P, v=P, n_pages=8, page_size=16, n_kv_heads=8, head_dim=128, dtype=1), **kw})


def _batch(hip, **kw):
    return hip.PagedBatch(**{**dict(page_table=P, seq_lens=P, q_starts=P, n_seqs=8, max_pages=1 << 16, max_q=1, max_keys=32768), **kw})


def _workspace(hip, pages, batch, rows, heads, prefix=None):
    n = C.c_size_t()
    if prefix is None:
        hip.check(hip.lib.lcmhip_paged_attention_workspace(pages, batch, rows, heads, C.byref(n)))
    else:
        hip.check(hip.lib.lcmhip_shared_prefix_attention_workspace(pages, batch, prefix, rows, heads, C.byref(n)))
    return n.value


def test_a_wrong_max_q_does_not_cost_gigabytes(hip):
    """Partial results are (rows, heads) times the parts of a list; the number of parts is chosen for few rows a sequence, and a
    max_q that understates them must not multiply it with all rows there are."""
    partial = 4 * 128 + 8
    for rows in (1 << 10, 1 << 14, 1 << 18, 1 << 22):
        assert _workspace(hip, _pages(hip), _batch(hip), rows, 32) <= (1 << 20) * partial + 256
        prefix = hip.SharedPrefix(page_table=P, lens=P, group_starts=P, n_groups=1 << 20, max_pages=1 << 16, max_keys=32768)
        assert _workspace(hip, _pages(hip), _batch(hip), rows, 32, prefix) <= 2 * max(1 << 20, rows * 32) * partial + 256
    # what a right max_q gives is as it was: 64 parts for two long sequences, padding rows among them, a few for many sequences
    for rows in (2, 64, 512):
        assert _workspace(hip, _pages(hip), _batch(hip, n_seqs=2, max_keys=131072), rows, 32) == 64 * rows * 32 * partial
    assert _workspace(hip, _pages(hip, n_kv_heads=16), _batch(hip, n_seqs=64, max_keys=3800), 64, 16) == 4 * 64 * 16 * partial


def test_bounds_that_32_bits_would_cut_are_refused():
    """The structs hold 32-bit numbers, and ctypes cuts what does not fit without a word: 2^32 + 16 would be 16."""
    from types import SimpleNamespace
    from lcm.nn import paged_attention as pa
    wide = SimpleNamespace(page_size=65536)
    for max_keys in (2**30 + 1, 2**31, 2**32 + 16):
        with pytest.raises(ValueError, match="max_keys"):
            pa._reach(max_keys, 1 << 20, wide)
    assert pa._reach(2**30, 1 << 20, wide) == 2**30 and pa._reach(None, 1 << 20, wide) == 2**30 and pa._reach(None, 2, wide) == 131072


@pytest.mark.parametrize("rotary_dim", [33, 127, 1, 0, -16, 24])
def test_a_rotary_table_of_an_odd_width_is_refused(rotary_dim):
    """An odd width would lose a dimension and turn the others by angles of another width; only multiples of 16 can be used at all."""
    from lcm.nn import paged_attention as pa
    with pytest.raises(ValueError, match="rotary_dim"):
        pa.RotaryTable.create(8, rotary_dim, device="cpu")


def _overlap(rows, heads, d, row, head):
    """Whether two (row, head) pieces of d values share one, by looking at all of them."""
    starts = sorted(t * row + h * head for t in range(rows) for h in range(heads))
    return any(b - a < d for a, b in zip(starts, starts[1:]))


def test_outputs_whose_rows_lie_on_each_other_are_refused(hip):
    """An expanded q_out, or one of overlapping rows, would be written by many waves at once.  Strides in units of 16 bytes."""
    def call(rows, heads, row, head, which):
        given, out, none = (P, heads * 128, 128), (P + (1 << 20), row, head), (None, 0, 0)
        tensors = (*given, *none, *out, *none) if which == "q" else (*none, *given, *none, *out)
        # a rotation of no positions ends every call that gets past the strides before it is launched
        rot = hip.Rotary(cos=P, sin=P, n_positions=0, rotary_dim=64, style=0)
        rc = hip.lib.lcmhip_head_norm_rope(*tensors, rows, heads, heads, 64, None, rot, P, 0, None)
        assert rc == -1
        return b"each other" in hip.lib.lcmhip_last_error()
    for which in ("q", "k"):
        for rows in (1, 2, 3, 7):
            for heads in (1, 2, 5):
                for row in (0, 32, 64, 128, 192, 256, 320, 448, 2240, -320):
                    for head in (0, 64, 60, 96, 128, 192, 448, 704, -64):
                        assert call(rows, heads, row, head, which) == _overlap(rows, heads, 64, row, head), (rows, heads, row, head)


def test_grids_past_the_launch_limit_are_refused(hip):
    """A launch holds fewer than 2^32 work items a dimension, 2^24 workgroups of 256: what needs more is refused by name and before
    anything is launched, not by the runtime behind the first kernel."""
    def refused(rc, text=b"workgroups"):
        return rc == -1 and text in hip.lib.lcmhip_last_error()
    one = dict(max_pages=1, max_keys=16)
    many_seqs = _batch(hip, n_seqs=1 << 21, q_starts=None)
    assert refused(hip.lib.lcmhip_paged_attention(_pages(hip), many_seqs, P, 1024, 128, P, 1 << 21, 8, 0.1, 1, P, 1 << 40, None))
    # the few-row kernel of one prefix's rows and the joining kernel behind it: rows of 128 heads, 2^27 results
    prefix = hip.SharedPrefix(page_table=P, lens=P, group_starts=P, n_groups=1 << 20, max_pages=1, max_keys=16)
    rows = (1 << 20) + 8
    wide = _pages(hip, n_kv_heads=1)
    assert refused(hip.lib.lcmhip_shared_prefix_attention(wide, _batch(hip, n_seqs=rows, q_starts=None, **one), prefix, P, 16384, 128, P, rows, 128, 0.1, 1,
                                                          P, 1 << 60, None))
    # heads: eight rows of eight heads a workgroup at head_dim 64, so 2^30 rows are 2^28 workgroups
    assert refused(hip.lib.lcmhip_head_norm_rope(P, 512, 64, None, 0, 0, P + (1 << 20), 512, 64, None, 0, 0, 1 << 30, 8, 0, 64, None, None, None, 1, None))
    assert refused(hip.lib.lcmhip_paged_append(_pages(hip), _batch(hip, **one), P, 1024, 128, P, 1024, 128, None, 0, 0, None, 1 << 28, 0,
                                               None, None, None, None))
