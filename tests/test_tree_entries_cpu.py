"""Arguments that the C entries of the speculative-decoding operators have to tell apart. Every call here ends in a
refusal of its own kind, so none is launched wherever this runs; addresses are never followed."""

import ctypes

import pytest


def _commit_args():
    import bdfp4

    a = bdfp4.CommitArgs()
    a.layers, a.rows, a.nodes, a.heads_kv, a.tail_slots, a.page_tokens, a.pages = 1, 2, 5, 2, 3, 128, 4
    for name in ("draft_key", "draft_value", "accepted", "accepted_counts", "seq_lens", "row_to_slot", "tail_key",
                 "tail_value", "page_table", "new_seq_lens", "seqused_fp4", "seqused_residual", "seqused_sink",
                 "source_tokens", "destination_pages"):
        setattr(a, name, 1 << 20)
    a.max_pages_per_row, a.page_table_stride = 2, 2
    return a


@pytest.mark.parametrize("change", [
    dict(source_tokens=0), dict(destination_pages=0), dict(source_tokens=0, destination_pages=0),
    dict(page_table=0), dict(pages=0), dict(max_pages_per_row=-1), dict(page_table=0, max_pages_per_row=0, pages=0),
])
def test_commit_work_table_goes_with_a_page_table(change):
    """Both halves of the work table or neither; a table of no columns may have no address, one of some may not."""
    import bdfp4

    a = _commit_args()
    for name, value in change.items():
        setattr(a, name, value)
    assert bdfp4.library().bdfp4_commit_drafts(ctypes.byref(a), None) == bdfp4.E_ARG


def test_tree_takes_a_table_of_no_columns():
    """No row reads a page: the check behind the table's is the one that refuses this call."""
    import bdfp4
    from test_tree_cpu import _tree_args

    a = _tree_args()
    a.page_table, a.page_table_stride, a.max_pages_per_row, a.page_tokens = 0, 1, 0, 32
    assert bdfp4.library().bdfp4_tree_decode(ctypes.byref(a), None) == bdfp4.E_UNSUPPORTED
    a.max_pages_per_row = 1
    assert bdfp4.library().bdfp4_tree_decode(ctypes.byref(a), None) == bdfp4.E_ARG


def test_strides_of_single_entries_mean_nothing():
    """A dimension of one entry may carry any stride; what reaches the kernels is that of a dense node."""
    import torch
    from nvfp4_decode_kernel.tree import _tree_tensor

    flat = torch.zeros(5000, dtype=torch.bfloat16)
    flat = flat[(-flat.data_ptr() % 16) // 2:]
    cpu = torch.device("cpu")
    for shape, strides, want in (
        ((1, 3, 2, 128), (1, 264, 128, 1), (256, 264)), ((3, 1, 2, 128), (512, 3, 128, 1), (512, 256)),
        ((1, 1, 1, 128), (7, 5, 3, 1), (128, 128)), ((2, 1, 2, 1, 128), (1024, 9, 136, 77, 1), (1024, 128, 136)),
    ):
        assert _tree_tensor(flat.as_strided(shape, strides), "x", shape, cpu)[1:] == want
    for shape, strides in (((2, 3, 2, 128), (771, 256, 128, 1)), ((1, 3, 2, 128), (8, 257, 128, 1))):
        with pytest.raises(ValueError):
            _tree_tensor(flat.as_strided(shape, strides), "x", shape, cpu)


def test_the_plugin_says_where_speculative_decoding_is():
    from nvfp4_vllm import guards
    from test_vllm_plugin import _config

    with pytest.raises(guards.UnsupportedConfigError, match="nvfp4_decode_kernel.tree"):
        guards.check_supported(_config(speculative_config=object()))


def test_sizes_past_32_bits_are_refused():
    """Query rows are counted in 32 bits: 64 nodes x 2^27 heads are none, or a tile of the wrong width."""
    import bdfp4
    from test_tree_cpu import _tree_args

    lib = bdfp4.library()
    for heads in (1 << 16, 1 << 26, 1 << 27, (1 << 31) - 1):
        assert lib.bdfp4_tree_workspace_bytes(1, 64, heads, 1) == 0
        a = _tree_args()
        a.heads_q, a.heads_kv, a.nodes, a.page_tokens = heads, 1, 64, 32
        assert lib.bdfp4_tree_decode(ctypes.byref(a), None) == bdfp4.E_UNSUPPORTED
    assert lib.bdfp4_tree_workspace_bytes(1, 64, 65535, 1) > 0


@pytest.mark.parametrize("rows,nodes,row,node,fine", [
    (2, 5, 5120, 1024, True), (2, 5, 1024, 2048, True), (2, 5, 0, 1024, False), (2, 5, 1024, 1024, False), (2, 5, 5120, 0, False),
    (2, 5, 4096, 1024, False), (1, 5, 8, 1024, True), (2, 1, 1024, 8, True), (2, 1, 1016, 8, False), (1, 1, 0, 0, True),
    (1, 5, 8, 1016, False), (3, 5, 1024, 2048, False),
])
def test_tree_output_has_its_own_elements(rows, nodes, row, node, fine):
    """Rows and nodes of the output that share memory would be written in any order. (The call's page size is one that is
    refused later, so none is launched.)"""
    import bdfp4
    from test_tree_cpu import _tree_args

    a = _tree_args()
    a.rows, a.nodes, a.out_row_stride, a.out_node_stride, a.page_tokens = rows, nodes, row, node, 32
    assert bdfp4.library().bdfp4_tree_decode(ctypes.byref(a), None) == (bdfp4.E_UNSUPPORTED if fine else bdfp4.E_ARG)
