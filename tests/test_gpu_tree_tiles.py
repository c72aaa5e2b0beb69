"""Tree attention at every width of a tile and where its work is cut: units that end next to a cut, units of many
parts, rows of nothing but drafts, and launches of fewer steps than CTAs."""

import pytest
import torch

from test_gpu_tree_decode import _call, _check, _inputs

pytestmark = pytest.mark.gpu


# query rows per KV head: on and next to the widths 16, 32, 64, 96 and 128, and several tiles
@pytest.mark.parametrize("page_tokens", [128, 64])
@pytest.mark.parametrize("nodes,ratio", [(16, 1), (17, 1), (8, 4), (11, 3), (64, 1), (13, 5), (24, 4), (49, 2), (64, 2),
                                         (43, 3), (61, 5)])
def test_tile_widths(page_tokens, nodes, ratio):
    w, x = _inputs([1, 15, 131, 640, 897, 1408], nodes, 2 * ratio, 2, seed=nodes, page_tokens=page_tokens)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("nodes,ratio", [(5, 4), (20, 4), (50, 2)])
def test_rotated_and_shifted_over_many_steps(nodes, ratio):
    gen = torch.Generator().manual_seed(nodes)
    shift = 0.3 * torch.randn(2, 128, generator=gen)
    w, x = _inputs([7000, 300, 4223], nodes, 2 * ratio, 2, seed=nodes)
    out = _call(w, x, query_rotation="hadamard", key_shift=shift.cuda())
    _check(w, x, out, rotate=True, shift=shift)


# the launch's steps over 296 CTAs (148 for wide tiles): below one each, just above, and with units a step or two
# longer or shorter than a CTA's share
@pytest.mark.parametrize("nodes", [3, 16])
@pytest.mark.parametrize("rows,length", [(1, 40), (3, 300), (74, 200), (75, 330), (37, 1000), (40, 900)])
def test_cuts(rows, length, nodes):
    lens = [max(1, length + 128 * ((r * 7) % 3 - 1)) for r in range(rows)]
    w, x = _inputs(lens, nodes, 8, 2, seed=rows)
    _check(w, x, _call(w, x), rows=range(0, rows, max(1, rows // 9)))


@pytest.mark.parametrize("nodes", [4, 40])
def test_rows_of_nothing_but_drafts(nodes):
    w, x = _inputs([130, 1, 257], nodes, 8, 2, seed=5)
    for lengths in (w.seqused_fp4, w.seqused_residual, w.seqused_sink):
        lengths.zero_()
    _check(w, x, _call(w, x))


def test_one_workspace_for_calls_in_turn():
    """Calls one after the other on a stream may share a workspace, whatever their sizes and kernels."""
    from nvfp4_decode_kernel import tree

    cases = [_inputs([900, 70, 2049], nodes, 8, 2, seed=nodes) for nodes in (2, 40, 7, 64)]
    alone = [_call(w, x) for w, x in cases]
    size = max(tree.tree_workspace_bytes(3, x["query"].shape[1], 8, 2) for _, x in cases)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(0xFF)
    for _ in range(2):
        for (w, x), want in zip(cases, alone):
            assert torch.equal(_call(w, x, workspace=workspace), want)
