"""Host side of the speculative-decoding operators, no GPU needed: argument checks of the C entries and of the
Python functions, struct sizes, and the plain statements themselves on small cases."""

import ctypes
import subprocess
import tempfile
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import tree_oracle

ROOT = Path(__file__).resolve().parent.parent


def test_struct_sizes_match_the_header():
    import bdfp4

    source = ('#include <stdio.h>\n#include "bdfp4.h"\nint main(void){printf("%zu %zu %zu\\n", sizeof(bdfp4_tree_args), '
              "sizeof(bdfp4_verify_args), sizeof(bdfp4_commit_args));return 0;}\n")
    with tempfile.TemporaryDirectory() as tmp:
        (Path(tmp) / "sizes.c").write_text(source)
        subprocess.run(["gcc", "-I", str(ROOT / "include"), f"{tmp}/sizes.c", "-o", f"{tmp}/sizes"], check=True)
        sizes = [int(x) for x in subprocess.run([f"{tmp}/sizes"], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(t) for t in (bdfp4.TreeArgs, bdfp4.VerifyArgs, bdfp4.CommitArgs)]


def _tree_args():
    """A call every check accepts, with addresses that are never followed."""
    import bdfp4

    a = bdfp4.TreeArgs()
    a.rows, a.nodes, a.heads_q, a.heads_kv, a.pages, a.page_tokens = 2, 5, 8, 2, 4, 128
    for name in ("query", "draft_key", "draft_value", "parents", "key_codes", "key_scales", "value_codes", "value_scales",
                 "page_table", "seqused_fp4", "out", "workspace"):
        setattr(a, name, 1 << 20)
    a.query_row_stride, a.query_node_stride = 5 * 1024, 1024
    for side in ("key", "value"):
        setattr(a, f"draft_{side}_row_stride", 5 * 256)
        setattr(a, f"draft_{side}_node_stride", 256)
        setattr(a, f"{side}_codes_pitch", 2 * 128 * 2 * 72)
        setattr(a, f"{side}_scales_pitch", 2 * 128 * 2 * 72)
    a.parents_row_stride, a.page_table_stride, a.max_pages_per_row = 5, 2, 2
    a.softmax_scale = 0.1
    a.out_row_stride, a.out_node_stride = 5 * 1024, 1024
    a.workspace_bytes = 1 << 40
    return a


@pytest.mark.parametrize("change", [
    dict(rows=0), dict(nodes=0), dict(heads_q=7), dict(heads_kv=0), dict(query=0), dict(query=(1 << 20) + 2),
    dict(draft_key=0), dict(parents=0), dict(out=0), dict(key_codes=0), dict(pages=0), dict(page_table=0),
    dict(page_table_stride=1), dict(max_pages_per_row=-1), dict(key_codes_pitch=128 * 64), dict(value_scales_pitch=24),
    dict(query_node_stride=1027), dict(out_node_stride=1000), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")),
    dict(key_tensor_scale=-1.0), dict(value_tensor_scale=float("inf")), dict(tail_key=1 << 20), dict(workspace=0),
    dict(workspace=(1 << 20) + 8), dict(workspace_bytes=0), dict(key_shift=4), dict(draft_value_row_stride=-8),
])
def test_tree_entry_refuses(change):
    import bdfp4

    a = _tree_args()
    for name, value in change.items():
        setattr(a, name, value)
    assert bdfp4.library().bdfp4_tree_decode(ctypes.byref(a), None) == bdfp4.E_ARG


def test_unsupported_requests_and_null_structs():
    import bdfp4

    lib = bdfp4.library()
    a = _tree_args()
    a.nodes = 65
    assert lib.bdfp4_tree_decode(ctypes.byref(a), None) == bdfp4.E_UNSUPPORTED
    a = _tree_args()
    a.page_tokens = 32
    assert lib.bdfp4_tree_decode(ctypes.byref(a), None) == bdfp4.E_UNSUPPORTED
    for entry in (lib.bdfp4_tree_decode, lib.bdfp4_verify_drafts, lib.bdfp4_commit_drafts):
        assert entry(None, None) == bdfp4.E_ARG
    assert lib.bdfp4_tree_workspace_bytes(1, 65, 8, 2) == 0 and lib.bdfp4_tree_workspace_bytes(1, 5, 7, 2) == 0
    assert lib.bdfp4_tree_workspace_bytes(1, 5, 8, 2) > 0
    v = bdfp4.VerifyArgs()
    v.rows, v.nodes, v.vocab = 1, 65, 10
    assert lib.bdfp4_verify_drafts(ctypes.byref(v), None) == bdfp4.E_UNSUPPORTED
    v.nodes = 4
    assert lib.bdfp4_verify_drafts(ctypes.byref(v), None) == bdfp4.E_ARG  # no tensors
    c = bdfp4.CommitArgs()
    c.layers, c.rows, c.nodes, c.heads_kv = 1, 1, 4, 2
    assert lib.bdfp4_commit_drafts(ctypes.byref(c), None) == bdfp4.E_ARG
    c.nodes = 65
    assert lib.bdfp4_commit_drafts(ctypes.byref(c), None) == bdfp4.E_UNSUPPORTED


def test_python_functions_refuse_cpu_tensors():
    from nvfp4_decode_kernel import tree

    x = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        tree.tree_decode(x, x, x, torch.zeros(1, 2, dtype=torch.int32), x, x, x, x, x, x)
    with pytest.raises(ValueError):
        tree.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32),
                           torch.zeros(1, 2))
    with pytest.raises(ValueError):
        tree.DraftCommitter(tail_key=torch.zeros(1, 1, 144, 2, 128), tail_value=torch.zeros(1, 1, 144, 2, 128))


def test_ancestors():
    seen = tree_oracle.ancestors([-1, 0, 0, 1, 3, 9, 5])
    assert [torch.nonzero(s)[:, 0].tolist() for s in seen] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [5], [5, 6]]


def test_walk_by_hand():
    """p accepts token 1 with probability 0.5 and token 2 with 0.3 / 0.5 after that; q halves the chance."""
    p = np.array([[0.2, 0.5, 0.3], [0.0, 0.0, 1.0], [0.6, 0.2, 0.2]])
    parents, tokens = [-1, 0, 0], [0, 1, 2]
    assert tree_oracle.verify(p, tokens, parents, [0.0, 0.4, 0.9])[:2] == ([0, 1], 2)
    assert tree_oracle.verify(p, tokens, parents, [0.7, 0.6, 0.5])[:2] == ([0, 2], 1)
    assert tree_oracle.verify(p, tokens, parents, [0.9, 0.6, 0.7])[:2] == ([0], 0)
    q = np.array([[0.1, 0.8, 0.1]] * 3)
    # 0.7 * 0.8 > 0.5: refused, w = (0.1, 0, 0.2), W = 0.3; then 0.9 * 0.1 * 0.3 < 0.2: taken
    assert tree_oracle.verify(p, tokens, parents, [0.5, 0.7, 0.9], q)[:2] == ([0, 2], 0)


def test_tree_attention_agrees_with_one_token_attention():
    """A single node over a tail only is plain attention over the tail and itself."""
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 2, 128, generator=gen).to(torch.bfloat16) for _ in range(3))
    tail_k, tail_v = (torch.randn(144, 2, 128, generator=gen).to(torch.bfloat16) for _ in range(2))
    out, allowed = tree_oracle.tree_attention(
        query=q, draft_key=k, draft_value=v, parents=[-1], key=None, value=None, page_ids=None, fp4=0, tail_key=tail_k,
        tail_value=tail_v, residual=30, sink=0, softmax_scale=128 ** -0.5)
    for h in range(2):
        keys = torch.cat([tail_k[:30, h], k[:, h]]).double()
        values = torch.cat([tail_v[:30, h], v[:, h]]).double()
        want = torch.softmax(q[0, h].double() @ keys.T * 128 ** -0.5, 0) @ values
        assert torch.allclose(out[0, h], want, rtol=1e-12, atol=1e-12)
    assert float((allowed / (out.abs() + 1)).max()) < 0.05
