"""Calls of the speculative-decoding operators at the edges of what their documentation allows."""

import pytest
import torch

from test_gpu_commit_drafts import _commit, _expect, _setup
from test_gpu_tree_decode import _call as _tree_call, _check as _tree_check, _inputs as _tree_inputs
from test_gpu_verify_drafts import _case as _verify_case, _check as _verify_check, _run as _verify_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page_tokens", [128, 64])
def test_commit_with_a_table_of_no_columns(page_tokens):
    """No row has a place for a page: a filled one is reported, and nothing is sealed wherever the allocator's
    recycled memory points."""
    import bdfp4

    s = _setup(3, 2, 6, 2, [126, 5, 250], [4, 3, 2], seed=61, page_tokens=page_tokens)
    before = [b.clone() for b in s["blocks"]]
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    for size in (3, 6, 12, 24):  # what the call's own buffers may be made of: valid page numbers
        torch.ones(size, dtype=torch.int32, device="cuda")
    tails, lengths = _commit(s, True, error=error, block_table=s["table"][:, :0].cuda())
    torch.cuda.synchronize()
    assert int(error) == bdfp4.DEV_BAD_PAGE
    assert all(torch.equal(a, b) for a, b in zip(s["blocks"], before))
    want_tails, _, want_lengths = _expect(s, True)
    for got, want in zip(tails, want_tails):
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    assert torch.stack([t.cpu() for t in lengths], 1).tolist() == [list(x) for x in want_lengths]
    # no row fills a page: nothing to report
    error.zero_()
    s["seq_lens"] = torch.tensor([100, 5, 200], dtype=torch.int32)
    _commit(s, True, error=error, block_table=s["table"][:, :0].cuda())
    assert int(error) == 0 and all(torch.equal(a, b) for a, b in zip(s["blocks"], before))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("drafter", [False, True])
def test_verify_clusters_that_start_one_by_one(dtype, drafter):
    """Rows of eight CTAs each while another stream's products keep every SM busy, so that the CTAs of a row start as
    places come free; every sum that crosses between them counts."""
    c = _verify_case(18, 5, 70000, dtype, drafter, seed=71)
    cuda = {k: None if v is None else v.cuda() for k, v in c.items()}
    want = _verify_run(cuda)
    _verify_check(c, want)
    busy, side = torch.randn(2048, 2048, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(side):
            for _ in range(4):
                busy @ busy
        for a, b in zip(_verify_run(cuda), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("nodes,heads", [(3, (4, 1)), (9, (8, 2)), (13, (8, 2)), (23, (8, 2)), (30, (8, 2))])
@pytest.mark.parametrize("rotate", [False, True])
def test_products_below_the_smallest_number(nodes, heads, rotate):
    """Queries, tail keys and draft keys of 2^-70: every score is zero to FP32, every token a node sees counts alike,
    and no masked one reaches it. (The tile widths of both kernels.)"""
    w, x = _tree_inputs([20, 300, 150], nodes, *heads, seed=72, rotate=rotate)
    w.tail_key.mul_(2.0 ** -70)
    tiny = dict(x, query=(x["query"].double() * 2.0 ** -70).to(torch.bfloat16),
                draft_key=(x["draft_key"].double() * 2.0 ** -70).to(torch.bfloat16))
    _tree_check(w, tiny, _tree_call(w, tiny, query_rotation="hadamard" if rotate else "none"), rotate=rotate)
