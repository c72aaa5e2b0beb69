"""Calls of the speculative-decoding operators at the edges of what their documentation allows."""

import pytest
import torch

from test_gpu_commit_drafts import _commit, _expect, _setup

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
