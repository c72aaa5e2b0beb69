"""What the checks of the tree attention's long rows can see: a result that lacks a page, the tail, the sink or an
ancestor, takes a wrong page, or sees what it may not, must lie outside the tolerance at every length they use."""

import pytest
import torch

from oracle import tree_oracle as oracle

HEADS, RATIO = 1, 2


def _row(tokens, nodes, rotate, seed):
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    fp4 = (tokens - 1) // 128 * 128
    outliers = torch.ones(128)
    outliers[torch.randperm(128, generator=gen)[:4]] = torch.exp(1.5 * randn(4))
    pages = fp4 // 128 + 1
    parents = (torch.rand(nodes, generator=gen) * torch.arange(nodes)).to(torch.int32).tolist()
    return dict(
        query=randn(nodes, HEADS * RATIO, 128).to(torch.bfloat16), draft_key=randn(nodes, HEADS, 128).to(torch.bfloat16),
        draft_value=randn(nodes, HEADS, 128).to(torch.bfloat16), parents=[-1] + parents[1:],
        key=(randn(pages, 128, HEADS, 128) * outliers).double(), value=randn(pages, 128, HEADS, 128).double(),
        page_ids=torch.arange(fp4 // 128), fp4=fp4, tail_key=(randn(144, HEADS, 128) * outliers).to(torch.bfloat16),
        tail_value=randn(144, HEADS, 128).to(torch.bfloat16), residual=tokens - fp4, sink=16,
        softmax_scale=128 ** -0.5, rotate=rotate)


@pytest.mark.parametrize("tokens,nodes,rotate", [(20000, 4, False), (20000, 40, False), (33001, 1, False), (7000, 16, True),
                                                 (2900, 6, False)])
def test_what_is_missing_is_seen(tokens, nodes, rotate):
    row = _row(tokens, nodes, rotate, seed=tokens + nodes)
    want, typical = oracle.tree_attention(**row, typical=True)

    def seen(**change):
        got = oracle.tree_attention(**{**row, **change})[0]
        return oracle.outside_typical(got, want, typical)

    assert not seen()
    assert oracle.outside_typical(want.to(torch.bfloat16).double(), want, typical) == 0
    pages = row["fp4"] // 128
    ids = row["page_ids"]
    assert oracle.outside_typical(torch.zeros_like(want), want, typical)
    assert seen(page_ids=torch.cat([ids[:pages // 2], ids[pages // 2 + 1:]]), fp4=row["fp4"] - 128)
    wrong = ids.clone()
    wrong[pages // 3] = pages
    assert seen(page_ids=wrong)
    if row["residual"] >= 32:
        assert seen(residual=0)
    # a node's few ancestors among thousands of tokens are below any rounding; a chain of all nodes in their place is not
    # (the tests that ask for single tokens see both)
    if nodes >= 16:
        assert seen(parents=list(range(-1, nodes - 1)))
