"""Verification of drafted trees against the 64-bit walk: whole numbers, equal in every entry. Inputs whose
decisions lie within 1e-9 of a border (where FP64 sums of another order may decide otherwise) would be skipped;
the seeds below have none."""

import math

import numpy as np
import pytest
import torch

from oracle import tree_oracle as oracle

pytestmark = pytest.mark.gpu


def _case(rows, nodes, vocab, dtype=torch.float32, drafter=False, seed=0, sharp=3.0, tree="random"):
    gen = torch.Generator().manual_seed(seed)
    logits = sharp * torch.randn(rows, nodes, vocab, generator=gen)
    target = torch.softmax(logits, -1).to(dtype)
    idea = torch.softmax(logits + 0.6 * torch.randn(rows, nodes, vocab, generator=gen), -1)
    parents = (torch.rand(rows, nodes, generator=gen) * torch.arange(nodes).clamp(max=6)).to(torch.int32)
    parents = (torch.arange(nodes) - 1 - parents).clamp(min=0).to(torch.int32)
    if tree == "star":
        parents.zero_()
    if tree == "chain":
        parents = torch.arange(-1, nodes - 1, dtype=torch.int32).expand(rows, nodes).contiguous()
    parents[:, 0] = -1
    tokens = torch.zeros(rows, nodes, dtype=torch.int32)
    for i in range(1, nodes):
        p = idea[torch.arange(rows), parents[:, i].long()]
        tokens[:, i] = torch.multinomial(p, 1, generator=gen)[:, 0].to(torch.int32)
    return dict(target=target, tokens=tokens, parents=parents, uniforms=torch.rand(rows, nodes, generator=gen),
                draft=idea.to(dtype) if drafter else None)


def _run(c, counts=None, **more):
    from nvfp4_decode_kernel import tree

    cuda = {k: None if v is None else v.cuda() for k, v in c.items()}
    return tree.verify_drafts(cuda["target"], cuda["tokens"], cuda["parents"], cuda["uniforms"], draft_probs=cuda["draft"],
                              node_counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"),
                              **more)


def _check(c, verdict, counts=None):
    rows, nodes, _ = c["target"].shape
    accepted, number, token = (t.cpu() for t in verdict)
    lengths = []
    for r in range(rows):
        path, want, margin = oracle.verify(
            c["target"][r].float().numpy(), c["tokens"][r].numpy(), c["parents"][r].numpy(), c["uniforms"][r].numpy(),
            None if c["draft"] is None else c["draft"][r].float().numpy(), None if counts is None else counts[r])
        assert margin > 1e-9, "an input next to a border: choose another seed"
        assert accepted[r].tolist() == path + [-1] * (nodes - len(path)), f"row {r}"
        assert int(number[r]) == len(path) and int(token[r]) == want, f"row {r}"
        lengths.append(len(path))
    return lengths


@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 31, 128, 1000, 4099, 50001, 70000])
def test_vocabularies(drafter, dtype, vocab):
    c = _case(3, 5, vocab, dtype, drafter, seed=vocab)
    _check(c, _run(c))


@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("nodes", [1, 2, 32, 33, 64])
@pytest.mark.parametrize("tree", ["random", "star", "chain"])
def test_trees(drafter, nodes, tree):
    c = _case(9, nodes, 300, torch.float32, drafter, seed=nodes + 7 * drafter, sharp=1.5, tree=tree)
    _check(c, _run(c))


def test_paths_of_every_length():
    """Sharp targets accept whole chains, and the refusals fall everywhere."""
    c = _case(40, 12, 64, torch.float32, True, seed=5, sharp=8.0, tree="chain")
    assert len(set(_check(c, _run(c)))) >= 6


@pytest.mark.parametrize("drafter", [False, True])
def test_many_rows(drafter):
    c = _case(300, 4, 5000, torch.float32, drafter, seed=6)
    _check(c, _run(c))


@pytest.mark.parametrize("drafter", [False, True])
def test_node_counts(drafter):
    counts = [0, 1, 2, 9, 5]
    c = _case(5, 9, 800, torch.float32, drafter, seed=8, sharp=6.0)
    c["parents"][2, 2:] = 0
    c["tokens"][2, 2:] = -5
    _check(c, _run(c, counts), counts)


def test_certain_and_impossible_tokens():
    """One-hot targets, a drafter that agrees exactly, refused siblings with one token, tokens outside the
    vocabulary, rows without any weight, uniforms of zero and next to one."""
    vocab, nodes = 40, 6
    c = _case(7, nodes, vocab, seed=9, tree="star")
    c["draft"] = c["target"].clone()
    c["target"][0] = 0.0
    c["target"][0, :, 11] = 1.0  # greedy: only token 11 can be taken
    c["tokens"][0] = torch.tensor([0, 3, 3, 11, 11, 5])
    c["draft"][0] = 1.0 / vocab
    c["tokens"][1] = torch.tensor([0, 4, 4, 4, 4, 4])
    c["tokens"][2] = torch.tensor([0, -1, vocab, 1 << 30, -7, 2])
    c["target"][3] = 0.0
    c["uniforms"][4] = 0.0
    c["uniforms"][5] = math.nextafter(1.0, 0.0)
    c["target"][6, 0] = 0.0
    c["target"][6, 0, vocab - 1] = 1.0
    c["tokens"][6] = 0
    c["uniforms"][6, 0] = float(np.nextafter(np.float32(1), np.float32(0)))
    for draft in (c["draft"], None):
        d = dict(c, draft=draft)
        verdict = _run(d)
        rows = range(7)
        accepted, number, token = (t.cpu() for t in verdict)
        for r in rows:
            path, want, _ = oracle.verify(d["target"][r].numpy(), d["tokens"][r].numpy(), d["parents"][r].numpy(),
                                          d["uniforms"][r].numpy(), None if draft is None else draft[r].numpy())
            assert accepted[r].tolist() == path + [-1] * (nodes - len(path)), f"row {r}"
            assert (int(number[r]), int(token[r])) == (len(path), want), f"row {r}"
        assert accepted[0].tolist()[:2] == [0, 3] and int(token[6]) == vocab - 1


def test_nan_probabilities_stay_in_range():
    c = _case(2, 4, 500, seed=10)
    c["target"][0] = float("nan")
    accepted, number, token = (t.cpu() for t in _run(c))
    assert 0 <= int(token[0]) < 500 and 1 <= int(number[0]) <= 4
    path, want, _ = oracle.verify(c["target"][1].numpy(), c["tokens"][1].numpy(), c["parents"][1].numpy(), c["uniforms"][1].numpy())
    assert int(number[1]) == len(path) and int(token[1]) == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_inputs(dtype):
    """A vocabulary padded behind its end, nodes taken out of a wider buffer, rows at any alignment."""
    c = _case(3, 5, 1003, dtype, True, seed=12)
    wide = torch.full((3, 7, 1010), 0.5, dtype=dtype, device="cuda")
    wide2 = torch.full((3, 6, 1021), 0.5, dtype=dtype, device="cuda")
    wide[:, 1:6, 3:1006] = c["target"].cuda()
    wide2[:, :5, 1:1004] = c["draft"].cuda()
    tokens = torch.zeros(3, 9, dtype=torch.int32, device="cuda")
    tokens[:, :5] = c["tokens"].cuda()
    d = dict(c, target=wide[:, 1:6, 3:1006], draft=wide2[:, :5, 1:1004], tokens=tokens[:, :5])
    _check(c, _run(d))


def test_tokens_follow_the_target():
    """20,000 rows of one tree: whatever the drafter proposed, the first token behind the root is distributed as
    the target's. Chi-square over 8 tokens: the 1e-6 quantile at 7 degrees of freedom is 40.5."""
    rows, vocab, nodes = 20000, 8, 4
    gen = torch.Generator().manual_seed(14)
    p = torch.softmax(torch.randn(vocab, generator=gen), 0)
    q = torch.softmax(torch.randn(vocab, generator=gen), 0)
    for drafter in (True, False):
        tokens = torch.zeros(rows, nodes, dtype=torch.int32)
        drawn = torch.multinomial(q, rows * 3, replacement=True, generator=gen).view(rows, 3)
        tokens[:, 1:] = drawn if drafter else torch.tensor([2, 5, 1])
        c = dict(target=p.expand(rows, nodes, vocab).contiguous(), tokens=tokens,
                 parents=torch.tensor([-1, 0, 0, 0], dtype=torch.int32).expand(rows, nodes).contiguous(),
                 uniforms=torch.rand(rows, nodes, generator=gen),
                 draft=q.expand(rows, nodes, vocab).contiguous() if drafter else None)
        accepted, number, token = (t.cpu() for t in _run(c))
        first = torch.where(number > 1, tokens.gather(1, accepted[:, 1:2].clamp(min=0).long())[:, 0], token)
        seen = torch.bincount(first.long(), minlength=vocab).double()
        expected = p.double() * rows
        assert float(((seen - expected) ** 2 / expected).sum()) < 40.5


def test_repeatable_and_captured():
    from nvfp4_decode_kernel import tree

    c = _case(6, 16, 20001, torch.float32, True, seed=15)
    cuda = {k: v.cuda() for k, v in c.items()}
    first = _run(c)
    out = tree.DraftVerdict(*(torch.zeros_like(t) for t in first))

    def call():
        return tree.verify_drafts(cuda["target"], cuda["tokens"], cuda["parents"], cuda["uniforms"],
                                  draft_probs=cuda["draft"], out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, out):
        assert torch.equal(a, b)


def test_refusals():
    c = _case(2, 4, 100, seed=16)
    good = {k: v for k, v in c.items()}

    def refused(error=ValueError, counts=None, **change):
        with pytest.raises(error):
            _run(dict(good, **change), counts)

    refused(target=c["target"].half())
    refused(target=c["target"].cuda()[..., ::2])
    refused(target=c["target"][0])
    refused(draft=c["target"].bfloat16())
    refused(draft=c["target"][..., :50])
    refused(tokens=c["tokens"].long())
    refused(tokens=c["tokens"][:, :3])
    refused(parents=c["parents"][:1])
    refused(uniforms=c["uniforms"].double())
    refused(counts=[1])
    refused(NotImplementedError, **{k: None if v is None else v.repeat_interleave(17, 1) for k, v in c.items()})
