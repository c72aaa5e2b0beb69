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


def _needles(w, nodes, heads_q, seed, loud):
    """Inputs whose every query asks for one token: along that token's key, with the workload's outlier channels evened
    out, so that its score stands far above all others. Query by query the token lies in the pages (spread over them),
    the tail, the sink, among the node's ancestors. Returns the inputs and the values asked for."""
    from oracle import tree_oracle as oracle
    from test_gpu_tree_decode import _trees

    gen = torch.Generator().manual_seed(seed)
    rows, heads = w.rows, w.heads_kv
    even = w.outlier_scale.cpu().double() ** -2
    x = dict(draft_key=(torch.randn(rows, nodes, heads, 128, generator=gen) * w.outlier_scale.cpu()).to(torch.bfloat16),
             draft_value=torch.randn(rows, nodes, heads, 128, generator=gen).to(torch.bfloat16),
             parents=_trees(rows, nodes, gen))
    key, value = oracle.cache_values(w.blocks, heads, w.page_tokens)
    query = torch.zeros(rows, nodes, heads_q, 128, dtype=torch.bfloat16)
    want = torch.zeros(rows, nodes, heads_q, 128, dtype=torch.float64)
    for r in range(rows):
        fp4, residual, sink = (int(t[r]) for t in (w.seqused_fp4, w.seqused_residual, w.seqused_sink))
        ids = w.page_table[r, :fp4 // w.page_tokens].cpu().long()
        tail_key, tail_value = w.tail_key[0, r].cpu().double(), w.tail_value[0, r].cpu().double()
        k = torch.cat([key[ids].reshape(-1, heads, 128), tail_key[:residual], tail_key[128:128 + sink], x["draft_key"][r].double()])
        v = torch.cat([value[ids].reshape(-1, heads, 128), tail_value[:residual], tail_value[128:128 + sink],
                       x["draft_value"][r].double()])
        first = [0, fp4, fp4 + residual, fp4 + residual + sink]
        cached = torch.ones(first[3], dtype=torch.bool)
        cached[:sink] = False
        cached[first[2]:] = True
        asked = []  # (node, head, token)
        for i, family in enumerate(oracle.ancestors(x["parents"][r].tolist())):
            for h in range(heads_q):
                n = i * heads_q + h
                choices = [torch.nonzero(cached[a:b])[:, 0] + a for a, b in zip(first, first[1:])] + [torch.nonzero(family)[:, 0] + first[3]]
                part = choices[(n + r) % 4]
                if not len(part):
                    part = choices[3]
                spread = (n * 0.6180339887) % 1.0
                asked.append((i, h, int(part[int(spread * len(part))]), family))
        for i, h, t, family in asked:
            kv = h * heads // heads_q
            direction = loud * k[t, kv] * even[kv]
            query[r, i, h] = direction.to(torch.bfloat16)
            want[r, i, h] = v[t, kv]
            score = query[r, i, h].double() @ k[:, kv].T * 128 ** -0.5 * 1.4427
            score[:first[3]][~cached] = -float("inf")
            score[first[3]:][~family] = -float("inf")
            best = float(score[t])
            score[t] = -float("inf")
            assert best - float(score.max()) > 40 + 0.05 * best, "an input that does not single out its token: choose another"
    return dict(x, query=query), want


def _check_needles(got, want):
    # the token's probability is rounded to BF16 at most (2^-8) against a sum that is not, and so is the result
    assert bool(((got.cpu().double() - want).abs() <= 1.05 * 2.0 ** -7 * want.abs() + 1e-6).all())


@pytest.mark.parametrize("nodes,heads", [(3, (4, 1)), (9, (6, 2)), (13, (8, 2)), (23, (8, 2)), (30, (8, 2))])
@pytest.mark.parametrize("factor", [1.0, 2.0 ** 22, 2.0 ** 60, 2.0 ** 100])
def test_scores_beyond_the_fraction_of_a_float(nodes, heads, factor):
    """Scores whose rounding is larger than any difference that FP16's exponents can hold: the token with the highest
    one is still the answer."""
    w, _ = _tree_inputs([700, 130, 20, 1300], 1, *heads, seed=74)
    x, want = _needles(w, nodes, heads[0], 75, 16.0 * factor)
    _check_needles(_tree_call(w, x), want)


@pytest.mark.parametrize("nodes,heads", [(3, (4, 1)), (9, (6, 2)), (13, (8, 2)), (23, (8, 2)), (30, (8, 2))])
@pytest.mark.parametrize("factor", [2.0 ** 10, 2.0 ** 20, 2.0 ** 60])
@pytest.mark.parametrize("rotate", [False, True])
def test_a_loud_query_leaves_the_others_alone(nodes, heads, factor, rotate):
    """One node, and one head of another, far louder than the rest of their tile: what is lost of a query goes by its
    own values (the allowance's terms are each query's own), not by the loudest."""
    w, x = _tree_inputs([700, 130, 20], nodes, *heads, seed=73, loud=4.0, rotate=rotate)
    loud = x["query"].double()
    loud[:, 1] *= factor
    loud[:, 2, -1] *= factor
    loud = dict(x, query=loud.to(torch.bfloat16))
    _tree_check(w, loud, _tree_call(w, loud, query_rotation="hadamard" if rotate else "none"), rotate=rotate)


@pytest.mark.parametrize("page_tokens", [128, 64])
@pytest.mark.parametrize("trusted", [False, True])
def test_tree_with_a_table_of_no_columns(page_tokens, trusted):
    """A batch whose rows have no page yet, the first steps of every sequence."""
    w, x = _tree_inputs([1, 20, 128], 5, 8, 2, seed=76, page_tokens=page_tokens)
    assert not bool(w.seqused_fp4.any())
    w.page_table = w.page_table[:, :0]
    _tree_check(w, x, _tree_call(w, x, trusted_metadata=trusted))


@pytest.mark.parametrize("rows,nodes", [(1, 1), (1, 4), (3, 1)])
def test_single_entries_of_any_stride(rows, nodes):
    """What broadcasting, slicing and transposing leave behind in dimensions of one entry."""
    def odd(t):  # every single entry's stride a 3
        return t.as_strided(t.shape, [3 if size == 1 and i < t.ndim - 1 else stride
                                      for i, (size, stride) in enumerate(zip(t.shape, t.stride()))])

    w, x = _tree_inputs([200, 20, 700][:rows], nodes, 4, 2, seed=77)
    want = _tree_call(w, x)
    device = {k: odd(v.cuda()) for k, v in x.items()}
    w.page_table = odd(w.page_table)
    w.tail_key, w.tail_value = w.tail_key.contiguous(), w.tail_value.contiguous()
    got = _tree_call(w, device, residual_key_pages_bf16=odd(w.tail_key[0]), residual_value_pages_bf16=odd(w.tail_value[0]),
                     out=odd(torch.zeros_like(want)))
    assert torch.equal(got, want)
    s = _setup(rows, 1, nodes, 2, [126, 5, 250][:rows], [1] * rows, seed=78)
    tails, lengths = _commit(s, True)
    s = dict(s, **{k: _Held(odd(s[k].cuda())) for k in ("key", "value", "accepted", "table")})
    again, others = _commit(s, True)
    assert all(torch.equal(a, b) for a, b in zip(tails, again))
    assert all(torch.equal(a, b) for a, b in zip(lengths, others))


class _Held:
    """A stand-in whose ``.cuda()`` hands out the tensor as it is, strides and all."""

    def __init__(self, t):
        self.t = t

    def cuda(self):
        return self.t


@pytest.mark.parametrize("sink", [0, 1, 4, 15])
@pytest.mark.parametrize("nodes", [3, 20])
def test_what_a_commit_with_a_short_sink_left(sink, nodes):
    """The lengths and tails of a committer with any sink are what the next step's attention takes."""
    from nvfp4_decode_kernel import tree
    from oracle import tree_oracle as oracle

    lens, counts = [0, 2, 100], [3, 3, 2]
    s = _setup(3, 1, 6, 2, lens, counts, seed=79, sink=sink, seal=False, shift=False)
    tails, lengths = _commit(s, False, sink=sink)
    w, x = _tree_inputs([1, 1, 1], nodes, 8, 2, seed=80)
    device = {k: v.cuda() for k, v in x.items()}
    for trusted in (False, True):
        out = tree.tree_decode(
            device["query"], device["draft_key"], device["draft_value"], device["parents"], *w.regions, w.page_table,
            lengths.seqused_fp4, residual_key_pages_bf16=tails[0][0], residual_value_pages_bf16=tails[1][0],
            residual_page_ids=s["row_to_slot"].cuda(), seqused_residual=lengths.seqused_residual,
            seqused_sink=lengths.seqused_sink, trusted_metadata=trusted).cpu().double()
        for r in range(3):
            n, slot = lens[r] + counts[r], int(s["row_to_slot"][r])
            want, allowed = oracle.tree_attention(
                query=x["query"][r], draft_key=x["draft_key"][r], draft_value=x["draft_value"][r],
                parents=x["parents"][r].tolist(), key=None, value=None, page_ids=None, fp4=0,
                tail_key=tails[0][0, slot].cpu(), tail_value=tails[1][0, slot].cpu(), residual=n, sink=min(n, sink),
                softmax_scale=128 ** -0.5)
            assert bool(((out[r] - want).abs() <= allowed).all()), f"row {r}"
    # a sink length beyond the rows there are is refused, and never followed
    args = (device["query"], device["draft_key"], device["draft_value"], device["parents"], *w.regions, w.page_table,
            lengths.seqused_fp4)
    more = dict(residual_key_pages_bf16=tails[0][0], residual_value_pages_bf16=tails[1][0],
                residual_page_ids=s["row_to_slot"].cuda(), seqused_residual=lengths.seqused_residual)
    with pytest.raises(ValueError):
        tree.tree_decode(*args, **more, seqused_sink=lengths.seqused_sink + sink + 1)
    over = tree.tree_decode(*args, **more, seqused_sink=torch.full_like(lengths.seqused_sink, 16), trusted_metadata=True)
    full = tree.tree_decode(*args, **more, seqused_sink=torch.full_like(lengths.seqused_sink, sink), trusted_metadata=True)
    assert torch.equal(over, full)


def test_a_commit_ends_at_a_number_that_is_no_node():
    """The row grows by what was written; nothing of the entries behind is, valid ones included, and it is reported."""
    import bdfp4

    s = _setup(4, 2, 40, 2, [10, 126, 126, 300], [5, 6, 38, 40], seed=81)
    s["accepted"][1, 1] = 40
    s["accepted"][2, 35] = -4
    s["accepted"][3, 0] = 1 << 30
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = [b.clone() for b in s["blocks"]]
    tails, lengths = _commit(s, True, error=error)
    assert int(error) == bdfp4.DEV_BAD_NODE
    cut = dict(s, counts=torch.tensor([5, 1, 35, 0], dtype=torch.int32))
    want_tails, sealed, want_lengths = _expect(cut, True)
    for got, want in zip(tails, want_tails):
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    assert torch.stack([t.cpu() for t in lengths], 1).tolist() == [list(x) for x in want_lengths]
    for block, old in zip(s["blocks"], before):
        assert (block != old).any(1).nonzero()[:, 0].tolist() == sorted(int(s["table"][r, c]) for r, c, _ in sealed)


def test_outputs_that_share_memory_are_refused():
    w, x = _tree_inputs([20, 300], 3, 4, 2, seed=82)
    want = _tree_call(w, x)
    for out in (torch.zeros(1, 3, 4, 128).expand(2, 3, 4, 128), torch.zeros(2, 1, 4, 128).expand(2, 3, 4, 128),
                torch.zeros(4096).as_strided((2, 3, 4, 128), (1024, 512, 128, 1))):
        with pytest.raises(ValueError):
            _tree_call(w, x, out=out.to(torch.bfloat16).cuda() if out.is_contiguous() else _like(out))
    by_node = torch.zeros(3, 2, 4, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(_tree_call(w, x, out=by_node), want)


def _like(t):
    return torch.zeros(4096, dtype=torch.bfloat16, device="cuda").as_strided(t.shape, t.stride())


def test_what_is_no_tensor_is_refused_as_such():
    from nvfp4_decode_kernel import tree

    w, x = _tree_inputs([20, 300], 3, 4, 2, seed=83)
    device = {k: v.cuda() for k, v in x.items()}
    args = [device["query"], device["draft_key"], device["draft_value"], device["parents"], *w.regions, w.page_table, w.seqused_fp4]
    tail = dict(residual_key_pages_bf16=w.tail_key[0], residual_value_pages_bf16=w.tail_value[0],
                residual_page_ids=w.slot_ids, seqused_residual=w.seqused_residual)
    for at in range(len(args)):
        with pytest.raises(ValueError):
            tree.tree_decode(*args[:at], None, *args[at + 1:], **tail)
    for name in (*tail, "key_shift", "workspace", "out", "node_counts", "seqused_sink", "error_word"):
        with pytest.raises(ValueError):
            tree.tree_decode(*args, **{**tail, name: [1]})
    probs, tokens = torch.full((2, 3, 8), 0.125, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(2, 3, device="cuda")
    for change in (dict(tokens=None), dict(parents=[0]), dict(uniforms=None), dict(draft_probs=[1])):
        with pytest.raises(ValueError):
            tree.verify_drafts(**{**dict(target_probs=probs, tokens=tokens, parents=tokens, uniforms=uniforms), **change})
    s = _setup(2, 1, 3, 2, [3, 4], [2, 2], seed=84)
    key, value = s["tail_key"].cuda(), s["tail_value"].cuda()
    for change in (dict(tail_value=None), dict(key_shift=[0.0])):
        with pytest.raises(ValueError):
            tree.DraftCommitter(**{**dict(tail_key=key, tail_value=value), **change})
    with pytest.raises(ValueError):
        _commit(s, True, block_table=[1])
