"""Attention of a drafted tree over the FP4 cache against its 64-bit statement, at the sizes, masks and layouts
where it can go wrong. The allowance per element is derived in ``oracle/tree_oracle.py``."""

import pytest
import torch

from oracle import tree_oracle as oracle

pytestmark = pytest.mark.gpu


def _trees(rows, nodes, gen, kind="random"):
    if kind == "chain":
        return torch.arange(-1, nodes - 1, dtype=torch.int32).expand(rows, nodes).contiguous()
    if kind == "roots":
        return torch.full((rows, nodes), -1, dtype=torch.int32)
    if kind == "star":
        parents = torch.zeros(rows, nodes, dtype=torch.int32)
        parents[:, 0] = -1
        return parents
    parents = (torch.rand(rows, nodes, generator=gen) * torch.arange(nodes)).to(torch.int32)
    parents[:, 0] = -1
    return parents


def _inputs(lens, nodes, heads_q, heads_kv, seed=0, tree="random", sink=16, loud=1.0, **cache):
    from bdfp4.workload import build_workload

    w = build_workload(rows=len(lens), heads_q=heads_q, heads_kv=heads_kv, seq_lens=lens, sink_tokens=sink, seed=seed, **cache)
    gen = torch.Generator().manual_seed(seed + 1)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    return w, dict(query=(loud * randn(len(lens), nodes, heads_q, 128)).to(torch.bfloat16),
                   draft_key=randn(len(lens), nodes, heads_kv, 128).to(torch.bfloat16),
                   draft_value=randn(len(lens), nodes, heads_kv, 128).to(torch.bfloat16),
                   parents=_trees(len(lens), nodes, gen, tree))


def _call(w, inputs, **more):
    from nvfp4_decode_kernel import tree

    args = dict(residual_key_pages_bf16=w.tail_key[0], residual_value_pages_bf16=w.tail_value[0],
                residual_page_ids=w.slot_ids, seqused_residual=w.seqused_residual,
                seqused_sink=w.seqused_sink if w.sink_tokens else None)
    args.update(more)
    device = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in inputs.items()}
    return tree.tree_decode(device["query"], device["draft_key"], device["draft_value"], device["parents"], *w.regions,
                            w.page_table, w.seqused_fp4, **args)


def _check(w, inputs, out, counts=None, rotate=False, shift=None, scale=128 ** -0.5, tail=True, rows=None):
    key, value = oracle.cache_values(w.blocks, w.heads_kv, w.page_tokens)
    key, value = key * w.tensor_scales[0], value * w.tensor_scales[2]
    out = out.cpu().double()
    worst = 0.0
    for r in range(w.rows) if rows is None else rows:
        n = inputs["query"].shape[1] if counts is None else counts[r]
        if n == 0:
            continue
        fp4 = int(w.seqused_fp4[r])
        want, allowed = oracle.tree_attention(
            query=inputs["query"][r, :n], draft_key=inputs["draft_key"][r, :n], draft_value=inputs["draft_value"][r, :n],
            parents=inputs["parents"][r, :n].tolist() if inputs["parents"].ndim == 2 else inputs["parents"][:n].tolist(),
            key=key, value=value, page_ids=w.page_table[r, :fp4 // w.page_tokens].cpu().long(), fp4=fp4,
            tail_key=w.tail_key[0, r].cpu(), tail_value=w.tail_value[0, r].cpu(),
            residual=int(w.seqused_residual[r]) if tail else 0, sink=int(w.seqused_sink[r]) if tail else 0,
            softmax_scale=scale, rotate=rotate, shift=shift)
        got = out[r, :n]
        assert torch.isfinite(got).all(), f"row {r}"
        ratio = float(((got - want).abs() / allowed).max())
        worst = max(worst, ratio)
        assert ratio <= 1.0, f"row {r}: {ratio:.2f} times the allowance"
    return worst


LENGTHS = [1, 5, 16, 17, 127, 128, 129, 144, 255, 257, 700]


@pytest.mark.parametrize("page_tokens", [128, 64])
@pytest.mark.parametrize("nodes", [1, 2, 7, 16, 33, 64])
def test_lengths_and_nodes(page_tokens, nodes):
    w, x = _inputs(LENGTHS, nodes, 8, 2, seed=nodes, page_tokens=page_tokens)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (4, 2), (3, 1), (10, 2), (14, 2), (21, 3), (16, 2), (16, 1), (40, 1)])
@pytest.mark.parametrize("nodes", [1, 5, 19])
def test_head_layouts(heads, nodes):
    w, x = _inputs([300, 1030], nodes, *heads, seed=heads[0] + nodes)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("tree", ["chain", "roots", "star"])
@pytest.mark.parametrize("nodes", [3, 64])
def test_tree_shapes(tree, nodes):
    w, x = _inputs([130, 513], nodes, 8, 2, seed=3, tree=tree)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("page_tokens", [128, 64])
def test_many_rows_of_many_lengths(page_tokens):
    lens = [1 + (137 * i) % 2900 for i in range(37)]
    w, x = _inputs(lens, 6, 8, 2, seed=11, page_tokens=page_tokens)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("nodes", [4, 40])
def test_long_row_is_split_over_the_gpu(nodes):
    w, x = _inputs([20000, 333], nodes, 8, 2, seed=12)
    _check(w, x, _call(w, x))


def test_one_node_over_a_long_row():
    w, x = _inputs([33001], 1, 4, 4, seed=13, page_tokens=64)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("rotate,shift", [(True, False), (True, True), (False, True)])
@pytest.mark.parametrize("nodes", [3, 50])
def test_rotation_and_shift(rotate, shift, nodes):
    w, x = _inputs([90, 700], nodes, 8, 2, seed=21, rotate=rotate, key_shift=True)
    s = w.key_shift[0] if shift else None
    out = _call(w, x, query_rotation="hadamard" if rotate else "none", key_shift=s)
    _check(w, x, out, rotate=rotate, shift=None if s is None else s.cpu())


@pytest.mark.parametrize("page_tokens", [128, 64])
def test_tensor_scales_and_softmax_scale(page_tokens):
    w, x = _inputs([90, 700, 1400], 9, 8, 2, seed=22, key_tensor_scale=0.37, value_tensor_scale=2.6, page_tokens=page_tokens)
    out = _call(w, x, tensor_scales=(w.tensor_scales[0], w.tensor_scales[2]), softmax_scale=0.21)
    _check(w, x, out, scale=0.21)


@pytest.mark.parametrize("loud", [8.0, 60.0, 1e-3])
def test_sharp_and_flat_scores(loud):
    """Scores whose maximum moves late and far (loud old pages, large queries), and nearly equal ones."""
    w, x = _inputs([1500, 200], 12, 8, 2, seed=23, loud=loud, loud_prefix=200)
    _check(w, x, _call(w, x))


@pytest.mark.parametrize("factor", [2.0 ** 90, 2.0 ** -90])
def test_far_query_magnitudes(factor):
    """A query far outside FP16 with a softmax scale that brings it back: the products must not lose it."""
    w, x = _inputs([300], 5, 4, 1, seed=24)
    scaled = dict(x, query=(x["query"].double() * factor).to(torch.bfloat16))
    got = _call(w, scaled, softmax_scale=128 ** -0.5 / factor)
    _check(w, scaled, got, scale=128 ** -0.5 / factor)


def test_small_and_large_tail_keys():
    """Tail and draft keys far from FP16's range, against queries that bring the scores back."""
    w, x = _inputs([60, 100], 5, 4, 1, seed=25)
    w.tail_key.mul_(2.0 ** 40)
    scaled = dict(x, draft_key=(x["draft_key"].double() * 2.0 ** 40).to(torch.bfloat16))
    _check(w, scaled, _call(w, scaled, softmax_scale=128 ** -0.5 * 2.0 ** -40), scale=128 ** -0.5 * 2.0 ** -40)
    w.tail_value.mul_(2.0 ** 60)
    scaled["draft_value"] = (x["draft_value"].double() * 2.0 ** 60).to(torch.bfloat16)
    _check(w, scaled, _call(w, scaled, softmax_scale=128 ** -0.5 * 2.0 ** -40), scale=128 ** -0.5 * 2.0 ** -40)


def test_without_tail_and_sink():
    w, x = _inputs([1, 128, 129, 513], 5, 8, 2, seed=31)
    none = dict(residual_key_pages_bf16=None, residual_value_pages_bf16=None, residual_page_ids=None,
                seqused_residual=None, seqused_sink=None)
    _check(w, x, _call(w, x, **none), tail=False)
    w, x = _inputs([70, 200], 5, 8, 2, seed=32, sink=0)
    _check(w, x, _call(w, x))


def test_node_counts_leave_the_rest_alone():
    nodes, counts = 11, [11, 0, 1, 7, 10]
    w, x = _inputs([300, 300, 20, 700, 129], nodes, 8, 2, seed=33)
    out = torch.full((5, nodes, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    # what lies behind a row's nodes may be anything
    for r, n in enumerate(counts):
        for name in ("query", "draft_key", "draft_value"):
            x[name][r, n:] = float("nan")
        x["parents"][r, n:] = 1 << 30
    got = _call(w, x, out=out, node_counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    assert got.data_ptr() == out.data_ptr()
    _check(w, x, got, counts=counts)
    for r, n in enumerate(counts):
        assert bool((out[r, n:] == 7.0).all()), f"row {r}"
    fresh = _call(w, x, node_counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    for r, n in enumerate(counts):
        assert torch.equal(fresh[r, :n], out[r, :n]) and not bool(fresh[r, n:].any())


def test_stale_bytes_behind_the_lengths_do_not_leak():
    """Tail rows past a row's length, the unused sink, other rows' slots and pages, page-table columns past the
    row's pages: NaN and infinity there change nothing."""
    w, x = _inputs([40, 300, 129], 6, 8, 2, seed=34)
    want = _call(w, x)
    for r, n in enumerate(w.seq_lens):
        residual, sink = int(w.seqused_residual[r]), int(w.seqused_sink[r])
        for t in (w.tail_key, w.tail_value):
            t[0, r, residual:128] = float("nan")
            t[0, r, 128 + sink:] = float("inf")
    w.blocks[0] = 0xFF  # the null block: NaN scales
    wide = torch.full((3, w.page_table.shape[1] + 3), 1 << 29, dtype=torch.int32, device="cuda")
    for r, n in enumerate(w.seqused_fp4.tolist()):
        wide[r, :n // 128] = w.page_table[r, :n // 128]
    w.page_table = wide
    assert torch.equal(_call(w, x, trusted_metadata=True), want)


def test_strided_queries_drafts_and_output():
    """Q, K and V as slices of one projection, a wider node axis, and a strided output."""
    rows, nodes, hq, hk = 3, 5, 8, 2
    w, x = _inputs([200, 300, 10], nodes, hq, hk, seed=35)
    qkv = torch.zeros(rows, nodes + 3, hq + 2 * hk, 128, dtype=torch.bfloat16, device="cuda")
    qkv[:, 1:1 + nodes, :hq], qkv[:, 1:1 + nodes, hq:hq + hk] = x["query"].cuda(), x["draft_key"].cuda()
    qkv[:, 1:1 + nodes, hq + hk:] = x["draft_value"].cuda()
    part = qkv[:, 1:1 + nodes]
    buffer = torch.full((rows, nodes, hq + 4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    got = _call(w, dict(x, query=part[:, :, :hq], draft_key=part[:, :, hq:hq + hk], draft_value=part[:, :, hq + hk:]),
                out=buffer[:, :, 2:2 + hq])
    assert torch.equal(got, _call(w, x))
    assert bool((buffer[:, :, :2] == 3.0).all()) and bool((buffer[:, :, 2 + hq:] == 3.0).all())
    _check(w, x, got)


def test_one_tree_for_all_rows():
    w, x = _inputs([200, 300], 9, 8, 2, seed=36)
    shared = x["parents"][0].contiguous()
    got = _call(w, dict(x, parents=shared))
    _check(w, dict(x, parents=shared), got)


def test_pages_shared_between_rows_and_slots_out_of_order():
    w, x = _inputs([400, 400, 50], 4, 8, 2, seed=37)
    w.page_table[1] = w.page_table[0]
    perm = torch.tensor([2, 0, 1], device="cuda")
    w.tail_key, w.tail_value = w.tail_key[:, perm].contiguous(), w.tail_value[:, perm].contiguous()
    ids = torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")
    got = _call(w, x, residual_page_ids=ids)
    back = ids.long()
    w.tail_key, w.tail_value = w.tail_key[:, back].contiguous(), w.tail_value[:, back].contiguous()
    _check(w, x, got)


def test_same_bits_again_and_under_a_graph():
    w, x = _inputs([5000, 700, 40], 16, 16, 2, seed=38)
    device = {k: v.cuda() for k, v in x.items()}
    first = _call(w, device)
    for _ in range(3):
        assert torch.equal(_call(w, device), first)
    out = torch.zeros_like(first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _call(w, device, out=out, trusted_metadata=True)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _call(w, device, out=out, trusted_metadata=True)
    out.zero_()
    # a replay follows what the device tensors hold by then: other lengths, another tree
    w.seqused_residual[0] = 3
    device["parents"].copy_(_trees(3, 16, torch.Generator().manual_seed(5)).cuda())
    graph.replay()
    torch.cuda.synchronize()
    _check(w, dict(x, parents=device["parents"].cpu()), out)


def test_two_streams_at_once():
    cases = [_inputs([3000, 90], 16, 8, 2, seed=s) for s in (40, 41)]
    inputs = [(w, {k: v.cuda() for k, v in x.items()}) for w, x in cases]
    want = [_call(w, x).clone() for w, x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (w, x) in enumerate(inputs):
            with torch.cuda.stream(streams[i]):
                got[i].append(_call(w, x, trusted_metadata=True))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_own_workspace_and_bad_pages():
    import bdfp4
    from nvfp4_decode_kernel import tree

    w, x = _inputs([700, 300], 5, 8, 2, seed=42)
    size = tree.tree_workspace_bytes(2, 5, 8, 2)
    buffer = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = _call(w, x)
    assert torch.equal(_call(w, x, workspace=buffer, error_word=error), want)
    assert int(error) == 0
    with pytest.raises(ValueError):
        _call(w, x, workspace=buffer[:-16])
    # a page id outside the cache is reported and never followed; the row that has it is garbage, the other is not
    w.page_table[0, 1] = w.blocks.shape[0] + 5
    with pytest.raises(ValueError):
        _call(w, x)
    got = _call(w, x, trusted_metadata=True, error_word=error)
    torch.cuda.synchronize()
    assert int(error) == bdfp4.DEV_BAD_PAGE
    assert torch.equal(got[1], want[1])


def test_refusals():
    from nvfp4_decode_kernel import tree

    w, x = _inputs([300, 40], 5, 8, 2, seed=43)
    x = {k: v.cuda() for k, v in x.items()}
    good = _call(w, x)

    def refused(error=ValueError, args=None, **more):
        with pytest.raises(error):
            _call(w, dict(x, **(args or {})), **more)

    refused(args=dict(query=x["query"].float()))
    refused(args=dict(query=x["query"][:, :, :7]))
    refused(args=dict(draft_key=x["draft_key"][:, :4]))
    refused(args=dict(draft_value=x["draft_value"].transpose(2, 3).contiguous().transpose(2, 3)))
    refused(args=dict(parents=x["parents"].long()))
    refused(args=dict(parents=x["parents"][:1]))
    refused(NotImplementedError, args={k: v.repeat_interleave(13, 1) for k, v in x.items()})
    refused(NotImplementedError, scale_mode="mxfp4_ocp")
    refused(scale_mode="fp4")
    refused(node_counts=torch.tensor([5, 6], dtype=torch.int32, device="cuda"))
    refused(node_counts=torch.tensor([5], dtype=torch.int32, device="cuda"))
    refused(residual_page_ids=None)
    refused(residual_page_ids=w.slot_ids + 1)
    refused(seqused_residual=w.seqused_residual + 128)
    refused(residual_key_pages_bf16=w.tail_key[0][:, :130])
    refused(key_shift=torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda"))
    refused(query_rotation="block_hadamard_64")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        refused(softmax_scale=bad)
        refused(tensor_scales=(1.0, bad))
    refused(out=torch.empty(2, 5, 8, 128, device="cuda"))
    refused(out=torch.empty(2, 5, 7, 128, dtype=torch.bfloat16, device="cuda"))
    refused(error_word=torch.zeros(1, device="cuda"))
    w.seqused_fp4 += 1
    refused()
    w.seqused_fp4 -= 1
    assert torch.equal(_call(w, x), good)
    for sizes in ((0, 5, 8, 2), (1, 65, 8, 2), (1, 5, 7, 2)):
        with pytest.raises(ValueError):
            tree.tree_workspace_bytes(*sizes)
