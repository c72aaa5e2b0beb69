"""Long rows of the tree attention, where thousands of tokens share the weight and a lost one hardly shows: results
within what independent roundings come to, and queries that ask for single tokens all over the cache."""

import pytest
import torch

from oracle import tree_oracle as oracle
from test_gpu_tree_decode import _call, _check, _inputs
from test_gpu_tree_edges import _check_needles, _needles

pytestmark = pytest.mark.gpu

CASES = [  # lengths, nodes, (heads, KV heads), page tokens: every tile width, rows that straddle CTAs, ragged batches
    ([20000, 333], 4, (8, 2), 128), ([20000, 333], 40, (8, 2), 128), ([33001], 1, (4, 4), 64), ([7000, 40, 3000], 16, (16, 2), 128),
    ([9000, 9001], 7, (8, 2), 64), ([12000], 12, (8, 1), 64), ([5000, 1, 700], 32, (16, 2), 64),
    ([1 + (137 * i) % 2900 for i in range(19)], 6, (8, 2), 128),
]


@pytest.mark.parametrize("lens,nodes,heads,page_tokens", CASES)
@pytest.mark.parametrize("rotate", [False, True])
def test_within_what_roundings_come_to(lens, nodes, heads, page_tokens, rotate):
    w, x = _inputs(lens, nodes, *heads, seed=91, page_tokens=page_tokens, rotate=rotate)
    got = _call(w, x, query_rotation="hadamard" if rotate else "none").cpu().double()
    key, value = oracle.cache_values(w.blocks, w.heads_kv, page_tokens)
    for r in range(len(lens)):
        fp4 = int(w.seqused_fp4[r])
        want, typical = oracle.tree_attention(
            query=x["query"][r], draft_key=x["draft_key"][r], draft_value=x["draft_value"][r],
            parents=x["parents"][r].tolist(), key=key, value=value, page_ids=w.page_table[r, :fp4 // page_tokens].cpu().long(),
            fp4=fp4, tail_key=w.tail_key[0, r].cpu(), tail_value=w.tail_value[0, r].cpu(),
            residual=int(w.seqused_residual[r]), sink=int(w.seqused_sink[r]), softmax_scale=128 ** -0.5, rotate=rotate,
            typical=True)
        off = ((got[r] - want) ** 2).mean(-1).sqrt() / typical
        print(f"{lens[r]} tokens, {nodes} nodes: rms error up to {float(off.max()):.2f} of what roundings come to")
        assert oracle.outside_typical(got[r], want, typical) == 0, f"row {r}: {float(off.max()):.2f}"


@pytest.mark.parametrize("lens,nodes,heads,page_tokens", CASES)
def test_single_tokens_are_found(lens, nodes, heads, page_tokens):
    w, _ = _inputs(lens, 1, *heads, seed=92, page_tokens=page_tokens)
    x, want = _needles(w, nodes, heads[0], 93, 16.0)
    _check_needles(_call(w, x), want)


@pytest.mark.parametrize("lens,nodes,heads,page_tokens", CASES)
def test_single_tokens_at_any_magnitude(lens, nodes, heads, page_tokens):
    """Each query by a power of two of its own: quiet beside loud in every tile, scores beyond 2^27 next to ordinary ones,
    in rows that straddle CTAs and in CTAs that hold many units."""
    w, _ = _inputs(lens, 1, *heads, seed=94, page_tokens=page_tokens)
    x, want = _needles(w, nodes, heads[0], 95, 16.0)
    power = torch.randint(0, 4, x["query"].shape[:3], generator=torch.Generator().manual_seed(96))
    by = torch.tensor([1.0, 2.0 ** 9, 2.0 ** 26, 2.0 ** 70], dtype=torch.float64)[power]
    x["query"] = (x["query"].double() * by[..., None]).to(torch.bfloat16)
    _check_needles(_call(w, x), want)


@pytest.mark.parametrize("nodes,heads", [(3, (8, 2)), (7, (8, 2)), (15, (8, 2)), (22, (8, 2)), (31, (8, 2))])
@pytest.mark.parametrize("page_tokens", [128, 64])
def test_many_units_per_cta_some_with_loud_queries(nodes, heads, page_tokens):
    """Hundreds of short units, so that a CTA goes from tiles of one scale to uneven ones and back."""
    lens = [1 + (211 * i) % 520 for i in range(220)]
    w, x = _inputs(lens, nodes, *heads, seed=97, page_tokens=page_tokens)
    loud = x["query"].double()
    loud[::3, nodes // 2] *= 2.0 ** 20
    loud[1::5, 0, 1] *= 2.0 ** -20
    x["query"] = loud.to(torch.bfloat16)
    _check(w, x, _call(w, x), rows=range(0, 220, 7))
