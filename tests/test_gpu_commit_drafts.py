"""The accepted path's way into tail, sink and pages: bit for bit what the one-token writers and the page
quantizer would have stored, and nothing else touched."""

import pytest
import torch

from oracle import nvfp4_oracle, tree_oracle

pytestmark = pytest.mark.gpu


def _setup(rows, layers, nodes, heads, lens, counts, seed, page_tokens=128, sink=16, seal=True, shift=True):
    from bdfp4.workload import carve_cache

    gen = torch.Generator().manual_seed(seed)

    def bf16(*shape):
        return torch.randn(*shape, generator=gen).to(torch.bfloat16)

    slots = rows + 2
    s = dict(tail_key=bf16(layers, slots, 128 + sink, heads, 128), tail_value=bf16(layers, slots, 128 + sink, heads, 128),
             key=bf16(layers, rows, nodes, heads, 128), value=bf16(layers, rows, nodes, heads, 128),
             row_to_slot=torch.randperm(slots, generator=gen)[:rows].to(torch.int32),
             seq_lens=torch.tensor(lens, dtype=torch.int32), counts=torch.tensor(counts, dtype=torch.int32),
             shift=0.25 * torch.randn(layers, heads, 128, generator=gen) if shift else None)
    accepted = torch.full((rows, nodes), -1, dtype=torch.int32)
    for r, c in enumerate(counts):
        if c:
            accepted[r, 0] = 0
            accepted[r, 1:c] = torch.randperm(nodes - 1, generator=gen)[:c - 1].sort().values.to(torch.int32) + 1
    s["accepted"] = accepted
    entries = 128 // page_tokens
    columns = (max(n + c for n, c in zip(lens, counts)) // 128 + 1) * entries
    blocks = [torch.full((1 + rows * columns, 2 * page_tokens * heads * 72), 0xAB, dtype=torch.uint8, device="cuda")
              for _ in range(layers)]
    s["table"] = (torch.randperm(rows * columns, generator=gen) + 1).to(torch.int32).view(rows, columns)
    s["blocks"], s["regions"] = blocks, [carve_cache(b, heads, page_tokens) for b in blocks] if seal else None
    return s


def _commit(s, rotate, sink=16, error=None, build=None, **more):
    from nvfp4_decode_kernel import tree

    tails = [s["tail_key"].cuda(), s["tail_value"].cuda()]
    committer = tree.DraftCommitter(tail_key=tails[0], tail_value=tails[1], sink_tokens=sink, rotate_key=rotate,
                                    key_shift=None if s["shift"] is None else s["shift"].cuda(), regions=s["regions"],
                                    error_word=error, **(build or {}))
    args = dict(seq_lens=s["seq_lens"].cuda(), row_to_slot=s["row_to_slot"].cuda(),
                block_table=s["table"].cuda() if s["regions"] is not None else None)
    args.update(more)
    lengths = committer(s["key"].cuda(), s["value"].cuda(), s["accepted"].cuda(), s["counts"].cuda(), **args)
    return tails, lengths


def _expect(s, rotate, sink=16, page_tokens=128, key_mode="amax6", value_mode="amax6"):
    """Tails token by token; a page is quantized the moment its last token arrives."""
    key = nvfp4_oracle.key_cache_basis(s["key"], rotate=rotate, shift=None) if s["shift"] is None else torch.stack(
        [nvfp4_oracle.key_cache_basis(s["key"][i], rotate=rotate, shift=s["shift"][i]) for i in range(s["key"].shape[0])])
    tails = [s["tail_key"].clone(), s["tail_value"].clone()]
    sealed, lengths = [], []
    for r in range(len(s["counts"])):
        n, count, slot = int(s["seq_lens"][r]), int(s["counts"][r]), int(s["row_to_slot"][r])
        if slot >= 0:
            for i, (position, at) in enumerate(tree_oracle.commit_positions(n, count)[0]):
                node = int(s["accepted"][r, i])
                for tail, source in zip(tails, (key, s["value"])):
                    tail[:, slot, at] = source[:, r, node]
                    if position < sink:
                        tail[:, slot, 128 + position] = source[:, r, node]
                if (position + 1) % 128 == 0:
                    page = [t[:, slot, :128].clone() for t in tails]
                    sealed.append((r, position // 128, page))
            n += count
        fp4 = (n - 1) // 128 * 128 if n else 0
        lengths.append((n, fp4, n - fp4, min(n, sink)))
    return tails, sealed, lengths


def _check(s, rotate, sink=16, page_tokens=128, key_mode="amax6", value_mode="amax6", build=None):
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = [b.cpu() for b in s["blocks"]]
    tails, lengths = _commit(s, rotate, sink, error, build)
    want_tails, sealed, want_lengths = _expect(s, rotate, sink, page_tokens)
    assert int(error) == 0
    for got, want in zip(tails, want_tails):
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    assert torch.stack([t.cpu() for t in lengths], 1).tolist() == [list(x) for x in want_lengths]
    if s["regions"] is None:
        return len(sealed)
    heads = s["key"].shape[3]
    codes, scales = page_tokens * 64 * heads, page_tokens * 8 * heads
    for layer, block in enumerate(s["blocks"]):
        want = before[layer].clone()
        for r, column, page in sealed:
            for e in range(128 // page_tokens):
                k, v = (t[layer, e * page_tokens:(e + 1) * page_tokens][None] for t in page)
                kc, ks = nvfp4_oracle.quantize_key_pages(k, key_mode)
                vc, vs = nvfp4_oracle.quantize_value_pages(v, value_mode)
                if page_tokens == 64:
                    kc = kc.permute(0, 2, 1, 3)
                at = int(s["table"][r, column * (128 // page_tokens) + e])
                want[at] = torch.cat([x.reshape(-1) for x in (kc, ks, vc, vs)])
        assert torch.equal(block.cpu(), want), f"layer {layer}"
    return len(sealed)


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("page_tokens", [128, 64])
@pytest.mark.parametrize("heads", [1, 2, 3])
def test_pages_fill_or_not(rotate, page_tokens, heads):
    lens, counts = [0, 10, 125, 126, 127, 128, 250, 383, 120], [3, 9, 2, 2, 2, 1, 9, 1, 9]
    s = _setup(9, 2, 9, heads, lens, counts, seed=heads, page_tokens=page_tokens)
    assert _check(s, rotate, page_tokens=page_tokens) == 5


@pytest.mark.parametrize("nodes", [1, 2, 31, 64])
def test_path_lengths(nodes):
    lens = [0, 1, 64, 127, 128 * 3 - nodes, 128 * 3 - nodes + 1]
    s = _setup(6, 1, nodes, 8, lens, [nodes, 1, nodes, nodes, nodes, max(1, nodes - 1)], seed=nodes)
    _check(s, True)


@pytest.mark.parametrize("shift", [False, True])
def test_without_rotation_or_pages(shift):
    s = _setup(4, 3, 7, 2, [5, 0, 300, 12], [7, 7, 3, 1], seed=3, seal=False, shift=shift)
    assert _check(s, False) == 0


@pytest.mark.parametrize("sink", [0, 4])
def test_sink_lengths(sink):
    s = _setup(3, 2, 7, 2, [0, 2, 125], [7, 7, 7], seed=4, sink=sink)
    _check(s, True, sink=sink)


def test_scale_modes():
    s = _setup(2, 1, 5, 2, [125, 126], [5, 5], seed=5)
    assert _check(s, True, key_mode="four_six", value_mode="four_six",
                  build=dict(key_scale_mode="four_six", value_scale_mode="four_six")) == 2


def test_inactive_rows_and_empty_paths():
    s = _setup(4, 1, 6, 2, [126, 126, 127, 300], [4, 0, 6, 3], seed=6)
    s["row_to_slot"][0] = -1
    _check(s, False)


def test_node_numbers_outside_the_tree_are_skipped():
    s = _setup(2, 1, 6, 2, [10, 10], [3, 3], seed=7, shift=False)
    tails, _ = _commit(s, False)
    s["accepted"][1, 1], s["accepted"][1, 2] = 6, -4
    again, _ = _commit(s, False)
    slot = int(s["row_to_slot"][1])
    assert torch.equal(again[0][:, slot, 10], tails[0][:, slot, 10])
    for at in (11, 12):
        assert torch.equal(again[0][:, slot, at].cpu(), s["tail_key"][:, slot, at])


def test_a_page_without_a_place_is_reported():
    import bdfp4

    s = _setup(2, 1, 6, 2, [126, 126], [4, 4], seed=8)
    s["table"][0, 0] = s["blocks"][0].shape[0] + 9
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = s["blocks"][0].clone()
    _commit(s, False, error=error)
    torch.cuda.synchronize()
    assert int(error) == bdfp4.DEV_BAD_PAGE
    changed = (s["blocks"][0] != before).any(1).nonzero()[:, 0].tolist()
    assert changed == [int(s["table"][1, 0])]
    error.zero_()
    _commit(s, False, error=error, block_table=s["table"][:, :0].cuda())
    assert int(error) == bdfp4.DEV_BAD_PAGE


def test_strided_drafts():
    """K and V as slices of a fused projection of every layer."""
    s = _setup(3, 2, 5, 2, [3, 200, 126], [5, 2, 4], seed=9)
    fused = torch.zeros(2, 3, 8, 10, 128, dtype=torch.bfloat16, device="cuda")
    fused[:, :, 1:6, 4:6], fused[:, :, 1:6, 6:8] = s["key"].cuda(), s["value"].cuda()
    want, _ = _commit(s, True)

    class On:
        """A CPU-side stand-in whose .cuda() hands out the strided view."""

        def __init__(self, t):
            self.t = t

        def cuda(self):
            return self.t

    got, _ = _commit(dict(s, key=On(fused[:, :, 1:6, 4:6]), value=On(fused[:, :, 1:6, 6:8])), True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured():
    from nvfp4_decode_kernel import tree

    s = _setup(3, 2, 5, 2, [3, 200, 126], [5, 2, 4], seed=10)
    want, lengths = _commit(s, True)
    tails = [s["tail_key"].cuda(), s["tail_value"].cuda()]
    committer = tree.DraftCommitter(tail_key=tails[0], tail_value=tails[1], rotate_key=True, key_shift=s["shift"].cuda(),
                                    regions=s["regions"])
    cuda = {k: s[k].cuda() for k in ("key", "value", "accepted", "counts", "seq_lens", "row_to_slot", "table")}
    zero = torch.zeros_like(cuda["counts"])

    def call(counts):
        return committer(cuda["key"], cuda["value"], cuda["accepted"], counts, seq_lens=cuda["seq_lens"],
                         row_to_slot=cuda["row_to_slot"], block_table=cuda["table"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(zero)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(cuda["counts"])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(tails[0], want[0]) and torch.equal(tails[1], want[1])
    for a, b in zip(got, lengths):
        assert torch.equal(a, b)


def test_refusals():
    from nvfp4_decode_kernel import tree

    s = _setup(2, 2, 5, 2, [3, 4], [2, 2], seed=11)
    key, value = s["tail_key"].cuda(), s["tail_value"].cuda()
    for change in (dict(tail_value=value[:1]), dict(tail_key=key.float()), dict(sink_tokens=17), dict(sink_tokens=4),
                   dict(key_shift=torch.zeros(2, 2, 128, dtype=torch.bfloat16, device="cuda")),
                   dict(key_shift=torch.zeros(2, 128, device="cuda")), dict(regions=s["regions"][:1]),
                   dict(tail_key=s["tail_key"])):
        with pytest.raises(ValueError):
            tree.DraftCommitter(**{**dict(tail_key=key, tail_value=value), **change})
    sealing = tree.DraftCommitter(tail_key=key, tail_value=value, regions=s["regions"])
    plain = tree.DraftCommitter(tail_key=key, tail_value=value)
    args = dict(draft_key=s["key"].cuda(), draft_value=s["value"].cuda(), accepted=s["accepted"].cuda(),
                accepted_counts=s["counts"].cuda(), seq_lens=s["seq_lens"].cuda(), row_to_slot=s["row_to_slot"].cuda())
    for committer, change in (
        (sealing, {}), (plain, dict(block_table=s["table"].cuda())), (plain, dict(draft_key=s["key"].cuda()[:1])),
        (plain, dict(draft_value=s["value"].cuda().float())), (plain, dict(accepted=s["accepted"].cuda().long())),
        (plain, dict(seq_lens=s["seq_lens"].cuda()[:1])), (plain, dict(row_to_slot=s["row_to_slot"])),
    ):
        with pytest.raises(ValueError):
            committer(**{**args, **change})
    big = {k: v.repeat_interleave(13, 2 if v.ndim == 5 else 1) if v.ndim > 1 else v for k, v in args.items()}
    with pytest.raises(NotImplementedError):
        plain(**big)
