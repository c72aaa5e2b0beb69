"""Whole speculative steps, as a serving loop takes them: the tree's attention in every layer, verification, commit,
and the next step over what the commit left. Attention within its derived allowance, all else bit for bit."""

import pytest
import torch

from oracle import nvfp4_oracle, tree_oracle

pytestmark = pytest.mark.gpu

SINK, LAYERS, HEADS, RATIO, VOCAB = 16, 2, 2, 4, 97


class _Sequences:
    """A small cache on the GPU and what should stand in it, token by token, on the CPU."""

    def __init__(self, lens, columns, page_tokens, gen):
        from bdfp4.workload import carve_cache

        def bf16(*shape):
            return torch.randn(*shape, generator=gen).to(torch.bfloat16)

        rows = len(lens)
        self.lens, self.page_tokens, self.entries = list(lens), page_tokens, 128 // page_tokens
        self.tails = [bf16(LAYERS, rows + 1, 128 + SINK, HEADS, 128) for _ in range(2)]
        self.slots = torch.randperm(rows + 1, generator=gen)[:rows].to(torch.int32)
        self.shift = 0.25 * torch.randn(LAYERS, HEADS, 128, generator=gen)
        pages = rows * columns * self.entries
        self.table = torch.randperm(pages, generator=gen).to(torch.int32).view(rows, -1)
        self.blocks = [torch.zeros(pages, 2 * page_tokens * HEADS * 72, dtype=torch.uint8) for _ in range(LAYERS)]
        for r, n in enumerate(lens):
            for page in range((n - 1) // 128 if n else 0):
                for layer in range(LAYERS):
                    self.seal(layer, r, page, [bf16(128, HEADS, 128) for _ in range(2)])
        self.gpu_blocks = [b.cuda() for b in self.blocks]
        self.gpu_tails = [t.cuda() for t in self.tails]
        self.regions = [carve_cache(b, HEADS, page_tokens) for b in self.gpu_blocks]

    def seal(self, layer, row, page, kv):
        for e in range(self.entries):
            k, v = (t[e * self.page_tokens:(e + 1) * self.page_tokens][None] for t in kv)
            kc, ks = nvfp4_oracle.quantize_key_pages(k, "amax6")
            vc, vs = nvfp4_oracle.quantize_value_pages(v, "amax6")
            if self.page_tokens == 64:
                kc = kc.permute(0, 2, 1, 3)
            self.blocks[layer][int(self.table[row, page * self.entries + e])] = torch.cat([x.reshape(-1) for x in (kc, ks, vc, vs)])

    def append(self, row, key, value):
        """One token of every layer, its key in the cache's basis already."""
        position, slot = self.lens[row], int(self.slots[row])
        for tail, token in zip(self.tails, (key, value)):
            tail[:, slot, position % 128] = token
            if position < SINK:
                tail[:, slot, 128 + position] = token
        if position % 128 == 127:
            for layer in range(LAYERS):
                self.seal(layer, row, position // 128, [t[layer, slot, :128] for t in self.tails])
        self.lens[row] += 1


@pytest.mark.parametrize("page_tokens", [128, 64])
@pytest.mark.parametrize("nodes", [6, 20])
def test_steps_of_a_serving_loop(page_tokens, nodes):
    from nvfp4_decode_kernel import tree

    gen = torch.Generator().manual_seed(100 * nodes + page_tokens)
    s = _Sequences([0, 1, 119, 250, 127], 4, page_tokens, gen)
    rows = len(s.lens)
    committer = tree.DraftCommitter(tail_key=s.gpu_tails[0], tail_value=s.gpu_tails[1], sink_tokens=SINK, rotate_key=True,
                                    key_shift=s.shift.cuda(), regions=s.regions)
    slots, table = s.slots.cuda(), s.table.cuda()
    lengths = tree.CommittedLengths(*(torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(
        *((n, (n - 1) // 128 * 128 if n else 0, n - ((n - 1) // 128 * 128 if n else 0), min(n, SINK)) for n in s.lens))))
    committed = 0
    for step in range(7):
        def bf16(*shape):
            return torch.randn(*shape, generator=gen).to(torch.bfloat16)

        query = bf16(LAYERS, rows, nodes, HEADS * RATIO, 128)
        key, value = bf16(LAYERS, rows, nodes, HEADS, 128), bf16(LAYERS, rows, nodes, HEADS, 128)
        parents = (torch.rand(rows, nodes, generator=gen) * torch.arange(nodes)).to(torch.int32)
        parents[:, 0] = -1
        draft_key, draft_value = key.cuda(), value.cuda()
        for layer in range(LAYERS):
            out = tree.tree_decode(
                query[layer].cuda(), draft_key[layer], draft_value[layer], parents.cuda(), *s.regions[layer], table,
                lengths.seqused_fp4, residual_key_pages_bf16=s.gpu_tails[0][layer], residual_value_pages_bf16=s.gpu_tails[1][layer],
                residual_page_ids=slots, seqused_residual=lengths.seqused_residual, seqused_sink=lengths.seqused_sink,
                query_rotation="hadamard", key_shift=s.shift[layer].cuda()).cpu().double()
            cached = tree_oracle.cache_values(s.blocks[layer], HEADS, page_tokens)
            for r, n in enumerate(s.lens):
                fp4 = (n - 1) // 128 * 128 if n else 0
                want, allowed = tree_oracle.tree_attention(
                    query=query[layer, r], draft_key=key[layer, r], draft_value=value[layer, r], parents=parents[r].tolist(),
                    key=cached[0], value=cached[1], page_ids=s.table[r, :fp4 // page_tokens].long(), fp4=fp4,
                    tail_key=s.tails[0][layer, int(s.slots[r])], tail_value=s.tails[1][layer, int(s.slots[r])],
                    residual=n - fp4, sink=min(n, SINK), softmax_scale=128 ** -0.5, rotate=True, shift=s.shift[layer])
                assert bool(((out[r] - want).abs() <= allowed).all()), f"step {step}, layer {layer}, row {r}"
        # a drafter that is close to the target, so that paths of several tokens are accepted
        logits = torch.randn(rows, nodes, VOCAB, generator=gen)
        target, draft = torch.softmax(3 * logits, -1), torch.softmax(3 * logits + 0.3 * torch.randn(logits.shape, generator=gen), -1)
        tokens = torch.zeros(rows, nodes, dtype=torch.int32)
        for i in range(1, nodes):
            tokens[:, i] = torch.multinomial(draft[torch.arange(rows), parents[:, i].long()], 1, generator=gen)[:, 0]
        uniforms = torch.rand(rows, nodes, generator=gen)
        verdict = tree.verify_drafts(target.cuda(), tokens.cuda(), parents.cuda(), uniforms.cuda(), draft_probs=draft.cuda())
        lengths = committer(draft_key, draft_value, verdict.accepted, verdict.accepted_counts, seq_lens=lengths.seq_lens,
                            row_to_slot=slots, block_table=table)
        basis = torch.stack([nvfp4_oracle.key_cache_basis(key[i], rotate=True, shift=s.shift[i]) for i in range(LAYERS)])
        for r in range(rows):
            path, token, margin = tree_oracle.verify(target[r].numpy(), tokens[r].numpy(), parents[r].numpy(), uniforms[r].numpy(),
                                                     draft[r].numpy(), None)
            assert margin > 1e-9, "an input next to a border: choose another seed"
            assert verdict.accepted[r].tolist() == path + [-1] * (nodes - len(path)) and int(verdict.next_tokens[r]) == token
            for node in path:
                s.append(r, basis[:, r, node], value[:, r, node])
            committed += len(path)
        assert lengths.seq_lens.tolist() == s.lens
        for got, want in zip(s.gpu_tails, s.tails):
            assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16)), f"step {step}"
        for got, want in zip(s.gpu_blocks, s.blocks):
            assert torch.equal(got.cpu(), want), f"step {step}"
    assert committed > 7 * rows and s.lens[2] > 128 and s.lens[4] > 128  # drafts were accepted, pages filled
