"""Timed cases of the speculative-decoding operators over the FP4 cache.

Three operators make one speculative step: ``tree_decode`` scores a tree of drafted tokens against a
paged NVFP4 cache (BF16 sink and rolling tail included), ``verify_drafts`` walks the tree with the
target's probabilities and given random numbers, and ``DraftCommitter`` moves the accepted path into
the cache. Each case can run in two forms: the operators' plain form in elementary torch operations
(``own`` false), or the framework's kernels (``own`` true).
"""

import math
import os
import sys

import torch

own = False

PAGE, DIM, SINK = 128, 128, 16
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    return [
        # the smallest call: one new token of one short sequence, where latency is all there is
        dict(name="tree: one token", op="tree", rows=1, nodes=1, heads_q=8, heads_kv=2, context=200, ragged=False,
             page_tokens=128, rotate=False, scaled=False),
        # a short chain of drafts for an interactive batch
        dict(name="tree: chain of 5", op="tree", rows=4, nodes=5, heads_q=32, heads_kv=8, context=4096, ragged=True,
             page_tokens=64, rotate=False, scaled=False),
        # the ordinary serving batch: 16 nodes, prompts of a few thousand tokens
        dict(name="tree: 16 nodes x 16 rows", op="tree", rows=16, nodes=16, heads_q=32, heads_kv=8, context=8192,
             ragged=True, page_tokens=128, rotate=False, scaled=False),
        # the long-context batch this cache is made for
        dict(name="tree: 8 nodes x 65536", op="tree", rows=16, nodes=8, heads_q=32, heads_kv=8, context=65536,
             ragged=False, page_tokens=64, rotate=False, scaled=False),
        # one very long sequence under a wide tree: 256 query rows per KV head
        dict(name="tree: one row x 262145", op="tree", rows=1, nodes=32, heads_q=64, heads_kv=8, context=262145,
             ragged=False, page_tokens=128, rotate=False, scaled=False),
        # a large tree of odd size over short ragged prompts, rotated and shifted keys, tensor scales
        dict(name="tree: 61 nodes, rotated", op="tree", rows=24, nodes=61, heads_q=40, heads_kv=8, context=2900,
             ragged=True, page_tokens=128, rotate=True, scaled=True),
        # one request, greedy drafts: nothing but latency
        dict(name="verify: chain of 5", op="verify", rows=1, nodes=5, vocab=32000, drafter=False, bf16=False),
        # a batch whose drafter sampled its tokens: rejections subtract the drafter's distribution
        dict(name="verify: 16 nodes, drafter", op="verify", rows=32, nodes=16, vocab=131072, drafter=True, bf16=False),
        # BF16 probabilities of an odd vocabulary
        dict(name="verify: 33 nodes, bf16", op="verify", rows=64, nodes=33, vocab=50001, drafter=False, bf16=True),
        # few rows of a small model, some of them filling a page, keys rotated on the way
        dict(name="commit: pages fill", op="commit", rows=3, layers=2, nodes=7, heads_kv=2, crossing=True, rotate=True),
        # every layer of a batch at once
        dict(name="commit: 64 rows x 32 layers", op="commit", rows=64, layers=32, nodes=16, heads_kv=8, crossing=False,
             rotate=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "tree", "verify", "commit"))
    if op == "tree":
        heads_kv = rng.choice((1, 2, 4, 8))
        ratio = rng.choice((1, 2, 4, 5, 7, 8, 16))
        nodes = _log(rng, 1, 64)
        context = _log(rng, 1, 262145)
        most = min(16 * 65536 * 8 // (context * heads_kv), 500_000_000 // ((context + 200) * nodes * heads_kv * ratio))
        return dict(op=op, rows=_log(rng, 1, max(1, min(64, most))), nodes=nodes, heads_q=heads_kv * ratio,
                    heads_kv=heads_kv, context=context, ragged=rng.random() < 0.5,
                    page_tokens=rng.choice((64, 128)), rotate=rng.random() < 0.5, scaled=rng.random() < 0.3)
    if op == "verify":
        nodes, vocab, drafter = _log(rng, 1, 64), _log(rng, 500, 160000), rng.random() < 0.5
        most = 32 * 16 * 131072 // (nodes * vocab)
        return dict(op=op, rows=_log(rng, 1, max(1, min(128, most))), nodes=nodes, vocab=vocab, drafter=drafter,
                    bf16=rng.random() < 0.5)
    crossing = rng.random() < 0.4
    rows, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
    layers = _log(rng, 1, 4 if crossing else max(1, min(32, 32 * 64 * 16 // (rows * nodes))))
    return dict(op=op, rows=min(rows, 8) if crossing else rows, layers=layers, nodes=nodes,
                heads_kv=rng.choice((1, 2, 8)), crossing=crossing, rotate=rng.random() < 0.5)


# ---- what a case's sizes are (the same for every seed) ---------------------------------------------


def _lengths(case):
    """Committed tokens of each row."""
    rows, context = case["rows"], case["context"]
    if not case["ragged"]:
        return [context] * rows
    return [max(1, int(context * (0.15 + 0.85 * ((0.618034 * (i + 1)) % 1.0)))) for i in range(rows)]


def _counts(case):
    """Valid nodes of each row."""
    if not case.get("ragged"):
        return [case["nodes"]] * case["rows"]
    return [case["nodes"] - (5 * i) % (case["nodes"] // 2 + 1) for i in range(case["rows"])]


def _split(n):
    fp4 = (n - 1) // PAGE * PAGE if n else 0
    return min(n, SINK), fp4, n - fp4


def _committed(case):
    """(length before, accepted nodes) of each row of a commit case."""
    out = []
    for i in range(case["rows"]):
        accepted = 1 + (5 * i + 2) % case["nodes"]
        if case["crossing"] and i % 2 == 0:  # this row's last accepted tokens lie past a page boundary, or fill it
            n = PAGE * (2 + i % 3) - 1 - (3 * i) % accepted
        else:
            n = PAGE * (i % 3) + 1 + (37 * i) % (PAGE - case["nodes"])
        out.append((n, accepted))
    return out


# ---- inputs ----------------------------------------------------------------------------------------


def _tree_parents(rows, nodes, gen, device):
    """Random trees: a node hangs on one of the four nodes before it (node 0 is the root)."""
    back = torch.randint(1, 5, (rows, nodes), generator=gen, device=device)
    at = torch.arange(nodes, device=device)
    parents = (at - back).clamp_min(0)
    parents[:, 0] = -1
    return parents.to(torch.int32).contiguous()


def _cache_views(blocks, heads, page_tokens):
    """The four regions of a flat block array: K codes, K scales, V codes, V scales."""
    num, pitch = blocks.shape
    codes, scales = page_tokens * 64 * heads, page_tokens * 8 * heads
    if page_tokens == PAGE:
        sizes = (num, 32, 4, 1, 4, 2, heads)
        key = blocks.as_strided((num, PAGE, heads, 64), (pitch, heads * 64, 64, 1), 0)
        key_scales = blocks.as_strided(sizes, (pitch, 16, 4, 1024, 1, 512, 1024), codes)
        value_scales = blocks.as_strided(sizes, (pitch, 16, 4, 1024, 1, 512, 1024), 2 * codes + scales)
    else:
        key = blocks.as_strided((num, 64, heads, 64), (pitch, 64, 4096, 1), 0)
        key_scales = blocks.as_strided((num, 32, 2, 1, 4, 2, heads), (pitch, 8, 4, 512, 1, 256, 512), codes)
        value_scales = blocks.as_strided((num, 32, 4, 1, 4, 1, heads), (pitch, 16, 4, 512, 1, 512, 512),
                                         2 * codes + scales)
    value = blocks.as_strided((num, heads, DIM, page_tokens // 2), (pitch, DIM * page_tokens // 2, page_tokens // 2, 1),
                              codes + scales)
    return key, key_scales, value, value_scales


def _random_blocks(num, heads, page_tokens, gen, device):
    """A cache as the quantizer leaves it: E2M1 codes over E4M3 scales near amax/6 of unit-variance data."""
    blocks = torch.randint(0, 256, (num, 2 * page_tokens * heads * 72), generator=gen, device=device, dtype=torch.uint8)
    codes, scales = page_tokens * 64 * heads, page_tokens * 8 * heads
    for start in (codes, 2 * codes + scales):
        z = torch.randn(num, scales, generator=gen, device=device)
        blocks[:, start:start + scales] = (0.3 * torch.exp(0.25 * z)).to(torch.float8_e4m3fn).view(torch.uint8)
    return blocks


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    return {"tree": _prepare_tree, "verify": _prepare_verify, "commit": _prepare_commit}[case["op"]](case, gen, device)


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _prepare_tree(case, gen, device):
    rows, nodes, hq, hk, pt = (case[k] for k in ("rows", "nodes", "heads_q", "heads_kv", "page_tokens"))
    lens = [_split(n) for n in _lengths(case)]
    per_row = [fp4 // pt for _, fp4, _ in lens]
    num, widest = 1 + sum(per_row), max(1, max(per_row))
    blocks = _random_blocks(num, hk, pt, gen, device)
    order = torch.randperm(num - 1, generator=gen, device=device).to(torch.int32) + 1
    table = torch.zeros(rows, widest, dtype=torch.int32, device=device)
    at = 0
    for i, n in enumerate(per_row):
        table[i, :n] = order[at:at + n]
        at += n

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    s = dict(case=case, blocks=blocks, regions=_cache_views(blocks, hk, pt), table=table,
             tail_key=randn(rows + 1, PAGE + SINK, hk, DIM).to(torch.bfloat16),
             tail_value=randn(rows + 1, PAGE + SINK, hk, DIM).to(torch.bfloat16),
             slots=torch.randperm(rows + 1, generator=gen, device=device)[:rows].to(torch.int32),
             sink=_ints([x[0] for x in lens], device), fp4=_ints([x[1] for x in lens], device),
             residual=_ints([x[2] for x in lens], device),
             # a few heads ask sharply, the others spread their weight over the context
             query=(randn(rows, nodes, hq, DIM) * torch.exp(0.5 * randn(1, 1, hq, 1))).to(torch.bfloat16),
             draft_key=randn(rows, nodes, hk, DIM).to(torch.bfloat16),
             draft_value=randn(rows, nodes, hk, DIM).to(torch.bfloat16),
             parents=_tree_parents(rows, nodes, gen, device),
             counts=_ints(_counts(case), device) if case["ragged"] else None,
             shift=0.25 * randn(hk, DIM) if case["rotate"] else None,
             tensor_scales=(0.8125, 1.375) if case["scaled"] else None,
             # node slots past a row's count are not written: the caller's buffer keeps what it had
             out=torch.zeros(rows, nodes, hq, DIM, dtype=torch.bfloat16, device=device))
    return s


def _prepare_verify(case, gen, device):
    rows, nodes, vocab = case["rows"], case["nodes"], case["vocab"]
    kind = torch.bfloat16 if case["bf16"] else torch.float32
    target = torch.empty(rows, nodes, vocab, dtype=kind, device=device)
    draft = torch.empty_like(target) if case["drafter"] else None
    parents = _tree_parents(rows, nodes, gen, device)
    tokens = torch.zeros(rows, nodes, dtype=torch.int32, device=device)
    guess = torch.empty(rows, nodes, vocab, dtype=torch.bfloat16, device=device)
    for i in range(nodes):  # a next-token distribution with one favourite, and the drafter's idea of it
        logits = 3.0 * torch.randn(rows, vocab, generator=gen, device=device)
        favourite = torch.randint(0, vocab, (rows, 1), generator=gen, device=device)
        logits.scatter_(1, favourite, torch.logsumexp(logits, 1, keepdim=True) + 0.8)
        target[:, i] = torch.softmax(logits, -1).to(kind)
        idea = torch.softmax(logits + 0.5 * torch.randn(rows, vocab, generator=gen, device=device), -1)
        if draft is not None:
            draft[:, i] = idea.to(kind)
        guess[:, i] = idea.to(torch.bfloat16)
    at = torch.arange(rows, device=device)
    for i in range(1, nodes):
        tokens[:, i] = torch.multinomial(guess[at, parents[:, i].long()].float(), 1, generator=gen)[:, 0].to(torch.int32)
    return dict(case=case, target=target, draft=draft, parents=parents, tokens=tokens,
                uniforms=torch.rand(rows, nodes, generator=gen, device=device))


def _prepare_commit(case, gen, device):
    rows, layers, nodes, hk = (case[k] for k in ("rows", "layers", "nodes", "heads_kv"))
    plan = _committed(case)

    def bf16(*shape):
        return torch.randn(*shape, generator=gen, device=device, dtype=torch.float32).to(torch.bfloat16)

    tail_key = torch.empty(layers, rows + 1, PAGE + SINK, hk, DIM, dtype=torch.bfloat16, device=device)
    tail_value = torch.empty_like(tail_key)
    for layer in range(layers):
        tail_key[layer], tail_value[layer] = bf16(*tail_key.shape[1:]), bf16(*tail_key.shape[1:])
    accepted = torch.full((rows, nodes), -1, dtype=torch.int32, device=device)
    for i, (_, count) in enumerate(plan):  # a path from the root: ascending node numbers
        rest = torch.randperm(nodes - 1, generator=gen, device=device)[:count - 1].sort().values + 1
        accepted[i, 0] = 0
        accepted[i, 1:count] = rest.to(torch.int32)
    columns = max(n + a for n, a in plan) // PAGE + 1
    blocks = [torch.zeros(1 + rows * columns, 2 * PAGE * hk * 72, dtype=torch.uint8, device=device)
              for _ in range(layers if case["crossing"] else 1)]
    order = torch.randperm(rows * columns, generator=gen, device=device).to(torch.int32) + 1
    return dict(case=case, draft_key=bf16(layers, rows, nodes, hk, DIM), draft_value=bf16(layers, rows, nodes, hk, DIM),
                accepted=accepted, counts=_ints([a for _, a in plan], device),
                seq_lens=_ints([n for n, _ in plan], device),
                slots=torch.randperm(rows + 1, generator=gen, device=device)[:rows].to(torch.int32),
                tail_key=tail_key, tail_value=tail_value, blocks=blocks, table=order.view(rows, columns),
                filled=[(i, (n + a) // PAGE - 1) for i, (n, a) in enumerate(plan) if (n + a) // PAGE > n // PAGE],
                shift=0.25 * torch.randn(layers, hk, DIM, generator=gen, device=device) if case["rotate"] else None)


# ---- one pass --------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if own:
        return _own(case["op"], s)
    return {"tree": _plain_tree, "verify": _plain_verify, "commit": _plain_commit}[case["op"]](s)


def _own(op, s):
    package = os.path.join(os.getcwd(), "bitdecoding-fp4_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from nvfp4_decode_kernel import tree

    case = s["case"]
    if op == "tree":
        return tree.tree_decode(
            s["query"], s["draft_key"], s["draft_value"], s["parents"], *s["regions"], s["table"], s["fp4"],
            node_counts=s["counts"], residual_key_pages_bf16=s["tail_key"], residual_value_pages_bf16=s["tail_value"],
            residual_page_ids=s["slots"], seqused_residual=s["residual"], seqused_sink=s["sink"],
            query_rotation="hadamard" if case["rotate"] else "none", key_shift=s["shift"],
            tensor_scales=s["tensor_scales"], out=s["out"], trusted_metadata=True)
    if op == "verify":
        v = tree.verify_drafts(s["target"], s["tokens"], s["parents"], s["uniforms"], draft_probs=s["draft"])
        return dict(accepted=v.accepted, counts=v.accepted_counts, next_tokens=v.next_tokens)
    if "committer" not in s:  # what a serving program builds once
        regions = None
        if s["filled"]:  # a path that ends on a page boundary fills a page too; layers that are not compared seal theirs aside
            aside = [torch.zeros_like(s["blocks"][0]) for _ in range(case["layers"] - len(s["blocks"]))]
            regions = [_cache_views(b, case["heads_kv"], PAGE) for b in s["blocks"] + aside]
        s["committer"] = tree.DraftCommitter(
            tail_key=s["tail_key"], tail_value=s["tail_value"], sink_tokens=SINK, rotate_key=case["rotate"],
            key_shift=s["shift"], regions=regions)
    new = s["committer"](s["draft_key"], s["draft_value"], s["accepted"], s["counts"], seq_lens=s["seq_lens"],
                         row_to_slot=s["slots"], block_table=s["table"] if s["filled"] else None)
    return _commit_outputs(s, new.seq_lens, new.seqused_fp4, new.seqused_residual, new.seqused_sink)


def _commit_outputs(s, seq, fp4, residual, sink):
    out = dict(tail_key=s["tail_key"], tail_value=s["tail_value"], seq_lens=seq, fp4=fp4, residual=residual, sink=sink)
    if s["filled"]:  # the pages that this step filled, as the values they stand for
        at = s["table"][[i for i, _ in s["filled"]], [c for _, c in s["filled"]]].long()
        pages = torch.stack([b[at] for b in s["blocks"]])
        key, value = _dequantize(pages.flatten(0, 1), s["case"]["heads_kv"], PAGE, torch.float32)
        out |= dict(key_pages=key, value_pages=value)
    return out


# ---- the plain forms -------------------------------------------------------------------------------


def _dequantize(pages, heads, page_tokens, kind):
    """Block bytes ``[n, bytes]`` -> K and V ``[n, tokens, heads, 128]``."""
    n, pt = pages.shape[0], page_tokens
    device = pages.device
    pair = torch.tensor([[E2M1[b & 15], E2M1[b >> 4]] for b in range(256)], dtype=kind, device=device)
    kc, ks, vc, vs = pages.split((pt * 64 * heads, pt * 8 * heads, pt * 64 * heads, pt * 8 * heads), 1)

    def scales(x):
        return x.contiguous().view(torch.float8_e4m3fn).to(kind)

    if pt == PAGE:
        kc, vc = kc.reshape(n, pt, heads, 64), vc.reshape(n, heads, DIM, 64)
        ks = scales(ks).view(n, heads, 2, 32, 4, 4).permute(0, 4, 3, 1, 2, 5).reshape(n, pt, heads, 8)
        vs = scales(vs).view(n, heads, 2, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(n, heads, DIM, 8)
    else:  # 64-token pages are head-major, their 16-byte chunks permuted
        t, c = torch.arange(64, device=device), torch.arange(DIM, device=device)
        place = torch.arange(4, device=device)[None] ^ ((t[:, None] >> 1) & 3)
        kc = kc.reshape(n, heads, 64, 4, 16)[:, :, t[:, None], place].reshape(n, heads, 64, 64).permute(0, 2, 1, 3)
        place = torch.arange(2, device=device)[None] ^ ((c[:, None] >> 2) & 1)
        vc = vc.reshape(n, heads, DIM, 2, 16)[:, :, c[:, None], place].reshape(n, heads, DIM, 32)
        ks = scales(ks).view(n, heads, 2, 32, 2, 4).permute(0, 4, 3, 1, 2, 5).reshape(n, 64, heads, 8)
        vs = scales(vs).view(n, heads, 32, 4, 4).permute(0, 1, 3, 2, 4).reshape(n, heads, DIM, 4)
    key = (pair[kc.long()].view(n, pt, heads, 8, 16) * ks[..., None]).view(n, pt, heads, DIM)
    value = (pair[vc.long()].view(n, heads, DIM, pt // 16, 16) * vs[..., None]).view(n, heads, DIM, pt)
    return key, value.permute(0, 3, 1, 2)


def _hadamard(kind, device):
    """The normalised Sylvester matrix of order 128."""
    i = torch.arange(DIM, device=device)
    bits = i[:, None] & i[None]
    parity = sum((bits >> k) & 1 for k in range(7)) & 1
    return (1 - 2 * parity).to(kind) / math.sqrt(DIM)


def _basis(key, rotate, shift, kind):
    """Keys as the cache stores them: rotated, the mean taken off, rounded to BF16 once."""
    if not rotate:
        return key
    return (key.to(kind) @ _hadamard(kind, key.device) - shift.to(kind)).to(torch.bfloat16)


def _ancestors(parents):
    """[rows, nodes, nodes]: node i sees node j."""
    rows, nodes = parents.shape
    up = torch.arange(nodes, device=parents.device).expand(rows, nodes).clone()
    seen = torch.zeros(rows, nodes, nodes + 1, dtype=torch.bool, device=parents.device)
    above = torch.cat([parents.long(), parents.new_full((rows, 1), -1).long()], 1)
    for _ in range(nodes):
        seen.scatter_(2, torch.where(up < 0, nodes, up)[:, :, None], True)
        up = above.gather(1, torch.where(up < 0, nodes, up))
    return seen[:, :, :nodes]


def _plain_tree(s):
    case = s["case"]
    kind = torch.float32
    rows, nodes, hq, hk, pt = (case[k] for k in ("rows", "nodes", "heads_q", "heads_kv", "page_tokens"))
    ts = s["tensor_scales"] or (1.0, 1.0)
    key, value = _dequantize(s["blocks"][s["table"].long()].flatten(0, 1), hk, pt, kind)
    key, value = key.reshape(rows, -1, hk, DIM) * ts[0], value.reshape(rows, -1, hk, DIM) * ts[1]
    slots = s["slots"].long()
    key = torch.cat([key, s["tail_key"][slots].to(kind), _basis(s["draft_key"], case["rotate"], s["shift"], kind).to(kind)], 1)
    value = torch.cat([value, s["tail_value"][slots].to(kind), s["draft_value"].to(kind)], 1)
    query = s["query"].to(kind)
    if case["rotate"]:
        query = query @ _hadamard(kind, query.device)
    # which tokens the row's cache holds: the sink stands in for the first tokens of page zero (of the
    # rolling tail while there is no page)
    fp4, residual, sink = (s[k].long()[:, None] for k in ("fp4", "residual", "sink"))
    at = torch.arange(s["table"].shape[1] * pt, device=query.device)[None]
    tail = torch.arange(PAGE + SINK, device=query.device)[None]
    first = torch.where(fp4 > 0, 0, sink)
    seen = torch.cat([(at < fp4) & (at >= sink),
                      torch.where(tail < PAGE, (tail < residual) & (tail >= first), tail - PAGE < sink)], 1)
    seen = torch.cat([seen[:, None].expand(-1, nodes, -1), _ancestors(s["parents"])], 2)
    scores = torch.matmul(query.view(rows, nodes, hk, hq // hk, DIM).permute(0, 2, 3, 1, 4).reshape(rows, hk, -1, DIM),
                          key.permute(0, 2, 3, 1)) * DIM ** -0.5
    del key
    scores = scores.view(rows, hk, hq // hk, nodes, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(rows, hk, -1, scores.shape[-1]), value.permute(0, 2, 1, 3)).view(rows, hk, hq // hk, nodes, DIM)
    out = (out / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(rows, nodes, hq, DIM).to(torch.bfloat16)
    if s["counts"] is None:
        return out
    return torch.where((torch.arange(nodes, device=out.device) < s["counts"][:, None])[..., None, None], out, s["out"])


def _plain_verify(s):
    # in 64 bits: acceptance and the drawn token are decisions next to borders
    target, draft, tokens, parents = s["target"], s["draft"], s["tokens"].long(), s["parents"].long()
    rows, nodes, vocab = target.shape
    u = s["uniforms"].double()
    at = torch.arange(rows, device=target.device)
    here = torch.zeros(rows, dtype=torch.long, device=target.device)
    weights, mass = target[:, 0].double(), torch.ones(rows, dtype=torch.float64, device=target.device)
    path = torch.full((rows, nodes), -1, dtype=torch.int32, device=target.device)
    path[:, 0] = 0
    depth = torch.ones(rows, dtype=torch.long, device=target.device)
    for i in range(1, nodes):
        asked = parents[:, i] == here
        token = tokens[:, i]
        weight = weights[at, token]
        chance = 1.0 if draft is None else draft[at, here, token].double()
        taken = asked & (u[:, i] * chance * mass < weight)
        refused = asked & ~taken
        if draft is None:
            weights = weights.scatter(1, token[:, None], torch.where(refused, 0.0, weight)[:, None])
            mass = torch.where(refused, (mass - weight).clamp_min(0), mass)
        else:
            left = (weights / mass[:, None] - draft[at, here].double()).clamp_min(0)
            total = left.sum(1)
            refused &= total > 0
            weights = torch.where(refused[:, None], left, weights)
            mass = torch.where(refused, total, mass)
        path[at, torch.where(taken, depth, 0)] = torch.where(taken, i, 0).to(torch.int32)
        depth += taken
        here = torch.where(taken, i, here)
        weights = torch.where(taken[:, None], target[:, i].double(), weights)
        mass = torch.where(taken, 1.0, mass)
    # what the refused children leave of it may be nothing at all: then the node's own distribution stands
    weights = torch.where(weights.sum(1, keepdim=True) > 0, weights, target[at, here].double())
    sums = weights.cumsum(1)
    drawn = (sums <= u[:, :1] * sums[:, -1:]).sum(1)
    last = torch.where(weights > 0, torch.arange(vocab, device=target.device), 0).amax(1)
    return dict(accepted=path, counts=depth.to(torch.int32), next_tokens=torch.minimum(drawn, last).to(torch.int32))


def _quantize(groups):
    """E2M1 codes and E4M3 scale bytes of ``[..., 16]`` groups under the amax/6 rule."""
    groups = groups.float()
    scale = (groups.abs().amax(-1) * torch.tensor(1.0 / 6.0, dtype=torch.float32, device=groups.device)).clamp(max=448.0)
    scale = scale.to(torch.float8_e4m3fn)
    x = groups * (1.0 / (scale.float() + 1.0e-30))[..., None]
    m = x.abs()
    code = sum(((m > mid) if k % 2 == 0 else (m >= mid)).to(torch.uint8)
               for k, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = code | (torch.signbit(x).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8)


def _plain_commit(s):
    case = s["case"]
    rows, nodes, hk = case["rows"], case["nodes"], case["heads_kv"]
    old, count = s["seq_lens"].long(), s["counts"].long()
    new = old + count
    step = torch.arange(nodes, device=old.device)[None]
    position = old[:, None] + step
    valid = step < count[:, None]
    boundary = new // PAGE * PAGE  # tokens before it end up in full pages
    node = s["accepted"].long().clamp_min(0)
    row = torch.arange(rows, device=old.device)[:, None].expand(rows, nodes)
    slot = s["slots"].long()[:, None].expand(rows, nodes)
    key = s["draft_key"][:, row, node]
    shift = s["shift"]
    key = _basis(key, case["rotate"], None if shift is None else shift[:, None, None], torch.float32)
    value = s["draft_value"][:, row, node]
    fills = boundary > old // PAGE * PAGE
    early = valid & (~fills[:, None] | (position < boundary[:, None]))
    for tail, source in ((s["tail_key"], key), (s["tail_value"], value)):
        tail[:, slot[early], position[early] % PAGE] = source[:, early]
        first = valid & (position < SINK)
        tail[:, slot[first], PAGE + position[first]] = source[:, first]
    if s["filled"]:
        at = torch.tensor([i for i, _ in s["filled"]], device=old.device)
        page = s["table"][at, torch.tensor([c for _, c in s["filled"]], device=old.device)].long()
        full_key, full_value = (t[:, s["slots"].long()[at], :PAGE] for t in (s["tail_key"], s["tail_value"]))
        layers, n = full_key.shape[:2]
        kc, ks = _quantize(full_key.reshape(layers, n, PAGE, hk, 8, 16))
        vc, vs = _quantize(full_value.permute(0, 1, 3, 4, 2).reshape(layers, n, hk, DIM, 8, 16))
        ks = ks.view(layers, n, 4, 32, hk, 2, 4).permute(0, 1, 4, 5, 3, 2, 6)
        vs = vs.view(layers, n, hk, 4, 32, 2, 4).permute(0, 1, 2, 5, 4, 3, 6)
        whole = torch.cat([x.reshape(layers, n, -1) for x in (kc, ks, vc, vs)], 2)
        for layer, blocks in enumerate(s["blocks"]):
            blocks[page] = whole[layer]
    late = valid & ~early
    for tail, source in ((s["tail_key"], key), (s["tail_value"], value)):
        tail[:, slot[late], position[late] % PAGE] = source[:, late]
    fp4 = torch.where(new > 0, (new - 1) // PAGE * PAGE, 0)
    return _commit_outputs(s, *(x.to(torch.int32) for x in (new, fp4, new - fp4, new.clamp_max(SINK))))


# ---- the floor of a pass, and its result in 64 bits ------------------------------------------------


def work(case):
    if case["op"] == "tree":
        hq, hk = case["heads_q"], case["heads_kv"]
        total = flops = 0
        for n, count in zip(_lengths(case), _counts(case)):
            sink, fp4, residual = _split(n)
            bf16 = residual + (sink if fp4 else 0) + count
            total += fp4 * hk * 144 + bf16 * hk * 512 + count * hq * DIM * 4
            flops += 4 * DIM * hq * count * (n + count / 2)
        return dict(bytes=total, flops=flops)
    if case["op"] == "verify":  # one distribution per row (two with a drafter) has to be read whole
        rows, size = case["rows"], 2 if case["bf16"] else 4
        return dict(bytes=rows * case["vocab"] * size * (2 if case["drafter"] else 1) + rows * case["nodes"] * 20,
                    flops=rows * case["vocab"] * (4 if case["drafter"] else 1))
    token = case["layers"] * case["heads_kv"] * DIM * 2 * 2
    total = 0
    for n, a in _committed(case):
        total += 2 * a * token
        if (n + a) // PAGE > n // PAGE:  # read a page's tokens, write its codes and scales
            total += PAGE * token + PAGE * case["layers"] * case["heads_kv"] * 144
    return dict(bytes=total, flops=total)


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers only
    s = prepare(case, seed)
    return _exact_tree(s) if case["op"] == "tree" else _exact_commit(s)


def _walsh(x):
    """x times the normalised Sylvester matrix, by butterflies, in 64 bits."""
    x = x.double()
    for k in range(7):
        y = x.unflatten(-1, (DIM >> (k + 1), 2, 1 << k))
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).flatten(-3)
    return x / math.sqrt(DIM)


def _exact_page_values(blocks, heads, pt):
    """K and V of whole blocks ``[n, bytes]`` in 64 bits, as [n, heads, tokens, 128]: byte by byte from the
    layout's own offsets."""
    device = blocks.device
    lut = torch.tensor(E2M1, dtype=torch.float64, device=device)
    h = torch.arange(heads, device=device)[:, None, None]
    t = torch.arange(pt, device=device)[None, :, None]
    c = torch.arange(DIM, device=device)[None, None, :]
    codes, scales = pt * 64 * heads, pt * 8 * heads

    def atom(row, group):  # (row, group) of a head's scale tile of 512-byte atoms
        return (group // 4) * 512 + (row % 32) * 16 + (row // 32) * 4 + group % 4

    if pt == PAGE:
        key_at = t * heads * 64 + h * 64 + c // 2
        key_scale_at = codes + h * 1024 + atom(t, c // 16)
        value_at = codes + scales + h * DIM * 64 + c * 64 + t // 2
        value_scale_at = 2 * codes + scales + h * 1024 + atom(c, t // 16)
    else:
        key_at = h * 4096 + t * 64 + (((c // 32) ^ ((t >> 1) & 3)) * 16) + (c // 2) % 16
        key_scale_at = codes + h * 512 + (c // 64) * 256 + (t % 32) * 8 + (t // 32) * 4 + (c // 16) % 4
        value_at = codes + scales + h * 4096 + c * 32 + (((t // 32) ^ ((c >> 2) & 1)) * 16) + (t // 2) % 16
        value_scale_at = 2 * codes + scales + h * 512 + atom(c, t // 16)

    def read(at, scale_at, odd):
        byte = blocks[:, at.expand(heads, pt, DIM).reshape(-1)].to(torch.int32)
        nibble = torch.where((odd.expand(heads, pt, DIM).reshape(-1) & 1) == 1, byte >> 4, byte & 15)
        scale = blocks[:, scale_at.expand(heads, pt, DIM).reshape(-1)].view(torch.float8_e4m3fn).double()
        return (lut[nibble] * scale).view(-1, heads, pt, DIM)

    return read(key_at, key_scale_at, c), read(value_at, value_scale_at, t)


def _exact_tree(s):
    """One row after another, one run of pages after another: sums of exp(score) and of exp(score) * value
    over everything a node sees, with one reference score per query."""
    case = s["case"]
    rows, nodes, hq, hk, pt = (case[k] for k in ("rows", "nodes", "heads_q", "heads_kv", "page_tokens"))
    ts = s["tensor_scales"] or (1.0, 1.0)
    out = s["out"].double()
    for r in range(rows):
        count = nodes if s["counts"] is None else int(s["counts"][r])
        fp4, residual, sink = (int(s[k][r]) for k in ("fp4", "residual", "sink"))
        query, draft = s["query"][r, :count].double(), s["draft_key"][r, :count].double()
        if case["rotate"]:
            query = _walsh(query)
            draft = (_walsh(draft) - s["shift"].double()).to(torch.bfloat16).double()
        query = query.view(count, hk, hq // hk, DIM).permute(1, 2, 0, 3) / math.sqrt(DIM)  # [hk, g, count, 128]
        slot = int(s["slots"][r])
        tail_key, tail_value = s["tail_key"][slot].double(), s["tail_value"][slot].double()
        lo = 0 if fp4 else sink  # without a page the sink is the head of the rolling tail
        key = torch.cat([tail_key[lo:residual], tail_key[PAGE:PAGE + sink], draft]).permute(1, 0, 2)
        value = torch.cat([tail_value[lo:residual], tail_value[PAGE:PAGE + sink],
                           s["draft_value"][r, :count].double()]).permute(1, 0, 2)
        parent = s["parents"][r].tolist()
        family = torch.zeros(count, count, dtype=torch.bool)
        for i in range(count):
            j = i
            while j >= 0:
                family[i, j] = True
                j = parent[j]
        blind = torch.zeros(count, key.shape[1], dtype=torch.bool)
        blind[:, key.shape[1] - count:] = ~family
        score = torch.einsum("hgnd,hld->hgnl", query, key).masked_fill(blind.to(key.device), -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = torch.exp(score - top)
        total, acc = weight.sum(-1, keepdim=True), torch.einsum("hgnl,hld->hgnd", weight, value)
        ids = s["table"][r, :fp4 // pt].long()
        step = max(1, 100_000_000 // (hk * DIM * pt))
        for start in range(0, ids.shape[0], step):
            key, value = _exact_page_values(s["blocks"][ids[start:start + step]], hk, pt)
            key = key.permute(1, 0, 2, 3).reshape(hk, -1, DIM)
            value = value.permute(1, 0, 2, 3).reshape(hk, -1, DIM)
            score = torch.matmul(query.reshape(hk, -1, DIM), key.transpose(1, 2)) * ts[0]
            if start == 0:
                score[..., :sink] = -math.inf
            score = score.view(*query.shape[:3], -1)
            peak = torch.maximum(top, score.amax(-1, keepdim=True))
            weight, back = torch.exp(score - peak), torch.exp(top - peak)
            total = total * back + weight.sum(-1, keepdim=True)
            acc = acc * back + torch.matmul(weight.view(hk, -1, weight.shape[-1]), value).view(acc.shape) * ts[1]
            top = peak
        out[r, :count] = (acc / total).permute(2, 0, 1, 3).reshape(count, hq, DIM)
    return out


def _exact_commit(s):
    """Token by token, at each token's own place; the filled pages' rounding has no value in 64 bits."""
    case = s["case"]
    key, value = s["tail_key"].double(), s["tail_value"].double()
    for r, (n, count) in enumerate(_committed(case)):
        slot = int(s["slots"][r])
        path = s["accepted"][r, :count].long()
        k = s["draft_key"][:, r, path].double()
        v = s["draft_value"][:, r, path].double()
        if case["rotate"]:
            k = _walsh(k) - s["shift"].double()[:, None]
        for i in range(count):
            rows = [(n + i) % PAGE] + ([PAGE + n + i] if n + i < SINK else [])
            for at in rows:
                key[:, slot, at], value[:, slot, at] = k[:, i], v[:, i]
    out = dict(tail_key=key, tail_value=value, seq_lens=None, fp4=None, residual=None, sink=None)
    if s["filled"]:
        out |= dict(key_pages=None, value_pages=None)
    return out
