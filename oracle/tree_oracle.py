"""Plain 64-bit statements of the speculative-decoding operators: attention of a drafted tree over the
dequantized cache, verification of the tree, and where a commit puts the accepted tokens.

The project this repository follows has none of them (its plugin refuses speculative decoding), so parity is
unpinned by construction; the cache layout and the keys' basis come from the pinned ``nvfp4_oracle``.
"""

import math

import numpy as np
import torch

from . import nvfp4_oracle as base

PAGE = 128
MAX_NODES = 64


def ancestors(parents):
    """[nodes, nodes] bool: node i sees node j. An entry that names no earlier node makes a root."""
    nodes = len(parents)
    seen = torch.zeros(nodes, nodes, dtype=torch.bool)
    for i, parent in enumerate(parents):
        if 0 <= parent < i:
            seen[i] = seen[parent]
        seen[i, i] = True
    return seen


def cache_values(blocks: torch.Tensor, heads: int, page_tokens: int):
    """A flat ``[blocks, bytes]`` cache -> FP64 K and V ``[blocks, tokens, H, 128]``."""
    b, pt, h = blocks.cpu(), page_tokens, heads
    codes, scales = pt * 64 * h, pt * 8 * h
    kc = b[:, :codes]
    kc = kc.reshape(-1, pt, h, 64) if pt == PAGE else kc.reshape(-1, h, pt, 64).permute(0, 2, 1, 3)
    key = base.dequantize_key_pages(kc, b[:, codes:codes + scales].reshape(-1, h, pt * 8))
    value = base.dequantize_value_pages(b[:, codes + scales:2 * codes + scales].reshape(-1, h, 128, pt // 2),
                                        b[:, 2 * codes + scales:].reshape(-1, h, pt * 8))
    return key.double(), value.double()


def tree_attention(*, query, draft_key, draft_value, parents, key, value, page_ids, fp4, tail_key, tail_value,
                   residual, sink, softmax_scale, rotate=False, shift=None, typical=False):
    """One row: ``query [nodes, Hq, 128]``, drafts ``[nodes, H, 128]`` (BF16), ``key`` / ``value`` the FP64 cache pages
    (tensor scales multiplied in), ``page_ids`` the row's pages, ``tail_* [>= 128, H, 128]`` BF16 (sink behind row
    128). Returns the FP64 result ``[nodes, Hq, 128]`` and how far a kernel may be from it.

    The allowance, per output element, first order with 5 % for the rest: the output's rounding to BF16 (2^-8
    relative); each probability's rounding to BF16 (2^-8; FP16 pages round by 2^-11); and the scores' errors. A
    score is a sum of 128 products in FP32 whose terms add up to A = sum |q||k| * scale: 2^-16 A covers the
    products' and sums' rounding (128 additions of 2^-24), its scaling and the exponential's argument; a rotated
    query is rounded to FP16 (2^-11), so its scores carry 2^-11 A more. Against FP4 pages a query is four FP4
    terms, each the rounding of what is left: the E4M3 scale of a group is at most 2^-4 off amax / 6, and half
    the widest E2M1 step is one scale, so a term leaves at most 17/16 / 6 < 0.178 of the group's largest value (a
    value clipped at six scales leaves less), four leave 0.178^4. Scaled so that the largest query value
    of its tile lies in [2^10, 2^11), or its own where that is below 2^-5 of the tile's, a term whose scale falls to
    E4M3's smallest (2^-9) or below leaves at most 3 x 2^-9, under 2^-16 of that value: of the head's largest, and of 32
    times the query's own. An error d in a score is a relative error d of its probability, and sum p v / sum p
    moves by at most sum p_t (d_t + mean d) |v_t|.

    That adds every token's error to every other's, so over thousands of tokens it exceeds the result. With ``typical``
    the second return is instead the root mean square error per (node, head) that independent roundings come to: the
    same bounds, a token's 128 products and the tokens added in squares, page probabilities by FP16's 2^-11."""
    nodes, hq, _ = query.shape
    h = draft_key.shape[1]
    g = hq // h
    q = query.double()
    if rotate:
        q = base_rotate(q)
    dk = base.key_cache_basis(draft_key, rotate=rotate, shift=shift).double()
    keys, values, seen = [], [], []

    def add(k, v, mask):
        keys.append(k)
        values.append(v)
        seen.append(mask)

    if fp4:
        k = key[page_ids].reshape(-1, h, 128)[:fp4]
        v = value[page_ids].reshape(-1, h, 128)[:fp4]
        add(k, v, (torch.arange(fp4) >= sink).expand(nodes, fp4))
    if residual:
        first = 0 if fp4 else sink
        add(tail_key[:residual].double(), tail_value[:residual].double(),
            (torch.arange(residual) >= first).expand(nodes, residual))
    if sink:
        add(tail_key[PAGE:PAGE + sink].double(), tail_value[PAGE:PAGE + sink].double(),
            torch.ones(nodes, sink, dtype=torch.bool))
    add(dk, draft_value.double(), ancestors(parents))
    k, v, mask = torch.cat(keys), torch.cat(values), torch.cat(seen, 1)
    left = q.abs().reshape(nodes, hq, 8, 16).amax(3) * 0.178 ** 4
    own = q.abs().amax(2)  # each query's largest value; below, the largest of each KV head
    tile = own.reshape(nodes, h, g).amax((0, 2)).repeat_interleave(g)
    left = torch.maximum(left, 2.0 ** -16 * torch.minimum(tile[None], 32 * own)[:, :, None])
    out = torch.empty(nodes, hq, 128, dtype=torch.float64)
    allowed = torch.empty_like(out)
    rms = torch.empty(nodes, hq, dtype=torch.float64)
    for head in range(hq):
        kh, vh = k[:, head // g], v[:, head // g]
        s = (q[:, head] @ kh.T * softmax_scale).masked_fill(~mask, -math.inf)
        p = torch.softmax(s, 1)
        terms = q[:, head].abs() @ kh.abs().T * softmax_scale
        d = terms * (2.0 ** -16 + (2.0 ** -11 if rotate else 0.0))
        d[:, :fp4] += left[:, head] @ kh[:fp4].abs().reshape(fp4, 8, 16).sum(2).T * softmax_scale
        d = torch.where(mask, d, 0.0)
        out[:, head] = p @ vh
        weight = p * (d + (p * d).sum(1, keepdim=True) + 2.0 ** -8)
        allowed[:, head] = 1.05 * (weight @ vh.abs() + 2.0 ** -8 * out[:, head].abs()) + 1e-7
        if typical:
            e = (terms * 2.0 ** -16) ** 2
            if rotate:
                e += (2.0 ** -11 * softmax_scale) ** 2 * (q[:, head] ** 2 @ kh.T ** 2)
            e[:, :fp4] += softmax_scale ** 2 * (left[:, head] ** 2 @ (kh[:fp4] ** 2).reshape(fp4, 8, 16).sum(2).T)
            e += torch.where(torch.arange(len(kh)) < fp4, 2.0 ** -22, 2.0 ** -16)
            variance = (p ** 2 * e) @ vh ** 2 + (2.0 ** -8 * out[:, head]) ** 2
            rms[:, head] = variance.mean(1).sqrt()
    return out, rms if typical else allowed


def base_rotate(x):
    """The normalised Sylvester Hadamard product in 64 bits."""
    n = x.shape[-1]
    i = np.arange(n)
    parity = np.zeros((n, n), dtype=np.int64)
    for b in range(7):
        parity ^= ((i[:, None] & i[None]) >> b) & 1
    return x @ torch.from_numpy((1.0 - 2.0 * parity) / math.sqrt(n))


def verify(target, tokens, parents, uniforms, draft=None, count=None):
    """One row's walk in FP64: ``target [nodes, vocab]``, the rest ``[nodes]``. Returns (path, next token, the
    smallest relative distance of any decision from its border)."""
    nodes, vocab = target.shape
    count = nodes if count is None else count
    if count == 0:
        return [], -1, math.inf
    target = target.astype(np.float64)
    draft = None if draft is None else draft.astype(np.float64)
    here, path, margin = 0, [0], math.inf
    w, mass = target[0].copy(), 1.0
    for c in range(1, count):
        if parents[c] != here:
            continue
        x = int(tokens[c])
        known = 0 <= x < vocab
        q = 1.0 if draft is None or not known else draft[here, x]
        weight = w[x] if known else 0.0
        left = float(uniforms[c]) * q * mass
        if left != weight:
            margin = min(margin, abs(left - weight) / max(left, weight))
        if left < weight:
            here = c
            path.append(c)
            w, mass = target[c].copy(), 1.0
        elif draft is None:
            mass = max(mass - weight, 0.0)
            if known:
                w[x] = 0.0
        else:
            rest = np.maximum(w / mass - draft[here], 0.0)
            if rest.sum() > 0:
                w, mass = rest, rest.sum()
    if not w.sum() > 0:
        w = target[here]
    sums = np.cumsum(w)
    positive = np.flatnonzero(w > 0)
    if not len(positive):
        return path, 0, margin
    goal = float(uniforms[0]) * sums[-1]
    over = np.flatnonzero((sums > goal) & (w > 0))
    if len(over):
        at = int(over[0])
        margin = min(margin, (sums[at] - goal) / sums[-1], (goal - (sums[at] - w[at])) / sums[-1] if goal > 0 else math.inf)
        return path, at, margin
    return path, int(positive[-1]), margin


def commit_positions(n, count):
    """(token number, tail row) of each accepted token of a row of ``n`` committed ones, and whether a page fills."""
    return [(n + i, (n + i) % PAGE) for i in range(count)], (n + count) // PAGE > n // PAGE


def outside_typical(got, want, typical):
    """How many (node, head) results of a row lie further from the FP64 one than three times what independent
    roundings come to. (Over a head's 128 channels and many tokens the root mean square is within a few percent of its
    expectation, and the roundings' bounds are taken for their spread, 1.7 times it for evenly spread errors: a right
    result stays below one.)"""
    off = ((got - want) ** 2).mean(-1).sqrt()
    return int((off > 3 * typical).sum())
