"""Speculative decoding over the paged NVFP4 cache: score a tree of drafted tokens, verify it, commit it.

OpenBitSys/BitDecoding-FP4 has no counterpart: its plugin refuses speculative decoding because its decode
kernel attends one query token per sequence (src/nvfp4_vllm/guards.py). The interface is this package's own,
shaped like the one-token path (``fp4_decode`` / ``KVCacheWriter``): the same cache regions, page table, BF16
tail and sink, lengths as device tensors, and no host synchronisation on a step.

One step of a batch, per layer and then once:

    out = tree_decode(query, draft_key, draft_value, parents, *regions, page_table, seqused_fp4, ...)
    verdict = verify_drafts(target_probs, tokens, parents, uniforms, draft_probs=...)
    lengths = committer(draft_keys, draft_values, verdict.accepted, verdict.accepted_counts, ...)

Node 0 of a tree is the sequence's newest token, decided in the step before but not in the cache yet; the
others are drafts. ``parents[r, i] < i`` is the parent of node ``i``. A row may use fewer than ``nodes`` nodes
(``node_counts``).
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

import bdfp4

from .interface import SINK_TOKENS
from .quantize_kv_kernel import HEAD_DIM, PAGE_SIZE, KVCacheWriter
from .scale_mode import DEFAULT_SCALE_MODE, scale_format

MAX_TREE_NODES = 64
ROTATIONS = ("none", "hadamard")


def _launch(call, args, device: torch.device) -> None:
    """``call`` on the device's current stream; the tensors' device is made current if it is not. (The stream's
    handle alone: making a stream object costs 4 us.)"""
    if device.index == torch._C._cuda_getDevice():
        call(args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            call(args, torch._C._cuda_getCurrentRawStream(device.index))


# The checks give the address back, so that a call asks each tensor once.


def _int32(tensor, name: str, shape: tuple, device) -> int:
    if (
        not isinstance(tensor, torch.Tensor) or tensor.dtype is not torch.int32 or tensor.device != device
        or tensor.shape != shape or (shape[-1] > 1 and tensor.stride(-1) != 1)
    ):
        raise ValueError(f"{name} must be INT32 {list(shape)} on {device}, dense along its last axis")
    return tensor.data_ptr()


def _tree_tensor(tensor, name: str, shape: tuple, device) -> tuple:
    """BF16 ``[..., nodes, heads, 128]`` with free leading strides: its address, then those strides (where a dimension
    has one entry its stride means nothing: that of a dense node stands in)."""
    if (
        isinstance(tensor, torch.Tensor) and tensor.dtype is torch.bfloat16 and tensor.device == device
        and tensor.shape == shape
    ):
        address, (*outer, head, inner) = tensor.data_ptr(), tensor.stride()
        ok = inner == 1 and (head == HEAD_DIM or shape[-2] == 1) and address % 16 == 0
        for i, size in enumerate(shape[:-2]):
            if size == 1:
                outer[i] = shape[-2] * HEAD_DIM
            elif outer[i] % 8:
                ok = False
        if ok:
            return address, *outer
    raise ValueError(f"{name} must be BF16 {list(shape)} on {device}, dense within a node and 16-byte aligned")


def _parents(parents, rows: int, nodes: int, device) -> tuple[int, int]:
    """``[rows, nodes]``, or ``[nodes]`` for one tree that every row shares: its address and row stride."""
    if isinstance(parents, torch.Tensor) and parents.ndim == 1 and nodes == parents.shape[0]:
        parents = parents.expand(rows, nodes)
    return _int32(parents, "parents", (rows, nodes), device), parents.stride(0)


def _cuda_device(tensor, name: str) -> torch.device:
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return tensor.device


def _check_values(bad: torch.Tensor, message: str) -> None:
    if bool(bad.any()):
        raise ValueError(message)


def _check_regions(key_pages_fp4, key_scales, value_pages_fp4, value_scales, device) -> tuple:
    """(pages, page tokens, KV heads, addresses, page pitches) of the four regions of an NVFP4 cache."""
    packed, scales = (torch.uint8, torch.float4_e2m1fn_x2), (torch.uint8, torch.float8_e4m3fn)
    if not isinstance(key_pages_fp4, torch.Tensor) or key_pages_fp4.device != device:
        raise ValueError(f"key_pages_fp4 must be a CUDA tensor on {device}")
    if key_pages_fp4.dtype not in packed or key_pages_fp4.ndim != 4 or key_pages_fp4.shape[3] * 2 != HEAD_DIM:
        raise ValueError("key_pages_fp4 must be packed FP4 with shape [pages, 128, heads_kv, 64]")
    pages, page, heads, _ = key_pages_fp4.shape
    if page == PAGE_SIZE:
        key_inner, scale_shape = (heads * 64, 64, 1), (pages, 32, 4, 1, 4, 2, heads)
        key_sf = value_sf = (16, 4, 1024, 1, 512, 1024)
        value_scale_shape = scale_shape
    elif page == 64:
        key_inner, scale_shape = (64, 64 * 64, 1), (pages, 32, 2, 1, 4, 2, heads)
        key_sf, value_sf = (8, 4, 512, 1, 256, 512), (16, 4, 512, 1, 512, 512)
        value_scale_shape = (pages, 32, 4, 1, 4, 1, heads)
    else:
        raise ValueError("key_pages_fp4 must be packed FP4 with shape [pages, 128, heads_kv, 64]")
    half = page // 2
    addresses, pitches = [], []
    for tensor, name, kinds, shape, inner in (
        (key_pages_fp4, "key_pages_fp4", packed, (pages, page, heads, 64), key_inner),
        (key_scales, "key_scales", scales, scale_shape, key_sf),
        (value_pages_fp4, "value_pages_fp4", packed, (pages, heads, HEAD_DIM, half), (HEAD_DIM * half, half, 1)),
        (value_scales, "value_scales", scales, value_scale_shape, value_sf),
    ):
        if not isinstance(tensor, torch.Tensor) or tensor.device != device:
            raise ValueError(f"{name} must be a CUDA tensor on {device}")
        if tensor.shape != shape or tensor.dtype not in kinds:
            held = "packed FP4" if kinds is packed else "E4M3 scale bytes"
            raise ValueError(f"{name} must hold {held} with shape {shape}")
        strides, address = tensor.stride(), tensor.data_ptr()
        pitch = strides[0] if pages > 1 else tensor.numel()
        if strides[1:] != inner or pitch % 16 or address % 16:
            raise ValueError(f"{name} must be in the quantizer's layout, dense within a page, with a 16-byte page pitch")
        addresses.append(address)
        pitches.append(pitch)
    return pages, page, heads, addresses, pitches


@functools.lru_cache(maxsize=1024)
def tree_workspace_bytes(rows: int, nodes: int, heads_q: int, heads_kv: int) -> int:
    """Bytes of the workspace :func:`tree_decode` needs for these sizes (any contents)."""
    size = int(bdfp4.library().bdfp4_tree_workspace_bytes(rows, nodes, heads_q, heads_kv))
    if size <= 0:
        raise ValueError(f"no tree decode for rows={rows}, nodes={nodes}, heads_q={heads_q}, heads_kv={heads_kv}")
    return size


def tree_decode(
    query: torch.Tensor,
    draft_key: torch.Tensor,
    draft_value: torch.Tensor,
    parents: torch.Tensor,
    key_pages_fp4: torch.Tensor,
    key_scales: torch.Tensor,
    value_pages_fp4: torch.Tensor,
    value_scales: torch.Tensor,
    fp4_page_table: torch.Tensor,
    seqused_fp4: torch.Tensor,
    *,
    node_counts: torch.Tensor | None = None,
    residual_key_pages_bf16: torch.Tensor | None = None,
    residual_value_pages_bf16: torch.Tensor | None = None,
    residual_page_ids: torch.Tensor | None = None,
    seqused_residual: torch.Tensor | None = None,
    seqused_sink: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    query_rotation: str = "none",
    key_shift: torch.Tensor | None = None,
    tensor_scales: tuple[float, float] | None = None,
    scale_mode: str = DEFAULT_SCALE_MODE,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    trusted_metadata: bool = False,
    error_word: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of a tree of drafted tokens per row over the FP4 cache, BF16 tail and sink included.

    ``query`` is BF16 ``[rows, nodes, heads_q, 128]`` and ``draft_key`` / ``draft_value`` BF16 ``[rows, nodes,
    heads_kv, 128]`` (1 to 64 nodes; strides between rows and nodes are free). Node ``i`` attends to the row's
    whole cache, to itself and to its ancestors under ``parents`` (INT32 ``[rows, nodes]``, or ``[nodes]`` for one
    tree that all rows share; an entry that is not the number of an earlier node makes a root). ``node_counts``
    (INT32 ``[rows]``, 0 to ``nodes``) gives each row's own number of nodes: what lies behind it is not read, and
    its output is left as it was (zeros without ``out``).

    The cache regions, ``fp4_page_table``, ``seqused_fp4`` and the ``residual_*`` / ``seqused_*`` arguments are
    those of :func:`nvfp4_decode_kernel.fp4_decode`; MXFP4 caches are not served. A tail may have any number of sink
    rows from 0 to 16 behind its 128 (``fp4_decode`` takes 16 with ``seqused_sink``, none without). Unlike there,
    neither the query nor the probabilities are rounded to one FP4 value: cache values enter the products exactly,
    queries as four FP4 terms (up to 1.0e-3 of the largest of 16 channels is lost; FP16 against BF16 tokens) and
    probabilities as FP16 (BF16 against BF16 tokens). A draft value that is not finite may reach every node of its
    row: its weight elsewhere is zero, not absent.

    Keys in the cache are rotated and shifted; ``query_rotation="hadamard"`` rotates the queries and the draft
    keys alike, and ``key_shift`` (FP32 ``[heads_kv, 128]``, already rotated) is subtracted from the draft keys,
    which are then rounded to BF16, as the tail writer does. ``tensor_scales`` is ``(key, value)`` of the pages.

    ``workspace`` (uint8, at least :func:`tree_workspace_bytes`, 16-byte aligned) makes the call allocation-free
    together with ``out`` (BF16 ``[rows, nodes, heads_q, 128]``, dense within a node, apart from the inputs); calls
    that may overlap on the GPU, captured ones included, need a workspace each. ``error_word`` (INT32 ``[1]``)
    collects ``bdfp4.DEV_*`` bits. ``trusted_metadata`` skips the checks that read device values.
    """
    device = _cuda_device(query, "query")
    if query.ndim != 4 or query.shape[3] != HEAD_DIM:
        raise ValueError("query must be BF16 [rows, nodes, heads_q, 128]")
    rows, nodes, heads_q, _ = query.shape
    if scale_mode != DEFAULT_SCALE_MODE and scale_format(scale_mode) != "nvfp4":
        raise NotImplementedError("tree decode is built for NVFP4 caches only")
    if rows < 1 or nodes < 1:
        raise ValueError("tree decode needs at least one row and one node")
    if nodes > MAX_TREE_NODES:
        raise NotImplementedError(f"a tree holds at most {MAX_TREE_NODES} nodes, got {nodes}")
    pages, page_tokens, heads_kv, addresses, pitches = _check_regions(
        key_pages_fp4, key_scales, value_pages_fp4, value_scales, device)
    if heads_kv < 1 or heads_q < 1 or heads_q % heads_kv:
        raise ValueError("heads_q must be divisible by heads_kv")
    a = bdfp4.TreeArgs()
    a.rows, a.nodes, a.heads_q, a.heads_kv = rows, nodes, heads_q, heads_kv
    a.key_codes, a.key_scales, a.value_codes, a.value_scales = addresses
    a.key_codes_pitch, a.key_scales_pitch, a.value_codes_pitch, a.value_scales_pitch = pitches
    a.pages, a.page_tokens = pages, page_tokens
    shape = (rows, nodes, heads_q, HEAD_DIM)
    a.query, a.query_row_stride, a.query_node_stride = _tree_tensor(query, "query", shape, device)
    draft_shape = (rows, nodes, heads_kv, HEAD_DIM)
    a.draft_key, a.draft_key_row_stride, a.draft_key_node_stride = _tree_tensor(draft_key, "draft_key", draft_shape, device)
    a.draft_value, a.draft_value_row_stride, a.draft_value_node_stride = _tree_tensor(
        draft_value, "draft_value", draft_shape, device)
    a.parents, a.parents_row_stride = _parents(parents, rows, nodes, device)
    if node_counts is not None:
        a.node_counts = _int32(node_counts, "node_counts", (rows,), device)
    if not isinstance(fp4_page_table, torch.Tensor) or fp4_page_table.ndim != 2:
        raise ValueError("fp4_page_table must be row-major INT32 with shape [rows, max_pages]")
    columns = fp4_page_table.shape[1]
    a.page_table = _int32(fp4_page_table, "fp4_page_table", (rows, columns), device)
    a.page_table_stride, a.max_pages_per_row = fp4_page_table.stride(0) if rows > 1 else columns, columns
    if a.page_table_stride < columns:
        raise ValueError("fp4_page_table must be row-major INT32 with shape [rows, max_pages]")
    a.seqused_fp4 = _int32(seqused_fp4, "seqused_fp4", (rows,), device)
    if query_rotation not in ROTATIONS:
        raise ValueError(f"query_rotation must be one of {list(ROTATIONS)}, got {query_rotation!r}")
    if key_shift is not None and (
        not isinstance(key_shift, torch.Tensor) or key_shift.dtype is not torch.float32 or key_shift.device != device or not key_shift.is_contiguous()
        or tuple(key_shift.shape) != (heads_kv, HEAD_DIM)
    ):
        raise ValueError(f"key_shift must be contiguous FP32 [{heads_kv}, {HEAD_DIM}] on {device}")
    a.rotate = int(query_rotation == "hadamard")
    if key_shift is not None:
        a.key_shift = key_shift.data_ptr()
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale) or scale <= 0.0:
        raise ValueError("softmax_scale must be finite and positive")
    key_ts = value_ts = 1.0
    if tensor_scales is not None:
        key_ts, value_ts = map(float, tensor_scales)
        if not (0.0 < key_ts < math.inf and 0.0 < value_ts < math.inf):
            raise ValueError("tensor_scales must be finite and positive")
    a.softmax_scale, a.key_tensor_scale, a.value_tensor_scale = scale, key_ts, value_ts

    residual = (residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, seqused_residual)
    has_residual = residual[0] is not None
    if has_residual != (residual[1] is not None) or has_residual != (residual[2] is not None) or has_residual != (
            residual[3] is not None):
        raise ValueError("residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, and "
                         "seqused_residual must be provided together")
    if seqused_sink is not None and not has_residual:
        raise ValueError("seqused_sink needs the BF16 residual arguments")
    slots = 0
    if has_residual:
        tail_shape = residual[0].shape if isinstance(residual[0], torch.Tensor) else ()
        slots = tail_shape[0] if tail_shape else 0
        for tensor, name in ((residual[0], "residual_key_pages_bf16"), (residual[1], "residual_value_pages_bf16")):
            if (
                not isinstance(tensor, torch.Tensor) or tensor.dtype is not torch.bfloat16 or tensor.device != device
                or not tensor.is_contiguous() or tensor.shape != tail_shape or len(tail_shape) != 4 or tail_shape[1] < PAGE_SIZE
                or tail_shape[2:] != (heads_kv, HEAD_DIM)
            ):
                raise ValueError(f"{name} must be contiguous BF16 [slots, {PAGE_SIZE} + sink tokens, {heads_kv}, {HEAD_DIM}] "
                                 f"on {device}")
        sink_rows = min(tail_shape[1] - PAGE_SIZE, SINK_TOKENS)
        a.tail_key, a.tail_value = residual[0].data_ptr(), residual[1].data_ptr()
        a.tail_slot_stride, a.tail_slots = tail_shape[1] * heads_kv * HEAD_DIM, slots
        a.tail_slot_ids = _int32(residual_page_ids, "residual_page_ids", (rows,), device)
        a.seqused_residual = _int32(seqused_residual, "seqused_residual", (rows,), device)
        if seqused_sink is not None:
            a.seqused_sink = _int32(seqused_sink, "seqused_sink", (rows,), device)
    if error_word is not None:
        a.error_word = _int32(error_word, "error_word", (1,), device)
    if not trusted_metadata:
        per_step = PAGE_SIZE // page_tokens
        most = columns // per_step * PAGE_SIZE
        _check_values((seqused_fp4 < 0) | (seqused_fp4 > most) | (seqused_fp4 % PAGE_SIZE != 0),
                      f"seqused_fp4 values must be page-aligned and in [0, {most}]")
        entry = torch.arange(columns, device=device)[None]
        _check_values((entry < (seqused_fp4 // page_tokens)[:, None]) & ((fp4_page_table < 0) | (fp4_page_table >= pages)),
                      f"fp4_page_table entries a row consumes must lie in [0, {pages})")
        if node_counts is not None:
            _check_values((node_counts < 0) | (node_counts > nodes), f"node_counts values must lie in [0, {nodes}]")
        if has_residual:
            _check_values((seqused_residual < 0) | (seqused_residual > PAGE_SIZE),
                          f"seqused_residual values must lie in [0, {PAGE_SIZE}]")
            _check_values((residual_page_ids < 0) | (residual_page_ids >= slots),
                          "residual_page_ids contains an out-of-range physical page ID")
            if seqused_sink is not None:
                _check_values((seqused_sink < 0) | (seqused_sink > sink_rows),
                              f"seqused_sink values must lie in [0, {sink_rows}]")
    if out is None:
        make = torch.empty if node_counts is None else torch.zeros
        out = make(shape, dtype=torch.bfloat16, device=device)
    a.out, by_row, by_node = _tree_tensor(out, "out", shape, device)
    extent = heads_q * HEAD_DIM
    if by_node < extent or by_row < (nodes - 1) * by_node + extent:  # not rows of nodes: nodes of rows, or they overlap
        for stride, size in sorted(((by_row, rows), (by_node, nodes))):
            if size > 1 and stride < extent:
                raise ValueError("out must have an element of its own for every result")
            extent += stride * (size - 1)
    a.out_row_stride, a.out_node_stride = by_row, by_node
    need = tree_workspace_bytes(rows, nodes, heads_q, heads_kv)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif (not isinstance(workspace, torch.Tensor) or workspace.dtype is not torch.uint8 or workspace.device != device or not workspace.is_contiguous()
          or workspace.numel() < need or workspace.data_ptr() % 16):
        raise ValueError(f"workspace must be a contiguous, 16-byte aligned uint8 buffer of at least {need} bytes on {device}")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    _launch(bdfp4.tree_decode, a, device)
    return out


class DraftVerdict(NamedTuple):
    """What became of each row's tree, on the device.

    ``accepted`` INT32 ``[rows, nodes]``: the accepted path as node numbers from the root (node 0) on, then -1;
    ``accepted_counts`` INT32 ``[rows]``: its length; ``next_tokens`` INT32 ``[rows]``: the token that follows it.
    """

    accepted: torch.Tensor
    accepted_counts: torch.Tensor
    next_tokens: torch.Tensor


def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, uniforms: torch.Tensor, *,
                  draft_probs: torch.Tensor | None = None, node_counts: torch.Tensor | None = None,
                  out: DraftVerdict | None = None) -> DraftVerdict:
    """Accept a path of the drafted tree and draw the token behind it, so that the tokens are distributed as
    if the target had been sampled one by one.

    ``target_probs`` FP32 or BF16 ``[rows, nodes, vocab]`` is the target's next-token distribution at every
    node; ``tokens`` INT32 ``[rows, nodes]`` the drafted tokens (entry 0 is not read as a draft). The walk starts
    at node 0 and tries the current node's children in order: child ``c`` with token ``x`` is accepted when
    ``uniforms[c] * q(x) * W < w(x)``, ``w`` being the target's distribution there and ``W = 1``. A refusal takes
    the drafter's share off: with ``draft_probs`` (same type and shape as ``target_probs``: the distribution
    each node's children were drawn from, independently of each other) ``w`` becomes ``max(w / W - q, 0)`` and
    ``W`` its sum; without, ``q(x) = 1``, ``w(x)`` becomes 0 and ``W`` loses it, so that in the end a child is
    accepted with exactly its target probability. When the children run out, ``uniforms[0]`` draws the next
    token from ``w``: the first index whose cumulative weight exceeds ``uniforms[0]`` times the total.

    ``uniforms`` FP32 ``[rows, nodes]`` in ``[0, 1)``; ``parents`` and ``node_counts`` as in :func:`tree_decode` (a
    row of no nodes gets ``-1`` everywhere and a count of 0). ``out`` takes the place of the allocated result.
    """
    device = _cuda_device(target_probs, "target_probs")
    if target_probs.ndim != 3 or target_probs.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("target_probs must be FP32 or BF16 [rows, nodes, vocab]")
    rows, nodes, vocab = target_probs.shape
    if rows < 1 or nodes < 1 or vocab < 1:
        raise ValueError("verify_drafts needs at least one row, one node and one token")
    if nodes > MAX_TREE_NODES:
        raise NotImplementedError(f"a tree holds at most {MAX_TREE_NODES} nodes, got {nodes}")
    for tensor, name in ((target_probs, "target_probs"), (draft_probs, "draft_probs")):
        if tensor is not None and (
            not isinstance(tensor, torch.Tensor) or tensor.dtype is not target_probs.dtype or tensor.device != device or tensor.shape != target_probs.shape
            or (vocab > 1 and tensor.stride(2) != 1)
        ):
            raise ValueError(f"{name} must be {target_probs.dtype} [{rows}, {nodes}, {vocab}] on {device}, dense along "
                             "the vocabulary")
    a = bdfp4.VerifyArgs()
    a.rows, a.nodes, a.vocab, a.bf16 = rows, nodes, vocab, int(target_probs.dtype is torch.bfloat16)
    a.tokens, a.tokens_row_stride = _int32(tokens, "tokens", (rows, nodes), device), tokens.stride(0)
    a.parents, a.parents_row_stride = _parents(parents, rows, nodes, device)
    if (not isinstance(uniforms, torch.Tensor) or uniforms.dtype is not torch.float32 or uniforms.device != device
            or tuple(uniforms.shape) != (rows, nodes) or (nodes > 1 and uniforms.stride(1) != 1)):
        raise ValueError(f"uniforms must be FP32 [{rows}, {nodes}] on {device}, dense along its last axis")
    a.uniforms, a.uniforms_row_stride = uniforms.data_ptr(), uniforms.stride(0)
    if node_counts is not None:
        a.node_counts = _int32(node_counts, "node_counts", (rows,), device)
    if out is None:
        path, number, token = torch.empty(rows * (nodes + 2), dtype=torch.int32, device=device).split((rows * nodes, rows, rows))
        out = DraftVerdict(path.view(rows, nodes), number, token)
    else:
        for tensor, name, shape in zip(out, DraftVerdict._fields, ((rows, nodes), (rows,), (rows,))):
            _int32(tensor, f"out.{name}", shape, device)
            if not tensor.is_contiguous():
                raise ValueError(f"out.{name} must be contiguous")
    a.target_probs = target_probs.data_ptr()
    a.target_row_stride, a.target_node_stride, _ = target_probs.stride()
    if draft_probs is not None:
        a.draft_probs = draft_probs.data_ptr()
        a.draft_row_stride, a.draft_node_stride, _ = draft_probs.stride()
    a.accepted, a.accepted_counts, a.next_tokens = (t.data_ptr() for t in out)
    _launch(bdfp4.verify_drafts, a, device)
    return out


class CommittedLengths(NamedTuple):
    """Each row's lengths after a commit, INT32 ``[rows]`` on the device: what the next step's
    :func:`tree_decode` takes (or ``fp4_decode``, whose sink is the whole 16 rows or, without ``seqused_sink``, none)."""

    seq_lens: torch.Tensor
    seqused_fp4: torch.Tensor
    seqused_residual: torch.Tensor
    seqused_sink: torch.Tensor


class DraftCommitter:
    """The accepted path's K/V of every layer into the cache.

    Built once with what does not change between steps: the tail buffers ``[layers, slots, 128 + sink_tokens,
    heads, 128]``, the basis of the cached keys (``rotate_key``, ``key_shift`` FP32 ``[layers, heads, 128]`` already
    rotated), and the layers' cache ``regions`` (a list of four-region tuples, one per layer) with their scale
    modes. A page that a row fills is sealed into the cache by the page writer, as the serving plugin's
    promotion does; without ``regions`` the caller sees to it that no row fills a page.
    """

    def __init__(self, *, tail_key: torch.Tensor, tail_value: torch.Tensor, sink_tokens: int = SINK_TOKENS,
                 rotate_key: bool = False, key_shift: torch.Tensor | None = None, regions: list | None = None,
                 key_scale_mode: str = DEFAULT_SCALE_MODE, value_scale_mode: str = DEFAULT_SCALE_MODE,
                 key_tensor_scale: float = 1.0, value_tensor_scale: float = 1.0,
                 error_word: torch.Tensor | None = None) -> None:
        device = _cuda_device(tail_key, "tail_key")
        if not 0 <= sink_tokens <= SINK_TOKENS:
            raise ValueError(f"sink_tokens must lie in [0, {SINK_TOKENS}], got {sink_tokens}")
        for tensor, name in ((tail_key, "tail_key"), (tail_value, "tail_value")):
            if (
                not isinstance(tensor, torch.Tensor) or tensor.dtype is not torch.bfloat16 or tensor.device != device
                or not tensor.is_contiguous() or tensor.ndim != 5 or tensor.shape[2] != PAGE_SIZE + sink_tokens or tensor.shape[4] != HEAD_DIM
                or tensor.shape != tail_key.shape
            ):
                raise ValueError(f"{name} must be contiguous BF16 [layers, slots, {PAGE_SIZE + sink_tokens}, heads, 128] "
                                 f"on {device}")
        layers, slots, _, heads, _ = tail_key.shape
        if key_shift is not None and (
            not isinstance(key_shift, torch.Tensor) or key_shift.dtype is not torch.float32 or key_shift.device != device or not key_shift.is_contiguous()
            or tuple(key_shift.shape) != (layers, heads, HEAD_DIM)
        ):
            raise ValueError(f"key_shift must be contiguous FP32 [{layers}, {heads}, {HEAD_DIM}] on {device}")
        if error_word is not None:
            _int32(error_word, "error_word", (1,), device)
        self.layers, self.slots, self.heads, self.sink_tokens = layers, slots, heads, int(sink_tokens)
        self._tail_key, self._tail_value, self._shift = tail_key, tail_value, key_shift
        self._rotate, self._device, self._error_word = bool(rotate_key), device, error_word
        self._seal = None
        self.page_tokens, self.pages = PAGE_SIZE, 0
        if regions is not None:
            if len(regions) != layers:
                raise ValueError(f"regions of {len(regions)} layers given, the tail has {layers}")
            bases = torch.tensor([[layer[i].data_ptr() for layer in regions] for i in range(4)], dtype=torch.int64,
                                 device=device)
            writer = KVCacheWriter(regions=regions[0], key_scale_mode=key_scale_mode, value_scale_mode=value_scale_mode,
                                   destination_bases=bases, key_tensor_scale=key_tensor_scale,
                                   value_tensor_scale=value_tensor_scale, error_word=error_word)
            if writer.heads != heads:
                raise ValueError(f"the cache has {writer.heads} KV heads, the tail {heads}")
            for layer in regions:  # one launch serves every layer, so their regions are laid out alike
                writer.bind_regions(*layer)
                if any(t.stride() != f.stride() or t.shape != f.shape for t, f in zip(layer, regions[0])):
                    raise ValueError("the layers' cache regions must have equal shapes and strides")
            self._seal = (writer, regions[0], regions)
            self.page_tokens, self.pages = writer.page_size, regions[0][0].shape[0]

    def __call__(self, draft_key: torch.Tensor, draft_value: torch.Tensor, accepted: torch.Tensor,
                 accepted_counts: torch.Tensor, *, seq_lens: torch.Tensor, row_to_slot: torch.Tensor,
                 block_table: torch.Tensor | None = None) -> CommittedLengths:
        """Append each row's accepted nodes (``accepted`` INT32 ``[rows, nodes]``, the first ``accepted_counts[r]``
        entries) to its sequence of ``seq_lens[r]`` tokens. A path ends before an entry that is not a node's number, and
        sets ``bdfp4.DEV_BAD_NODE`` in the error word.

        ``draft_key`` / ``draft_value`` are BF16 ``[layers, rows, nodes, heads, 128]`` as the model made them (the
        same tensors :func:`tree_decode` read, all layers). Token ``p`` goes to row ``p % 128`` of slot
        ``row_to_slot[r]`` and, below ``sink_tokens``, to the sink; a negative slot (or one the tail does not have)
        leaves its row alone, and no two rows may name one slot.
        ``block_table`` INT32 ``[rows, columns]`` names the pages that filled tails are sealed into and is required
        when the committer was built with ``regions``; a page without a valid entry there (or behind the last
        column) is not sealed and sets ``bdfp4.DEV_BAD_PAGE`` in the error word. Returns the new lengths;
        ``seq_lens`` is not changed.
        """
        device = self._device
        if not isinstance(draft_key, torch.Tensor) or draft_key.ndim != 5:
            raise ValueError("draft_key must be BF16 [layers, rows, nodes, heads, 128]")
        _, rows, nodes = draft_key.shape[:3]
        if rows < 1 or nodes < 1:
            raise ValueError("a commit needs at least one row and one node")
        if nodes > MAX_TREE_NODES:
            raise NotImplementedError(f"a tree holds at most {MAX_TREE_NODES} nodes, got {nodes}")
        shape = (self.layers, rows, nodes, self.heads, HEAD_DIM)
        a = bdfp4.CommitArgs()
        a.layers, a.rows, a.nodes, a.heads_kv = self.layers, rows, nodes, self.heads
        a.draft_key, a.key_layer_stride, a.key_row_stride, a.key_node_stride = _tree_tensor(
            draft_key, "draft_key", shape, device)
        a.draft_value, a.value_layer_stride, a.value_row_stride, a.value_node_stride = _tree_tensor(
            draft_value, "draft_value", shape, device)
        a.accepted, a.accepted_row_stride = _int32(accepted, "accepted", (rows, nodes), device), accepted.stride(0)
        a.accepted_counts = _int32(accepted_counts, "accepted_counts", (rows,), device)
        a.seq_lens = _int32(seq_lens, "seq_lens", (rows,), device)
        a.row_to_slot = _int32(row_to_slot, "row_to_slot", (rows,), device)
        if (block_table is not None) != (self._seal is not None):
            raise ValueError("block_table goes with a committer that was built with regions, and only with one")
        lengths = torch.empty(4, rows, dtype=torch.int32, device=device)
        a.tail_key, a.tail_value = self._tail_key.data_ptr(), self._tail_value.data_ptr()
        a.tail_slot_stride = (PAGE_SIZE + self.sink_tokens) * self.heads * HEAD_DIM
        a.tail_layer_stride = self.slots * a.tail_slot_stride
        a.tail_slots, a.sink_tokens, a.rotate = self.slots, self.sink_tokens, int(self._rotate)
        a.key_shift = bdfp4.ptr(self._shift)
        address = lengths.data_ptr()
        a.new_seq_lens, a.seqused_fp4, a.seqused_residual, a.seqused_sink = range(address, address + 16 * rows, 4 * rows)
        a.error_word = bdfp4.ptr(self._error_word)
        if self._seal is None:
            a.part = bdfp4.COMMIT_ALL
            _launch(bdfp4.commit_drafts, a, device)
            return CommittedLengths(*lengths.unbind())
        if not isinstance(block_table, torch.Tensor) or block_table.ndim != 2:
            raise ValueError("block_table must be row-major INT32 with shape [rows, columns]")
        columns = block_table.shape[1]
        a.page_table = _int32(block_table, "block_table", (rows, columns), device)
        a.page_table_stride = block_table.stride(0)
        work = torch.empty(2, rows * (PAGE_SIZE // self.page_tokens), dtype=torch.int32, device=device)
        a.max_pages_per_row, a.pages, a.page_tokens = columns, self.pages, self.page_tokens
        a.source_tokens, a.destination_pages = work[0].data_ptr(), work[1].data_ptr()
        # the tokens behind a page boundary reuse tail rows that the seal reads, so they wait for it
        with torch.cuda.device(device):
            a.part = bdfp4.COMMIT_HEAD
            _launch(bdfp4.commit_drafts, a, device)
            writer, regions, _ = self._seal
            writer(self._tail_key.view(-1, self.heads, HEAD_DIM), self._tail_value.view(-1, self.heads, HEAD_DIM), regions,
                   work[0], work[1])
            a.part = bdfp4.COMMIT_REST
            _launch(bdfp4.commit_drafts, a, device)
        return CommittedLengths(*lengths.unbind())
