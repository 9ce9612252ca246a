"""Tensor-level wrappers over the C ABI: shape/dtype/device checks, then one launch.

Every function here requires device tensors on a ROCm GPU and launches on the
current torch stream of that device.  None of them has a CPU or PyTorch
fallback; a missing library or a CPU tensor raises.
"""

from __future__ import annotations

import ctypes
import functools
import math
from array import array
from dataclasses import dataclass

import numpy as np
import torch

from nanoengine_amd import _native
from nanoengine_amd._native import (
    DTYPE_BF16,
    DTYPE_FP16,
    DTYPE_FP32,
    DTYPE_INT8,
    EPILOGUE_STORE,
    EPILOGUE_SWIGLU,
)

_DTYPE_CODES = {
    torch.bfloat16: DTYPE_BF16,
    torch.float16: DTYPE_FP16,
    torch.float32: DTYPE_FP32,
    torch.int8: DTYPE_INT8,
}

HEAD_DIM = 128


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODES[dtype]
    except KeyError as error:
        raise TypeError(f"unsupported dtype {dtype}") from error


def _ptr(tensor: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if tensor is None else ctypes.c_void_p(tensor.data_ptr())


def _require_gpu(*tensors: torch.Tensor | None) -> torch.device:
    device = None
    for tensor in tensors:
        if tensor is None:
            continue
        if tensor.device.type != "cuda":
            raise RuntimeError(
                f"nanoengine HIP kernels need GPU tensors; got one on {tensor.device}"
            )
        if device is None:
            device = tensor.device
        elif tensor.device != device:
            raise RuntimeError(f"tensors on different devices: {device} and {tensor.device}")
    if device is None:
        raise RuntimeError("no GPU tensor given")
    return device


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _check(cond: bool, message: str) -> None:
    if not cond:
        raise ValueError(message)


def _contig(tensor: torch.Tensor, name: str) -> None:
    _check(tensor.is_contiguous(), f"{name} must be contiguous")


def _int32(tensor: torch.Tensor, name: str) -> None:
    _check(tensor.dtype == torch.int32, f"{name} must be int32, got {tensor.dtype}")
    _contig(tensor, name)


# --------------------------------------------------------------------------- A1
def ngram_propose(
    history: torch.Tensor,
    history_len: torch.Tensor,
    num_tokens: torch.Tensor,
    max_ngram: int,
    max_drafts: int,
    min_ngram: int = 1,
    drafts: torch.Tensor | None = None,
    num_drafts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Drafts ``[b, max_drafts]`` (tail unused) and their counts ``[b]`` from each history."""
    device = _require_gpu(history, history_len, num_tokens)
    _int32(history, "history")
    _int32(history_len, "history_len")
    _int32(num_tokens, "num_tokens")
    _check(history.dim() == 2, "history must be [num_seqs, capacity]")
    num_seqs = history.shape[0]
    if drafts is None:
        drafts = torch.zeros((num_seqs, max_drafts), dtype=torch.int32, device=device)
    if num_drafts is None:
        num_drafts = torch.empty((num_seqs,), dtype=torch.int32, device=device)
    _native.call(
        "ne_ngram_propose",
        _ptr(history), history.stride(0), _ptr(history_len), _ptr(num_tokens), num_seqs,
        max_ngram, min_ngram, max_drafts, _ptr(drafts), _ptr(num_drafts), _stream(device),
    )
    return drafts, num_drafts


# --------------------------------------------------------------------------- A7
def kv_write(
    vectors: torch.Tensor,
    slot_mapping: torch.Tensor,
    cache: torch.Tensor,
    scales: torch.Tensor | None,
) -> None:
    """Write ``vectors [n, heads, 128]`` to ``cache`` at ``slot_mapping`` (quantising to int8)."""
    device = _require_gpu(vectors, slot_mapping, cache, scales)
    _contig(vectors, "vectors")
    _int32(slot_mapping, "slot_mapping")
    _check(vectors.dim() == 3 and vectors.shape[2] == HEAD_DIM, "vectors must be [n, heads, 128]")
    _check(cache.dim() == 3 and cache.shape[1:] == vectors.shape[1:], "cache shape mismatch")
    _check(slot_mapping.numel() == vectors.shape[0], "one slot per vector row")
    if cache.dtype == torch.int8:
        _check(scales is not None and scales.shape[0] == cache.shape[0], "int8 cache needs scales")
    _native.call(
        "ne_kv_write",
        _ptr(vectors), dtype_code(vectors.dtype), vectors.shape[0], vectors.shape[1], HEAD_DIM,
        _ptr(slot_mapping), _ptr(cache), dtype_code(cache.dtype), _ptr(scales),
        dtype_code(scales.dtype) if scales is not None else DTYPE_BF16, _stream(device),
    )


def _call_on(device: torch.device, name: str, *args) -> None:
    """``_native.call`` with ``device`` current: a launch goes to the current device, whichever
    device its stream belongs to."""
    if torch.cuda.current_device() == device.index:
        _native.call(name, *args)
    else:
        with torch.cuda.device(device):
            _native.call(name, *args)


# ------------------------------------------------------------------- block copies
def copy_kv_blocks(buffers: list[torch.Tensor], block_size: int, src: list[int], dst: list[int]) -> None:
    """Copy block ``src[i]`` to block ``dst[i]`` in every buffer: caches and scales
    ``[num_slots (+ 1), ...]`` whose slots ``b * block_size ..`` are block ``b``, as a
    :class:`~nanoengine_amd.memory.KVCachePool` holds them, all layers in one launch.

    ``src`` and ``dst`` are host lists.  The copies are unordered, so no block may be a
    destination twice or the destination of one copy and the source of another.  Under graph
    capture the graph keeps the blocks of this call."""
    _check(block_size >= 1, "block_size must be at least 1")
    _check(len(src) == len(dst), f"{len(src)} sources for {len(dst)} destinations")
    if not buffers:
        raise ValueError("no buffers to copy in")
    first = buffers[0]
    if not first.is_cuda or len(set(map(torch.Tensor.get_device, buffers))) > 1:
        _require_gpu(*buffers)  # names the tensor
    # (one call per tensor and check: a pool has four tensors per layer)
    shapes = [t.shape for t in buffers]
    num_slots = shapes[0][0] if shapes[0] else 0
    _check(all(map(torch.Tensor.is_contiguous, buffers)) and all([s and s[0] == num_slots for s in shapes]),
           "buffers must be contiguous and hold the same slots")
    _check(num_slots > 0, "buffers hold no slots")
    n = len(buffers)
    block_bytes = array("q", [t.nbytes // num_slots * block_size for t in buffers])
    pointers = array("Q", map(torch.Tensor.data_ptr, buffers))
    _copy_blocks(first.device, pointers, block_bytes, n, num_slots // block_size, src, dst)


def _block_list(blocks: list[int]) -> array:
    try:
        return array("i", blocks)
    except TypeError as error:
        raise TypeError("blocks must be a list of ints") from error


def _copy_blocks(device: torch.device, pointers: array, block_bytes: array, num_buffers: int, num_blocks: int,
                 src: list[int], dst: list[int]) -> None:
    if len(src) and (max(max(src), max(dst)) >= num_blocks or min(min(src), min(dst)) < 0):
        raise ValueError(f"blocks outside [0, {num_blocks})")
    sources, targets = _block_list(src), _block_list(dst)
    _call_on(device, "ne_kv_copy_blocks", pointers.buffer_info()[0], block_bytes.buffer_info()[0], num_buffers,
             num_blocks, sources.buffer_info()[0], targets.buffer_info()[0], len(src), _stream(device))


# --------------------------------------------------------------------------- A6
@dataclass
class AttentionWorkspace:
    """Caller-owned scratch for split-K attention; re-zeroed when its layout changes.

    ``plan_key`` names the metadata the last :func:`paged_attention_plan` call used, so
    that a planned attention call on other metadata is refused.  ``frozen`` is set once a
    captured HIP graph holds the buffers' addresses: from then on a call that would need a
    larger one raises instead of reallocating under the graph (a graph holds no buffer that
    was not there yet)."""

    buffer: torch.Tensor | None = None
    layout: tuple | None = None
    plan_key: tuple | None = None
    runs_key: tuple | None = None  # metadata of the last paged_kv_runs_plan (measurement)
    frozen: bool = False
    prefix_buffer: torch.Tensor | None = None  # of shared-prefix plans

    def get(self, device: torch.device, nbytes: int, layout: tuple) -> torch.Tensor:
        if self.buffer is None or self.buffer.numel() < nbytes or self.buffer.device != device:
            if self.frozen and self.buffer is not None:
                raise RuntimeError(f"attention workspace of {self.buffer.numel()} bytes is held by a captured HIP graph; "
                                   f"this call needs {nbytes} bytes on {device}: size it before capture")
            self.buffer = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            self.layout = layout
            self.plan_key = self.runs_key = None
        elif self.layout != layout:
            self.buffer.zero_()
            self.layout = layout
            self.plan_key = self.runs_key = None
        return self.buffer

    def get_prefix(self, device: torch.device, nbytes: int) -> torch.Tensor:
        """A buffer for :func:`shared_prefix_plan`, under the same rule."""
        have = self.prefix_buffer
        if have is None or have.numel() < nbytes or have.device != device:
            if self.frozen and have is not None:
                raise RuntimeError(f"shared-prefix workspace of {have.numel()} bytes is held by a captured HIP graph; "
                                   f"this call needs {nbytes} bytes on {device}: size it before capture")
            self.prefix_buffer = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
        return self.prefix_buffer

    def error_flag(self) -> int:
        words = [int(b[:4].view(torch.int32).item()) for b in (self.buffer, self.prefix_buffer) if b is not None]
        return words[0] | words[-1] if words else 0


_default_workspaces: dict[torch.device, AttentionWorkspace] = {}


def default_workspace(device: torch.device) -> AttentionWorkspace:
    return _default_workspaces.setdefault(device, AttentionWorkspace())


def paged_verify_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    block_tables: torch.Tensor,
    block_size: int,
    ctx_len: torch.Tensor,
    q_start: torch.Tensor,
    q_len: torch.Tensor,
    max_q_len: int,
    max_ctx_len: int,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: AttentionWorkspace | None = None,
    split_len: int = 0,
    planned: bool = False,
) -> torch.Tensor:
    """Paged multi-query attention; ``q``/``out`` are ``[rows, q_heads, 128]`` bf16.

    ``planned=True`` reads the work plan that :func:`paged_attention_plan` wrote into
    the same ``workspace`` for the same metadata (once per step, shared by the layers)."""
    device = _require_gpu(q, k_cache, v_cache, k_scale, v_scale, block_tables, ctx_len, q_start,
                          q_len)
    _check(q.dtype == torch.bfloat16 and q.dim() == 3 and q.shape[2] == HEAD_DIM,
           "q must be [rows, heads, 128] bf16")
    _check(q.stride(2) == 1, "q head_dim must be contiguous")
    _check(k_cache.shape == v_cache.shape and k_cache.dim() == 3, "k/v cache shape mismatch")
    _check(k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous")
    is_int8 = k_cache.dtype == torch.int8
    if is_int8:
        _check(k_scale is not None and v_scale is not None, "int8 cache needs scales")
        _check(k_scale.is_contiguous() and v_scale.is_contiguous(), "scales must be contiguous")
        _check(k_scale.numel() == k_cache.shape[0] * k_cache.shape[1], "k_scale shape mismatch")
    else:
        _check(k_cache.dtype == torch.bfloat16, "cache must be int8 or bf16")
    _int32(block_tables, "block_tables")
    for name, t in (("ctx_len", ctx_len), ("q_start", q_start), ("q_len", q_len)):
        _int32(t, name)
    num_seqs = ctx_len.shape[0]
    num_q_heads = q.shape[1]
    num_kv_heads = k_cache.shape[1]
    if out is None:
        out = torch.empty_like(q)
    _check(out.shape == q.shape and out.dtype == torch.bfloat16 and out.stride(2) == 1,
           "out must match q")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(HEAD_DIM)
    nbytes = _native.load().ne_paged_attention_workspace_size(
        num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, split_len
    )
    _check(nbytes > 0, "bad attention shape")
    workspace = workspace or default_workspace(device)
    ws = workspace.get(device, nbytes, (num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, split_len))
    if planned:
        _check(workspace.plan_key == _plan_key(block_tables, block_size, ctx_len, q_start, q_len, max_q_len,
                                               max_ctx_len, split_len),
               "planned attention needs paged_attention_plan on the same metadata and workspace first")
    _native.call(
        "ne_paged_verify_attention_planned" if planned else "ne_paged_verify_attention",
        _ptr(q), q.stride(0), q.stride(1),
        _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
        dtype_code(k_cache.dtype), dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16,
        _ptr(block_tables), block_tables.stride(0), block_size,
        _ptr(ctx_len), _ptr(q_start), _ptr(q_len),
        num_seqs, num_q_heads, num_kv_heads, HEAD_DIM, max_q_len, max_ctx_len,
        float(softmax_scale),
        _ptr(out), out.stride(0), out.stride(1),
        split_len, _ptr(ws), ws.numel(), _stream(device),
    )
    return out


def paged_verify_attention_noalloc(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    block_tables: torch.Tensor,
    block_size: int,
    ctx_len: torch.Tensor,
    q_start: torch.Tensor,
    q_len: torch.Tensor,
    max_q_len: int,
    max_ctx_len: int,
    error_flag: torch.Tensor,
    out: torch.Tensor,
    softmax_scale: float | None = None,
    split_len: int = 0,
) -> torch.Tensor:
    """:func:`paged_verify_attention` without a workspace: the work plan and split partials
    live in the library's per-GPU scratch (``NOALLOC_SCRATCH_BYTES``), ``error_flag`` is a
    caller-owned int32 device word that receives the error bits, and ``out`` is given, so
    the call allocates nothing (usable where allocation is not allowed).  Calls that
    overlap on one GPU share the scratch and race."""
    device = _require_gpu(q, k_cache, v_cache, k_scale, v_scale, block_tables, ctx_len, q_start, q_len,
                          error_flag, out)
    _check(q.dtype == torch.bfloat16 and q.dim() == 3 and q.shape[2] == HEAD_DIM and q.stride(2) == 1,
           "q must be [rows, heads, 128] bf16")
    _check(out.shape == q.shape and out.dtype == torch.bfloat16 and out.stride(2) == 1, "out must match q")
    _check(error_flag.dtype == torch.int32 and error_flag.numel() >= 1, "error_flag must be an int32 word")
    is_int8 = k_cache.dtype == torch.int8
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(HEAD_DIM)
    _native.call(
        "ne_paged_verify_attention_noalloc",
        _ptr(q), q.stride(0), q.stride(1),
        _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
        dtype_code(k_cache.dtype), dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16,
        _ptr(block_tables), block_tables.stride(0), block_size,
        _ptr(ctx_len), _ptr(q_start), _ptr(q_len),
        ctx_len.shape[0], q.shape[1], k_cache.shape[1], HEAD_DIM, max_q_len, max_ctx_len,
        float(softmax_scale),
        _ptr(out), out.stride(0), out.stride(1),
        split_len, _ptr(error_flag), _stream(device),
    )
    return out


def _plan_key(block_tables, block_size, ctx_len, q_start, q_len, max_q_len, max_ctx_len, split_len) -> tuple:
    return (block_tables.data_ptr(), tuple(block_tables.shape), block_tables.stride(0), block_size,
            ctx_len.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), ctx_len.shape[0], max_q_len, max_ctx_len,
            split_len)


def paged_attention_plan(
    block_tables: torch.Tensor,
    block_size: int,
    ctx_len: torch.Tensor,
    q_start: torch.Tensor,
    q_len: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    max_q_len: int,
    max_ctx_len: int,
    workspace: AttentionWorkspace,
    split_len: int = 0,
) -> None:
    """Write the attention work plan for this metadata into ``workspace`` (8 KV heads and
    at most 32 query rows per KV head; bf16 pools or int8 ones with 2-byte scales)."""
    device = _require_gpu(block_tables, ctx_len, q_start, q_len)
    _int32(block_tables, "block_tables")
    for name, t in (("ctx_len", ctx_len), ("q_start", q_start), ("q_len", q_len)):
        _int32(t, name)
    num_seqs = ctx_len.shape[0]
    nbytes = _native.load().ne_paged_attention_workspace_size(
        num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, split_len
    )
    _check(nbytes > 0, "bad attention shape")
    ws = workspace.get(device, nbytes, (num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, split_len))
    _native.call(
        "ne_paged_attention_plan",
        _ptr(block_tables), block_tables.stride(0), block_size, _ptr(ctx_len), _ptr(q_start), _ptr(q_len),
        num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, split_len, _ptr(ws), ws.numel(),
        _stream(device),
    )
    workspace.plan_key = _plan_key(block_tables, block_size, ctx_len, q_start, q_len, max_q_len, max_ctx_len,
                                   split_len)
    workspace.runs_key = None


def paged_kv_stream_planned(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    num_seqs: int,
    num_q_heads: int,
    max_q_len: int,
    max_ctx_len: int,
    workspace: AttentionWorkspace,
    split_len: int = 0,
) -> None:
    """Measurement: the K/V reads of the planned attention call alone (its plan, tiles, ring
    and copies; nothing computed or stored), on the plan ``workspace`` holds for the same
    metadata.  Its time is the memory ceiling of that call's access pattern."""
    device = _require_gpu(k_cache, v_cache, k_scale, v_scale)
    _check(workspace.buffer is not None and workspace.plan_key is not None,
           "the stream reads the plan paged_attention_plan wrote into the workspace")
    num_kv_heads = k_cache.shape[1]
    is_int8 = k_cache.dtype == torch.int8
    _native.call(
        "ne_paged_kv_stream_planned",
        _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), dtype_code(k_cache.dtype),
        dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16, num_seqs, num_q_heads, num_kv_heads, max_q_len,
        max_ctx_len, split_len, _ptr(workspace.buffer), workspace.buffer.numel(), _stream(device),
    )


def paged_kv_runs_plan(
    block_tables: torch.Tensor,
    block_size: int,
    ctx_len: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    max_q_len: int,
    max_ctx_len: int,
    workspace: AttentionWorkspace,
) -> None:
    """Measurement: cut the sequences' 16-key tiles, in order, into the workspace's
    plan_grid runs of near-equal length across sequence boundaries, for
    :func:`paged_kv_stream_runs`.  The runs take the place of the attention work plan,
    so a planned call afterwards needs :func:`paged_attention_plan` again."""
    device = _require_gpu(block_tables, ctx_len)
    _int32(block_tables, "block_tables")
    _int32(ctx_len, "ctx_len")
    num_seqs = ctx_len.shape[0]
    nbytes = _native.load().ne_paged_attention_workspace_size(
        num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, 0
    )
    _check(nbytes > 0, "bad attention shape")
    ws = workspace.get(device, nbytes, (num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, 0))
    _native.call(
        "ne_paged_kv_runs_plan",
        _ptr(block_tables), block_tables.stride(0), block_size, _ptr(ctx_len), num_seqs, num_q_heads,
        num_kv_heads, max_q_len, max_ctx_len, _ptr(ws), ws.numel(), _stream(device),
    )
    workspace.plan_key = None
    workspace.runs_key = (num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len)


def paged_kv_stream_runs(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    num_seqs: int,
    num_q_heads: int,
    max_q_len: int,
    max_ctx_len: int,
    workspace: AttentionWorkspace,
) -> None:
    """Measurement: the same K/V bytes as the planned call, read in the balanced whole-slot
    runs that :func:`paged_kv_runs_plan` wrote (work-group w reads all 8 KV heads of every
    tile of run w through the planned call's ring and copies; nothing computed or stored)."""
    device = _require_gpu(k_cache, v_cache, k_scale, v_scale)
    num_kv_heads = k_cache.shape[1]
    _check(workspace.buffer is not None
           and workspace.runs_key == (num_seqs, num_q_heads, num_kv_heads, max_q_len, max_ctx_len),
           "the stream reads the runs paged_kv_runs_plan wrote into the workspace for this shape")
    is_int8 = k_cache.dtype == torch.int8
    _native.call(
        "ne_paged_kv_stream_runs",
        _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), dtype_code(k_cache.dtype),
        dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16, num_seqs, num_q_heads, num_kv_heads, max_q_len,
        max_ctx_len, _ptr(workspace.buffer), workspace.buffer.numel(), _stream(device),
    )


# ----------------------------------------------------------- shared prefixes
@dataclass(frozen=True)
class PrefixGroups:
    """Which sequences of a batch hold the same tokens in the same blocks from the start on:
    device tensors that a step reads, so their contents may change between replays of a graph."""

    seqs: torch.Tensor  # [b] int32: every sequence's index, group after group
    start: torch.Tensor  # [groups + 1] int32: first entry of each group; 0 first, b last
    prefix_len: torch.Tensor  # [groups] int32: tokens the group's tables have in common
    max_prefix_len: int  # bound on prefix_len

    @classmethod
    def from_lists(cls, groups: list[list[int]], prefix_lens: list[int], device: torch.device) -> "PrefixGroups":
        """From host lists: each group's sequences, and the tokens each shares."""
        _check(len(groups) == len(prefix_lens), "one prefix length per group")
        seqs = [s for members in groups for s in members]
        _check(sorted(seqs) == list(range(len(seqs))), "every sequence belongs to one group")
        start = [0]
        for members in groups:
            start.append(start[-1] + len(members))
        flat = torch.tensor(seqs + start + prefix_lens, dtype=torch.int32).to(device)
        n, g = len(seqs), len(groups)
        return cls(flat[:n], flat[n : n + g + 1], flat[n + g + 1 :], max(prefix_lens, default=0))


@dataclass(frozen=True)
class SharedPrefixPlan:
    """The work plan of one step (:func:`shared_prefix_plan`) and what it was made for."""

    workspace: torch.Tensor
    block_tables: torch.Tensor
    block_size: int
    num_rows: int
    num_q_heads: int
    num_kv_heads: int
    max_q_len: int
    max_ctx_len: int
    num_blocks: int
    groups: PrefixGroups

    @functools.cached_property
    def _sizes(self) -> tuple:
        """What every layer's call passes: sequences to the prefix bound, as the entry point takes them."""
        return (self.groups.seqs.shape[0], self.groups.prefix_len.shape[0], self.num_q_heads, self.num_kv_heads, HEAD_DIM,
                self.max_q_len, self.max_ctx_len, self.groups.max_prefix_len)

    def error_flag(self) -> int:
        """The error word of the plan and the calls on it (waits for them)."""
        return self._word(0)

    def _word(self, i: int) -> int:
        if self.groups.seqs.shape[0] == 0:  # nothing was planned, nor written
            return 0
        return int(self.workspace[4 * i : 4 * i + 4].view(torch.int32).item())

    def shared_items(self) -> int:
        """Work items that read a prefix for its whole group (waits for the plan): 0 where sharing
        would cost more than it saves, as for few sequences or short prefixes."""
        return self._word(2)


SHARED_PREFIX_MAX_SEQS = 1024  # a plan's sequences
# Sharing has to save more than this many bytes of keys and values per layer for a step to be faster with it
# (at the border itself one measured case gains and one loses).  28 layers of
# 16 query and 8 KV heads, verify steps of 5 rows, us per layer without and with: 64 sequences on 512 tokens
# (66 MB saved, int8) 66.7 / 67.6, on 1,024 (132 MB) 72.4 / 69.0, on 2,048 (264 MB) 86 / 72, on 8,192 161 / 84;
# 16 on 2,048 (126 MB, bf16) 58.8 / 59.5, on 4,096 (126 MB, int8) 65.3 / 64.4; 60 on nine prefixes of 1,024
# (107 MB, int8) 70.5 / 71.2, of 2,048 (428 MB, bf16) 88.5 / 80.5.
SHARED_PREFIX_MIN_BYTES = 120 << 20


def shared_prefix_pays(saved_tokens: int, num_kv_heads: int, kv_dtype: torch.dtype) -> bool:
    """Whether a batch that need not read ``saved_tokens`` cached tokens again (a prefix's tokens
    times its members but one, over the groups) is faster with :func:`shared_prefix_attention`."""
    return saved_tokens * num_kv_heads * 2 * HEAD_DIM * kv_dtype.itemsize > SHARED_PREFIX_MIN_BYTES


def shared_prefix_supported(k_cache: torch.Tensor, k_scale: torch.Tensor | None) -> bool:
    """Whether :func:`shared_prefix_attention` takes this cache (bf16, or int8 with bf16 or fp16 scales)."""
    if k_cache.dtype == torch.bfloat16:
        return True
    return k_cache.dtype == torch.int8 and k_scale is not None and k_scale.dtype in (torch.bfloat16, torch.float16)


def shared_prefix_workspace_bytes(num_seqs: int, num_groups: int, num_q_heads: int, num_kv_heads: int, max_q_len: int,
                                  max_ctx_len: int, max_prefix_len: int) -> int:
    return _native.load().ne_shared_prefix_workspace_size(num_seqs, num_groups, num_q_heads, num_kv_heads, max_q_len,
                                                          max_ctx_len, max_prefix_len)


def shared_prefix_plan(
    block_tables: torch.Tensor,
    block_size: int,
    ctx_len: torch.Tensor,
    q_start: torch.Tensor,
    q_len: torch.Tensor,
    groups: PrefixGroups,
    num_q_heads: int,
    num_kv_heads: int,
    max_q_len: int,
    max_ctx_len: int,
    num_rows: int | None = None,
    num_blocks: int | None = None,
    workspace: torch.Tensor | None = None,
) -> SharedPrefixPlan:
    """Plan a step's :func:`shared_prefix_attention` calls (one per layer) from its lengths and
    groups on the device.  ``num_rows`` (default: those of each call's ``q``) bounds the query
    rows, ``num_blocks`` (default: those of each call's cache) the block tables' entries; a
    sequence with rows past the bound is not computed, and flagged.  ``workspace``
    (default: allocated here) is a uint8 tensor of :func:`shared_prefix_workspace_bytes` that no
    other plan uses until this one's calls are done."""
    device = _require_gpu(block_tables, ctx_len, q_start, q_len, groups.seqs, groups.start, groups.prefix_len)
    named = (("block_tables", block_tables), ("ctx_len", ctx_len), ("q_start", q_start), ("q_len", q_len),
             ("group seqs", groups.seqs), ("group start", groups.start), ("prefix_len", groups.prefix_len))
    for name, t in named:
        if t.dtype != torch.int32 or not t.is_contiguous():
            _int32(t, name)
    num_seqs, num_groups = ctx_len.shape[0], groups.prefix_len.shape[0]
    _check(block_tables.dim() == 2 and block_tables.shape[0] >= num_seqs, "block_tables must be [b, max_blocks]")
    _check(q_start.shape[0] == num_seqs and q_len.shape[0] == num_seqs and groups.seqs.shape[0] == num_seqs
           and groups.start.shape[0] == num_groups + 1, "lengths and groups of different batches")
    nbytes = _native.load().ne_shared_prefix_workspace_size(num_seqs, num_groups, num_q_heads, num_kv_heads, max_q_len,
                                                            max_ctx_len, groups.max_prefix_len)
    _check(nbytes > 0 or num_seqs == 0, "bad attention shape")
    if workspace is None:
        workspace = torch.empty((max(nbytes, 256),), dtype=torch.uint8, device=device)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.device != device:
        raise ValueError(f"workspace must be contiguous uint8 on {device}")
    if num_rows is None:
        num_rows = (1 << 31) - 1
    if num_blocks is None:
        num_blocks = ((1 << 31) - 1) // max(block_size, 1)
    plan = SharedPrefixPlan(workspace, block_tables, block_size, num_rows, num_q_heads, num_kv_heads, max_q_len, max_ctx_len,
                            num_blocks, groups)
    _call_on(device, "ne_shared_prefix_plan", ctx_len.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), num_rows,
             groups.seqs.data_ptr(), groups.start.data_ptr(), groups.prefix_len.data_ptr(), num_seqs, num_groups,
             num_q_heads, num_kv_heads, max_q_len, max_ctx_len, groups.max_prefix_len, block_tables.stride(0), block_size,
             num_blocks, workspace.data_ptr(), workspace.numel(), _stream(device))
    return plan


def shared_prefix_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    plan: SharedPrefixPlan,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Paged attention of a batch whose sequences share prefixes: :func:`paged_verify_attention`'s
    function of the same pool, a prefix's keys read once for its whole group.  ``q`` / ``out``
    are ``[rows, q_heads, 128]`` bf16; the pool is bf16, or int8 with bf16 or fp16 scales.  The
    block tables and lengths the plan was made from must not have changed."""
    index = plan.workspace.get_device()
    if q.get_device() != index or k_cache.get_device() != index or v_cache.get_device() != index:
        _require_gpu(q, k_cache, v_cache, plan.workspace)  # names the devices
    _check(q.dtype == torch.bfloat16 and q.dim() == 3 and q.shape[2] == HEAD_DIM and q.stride(2) == 1,
           "q must be [rows, heads, 128] bf16")
    # (a step calls this once per layer: no message is built unless it is raised)
    if q.shape[1] != plan.num_q_heads:
        raise ValueError(f"the plan is for {plan.num_q_heads} query heads")
    slots = k_cache.shape
    if (slots != v_cache.shape or k_cache.dtype != v_cache.dtype or len(slots) != 3 or slots[1] != plan.num_kv_heads
            or slots[2] != HEAD_DIM):
        raise ValueError(f"caches must be [slots, {plan.num_kv_heads}, 128]")
    _check(k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous")
    is_int8 = k_cache.dtype == torch.int8
    scale_code = DTYPE_BF16
    if is_int8:
        _check(k_scale is not None and v_scale is not None, "int8 cache needs scales")
        _require_gpu(plan.workspace, k_scale, v_scale)
        _check(k_scale.dtype == v_scale.dtype and k_scale.is_contiguous() and v_scale.is_contiguous()
               and k_scale.numel() == v_scale.numel() == slots[0] * slots[1],
               "scales must be contiguous, one per slot and KV head")
        scale_code = dtype_code(k_scale.dtype)
    else:
        _check(k_cache.dtype == torch.bfloat16, "cache must be int8 or bf16")
    if q.shape[0] < plan.num_rows != (1 << 31) - 1:
        raise ValueError(f"q has {q.shape[0]} rows, the plan {plan.num_rows}")
    if out is None:
        out = torch.empty_like(q)
    _check(out.shape == q.shape and out.dtype == torch.bfloat16 and out.stride(2) == 1 and out.get_device() == index,
           "out must match q")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(HEAD_DIM)
    device = plan.workspace.device
    _call_on(device, "ne_shared_prefix_attention_rows", q.data_ptr(), q.stride(0), q.stride(1), q.shape[0], k_cache.data_ptr(),
             v_cache.data_ptr(), k_scale.data_ptr() if is_int8 else None, v_scale.data_ptr() if is_int8 else None,
             DTYPE_INT8 if is_int8 else DTYPE_BF16, scale_code, plan.block_tables.data_ptr(), plan.block_tables.stride(0),
             plan.block_size, min(plan.num_blocks, slots[0] // plan.block_size), *plan._sizes, softmax_scale,
             out.data_ptr(), out.stride(0), out.stride(1), plan.workspace.data_ptr(), plan.workspace.numel(),
             _stream(device))
    return out


def plan_supported(num_q_heads: int, num_kv_heads: int, max_q_len: int, num_seqs: int, kv_dtype, scale_dtype) -> bool:
    """Whether :func:`paged_attention_plan` / ``planned=True`` serve this shape."""
    cache_ok = kv_dtype == torch.bfloat16 or (kv_dtype == torch.int8 and scale_dtype in (torch.bfloat16,
                                                                                        torch.float16))
    return (cache_ok and num_kv_heads == 8 and num_q_heads % num_kv_heads == 0
            and (num_q_heads // num_kv_heads) * max_q_len <= 32 and num_seqs <= 1024)


# --------------------------------------------------------------------------- A8
def w8a16_gemm(
    x: torch.Tensor,
    weight_int8: torch.Tensor,
    weight_scale: torch.Tensor,
    epilogue: int = EPILOGUE_STORE,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``bf16(x @ (int8 * scale).T)``; SwiGLU epilogue pairs 16 gate rows with 16 up rows."""
    device = _require_gpu(x, weight_int8, weight_scale)
    _check(x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1, "x must be [m, k] bf16")
    _check(weight_int8.dtype == torch.int8 and weight_int8.dim() == 2, "weight must be [n, k] int8")
    _contig(weight_int8, "weight_int8")
    _contig(weight_scale, "weight_scale")
    m, k = x.shape
    n = weight_int8.shape[0]
    _check(weight_int8.shape[1] == k, f"k mismatch: x has {k}, weight {weight_int8.shape[1]}")
    _check(weight_scale.numel() == n, "one scale per weight row")
    n_out = n // 2 if epilogue == EPILOGUE_SWIGLU else n
    if out is None:
        out = torch.empty((m, n_out), dtype=torch.bfloat16, device=device)
    _check(out.shape == (m, n_out) and out.stride(1) == 1, "bad out shape")
    _native.call(
        "ne_w8a16_gemm",
        _ptr(x), x.stride(0), _ptr(weight_int8), _ptr(weight_scale),
        dtype_code(weight_scale.dtype), m, n, k, _ptr(out), out.stride(0), epilogue,
        _stream(device),
    )
    return out


# ------------------------------------------------------------------------- W8A8
def _launch(index: int, name: str, *args) -> None:
    """An entry point on device ``index``'s current torch stream (the last argument), that device current."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        _native.call(name, *args, stream)
    else:
        with torch.cuda.device(index):
            _native.call(name, *args, stream)


def _code_outputs(x: torch.Tensor, rows: int, k: int, codes, scales) -> tuple[torch.Tensor, torch.Tensor]:
    if codes is None:
        codes = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    elif codes.dtype != torch.int8 or codes.shape != x.shape or not codes.is_contiguous() or codes.device != x.device:
        raise ValueError(f"codes must be contiguous int8 [{rows}, {k}] on {x.device}")
    if scales is None:
        scales = x.new_empty(rows, dtype=torch.float32)
    elif scales.dtype != torch.float32 or scales.shape != (rows,) or not scales.is_contiguous() or scales.device != x.device:
        raise ValueError(f"scales must be contiguous fp32 [{rows}] on {x.device}")
    return codes, scales


def quantize_rows(x: torch.Tensor, codes: torch.Tensor | None = None,
                  scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 codes ``[m, k]`` of the rows of ``x [m, k]`` (bf16 or fp16) and fp32 scales ``[m]``: the
    formula of :func:`~nanoengine_amd.int8_quantization.quantize_vectors` per row, for
    :func:`w8a8_gemm`.  A row with a NaN or an infinity gets the scale NaN and codes 0."""
    if not x.is_cuda:
        _require_gpu(x)
    whole = x.is_contiguous()
    if x.dim() != 2 or not whole and x.stride(1) != 1 and x.shape[1] != 1:
        raise ValueError("x must be [m, k] with contiguous rows")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("x must be bf16 or fp16")
    rows, k = x.shape
    codes, scales = _code_outputs(x, rows, k, codes, scales)
    _launch(x.get_device(), "ne_quantize_rows", x.data_ptr(), _DTYPE_CODES[x.dtype], k if whole else x.stride(0), rows, k,
            codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _check_norm_rows(weight: torch.Tensor, rows: torch.Tensor) -> None:
    if rows.get_device() != weight.get_device() or not rows.is_cuda:
        _require_gpu(rows, weight)
    if (rows.dim() != 2 or weight.dim() != 1 or weight.numel() != rows.shape[1] or rows.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16
            or not rows.is_contiguous() or not weight.is_contiguous()):
        raise ValueError("rows must be contiguous [rows, hidden] bf16, the weight [hidden]")


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float, codes: torch.Tensor | None = None,
                     scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`quantize_rows` of :func:`rmsnorm`'s rows (the same bits), in one pass; hidden at most 4,096."""
    _check_norm_rows(weight, x)
    rows, hidden = x.shape
    codes, scales = _code_outputs(x, rows, hidden, codes, scales)
    _launch(x.get_device(), "ne_rmsnorm_quantize", x.data_ptr(), weight.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, hidden,
            eps)
    return codes, scales


def add_rmsnorm_quantize(residual: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, eps: float,
                         codes: torch.Tensor | None = None,
                         scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``residual += delta`` (bf16) in place, then :func:`quantize_rows` of its RMSNorm:
    :func:`add_rmsnorm` with the same bits and its rows as codes."""
    _check_norm_rows(weight, residual)
    _check_norm_rows(weight, delta)
    _check(residual.shape == delta.shape, "residual and delta must be of one shape")
    codes, scales = _code_outputs(residual, *residual.shape, codes, scales)
    _launch(residual.get_device(), "ne_add_rmsnorm_quantize", residual.data_ptr(), delta.data_ptr(), weight.data_ptr(),
            codes.data_ptr(), scales.data_ptr(), *residual.shape, eps)
    return codes, scales


def w8a8_gemm(
    codes: torch.Tensor,
    scales: torch.Tensor,
    weight_int8: torch.Tensor,
    weight_scale: torch.Tensor,
    epilogue: int = EPILOGUE_STORE,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``bf16((codes @ int8.T) * scales[:, None] * weight_scale)`` with an exact integer sum, on the
    weights of :func:`w8a16_gemm`; SwiGLU epilogue pairs 16 gate rows with 16 up rows.  ``k`` is a
    multiple of 16, at most 131,056; ``n`` is any number (SwiGLU: a multiple of 32)."""
    index = codes.get_device()
    if index < 0 or scales.get_device() != index or weight_int8.get_device() != index or weight_scale.get_device() != index:
        _require_gpu(codes, scales, weight_int8, weight_scale)  # names the devices
    whole = codes.is_contiguous()
    if codes.dtype != torch.int8 or codes.dim() != 2 or not whole and codes.stride(1) != 1:
        raise ValueError("codes must be [m, k] int8 with contiguous rows")
    if weight_int8.dtype != torch.int8 or weight_int8.dim() != 2 or not weight_int8.is_contiguous():
        raise ValueError("weight must be contiguous [n, k] int8")
    m, k = codes.shape
    n, k_weight = weight_int8.shape
    if k != k_weight:
        raise ValueError(f"k mismatch: codes have {k}, weight {k_weight}")
    if scales.dtype != torch.float32 or scales.numel() != m or not scales.is_contiguous():
        raise ValueError("scales must be contiguous fp32, one per row")
    if weight_scale.numel() != n or not weight_scale.is_contiguous():
        raise ValueError("weight_scale must be contiguous, one per weight row")
    n_out = n // 2 if epilogue == EPILOGUE_SWIGLU else n
    if out is None:
        out, ldy = codes.new_empty(m, n_out, dtype=torch.bfloat16), n_out
    elif out.shape != (m, n_out) or out.dtype != torch.bfloat16 or out.stride(1) != 1 and n_out > 1 or out.get_device() != index:
        raise ValueError(f"out must be bf16 [{m}, {n_out}] with contiguous rows on cuda:{index}")
    else:
        ldy = out.stride(0) if m > 1 else n_out
    _launch(index, "ne_w8a8_gemm", codes.data_ptr(), k if whole else codes.stride(0), scales.data_ptr(), weight_int8.data_ptr(),
            weight_scale.data_ptr(), dtype_code(weight_scale.dtype), m, n, k, out.data_ptr(), ldy, epilogue)
    return out


PROJ_TILE_ROWS = 80  # token rows per work-group of the W8A16 kernels
SPLITK_TILE_ROWS = 48  # token rows per work-group of the split-K product
PROJ_TILE_COLS = 64  # weight rows per work-group of the store / split-K kernels
TARGET_WORK_GROUPS = 256  # one per CU


def splitk_splits(m: int, n: int, k: int, max_splits: int = 4) -> int:
    """K splits that bring a narrow projection to about one work-group per CU (at most; 320
    rows of o / down give 7 x 16 tiles of 48 rows and 2 splits)."""
    tiles = -(-m // SPLITK_TILE_ROWS) * (n // PROJ_TILE_COLS)
    splits = max(1, min(max_splits, TARGET_WORK_GROUPS // max(tiles, 1)))
    while splits > 1 and k % (128 * splits):
        splits -= 1
    return splits


def w8a16_gemm_splitk(
    x: torch.Tensor,
    weight_int8: torch.Tensor,
    weight_scale: torch.Tensor,
    splits: int,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """fp32 ``[splits, m, n]`` partial products over K parts (scale applied), summed by
    ``splitk_add_rmsnorm``."""
    device = _require_gpu(x, weight_int8, weight_scale)
    _check(x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1, "x must be [m, k] bf16")
    _check(weight_int8.dtype == torch.int8 and weight_int8.dim() == 2, "weight must be [n, k] int8")
    _contig(weight_int8, "weight_int8")
    _contig(weight_scale, "weight_scale")
    m, k = x.shape
    n = weight_int8.shape[0]
    _check(weight_int8.shape[1] == k, f"k mismatch: x has {k}, weight {weight_int8.shape[1]}")
    _check(weight_scale.numel() == n, "one scale per weight row")
    if out is None:
        out = torch.empty((splits, m, n), dtype=torch.float32, device=device)
    _check(out.dtype == torch.float32 and out.is_contiguous() and out.numel() >= splits * m * n,
           "partials must be contiguous fp32 with room for [splits, m, n]")
    _native.call(
        "ne_w8a16_gemm_splitk",
        _ptr(x), x.stride(0), _ptr(weight_int8), _ptr(weight_scale),
        dtype_code(weight_scale.dtype), m, n, k, splits, _ptr(out), _stream(device),
    )
    return out


def lm_head_num_tiles(vocab: int) -> int:
    return int(_native.load().ne_lm_head_num_tiles(vocab))


def lm_head(
    x: torch.Tensor,
    weight: torch.Tensor,
    logits: torch.Tensor | bool = True,
    argmax_partials: torch.Tensor | bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``x [m, k] @ weight[n, k].T`` in bf16; optionally only per-tile argmax partials."""
    device = _require_gpu(x, weight)
    _check(x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16, "bf16 inputs required")
    _check(x.dim() == 2 and x.stride(1) == 1, "x must be [m, k]")
    _contig(weight, "weight")
    m, k = x.shape
    _check(weight.dim() == 2 and weight.shape[1] == k, f"k mismatch: x has {k}, weight {tuple(weight.shape)}")
    n = weight.shape[0]
    if logits is True:
        logits = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    elif logits is False:
        logits = None
    if argmax_partials is True:
        argmax_partials = torch.empty((m, lm_head_num_tiles(n)), dtype=torch.int64, device=device)
    elif argmax_partials is False:
        argmax_partials = None
    _native.call(
        "ne_lm_head",
        _ptr(x), x.stride(0), _ptr(weight), m, n, k, _ptr(logits),
        logits.stride(0) if logits is not None else 0, _ptr(argmax_partials), _stream(device),
    )
    return logits, argmax_partials


# ------------------------------------------------------------------- norms, RoPE
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out=None) -> torch.Tensor:
    device = _require_gpu(x, weight)
    _contig(x, "x")
    out = torch.empty_like(x) if out is None else out
    rows, hidden = x.shape
    _native.call("ne_rmsnorm", _ptr(x), _ptr(weight), _ptr(out), rows, hidden, float(eps),
                 _stream(device))
    return out


def add_rmsnorm(residual: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, eps: float,
                out=None) -> torch.Tensor:
    """``residual += delta`` (bf16) in place, then RMSNorm of the new residual."""
    device = _require_gpu(residual, delta, weight)
    _contig(residual, "residual")
    _contig(delta, "delta")
    out = torch.empty_like(residual) if out is None else out
    rows, hidden = residual.shape
    _native.call("ne_add_rmsnorm", _ptr(residual), _ptr(delta), _ptr(weight), _ptr(out), rows,
                 hidden, float(eps), _stream(device))
    return out


def splitk_add_rmsnorm(residual: torch.Tensor, partials: torch.Tensor, splits: int, weight: torch.Tensor,
                       eps: float, out=None) -> torch.Tensor:
    """``residual += bf16(sum of the split-K partials)`` in place, then RMSNorm."""
    device = _require_gpu(residual, partials, weight)
    _contig(residual, "residual")
    rows, hidden = residual.shape
    _check(partials.dtype == torch.float32 and partials.is_contiguous()
           and partials.numel() >= splits * rows * hidden, "partials must be fp32 [splits, rows, hidden]")
    out = torch.empty_like(residual) if out is None else out
    _native.call("ne_splitk_add_rmsnorm", _ptr(residual), _ptr(partials), splits, _ptr(weight), _ptr(out),
                 rows, hidden, float(eps), _stream(device))
    return out


def embed_rmsnorm(tokens: torch.Tensor, embed: torch.Tensor, weight: torch.Tensor, eps: float,
                  residual=None, out=None) -> tuple[torch.Tensor, torch.Tensor]:
    device = _require_gpu(tokens, embed, weight)
    _int32(tokens, "tokens")
    rows = tokens.numel()
    hidden = embed.shape[1]
    if residual is None:
        residual = torch.empty((rows, hidden), dtype=embed.dtype, device=device)
    if out is None:
        out = torch.empty((rows, hidden), dtype=embed.dtype, device=device)
    _native.call("ne_embed_rmsnorm", _ptr(tokens), _ptr(embed), _ptr(weight), _ptr(residual),
                 _ptr(out), rows, hidden, float(eps), _stream(device))
    return residual, out


def rope_table(positions: int, rope_theta: float, head_dim: int = HEAD_DIM) -> torch.Tensor:
    """[positions, 2, head_dim / 2] bf16 cos | sin on the CPU, built exactly as
    build_rotary_tables does (ne/models/qwen3.py:47-57): fp32 inverse frequencies,
    fp32 angles position * inv_freq, cos/sin in fp32, then rounded to bf16."""
    exps = torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim
    inv_freq = 1.0 / (rope_theta**exps)
    angles = torch.arange(positions).float()[:, None] * inv_freq
    return torch.stack([angles.cos(), angles.sin()], dim=1).to(torch.bfloat16).contiguous()


def qk_norm_rope_kv_write(
    qkv: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    eps: float,
    positions: torch.Tensor,
    rope_cos_sin: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    device = _require_gpu(qkv, q_norm_weight, k_norm_weight, positions, rope_cos_sin, slot_mapping,
                          k_cache, v_cache)
    _contig(qkv, "qkv")
    _int32(positions, "positions")
    _int32(slot_mapping, "slot_mapping")
    _check(rope_cos_sin.dtype == torch.bfloat16 and rope_cos_sin.dim() == 3 and rope_cos_sin.shape[1:] == (2, 64)
           and rope_cos_sin.is_contiguous(), "rope_cos_sin must be contiguous [positions, 2, 64] bf16")
    rows = qkv.shape[0]
    _check(qkv.shape[1] == (num_q_heads + 2 * num_kv_heads) * HEAD_DIM, "qkv width mismatch")
    if q_out is None:
        q_out = torch.empty((rows, num_q_heads, HEAD_DIM), dtype=torch.bfloat16, device=device)
    is_int8 = k_cache.dtype == torch.int8
    _native.call(
        "ne_qk_norm_rope_kv_write",
        _ptr(qkv), rows, num_q_heads, num_kv_heads, HEAD_DIM,
        _ptr(q_norm_weight), _ptr(k_norm_weight), float(eps),
        _ptr(positions), _ptr(rope_cos_sin), rope_cos_sin.shape[0], _ptr(slot_mapping),
        _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
        dtype_code(k_cache.dtype), dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16,
        _ptr(q_out), _stream(device),
    )
    return q_out


def w8a16_qkv_norm_rope_kv(
    x: torch.Tensor,
    w_int8: torch.Tensor,
    w_scale: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    eps: float,
    positions: torch.Tensor,
    rope_cos_sin: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    q_out: torch.Tensor,
) -> torch.Tensor:
    """The QKV projection with QK-norm, RoPE and the KV write fused into its epilogue:
    the same bits as :func:`w8a16_gemm` followed by :func:`qk_norm_rope_kv_write`."""
    device = _require_gpu(x, w_int8, w_scale, q_norm_weight, k_norm_weight, positions, rope_cos_sin,
                          slot_mapping, k_cache, v_cache, q_out)
    _check(x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1, "x must be [m, k] bf16")
    _check(w_int8.dtype == torch.int8 and w_int8.is_contiguous(), "w must be contiguous int8")
    _int32(positions, "positions")
    _int32(slot_mapping, "slot_mapping")
    _check(rope_cos_sin.dtype == torch.bfloat16 and rope_cos_sin.dim() == 3 and rope_cos_sin.shape[1:] == (2, 64)
           and rope_cos_sin.is_contiguous(), "rope_cos_sin must be contiguous [positions, 2, 64] bf16")
    rows, kdim = x.shape
    _check(w_int8.shape == ((num_q_heads + 2 * num_kv_heads) * HEAD_DIM, kdim), "w shape mismatch")
    _check(q_out.shape == (rows, num_q_heads, HEAD_DIM) and q_out.dtype == torch.bfloat16 and q_out.is_contiguous(),
           "q_out must be contiguous [rows, q_heads, 128] bf16")
    is_int8 = k_cache.dtype == torch.int8
    _native.call(
        "ne_w8a16_qkv_norm_rope_kv",
        _ptr(x), x.stride(0), _ptr(w_int8), _ptr(w_scale), dtype_code(w_scale.dtype), rows,
        num_q_heads, num_kv_heads, kdim,
        _ptr(q_norm_weight), _ptr(k_norm_weight), float(eps),
        _ptr(positions), _ptr(rope_cos_sin), rope_cos_sin.shape[0], _ptr(slot_mapping),
        dtype_code(k_cache.dtype), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
        dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16,
        _ptr(q_out), _stream(device),
    )
    return q_out


def w8a8_qkv_norm_rope_kv(
    codes: torch.Tensor,
    scales: torch.Tensor,
    w_int8: torch.Tensor,
    w_scale: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    eps: float,
    positions: torch.Tensor,
    rope_cos_sin: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    q_out: torch.Tensor,
) -> torch.Tensor:
    """:func:`w8a16_qkv_norm_rope_kv` from rows in 8 bits (:func:`quantize_rows`): the same bits as
    :func:`w8a8_gemm` followed by :func:`qk_norm_rope_kv_write` (of finite rows)."""
    device = _require_gpu(codes, scales, w_int8, w_scale, q_norm_weight, k_norm_weight, positions, rope_cos_sin,
                          slot_mapping, k_cache, v_cache, k_scale, v_scale, q_out)
    _check(codes.dtype == torch.int8 and codes.dim() == 2 and codes.stride(1) == 1, "codes must be [m, k] int8 with contiguous rows")
    rows, kdim = codes.shape
    _check(scales.dtype == torch.float32 and scales.numel() == rows and scales.is_contiguous(),
           "scales must be contiguous fp32, one per row")
    channels = (num_q_heads + 2 * num_kv_heads) * HEAD_DIM
    _check(w_int8.dtype == torch.int8 and w_int8.is_contiguous() and w_int8.shape == (channels, kdim),
           f"w must be contiguous int8 [{channels}, {kdim}]")
    _check(w_scale.numel() == channels and w_scale.is_contiguous(), "w_scale must be contiguous, one per weight row")
    for norm in (q_norm_weight, k_norm_weight):
        _check(norm.dtype == torch.bfloat16 and norm.numel() == HEAD_DIM and norm.is_contiguous(),
               f"norm weights must be contiguous bf16 [{HEAD_DIM}]")
    _int32(positions, "positions")
    _int32(slot_mapping, "slot_mapping")
    _check(positions.numel() >= rows and slot_mapping.numel() >= rows, "a position and a slot per row")
    _check(rope_cos_sin.dtype == torch.bfloat16 and rope_cos_sin.dim() == 3 and rope_cos_sin.shape[1:] == (2, 64)
           and rope_cos_sin.is_contiguous(), "rope_cos_sin must be contiguous [positions, 2, 64] bf16")
    _check(q_out.shape == (rows, num_q_heads, HEAD_DIM) and q_out.dtype == torch.bfloat16 and q_out.is_contiguous(),
           "q_out must be contiguous [rows, q_heads, 128] bf16")
    for cache in (k_cache, v_cache):
        _check(cache.dtype == k_cache.dtype and cache.dim() == 3 and cache.shape[1:] == (num_kv_heads, HEAD_DIM)
               and cache.is_contiguous(), f"caches must be contiguous [slots, {num_kv_heads}, {HEAD_DIM}] of one type")
    is_int8 = k_cache.dtype == torch.int8
    if is_int8:
        _check(k_scale is not None and v_scale is not None, "an int8 cache needs its scales")
        for cache, scale in ((k_cache, k_scale), (v_cache, v_scale)):
            _check(scale.dtype == k_scale.dtype and scale.shape == cache.shape[:2] and scale.is_contiguous(),
                   "cache scales must be contiguous [slots, kv_heads] of one type")
    _launch(device.index, "ne_w8a8_qkv_norm_rope_kv", codes.data_ptr(), codes.stride(0) if rows > 1 else kdim, scales.data_ptr(),
            w_int8.data_ptr(), w_scale.data_ptr(), dtype_code(w_scale.dtype), rows, num_q_heads, num_kv_heads, kdim,
            q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), float(eps), positions.data_ptr(), rope_cos_sin.data_ptr(),
            rope_cos_sin.shape[0], slot_mapping.data_ptr(), dtype_code(k_cache.dtype), k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr() if is_int8 else None, v_scale.data_ptr() if is_int8 else None,
            dtype_code(k_scale.dtype) if is_int8 else DTYPE_BF16, q_out.data_ptr())
    return q_out


def qkv_fusion_supported(k_cache: torch.Tensor, k_scale: torch.Tensor | None) -> bool:
    """Whether the fused QKV projections take this cache (bf16, or int8 with bf16/fp16 scales)."""
    if k_cache.dtype == torch.bfloat16:
        return True
    return k_cache.dtype == torch.int8 and k_scale is not None and k_scale.dtype in (torch.bfloat16, torch.float16)


# ------------------------------------------------------------------------ A9/A10
def accept(
    drafts: torch.Tensor,
    num_drafts: torch.Tensor,
    row_start: torch.Tensor,
    vocab: int,
    logits: torch.Tensor | None = None,
    argmax_partials: torch.Tensor | None = None,
    temperature: float | torch.Tensor = 0.0,
    top_p: float | torch.Tensor = 1.0,
    seeds: torch.Tensor | None = None,
    steps: torch.Tensor | None = None,
    out_tokens: torch.Tensor | None = None,
    num_out: torch.Tensor | None = None,
    history: torch.Tensor | None = None,
    history_len: torch.Tensor | None = None,
    num_cached: torch.Tensor | None = None,
    draft_logits: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
    draft_row_start: torch.Tensor | None = None,
    any_sampled: bool | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Accepted guesses plus one target token per sequence: ``(out_tokens [b, k+1], num_out [b])``.

    ``temperature`` / ``top_p``: one value for every sequence, or per-sequence fp32 device
    tensors (0 = greedy); with tensors, ``any_sampled`` says whether any temperature is
    positive (the host knows it without reading the device).  The draft distribution of
    each guess (sampled sequences): ``draft_logits`` (bf16, the draft model's logits; its
    distribution is the same temperature/top-p softmax) or ``draft_probs`` (fp32
    probabilities used as given), row ``draft_row_start[b] + i`` for guess i of sequence b;
    neither: the guesses count as deterministic (one-hot draft distribution)."""
    device = _require_gpu(drafts, num_drafts, row_start, logits, argmax_partials)
    _int32(drafts, "drafts")
    _int32(num_drafts, "num_drafts")
    _int32(row_start, "row_start")
    num_seqs, max_drafts = drafts.shape
    if isinstance(temperature, torch.Tensor):
        _check(temperature.dtype == torch.float32 and temperature.numel() >= num_seqs, "temperature [b] fp32")
        _check(any_sampled is not None, "per-sequence temperatures need any_sampled")
        temps = temperature
    else:
        any_sampled = float(temperature) > 0.0
        temps = torch.full((num_seqs,), float(temperature), dtype=torch.float32, device=device) if any_sampled \
            else None
    if isinstance(top_p, torch.Tensor):
        _check(top_p.dtype == torch.float32 and top_p.numel() >= num_seqs, "top_p [b] fp32")
        top_ps = top_p
    else:
        top_ps = None if float(top_p) >= 1.0 else torch.full((num_seqs,), float(top_p), dtype=torch.float32,
                                                                device=device)
    if logits is not None:
        _check(logits.dtype == torch.bfloat16 and logits.stride(1) == 1, "logits must be bf16 rows")
        _check(logits.shape[1] == vocab, "logits width must equal vocab")
    if any_sampled:
        _check(logits is not None, "sampled acceptance needs logits")
        _check(seeds is not None and steps is not None, "sampled acceptance needs seeds and steps")
        _check(seeds.dtype == torch.int64 and steps.dtype == torch.int64, "seeds/steps int64")
    _check(draft_logits is None or draft_probs is None, "give draft logits or draft probabilities, not both")
    draft = draft_logits if draft_logits is not None else draft_probs
    draft_dtype = DTYPE_BF16
    if draft is not None:
        _check(any_sampled, "draft distributions need sampled acceptance")
        want = torch.bfloat16 if draft_logits is not None else torch.float32
        _check(draft.dtype == want and draft.stride(1) == 1, f"draft rows must be {want} rows")
        _check(draft.shape[1] == vocab, "draft rows' width must equal vocab")
        _check(draft_row_start is not None, "draft rows need draft_row_start")
        _int32(draft_row_start, "draft_row_start")
        draft_dtype = dtype_code(draft.dtype)
    if out_tokens is None:
        out_tokens = torch.empty((num_seqs, max_drafts + 1), dtype=torch.int32, device=device)
    if num_out is None:
        num_out = torch.empty((num_seqs,), dtype=torch.int32, device=device)
    num_tiles = argmax_partials.shape[1] if argmax_partials is not None else 0
    _native.call(
        "ne_accept",
        _ptr(logits), logits.stride(0) if logits is not None else 0,
        _ptr(argmax_partials), num_tiles, vocab,
        _ptr(drafts), max_drafts, _ptr(num_drafts), _ptr(row_start), num_seqs,
        _ptr(temps), _ptr(top_ps), int(bool(any_sampled)), _ptr(seeds), _ptr(steps),
        _ptr(out_tokens), _ptr(num_out),
        _ptr(history), history.stride(0) if history is not None else 0,
        _ptr(history_len), _ptr(num_cached),
        _ptr(draft), draft_dtype, draft.stride(0) if draft is not None else 0, _ptr(draft_row_start),
        _stream(device),
    )
    return out_tokens, num_out


# ------------------------------------------------------------ adjusting logits
@dataclass(slots=True)  # (one is made per step; frozen would take twice as long)
class TokenPenalties:
    """Penalties for the tokens of each sequence so far, for :func:`adjust_logits`: device tensors that a
    step reads, so their contents may change between replays of a graph.

    ``repetition`` divides positive logits (and multiplies others) of tokens anywhere in the history,
    ``frequency`` times its count and ``presence`` are taken off a token of the output (what follows
    ``prompt_len``; None: the whole history).  Each is one value, or an fp32 tensor with one per row.
    Rows are the sequences' own (row i of sequence i) unless ``row_seq`` names them; ``row_drafts``
    of the guesses in ``drafts`` count as output too (a verify step's row i: the i guesses before it)."""

    history: torch.Tensor  # [seqs, capacity] int32
    history_len: torch.Tensor  # [seqs] int32
    prompt_len: torch.Tensor | None = None  # [seqs] int32
    repetition: float | torch.Tensor = 1.0
    presence: float | torch.Tensor = 0.0
    frequency: float | torch.Tensor = 0.0
    drafts: torch.Tensor | None = None  # [seqs, max_drafts] int32
    row_seq: torch.Tensor | None = None  # [rows] int32
    row_drafts: torch.Tensor | None = None  # [rows] int32


@dataclass(slots=True)  # (one is made per step; frozen would take twice as long)
class TokenBias:
    """Biases of single tokens, for :func:`adjust_logits`: entries ``start[r] .. start[r + 1]`` are row r's."""

    start: torch.Tensor  # [rows + 1] int32
    tokens: torch.Tensor  # [entries] int32
    values: torch.Tensor  # [entries] fp32

    @classmethod
    def from_dicts(cls, rows: list[dict[int, float] | None], device: torch.device) -> "TokenBias":
        """From each row's token -> bias on the host (None: no biases)."""
        start, tokens, values = [0], [], []
        for biases in rows:
            tokens += (biases or {}).keys()
            values += (biases or {}).values()
            start.append(len(tokens))
        flat = torch.tensor(start + tokens, dtype=torch.int32).to(device)
        return cls(flat[: len(start)], flat[len(start) :], torch.tensor(values, dtype=torch.float32).to(device))


def allowed_words(vocab: int) -> int:
    """32-bit words of a mask of ``vocab`` tokens."""
    return (vocab + 31) // 32


def allowed_mask(rows: list[list[int] | None], vocab: int, device: torch.device) -> torch.Tensor:
    """Masks ``[rows, words]`` int32 for :func:`adjust_logits` from each row's allowed tokens on the host
    (None: all): bit j of word w is token 32 w + j."""
    bits = np.zeros((len(rows), allowed_words(vocab) * 32), dtype=np.uint8)
    for row, tokens in zip(bits, rows):
        if tokens is None:
            row[:] = 1
        elif len(tokens):
            index = np.asarray(tokens, dtype=np.int64)
            _check(index.min() >= 0 and index.max() < vocab, f"allowed tokens outside [0, {vocab})")
            row[index] = 1
    words = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    return torch.from_numpy(words).to(device)


def _int32_pointer(tensor: torch.Tensor | None, shape: tuple, name: str, index: int) -> int | None:
    """The address (None for None) of a contiguous int32 argument of a given shape on device ``index``."""
    if tensor is None:
        return None
    if tensor.dtype != torch.int32 or tensor.shape != shape or not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}, got {tensor.dtype} {list(tensor.shape)}")
    if tensor.get_device() != index:
        raise RuntimeError(f"{name} is on {tensor.device}, the logits on cuda:{index}")
    return tensor.data_ptr()


def _int32_vector(tensor: torch.Tensor | None, n: int, name: str, index: int) -> int | None:
    """:func:`_int32_pointer` of ``n`` values in a row."""
    if tensor is None:
        return None
    if tensor.dtype != torch.int32 or tensor.dim() != 1 or tensor.numel() != n or not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{n}], got {tensor.dtype} {list(tensor.shape)}")
    if tensor.get_device() != index:
        raise RuntimeError(f"{name} is on {tensor.device}, the logits on cuda:{index}")
    return tensor.data_ptr()


def _row_values(value, rows: int, name: str, index: int) -> tuple:
    """(address or None, scalar) of a penalty: one value, or an fp32 one per row."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.dtype != torch.float32 or value.dim() != 1 or value.numel() != rows or not value.is_contiguous():
        raise ValueError(f"{name} must be one value or contiguous fp32 [{rows}]")
    if value.get_device() != index:
        raise RuntimeError(f"{name} is on {value.device}, the logits on cuda:{index}")
    return value.data_ptr(), 0.0


_NO_PENALTIES = (None, 0, 0, None, None, 0, None, 0, None, None, None, 1.0, None, 0.0, None, 0.0)


def _penalty_arguments(p: TokenPenalties, rows: int, index: int) -> tuple:
    h, drafts = p.history, p.drafts
    whole = h.is_contiguous()
    if h.dtype != torch.int32 or h.dim() != 2 or not whole and h.stride(1) != 1 and h.shape[1] > 1:
        raise ValueError("history must be [seqs, capacity] int32 with contiguous rows")
    if h.get_device() != index:
        raise RuntimeError(f"history is on {h.device}, the logits on cuda:{index}")
    seqs, capacity = h.shape
    if seqs == 0:  # whose row_seq could name no sequence
        _check(rows == 0 or p.row_seq is not None, "no sequences")
        return _NO_PENALTIES
    length = _int32_vector(p.history_len, seqs, "history_len", index)
    max_drafts = 0
    if drafts is not None:
        max_drafts = drafts.shape[-1] if drafts.dim() else 0
        _check(p.row_drafts is not None, "drafts need row_drafts")
    return (
        # (an empty tensor has no address, and its rows' guesses may still count)
        h.data_ptr() if capacity else length, capacity if whole else h.stride(0), capacity, length,
        _int32_vector(p.prompt_len, seqs, "prompt_len", index), seqs,
        _int32_pointer(drafts, (seqs, max_drafts), "drafts", index), max_drafts,
        _int32_vector(p.row_seq, rows, "row_seq", index), _int32_vector(p.row_drafts, rows, "row_drafts", index),
        *_row_values(p.repetition, rows, "repetition", index), *_row_values(p.presence, rows, "presence", index),
        *_row_values(p.frequency, rows, "frequency", index))


def _bias_arguments(bias: TokenBias, rows: int, index: int) -> tuple:
    entries = bias.tokens.numel()
    if (bias.values.dtype != torch.float32 or bias.values.dim() != 1 or bias.values.numel() != entries
            or not bias.values.is_contiguous()):
        raise ValueError(f"bias values must be contiguous fp32 [{entries}]")
    if bias.values.get_device() != index:
        raise RuntimeError(f"bias values are on {bias.values.device}, the logits on cuda:{index}")
    start = _int32_vector(bias.start, rows + 1, "bias start", index)
    tokens = _int32_vector(bias.tokens, entries, "bias tokens", index)
    return (start, tokens, bias.values.data_ptr(), entries) if entries else (None, None, None, 0)


def adjust_logits(
    logits: torch.Tensor,
    penalties: TokenPenalties | None = None,
    bias: TokenBias | None = None,
    allowed: torch.Tensor | None = None,
    allowed_rows: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``logits [rows, vocab]`` (bf16, fp16 or fp32) under penalties, then biases, then a mask, before
    :func:`sample` or :func:`accept`: in fp32, rounded once to ``out``'s type.

    ``out`` (default: allocated) is of the logits' type, fp32, or ``logits`` itself.  ``allowed`` is
    int32 ``[masks, allowed_words(vocab)]`` (:func:`allowed_mask`); a token whose bit is not set
    becomes -inf, whatever its logit was.  ``allowed_rows [rows]`` int32 names each row's mask (default:
    its own index; negative: no mask, one past the masks: no token).  Tokens outside the vocabulary
    count nowhere."""
    if not logits.is_cuda:
        _require_gpu(logits)
    index, dtype = logits.get_device(), logits.dtype
    whole = logits.is_contiguous()
    if logits.dim() != 2 or not whole and logits.stride(1) != 1 and logits.shape[1] != 1:
        raise ValueError("logits must be [rows, vocab] with contiguous rows")
    code = dtype_code(dtype)
    if code == DTYPE_INT8:
        raise ValueError("logits must be bf16, fp16 or fp32")
    rows, vocab = logits.shape
    if out is None:
        out = logits.new_empty(rows, vocab)
    elif out is not logits:
        if (out.dtype not in (dtype, torch.float32) or out.shape != logits.shape or out.get_device() != index
                or out.stride(1) != 1 and vocab > 1):
            raise ValueError(f"out must be {dtype} or fp32 [{rows}, {vocab}] with contiguous rows on cuda:{index}")
    allowed_arguments = (None, 0, 0, None)
    if allowed is not None:
        masks, words = allowed.shape[0], allowed_words(vocab)
        if masks == 0 and rows > 0:
            raise ValueError("no masks")
        allowed_arguments = (_int32_pointer(allowed, (masks, words), "allowed", index), words, masks,
                             _int32_vector(allowed_rows, rows, "allowed_rows", index))
    _launch(index, "ne_adjust_logits", logits.data_ptr(), code, vocab if whole else logits.stride(0), rows, vocab,
            *(_NO_PENALTIES if penalties is None else _penalty_arguments(penalties, rows, index)),
            *((None, None, None, 0) if bias is None else _bias_arguments(bias, rows, index)), *allowed_arguments,
            out.data_ptr(), _DTYPE_CODES[out.dtype], vocab if out.is_contiguous() else out.stride(0))
    return out


# ---------------------------------------------------------------------- sampling
def _row_parameter(value, rows: int, dtype: torch.dtype, name: str, device: torch.device):
    """(device pointer or None, scalar) of a sampling parameter: one value, or one per row."""
    if not isinstance(value, torch.Tensor):
        return None, value
    _check(value.dtype == dtype and value.dim() == 1 and value.shape[0] == rows and value.is_contiguous(),
           f"{name} must be one value or contiguous {dtype} [{rows}]")
    if value.device != device:
        raise RuntimeError(f"{name} is on {value.device}, the logits on {device}")
    return value.data_ptr(), 0


def sample(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
    out: torch.Tensor | None = None,
    probs: bool | torch.Tensor = False,
    workspace: torch.Tensor | None = None,
):
    """A token per row of ``logits [rows, vocab]`` (bf16, fp16 or fp32) from ``uniforms [rows]``
    fp32 in [0, 1): int32 ``[rows]``, and with ``probs`` (True, or an fp32 tensor to write) the
    filtered distribution ``[rows, vocab]`` too, as :func:`accept` takes it for ``draft_probs``.

    Tokens are ordered by logit, equal ones by index.  Kept are the first ``top_k`` (0: all), of
    those the fewest that reach ``top_p`` of their weight, of those the ones at least ``min_p``
    times as likely as the first (above 1: the first alone); the token is the first whose running
    weight exceeds the uniform's share of the kept weight.  ``temperature`` 0 takes the argmax.  Each parameter is
    one value or a tensor ``[rows]`` (fp32; ``top_k`` int32).  Weights are integers in units of
    2^-45 (151,936 tokens) of the row's largest, so a call repeated gives the same bits; a batch of
    another size splits its rows otherwise, and rounds a border's sum by other units.  NaN and -inf logits are never
    drawn; a row without any other gives -1.  ``workspace`` (default: allocated here) is uint8 of
    :func:`sample_workspace_bytes`, of one call at a time."""
    device = _require_gpu(logits, uniforms)
    _check(logits.dim() == 2 and logits.stride(1) == 1 or logits.dim() == 2 and logits.shape[1] == 1,
           "logits must be [rows, vocab] with contiguous rows")
    _check(logits.dtype in (torch.bfloat16, torch.float16, torch.float32), "logits must be bf16, fp16 or fp32")
    rows, vocab = logits.shape
    if uniforms.dtype != torch.float32 or uniforms.dim() != 1 or uniforms.shape[0] != rows or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be contiguous fp32 [{rows}]")
    t_ptr, t = _row_parameter(temperature, rows, torch.float32, "temperature", device)
    k_ptr, k = _row_parameter(top_k, rows, torch.int32, "top_k", device)
    p_ptr, p = _row_parameter(top_p, rows, torch.float32, "top_p", device)
    m_ptr, m = _row_parameter(min_p, rows, torch.float32, "min_p", device)
    if t_ptr is None and not 0.0 <= t < math.inf:
        raise ValueError(f"temperature must be finite and >= 0, got {t}")
    _check(p == p and m == m, "top_p and min_p must not be NaN")
    k = max(0, min(int(k), vocab))
    if out is None:
        out = torch.empty((rows,), dtype=torch.int32, device=device)
    elif out.dtype != torch.int32 or tuple(out.shape) != (rows,) or not out.is_contiguous() or out.device != device:
        raise ValueError(f"out must be contiguous int32 [{rows}] on {device}")
    table = None
    if isinstance(probs, torch.Tensor):
        table = probs
        _check(table.dtype == torch.float32 and tuple(table.shape) == (rows, vocab) and table.device == device
               and (table.stride(1) == 1 or vocab == 1), f"probs must be fp32 [{rows}, {vocab}] on {device}")
    elif probs:
        table = torch.empty((rows, vocab), dtype=torch.float32, device=device)
    if rows > 0:
        code = dtype_code(logits.dtype)
        nbytes = _native.load().ne_sample_workspace_size(rows, vocab, code)
        if nbytes == 0:
            raise ValueError(f"unsupported sampling shape: {rows} rows of {vocab}")
        if workspace is None:
            workspace = torch.empty((nbytes,), dtype=torch.uint8, device=device)
        elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.device != device:
            raise ValueError(f"workspace must be contiguous uint8 on {device}")
        _call_on(device, "ne_sample", logits.data_ptr(), code, logits.stride(0) if rows > 1 else vocab, rows, vocab,
                 uniforms.data_ptr(), t_ptr, t, k_ptr, k, p_ptr, p, m_ptr, m, out.data_ptr(),
                 None if table is None else table.data_ptr(), 0 if table is None or rows < 2 else table.stride(0),
                 workspace.data_ptr(), workspace.numel(), _stream(device))
    return out if table is None else (out, table)


def sample_workspace_bytes(rows: int, vocab: int, dtype: torch.dtype) -> int:
    """Bytes of workspace that :func:`sample` needs for these logits (by itself it allocates them)."""
    return _native.load().ne_sample_workspace_size(rows, vocab, dtype_code(dtype))


def prepare_verify_step(
    history: torch.Tensor,
    history_len: torch.Tensor,
    drafts: torch.Tensor,
    num_drafts: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    scratch_slot: int,
    tokens: torch.Tensor,
    positions: torch.Tensor,
    slot_mapping: torch.Tensor,
    q_start: torch.Tensor,
    q_len: torch.Tensor,
    ctx_len: torch.Tensor,
) -> None:
    """Pack a batched verify step on the device: rows, positions, slots, attention metadata."""
    device = _require_gpu(history, history_len, drafts, num_drafts, block_tables, tokens, positions,
                          slot_mapping, q_start, q_len, ctx_len)
    for name, t in (("history", history), ("history_len", history_len), ("drafts", drafts),
                    ("num_drafts", num_drafts), ("block_tables", block_tables), ("tokens", tokens),
                    ("positions", positions), ("slot_mapping", slot_mapping), ("q_start", q_start),
                    ("q_len", q_len), ("ctx_len", ctx_len)):
        _int32(t, name)
    num_seqs, max_drafts = drafts.shape
    _check(tokens.numel() >= num_seqs * (max_drafts + 1), "tokens too small for the padded rows")
    _native.call(
        "ne_prepare_verify_step",
        _ptr(history), history.stride(0), _ptr(history_len), _ptr(drafts), max_drafts, _ptr(num_drafts),
        _ptr(block_tables), block_tables.stride(0), block_size, scratch_slot, num_seqs,
        _ptr(tokens), _ptr(positions), _ptr(slot_mapping), _ptr(q_start), _ptr(q_len), _ptr(ctx_len),
        _stream(device),
    )


def advance_step_counts(history_len: torch.Tensor, num_out: torch.Tensor, max_new_tokens: torch.Tensor,
                        num_generated: torch.Tensor, steps: torch.Tensor, num_guesses: torch.Tensor,
                        k: int) -> None:
    """After a verify step: active sequences add their emitted tokens to the generated
    count, advance the sampling step and get the next step's guess count
    (speculative_generator.py:71-72); inactive ones (history_len 0) get 0 guesses."""
    device = _require_gpu(history_len, num_out, max_new_tokens, num_generated, steps, num_guesses)
    for name, t in (("history_len", history_len), ("num_out", num_out), ("max_new_tokens", max_new_tokens),
                    ("num_generated", num_generated), ("num_guesses", num_guesses)):
        _int32(t, name)
    _check(steps.dtype == torch.int64 and steps.is_contiguous(), "steps must be contiguous int64")
    n = history_len.numel()
    _check(all(t.numel() >= n for t in (num_out, max_new_tokens, num_generated, steps, num_guesses)),
           "per-sequence arrays shorter than history_len")
    _native.call("ne_advance_step_counts", _ptr(history_len), _ptr(num_out), _ptr(max_new_tokens),
                 _ptr(num_generated), _ptr(steps), _ptr(num_guesses), k, n, _stream(device))


def advance_and_propose(history: torch.Tensor, history_len: torch.Tensor, num_out: torch.Tensor,
                        max_new_tokens: torch.Tensor, num_generated: torch.Tensor, steps: torch.Tensor,
                        num_guesses: torch.Tensor, k: int, max_ngram: int, drafts: torch.Tensor,
                        num_drafts: torch.Tensor, min_ngram: int = 1) -> None:
    """:func:`advance_step_counts` then :func:`ngram_propose` with ``num_tokens =
    num_guesses`` in one launch (the same results): the tail of a verify step."""
    device = _require_gpu(history, history_len, num_out, max_new_tokens, num_generated, steps, num_guesses,
                          drafts, num_drafts)
    for name, t in (("history", history), ("history_len", history_len), ("num_out", num_out),
                    ("max_new_tokens", max_new_tokens), ("num_generated", num_generated),
                    ("num_guesses", num_guesses), ("drafts", drafts), ("num_drafts", num_drafts)):
        _int32(t, name)
    _check(steps.dtype == torch.int64 and steps.is_contiguous(), "steps must be contiguous int64")
    _check(history.dim() == 2 and drafts.dim() == 2 and drafts.is_contiguous(),
           "history [num_seqs, capacity], drafts [num_seqs, max_drafts]")
    n = history.shape[0]
    _check(all(t.numel() >= n for t in (history_len, num_out, max_new_tokens, num_generated, steps, num_guesses,
                                        num_drafts)) and drafts.shape[0] >= n,
           "per-sequence arrays shorter than the histories")
    _native.call("ne_advance_and_propose", _ptr(history), history.stride(0), _ptr(history_len), _ptr(num_out),
                 _ptr(max_new_tokens), _ptr(num_generated), _ptr(steps), _ptr(num_guesses), k, n, max_ngram,
                 min_ngram, drafts.shape[1], _ptr(drafts), _ptr(num_drafts), _stream(device))


def copy_bytes(src: torch.Tensor, dst: torch.Tensor) -> None:
    device = _require_gpu(src, dst)
    nbytes = src.numel() * src.element_size()
    _check(dst.numel() * dst.element_size() >= nbytes, "dst too small")
    _native.call("ne_copy_bytes", _ptr(src), _ptr(dst), nbytes, _stream(device))
