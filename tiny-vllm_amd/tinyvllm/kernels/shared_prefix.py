"""Paged decode attention over shared prefixes (no reference counterpart: the
reference's decode reads a page once for every row that points at it,
tinyvllm/kernels/paged_decode.cu:92-466)."""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

import numpy as np
import torch

from tinyvllm._validation import _check_positive_int
from tinyvllm.kernels._extension import (
    cache_format, check, dtype_code, load_kernels, on_device, require_gpu, stream_of,
)
from tinyvllm.paged_kv import PagedKVCache
from tinyvllm.runtime.contracts import SingleQueryMetadata

_HEADER = 16     # words of a plan ahead of its lists
_TASK_WORDS = 8
_capturing = torch._C._cuda_isCurrentStreamCapturing


def takes_shared_prefix(num_heads: int, num_kv_heads: int, head_dim: int) -> bool:
    """Whether the shared-prefix kernels have this geometry."""
    return (0 < head_dim <= 256 and head_dim % 8 == 0 and 0 < num_kv_heads
            and num_heads % num_kv_heads == 0 and num_heads <= 4096)


class SharedPrefixPlan:
    """How one decode step's attention is cut into tasks, kept on the device
    for every layer of the step.

    ``update`` replaces the plan in place (same device address), so a captured
    call replays over whatever plan was last uploaded, as long as that has the
    captured number of rows. Its upload is ordered on the current stream: calls
    by the old plan on other streams must be done, and calls by the new one
    there must wait for it. It is refused under graph capture."""

    def __init__(self, *, num_heads: int, num_kv_heads: int, head_dim: int, block_size: int,
                 max_rows: int, device: torch.device | str) -> None:
        for name, value in (("num_heads", num_heads), ("num_kv_heads", num_kv_heads),
                            ("head_dim", head_dim), ("block_size", block_size),
                            ("max_rows", max_rows)):
            _check_positive_int(name, value)
        lib = load_kernels()
        geometry = (max_rows, num_heads, num_kv_heads)
        words = int(lib.tvllm_shared_prefix_plan_words(*geometry))
        if not words or not takes_shared_prefix(num_heads, num_kv_heads, head_dim):
            raise ValueError("no shared-prefix kernel for this geometry (head_dim a multiple of "
                             "8 up to 256, heads a multiple of the KV heads)")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.block_size, self.max_rows = block_size, max_rows
        self.max_tasks = int(lib.tvllm_shared_prefix_max_tasks(*geometry))
        self.max_workspace_bytes = int(lib.tvllm_shared_prefix_workspace_size(*geometry, head_dim))
        self.device = torch.device(device)
        on_gpu = self.device.type == "cuda"
        if on_gpu and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.host = torch.zeros(words, dtype=torch.int32, pin_memory=on_gpu)
        self.data = torch.zeros(words, dtype=torch.int32, device=self.device)
        self._uploaded = torch.cuda.Event() if on_gpu else None
        self._pending = False
        self.num_rows = 0        # of the plan last made; the grid and the
        self.num_tasks = 0       # workspace that it needs
        self.workspace_bytes = 0
        self._least = 0          # of a workspace: rows without keys need one too

    def update(self, context_lens: Sequence[int], row_groups: Sequence[int],
               prefix_lens: Sequence[int]) -> None:
        """Plan a step: row r has ``context_lens[r]`` tokens (0: padding) and is
        in group ``row_groups[r]`` (-1: none); the first ``prefix_lens[g]``
        tokens, whole blocks, of group g's rows lie in the same blocks."""
        lengths, groups, prefixes = (np.ascontiguousarray(x, dtype=np.int64)
                                     for x in (context_lens, row_groups, prefix_lens))
        if lengths.ndim != 1 or groups.shape != lengths.shape or prefixes.ndim != 1:
            raise ValueError("context_lens and row_groups must be vectors of one length")
        if len(lengths) > self.max_rows:
            raise ValueError("more rows than the plan holds")
        if self._uploaded is not None and _capturing():
            raise RuntimeError("a plan cannot be updated under graph capture")
        if self._pending:  # stream order does not hold back the CPU's writes
            self._uploaded.synchronize()
            self._pending = False
        tasks, need = ctypes.c_int64(), ctypes.c_int64()
        try:
            check(load_kernels().tvllm_shared_prefix_plan(
                lengths.ctypes.data, groups.ctypes.data, prefixes.ctypes.data, len(lengths),
                len(prefixes), self.max_rows, self.num_heads, self.num_kv_heads, self.head_dim,
                self.block_size, self.host.data_ptr(), self.host.numel(), ctypes.byref(tasks),
                ctypes.byref(need)))
        except RuntimeError as exc:
            raise ValueError(str(exc)) from None
        used = _HEADER + 3 * self.max_rows + _TASK_WORDS * tasks.value
        if self._uploaded is None:
            self.data[:used].copy_(self.host[:used])
        else:
            with torch.cuda.device(self.device):
                self.data[:used].copy_(self.host[:used], non_blocking=True)
                self._uploaded.record()
            self._pending = True
        self.num_rows, self.num_tasks = len(lengths), tasks.value
        self.workspace_bytes = need.value
        self._least = need.value if need.value or lengths.all() else 16


def find_shared_prefixes(table_ids, table_offsets, context_lens, block_size: int
                         ) -> tuple[np.ndarray, np.ndarray]:
    """(group of each row or -1, prefix tokens of each group) of a batch whose
    row r's block ids are ``table_ids[table_offsets[r]:table_offsets[r + 1]]``:
    rows with the same first block form a group, whose prefix is the longest
    run of leading blocks that they all have, the block of a row's newest token
    (which the step writes) left out."""
    ids = np.asarray(table_ids, dtype=np.int64)
    offsets = np.asarray(table_offsets, dtype=np.int64)
    lengths = np.asarray(context_lens, dtype=np.int64)
    groups = np.full(len(lengths), -1, dtype=np.int64)
    usable = np.maximum(lengths - 1, 0) // block_size
    rows = np.flatnonzero(usable)
    prefixes = []
    if len(rows) > 1:
        _, inverse, counts = np.unique(ids[offsets[rows]], return_inverse=True,
                                       return_counts=True)
        for g in np.flatnonzero(counts > 1):
            members = rows[inverse == g]
            common = int(usable[members].min())
            tables = ids[offsets[members][:, None] + np.arange(common)]
            differ = np.flatnonzero((tables != tables[0]).any(axis=0))
            groups[members] = len(prefixes)
            prefixes.append((int(differ[0]) if len(differ) else common) * block_size)
    return groups, np.asarray(prefixes, dtype=np.int64)


def paged_decode_shared_prefix(
    q: torch.Tensor,
    cache: PagedKVCache,
    layer_idx: int,
    metadata: SingleQueryMetadata,
    plan: SharedPrefixPlan,
    output: torch.Tensor,
    *,
    scale: float,
    workspace: torch.Tensor | None = None,
) -> None:
    """``paged_decode_attention`` by a plan: keys that the rows of a group
    share are read and multiplied once for all of them.

    The context lengths are those of ``plan.update`` (``metadata.context_lens``
    is not read); ``output`` is memory of its own, and no row of it is listed
    twice. ``workspace`` (optional, uint8, 16-byte aligned): at least
    ``plan.workspace_bytes``, under capture ``plan.max_workspace_bytes``; when
    omitted it is allocated from torch's caching allocator (inside graph
    capture that is the graph's private pool)."""
    key, value, layers = cache.key, cache.value, cache.num_layers
    rows, blocks = metadata.query_rows, metadata.block_table_ids
    offsets, data = metadata.block_table_offsets, plan.data
    if not -layers <= layer_idx < layers:
        raise IndexError("layer_idx is not a layer of the cache")
    device = require_gpu(q, key, value, output, rows, blocks, offsets, data)
    if q.dim() != 3:
        raise RuntimeError("Q must be a GPU [tokens, heads, dim] tensor")
    strides = key.stride()
    if strides != value.stride():
        raise RuntimeError("K/V caches must share one layout")
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("Q must use float16 or bfloat16")
    if (key.dtype != dtype and not cache.fp8) or output.dtype != dtype:
        raise RuntimeError("Q/K/V/output must share device and dtype")
    q_token, q_head, q_dim = q.stride()
    if output.shape != q.shape or q_dim != 1 or output.stride(2) != 1:
        raise RuntimeError("output must match Q shape with unit last stride")
    for tensor in (rows, blocks, offsets):
        if tensor.dtype != torch.long or tensor.dim() != 1 or not tensor.is_contiguous():
            raise RuntimeError("metadata must be contiguous GPU int64 vectors on Q's device")
    num_rows = rows.numel()
    if offsets.numel() != num_rows + 1:
        raise RuntimeError("metadata lengths must align")
    _, heads, dim = q.shape
    if (plan.num_heads, plan.num_kv_heads, plan.head_dim, plan.block_size) != (
            heads, cache.num_kv_heads, dim, cache.block_size):
        raise RuntimeError("the plan was made for another geometry")
    if plan.num_rows != num_rows:
        raise RuntimeError("the plan was made for another number of rows")
    if num_rows == 0:
        return
    with on_device(device):
        # A captured call is replayed over later plans: it takes the bounds.
        if _capturing():
            tasks, need = plan.max_tasks, plan.max_workspace_bytes
        else:
            tasks, need = plan.num_tasks, plan._least
        if need and (workspace is None or workspace.numel() < need):
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        elif workspace is not None and (
                require_gpu(q, workspace) != device or workspace.dtype != torch.uint8
                or not workspace.is_contiguous()):
            raise RuntimeError("workspace must be contiguous uint8 on Q's device")
        # Addresses of the layer, without views of it (1.2 us each).
        skip = layer_idx % layers * strides[0] * key.element_size()
        check(load_kernels().tvllm_paged_decode_shared_prefix(
            q.data_ptr(), q_token, q_head, key.data_ptr() + skip, value.data_ptr() + skip,
            output.data_ptr(), output.stride(0), output.stride(1), rows.data_ptr(),
            blocks.data_ptr(), offsets.data_ptr(), data.data_ptr(), num_rows, plan.max_rows,
            tasks, heads, plan.num_kv_heads, dim, cache.num_slots, strides[1], strides[2],
            cache.block_size, float(scale), workspace.data_ptr() if need else None, need,
            dtype_code(dtype), *cache_format(cache), stream_of(device),
        ))
