"""Logit controls in front of the sampler: penalties, biases and token masks
(no reference counterpart: the reference samples from the logits as they are,
tinyvllm/sampling.py:21-72)."""
from __future__ import annotations

import torch

from tinyvllm.kernels._extension import (
    check, dtype_code, load_kernels, on_device, require_gpu, stream_of,
)
from tinyvllm.kernels.sampling import _check_logits


def _vector(tensor: torch.Tensor | None, dtype: torch.dtype, size: int, index: int,
            name: str) -> int | None:
    """Address of a vector of ``size`` (-1: any) elements, None without one."""
    if tensor is None:
        return None
    if (tensor.dtype != dtype or tensor.dim() != 1 or not tensor.is_contiguous()
            or (tensor.numel() != size and size >= 0)):
        raise RuntimeError(f"{name} must be a contiguous {dtype} vector"
                           + ("" if size < 0 else f" of {size}"))
    if tensor.get_device() != index:
        raise RuntimeError("tensors must share one GPU device")
    return tensor.data_ptr() or None  # (0: empty)


def apply_logit_controls(
    logits: torch.Tensor,
    *,
    repetition: torch.Tensor | None = None,
    presence: torch.Tensor | None = None,
    frequency: torch.Tensor | None = None,
    history: torch.Tensor | None = None,
    slots: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    prompt_lens: torch.Tensor | None = None,
    newest: torch.Tensor | None = None,
    bias_tokens: torch.Tensor | None = None,
    bias_values: torch.Tensor | None = None,
    bias_offsets: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    mask_rows: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Each row's controls applied to its logits [rows, vocab], in this order:

    * tokens in the row's history: positive logits divided by ``repetition[r]``,
      others multiplied by it; then ``frequency[r]`` times the number of times
      the token stands in the answer part subtracted, and ``presence[r]`` if
      it stands there (float32 [rows]; None: 1, 0 and 0);
    * ``bias_values[j]`` added to token ``bias_tokens[j]`` for
      ``bias_offsets[r] <= j < bias_offsets[r + 1]`` (int32, float32, int64
      [rows + 1]); of a token that a row lists twice the last entry counts;
    * tokens whose bit in ``mask[mask_rows[r]]`` is 0 set to -inf (token i: bit
      i % 32 of word i // 32; int32 [masks, words], int64 [rows], -1: no mask).

    ``history`` (int32 [slots, capacity]) holds token ids by position; row r's
    is ``history[slots[r], :lengths[r]]`` (int64 [rows]; slot -1: none), of
    which the first ``prompt_lens[r]`` are its prompt. ``newest`` (int64
    [rows]), where given, is the token at position ``lengths[r] - 1``: it is
    counted and written into the history (rows then need slots of their own).
    Ids outside the vocabulary, slots and mask rows outside their tensors count
    as none.

    ``out`` receives the result: None for a new tensor of the logits' type, a
    float32 or same-type tensor of their shape, or ``logits`` itself. Computed
    in float32 and rounded once to ``out``'s type."""
    _check_logits(logits)
    rows, vocab = logits.shape
    device = require_gpu(logits)
    index = device.index
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=device)
    elif (out.shape != logits.shape or out.stride(1) != 1
          or out.dtype not in (logits.dtype, torch.float32)):
        raise RuntimeError("out must be float32 or of the logits' type, of their shape, with "
                           "unit last stride")
    elif out.get_device() != index:
        raise RuntimeError("tensors must share one GPU device")
    if history is None:
        if not (repetition is presence is frequency is newest is None):
            raise RuntimeError("penalties need a history")
    elif slots is None or lengths is None or prompt_lens is None:
        raise RuntimeError("a history needs slots, lengths and prompt_lens")
    elif history.dtype != torch.int32 or history.dim() != 2 or not history.is_contiguous():
        raise RuntimeError("history must be contiguous int32 [slots, capacity]")
    if (bias_offsets is None) != (bias_tokens is None) or (bias_tokens is None) != (
            bias_values is None):
        raise RuntimeError("biases need tokens, values and offsets")
    if bias_tokens is not None and bias_tokens.numel() != bias_values.numel():
        raise RuntimeError("bias_tokens and bias_values must align")
    if (mask is None) != (mask_rows is None):
        raise RuntimeError("masks need mask_rows")
    if mask is not None and (mask.dtype != torch.int32 or mask.dim() != 2 or mask.stride(1) != 1
                             or (mask.shape[0] and mask.shape[1] < -(-vocab // 32))):
        raise RuntimeError("mask must be int32 [masks, words] with unit last stride and a bit "
                           "for every token")
    history_ptr = mask_ptr = None
    num_slots = capacity = masks = mask_stride = num_bias = 0
    if history is not None:
        if history.get_device() != index:
            raise RuntimeError("tensors must share one GPU device")
        num_slots, capacity = history.shape
        history_ptr = history.data_ptr() or None
    if mask is not None:
        if mask.get_device() != index:
            raise RuntimeError("tensors must share one GPU device")
        masks, mask_stride, mask_ptr = mask.shape[0], mask.stride(0), mask.data_ptr() or None
    if bias_tokens is not None:
        num_bias = bias_values.numel()
    f32, i64 = torch.float32, torch.long
    args = (
        _vector(repetition, f32, rows, index, "repetition"),
        _vector(presence, f32, rows, index, "presence"),
        _vector(frequency, f32, rows, index, "frequency"),
        history_ptr, num_slots, capacity,
        _vector(slots, i64, rows, index, "slots"),
        _vector(lengths, i64, rows, index, "lengths"),
        _vector(prompt_lens, i64, rows, index, "prompt_lens"),
        _vector(newest, i64, rows, index, "newest"),
        _vector(bias_tokens, torch.int32, num_bias, index, "bias_tokens"),
        _vector(bias_values, f32, -1, index, "bias_values"),
        _vector(bias_offsets, i64, rows + 1, index, "bias_offsets"), num_bias,
        mask_ptr, masks, mask_stride, _vector(mask_rows, i64, rows, index, "mask_rows"))
    if rows == 0:
        return out
    with on_device(device):
        check(load_kernels().tvllm_logit_controls(
            logits.data_ptr(), rows, vocab, logits.stride(0), *args, out.data_ptr(),
            out.stride(0), dtype_code(logits.dtype), dtype_code(out.dtype), stream_of(device),
        ))
    return out
