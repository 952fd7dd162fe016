"""Logit controls of a batch's requests, with what they need on the device (no
reference counterpart: its requests carry no penalties, biases or masks).

One row per request slot: the request's token ids by position and, where it
has ``allowed_token_ids``, their bit mask. A row is filled when a request's
first sampled step comes; from then on the kernel itself appends each step's
newest token, which in a pipelined engine the host does not know yet.
"""
from __future__ import annotations

import numpy as np
import torch

from tinyvllm.batch import PreparedBatch
from tinyvllm.kernels.logits import apply_logit_controls


class RequestControls:
    def __init__(self, *, max_num_seqs: int, max_model_len: int, vocab_size: int,
                 device: torch.device) -> None:
        self.device = device
        self.capacity = max_num_seqs
        self.vocab_size = vocab_size
        self.history = torch.zeros((max_num_seqs, max_model_len), dtype=torch.int32,
                                   device=device)
        self.masks = torch.zeros((max_num_seqs, -(-vocab_size // 32)), dtype=torch.int32,
                                 device=device)
        # What each row holds: its request, its tokens, whose mask.
        self._owner = [-1] * max_num_seqs
        self._tokens = [0] * max_num_seqs
        self._mask_owner = [-1] * max_num_seqs

    def forget(self, request_id: int) -> None:
        """The request ended: a later one of that id starts anew."""
        for owners in (self._owner, self._mask_owner):
            for slot, owner in enumerate(owners):
                if owner == request_id:
                    owners[slot] = -1

    def _fill_history(self, slot: int, request_id: int, history, length: int) -> None:
        """Upload what row ``slot`` lacks of the request's first ``length`` - 1
        tokens (the kernel writes the last)."""
        kept = self._tokens[slot] if self._owner[slot] == request_id else 0
        if kept != length - 1:
            if kept > length - 1:
                kept = 0
            prompt, answer = history
            ids = np.asarray((list(prompt) + list(answer))[kept:length - 1], dtype=np.int64)
            if len(ids) != length - 1 - kept or (len(ids) and ids.min() < 0):
                raise ValueError("a controlled request's tokens are not known yet")
            self.history[slot, kept:length - 1].copy_(
                torch.from_numpy(ids.astype(np.int32)), non_blocking=True)
        self._owner[slot] = request_id
        self._tokens[slot] = length

    def _fill_mask(self, slot: int, request_id: int, allowed) -> None:
        if self._mask_owner[slot] == request_id:
            return
        ids = np.fromiter(allowed, dtype=np.int64, count=len(allowed))
        if ids.max() >= self.vocab_size:
            raise ValueError("allowed token ID is out of vocabulary range")
        words = np.zeros(self.masks.shape[1], dtype=np.uint32)
        np.bitwise_or.at(words, ids // 32, np.uint32(1) << (ids % 32).astype(np.uint32))
        self.masks[slot].copy_(torch.from_numpy(words.view(np.int32)), non_blocking=True)
        self._mask_owner[slot] = request_id

    def apply(self, logits: torch.Tensor, batch: PreparedBatch, newest: torch.Tensor) -> None:
        """Change the sampled rows' logits in place. ``newest`` (int64 on the
        device): each sampled row's last input token."""
        rows = batch.num_samples
        item_of = {rid: i for i, rid in enumerate(batch.request_ids)}
        ints = np.zeros((4, rows), dtype=np.int64)  # slots, lengths, prompt lengths, mask rows
        ints[0] = ints[3] = -1
        floats = np.zeros((3, rows), dtype=np.float32)
        floats[0] = 1.0
        offsets = np.zeros(rows + 1, dtype=np.int64)
        tokens: list[int] = []
        values: list[float] = []
        any_mask = False
        for r, (rid, params, history) in enumerate(zip(
                batch.sample_request_ids, batch.sampling_params, batch.sample_histories)):
            if params.controlled:
                item = item_of[rid]
                if batch.request_slots is None:  # rows in batch order, filled anew each step
                    slot = item
                    self._owner[slot] = self._mask_owner[slot] = -1
                else:
                    slot = batch.request_slots[item]
                if not 0 <= slot < self.capacity:
                    raise ValueError("request slots must be below capacity")
                if params.penalised:
                    length = batch.context_lens_after[item]
                    self._fill_history(slot, rid, history, length)
                    ints[:3, r] = slot, length, len(history[0])
                    floats[:, r] = (params.repetition_penalty, params.presence_penalty,
                                    params.frequency_penalty)
                if params.allowed_token_ids is not None:
                    self._fill_mask(slot, rid, params.allowed_token_ids)
                    ints[3, r] = slot
                    any_mask = True
                for token, value in params.logit_bias:
                    tokens.append(token)
                    values.append(value)
            offsets[r + 1] = len(tokens)
        # One upload, carved up on the device (8-byte fields first).
        fields = [ints, offsets, floats, np.asarray(tokens, dtype=np.int32),
                  np.asarray(values, dtype=np.float32)]
        packed = torch.from_numpy(np.concatenate([f.reshape(-1).view(np.uint8) for f in fields]))
        data = packed.to(self.device, non_blocking=True)
        parts, at = [], 0
        for f in fields:
            parts.append(data[at:at + f.nbytes].view(
                {"int64": torch.long, "int32": torch.int32,
                 "float32": torch.float32}[f.dtype.name]).view(f.shape))
            at += f.nbytes
        ints_d, offsets_d, floats_d, tokens_d, values_d = parts
        biases = {} if not tokens else dict(bias_tokens=tokens_d, bias_values=values_d,
                                            bias_offsets=offsets_d)
        masks = {} if not any_mask else dict(mask=self.masks, mask_rows=ints_d[3])
        apply_logit_controls(logits, repetition=floats_d[0], presence=floats_d[1],
                             frequency=floats_d[2], history=self.history, slots=ints_d[0],
                             lengths=ints_d[1], prompt_lens=ints_d[2], newest=newest,
                             out=logits, **biases, **masks)
