"""Penalties, biases and masks on logits against the formula in 64 bits."""
import math
import random

import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS32 = 2.0 ** -24


def make(seed, rows, vocab, *, dtype=BF16, longest=200, slots=None, capacity=None, masks=3):
    """Rows with every mix of controls; CPU tensors and lists."""
    r = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    count = slots or rows + 2
    capacity = capacity or longest + 5
    pool = r.sample(range(count), min(rows, count))
    c = dict(
        logits=(torch.randn(rows, vocab, generator=g) * 5).to(dtype),
        history=torch.randint(0, vocab, (count, capacity), generator=g, dtype=torch.int32),
        slots=[pool[i] if r.random() < 0.8 else -1 for i in range(rows)],
        lengths=[r.choice([0, 1, 2, r.randint(1, longest), longest]) for _ in range(rows)],
        newest=[r.randrange(vocab) for _ in range(rows)],
        repetition=[r.choice([1.0, 1.3, 0.7]) for _ in range(rows)],
        presence=[r.choice([0.0, 0.6, -0.4]) for _ in range(rows)],
        frequency=[r.choice([0.0, 0.25, -0.1]) for _ in range(rows)],
        bias=[[] if r.random() < 0.4 else
              [(r.randrange(vocab), r.uniform(-9, 9)) for _ in range(r.choice([1, 2, 40]))]
              for _ in range(rows)],
        mask=torch.randint(-2 ** 31, 2 ** 31, (masks, -(-vocab // 32)), generator=g).int(),
        mask_rows=[r.randint(-1, masks - 1) for _ in range(rows)])
    c["prompts"] = [r.choice([0, n // 2, n]) for n in c["lengths"]]
    # Repeats: words of a text come again.
    c["history"][:, ::3] = c["history"][:, :1] % max(1, vocab // 7)
    return c


def formula(c, use_newest=True):
    """(result, error allowed in 32 bits, history after the call) in 64 bits."""
    x = c["logits"].double()
    off = torch.zeros_like(x)
    rows, vocab = x.shape
    history = c["history"].clone()
    for r in range(rows):
        slot, n = c["slots"][r], c["lengths"][r]
        if 0 <= slot < history.shape[0] and n > 0:
            ids = history[slot, :min(n, history.shape[1])].tolist()
            if use_newest:
                ids = ids[:n - 1] + [c["newest"][r]]
                if n <= history.shape[1]:
                    history[slot, n - 1] = c["newest"][r]
            rho, pres, freq = (torch.tensor(c[k][r], dtype=F32).double()
                               for k in ("repetition", "presence", "frequency"))
            times, seen = {}, set(ids)
            for p, i in enumerate(ids):
                if p >= c["prompts"][r]:
                    times[i] = times.get(i, 0) + 1
            for i in seen:
                if 0 <= i < vocab:
                    k = times.get(i, 0)
                    x[r, i] = x[r, i] / rho if x[r, i] > 0 else x[r, i] * rho
                    off[r, i] += abs(x[r, i]) + 2 * abs(freq) * k + abs(pres)
                    x[r, i] -= freq * k + (pres if k else 0.0)
        last = dict(c["bias"][r])  # of a token listed twice the last entry
        for i, b in last.items():
            if 0 <= i < vocab:
                x[r, i] += float(torch.tensor(b, dtype=F32))
                off[r, i] += abs(b) + abs(x[r, i])
        m = c["mask_rows"][r]
        if 0 <= m < c["mask"].shape[0]:
            bits = torch.stack([(c["mask"][m].long() >> j) & 1 for j in range(32)], 1).flatten()
            x[r, bits[:vocab] == 0] = -math.inf
    # Every operation is half a step off its own result at most; four of them.
    return x, 4 * EPS32 * off, history


def call(c, device, *, out=None, use_newest=True, logits=None, **over):
    from tinyvllm.kernels.logits import apply_logit_controls

    def t(values, dtype):
        return torch.tensor(values, dtype=dtype, device=device)

    flat = [e for b in c["bias"] for e in b]
    offsets = [0]
    for b in c["bias"]:
        offsets.append(offsets[-1] + len(b))
    history = c["history"].to(device)
    args = dict(
        repetition=t(c["repetition"], F32), presence=t(c["presence"], F32),
        frequency=t(c["frequency"], F32), history=history, slots=t(c["slots"], torch.long),
        lengths=t(c["lengths"], torch.long), prompt_lens=t(c["prompts"], torch.long),
        newest=t(c["newest"], torch.long) if use_newest else None,
        bias_tokens=t([i for i, _ in flat], torch.int32),
        bias_values=t([v for _, v in flat], F32), bias_offsets=t(offsets, torch.long),
        mask=c["mask"].to(device), mask_rows=t(c["mask_rows"], torch.long), out=out)
    args.update(over)
    got = apply_logit_controls(c["logits"].to(device) if logits is None else logits, **args)
    torch.cuda.synchronize()
    return got, history


def check(got, want, slack):
    got = got.cpu()
    assert torch.equal(got.isinf(), want.to(got.dtype).isinf())
    fine = want.isfinite()
    err = (got.double() - want).abs()[fine]
    limit = (torch.finfo(got.dtype).eps / 2 * want.abs() + slack * (1 + torch.finfo(got.dtype).eps)
             + torch.finfo(got.dtype).tiny)[fine]
    assert (err <= limit).all(), f"{float((err / limit).max()):.2f} times the bound"


TYPES = [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)]


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (2, 8191), (5, 8192), (4, 8200),
                                        (3, 16391), (40, 1000)])
def test_controls(device, types, rows, vocab):
    dtype, out_dtype = types
    c = make(rows * vocab, rows, vocab, dtype=dtype)
    want, slack, history = formula(c)
    out = torch.full((rows, vocab), float("nan"), dtype=out_dtype, device=device)
    got, kept = call(c, device, out=out)
    assert got is out
    check(got, want, slack)
    assert torch.equal(kept.cpu(), history)
