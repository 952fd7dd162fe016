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
                    history[slot, n - 1] = c["newest"][r] if 0 <= c["newest"][r] < vocab else -1
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1000, 1001])
def test_in_place_and_as_a_slice(device, dtype, vocab):
    """Columns of a wider tensor, changed in place: the rest stays."""
    c = make(3, 9, vocab, dtype=dtype)
    want, slack, _ = formula(c)
    wide = torch.full((9, vocab + 33), 5.0, dtype=dtype, device=device)
    part = wide[:, 16:16 + vocab]
    part.copy_(c["logits"])
    got, _ = call(c, device, logits=part, out=part)
    assert got is part
    check(got, want, slack)
    assert (wide[:, :16] == 5.0).all() and (wide[:, 16 + vocab:] == 5.0).all()


@pytest.mark.gpu
def test_rows_without_controls_are_copied_bit_for_bit(device):
    c = make(4, 6, 9000)
    c["logits"][0, 5] = float("nan")
    c["logits"][1, 8999] = float("inf")
    c["logits"][2] = torch.finfo(BF16).min
    off = dict(c, slots=[-1] * 6, bias=[[]] * 6, mask_rows=[-1] * 6)
    got, history = call(off, device)
    assert torch.equal(got.view(torch.int16).cpu(), c["logits"].view(torch.int16))
    assert torch.equal(history.cpu(), c["history"])
    got, _ = call(dict(off, slots=[99, -5, 8, 1000, -1, 10 ** 12]), device)  # no such slots
    assert torch.equal(got.view(torch.int16).cpu(), c["logits"].view(torch.int16))
    got, _ = call(dict(off, mask_rows=[3, 99, -7, 10 ** 12, 4, -1]), device)  # no such masks
    assert torch.equal(got.view(torch.int16).cpu(), c["logits"].view(torch.int16))


@pytest.mark.gpu
def test_masks_that_leave_nothing_or_one_token(device):
    """Through the sampler too: nothing left answers token 0, as a row of equal
    logits does; one left answers that one at any temperature."""
    from tinyvllm.kernels.sampling import argmax, sample

    rows, vocab = 4, 20011
    c = make(5, rows, vocab, masks=2)
    c["mask"][0] = 0
    c["mask"][1] = 0
    c["mask"][1, 17000 // 32] = 1 << (17000 % 32)
    c.update(slots=[-1] * rows, bias=[[]] * rows, mask_rows=[0, 1, 0, 1])
    want, slack, _ = formula(c)
    got, _ = call(c, device)
    check(got, want, slack)
    assert argmax(got).tolist() == [0, 17000, 0, 17000]
    t = torch.tensor([0.0, 0.0, 1.0, 1.0], device=device)
    zeros = torch.zeros(rows, dtype=torch.long, device=device)
    drawn = sample(got, t, zeros, torch.ones(rows, device=device), zeros, zeros)
    assert drawn.tolist() == [0, 17000, 0, 17000]


@pytest.mark.gpu
def test_infinite_and_nan_logits_keep_to_the_formula(device):
    c = make(6, 3, 512, dtype=F32)
    c["logits"][:, 0] = float("inf")
    c["logits"][:, 1] = -float("inf")
    c["logits"][:, 2] = float("nan")
    c["logits"][:, 3] = torch.finfo(F32).min / 4
    c["history"][:, :] = torch.arange(c["history"].shape[1], dtype=torch.int32) % 8
    c.update(slots=[0, 1, 2], lengths=[50] * 3, prompts=[10] * 3, newest=[3] * 3,
             repetition=[1.5] * 3, presence=[0.5] * 3, frequency=[0.1] * 3,
             bias=[[(0, -3.0), (1, 4.0), (2, 5.0)]] * 3, mask_rows=[-1] * 3)
    want, slack, _ = formula(c)
    got, _ = call(c, device)
    got = got.cpu()
    assert torch.equal(got.isnan(), want.isnan()) and got[:, 2].isnan().all()
    assert (got[:, 0] == float("inf")).all() and (got[:, 1] == -float("inf")).all()
    fine = want.isfinite()
    err = (got.double() - want).abs()[fine]
    assert (err <= (2.0 ** -24 * want.abs() + slack)[fine]).all()
    c["mask"][0] = 0  # a masked NaN or infinity is -inf
    got, _ = call(dict(c, mask_rows=[0] * 3), device)
    assert (got == -float("inf")).all()


@pytest.mark.gpu
def test_ids_outside_the_vocabulary_count_as_none(device):
    c = make(7, 2, 300)
    c.update(slots=[0, 1], lengths=[40, 40], prompts=[5, 5], newest=[-1, 10 ** 10],
             repetition=[2.0, 2.0], bias=[[(299, 1.0)], [(0, 1.0)]], mask_rows=[-1, -1])
    c["history"][0, :20] = 300
    c["history"][1, :20] = -7
    c["history"][1, 20:30] = 2 ** 31 - 1
    keep = c["history"].clone()
    want, slack, _ = formula(c)
    bad = torch.tensor([-3, 300, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=device)
    got, history = call(c, device)
    check(got, want, slack)
    keep[0, 39] = keep[1, 39] = -1  # no token
    assert torch.equal(history.cpu(), keep)
    got, _ = call(dict(c, bias=[[], []]), device, bias_tokens=bad,
                  bias_values=torch.ones(4, device=device),
                  bias_offsets=torch.tensor([-5, 2, 99], device=device))
    check(got, *formula(dict(c, bias=[[], []]))[:2])


@pytest.mark.gpu
@pytest.mark.parametrize("longest,capacity", [(5000, 5001), (70000, 70004), (64, 40)])
def test_long_histories(device, longest, capacity):
    """Lists of many rounds, unaligned ones, and requests longer than the list
    (their tokens past it do not count but the newest, which is not kept)."""
    c = make(8, 5, 12000, longest=longest, capacity=capacity)
    c["lengths"] = [longest, longest - 1, max(1, longest - 2), longest // 2, 1]
    c["prompts"] = [longest // 3] * 5
    want, slack, history = formula(c)
    got, kept = call(c, device)
    if capacity >= longest:
        check(got, want, slack)
        assert torch.equal(kept.cpu(), history)
    else:
        wide = dict(c, history=torch.cat([c["history"], torch.full(
            (len(c["history"]), longest - capacity), -1, dtype=torch.int32)], 1))
        want, slack, history = formula(wide)
        check(got, want, slack)
        assert torch.equal(kept.cpu(), history[:, :capacity])


@pytest.mark.gpu
def test_histories_without_a_newest_token(device):
    c = make(9, 12, 700)
    want, slack, history = formula(c, use_newest=False)
    got, kept = call(c, device, use_newest=False)
    check(got, want, slack)
    assert torch.equal(kept.cpu(), c["history"]) and torch.equal(history, c["history"])


@pytest.mark.gpu
def test_every_control_alone(device):
    none = dict(repetition=None, presence=None, frequency=None, history=None, slots=None,
                lengths=None, prompt_lens=None, newest=None, bias_tokens=None, bias_values=None,
                bias_offsets=None, mask=None, mask_rows=None)
    c = make(10, 8, 2000)
    off = dict(c, slots=[-1] * 8, bias=[[]] * 8, mask_rows=[-1] * 8)
    for keep, case in (
            ((), off), (("bias_tokens", "bias_values", "bias_offsets"), dict(off, bias=c["bias"])),
            (("mask", "mask_rows"), dict(off, mask_rows=c["mask_rows"])),
            (("repetition", "history", "slots", "lengths", "prompt_lens", "newest"),
             dict(off, slots=c["slots"], presence=[0.0] * 8, frequency=[0.0] * 8)),
            (("presence", "history", "slots", "lengths", "prompt_lens", "newest"),
             dict(off, slots=c["slots"], repetition=[1.0] * 8, frequency=[0.0] * 8)),
            (("frequency", "history", "slots", "lengths", "prompt_lens", "newest"),
             dict(off, slots=c["slots"], repetition=[1.0] * 8, presence=[0.0] * 8))):
        over = {k: v for k, v in none.items() if k not in keep}
        got, _ = call(case, device, **over)
        check(got, *formula(case)[:2])


@pytest.mark.gpu
def test_captured_call_keeps_its_history(device):
    """A decode loop's three calls, captured and replayed as the host would:
    lengths and newest tokens change, the history grows on the device."""
    from tinyvllm.kernels.logits import apply_logit_controls

    rows, vocab = 3, 9001
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(rows, vocab, generator=g).to(device)
    history = torch.zeros(rows, 64, dtype=torch.int32, device=device)
    prompts = [4, 1, 9]
    ids = [torch.randint(0, 50, (n,), generator=g).tolist() for n in prompts]
    for r, x in enumerate(ids):
        history[r, :len(x) - 1] = torch.tensor(x[:-1], dtype=torch.int32, device=device)
    lengths = torch.tensor(prompts, device=device)
    newest = torch.tensor([x[-1] for x in ids], device=device)
    args = dict(repetition=torch.full((rows,), 1.2, device=device),
                presence=torch.full((rows,), 0.3, device=device),
                frequency=torch.full((rows,), 0.2, device=device), history=history,
                slots=torch.arange(rows, device=device), lengths=lengths,
                prompt_lens=torch.tensor(prompts, device=device), newest=newest)
    out = torch.empty_like(logits)
    apply_logit_controls(logits, out=out, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply_logit_controls(logits, out=out, **args)
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        c = dict(logits=logits.cpu(), history=torch.zeros(rows, 64, dtype=torch.int32),
                 slots=[0, 1, 2], lengths=[len(x) for x in ids], newest=[x[-1] for x in ids],
                 repetition=[1.2] * rows, presence=[0.3] * rows, frequency=[0.2] * rows,
                 bias=[[]] * rows, mask_rows=[-1] * rows, mask=torch.zeros(0, 1),
                 prompts=prompts)
        for r, x in enumerate(ids):
            c["history"][r, :len(x)] = torch.tensor(x, dtype=torch.int32)
        check(out, *formula(c)[:2])
        logits.add_(0.25)
        step = torch.randint(0, 50, (rows,), generator=g)
        for x, t in zip(ids, step.tolist()):
            x.append(t)
        newest.copy_(step)
        lengths.add_(1)


@pytest.mark.gpu
def test_wrapper_refusals(device):
    from tinyvllm.kernels.logits import apply_logit_controls

    c = make(11, 3, 100)
    call(c, device)
    x = c["logits"].to(device)
    longs = torch.zeros(3, dtype=torch.long, device=device)
    floats = torch.ones(3, device=device)
    history = torch.zeros(4, 8, dtype=torch.int32, device=device)
    mask = torch.zeros(2, 4, dtype=torch.int32, device=device)
    for args, message in (
            (dict(logits=x.double()), "float16, bfloat16 or float32"),
            (dict(logits=x[0]), "rows, vocab"), (dict(logits=x.T), "unit last stride"),
            (dict(logits=x.cpu()), "GPU"), (dict(repetition=floats), "history"),
            (dict(newest=longs), "history"), (dict(history=history), "slots"),
            (dict(history=history.long(), slots=longs, lengths=longs, prompt_lens=longs), "int32"),
            (dict(history=history, slots=longs.int(), lengths=longs, prompt_lens=longs), "slots"),
            (dict(history=history, slots=longs, lengths=longs[:2], prompt_lens=longs), "lengths"),
            (dict(history=history.cpu(), slots=longs, lengths=longs, prompt_lens=longs), "one GPU"),
            (dict(history=history, slots=longs, lengths=longs, prompt_lens=longs,
                  presence=floats.double()), "presence"),
            (dict(bias_tokens=longs.int()), "biases"),
            (dict(bias_tokens=longs.int(), bias_values=floats, bias_offsets=longs), "of 4"),
            (dict(bias_tokens=longs.int(), bias_values=floats[:2],
                  bias_offsets=torch.zeros(4, dtype=torch.long, device=device)), "align"),
            (dict(mask=mask), "mask_rows"), (dict(mask=mask[:, :3], mask_rows=longs), "bit"),
            (dict(mask=mask.long(), mask_rows=longs), "int32"),
            (dict(out=x.half()), "out"), (dict(out=x[:2]), "out"),
            (dict(out=torch.empty(3, 100)), "one GPU")):
        with pytest.raises(RuntimeError, match=message):
            apply_logit_controls(**{**dict(logits=x), **args})
    assert apply_logit_controls(x[:0]).shape == (0, 100)


@pytest.mark.gpu
def test_launches_go_to_the_tensors_device(device, monkeypatch):
    """With another device current, the logits' own is made current for the call."""
    from tinyvllm.kernels import _extension

    c = make(12, 3, 100)
    entered = []

    class Recorded(torch.cuda.device):
        def __init__(self, where):
            entered.append(where)
            super().__init__(where)

    monkeypatch.setattr(_extension, "_current_device", lambda: 99)
    monkeypatch.setattr(torch.cuda, "device", Recorded)
    out, _ = call(c, device)
    assert out.device in entered
    check(out, *formula(c)[:2])


@pytest.mark.gpu
def test_outputs_beside_the_logits_in_one_buffer_or_over_them(device):
    """Columns of one buffer are apart; rows that overlap others are refused."""
    from tinyvllm.kernels.logits import apply_logit_controls

    c = make(13, 4, 100)
    both = torch.zeros(4, 240, device=device)
    logits, out = both[:, :100], both[:, 120:220]
    logits.copy_(c["logits"])
    call(c, device, logits=logits, out=out)
    check(out, *formula(c)[:2])
    flat = torch.zeros(1000, device=device)
    for first, second in ((flat[:400].view(4, 100), flat[100:500].view(4, 100)),
                          (flat[:400].view(4, 100), flat[60:460].view(4, 100)),
                          (both[:, :100], both[:, 60:160]), (both[:, 140:240], both[:, 60:160])):
        with pytest.raises(RuntimeError, match="overlap"):
            apply_logit_controls(first, out=second)
    apply_logit_controls(flat[:400].view(4, 100), out=flat[400:800].view(4, 100))
