"""Operator cases: decode attention over a shared prompt, and logit controls.

Both serve a decode batch whose requests share one long prompt and are held
apart, or held to a form, by their own controls:

* ``prefix``: one token per request attends its whole context, of which the
  first tokens lie in pages that the requests of a group share;
* ``logits``: repetition, presence and frequency penalties from each request's
  tokens, additive biases and allowed-token masks, in front of the sampler.

``listed()`` holds the sizes of the benchmark and test configurations, ``draw``
spreads further cases over the same ranges. Where ``own`` is false ``run``
computes the operators from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path.cwd() / "tiny-vllm_amd"))

own = False

PAGE = 16
VOCAB = 151936
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8_SCALES = (0.0625, 0.03125)


# ---------------------------------------------------------------- the cases --

def listed():
    return [
        # Two answers to one chat request, just begun: the smallest call.
        dict(name="prefix_2x512", kind="prefix", rows=2, groups=1, alone=0, prefix=512, low=1,
             high=32, heads=16, kv_heads=8, dim=128, dtype="bf16", cache="same",
             layout="head_major"),
        # The headline batch behind one system prompt of its usual length.
        dict(name="prefix_64x2048", kind="prefix", rows=64, groups=1, alone=0, prefix=2048, low=64,
             high=512, heads=32, kv_heads=8, dim=128, dtype="bf16", cache="same",
             layout="token_major"),
        # Several applications on one server: six prompts of their own lengths,
        # and a tenth of the requests with none.
        dict(name="prefix_49_in_6", kind="prefix", rows=49, groups=6, alone=5, prefix=4096, low=1,
             high=1024, heads=32, kv_heads=8, dim=128, dtype="bf16", cache="same",
             layout="token_major"),
        # Questions about one long document over the FP8 cache, 32B heads.
        dict(name="prefix_16x32k_fp8", kind="prefix", rows=16, groups=1, alone=0, prefix=32768,
             low=16, high=256, heads=64, kv_heads=8, dim=128, dtype="bf16", cache="fp8",
             layout="head_major"),
        # Models with 64-wide heads in fp16, an odd batch.
        dict(name="prefix_33x3k_dim64", kind="prefix", rows=33, groups=2, alone=1, prefix=3008,
             low=1, high=777, heads=32, kv_heads=8, dim=64, dtype="fp16", cache="same",
             layout="token_major"),
        # 256-wide heads, two KV heads.
        dict(name="prefix_24x1k_dim256", kind="prefix", rows=24, groups=1, alone=0, prefix=1024,
             low=32, high=300, heads=16, kv_heads=2, dim=256, dtype="bf16", cache="same",
             layout="token_major"),
        # Offline extraction: 256 inputs behind one long instruction.
        dict(name="prefix_256x32k", kind="prefix", rows=256, groups=1, alone=0, prefix=32768,
             low=1, high=1024, heads=32, kv_heads=8, dim=128, dtype="bf16", cache="same",
             layout="token_major"),
        # One chat request with a repetition penalty.
        dict(name="logits_1", kind="logits", rows=1, vocab=VOCAB, low=300, high=300,
             penalised=1.0, biased=0.0, bias=0, masked=0.0, allowed=1.0, dtype="bf16", out="bf16"),
        # A served batch: most requests penalised, some with biases, some held to a form.
        dict(name="logits_64", kind="logits", rows=64, vocab=VOCAB, low=64, high=4096,
             penalised=0.75, biased=0.25, bias=16, masked=0.25, allowed=0.02, dtype="bf16",
             out="bf16"),
        # Constrained answers only: every request behind a mask, few tokens allowed.
        dict(name="logits_33_masks", kind="logits", rows=33, vocab=49999, low=1, high=1024,
             penalised=0.0, biased=0.0, bias=0, masked=1.0, allowed=0.001, dtype="fp16",
             out="fp32"),
        # Offline batch with long histories, fp32 logits, all controls.
        dict(name="logits_256x32k", kind="logits", rows=256, vocab=VOCAB, low=2048, high=32768,
             penalised=1.0, biased=0.5, bias=300, masked=0.5, allowed=0.5, dtype="fp32",
             out="fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    cap = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("prefix", "logits")}
    while True:
        case = _draw(rng)
        if _cost(case) <= cap[case["kind"]]:
            return case


def _draw(rng):
    if rng.random() < 0.6:
        rows = _log(rng, 2, 256)
        groups = min(rng.choice([1, 1, _log(rng, 2, 16)]), max(1, rows // 2))
        high = _log(rng, 2, 2048)
        dim = rng.choice([128, 128, 128, 64, 256, 32, 96])
        kv_heads = rng.choice([8, 8, 2, 4])
        return dict(kind="prefix", rows=rows, groups=groups,
                    alone=rng.choice([0, rng.randint(0, rows - 2 * groups)]),
                    prefix=PAGE * _log(rng, 1, 2048), low=rng.choice([1, max(1, high // 2)]),
                    high=high, heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 16]),
                    kv_heads=kv_heads, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    cache=rng.choice(["same", "same", "fp8"]),
                    layout=rng.choice(["token_major", "head_major"]))
    high = _log(rng, 2, 32768)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return dict(kind="logits", rows=_log(rng, 1, 256), vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]),
                low=rng.choice([1, max(1, high // 2), high]), high=high,
                penalised=rng.choice([0.0, 0.5, 1.0]), biased=rng.choice([0.0, 0.3, 1.0]),
                bias=_log(rng, 1, 300), masked=rng.choice([0.0, 0.3, 1.0]),
                allowed=rng.choice([0.001, 0.5, 0.99]), dtype=dtype,
                out=rng.choice([dtype, "fp32"]))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# --------------------------------------------------------- inputs from a seed --

def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed) * 7919 + 31)


def _shape(case):
    """The rows' groups (-1: none), the groups' shared tokens and the contexts:
    the case's own, the same ones for every seed."""
    g = _gen(case["rows"] * 100003 + case["prefix"], "cpu")
    rows, groups, alone = case["rows"], case["groups"], case["alone"]
    member = torch.randint(0, groups, (rows - alone,), generator=g)
    member[:2 * groups] = torch.arange(groups).repeat(2)  # two rows at least in each
    member = torch.cat([member, torch.full((alone,), -1)])[torch.randperm(rows, generator=g)]
    pages = case["prefix"] // PAGE
    shared = torch.randint(max(1, pages // 8), pages + 1, (groups,), generator=g) * PAGE
    shared[0] = pages * PAGE
    tail = torch.randint(case["low"], case["high"] + 1, (rows,), generator=g)
    tail[int(torch.randint(0, rows, (1,), generator=g))] = case["high"]
    lengths = tail + torch.where(member >= 0, shared[member.clamp(min=0)], 0)
    return member, shared, lengths


def _prefix_inputs(case, seed):
    member, shared, lengths = _shape(case)
    pages = torch.div(lengths + PAGE - 1, PAGE, rounding_mode="floor")
    common = torch.where(member >= 0, shared[member.clamp(min=0)] // PAGE, 0)
    pool = int((shared // PAGE).sum() + (pages - common).sum()) + 7
    order = torch.randperm(pool, generator=_gen(seed + 1, "cpu"))
    heads, at = [], 0
    for n in (shared // PAGE).tolist():
        heads.append(order[at:at + n])
        at += n
    tables = []
    for g, n, c in zip(member.tolist(), pages.tolist(), common.tolist()):
        tables.append(torch.cat([heads[g][:c] if g >= 0 else order[:0], order[at:at + n - c]]))
        at += n - c
    dt = DTYPES[case["dtype"]]
    g = _gen(seed)
    q = (torch.randn((case["rows"], case["heads"], case["dim"]), generator=g, device="cuda")
         * 1.5).to(dt)
    fp8 = case["cache"] == "fp8"
    scales = FP8_SCALES if fp8 else (1.0, 1.0)
    kv = []
    for scale in scales:
        x = torch.randn((pool * PAGE, case["kv_heads"], case["dim"]), generator=g, device="cuda",
                        dtype=torch.float32 if dt == torch.float16 or fp8 else dt)
        kv.append((x / scale).to(torch.float8_e4m3fn) if fp8 else x.to(dt))
    return member, shared, lengths, pool, tables, q, kv, scales


def _logits_inputs(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    shape = _gen(rows * 100003 + case["high"], "cpu")
    lengths = torch.randint(case["low"], case["high"] + 1, (rows,), generator=shape)
    lengths[int(torch.randint(0, rows, (1,), generator=shape))] = case["high"]
    prompts = (lengths * torch.rand(rows, generator=shape)).long()

    def some(share):  # about that share of the rows, all of them at 1
        return torch.rand(rows, generator=shape) < share

    penalised, biased, masked = (some(case[n]) for n in ("penalised", "biased", "masked"))
    g, c = _gen(seed), _gen(seed + 2, "cpu")
    dt = DTYPES[case["dtype"]]
    logits = (torch.randn((rows, vocab), generator=g, device="cuda") * 4).to(dt)
    # Words repeat as they do in text: low ids far more often than high ones.
    capacity = case["high"] + 16
    history = (torch.rand((rows, capacity), generator=g, device="cuda") ** 4 * vocab).to(torch.int32)
    newest = (torch.rand(rows, generator=g, device="cuda") ** 4 * vocab).to(torch.int64)
    slots = torch.where(penalised, torch.randperm(rows, generator=c), -1)
    counts = torch.where(biased, case["bias"], 0)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    # Distinct tokens in a row's list, as a mapping from tokens to biases has.
    step = max(1, vocab // max(1, case["bias"]))
    rank = torch.cat([torch.arange(n) for n in counts.tolist()] or [counts])
    tokens = (rank * step + torch.randint(0, step, rank.shape, generator=c)).to(torch.int32)
    values = torch.randn(rank.shape, generator=c) * 5
    where = torch.where(masked, masked.long().cumsum(0) - 1, -1)
    bits = torch.rand((int(masked.sum()), -(-vocab // 32), 32), generator=g,
                      device="cuda") < case["allowed"]
    weights = 2 ** torch.arange(32, device="cuda", dtype=torch.int64)
    words = (bits.long() * weights).sum(-1).to(torch.int32)
    return dict(logits=logits, history=history, newest=newest, slots=slots.cuda(),
                lengths=lengths.cuda(), prompts=prompts.cuda(),
                repetition=(1 + 0.5 * torch.rand(rows, generator=c)).cuda(),
                presence=torch.rand(rows, generator=c).cuda(),
                frequency=(0.5 * torch.rand(rows, generator=c)).cuda(),
                bias_tokens=tokens.cuda(), bias_values=values.cuda(),
                bias_offsets=offsets.cuda(), mask=words, mask_rows=where.cuda(),
                out=DTYPES[case["out"]])


def prepare(case, seed):
    if case["kind"] == "logits":
        return dict(kind="logits", **_logits_inputs(case, seed))
    member, shared, lengths, pool, tables, q, (k, v), (ks, vs) = _prefix_inputs(case, seed)
    scale = case["dim"] ** -0.5
    if case["layout"] == "head_major":  # storage [heads, slots, dim] behind the same view
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    state = dict(kind="prefix", q=q, k=k, v=v, ks=ks, vs=vs, scale=scale)
    if own:
        from tinyvllm.kernels.shared_prefix import SharedPrefixPlan
        from tinyvllm.paged_kv import PagedKVCache
        from tinyvllm.runtime.contracts import SingleQueryMetadata

        cache = PagedKVCache(num_layers=1, num_blocks=pool, block_size=PAGE,
                             num_kv_heads=case["kv_heads"], head_dim=case["dim"], device="cuda",
                             dtype=k.dtype, k_scale=ks, v_scale=vs, layout=case["layout"])
        cache.key[0].copy_(k)
        cache.value[0].copy_(v)
        plan = SharedPrefixPlan(num_heads=case["heads"], num_kv_heads=case["kv_heads"],
                                head_dim=case["dim"], block_size=PAGE, max_rows=case["rows"],
                                device="cuda")
        plan.update(lengths.tolist(), member.tolist(), shared.tolist())
        offsets = torch.tensor([0] + [len(t) for t in tables]).cumsum(0)
        metadata = SingleQueryMetadata(
            query_rows=torch.arange(case["rows"]).cuda(), block_table_ids=torch.cat(tables).cuda(),
            block_table_offsets=offsets.cuda(), context_lens=lengths.cuda(),
            max_context_len=int(lengths.max()))
        return dict(kind="prefix", q=q, cache=cache, plan=plan, metadata=metadata, scale=scale,
                    out=torch.empty_like(q))
    # The plain form's plan: each group's slots and rows, each row's own slots,
    # padded to the longest, with what is padding marked.
    groups, rows = case["groups"], case["rows"]
    first = [int((member == g).nonzero()[0]) for g in range(groups)]
    p = torch.arange(int(shared.max()))
    prefix_slots = torch.stack([tables[r][(p // PAGE).clamp(max=len(tables[r]) - 1)] * PAGE
                                + p % PAGE for r in first])
    begin = torch.where(member >= 0, shared[member.clamp(min=0)], 0)
    t = torch.arange(int((lengths - begin).max()))
    own_slots = torch.stack([tables[r][((begin[r] + t) // PAGE).clamp(max=len(tables[r]) - 1)] * PAGE
                             + (begin[r] + t) % PAGE for r in range(rows)])
    lists = [(member == g).nonzero()[:, 0] for g in range(groups)]
    most = max(len(x) for x in lists)
    place = torch.zeros(rows, dtype=torch.long)
    for x in lists:
        place[x] = torch.arange(len(x))
    state.update(
        prefix_slots=prefix_slots.cuda(), prefix_out=(p >= shared[:, None]).cuda(),
        own_slots=own_slots.cuda(), own_out=(t >= (lengths - begin)[:, None]).cuda(),
        members=torch.stack([torch.cat([x, x[:1].repeat(most - len(x))]) for x in lists]).cuda(),
        member=member.clamp(min=0).cuda(), grouped=(member >= 0).cuda(), place=place.cuda())
    return state


# ---------------------------------------------------------------------- run --

@torch.inference_mode()
def run(state):
    if own:
        return _own_prefix(state) if state["kind"] == "prefix" else _own_logits(state)
    return _plain_prefix(state) if state["kind"] == "prefix" else _plain_logits(state)


def _own_prefix(s):
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    paged_decode_shared_prefix(s["q"], s["cache"], 0, s["metadata"], s["plan"], s["out"],
                               scale=s["scale"])
    return s["out"]


def _own_logits(s):
    from tinyvllm.kernels.logits import apply_logit_controls

    out = torch.empty(s["logits"].shape, dtype=s["out"], device=s["logits"].device)
    apply_logit_controls(
        s["logits"], repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
        history=s["history"], slots=s["slots"], lengths=s["lengths"], prompt_lens=s["prompts"],
        newest=s["newest"], bias_tokens=s["bias_tokens"], bias_values=s["bias_values"],
        bias_offsets=s["bias_offsets"], mask=s["mask"], mask_rows=s["mask_rows"], out=out)
    return dict(logits=out, history=s["history"])


def _part(q, k, v, out, scale):
    """Running maximum, sum and unnormalised output of one part of the keys:
    q [n, Hkv, queries, D], k and v [n, keys, Hkv, D], out [n, keys] (not seen)."""
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * scale
    s = s.masked_fill(out[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0, m))
    return m, e.sum(-1, keepdim=True), torch.matmul(e, v.permute(0, 2, 1, 3))


def _plain_prefix(s):
    q = s["q"].float()
    rows, heads, dim = q.shape
    kv_heads = s["k"].shape[1]
    group = heads // kv_heads
    q = q.view(rows, kv_heads, group, dim)
    scale = s["scale"] * s["ks"]
    # The shared parts: every query of a group in one product.
    groups, most = s["members"].shape
    qg = q[s["members"]].transpose(1, 2).reshape(groups, kv_heads, most * group, dim)
    parts = _part(qg, s["k"][s["prefix_slots"]].float(), s["v"][s["prefix_slots"]].float(),
                  s["prefix_out"], scale)
    mp, lp, ap = (x.view(groups, kv_heads, most, group, -1).transpose(1, 2)[s["member"], s["place"]]
                  for x in parts)
    none = ~s["grouped"][:, None, None, None]
    mp, lp, ap = mp.masked_fill(none, -math.inf), lp.masked_fill(none, 0), ap.masked_fill(none, 0)
    # The rows' own parts, and both together.
    mo, lo, ao = _part(q, s["k"][s["own_slots"]].float(), s["v"][s["own_slots"]].float(),
                       s["own_out"], scale)
    m = torch.maximum(mp, mo)
    wp, wo = torch.exp(mp - m), torch.exp(mo - m)
    out = (ap * wp + ao * wo) / (lp * wp + lo * wo) * s["vs"]
    return out.view(rows, heads, dim).to(s["q"].dtype)


def _plain_logits(s):
    rows, vocab = s["logits"].shape
    has, slot = s["slots"] >= 0, s["slots"].clamp(min=0)
    # The newest token joins the history, then every token is counted.
    last = s["lengths"] - 1
    history = s["history"]
    history[slot[has], last[has]] = s["newest"][has].to(torch.int32)
    t = torch.arange(history.shape[1], device=history.device)
    seen = (t < s["lengths"][:, None]) & has[:, None]
    tokens = history[slot].long()
    total = torch.zeros((rows, vocab), device=history.device)
    total.scatter_add_(1, tokens, seen.float())
    answer = torch.zeros((rows, vocab), device=history.device)
    answer.scatter_add_(1, tokens, (seen & (t >= s["prompts"][:, None])).float())
    x = s["logits"].float()
    rho = s["repetition"][:, None]
    x = torch.where(total > 0, torch.where(x > 0, x / rho, x * rho), x)
    x = x - s["frequency"][:, None] * answer - s["presence"][:, None] * (answer > 0)
    counts = s["bias_offsets"].diff()
    row = torch.repeat_interleave(torch.arange(rows, device=x.device), counts,
                                  output_size=s["bias_tokens"].numel())
    bias = torch.zeros_like(x)
    bias[row, s["bias_tokens"].long()] = s["bias_values"]
    x = x + bias
    if s["mask"].numel():
        i = torch.arange(vocab, device=x.device)
        words = s["mask"][s["mask_rows"].clamp(min=0)][:, i // 32]
        allowed = ((words >> (i % 32)) & 1).bool() | (s["mask_rows"] < 0)[:, None]
        x = x.masked_fill(~allowed, -math.inf)
    return dict(logits=x.to(s["out"]), history=history)


# --------------------------------------------------------------------- work --

def work(case):
    if case["kind"] == "prefix":
        member, shared, lengths = _shape(case)
        begin = torch.where(member >= 0, shared[member.clamp(min=0)], 0)
        keys = int(shared.sum()) + int((lengths - begin).sum())
        element = 1 if case["cache"] == "fp8" else 2
        return dict(bytes=2 * keys * case["kv_heads"] * case["dim"] * element
                    + 4 * case["rows"] * case["heads"] * case["dim"],
                    flops=4 * int(lengths.sum()) * case["heads"] * case["dim"])
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    rows, vocab = case["rows"], case["vocab"]
    tokens = rows * case["penalised"] * (case["low"] + case["high"]) / 2
    return dict(bytes=rows * vocab * (size[case["dtype"]] + size[case["out"]])
                + 4 * tokens + rows * case["masked"] * vocab / 8
                + 8 * rows * case["biased"] * case["bias"],
                flops=6 * rows * vocab + 2 * tokens)


# -------------------------------------------------------------------- exact --

@torch.inference_mode()
def exact(case, seed):
    if case["kind"] == "prefix":
        member, shared, lengths, _, tables, q, (k, v), (ks, vs) = _prefix_inputs(case, seed)
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for r, n in enumerate(lengths.tolist()):
            t = torch.arange(n)
            slots = (tables[r][t // PAGE] * PAGE + t % PAGE).cuda()
            keys = (k[slots].float() if case["cache"] == "fp8" else k[slots]).double() * ks
            values = (v[slots].float() if case["cache"] == "fp8" else v[slots]).double() * vs
            x = q[r].double().view(case["kv_heads"], group, -1)
            weights = torch.softmax(
                torch.bmm(x, keys.permute(1, 2, 0).contiguous()) * case["dim"] ** -0.5, -1)
            out[r] = torch.bmm(weights, values.transpose(0, 1).contiguous()).flatten(0, 1)
        return out
    d = _logits_inputs(case, seed)
    x = d["logits"].double()
    history = d["history"].clone()
    vocab = case["vocab"]
    for r, (slot, n, prompt) in enumerate(zip(d["slots"].tolist(), d["lengths"].tolist(),
                                              d["prompts"].tolist())):
        if slot >= 0:
            history[slot, n - 1] = d["newest"][r]
            ids = history[slot, :n].long()
            answer = torch.bincount(ids[prompt:], minlength=vocab).double()
            there = torch.bincount(ids, minlength=vocab) > 0
            rho = d["repetition"][r].double()
            x[r] = torch.where(there, torch.where(x[r] > 0, x[r] / rho, x[r] * rho), x[r])
            x[r] -= d["frequency"][r].double() * answer
            x[r] -= d["presence"][r].double() * (answer > 0)
        a, b = d["bias_offsets"][r:r + 2].tolist()
        x[r, d["bias_tokens"][a:b].long()] += d["bias_values"][a:b].double()
        row = int(d["mask_rows"][r])
        if row >= 0:
            bits = torch.stack([(d["mask"][row] >> j) & 1 for j in range(32)], 1).flatten()
            x[r, bits[:vocab] == 0] = -math.inf
    return dict(logits=x, history=history)
