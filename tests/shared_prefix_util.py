"""Batches whose rows share prefixes, and their attention in 64 bits."""
from __future__ import annotations

import random

import torch


def make_batch(*, seed, heads, kv_heads, dim, dtype, prefixes, rows, block_size=16, fp8=False,
               layout="token_major", spare=3, std=1.0):
    """``prefixes[g]``: group g's shared tokens; ``rows``: (group or -1, own
    tokens) each; a group row has ``prefixes[g]`` tokens more. CPU tensors and
    lists, blocks drawn from a shuffled pool with ``spare`` blocks left over."""
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    lengths = [(prefixes[x] if x >= 0 else 0) + n for x, n in rows]
    shared = [p // block_size for p in prefixes]
    pages = [-(-n // block_size) for n in lengths]
    pool = sum(shared) + sum(p - (shared[x] if x >= 0 else 0)
                             for p, (x, _) in zip(pages, rows)) + spare
    order = list(range(pool))
    r.shuffle(order)
    heads_of = [[order.pop() for _ in range(n)] for n in shared]
    tables = [(heads_of[x] if x >= 0 else []) for x, _ in rows]
    tables = [t + [order.pop() for _ in range(p - len(t))] for t, p in zip(tables, pages)]
    q = (torch.randn(len(rows), heads, dim, generator=g) * std).to(dtype)
    scales = (0.0625, 0.03125) if fp8 else (1.0, 1.0)
    kv = []
    for scale in scales:
        x = torch.randn(pool * block_size, kv_heads, dim, generator=g)
        kv.append((x / scale).to(torch.float8_e4m3fn) if fp8 else x.to(dtype))
    return dict(q=q, k=kv[0], v=kv[1], scales=scales, lengths=lengths, pool=pool,
                groups=[x for x, _ in rows], prefixes=list(prefixes), tables=tables,
                block_size=block_size, layout=layout, scale=dim ** -0.5, fp8=fp8)


def attend64(b):
    """(outputs, weighted sums of |v|, largest sum of |q k|) in 64 bits."""
    q = b["q"].double()
    rows, heads, dim = q.shape
    k, v = (b[n].float().double() * s for n, s in zip("kv", b["scales"]))
    group = heads // k.shape[1]
    out, mass, qk = torch.zeros_like(q), torch.zeros_like(q), 0.0
    bs = b["block_size"]
    for i, (table, n) in enumerate(zip(b["tables"], b["lengths"])):
        if n == 0:
            continue
        slots = torch.tensor([table[t // bs] * bs + t % bs for t in range(n)])
        for h in range(heads):
            kk, vv = k[slots, h // group], v[slots, h // group]
            w = torch.softmax(kk @ q[i, h] * b["scale"], 0)
            out[i, h], mass[i, h] = w @ vv, w @ vv.abs()
            qk = max(qk, float((kk.abs() @ q[i, h].abs()).max()) * b["scale"])
    return out, mass, qk


def allowed(b, out, mass, qk, dtype):
    """Largest error of a right evaluation, element by element: the output's
    rounding (half a step); each weight within a relative w, so that the
    quotient of two sums of weights is within 2 w of sum p|v| - w being half a
    step of fp16 (the least precise form weights take), the fp32 error of a
    score of ``dim`` products (2^-24 each way of the sum of their magnitudes,
    for every addition) in the exponent, and fp32 sums of n terms; weights below
    2^-32 of the largest are lost: n of them, at the values' magnitude."""
    dim, n = out.shape[-1], max(b["lengths"] + [1])
    w = 2.0 ** -11 + (dim + 4) * 2.0 ** -24 * qk + n * 2.0 ** -24
    top = float(b["v"].float().abs().max()) * b["scales"][1]
    return (torch.finfo(dtype).eps / 2 * out.abs() + 2 * w * mass * (1 + torch.finfo(dtype).eps)
            + n * 2.0 ** -32 * top + 2.0 ** -25)


def on_device(b, device, *, plan=None, max_rows=None):
    """(q, cache, metadata, plan, output) of a batch, the output full of NaN."""
    from tinyvllm.kernels.shared_prefix import SharedPrefixPlan
    from tinyvllm.paged_kv import PagedKVCache
    from tinyvllm.runtime.contracts import SingleQueryMetadata

    q = b["q"].to(device)
    rows, heads, dim = q.shape
    cache = PagedKVCache(num_layers=1, num_blocks=b["pool"], block_size=b["block_size"],
                         num_kv_heads=b["k"].shape[1], head_dim=dim, device=device,
                         dtype=b["k"].dtype, k_scale=b["scales"][0], v_scale=b["scales"][1],
                         layout=b["layout"])
    cache.key[0].copy_(b["k"])
    cache.value[0].copy_(b["v"])
    ids = [x for t in b["tables"] for x in t]
    offsets = [0]
    for t in b["tables"]:
        offsets.append(offsets[-1] + len(t))
    meta = SingleQueryMetadata(
        query_rows=torch.arange(rows, device=device),
        block_table_ids=torch.tensor(ids or [0], dtype=torch.long, device=device),
        block_table_offsets=torch.tensor(offsets, device=device),
        context_lens=torch.tensor(b["lengths"], dtype=torch.long, device=device),
        max_context_len=max(b["lengths"] + [1]))
    if plan is None:
        plan = SharedPrefixPlan(num_heads=heads, num_kv_heads=cache.num_kv_heads, head_dim=dim,
                                block_size=b["block_size"], max_rows=max_rows or rows,
                                device=device)
    plan.update(b["lengths"], b["groups"], b["prefixes"])
    return q, cache, meta, plan, torch.full_like(q, float("nan"))
