"""Decode attention over shared prefixes against attention in 64 bits."""
import pytest
import torch

from shared_prefix_util import allowed, attend64, make_batch, on_device

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def run(b, device):
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    q, cache, meta, plan, out = on_device(b, device)
    paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=b["scale"])
    torch.cuda.synchronize()
    return out


def check(b, out):
    want, mass, qk = attend64(b)
    err = (out.cpu().double() - want).abs()
    limit = allowed(b, want, mass, qk, out.dtype)
    assert torch.isfinite(out).all()
    assert (err <= limit).all(), f"{float((err / limit).max()):.2f} times the bound"


SHAPES = [  # heads, kv heads, dim, dtype, fp8, layout, block size
    (8, 8, 128, BF16, False, "token_major", 16),
    (32, 8, 128, BF16, False, "head_major", 16),
    (16, 2, 128, F16, False, "token_major", 16),
    (10, 2, 128, BF16, True, "token_major", 16),
    (12, 4, 64, F16, False, "head_major", 8),
    (8, 2, 64, BF16, True, "head_major", 1),
    (8, 2, 32, BF16, False, "token_major", 24),
    (6, 2, 32, F16, True, "token_major", 16),
    (8, 1, 256, BF16, False, "token_major", 32),
    (4, 2, 256, F16, True, "head_major", 256),
    (8, 2, 96, BF16, False, "token_major", 16),
    (40, 2, 80, F16, False, "token_major", 7),
    (9, 3, 8, BF16, False, "token_major", 16),
    (4, 2, 200, BF16, True, "token_major", 16),
    (150, 1, 128, BF16, False, "token_major", 16),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("count", [2, 5, 40])
def test_one_group(device, shape, count):
    """A group of rows behind one prefix of several tiles, own parts of every
    kind of end (none, one token, odd, several chunks), and rows apart."""
    heads, kv_heads, dim, dtype, fp8, layout, bs = shape
    prefix = -(-330 // bs) * bs
    own = [0, 1, 2, 17, 63, 64, 65, 130, 300]
    rows = [(0, own[i % len(own)]) for i in range(count)] + [(-1, 77), (-1, 0), (-1, 1)]
    b = make_batch(seed=count, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, fp8=fp8,
                   layout=layout, block_size=bs, prefixes=[prefix], rows=rows)
    out = run(b, device)
    assert (out[count + 1] == 0).all()
    check(b, out)


def test_several_groups_and_scattered_rows(device):
    """Groups of their own sizes and prefixes (one of a single row, one empty),
    rows of a group anywhere in the batch, query rows not in batch order."""
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    rows = [(g, n) for g, n in ((0, 5), (1, 40), (-1, 90), (0, 0), (2, 3), (1, 1), (0, 64),
                                (3, 200), (1, 7), (-1, 1), (0, 129), (1, 0), (3, 2))]
    b = make_batch(seed=4, heads=16, kv_heads=4, dim=128, dtype=BF16,
                   prefixes=[160, 1040, 48, 16, 64], rows=rows)
    b["q"] = torch.cat([b["q"], torch.zeros(5, 16, 128, dtype=BF16)])  # tokens of nobody
    q, cache, meta, plan, out = on_device(dict(b, q=b["q"][:len(rows)]), device)
    order = torch.randperm(len(rows) + 5, generator=torch.Generator().manual_seed(1))[:len(rows)]
    wide_q = torch.randn(len(rows) + 5, 16, 128, dtype=BF16, device=device)
    wide_q[order.to(device)] = q
    wide_out = torch.full_like(wide_q, 7.0)
    import dataclasses

    meta = dataclasses.replace(meta, query_rows=order.to(device))
    paged_decode_shared_prefix(wide_q, cache, 0, meta, plan, wide_out, scale=b["scale"])
    check(dict(b, q=b["q"][:len(rows)]), wide_out[order.to(device)])
    others = torch.ones(len(rows) + 5, dtype=torch.bool)
    others[order] = False
    assert (wide_out[others.to(device)] == 7.0).all()  # tokens of no row stay as they were


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_strided_queries_and_outputs(device, dtype, fp8):
    """Q as the head slice of a packed projection, the output likewise."""
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    b = make_batch(seed=8, heads=8, kv_heads=2, dim=64, dtype=dtype, fp8=fp8, prefixes=[512],
                   rows=[(0, n) for n in range(1, 31)])
    q, cache, meta, plan, out = on_device(b, device)
    packed = torch.randn(30, 12, 72, device=device).to(dtype)
    packed[:, 2:10, :64] = q
    spaced = torch.zeros(30, 10, 72, device=device, dtype=dtype)
    paged_decode_shared_prefix(packed[:, 2:10, :64], cache, 0, meta, plan, spaced[:, 1:9, :64],
                               scale=b["scale"])
    check(b, spaced[:, 1:9, :64])
    assert (spaced[:, 0] == 0).all() and (spaced[:, 9] == 0).all()
    assert (spaced[..., 64:] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("count", [3, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_slots_that_no_row_attends_do_not_matter(device, bad, count, dim):
    """NaNs and infinities in the rest of the last pages, in unused blocks and
    in another layer leave every result as it is."""
    rows = [(0, n) for n in (1, 3, 9, 15, 17, 31, 33, 50)] * 5
    b = make_batch(seed=11, heads=8, kv_heads=2, dim=dim, dtype=BF16, prefixes=[208],
                   rows=rows[:count])
    want = run(b, device)
    used = torch.zeros(len(b["k"]), dtype=torch.bool)
    for table, n in zip(b["tables"], b["lengths"]):
        for t in range(n):
            used[table[t // 16] * 16 + t % 16] = True
    assert (~used).any()
    for name in "kv":
        b[name][~used] = bad
    assert torch.equal(run(b, device), want)


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), 1e30])
def test_extreme_values_reach_only_who_attends_them(device, where, value):
    """A value of V beyond fp16, an infinity or a NaN in one dim of one KV head:
    that dim of the rows that attend it, and nothing else, changes."""
    rows = [(0, 20 + i) for i in range(24)] + [(-1, 70)]
    b = make_batch(seed=12, heads=8, kv_heads=2, dim=128, dtype=BF16, prefixes=[400], rows=rows)
    plain = run(b, device).cpu()
    owner = 5
    t = 130 if where == "prefix" else 405
    slot = b["tables"][owner][t // 16] * 16 + t % 16
    b["v"][slot, 1, 77] = value
    got = run(b, device).cpu()
    hit = torch.zeros(25, 8, 128, dtype=torch.bool)
    hit[:24 if where == "prefix" else 0, 4:, 77] = True
    hit[owner, 4:, 77] = True
    if value == 1e30:
        check(b, got.to(device))
    else:
        assert not torch.isfinite(got[hit]).any()
    # The others agree to their rounding: the task was done again another way.
    want, mass, qk = attend64(dict(b, v=torch.where(b["v"].abs() < 1e29, b["v"], 0)))
    limit = allowed(dict(b, v=torch.where(b["v"].abs() < 1e29, b["v"], 0)), want, mass, qk, BF16)
    assert ((got.double() - want).abs()[~hit] <= limit[~hit]).all()
    assert torch.equal(got[24], plain[24])


def test_weights_far_below_the_largest_keep_their_value(device):
    """One key of a prefix far above the others, which are many and all alike:
    fp16 weights would lose or bias them without room below the largest."""
    count, prefix, dim = 20, 4096, 64
    b = make_batch(seed=13, heads=8, kv_heads=2, dim=dim, dtype=F16, prefixes=[prefix],
                   rows=[(0, 1)] * count)
    # Scores 0 everywhere but one key at 12 ln 2: the many weigh 2^-12 each.
    b["q"].zero_()
    b["q"][..., 0] = 1.0
    b["k"].zero_()
    top = b["tables"][0][7] * 16 + 3
    b["k"][top, :, 0] = 12 * 0.6931471805599453 / b["scale"]
    check(b, run(b, device))


def test_long_prefix_and_many_rows(device):
    b = make_batch(seed=14, heads=8, kv_heads=1, dim=128, dtype=BF16, prefixes=[20000],
                   rows=[(0, i % 90) for i in range(70)], std=2.0)
    check(b, run(b, device))


def test_single_tokens_and_empty_batches(device):
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    b = make_batch(seed=15, heads=4, kv_heads=2, dim=128, dtype=BF16, prefixes=[16],
                   rows=[(0, 0), (0, 0), (-1, 1), (-1, 0)])
    out = run(b, device)
    check(b, out)
    assert (out[3] == 0).all()
    empty = make_batch(seed=16, heads=4, kv_heads=2, dim=128, dtype=BF16, prefixes=[],
                       rows=[(-1, 0)] * 3)
    assert (run(empty, device) == 0).all()
    none = make_batch(seed=17, heads=4, kv_heads=2, dim=128, dtype=BF16, prefixes=[], rows=[])
    q, cache, meta, plan, out = on_device(none, device, max_rows=1)
    paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=1.0)


def test_same_result_every_time_and_on_another_stream(device):
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    b = make_batch(seed=18, heads=32, kv_heads=8, dim=128, dtype=BF16, prefixes=[1024],
                   rows=[(0, 50 + i) for i in range(33)])
    q, cache, meta, plan, out = on_device(b, device)
    paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=b["scale"])
    first = out.clone()
    check(b, first)
    side = torch.cuda.Stream(device=device)
    side.wait_stream(torch.cuda.current_stream(device))
    outs = [torch.empty_like(out) for _ in range(2)]
    with torch.cuda.stream(side):  # two calls that may overlap: each has its own workspace
        paged_decode_shared_prefix(q, cache, 0, meta, plan, outs[0], scale=b["scale"])
    paged_decode_shared_prefix(q, cache, 0, meta, plan, outs[1], scale=b["scale"])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)


def test_captured_call_follows_the_plan_that_is_uploaded(device):
    """One graph of two calls (so their private workspaces come from one pool),
    replayed over later plans, caches and tables, with eager work between."""
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    shape = dict(heads=16, kv_heads=4, dim=128, dtype=BF16)
    first = make_batch(seed=20, prefixes=[320], rows=[(0, 9 + i) for i in range(12)], spare=200,
                       **shape)
    q, cache, meta, plan, out = on_device(first, device)
    blocks = torch.zeros(2000, dtype=torch.long, device=device)
    offsets = torch.zeros(13, dtype=torch.long, device=device)
    import dataclasses

    meta = dataclasses.replace(meta, block_table_ids=blocks, block_table_offsets=offsets)
    again = torch.empty_like(out)

    def both():
        paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=first["scale"])
        paged_decode_shared_prefix(q, cache, 0, meta, plan, again, scale=first["scale"])

    side = torch.cuda.Stream(device=device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    steps = [first]
    for seed, prefixes, rows in (
            (21, [], [(-1, n) for n in range(12)]),
            (22, [320, 640], [(i % 2, i) for i in range(12)]),
            (23, [64], [(0, 3)] * 7 + [(-1, 0)] * 5),
            (24, [1600], [(0, 40)] * 12)):
        steps.append(make_batch(seed=seed, prefixes=prefixes, rows=rows, **shape))
    for b in steps:
        slots = len(b["k"])
        assert slots <= len(first["k"])
        q.copy_(b["q"])
        cache.key[0][:slots].copy_(b["k"])
        cache.value[0][:slots].copy_(b["v"])
        ids = torch.tensor([x for t in b["tables"] for x in t] or [0])
        blocks[:len(ids)].copy_(ids)
        offsets.copy_(torch.tensor([0] + [len(t) for t in b["tables"]]).cumsum(0))
        plan.update(b["lengths"], b["groups"], b["prefixes"])
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(b, out)
        assert torch.equal(again, out)
        both()  # the same calls outside the graph
        check(b, out)


def test_wrapper_refusals(device):
    import dataclasses

    from tinyvllm.kernels.shared_prefix import SharedPrefixPlan, paged_decode_shared_prefix

    b = make_batch(seed=30, heads=8, kv_heads=2, dim=128, dtype=BF16, prefixes=[32],
                   rows=[(0, 3), (0, 5)])
    q, cache, meta, plan, out = on_device(b, device)

    def call(**over):
        args = dict(q=q, cache=cache, layer_idx=0, metadata=meta, plan=plan, output=out,
                    scale=b["scale"])
        args.update(over)
        paged_decode_shared_prefix(**args)

    call()
    other = SharedPrefixPlan(num_heads=8, num_kv_heads=2, head_dim=64, block_size=16, max_rows=2,
                             device=device)
    short = SharedPrefixPlan(num_heads=8, num_kv_heads=2, head_dim=128, block_size=16, max_rows=2,
                             device=device)
    short.update([5], [-1], [])
    host = SharedPrefixPlan(num_heads=8, num_kv_heads=2, head_dim=128, block_size=16, max_rows=2,
                            device="cpu")
    host.update(b["lengths"], b["groups"], b["prefixes"])
    for over, message in (
            (dict(q=q.float()), "float16 or bfloat16"), (dict(q=q[0]), "heads, dim"),
            (dict(output=out.half()), "dtype"), (dict(output=out[:, :4]), "match Q"),
            (dict(plan=other), "geometry"), (dict(plan=short), "number of rows"),
            (dict(plan=host), "one GPU"), (dict(q=q.cpu()), "GPU"),
            (dict(scale=-1.0), "scale"),
            (dict(metadata=dataclasses.replace(meta, query_rows=meta.query_rows.int())),
             "int64"),
            (dict(metadata=dataclasses.replace(
                meta, block_table_offsets=meta.block_table_offsets[:2])), "align"),
            (dict(workspace=torch.empty(1 << 20, dtype=torch.float32, device=device)), "uint8"),
            (dict(q=torch.empty(2, 8, 132, dtype=BF16, device=device)[..., 2:130],), "Q rows")):
        with pytest.raises(RuntimeError, match=message):
            call(**over)
    with pytest.raises(RuntimeError, match="match Q shape"):
        call(q=q.transpose(0, 2))


def test_launches_go_to_the_tensors_device(device, monkeypatch):
    """With another device current, the queries' own is made current for the call."""
    from tinyvllm.kernels import _extension

    b = make_batch(seed=31, heads=8, kv_heads=2, dim=128, dtype=BF16, prefixes=[32],
                   rows=[(0, 3), (0, 5)])
    entered = []

    class Recorded(torch.cuda.device):
        def __init__(self, where):
            entered.append(where)
            super().__init__(where)

    args = on_device(b, device)
    monkeypatch.setattr(_extension, "_current_device", lambda: 99)
    monkeypatch.setattr(torch.cuda, "device", Recorded)
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    q, cache, meta, plan, out = args
    paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=b["scale"])
    assert q.device in entered
    check(b, out)


def test_layers_of_a_cache(device):
    """Every layer by its index, from either end; indexes past them are refused."""
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix
    from tinyvllm.paged_kv import PagedKVCache

    for layout in ("token_major", "head_major"):
        b = make_batch(seed=32, heads=8, kv_heads=2, dim=64, dtype=BF16, prefixes=[48],
                       rows=[(0, 3), (0, 5), (-1, 20)])
        q, cache, meta, plan, out = on_device(b, device)
        deep = PagedKVCache(num_layers=3, num_blocks=b["pool"], block_size=16, num_kv_heads=2,
                            head_dim=64, device=device, dtype=BF16, layout=layout)
        for layer in range(3):
            deep.key[layer].copy_(cache.key[0] * 2 ** layer)
            deep.value[layer].copy_(cache.value[0] + layer)
        for layer in (0, 1, 2, -1, -3):
            n = layer % 3
            paged_decode_shared_prefix(q, deep, layer, meta, plan, out, scale=b["scale"])
            check(dict(b, k=deep.key[n].cpu(), v=deep.value[n].cpu()), out)
        for layer in (3, -4):
            with pytest.raises(IndexError):
                paged_decode_shared_prefix(q, deep, layer, meta, plan, out, scale=b["scale"])


def test_refused_over_the_queries_and_under_capture(device):
    """The output over Q is refused; so is an update that a graph would record
    (its upload would be replayed from a buffer that later updates rewrite)."""
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    b = make_batch(seed=33, heads=8, kv_heads=2, dim=128, dtype=BF16, prefixes=[32],
                   rows=[(0, 3), (0, 5)])
    q, cache, meta, plan, out = on_device(b, device)
    with pytest.raises(RuntimeError, match="output"):
        paged_decode_shared_prefix(q, cache, 0, meta, plan, q, scale=b["scale"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.fill_(0)
        with pytest.raises(RuntimeError, match="capture"):
            plan.update(b["lengths"], b["groups"], b["prefixes"])
    graph.replay()
    torch.cuda.synchronize()
    paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=b["scale"])
    check(b, out)


# Few short rows are planned without sharing; a long row beside them has the
# groups' keys shared and their parts merged.
LONG = (-1, 700)


def shares(b, device):
    """Whether the batch's plan shares a prefix (a task of more than one row)."""
    plan = on_device(b, device)[3]
    return plan.workspace_bytes > 0


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("count", [2, 5, 40])
def test_one_group_beside_a_long_row(device, shape, count):
    heads, kv_heads, dim, dtype, fp8, layout, bs = shape
    own = [0, 1, 2, 17, 63, 64, 65, 130, 300]
    rows = [(0, own[i % len(own)]) for i in range(count)] + [(-1, 77), (-1, 0), (-1, 1), LONG]
    b = make_batch(seed=40 + count, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, fp8=fp8,
                   layout=layout, block_size=bs, prefixes=[-(-330 // bs) * bs], rows=rows)
    assert shares(b, device)
    out = run(b, device)
    assert (out[count + 1] == 0).all()
    check(b, out)


@pytest.mark.parametrize("dtype,fp8", [(BF16, False), (F16, False), (BF16, True)])
def test_strided_queries_and_outputs_beside_a_long_row(device, dtype, fp8):
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    b = make_batch(seed=50, heads=8, kv_heads=2, dim=64, dtype=dtype, fp8=fp8, prefixes=[512],
                   rows=[(0, n) for n in range(1, 30)] + [LONG])
    q, cache, meta, plan, out = on_device(b, device)
    packed = torch.randn(30, 12, 72, device=device).to(dtype)
    packed[:, 2:10, :64] = q
    spaced = torch.zeros(30, 10, 72, device=device, dtype=dtype)
    paged_decode_shared_prefix(packed[:, 2:10, :64], cache, 0, meta, plan, spaced[:, 1:9, :64],
                               scale=b["scale"])
    check(b, spaced[:, 1:9, :64])
    assert (spaced[:, 0] == 0).all() and (spaced[:, 9] == 0).all()
    assert (spaced[..., 64:] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("count", [3, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_unattended_slots_do_not_matter_beside_a_long_row(device, bad, count, dim):
    rows = [(0, n) for n in (1, 3, 9, 15, 17, 31, 33, 50)] * 5
    b = make_batch(seed=51, heads=8, kv_heads=2, dim=dim, dtype=BF16, prefixes=[208],
                   rows=rows[:count] + [LONG])
    assert shares(b, device)
    want = run(b, device)
    used = torch.zeros(len(b["k"]), dtype=torch.bool)
    for table, n in zip(b["tables"], b["lengths"]):
        for t in range(n):
            used[table[t // 16] * 16 + t % 16] = True
    for name in "kv":
        b[name][~used] = bad
    assert torch.equal(run(b, device), want)


@pytest.mark.parametrize("value", [float("inf"), float("nan"), 1e30])
def test_extreme_values_of_a_shared_prefix(device, value):
    """V beyond fp16, an infinity or a NaN in one dim of one KV head's shared
    keys: the wide tasks that meet it are done again, others keep their values."""
    rows = [(0, 20 + i) for i in range(24)] + [LONG]
    b = make_batch(seed=52, heads=8, kv_heads=2, dim=128, dtype=BF16, prefixes=[400], rows=rows)
    assert shares(b, device)
    plain = run(b, device).cpu()
    b["v"][b["tables"][5][130 // 16] * 16 + 130 % 16, 1, 77] = value
    got = run(b, device).cpu()
    hit = torch.zeros(25, 8, 128, dtype=torch.bool)
    hit[:24, 4:, 77] = True
    if value == 1e30:
        check(b, got.to(device))
    else:
        assert not torch.isfinite(got[hit]).any()
    clean = dict(b, v=torch.where(b["v"].abs() < 1e29, b["v"], 0))
    want, mass, qk = attend64(clean)
    limit = allowed(clean, want, mass, qk, BF16)
    assert ((got.double() - want).abs()[~hit] <= limit[~hit]).all()
    assert torch.equal(got[24], plain[24])


def test_calls_without_parts_need_no_workspace(device):
    """Few short rows: one launch, no workspace; with a row without keys, its
    zeros come from the second one."""
    rows = [(0, 5), (0, 40), (-1, 33)]
    for more, empty in (([], False), ([(-1, 0)], True)):
        b = make_batch(seed=53, heads=8, kv_heads=2, dim=128, dtype=BF16, prefixes=[64],
                       rows=rows + more)
        q, cache, meta, plan, out = on_device(b, device)
        assert plan.workspace_bytes == 0
        from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

        for workspace in (None, torch.empty(0, dtype=torch.uint8, device=device)):
            out.fill_(float("nan"))
            paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=b["scale"],
                                       workspace=workspace)
            check(b, out)
            assert not empty or (out[3] == 0).all()
