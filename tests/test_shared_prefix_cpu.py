"""Shared-prefix planning on the host: the plan's tasks cover every key of every
row once, within the stated bounds, and wrong arguments are refused."""
import ctypes
import random

import numpy as np
import pytest

from tinyvllm.kernels._extension import load_kernels
from tinyvllm.kernels.shared_prefix import SharedPrefixPlan, find_shared_prefixes

HEADER, TASK_WORDS = 16, 8
LONGEST = (1 << 31) - 1 - 4096  # tokens of a context


def read_plan(plan):
    """(rows' (first part, parts), members, tasks) of the plan last made."""
    host = plan.host.numpy()
    n = plan.max_rows
    rows = host[HEADER:HEADER + 2 * n].reshape(n, 2)[:plan.num_rows]
    members = host[HEADER + 2 * n:HEADER + 3 * n]
    at = HEADER + 3 * n
    return rows, members, host[at:at + TASK_WORDS * plan.num_tasks].reshape(-1, TASK_WORDS)


def check_plan(plan, lengths, groups, prefixes):
    rows, members, tasks = read_plan(plan)
    assert sorted(members[:len(lengths)]) == list(range(len(lengths)))
    assert plan.num_tasks <= plan.max_tasks and plan.workspace_bytes <= plan.max_workspace_bytes
    group = plan.num_heads // plan.num_kv_heads
    parts = {}  # (row, query head) -> [(part, k0, k1)]
    for member, queries, kvh, heads, k0, k1, part, table_row in tasks.tolist():
        begin, count = (queries >> 8) * 16, queries & 0xFF
        assert 0 < count <= 128 and heads in (1, 2, 4) and 0 <= k0 < k1
        assert heads == 1 or count <= 16
        assert kvh + heads <= plan.num_kv_heads
        assert table_row == members[member + begin // group]
        for x in range(heads):
            for i in range(begin, begin + count):
                row = int(members[member + i // group])
                head = (kvh + x) * group + i % group
                parts.setdefault((row, head), []).append((part, k0, k1))
                if groups[row] < 0 or groups[row] != groups[table_row] or row == table_row:
                    assert row == table_row
                else:  # a row reads another's table within their prefix only
                    assert k1 <= prefixes[groups[row]]
    entries = 0
    for r, n in enumerate(lengths):
        first, count = rows[r].tolist()
        if n == 0:
            assert count == 0
        for h in range(plan.num_heads):
            mine = sorted(parts.get((r, h), []))
            assert [p for p, _, _ in mine] == list(range(count))  # each part once
            edges = sorted((a, b) for _, a, b in mine)
            assert [a for a, _ in edges] == [0] * (n > 0) + [b for _, b in edges[:-1]]
            assert not edges or edges[-1][1] == n
        if count > 1:
            assert first == entries
            entries += count
    assert plan.workspace_bytes == entries * plan.num_heads * (plan.head_dim + 2) * 4


def random_step(r, max_rows, bs):
    count = r.randint(1, max_rows)
    groups_n = r.randint(0, 5)
    prefixes = [bs * r.choice([0, 1, 7, r.randint(1, 4000 // bs + 1)]) for _ in range(groups_n)]
    groups = [r.randint(-1, groups_n - 1) for _ in range(count)]
    lengths = [(prefixes[g] if g >= 0 else 0) + r.choice([0, 1, 17, 64, r.randint(1, 3000)])
               for g in groups]
    return lengths, groups, prefixes


@pytest.mark.parametrize("heads,kv_heads,dim", [
    (1, 1, 8), (8, 8, 128), (32, 8, 128), (64, 8, 128), (40, 2, 80), (150, 1, 64), (17, 17, 256),
    (12, 6, 128), (300, 2, 96)])
def test_tasks_cover_every_key_once(heads, kv_heads, dim):
    r = random.Random(heads * 1000 + dim)
    for bs in (1, 16, 24):
        plan = SharedPrefixPlan(num_heads=heads, num_kv_heads=kv_heads, head_dim=dim,
                                block_size=bs, max_rows=9, device="cpu")
        for _ in range(6):
            step = random_step(r, 9, bs)
            plan.update(*step)
            check_plan(plan, *step)


@pytest.mark.parametrize("lengths,groups,prefixes", [
    ([0], [-1], []), ([0, 0, 0], [-1, -1, -1], [160]),
    ([160, 160], [0, 0], [160]),            # nothing beyond the prefix
    ([161], [0], [160]),                    # a group of one
    ([32768 + 5] * 200, [0] * 200, [32768]),
    ([1] * 256, [-1] * 256, []),
    ([LONGEST], [-1], []),
    ([LONGEST] * 2, [0, 0], [LONGEST // 16 * 16]),
])
def test_extreme_steps(lengths, groups, prefixes):
    plan = SharedPrefixPlan(num_heads=8, num_kv_heads=2, head_dim=128, block_size=16,
                            max_rows=256, device="cpu")
    plan.update(lengths, groups, prefixes)
    check_plan(plan, lengths, groups, prefixes)


def test_update_refuses_wrong_steps():
    plan = SharedPrefixPlan(num_heads=8, num_kv_heads=2, head_dim=128, block_size=16, max_rows=4,
                            device="cpu")
    plan.update([40, 33], [0, 0], [32])
    before = plan.host.clone()
    for step, message in (
            (([40] * 5, [-1] * 5, []), "more rows"),
            (([40, 33], [0], [32]), "one length"),
            (([40, 33], [0, 1], [32]), "out of range"),
            (([40, 33], [0, -2], [32]), "out of range"),
            (([40, 31], [0, 0], [32]), "shorter"),
            (([40, 0], [0, 0], [32]), "shorter"),
            (([40, 33], [0, 0], [30]), "whole blocks"),
            (([40, 33], [0, 0], [-16]), "whole blocks"),
            (([-1, 33], [-1, -1], []), "context length"),
            (([LONGEST + 1, 33], [-1, -1], []), "context length")):
        with pytest.raises(ValueError, match=message):
            plan.update(*step)
    assert (plan.num_rows, plan.num_tasks > 0) == (2, True)
    assert plan.host.equal(before)  # a refused step leaves the plan as it was
    plan.update([40, 33], [0, 0], [32])
    assert plan.host.equal(before) and load_kernels().tvllm_last_error() == b""


def test_geometries_without_a_kernel_are_refused():
    good = dict(num_heads=8, num_kv_heads=2, head_dim=128, block_size=16, max_rows=4,
                device="cpu")
    for wrong in (dict(head_dim=130), dict(head_dim=264), dict(num_kv_heads=3),
                  dict(num_heads=8192, num_kv_heads=8), dict(max_rows=1 << 21)):
        with pytest.raises(ValueError):
            SharedPrefixPlan(**{**good, **wrong})
    for wrong in (dict(head_dim=0), dict(block_size=0), dict(max_rows=0)):
        with pytest.raises(ValueError):
            SharedPrefixPlan(**{**good, **wrong})
    with pytest.raises(TypeError):
        SharedPrefixPlan(**{**good, "num_heads": 8.0})


def entry_args(**over):
    """Arguments of tvllm_paged_decode_shared_prefix with no rows."""
    args = dict(q=None, qts=1024, qhs=128, k=None, v=None, out=None, ots=1024, ohs=128, rows=None,
                blocks=None, offsets=None, plan=None, num_rows=0, max_rows=4, num_tasks=0,
                heads=8, kv_heads=2, dim=128, slots=64, css=256, chs=128, bs=16, scale=0.1,
                ws=None, ws_bytes=0, dtype=0, cache=0, ks=1.0, vs=1.0, stream=None)
    args.update(over)
    return list(args.values())


def test_entry_point_refuses_wrong_arguments():
    lib = load_kernels()
    assert lib.tvllm_paged_decode_shared_prefix(*entry_args()) == 0
    for over, message in (
            (dict(dtype=2), b"float16 or bfloat16"), (dict(cache=1), b"cache dtype"),
            (dict(ks=0.0, cache=3), b"positive"), (dict(vs=2.0), b"FP8 cache only"),
            (dict(kv_heads=3), b"GQA"), (dict(dim=12), b"head_dim"), (dict(bs=0), b"block"),
            (dict(slots=65), b"block"), (dict(css=100), b"non-overlapping"),
            (dict(scale=0.0), b"scale"), (dict(num_rows=5), b"more rows"),
            (dict(num_tasks=1 << 20), b"more tasks"), (dict(ws_bytes=-1), b"negative"),
            (dict(num_rows=1), b"null pointer")):
        assert lib.tvllm_paged_decode_shared_prefix(*entry_args(**over)) == -1, over
        assert message in lib.tvllm_last_error(), (over, lib.tvllm_last_error())
    ptr = 1 << 20  # aligned; refused before anything is launched
    some = dict(num_rows=1, q=ptr, k=ptr, v=ptr, out=ptr, rows=ptr, blocks=ptr, offsets=ptr,
                plan=ptr)
    for over, message in (
            (dict(q=ptr + 2), b"Q rows"), (dict(qts=1020), b"Q rows"),
            (dict(k=ptr + 8), b"cache rows"), (dict(out=ptr + 4), b"output rows"),
            (dict(ohs=130), b"output rows"), (dict(ws_bytes=64), b"null workspace"),
            (dict(ws=ptr + 4, ws_bytes=64), b"workspace")):
        assert lib.tvllm_paged_decode_shared_prefix(*entry_args(**{**some, **over})) == -1, over
        assert message in lib.tvllm_last_error(), (over, lib.tvllm_last_error())
    assert lib.tvllm_paged_decode_shared_prefix(*entry_args()) == 0
    assert lib.tvllm_last_error() == b""


def test_planner_entry_point_refuses_small_buffers():
    lib = load_kernels()
    one = (ctypes.c_int64 * 1)(5)
    group = (ctypes.c_int64 * 1)(-1)
    tasks, need = ctypes.c_int64(), ctypes.c_int64()
    words = lib.tvllm_shared_prefix_plan_words(1, 8, 2)
    buffer = (ctypes.c_int32 * words)()
    call = lambda n: lib.tvllm_shared_prefix_plan(  # noqa: E731
        one, group, None, 1, 0, 1, 8, 2, 128, 16, buffer, n, ctypes.byref(tasks),
        ctypes.byref(need))
    assert call(words - 1) == -1 and b"too small" in lib.tvllm_last_error()
    assert call(words) == 0 and tasks.value >= 1
    assert lib.tvllm_shared_prefix_plan_words(0, 8, 2) == 0
    assert lib.tvllm_shared_prefix_workspace_size(4, 8, 3, 128) == 0


def brute_groups(tables, lengths, bs):
    """Row pairs with the same first block, and their groups' common blocks."""
    usable = [max(n - 1, 0) // bs for n in lengths]
    found = {}
    for r, t in enumerate(tables):
        if usable[r]:
            found.setdefault(t[0], []).append(r)
    out = {}
    for members in found.values():
        if len(members) > 1:
            limit = min(usable[r] for r in members)
            common = next((i for i in range(limit)
                           if len({tables[r][i] for r in members}) > 1), limit)
            for r in members:
                out[r] = (tuple(members), common * bs)
    return out


def test_find_shared_prefixes_matches_brute_force():
    r = random.Random(3)
    for _ in range(40):
        bs = r.choice([1, 4, 16])
        heads = [[r.randrange(10 ** 6) for _ in range(9)] for _ in range(3)]
        tables, lengths = [], []
        for _ in range(r.randint(1, 12)):
            base = r.choice(heads)[:r.randint(0, 9)]
            t = base + [r.randrange(10 ** 6) for _ in range(r.randint(0 if base else 1, 5))]
            tables.append(t)
            lengths.append(r.choice([0, 1, (len(t) - 1) * bs + r.randint(1, bs), len(t) * bs]))
        offsets = np.cumsum([0] + [len(t) for t in tables])
        ids = np.concatenate(tables)
        groups, prefixes = find_shared_prefixes(ids, offsets, lengths, bs)
        want = brute_groups(tables, lengths, bs)
        for row in range(len(tables)):
            if row in want:
                members, common = want[row]
                assert tuple(np.flatnonzero(groups == groups[row])) == members
                assert prefixes[groups[row]] == common
            else:
                assert groups[row] == -1
