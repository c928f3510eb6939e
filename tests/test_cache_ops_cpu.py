"""The cache operators' host side: step plans and what they refuse, and the entry points'
refusals, without a GPU; and the reference the GPU tests compare with, checked on its own."""
import ctypes
import math

import pytest
import torch

import cache_reference as ref
from distserve_amd import cabi


def section(words, at, n, width):
    return [tuple(words[at + width * i:at + width * (i + 1)]) for i in range(n)]


def pieces_of(step, words, heads):
    """What the kernels make of a plan: {(q_start, row0, head): [(kv_begin, kv_end, part_row)]} of the kernel
    for few rows and of the one for many, walked as the kernels walk it."""
    few, many = {}, {}
    tiles = section(words, step.row_tiles_at, step.num_row_tiles, 8)
    height = 16 * step.row_tiles
    at = (0, 0, 0)
    for group, (*copy, tile, head, unit, units) in enumerate(section(words, step.row_starts_at, step.num_row_groups, 12)):
        assert (tile, head, unit) == at and units > 0 and tuple(copy) == tiles[tile]          # each group goes on where the one before stopped
        while units:
            q_start, rows, first, table_at, row0, kv_end, total, _ = tiles[tile]
            n = min(units, total - unit)
            part = -1 if n == total else (step.num_row_groups * height if unit == 0 else 0) + group * height
            few.setdefault((q_start, row0, head), []).append((unit * 128, min(kv_end, (unit + n) * 128), part))
            units -= n
            unit += n
            if unit == total:
                unit, head = 0, head + 1
                if head == heads:
                    head, tile = 0, tile + 1
        at = (tile, head, unit)
    assert at == (step.num_row_tiles, 0, 0)                    # and nothing is left over
    for q_start, rows, first, table_at, row0, kv0, kv1, part, head0, *_ in section(words, step.tile_items_at, step.num_tile_items, 12):
        assert kv0 % 64 == 0 and head0 % 8 == 0
        for head in range(head0, min(heads, head0 + 8)):
            at_head = -1 if part < 0 else step.row_part_rows + head * step.item_part_rows + part
            many.setdefault((q_start, row0, head), []).append((kv0, kv1, at_head))
    return few, many


def plan(first, new, table, num_blocks=64, block_size=16, heads=8, kv_heads=2, head_dim=64, dtype=cabi.KVM_F16, format=cabi.KVM_CACHE_PLAIN):
    return cabi.plan_step(first, new, table, num_blocks, block_size, heads, kv_heads, head_dim, dtype, format)


def test_a_plan_names_every_slot_and_page():
    step, words = plan([0, 15, 40, 3], [17, 2, 0, 1], [[5, 9], [7, 1], [2, 3, 4], [11]])
    assert (step.num_seqs, step.num_tokens, step.num_kv_tokens, step.num_pages) == (4, 20, 17 + 17 + 40 + 4, 8)
    assert list(words[step.table_at:step.table_at + 8]) == [5, 9, 7, 1, 2, 3, 4, 11]
    slots = list(words[step.slots_at:step.slots_at + 20])
    assert slots == [5 * 16 + i for i in range(16)] + [9 * 16] + [7 * 16 + 15, 1 * 16] + [11 * 16 + 3]
    pages = [tuple(words[step.pages_at + 2 * i:step.pages_at + 2 * i + 2]) for i in range(8)]
    assert pages == [(0, 16), (16, 1), (17, 16), (33, 1), (34, 16), (50, 16), (66, 8), (74, 4)]
    assert step.all_new == 0 and plan([0, 0], [1, 2], [[0], [1]])[0].all_new == 1


@pytest.mark.parametrize("heads,kv_heads,head_dim,dtype", [(8, 8, 64, 0), (64, 8, 128, 1), (71, 1, 64, 0), (6, 2, 256, 2),
                                                           (12, 12, 80, 1)])
def test_the_pieces_of_a_plan_cover_every_row_and_key_once(heads, kv_heads, head_dim, dtype):
    import random

    rng = random.Random(heads + head_dim)
    for case in range(30):
        n = rng.choice([1, 2, 7, 40])
        new = [rng.choice([0, 1, 1, 1, 2, 5, 33, 200]) for _ in range(n)]
        first = [rng.choice([0, 1, 15, 16, 17, 700, 5000, 70000]) for _ in range(n)]
        pages = [-(-(a + b) // 16) + rng.choice([0, 0, 3]) for a, b in zip(first, new)]
        order = list(range(sum(pages) + 2))
        rng.shuffle(order)
        table, at = [], 0
        for p in pages:
            table.append(order[at:at + p])
            at += p
        step, words = plan(first, new, table, len(order), 16, heads, kv_heads, head_dim, dtype, case % 2)
        group = heads // kv_heads
        starts, table_at = [0], [0]
        for b, p in zip(new, pages):
            starts.append(starts[-1] + b)
            table_at.append(table_at[-1] + p)
        tile_of = [128 if dtype != cabi.KVM_F32 and m * group > 32 else 16 * step.row_tiles for m in new]
        # the tiles' and items' own fields
        for at, count, width in ((step.row_tiles_at, step.num_row_tiles, 8), (step.tile_items_at, step.num_tile_items, 12)):
            for q_start, total, begin, table_start, row0, *_ in section(words, at, count, width):
                s = next(s for s in range(n) if starts[s] == q_start and new[s] > 0)
                assert total == new[s] * group and begin == first[s] and table_start == table_at[s]
                assert (tile_of[s] == 128) == (at == step.tile_items_at) and row0 % tile_of[s] == 0
        few, many = pieces_of(step, words, kv_heads)
        joins = {(j[0], j[1], j[3]): j for j in section(words, step.joins_at, step.num_joins, 8)}
        assert len(joins) == step.num_joins
        used = []
        for s in range(n):
            for row0 in range(0, new[s] * group, tile_of[s]):
                here = min(tile_of[s], new[s] * group - row0)
                for head in range(kv_heads):
                    key = (starts[s], row0, head)
                    pieces = (many if tile_of[s] == 128 else few).pop(key)
                    assert pieces[0][0] == 0 and pieces[-1][1] == first[s] + (row0 + here - 1) // group + 1
                    assert all(a[1] == b[0] and a[0] < a[1] for a, b in zip(pieces, pieces[1:]))
                    if len(pieces) == 1:
                        assert pieces[0][2] == -1 and key not in joins
                    else:
                        _, _, rows_here, _, part, after, pitch, count = joins.pop(key)
                        assert rows_here == here <= step.join_rows and count == len(pieces)
                        assert [p[2] for p in pieces] == [part] + [after + i * pitch for i in range(count - 1)]
                        used += [r for p in pieces for r in range(p[2], p[2] + here)]
        assert not few and not many and not joins
        assert len(set(used)) == len(used) and all(0 <= r < step.part_rows for r in used)
        assert cabi.attention_workspace(step) == step.part_rows * (head_dim + 2) * 4
        # every group of the kernel for few rows has the same amount to read, give or take a unit
        shares = [g[11] for g in section(words, step.row_starts_at, step.num_row_groups, 12)]
        assert not shares or max(shares) - min(shares) <= 1


def test_plans_refuse_what_a_kernel_could_trip_over():
    def refused(code, *args, **kwargs):
        with pytest.raises(cabi.KvmError) as e:
            plan(*args, **kwargs)
        assert e.value.code == code, e.value
        return str(e.value)

    ok = ([3], [2], [[0]])
    plan(*ok)
    assert "block_table[0][1] = 64" in refused(cabi.KVM_ERANGE, [0], [20], [[0, 64]])
    refused(cabi.KVM_ERANGE, [0], [20], [[0, -1]])
    refused(cabi.KVM_ERANGE, [0], [1], [[0, 99]])                       # not needed, still a bad table
    assert "17 tokens" in refused(cabi.KVM_ERANGE, [15], [2], [[0]])
    refused(cabi.KVM_ERANGE, [-1], [2], [[0]])
    refused(cabi.KVM_ERANGE, [1], [-2], [[0]])
    assert "two tokens" in refused(cabi.KVM_EDUP, [3, 3], [1, 1], [[7], [7]])
    refused(cabi.KVM_EDUP, [0], [32], [[7, 7]])
    plan([16, 16], [1, 1], [[7, 8], [7, 9]])                            # a shared prefix is fine
    plan([3, 4], [1, 1], [[7], [7]])                                    # and so are two slots of one block
    for bad in (dict(heads=7), dict(heads=0), dict(kv_heads=0), dict(head_dim=72), dict(head_dim=0), dict(head_dim=272),
                dict(dtype=3), dict(format=2), dict(block_size=0), dict(block_size=70000), dict(num_blocks=-1),
                dict(num_blocks=2**27, block_size=16)):
        refused(cabi.KVM_EINVAL, *ok, **bad)
    refused(cabi.KVM_ERANGE, [2**31], [1], [[0]])
    with pytest.raises(cabi.KvmError):
        cabi.plan_step([1], [1], [], 0, 0, 8, 8, 64, cabi.KVM_F16)      # earlier tokens need a cache
    step, _ = cabi.plan_step([0, 0], [3, 4], [], 0, 0, 8, 8, 64, cabi.KVM_F16)
    assert step.num_blocks == 0 and step.num_tokens == 7
    # an empty step is a plan like any other
    step, _ = plan([], [], [])
    assert step.num_tokens == 0 and step.num_row_groups == 0 and step.num_tile_items == 0
    # too little room is refused, not overrun
    words, first, new = (ctypes.c_int32 * 64)(), (ctypes.c_int64 * 1)(0), (ctypes.c_int64 * 1)(40)
    table, lens, out = (ctypes.c_int64 * 3)(0, 1, 2), (ctypes.c_int64 * 1)(3), cabi.KvmStep()
    rc = cabi.lib.kvm_plan_step(first, new, 1, table, lens, 8, 16, 8, 2, 64, 0, 0, words, 30, ctypes.byref(out))
    assert rc == cabi.KVM_EINVAL and b"kvm_plan_words" in cabi.lib.kvm_last_error()


def test_entry_points_refuse_before_they_touch_a_device():
    step, words = plan([3], [2], [[0]])
    at = ctypes.addressof(words)
    pools = cabi.KvmCache(4096, 8192, 64, 2, 0, 2, 16, 64, cabi.KVM_F16, cabi.KVM_CACHE_PLAIN)
    rows = cabi.KvmRows(4096, 128, 64)

    def refused(code, call, *args):
        with pytest.raises(cabi.KvmError) as e:
            call(*args)
        assert e.value.code == code, e.value

    # host memory in the place of the device copy of the plan
    refused(cabi.KVM_EINVAL, cabi.write_kv, step, at, pools, rows, rows)
    refused(cabi.KVM_EINVAL, cabi.paged_attention, step, at, pools, rows, rows, 1.0)
    # a step that was changed, or never made
    step.num_tokens = 3
    for call, args in ((cabi.write_kv, (pools, rows, rows)), (cabi.read_kv, (pools, rows, rows)),
                       (cabi.paged_attention, (pools, rows, rows, 1.0)), (cabi.prompt_attention, (rows, rows, rows, rows, 1.0))):
        refused(cabi.KVM_EINVAL, call, step, at, *args)
        refused(cabi.KVM_EINVAL, call, cabi.KvmStep(), at, *args)
    refused(cabi.KVM_EINVAL, cabi.attention_workspace, step)
    # nothing to do is nothing done, whatever else the call says
    empty, _ = plan([5], [0], [[0]])
    cabi.write_kv(empty, 0, pools, rows, rows)
    cabi.paged_attention(empty, 0, pools, rows, rows, 1.0)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: only for a machine where nothing can be launched")
def test_entry_points_refuse_memory_that_is_written_and_used():
    step, _ = plan([0], [3], [[0]], num_blocks=4)          # 3 tokens, 8 heads, 2 KV heads of 64 in fp16: rows of 128 bytes
    step.device = 0                                        # the caller vouches for extents: no question to the runtime
    K, V, Q, O, S, W = (i << 24 for i in range(1, 7))
    pool = 4 * 2 * 2 * 16 * 64 * 2

    def pools(k=K, v=V):
        return cabi.KvmCache(k, v, 4, 2, 0, 2, 16, 64, cabi.KVM_F16, cabi.KVM_CACHE_PLAIN, pool)

    def rows(at, token, head=64, extent=1 << 20):
        return cabi.KvmRows(at, token, head, extent)

    def refused(code, text, call, *args):
        with pytest.raises(cabi.KvmError, match=text) as e:
            call(step, W, *args)
        assert e.value.code == code, e.value

    q, k, v = rows(Q, 512), rows(S, 128), rows(S + 4096, 128)
    for out in (rows(Q, 512), rows(Q + 128, 512), rows(Q + 2048, 512), rows(Q, 1024), rows(Q + 1024, 1024 + 64),
                rows(Q + 128, 64, 3 * 64), rows(Q - 1024 + 128, 512)):
        refused(cabi.KVM_EINVAL, "out and q share memory", cabi.paged_attention, pools(), q, out, 1.0)
    refused(cabi.KVM_EINVAL, "out and a pool", cabi.paged_attention, pools(), q, rows(V + pool - 16, 512), 1.0)
    refused(cabi.KVM_EINVAL, "out and a pool", cabi.paged_attention, pools(), q, rows(K - 16, 512), 1.0)
    refused(cabi.KVM_EINVAL, "out and k", cabi.prompt_attention, q, k, v, rows(S - 2048, 512), 1.0)
    refused(cabi.KVM_EINVAL, "out and v", cabi.prompt_attention, q, k, rows(O + 1024, 128), rows(O, 512), 1.0)
    refused(cabi.KVM_EINVAL, "k and a pool", cabi.write_kv, pools(), rows(K, 128), v)
    refused(cabi.KVM_EINVAL, "v and a pool", cabi.write_kv, pools(), k, rows(K + pool - 128, 128))
    refused(cabi.KVM_EINVAL, "the K pool and the V pool", cabi.write_kv, pools(v=K), k, v)
    refused(cabi.KVM_EINVAL, "the K pool and the V pool", cabi.write_kv, pools(v=K + pool - 16), k, v)
    refused(cabi.KVM_EINVAL, "k_out and v_out", cabi.read_kv, pools(), rows(O, 128), rows(O, 128))
    refused(cabi.KVM_EINVAL, "k_out and v_out", cabi.read_kv, pools(), rows(O, 256), rows(O + 128, 256))
    refused(cabi.KVM_EINVAL, "k_out and a pool", cabi.read_kv, pools(), rows(K + 256, 128), rows(O, 128))
    # strides whose reach passes 64 bits
    refused(cabi.KVM_ERANGE, "too large", cabi.write_kv, pools(), rows(S, 1 << 62), v)
    refused(cabi.KVM_ERANGE, "too large", cabi.paged_attention, pools(), q, rows(O, 1 << 62), 1.0)


def test_a_plan_that_memory_does_not_suffice_for_is_refused():
    code = """
import ctypes, resource
from distserve_amd import cabi
now = int(open('/proc/self/statm').read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (now + (64 << 20), now + (64 << 20)))
try:
    cabi.plan_step([0], [1], [[0]], 1 << 26, 31, 8, 2, 64, cabi.KVM_F16)       # a bit for each of 2^31 slots
except cabi.KvmError as e:
    assert e.code == cabi.KVM_EINVAL and 'alloc' in str(e), e
    print('refused')
"""
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout == "refused\n", (done.returncode, done.stdout, done.stderr)


def test_the_words_of_impossible_steps_are_refused():
    for bad in ((-1, 1, 1, 8, 2), (1, 1 << 40, 1, 8, 2), (1, 1, 1 << 40, 8, 2), (1, 1, 1, 8, 9), (1, 1, 1, 1 << 21, 1), (1, 1, 1, 8, 0)):
        assert cabi.lib.kvm_plan_words(*bad) == cabi.KVM_EINVAL


def test_the_op_layer_refuses_cpu_tensors_and_plans_without_a_gpu():
    import distserve_amd

    z = torch.zeros(4, 1, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        distserve_amd.plan_step(z, [1], [0], [[0]], 4)
    with pytest.raises(RuntimeError, match="not torch.float64"):
        distserve_amd.plan_prompt([1], 2, 2, 64, torch.float64, "cuda:0")
    held = distserve_amd.StepPlan([0], [3], [1], [1], 4, 16, 4, 2, 64, 5, False, -1)      # a plan to look at
    assert held.num_tokens() == 3 and held.device_index() == -1
    row = torch.zeros(3, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="without a GPU"):
        distserve_amd.write_kv(held, 0, row, row, z, z)
    for bad in (([0], [3], [1], [2], 4), ([0, 0], [3], [1], [1], 4), ([0], [3], [1], [], 4), ([0], [-3], [1], [1], 4),
                ([0], [3], [4], [1], 4)):
        with pytest.raises(RuntimeError):
            distserve_amd.StepPlan(*bad, 16, 4, 2, 64, 5, False, -1)


def test_the_alternate_namespace_has_the_cache_ops_too():
    import os

    import distserve_amd

    torch.ops.load_library(os.path.join(os.path.dirname(distserve_amd.TORCH_LIB_PATH), "libkvmove_torch_alt.so"))
    for name in ("write_kv", "read_kv", "paged_attention", "prompt_attention"):
        ours = str(getattr(torch.ops.kvcache_ops, name).default._schema)
        theirs = str(getattr(torch.ops.kvmove_kvcache_ops, name).default._schema)
        assert theirs.replace("kvmove_kvcache_ops", "kvcache_ops") == ours
    plan = torch.classes.kvmove_kvcache_ops.StepPlan([0], [3], [1], [1], 4, 16, 4, 2, 64, 5, False, -1)
    assert plan.num_kv_tokens() == 3


def test_the_reference_quantiser_agrees_with_the_cast_and_with_its_bound():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(200, 64, generator=g) * torch.exp(torch.randn(200, 1, generator=g) * 5)
    x[3] = 0.0
    x[4, 5], x[4, 6], x[4, 7] = math.inf, -math.inf, math.nan
    x[5] = 448.0
    x[6] = 449.0
    x[7, :] = torch.tensor([2.0 ** -140])
    values, e = ref.quantise(x)
    assert e[3] == 0 and e[5] == 0 and e[6] == 1 and e[7] == -126
    scale = torch.ldexp(torch.ones(200, dtype=torch.float64), e)[:, None]
    cast = (x.double() / scale).clamp(-448, 448).float().to(torch.float8_e4m3fn).double() * scale
    assert torch.equal(values.nan_to_num(1e9), cast.nan_to_num(1e9))
    assert torch.isnan(values[4, 7]) and values[4, 5] == 448 * scale[4] and values[4, 6] == -448 * scale[4]
    finite = torch.isfinite(x)
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, 2.0 ** -10 * scale.expand_as(x))
    assert ((values - x.double()).abs()[finite] <= bound[finite]).all()


def test_the_two_forms_of_the_reference_attention_agree():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(s, generator=g) for s in ((5, 6, 32), (12, 2, 32), (12, 2, 32)))
    a, ta = ref.attention(q, k, v, 7, 0.3, torch.float16)
    b, tb = ref.attention_fast(q, k, v, 7, 0.3, torch.float16)
    assert torch.allclose(a, b, atol=1e-12) and torch.allclose(ta, tb, rtol=1e-9)
