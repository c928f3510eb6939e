"""What the cache operators' entry points make of arguments at the edge of what they take, without a GPU."""
import ctypes
import math

import pytest
import torch

from distserve_amd import cabi

NO_GPU = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="the addresses are made up: only for a machine where nothing can be launched")

K, V, Q, O, S, W, X = (i << 24 for i in range(1, 8))       # made-up addresses, 16 MiB apart
POOL = 4 * 2 * 2 * 16 * 64 * 2


def a_step(new=3, first=0, **kwargs):
    args = dict(num_blocks=4, block_size=16, num_heads=8, num_kv_heads=2, head_dim=64, dtype=cabi.KVM_F16)
    args.update(kwargs)
    step, words = cabi.plan_step([first], [new], [list(range(-(-(first + new) // args["block_size"])))], **args)
    step.device = 0                                        # the caller vouches for extents: no question to the runtime
    return step


def pools(**change):
    args = dict(k=K, v=V, num_blocks=4, num_layers=2, layer=0, num_kv_heads=2, block_size=16, head_dim=64,
                dtype=cabi.KVM_F16, format=cabi.KVM_CACHE_PLAIN, extent=POOL)
    args.update(change)
    return cabi.KvmCache(**args)


def rows(at, token, head=64, extent=1 << 20):
    return cabi.KvmRows(at, token, head, extent)


def refused(code, text, call, *args):
    with pytest.raises(cabi.KvmError, match=text) as e:
        call(*args)
    assert e.value.code == code, e.value


@NO_GPU
def test_scales_that_are_no_number_in_powers_of_two_are_refused():
    step = a_step()
    q, k, v, out = rows(Q, 512), rows(S, 128), rows(S + 4096, 128), rows(O, 512)
    for scale in (3.0e38, -3.0e38, math.inf, math.nan):
        refused(cabi.KVM_EINVAL, "scale", cabi.paged_attention, step, W, pools(), q, out, scale)
        refused(cabi.KVM_EINVAL, "scale", cabi.prompt_attention, step, W, q, k, v, out, scale)


@NO_GPU
def test_sizes_whose_product_passes_64_bits_are_refused():
    step = a_step()
    q, k, v, out = rows(Q, 512), rows(S, 128), rows(S + 4096, 128), rows(O, 512)
    for layers, layer in ((1 << 52, 1 << 50), (1 << 62, 3), ((1 << 63) - 1, 1 << 61), (1 << 50, 0)):
        bad = pools(num_layers=layers, layer=layer, extent=(1 << 63) - 1)
        refused(cabi.KVM_ERANGE, "pool", cabi.write_kv, step, W, bad, k, v)
        refused(cabi.KVM_ERANGE, "pool", cabi.read_kv, step, W, bad, rows(O, 128), rows(O + 4096, 128))
        refused(cabi.KVM_ERANGE, "pool", cabi.paged_attention, step, W, bad, q, out, 1.0)
    # strides that are multiples of 2^64 bytes
    for stride in (1 << 62, 3 << 61, (1 << 63) - 8):
        refused(cabi.KVM_ERANGE, "too large", cabi.write_kv, step, W, pools(), rows(S, stride), v)
        refused(cabi.KVM_ERANGE, "too large", cabi.write_kv, step, W, pools(), k, rows(S, 128, stride))


@NO_GPU
def test_outputs_on_the_workspace_or_the_plan_are_refused():
    step = a_step(1, 16 * 200, num_blocks=256)             # a long sequence: its keys are cut into pieces
    need = cabi.attention_workspace(step)
    assert need > 0
    pool = dict(num_blocks=256, extent=64 * POOL)
    words = step.words * 4
    at = X + (1 << 24)                                     # workspace
    q, out = rows(Q, 512), rows(O, 512)
    for where in (at, at + need - 16, at - 16):
        refused(cabi.KVM_EINVAL, "share memory", cabi.paged_attention, step, W, pools(**pool), q, rows(where, 512), 1.0, at, need)
        refused(cabi.KVM_EINVAL, "share memory", cabi.paged_attention, step, W, pools(**pool), rows(where, 512), out, 1.0, at, need)
    for where in (W - 16, W, W + words - 4 & ~15):
        refused(cabi.KVM_EINVAL, "share memory", cabi.paged_attention, step, W, pools(**pool), q, rows(where, 512), 1.0, at, need)
        refused(cabi.KVM_EINVAL, "share memory", cabi.paged_attention, step, W, pools(**pool), q, out, 1.0, where, need)
    # the workspace on the pools
    for where in (K, K + 64 * POOL - 16, V - 16):
        refused(cabi.KVM_EINVAL, "share memory", cabi.paged_attention, step, W, pools(**pool), q, out, 1.0, where, need)
    prompt = a_step(2000, num_blocks=256, num_kv_heads=8, dtype=cabi.KVM_F32)
    need = cabi.attention_workspace(prompt)
    assert need > 0
    far = 1 << 40                                          # rows of 512 * 4 bytes, apart from each other
    q, k, v, out = (cabi.KvmRows(far + (i << 28), 512, 64, 1 << 28) for i in range(4))
    for where in (k.ptr, v.ptr + 4096, q.ptr + 2000 * 2048 - 16):
        refused(cabi.KVM_EINVAL, "share memory", cabi.prompt_attention, prompt, W, q, k, v, out, 1.0, where, need)
    refused(cabi.KVM_EINVAL, "share memory", cabi.prompt_attention, prompt, W, q, k, v, rows(W, 512, 64, 1 << 28), 1.0, far >> 1, need)
    step = a_step()
    refused(cabi.KVM_EINVAL, "share memory", cabi.write_kv, step, K + 4096, pools(), rows(S, 128), rows(S + 4096, 128))
    refused(cabi.KVM_EINVAL, "share memory", cabi.read_kv, step, W, pools(), rows(W, 128), rows(O, 128))
    refused(cabi.KVM_EINVAL, "share memory", cabi.read_kv, step, W, pools(), rows(O, 128), rows(W, 128))


def test_tensors_with_gradients_are_refused_wherever_they_stand():
    """Rows, outputs and pools that require a gradient, and any of them with a forward-mode tangent."""
    import distserve_amd
    from torch.autograd import forward_ad

    plan = distserve_amd.StepPlan([0], [3], [1], [1], 4, 16, 4, 2, 64, 5, False, -1)      # a plan to look at, without a GPU
    pool = torch.zeros(4, 1, 2, 16, 64, dtype=torch.float16)
    row, q = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, 4, 64, dtype=torch.float16)
    calls = [
        (lambda *t: distserve_amd.write_kv(plan, 0, *t), [row, row, pool, pool]),
        (lambda *t: distserve_amd.read_kv(plan, 0, *t), [pool, pool]),
        (lambda *t: distserve_amd.paged_attention(plan, 0, *t[:3], out=t[3]), [q, pool, pool, q]),
        (lambda *t: distserve_amd.prompt_attention(plan, *t[:3], out=t[3]), [q, row, row, q]),
    ]
    ops = torch.ops.kvcache_ops
    calls += [
        (lambda *t: ops.write_kv(plan, 0, *t), [row, row, pool, pool]),
        (lambda *t: ops.paged_attention(plan, 0, *t[:3], None, t[3]), [q, pool, pool, q]),
    ]
    for call, tensors in calls:
        for i in range(len(tensors)):
            wanted = [t.clone().requires_grad_() if i == j else t for j, t in enumerate(tensors)]
            with pytest.raises(RuntimeError, match="no gradient"):
                call(*wanted)
            with torch.no_grad(), pytest.raises(RuntimeError, match="without a GPU"):       # as far as a machine without one gets
                call(*wanted)
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(tensors)]
                with pytest.raises(RuntimeError, match="no gradient"):
                    call(*dual)


@pytest.mark.parametrize("name", ["paged_attention", "prompt_attention"])
@pytest.mark.parametrize("space", ["kvcache_ops", "kvmove_kvcache_ops"])
def test_the_attention_ops_schemas_say_that_out_is_written_and_returned(space, name):
    import os

    import distserve_amd

    if space != "kvcache_ops":
        torch.ops.load_library(os.path.join(os.path.dirname(distserve_amd.TORCH_LIB_PATH), "libkvmove_torch_alt.so"))
    schema = getattr(getattr(torch.ops, space), name).default._schema
    out = schema.arguments[-1]
    assert out.name == "out" and out.default_value is None and schema.is_mutable
    assert out.alias_info is not None and out.alias_info.is_write
    back = schema.returns[0].alias_info
    assert back is not None and back.is_write and back.after_set == out.alias_info.before_set
    assert [a.name for a in schema.arguments if a.alias_info is not None] == ["out"]


@pytest.mark.parametrize("block", [16, 32, 8, 24, 1])
@pytest.mark.parametrize("dtype", [cabi.KVM_F16, cabi.KVM_BF16, cabi.KVM_F32])
def test_which_kernel_a_sequences_rows_go_to(dtype, block):
    """More than 16 rows of 16 bits for a KV head go to the kernel for many rows, where blocks are whole sixteens; all
    others to the one for few, two row tiles at a time if one of them has more than 16 and head_dim is 128 at most.
    Either way every row's keys are covered once, from the first to its own."""
    for heads, kv_heads, head_dim in ((1, 1, 64), (8, 8, 128), (12, 3, 64), (17, 1, 128), (16, 2, 256), (48, 2, 80)):
        group = heads // kv_heads
        news = sorted({n for rows in (1, 15, 16, 17, 23, 24, 31, 32, 33, 48, 129) for n in (rows // group, -(-rows // group)) if n})
        for new in ([n] for n in news):
            new = new + [1, 0, 2]
            first = [100, 0, 7, 3000]
            pages = [-(-(a + b) // block) for a, b in zip(first, new)]
            at, table = 0, []
            for p in pages:
                table.append(list(range(at, at + p)))
                at += p
            step, words = cabi.plan_step(first, new, table, at + 1, block, heads, kv_heads, head_dim, dtype)
            many = [dtype != cabi.KVM_F32 and n * group > 16 and block % 16 == 0 for n in new]
            few_rows = [n * group for n, m in zip(new, many) if not m]
            assert step.row_tiles == (2 if max(few_rows, default=0) > 16 and head_dim <= 128 else 1)
            height = 16 * step.row_tiles
            tiles = [tuple(words[step.row_tiles_at + 8 * i:step.row_tiles_at + 8 * i + 8]) for i in range(step.num_row_tiles)]
            items = [tuple(words[step.tile_items_at + 12 * i:step.tile_items_at + 12 * i + 12]) for i in range(step.num_tile_items)]
            want_tiles, starts = [], [sum(new[:s]) for s in range(len(new))]
            for s, n in enumerate(new):
                for r in range(0, 0 if many[s] else n * group, height):
                    end = first[s] + (min(r + height, n * group) - 1) // group + 1
                    want_tiles.append((starts[s], n * group, first[s], sum(pages[:s]), r, end, -(-end // 128)))
            assert [t[:7] for t in tiles] == want_tiles
            for s, n in enumerate(new):
                mine = [i for i in items if i[0] == starts[s] and i[1] == n * group and n]
                if not many[s]:
                    assert not mine
                    continue
                for r in range(0, n * group, 128):
                    for head0 in range(0, kv_heads, 8):
                        cut = sorted((i[5], i[6]) for i in mine if i[4] == r and i[8] == head0)
                        assert cut[0][0] == 0 and all(a[1] == b[0] for a, b in zip(cut, cut[1:]))
                        assert cut[-1][1] == first[s] + (min(r + 128, n * group) - 1) // group + 1
