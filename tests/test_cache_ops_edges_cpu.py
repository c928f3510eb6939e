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
