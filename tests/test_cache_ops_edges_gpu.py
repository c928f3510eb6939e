"""The cache operators at the edges of their types and arguments, on the GPU."""
import gc
import math

import pytest
import torch

import cache_reference as ref
from test_cache_ops_gpu import Case
from distserve_amd import paged_attention, plan_prompt, plan_step, prompt_attention, read_kv, write_kv

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module", autouse=True)
def _memory_goes_back():
    """Large allocations are not left cached: later tests count on small ones of their own."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def say(*what):
    print(*what, flush=True)


# first tokens, new tokens: one piece of the kernel for few rows, several that are joined, and the same of the one for many
STEPS = {"row": (299, 1), "rows-joined": (5000, 2), "tile": (260, 40), "tiles-joined": (6000, 130)}


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("fmt", ["plain", "e4m3"])
@pytest.mark.parametrize("every", [16, 1 << 30])
def test_values_at_fp16s_largest_stay_numbers(step, fmt, d, every):
    """Every value is fp16's largest, so every mean of them is.  The weights (1 for the first of every so many keys, just
    above the middle of two fp16 numbers for the others) round up by nearly 2^-11 of themselves, and a mean that is
    past 65520 by that would round to an infinity."""
    say("largest", step, fmt, d, every)
    first, new = STEPS[step]
    n, block = first + new, 16
    pages = -(-n // block)
    weight = 0.5 + 1.05 * 2.0 ** -12
    shape = (pages, 1, 1, block, d)
    if fmt == "plain":
        kc, vc = (torch.zeros(shape, dtype=torch.float16) for _ in range(2))
        kc[..., 0] = -1.0
        kc[0::max(1, every // 16), 0, 0, 0, 0] = 0.0
        vc[..., ::2], vc[..., 1::2] = 65504.0, -65504.0
    else:
        kc, vc = (torch.zeros(*shape[:-1], d + 1, dtype=torch.uint8) for _ in range(2))
        flat_k, flat_v = (x.view(pages, block * (d + 1)) for x in (kc, vc))
        flat_k[:, 0:block * d:d] = 0xb8                   # -1
        flat_k[0::max(1, every // 16), 0] = 0
        flat_k[:, block * d:] = 127
        flat_v[:, 0:block * d:2], flat_v[:, 1:block * d:2] = 0x7e, 0xfe      # 448 * 2^8, held as 65504
        flat_v[:, block * d:] = 127 + 8
    kc, vc = kc.cuda(), vc.cuda()
    plan = plan_step(kc, [new], [first], [list(range(pages))], 1, torch.float16)
    q = torch.zeros(new, 1, d, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    out = paged_attention(plan, 0, q, kc, vc, scale=-math.log(weight)).cpu().double()
    # weights off by 2^-11 of themselves at most, and one rounding of the result
    assert (out[..., ::2] - 65504.0).abs().max() <= 2 * 2.0 ** -11 * 65504.0
    assert (out[..., 1::2] + 65504.0).abs().max() <= 2 * 2.0 ** -11 * 65504.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantising_the_smallest_numbers(dtype):
    """Rows whose scale is 2^-126 or near it: codes times the scale are subnormal numbers of 32 bits."""
    say("smallest", dtype)
    d = 64
    g = torch.Generator().manual_seed(3)
    x = torch.empty(32, 1, d)
    for i in range(32):                                  # largest magnitudes of about 2^-114 - i
        x[i] = torch.randn(d, generator=g) * 2.0 ** (-114 - i)
    x[30, 0] = torch.arange(64) * 2.0 ** -136            # multiples of half the smallest code's value
    x[31, 0] = torch.arange(64) * 2.0 ** -133
    x = x.to(dtype)
    kc, vc = (torch.zeros(2, 1, 1, 16, d + 1, dtype=torch.uint8, device="cuda") for _ in range(2))
    plan = plan_step(kc, [32], [0], [[1, 0]], 1, dtype)
    write_kv(plan, 0, x.cuda(), x.cuda(), kc, vc)
    k, v = read_kv(plan, 0, kc, vc)
    want, e = ref.quantise(x)
    assert e.min() == -126
    for got in (k, v):
        bad = (got.cpu().double() != want.to(dtype).double()).view(32, d)
        assert not bad.any(), [(i, x[i, 0][bad[i]][:3].tolist(), got.cpu()[i, 0][bad[i]][:3].tolist()) for i in range(32) if bad[i].any()]


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_scale_of_zero_or_next_to_it_over_large_scores(dtype, new):
    """Scores of +-1.6e37: nothing of them is left under a scale of 0 or of 2^-149."""
    d, first = 16, 300
    n = first + new
    k = torch.full((n, 1, d), 1e18, dtype=dtype)
    k[::2] = -1e18
    v = torch.zeros(n, 1, d, dtype=dtype)
    v[::2] = 1.0
    q = torch.full((new, 1, d), 1e18, dtype=dtype)
    kc, vc = (torch.zeros(-(-n // 16), 1, 1, 16, d, dtype=dtype, device="cuda") for _ in range(2))
    table = [list(range(kc.shape[0]))]
    whole = plan_step(kc, [n], [0], table, 1)
    write_kv(whole, 0, k.cuda(), v.cuda(), kc, vc)
    plan = plan_step(kc, [new], [first], table, 1)
    for scale in (0.0, 2.0 ** -149, -2.0 ** -149):
        say("scale", dtype, new, scale)
        out = paged_attention(plan, 0, q.cuda(), kc, vc, scale=scale)
        want, tol = ref.attention(q, k, v, first, scale, dtype)
        assert ((out.cpu().double() - want).abs() <= tol).all(), scale


@pytest.mark.parametrize("through", ["functions", "ops"])
def test_writes_raise_the_versions_of_what_they_write(through):
    """A backward pass that kept a pool or an output from before the call is refused, not wrong."""
    ops = torch.ops.kvcache_ops
    pools = [torch.zeros(2, 1, 2, 16, 64, device="cuda") for _ in range(2)]
    row, q = torch.ones(3, 2, 64, device="cuda"), torch.ones(3, 4, 64, device="cuda")
    out = torch.zeros_like(q)
    plan, prompt = plan_step(pools[0], [3], [0], [[1]], 4), plan_prompt([3], 4, 2, 64, torch.float32)
    w = torch.ones((), device="cuda", requires_grad=True)
    kept = [(w * t).sum() for t in (*pools, out)]
    with torch.no_grad():
        if through == "functions":
            write_kv(plan, 0, row, row, *pools)
            assert paged_attention(plan, 0, q, *pools, out=out) is not None
            versions = [t._version for t in (row, q, out, *pools)]
            prompt_attention(prompt, q, row, row, out=out)
        else:
            ops.write_kv(plan, 0, row, row, *pools)
            ops.paged_attention(plan, 0, q, *pools, None, out)
            versions = [t._version for t in (row, q, out, *pools)]
            ops.prompt_attention(prompt, q, row, row, None, out)
    assert versions[:2] == [0, 0] and [t._version for t in (row, q, out, *pools)] == [0, 0, versions[2] + 1, *versions[3:]]
    for y in kept:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():                           # tensors without a version stay usable, inside and out
        made = [torch.zeros_like(p) for p in pools]
        write_kv(plan, 0, row, row, *made)
    write_kv(plan, 0, row, row, *made)
    assert torch.equal(paged_attention(plan, 0, q, *made), q)


def long_step(seqs, seed=0):
    """Pools of random values and a plan of one new token for each of some sequences, in scattered blocks."""
    g = torch.Generator().manual_seed(seed)
    pools = [torch.randn(seqs * 20, 1, 2, 16, 64, generator=g).half().cuda() for _ in range(2)]
    table = torch.randperm(seqs * 20, generator=g).view(seqs, 20).tolist()
    make = lambda: plan_step(pools[0], [1] * seqs, [319 - i % 50 for i in range(seqs)], table, 4)
    q = torch.randn(seqs, 4, 64, generator=g).half().cuda()
    return pools, make, q


def test_plans_are_made_whichever_stream_is_busy():
    """The stream that the plan is for, and torch's pool of 32 once around and more, each busy in its turn."""
    pools, make, q = long_step(8)
    want = paged_attention(make(), 0, q, *pools)
    torch.cuda.synchronize()
    for i in range(41):
        stream = torch.cuda.Stream() if i else torch.cuda.current_stream()
        done = torch.cuda.Event()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(100_000_000)                 # some 40 ms, a plan takes 0.1
        done.record(stream)
        plan = make()
        assert not done.query(), f"the plan waited for stream {i}"
        out = paged_attention(plan, 0, q, *pools)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_plans_made_on_a_busy_stream_are_used_on_others_and_in_graphs():
    """The words are still on their way when the plan is used: on another stream, in a capture, and when it is gone."""
    pools, make, q = long_step(8, 2)
    want = paged_attention(make(), 0, q, *pools)
    others = [long_step(8, 3 + i) for i in range(4)]
    torch.cuda.synchronize()
    for turn in range(6):
        busy, user = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(25_000_000)
            plan = make()
        if turn % 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=user):
                out = paged_attention(plan, 0, q, *pools)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3):
                    graph.replay()
        else:
            with torch.cuda.stream(user):
                out = paged_attention(plan, 0, q, *pools)
                torch.cuda._sleep(100_000_000)
                again = paged_attention(plan, 0, q, *pools)
            del plan
            # plans of the same size, made on the stream whose memory the words are: theirs is not to be given away while a
            # call of another stream is yet to run
            with torch.cuda.stream(busy):
                kept = [m() for _, m, _ in others for _ in range(4)]
            torch.cuda.synchronize()
            assert torch.equal(again, want) and len(kept) == 16
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn


def test_plans_are_made_while_another_thread_captures():
    import threading

    pools, make, q = long_step(8, 1)
    first = make()
    want = paged_attention(first, 0, q, *pools)
    made, errors = [], []

    def plan(turn):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if turn % 2 else torch.cuda.default_stream()):
                made.append(make())
        except Exception as e:                             # told in the assertion below
            errors.append(e)

    for turn in range(40):                                 # the capture streams go round torch's pool
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            thread = threading.Thread(target=plan, args=(turn,))
            thread.start()
            thread.join()
            out = paged_attention(first, 0, q, *pools)
        assert not errors, errors
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(paged_attention(made[-1], 0, q, *pools), want), turn


@pytest.mark.parametrize("ctx_dtype,dec_dtype", [("auto", "e4m3"), ("e4m3", "auto")])
def test_instances_with_pools_of_different_kinds_are_not_bound(ctx_dtype, dec_dtype):
    from distserve_amd import CacheConfig, ContextStageLLMEngine, DecodingStageLLMEngine, ModelConfig, ParallelConfig, cabi

    cabi.reset()
    model = ModelConfig.from_kv_shape(2, 8, 64, 4)
    ctx = ContextStageLLMEngine(model, ParallelConfig(2, 0, 1, 0), CacheConfig(16, 64, cache_dtype=ctx_dtype))
    dec = DecodingStageLLMEngine(model, ParallelConfig(), CacheConfig(16, 64, cache_dtype=dec_dtype))
    ctx._init_kvcache(256, 0)                              # of 65 or 128 bytes a row: either divides the other's pool
    dec._init_kvcache(65, 2)
    with pytest.raises(RuntimeError, match="same cache_dtype"):
        dec.register_kvcache_mem_handles(ctx.parallel_config, ctx.kv_cache_mem_handles)
    cabi.reset()


# ---- chunks and prompts over blocks that are not multiples of 16: the kernel for few rows, two row tiles at a time

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [8, 24])
@pytest.mark.parametrize("hq,h,d", [(8, 2, 64), (4, 4, 96), (8, 1, 128), (4, 2, 256)])
def test_chunks_over_other_block_sizes(dtype, block, hq, h, d):
    say("chunks, blocks of", block, dtype, hq, h, d)
    case = Case(dtype, "plain", hq, h, d, block, [0, 300, 77, 1500, 40], [70, 33, 1, 2, 0], seed=d + block)
    case.check(case.attend(), fast=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [8, 16])
@pytest.mark.parametrize("hq,h,d", [(8, 2, 64), (4, 4, 80), (8, 1, 128), (2, 2, 256)])
def test_prompts_under_a_plan_with_a_pool(dtype, block, hq, h, d):
    """K and V are rows at hand; the plan is the step's, with the pool that they are written to."""
    say("prompts, blocks of", block, dtype, hq, h, d)
    lens = [1, 130, 0, 63, 17]
    case = Case(dtype, "plain", hq, h, d, block, [0] * 5, lens, seed=d)
    k, v = (torch.cat(parts).to(dtype) for parts in case.seqs)
    case.check(prompt_attention(case.plan, case.q.cuda(), k.cuda(), v.cuda()), fast=True)
    case.check(case.attend(), fast=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [15, 16, 17, 24, 32, 33])
@pytest.mark.parametrize("fmt", ["plain", "e4m3"])
def test_both_sides_of_the_border_between_the_kernels(dtype, rows, fmt):
    """16 rows of a KV head (tokens and heads of its group) go to the kernel for few rows, 17 to the one for many."""
    say("border", dtype, rows, fmt)
    for hq, new in {(1, rows), (rows, 1)} | ({(3, rows // 3)} if rows % 3 == 0 else set()):
        case = Case(dtype, fmt, 2 * hq, 2, 64, 16, [200, 0, 1000], [new, new, 1], seed=rows)
        case.check(case.attend(), fast=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_under_every_scale(dtype):
    """A quantised pool's values as its format defines them, rounded to the rows' type once (past fp16's largest: that)."""
    say("codes", dtype)
    d = 256
    pool = torch.zeros(16, 1, 1, 16, d + 1, dtype=torch.uint8)
    flat = pool.view(16, 16 * (d + 1))
    flat[:, :16 * d] = torch.arange(256, dtype=torch.uint8).repeat(16)
    flat[:, 16 * d:] = torch.arange(256, dtype=torch.uint8).view(16, 16)
    want = ref.decode_pool(pool, d).view(256, d)[:255]
    if dtype == torch.float16:
        want = want.clamp(-65504.0, 65504.0)
    want = want.to(dtype)
    plan = plan_step(pool.cuda(), [1], [254], [list(range(16))], 1, dtype)
    for got in read_kv(plan, 0, pool.cuda(), pool.cuda()):
        got = got.cpu().view(255, d)
        bad = ~((got == want) | (got.isnan() & want.isnan()))
        assert not bad.any(), [(s - 127, hex(c), got[s, c].item(), want[s, c].item()) for s, c in bad.nonzero()[:8].tolist()]


def test_a_capture_on_the_stream_that_still_copies_the_plan():
    pools, make, q = long_step(8, 8)
    want = paged_attention(make(), 0, q, *pools)
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(50_000_000)
        plan = make()
        graph.capture_begin()                              # without the wait for the GPU that torch.cuda.graph begins with
        try:
            out = paged_attention(plan, 0, q, *pools)
        finally:
            graph.capture_end()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_plan_is_used_while_the_stream_it_was_made_on_captures_elsewhere():
    """One thread captures on the stream that a plan was made on, in the mode that lets other threads work; another uses that
    plan and makes plans meanwhile."""
    import threading

    pools, make, q = long_step(8, 10)
    want = paged_attention(make(), 0, q, *pools)
    torch.cuda.synchronize()
    for turn in range(4):
        stream, graph, got, errors = torch.cuda.Stream(), torch.cuda.CUDAGraph(), [], []
        with torch.cuda.stream(stream):
            torch.cuda._sleep(25_000_000)
            first, second = make(), make()

        def work():
            try:
                with torch.cuda.stream(torch.cuda.Stream()):
                    got.append(paged_attention(second, 0, q, *pools))
                    got.append(paged_attention(make(), 0, q, *pools))
            except Exception as e:                         # told in the assertion below
                errors.append(e)

        with torch.cuda.stream(stream):
            graph.capture_begin(capture_error_mode="thread_local")
            try:
                thread = threading.Thread(target=work)
                if turn % 2:                               # before the copy has ended, or after the captured call has waited for it
                    thread.start()
                    thread.join()
                out = paged_attention(first, 0, q, *pools)
                if turn % 2 == 0:
                    thread.start()
                    thread.join()
            finally:
                graph.capture_end()
        assert not errors, errors
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and len(got) == 2 and all(torch.equal(g, want) for g in got), turn


def test_plans_made_in_inference_mode_are_used_outside_of_it():
    pools, make, q = long_step(4, 9)
    want = paged_attention(make(), 0, q, *pools)
    with torch.inference_mode():
        plan = make()
        inside = paged_attention(plan, 0, q, *pools)
    with torch.cuda.stream(torch.cuda.Stream()):
        outside = paged_attention(plan, 0, q, *pools)
    torch.cuda.synchronize()
    assert torch.equal(inside, want) and torch.equal(outside, want)


def test_graphs_keep_the_words_of_the_plans_they_were_captured_with():
    """A plan dropped after the capture: its words stay as long as the graph does, and no longer."""
    pools, make, q = long_step(8, 7)
    want = paged_attention(make(), 0, q, *pools)
    gc.collect()
    torch.cuda.synchronize()
    make()                                                 # (whatever earlier graphs let go is given back)
    start = torch.cuda.memory_allocated()
    plan = make()
    size = torch.cuda.memory_allocated() - start
    assert size > 0
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            outs.append([paged_attention(plan, 0, q, *pools) for _ in range(2)])
    held = torch.cuda.memory_allocated()
    del plan
    gc.collect()
    assert torch.cuda.memory_allocated() == held           # nothing below replays if this does not hold
    junk = [torch.full((size // 4,), -1, dtype=torch.int32, device="cuda") for _ in range(16)]
    for turn in range(3):
        for i in range(2):
            for out in outs[i]:
                out.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out, want) for out in outs[i]), turn
            assert torch.equal(paged_attention(make(), 0, q, *pools), want)
    del junk
    graphs.pop()
    gc.collect()
    make()
    graphs[0].replay()                                     # the other graph's are still there
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs[0])
    before = torch.cuda.memory_allocated()
    del graph
    graphs.clear()
    gc.collect()
    make()
    assert torch.cuda.memory_allocated() <= before - size   # (a graph has a little of its own)
