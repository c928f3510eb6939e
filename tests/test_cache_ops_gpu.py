"""The cache operators against their definition in 64 bits (cache_reference), on the GPU."""
import gc
import math
import random

import pytest
import torch

import cache_reference as ref
from distserve_amd import (cabi, paged_attention, plan_prompt, plan_step, prompt_attention, quantized_pool_shape, read_kv,
                           write_kv)

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
CANARY = 0x5B


@pytest.fixture(scope="module", autouse=True)
def _memory_goes_back():
    """Large allocations are not left cached: later tests count on small ones of their own."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def say(*what):
    print(*what, flush=True)


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def tables_for(lens, block, seed, spare=3):
    """Scattered block tables for sequences of these lengths, and the pool's block count."""
    pages = [-(-n // block) for n in lens]
    order = list(range(sum(pages) + spare))
    random.Random(seed).shuffle(order)
    out, at = [], 0
    for p in pages:
        out.append(order[at:at + p])
        at += p
    return out, len(order)


class Case:
    """Pools filled with random K and V for some sequences; what lies in no sequence's tokens is NaN
    (plain pools) or the NaN code under a NaN scale (quantised ones)."""

    def __init__(self, dtype, fmt, hq, h, d, block, first, new, layers=2, layer=1, seed=0):
        self.dtype, self.fmt, self.hq, self.h, self.d, self.block = dtype, fmt, hq, h, d, block
        self.first, self.new, self.layer = first, new, layer
        lens = [a + b for a, b in zip(first, new)]
        self.table, blocks = tables_for(lens, block, seed)
        self.tokens = sum(new)
        self.q = rand((self.tokens, hq, d), dtype, seed + 1)
        k, v = (rand((sum(lens), h, d), dtype, seed + 2 + i) for i in range(2))
        shape = (blocks, layers, h, block, d)
        pools, self.seqs = [], [[], []]
        for which, x in enumerate((k, v)):
            if fmt == "plain":
                pool = torch.full(shape, math.nan, dtype=dtype)
            else:
                pool = torch.full(quantized_pool_shape(shape), 255, dtype=torch.uint8)
                flat = pool.view(blocks, layers, h, block * (d + 1))
                x, e = ref.quantise(x)
                codes = (x / torch.pow(2.0, e.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
            at = 0
            for table, n in zip(self.table, lens):
                for j in range(n):
                    p, off = table[j // block], j % block
                    if fmt == "plain":
                        pool[p, layer, :, off] = x[at + j]
                    else:
                        flat[p, layer, :, off * d:(off + 1) * d] = codes[at + j]
                        flat[p, layer, :, block * d + off] = (e[at + j] + 127).to(torch.uint8)
                self.seqs[which].append(x[at:at + n])
                at += n
            pools.append(pool)
        self.k_cache, self.v_cache = (p.cuda() for p in pools)
        self.plan = plan_step(self.k_cache, new, first, self.table, hq, dtype)

    def attend(self, **kw):
        return paged_attention(self.plan, self.layer, self.q.cuda(), self.k_cache, self.v_cache, **kw)

    def check(self, out, scale=None, fast=False):
        scale = self.d ** -0.5 if scale is None else scale
        at = 0
        for s, n in enumerate(self.new):
            want, tol = (ref.attention_fast if fast else ref.attention)(
                self.q[at:at + n], self.seqs[0][s], self.seqs[1][s], self.first[s], scale, self.dtype)
            got = out[at:at + n].cpu().double()
            worst = ((got - want).abs() / tol).max().item() if n else 0.0
            assert not torch.isnan(got).any() and worst <= 1.0, f"sequence {s}: {worst} times the allowed error"
            at += n


# ---- write and read back

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [16, 64, 80, 128, 240, 256])
@pytest.mark.parametrize("fmt", ["plain", "e4m3"])
def test_write_fills_the_named_slots_and_no_others(dtype, d, fmt):
    say("write", dtype, d, fmt)
    h, block, layers, layer = 3, 16, 3, 1
    first, new = [0, 15, 33, 7, 0], [17, 2, 0, 1, 16]
    table, blocks = tables_for([a + b for a, b in zip(first, new)], block, d)
    shape = (blocks, layers, h, block, d)
    if fmt == "e4m3":
        shape, pool_type = quantized_pool_shape(shape), torch.uint8
    else:
        pool_type = dtype
    n = sum(new)
    # K and V are slices of a fused projection: strides that are not the heads' own
    fused = rand((n + 2, 5 * h, d), dtype, d, 30.0).cuda()
    k, v = fused[:, h:2 * h], fused[:, 3 * h:4 * h]
    size = math.prod(shape) * torch.empty((), dtype=pool_type).element_size()
    bytes_k, bytes_v = (torch.full((size + 8192,), CANARY, dtype=torch.uint8, device="cuda") for _ in range(2))
    k_cache, v_cache = (b[4096:-4096].view(pool_type).view(shape) for b in (bytes_k, bytes_v))
    plan = plan_step(k_cache, new, first, table, h, dtype)
    write_kv(plan, layer, k, v, k_cache, v_cache)
    torch.cuda.synchronize()
    for x, whole in ((k, bytes_k), (v, bytes_v)):
        want = torch.full((size,), CANARY, dtype=torch.uint8)
        pool = want.view(pool_type).view(shape)
        if fmt == "e4m3":
            values, e = ref.quantise(x[:n].cpu())
            codes = (values / torch.pow(2.0, e.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
            flat = pool.view(blocks, layers, h, block * (d + 1))
        at = 0
        for s in range(len(new)):
            for i in range(new[s]):
                j = first[s] + i
                p, off = table[s][j // block], j % block
                if fmt == "plain":
                    pool[p, layer, :, off] = x[at].cpu()
                else:
                    flat[p, layer, :, off * d:(off + 1) * d] = codes[at]
                    flat[p, layer, :, block * d + off] = (e[at] + 127).to(torch.uint8)
                at += 1
        got = whole.cpu()
        assert (got[:4096] == CANARY).all() and (got[-4096:] == CANARY).all()
        assert torch.equal(got[4096:-4096], want)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantising_at_the_borders(dtype):
    """Ties, rows at the scale's borders, zeros, the type's largest and smallest, infinities and NaN."""
    say("borders", dtype)
    d, block = 64, 16
    info = torch.finfo(dtype)
    x = rand((32, 1, d), dtype, 5)
    x[0] = 0.0
    x[1, 0, 3], x[1, 0, 4], x[1, 0, 5] = math.inf, -math.inf, math.nan
    x[2] = math.nan
    x[3] = math.inf
    x[4] = info.max
    x[5] = -info.max
    x[6] = info.smallest_normal * info.eps                       # the type's smallest
    x[7, 0, 0] = info.max
    x[8] = 448.0
    x[9] = 450.0
    x[10] = torch.arange(64).to(dtype) * 0.0625 + 16              # ties of the grid at 16 .. 32
    x[11] = -0.0
    x[12, 0] = torch.tensor([2.0 ** -i for i in range(24)] + [0.0] * 40).to(dtype)
    x[13, 0] = torch.tensor([1.5 * 2.0 ** -i for i in range(24)] + [448.0] * 40).to(dtype)
    pool = torch.zeros((2, 1, 1, block, d + 1), dtype=torch.uint8, device="cuda")
    k_cache, v_cache = pool, pool.clone()
    plan = plan_step(k_cache, [32], [0], [[1, 0]], 1, dtype)
    write_kv(plan, 0, x.cuda(), x.cuda(), k_cache, v_cache)
    k, v = read_kv(plan, 0, k_cache, v_cache)
    want, _ = ref.quantise(x)
    if dtype == torch.float16:
        want = want.clamp(-65504.0, 65504.0)
    for got in (k, v):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0), want.to(dtype).double().nan_to_num(7.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,h,block", [(64, 12, 16), (128, 8, 32), (80, 5, 48), (256, 1, 16)])
@pytest.mark.parametrize("fmt", ["plain", "e4m3"])
def test_read_back_packs_the_sequences(dtype, d, h, block, fmt):
    say("read", dtype, d, h, block, fmt)
    case = Case(dtype, fmt, h, h, d, block, [0, 40, 3, 0, 95], [5, 0, 1, 16, 2], seed=d)
    k, v = read_kv(case.plan, case.layer, case.k_cache, case.v_cache)
    for got, parts in ((k, case.seqs[0]), (v, case.seqs[1])):
        assert torch.equal(got.cpu().double(), torch.cat(parts).to(dtype).double())


def test_plain_pools_take_any_block_size():
    for block in (1, 3, 8, 17, 128):
        say("block", block)
        case = Case(torch.float16, "plain", 4, 2, 32, block, [0, 40, 2], [5, 1, 33], seed=block)
        k, _ = read_kv(case.plan, case.layer, case.k_cache, case.v_cache)
        assert torch.equal(k.cpu(), torch.cat(case.seqs[0]))
        case.check(case.attend())


# ---- attention over the cache

SHAPES = [  # hq, h, d, block
    (12, 12, 64, 16), (8, 1, 128, 16), (32, 4, 128, 32), (4, 4, 80, 16), (14, 2, 96, 48), (2, 2, 256, 16), (16, 2, 16, 16),
    (71, 1, 64, 16), (10, 2, 240, 16),
]
BATCHES = {
    "one": ([0], [1]),
    "tokens": ([0, 1, 15, 16, 17, 31, 130, 257, 600], [1] * 9),
    "ragged": ([0, 300, 5, 0, 31, 64], [3, 1, 0, 40, 2, 5]),
    "long": ([3000, 10], [2, 1]),
}


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("hq,h,d,block", SHAPES)
@pytest.mark.parametrize("fmt", ["plain", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
def test_paged_attention(dtype, fmt, hq, h, d, block, batch):
    say("paged", dtype, fmt, hq, h, d, block, batch)
    first, new = BATCHES[batch]
    case = Case(dtype, fmt, hq, h, d, block, first, new, seed=hq + d)
    case.check(case.attend(), fast=True)


@pytest.mark.parametrize("fmt", ["plain", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,h,d", [(8, 2, 128), (3, 3, 64), (4, 1, 256)])
def test_paged_attention_of_chunks(dtype, fmt, hq, h, d):
    say("chunk", dtype, fmt, hq, h, d)
    case = Case(dtype, fmt, hq, h, d, 16, [0, 700, 129, 64], [200, 333, 1, 64], seed=d)
    case.check(case.attend(), fast=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,h,d", [(12, 12, 64), (16, 2, 128), (4, 4, 80), (2, 1, 256), (5, 1, 112)])
def test_prompt_attention(dtype, hq, h, d):
    lens = [1, 130, 0, 63, 257, 2, 64]
    say("prompt", dtype, hq, h, d)
    q, k, v = (rand((sum(lens), n, d), dtype, i + d) for i, n in enumerate((hq, h, h)))
    plan = plan_prompt(lens, hq, h, d, dtype)
    out = prompt_attention(plan, q.cuda(), k.cuda(), v.cuda()).cpu().double()
    at = 0
    for n in lens:
        want, tol = ref.attention_fast(q[at:at + n], k[at:at + n], v[at:at + n], 0, d ** -0.5, dtype)
        assert ((out[at:at + n] - want).abs() <= tol).all(), n
        at += n


def test_large_and_odd_scores():
    """Scores that would overflow without the running maximum, a scale of zero and a negative one."""
    for scale in (30.0, 0.0, -0.7):
        for dtype in TYPES:
            say("scale", scale, dtype)
            case = Case(dtype, "plain", 4, 2, 64, 16, [100, 0], [3, 40], seed=3)
            case.check(case.attend(scale=scale), scale=scale)


# ---- what must not reach a result

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("hq,h,d,new", [(4, 4, 64, 20), (8, 1, 128, 5), (2, 2, 128, 200), (2, 1, 256, 40)])
def test_later_tokens_do_not_reach_earlier_rows(dtype, value, hq, h, d, new):
    """An infinity or NaN in one new token's K and V: rows before it come out as if it were not there,
    rows from it on as the formula says.  (As everywhere, within the error that cache_reference derives: a
    workgroup that meets such a value takes another order of sums than one that does not, and each of
    the two is that close to the definition.)"""
    say("later", dtype, value, hq, h, d, new)
    first = 37
    case = Case(dtype, "plain", hq, h, d, 16, [first], [new], seed=9)
    case.check(case.attend(), fast=True)
    want, tol = ref.attention_fast(case.q, case.seqs[0][0], case.seqs[1][0], first, d ** -0.5, dtype)

    def close(got, rows, cols=slice(None)):
        return ((got.cpu().double()[rows] - want[rows]).abs() <= tol[rows])[:, :, cols].all()

    at = first + new // 2
    spots = {at: slice(3, 5), at + 2: slice(0, 1)} if new > 6 else {at: slice(0, 2)}
    for j, cols in spots.items():
        p, off = case.table[0][j // 16], j % 16
        case.v_cache[p, case.layer, :, off, cols] = value
    out = case.attend()
    rows = new // 2
    assert close(out, slice(0, rows))
    after = out[rows:].cpu()
    assert not torch.isfinite(after[:, :, spots[at]]).any()
    # columns that hold no such value stay what they were
    untouched = torch.ones(d, dtype=torch.bool)
    for cols in spots.values():
        untouched[cols] = False
    assert close(out, slice(rows, None), untouched)
    for j in spots:
        p, off = case.table[0][j // 16], j % 16
        case.v_cache[p, case.layer, :, off] = 1.0
        case.k_cache[p, case.layer, :, off] = math.nan
    out = case.attend()
    assert close(out, slice(0, rows)) and torch.isnan(out[rows:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [33, 200])
def test_prompts_keep_later_infinities_out_of_earlier_rows(dtype, new):
    say("prompt later", dtype, new)
    q, k, v = (rand((new + 7, 2, 64), dtype, i) for i in range(3))
    plan = plan_prompt([new, 7], 2, 2, 64, dtype)
    parts = [ref.attention_fast(q[a:b], k[a:b], v[a:b], 0, 64 ** -0.5, dtype) for a, b in ((0, new), (new, new + 7))]
    want, tol = (torch.cat([p[i] for p in parts]) for i in range(2))
    v[new - 2, :, 5] = math.inf
    out = prompt_attention(plan, q.cuda(), k.cuda(), v.cuda())
    good = (out.cpu().double() - want).abs() <= tol
    assert good[:new - 2].all() and good[new:].all() and good[new - 2:new, :, :5].all() and good[new - 2:new, :, 6:].all()
    assert not torch.isfinite(out[new - 2:new, :, 5]).any()


def test_a_quantised_nan_reaches_only_the_rows_that_see_it():
    case = Case(torch.float16, "e4m3", 4, 2, 64, 16, [20], [10], seed=4)
    want, tol = ref.attention(case.q, case.seqs[0][0], case.seqs[1][0], 20, 64 ** -0.5, torch.float16)
    p, off = case.table[0][25 // 16], 25 % 16
    flat = case.v_cache.view(*case.v_cache.shape[:3], 16 * 65)
    flat[p, case.layer, :, off * 64 + 7] = 0x7f
    out = case.attend()
    assert ((out.cpu().double() - want).abs() <= tol)[:5].all()
    assert torch.isnan(out[5:, :, 7]).all() and not torch.isnan(out[5:, :, :7]).any()


# ---- how a program calls them

@pytest.mark.parametrize("new", [3, 64])
def test_codes_past_fp16_beside_a_nan_are_the_largest_number(new):
    """Keys 0..5 hold 448 * 2^8 in V's column 3, which fp16 does not; the last key holds a NaN in column 5."""
    table, last = [3, 1, 4, 2, 0], 5 + new - 1
    kc = torch.zeros(5, 1, 1, 16, 65, dtype=torch.uint8)
    kc.view(5, 16 * 65)[:, 16 * 64:] = 127                                    # scales of one
    vc = kc.clone()
    for key in range(6):
        vc.view(5, 16 * 65)[table[0], key * 64 + 3] = 0x7e
        vc.view(5, 16 * 65)[table[0], 16 * 64 + key] = 127 + 8
    vc.view(5, 16 * 65)[table[last // 16], last % 16 * 64 + 5] = 0x7f
    kc, vc = kc.cuda(), vc.cuda()
    plan = plan_step(kc, [new], [5], [table], 1)
    got = paged_attention(plan, 0, torch.zeros(new, 1, 64, dtype=torch.float16, device="cuda"), kc, vc).cpu()[:, 0].double()
    want = 65504.0 * 6 / (6 + torch.arange(new, dtype=torch.float64))         # all scores are zero: plain means
    # one rounding to fp16 (half a step, 2^-11), and sums and a quotient in 32 bits
    assert ((got[:, 3] - want).abs() <= want * 2.0**-10).all()
    assert got[:-1].isfinite().all() and got[-1, 5].isnan() and got[-1, :5].isfinite().all()


def test_padded_batches_and_given_outputs_keep_what_lies_behind():
    case = Case(torch.bfloat16, "plain", 8, 2, 128, 16, [50, 0], [1, 30], seed=6)
    n = case.tokens
    wide = torch.full((n + 9, 3, 8, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:n, 1] = case.q.cuda()
    q = wide[:, 1]
    out = torch.full((n + 9, 8, 256), 3.0, dtype=torch.bfloat16, device="cuda")
    got = paged_attention(case.plan, case.layer, q, case.k_cache, case.v_cache, out=out[:, :, 64:192])
    assert got.data_ptr() == out[:, :, 64:192].data_ptr()
    case.check(out[:n, :, 64:192])
    assert (out[n:] == 3.0).all() and (out[:, :, :64] == 3.0).all() and (out[:, :, 192:] == 3.0).all()
    made = paged_attention(case.plan, case.layer, q, case.k_cache, case.v_cache)
    assert torch.equal(made[:n], out[:n, :, 64:192]) and (made[n:] == 0).all()


def test_calls_repeat_bit_for_bit():
    case = Case(torch.float16, "plain", 16, 2, 128, 16, [4000, 100, 0], [1, 300, 5], seed=8)
    outs = [case.attend() for _ in range(4)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_on_another_stream_than_the_plan_was_made_on():
    case = Case(torch.float16, "e4m3", 8, 2, 64, 16, [2000, 3], [1, 40], seed=11)
    want = case.attend()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [case.attend() for _ in range(3)]
    del case.plan                      # its memory must not be reused before the side stream is done
    junk = [torch.full((4096,), -1, dtype=torch.int32, device="cuda") for _ in range(8)]
    side.synchronize()
    assert all(torch.equal(want, o) for o in outs) and len(junk) == 8


def test_captured_graphs_replay_with_what_the_pools_hold():
    """Write and attend in two graphs whose replays alternate on two streams, each with workspace of its own."""
    first, new = [700, 2500], [1, 1]
    cases = [Case(torch.float16, "plain", 8, 2, 64, 16, first, new, seed=20 + i) for i in range(2)]
    held = []
    for case in cases:
        k, v = (rand((2, 2, 64), torch.float16, 40 + i).cuda() for i in range(2))
        q = case.q.cuda()
        for _ in range(2):
            write_kv(case.plan, case.layer, k, v, case.k_cache, case.v_cache)
            paged_attention(case.plan, case.layer, q, case.k_cache, case.v_cache)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            write_kv(case.plan, case.layer, k, v, case.k_cache, case.v_cache)
            out = paged_attention(case.plan, case.layer, q, case.k_cache, case.v_cache)
        held.append((graph, k, v, q, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for case, (graph, k, v, q, out) in zip(cases, held):
            k.copy_(rand((2, 2, 64), torch.float16, 60 + turn))
            q.copy_(rand((2, 8, 64), torch.float16, 80 + turn))
        torch.cuda.synchronize()
        for stream, (graph, *_) in zip(streams, held):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for case, (graph, k, v, q, out) in zip(cases, held):
            replayed = out.clone()
            write_kv(case.plan, case.layer, k, v, case.k_cache, case.v_cache)
            eager = paged_attention(case.plan, case.layer, q, case.k_cache, case.v_cache)
            assert torch.equal(replayed, eager), turn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="before the graph capture"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            plan_step(cases[0].k_cache, new, first, cases[0].table, 8)
    torch.cuda.synchronize()


def test_two_threads_at_once():
    import threading

    cases = [Case(torch.float16, "plain", 8, 8, 64, 16, [900 + i], [1], seed=30 + i) for i in range(2)]
    want = [c.attend() for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                plan = plan_step(cases[i].k_cache, cases[i].new, cases[i].first, cases[i].table, 8)
                out = paged_attention(plan, 1, cases[i].q.cuda(), cases[i].k_cache, cases[i].v_cache)
                if not torch.equal(out, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_offsets_past_32_bits():
    """Pools of more than 4 GiB, used at both ends; few blocks are ever touched."""
    d, h, block, layers = 128, 32, 16, 20
    blocks = 2000                                        # 2.6 MiB a block: 5.2 GB a pool
    shape = (blocks, layers, h, block, d)
    k_cache, v_cache = (torch.empty(shape, dtype=torch.float16, device="cuda") for _ in range(2))
    assert k_cache.numel() * 2 > 1 << 32
    table = [[1999, 0, 1998, 1]]
    n = 60
    k, v, q = (rand((n, h, d), torch.float16, i) for i in range(3))
    plan = plan_step(k_cache, [n], [0], table, h)
    write_kv(plan, layers - 1, k.cuda(), v.cuda(), k_cache, v_cache)
    back = read_kv(plan, layers - 1, k_cache, v_cache)
    assert torch.equal(back[0].cpu(), k) and torch.equal(back[1].cpu(), v)
    out = paged_attention(plan, layers - 1, q.cuda(), k_cache, v_cache).cpu().double()
    want, tol = ref.attention_fast(q, k, v, 0, d ** -0.5, torch.float16)
    assert ((out - want).abs() <= tol).all()


# ---- refusals on GPU tensors (all of them on the host, before any launch)

def test_refusals():
    case = Case(torch.float16, "plain", 4, 2, 64, 16, [20], [3], seed=1)
    q, kc, vc, plan = case.q.cuda(), case.k_cache, case.v_cache, case.plan
    row = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")

    def refused(match, call, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            call(*args, **kw)

    refused("layer 2", paged_attention, plan, 2, q, kc, vc)
    refused("layer -1", write_kv, plan, -1, row, row, kc, vc)
    refused("must be", paged_attention, plan, 1, q[:2], kc, vc)
    refused("must be", paged_attention, plan, 1, q[:, :3], kc, vc)
    refused("plan is for", paged_attention, plan, 1, q.float(), kc, vc)
    refused("plan is for", paged_attention, plan, 1, q, kc.bfloat16(), vc.bfloat16())
    refused("agree", paged_attention, plan, 1, q, kc, vc[:-1])
    refused("the plan is for", paged_attention, plan, 1, q, kc[:-1].contiguous(), vc[:-1].contiguous())
    refused("contiguous", paged_attention, plan, 1, q, kc.transpose(1, 2), vc.transpose(1, 2))
    refused("last stride", paged_attention, plan, 1, torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")[:, :, ::2], kc, vc)
    refused("16 bytes", paged_attention, plan, 1, torch.zeros(3, 4, 68, dtype=torch.float16, device="cuda")[:, :, :64], kc, vc)
    refused("16 bytes", paged_attention, plan, 1, torch.zeros(800, dtype=torch.float16, device="cuda")[4:772].view(3, 4, 64), kc, vc)
    refused("on the GPU|on cpu|on cuda", paged_attention, plan, 1, case.q, kc, vc)
    refused("out is", paged_attention, plan, 1, q, kc, vc, out=row)
    refused("overlap", paged_attention, plan, 1, q, kc, vc, out=row[:1, :1].expand(3, 4, 64))
    refused("finite", paged_attention, plan, 1, q, kc, vc, scale=math.nan)
    refused("earlier tokens", prompt_attention, plan, q, row, row)
    refused("gradient", paged_attention, plan, 1, q.clone().requires_grad_(), kc, vc)
    with torch.no_grad():
        paged_attention(plan, 1, q.clone().requires_grad_(), kc, vc)
    refused("multiple of 16", plan_step, torch.zeros(4, 1, 2, 16, 72, dtype=torch.float16, device="cuda"), [1], [0], [[0]], 2)
    refused("no blocks", plan_step, kc[:0], [1], [0], [[0]], 2)
    coded = torch.zeros(4, 1, 2, 8, 65, dtype=torch.uint8, device="cuda")
    odd = plan_step(coded, [1], [0], [[0]], 2)
    refused("block_size", write_kv, odd, 0, row, row, coded, coded.clone())
    prompt = plan_prompt([3], 4, 2, 64, torch.float16)
    refused("without a cache", paged_attention, prompt, 0, q, kc, vc)
    # K and V may broadcast (a stride of zero); an output may not
    shared = rand((1, 2, 64), torch.float16, 3).cuda().expand(3, 2, 64)
    out = prompt_attention(prompt, q, shared, shared)
    assert torch.equal(out, prompt_attention(prompt, q, shared.contiguous(), shared.contiguous()))


def test_outputs_that_lie_on_inputs_are_refused_and_fused_ones_are_not():
    case = Case(torch.float16, "plain", 4, 2, 64, 16, [20, 300], [3, 40], seed=1)
    kc, vc, plan = case.k_cache, case.v_cache, case.plan
    q = case.q.cuda()
    wide = torch.zeros(43, 12, 64, dtype=torch.float16, device="cuda")           # q, out and others in one row
    wide[:, :4] = q
    side = torch.zeros(43, 4, 2, 64, dtype=torch.float16, device="cuda")         # q and out in turns, head by head
    side[:, :, 0] = q
    row = torch.zeros(43, 2, 64, dtype=torch.float16, device="cuda")
    for rows, out in ((q, q), (wide[:, :4], wide[:, :4]), (wide[:, :4], wide[:, 3:7]), (side[:, :, 0], side[:, :, 0])):
        with pytest.raises(RuntimeError, match="share memory"):
            paged_attention(plan, 1, rows, kc, vc, out=out)
    for call in (lambda: write_kv(plan, 1, row, row, kc, kc), lambda: write_kv(plan, 1, kc.view(-1, 2, 64)[:43], row, kc, vc)):
        with pytest.raises(RuntimeError, match="share memory"):
            call()
    want = paged_attention(plan, 1, q, kc, vc)
    assert torch.equal(paged_attention(plan, 1, wide[:, :4], kc, vc, out=wide[:, 4:8]), want)
    assert torch.equal(paged_attention(plan, 1, side[:, :, 0], kc, vc, out=side[:, :, 1]), want)
    assert torch.equal(wide[:, 4:8], want) and torch.equal(side[:, :, 1], want) and not wide[:, 8:].any()
    assert torch.equal(wide[:, :4], q) and torch.equal(side[:, :, 0], q)


def test_the_c_interface_checks_extents_and_workspaces():
    case = Case(torch.float16, "plain", 2, 2, 64, 16, [3000], [1], seed=1)
    step, words = cabi.plan_step(case.first, case.new, case.table, case.k_cache.shape[0], 16, 2, 2, 64, cabi.KVM_F16)
    dev = torch.tensor(list(words[:step.words]), dtype=torch.int32, device="cuda")
    q = case.q.cuda()
    out = torch.empty_like(q)
    stream = torch.cuda.current_stream().cuda_stream
    need = cabi.attention_workspace(step)
    assert need > 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda")

    def cache(**change):
        args = dict(k=case.k_cache.data_ptr(), v=case.v_cache.data_ptr(), num_blocks=case.k_cache.shape[0], num_layers=2,
                    layer=1, num_kv_heads=2, block_size=16, head_dim=64, dtype=cabi.KVM_F16, format=cabi.KVM_CACHE_PLAIN)
        args.update(change)
        return cabi.KvmCache(**args)

    rows = lambda t: cabi.KvmRows(t.data_ptr(), t.stride(0), t.stride(1))
    cabi.paged_attention(step, dev.data_ptr(), cache(), rows(q), rows(out), 0.125, work.data_ptr(), need, stream)
    assert torch.equal(out, case.attend())
    for code, args in ((cabi.KVM_EINVAL, (cache(), rows(q), rows(out), 0.125, work.data_ptr(), need - 1, stream)),
                       (cabi.KVM_EINVAL, (cache(), rows(q), rows(out), 0.125, 0, 0, stream)),
                       (cabi.KVM_ERANGE, (cache(num_layers=1 << 20), rows(q), rows(out), 0.125, work.data_ptr(), need, stream)),
                       (cabi.KVM_EMISMATCH, (cache(head_dim=128), rows(q), rows(out), 0.125, work.data_ptr(), need, stream)),
                       (cabi.KVM_EMISMATCH, (cache(dtype=cabi.KVM_BF16), rows(q), rows(out), 0.125, work.data_ptr(), need, stream)),
                       (cabi.KVM_EMISMATCH, (cache(format=cabi.KVM_CACHE_E4M3), rows(q), rows(out), 0.125, work.data_ptr(), need, stream)),
                       (cabi.KVM_EINVAL, (cache(k=0), rows(q), rows(out), 0.125, work.data_ptr(), need, stream))):
        with pytest.raises(cabi.KvmError) as e:
            cabi.paged_attention(step, dev.data_ptr(), *args)
        assert e.value.code == code


def test_empty_steps_launch_nothing():
    case = Case(torch.float16, "plain", 4, 2, 64, 16, [20], [1], seed=1)
    plan = plan_step(case.k_cache, [0], [21], case.table, 4)
    none = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    assert paged_attention(plan, 1, none, case.k_cache, case.v_cache).shape == (0, 4, 64)
    write_kv(plan, 1, none[:, :2], none[:, :2], case.k_cache, case.v_cache)
    k, _ = read_kv(plan, 1, case.k_cache, case.v_cache)
    assert torch.equal(k.cpu(), case.seqs[0][0])
    plan = plan_step(case.k_cache, [], [], [], 4)
    assert read_kv(plan, 1, case.k_cache, case.v_cache)[0].shape == (0, 2, 64)
    assert prompt_attention(plan_prompt([], 4, 2, 64, torch.float16), none, none[:, :2], none[:, :2]).shape == (0, 4, 64)


# ---- together, as a deployment runs them

@pytest.mark.parametrize("cache_dtype", ["auto", "e4m3"])
def test_a_request_through_both_instances(cache_dtype):
    """Prefill on a two-rank context instance (write, prompt attention), migration to a decoding instance,
    decoding steps, swap out and back in, more steps: every step's attention is what the whole
    sequence's K and V give."""
    from distserve_amd import (CacheConfig, ContextStageLLMEngine, DecodingStageLLMEngine, ModelConfig, ParallelConfig,
                               create_request)

    cabi.reset()
    layers, hq, h, d, block = 2, 8, 4, 64, 16
    model = ModelConfig.from_kv_shape(layers, hq, d, h)
    cache_config = CacheConfig(block, 64, cache_dtype=cache_dtype)
    ctx = ContextStageLLMEngine(model, ParallelConfig(2, 0, 1, 0), cache_config)
    dec = DecodingStageLLMEngine(model, ParallelConfig(), cache_config,
                                 clear_migrated_blocks_callback=ctx.clear_migrated_blocks_callback)
    ctx._init_kvcache(24, 0)
    dec._init_kvcache(24, 24)
    dec.register_kvcache_mem_handles(ctx.parallel_config, ctx.kv_cache_mem_handles)
    lens = [37, 16, 50]
    requests = [create_request(n, i) for i, n in enumerate(lens)]
    dtype = model.get_torch_dtype()
    total = [n + 6 for n in lens]
    k, v, q = ([[rand((n, heads, d), dtype, 100 * i + 10 * s + j) for s, n in enumerate(total)] for i in range(layers)]
               for j, heads in enumerate((h, h, hq)))
    held = lambda x: ref.quantise(x)[0] if cache_dtype == "e4m3" else x

    for r in requests:
        ctx.block_manager.allocate_blocks(r)
    tables = ctx.block_manager.get_partial_block_table([0, 1, 2])
    for rank, worker in enumerate(ctx.workers[0]):
        plan = worker.plan_step(lens, [0, 0, 0], tables)
        hs, qs = slice(rank * 2, rank * 2 + 2), slice(rank * 4, rank * 4 + 4)
        for layer in range(layers):
            pack = lambda x, cols: torch.cat([x[layer][s][:lens[s], cols] for s in range(3)]).cuda()
            kk, vv, qq = pack(k, hs), pack(v, hs), pack(q, qs)
            worker.write_kv(plan, layer, kk, vv)
            out = worker.prompt_attention(plan, qq, kk, vv).cpu().double()
            at = 0
            for s, n in enumerate(lens):
                want, tol = ref.attention_fast(q[layer][s][:n, qs], k[layer][s][:n, hs], v[layer][s][:n, hs], 0, d ** -0.5, dtype)
                assert ((out[at:at + n] - want).abs() <= tol).all(), (rank, layer, s)
                at += n
    for r in requests:
        migrating = ctx.on_prefill_finished(r)
        dec._migrate_blocks(migrating)
    assert ctx.block_manager.get_num_avail_gpu_blocks() == 24
    worker = dec.workers[0][0]
    at_len = list(lens)

    def step():
        for r, n in zip(requests, at_len):      # the token whose K and V this step writes
            r.add_generated_token("", n)
            dec.block_manager.allocate_blocks(r)
        worker.step([r.request_id for r in requests])        # waits for the requests' swaps, if any
        plan = worker.plan_step([1, 1, 1], at_len, dec.block_manager.get_partial_block_table([0, 1, 2]))
        for layer in range(layers):
            pack = lambda x: torch.cat([x[layer][s][n:n + 1] for s, n in enumerate(at_len)]).cuda()
            worker.write_kv(plan, layer, pack(k), pack(v))
            out = worker.paged_attention(plan, layer, pack(q)).cpu().double()
            kk, vv = worker.read_kv(plan, layer)
            row = 0
            for s, n in enumerate(at_len):
                keys, values = held(k[layer][s][:n + 1]), held(v[layer][s][:n + 1])
                assert torch.equal(kk[row:row + n + 1].cpu().double(), keys.double())
                assert torch.equal(vv[row:row + n + 1].cpu().double(), values.double())
                row += n + 1
                want, tol = ref.attention_fast(q[layer][s][n:n + 1], keys, values, n, d ** -0.5, dtype)
                assert ((out[s] - want[0]).abs() <= tol[0]).all(), (layer, s, n)
        for s in range(3):
            at_len[s] += 1

    step()
    step()
    dec.block_manager.swap_out_requests(requests)
    dec.block_manager.swap_in_requests(requests)
    step()
    step()
    if cache_dtype == "e4m3":
        assert worker._get_block_size_in_bytes(block, model, ParallelConfig()) == 2 * layers * h * block * (d + 1)
    torch.cuda.synchronize()
    cabi.reset()
