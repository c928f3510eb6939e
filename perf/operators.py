"""The cache operators' cases: what one pass of each costs on the GPU.

Four operators over the paged KV pools ``[blocks, layers, kv_heads, block_size, head_dim]``:

``store``    new tokens' K and V written into their blocks (``write_kv``)
``quant``    the same into a quantised pool, and the sequences read back (``write_kv``, ``read_kv``)
``paged``    new tokens' queries attending over the paged cache (``paged_attention``)
``prompt``   causal attention of whole packed prompts (``prompt_attention``)

A case gives sizes; the sequences' lengths follow from its ``layout`` number, block tables
and values from the seed.  A quantised pool is uint8 ``[blocks, layers, heads, B, D + 1]``: each
(block, layer, head) slab holds B*D e4m3 codes, token by token, and then B scale bytes, one
for each token, that stand for ``2 ** (byte - 127)``.

With ``own`` false ``run`` computes in elementary torch operations in 32 bits; with ``own``
true it calls ``distserve_amd``.
"""
import math
import random

import torch

own = False

LAYERS, LAYER = 2, 1          # pools of two layers; the pass works on the second (strided blocks)
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def _case(name, op, dtype, heads, kv_heads, head_dim, block, seqs, new, ctx, layout, cache="plain", chunks=0):
    """``seqs`` sequences; each brings new[0]..new[1] tokens behind ctx[0]..ctx[1] cached ones.
    ``chunks`` > 0: only that many bring ``new`` tokens, the others one each."""
    return {"name": name, "op": op, "dtype": dtype, "cache": cache, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "block": block, "seqs": seqs, "new_lo": new[0], "new_hi": new[1],
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "chunks": chunks, "layout": layout}


def listed():
    return [
        # one decoding step's tokens of a 7B model's batch
        _case("store-step", "store", "fp16", 32, 32, 128, 16, 96, (1, 1), (0, 1500), 1),
        # a context step: the prompts of a batch, 13B heads on one of two tensor ranks
        _case("store-prompts", "store", "bf16", 20, 20, 128, 16, 16, (64, 2048), (0, 0), 2),
        # a small model's decoding step on a quantised pool, and its sequences read back
        _case("quant-step", "quant", "fp16", 12, 12, 64, 16, 32, (1, 1), (0, 600), 3, "e4m3"),
        # prompts into a quantised pool, grouped heads, read back to recompute from
        _case("quant-prompts", "quant", "bf16", 64, 8, 128, 16, 12, (256, 4096), (0, 0), 4, "e4m3"),
        # one user, one token, a small model: the latency of a call
        _case("token-one", "paged", "fp16", 12, 12, 64, 16, 1, (1, 1), (777, 777), 5),
        # a decoding batch of a 7B model
        _case("token-batch", "paged", "fp16", 32, 32, 128, 16, 32, (1, 1), (64, 2048), 6),
        # few long sequences, grouped heads: the long axis has to be split
        _case("token-long", "paged", "bf16", 64, 8, 128, 16, 8, (1, 1), (8000, 48000), 7),
        # a decoding batch over a quantised pool
        _case("token-quant", "paged", "fp16", 64, 8, 128, 16, 64, (1, 1), (256, 4096), 8, "e4m3"),
        # chunks of long prompts over what is cached of them
        _case("chunk-grouped", "paged", "fp16", 64, 8, 128, 16, 4, (512, 512), (1000, 8000), 9),
        # decoding steps with two chunks riding along, quantised pool
        _case("chunk-mixed", "paged", "bf16", 32, 8, 128, 32, 26, (700, 777), (300, 6000), 10, "e4m3", 2),
        # a context batch of a 7B model
        _case("prompts-packed", "prompt", "fp16", 32, 32, 128, 16, 16, (64, 2048), (0, 0), 11),
        # one long prompt, grouped heads
        _case("prompt-long", "prompt", "bf16", 64, 8, 128, 16, 1, (8192, 8192), (0, 0), 12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    limit = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["store", "quant", "paged", "paged", "paged", "prompt"])
        cache = "e4m3" if op == "quant" else rng.choice(["plain", "plain", "e4m3"]) if op == "paged" else "plain"
        dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
        head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 12, 20, 32])
        group = rng.choice([1, 1, 1, 2, 4, 7, 8])
        if kv_heads * group > 80:
            group = 1
        block = rng.choice([16, 16, 32]) if cache == "e4m3" else rng.choice([8, 16, 16, 32])
        seqs = _log_int(rng, 1, 128)
        top = _log_int(rng, 1, 16384)
        chunks = 0
        if op == "prompt":
            new, ctx = (_log_int(rng, 1, top), top), (0, 0)
        elif op == "paged":
            ctx = (_log_int(rng, 1, top) - 1, top)
            new = rng.choice([(1, 1), (1, 1), (1, 5), (3, 200), (64, 900)])
            chunks = rng.choice([0, 0, 1, 2]) if new[1] > 5 else 0
        else:
            new, ctx = rng.choice([((1, 1), (0, top)), ((1, min(top, 4096)), (0, 300))])
        case = _case("", op, dtype, kv_heads * group, kv_heads, head_dim, block, seqs, new, ctx,
                     rng.randrange(1 << 30), cache, min(chunks, seqs))
        del case["name"]
        kv = sum(_kv_lens(case))
        wide = 2 * kv_heads * head_dim * 4
        # no dearer than the largest listed case: in arithmetic (32-bit products run at a fraction of the
        # 16-bit rate), in the cache and in the rows
        rows = sum(_new_lens(case)) * kv_heads * group * head_dim
        if work(case)["flops"] * (8 if dtype == "fp32" else 1) <= limit and kv * wide <= 2 << 30 and rows <= 1 << 27:
            return case


def _new_lens(case):
    rng = random.Random(case["layout"])
    lens = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    if case["chunks"]:
        lens = [n if i % max(1, case["seqs"] // case["chunks"]) == 0 else 1 for i, n in enumerate(lens)]
    return lens


def _ctx_lens(case):
    rng = random.Random(case["layout"] + 1)
    return [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]


def _kv_lens(case):
    return [c + n for c, n in zip(_ctx_lens(case), _new_lens(case))]


def work(case):
    size, d, h, hq = _SIZE[case["dtype"]], case["head_dim"], case["kv_heads"], case["heads"]
    new, ctx, kv = _new_lens(case), _ctx_lens(case), _kv_lens(case)
    row = d + 1 if case["cache"] == "e4m3" else d * size       # bytes of one token's head in the pool
    tokens, cached = sum(new), sum(kv)
    if case["op"] == "store":
        return {"bytes": 2 * tokens * h * (d * size + row), "flops": 0}
    if case["op"] == "quant":
        # the new tokens in and their codes out; the older tokens' codes in and every value out
        return {"bytes": 2 * h * (tokens * (d * size + row) + (cached - tokens) * row + cached * d * size),
                "flops": 2 * h * d * (2 * tokens + cached)}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    flops = 4 * pairs * hq * d
    if case["op"] == "prompt":
        return {"bytes": 2 * tokens * d * size * (h + hq), "flops": flops}
    return {"bytes": 2 * h * cached * row + 2 * tokens * hq * d * size, "flops": flops}


# ---- inputs

def _normal(shape, dtype, gen):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)


def _keys(shape, dtype, gen):
    """Keys have a few channels that are much larger than the rest."""
    gain = 1.0 + 3.0 * (torch.rand(shape[-1], device="cuda", generator=gen) < 0.03).float()
    return (torch.randn(shape, device="cuda", generator=gen) * gain).to(dtype)


def _quantised_pool(blocks, case, gen):
    """A pool as quantised writes leave it: every row's largest code lies in the top binade."""
    h, b, d = case["kv_heads"], case["block"], case["head_dim"]
    pool = torch.empty(blocks, LAYERS, h, b, d + 1, dtype=torch.uint8, device="cuda")
    flat = pool.view(blocks, LAYERS, h, b * (d + 1))
    for layer in range(LAYERS):
        values = torch.randn((blocks, h, b, d), device="cuda", generator=gen) * 100.0
        top = values.abs().amax(-1, keepdim=True)
        codes = (values * (440.0 / top)).to(torch.float8_e4m3fn)
        flat[:, layer, :, :b * d] = codes.view(torch.uint8).view(blocks, h, b * d)
        flat[:, layer, :, b * d:] = torch.randint(117, 122, (blocks, h, b), device="cuda", generator=gen,
                                                  dtype=torch.uint8)
    return pool


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + case["layout"])
    dtype = _DTYPES[case["dtype"]]
    hq, h, d, b = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    new, ctx, kv = _new_lens(case), _ctx_lens(case), _kv_lens(case)
    tokens = sum(new)
    state = {"case": case, "dtype": dtype, "new": new, "ctx": ctx, "kv": kv}
    if case["op"] in ("paged", "prompt"):
        state["q"] = _normal((tokens, hq, d), dtype, gen)
    if case["op"] != "paged":
        state["k"] = _keys((tokens, h, d), dtype, gen)
        state["v"] = _normal((tokens, h, d), dtype, gen)
    if case["op"] != "prompt":
        pages = [-(-n // b) for n in kv]
        blocks = sum(pages) + sum(pages) // 8 + 3
        order = list(range(blocks))
        random.Random(seed).shuffle(order)
        table, at = [], 0
        for n in pages:
            table.append(order[at:at + n])
            at += n
        state["table"] = table
        if case["cache"] == "e4m3":
            state["k_cache"], state["v_cache"] = (_quantised_pool(blocks, case, gen) for _ in range(2))
        else:
            state["k_cache"] = _keys((blocks, LAYERS, h, b, d), dtype, gen)
            state["v_cache"] = _normal((blocks, LAYERS, h, b, d), dtype, gen)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    dtype, new, ctx, kv = state["dtype"], state["new"], state["ctx"], state["kv"]
    hq, h, d, b = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    if own:
        import distserve_amd

        if case["op"] == "prompt":
            state["plan"] = distserve_amd.plan_prompt(new, hq, h, d, dtype)
        else:
            state["plan"] = distserve_amd.plan_step(state["k_cache"], new, ctx, state["table"], hq, dtype)
    else:
        # the index tensors that a plain program keeps for a step
        state["starts"] = [sum(new[:i]) for i in range(len(new))]
        if case["op"] != "prompt":
            state["pages"] = [torch.tensor(t, device="cuda", dtype=torch.int64) for t in state["table"]]
            page = [state["table"][s][(ctx[s] + i) // b] for s in range(len(new)) for i in range(new[s])]
            off = [(ctx[s] + i) % b for s in range(len(new)) for i in range(new[s])]
            state["page"] = torch.tensor(page, device="cuda", dtype=torch.int64)
            state["off"] = torch.tensor(off, device="cuda", dtype=torch.int64)
            # sequences of one new token are taken together, padded to the longest
            ones = [s for s in range(len(new)) if new[s] == 1]
            width = max([len(state["table"][s]) for s in ones], default=0)
            padded = [state["table"][s] + [0] * (width - len(state["table"][s])) for s in ones]
            state["ones"] = ones
            state["ones_pages"] = torch.tensor(padded, device="cuda", dtype=torch.int64)
            state["ones_rows"] = torch.tensor([state["starts"][s] for s in ones], device="cuda", dtype=torch.int64)
            state["ones_kv"] = torch.tensor([kv[s] for s in ones], device="cuda", dtype=torch.int64)
    return state


# ---- plain forms

def _power(e):
    """2 ** e for -126 <= e <= 127, exactly: the bits of a 32-bit number with that exponent."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _plain_quantise(x):
    """(codes as e4m3, scale bytes) of rows along the last axis."""
    x = x.float()
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    top = finite.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(-126, 126)
    codes = (x * _power(-e)[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _plain_values(pool, pages, case):
    """Blocks ``pages`` of the pool's layer as 32-bit values [..., heads, B, D]."""
    if case["cache"] == "plain":
        return pool[pages, LAYER].float()
    b, d = case["block"], case["head_dim"]
    slabs = pool[pages, LAYER]
    slabs = slabs.reshape(*slabs.shape[:-2], b * (d + 1))
    codes = slabs[..., :b * d].contiguous().view(torch.float8_e4m3fn).float()
    scale = _power(slabs[..., b * d:].int() - 127)
    return codes.view(*codes.shape[:-1], b, d) * scale[..., None]


def _plain_store(state):
    case = state["case"]
    page, off = state["page"], state["off"]
    for x, pool in ((state["k"], state["k_cache"]), (state["v"], state["v_cache"])):
        if case["cache"] == "plain":
            pool[page, LAYER, :, off] = x
            continue
        b, d = case["block"], case["head_dim"]
        codes, scales = _plain_quantise(x)
        flat = pool.view(pool.shape[0], LAYERS, pool.shape[2], b * (d + 1))[:, LAYER]
        head = torch.arange(pool.shape[2], device="cuda")
        at = (off * d)[:, None, None] + torch.arange(d, device="cuda")
        flat[page[:, None, None], head[None, :, None], at.expand(-1, head.numel(), -1)] = codes.view(torch.uint8)
        flat[page[:, None], head[None, :], (b * d + off)[:, None].expand(-1, head.numel())] = scales


def _plain_read(state):
    case, outs = state["case"], []
    for pool in (state["k_cache"], state["v_cache"]):
        parts = []
        for pages, n in zip(state["pages"], state["kv"]):
            values = _plain_values(pool, pages, case).transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"])
            parts.append(values[:n])
        values = torch.cat(parts)
        if state["dtype"] == torch.float16:
            values = values.clamp(-65504.0, 65504.0)      # a code may round a large value past the type's largest
        outs.append(values.to(state["dtype"]))
    return outs


def _plain_softmax_product(q, k, v, allowed, scale):
    """q [h, rows, D], k and v [h, keys, D], all 32-bit; allowed broadcasts to [h, rows, keys]."""
    scores = torch.bmm(q * scale, k.transpose(1, 2).contiguous())
    scores = torch.where(allowed, scores, torch.full((), float("-inf"), device="cuda"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.bmm(weights, v) / weights.sum(-1, keepdim=True)


def _plain_rows(q, k, v, first, group, scale):
    """One sequence: q [n, Hq, D] behind ``first`` cached tokens, k and v [H, keys, D]."""
    n, hq, d = q.shape
    h = hq // group
    out = torch.empty(n, hq, d, device="cuda", dtype=torch.float32)
    key = torch.arange(k.shape[1], device="cuda")
    last = first + torch.arange(n, device="cuda")
    heads = max(1, min(h, (1 << 30) // (group * n * k.shape[1])))    # so that the scores stay at 4 GiB
    for h0 in range(0, h, heads):
        h1 = min(h, h0 + heads)
        rows = q[:, h0 * group:h1 * group].float().reshape(n, h1 - h0, group, d).permute(1, 2, 0, 3)
        allowed = (key[None, :] <= last[:, None]).repeat(group, 1)[None]
        got = _plain_softmax_product(rows.reshape(h1 - h0, group * n, d), k[h0:h1].float(), v[h0:h1].float(),
                                     allowed, scale)
        out[:, h0 * group:h1 * group] = got.view(h1 - h0, group, n, d).permute(2, 0, 1, 3).reshape(n, -1, d)
    return out


def _plain_paged(state):
    case = state["case"]
    q, hq, h, d, b = state["q"], case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    group, scale = hq // h, d ** -0.5
    out = torch.empty(q.shape, device="cuda", dtype=torch.float32)
    ones = state["ones"]
    if ones:
        width = state["ones_pages"].shape[1]
        step = max(1, (1 << 29) // (width * b * h * d))              # so that the gathered keys stay at 2 GiB
        for at in range(0, len(ones), step):
            pages = state["ones_pages"][at:at + step]
            n = pages.shape[0]
            k, v = (_plain_values(p, pages, case).transpose(1, 2).reshape(n * h, width * b, d)
                    for p in (state["k_cache"], state["v_cache"]))
            rows = state["ones_rows"][at:at + step]
            keep = torch.arange(width * b, device="cuda")[None, :] < state["ones_kv"][at:at + step, None]
            got = _plain_softmax_product(q[rows].float().reshape(n * h, group, d), k, v,
                                         keep.repeat_interleave(h, 0)[:, None], scale)
            out[rows] = got.view(n, hq, d)
    for s, n in enumerate(state["new"]):
        if n != 1:
            k, v = (_plain_values(p, state["pages"][s], case).transpose(0, 1).reshape(h, -1, d)
                    for p in (state["k_cache"], state["v_cache"]))
            at = state["starts"][s]
            out[at:at + n] = _plain_rows(q[at:at + n], k[:, :state["kv"][s]], v[:, :state["kv"][s]], state["ctx"][s],
                                         group, scale)
    return out.to(state["dtype"])


def _plain_prompt(state):
    case, q = state["case"], state["q"]
    group, scale = case["heads"] // case["kv_heads"], case["head_dim"] ** -0.5
    out = torch.empty(q.shape, device="cuda", dtype=torch.float32)
    for at, n in zip(state["starts"], state["new"]):
        k, v = (x[at:at + n].transpose(0, 1) for x in (state["k"], state["v"]))
        out[at:at + n] = _plain_rows(q[at:at + n], k, v, 0, group, scale)
    return out.to(state["dtype"])


def run(state):
    op = state["case"]["op"]
    if own:
        import distserve_amd as kv

        if op == "prompt":
            return kv.prompt_attention(state["plan"], state["q"], state["k"], state["v"])
        if op == "paged":
            return kv.paged_attention(state["plan"], LAYER, state["q"], state["k_cache"], state["v_cache"])
        kv.write_kv(state["plan"], LAYER, state["k"], state["v"], state["k_cache"], state["v_cache"])
        if op == "store":
            return [state["k_cache"], state["v_cache"]]
        return list(kv.read_kv(state["plan"], LAYER, state["k_cache"], state["v_cache"]))
    if op == "prompt":
        return _plain_prompt(state)
    if op == "paged":
        return _plain_paged(state)
    _plain_store(state)
    return [state["k_cache"], state["v_cache"]] if op == "store" else _plain_read(state)


# ---- the definition in 64 bits

def _e4m3_table():
    """The value of every 8-bit code: sign, four exponent bits (bias 7), three mantissa bits."""
    values = []
    for code in range(256):
        sign, exponent, mantissa = -1.0 if code & 128 else 1.0, (code >> 3) & 15, code & 7
        if exponent == 15 and mantissa == 7:
            values.append(math.nan)
        elif exponent == 0:
            values.append(sign * mantissa * 2.0 ** -9)
        else:
            values.append(sign * (1.0 + mantissa / 8.0) * 2.0 ** (exponent - 7))
    return torch.tensor(values, dtype=torch.float64, device="cuda")


def _exact_powers(e):
    return torch.tensor([2.0 ** k for k in range(-200, 201)], dtype=torch.float64, device="cuda")[e.long() + 200]


def _exact_tokens(pool, table, n, case):
    """The first ``n`` tokens of a block table as 64-bit values [n, heads, D]."""
    b, d, h = case["block"], case["head_dim"], case["kv_heads"]
    where = torch.arange(n, device="cuda")
    page = torch.tensor(table, device="cuda")[where // b]
    off = where % b
    if case["cache"] == "plain":
        return pool[page, LAYER, :, off].double()
    blocks = pool.shape[0]
    flat = pool.reshape(blocks, LAYERS, h, b * (d + 1))
    rows = flat[page, LAYER]                                                       # [n, h, B*(D+1)]
    codes = torch.gather(rows, 2, (off[:, None, None] * d + torch.arange(d, device="cuda")).expand(n, h, d))
    byte = torch.gather(rows, 2, (b * d + off)[:, None, None].expand(n, h, 1))
    return _e4m3_table()[codes.long()] * _exact_powers(byte.long() - 127)


def _exact_nearest(x):
    """x (64-bit rows) on the grid of e4m3 times its row's power of two."""
    top = x.abs().amax(-1, keepdim=True)
    part, e = torch.frexp(top / 448.0)                                             # top / 448 = part * 2**e
    e = torch.where(top > 0, torch.where(part > 0.5, e, e - 1), 0)
    y = x * _exact_powers(-e)
    step = _exact_powers(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(y / step) * step * _exact_powers(e)                         # halves go to even


def exact(case, seed):
    state = _inputs(case, seed)
    new, ctx, kv = state["new"], state["ctx"], state["kv"]
    b, d, h, hq = case["block"], case["head_dim"], case["kv_heads"], case["heads"]
    if case["op"] == "store":
        outs = []
        for x, pool in ((state["k"], state["k_cache"]), (state["v"], state["v_cache"])):
            pool, at = pool.double(), 0
            for s in range(len(new)):
                where = ctx[s] + torch.arange(new[s], device="cuda")
                page = torch.tensor(state["table"][s], device="cuda")[where // b]
                pool[page, LAYER, :, where % b] = x[at:at + new[s]].double()
                at += new[s]
            outs.append(pool)
        return outs
    if case["op"] == "quant":
        outs = []
        for x, pool in ((state["k"], state["k_cache"]), (state["v"], state["v_cache"])):
            parts, at = [], 0
            for s in range(len(new)):
                old = _exact_tokens(pool, state["table"][s], ctx[s], case)
                parts += [old, _exact_nearest(x[at:at + new[s]].double())]
                at += new[s]
            outs.append(torch.cat(parts))
        return outs
    if work(case)["flops"] > 2e13:
        return None
    group, outs, at = hq // h, [], 0
    for s, n in enumerate(new):
        if case["op"] == "prompt":
            k, v = state["k"][at:at + n].double(), state["v"][at:at + n].double()
        else:
            k, v = (_exact_tokens(state[p], state["table"][s], kv[s], case) for p in ("k_cache", "v_cache"))
        out = torch.empty(n, hq, d, dtype=torch.float64, device="cuda")
        span = max(1, (1 << 27) // kv[s])
        for r0 in range(0, n, span):
            r1 = min(n, r0 + span)
            limit = ctx[s] + torch.arange(r0, r1, device="cuda")
            hidden = torch.arange(kv[s], device="cuda")[None, :] > limit[:, None]
            for head in range(hq):
                score = state["q"][at + r0:at + r1, head].double() @ k[:, head // group].T / math.sqrt(d)
                out[r0:r1, head] = torch.softmax(score.masked_fill(hidden, float("-inf")), -1) @ v[:, head // group]
        outs.append(out)
        at += n
    return torch.cat(outs)
