"""The cache operators' definition in 64 bits on the CPU, and how far a kernel may be from it."""
from __future__ import annotations

import math

import torch


def e4m3_grid() -> torch.Tensor:
    """The non-negative finite e4m3 values, ascending, so that index parity is the mantissa's last bit."""
    return torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                        [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)],
                        dtype=torch.float64)


def quantise(x: torch.Tensor):
    """(values on the grid, exponents) of rows of x; independent of any cast: nearest of the grid's
    values by comparison, ties to the even one."""
    x = x.double()
    finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros((), dtype=torch.float64))
    top = finite.amax(-1)
    e = torch.full(top.shape, -126, dtype=torch.int64)
    for k in range(-126, 128):                       # smallest exponent that covers the row
        e = torch.where((top > 448.0 * 2.0 ** (k - 1)) & (e < k), torch.full_like(e, k), e)
    e = torch.where(top > 0, e, torch.zeros_like(e))
    scale = torch.tensor([2.0 ** k for k in range(-126, 128)], dtype=torch.float64)[e + 126][..., None]
    y = (x.abs() / scale).clamp(max=448.0)
    grid = e4m3_grid()
    upper = torch.searchsorted(grid, y.nan_to_num(0.0)).clamp(max=len(grid) - 1)
    lower = (upper - 1).clamp(min=0)
    down, up = (y - grid[lower]).abs(), (grid[upper] - y).abs()
    pick = torch.where((down < up) | ((down == up) & (lower % 2 == 0)), lower, upper)
    values = grid[pick] * scale * torch.sign(x)
    return torch.where(torch.isnan(x), x, values), e


def decode_pool(pool: torch.Tensor, head_dim: int) -> torch.Tensor:
    """A quantised pool's values, [blocks, layers, heads, B, D] in 64 bits (CPU tensor)."""
    n, layers, heads, b, _ = pool.shape
    flat = pool.reshape(n, layers, heads, b * (head_dim + 1))
    grid = torch.cat([e4m3_grid(), torch.tensor([math.nan], dtype=torch.float64)])
    table = torch.cat([grid, -grid])
    codes = table[flat[..., :b * head_dim].long()].view(n, layers, heads, b, head_dim)
    scale = torch.tensor([2.0 ** (k - 127) for k in range(256)], dtype=torch.float64)[flat[..., b * head_dim:].long()]
    return codes * scale[..., None]


def gather(pool: torch.Tensor, layer: int, table, n: int) -> torch.Tensor:
    """The first n tokens of a block table out of a plain-valued pool: [n, heads, D]."""
    b = pool.shape[3]
    where = torch.arange(n)
    page = torch.tensor(list(table), dtype=torch.int64)[where // b] if n else torch.zeros(0, dtype=torch.int64)
    return pool[page, layer, :, where % b]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first: int, scale: float, dtype: torch.dtype):
    """(out, allowed error): rows q [n, Hq, D] behind ``first`` tokens over k, v [first + n, H, D], in 64 bits.

    The error allowed to a kernel that keeps scores, weights' sums and accumulators in 32 bits
    and rounds weights and results to ``dtype``.  With u half a step of dtype and w = 2^-24
    half a step of 32 bits, for row i and column d:
      weights rounded to dtype             u * sum_j p_j |v_jd|   (p the softmax; in 32 bits too)
      result rounded                       u * |out|
      scores: D products and sums          s = (2 D + 8) w * max_j scale * sum |q||k|, and the exponential (2 w);
                                           weights and their sum move by exp(s) each: 2 (s + 2 w) sum p|v|
      sums over n keys, rescaled           (2 n + 64) w sum p|v|, and the same for the weights' sum
      weights below dtype's normal range   half its smallest step each: t sum_j |v_j| / l, with l >= 1
    """
    n, hq, d = q.shape
    group = hq // k.shape[1]
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps / 2
    out = torch.empty(n, hq, d, dtype=torch.float64)
    tol = torch.empty(n, hq, d, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for h in range(hq):
        for i in range(n):
            seen = first + i + 1
            kk, vv = k[:seen, h // group], v[:seen, h // group]
            score = scale * (kk @ q[i, h])
            p = torch.softmax(score, 0)
            out[i, h] = p @ vv
            spread = p @ vv.abs()
            s = (2 * d + 8) * w * float((abs(scale) * (kk.abs() @ q[i, h].abs())).max())
            tol[i, h] = (u * spread + u * out[i, h].abs() + 2 * (s + 2 * w) * spread + 2 * (2 * seen + 64) * w * spread
                         + tiny * vv.abs().sum(0) + tiny)
    return out, tol


def attention_fast(q, k, v, first, scale, dtype):
    """The same on whole matrices, for finite inputs of some size."""
    n, hq, d = q.shape
    if n == 0:
        return torch.empty(0, hq, d, dtype=torch.float64), torch.empty(0, hq, d, dtype=torch.float64)
    group = hq // k.shape[1]
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps / 2
    hidden = torch.arange(k.shape[0])[None, :] > first + torch.arange(n)[:, None]
    out = torch.empty(n, hq, d, dtype=torch.float64)
    tol = torch.empty(n, hq, d, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for h in range(hq):
        kk, vv = k[:, h // group], v[:, h // group]
        p = torch.softmax((scale * (q[:, h] @ kk.T)).masked_fill(hidden, -math.inf), 1)
        out[:, h] = p @ vv
        spread = p @ vv.abs()
        most = (abs(scale) * (q[:, h].abs() @ kk.abs().T)).masked_fill(hidden, 0).amax(1)
        s = ((2 * d + 8) * w * most)[:, None]
        seen = (first + 1 + torch.arange(n)).double()[:, None]
        total = (~hidden).double() @ vv.abs()
        tol[:, h] = (u * spread + u * out[:, h].abs() + 2 * (s + 2 * w) * spread + 2 * (2 * seen + 64) * w * spread
                     + tiny * total + tiny)
    return out, tol
