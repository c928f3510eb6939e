"""The cache operators: what a model's layers do with the paged KV pools.

A step brings new tokens to some sequences.  ``plan_step`` takes what ``Worker.step`` gets for
it (reference distserve/worker.py:194-203: how many new tokens each request has, the index
of its first new token, its block table), checks it once on the host and puts it on the GPU;
each layer then calls

    write_kv(plan, layer, k, v, k_cache, v_cache)            new tokens' K and V into their blocks
    paged_attention(plan, layer, q, k_cache, v_cache)        the new tokens attend over the cache

or, where every sequence is new (a context instance's step), ``prompt_attention(plan, q, k, v)``
over the rows at hand.  ``read_kv`` gives the sequences' K and V back.

Rows are ``[tokens, heads, head_dim]``, float16, bfloat16 or float32, all sequences' new
tokens one after the other; slices of a fused projection are fine (any token and head
strides that keep rows at multiples of 16 bytes).  Tensors may have more rows than the step has
tokens (a batch padded to a fixed size): those behind the last sequence are neither read nor
written (a new output holds zeros there).
An ``out`` may be a slice of the tensor that q is a slice of, but must not share memory with what the call
reads; the K and the V pool of a write must be two.  Such calls are refused.

A pool is plain, ``[num_blocks, layers, kv_heads, block_size, head_dim]`` of the rows' type, or
quantised: uint8 with last dimension ``head_dim + 1`` (``quantized_pool_shape``), e4m3 codes with a
power-of-two scale for each token and head.  Migration and swap move both.  Chunks and prompts are fastest where
``block_size`` is a multiple of 16: over other blocks every row of a plan goes to the kernel for few rows
(512 tokens behind thousands, 64 heads over 8: 1.5 ms instead of 0.35).

Everything, a plan's copy to the GPU too, runs on the current stream of the tensors' device and returns
without waiting; a plan made on one stream can be used on any other, which then waits for its copy.
Calls can be captured into a graph; the plan must have been made before the capture, and the graph keeps
what it needs of it.  There are no gradients: a call on tensors that require one (rows, pools or ``out``),
or that have a forward-mode tangent, is refused, and what a call writes has its version raised.

Scores, softmax sums and accumulators are 32-bit.  The softmax weights of float16 and bfloat16 rows are rounded to
the rows' type for the product with V, half a step of each, which adds about as much error as the
rounding of the result does (relative to the definition, 2.9e-4 instead of 2.1e-4 in float16, 2.1e-3 instead of 1.6e-3 in bfloat16).
"""
from __future__ import annotations

from itertools import chain
from typing import Optional, Sequence, Tuple

import torch

# ``torch.ops.kvcache_ops.*`` are the same functions with schemas; the plan's methods, which the functions
# below call, cost a third of their host time.
StepPlan = torch.classes.kvcache_ops.StepPlan

# torch's numbers of the types (what C++ calls a ScalarType)
_TYPE_NUMBER = {torch.float16: 5, torch.bfloat16: 15, torch.float32: 6}


def quantized_pool_shape(shape: Sequence[int]) -> Tuple[int, ...]:
    """The uint8 pool that holds what a plain pool of ``shape`` holds: one byte more than head_dim a token."""
    return (*shape[:-1], shape[-1] + 1)


def _type_number(dtype: torch.dtype) -> int:
    if dtype not in _TYPE_NUMBER:
        raise RuntimeError(f"the cache operators work on float16, bfloat16 and float32, not {dtype}")
    return _TYPE_NUMBER[dtype]


def plan_step(k_cache: torch.Tensor, input_lens: Sequence[int], first_token_indexes: Sequence[int],
              block_table: Sequence[Sequence[int]], num_heads: int, dtype: Optional[torch.dtype] = None) -> StepPlan:
    """The plan of a step over pools shaped like ``k_cache``: sequence ``i`` brings ``input_lens[i]``
    tokens behind the ``first_token_indexes[i]`` that its blocks ``block_table[i]`` hold already.
    ``num_heads`` query heads share the pool's KV heads.  ``dtype`` is the rows' type (a quantised
    pool does not tell; default: the pool's, float16 for a quantised one)."""
    if k_cache.dim() != 5:
        raise RuntimeError(f"a pool must be [num_blocks, layers, kv_heads, block_size, head_dim], got {tuple(k_cache.shape)}")
    if not k_cache.is_cuda:
        raise RuntimeError("plan_step: the pools must live on the GPU")
    coded = k_cache.dtype == torch.uint8
    if dtype is None:
        dtype = torch.float16 if coded else k_cache.dtype
    num_blocks, _, num_kv_heads, block_size, width = k_cache.shape
    if num_blocks == 0:
        raise RuntimeError("plan_step: the pool has no blocks")
    return StepPlan(list(first_token_indexes), list(input_lens), list(chain.from_iterable(block_table)),
                    [len(t) for t in block_table], num_blocks, block_size, num_heads, num_kv_heads,
                    width - 1 if coded else width, _type_number(dtype), coded, k_cache.device.index)


def plan_prompt(input_lens: Sequence[int], num_heads: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype,
                device: Optional[torch.device] = None) -> StepPlan:
    """The plan of a step of whole prompts without a cache, for ``prompt_attention``."""
    device = torch.device("cuda") if device is None else torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("plan_prompt: the operators run on the GPU")
    index = torch.cuda.current_device() if device.index is None else device.index
    lens = list(input_lens)
    return StepPlan([0] * len(lens), lens, [], [], 0, 0, num_heads, num_kv_heads, head_dim, _type_number(dtype), False, index)


def write_kv(plan: StepPlan, layer: int, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
             v_cache: torch.Tensor) -> None:
    """The step's new K and V rows ``[tokens, kv_heads, head_dim]`` into layer ``layer`` of the pools."""
    plan.write_kv(layer, k, v, k_cache, v_cache)


def read_kv(plan: StepPlan, layer: int, k_cache: torch.Tensor, v_cache: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V of all tokens of the step's sequences, earlier and new, ``[kv_tokens, kv_heads, head_dim]``
    each, one sequence after the other."""
    return plan.read_kv(layer, k_cache, v_cache)


def paged_attention(plan: StepPlan, layer: int, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the step's new tokens ``q`` ``[tokens, heads, head_dim]`` over the cache, each over its
    sequence up to itself; the new tokens' K and V must have been written.  ``scale``: of the scores,
    default ``head_dim ** -0.5``."""
    return plan.paged_attention(layer, q, k_cache, v_cache, scale, out)


def prompt_attention(plan: StepPlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of whole prompts packed one after the other, every sequence of the plan being new."""
    return plan.prompt_attention(q, k, v, scale, out)
