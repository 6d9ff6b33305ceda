"""Block tables, slot maps, positions and lengths of one serving step, built on the GPU.

``plan_step`` stands in front of ``cache_write`` and the attention entry points: from how many
tokens each request has in the cache and how many it gets now, it takes the pages they lack from a
free list, enters them into the block table, and returns where every new token goes.  Nothing is
read back to the host, so a step (or a captured graph of steps) needs no synchronisation.
"""

from __future__ import annotations

import typing

import torch

from . import _cabi
from .decode import _call_on_index, _current_stream

MAX_BATCH = 8192

_PACK = _cabi.packer(_cabi.PdPlanArgs)


class StepPlan(typing.NamedTuple):
    """What ``plan_step`` returns; the names are those the other entry points use."""

    slot_mapping: torch.Tensor  # [num_tokens] int64, -1: padding, or a token of a request not served
    positions: torch.Tensor  # [num_tokens] int64, 0 for padding
    query_start_loc: torch.Tensor  # [B + 1] int32
    seq_lens: torch.Tensor  # [B] int32
    num_free: torch.Tensor  # [1] int32


def _vector(t: torch.Tensor, what: str, dtype: torch.dtype, size: int | None, index: int) -> int:
    """Address of a checked vector; cheap where all is well (a plan is microseconds of work)."""
    if (t.dtype is not dtype or t.dim() != 1 or t.get_device() != index or not t.is_contiguous()
            or (size is not None and t.numel() != size)):
        if t.get_device() != index:
            raise ValueError(f"{what} must be on the block table's device")
        raise ValueError(f"{what} must be a contiguous vector of {dtype}"
                         + ("" if size is None else f" with {size} entries"))
    return t.data_ptr()


def plan_step(block_table: torch.Tensor, context_lens: torch.Tensor, new_tokens: torch.Tensor,
              free_blocks: torch.Tensor, num_free: torch.Tensor, *, block_size: int, num_tokens: int,
              out: StepPlan | None = None, status: torch.Tensor | None = None) -> StepPlan:
    """Plan one step of a batch.

    ``block_table`` ``[B, max_blocks]``, ``context_lens`` ``[B]`` (tokens already cached) and
    ``new_tokens`` ``[B]`` are int32; ``free_blocks`` holds the free block ids as a stack whose top
    is entry ``num_free[0] - 1`` (both int32).  ``num_tokens`` is the length of the per-token
    outputs: the sum of ``new_tokens``, or more for a padded batch.

    Request b lacks ``ceil((c + n) / block_size) - ceil(c / block_size)`` pages; they are popped from
    the stack in request order and written into its row of ``block_table`` (the only input that is
    changed).  A request is served when its row has room for all its pages and the stack holds the
    pages of all such requests up to and including it (or it needs none); one that is not served
    keeps its length and row, its tokens get slot -1, and ``status`` (an int32 word) gets
    ``DEV_NO_BLOCKS``.  ``query_start_loc`` counts its tokens all the same (their rows of the batch stay
    where they are), so an attention call of the same step takes them for the last of the cached ones and
    what it gives for them means nothing: read ``status`` before the results are used.  Block ids are taken as they are; ``cache_write`` and the attention kernels
    check them.

    ``out`` receives the results in buffers of the caller, for captured graphs: ``out.seq_lens`` may
    be ``context_lens`` and ``out.num_free`` may be ``num_free``, so a replayed step carries its state
    on; otherwise nothing may overlap.  At most 8192 requests and fewer than 2**31 new tokens.
    """
    if not block_table.is_cuda:
        raise _cabi.NativeLibraryError("plan_step runs on CUDA tensors only; there is no CPU path")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [batch, max_blocks]")
    b, width = block_table.shape
    stride, inner = block_table.stride()
    if width < 1:
        raise ValueError("block_table must be int32 [batch, max_blocks]")
    if inner != 1 and width > 1:
        raise ValueError("block_table rows must be contiguous")
    if stride < width:
        if b > 1:
            raise ValueError("block_table rows must not overlap")
        stride = width
    if num_tokens < 0 or block_size <= 0:
        raise ValueError("num_tokens must not be negative and block_size must be positive")
    if b > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} requests")
    index = block_table.get_device()
    i32 = torch.int32
    ctx = _vector(context_lens, "context_lens", i32, b, index)
    new = _vector(new_tokens, "new_tokens", i32, b, index)
    free = _vector(free_blocks, "free_blocks", i32, None, index)
    nfree = _vector(num_free, "num_free", i32, 1, index)
    if out is None:
        make = num_free.new_empty
        out = StepPlan(make(num_tokens, dtype=torch.int64), make(num_tokens, dtype=torch.int64), make(b + 1), make(b), make(1))
        ptrs = [t.data_ptr() for t in out]
    else:
        ptrs = (_vector(out.slot_mapping, "out.slot_mapping", torch.int64, num_tokens, index),
                _vector(out.positions, "out.positions", torch.int64, num_tokens, index),
                _vector(out.query_start_loc, "out.query_start_loc", i32, b + 1, index),
                _vector(out.seq_lens, "out.seq_lens", i32, b, index),
                _vector(out.num_free, "out.num_free", i32, 1, index))
        _refuse_overlap(block_table, context_lens, new_tokens, free_blocks, num_free, out)
    word = 0
    if status is not None:
        if status.dtype is not i32 or status.numel() < 1 or status.get_device() != index:
            raise ValueError("status must be an int32 tensor on the same device")
        word = status.data_ptr()
    block = _PACK.pack(block_table.data_ptr(), stride, ctx, new, free, nfree, *ptrs, b, width, block_size,
                       free_blocks.numel(), num_tokens, word, _current_stream(index))
    rc = _call_on_index(index, _cabi.load().pd_plan_step, block)
    if rc != 0:
        _cabi.check(rc, "pd_plan_step")
    return out


def _span(t: torch.Tensor) -> tuple[int, int]:
    first = t.data_ptr()
    last = first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else first
    return first, last


def _refuse_overlap(block_table, context_lens, new_tokens, free_blocks, num_free, out: StepPlan) -> None:
    """No output shares memory with an input or another output, but for the two updates in place."""
    inputs = [("block_table", block_table), ("context_lens", context_lens), ("new_tokens", new_tokens),
              ("free_blocks", free_blocks), ("num_free", num_free)]
    outputs = [(f"out.{n}", t) for n, t in zip(StepPlan._fields, out)]
    for i, (name, t) in enumerate(outputs):
        lo, hi = _span(t)
        for other, u in inputs + outputs[:i]:
            a, z = _span(u)
            if lo < z and a < hi:
                whole = (lo, hi) == (a, z)
                if whole and (name, other) in (("out.seq_lens", "context_lens"), ("out.num_free", "num_free")):
                    continue
                raise ValueError(f"{name} overlaps {other}")
