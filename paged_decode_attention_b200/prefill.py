"""Attention over the paged cache beyond one plain new token per request.

* ``paged_prefill``: causal attention of many new tokens per request (prompts, chunks of prompts,
  drafted tokens), a ragged batch in one call;
* ``paged_diff_decode``: differential attention of one new token per request;
* ``paged_diff_prefill``: differential attention of many new tokens per request.

They read the cache that ``paged_decode`` reads, after ``cache_write`` has stored the new tokens.
``kernel="auto"`` takes the kernels on the matrix units where they serve the request (head_dim 64
and 128, q of the cache's own 16-bit type or fp16 with 8-bit pages, 16-byte aligned rows; single tokens:
pages of a multiple of 16 tokens up to 256, groups of up to 16 heads) and a general kernel on the CUDA cores everywhere else.  There
is no CPU or PyTorch fallback and no autograd.

What lies behind a request's last token in its pages is never used.  The values of its own tokens
have to be finite: one that is not may reach query rows in front of it.  With 8-bit pages on the matrix
units a value scale is below 255.  The new tokens of a request that ``plan_step``
refused are not in the cache: its status word tells, and what comes out for their rows means nothing.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _cabi
from .cache import PagedKVCache
from .config import KV_CODE, torch_dtype
from .decode import _call_on_index, _current_stream

_PACK = _cabi.packer(_cabi.PdPrefillArgs)
_INDEX = {name: i for i, (name, _) in enumerate(_cabi.PdPrefillArgs._fields_)}
_SCRATCH, _SCRATCH_AT = struct.Struct("@PQ"), _cabi.PdPrefillArgs.workspace.offset


def build_prefill_args(q: torch.Tensor, cache: PagedKVCache, out: torch.Tensor, query_start_loc: torch.Tensor | None, *,
                       maps: int = 1, lam=None, norm: bool = False, norm_weight: torch.Tensor | None = None,
                       eps: float = 1e-5, out_scale: float = 1.0, sm_scale: float | None = None, kernel: str = "auto",
                       max_seq_len: int = 0, status: torch.Tensor | None = None, sm_count: int = 0,
                       stream: int = 0) -> list:
    """The checked values of a ``PdPrefillArgs`` block, in its field order, without scratch."""
    k, v, bt, sl, shape = cache.k_cache, cache.v_cache, cache.block_table, cache.seq_lens, cache.shape
    dev = k.get_device()
    k_stride = k.stride()
    if k.dim() != 4 or k.shape != v.shape or k_stride != v.stride() or k.dtype is not v.dtype or k_stride[3] != 1:
        raise ValueError("k_cache and v_cache must be alike [num_blocks, block_size, H_kv, D] with head_dim contiguous")
    if k.dtype is not torch_dtype(cache.kv_dtype):
        raise ValueError(f"cache tensors are {k.dtype}, kv_dtype says {cache.kv_dtype}")
    num_blocks, page, hkv, d = k.shape
    hq = shape.num_q_heads
    if hkv != shape.num_kv_heads or page != cache.block_size or d != shape.head_dim:
        raise ValueError("cache tensors disagree with cache.shape / cache.block_size")
    if hq % maps or hkv % maps or hq % hkv:
        raise ValueError(f"{hq} query heads and {hkv} kv heads do not form whole groups" + (" of pairs" if maps == 2 else ""))
    q_shape, q_stride = q.shape, q.stride()
    rows = q_shape[0] if q_shape else 0
    want = (rows, hq, d) if maps == 1 else (rows, hq // 2, 2, d)
    if q_shape != want:
        raise ValueError(f"q must be [rows, {', '.join(map(str, want[1:]))}]")
    map_stride = q_stride[2] if maps == 2 else 0
    io = _cabi.IO_CODE.get(q.dtype)
    if io is None:
        raise ValueError(f"q dtype {q.dtype} not supported (fp16 or bf16)")
    if q_stride[-1] != 1:
        raise ValueError("head_dim must be contiguous in q")
    out_stride = out.stride()
    if out.shape != (rows, hq // maps, maps * d) or out.dtype is not q.dtype or out_stride[2] != 1:
        raise ValueError(f"out must be {q.dtype} [{rows}, {hq // maps}, {maps * d}] with the last dimension contiguous")
    if bt.dtype is not torch.int32 or sl.dtype is not torch.int32 or bt.dim() != 2 or sl.dim() != 1:
        raise ValueError("block_table [B, max_blocks] and seq_lens [B] must be int32")
    b, width = bt.shape
    bt_stride, inner = bt.stride()
    if (width > 1 and inner != 1) or not sl.is_contiguous():
        raise ValueError("block_table rows and seq_lens must be contiguous")
    if b > 1 and bt_stride < width:
        raise ValueError("block_table rows must not overlap")
    if sl.numel() != b:
        raise ValueError(f"seq_lens has {sl.shape[0]} entries for {b} block_table rows")
    tensors = [q, out, v, bt, sl]
    starts = 0
    if query_start_loc is not None:
        if query_start_loc.dtype is not torch.int32 or query_start_loc.dim() != 1 \
                or query_start_loc.numel() != b + 1 or not query_start_loc.is_contiguous():
            raise ValueError(f"query_start_loc must be a contiguous int32 vector of {b + 1} entries")
        starts = query_start_loc.data_ptr()
        tensors.append(query_start_loc)
    elif rows != b:
        raise ValueError(f"q batch {rows} != block_table rows {b}")
    ks, vs = cache.k_scale, cache.v_scale
    scales = (0, 0, 0, 0)
    if (ks is None) != (vs is None):
        raise ValueError("k_scale and v_scale must both be given or both be None")
    if ks is not None:
        s_stride = ks.stride()
        if ks.dtype is not torch.float16 or vs.dtype is not torch.float16 or ks.shape != (num_blocks, page, hkv) \
                or ks.shape != vs.shape or s_stride != vs.stride() or (hkv > 1 and s_stride[2] != 1):
            raise ValueError("scales must be fp16 [num_blocks, block_size, H_kv], alike, with the head index contiguous")
        scales = (ks.data_ptr(), vs.data_ptr(), s_stride[0], s_stride[1])
        tensors += (ks, vs)
    lam_ptr, lam_t, lam_h, lam_value, weight = 0, 0, 0, 0.0, 0
    if maps == 2:
        if norm and not eps > 0:
            raise ValueError("eps must be positive: a row without keys is all zeros")
        if lam is None:
            raise ValueError("lam must be a float or an fp32 tensor")
        if isinstance(lam, torch.Tensor):
            if lam.dtype != torch.float32 or lam.dim() > 2:
                raise ValueError("lam must be fp32: one value, [pairs] or [rows, pairs]")
            if lam.dim() == 1 and lam.numel() == hq // 2:  # the usual form, one value a pair
                lam_ptr, lam_t, lam_h = lam.data_ptr(), 0, lam.stride(0)
            else:
                wide = lam.expand(rows, hq // 2)  # raises when the shape does not broadcast
                lam_ptr, lam_t, lam_h = wide.data_ptr(), wide.stride(0), wide.stride(1)
            tensors.append(lam)
        else:
            lam_value = float(lam)
        if norm_weight is not None:
            if not norm:
                raise ValueError("norm_weight without norm")
            if norm_weight.dtype is not torch.float32 or norm_weight.shape != (2 * d,) or not norm_weight.is_contiguous():
                raise ValueError(f"norm_weight must be a contiguous fp32 vector of {2 * d} entries")
            weight = norm_weight.data_ptr()
            tensors.append(norm_weight)
    word = 0
    if status is not None:
        if status.dtype != torch.int32 or status.numel() < 1:
            raise ValueError("status must be an int32 tensor")
        word = status.data_ptr()
        tensors.append(status)
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError("all tensors must be on the cache's device")
    if kernel not in _cabi.KERNEL_CODE:
        raise ValueError(f"kernel must be one of {sorted(_cabi.KERNEL_CODE)}")
    return [q.data_ptr(), out.data_ptr(), q_stride[0], q_stride[1], map_stride, out_stride[0], out_stride[1],
            k.data_ptr(), v.data_ptr(), k_stride[0], k_stride[1], k_stride[2], *scales,
            bt.data_ptr(), max(bt_stride, width), sl.data_ptr(), starts,
            rows, b, hq, hkv, d, page, num_blocks, width, KV_CODE[cache.kv_dtype], io,
            shape.softmax_scale if sm_scale is None else float(sm_scale), maps,
            lam_ptr, lam_t, lam_h, lam_value, weight, float(eps), float(out_scale), int(bool(norm)),
            _cabi.KERNEL_CODE[kernel], int(sm_count), int(max_seq_len), 0, 0, word, stream]


def selected_prefill_kernel(values: list) -> str:
    """Which kernel a block of ``build_prefill_args`` values runs on ("simple" or "stream")."""
    rc = _cabi.load().pd_prefill_select_kernel(_PACK.pack(*values))
    if rc < 0:
        _cabi.check(rc, "pd_prefill_select_kernel")
    return _cabi.KERNEL_NAME[rc]


def _run(entry: str, q: torch.Tensor, cache: PagedKVCache, out: torch.Tensor | None,
         query_start_loc: torch.Tensor | None, maps: int, **kw) -> torch.Tensor:
    if not q.is_cuda:
        raise _cabi.NativeLibraryError(f"{entry} runs on CUDA tensors only; there is no CPU path")
    index = q.get_device()
    if out is None:
        out = q.new_empty((q.shape[0], q.shape[1], maps * q.shape[-1]))
    values = build_prefill_args(q, cache, out, query_start_loc, maps=maps, stream=_current_stream(index), **kw)
    if q.shape[0] == 0 or cache.batch == 0:
        return out
    lib = _cabi.load()
    need = ctypes.c_uint64(0)
    block = _PACK.pack(*values)
    rc = _call_on_index(index, lib.pd_prefill_workspace_bytes, block, ctypes.byref(need))
    if rc != 0:
        _cabi.check(rc, "pd_prefill_workspace_bytes")
    if need.value:
        # Scratch of this call alone, from torch's allocator: ordered by the stream, and inside a
        # capture a part of that graph, so no two graphs or streams share it.
        ws = q.new_empty(need.value, dtype=torch.uint8)
        block = block[:_SCRATCH_AT] + _SCRATCH.pack(ws.data_ptr(), need.value) + block[_SCRATCH_AT + _SCRATCH.size:]
    rc = _call_on_index(index, getattr(lib, entry), block)
    if rc != 0:
        _cabi.check(rc, entry)
    return out


def paged_prefill(q: torch.Tensor, cache: PagedKVCache, query_start_loc: torch.Tensor, out: torch.Tensor | None = None, *,
                  sm_scale: float | None = None, kernel: str = "auto", max_seq_len: int = 0,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of many new tokens per request: q ``[T, Hq, D]`` -> ``[T, Hq, D]``.

    Request b owns the rows ``query_start_loc[b] : query_start_loc[b + 1]`` (int32 ``[B + 1]``); they are
    the last of its ``cache.seq_lens[b]`` cached tokens, and each attends to the keys up to its own
    position.  Rows behind ``query_start_loc[B]`` are left as they were in ``out``; rows that it names behind
    the last of q are cut off, and the others keep their positions; a request with more
    rows than cached tokens has rows that attend to nothing, which are zero.  ``max_seq_len`` is an
    optional host-side bound on ``seq_lens`` that decides how the keys are split; without it the width of the
    block table does.  Give it where the table is wider than the contexts (prompts of 512 and 2048 tokens with
    tables of 32768 take 1.7 and 2 times as long without).
    ``kernel`` and ``status`` are as for ``paged_decode``.
    """
    return _run("pd_prefill", q, cache, out, query_start_loc, 1, sm_scale=sm_scale, kernel=kernel,
                max_seq_len=max_seq_len, status=status)


def paged_diff_decode(q: torch.Tensor, cache: PagedKVCache, lam, out: torch.Tensor | None = None, *, norm: bool = True,
                      norm_weight: torch.Tensor | None = None, eps: float = 1e-5, out_scale: float = 1.0,
                      sm_scale: float | None = None, kernel: str = "auto",
                      status: torch.Tensor | None = None) -> torch.Tensor:
    """Differential attention of one new token per request: q ``[B, H, 2, D]`` -> ``[B, H, 2 * D]``.

    The cache has two kv heads per kv pair: heads 2j and 2j + 1 are the keys K1 and K2 of pair j, and
    their value rows side by side are its value V, ``2 * D`` wide.  ``cache.shape`` counts heads (``2 * H``
    query heads).  With s = ``sm_scale`` (``D ** -0.5``) and ``lam`` a float or an fp32 tensor that
    broadcasts to ``[B, H]``::

        x   = softmax(q[:, :, 0] K1^T s) V - lam * softmax(q[:, :, 1] K2^T s) V
        out = x * rsqrt(mean(x ** 2) + eps) * norm_weight * out_scale

    ``norm=False`` leaves the norm out, ``norm_weight=None`` (fp32 ``[2 * D]``) its weight; a model's
    constant factor behind the norm, one minus its initial lambda, is ``out_scale``.  A request of
    length zero gives zeros.
    """
    return _run("pd_diff_decode", q, cache, out, None, 2, lam=lam, norm=norm, norm_weight=norm_weight, eps=eps,
                out_scale=out_scale, sm_scale=sm_scale, kernel=kernel, status=status)


def paged_diff_prefill(q: torch.Tensor, cache: PagedKVCache, query_start_loc: torch.Tensor, lam,
                       out: torch.Tensor | None = None, *, norm: bool = True, norm_weight: torch.Tensor | None = None,
                       eps: float = 1e-5, out_scale: float = 1.0, sm_scale: float | None = None, kernel: str = "auto",
                       max_seq_len: int = 0, status: torch.Tensor | None = None) -> torch.Tensor:
    """Differential attention of many new tokens per request: q ``[T, H, 2, D]`` -> ``[T, H, 2 * D]``.

    Rows and lengths as in ``paged_prefill``, the rest as in ``paged_diff_decode`` (``lam`` broadcasts to
    ``[T, H]``).
    """
    return _run("pd_prefill", q, cache, out, query_start_loc, 2, lam=lam, norm=norm, norm_weight=norm_weight, eps=eps,
                out_scale=out_scale, sm_scale=sm_scale, kernel=kernel, max_seq_len=max_seq_len, status=status)
