"""Attention over the paged cache where its rows, keys and workers are laid out at an edge: against
the definitions in 64 bits, with the bounds derived in operators_ref."""

from __future__ import annotations

import ctypes
import dataclasses

import pytest
import torch

import operators_ref as ref
from paged_decode_attention_b200 import _cabi, prefill as pre

pytestmark = pytest.mark.gpu


def check_rows(got, c, r, rows, what=""):
    """The first ``rows`` rows of ``got`` against the same rows of ``r``, all of which have to be finite."""
    out, bound = (x[:rows] for x in r)
    assert rows > 0 and out.isfinite().all() and bound.isfinite().all()
    off = (got[:rows].double() - out).abs()
    assert (off <= bound).all(), f"{what}: off by {float(off.nan_to_num(float('inf')).max()):.3e}"


@pytest.mark.parametrize("kernel", ["simple", "stream"])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("kv", ["fp16", "bf16", "int8"])
@pytest.mark.parametrize("lens,new,rows", [([35], [30], 11), ([300, 520], [300, 520], 401), ([9000, 8000], [40, 30], 45)])
def test_rows_are_cut_off_where_the_starts_name_more(kernel, maps, kv, lens, new, rows):
    """q holds fewer rows than query_start_loc names: those it holds see the keys they would see in the whole."""
    c = ref.make(lens, new, heads=4, kv_heads=2, dim=64, kv=kv, maps=maps, lam="heads", seed=3)
    r = ref.reference(c)
    c.q = c.q[:rows].contiguous()
    check_rows(c.call(kernel=kernel), c, r, rows, kernel)


@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("kv_heads", [1, 2, 4])
@pytest.mark.parametrize("sm_count,requests", [(2, 3), (2, 4), (5, 10), (8, 9), (140, 141), (140, 280), (148, 296)])
def test_short_requests_dealt_whole_to_any_number_of_sms(sm_count, requests, kv_heads, kv):
    """Fewer requests than workers, none longer than 256 tokens, no room in the table for longer ones: each worker
    has one, and the two maps of a pair meet in scratch rows that nobody else may touch."""
    c = ref.make([96 + 7 * (i % 5) for i in range(requests)], heads=2 * kv_heads, kv_heads=kv_heads, dim=64, kv=kv, maps=2,
                 seed=requests)
    r = ref.reference(c)
    out = torch.empty(requests, c.q.shape[1], 128, dtype=c.q.dtype, device="cuda")
    lib, need = _cabi.load(), ctypes.c_uint64(0)
    values = pre.build_prefill_args(c.q, c.cache, out, None, maps=2, lam=c.lam, kernel="stream", sm_count=sm_count,
                                    stream=torch.cuda.current_stream().cuda_stream, **c.kwargs())
    names = [n for n, _ in _cabi.PdPrefillArgs._fields_]
    _cabi.check(lib.pd_prefill_workspace_bytes(pre._PACK.pack(*values), ctypes.byref(need)), "pd_prefill_workspace_bytes")
    scratch = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    values[names.index("workspace")], values[names.index("workspace_bytes")] = scratch.data_ptr(), need.value
    block = pre._PACK.pack(*values)
    for _ in range(30):
        out.fill_(float("nan"))
        _cabi.check(lib.pd_diff_decode(block), "pd_diff_decode")
        check_rows(out, c, r, requests)


@pytest.mark.parametrize("kernel", ["simple", "stream"])
@pytest.mark.parametrize("kv", ["fp16", "bf16", "int8", "fp8_e5m2"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cached,new", [(100, 200), (40, 101), (1, 64), (200, 300)])
def test_many_rows_without_keys_beside_rows_with_keys(kernel, kv, dim, cached, new):
    """More new tokens than cached ones, by so many that 128 packed rows and more attend to nothing while others of
    their CTA have keys: those rows are zeros in every call."""
    batch = 40
    c = ref.make([cached] * batch, [new] * batch, heads=8, kv_heads=2, dim=dim, kv=kv, seed=new)
    r = ref.reference(c)
    empty = (torch.arange(new, device="cuda") < new - cached).repeat(batch)
    assert int(empty.sum()) * 4 // batch >= 128 and (r[0][empty] == 0).all()
    out = torch.empty(c.q.shape, dtype=c.q.dtype, device="cuda")
    for _ in range(1 if kernel == "simple" else 20):
        out.fill_(float("nan"))
        c.call(out=out, kernel=kernel)
        assert (out[empty] == 0).all()
        check_rows(out, c, r, batch * new, kernel)


def without_poison(c):
    """The same case with finite values wherever it has NaN, so that a page left out counts as nothing in the
    reference: zero times what stands in the page read in its place."""
    def clean(t):
        return t if t is None or t.dtype is torch.int8 else torch.nan_to_num(t.float(), 0.0).to(t.dtype)

    tensors = {n: clean(getattr(c.cache, n)) for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    return dataclasses.replace(c, cache=dataclasses.replace(c.cache, **tensors))


@pytest.mark.parametrize("kernel", ["simple", "stream"])
@pytest.mark.parametrize("kv", ["fp16", "bf16", "int8", "fp8_e5m2"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("maps,new", [(1, [300, 10, 20, 64]), (2, [300, 10, 20, 64]), (2, None)])
def test_pages_outside_the_pool_count_as_nothing(kernel, kv, dim, maps, new):
    """Every row is compared, also those of requests that lose a page, and the one that loses all of them gives zeros."""
    for seed in range(3):
        c = ref.make([300, 64, 2500, 64], new, heads=4, kv_heads=2, dim=dim, kv=kv, maps=maps, seed=seed)
        table = c.cache.block_table
        table[0, 3], table[1, 0], table[2, 1], table[2, 100] = 10 ** 6, -1, -3, c.cache.num_blocks
        table[3] = -1
        r = ref.reference(without_poison(c))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = c.call(kernel=kernel, status=status)
        assert int(status) == _cabi.DEV_BAD_BLOCK
        check_rows(got, c, r, got.shape[0], kernel)
        assert (got[-(64 if new else 1):] == 0).all()


@pytest.mark.parametrize("kernel", ["simple", "stream"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [None, [30, 4], [130, 200]])
def test_without_the_norm_its_weight_is_not_applied(kernel, dim, new):
    """The C ABI's formula: a weight that stands in an argument block whose ``norm`` is 0 is no part of the result."""
    c = ref.make([700, 260], new, heads=4, kv_heads=2, dim=dim, maps=2)
    kw = c.kwargs()
    weight = c.weight
    c.norm, c.weight = False, None
    r = ref.reference(c)
    out = torch.full((c.q.shape[0], c.q.shape[1], 2 * dim), float("nan"), dtype=c.q.dtype, device="cuda")
    lib, need = _cabi.load(), ctypes.c_uint64(0)
    values = pre.build_prefill_args(c.q, c.cache, out, c.starts, maps=2, lam=c.lam, kernel=kernel,
                                    stream=torch.cuda.current_stream().cuda_stream, **{**kw, "norm_weight": weight})
    at = {n: i for i, (n, _) in enumerate(_cabi.PdPrefillArgs._fields_)}
    values[at["norm"]] = 0
    _cabi.check(lib.pd_prefill_workspace_bytes(pre._PACK.pack(*values), ctypes.byref(need)), "pd_prefill_workspace_bytes")
    scratch = torch.empty(max(need.value, 1), dtype=torch.uint8, device="cuda")
    values[at["workspace"]], values[at["workspace_bytes"]] = scratch.data_ptr(), need.value
    entry = lib.pd_diff_decode if new is None else lib.pd_prefill
    _cabi.check(entry(pre._PACK.pack(*values)), "call")
    check_rows(out, c, r, out.shape[0], kernel)
