"""What the step plan and the prefill entry points refuse, and the kernel choice: no device needed."""

from __future__ import annotations

import ctypes
import pathlib
import re

import pytest
import torch

import operators_ref as ref
import paged_decode_attention_b200 as pda
from paged_decode_attention_b200 import _cabi, plan as ppl, prefill as pre

ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("name", ["PdPrefillArgs", "PdPlanArgs"])
def test_struct_layouts_match_the_header(name):
    header = (ROOT / "include" / "paged_decode.h").read_text()
    body = re.sub(r"/\*.*?\*/", "", header.split(f"typedef struct {name} {{")[1].split(f"}} {name};")[0], flags=re.S)
    names = [re.findall(r"(\w+)\s*$", part.strip())[0] for stmt in body.split(";") if stmt.strip() for part in stmt.split(",")]
    struct = getattr(_cabi, name)
    assert names == [f[0] for f in struct._fields_]
    packed = _cabi.packer(struct)
    values = [float(i) if t is ctypes.c_float else i for i, (_, t) in enumerate(struct._fields_)]
    back = struct.from_buffer_copy(packed.pack(*values))
    assert [getattr(back, n) or 0 for n in names] == values


def test_flag_matches_the_header():
    header = (ROOT / "include" / "paged_decode.h").read_text()
    assert int(re.search(r"#define PD_DEV_NO_BLOCKS (\d+)u", header).group(1)) == _cabi.DEV_NO_BLOCKS


def values(c, **more):
    shape = (c.q.shape[0], c.q.shape[1], c.maps * c.q.shape[-1])
    kw = {**c.kwargs(), **more}
    if c.maps == 2:
        kw.setdefault("lam", c.lam)
    out = kw.pop("out", None)
    out = torch.empty(shape, dtype=c.q.dtype) if out is None else out
    return pre.build_prefill_args(c.q, c.cache, out, c.starts, maps=c.maps, sm_count=148, **kw)


def case(lens=(40, 7), new=(5, 7), **kw):
    kw = {"heads": 4, "kv_heads": 2, "dim": 64, "device": "cpu", **kw}
    return ref.make(list(lens), None if new is None else list(new), **kw)


def test_cpu_tensors_are_refused():
    c = case()
    for call in (c.call, case(maps=2).call, case(new=None, maps=2).call):
        with pytest.raises(_cabi.NativeLibraryError):
            call()
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_cabi.NativeLibraryError):
        pda.plan_step(torch.zeros(2, 3, dtype=torch.int32), i, i, i, i[:1], block_size=16, num_tokens=0)


@pytest.mark.parametrize("kw,expect", [
    (dict(new=None, maps=2), "stream"), (dict(new=None, maps=2, dim=128, kv="int8"), "stream"),
    (dict(new=None, maps=2, dim=32), "simple"), (dict(new=None, maps=2, dim=256), "simple"),
    (dict(new=None, maps=2, page=8), "simple"), (dict(new=None, maps=2, heads=34, kv_heads=2), "simple"),
    (dict(), "stream"), (dict(dim=128, maps=2, kv="int8"), "stream"), (dict(kv="bf16"), "stream"), (dict(page=48), "stream"),
    (dict(page=5), "stream"), (dict(sm_scale=-0.1), "simple"), (dict(heads=129, kv_heads=1), "simple"),
    (dict(dim=32), "simple"), (dict(dim=256), "simple"), (dict(io=torch.bfloat16), "simple")])
def test_kernel_choice(kw, expect):
    kw = dict(kw)
    scale = kw.pop("sm_scale", None)
    assert pre.selected_prefill_kernel(values(case(**kw), **({} if scale is None else {"sm_scale": scale}))) == expect


def test_a_kernel_that_does_not_serve_the_request_is_refused_by_name():
    with pytest.raises(RuntimeError, match="unsupported"):
        pre.selected_prefill_kernel(values(case(dim=32), kernel="stream"))
    with pytest.raises(RuntimeError, match="unsupported"):
        pre.selected_prefill_kernel(values(case(dim=32, new=None, maps=2), kernel="stream"))


@pytest.mark.parametrize("break_it", [
    lambda c: setattr(c, "q", c.q[:, :3]), lambda c: setattr(c, "q", c.q.float()), lambda c: setattr(c, "q", c.q[..., :32]),
    lambda c: setattr(c, "q", c.q[..., 0]), lambda c: setattr(c, "q", c.q.transpose(1, 2).contiguous().transpose(1, 2)),
    lambda c: setattr(c, "starts", c.starts.long()), lambda c: setattr(c, "starts", c.starts[:-1]),
    lambda c: setattr(c, "starts", torch.zeros(6, dtype=torch.int32)[::2]),
    lambda c: setattr(c.cache, "seq_lens", c.cache.seq_lens.long()), lambda c: setattr(c.cache, "seq_lens", c.cache.seq_lens[:1]),
    lambda c: setattr(c.cache, "block_table", c.cache.block_table.t().contiguous().t()),
    lambda c: setattr(c.cache, "v_cache", c.cache.v_cache[:-1]), lambda c: setattr(c.cache, "block_size", 32),
    lambda c: setattr(c.cache, "k_scale", torch.zeros(3)),
    lambda c: setattr(c.cache, "shape", pda.ModelShape(6, 2, 64)), lambda c: setattr(c.cache, "shape", pda.ModelShape(4, 4, 64))])
def test_prefill_refuses(break_it):
    c = case()
    break_it(c)
    with pytest.raises(ValueError):
        values(c)


@pytest.mark.parametrize("more", [dict(lam=torch.zeros(3)), dict(lam=torch.zeros(4).double()), dict(lam=torch.zeros(1, 2, 4)),
                                  dict(norm_weight=torch.zeros(64)), dict(norm_weight=torch.zeros(128).half()),
                                  dict(norm=False), dict(eps=0.0), dict(eps=-1e-5), dict(lam=None), dict(kernel="fast"), dict(status=torch.zeros(1)),
                                  dict(out=torch.empty(12, 4, 64, dtype=torch.float16)),
                                  dict(out=torch.empty(12, 4, 128, dtype=torch.bfloat16))])
def test_differential_arguments_refused(more):
    with pytest.raises((ValueError, RuntimeError)):
        values(case(maps=2), **more)


def test_one_row_per_request_where_there_are_no_starts():
    c = case(new=None, maps=2)
    c.q = c.q[:1]
    with pytest.raises(ValueError):
        values(c)


def test_an_odd_number_of_heads_forms_no_pairs():
    c = case(maps=2)
    c.cache.shape = pda.ModelShape(8, 3, 64)
    c.cache.k_cache, c.cache.v_cache = c.cache.k_cache[:, :, :3], c.cache.v_cache[:, :, :3]
    with pytest.raises(ValueError):
        values(c)


def test_c_entries_check_for_themselves():
    lib = _cabi.load()
    good = values(case())
    pack = _cabi.packer(_cabi.PdPrefillArgs)

    def rc(**kw):
        v = list(good)
        for name, x in kw.items():
            v[pre._INDEX[name]] = x
        return lib.pd_prefill_select_kernel(pack.pack(*v))

    assert rc() in (1, 2)
    for kw in (dict(q=0), dict(out=0), dict(k_cache=0), dict(block_table=0), dict(seq_lens=0), dict(num_rows=-1), dict(batch=-1),
               dict(num_q_heads=3), dict(num_kv_heads=0), dict(maps=3), dict(maps=2, num_kv_heads=1), dict(block_size=0),
               dict(num_blocks=0), dict(max_blocks_per_seq=0), dict(kv_dtype=4), dict(kv_dtype=3), dict(io_dtype=2), dict(kernel=3),
               dict(max_seq_len=-1), dict(maps=2, norm=1, eps=0.0), dict(k_scale=16), dict(block_table_stride=0), dict(query_start=0)):
        assert rc(**kw) == -1, kw
    for kw in (dict(head_dim=96), dict(kv_stride_token=100), dict(k_cache=8)):
        assert rc(**kw) == -2, kw
    assert rc(workspace=128) == -3
    assert lib.pd_prefill(None) == -1 and lib.pd_diff_decode(None) == -1 and lib.pd_plan_step(None) == -1
    assert lib.pd_diff_decode(pack.pack(*good)) == -1  # starts given
    n = ctypes.c_uint64(7)
    assert lib.pd_prefill_workspace_bytes(None, ctypes.byref(n)) == -1
    assert lib.pd_prefill_workspace_bytes(pack.pack(*good), None) == -1


def plan_args():
    i = lambda *n: torch.zeros(n, dtype=torch.int32)
    return dict(block_table=i(3, 4), context_lens=i(3), new_tokens=i(3), free_blocks=i(9), num_free=i(1), block_size=16,
                num_tokens=5)


def on_meta(x):
    """A stand-in that says it is on the GPU, for checks that come before any address is used."""
    return x.as_subclass(type("Fake", (torch.Tensor,), {"is_cuda": property(lambda self: True)}))


@pytest.mark.parametrize("change", [
    dict(block_table=torch.zeros(3, 4)), dict(block_table=torch.zeros(4, dtype=torch.int32)),
    dict(block_table=torch.zeros(4, 3, dtype=torch.int32).t()), dict(block_table=torch.zeros(3, 0, dtype=torch.int32)),
    dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), dict(block_table=torch.zeros(8193, 1, dtype=torch.int32)),
    dict(context_lens=torch.zeros(2, dtype=torch.int32)), dict(context_lens=torch.zeros(3, dtype=torch.int64)),
    dict(new_tokens=torch.zeros(6, dtype=torch.int32)[::2]), dict(free_blocks=torch.zeros(3, 3, dtype=torch.int32)),
    dict(num_free=torch.zeros(2, dtype=torch.int32)), dict(block_size=0), dict(num_tokens=-1), dict(status=torch.zeros(1))])
def test_plan_refuses(change):
    a = {**plan_args(), **change}
    a["block_table"] = on_meta(a["block_table"])
    with pytest.raises(ValueError):
        pda.plan_step(**a)


def test_plan_refuses_overlapping_outputs():
    a = plan_args()
    i = lambda *n: torch.zeros(n, dtype=torch.int32)
    good = pda.StepPlan(torch.zeros(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int64), i(4), a["context_lens"], a["num_free"])
    inputs = [a[k] for k in ("block_table", "context_lens", "new_tokens", "free_blocks", "num_free")]
    ppl._refuse_overlap(*inputs, good)  # the two updates in place
    both = torch.zeros(8, dtype=torch.int64)
    words = i(8)
    for bad in (good._replace(seq_lens=a["new_tokens"]), good._replace(num_free=a["free_blocks"][3:4]),
                good._replace(slot_mapping=both[:5], positions=both[3:]), good._replace(positions=good.slot_mapping),
                good._replace(query_start_loc=a["block_table"][0]), good._replace(query_start_loc=words[:4], seq_lens=words[3:6])):
        with pytest.raises(ValueError, match="overlaps"):
            ppl._refuse_overlap(*inputs, bad)
    shifted = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="overlaps"):
        ppl._refuse_overlap(a["block_table"], shifted[:3], *inputs[2:], good._replace(seq_lens=shifted[1:]))


def test_plan_c_entry_checks():
    lib = _cabi.load()
    pack = _cabi.packer(_cabi.PdPlanArgs)
    names = [n for n, _ in _cabi.PdPlanArgs._fields_]
    good = dict(block_table=16, block_table_stride=4, context_lens=16, new_tokens=16, free_blocks=16, num_free=16, slot_mapping=16,
                positions=16, query_start=16, seq_lens=16, num_free_out=16, batch=3, max_blocks_per_seq=4, block_size=16,
                free_capacity=9, num_tokens=5, status=0, stream=0)

    def rc(**kw):
        return lib.pd_plan_step(pack.pack(*[{**good, **kw}[n] for n in names]))

    for kw in (dict(block_table=0), dict(context_lens=0), dict(new_tokens=0), dict(free_blocks=0), dict(num_free=0),
               dict(slot_mapping=0), dict(positions=0), dict(query_start=0), dict(seq_lens=0), dict(num_free_out=0), dict(batch=-1),
               dict(max_blocks_per_seq=0), dict(block_size=0), dict(free_capacity=-1), dict(num_tokens=-1),
               dict(block_table_stride=3)):
        assert rc(**kw) == -1, kw
    for kw in (dict(batch=8193), dict(max_blocks_per_seq=2 ** 30, block_table_stride=2 ** 30), dict(block_size=2 ** 30)):
        assert rc(**kw) == -2, kw
