"""paged_prefill, paged_diff_decode and paged_diff_prefill against their definitions in 64 bits, with
the bounds derived in operators_ref.  Everything that must not be read is NaN."""

from __future__ import annotations

import pytest
import torch

import operators_ref as ref
import paged_decode_attention_b200 as pda
from paged_decode_attention_b200 import _cabi, prefill as pre

pytestmark = pytest.mark.gpu

KVS = ["fp16", "bf16", "int8", "fp8_e5m2"]


def selected(c, kernel="auto"):
    shape = (c.q.shape[0], c.q.shape[1], c.maps * c.q.shape[-1])
    kw = c.kwargs()
    if c.maps == 2:
        kw["lam"] = c.lam
    values = pre.build_prefill_args(c.q, c.cache, torch.empty(shape, dtype=c.q.dtype, device="cuda"), c.starts, maps=c.maps,
                                    kernel=kernel, **kw)
    return pre.selected_prefill_kernel(values)


def both(c, want=None, what=""):
    """The general kernel and, where it differs, the chosen one; both raise no flag."""
    r = ref.reference(c)
    chosen = selected(c)
    if want is not None:
        assert chosen == want
    for kernel in ("simple",) if chosen == "simple" else ("simple", "stream"):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = c.call(kernel=kernel, status=status)
        torch.cuda.synchronize()
        assert int(status) == 0
        ref.check(got, c, f"{what}/{kernel}", r)
    return r


# ---- differential decode ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (4, 2), (8, 4), (12, 1), (32, 2), (6, 3), (16, 8)])
def test_diff_decode_heads_and_types(kv, dim, heads, kv_heads):
    both(ref.make([1, 15, 16, 17, 0, 333], heads=heads, kv_heads=kv_heads, dim=dim, kv=kv, maps=2, seed=heads), "stream")


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 5], [5000], [40000, 3], [1, 16, 255, 256, 257, 4096], [700] * 40,
                                  list(range(1, 160))])
@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_diff_decode_lengths(lens, kv):
    both(ref.make(lens, heads=4, kv_heads=2, dim=128, kv=kv, maps=2, seed=len(lens)), "stream")


@pytest.mark.parametrize("page", [16, 32, 48, 128, 256])
def test_diff_decode_pages(page):
    both(ref.make([1, page - 1, page, page + 1, 3 * page + 5], heads=4, kv_heads=2, page=page, maps=2), "stream")


@pytest.mark.parametrize("how", [dict(norm=False), dict(weight=False), dict(lam="float"), dict(lam="rows"), dict(interleaved=True)])
def test_diff_decode_options(how):
    both(ref.make([3, 100, 0, 61], heads=4, kv_heads=2, dim=64, maps=2, seed=8, **how), "stream")


@pytest.mark.parametrize("dim,page,kv,io", [(32, 16, "fp16", None), (256, 16, "fp16", None), (64, 8, "fp16", None),
                                            (64, 5, "int8", None), (64, 16, "fp16", torch.bfloat16), (128, 16, "bf16", torch.float16),
                                            (32, 16, "int8", None), (128, 512, "bf16", None)])
def test_diff_decode_on_the_general_kernel(dim, page, kv, io):
    both(ref.make([1, 40, 0, 333], heads=3, kv_heads=1, dim=dim, page=page, kv=kv, io=io, maps=2), "simple")


def test_diff_decode_values_with_a_mean():
    """Both maps then agree in most of what they give, and the difference is what is left."""
    both(ref.make([700, 90, 1], heads=4, kv_heads=2, dim=64, maps=2, v_mean=1.0, seed=2), "stream")


def test_diff_decode_is_reproducible():
    c = ref.make([4000, 17, 900, 20000], heads=8, kv_heads=4, dim=128, maps=2)
    a = c.call()
    for _ in range(5):
        assert torch.equal(a, c.call())


def test_diff_decode_layouts():
    """The two maps side by side or one behind the other; q and out as parts of larger buffers."""
    c = ref.make([100, 40, 7], heads=4, kv_heads=2, dim=64, maps=2)
    r = ref.reference(c)
    behind = torch.empty(3, 2, 4, 64, dtype=torch.float16, device="cuda")
    behind.copy_(c.q.transpose(1, 2))
    padded = torch.full((3, 6, 144), 9.0, dtype=torch.float16, device="cuda")
    c.q = behind.transpose(1, 2)
    got = c.call(out=padded[:, 1:5, 8:136])
    ref.check(got, c, "strided", r)
    edge = padded.clone()
    edge[:, 1:5, 8:136] = 9.0
    assert (edge == 9.0).all()


def test_diff_decode_bad_blocks_are_left_out_and_flagged():
    for kernel in ("simple", "stream"):
        c = ref.make([100, 64], heads=4, kv_heads=2, dim=64, maps=2)
        c.cache.block_table[0, 2] = 10 ** 6
        c.cache.block_table[1, 0] = -1
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = c.call(kernel=kernel, status=status)
        assert int(status) == _cabi.DEV_BAD_BLOCK
        ref.check(got, c, kernel)


# ---- prefill and differential prefill ----------------------------------------------------------------

@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (4, 2), (8, 1), (3, 3)])
def test_prefill_heads_and_types(maps, kv, dim, heads, kv_heads):
    both(ref.make([1, 17, 200, 130, 300], [1, 17, 200, 3, 129], heads=heads, kv_heads=kv_heads, dim=dim, kv=kv, maps=maps), "stream")


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("lens,new", [
    ([1], [1]), ([5], [0]), ([0], [0]), ([0, 3], [0, 3]), ([128], [128]), ([129], [129]), ([127, 256], [127, 255]),
    ([1000], [1000]), ([2000, 5], [3, 5]), ([4096], [1]), ([9000, 8000], [2, 4]), ([64] * 30, [64] * 30),
    ([300, 0, 300], [300, 0, 1]), ([3, 10], [7, 20]), ([0], [4])])
def test_prefill_lengths(maps, lens, new):
    """Among them: no rows, no keys, more rows than keys (the first attend to nothing)."""
    both(ref.make(lens, new, heads=4, kv_heads=2, dim=128, kv="bf16", maps=maps, seed=sum(lens)), "stream")


@pytest.mark.parametrize("page", [1, 5, 16, 32, 48, 128, 256, 500])
@pytest.mark.parametrize("kv", ["fp16", "fp8_e5m2"])
def test_prefill_pages(page, kv):
    both(ref.make([1, page - 1, page, page + 1, 3 * page + 5], [1, page - 1, 1, page + 1, 2 * page], heads=4, kv_heads=2,
                  page=page, kv=kv), "stream")


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("dim,page,kv,io", [(32, 16, "fp16", None), (256, 16, "bf16", None), (64, 16, "fp16", torch.bfloat16),
                                            (128, 16, "bf16", torch.float16), (32, 16, "int8", None)])
def test_prefill_on_the_general_kernel(maps, dim, page, kv, io):
    both(ref.make([30, 40, 133], [30, 4, 20], heads=3, kv_heads=1, dim=dim, page=page, kv=kv, io=io, maps=maps), "simple")


@pytest.mark.parametrize("how", [dict(norm=False), dict(weight=False), dict(lam="float"), dict(lam="rows"), dict(interleaved=True)])
@pytest.mark.parametrize("dim", [64, 128])
def test_diff_prefill_options(how, dim):
    both(ref.make([90, 200, 61], [90, 5, 40], heads=4, kv_heads=2, dim=dim, maps=2, seed=8, **how), "stream")


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("kernel", ["simple", "auto"])
def test_rows_of_nobody_are_left_as_they_were(maps, kernel):
    c = ref.make([50, 20], [30, 20], heads=4, kv_heads=2, dim=64, maps=maps)
    pad = torch.zeros((70, *c.q.shape[1:]), dtype=c.q.dtype, device="cuda")
    pad[:50] = c.q
    c.q = pad
    out = torch.full((70, 4, 64 * maps), 7.0, dtype=torch.float16, device="cuda")
    got = c.call(out=out, kernel=kernel)
    assert got.data_ptr() == out.data_ptr() and (out[50:] == 7.0).all()
    ref.check(got, c)


@pytest.mark.parametrize("kernel", ["simple", "auto"])
@pytest.mark.parametrize("kv,page", [("fp16", 16), ("bf16", 5), ("int8", 16), ("fp8_e5m2", 7)])
def test_prefill_bad_blocks_are_left_out_and_flagged(kernel, kv, page):
    """The last of the lengths passes more blocks than the kernel keeps masks of."""
    for maps in (1, 2):
        c = ref.make([300, 64, 2500], [300, 10, 20], heads=4, kv_heads=2, dim=64, kv=kv, page=page, maps=maps)
        c.cache.block_table[2, 1] = -3
        c.cache.block_table[0, 3] = 10 ** 6
        c.cache.block_table[1, 0] = -1
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = c.call(kernel=kernel, status=status)
        assert int(status) == _cabi.DEV_BAD_BLOCK
        ref.check(got, c, kernel)


@pytest.mark.parametrize("kernel", ["simple", "auto"])
def test_prefill_length_beyond_the_table_is_cut_and_flagged(kernel):
    c = ref.make([32, 40], [4, 40], heads=4, kv_heads=2, dim=64, table_extra=0)
    c.cache.seq_lens[1] = 1000  # the row names 48 tokens; the last eight lie in the page but were never written
    c.cache.k_cache.nan_to_num_(0.0)
    c.cache.v_cache.nan_to_num_(0.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = c.call(kernel=kernel, status=status)
    assert int(status) == _cabi.DEV_BAD_BLOCK
    c.cache.seq_lens[1] = 48
    ref.check(got, c, kernel)


def test_prefill_sm_scale_and_layouts():
    c = ref.make([90, 200], [90, 20], heads=6, kv_heads=2, dim=64)
    c.sm_scale = 0.3
    r = both(c)
    turned = c.q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    padded = torch.full((110, 8, 80), 9.0, dtype=torch.float16, device="cuda")
    c.q = turned
    for kernel in ("simple", "auto"):
        padded.fill_(9.0)
        ref.check(c.call(out=padded[:, 1:7, 8:72], kernel=kernel), c, kernel, r)
        padded[:, 1:7, 8:72] = 9.0
        assert (padded == 9.0).all()
    odd = torch.empty(110 * 6 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(110, 6, 64)  # 2-byte aligned only
    odd.copy_(turned)
    c.q = odd
    ref.check(c.call(), c, "odd", r)


@pytest.mark.parametrize("kv", ["fp16", "bf16", "int8", "fp8_e5m2"])
def test_prefill_large_scores(kv):
    """Scores of some hundreds: the running maximum moves, probabilities underflow."""
    for maps in (1, 2):
        c = ref.make([700], [400], heads=2, kv_heads=1, dim=64, kv=kv, maps=maps, norm=False)
        c.q *= 16
        both(c)


@pytest.mark.parametrize("dim", [64, 128])
def test_unscaled_fp8_pages(dim):
    for maps in (1, 2):
        both(ref.make([1, 17, 200, 300], [1, 17, 3, 129], heads=4, kv_heads=2, dim=dim, kv="fp8_e5m2", scaled=False, maps=maps), "stream")
    both(ref.make([1, 17, 0, 333], heads=4, kv_heads=2, dim=dim, kv="fp8_e5m2", scaled=False, maps=2), "stream")


@pytest.mark.parametrize("maps", [1, 2])
def test_prefill_many_requests(maps):
    """More requests than one probe of 32 finds, some without rows or keys."""
    lens = [(i * 7) % 23 for i in range(1100)]
    new = [n if i % 3 else min(n, 1) for i, n in enumerate(lens)]
    both(ref.make(lens, new, heads=2, kv_heads=1, dim=64, maps=maps), "stream")


@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("maps", [1, 2])
def test_prefill_split_contexts_of_different_lengths(maps, kv):
    """Few rows and long keys: the keys are split, the short request has fewer pieces than there are splits."""
    both(ref.make([20000, 130, 7000, 0], [3, 4, 130, 0], heads=4, kv_heads=2, dim=128, kv=kv, maps=maps), "stream")


def test_out_may_be_q():
    c = ref.make([300, 40], [200, 40], heads=4, kv_heads=2, dim=64)
    r = ref.reference(c)
    q = c.q
    c.q = q.clone()
    ref.check(c.call(out=c.q), c, "in place", r)


def test_empty_calls():
    c = ref.make([5, 6], [0, 0], heads=2, kv_heads=1, dim=64)
    assert tuple(c.call().shape) == (0, 2, 64)
    c = ref.make([5], heads=2, kv_heads=1, dim=64, maps=2)
    c.q = c.q[:0]
    c.cache.block_table, c.cache.seq_lens = c.cache.block_table[:0], c.cache.seq_lens[:0]
    c.lam = 0.5
    assert tuple(c.call().shape) == (0, 2, 128)


@pytest.mark.parametrize("maps,new", [(1, [40, 3]), (2, [40, 3]), (2, None)])
def test_two_captured_graphs_replayed_side_by_side(maps, new):
    """Each graph has its own scratch: replays on two streams at once give what single calls give."""
    cases = [ref.make([2000, 900], new, heads=4, kv_heads=2, dim=64, maps=maps, seed=s) for s in (1, 2)]
    want = [c.call() for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.call())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("maps,new", [(1, [40, 3]), (2, None)])
def test_calls_on_two_streams_at_once(maps, new):
    cases = [ref.make([3000, 900], new, heads=4, kv_heads=2, dim=64, maps=maps, seed=s) for s in (1, 2)]
    want = [c.call() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.call())
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_a_pool_beyond_32_bit_offsets():
    """A page whose elements lie past 2^31 of the pool."""
    page, hkv, d = 256, 8, 128
    blocks = 2 ** 31 // (page * hkv * d) + 8
    k = torch.zeros((blocks, page, hkv, d), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in (k, v):
        t[-3:] = torch.randn((3, page, hkv, d), generator=g, device="cuda").half()
    table = torch.tensor([[blocks - 1, blocks - 3, blocks - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    cache = pda.PagedKVCache(pda.ModelShape(8, 8, d, "far"), page, "fp16", k, v, None, None, table, lens)
    starts = torch.tensor([0, 50], dtype=torch.int32, device="cuda")
    q = torch.randn((50, 8, d), generator=g, device="cuda").half()
    both(ref.Case(q, cache, starts))
    both(ref.Case(q.view(50, 4, 2, d), cache, starts, lam=0.4, maps=2))
    both(ref.Case(q.view(50, 4, 2, d)[:1], cache, None, lam=0.4, maps=2))


# ---- together ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("maps", [1, 2])
def test_a_serving_run(kv, maps):
    """Prompts, then single tokens, each step planned, written and attended to on the GPU; at the end every
    request's cache holds what was written and its last result is that of its whole history."""
    page, d, heads, hk, b = 16, 64, 4 * maps, 2 * maps, 5
    g = torch.Generator(device="cuda").manual_seed(4)
    pool = 60
    shape = (pool, page, hk, d)
    store = pda.torch_dtype(kv)
    k, v = torch.zeros(shape, dtype=store, device="cuda"), torch.zeros(shape, dtype=store, device="cuda")
    ks, vs = (torch.zeros(shape[:3], dtype=torch.float16, device="cuda") for _ in range(2)) if kv == "int8" else (None, None)
    table = torch.zeros((b, 12), dtype=torch.int32, device="cuda")
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    free = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    left = torch.tensor([pool], dtype=torch.int32, device="cuda")
    history = [([], []) for _ in range(b)]
    for step in ([20, 1, 47, 16, 33], [1] * b, [1, 0, 1, 1, 1], [1] * b, [3, 1, 1, 40, 2]):
        new = torch.tensor(step, dtype=torch.int32, device="cuda")
        n = sum(step)
        plan = pda.plan_step(table, lens, new, free, left, block_size=page, num_tokens=n + 3)
        key, value = (torch.randn((n, hk, d), generator=g, device="cuda").half() for _ in range(2))
        cache = pda.PagedKVCache(pda.ModelShape(heads, hk, d, "run"), page, kv, k, v, ks, vs, table, plan.seq_lens)
        pda.cache_write(key, value, cache, plan.slot_mapping)
        q = torch.randn((n, heads, d), generator=g, device="cuda").half()
        at = 0
        for r, m in enumerate(step):
            history[r][0].append(key[at:at + m])
            history[r][1].append(value[at:at + m])
            at += m
        if maps == 2:
            c = ref.Case(q.view(n, heads // 2, 2, d), cache, plan.query_start_loc, lam=0.5, maps=2)
        else:
            c = ref.Case(q, cache, plan.query_start_loc)
        ref.check(c.call(), c, "prefill")
        if step == [1] * b:
            c.starts = None
            if maps == 2:
                ref.check(c.call(), c, "decode")
            else:
                one = pda.paged_decode(q, cache)
                c.starts = plan.query_start_loc
                out, _ = ref.reference(c)
                assert float((one.double() - out).abs().max()) < 2e-3
        lens, left = plan.seq_lens, plan.num_free
    for r in range(b):
        hk_, hv_ = torch.cat(history[r][0]), torch.cat(history[r][1])
        n = int(lens[r])
        assert n == hk_.shape[0]
        got_k, got_v, _ = ref.dense(cache, r, n)
        for x, y in ((got_k, hk_), (got_v, hv_)):
            if kv == "fp16":
                assert torch.equal(x, y.double())
            else:  # int8: half a step of the row's scale, and the scale's own rounding (2^-11 of 127 steps)
                peak = y.double().abs().amax(-1, keepdim=True)
                assert ((x - y.double()).abs() <= peak / 127 * (0.5 + 127 * 2.0 ** -11) + 1e-6).all()
