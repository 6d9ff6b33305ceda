"""plan_step against a plain restatement in Python integers: all outputs are whole numbers and have
to be equal."""

from __future__ import annotations

import random

import pytest
import torch

import paged_decode_attention_b200 as pda
from paged_decode_attention_b200 import _cabi

pytestmark = pytest.mark.gpu


def plain(table, ctx, new, free, num_free, page, tokens):
    table = [list(r) for r in table]
    num_free = min(max(num_free, 0), len(free))
    width = len(table[0]) if table else 0
    upto, taken, ok = 0, 0, True
    slots, positions, starts, lens = [], [], [0], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        held, want = -(-c // page), -(-(c + n) // page)
        before, served = upto, False
        if want <= width:
            upto += want - held
            served = want == held or upto <= num_free
        if served:
            for k in range(want - held):
                table[b][held + k] = free[num_free - 1 - (before + k)]
            if want > held:
                taken = upto
        ok = ok and served
        for p in range(c, c + n):
            block = table[b][p // page] if served else -1
            slots.append(block * page + p % page if block >= 0 else -1)
            positions.append(p)
        starts.append(starts[-1] + n)
        lens.append(c + n if served else c)
    slots, positions = slots[:tokens], positions[:tokens]
    slots += [-1] * (tokens - len(slots))
    positions += [0] * (tokens - len(positions))
    return table, slots, positions, starts, lens, num_free - taken, ok


def run_both(table, ctx, new, free, num_free, page, tokens, **kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    t = i32(table)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    plan = pda.plan_step(t, i32(ctx), i32(new), i32(free), i32([num_free]), block_size=page, num_tokens=tokens,
                         status=status, **kw)
    want = plain(table, ctx, new, free, num_free, page, tokens)
    got = (t.tolist(), plan.slot_mapping.tolist(), plan.positions.tolist(), plan.query_start_loc.tolist(),
           plan.seq_lens.tolist(), int(plan.num_free), int(status) == 0)
    for name, g, w in zip(("table", "slots", "positions", "starts", "lens", "num_free", "served"), got, want):
        assert g == w, name
    assert int(status) in (0, _cabi.DEV_NO_BLOCKS)


def draw(rng, batch, page, ctx_hi, new_hi, slack=3, width_extra=0):
    ctx = [rng.randint(0, ctx_hi) for _ in range(batch)]
    new = [rng.randint(0, new_hi) for _ in range(batch)]
    held = [-(-c // page) for c in ctx]
    want = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    width = max(1, max(want) + width_extra)
    need = sum(w - h for w, h in zip(want, held))
    ids = list(range(sum(held) + need + max(slack, 0)))
    rng.shuffle(ids)
    table = [[-7] * width for _ in range(batch)]
    at = 0
    for b, h in enumerate(held):
        table[b][:h] = ids[at:at + h]
        at += h
    free = ids[at:]
    return table, ctx, new, free, need + slack


@pytest.mark.parametrize("batch,page,ctx_hi,new_hi,pad", [
    (1, 16, 0, 1, 0), (1, 1, 5, 3, 2), (3, 16, 40, 1, 0), (24, 16, 160, 1, 8), (256, 32, 4000, 1, 0), (64, 16, 1000, 400, 5),
    (33, 7, 50, 90, 3), (513, 16, 33, 2, 1), (2000, 8, 20, 3, 0), (8192, 16, 40, 2, 7), (5, 64, 100, 20000, 0)])
def test_matches_the_plain_form(batch, page, ctx_hi, new_hi, pad):
    rng = random.Random(batch * 131 + page)
    table, ctx, new, free, num_free = draw(rng, batch, page, ctx_hi, new_hi)
    run_both(table, ctx, new, free, num_free, page, sum(new) + pad)


@pytest.mark.parametrize("batch,missing", [(1, 1), (5, 1), (40, 20), (300, 200)])
def test_an_exhausted_pool_serves_requests_in_order(batch, missing):
    rng = random.Random(batch)
    table, ctx, new, free, num_free = draw(rng, batch, 16, 60, 50, slack=0)
    run_both(table, ctx, new, free, max(0, num_free - missing), 16, sum(new))


def test_edges():
    # nothing new, everything new, a full row, a row without room, negative counts, an empty pool
    run_both([[3, 4], [5, 6]], [32, 0], [0, 0], [], 0, 16, 0)
    run_both([[3, 4], [5, 6]], [32, 0], [0, 0], [], 0, 16, 4)
    run_both([[0, 0], [0, 0]], [0, 0], [32, 17], [9, 8, 7, 6], 4, 16, 49)
    run_both([[3, 4], [5, 6], [1, 2]], [32, 16, 3], [1, 2, 1], [9, 8, 7], 3, 16, 4)
    run_both([[3, 4], [5, 6]], [-4, 20], [5, -2], [9, 8], 2, 16, 5)
    run_both([[3], [5]], [4, 9], [1, 1], [], 0, 16, 2)
    run_both([[3], [-1]], [4, 9], [1, 1], [2], -5, 16, 2)  # a count below zero is none, an unset entry gives no slot
    run_both([[3], [5]], [16, 9], [0, 9], [2], 7, 16, 9)  # a count beyond the list is the list
    # fewer per-token entries than tokens: the rest is cut off
    run_both([[0, 0, 0]], [5], [30], [9, 8, 7, 6], 4, 16, 11)


def test_lengths_near_the_largest_are_refused_not_wrapped():
    big = 2 ** 31 - 1
    run_both([[3, 4], [5, 6]], [big, 1], [0, 1], [9, 8], 2, 16, 1)


def test_odd_addresses_and_strided_rows():
    rng = random.Random(3)
    table, ctx, new, free, num_free = draw(rng, 9, 16, 100, 30)
    tokens = sum(new)
    wide = torch.full((9, len(table[0]) + 5), -9, dtype=torch.int32, device="cuda")
    t = wide[:, 2:2 + len(table[0])]
    t.copy_(torch.tensor(table, dtype=torch.int32))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    store = torch.full((2 * tokens + 3,), 5, dtype=torch.int64, device="cuda")
    out = pda.StepPlan(store[1:1 + tokens], store[2 + tokens:2 + 2 * tokens], i32([0] * 10), i32([0] * 9), i32([0]))
    pda.plan_step(t, i32(ctx), i32(new), i32(free), i32([num_free]), block_size=16, num_tokens=tokens, out=out)
    want = plain(table, ctx, new, free, num_free, 16, tokens)
    assert t.tolist() == want[0] and out.slot_mapping.tolist() == want[1] and out.positions.tolist() == want[2]
    assert store[0] == 5 and store[1 + tokens] == 5 and store[-1] == 5
    assert (wide[:, :2] == -9).all() and (wide[:, -3:] == -9).all()


def test_a_captured_step_carries_its_state_on():
    """seq_lens and num_free updated in place: each replay is the next step."""
    b, page, steps = 70, 4, 9
    rng = random.Random(1)
    ctx = [rng.randint(0, 30) for _ in range(b)]
    held = [-(-c // page) for c in ctx]
    ids = list(range(sum(held) + b * 4))
    rng.shuffle(ids)
    table = [[0] * 12 for _ in range(b)]
    at = 0
    for r, h in enumerate(held):
        table[r][:h] = ids[at:at + h]
        at += h
    free = ids[at:]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    t, lens, new, f, left = i32(table), i32(ctx), i32([1] * b), i32(free), i32([len(free)])
    out = pda.StepPlan(torch.zeros(b, dtype=torch.int64, device="cuda"), torch.zeros(b, dtype=torch.int64, device="cuda"),
                       i32([0] * (b + 1)), lens, left)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pda.plan_step(t, lens, new, f, left, block_size=page, num_tokens=b, out=out)
    count = len(free)
    for _ in range(steps):
        table, slots, positions, _, ctx, count, _ = plain(table, ctx, [1] * b, free, count, page, b)
        graph.replay()
        assert t.tolist() == table and out.slot_mapping.tolist() == slots and out.positions.tolist() == positions
        assert lens.tolist() == ctx and int(left) == count


def test_on_a_stream_of_its_own():
    rng = random.Random(5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        table, ctx, new, free, num_free = draw(rng, 30, 16, 200, 10)
        run_both(table, ctx, new, free, num_free, 16, sum(new))
