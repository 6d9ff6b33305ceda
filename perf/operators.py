"""Operators around a paged KV cache, with their plain forms: what a serving step needs besides
single-token attention.

  plan          block tables, slot maps, positions and lengths of one step, from request lengths
  diff_decode   differential attention of one new token per request over the paged cache
  prefill       causal attention of many new tokens per request over the paged cache
  diff_prefill  the same for differential attention

``run`` computes the plain forms in elementary torch operations, in 32 bits, or (``own``) calls the
package.  ``exact`` restates the definitions in 64 bits, request by request.
"""

import math
import random

import torch

own = False

EPS = 1e-5
OUT_SCALE = 0.2  # 1 - lambda_init of a deep layer


def listed():
    return [
        # one decode step of a ragged serving batch: every request gets one token
        {"name": "plan_decode_b256", "op": "plan", "batch": 256, "page": 32, "ctx_lo": 1, "ctx_hi": 32768,
         "new_lo": 1, "new_hi": 1},
        # a step that admits prompts beside chunks of longer ones: tens of thousands of slots
        {"name": "plan_prompts_b64", "op": "plan", "batch": 64, "page": 16, "ctx_lo": 0, "ctx_hi": 4096,
         "new_lo": 1, "new_hi": 2048},
        # a small model's chat batch: 1.4 MB of cache, latency counts
        {"name": "diff_decode_small_fp16", "op": "diff_decode", "batch": 24, "pairs": 7, "kv_pairs": 1, "dim": 64,
         "page": 16, "kv": "fp16", "ctx_lo": 64, "ctx_hi": 160},
        # a medium batch with grouped heads: 1.4 GB of cache streamed once
        {"name": "diff_decode_b64_fp16", "op": "diff_decode", "batch": 64, "pairs": 16, "kv_pairs": 4, "dim": 128,
         "page": 16, "kv": "fp16", "ctx_lo": 2048, "ctx_hi": 8192},
        # int8 cache with a scale for each token and head, eight query pairs to a kv pair
        {"name": "diff_decode_b32_int8", "op": "diff_decode", "batch": 32, "pairs": 32, "kv_pairs": 4, "dim": 128,
         "page": 16, "kv": "int8", "ctx_lo": 1000, "ctx_hi": 4096},
        # two long documents in scaled fp8: the cache's length has to be split over the machine
        {"name": "diff_decode_long_fp8", "op": "diff_decode", "batch": 2, "pairs": 16, "kv_pairs": 4, "dim": 128,
         "page": 16, "kv": "fp8_e5m2", "ctx_lo": 131072, "ctx_hi": 131072},
        # a chat batch's first step: short prompts of a small model, nothing cached yet
        {"name": "prefill_short_fp16", "op": "prefill", "batch": 24, "heads": 14, "kv_heads": 2, "dim": 64,
         "page": 16, "kv": "fp16", "ctx_lo": 0, "ctx_hi": 0, "new_lo": 64, "new_hi": 160},
        # one long prompt at once: the matrix products bound it
        {"name": "prefill_8192_bf16", "op": "prefill", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "kv": "bf16", "ctx_lo": 0, "ctx_hi": 0, "new_lo": 8192, "new_hi": 8192},
        # chunks of prompts behind what is cached, int8 pages, ragged
        {"name": "prefill_chunks_int8", "op": "prefill", "batch": 6, "heads": 28, "kv_heads": 4, "dim": 128,
         "page": 32, "kv": "int8", "ctx_lo": 1024, "ctx_hi": 16384, "new_lo": 100, "new_hi": 512},
        # drafted tokens of a few requests checked against long contexts: few rows, a long axis
        {"name": "diff_prefill_drafts_fp16", "op": "diff_prefill", "batch": 4, "pairs": 16, "kv_pairs": 4, "dim": 64,
         "page": 16, "kv": "fp16", "ctx_lo": 16384, "ctx_hi": 32768, "new_lo": 3, "new_hi": 5},
        # ragged prompts of a differential model whose value heads are 128 wide
        {"name": "diff_prefill_b4_bf16", "op": "diff_prefill", "batch": 4, "pairs": 16, "kv_pairs": 4, "dim": 64,
         "page": 16, "kv": "bf16", "ctx_lo": 0, "ctx_hi": 0, "new_lo": 500, "new_hi": 2048},
        # one prompt with value heads 256 wide
        {"name": "diff_prefill_4096_fp16", "op": "diff_prefill", "batch": 1, "pairs": 16, "kv_pairs": 4, "dim": 128,
         "page": 32, "kv": "fp16", "ctx_lo": 0, "ctx_hi": 0, "new_lo": 4096, "new_hi": 4096},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "diff_decode", "diff_decode", "prefill", "prefill", "diff_prefill", "diff_prefill"])
    page = rng.choice([16, 32, 64])
    if op == "plan":
        new_hi = _log_between(rng, 1, 1500)
        return {"op": op, "batch": _log_between(rng, 1, 400 if new_hi < 100 else 64), "page": page, "ctx_lo": rng.randint(0, 50),
                "ctx_hi": _log_between(rng, 51, 20000), "new_lo": rng.randint(0, 1), "new_hi": new_hi}
    dim = rng.choice([64, 128])
    kv = rng.choice(["fp16", "bf16", "int8", "fp8_e5m2"])
    kv_heads = rng.choice([1, 2, 3, 4])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    if op == "diff_decode":
        # at most 300 000 tokens of at most four pairs of heads
        batch = _log_between(rng, 1, 100)
        hi = max(2, min(100000, _log_between(rng, 30, 300000) // batch))
        return {"op": op, "batch": batch, "pairs": kv_heads * group, "kv_pairs": kv_heads, "dim": dim, "page": page,
                "kv": kv, "ctx_lo": rng.randint(1, hi), "ctx_hi": hi}
    # new tokens times keys times query heads stay below those of one long prompt
    batch = _log_between(rng, 1, 24)
    new_hi = max(1, min(4000, _log_between(rng, 2, 6000) // batch))
    ctx_hi = rng.choice([0, max(1, min(16000, _log_between(rng, 16, 60000) // batch))])
    while batch * new_hi * (new_hi + ctx_hi) * kv_heads * group > 4e8:
        new_hi, ctx_hi = max(1, new_hi * 2 // 3), ctx_hi * 2 // 3
    case = {"op": op, "batch": batch, "dim": dim, "page": page, "kv": kv, "ctx_lo": rng.randint(0, ctx_hi), "ctx_hi": ctx_hi,
            "new_lo": rng.randint(1, new_hi), "new_hi": new_hi}
    if op == "prefill":
        return dict(case, heads=kv_heads * group, kv_heads=kv_heads)
    return dict(case, pairs=kv_heads * group, kv_pairs=kv_heads)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _spread(what, lo, hi, n):
    """n lengths in [lo, hi], log-uniform, a function of the case alone."""
    r = random.Random("%s %d %d %d" % (what, lo, hi, n))
    return [min(hi, max(lo, int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1)))) - 1))) for _ in range(n)]


def _lengths(case):
    """(tokens already cached, new tokens) of each request."""
    ctx = _spread("ctx", case["ctx_lo"], case["ctx_hi"], case["batch"])
    if "new_lo" not in case:
        return ctx, [0] * len(ctx)
    return ctx, _spread("new", case["new_lo"], case["new_hi"], case["batch"])


_STORED = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "fp8_e5m2": torch.float8_e5m2}


def _pages(gen, kv, shape):
    if kv == "int8":
        return torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).to(_STORED[kv])


def _scales(gen, kv, shape):
    if kv == "int8":
        return (torch.randn(shape, generator=gen, device="cuda").abs() / 127.0 + 1e-4).half()
    if kv == "fp8_e5m2":
        return (torch.rand(shape, generator=gen, device="cuda") * 1.5 + 0.5).half()
    return None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.Generator(device="cpu").manual_seed(seed)
    ctx, new = _lengths(case)
    perm = torch.randperm(len(ctx), generator=order).tolist()
    ctx, new = [ctx[i] for i in perm], [new[i] for i in perm]
    page, op = case["page"], case["op"]
    s = {"op": op, "page": page, "case": case}
    if op == "plan":
        held = [-(-c // page) for c in ctx]
        width = max(1, max(-(-(c + n) // page) for c, n in zip(ctx, new)))
        need = sum(-(-(c + n) // page) - h for c, n, h in zip(ctx, new, held))
        pool = torch.randperm(sum(held) + need + 17, generator=order).to(torch.int32)
        table = torch.zeros(len(ctx), width, dtype=torch.int32)
        at = 0
        for row, h in enumerate(held):
            table[row, :h] = pool[at:at + h]
            at += h
        s.update(table=table.cuda(), ctx=torch.tensor(ctx, dtype=torch.int32).cuda(),
                 new=torch.tensor(new, dtype=torch.int32).cuda(), free=pool[at:].contiguous().cuda(),
                 num_free=torch.tensor([need + 17], dtype=torch.int32).cuda(), tokens=sum(new))
        return s
    diff = op.startswith("diff")
    heads, kv_heads = (2 * case["pairs"], 2 * case["kv_pairs"]) if diff else (case["heads"], case["kv_heads"])
    d, kv = case["dim"], case["kv"]
    lens = [c + n for c, n in zip(ctx, new)]
    pages = [-(-n // page) for n in lens]
    used = sum(pages)
    blocks = torch.randperm(used, generator=order).to(torch.int32)
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32)
    at = 0
    for row, n in enumerate(pages):
        table[row, :n] = blocks[at:at + n]
        at += n
    shape = (used, page, kv_heads, d)
    s.update(table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda(), k=_pages(gen, kv, shape),
             v=_pages(gen, kv, shape), ks=_scales(gen, kv, shape[:3]), vs=_scales(gen, kv, shape[:3]), kv=kv,
             heads=heads, kv_heads=kv_heads, d=d, max_len=max(lens), max_new=max(new))
    rows = len(lens) if op == "diff_decode" else sum(new)
    io = torch.bfloat16 if kv == "bf16" else torch.float16
    q = torch.randn((rows, heads, d), generator=gen, device="cuda").to(io)
    if diff:
        s["lam"] = torch.rand(case["pairs"], generator=gen, device="cuda") * 0.6 + 0.2
        s["weight"] = 1 + 0.1 * torch.randn(2 * d, generator=gen, device="cuda")
        q = q.view(rows, case["pairs"], 2, d)
    s["q"] = q
    if op != "diff_decode":
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
    return s


# ---------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------

def run(s):
    return _calls(s) if own else _plain(s)


def _calls(s):
    import paged_decode_attention_b200 as pda

    if s["op"] == "plan":
        plan = pda.plan_step(s["table"], s["ctx"], s["new"], s["free"], s["num_free"], block_size=s["page"],
                             num_tokens=s["tokens"])
        return {"table": s["table"], "slots": plan.slot_mapping, "positions": plan.positions,
                "starts": plan.query_start_loc, "lens": plan.seq_lens, "num_free": plan.num_free}
    cache = pda.PagedKVCache(pda.ModelShape(s["heads"], s["kv_heads"], s["d"], "case"), s["page"], s["kv"], s["k"], s["v"],
                             s["ks"], s["vs"], s["table"], s["lens"])
    if s["op"] == "prefill":
        return pda.paged_prefill(s["q"], cache, s["starts"])
    if s["op"] == "diff_decode":
        return pda.paged_diff_decode(s["q"], cache, s["lam"], norm_weight=s["weight"], eps=EPS, out_scale=OUT_SCALE)
    return pda.paged_diff_prefill(s["q"], cache, s["starts"], s["lam"], norm_weight=s["weight"], eps=EPS, out_scale=OUT_SCALE)


def _plain(s):
    if s["op"] == "plan":
        return _plain_plan(s)
    q = s["q"].float()
    if s["op"] == "diff_decode":
        at = torch.arange(q.shape[0], device=q.device)[:, None]  # request b: row b, at its last position
        live = torch.ones_like(at, dtype=torch.bool)
        pos = s["lens"].long()[:, None] - 1
    else:
        starts = s["starts"].long()
        n = starts[1:] - starts[:-1]
        i = torch.arange(s["max_new"], device=q.device)[None]
        live = i < n[:, None]
        at = torch.where(live, starts[:-1, None] + i, 0)
        pos = s["lens"].long()[:, None] - n[:, None] + i
    q = q[at]  # [B, Q, heads.., D]
    out = _attend(s, q, pos)
    if s["op"].startswith("diff"):
        out = out[..., 0, :] - s["lam"][:, None] * out[..., 1, :]
        out = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + EPS) * s["weight"] * OUT_SCALE
    return out[live].to(s["q"].dtype)


def _dense(s, pages, scales):
    """[B, S, heads, D] in 32 bits of the pages that the block table names."""
    t = s["table"].long()
    x = pages[t].float()
    if scales is not None:
        x = x * scales[t].float()[..., None]
    return x.flatten(1, 2)[:, :s["max_len"]]


def _attend(s, q, pos):
    """Causal attention of q [B, Q, H, D] (or [B, Q, H, 2, D]) at positions pos [B, Q]."""
    k, v = _dense(s, s["k"], s["ks"]), _dense(s, s["v"], s["vs"])
    b, n, d = q.shape[0], q.shape[1], s["d"]
    beyond = torch.arange(k.shape[1], device=k.device) > pos[:, :, None]  # [B, Q, S]
    v = torch.where((torch.arange(k.shape[1], device=k.device) < s["lens"][:, None])[:, :, None, None], v, 0)
    if q.dim() == 5:
        hk = k.shape[2] // 2
        q = q.view(b, n, hk, -1, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(b, hk, 2, -1, d)  # rows (group, query)
        k = k.view(b, -1, hk, 2, d).permute(0, 2, 3, 4, 1)
        v = v.view(b, -1, hk, 2 * d).permute(0, 2, 1, 3)[:, :, None]
    else:
        hk = k.shape[2]
        q = q.view(b, n, hk, -1, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
        k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)
    x = torch.matmul(q, k).mul_(d ** -0.5)
    x = x.view(*x.shape[:-2], -1, n, x.shape[-1])  # [.., G, Q, S]
    x.masked_fill_(beyond.view(b, *([1] * (x.dim() - 3)), n, -1), float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.flatten(-3, -2), v).view(*x.shape[:-1], -1) / total
    if o.dim() == 6:  # [B, Hk, 2, G, Q, 2D] -> [B, Q, H, 2, 2D]
        return o.permute(0, 4, 1, 3, 2, 5).flatten(2, 3)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)


def _plain_plan(s):
    table, ctx, new, free, page = s["table"], s["ctx"].long(), s["new"].long(), s["free"], s["page"]
    num_free = s["num_free"].long()
    held, want = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    fits = want <= table.shape[1]
    need = torch.where(fits, want - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= num_free))
    col = torch.arange(table.shape[1], device=table.device)
    k = (upto - need)[:, None] + col - held[:, None]
    fresh = served[:, None] & (col >= held[:, None]) & (col < want[:, None])
    table = torch.where(fresh, free[(num_free - 1 - k).clamp(0, free.numel() - 1)], table)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["tokens"], device=table.device)
    r = torch.searchsorted(starts[1:], t, right=True).clamp(max=ctx.numel() - 1)
    pos = ctx[r] + t - starts[r]
    block = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(served[r], block * page + pos % page, -1)
    taken = torch.where(served, upto, 0).amax()
    lens = torch.where(served, ctx + new, ctx)
    return {"table": table, "slots": slots, "positions": pos, "starts": starts.int(), "lens": lens.int(),
            "num_free": (num_free - taken).int()}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------------------------

_BYTES = {"fp16": 2, "bf16": 2, "int8": 1, "fp8_e5m2": 1}


def work(case):
    ctx, new = _lengths(case)
    b, page, op = case["batch"], case["page"], case["op"]
    if op == "plan":
        # a page's entry is read or written where a new token lies in it
        entries = sum(-(-(c + n) // page) - c // page for c, n in zip(ctx, new) if n)
        return {"bytes": 16 * sum(new) + 4 * entries + 4 * (4 * b + 3), "flops": 0}
    diff = op.startswith("diff")
    hq, hk = (2 * case["pairs"], 2 * case["kv_pairs"]) if diff else (case["heads"], case["kv_heads"])
    d = case["dim"]
    if op == "diff_decode":
        new, rows = [1] * b, b
        lens, pairs_of_keys = ctx, sum(ctx)
    else:
        lens, rows = [c + n for c, n in zip(ctx, new)], sum(new)
        pairs_of_keys = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    token = 2 * hk * (d * _BYTES[case["kv"]] + (2 if case["kv"] in ("int8", "fp8_e5m2") else 0))
    byts = sum(lens) * token + 2 * rows * hq * d * 2 + sum(-(-n // page) for n in lens) * 4 + 8 * b
    return {"bytes": byts, "flops": pairs_of_keys * hq * 2 * (d + (2 * d if diff else d))}


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    q, d, diff = s["q"].double(), s["d"], case["op"].startswith("diff")
    lens = s["lens"].tolist()
    starts = list(range(len(lens) + 1)) if case["op"] == "diff_decode" else s["starts"].tolist()
    rows = []
    for b, n in enumerate(lens):
        ids = s["table"][b, :-(-n // s["page"])].long()
        k, v = s["k"][ids].double(), s["v"][ids].double()
        if s["ks"] is not None:
            k, v = k * s["ks"][ids].double().unsqueeze(-1), v * s["vs"][ids].double().unsqueeze(-1)
        k, v = k.reshape(-1, s["kv_heads"], d)[:n], v.reshape(-1, s["kv_heads"], d)[:n]
        x = q[starts[b]:starts[b + 1]]
        m = x.shape[0]
        hidden = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)

        def soft(query, key):  # [m, D], [n, D]
            w = (query @ key.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            return torch.softmax(w, dim=1)

        outs = []
        if diff:
            group = case["pairs"] // case["kv_pairs"]
            for h in range(case["pairs"]):
                j = h // group
                wide = torch.cat([v[:, 2 * j], v[:, 2 * j + 1]], dim=1)
                o = soft(x[:, h, 0], k[:, 2 * j]) @ wide - s["lam"][h].double() * (soft(x[:, h, 1], k[:, 2 * j + 1]) @ wide)
                o = o / torch.sqrt((o * o).mean(dim=1, keepdim=True) + EPS)
                outs.append(o * s["weight"].double() * OUT_SCALE)
        else:
            group = case["heads"] // case["kv_heads"]
            for h in range(case["heads"]):
                outs.append(soft(x[:, h], k[:, h // group]) @ v[:, h // group])
        rows.append(torch.stack(outs, dim=1))
    return torch.cat(rows)
