"""The definitions of the paged operators in 64 bits, request by request, with bounds on how far a
kernel may be from them (tests only).

Bounds.  Let p_k be the probabilities of one row, A = sum p_k |v_k| and n its number of keys.
  * the result is rounded to its type: u |out| with u = finfo.eps / 2;
  * the kernels on the matrix units round every probability to that type: at most u A; below the
    smallest normal fp16 (relative to the row's largest, which is 1) by at most 2^-25 each, so
    n 2^-25 max|v| / l with l = sum exp(s - max) more;
  * a score is off by ds: D + 8 roundings of 2^-24 in 32 bits, relative to sum |q_i k_i|, and by the
    step of the query digits where int8 keys meet the query in integers (half of max|q| / 16256 per
    element); the exponential adds 2^-21 (two instructions' error); a probability is then off by
    2 (ds + 2^-21) relative, numerator and denominator;
  * 32-bit sums of n terms: n 2^-24 A, twice (numerator and denominator).
Differential: the errors of the maps add up as dx = d1 + |lam| d2, the norm's factor r is off by
r rms(dx) relative to the first order (times 1 + that for the second).
"""

from __future__ import annotations

import dataclasses
import math

import torch

import paged_decode_attention_b200 as pda

U32 = 2.0 ** -24


@dataclasses.dataclass
class Case:
    q: torch.Tensor
    cache: pda.PagedKVCache
    starts: torch.Tensor | None  # None: one row per request
    lam: object = None
    weight: torch.Tensor | None = None
    norm: bool = True
    eps: float = 1e-5
    out_scale: float = 0.2
    maps: int = 1
    sm_scale: float | None = None

    def kwargs(self):
        kw = {} if self.sm_scale is None else {"sm_scale": self.sm_scale}
        if self.maps == 2:
            kw.update(norm=self.norm, norm_weight=self.weight, eps=self.eps, out_scale=self.out_scale)
        return kw

    def call(self, **more):
        kw = {**self.kwargs(), **more}
        if self.maps == 1:
            return pda.paged_prefill(self.q, self.cache, self.starts, **kw)
        if self.starts is None:
            return pda.paged_diff_decode(self.q, self.cache, self.lam, **kw)
        return pda.paged_diff_prefill(self.q, self.cache, self.starts, self.lam, **kw)


def make(lens, new=None, *, heads=8, kv_heads=2, dim=64, page=16, kv="fp16", io=None, maps=1, seed=0, spare=3,
         interleaved=False, table_extra=2, norm=True, weight=True, lam="heads", v_mean=0.0, scaled=True, device="cuda"):
    """A seeded case; ``new`` None makes it single-token.  Heads are counted in pairs for maps = 2.

    Everything the operators must not read is poisoned: tokens behind a request's length and pages
    nobody owns hold NaN (127 in int8), block-table entries behind the last page name no block.
    """
    gen = torch.Generator(device="cpu").manual_seed(seed)
    heads, kv_heads = heads * maps, kv_heads * maps
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + spare
    ids = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(1, max(pages, default=1) + table_extra)), 2 ** 30, dtype=torch.int32)
    dead = torch.ones(pool, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = ids[at:at + n]
        flat = torch.arange(lens[b])
        dead[ids[at:at + n].long()[flat // page], flat % page] = False
        at += n
    stored = pda.torch_dtype(kv)
    ten = []
    for _ in range(2):
        if kv == "int8":
            x = torch.randint(-127, 128, (pool, page, kv_heads, dim), generator=gen).to(torch.int8)
            x[dead] = 127
        else:
            x = torch.randn(pool, page, kv_heads, dim, generator=gen)
            x = (x + v_mean if len(ten) else x).to(stored)
            x.view(torch.uint8 if x.element_size() == 1 else torch.int16)[dead] = 0x7F if x.element_size() == 1 else 0x7FFF
        ten.append(x)
    scales = [None, None]
    if kv == "int8" or (kv == "fp8_e5m2" and scaled):
        for i in range(2):
            s = torch.randn(pool, page, kv_heads, generator=gen).abs() / 127 + 1e-4 if kv == "int8" else \
                torch.rand(pool, page, kv_heads, generator=gen) * 1.5 + 0.5
            s = s.half()
            s[dead] = float("nan")
            scales[i] = s.to(device)
    if interleaved:
        both = torch.stack(ten, dim=1).to(device)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (x.to(device) for x in ten)
    io = io or (torch.bfloat16 if kv == "bf16" else torch.float16)
    rows = len(lens) if new is None else sum(new)
    shape = (rows, heads, dim) if maps == 1 else (rows, heads // 2, 2, dim)
    q = torch.randn(shape, generator=gen).to(io).to(device)
    starts = None
    if new is not None:
        starts = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32).to(device)
    lam_value, w = None, None
    if maps == 2:
        pairs = heads // 2
        lam_value = 0.65 if lam == "float" else torch.rand((rows, pairs) if lam == "rows" else (pairs,), generator=gen).to(device) * 0.6 + 0.2
        w = (1 + 0.3 * torch.randn(2 * dim, generator=gen)).to(device) if weight and norm else None
    cache = pda.PagedKVCache(pda.ModelShape(heads, kv_heads, dim, "case"), page, kv, k, v, scales[0], scales[1],
                             table.to(device), torch.tensor(lens, dtype=torch.int32).to(device))
    return Case(q, cache, starts, lam_value, w, norm, maps=maps)


def dense(cache, b, n):
    """[n, heads, D] keys and values of request b in 64 bits (a block id outside the pool: absent)."""
    page = cache.block_size
    ids = cache.block_table[b, :-(-n // page)].long()
    ok = (ids >= 0) & (ids < cache.num_blocks)
    ids = torch.where(ok, ids, 0)
    k, v = cache.k_cache[ids].double(), cache.v_cache[ids].double()
    if cache.k_scale is not None:
        k, v = k * cache.k_scale[ids].double()[..., None], v * cache.v_scale[ids].double()[..., None]
    h, d = k.shape[2], k.shape[3]
    return k.reshape(-1, h, d)[:n], v.reshape(-1, h, d)[:n], ok.repeat_interleave(page)[:n]


def reference(c: Case):
    """(out, bound): the definition in 64 bits and how far a kernel may be from it, per element; rows
    that belong to nobody are NaN in both."""
    d, maps = c.cache.shape.head_dim, c.maps
    scale = d ** -0.5 if c.sm_scale is None else c.sm_scale
    u = torch.finfo(c.q.dtype).eps / 2
    lens = c.cache.seq_lens.tolist()
    starts = list(range(len(lens) + 1)) if c.starts is None else c.starts.tolist()
    rows, hq = c.q.shape[0], c.q.shape[1]
    out = torch.full((rows, hq, maps * d), float("nan"), dtype=torch.float64, device=c.q.device)
    bound = out.clone()
    group = c.cache.shape.num_q_heads // c.cache.shape.num_kv_heads
    eye = c.cache.k_cache.device
    for b, n in enumerate(lens):
        n = max(n, 0)
        m = starts[b + 1] - starts[b]
        if m <= 0:
            continue
        q = c.q[starts[b]:starts[b + 1]].double()
        k, v, present = dense(c.cache, b, n)
        last = torch.arange(m, device=eye) + n - m  # position of each row
        seen = (torch.arange(n, device=eye)[None] <= last[:, None]) & present[None]

        def soft(x, key, val):
            """One map: (o, error of o) of queries [m, D] against keys [n, D], values [n, W]."""
            if n == 0:
                z = torch.zeros(m, val.shape[1], dtype=torch.float64, device=eye)
                return z, z
            s = x @ key.T * scale
            ds = (d + 8) * U32 * (x.abs() @ key.abs().T) * scale
            if c.cache.kv_dtype == "int8" and c.starts is None:
                ds = ds + scale * x.abs().amax(1, keepdim=True) / 32512 * key.abs().sum(1)
            s = torch.where(seen, s, -math.inf)
            top = s.amax(1, keepdim=True)
            top = torch.where(top.isinf(), 0.0, top)
            e = torch.exp(s - top)
            total = e.sum(1, keepdim=True)
            p = torch.where(total > 0, e / total, 0.0)
            o = p @ val
            a = p @ val.abs()
            off = 2 * (p * (ds + 2.0 ** -21)) @ val.abs() + a * 2 * (p * (ds + 2.0 ** -21)).sum(1, keepdim=True)
            off = off + u * a + 2 * n * U32 * a
            # only the keys the row sees count, and only their values
            top_v = (seen[:, :, None] * val.abs()[None]).amax(1) if m * n * val.shape[1] < 2 ** 24 else val.abs().amax(0)[None]
            return o, off + n * 2.0 ** -25 * top_v / total.clamp_min(1)

        for h in range(hq):
            j = h // group
            if maps == 1:
                o, off = soft(q[:, h], k[:, j], v[:, j])
            else:
                wide = torch.cat([v[:, 2 * j], v[:, 2 * j + 1]], 1)
                o1, e1 = soft(q[:, h, 0], k[:, 2 * j], wide)
                o2, e2 = soft(q[:, h, 1], k[:, 2 * j + 1], wide)
                if isinstance(c.lam, torch.Tensor):
                    lam = c.lam.double().expand(rows, hq)[starts[b]:starts[b + 1], h, None]
                else:
                    lam = torch.tensor(float(torch.tensor(c.lam, dtype=torch.float32)), dtype=torch.float64, device=eye)
                o, off = o1 - lam * o2, e1 + lam.abs() * e2 + 4 * U32 * (o1.abs() + o2.abs())
                factor = torch.full((m, 1), c.out_scale, dtype=torch.float64, device=eye)
                if c.norm:
                    r = torch.rsqrt(o.square().mean(1, keepdim=True) + c.eps)
                    shift = r * off.square().mean(1, keepdim=True).sqrt()
                    off = off + o.abs() * shift * (1 + shift)
                    factor = factor * r
                w = c.weight.double() if c.weight is not None else torch.ones(2 * d, dtype=torch.float64, device=eye)
                o, off = o * factor * w, off * factor.abs() * w.abs() * (1 + 16 * U32)
            out[starts[b]:starts[b + 1], h] = o
            # the last rounding; below the smallest normal fp16 it is absolute
            bound[starts[b]:starts[b + 1], h] = off + u * (o.abs() + off) + (2.0 ** -25 if c.q.dtype == torch.float16 else 0.0)
    return out, bound


def check(got: torch.Tensor, c: Case, what: str = "", ref=None):
    out, bound = reference(c) if ref is None else ref
    mine = ~out.isnan()
    g = got.double()
    assert not g[mine].isnan().any(), f"{what}: NaN"
    over = ((g - out).abs() - bound)[mine]
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{what}: off by {float((g - out).abs()[mine].max()):.3e}, {int((over > 0).sum())} of {over.numel()} beyond their bounds"
