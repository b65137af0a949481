"""Shared by the paged-cache tests: caches with poisoned unused rows, page tables, and plain 64-bit forms."""
from __future__ import annotations

import torch

D = 128
E4M3 = torch.float8_e4m3fn
TINY = 2.0 ** -100


def half_step(t):
    """Largest relative error of one rounding to t."""
    return {E4M3: 2.0 ** -4}.get(t) or torch.finfo(t).eps / 2


def empty_cache(pages, page_size, hk, dtype, layout="hnd", fill=float("nan")):
    """(k, v, k_scale, v_scale) filled with `fill`."""
    def one(shape, dt):
        n, ps, h = shape
        tail = (D,) if dt is not torch.float32 else ()
        if layout == "nhd":
            t = torch.empty(n, ps, h, *tail, dtype=dt, device="cuda")
        else:
            t = torch.empty(n, h, ps, *tail, dtype=dt, device="cuda").transpose(1, 2)
        t.copy_(torch.full((), fill, device="cuda").to(dt))
        return t
    shape = (pages, page_size, hk)
    s = (one(shape, torch.float32), one(shape, torch.float32)) if dtype is E4M3 else (None, None)
    return one(shape, dtype), one(shape, dtype), *s


def quantise(x):
    """x in fp32 -> (codes, scale), the definition."""
    amax = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return (x * (448.0 / amax)).to(E4M3), (amax / 448.0).squeeze(-1)


def fill_sequences(lens, hq, hk, dtype, cache_dtype, page_size, layout="hnd", seed=0, spare=2, k_gain=1.0, room=0):
    """Random sequences in pages of mixed order.  Rows that no sequence holds are NaN; table entries behind a sequence point
    outside the cache, and the table is wide enough for `room` tokens.  Returns a dict with the caches, table, lengths, q, and the rows' values in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-n // page_size) for n in lens]
    pages = sum(counts) + spare
    k, v, ks, vs = empty_cache(pages, page_size, hk, cache_dtype, layout)
    order = torch.randperm(pages, generator=g, device="cuda")
    width = max(max(counts) + 1, -(-room // page_size))
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32, device="cuda")
    rows = []
    used = 0
    for b, n in enumerate(lens):
        table[b, :counts[b]] = order[used:used + counts[b]].to(torch.int32)
        used += counts[b]
        pos = torch.arange(n, device="cuda")
        page, at = table[b].long()[pos // page_size], pos % page_size
        got = []
        for cache, scale, gain in ((k, ks, k_gain), (v, vs, 1.0)):
            x = torch.randn(n, hk, D, generator=g, device="cuda") * gain
            if scale is None:
                cache[page, at] = x.to(cache.dtype)
                got.append(x.to(cache.dtype).double())
            else:
                x = x * torch.exp2(3 * torch.randn(n, hk, 1, generator=g, device="cuda"))  # rows of different sizes
                codes, s = quantise(x)
                cache.view(torch.uint8)[page, at] = codes.view(torch.uint8)
                scale[page, at] = s
                got.append(codes.double() * s.double()[..., None])
        rows.append(got)
    q = (1.5 * torch.randn(len(lens), hq, D, generator=g, device="cuda")).to(dtype)
    return dict(k=k, v=v, k_scale=ks, v_scale=vs, page_table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                q=q, rows=rows, pages=pages)


def attend64(q, k, v, sm_scale=D ** -0.5):
    """One token's attention in 64 bits.  q (hq, D); k, v (n, hk, D).  Returns out, lse and, for the tolerances, sum p |v| and
    the largest sum_d |q_d k_d| * sm_scale of each head."""
    hq, hk = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        z = torch.zeros(hq, D, dtype=torch.float64, device=q.device)
        return z, torch.full((hq,), -float("inf"), dtype=torch.float64, device=q.device), z, z[:, 0]
    qd = q.double().view(hk, hq // hk, D)
    s = torch.einsum("hgd,nhd->hgn", qd, k) * sm_scale
    size = (torch.einsum("hgd,nhd->hgn", qd.abs(), k.abs()) * abs(sm_scale)).amax(-1).reshape(hq)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    p = w / total
    flat = lambda x: x.reshape(hq, -1)
    return (flat(torch.einsum("hgn,nhd->hgd", p, v)), flat(top + torch.log(total))[:, 0],
            flat(torch.einsum("hgn,nhd->hgd", p, v.abs())), size)


def decode_bounds(ref, lse, weight, size, n, dtype, cache_dtype, q, k, v, sm_scale=D ** -0.5):
    """Tolerances of out and lse from the roundings the kernel makes:
      score: 128 products summed in fp32 and a few factors, at most (128 + 6) 2^-24 of sum |q_d k_d|, and for an e4m3 cache
        q's own step as fp16 below 2^-14 of its largest element, 2^-24 of that element for each d;
      exp2: 2^-22 relative, and its argument's rounding 2^-23 |s| (s in log2 units, bounded by the size of the score);
      weights: two bf16 parts 2^-16, two fp16 parts 2^-21, one fp16 part (e4m3 to bf16) 2^-11, and fp16 steps of 2^-25 against
        a largest weight of 2^15 times the row's V scale;
      sums over n tokens in fp32: n 2^-24;  output: one rounding to its type."""
    if n == 0:
        return torch.zeros_like(ref), torch.zeros_like(lse)
    ds = 2.0 ** -24 * (134 + 2 * 1.4427) * size
    if cache_dtype is E4M3:
        hq, hk = q.shape[0], k.shape[1]
        per_head = k.abs().sum(-1).amax(0).repeat_interleave(hq // hk)
        ds = ds + 2.0 ** -24 * q.double().abs().amax(-1) * per_head * abs(sm_scale)
    sums = (n + 16) * 2.0 ** -24
    rel = 2 * ds + sums + 2.0 ** -21
    fp16 = dtype is torch.float16 or cache_dtype is E4M3
    wstep = 2.0 ** -11 if dtype is torch.bfloat16 and fp16 else 2.0 ** -21 if fp16 else 2.0 ** -16
    top = v.abs().amax().item()
    out_tol = half_step(dtype) * ref.abs() + (rel[:, None] + wstep) * weight + (n * 2.0 ** -40 * top if fp16 else 0.0) + \
        2.0 ** -25 * (dtype is torch.float16)
    return out_tol * 1.001 + 1e-30, ds + sums + 2.0 ** -20 + 2.0 ** -22 * lse.abs()
