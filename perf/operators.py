"""What is measured of the paged key/value cache: writing rows into it (copied, or quantised to e4m3 with a scale for each
token and head), reading a cached prefix back as contiguous keys and values, and attention of one new token for each
sequence over its pages.

Caches are (pages, page_size, kv_heads, 128); storage is either token-major ("nhd") or head-major within a page ("hnd").
Scales are (pages, page_size, kv_heads) in fp32, stored head-major."""
import random

import torch

own = False

D = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # least absolute maximum that a scale stands for, so that a row of zeros has a scale too
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SLOT_POOL = 65536  # slots of the pool that single tokens are written into


def listed():
    return [
        # one user's chat turn: a short history, where latency is all there is
        dict(name="decode_1x500", op="decode", batch=1, least=500, most=500, q_heads=32, kv_heads=8, dtype="bf16", cache="same",
             layout="nhd", page_size=16),
        # many short chats with few heads on each GPU (a head shard)
        dict(name="decode_256x600_shard", op="decode", batch=256, least=1, most=600, q_heads=8, kv_heads=2, dtype="fp16", cache="same",
             layout="nhd", page_size=16),
        # a serving batch of mixed lengths
        dict(name="decode_64x8k", op="decode", batch=64, least=64, most=8192, q_heads=32, kv_heads=8, dtype="bf16", cache="same",
             layout="nhd", page_size=16),
        # the same for a quantised cache and 7 query heads on each key head, lengths odd
        dict(name="decode_33x16k_e4m3", op="decode", batch=33, least=777, most=16001, q_heads=28, kv_heads=4, dtype="bf16", cache="e4m3",
             layout="hnd", page_size=64),
        # the answer to one long prompt: the headline prefill's length
        dict(name="decode_1x128k", op="decode", batch=1, least=131072, most=131072, q_heads=32, kv_heads=8, dtype="bf16", cache="same",
             layout="hnd", page_size=128),
        # the longest prompts, quantised
        dict(name="decode_2x256k_e4m3", op="decode", batch=2, least=200003, most=262144, q_heads=28, kv_heads=4, dtype="bf16", cache="e4m3",
             layout="hnd", page_size=128),
        # the new tokens of a decode step
        dict(name="write_64_single", op="write", tokens=64, start=0, single=True, q_heads=32, kv_heads=8, dtype="bf16", cache="same",
             layout="nhd", page_size=16),
        # a prompt's chunk that starts inside a page, quantised
        dict(name="write_4099_e4m3", op="write", tokens=4099, start=37, single=False, q_heads=8, kv_heads=2, dtype="fp16", cache="e4m3",
             layout="hnd", page_size=64),
        # a whole long prompt, quantised
        dict(name="write_128k_e4m3", op="write", tokens=131072, start=0, single=False, q_heads=32, kv_heads=8, dtype="bf16", cache="e4m3",
             layout="hnd", page_size=128),
        # a short cached prefix
        dict(name="read_1x700_e4m3", op="read", batch=1, least=700, most=700, kv_heads=2, dtype="fp16", cache="e4m3", layout="hnd",
             page_size=16),
        # prefixes of several sequences, one padded batch
        dict(name="read_7x5k", op="read", batch=7, least=300, most=5003, kv_heads=8, dtype="bf16", cache="same", layout="nhd", page_size=16),
        # a long cached prefix before the next chunk of its prompt
        dict(name="read_1x128k_e4m3", op="read", batch=1, least=131072, most=131072, kv_heads=8, dtype="bf16", cache="e4m3", layout="hnd",
             page_size=128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["decode", "decode", "write", "read"])
    kv_heads = rng.choice([1, 2, 4, 8])
    case = dict(op=op, kv_heads=kv_heads, dtype=rng.choice(["bf16", "fp16"]), cache=rng.choice(["same", "e4m3"]),
                layout=rng.choice(["nhd", "hnd"]), page_size=rng.choice([16, 32, 48, 64, 128, 256]))
    if op == "write":
        single = rng.random() < 0.4
        tokens = _log_int(rng, 1, 1024 if single else 1000000 // kv_heads)
        return dict(case, single=single, tokens=tokens, start=0 if single else rng.randrange(0, 300),
                    q_heads=kv_heads * rng.choice([1, 2, 4, 7, 8]))
    # rows of all sequences and heads together, padded to the longest: up to 2^20 to read, 2^22 to attend over
    rows = 2 ** 20 // kv_heads if op == "read" else 2 ** 21 // kv_heads
    most = _log_int(rng, 1, 200000 if op == "decode" else rows)
    most = min(most, rows)
    batch = _log_int(rng, 1, max(1, min(512, rows // most)))
    case |= dict(batch=batch, most=most, least=rng.randint(1, most))
    return dict(case, q_heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12, 16])) if op == "decode" else case


def _lens(case):
    """Lengths between least and most, spread evenly (fractions of multiples of the golden ratio); the first is the longest."""
    span = case["most"] - case["least"] + 1
    return [case["most"]] + [case["least"] + int(span * ((i * 0.6180339887498949) % 1.0)) for i in range(1, case["batch"])]


def _pages(length, page_size):
    return -(-length // page_size)


def _empty_cache(case, pages, dtype):
    ps, hk = case["page_size"], case["kv_heads"]
    if case["layout"] == "nhd":
        return torch.zeros(pages, ps, hk, D, dtype=dtype, device="cuda")
    return torch.zeros(pages, hk, ps, D, dtype=dtype, device="cuda").transpose(1, 2)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _put_codes(cache, scale, x):
    """Quantises x into a cache that prepare() fills."""
    amax = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    cache.copy_((x * (E4M3_MAX / amax)).to(torch.float8_e4m3fn))
    scale.copy_((amax / E4M3_MAX).squeeze(-1))


def _filled(case, gen, lens):
    """A pool that holds the sequences in pages of mixed order, and the table of their pages. Keys have channels that stand
    out (the same for every token), as rotated keys do."""
    ps, hk = case["page_size"], case["kv_heads"]
    counts = [_pages(n, ps) for n in lens]
    pages = sum(counts) + 3
    dtype = DTYPES[case["dtype"]]
    quant = case["cache"] == "e4m3"
    channels = 2.0 * _normal(gen, hk, D)
    state = {}
    for name, shift in (("k", channels), ("v", 0.0)):
        cache = _empty_cache(case, pages, torch.float8_e4m3fn if quant else dtype)
        scale = torch.zeros(pages, hk, ps, device="cuda").transpose(1, 2) if quant else None
        step = max(1, (1 << 27) // (ps * hk * D))
        for a in range(0, pages, step):
            x = _normal(gen, min(step, pages - a), ps, hk, D) + shift
            if quant:
                _put_codes(cache[a:a + step], scale[a:a + step], x)
            else:
                cache[a:a + step].copy_(x)
        state[name + "_cache"], state[name + "_scale"] = cache, scale
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    col = torch.arange(max(counts), device="cuda")
    first = torch.tensor(starts[:-1], device="cuda")[:, None]
    at = torch.where(col < torch.tensor(counts, device="cuda")[:, None], first + col, 0)
    state["page_table"] = order[at].contiguous()
    state["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    hk, ps = case["kv_heads"], case["page_size"]
    if case["op"] == "decode":
        state = _filled(case, gen, _lens(case))
        # queries of about twice unit length a channel: softmax rows with a few large weights and a long tail
        state["q"] = (2.0 * _normal(gen, case["batch"], case["q_heads"], D)).to(dtype)
        state["out"] = torch.zeros_like(state["q"])
        state["lse"] = torch.zeros(case["batch"], case["q_heads"], device="cuda")
    elif case["op"] == "read":
        state = _filled(case, gen, _lens(case))
        shape = (case["batch"], case["most"], hk, D)
        state["k"] = torch.zeros(shape, dtype=dtype, device="cuda")
        state["v"] = torch.zeros(shape, dtype=dtype, device="cuda")
    else:
        t = case["tokens"]
        quant = case["cache"] == "e4m3"
        pages = _pages(SLOT_POOL, ps) if case["single"] else _pages(case["start"] + t, ps) + 3
        state = {}
        for name in ("k", "v"):
            state[name + "_cache"] = _empty_cache(case, pages, torch.float8_e4m3fn if quant else dtype)
            state[name + "_scale"] = torch.zeros(pages, hk, ps, device="cuda").transpose(1, 2) if quant else None
        # keys come rotated from the projection, values are its last columns
        qkv = torch.empty(t, (case["q_heads"] + 2 * hk) * D, dtype=dtype, device="cuda")
        for a in range(0, t, 16384):
            qkv[a:a + 16384] = _normal(gen, min(16384, t - a), qkv.shape[1])
        state["k"] = (qkv[:, case["q_heads"] * D:-hk * D].reshape(t, hk, D) + 2.0 * _normal(gen, hk, D)).to(dtype)
        state["v"] = qkv[:, -hk * D:].view(t, hk, D)
        state["qkv"] = qkv
        if case["single"]:
            state["slots"] = torch.randperm(pages * ps, generator=gen, device="cuda")[:t]
        else:
            order = torch.randperm(pages, generator=gen, device="cuda")
            at = torch.arange(case["start"], case["start"] + t, device="cuda")
            state["slots"] = order[at // ps] * ps + at % ps
    state["op"] = case["op"]
    return state


def _gathered(state, name, length):
    """The cache's rows of every sequence as (batch, length, kv_heads, 128) in 32 bits."""
    cache, scale, table = state[name + "_cache"], state[name + "_scale"], state["page_table"].long()
    pos = torch.arange(length, device=cache.device)
    page, at = table[:, pos // cache.shape[1]], pos % cache.shape[1]
    if scale is None:
        return cache[page, at].float()
    codes = cache.view(torch.uint8)[page, at].view(torch.float8_e4m3fn)
    return codes.float() * scale[page, at][..., None]


def _plain_decode(state):
    q, lens = state["q"], state["seq_lens"]
    batch, hq, _ = q.shape
    length = state["page_table"].shape[1] * state["k_cache"].shape[1]
    hk = state["k_cache"].shape[2]
    k = _gathered(state, "k", length)
    s = torch.einsum("bhgd,blhd->bhgl", q.float().view(batch, hk, hq // hk, D), k) * D ** -0.5
    del k
    s.masked_fill_((torch.arange(length, device=q.device) >= lens[:, None])[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("bhgl,blhd->bhgd", p / total, _gathered(state, "v", length))
    return {"out": out.reshape(q.shape).to(q.dtype), "lse": (top + torch.log(total)).reshape(batch, hq)}


def _plain_write(state):
    slots = state["slots"]
    outs = {}
    for name in ("k", "v"):
        x, cache, scale = state[name], state[name + "_cache"], state[name + "_scale"]
        page, at = slots // cache.shape[1], slots % cache.shape[1]
        if scale is None:
            cache[page, at] = x
        else:
            x = x.float()
            amax = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
            codes = (x * (E4M3_MAX / amax)).to(torch.float8_e4m3fn)
            cache.view(torch.uint8)[page, at] = codes.view(torch.uint8)
            scale[page, at] = (amax / E4M3_MAX).squeeze(-1)
            outs[name + "_scale"] = scale
        outs[name + "_cache"] = cache
    return outs


def _plain_read(state):
    outs = {}
    for name in ("k", "v"):
        to = state[name]
        rows = _gathered(state, name, to.shape[1]).to(to.dtype)
        there = torch.arange(to.shape[1], device=to.device) < state["seq_lens"][:, None]
        outs[name] = torch.where(there[..., None, None], rows, to)
    return outs


def run(state):
    if own:
        import flashprefill_b200 as fp
        scales = {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        if state["op"] == "decode":
            fp.paged_decode(state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["seq_lens"], state["out"],
                            lse=state["lse"], **scales)
            return {"out": state["out"], "lse": state["lse"]}
        if state["op"] == "write":
            fp.kv_cache_write(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"], **scales)
            return {name: state[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale") if state[name] is not None}
        fp.kv_cache_read(state["k_cache"], state["v_cache"], state["page_table"], state["seq_lens"], state["k"], state["v"], **scales)
        return {"k": state["k"], "v": state["v"]}
    return {"decode": _plain_decode, "write": _plain_write, "read": _plain_read}[state["op"]](state)


def work(case):
    hk = case["kv_heads"]
    held = 2 * hk * (D + 4 if case["cache"] == "e4m3" else 2 * D)  # bytes of one token in the cache
    if case["op"] == "write":
        return {"bytes": case["tokens"] * (2 * hk * D * 2 + held + 8), "flops": 0}
    lens = _lens(case)
    table = sum(4 * _pages(n, case["page_size"]) + 4 for n in lens)
    if case["op"] == "read":
        return {"bytes": sum(lens) * (2 * hk * D * 2 + held) + table, "flops": 0}
    hq = case["q_heads"]
    return {"bytes": sum(lens) * held + table + case["batch"] * hq * (2 * D * 2 + 4), "flops": 4 * sum(lens) * hq * D}


def _rows64(state, name, b, length):
    """Sequence b's cached rows in 64 bits, (kv_heads, length, 128)."""
    cache, scale, ps = state[name + "_cache"], state[name + "_scale"], state["k_cache"].shape[1]
    pages = state["page_table"][b, :_pages(length, ps)].long()
    x = cache.view(torch.uint8)[pages].view(cache.dtype).double() if scale is not None else cache[pages].double()
    if scale is not None:
        x = x * scale[pages].double().unsqueeze(-1)
    return x.flatten(0, 1)[:length].transpose(0, 1)


def _e4m3_64(x):
    """x in 64 bits rounded to e4m3's values: 3 bits after the leading one, steps of 2^-9 at the least."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -40))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "decode":
        q = state["q"].double()
        outs, lses = [], []
        for b, n in enumerate(_lens(case)):
            heads = q[b].view(case["kv_heads"], -1, D)
            s = torch.matmul(heads, _rows64(state, "k", b, n).transpose(1, 2)) / 128 ** 0.5
            lses.append(torch.logsumexp(s, -1).reshape(-1))
            outs.append(torch.matmul(torch.softmax(s, -1), _rows64(state, "v", b, n)).reshape(-1, D))
        return {"out": torch.stack(outs), "lse": torch.stack(lses)}
    got = {}
    for name in ("k", "v"):
        if case["op"] == "read":
            to = state[name].double()
            for b, n in enumerate(_lens(case)):
                to[b, :n] = _rows64(state, name, b, n).transpose(0, 1)
            got[name] = to
            continue
        cache, scale = state[name + "_cache"], state[name + "_scale"]
        pages, ps, hk, _ = cache.shape
        x = state[name].double()
        flat = torch.zeros(pages * ps, hk, D, dtype=torch.float64, device="cuda")
        if scale is not None:
            most = x.abs().max(-1, keepdim=True).values.clamp_min(TINY)
            flat_scale = torch.zeros(pages * ps, hk, dtype=torch.float64, device="cuda")
            flat_scale[state["slots"]] = (most / E4M3_MAX).squeeze(-1)
            got[name + "_scale"] = flat_scale.view(pages, ps, hk)
            x = _e4m3_64(x / most * E4M3_MAX)
        flat[state["slots"]] = x
        got[name + "_cache"] = flat.view(pages, ps, hk, D)
    return got
