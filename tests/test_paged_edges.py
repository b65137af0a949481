"""Paged cache and decode attention where the work is cut: more items than pieces, workspaces with stale contents."""
import os

import pytest
import torch

import flashprefill_b200 as fp
from flashprefill_b200 import _lib
from tests import paged_util as pu
from tests.test_paged_cache import check_decode, same_bits

E4M3 = torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16

# A GPU of 148 SMs holds 444 CTAs of items of up to 8 heads and 296 of items of 9 to 16: lens, q heads, kv heads, page size, layout
MANY_ITEMS = [
    ([0, 1, 700, 64, 65, 17, 300, 2] * 8, 16, 8, 16, "nhd"),                   # 512 items
    ([33, 0, 129] * 29 + [5, 1000], 15, 5, 48, "hnd"),                         # 445 items, one more than pieces
    ([9000] + [0, 3, 0, 70, 1] * 60, 2, 2, 64, "hnd"),                         # 602 items, one of them in many pieces
    ([0] * 299 + [1], 4, 2, 16, "nhd"),                                        # 600 items that hold one token
    ([257, 0, 31, 16, 1] * 30, 24, 2, 16, "hnd"),                              # 300 items of 12 heads
    ([5000, 0] + [40, 200, 0] * 99, 16, 1, 5, "nhd"),                          # 299 items of 16 heads
    ([100, 7, 0, 900] * 38, 20, 1, 32, "nhd"),                                 # 304 items: 20 heads in two groups
    ([0, 1], 32, 8, 16, "hnd"),                                                # fewer units than CTAs: most leave early
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("case", range(len(MANY_ITEMS)))
def test_more_items_than_pieces(case, quant, dtype):
    """Items that no piece begins alone, pieces that span several whole items and two cut ones, lengths of zero among them; in
    workspaces of zeros, of ones and of an earlier call's sums."""
    lens, hq, hk, ps, layout = MANY_ITEMS[case]
    cd = E4M3 if quant else dtype
    f = pu.fill_sequences(lens, hq, hk, dtype, cd, ps, layout, seed=30 + case, room=70000)
    n = fp.paged_decode_workspace_bytes(len(lens), hq, hk, cd, f["page_table"].shape[1], ps)
    assert n > 0  # in pieces, not clusters
    cache = (f["k"], f["v"])
    back = torch.arange(len(lens) - 1, -1, -1, device="cuda")
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    first = None
    for fill in (0, 255, None):
        if fill is not None:
            ws.fill_(fill)
        else:  # the sums and descriptors of other lengths
            fp.paged_decode(f["q"], *cache, f["page_table"][back], f["lens"][back], torch.empty_like(f["q"]), None, f["k_scale"],
                            f["v_scale"], workspace=ws)
        out = torch.full_like(f["q"], float("nan"))
        lse = torch.full((len(lens), hq), float("nan"), device="cuda")
        fp.paged_decode(f["q"], *cache, f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"], workspace=ws)
        fp.check_paged_error()
        if first is None:
            first = out, lse
            check_decode(f, out, lse, dtype, cd)
        assert same_bits(out, first[0]) and same_bits(lse, first[1])


# ------------------------------------------------------------------ memory that two tensors of one call share
@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from flashprefill_b200 import build
        build.build()
    return _lib.load()


def test_c_entries_refuse_one_memory_for_keys_and_values(lib):
    i = _lib.i64arr
    def write(kc, vc, cd, ks, vs):
        ss = i([32, 1, 16]) if cd else None
        return lib.fpb_kv_cache_write(256, 512, 0, 4, 2, 128, i([256, 128]), i([256, 128]), kc, vc, cd, 8, 16, i([4096, 128, 2048]), ks,
                                      vs, ss, 1024, 8, None)
    assert write(4096, 4096, _lib.FPB_BF16, None, None) == _lib.FPB_EINVAL and b"k_cache and v_cache" in lib.fpb_last_error()
    assert write(4096, 8192, _lib.FPB_E4M3, 64, 64) == _lib.FPB_EINVAL and b"k_scale and v_scale" in lib.fpb_last_error()
    s = i([40 * 256, 256, 128])
    assert lib.fpb_kv_cache_read(4096, 8192, 0, 8, 16, 2, 128, i([4096, 128, 2048]), None, None, None, 256, 4, 4, 512, 2, 1024, 1024, 0,
                                 40, s, s, None) == _lib.FPB_EINVAL and b"k and v must not" in lib.fpb_last_error()


@pytest.mark.gpu
def test_write_refuses_one_scale_tensor_for_keys_and_values():
    """Keys would be read back with the values' scales."""
    c = fp.kv_cache_alloc(2, 16, 2, E4M3)
    rows = torch.ones(3, 2, 128, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="k_scale and v_scale must not be the same memory"):
        fp.kv_cache_write(rows, rows, c.k, c.v, torch.arange(3, device="cuda"), c.k_scale, c.k_scale)


# ------------------------------------------------------------------ launches that are prepared while their predecessors run
def test_kernels_behind_a_stream_wait_use_no_read_only_loads():
    """A kernel that is launched while its inputs are still being written must not read them as memory that is constant for its
    lifetime: __ldg, ld.global.nc and const __restrict__ are free to be moved in front of the wait."""
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    for name in ("fp_paged.cu", "fp_decode.cu"):
        with open(os.path.join(csrc, name)) as f:
            code = "\n".join(line.split("//")[0] for line in f)
        assert "await_stream()" in code
        for word in ("__ldg", "ld.global.nc", "__restrict__", "__ldca", "ld.const"):
            assert word not in code, (name, word)


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
def test_every_step_sees_what_the_one_before_it_wrote(quant):
    """Lengths, tables, slots, rows and queries changed on the stream just before each call, a step right behind the other, eagerly
    and from one captured graph (behind copies and a join of two streams): every step equals the same calls made one by one."""
    dtype, cd, n = BF16, E4M3 if quant else BF16, 200
    g = torch.Generator(device="cuda").manual_seed(4)
    steps = 12
    rows = torch.randn(steps, 2, n, 2, 128, generator=g, device="cuda").to(dtype)
    qs = torch.randn(steps, 1, 8, 128, generator=g, device="cuda").to(dtype)
    orders = torch.stack([torch.randperm(16, generator=g, device="cuda") for _ in range(steps)])
    tables, lengths = orders.int()[:, None], torch.randint(1, n + 1, (steps, 1), generator=g, device="cuda").int()
    pos = torch.arange(n, device="cuda")

    def run(apart, stages=None):
        c = fp.kv_cache_alloc(16, 16, 2, cd)
        for t in c:
            if t is not None:
                t.zero_()
        table, lens, slots = torch.zeros_like(tables[0]), torch.zeros_like(lengths[0]), torch.zeros(n, dtype=torch.int64, device="cuda")
        kv, q = torch.zeros_like(rows[0]), torch.zeros_like(qs[0])
        outs = torch.empty(steps, 1, 8, 128, dtype=dtype, device="cuda")
        back = torch.empty(steps, 2, 1, n, 2, 128, dtype=dtype, device="cuda").fill_(1.0)
        wait = torch.cuda.synchronize if apart else lambda: None
        side = torch.cuda.Stream()

        def all_steps():
            for i in range(steps):
                here = torch.cuda.current_stream()
                side.wait_stream(here)
                with torch.cuda.stream(side):
                    table.copy_(tables[i])
                    lens.copy_(lengths[i])
                slots.copy_(orders[i][pos // 16] * 16 + pos % 16)
                kv.copy_(rows[i])
                q.copy_(qs[i])
                wait()
                fp.kv_cache_write(kv[0], kv[1], c.k, c.v, slots, c.k_scale, c.v_scale)
                wait()
                here.wait_stream(side)
                fp.paged_decode(q, c.k, c.v, table, lens, outs[i], None, c.k_scale, c.v_scale)
                wait()
                fp.kv_cache_read(c.k, c.v, table, lens, back[i, 0], back[i, 1], c.k_scale, c.v_scale)
                wait()

        if stages is None:
            all_steps()
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                all_steps()
            for _ in range(stages):
                outs.zero_()
                back.fill_(1.0)
                graph.replay()
        torch.cuda.synchronize()
        fp.check_paged_error()
        return outs, back

    want = run(True)
    for got in (run(False), run(False), run(False, stages=4)):
        assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])


# ------------------------------------------------------------------ values that are not finite, scales far apart
def check_rows(f, out, lse, dtype, cache_dtype):
    """Infinities and NaN where the definition in 64 bits has them, all else within its bounds."""
    for b, (k, v) in enumerate(f["rows"]):
        ref, rl, _, _ = pu.attend64(f["q"][b], k, v)
        finite, _, weight, size = pu.attend64(f["q"][b], k, torch.where(v.isfinite(), v, 0.0))
        to, tl = pu.decode_bounds(finite, rl, weight, size, k.shape[0], dtype, cache_dtype, f["q"][b], k, torch.where(v.isfinite(), v, 0.0))
        got, there = out[b].double(), ref.isfinite()
        assert torch.equal(got[~there].nan_to_num(7.0, 8.0, 9.0), ref[~there].nan_to_num(7.0, 8.0, 9.0)), b
        err = (got - ref).abs()[there]
        assert (err <= to[there]).all(), (b, (err / to[there]).max().item())
        assert ((lse[b].double() - rl).abs() <= tl).all(), b


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 50000])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_infinite_values_follow_the_softmax(dtype, room):
    """An infinite value with any weight makes its channel infinite, with its sign (the token of the largest weight, of ordinary
    ones, a sequence of one token); two of opposite signs make NaN; nothing else changes."""
    f = pu.fill_sequences([700, 300, 1, 65], 8, 2, dtype, dtype, 16, seed=40, k_gain=0.3, room=room)

    def put(b, at, head, channel, x):
        f["v"][f["page_table"][b, at // 16].long(), at % 16, head, channel] = x
        f["rows"][b][1][at, head, channel] = x

    inf = float("inf")
    k, q = f["rows"][0][0], f["q"][0].double()
    top = torch.einsum("gd,nd->gn", q[:4], k[:, 0]).argmax(-1).tolist()  # heaviest token of each head of KV head 0
    for i, at in enumerate(top):
        put(0, at, 0, i, inf)
        put(0, at, 0, 40 + i, -inf)
    for i, at in enumerate(range(0, 700, 33)):
        put(0, at, 1, i, inf if i % 2 else -inf)
    put(0, 5, 1, 100, inf)
    put(0, 690, 1, 100, -inf)
    put(0, 5, 1, 101, inf)
    put(0, 690, 1, 101, inf)
    put(2, 0, 0, 3, inf)
    put(2, 0, 1, 4, -inf)
    put(3, 64, 0, 127, inf)
    out, lse = torch.empty_like(f["q"]), torch.empty(4, 8, device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse)
    assert out[0].isinf().any() and out[0, 4:, 100].isnan().all() and out[2, :4, 3].eq(inf).all()
    check_rows(f, out, lse, dtype, dtype)


def weighted_bounds(q, k, v, dtype, cache_dtype):
    """attend64's results with bounds whose fp16 steps, 2^-40 of each, are those of the largest product of a head's weight and a row's
    largest value."""
    ref, lse, weight, size = pu.attend64(q, k, v)
    n, hk = k.shape[0], k.shape[1]
    to, tl = pu.decode_bounds(ref, lse, weight, size, n, dtype, cache_dtype, q, k, torch.zeros_like(v))
    s = torch.einsum("hgd,nhd->hgn", q.double().view(hk, -1, 128), k) * 128 ** -0.5
    largest = (torch.softmax(s, -1) * v.abs().amax(-1).t()[:, None]).amax(-1).reshape(-1, 1)
    return ref, lse, to + n * 2.0 ** -40 * largest, tl


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 70000])
@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_value_scales_far_apart(dtype, heads, room):
    """A quantised row keeps its bits whatever the scales of the others: rows of values up to 2^90 times as large that the softmax
    gives no weight (in front, behind and between), scales that rise and fall through the sequence, and weights that make up
    for the scales."""
    f = pu.fill_sequences([300, 300, 513, 600, 40], heads, 1, dtype, E4M3, 16, seed=50, k_gain=0.2, room=room)
    f["q"] = f["q"].abs() + 0.1  # so that a key of like values has a score of its sign for every head

    def at(b, i):
        i = torch.as_tensor(i, device="cuda")
        return f["page_table"][b].long()[i // 16], i % 16

    def gain(b, i, x):
        p = at(b, i)
        f["v_scale"][p[0], p[1]] *= x[:, None]
        f["rows"][b][1][i] *= x.double()[:, None, None]

    def no_weight(b, i):
        p = at(b, i)
        f["k"].view(torch.uint8)[p[0], p[1]] = torch.tensor(-448.0).to(E4M3).view(torch.uint8).item()
        f["k_scale"][p[0], p[1]] = 1.0  # score below -448 * 0.1 * sqrt(128) = -500
        f["rows"][b][0][i] = -448.0

    for b, i in ((0, [0, 1, 40]), (1, [299]), (2, list(range(31, 513, 64)))):
        no_weight(b, i)
        gain(b, i, torch.full((len(i),), 2.0 ** (90 if b else 45), device="cuda"))
    n = 600
    i = torch.arange(n, device="cuda")
    gain(3, i, torch.exp2(-20.0 * torch.sin(i / 25.0).abs()))
    i = torch.arange(40, device="cuda")
    gain(4, i, torch.exp2(-2.0 * i))
    # a key of like values c has the score c * sum(q) / sqrt(128): about 1.5 nats a token, more than the 1.4 that its values lose
    p = at(4, i)
    c = 1.5 / (f["q"][4].float().sum(-1).min() * 128 ** -0.5)
    f["k"].view(torch.uint8)[p[0], p[1]] = torch.tensor(1.0).to(E4M3).view(torch.uint8).item()
    f["k_scale"][p[0], p[1]] = (c * i)[:, None]
    f["rows"][4][0][i] = (c * i).float().double()[:, None, None].expand(40, 1, 128)
    out, lse = torch.empty_like(f["q"]), torch.empty(5, heads, device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"])
    fp.check_paged_error()
    for b, (k, v) in enumerate(f["rows"]):
        ref, rl, to, tl = weighted_bounds(f["q"][b], k, v, dtype, E4M3)
        err = (out[b].double() - ref).abs()
        assert (err <= to).all(), (b, (err / to).max().item(), ref.abs().max().item())
        assert ((lse[b].double() - rl).abs() <= tl).all(), b


@pytest.mark.gpu
@pytest.mark.parametrize("small", [2.0 ** -13, 2.0 ** -20, 2.0 ** -26])
def test_small_elements_of_a_query_beside_large_ones(small):
    """bfloat16 queries over a quantised cache, multiplied in fp16: elements far below their row's largest keep their bits where the
    keys do not meet the large one.  An element is off by 2^-39 of the largest at the most."""
    f = pu.fill_sequences([90, 700], 6, 2, BF16, E4M3, 16, seed=60)
    f["q"] *= small
    f["q"][:, :, 17] = 1.0
    f["k"].view(torch.uint8)[..., 17] = 0
    for k, _ in f["rows"]:
        k[..., 17] = 0.0
    scale = 128 ** -0.5 / small
    out, lse = torch.empty_like(f["q"]), torch.empty(2, 6, device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"], sm_scale=scale)
    for b, (k, v) in enumerate(f["rows"]):
        ref, rl, weight, size = pu.attend64(f["q"][b], k, v, scale)
        to, tl = pu.decode_bounds(ref, rl, weight, size, k.shape[0], BF16, E4M3, f["q"][b] * 2.0 ** -15, k, v, scale)
        assert ((out[b].double() - ref).abs() <= to).all() and ((lse[b].double() - rl).abs() <= tl).all(), b


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 70000])
def test_weights_keep_more_bits_than_their_products_type(room):
    """Rows of 1 and of -(1 + 2^-13) in equal parts: what is left of their sum, 2^-14, is below one rounding of a weight to fp16 (which
    is all that an e4m3 cache's weights get for bfloat16 output)."""
    n, dtype = 64, FP16
    f = pu.fill_sequences([n], 4, 1, dtype, E4M3, 16, seed=61, room=room)
    page, at = f["page_table"][0].long()[torch.arange(n, device="cuda") // 16], torch.arange(n, device="cuda") % 16
    f["k"].view(torch.uint8)[page, at] = 0
    sign = torch.where(torch.arange(n, device="cuda") % 2 == 0, 1.0, -1.0)
    scale = torch.where(sign > 0, 1.0, 1.0 + 2.0 ** -13)
    f["v"].view(torch.uint8)[page, at] = sign[:, None, None].expand(n, 1, 128).to(E4M3).view(torch.uint8)
    f["v_scale"][page, at] = scale[:, None]
    k, v = torch.zeros(n, 1, 128, dtype=torch.float64, device="cuda"), (sign * scale).double()[:, None, None].expand(n, 1, 128)
    out = torch.empty_like(f["q"])
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, None, f["k_scale"], f["v_scale"])
    ref, _, weight, size = pu.attend64(f["q"][0], k, v)
    # weights as two fp16 parts, 2^-21; their sum in fp32, n 2^-24; exp2 and the scale's product, 2^-21
    bound = (2.0 ** -21 + (n + 16) * 2.0 ** -24 + 2.0 ** -21) * weight + pu.half_step(dtype) * ref.abs()
    assert (ref.abs() > 4 * bound).all() and ((out[0].double() - ref).abs() <= bound).all()


# ------------------------------------------------------------------ the checked mode, several callers at once
def test_checked_calls_report_their_own_errors(monkeypatch):
    """The device's error word is one for all: a checked call must not clear what another's raised.  The word is a variable here."""
    import threading
    import time
    from flashprefill_b200 import _ops
    word = []

    class Ext:
        @staticmethod
        def paged_decode(q, *rest):
            time.sleep(0.001)
            if q.bad:
                word.append("bad")

    class Q:
        device = torch.device("cpu")

        def __init__(self, bad):
            self.bad = bad

    def check(device=None):
        time.sleep(0.001)
        found, word[:] = list(word), []
        if found:
            raise fp.FlashPrefillError("bad")

    class Anywhere:
        def __init__(self, device): pass
        def __enter__(self): pass
        def __exit__(self, *a): pass

    monkeypatch.setattr(_ops, "CHECK", True)
    monkeypatch.setattr(_ops, "check_paged_error", check)
    monkeypatch.setattr(_lib, "_ext", Ext)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", Anywhere)
    raised = {}

    def work(name, bad):
        n = 0
        for _ in range(30):
            try:
                fp.paged_decode(Q(bad), *[None] * 5)
            except fp.FlashPrefillError:
                n += 1
        raised[name] = n

    threads = [threading.Thread(target=work, args=(i, i % 2 == 0)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert raised == {0: 30, 1: 0, 2: 30, 3: 0}


@pytest.mark.gpu
def test_checked_mode_of_two_threads():
    """FLASHPREFILL_B200_CHECK=1 in two threads on streams of their own: each call with a slot outside the cache raises, no other."""
    import subprocess
    import sys
    code = """
import threading, torch, flashprefill_b200 as fp
r = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device="cuda")
raised = [0, 0]
def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        c = fp.kv_cache_alloc(4, 16, 1)
        slots = torch.tensor([1, 3 if i else 64], device="cuda")
        for _ in range(200):
            try:
                fp.kv_cache_write(r, r, c.k, c.v, slots)
            except fp.FlashPrefillError:
                raised[i] += 1
torch.cuda.synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
[t.start() for t in threads]
[t.join() for t in threads]
print(raised)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, FLASHPREFILL_B200_CHECK="1", PYTHONPATH=root), capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split("\n")[0] == "[200, 0]", r.stdout + r.stderr


# ------------------------------------------------------------------ registered ops
@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
def test_registered_write_read_and_decode_match_the_entry_points(quant):
    """A run of the three through torch.ops, eagerly and traced by torch.compile, against the Python entry points."""
    cd, n = E4M3 if quant else BF16, 100
    g = torch.Generator(device="cuda").manual_seed(70)
    k, v = (torch.randn(n, 2, 128, generator=g, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn(1, 8, 128, generator=g, device="cuda").to(BF16)
    slots = torch.randperm(128, generator=g, device="cuda")[:n]
    table, lens = torch.tensor([[3, 1, 7, 0]], dtype=torch.int32, device="cuda"), torch.tensor([60], dtype=torch.int32, device="cuda")

    def run(write, read, decode):
        c = fp.KVCache(*(None if t is None else t.zero_() for t in fp.kv_cache_alloc(8, 16, 2, cd)))
        kr, vr, out, lse = (torch.zeros(1, 64, 2, 128, dtype=BF16, device="cuda"), torch.zeros(1, 64, 2, 128, dtype=BF16, device="cuda"),
                            torch.zeros_like(q), torch.zeros(1, 8, device="cuda"))
        write(k, v, c.k, c.v, slots, c.k_scale, c.v_scale)
        read(c.k, c.v, table, lens, kr, vr, c.k_scale, c.v_scale)
        decode(q, c.k, c.v, table, lens, out, lse, c.k_scale, c.v_scale)
        return [*(t for t in c if t is not None), kr, vr, out, lse]

    ops = torch.ops.flashprefill
    want = run(fp.kv_cache_write, fp.kv_cache_read, fp.paged_decode)
    got = run(ops.kv_cache_write, ops.kv_cache_read, ops.paged_decode)
    for a, b in zip(got, want):
        assert same_bits(a, b)

    def traced(kr, vr, out, lse, *cache):
        ks, vs = cache[2:] if quant else (None, None)
        ops.kv_cache_write(k, v, cache[0], cache[1], slots, ks, vs)
        ops.kv_cache_read(cache[0], cache[1], table, lens, kr, vr, ks, vs)
        ops.paged_decode(q, cache[0], cache[1], table, lens, out, lse, ks, vs)
        return out * 1.0

    outs = [torch.zeros_like(t) for t in want[-4:]]
    cache = [t.zero_() for t in fp.kv_cache_alloc(8, 16, 2, cd) if t is not None]
    torch.compile(traced, backend="aot_eager", fullgraph=True)(*outs, *cache)
    for a, b in zip(cache + outs, want):
        assert same_bits(a, b)
    fp.check_paged_error()


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 70000])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_of_millions_and_more(dtype, quant, room):
    """Scores whose steps in fp32 are whole powers of two: the tokens of the largest share the weight, all others have none.  Scores are
    exact products of one channel, so equal ones are equal."""
    cd = E4M3 if quant else dtype
    n = 200
    f = pu.fill_sequences([n] * 6, 4, 1, dtype, cd, 16, seed=80, room=room)
    f["q"][:] = 0
    size = torch.tensor([2.0 ** 20, 2.0 ** 22, 2.0 ** 24, 2.0 ** 27, -2.0 ** 24, 2.0 ** 32], dtype=torch.float64)
    g = torch.Generator().manual_seed(1)
    for b in range(6):
        # keys of 1 to 15 in one channel, the query's value times sm_scale 1 gives the size
        value = torch.randint(1, 16, (n,), generator=g).double().cuda()
        at = torch.arange(n, device="cuda")
        page, at = f["page_table"][b].long()[at // 16], at % 16
        k = torch.zeros(n, 1, 128, dtype=torch.float64, device="cuda")
        gain = 2.0 ** (10 if quant else 0)
        k[:, 0, 5] = value * (1.0 if quant else 2.0 ** 10)
        if quant:
            f["k"].view(torch.uint8)[page, at] = k.to(E4M3).view(torch.uint8)
            f["k_scale"][page, at] = gain
        else:
            f["k"][page, at] = k.to(cd)
        f["rows"][b][0][:] = k * gain
        f["q"][b, :, 5] = (size[b] * 2.0 ** -24).to(dtype)  # 2^-4 to 2^8; the sm_scale below has the rest
    scale = 2.0 ** 14
    out, lse = torch.empty_like(f["q"]), torch.empty(6, 4, device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"], sm_scale=scale)
    fp.check_paged_error()
    for b, (k, v) in enumerate(f["rows"]):
        ref, rl, weight, _ = pu.attend64(f["q"][b], k, v, scale)
        to, _ = pu.decode_bounds(ref, rl, weight, torch.zeros_like(rl), n, dtype, cd, f["q"][b] * 0, k, v, scale)
        err = (out[b].double() - ref).abs()
        assert (err <= to).all(), (b, (err / to).max().item())
        # the product with sm_scale * log2(e) and its way back, each off by 2^-24
        assert ((lse[b].double() - rl).abs() <= 2.0 ** -21 * rl.abs() + 2.0 ** -20).all(), b


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 70000])
@pytest.mark.parametrize("hq,page_size", [(8, 16), (24, 5), (24, 48)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_one_head_of_large_scores_beside_ordinary_ones(dtype, hq, page_size, room):
    """A quantised cache where one head's scores reach tens of thousands, at some place in the sequence: it and its neighbours in the
    same warps keep to the definition, as does a sequence with none."""
    f = pu.fill_sequences([3000, 0, 65, 900, 1], hq, 2, dtype, E4M3, page_size, "nhd", seed=81, room=room)
    f["q"][0, 1] *= 4000.0
    f["q"][2, hq - 1] *= -3000.0
    at = 777
    page, off = f["page_table"][3, at // page_size].long(), at % page_size
    f["k_scale"][page, off] *= 5000.0  # one token whose key is large for every head
    f["rows"][3][0][at] = f["k"].view(torch.uint8)[page, off].view(E4M3).double() * f["k_scale"][page, off].double()[:, None]
    out, lse = torch.full_like(f["q"], float("nan")), torch.full((5, hq), float("nan"), device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"])
    fp.check_paged_error()
    check_decode(f, out, lse, dtype, E4M3)
    again = torch.empty_like(out)
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], again, None, f["k_scale"], f["v_scale"])
    assert same_bits(out, again)


# ------------------------------------------------------------------ refusals
def test_workspace_of_a_type_that_no_cache_holds_is_refused(lib):
    with pytest.raises(TypeError, match="float32"):
        fp.paged_decode_workspace_bytes(1, 8, 2, torch.float32, 64, 16)


@pytest.mark.gpu
def test_a_scale_that_is_no_number_is_refused():
    f = pu.fill_sequences([20], 4, 2, BF16, BF16, 16, seed=90)
    for bad in ("0.1", [0.1], object()):
        with pytest.raises(TypeError):
            fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], torch.empty_like(f["q"]), sm_scale=bad)
    with pytest.raises(ValueError, match="sm_scale"):
        fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], torch.empty_like(f["q"]), sm_scale=1e300)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_lse_does_not_depend_on_the_scale_of_the_values(dtype):
    """Short rows of small scores over a quantised cache: the log of the sum is as near as a 16-bit cache's, for values of any size."""
    f = pu.fill_sequences([1, 2, 3, 5, 17] * 40, 24, 2, dtype, E4M3, 16, seed=91, k_gain=0.01)
    f["v_scale"] *= torch.exp2(torch.randint(-6, 7, f["v_scale"].shape, generator=torch.Generator("cuda").manual_seed(1), device="cuda").float())
    out, lse = torch.empty_like(f["q"]), torch.empty(200, 24, device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"], sm_scale=0.01)
    for b, (k, v) in enumerate(f["rows"]):
        ref, rl, weight, size = pu.attend64(f["q"][b], k, v, 0.01)
        _, tl = pu.decode_bounds(ref, rl, weight, size, k.shape[0], dtype, E4M3, f["q"][b], k, v, 0.01)
        assert ((lse[b].double() - rl).abs() <= tl).all(), (b, ((lse[b].double() - rl).abs() / tl).max().item())
