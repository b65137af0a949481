"""Paged key/value cache and decode attention.

CPU: the C entry points refuse bad arguments before any CUDA call, the workspace bound, the Python entry points refuse CPU
tensors.  GPU: every entry point against its plain form in 64 bits (copies and codes bit for bit), at the lengths, page
sizes, head layouts and strides where a tile, a page or a split ends; stale rows are NaN and table entries behind a sequence
point outside the cache, so that anything read beyond a sequence shows."""
import ctypes
import os

import pytest
import torch

import flashprefill_b200 as fp
from flashprefill_b200 import _lib
from tests import paged_util as pu

E4M3 = torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16


# ------------------------------------------------------------------ host checks
@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from flashprefill_b200 import build
        build.build()
    return _lib.load()


CS = [16 * 2 * 128, 128, 16 * 128]  # head-major pages of 16
SS = [32, 1, 16]


def _write(lib, **over):
    a = dict(k=256, v=512, dtype=0, t=4, hk=2, d=128, ks=[256, 128], kc=4096, vc=8192, cd=0, pages=8, ps=16, cs=CS, ksc=None,
             vsc=None, ss=None, slots=1024, sb=8)
    a.update(over)
    arr = lambda x: None if x is None else _lib.i64arr(x)
    return lib.fpb_kv_cache_write(a["k"], a["v"], a["dtype"], a["t"], a["hk"], a["d"], arr(a["ks"]), arr(a["ks"]), a["kc"],
                                  a["vc"], a["cd"], a["pages"], a["ps"], arr(a["cs"]), a["ksc"], a["vsc"], arr(a["ss"]),
                                  a["slots"], a["sb"], None)


@pytest.mark.parametrize("over,msg", [
    (dict(d=64), "head_dim"), (dict(dtype=2), "dtype"), (dict(cd=1), "16-bit type"), (dict(cd=5), "16-bit type"),
    (dict(pages=0), "num_pages"), (dict(ps=0), "page_size"), (dict(hk=0), "num_kv_heads"), (dict(kc=0), "k_cache is NULL"),
    (dict(vc=8200), "16-byte"), (dict(cs=[4096, 127, 2048]), "cache stride[1]"), (dict(cs=[-4096, 128, 2048]), "cache stride[0]"),
    (dict(cs=None), "cache strides"), (dict(cd=2, ss=SS), "needs k_scale"), (dict(cd=2, ksc=64, vsc=66, ss=SS), "aligned float"),
    (dict(cd=2, ksc=64, vsc=128), "scale strides"), (dict(cd=2, ksc=64, vsc=128, ss=[-1, 1, 1]), "scale stride[0]"),
    (dict(cd=2, cs=[4096, 8, 2048], ksc=64, vsc=128, ss=SS), "cache stride[1]"),
    (dict(ksc=64, vsc=128), "takes no scales"), (dict(t=-1), "tokens"), (dict(t=1 << 30, hk=2), "2^31"), (dict(sb=2), "slot_bytes"),
    (dict(k=0), "k is NULL"), (dict(ks=[255, 128]), "k stride"), (dict(slots=0), "slots"), (dict(slots=1028), "slots"),
])
def test_write_refuses_on_the_host(lib, over, msg):
    assert _write(lib, **over) == _lib.FPB_EINVAL
    assert msg in lib.fpb_last_error().decode()


def test_write_of_no_rows_launches_nothing(lib):
    assert _write(lib, t=0, k=0, v=0, slots=0) == _lib.FPB_OK


def _read(lib, **over):
    a = dict(kc=4096, vc=8192, cd=0, pages=8, ps=16, hk=2, d=128, cs=CS, table=256, tst=4, mp=4, lens=512, b=2, k=1024, v=2048,
             dtype=0, s=40, ks=[40 * 256, 256, 128])
    a.update(over)
    arr = lambda x: None if x is None else _lib.i64arr(x)
    return lib.fpb_kv_cache_read(a["kc"], a["vc"], a["cd"], a["pages"], a["ps"], a["hk"], a["d"], arr(a["cs"]), None, None, None,
                                 a["table"], a["tst"], a["mp"], a["lens"], a["b"], a["k"], a["v"], a["dtype"], a["s"],
                                 arr(a["ks"]), arr(a["ks"]), None)


@pytest.mark.parametrize("over,msg", [
    (dict(table=0), "page_table"), (dict(table=258), "page_table"), (dict(lens=0), "seq_lens"), (dict(b=0), "batch"),
    (dict(mp=0), "max_pages"), (dict(mp=1 << 30, ps=16), "max_pages * page_size"), (dict(tst=-4), "table stride"),
    (dict(b=70000), "65535"), (dict(s=0), "out_len"), (dict(s=1 << 30), "out_len"), (dict(k=1032), "16-byte"),
    (dict(ks=[40 * 256, 256, 4]), "k stride[2]"), (dict(d=96), "head_dim"), (dict(cd=2), "needs k_scale"),
])
def test_read_refuses_on_the_host(lib, over, msg):
    assert _read(lib, **over) == _lib.FPB_EINVAL
    assert msg in lib.fpb_last_error().decode()


def _decode(lib, **over):
    a = dict(q=256, dtype=0, b=2, hq=8, hk=2, d=128, qs=[1024, 128], kc=4096, vc=8192, cd=0, pages=64, ps=16, cs=CS, table=256,
             tst=64, mp=64, lens=512, out=1024, os=[1024, 128], lse=None, scale=0.1, ws=4096, wsb=1 << 30)
    a.update(over)
    arr = lambda x: None if x is None else _lib.i64arr(x)
    return lib.fpb_paged_decode(a["q"], a["dtype"], a["b"], a["hq"], a["hk"], a["d"], arr(a["qs"]), a["kc"], a["vc"], a["cd"],
                                a["pages"], a["ps"], arr(a["cs"]), None, None, None, a["table"], a["tst"], a["mp"], a["lens"],
                                a["out"], arr(a["os"]), a["lse"], a["scale"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,msg", [
    (dict(hq=7), "multiple"), (dict(hq=0), "multiple"), (dict(b=0), "batch"), (dict(q=8), "q must be 16-byte"), (dict(qs=[1024, 4]), "q stride"),
    (dict(out=0), "out"), (dict(out=1025), "out"), (dict(os=None), "out strides"), (dict(os=[-1, 128]), "out stride[0]"),
    (dict(lse=1026), "lse"), (dict(scale=float("nan")), "sm_scale"), (dict(ws=0, mp=8192), "workspace"), (dict(ws=4100, mp=8192), "workspace"),
    (dict(wsb=100, mp=8192), "workspace too small"), (dict(table=0), "page_table"), (dict(lens=2), "seq_lens"), (dict(d=256), "head_dim"),
    (dict(cd=1), "16-bit type"), (dict(b=1 << 28), "2^31"),
])
def test_decode_refuses_on_the_host(lib, over, msg):
    assert _decode(lib, **over) == _lib.FPB_EINVAL
    assert msg in lib.fpb_last_error().decode()


def test_decode_workspace_is_bounded():
    n = fp.paged_decode_workspace_bytes
    assert n(1, 32, 8, BF16, 8, 16) == n(256, 32, 8, BF16, 32, 16) == 0  # short sequences: one cluster an item
    few, many = n(1, 32, 8, BF16, 8192, 128), n(256, 32, 8, BF16, 8192, 128)
    # by the GPU's blocks and an item's heads, not by batch or length
    assert 0 < few < many < 4 << 20 and n(4096, 32, 8, BF16, 8192, 128) == n(256, 32, 8, BF16, 16384, 128) == many
    assert n(256, 128, 8, BF16, 8192, 128) > many  # 16 heads an item
    assert n(0, 32, 8, BF16, 8, 16) == n(1, 7, 2, BF16, 8, 16) == 0


def test_python_entries_refuse_cpu_tensors_and_bad_allocations():
    k = torch.zeros(4, 2, 128, dtype=BF16)
    cache = torch.zeros(8, 16, 2, 128, dtype=BF16)
    table, lens = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fp.kv_cache_write(k, k, cache, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        fp.kv_cache_read(cache, cache, table, lens, k[:, None], k[:, None])
    with pytest.raises(ValueError, match="CUDA"):
        fp.paged_decode(k, cache, cache, table, lens, torch.empty_like(k))
    with pytest.raises(TypeError):
        fp.kv_cache_alloc(4, 16, 2, torch.float32, device="cpu")
    with pytest.raises(ValueError):
        fp.kv_cache_alloc(0, 16, 2, device="cpu")
    c = fp.kv_cache_alloc(4, 16, 2, E4M3, device="cpu")
    assert c.k.shape == (4, 16, 2, 128) and c.k_scale.shape == (4, 16, 2) and c.k.stride() == c.v.stride()
    assert fp.kv_cache_alloc(4, 16, 2, device="cpu").k_scale is None


# ------------------------------------------------------------------ write
def same_bits(a, b):
    as_int = lambda t: t.contiguous().view(torch.uint8)
    return torch.equal(as_int(a), as_int(b))


WRITE_CASES = [  # rows, kv heads, page size, layout
    (1, 1, 16, "hnd"), (3, 8, 16, "nhd"), (33, 5, 1, "hnd"), (257, 2, 48, "nhd"), (1030, 4, 128, "hnd"), (64, 7, 3, "nhd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("t,hk,ps,layout", WRITE_CASES)
def test_write_matches_the_definition(t, hk, ps, layout, quant, dtype):
    g = torch.Generator(device="cuda").manual_seed(t)
    pages = -(-t // ps) + 2
    cd = E4M3 if quant else dtype
    cache = pu.empty_cache(pages, ps, hk, cd, layout, fill=3.0)
    qkv = torch.randn(t, (hk + 3) * 128 * 2, generator=g, device="cuda").to(dtype)
    k = qkv[:, 128:(hk + 1) * 128].view(t, hk, 128)  # columns of a projection
    v = torch.randn(t, hk, 128, generator=g, device="cuda").to(dtype) * 2.0 ** (torch.arange(t, device="cuda") % 30 - 15).to(dtype)[:, None, None]
    slots = torch.randperm(pages * ps, generator=g, device="cuda")[:t]
    slots[::5] = -1 - slots[::5]  # padding of a captured batch
    want = [None if c is None else c.clone() for c in cache]
    at = slots >= 0
    page, off = slots[at] // ps, slots[at] % ps
    for x, i in ((k, 0), (v, 1)):
        if not quant:
            want[i][page, off] = x[at]
            continue
        x = x[at].double()
        amax = x.abs().amax(-1, keepdim=True).clamp_min(pu.TINY)
        want[i + 2][page, off] = (amax / 448).squeeze(-1).float()
        codes, old = cache[i].clone(), x
        fp.kv_cache_write(k, v, cache[0], cache[1], slots, cache[2], cache[3])
        got = cache[i].view(torch.uint8)[page, off].view(E4M3).double()
        exact = old / amax * 448
        # fp16 rows of the largest factor, 2^14, overflow to inf where |x| >= 4: such a row reads back as NaN
        finite = old.isfinite().all(-1)
        assert (got * cache[i + 2][page, off].double()[..., None])[~finite].isnan().all().item()
        # half an e4m3 step: 2^-4 of the value, 2^-10 among the denormals; 2^-23 for the factor and the product in fp32
        near = (got - exact).abs() <= (exact.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * (1 + 2.0 ** -10) + exact.abs() * 2.0 ** -22
        assert near[finite].all().item()
        want[i].view(torch.uint8)[page, off] = cache[i].view(torch.uint8)[page, off]  # the others stay as they were
    fp.kv_cache_write(k, v, cache[0], cache[1], slots.int() if t % 2 else slots, cache[2], cache[3])
    fp.check_paged_error()
    for got, exp in zip(cache[:2], want[:2]):
        assert same_bits(got, exp)
    for got, exp in zip(cache[2:], want[2:]):
        assert got is None or ((got == exp) | ((got - exp).abs() <= 2.0 ** -23 * exp)).all().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_write_of_extreme_rows(dtype):
    """Zeros, the type's least and largest values, infinities and NaN: a row with one that is not finite reads back as NaN, any
    other within half a step."""
    big, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = torch.zeros(8, 1, 128, dtype=dtype, device="cuda")
    rows[1] = big
    rows[1, 0, ::2] = -big
    rows[2] = least
    rows[3, 0, 5] = least * torch.finfo(dtype).eps  # the least denormal
    rows[4, 0, 7] = float("inf")
    rows[5] = 1.0
    rows[5, 0, 127] = -float("inf")
    rows[6] = 1.0
    rows[6, 0, 0] = float("nan")
    rows[7] = torch.linspace(-1, 1, 128, dtype=dtype, device="cuda")
    cache = pu.empty_cache(1, 8, 1, E4M3)
    fp.kv_cache_write(rows, rows, cache[0], cache[1], torch.arange(8, device="cuda"), cache[2], cache[3])
    k, v = torch.empty(1, 8, 1, 128, dtype=dtype, device="cuda"), torch.empty(1, 8, 1, 128, dtype=dtype, device="cuda")
    fp.kv_cache_read(cache[0], cache[1], torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                     torch.tensor([8], dtype=torch.int32, device="cuda"), k, v, cache[2], cache[3])
    fp.check_paged_error()
    assert same_bits(k, v)
    got = k[0].double()
    assert got[[4, 5, 6]].isnan().all()
    assert (got[0] == 0).all()
    for r in (1, 2, 3, 7):
        want = rows[r].double()
        amax = want.abs().max()
        # rows below the floor of 2^-100 count as rows of that size
        tol = want.abs() * (2.0 ** -4 + pu.half_step(dtype)) * 1.001 + max(amax, pu.TINY) / 448 * 2.0 ** -10 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((got[r] - want).abs() <= tol).all(), r


# ------------------------------------------------------------------ read
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("lens,hk,ps,layout", [
    ([1], 1, 16, "hnd"), ([0, 5, 16, 17], 8, 16, "nhd"), ([300, 0, 129], 3, 48, "hnd"), ([1, 2, 3], 2, 1, "nhd"),
    ([2050], 4, 128, "hnd"),
    # calls large enough for the kernel that takes 4 tokens at a time, where 4 divides page_size
    ([3001, 0, 2998, 4099], 8, 16, "nhd"), ([2, 4099, 4098, 4097], 5, 4, "hnd"), ([4099, 3, 4096, 4000], 5, 6, "nhd"),
])
def test_read_matches_the_definition(lens, hk, ps, layout, quant, dtype):
    f = pu.fill_sequences(lens, hk, hk, dtype, E4M3 if quant else dtype, ps, layout, seed=len(lens))
    B, S = len(lens), max(lens) + 3
    big = torch.full((B, S + 1, 2 * hk, 128), 7.0, dtype=dtype, device="cuda")
    k, v = big[:, :S, ::2], torch.full((B, S, hk, 128), 7.0, dtype=dtype, device="cuda")  # heads of a wider tensor; rows of its own
    fp.kv_cache_read(f["k"], f["v"], f["page_table"], f["lens"], k, v, f["k_scale"], f["v_scale"])
    fp.check_paged_error()
    for b, n in enumerate(lens):
        for got, want in ((k, f["rows"][b][0]), (v, f["rows"][b][1])):
            assert same_bits(got[b, :n], want.float().to(dtype))  # code * scale is rounded once to fp32, once to 16 bits
            assert (got[b, n:] == 7.0).all()
    assert (big[:, :, 1::2] == 7.0).all() and (big[:, S] == 7.0).all()


# ------------------------------------------------------------------ decode
def check_decode(f, out, lse, dtype, cache_dtype, sm_scale=128 ** -0.5, lse_too=True):
    for b, (k, v) in enumerate(f["rows"]):
        ref, rl, weight, size = pu.attend64(f["q"][b], k, v, sm_scale)
        to, tl = pu.decode_bounds(ref, rl, weight, size, k.shape[0], dtype, cache_dtype, f["q"][b], k, v, sm_scale)
        err = (out[b].double() - ref).abs()
        assert (err <= to).all(), (b, k.shape[0], (err / to.clamp_min(1e-30)).max().item())
        if not lse_too:
            continue
        if k.shape[0] == 0:
            assert (lse[b] == -float("inf")).all()
        else:
            assert ((lse[b].double() - rl).abs() <= tl).all(), (b, ((lse[b].double() - rl).abs() / tl).max().item())


DECODE_CASES = [  # lens, q heads, kv heads, page size, layout
    ([1], 1, 1, 16, "hnd"),
    ([0, 1, 15, 16, 17, 31, 32, 33], 8, 2, 16, "nhd"),
    ([63, 64, 65, 127, 128, 129, 0, 257], 32, 8, 16, "nhd"),
    ([500, 3, 1000], 28, 4, 64, "hnd"),
    ([777], 7, 7, 48, "hnd"),
    ([5, 40], 12, 1, 1, "nhd"),
    ([1100, 90], 16, 1, 5, "hnd"),
    ([300, 200], 40, 2, 16, "nhd"),   # 20 heads a KV head: two groups
    ([130], 33, 1, 128, "hnd"),       # three groups of 11
    ([6000, 1], 8, 8, 128, "hnd"),
    ([40000], 4, 1, 256, "nhd"),
    ([20000, 0, 3, 9000, 65, 17001], 8, 2, 64, "hnd"),
    ([100] * 150, 8, 2, 16, "nhd"),
    ([70, 0, 9, 300] * 10, 24, 2, 32, "hnd"),  # 12 heads a KV head, more items than half the SMs
    ([2000, 5], 128, 4, 16, "nhd"),            # 32 heads a KV head
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("wide", [False, True])  # the table's width decides between clusters and stretches
@pytest.mark.parametrize("case", range(len(DECODE_CASES)))
def test_decode_matches_the_definition(case, wide, quant, dtype):
    lens, hq, hk, ps, layout = DECODE_CASES[case]
    cd = E4M3 if quant else dtype
    f = pu.fill_sequences(lens, hq, hk, dtype, cd, ps, layout, seed=case, room=70000 if wide else 0)
    assert not wide or fp.paged_decode_workspace_bytes(len(lens), hq, hk, cd, f["page_table"].shape[1], ps) > 0
    out = torch.full_like(f["q"], float("nan"))
    lse = torch.full((len(lens), hq), float("nan"), device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"])
    fp.check_paged_error()
    check_decode(f, out, lse, dtype, cd)


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("gain", [1e-3, 8.0])
def test_decode_flat_and_peaked_rows(quant, gain):
    """Weights that are all alike, and rows where one token takes nearly all of the weight."""
    for dtype in (BF16, FP16):
        f = pu.fill_sequences([3000, 70], 8, 2, dtype, E4M3 if quant else dtype, 16, seed=5, k_gain=gain)
        out, lse = torch.empty_like(f["q"]), torch.empty(2, 8, device="cuda")
        fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"], sm_scale=0.3)
        check_decode(f, out, lse, dtype, E4M3 if quant else dtype, 0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
def test_decode_of_large_bf16_queries(quant):
    """Queries beyond fp16's range (an e4m3 cache is multiplied in fp16) and very small ones."""
    for mult in (2.0 ** 20, 2.0 ** -27):
        f = pu.fill_sequences([200], 4, 1, BF16, E4M3 if quant else BF16, 16, seed=6)
        f["q"] = f["q"] * mult
        out, lse = torch.empty_like(f["q"]), torch.empty(1, 4, device="cuda")
        fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, f["k_scale"], f["v_scale"],
                        sm_scale=0.1 / mult)
        check_decode(f, out, lse, BF16, E4M3 if quant else BF16, 0.1 / mult)


@pytest.mark.gpu
def test_decode_without_lse_strided_and_in_place():
    f = pu.fill_sequences([900, 33, 0], 8, 2, BF16, BF16, 16, seed=8)
    args = (f["k"], f["v"], f["page_table"], f["lens"])
    want = torch.empty_like(f["q"])
    fp.paged_decode(f["q"], *args, want)
    wide = torch.full((3, 20, 256), 5.0, dtype=BF16, device="cuda")
    wide[:, 2:18:2, :128] = f["q"]
    fp.paged_decode(wide[:, 2:18:2, :128], *args, wide[:, 2:18:2, :128])  # strided, out over q
    assert same_bits(wide[:, 2:18:2, :128], want)
    assert (wide[:, ::2][:, [0, 9]] == 5.0).all() and (wide[:, 1::2] == 5.0).all() and (wide[:, :, 128:] == 5.0).all()
    odd = torch.empty(3, 8, 129, dtype=BF16, device="cuda")[:, :, 1:]  # rows at odd addresses
    odd.copy_(f["q"])
    out = torch.empty(3, 8, 129, dtype=BF16, device="cuda")[:, :, 1:]
    fp.paged_decode(odd, *args, out)
    assert same_bits(out, want)
    table = torch.full((3, 200), 2 ** 30, dtype=torch.int32, device="cuda")  # part of a wider table
    table[:, :f["page_table"].shape[1]] = f["page_table"]
    fp.paged_decode(f["q"], f["k"], f["v"], table[:, :f["page_table"].shape[1]], f["lens"], out)
    assert same_bits(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("room", [0, 50000])
def test_bad_pages_lengths_and_slots_are_reported_and_skipped(room, quant):
    dtype = BF16
    cd = E4M3 if quant else dtype
    f = pu.fill_sequences([200, 90, 64], 8, 2, dtype, cd, 16, seed=9, room=room)
    scales = (f["k_scale"], f["v_scale"])
    # a page that is not in the cache: its tokens are left out
    for bad in (-1, f["pages"], 2 ** 31 - 1):
        f["page_table"][0, 3] = bad
        out, lse = torch.empty_like(f["q"]), torch.empty(3, 8, device="cuda")
        fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse, *scales)
        with pytest.raises(fp.FlashPrefillError, match="outside the paged cache"):
            fp.check_paged_error()
        fp.check_paged_error()  # reported once
        g = dict(f, rows=[[torch.cat([x[:48], x[64:]]) for x in f["rows"][0]]] + f["rows"][1:])
        check_decode(g, out, lse, dtype, cd)
    # lengths outside the room: zeros, -inf, and no other sequence touched
    for bad in (-1, f["page_table"].shape[1] * 16 + 1, 2 ** 31 - 1):
        lens = f["lens"].clone()
        lens[1] = bad
        out, lse = torch.full_like(f["q"], float("nan")), torch.empty(3, 8, device="cuda")
        fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], lens, out, lse, *scales)
        with pytest.raises(fp.FlashPrefillError, match="sequence length"):
            fp.check_paged_error()
        assert (out[1] == 0).all() and (lse[1] == -float("inf")).all() and not out.isnan().any()
        k = torch.full((3, 200, 2, 128), 7.0, dtype=dtype, device="cuda")
        v = k.clone()
        fp.kv_cache_read(f["k"], f["v"], f["page_table"], lens, k, v, *scales)
        with pytest.raises(fp.FlashPrefillError, match="sequence length"):
            fp.check_paged_error()
        assert (k[1] == 7.0).all() and (v[1] == 7.0).all() and (k[2, 64:] == 7.0).all() and (k[2, :64] != 7.0).any()
    # slots beyond the cache
    before = [None if t is None else t.clone() for t in (f["k"], f["v"], *scales)]
    rows = torch.ones(3, 2, 128, dtype=dtype, device="cuda")
    fp.kv_cache_write(rows, rows, f["k"], f["v"], torch.tensor([f["pages"] * 16, -1, 2 ** 40], device="cuda"), *scales)
    with pytest.raises(fp.FlashPrefillError, match="outside the paged cache"):
        fp.check_paged_error()
    for a, b in zip((f["k"], f["v"], *scales), before):
        assert a is None or same_bits(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 100000])
def test_decode_is_deterministic_and_captured_graphs_serve_other_lengths(room):
    """One capture, replayed for other lengths, tables and queries; a second graph on another stream beside it."""
    f = pu.fill_sequences([4000, 130, 700, 64], 32, 8, BF16, BF16, 16, seed=10, room=room)
    q, table, lens = f["q"].clone(), f["page_table"].clone(), f["lens"].clone()
    args = (f["k"], f["v"], table, lens)
    outs = [torch.empty_like(q) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    fp.paged_decode(q, *args, outs[0])  # loads the kernels
    torch.cuda.synchronize()
    graphs = []
    for s, o in zip(streams, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            fp.paged_decode(q, *args, o)
        graphs.append(g)
    for perm in ([0, 1, 2, 3], [3, 0, 2, 1], [2, 2, 0, 0]):
        q.copy_(f["q"][perm])
        table.copy_(f["page_table"][perm])
        lens.copy_(f["lens"][perm])
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(3):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(q)
        fp.paged_decode(q, *args, want)
        for o in outs:
            assert same_bits(o, want)
    fp.check_paged_error()


@pytest.mark.gpu
def test_given_workspace_needs_no_initialisation_and_small_ones_are_refused():
    f = pu.fill_sequences([3000, 10], 8, 2, FP16, FP16, 16, seed=11, room=40000)
    n = fp.paged_decode_workspace_bytes(2, 8, 2, FP16, f["page_table"].shape[1], 16)
    args = (f["q"], f["k"], f["v"], f["page_table"], f["lens"])
    want, out = torch.empty_like(f["q"]), torch.empty_like(f["q"])
    fp.paged_decode(*args, want)
    for fill in (0, 255):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        fp.paged_decode(*args, out, workspace=ws)
        fp.paged_decode(*args, out, workspace=ws)
        assert same_bits(out, want)
    with pytest.raises(ValueError, match="workspace too small"):
        fp.paged_decode(*args, out, workspace=ws[:n - 256])
    with pytest.raises(ValueError, match="CUDA"):
        fp.paged_decode(*args, out, workspace=ws.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
def test_offsets_beyond_32_bits(quant):
    """Pages further apart than 2^31 elements together: writing, reading back and attending to the last of them."""
    dtype, cd = BF16, E4M3 if quant else BF16
    pages, ps, hk, gap = 20, 16, 2, 1 << 28
    def pool():
        flat = torch.empty((pages - 1) * gap + ps * hk * 128, dtype=torch.uint8 if quant else dtype, device="cuda")
        flat = flat.view(cd) if quant else flat
        return flat.as_strided((pages, ps, hk, 128), (gap, hk * 128, 128, 1))
    k_cache, v_cache = pool(), pool()
    scales = [torch.empty(pages, ps, hk, device="cuda") for _ in range(2)] if quant else [None, None]
    n = pages * ps
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(n, hk, 128, generator=g, device="cuda").to(dtype) for _ in range(2))
    fp.kv_cache_write(k, v, k_cache, v_cache, torch.arange(n, device="cuda"), *scales)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    kr, vr = torch.empty(1, n, hk, 128, dtype=dtype, device="cuda"), torch.empty(1, n, hk, 128, dtype=dtype, device="cuda")
    fp.kv_cache_read(k_cache, v_cache, table, lens, kr, vr, *scales)
    if not quant:
        assert same_bits(kr[0], k) and same_bits(vr[0], v)
    q = torch.randn(1, 8, 128, generator=g, device="cuda").to(dtype)
    out, lse = torch.empty_like(q), torch.empty(1, 8, device="cuda")
    fp.paged_decode(q, k_cache, v_cache, table, lens, out, lse, *scales)
    fp.check_paged_error()
    if quant:
        rows = [c.view(torch.uint8).reshape(n, hk, 128).view(E4M3).double() * s.reshape(n, hk, 1).double()
                for c, s in zip((k_cache, v_cache), scales)]
    else:
        rows = [k.double(), v.double()]
    check_decode(dict(q=q, rows=[rows]), out, lse, dtype, cd)


@pytest.mark.gpu
def test_values_that_are_not_finite_follow_the_softmax():
    """A NaN in a cached row of a sequence spoils that sequence's heads only; a key with -inf score has no weight; a query of
    zeros averages; stale NaN rows behind the length never count (every other test has them)."""
    f = pu.fill_sequences([100, 100, 100], 4, 2, FP16, FP16, 16, seed=12)
    page = f["page_table"]
    f["v"][page[0, 1].long(), 3, 1, 5] = float("nan")
    f["k"][page[1, 2].long(), 4] = -float("inf")
    f["q"][1] = f["q"][1].abs() + 0.1
    f["q"][2] = 0
    out, lse = torch.empty_like(f["q"]), torch.empty(3, 4, device="cuda")
    fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], out, lse)
    assert out[0, 2:, 5].isnan().all() and not out[0, :2].isnan().any() and not out[0, 2:, :5].isnan().any()
    keep = [i for i in range(100) if i != 36]
    g = dict(q=f["q"][1:], rows=[[x[keep] for x in f["rows"][1]], f["rows"][2]])
    for b, h in ((0, slice(0, 2)), (1, slice(0, 4))):
        k, v = g["rows"][b]
        ref, rl, weight, size = pu.attend64(g["q"][b], k, v)
        to, tl = pu.decode_bounds(ref, rl, weight, size, k.shape[0], FP16, FP16, g["q"][b], k, v)
        assert ((out[1 + b].double() - ref).abs() <= to)[h].all() and ((lse[1 + b].double() - rl).abs() <= tl)[h].all()


@pytest.mark.gpu
def test_python_refusals():
    f = pu.fill_sequences([20, 30], 8, 2, BF16, E4M3, 16, seed=13)
    q, k, v, t, n, ks, vs = (f[x] for x in ("q", "k", "v", "page_table", "lens", "k_scale", "v_scale"))
    out = torch.empty_like(q)
    ok = dict(q=q, k_cache=k, v_cache=v, page_table=t, seq_lens=n, out=out, k_scale=ks, v_scale=vs)
    fp.paged_decode(**ok)
    for over, err, msg in [
        (dict(q=q.float()), TypeError, "bfloat16"), (dict(q=q[0]), ValueError, "dimensions"), (dict(out=out[:1]), ValueError, "out"),
        (dict(out=out.half()), ValueError, "out"), (dict(out=out[:, :1].expand(2, 8, 128)), ValueError, "expanded"),
        (dict(out=torch.empty(2, 8, 256, dtype=BF16, device="cuda")[:, :, ::2]), ValueError, "contiguous"),
        (dict(k_scale=None), ValueError, "k_scale"), (dict(k_scale=ks[:1]), ValueError, "shape"),
        (dict(k_scale=ks.double(), v_scale=vs.double()), TypeError, "float32"), (dict(v_scale=vs.contiguous()), ValueError, "strides"),
        (dict(v_cache=v.contiguous()), ValueError, "share"), (dict(k_cache=k[..., :64], v_cache=v[..., :64]), ValueError, "128"),
        (dict(k_cache=k.half(), v_cache=v.half(), k_scale=None, v_scale=None), TypeError, "float8"),
        (dict(k_cache=k.to(BF16), v_cache=v.to(BF16)), ValueError, "no scales"),
        (dict(page_table=t.long()), TypeError, "int32"), (dict(seq_lens=n.long()), TypeError, "int32"),
        (dict(page_table=t[:1]), ValueError, "rows"), (dict(seq_lens=n[:1]), ValueError, "rows"),
        (dict(page_table=t.t().contiguous().t()), ValueError, "contiguous"), (dict(seq_lens=n.cpu()), ValueError, "CUDA"),
        (dict(lse=torch.empty(2, 8, dtype=torch.float64, device="cuda")), ValueError, "lse"),
        (dict(lse=torch.empty(8, 2, device="cuda").t()), ValueError, "lse"), (dict(q=q[:, :7], out=out[:, :7]), ValueError, "multiple"),
        (dict(sm_scale=float("inf")), ValueError, "sm_scale"),
    ]:
        with pytest.raises(err, match=msg):
            fp.paged_decode(**{**ok, **over})
    rows = torch.zeros(3, 2, 128, dtype=BF16, device="cuda")
    slots = torch.arange(3, device="cuda")
    for a, err, msg in [
        ((rows, rows[:2], k, v, slots, ks, vs), ValueError, "shape"), ((rows, rows.half(), k, v, slots, ks, vs), TypeError, "dtype"),
        ((rows[:, :1], rows[:, :1], k, v, slots, ks, vs), ValueError, "KV heads"), ((rows, rows, k, v, slots[:2], ks, vs), ValueError, "slots"),
        ((rows, rows, k, v, slots.float(), ks, vs), TypeError, "slots"), ((rows, rows, k, v, slots[None], ks, vs), ValueError, "dimensions"),
        ((rows, rows, k[:1].expand_as(k), v[:1].expand_as(v), slots, ks, vs), ValueError, "expanded"),
        ((rows, rows, k, k, slots, ks, vs), ValueError, "same memory"),
    ]:
        with pytest.raises(err, match=msg):
            fp.kv_cache_write(*a)
    to, to2 = (torch.zeros(2, 40, 2, 128, dtype=BF16, device="cuda") for _ in range(2))
    for a, err, msg in [
        ((k, v, t, n, to, to[:, :20], ks, vs), ValueError, "share"), ((k, v, t, n, to[..., ::2], to[..., ::2], ks, vs), ValueError, "contiguous"),
        ((k, v, t, n, to.float(), to.float(), ks, vs), TypeError, "bfloat16"), ((k, v, t[:1], n, to, to2, ks, vs), ValueError, "rows"),
        ((k, v, t, n, to[:, :1].expand_as(to), to, ks, vs), ValueError, "expanded"), ((k, v, t, n, to, to, ks, vs), ValueError, "same memory"),
    ]:
        with pytest.raises(err, match=msg):
            fp.kv_cache_read(*a)
    fp.check_paged_error()


@pytest.mark.gpu
def test_empty_calls_do_nothing():
    c = fp.kv_cache_alloc(4, 16, 2)
    none = torch.empty(0, 2, 128, dtype=BF16, device="cuda")
    table, lens = torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    fp.kv_cache_write(none, none, *c[:2], torch.empty(0, dtype=torch.int64, device="cuda"))
    fp.paged_decode(none, *c[:2], table, lens, torch.empty_like(none))
    fp.kv_cache_read(*c[:2], table, lens, none[:, None], none[:, None])
    fp.check_paged_error()


@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own():
    """Calls from two threads at once, each on its own stream with a workspace from the allocator: each gets its own result."""
    import threading
    fs = [pu.fill_sequences([9000 + 50 * i, 130, 0], 8, 2, BF16, E4M3 if i else BF16, 16, seed=20 + i, room=60000) for i in range(2)]
    want = []
    for f in fs:
        o = torch.empty_like(f["q"])
        fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], o, None, f["k_scale"], f["v_scale"])
        want.append(o)
    torch.cuda.synchronize()
    bad = []

    def work(i):
        f = fs[i]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                o = torch.empty_like(f["q"])
                fp.paged_decode(f["q"], f["k"], f["v"], f["page_table"], f["lens"], o, None, f["k_scale"], f["v_scale"])
                if not same_bits(o, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad
    fp.check_paged_error()


@pytest.mark.gpu
def test_a_call_waits_for_what_the_stream_holds():
    """Rows written, read and attended to in one go behind a long kernel, many times over: no call may see what its predecessors
    on the stream have not finished (its launch is prepared while they run)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(4096, 4096, generator=g, device="cuda", dtype=BF16)
    cache = fp.kv_cache_alloc(64, 16, 2)
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    n = 1000
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    slots = torch.arange(n, device="cuda")
    q = torch.randn(1, 8, 128, generator=g, device="cuda").to(BF16)
    for i in range(20):
        k, v = (torch.randn(n, 2, 128, generator=g, device="cuda").to(BF16) for _ in range(2))
        torch.cuda.synchronize()
        big @ big
        late_k, late_v = k * 1.0, v * 1.0  # made on the stream just before the write
        kr, vr, out = torch.empty(1, n, 2, 128, dtype=BF16, device="cuda"), torch.empty(1, n, 2, 128, dtype=BF16, device="cuda"), torch.empty_like(q)
        fp.kv_cache_write(late_k, late_v, cache.k, cache.v, slots)
        fp.paged_decode(q, cache.k, cache.v, table, lens, out)
        fp.kv_cache_read(cache.k, cache.v, table, lens, kr, vr)
        after = out + 0  # and nothing behind a call may run ahead of it
        torch.cuda.synchronize()
        assert same_bits(kr[0], k) and same_bits(vr[0], v)
        check_decode(dict(q=q, rows=[[k.double(), v.double()]]), after, torch.full((1, 8), float("nan"), device="cuda"), BF16, BF16, lse_too=False)


@pytest.mark.gpu
def test_checked_mode_raises_from_the_call(tmp_path):
    """FLASHPREFILL_B200_CHECK=1 (read at import): two rows for one slot and a slot outside the cache raise from the call."""
    import subprocess
    import sys
    code = """
import torch, flashprefill_b200 as fp
c = fp.kv_cache_alloc(4, 16, 1)
r = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device="cuda")
fp.kv_cache_write(r, r, c.k, c.v, torch.tensor([3, 4], device="cuda"))
for slots, err in (([5, 5], ValueError), ([1, 64], fp.FlashPrefillError)):
    try:
        fp.kv_cache_write(r, r, c.k, c.v, torch.tensor(slots, device="cuda"))
    except err as e:
        print(type(e).__name__)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, FLASHPREFILL_B200_CHECK="1", PYTHONPATH=root), capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["ValueError", "FlashPrefillError"], r.stdout + r.stderr
