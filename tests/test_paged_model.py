"""The paged cache's operators together, as a server runs them: a prompt in chunks (flash_prefill over a prefix read back from the
cache), then tokens one by one; and the Llama model's prefill / decode methods against its whole-sequence forward."""
import pytest
import torch

import flashprefill_b200 as fp
from flashprefill_b200.llama_prefill import LlamaCache, LlamaConfig, TPLlamaPrefill
from tests import paged_util as pu

E4M3 = torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16


def test_cache_slots_follow_the_page_table():
    table = torch.tensor([[3, 0], [2, 5]], dtype=torch.int32)
    k = torch.empty(6, 16, 2, 128)
    cache = LlamaCache([fp.KVCache(k, k, None, None)], table, torch.zeros(2, dtype=torch.int32), [0, 0], (None, None))
    assert cache.page_size == 16 and cache.max_len == 32
    got = cache.slots(torch.tensor([0, 0, 1]), torch.tensor([1, 17, 31]))
    assert got.tolist() == [3 * 16 + 1, 1, 5 * 16 + 15]


def test_prefill_refuses_sequences_that_are_not_there():
    m = TPLlamaPrefill(LlamaConfig(layers=1, hidden=128, q_heads=1, kv_heads=1, ffn=128, vocab=16), device="cpu", dtype=torch.float32)
    cache = m.new_cache(2, 32, page_size=16, dtype=BF16)
    for seq in (-1, 2):
        with pytest.raises(ValueError, match="sequence"):
            m.prefill(torch.zeros(3, dtype=torch.int64), cache, seq)
    with pytest.raises(ValueError, match="fit"):
        m.prefill(torch.zeros(33, dtype=torch.int64), cache, 1)
    with pytest.raises(ValueError, match="fit"):
        m.prefill(torch.zeros(0, dtype=torch.int64), cache, 1)


def test_registered_ops_trace_and_mutate():
    from torch._subclasses.fake_tensor import FakeTensorMode
    for name, muts in (("kv_cache_write", ("k_cache", "v_cache", "k_scale", "v_scale")), ("kv_cache_read", ("k", "v")),
                       ("paged_decode", ("out", "lse"))):
        args = {a.name: a for a in getattr(torch.ops.flashprefill, name).default._schema.arguments}
        for m in muts:
            assert args[m].alias_info is not None and args[m].alias_info.is_write
    with FakeTensorMode():
        e = lambda *s, dt=BF16: torch.empty(*s, dtype=dt, device="cuda")
        kc, table, lens = e(8, 16, 2, 128), e(4, 2, dt=torch.int32), e(4, dt=torch.int32)
        torch.ops.flashprefill.kv_cache_write(e(4, 2, 128), e(4, 2, 128), kc, kc, e(4, dt=torch.int64), None, None)
        torch.ops.flashprefill.kv_cache_read(kc, kc, table, lens, e(4, 32, 2, 128), e(4, 32, 2, 128))
        torch.ops.flashprefill.paged_decode(e(4, 8, 128), kc, kc, table, lens, e(4, 8, 128), None)


@pytest.mark.gpu
def test_registered_ops_match_the_entry_points():
    f = pu.fill_sequences([40, 700], 8, 2, BF16, E4M3, 16, seed=3)
    args = (f["q"], f["k"], f["v"], f["page_table"], f["lens"])
    a, b = torch.empty_like(f["q"]), torch.empty_like(f["q"])
    la, lb = torch.empty(2, 8, device="cuda"), torch.empty(2, 8, device="cuda")
    fp.paged_decode(*args, a, la, f["k_scale"], f["v_scale"])
    torch.ops.flashprefill.paged_decode(*args, b, lb, f["k_scale"], f["v_scale"])
    assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("quant", [False, True])
def test_prompt_in_chunks_then_tokens(quant, layout):
    """Every step against the definition: the cache holds each row as written (quantised where it is), a chunk attends to the
    rows read back and its own, a token to the rows in the cache."""
    dtype, cd, hq, hk, ps = BF16, E4M3 if quant else BF16, 8, 2, 48
    chunks, steps = [700, 133, 1], 4
    total = sum(chunks) + steps
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(total, h, 128, generator=g, device="cuda").to(dtype) for h in (hq, hk, hk))
    pages = -(-total // ps)
    kc, vc, ks, vs = pu.empty_cache(pages + 2, ps, hk, cd, layout)
    order = torch.randperm(pages + 2, generator=g, device="cuda")[:pages]
    table = order.to(torch.int32)[None]
    pos = torch.arange(total, device="cuda")
    slots = order[pos // ps] * ps + pos % ps

    def held(x):  # a row as the cache stands for it, in 64 bits
        if not quant:
            return x.double()
        codes, s = pu.quantise(x.float())
        return codes.double() * s.double()[..., None]

    n = 0
    for c in chunks:
        out = torch.empty(1, c, hq, 128, dtype=dtype, device="cuda")
        kw, vw = (torch.full((1, n + c, hk, 128), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        fp.kv_cache_read(kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"), kw, vw, ks, vs)
        want = held(k[:n])
        # read back: one step of the scale's quotient and product in fp32 and one rounding to 16 bits
        # a code may be the neighbour of the definition's where fp32 rounds to another side of a tie: one e4m3 step, 2^-3
        step = 2.0 ** -3 if quant else 0.0
        floor = want.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -9 if quant else 0.0
        assert ((kw[0, :n].double() - want).abs() <= want.abs() * (step + pu.half_step(dtype)) * 1.01 + floor).all().item()
        kw[0, n:], vw[0, n:] = k[n:n + c], v[n:n + c]
        assert not kw.isnan().any() and not vw.isnan().any()
        fp.flash_prefill(q[None, n:n + c], kw, vw, out, 128, 2, 4, 0.0, 2, 0)  # alpha 0: every block
        for i in (0, c - 1):
            ref, _, _, _ = pu.attend64(q[n + i], kw[0, :n + i + 1].double(), vw[0, :n + i + 1].double())
            assert ((out[0, i].double() - ref).abs() <= 2e-2).all()  # the prefill's own tolerance
        fp.kv_cache_write(k[n:n + c], v[n:n + c], kc, vc, slots[n:n + c], ks, vs)
        n += c
    for _ in range(steps):
        fp.kv_cache_write(k[n:n + 1], v[n:n + 1], kc, vc, slots[n:n + 1], ks, vs)
        n += 1
        out, lse = torch.empty(1, hq, 128, dtype=dtype, device="cuda"), torch.empty(1, hq, device="cuda")
        fp.paged_decode(q[n - 1:n], kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"), out, lse, ks, vs)
        page, at = slots[:n] // ps, slots[:n] % ps
        rows = [c.view(torch.uint8)[page, at].view(E4M3).double() * s[page, at].double()[..., None] if quant
                else c[page, at].double() for c, s in ((kc, ks), (vc, vs))]
        ref, rl, weight, size = pu.attend64(q[n - 1], *rows)
        to, tl = pu.decode_bounds(ref, rl, weight, size, n, dtype, cd, q[n - 1], *rows)
        assert ((out[0].double() - ref).abs() <= to).all() and ((lse[0].double() - rl).abs() <= tl).all()
    fp.check_paged_error()


def _small(device):
    cfg = LlamaConfig(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=4096, alpha=0.0)
    return cfg, TPLlamaPrefill(cfg, 0, 1, device=device, seed=7)


@pytest.mark.gpu
def test_model_answers_as_its_forward_does():
    """Two prompts of different lengths, one in two chunks, then tokens together: each step's logits against the whole sequence's
    forward (every block selected), at the tolerance of the forward's own test."""
    cfg, m = _small("cuda:0")
    g = torch.Generator().manual_seed(2)
    ids = [torch.randint(0, cfg.vocab, (n,), generator=g).cuda() for n in (300, 77)]
    new = torch.randint(0, cfg.vocab, (2, 3), generator=g).cuda()
    cache = m.new_cache(2, 400, page_size=16)
    m.prefill(ids[0][:190], cache, 0)
    got = [m.prefill(ids[0][190:], cache, 0), m.prefill(ids[1], cache, 1)]
    near = lambda a, b: (a - b).abs().max().item() / b.abs().max().item() < 2e-2
    assert near(got[0], m.forward(ids[0])) and near(got[1], m.forward(ids[1]))
    for t in range(new.shape[1]):
        logits = m.decode(new[:, t], cache)
        for b in range(2):
            assert near(logits[b], m.forward(torch.cat([ids[b], new[b, :t + 1]])))
    assert cache.lens == [303, 80] and cache.seq_lens.tolist() == [303, 80]
    with pytest.raises(ValueError, match="fit"):
        m.prefill(ids[0], cache, 0)
    with pytest.raises(ValueError, match="sequences"):
        m.decode(new[:1, 0], cache)
    fp.check_paged_error()


@pytest.mark.gpu
def test_model_with_a_quantised_cache_runs():
    """An e4m3 cache changes the logits by what its values' rounding does to them: the model run on keys and values rounded the
    same way, by the definition, gives the same logits."""
    cfg, m = _small("cuda:0")
    ids = torch.randint(0, cfg.vocab, (150,), generator=torch.Generator().manual_seed(4)).cuda()
    cache = m.new_cache(1, 200, dtype=E4M3)
    m.prefill(ids[:-1], cache)
    got = m.decode(ids[-1:], cache)[0]

    # the same two steps in plain form: the prompt attends to its own rows, the token to the rounded ones
    kept = []
    def attention(q, k, v, out, c):
        n = len(kept)
        if q.shape[1] > 1:
            kept.append([k, v])
            for i in range(q.shape[1]):
                out[0, i] = pu.attend64(q[0, i], k[0, :i + 1].double(), v[0, :i + 1].double())[0].to(out.dtype)
    whole = TPLlamaPrefill(cfg, 0, 1, device="cuda:0", seed=7, attention=attention)
    whole.forward(ids[:-1])
    layer = iter(kept)
    def token(q, k, v):
        rows = []
        for x, new in zip(next(layer), (k, v)):
            codes, s = pu.quantise(torch.cat([x[0], new]).float())
            rows.append(codes.double() * s.double()[..., None])
        return pu.attend64(q[0], *rows)[0].to(q.dtype).reshape(1, -1)
    x = whole.embed[ids[-1:]]
    cos, sin = (t[149:150] for t in cache.rope)
    with torch.no_grad():
        for L in whole.layers:
            x = whole._layer(L, x, cos, sin, token)
        want = whole._logits(x)[0]
    assert (got - want).abs().max().item() / want.abs().max().item() < 2e-2
