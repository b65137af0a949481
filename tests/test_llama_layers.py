"""What the Llama harness holds and moves beside its kernels: hidden states of a layer, the LM head of a token."""
import gc

import pytest
import torch

from flashprefill_b200.llama_prefill import LlamaConfig, TPLlamaPrefill
from tests.test_llama_prefill import SMALL, dense_causal


def test_forward_holds_one_hidden_state(monkeypatch):
    """Where a layer's products are reduced, the hidden rows, their normalised form and the product are alive, and no second hidden
    state."""
    cfg = LlamaConfig(**SMALL)
    m = TPLlamaPrefill(cfg, 0, 1, device="cpu", dtype=torch.float32, seed=3, attention=dense_causal)
    tokens = torch.randint(0, cfg.vocab, (77,), generator=torch.Generator().manual_seed(1))
    alive = []

    def reduce(x):
        gc.collect()
        alive.append(len({t.data_ptr() for t in gc.get_objects() if type(t) is torch.Tensor and tuple(t.shape) == (77, cfg.hidden)}))
        return x

    monkeypatch.setattr(m, "_reduce", reduce)
    m.forward(tokens)
    assert len(alive) == 2 * cfg.layers and max(alive) == 3


def test_layers_leave_the_embedding_alone():
    cfg = LlamaConfig(**SMALL)
    m = TPLlamaPrefill(cfg, 0, 1, device="cpu", dtype=torch.float32, seed=3, attention=dense_causal)
    before = m.embed.clone()
    tokens = torch.arange(cfg.vocab)[-50:]
    first = m.forward(tokens)
    assert torch.equal(m.embed, before) and torch.equal(m.forward(tokens), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 3, 33])
def test_token_logits_are_summed_in_32_bits_without_a_wide_head(rows, dtype):
    cfg = LlamaConfig(layers=0, hidden=1024, q_heads=8, kv_heads=2, ffn=2048, vocab=20001)
    m = TPLlamaPrefill(cfg, device="cuda:0", dtype=dtype, seed=4)
    x = torch.randn(rows, cfg.hidden, generator=torch.Generator("cuda").manual_seed(rows), device="cuda").to(dtype)
    m._token_logits(x)  # cuBLAS takes its workspace
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = m._token_logits(x)
    assert torch.cuda.max_memory_allocated() - before < 2 * m.lm_head.numel()  # bytes: less than a second head, let alone a wide one
    assert got.dtype is torch.float32 and got.shape == (rows, cfg.vocab)
    last = x.float()
    last = (last * torch.rsqrt(last.pow(2).mean(-1, keepdim=True) + cfg.eps)).to(dtype).double()
    head = m.lm_head.double()
    # exact products; 1024 of them summed in fp32, each step off by 2^-23 at the most (tensor cores truncate)
    bound = cfg.hidden * 2.0 ** -23 * (last.abs() @ head.abs().t())
    assert ((got.double() - last @ head.t()).abs() <= bound).all()


def test_token_logits_on_the_cpu_are_the_prompts():
    m = TPLlamaPrefill(LlamaConfig(**SMALL), device="cpu", dtype=torch.float32, seed=3, attention=dense_causal)
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1))
    assert torch.equal(m._token_logits(x), m._logits(x))


def test_cached_steps_refuse_to_be_captured(monkeypatch):
    m = TPLlamaPrefill(LlamaConfig(**SMALL), device="cpu", dtype=torch.float32, seed=3, attention=dense_causal)
    cache = m.new_cache(2, 64, page_size=16, dtype=torch.bfloat16)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="prefill .*captured"):
        m.prefill(torch.zeros(3, dtype=torch.int64), cache)
    with pytest.raises(RuntimeError, match="decode .*captured"):
        m.decode(torch.zeros(2, dtype=torch.int64), cache)
    assert cache.lens == [0, 0]
