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
