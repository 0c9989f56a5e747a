"""The engine in 8-bit integers on the CPU: the int8 cache and 8-bit projections through the generate loop."""

from __future__ import annotations

import pytest
import torch

from liteinfer_amd.attention import eager_attention
from liteinfer_amd.engine import model as model_module
from liteinfer_amd.engine.llm import LLM, EngineConfig
from liteinfer_amd.engine.model import LlamaShape, RandomLlama
from liteinfer_amd.engine.ops import Int8Weight
from tests.engine_helpers import random_prompts

TINY = LlamaShape(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=96,
                  vocab_size=200)



@pytest.fixture(autouse=True)
def dense_attention_on_the_cpu(monkeypatch):
    """The model calls the paged kernels; a CPU model attends with the dense ones."""
    paged = model_module.paged_attention

    def attend(query, kv, scaling, groups):
        return (paged if query.is_cuda else eager_attention)(query, kv, scaling, groups)

    monkeypatch.setattr(model_module, "paged_attention", attend)


def _generate(model, **kw):
    config = EngineConfig(max_num_seqs=4, max_model_len=128, max_num_batched_tokens=24, num_gpu_blocks=64, use_graphs=False,
                          **kw)
    llm = LLM(model, config)
    return llm.generate_ids(random_prompts(6, 3, 40, TINY.vocab_size), max_tokens=5), llm


@pytest.mark.parametrize("weight_quant", [None, "int8"])
def test_the_engine_generates_over_an_int8_cache(weight_quant):
    model = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=1, std=0.1, weight_quant=weight_quant)
    (outputs, stats), llm = _generate(model, cache_quant="int8")
    assert stats.output_tokens == 30 and stats.logits_finite
    assert llm.cache.pool.slots(0)[0].dtype == torch.int8
    assert llm.cache.pool.num_free_blocks == 63  # (the padding slot's block stays)
    again, _ = _generate(model, cache_quant="int8")
    assert again[0] == outputs


def test_eight_bit_weights_are_the_models_rounded():
    plain = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=2)
    model = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=2, weight_quant="int8")
    assert torch.equal(model.embed, plain.embed) and torch.equal(model.lm_head, plain.lm_head)
    for a, b in zip(plain.layers, model.layers):
        for name in ("w_qkv", "w_o", "w_gate_up", "w_down"):
            w, q = getattr(a, name), getattr(b, name)
            assert isinstance(q, Int8Weight)
            off = (q.codes * q.scales[:, None] - w).abs()
            assert (off <= q.scales[:, None] / 2 * (1 + 2.0 ** -16)).all()
    assert model.parameter_bytes() < plain.parameter_bytes()


def test_an_unknown_format_is_refused():
    with pytest.raises(ValueError, match="weight_quant"):
        RandomLlama(TINY, device="cpu", weight_quant="int4")
