"""GraphedDecoder and PagedDecoder refuse models whose steps they would compute differently (no GPU needed)."""
import pytest
import torch

import decoder
from decoder import GraphedDecoder, PagedDecoder

CONFIG = dict(vocab_size=64, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, head_dim=16, max_position_embeddings=128)


def model(**kw):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    return LlamaForCausalLM(LlamaConfig(**CONFIG, **kw)).eval()


def filled(m, *names):
    """The named biases of the last layer, no longer zero."""
    at = m.model.layers[-1]
    for name in names:
        at.get_submodule(name).bias.data.fill_(0.5)
    return m


def refused(m, match, max_tokens=64, graphed=True):
    with pytest.raises(ValueError, match=match):
        PagedDecoder(m, batch=2, max_tokens=max_tokens)
    if graphed:
        with pytest.raises(ValueError, match=match):
            GraphedDecoder(m, max_tokens=max_tokens)


def head_norms(m, q_eps=1e-6, k_eps=1e-6, width=16, layers=None):
    for layer in m.model.layers if layers is None else layers:
        for name, eps in (("q_norm", q_eps), ("k_norm", k_eps)):
            norm = torch.nn.Module()
            norm.weight = torch.nn.Parameter(torch.ones(width))
            norm.variance_epsilon = eps
            setattr(layer.self_attn, name, norm)
    return m


@pytest.mark.parametrize("name", ["q_proj", "k_proj", "v_proj", "o_proj"])
def test_attention_biases(name):
    refused(filled(model(attention_bias=True), f"self_attn.{name}"), "bias")


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_mlp_biases(name):
    refused(filled(model(mlp_bias=True), f"mlp.{name}"), "bias")


def test_lm_head_bias():
    m = model()
    m.lm_head = torch.nn.Linear(64, 64)
    refused(m, "bias")


@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_activations(act):
    refused(model(hidden_act=act), "SiLU")


def test_sliding_windows():
    m = model()
    m.config.sliding_window = 48
    refused(m, "sliding window", max_tokens=64)
    decoder.check_model(m, 48)  # a window that no query reaches past
    m.config.use_sliding_window = False
    decoder.check_model(m, 64)
    m = model()
    m.model.layers[1].self_attn.sliding_window = 32
    refused(m, "sliding window")


def test_attention_scale():
    m = model()
    m.model.layers[0].self_attn.scaling = 1.0
    refused(m, "scale")


def test_head_norms():
    refused(head_norms(model(), 1e-6, 1e-5), "epsilon", graphed=False)
    refused(head_norms(model(), width=64), "norms", graphed=False)  # over all heads at once
    m = head_norms(model())
    m.model.layers[0].self_attn.q_norm.bias = torch.nn.Parameter(torch.ones(16))
    refused(m, "norms", graphed=False)
    with pytest.raises(ValueError, match="norms"):  # the one-sequence decoder has no per-head norms
        GraphedDecoder(head_norms(model()), max_tokens=64)


def test_models_that_are_served():
    decoder.check_model(model(), 64)
    decoder.check_model(model(attention_bias=True, mlp_bias=True), 64)  # biases of zeros change nothing
    decoder.check_model(head_norms(model(), 1e-5, 1e-5), 64, head_norms=True)
    only_q = head_norms(model())
    for layer in only_q.model.layers:
        del layer.self_attn.k_norm
    decoder.check_model(only_q, 64, head_norms=True)
