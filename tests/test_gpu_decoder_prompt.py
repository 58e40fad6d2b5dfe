"""The logits that a prompt leaves, and what follows, for a model whose norms have weights that differ."""
import pytest
import torch

import popkv
from decoder import GraphedDecoder, PagedDecoder
from test_gpu_paged_decoder import CONFIG, Judge, ids, tiny_model

pytestmark = pytest.mark.gpu


def uneven_model(head_norms=False):
    """Norm weights spread over 0.2 to 2.2, as a trained model's are spread."""
    model = tiny_model(head_norms)
    g = torch.Generator().manual_seed(7)
    norms = [model.model.norm]
    for layer in model.model.layers:
        norms += [layer.input_layernorm, layer.post_attention_layernorm]
    for norm in norms:
        norm.weight.data.copy_(0.2 + 2.0 * torch.rand(CONFIG["hidden_size"], generator=g))
    return model


@pytest.mark.parametrize("head_norms", [False, True])
@pytest.mark.parametrize("method", ["full", "quest"])
def test_paged_decoder_prompt(head_norms, method):
    model = uneven_model(head_norms)
    judge = Judge(model)
    prompts = [ids(n, 20 + i) for i, n in enumerate((1, 37, 160))]
    # Quest with a budget for everything, so that the model's own forward is the reference.
    dec = PagedDecoder(model, popkv.RetrievalConfig(budget=256, full_layers=(0,)), batch=3, max_tokens=256, method=method)
    for b, p in enumerate(prompts):
        dec.prefill(b, p)
        judge.close(dec.logits[b], p.tolist())
        assert int(dec.token[b]) == int(dec.logits[b].argmax())
    seqs = [p.tolist() for p in prompts]
    for _ in range(2):
        for s, t in zip(seqs, dec.token.tolist()):
            s.append(t)
        dec.step()
        for b, s in enumerate(seqs):
            judge.close(dec.logits[b], s)


@pytest.mark.parametrize("method", ["full", "popkv"])
def test_graphed_decoder_prompt(method):
    model = uneven_model()
    judge = Judge(model)
    dec = GraphedDecoder(model, popkv.RetrievalConfig(budget=256, full_layers=(0,)), max_tokens=200, method=method)
    prompt = ids(150, 31)
    dec.prefill(prompt)
    judge.close(dec.logits[0], prompt.tolist())
    assert int(dec.token) == int(dec.logits.argmax())
    if method == "full":
        seq = prompt.tolist() + [int(dec.token)]
        dec.step()
        judge.close(dec.logits[0], seq)
