"""The gated delta rule and draft verification together: a language model on
the one, decoded speculatively with the other."""
from __future__ import annotations

import pytest
import torch

DEV = "cuda"


def _model(seed=3, layers=2, vocab=96, std=0.02, **sizes):
    from ramnet_harness import DeltaConfig, DeltaLM
    cfg = DeltaConfig(**{**dict(vocab=vocab, layers=layers, d_model=64, key_heads=2, heads=4, key_dim=32, value_dim=24,
                                mlp_width=128), **sizes})
    torch.manual_seed(seed)
    model = DeltaLM(cfg)
    model.init_weights(std)
    return model


def test_shapes_and_no_cpu_fallback():
    model = _model()
    states = model.fresh_state(2, "cpu")
    assert len(states) == 2 and states[0].shape == (2, 4, 32, 24)
    q, k, v, g, beta = model.blocks[0].delta.op_inputs(torch.randn(2, 5, 64))
    assert q.shape == k.shape == (2, 5, 2, 32) and v.shape == (2, 5, 4, 24) and g.shape == beta.shape == (2, 5, 4)
    assert bool((g < 0).all()) and bool((beta > 0).all()) and bool((beta < 1).all())
    with pytest.raises(RuntimeError):
        model(torch.zeros(2, 5, dtype=torch.long), states)  # the operator refuses host tensors


def test_refusals():
    from ramnet_harness import speculative_generate
    with pytest.raises(ValueError):
        _model(heads=3)
    with pytest.raises(ValueError):
        speculative_generate(_model(), _model(), torch.zeros(1, 1, dtype=torch.long), 4, drafts=0)


@pytest.mark.gpu
def test_drafts_of_the_model_itself_all_stay():
    from ramnet_harness import speculative_generate
    model = _model().to(DEV)
    prompt = torch.randint(0, 96, (5, 70), device=DEV)
    gen = torch.Generator(DEV).manual_seed(1)
    out, _, steps = speculative_generate(model, model, prompt, 16, drafts=4, generator=gen)
    assert out.shape == (5, 16) and int(out.min()) >= 0 and int(out.max()) < 96
    assert steps == 3  # the first token with the prompt, then 5 a step


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [1, 4, 40])
@pytest.mark.parametrize("T", [1, 100])
def test_states_are_those_of_the_tokens_that_stayed(T, drafts):
    """What the steps leave is what a prefill over the same tokens leaves.

    The two differ by the order of fp32 sums: a Linear map of 64 to 128 inputs
    is off by up to 128 * 2^-24 = 8e-6 of its sum of magnitudes, and about
    eight of them lie one behind the other here: 6e-5 of the largest value."""
    from ramnet_harness import speculative_generate
    model, drafter = _model().to(DEV), _model(seed=4, layers=1).to(DEV)
    prompt = torch.randint(0, 96, (3, T), device=DEV)
    gen = torch.Generator(DEV).manual_seed(2)
    out, states, _ = speculative_generate(model, drafter, prompt, 21, drafts=drafts, generator=gen)
    whole = torch.cat((prompt, out[:, :-1]), dim=1)
    with torch.no_grad():
        _, want = model(whole, model.fresh_state(3, DEV))
    for a, b in zip(states, want):
        assert float((a - b).abs().max()) <= 6e-5 * float(b.abs().max())


@pytest.mark.gpu
def test_tokens_are_distributed_as_the_models_own():
    """Frequencies of the third token over many rows of one prompt, within 5
    standard deviations of what the model says exactly."""
    from ramnet_harness import speculative_generate
    V, rows = 12, 8192
    model, drafter = _model(vocab=V, std=0.3).to(DEV), _model(seed=4, layers=1, vocab=V, std=0.3).to(DEV)
    prompt = torch.randint(0, V, (1, 9), device=DEV)
    gen = torch.Generator(DEV).manual_seed(5)
    out, _, _ = speculative_generate(model, drafter, prompt.expand(rows, -1), 3, drafts=2, generator=gen)
    pairs = torch.cartesian_prod(torch.arange(V), torch.arange(V)).to(DEV)
    with torch.no_grad():
        logits, _ = model(torch.cat((prompt.expand(V * V, -1), pairs), dim=1), model.fresh_state(V * V, DEV))
    p = torch.softmax(logits[:, -3:].double(), -1)
    at = torch.arange(V * V, device=DEV)
    want = ((p[at, 0, pairs[:, 0]] * p[at, 1, pairs[:, 1]]).unsqueeze(-1) * p[:, 2]).sum(0)
    seen = torch.bincount(out[:, 2], minlength=V).double() / rows
    assert bool(((seen - want).abs() <= 5 * (want * (1 - want) / rows).sqrt()).all())


@pytest.mark.gpu
def test_it_trains():
    model = _model().to(DEV)
    tokens = torch.randint(0, 96, (2, 130), device=DEV)
    adam = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(30):
        logits, _ = model(tokens[:, :-1], model.fresh_state(2, DEV))
        loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())
        adam.zero_grad()
        loss.backward()
        assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in model.parameters())
        adam.step()
        losses.append(float(loss))
    assert losses[-1] < 0.5 * losses[0]
