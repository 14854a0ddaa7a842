"""The convolution, the selective scan and sampling together: a language model on them, and the delta rule's with a
convolution before it, decoded with filters."""
from __future__ import annotations

import pytest
import torch

DEV = "cuda"


def _model(seed=3, layers=2, vocab=96, std=0.02, **sizes):
    from ramnet_harness import ScanConfig, ScanLM
    cfg = ScanConfig(**{**dict(vocab=vocab, layers=layers, d_model=48, inner=72, states=10, groups=2, step_rank=5,
                               conv_width=3), **sizes})
    torch.manual_seed(seed)
    model = ScanLM(cfg)
    model.init_weights(std)
    return model


def _delta_model(seed=3, layers=2, vocab=96, std=0.02, **sizes):
    from ramnet_harness import DeltaConfig, DeltaLM
    cfg = DeltaConfig(**{**dict(vocab=vocab, layers=layers, d_model=64, key_heads=2, heads=4, key_dim=32, value_dim=24,
                                mlp_width=128, conv_width=4), **sizes})
    torch.manual_seed(seed)
    model = DeltaLM(cfg)
    model.init_weights(std)
    return model


def _near(a, b, rel=6e-5):
    """The same by another order of fp32 sums: a Linear map of 48 to 128 inputs is off by up to 128 * 2^-24 = 8e-6 of
    its sum of magnitudes, and about eight of them lie one behind the other here: 6e-5 of the largest value."""
    return float((a - b).abs().max()) <= rel * float(b.abs().max())


def test_shapes_and_no_cpu_fallback():
    model = _model()
    states = model.fresh_state(2, "cpu")
    assert len(states) == 2 and states[0][0].shape == (2, 72, 10) and states[0][1].shape == (2, 2, 72)
    with pytest.raises(RuntimeError):
        model(torch.zeros(2, 5, dtype=torch.long), states)  # the operators refuse host tensors
    delta = _delta_model().fresh_state(2, "cpu")
    assert delta[0][0].shape == (2, 4, 32, 24) and delta[0][1].shape == (2, 3, 2 * 64 + 96)


def test_refusals():
    from ramnet_harness import sample_generate
    with pytest.raises(ValueError):
        _model(groups=5)
    with pytest.raises(ValueError):
        sample_generate(_model(), torch.zeros(1, 1, dtype=torch.long), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("make", [_model, _delta_model])
@pytest.mark.parametrize("cut", [1, 3, 69])
def test_a_prompt_in_parts(make, cut):
    """Prefill and steps in place give what one call gives."""
    model = make().to(DEV)
    tokens = torch.randint(0, 96, (3, 70), device=DEV)
    with torch.no_grad():
        want, end = model(tokens, model.fresh_state(3, DEV))
        got, states = model(tokens[:, :cut], model.fresh_state(3, DEV))
        parts = [got]
        for t in range(cut, 70):
            got, states = model(tokens[:, t:t + 1], states, inplace=True)
            parts.append(got)
    assert _near(torch.cat(parts, 1), want)
    for a, b in zip(states, end):
        assert all(_near(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_padded_prompts():
    """Rows of unequal lengths in one call are the rows one by one."""
    from ramnet_harness import sample_generate
    model = _model().to(DEV)
    lengths = torch.tensor([40, 1, 17], device=DEV)
    tokens = torch.randint(0, 96, (3, 40), device=DEV)
    out, states = sample_generate(model, tokens, 9, lengths, temperature=0.0)
    for row, n in enumerate(lengths.tolist()):
        alone, state = sample_generate(model, tokens[row:row + 1, :n], 9, temperature=0.0)
        assert torch.equal(alone[0], out[row])
        for a, b in zip(states, state):
            assert _near(a[0][row], b[0][0]) and _near(a[1][row], b[1][0])


@pytest.mark.gpu
def test_settings_of_each_row():
    from ramnet_harness import sample_generate
    model = _model(std=0.3).to(DEV)
    tokens = torch.randint(0, 96, (4, 12), device=DEV)
    kw = dict(temperature=torch.tensor([0.0, 1.0, 1.0, 1.5], device=DEV), top_k=torch.tensor([0, 1, 5, 0], device=DEV),
              top_p=torch.tensor([1.0, 1.0, 0.9, 0.5], device=DEV), min_p=torch.tensor([0.0, 0.0, 0.1, 0.0], device=DEV))
    out, _ = sample_generate(model, tokens, 6, **kw, generator=torch.Generator(DEV).manual_seed(1))
    greedy, _ = sample_generate(model, tokens, 6, temperature=0.0)
    assert torch.equal(out[:2], greedy[:2])
    again, _ = sample_generate(model, tokens, 6, **kw, generator=torch.Generator(DEV).manual_seed(1))
    assert torch.equal(out, again)


@pytest.mark.gpu
def test_decoding_as_a_graph():
    """A step captured once, its states updated in place at every replay, is the step itself."""
    from ramnet_ops import sample_tokens
    model = _model().to(DEV).bfloat16()
    prompt = torch.randint(0, 96, (4, 20), device=DEV)
    random = torch.rand(8, 4, device=DEV)

    @torch.no_grad()
    def start():
        logits, states = model(prompt, model.fresh_state(4, DEV))
        return logits[:, -1].argmax(-1, keepdim=True), states

    @torch.no_grad()
    def step(token, states, u):
        logits, _ = model(token, states, inplace=True)
        return sample_tokens(logits[:, -1], u, temperature=0.9, top_k=20, top_p=0.95).unsqueeze(1)
    token, states = start()
    want = []
    for u in random:
        token = step(token, states, u)
        want.append(token)
    token, states = start()
    held, u = token.clone(), random[0].clone()
    spare = [tuple(t.clone() for t in s) for s in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, spare, u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.copy_(step(held, states, u))
    for n in range(8):
        u.copy_(random[n])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want[n])


@pytest.mark.gpu
@pytest.mark.parametrize("make", [_model, _delta_model])
def test_gradients(make):
    """Every parameter has a gradient, and it is that of central differences along it. A difference over a step h is
    off by c h^2 + O(h^4): over half of it by a quarter, a third of what the two differ by. A loss near log(96)
    through some 20 layers of fp32 sums is off by up to 2^-19, a slope by that over the step."""
    model = make(std=0.2).to(DEV)
    tokens = torch.randint(0, 96, (2, 60), device=DEV)

    def loss():
        logits, _ = model(tokens[:, :-1], model.fresh_state(2, DEV))
        return torch.nn.functional.cross_entropy(logits.flatten(0, 1).double(), tokens[:, 1:].flatten())
    loss().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), name
        norm = float(p.grad.norm())
        kept, step = p.detach().clone(), p.grad / max(norm, 1e-30)

        def slope(h):
            out = []
            with torch.no_grad():
                for sign in (h, -h):
                    p.copy_(kept + sign * step)
                    out.append(float(loss()))
                p.copy_(kept)
            return (out[0] - out[1]) / (2 * h)
        h = 2.0 ** -9 * max(float(kept.norm()), 1.0)
        wide, narrow = slope(h), slope(h / 2)
        assert abs(narrow - norm) <= abs(wide - narrow) + 2 * 2.0 ** -19 / h, (name, wide, narrow, norm)


@pytest.mark.gpu
def test_speculation_with_filters():
    from ramnet_harness import speculative_generate
    model, drafter = _delta_model().to(DEV), _delta_model(seed=4, layers=1).to(DEV)
    prompt = torch.randint(0, 96, (3, 20), device=DEV)
    for kw in (dict(top_k=8), dict(top_p=0.8, min_p=0.01), {}):
        gen = torch.Generator(DEV).manual_seed(2)
        out, states, _ = speculative_generate(model, drafter, prompt, 21, drafts=4, generator=gen, **kw)
        with torch.no_grad():
            logits, want = model(torch.cat((prompt, out[:, :-1]), dim=1), model.fresh_state(3, DEV))
        for a, b in zip(states, want):
            assert all(_near(x, y) for x, y in zip(a, b))
        if "top_k" in kw:  # every token is among those that the filter leaves (by the reordered sums: one more)
            best = logits[:, 19:].topk(kw["top_k"] + 1, dim=-1).indices
            assert bool((best == out.unsqueeze(-1)).any(-1).all())
    own, _, steps = speculative_generate(model, model, prompt, 16, drafts=4, top_k=1)
    with torch.no_grad():
        logits, _ = model(torch.cat((prompt, own[:, :-1]), dim=1), model.fresh_state(3, DEV))
    best = logits[:, 19:].topk(2, dim=-1)
    greedy = best.indices[..., 0] == own
    close = best.values[..., 0] - best.values[..., 1] <= 6e-5 * logits.abs().max()
    assert bool((greedy | close).all()) and steps <= 6


@pytest.mark.gpu
def test_filtered_tokens_are_distributed_as_the_models_own():
    """Frequencies of the second token over many rows of one prompt, within 5 standard deviations of what the
    filtered model says exactly."""
    from ramnet_harness import speculative_generate
    from ramnet_ops import token_probabilities
    V, rows = 12, 8192
    model, drafter = _delta_model(vocab=V, std=0.3).to(DEV), _delta_model(seed=4, layers=1, vocab=V, std=0.3).to(DEV)
    prompt = torch.randint(0, V, (1, 9), device=DEV)
    kw = dict(top_k=6, top_p=0.9)
    out, _, _ = speculative_generate(model, drafter, prompt.expand(rows, -1), 2, drafts=2, temperature=1.3,
                                     generator=torch.Generator(DEV).manual_seed(5), **kw)
    with torch.no_grad():
        logits, _ = model(torch.cat((prompt.expand(V, -1), torch.arange(V, device=DEV).view(V, 1)), dim=1),
                          model.fresh_state(V, DEV))
    p = token_probabilities(logits[:, -2:], temperature=1.3, **kw).double()
    want = (p[:, 0].diagonal().unsqueeze(-1) * p[:, 1]).sum(0)
    seen = torch.bincount(out[:, 1], minlength=V).double() / rows
    assert bool(((seen - want).abs() <= 5 * (want * (1 - want) / rows).sqrt() + 1e-6).all())
