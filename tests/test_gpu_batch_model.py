"""Continuations of one prompt drawn together (model.ParallelDecoder: 8-bit or
f16 caches, shared-prefix attention, sampling) against the one-sequence decoder
fed the same tokens."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from ramvamp_b200.model import ModelConfig, Qwen3Weights

    cfg = ModelConfig(n_layers=3, hidden=256, n_heads=4, n_kv_heads=2, head_dim=128, moe=512, n_experts=8, top_k=2,
                      vocab=1000)
    return Qwen3Weights.synthetic(cfg, seed=3)


PROMPT = [5, 17, 900, 3, 44, 251, 7]


def logits_of(model, tokens):
    """The one-sequence decoder's logits after each token."""
    from ramvamp_b200.model import Decoder

    dec, out = Decoder(model, max_positions=64), []
    dec.reset()
    for t in tokens:
        dec.token.fill_(t)
        dec.step()
        out.append(dec.logits.clone())
    return torch.stack(out)


@pytest.mark.parametrize("fmt,bound", [("KV_F16", 0.01), ("KV_Q8", 0.1)])
def test_logits_follow_the_one_sequence_decoder(model, fmt, bound):
    """RMS of the difference over RMS of the logits.  With f16 caches the
    attention differs by f32 rounding alone, which may move Q8_K activations by
    one of 127 levels (about 0.002 of a layer's output: 0.01 for three).  8-bit
    rows are off by up to half of one of 127 levels (about 0.008 of a row's RMS,
    in keys and in values: at most some 0.03 a layer)."""
    import ramvamp_b200 as rv
    from ramvamp_b200.model import ParallelDecoder

    par = ParallelDecoder(model, 3, max_prompt=16, max_new=12, kv_format=getattr(rv, fmt))
    first = par.prefill(PROMPT).clone()
    rng = np.random.default_rng(1)
    tokens = rng.integers(0, model.cfg.vocab, (3, 12))
    steps = [par.step(torch.tensor(tokens[:, i], dtype=torch.int32, device="cuda")).clone() for i in range(12)]
    for b in range(3):
        want = logits_of(model, PROMPT + [int(t) for t in tokens[b]])
        assert torch.equal(want[len(PROMPT) - 1], first)
        for i in range(12):
            w = want[len(PROMPT) + i]
            assert float((steps[i][b] - w).norm() / w.norm()) < bound, (b, i)
    with pytest.raises(ValueError):
        par.step(torch.zeros(3, dtype=torch.int32, device="cuda"))
    rv.device_status(0)


def test_generate_draws_and_repeats(model):
    import ramvamp_b200 as rv
    from ramvamp_b200.model import ParallelDecoder

    par = ParallelDecoder(model, 16, max_prompt=16, max_new=8)
    tokens, logprobs = par.generate(PROMPT, 8, seed=4, temperature=0.9, top_k=200, top_p=0.95)
    again = par.generate(PROMPT, 8, seed=4, temperature=0.9, top_k=200, top_p=0.95)
    assert torch.equal(tokens, again[0]) and torch.equal(logprobs, again[1])
    other, _ = par.generate(PROMPT, 8, seed=5, temperature=0.9, top_k=200, top_p=0.95)
    assert not torch.equal(tokens, other)
    assert tokens.shape == (16, 8) and int(tokens.min()) >= 0 and int(tokens.max()) < model.cfg.vocab
    assert torch.isfinite(logprobs).all() and float(logprobs.max()) <= 0.0
    assert len({tuple(t) for t in tokens.tolist()}) > 1  # the continuations differ
    greedy, lp = par.generate(PROMPT, 3, temperature=0.0)
    assert (greedy == greedy[:1]).all() and not lp.any()
    assert int(greedy[0, 0]) == int(par.prefill(PROMPT).argmax())
    rv.device_status(0)
