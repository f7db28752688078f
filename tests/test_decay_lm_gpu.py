"""The example model: training lowers its loss, and generation (chunked prefill,
one-token steps in a CUDA graph, sampler) agrees with the whole-sequence form."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "decay_lm", Path(__file__).resolve().parents[1] / "examples" / "decay_lm.py")


@pytest.fixture(scope="module")
def lm():
    module = importlib.util.module_from_spec(_spec)
    import sys

    sys.modules["decay_lm"] = module
    _spec.loader.exec_module(module)
    return module


def _model(lm, layers=2):
    torch.manual_seed(0)
    cfg = lm.DecayConfig(vocab_size=300, d_model=256, layers=layers, heads=4, kv_heads=2, key_dim=64, value_dim=64)
    return lm.DecayLM(cfg).cuda(), cfg


def test_training_lowers_the_loss(lm):
    model, cfg = _model(lm)
    trainer = lm.DataParallelTrainer(model, lm.TrainSettings(learning_rate=2e-3, warmup_steps=2, total_steps=30))
    batch = lm.synthetic_batch(2, 96, cfg.vocab_size, seed=1, device="cuda")
    losses = [float(trainer.step(*batch)[0]) for _ in range(30)]
    assert all(map(lambda x: x == x, losses)) and losses[-1] < losses[0] - 1.0


def test_prefill_and_steps_equal_the_whole_sequence(lm):
    """Ragged prompts, then forced tokens one by one: the logits are those of
    the whole sequence, up to the bfloat16 rounding of the activations (their
    order of rounding differs; 2 layers, logits of size about 1)."""
    model, cfg = _model(lm)
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, cfg.vocab_size, (3, 90), generator=g).cuda()
    lengths = torch.tensor([70, 1, 64], dtype=torch.int32, device="cuda")
    prompts = tokens[:, :70].clone()
    prompts[torch.arange(70, device="cuda") >= lengths[:, None]] = -1
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        logits, states = model.prefill(prompts, lengths)
        got = [logits]
        rows = torch.arange(3, device="cuda")
        for t in range(10):
            got.append(model.step(tokens[rows, lengths.long() + t], states))
        whole = model(tokens)
    for t, logits in enumerate(got):
        want = whole[rows, lengths.long() - 1 + t]
        assert float((logits - want).norm()) <= 0.03 * float(want.norm()), t


def test_the_graph_generates_what_eager_steps_do(lm):
    model, cfg = _model(lm)
    settings = dict(temperature=0.9, top_k=40, top_p=0.9)
    prompts = torch.randint(0, cfg.vocab_size, (3, 40), generator=torch.Generator().manual_seed(3)).cuda()
    lengths = torch.tensor([40, 40, 12], dtype=torch.int32, device="cuda")
    tokens, log_probs = lm.Generator(model, **settings)(prompts, lengths, 12, seed=5)
    uniform = torch.rand(12, 3, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits, states = model.prefill(prompts, lengths)
        for t in range(12):
            got = lm.sample_tokens(logits, uniform[t], **settings)
            assert torch.equal(got.tokens, tokens[:, t]) and torch.equal(got.log_prob, log_probs[:, t])
            logits = model.step(got.tokens, states)
