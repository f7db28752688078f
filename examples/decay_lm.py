"""A small language model of decay attention blocks: train, prefill, generate.

Runs this package's decay attention, embedding lookup and sampler together as a
program would:

  training    embedding_lookup -> blocks (decay_attention over the sequence) ->
              the tied head's cross-entropy, stepped by DataParallelTrainer
  prompts     one chunked pass over a ragged batch (`lengths`): every row's
              state after its own last token
  generation  one token per step against the states (decay_attention_step,
              updated in place), sampled with sample_tokens; the whole step,
              sampler included, is one CUDA graph

    python examples/decay_lm.py
"""

from __future__ import annotations

import math
import sys
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn as nn
import torch.nn.functional as F

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from mamba4_b200 import decay_attention, decay_attention_step, embedding_lookup, sample_tokens  # noqa: E402
from mamba4_b200.glue import head_cross_entropy  # noqa: E402
from mamba4_b200.model import RMSNorm  # noqa: E402
from mamba4_b200.train import DataParallelTrainer, TrainSettings, synthetic_batch  # noqa: E402


@dataclass(frozen=True)
class DecayConfig:
    vocab_size: int = 4096
    d_model: int = 512
    layers: int = 4
    heads: int = 8
    kv_heads: int = 4      # key/value heads, each shared by heads / kv_heads query heads
    key_dim: int = 64
    value_dim: int = 128


class DecayMixer(nn.Module):
    """Decay attention between two projections, with a SiLU gate. Head h
    forgets at rate 2^-(4 + 6 h / heads): half lives of 11 to about 700 tokens."""

    def __init__(self, cfg: DecayConfig):
        super().__init__()
        self.cfg = cfg
        inner = cfg.heads * cfg.value_dim
        self.sizes = [inner, cfg.heads * cfg.key_dim, cfg.kv_heads * cfg.key_dim, cfg.kv_heads * cfg.value_dim]
        self.in_proj = nn.Linear(cfg.d_model, sum(self.sizes), bias=False)
        self.out_proj = nn.Linear(inner, cfg.d_model, bias=False)
        nn.init.normal_(self.in_proj.weight, 0.0, 0.02)
        nn.init.normal_(self.out_proj.weight, 0.0, 0.02 / math.sqrt(2 * cfg.layers))
        rate = 2.0 ** -(4 + 6 * torch.arange(cfg.heads) / cfg.heads)
        self.register_buffer("log_decay", torch.log1p(-rate))

    def split(self, x):
        """gate, q, k, v of x [..., d_model]: slices of one projection, read in place by the kernels."""
        cfg = self.cfg
        gate, q, k, v = self.in_proj(x).to(torch.bfloat16).split(self.sizes, dim=-1)
        lead = x.shape[:-1]
        return (gate, q.view(*lead, cfg.heads, cfg.key_dim), k.view(*lead, cfg.kv_heads, cfg.key_dim),
                v.view(*lead, cfg.kv_heads, cfg.value_dim))

    def forward(self, x, lengths=None):
        gate, q, k, v = self.split(x)
        res = decay_attention(q, k, v, self.log_decay, lengths=lengths)
        return self.out_proj(res.output.flatten(-2) * F.silu(gate)), res.state

    def step(self, x, state):
        gate, q, k, v = self.split(x)
        res = decay_attention_step(state, q, k, v, self.log_decay, inplace=True)
        return self.out_proj(res.output.flatten(-2) * F.silu(gate))


class DecayLM(nn.Module):
    def __init__(self, cfg: DecayConfig):
        super().__init__()
        self.cfg = cfg
        self.embedding = nn.Parameter(0.02 * torch.randn(cfg.vocab_size, cfg.d_model))
        self.scale = math.sqrt(cfg.d_model)
        self.norms = nn.ModuleList(RMSNorm(cfg.d_model, 1e-5) for _ in range(cfg.layers))
        self.mixers = nn.ModuleList(DecayMixer(cfg) for _ in range(cfg.layers))
        self.final_norm = RMSNorm(cfg.d_model, 1e-5)
        self.fused_loss = True  # forward(tokens, targets) returns per-token losses

    def embed(self, tokens):
        return embedding_lookup(tokens, self.embedding, scale=self.scale, dtype=torch.bfloat16)

    def hidden(self, tokens, lengths=None):
        x, states = self.embed(tokens), []
        for norm, mixer in zip(self.norms, self.mixers):
            out, state = mixer(norm(x), lengths)
            x = x + out.to(x.dtype)
            states.append(state)
        return self.final_norm(x), states

    def logits(self, x):
        return F.linear(x, self.embedding.to(x.dtype)).float()

    def forward(self, tokens, targets=None):
        x, _ = self.hidden(tokens)
        return self.logits(x) if targets is None else head_cross_entropy(x, self.embedding, targets)

    @torch.no_grad()
    def prefill(self, tokens, lengths):
        """tokens [B, T] (any id outside the vocabulary as padding), lengths [B]
        (at least 1): logits after each row's last token, and the states."""
        x, states = self.hidden(tokens, lengths)
        last = x[torch.arange(x.shape[0], device=x.device), lengths.long() - 1]
        return self.logits(last), states

    @torch.no_grad()
    def step(self, tokens, states):
        """tokens [B] -> logits [B, V]; `states` are updated in place."""
        x = self.embed(tokens)
        for norm, mixer, state in zip(self.norms, self.mixers, states):
            x = x + mixer.step(norm(x), state).to(x.dtype)
        return self.logits(self.final_norm(x))


class Generator:
    """Prompts through the chunked form once, then one CUDA graph per token:
    step, sampler and state updates."""

    def __init__(self, model: DecayLM, **sampling):
        self.model, self.sampling = model, sampling
        self.graph = None

    def _body(self):
        logits = self.model.step(self.tokens, self.states)
        got = sample_tokens(logits, self.uniform, **self.sampling)
        self.tokens.copy_(got.tokens)
        self.log_prob.copy_(got.log_prob)

    def _capture(self, batch, device):
        cfg = self.model.cfg
        self.states = [torch.zeros(batch, cfg.heads, cfg.key_dim, cfg.value_dim, device=device)
                       for _ in range(cfg.layers)]
        self.tokens = torch.zeros(batch, dtype=torch.int64, device=device)
        self.uniform, self.log_prob = torch.zeros(batch, device=device), torch.zeros(batch, device=device)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            for _ in range(2):
                self._body()
        torch.cuda.current_stream(device).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self._body()

    @torch.no_grad()
    def __call__(self, prompts, lengths, new_tokens, seed=0):
        """-> tokens [B, new_tokens], log-probabilities [B, new_tokens]."""
        batch, device = prompts.shape[0], prompts.device
        uniform = torch.rand(new_tokens, batch, generator=torch.Generator(device=device).manual_seed(seed),
                             device=device)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            if self.graph is None or self.tokens.shape[0] != batch:
                self._capture(batch, device)
            logits, states = self.model.prefill(prompts, lengths)
        for held, state in zip(self.states, states):
            held.copy_(state)
        got = sample_tokens(logits, uniform[0], **self.sampling)
        self.tokens.copy_(got.tokens)
        tokens, log_probs = [got.tokens], [got.log_prob]
        for t in range(1, new_tokens):
            self.uniform.copy_(uniform[t])
            self.graph.replay()
            tokens.append(self.tokens.clone())
            log_probs.append(self.log_prob.clone())
        return torch.stack(tokens, 1), torch.stack(log_probs, 1)


def main():
    torch.manual_seed(0)
    cfg = DecayConfig()
    model = DecayLM(cfg).cuda()
    trainer = DataParallelTrainer(model, TrainSettings(learning_rate=1e-3, warmup_steps=5, total_steps=40))
    batch = synthetic_batch(8, 512, cfg.vocab_size, seed=1, device="cuda")  # one batch, to be memorised
    for step in range(40):
        loss, _, norm = trainer.step(*batch)
        if step % 10 == 0 or step == 39:
            print(f"step {step:2d}  loss {float(loss):.3f}  gradient norm {float(norm):.3f}")
    prompts = batch[0][:4, :100].clone()
    lengths = torch.tensor([100, 17, 64, 1], dtype=torch.int32, device="cuda")
    prompts[torch.arange(100, device="cuda") >= lengths[:, None]] = -1
    generate = Generator(model, temperature=0.8, top_k=50, top_p=0.95)
    tokens, log_probs = generate(prompts, lengths, new_tokens=32)
    for row, lp in zip(tokens.tolist(), log_probs.sum(1).tolist()):
        print(f"log p {lp:8.2f}  tokens {row[:12]} ...")


if __name__ == "__main__":
    main()
