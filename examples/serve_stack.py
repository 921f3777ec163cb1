"""A stack of decoder layers serving several requests at once: attention with a
rotary encoding over the paged 8-bit or 4-bit K/V cache next to the routed NF4
MLP, NF4 projections and LM head; random weights, greedy tokens and their log
probabilities.

    python examples/serve_stack.py [--layers 4] [--prompts 700,33,1,250] [--new 16] [--chunk 256] [--format int8]

Every step takes a token of each request that is answering and up to ``chunk``
tokens of a prompt that is not yet read; finished requests leave and give
their blocks back.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from next_step_ai_amd._runtime import nf4_code  # noqa: E402
from next_step_ai_amd.kv_cache import KvBatch, KvCache, KvStep, paged_attention  # noqa: E402
from next_step_ai_amd.lm_head import dense_linear_nf4, lm_head_forward, lm_head_nf4_meta, token_logprobs  # noqa: E402
from next_step_ai_amd.rotary import Rotary  # noqa: E402
from next_step_ai_amd.synth import make_synthetic_layer, synth_nf4, synth_normal_f16  # noqa: E402


def norm(x: torch.Tensor) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).half()


class Linear:
    """A random NF4 projection [out, in]."""

    def __init__(self, out_features: int, in_features: int, seed: int, device: torch.device):
        self.shape = (out_features, in_features)
        self.packed, self.absmax = synth_nf4(seed, out_features * in_features, 64, in_features ** -0.5, device)
        self.code = nf4_code(device)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return dense_linear_nf4(x, self.packed, self.absmax, self.code, *self.shape, 64)


class Stack:
    def __init__(self, *, layers: int, hidden: int, intermediate: int, q_heads: int, kv_heads: int, head_dim: int, vocab: int,
                 top_k: int, blocks: int, fmt: str, device: torch.device, seed: int = 1, base: float = 500000.0):
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.embed = synth_normal_f16(seed, (vocab, hidden), 1.0, device)
        head = Linear(vocab, hidden, seed + 1, device)
        self.head = lm_head_nf4_meta(head.packed, head.absmax, head.code, vocab, hidden, 64)
        self.qkv = [Linear((q_heads + 2 * kv_heads) * head_dim, hidden, seed + 10 * i + 2, device) for i in range(layers)]
        self.proj = [Linear(hidden, q_heads * head_dim, seed + 10 * i + 3, device) for i in range(layers)]
        self.mlp = [make_synthetic_layer(H=hidden, I=intermediate, R=64, seed=seed + 10 * i + 4, device=device, double_quant=True,
                                         keep_f32_absmax=False).layer(top_k) for i in range(layers)]
        self.cache = [KvCache(blocks, kv_heads, head_dim, fmt=fmt, device=device) for _ in range(layers)]
        self.rotary = Rotary(head_dim, blocks * self.cache[0].block_tokens, base=base, device=device)

    def attend(self, i: int, q: torch.Tensor, step: KvStep) -> torch.Tensor:
        return paged_attention(q, self.cache[i], step)

    def forward(self, tokens: torch.Tensor, step: KvStep) -> torch.Tensor:
        """The step's tokens [total] -> hidden states [total, hidden]."""
        n, D = tokens.shape[0], self.head_dim
        x = self.embed[tokens]
        for i in range(len(self.mlp)):
            # one product for q, k and v: the kernels read the three where they lie
            q, k, v = (t.view(n, -1, D) for t in self.qkv[i](norm(x)).split(
                [self.q_heads * D, self.kv_heads * D, self.kv_heads * D], dim=1))
            q = self.cache[i].append_rotated(k, v, step.slots, step.positions, self.rotary, q=q, q_out=q)
            x = x + self.proj[i](self.attend(i, q, step).view(n, -1))
            y = norm(x)
            x = x + (self.mlp[i].forward(y[0])[0] if n == 1 else self.mlp[i].prefill(y)[0])
        return x

    def next_tokens(self, x: torch.Tensor) -> dict[str, torch.Tensor]:
        """The most likely tokens, their log probabilities and the entropies."""
        got = token_logprobs(lm_head_forward(norm(x)[None], self.head)[0], top=1)
        return {"token": got["top_ids"][:, 0], "logprob": got["top_logprobs"][:, 0], "entropy": got["entropy"]}


def serve(stack: Stack, prompts: list[torch.Tensor], new: int, chunk: int, batch: KvBatch,
          scores: list[list[float]] | None = None) -> tuple[list[list[int]], list]:
    """Answers of ``new`` tokens to every prompt, and (tokens, ms) of the
    steps.  ``scores``: receives a list of each answer's log probabilities."""
    R, device = len(prompts), batch.device
    answers: list[list[int]] = [[] for _ in range(R)]
    if scores is not None:
        scores[:] = [[] for _ in range(R)]
    read = [0] * R  # tokens of a prompt that are in the cache
    steps = []
    while any(len(a) < new for a in answers):
        lengths, parts, left = [], [], chunk
        for r in range(R):
            if len(answers[r]) >= new:
                n = 0
            elif answers[r]:
                n = 1
                parts.append(torch.tensor(answers[r][-1:]))
            else:
                n = min(left, len(prompts[r]) - read[r])
                parts.append(prompts[r][read[r]: read[r] + n])
                read[r] += n
                left -= n
            lengths.append(n)
        total = sum(lengths)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        step = batch.plan(torch.tensor(lengths, dtype=torch.int32, device=device), total, max_new=max(lengths))
        x = stack.forward(torch.cat(parts).to(device), step)
        # requests whose prompt is read answer with their last token
        ready = [r for r in range(R) if lengths[r] and read[r] == len(prompts[r])]
        ends = torch.tensor(lengths).cumsum(0) - 1
        got = stack.next_tokens(x[ends[ready].to(device)]) if ready else None
        for r, token, score in zip(ready, got["token"].tolist(), got["logprob"].tolist()) if ready else ():
            answers[r].append(token)
            if scores is not None:
                scores[r].append(score)
        ended = torch.tensor([int(r in ready and len(answers[r]) == new) for r in range(R)], dtype=torch.int32)
        step.check()
        batch.commit(ended.to(device))
        torch.cuda.synchronize()
        steps.append((total, (time.perf_counter() - t0) * 1e3))
    return answers, steps


def main(argv: list[str] | None = None) -> tuple[list[list[int]], KvBatch]:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--intermediate", type=int, default=14336)
    p.add_argument("--heads", default="32,8", help="query and K/V heads")
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--vocab", type=int, default=32000)
    p.add_argument("--top-k", type=int, default=64, help="MLP blocks per token")
    p.add_argument("--prompts", default="700,33,1,250", help="prompt lengths")
    p.add_argument("--new", type=int, default=16, help="tokens per answer")
    p.add_argument("--chunk", type=int, default=256, help="prompt tokens per step")
    p.add_argument("--format", default="int8", choices=("int8", "e4m3", "e2m1"))
    a = p.parse_args(argv)
    device = torch.device("cuda", 0)
    q_heads, kv_heads = (int(v) for v in a.heads.split(","))
    lengths = [int(v) for v in a.prompts.split(",")]
    need = [(n + a.new + 15) // 16 for n in lengths]
    stack = Stack(layers=a.layers, hidden=a.hidden, intermediate=a.intermediate, q_heads=q_heads, kv_heads=kv_heads,
                  head_dim=a.head_dim, vocab=a.vocab, top_k=a.top_k, blocks=sum(need), fmt=a.format, device=device)
    batch = KvBatch(sum(need), 16, max_requests=len(lengths), max_blocks=max(need), q_heads=q_heads, kv_heads=kv_heads,
                    head_dim=a.head_dim, device=device)
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(a.vocab, (n,), generator=g) for n in lengths]
    serve(stack, [q[:3] for q in prompts], 2, a.chunk, batch)  # kernels loaded, workspaces allocated
    scores: list[list[float]] = []
    answers, steps = serve(stack, prompts, a.new, a.chunk, batch, scores)
    for n, ms in steps:
        print(f"step of {n:4d} tokens: {ms:7.2f} ms")
    for r, out in enumerate(answers):
        print(f"request {r} ({lengths[r]} tokens, log probability {sum(scores[r]):.2f}): {out}")
    print(f"free blocks: {int(batch.state[1])} of {sum(need)}", flush=True)
    return answers, batch


if __name__ == "__main__":
    main()
