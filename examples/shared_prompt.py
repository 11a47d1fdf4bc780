"""Several answers to one prompt through one decoder layer on the GPU.

    python examples/shared_prompt.py [--answers 8] [--prompt 500] [--steps 16]

The prompt's keys and values are computed once and lie in pages that all answers share; each
answer appends its own tokens to pages of its own. A step is what a decoder layer runs: the
quantized projections (`matmul_many`, `matmul`, `matmul_gated`), the norms and the rotation of
the heads (`qk_norm_rope`, `kv_append`) and the attention between them (`shared_attention`). As
a check every answer is computed again with the whole context in pages of its own.

The weights are random Q8_0 rows; PyTorch supplies device memory, the stream, the residual
adds and the layer norms.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import dynalm_amd as dq  # noqa: E402

WIDTH, HEADS, KV_HEADS, DIM, FFN = 1536, 12, 2, 128, 8960
PAGE, EPS, LONGEST = 16, 1e-6, 8192


def q8_rows(rng, n: int, k: int) -> np.ndarray:
    """n random Q8_0 rows of k values with a standard deviation of about 1 / sqrt(k)."""
    blocks = np.empty((n, k // 32, 34), np.uint8)
    blocks[..., :2] = np.full((n, k // 32, 1), 1.0 / (73 * k**0.5), np.float16).view(np.uint8)
    blocks[..., 2:] = rng.integers(-127, 128, (n, k // 32, 32), dtype=np.int8).view(np.uint8)
    return blocks.reshape(n, -1)


class Layer:
    def __init__(self, seed: int = 0, cache_type: torch.dtype = torch.bfloat16, pages: int = 256):
        rng = np.random.default_rng(seed)
        shapes = {"q": (HEADS * DIM, WIDTH), "k": (KV_HEADS * DIM, WIDTH), "v": (KV_HEADS * DIM, WIDTH), "o": (WIDTH, HEADS * DIM),
                  "gate": (FFN, WIDTH), "up": (FFN, WIDTH), "down": (WIDTH, FFN)}
        self.w = {name: dq.Weight.upload(dq.Q8_0, q8_rows(rng, n, k), k) for name, (n, k) in shapes.items()}
        self.q_norm, self.k_norm = (torch.from_numpy(rng.uniform(0.5, 1.5, DIM).astype(np.float32)).cuda() for _ in range(2))
        angle = torch.arange(LONGEST, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(DIM // 2, dtype=torch.float64) * 2 / DIM)
        self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        self.rope = dq.Rope(self.cos.data_ptr(), self.sin.data_ptr(), LONGEST, DIM, dq.ROPE_HALVES)
        self.k = torch.zeros((pages, PAGE, KV_HEADS, DIM), dtype=cache_type, device="cuda")
        self.v = torch.zeros_like(self.k)
        kind = dq.BF16 if cache_type == torch.bfloat16 else dq.F16
        self.cache = dq.KvCache(self.k.data_ptr(), self.v.data_ptr(), kind, KV_HEADS, DIM, PAGE, pages, *self.k.stride()[:3])
        self.workspace = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    @staticmethod
    def _rows(tokens: int, n: int) -> torch.Tensor:
        return torch.empty((tokens, n), dtype=torch.float32, device="cuda")

    @staticmethod
    def _norm(x: torch.Tensor) -> torch.Tensor:
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)

    def step(self, x: torch.Tensor, positions, slots, prefix_pages, prefix_len: int, offsets, most_new: int, pages, lens,
             most_own: int) -> torch.Tensor:
        """One pass of x [tokens, WIDTH] (sequences' new tokens one after another) through the layer."""
        t, stream = x.shape[0], torch.cuda.current_stream().cuda_stream
        q, k, v, attended, mixed = (self._rows(t, n) for n in (HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM, HEADS * DIM, WIDTH))
        h = self._norm(x)
        dq.matmul_many([(self.w[n], h, t, WIDTH, y, y.shape[1], None) for n, y in (("q", q), ("k", k), ("v", v))], stream)
        q_heads = dq.Heads(q.data_ptr(), dq.F32, HEADS, q.stride(0), DIM)
        kv_heads = [dq.Heads(y.data_ptr(), dq.F32, KV_HEADS, y.stride(0), DIM) for y in (k, v)]
        dq.qk_norm_rope(t, DIM, q_heads, q_heads, self.q_norm, eps=EPS, rope=self.rope, positions=positions, stream=stream)
        dq.kv_append(self.cache, t, *kv_heads, slots, self.k_norm, EPS, self.rope, positions, stream)
        out = dq.Heads(attended.data_ptr(), dq.F32, HEADS, attended.stride(0), DIM)
        dq.shared_attention(self.cache, q_heads, out, None, t, lens.shape[0], offsets, most_new, prefix_pages, prefix_len, pages,
                            pages.stride(0), lens, most_own, DIM**-0.5, self.workspace, self.workspace.numel(), stream)
        dq.matmul(self.w["o"], attended, t, HEADS * DIM, mixed, WIDTH, None, stream)
        x = x + mixed
        h, gated, down = self._norm(x), self._rows(t, FFN), self._rows(t, WIDTH)
        dq.matmul_gated(dq.SILU, h, t, WIDTH, self.w["gate"], self.w["up"], gated, FFN, stream=stream)
        dq.matmul(self.w["down"], gated, t, FFN, down, WIDTH, None, stream)
        return x + down


def _ints(values, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(values, dtype=dtype, device="cuda")


def prefill(layer: Layer, prompt: torch.Tensor, pages: list[int]) -> torch.Tensor:
    """The prompt's rows through the layer, its keys and values into `pages`."""
    n = prompt.shape[0]
    slots = _ints([pages[i // PAGE] * PAGE + i % PAGE for i in range(n)], torch.int64)
    return layer.step(prompt, _ints(list(range(n))), slots, None, 0, _ints([0, n]), n, _ints([pages]), _ints([n]), n)


def decode(layer: Layer, tokens: torch.Tensor, done: int, prompt_len: int, prefix_pages: list[int], own_pages: list[list[int]],
           prefix_len: int) -> torch.Tensor:
    """Step `done` of the answers: tokens [answers, WIDTH]. prefix_len 0: the prompt lies in own_pages too."""
    answers, own = tokens.shape[0], prompt_len - prefix_len + done + 1
    at = own - 1
    slots = _ints([p[at // PAGE] * PAGE + at % PAGE for p in own_pages], torch.int64)
    return layer.step(tokens, _ints([prompt_len + done] * answers), slots, _ints(prefix_pages) if prefix_len else None, prefix_len,
                      None, 1, _ints(own_pages), _ints([own] * answers), own)


def run(answers: int = 8, prompt_len: int = 500, steps: int = 16, seed: int = 0) -> float:
    """The largest difference, relative to the rows' size, between shared and separate prompts."""
    shared, own = -(-prompt_len // PAGE), -(-steps // PAGE)
    whole = -(-(prompt_len + steps) // PAGE)
    layer = Layer(seed, pages=shared + answers * own + answers * whole)
    free = torch.randperm(layer.k.shape[0], generator=torch.Generator().manual_seed(seed)).tolist()

    def take(n: int) -> list[int]:
        return [free.pop() for _ in range(n)]

    gen = torch.Generator(device="cuda").manual_seed(seed)
    prompt = torch.randn((prompt_len, WIDTH), generator=gen, device="cuda")
    first = torch.randn((answers, WIDTH), generator=gen, device="cuda")
    prefix_pages = take(shared)
    prefill(layer, prompt, prefix_pages)
    own_pages, whole_pages = [take(own) for _ in range(answers)], [take(whole) for _ in range(answers)]
    for pages in whole_pages:
        prefill(layer, prompt, pages)
    worst, x, y = 0.0, first, first
    for i in range(steps):
        x = decode(layer, x, i, prompt_len, prefix_pages, own_pages, prompt_len)
        y = decode(layer, y, i, prompt_len, prefix_pages, whole_pages, 0)
        worst = max(worst, ((x - y).norm() / y.norm()).item())
        x = y = Layer._norm(x)  # (both go on from the same rows)
    return worst


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--answers", type=int, default=8)
    p.add_argument("--prompt", type=int, default=500)
    p.add_argument("--steps", type=int, default=16)
    a = p.parse_args()
    off = run(a.answers, a.prompt, a.steps)
    print(f"{a.answers} answers of {a.steps} tokens behind a prompt of {a.prompt}: shared and separate prompts differ by {off:.2g}")
