#!/usr/bin/env python3
"""Frames -> tokens -> a small language decoder, all on one GPU.

    python examples/video_decoder.py [--frames 4] [--steps 24]

A MobileNetV3-small plan (`PlanModel`) turns video frames into 7 x 7 x 576
feature maps; every cell becomes a token with a (time, height, width) position.
A decoder with random weights reads them as its prompt and then produces tokens
one by one.  Its attention runs on the language-model operators: `append` turns
keys and queries and puts keys and values into the 8-bit paged cache, `attend`
reads the cache; a decode step of all layers is captured into a CUDA graph once
and replayed.  Projections and norms are plain torch.
"""
from __future__ import annotations

import argparse
import os
import sys
import tempfile

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import infvino_b200 as ivb  # noqa: E402
from infvino_b200 import plangen  # noqa: E402

CELLS = 7  # the backbone's output is 7 x 7


def frame_tokens(frames: np.ndarray, plan_dir: str) -> torch.Tensor:
    """[frames, 3, 224, 224] float32 in 0..1 -> [frames * 49, 576] half on the GPU."""
    plan = plangen.mobilenetv3_small(plan_dir)
    n = len(frames)
    with ivb.PlanModel(plan, max_batch=n, flags=ivb.FLAG_NO_POOL) as m:
        m.setInput(ivb.f32_to_f16(frames), n)
        m.run(n)
        maps = m.readTensor("features.12.out", n).view(np.float16).reshape(n, 576, CELLS * CELLS)
    return torch.from_numpy(np.ascontiguousarray(maps.transpose(0, 2, 1))).reshape(-1, 576).cuda()


class Decoder:
    """`layers` blocks of attention (grouped queries, rotary with three axes, a
    sliding window with sinks) and a gated feed-forward part, one sequence."""

    def __init__(self, layers=4, dim=512, q_heads=8, kv_heads=2, head_dim=64, vocab=1024, window=256, sinks=4, max_len=1024, page=32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(i, o):
            return (torch.randn((i, o), generator=g, device="cuda") * i ** -0.5).half()

        self.q_heads, self.kv_heads, self.head_dim, self.window, self.sinks, self.max_len = q_heads, kv_heads, head_dim, window, sinks, max_len
        self.embed_frame, self.embed = weight(576, dim), torch.randn((vocab, dim), generator=g, device="cuda").half()
        self.blocks = [{"qkv": weight(dim, (q_heads + 2 * kv_heads) * head_dim), "o": weight(q_heads * head_dim, dim),
                        "up": weight(dim, 4 * dim), "down": weight(2 * dim, dim)} for _ in range(layers)]
        self.head = weight(dim, vocab)
        self.ops, self.side = ivb.KvOps(0), torch.cuda.Stream()  # (captures are made on one stream: each has a workspace)
        pairs = head_dim // 2
        table = torch.empty((max_len, pairs, 2), device="cuda")
        self.ops.rope_table([10000.0 ** (-i / pairs) for i in range(pairs)], table, self.stream())
        self.axis_of = [0] * (pairs // 4) + [1] * (pairs * 3 // 8) + [2] * (pairs - pairs // 4 - pairs * 3 // 8)  # time, height, width
        self.rotary = ivb.Rotary(table, self.axis_of)
        pages = -(-max_len // page)
        self.caches = []
        for _ in range(layers):
            codes = [torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.int8, device="cuda") for _ in range(2)]
            scales = [torch.zeros((pages, kv_heads, page // 16), device="cuda") for _ in range(2)]
            self.caches.append(ivb.KvCache(*codes, *scales))
        self.pages = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()[None].contiguous()

    @staticmethod
    def stream() -> int:
        return torch.cuda.current_stream().cuda_stream

    def forward(self, x, pos, offsets, starts, lens):
        """Logits of the last of x [tokens, dim], whose keys and values go to the cache at starts."""
        t, qh, kh, d = x.shape[0], self.q_heads, self.kv_heads, self.head_dim
        for block, cache in zip(self.blocks, self.caches):
            qkv = (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ block["qkv"]).view(t, qh + 2 * kh, d)
            q, k, v = qkv[:, :qh], qkv[:, qh:qh + kh], qkv[:, qh + kh:]  # strided: the operators read them in place
            turned, out = torch.empty((t, qh, d), dtype=x.dtype, device="cuda"), torch.empty((t, qh, d), dtype=x.dtype, device="cuda")
            self.ops.append(cache, k, v, offsets, starts, self.pages, rotary=self.rotary, pos=pos, q=q, q_out=turned, stream=self.stream())
            self.ops.attend(cache, turned, out, offsets, lens, self.pages, max_new=t, window=self.window, sinks=self.sinks, stream=self.stream())
            x = x + out.view(t, qh * d) @ block["o"]
            a, b = (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ block["up"]).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ block["down"]
        return torch.nn.functional.rms_norm(x[-1:], x.shape[-1:]) @ self.head

    def prompt(self, frames_tokens: torch.Tensor):
        """Runs the frames; returns the logits and what the next token's position is."""
        t = frames_tokens.shape[0]
        i = torch.arange(t, device="cuda")
        pos = torch.stack([i // (CELLS * CELLS), i // CELLS % CELLS, i % CELLS]).to(torch.int32)
        one = torch.tensor([t], dtype=torch.int32, device="cuda")
        logits = self.forward(frames_tokens @ self.embed_frame, pos, torch.tensor([0, t], dtype=torch.int32, device="cuda"),
                              torch.zeros(1, dtype=torch.int32, device="cuda"), one)
        return logits, max(t // (CELLS * CELLS), CELLS)

    def generate(self, frames_tokens: torch.Tensor, steps: int):
        """Greedy tokens and each step's logits: the prompt, then one captured step replayed."""
        length = frames_tokens.shape[0]
        if length + steps > self.max_len:
            raise ValueError(f"{length} prompt tokens and {steps} steps exceed max_len {self.max_len}")
        logits, at = self.prompt(frames_tokens)
        token = logits.argmax(-1)
        start = torch.tensor([length], dtype=torch.int32, device="cuda")
        lens, pos = start + 1, torch.full((3, 1), at, dtype=torch.int32, device="cuda")
        offsets = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        self.ops.reserve(self.side.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=self.side):
            out = self.forward(self.embed[token], pos, offsets, start, lens)
        tokens, seen = [], []
        for _ in range(steps):
            tokens.append(int(token))
            graph.replay()
            seen.append(out.clone())
            token.copy_(out.argmax(-1))
            start += 1
            lens += 1
            pos += 1
        self.ops.synchronize(self.stream())  # reports page numbers or positions that do not fit
        return tokens, torch.cat(seen)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--frames", type=int, default=4)
    ap.add_argument("--steps", type=int, default=24)
    a = ap.parse_args()
    frames = np.random.default_rng(0).random((a.frames, 3, 224, 224), dtype=np.float32)
    with tempfile.TemporaryDirectory() as plan_dir:
        x = frame_tokens(frames, plan_dir)
    tokens, _ = Decoder().generate(x, a.steps)
    print(f"{a.frames} frames, {x.shape[0]} prompt tokens ->", *tokens)


if __name__ == "__main__":
    main()
