"""Qwen3-MoE decoder layers on the GPU: prompts in, then tokens one by one.

Per layer (src/qwen3moe/model.zig:212-232 around src/qwen3moe/attn.zig):
    n = rms(h);  q, k, v = FP8 projections of n
    q, k, v normed per head, rotated, k and v written to the paged cache     attn.append
    a = attention over the prompts, or of the new token over the cache        attn.prefill / attn.DecodePlan
    h += FP8 projection of a
    h += MoE(rms(h))                                                          moe.stack_forward
on synthetic weights of the model's layer shape.  Embedding and output head are left out: hidden
states go in and come out.

    python examples/decoder.py --layers 2 --prompts 300,77,1024 --tokens 32 [--cache e4m3]
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from colizig_b200 import _abi, attn, gpu, moe, synth  # noqa: E402

EPS = 1e-6


def matmul_fp8(x, w, scales):
    """x f32 [T, I] times a block-FP8 weight [O, I], on the current stream."""
    y = torch.empty((x.shape[0], w.shape[0]), dtype=torch.float32, device=x.device)
    if x.shape[0]:
        _abi.check("colizig_cuda_matmul_fp8_device", _abi.load().colizig_cuda_matmul_fp8_device(
            y.data_ptr(), x.data_ptr(), w.data_ptr(), scales.data_ptr(), x.shape[0], w.shape[1], w.shape[0],
            torch.cuda.current_stream().cuda_stream))
    return y


def rms(h, w):
    return h * torch.rsqrt(h.double().square().mean(-1, keepdim=True) + EPS).float() * w


class Layer:
    """One decoder layer's weights and its part of the cache."""

    def __init__(self, index, dims, q_heads, kv_heads, head_dim, pages, page_size, cache_dtype, max_batch):
        g = torch.Generator(device="cuda").manual_seed(index)
        self.index, self.hq, self.hk, self.d = index, q_heads, kv_heads, head_dim
        H = dims.hidden

        def fp8(O, I):
            w = (torch.randn((O, I), generator=g, device="cuda") * 0.5).to(torch.float8_e4m3fn).view(torch.uint8)
            s = torch.rand((synth.nblk(O), synth.nblk(I)), generator=g, device="cuda") * 0.02 + 0.04
            return w, s

        # q, k and v stacked: one product per token batch
        self.qkv = fp8((q_heads + 2 * kv_heads) * head_dim, H)
        self.o = fp8(H, q_heads * head_dim)
        self.in_norm = torch.ones(H, device="cuda")
        self.post_norm = torch.ones((1, H), device="cuda")
        self.q_norm = 1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")
        self.k_norm = 1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")
        scale = torch.full((kv_heads,), 1 / 32, device="cuda") if cache_dtype == attn.E4M3 else None
        self.cache = attn.KvCache.empty(pages, kv_heads, page_size, head_dim, cache_dtype, k_scale=scale, v_scale=scale)
        self.plan = attn.DecodePlan(self.cache, q_heads, max_batch)
        self.moe = moe.Layer.from_weights(index, dims, synth.make_layer(dims, seed=100 + index, device="cuda"))

    def attention(self, h, positions, slots, rope, cu=None, table=None, lens=None):
        """h += attention sublayer; whole prompts (cu) or one token per sequence (table, lens)."""
        hq, hk, d = self.hq, self.hk, self.d
        qkv = matmul_fp8(rms(h, self.in_norm), *self.qkv)
        q = qkv[:, : hq * d].unflatten(1, (hq, d))
        k = qkv[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
        v = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
        q, k, v = attn.append(self.cache, q, k, v, positions, slots, rope, self.q_norm, self.k_norm, EPS,
                              packed=cu is not None)
        a = attn.prefill(q, k, v, cu) if cu is not None else self.plan.run(q, table, lens)
        return h.add_(matmul_fp8(a.float().flatten(1), *self.o))

    def forward(self, h, *args, **kw):
        self.attention(h, *args, **kw)
        return moe.stack_forward(self.index, 1, h, self.post_norm, EPS)


class Decoder:
    """Layers, and the page table their caches share."""

    def __init__(self, layers=2, dims=synth.CONFIGS["c2"], q_heads=32, kv_heads=4, head_dim=128, page_size=64,
                 max_len=2048, max_batch=8, cache_dtype=torch.bfloat16):
        gpu.init(torch.cuda.current_device())
        self.page_size, self.width = page_size, -(-max_len // page_size)
        pages = self.width * max_batch
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).tolist()
        self.table = torch.zeros((max_batch, self.width), dtype=torch.int32)
        self.lens = []
        self.rope = attn.rope_table(max_len, head_dim)
        self.layers = [Layer(i, dims, q_heads, kv_heads, head_dim, pages, page_size, cache_dtype, max_batch)
                       for i in range(layers)]

    def _grow(self, b, n):
        """Room for n tokens of sequence b."""
        have = -(-self.lens[b] // self.page_size) if b < len(self.lens) else 0
        for i in range(have, -(-n // self.page_size)):
            self.table[b, i] = self.free.pop()

    def prompt(self, hidden):
        """hidden: one f32 [n, H] per sequence.  Returns their states, one after the other."""
        pos = []
        for b, x in enumerate(hidden):
            self._grow(b, x.shape[0])
            pos.append(torch.arange(x.shape[0]))
        self.lens = [x.shape[0] for x in hidden]
        seq = torch.repeat_interleave(torch.arange(len(hidden)), torch.tensor(self.lens))
        pos = torch.cat(pos)
        slots = self.table[seq, pos // self.page_size].long() * self.page_size + pos % self.page_size
        cu = torch.tensor([0] + self.lens).cumsum(0).int().cuda()
        h = torch.cat(hidden).cuda()
        pos, slots = pos.int().cuda(), slots.cuda()
        for layer in self.layers:
            layer.forward(h, pos, slots, self.rope, cu=cu)
        return h

    def step(self, h):
        """One new token per sequence, f32 [B, H]; returns its states."""
        B = len(self.lens)
        pos = torch.tensor(self.lens)
        for b in range(B):
            self._grow(b, self.lens[b] + 1)
        self.lens = [n + 1 for n in self.lens]
        slots = (self.table[torch.arange(B), pos // self.page_size].long() * self.page_size + pos % self.page_size).cuda()
        table, lens = self.table[:B].cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        h = h.clone()
        pos = pos.int().cuda()
        for layer in self.layers:
            layer.forward(h, pos, slots, self.rope, table=table, lens=lens)
        return h


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prompts", default="300,77,1024")
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--cache", choices=("bf16", "e4m3"), default="bf16")
    a = ap.parse_args()
    lens = [int(n) for n in a.prompts.split(",")]
    dec = Decoder(a.layers, max_len=max(lens) + a.tokens, max_batch=len(lens),
                  cache_dtype=torch.bfloat16 if a.cache == "bf16" else attn.E4M3)
    H = synth.CONFIGS["c2"].hidden
    g = torch.Generator().manual_seed(1)
    torch.cuda.synchronize()
    t = time.perf_counter()
    h = dec.prompt([torch.randn((n, H), generator=g) for n in lens])
    torch.cuda.synchronize()
    print(f"prompts {lens}: {a.layers} layers in {(time.perf_counter() - t) * 1e3:.2f} ms")
    last = h[torch.tensor(lens).cumsum(0) - 1]
    t = time.perf_counter()
    for _ in range(a.tokens):
        last = dec.step(rms(last, torch.ones(H, device="cuda")))
    torch.cuda.synchronize()
    attn.check()
    moe.check()
    print(f"{a.tokens} tokens for {len(lens)} sequences: {(time.perf_counter() - t) / a.tokens * 1e3:.3f} ms a token, "
          f"|h| {float(last.norm()):.3f}")


if __name__ == "__main__":
    main()
