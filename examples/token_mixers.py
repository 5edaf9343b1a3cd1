"""The token mixers of a hybrid layer pair, as a serving loop would call them.

A prompt batch and a few single-token steps go through (1) the grouped INT8 projection split into q, k, v and z and the
gated delta rule behind it, and (2) the paged INT8 cache and the attention over it.  Weights are random; run it on a B200:

    python examples/token_mixers.py
"""
from __future__ import annotations

import os
import sys
from types import SimpleNamespace

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from reax_engine_runtime_v3_b200 import gated_delta  # noqa: E402
from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache  # noqa: E402
from reax_engine_runtime_v3_b200.runtime.split_gated_projection import project_split  # noqa: E402

WIDTH = 2560                                # activations
K_HEADS, V_HEADS, D = 16, 32, 128           # gated delta rule: 2 * 16 * 128 + 32 * 128 = 8192 rows of q, k, v, 4096 of z
KV_HEADS, GROUP, DIM, PAGE = 4, 4, 256, 64  # attention


def projection_bank(device, gen):
    """A grouped INT8 bank of 12288 rows in one group, as the split z branch takes it (random weights)."""
    rows = (2 * K_HEADS + V_HEADS) * D + V_HEADS * D
    return SimpleNamespace(
        width=WIDTH, parts=1, group=WIDTH, hp=0, low_columns=torch.arange(WIDTH, dtype=torch.int32, device=device),
        high_columns=torch.zeros(0, dtype=torch.int32, device=device),
        low_weight=torch.randint(-127, 128, (rows, WIDTH), generator=gen, device=device, dtype=torch.int32).to(torch.int8),
        high_weight=torch.zeros(rows, 0, dtype=torch.bfloat16, device=device),
        smoothing=torch.ones(WIDTH, device=device), centers=torch.zeros(WIDTH, device=device),
        scales=torch.full((1, rows), 2e-4, device=device), bias=torch.zeros(1, rows, device=device))


def gates(rows, gen, device):
    """log decays and betas, as the control projection's activations give them."""
    g = -torch.rand(rows, V_HEADS, generator=gen, device=device)
    return g, torch.sigmoid(torch.randn(rows, V_HEADS, generator=gen, device=device))


def split_heads(qkv):
    n, kd = len(qkv), K_HEADS * D
    return qkv[:, :kd].view(n, K_HEADS, D), qkv[:, kd:2 * kd].view(n, K_HEADS, D), qkv[:, 2 * kd:].view(n, V_HEADS, D)


def main(lengths=(70, 1, 200), steps=4, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(0)
    batch, total = len(lengths), sum(lengths)
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=device)
    bank = projection_bank(device, gen)
    state = torch.zeros(batch, V_HEADS, D, D, device=device)
    most = max(lengths) + steps
    cache = Int8Cache.empty(batch * -(-most // PAGE), KV_HEADS, DIM, PAGE, device)
    tables = torch.arange(cache.pages, dtype=torch.int32, device=device).view(batch, -1)
    cached = torch.zeros(batch, dtype=torch.int32, device=device)

    def layer_pair(x, prompt):
        rows = len(x)
        qkv, _ = project_split(x, bank, 8192, "slice_m128n128")
        q, k, v = split_heads(qkv)
        g, beta = gates(rows, gen, device)
        if prompt:
            mixed = gated_delta.prefill(q, k, v, g, beta, state, cu_seqlens=cu, carry=False)
        else:
            mixed = gated_delta.decode(q, k, v, g, beta, state)
        new = [torch.randn(rows, KV_HEADS, DIM, generator=gen, device=device).bfloat16() for _ in "kv"]
        queries = torch.randn(rows, KV_HEADS * GROUP, DIM, generator=gen, device=device).bfloat16()
        spans = dict(cu_seqlens=cu) if prompt else {}
        cache.append(*new, tables, cached, **spans)
        cached.add_((cu[1:] - cu[:-1]) if prompt else 1)
        seen = cache.attend(queries, tables, cached, max_rows=max(lengths) if prompt else 1, **spans)
        return mixed, seen

    outs = [layer_pair(torch.randn(total, WIDTH, generator=gen, device=device).bfloat16(), True)]
    for _ in range(steps):
        outs.append(layer_pair(torch.randn(batch, WIDTH, generator=gen, device=device).bfloat16(), False))
    return outs, state, cached


if __name__ == "__main__":
    outs, state, cached = main()
    torch.cuda.synchronize()
    for mixed, seen in outs:
        print(f"{len(mixed):4d} rows: mixed {tuple(mixed.shape)} rms {mixed.float().square().mean().sqrt():.4f}, "
              f"attended {tuple(seen.shape)} rms {seen.float().square().mean().sqrt():.4f}")
    print("cached rows", cached.tolist(), "state rms", f"{state.square().mean().sqrt():.4f}")
