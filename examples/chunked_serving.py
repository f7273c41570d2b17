"""Serving loop over a paged, quantised KV cache: prompts in pieces, mixed with decodes.

    python examples/chunked_serving.py [--dtype bf16] [--no-quant] [--budget 512]

A random-init stack of attention layers serves a few prompts of different lengths.  Every step packs up to ``--budget``
prompt tokens with one token of each sequence that already decodes, and runs per layer

    kvcache_append_varlen           the step's K and V into their pages, e4m3 with a scale per token and KV head
    flash_attn_varlen_with_kvcache  the step's queries over everything cached

with one ``kvcache_chunk_plan`` per step.  At the end the cached tokens of one sequence are read back
(``kvcache_gather_varlen``) and attended with ``flash_attn_varlen_func``; the outputs of the last layer must agree with
what the loop produced for them in pieces.
"""

from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

import mxflashattn_b200 as fa


class Cache:
    """Pages of every layer and one block table; pages are taken from a free list as sequences grow."""

    def __init__(self, layers, pages, page_size, kv_heads, dim, dtype, quant, batch, max_len, device):
        store = torch.float8_e4m3fn if quant else dtype
        shape = (layers, pages, page_size, kv_heads, dim)
        self.k, self.v = torch.zeros(shape, device=device).to(store), torch.zeros(shape, device=device).to(store)
        self.ks = self.vs = [None] * layers
        if quant:
            unit = torch.full((layers, pages, kv_heads, page_size), 127, device=device, dtype=torch.uint8)
            self.ks, self.vs = unit.view(torch.float8_e8m0fnu), unit.clone().view(torch.float8_e8m0fnu)
        self.page_size = page_size
        self.free = list(torch.randperm(pages).tolist())
        self.table = torch.full((batch, -(-max_len // page_size)), -1, dtype=torch.int32)
        self.used = [0] * batch

    def grow(self, seq, length):
        """Pages for ``length`` tokens of ``seq`` (host side)."""
        while self.used[seq] * self.page_size < length:
            self.table[seq, self.used[seq]] = self.free.pop()
            self.used[seq] += 1


def serve(*, prompts=(700, 37, 1300, 5), decode=8, budget=512, layers=2, q_heads=16, kv_heads=4, dim=128, page_size=16,
          dtype=torch.bfloat16, quant=True, seed=0, device="cuda"):
    """Serve the prompts; (steps, tokens, seconds, largest difference to the whole-sequence attention)."""
    torch.manual_seed(seed)
    batch, hidden = len(prompts), q_heads * dim
    total = [n + decode for n in prompts]
    heads = q_heads + 2 * kv_heads
    w_qkv = [torch.randn(hidden, heads * dim, device=device, dtype=dtype) / hidden ** 0.5 for _ in range(layers)]
    w_out = [torch.randn(hidden, hidden, device=device, dtype=dtype) / hidden ** 0.5 for _ in range(layers)]
    # the "token embeddings" of the whole run: what a sampler would choose is not the point here
    inputs = [torch.randn(n, hidden, device=device, dtype=dtype) for n in total]
    pages = sum(-(-n // page_size) for n in total) + 2
    cache = Cache(layers, pages, page_size, kv_heads, dim, dtype, quant, batch, max(total), device)
    done = [0] * batch
    steps, last_q, last_out = 0, [], []
    torch.cuda.synchronize()
    began = time.perf_counter()
    while any(d < t for d, t in zip(done, total)):
        # this step's tokens: one of each decoding sequence, prompt pieces for the rest of the budget
        left, take = budget, []
        for b in range(batch):
            want = 1 if done[b] >= prompts[b] else prompts[b] - done[b]
            n = 0 if done[b] == total[b] else min(want, max(left, 1) if want == 1 else left)
            take.append(n)
            left -= n
        lengths = [d + n for d, n in zip(done, take)]
        for b in range(batch):
            cache.grow(b, lengths[b])
        offsets = [0]
        for n in take:
            offsets.append(offsets[-1] + n)
        cu = torch.tensor(offsets, dtype=torch.int32).to(device, non_blocking=True)
        lens = torch.tensor(lengths, dtype=torch.int32).to(device, non_blocking=True)
        table = cache.table.to(device, non_blocking=True)
        tokens, longest = offsets[-1], max(take)
        plan = fa.kvcache_chunk_plan(cu, lens, tokens, longest, q_heads=q_heads, kv_heads=kv_heads, causal=True)
        x = torch.cat([inputs[b][done[b]:lengths[b]] for b in range(batch)])
        for i in range(layers):
            qkv = (x @ w_qkv[i]).view(tokens, heads, dim)
            q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv_heads], qkv[:, q_heads + kv_heads:]
            fa.kvcache_append_varlen(k, v, cache.k[i], cache.v[i], cu, lens, table, k_scales=cache.ks[i],
                                     v_scales=cache.vs[i])
            o = fa.flash_attn_varlen_with_kvcache(q, cache.k[i], cache.v[i], cu, lens, table, longest, max(lengths),
                                                  causal=True, k_scales=cache.ks[i], v_scales=cache.vs[i], plan=plan)
            if i == layers - 1:
                last_q.append((offsets, q.clone()))
                last_out.append(o)
            x = x + o.reshape(tokens, hidden) @ w_out[i]
        done, steps = lengths, steps + 1
    torch.cuda.synchronize()
    seconds = time.perf_counter() - began

    # the longest sequence's last layer again, in one piece, over the values read back from the cache
    seq = max(range(batch), key=lambda b: total[b])
    n = total[seq]
    cu = torch.tensor([0, n], dtype=torch.int32, device=device)
    lens = torch.tensor([n], dtype=torch.int32, device=device)
    table = cache.table[seq:seq + 1].to(device)
    k, v = fa.kvcache_gather_varlen(cache.k[-1], cache.v[-1], cu, lens, table, n, k_scales=cache.ks[-1],
                                    v_scales=cache.vs[-1], dtype=dtype)
    q = torch.cat([t[o[seq]:o[seq + 1]] for o, t in last_q])
    pieces = torch.cat([t[o[0][seq]:o[0][seq + 1]] for o, t in zip(last_q, last_out)])
    whole = fa.flash_attn_varlen_func(q, k, v, cu, cu, n, n, causal=True)
    return steps, sum(total), seconds, float((whole.float() - pieces.float()).abs().max())


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dtype", choices=("bf16", "fp16"), default="bf16")
    ap.add_argument("--no-quant", action="store_true", help="keep the cache in 16 bits")
    ap.add_argument("--budget", type=int, default=512, help="prompt tokens a step may take")
    a = ap.parse_args()
    steps, tokens, seconds, diff = serve(dtype=torch.bfloat16 if a.dtype == "bf16" else torch.float16,
                                         quant=not a.no_quant, budget=a.budget)
    print(f"{steps} steps, {tokens} tokens in {seconds * 1e3:.1f} ms; pieces against the whole sequence: "
          f"largest difference {diff:.2e}")


if __name__ == "__main__":
    main()
