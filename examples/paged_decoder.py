"""Serving a small decoder over a paged key/value cache: residual + RMS norm, the quantised cache write, attention
over the cache, and the int2 LM head with the sampler, as one loop.

    python examples/paged_decoder.py --format e4m3 --prompts 700 33 256 --new 32

The weights are random (there is no checkpoint here), so the text means nothing: the example shows how the
operators are called together.  Prompts enter in chunks, several sequences to a call; then every sequence gets one token a
step.  The products between the operators are plain torch matmuls.
"""
from __future__ import annotations

import argparse
import importlib
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
gs = importlib.import_module("gemma-webgpu-engine_b200")


class PagedDecoder:
    """Pre-norm decoder layers over one cache each; every second layer sees a window of the context."""

    def __init__(self, sampler, *, layers=4, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, inner=4096, vocab=8192,
                 format="bf16", pages=256, page_size=16, window=512, sinks=4, seed=0):
        dev = torch.device("cuda", sampler.device)
        gen = torch.Generator(device=dev).manual_seed(seed)

        def mat(rows, cols):
            return (torch.randn((rows, cols), generator=gen, device=dev) * rows ** -0.5).to(torch.bfloat16)

        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.embed = torch.randn((vocab, hidden), generator=gen, device=dev)
        self.layers = []
        for i in range(layers):
            norms = [1.0 + 0.1 * torch.randn(hidden, generator=gen, device=dev) for _ in range(2)]
            self.layers.append(dict(
                norm1=gs.GpuRmsNorm(sampler, norms[0]), norm2=gs.GpuRmsNorm(sampler, norms[1]), weights=norms,
                qkv=mat(hidden, (q_heads + 2 * kv_heads) * head_dim), out=mat(q_heads * head_dim, hidden),
                up=mat(hidden, 2 * inner), down=mat(inner, hidden),
                cache=gs.GpuKvCache.allocate(sampler, pages, kv_heads, page_size, head_dim, format),
                window=window if i % 2 else 0, sinks=sinks if i % 2 else 0))
        # the last norm writes the int8 grid that the LM head reads
        self.grid = 1.0 / 32
        self.norm = gs.GpuRmsNorm(sampler, hidden=hidden, out="srq", srq_scale=self.grid)
        codes = np.random.default_rng(seed).integers(0, 1 << 32, size=(vocab, hidden // 16), dtype=np.uint64)
        self.head = gs.GpuLmHead(sampler, codes.astype(np.uint32), np.full(vocab, hidden ** -0.5, np.float32), self.grid)

    def forward(self, tokens, slots, q_start, kv_len, table, max_q, max_kv):
        """The residual stream's last sum as (h, branch), both [tokens, hidden] float32."""
        h, branch = self.embed[tokens], None
        n, qh, kh, d = tokens.shape[0], self.q_heads, self.kv_heads, self.head_dim
        for layer in self.layers:
            r = layer["norm1"](h, branch)
            h = h if branch is None else r.residual
            qkv = (r.out @ layer["qkv"]).view(n, qh + 2 * kh, d)
            q, k, v = qkv[:, :qh], qkv[:, qh:qh + kh], qkv[:, qh + kh:]  # (read where they lie)
            cache = layer["cache"]
            cache.write(k, v, slots)
            a, _ = cache.attend(q, q_start, kv_len, table, max_q=max_q, max_kv=max_kv, scale=d ** -0.5,
                                window=layer["window"], sinks=layer["sinks"])
            r = layer["norm2"]((a.view(n, qh * d) @ layer["out"]).float(), h)
            h = r.residual
            gate, up = (r.out @ layer["up"]).chunk(2, dim=1)
            branch = ((torch.nn.functional.silu(gate) * up) @ layer["down"]).float()
        return h, branch

    def sample(self, h, branch, params, rng_state=None):
        """One token id per row of the stream."""
        r = self.norm(h, branch)
        return self.head.sample(r.out, r.row_sum, params, rng_state=rng_state).ids


def generate(model, prompts, new_tokens, params, chunk=512, rng_state=None):
    """``new_tokens`` ids for each prompt (lists of ids): the prompts in chunks, then one token a step."""
    dev, page = model.embed.device, model.page_size
    seqs = len(prompts)
    cols = max(-(-(len(p) + new_tokens) // page) for p in prompts)
    table = torch.full((seqs, cols), -1, dtype=torch.int32)
    used = 0
    for b, p in enumerate(prompts):
        need = -(-(len(p) + new_tokens) // page)
        table[b, :need] = torch.arange(used, used + need, dtype=torch.int32)
        used += need
    if used > model.layers[0]["cache"].pages:
        raise ValueError(f"the prompts need {used} pages")
    table_dev = table.to(dev)

    def call(rows):  # rows: (sequence, first position, ids)
        ids = [t for _, _, x in rows for t in x]
        slots = [int(table[b, p // page]) * page + p % page for b, p0, x in rows for p in range(p0, p0 + len(x))]
        starts = np.cumsum([0] + [len(x) for _, _, x in rows]).tolist()
        lens = [p0 + len(x) for _, p0, x in rows]
        i32 = dict(dtype=torch.int32, device=dev)
        h, branch = model.forward(torch.tensor(ids, device=dev), torch.tensor(slots, **i32), torch.tensor(starts, **i32),
                                  torch.tensor(lens, **i32), table_dev[[b for b, _, _ in rows]],
                                  max(len(x) for _, _, x in rows), max(lens))
        last = torch.tensor(starts[1:], device=dev) - 1
        return h[last], branch[last]

    stream = [None] * seqs
    for p0 in range(0, max(len(p) for p in prompts), chunk):
        rows = [(b, p0, p[p0:p0 + chunk]) for b, p in enumerate(prompts) if p0 < len(p)]
        h, branch = call(rows)
        for i, (b, _, _) in enumerate(rows):
            stream[b] = h[i], branch[i]
    h, branch = (torch.stack(x) for x in zip(*stream))
    # decode: the tokens stay on the device, and so do the positions
    at = torch.tensor([len(p) for p in prompts], device=dev)
    longest = max(len(p) for p in prompts)
    row = torch.arange(seqs, device=dev)
    out = []
    for i in range(new_tokens):
        token = model.sample(h, branch, params, rng_state).long()
        out.append(token)
        if i + 1 == new_tokens:
            break
        slots = (table_dev[row, at // page] * page + at % page).to(torch.int32)
        at = at + 1
        h, branch = model.forward(token, slots, None, at.to(torch.int32), table_dev, 1, longest + i + 1)
    for layer in model.layers:
        layer["cache"].check()
    return torch.stack(out, dim=1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--format", choices=["bf16", "e4m3", "int8"], default="e4m3")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompts", type=int, nargs="+", default=[700, 33, 256], help="prompt lengths")
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--chunk", type=int, default=512)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    sampler = gs.GpuSampler(0)
    pages = sum(-(-(n + a.new) // 16) for n in a.prompts)
    model = PagedDecoder(sampler, layers=a.layers, format=a.format, pages=pages)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, model.embed.shape[0], n).tolist() for n in a.prompts]
    params = gs.params_from_config(dict(gs.DEFAULT_DECODING_CONFIG, temperature=a.temperature, topK=40))
    state = None
    if a.temperature:
        state = torch.arange(1, len(prompts) + 1, dtype=torch.float64, device="cuda")
    generate(model, prompts, 2, params, a.chunk, state)
    torch.cuda.synchronize()
    t = time.perf_counter()
    ids = generate(model, prompts, a.new, params, a.chunk, state)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t) * 1e3
    for p, row in zip(prompts, ids.tolist()):
        print(f"prompt of {len(p):5d}: {row[:12]}{' ...' if len(row) > 12 else ''}")
    print(f"{sum(map(len, prompts))} prompt tokens and {ids.numel()} new ones in {ms:.1f} ms ({a.format} cache)")


if __name__ == "__main__":
    main()
