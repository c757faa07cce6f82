"""Streaming requests through a small decoder over the paged KV cache.

Several requests' prompts arrive in pieces while other requests already decode: every step takes one ragged batch
(a prompt chunk here, a single token there), appends its keys and values to the cache with the position rotation
on the way (Context.op_kv_append) and attends over everything cached so far (Context.op_chunk_attention). Projections
are plain torch products; weights are random. The hidden states are checked against the same requests fed whole.

    python examples/chunked_decoder.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "gsv.cpp_b200"))
import gsvcu  # noqa: E402

LAYERS, WIDTH, HEADS, KV_HEADS, DIM, PAGE = 2, 512, 8, 2, 64, 64


class Decoder:
    """LAYERS blocks of normalisation, grouped-query attention and a residual connection, in BF16."""

    def __init__(self, ctx, pages, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[0] ** -0.5).bfloat16()  # noqa: E731
        self.ctx = ctx
        self.qkv = [rand(WIDTH, (HEADS + 2 * KV_HEADS) * DIM) for _ in range(LAYERS)]
        self.out = [rand(HEADS * DIM, WIDTH) for _ in range(LAYERS)]
        self.cache = gsvcu.PagedKV(torch.zeros(pages, LAYERS, 2, KV_HEADS, PAGE, DIM, dtype=torch.bfloat16, device="cuda"))
        angle = torch.arange(4096, dtype=torch.float64, device="cuda")[:, None] * \
            10000.0 ** (-torch.arange(DIM // 2, dtype=torch.float64, device="cuda") * 2 / DIM)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def step(self, x, batch):
        """x [rows][WIDTH]: the new tokens' inputs, packed by sequence."""
        n = x.shape[0]
        q = torch.empty(n, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        a = torch.empty_like(q)
        for layer in range(LAYERS):
            y = torch.nn.functional.layer_norm(x, (WIDTH,)) @ self.qkv[layer]
            y = y.view(n, HEADS + 2 * KV_HEADS, DIM)
            self.ctx.op_kv_append(self.cache, batch, layer, y[:, :HEADS], y[:, HEADS:HEADS + KV_HEADS],
                                  y[:, HEADS + KV_HEADS:], q, cos=self.cos, sin=self.sin)
            self.ctx.op_chunk_attention(self.cache, batch, layer, q, a)
            x = x + a.view(n, HEADS * DIM) @ self.out[layer]
        return x


def batch_of(chunks, lengths, table):
    """One step's batch: chunk sizes and total lengths of every sequence (host lists), its page table."""
    starts = [0]
    for n in chunks:
        starts.append(starts[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return gsvcu.ChunkBatch(i32(starts), i32(lengths), table, starts[-1], max(chunks), max(lengths))


def main(lengths=(300, 77, 1024, 40), pieces=(64, 200, 128, 1)):
    """Feeds request i in chunks of pieces[i] tokens; returns the largest relative difference from feeding it whole."""
    ctx = gsvcu.Context(0)
    pages = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(pages), device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), max(pages), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream_handle())):   # the operators run on the context's stream
        x = [torch.randn(n, WIDTH, device="cuda").bfloat16() for n in lengths]
        whole = Decoder(ctx, sum(pages)).step(torch.cat(x), batch_of(lengths, lengths, table)).split(list(lengths))
        decoder = Decoder(ctx, sum(pages))
        done, steps = [0] * len(lengths), 0
        got = [[] for _ in lengths]
        while any(d < n for d, n in zip(done, lengths)):
            chunks = [min(p, n - d) for p, n, d in zip(pieces, lengths, done)]
            rows = torch.cat([s[d:d + c] for s, d, c in zip(x, done, chunks)])
            done = [d + c for d, c in zip(done, chunks)]
            y = decoder.step(rows, batch_of(chunks, done, table)).split(chunks)
            for g, part in zip(got, y):
                g.append(part)
            steps += 1
        worst = max(float((torch.cat(g).float() - w.float()).norm() / w.float().norm()) for g, w in zip(got, whole))
    ctx.sync()
    print(f"{len(lengths)} requests of {list(lengths)} tokens in {steps} steps, {ctx.kernel_launches()} operator kernels: "
          f"relative difference from whole prompts {worst:.1e}")
    ctx.close()
    return worst


if __name__ == "__main__":
    main()
