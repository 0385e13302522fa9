"""One attention layer over long contexts: prompts in chunks, then single tokens from a HIP graph.

    python examples/long_context.py --sequences 8 --context 32768 --chosen 32

Random weights, synthetic tokens. Every token attends to the ``--chosen`` blocks of 64 keys whose
bounds score highest with its query (the first and the last two always among them); the last step is
repeated over all blocks, and the weight that the chosen ones hold of it is printed.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from retrieve_amd.kv import PagedCache, block_attention, rotary_table  # noqa: E402

PAGE = 64


class Layer(torch.nn.Module):
    """Projections around the cache's three calls."""

    def __init__(self, heads: int, heads_kv: int, dim: int, cache: PagedCache, cos_sin,
                 chosen: int):
        super().__init__()
        width = heads * dim
        self.heads, self.heads_kv, self.dim, self.chosen = heads, heads_kv, dim, chosen
        self.qkv = torch.nn.Linear(width, (heads + 2 * heads_kv) * dim, bias=False)
        self.out = torch.nn.Linear(width, width, bias=False)
        self.cache, self.cos_sin = cache, cos_sin

    def forward(self, x, positions, seq_ids, sequences):
        rows = self.qkv(x).view(len(x), -1, self.dim)
        q, k, v = rows.split([self.heads, self.heads_kv, self.heads_kv], 1)  # (strided views)
        q = self.cache.append(q, k, v, self.cos_sin, positions, seq_ids)
        out, lse = self.cache.attend(q, positions, seq_ids, self.chosen, sink=1, recent=2,
                                     sequences=sequences)
        return self.out(out.view(len(x), -1)), q, lse


@torch.inference_mode()
def run(sequences: int, context: int, chosen: int, steps: int, heads: int = 32, heads_kv: int = 8,
        dim: int = 128, chunk: int = 4096) -> dict:
    torch.manual_seed(0)
    dev = torch.device("cuda", torch.cuda.current_device())
    total = context + steps
    blocks = -(-total // PAGE)
    cache = PagedCache(sequences * blocks, heads_kv, dim, PAGE, sequences, blocks, device=dev)
    for s in range(sequences):
        cache.reserve(s, total)
    layer = Layer(heads, heads_kv, dim, cache, rotary_table(total, dim, device=dev), chosen)
    layer = layer.to(dev, torch.bfloat16)
    begin, mid, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))

    # prompts: a chunk of each sequence in turn
    positions = torch.arange(total, dtype=torch.int32, device=dev)
    begin.record()
    for first in range(0, context, chunk):
        n = min(chunk, context - first)
        for s in range(sequences):
            x = torch.randn(n, heads * dim, device=dev, dtype=torch.bfloat16)
            seq_ids = torch.full((n,), s, dtype=torch.int32, device=dev)
            layer(x, positions[first:first + n], seq_ids, 1)
    mid.record()

    # single tokens: one graph, replayed with its inputs rewritten in place
    x = torch.randn(sequences, heads * dim, device=dev, dtype=torch.bfloat16)
    pos = torch.full((sequences,), context, dtype=torch.int32, device=dev)
    seq_ids = torch.arange(sequences, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, pos, seq_ids, sequences)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, q, lse = layer(x, pos, seq_ids, sequences)
    graph.replay()  # (the first replay sends the graph to the GPU)
    decode = torch.cuda.Event(enable_timing=True)
    decode.record()
    for i in range(steps):
        pos.fill_(context + i)
        graph.replay()
        x.copy_(torch.nn.functional.rms_norm(y, y.shape[1:]))
    end.record()

    every = torch.arange(blocks, dtype=torch.int32, device=dev)
    every = every.expand(sequences, heads_kv, blocks).contiguous()
    _, lse_all = block_attention(q, cache.k, cache.v, every, pos, seq_ids, cache.page_table)
    torch.cuda.synchronize()
    return {
        "prompt_tokens_per_s": sequences * context / begin.elapsed_time(mid) * 1e3,
        "decode_us_per_step": decode.elapsed_time(end) / steps * 1e3,
        "weight_of_the_chosen": float((lse - lse_all).exp().mean()),
        "share_of_the_blocks": min(1.0, chosen / blocks),
        "finite": bool(torch.isfinite(y).all()),
    }


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--sequences", type=int, default=8)
    p.add_argument("--context", type=int, default=32768)
    p.add_argument("--chosen", type=int, default=32)
    p.add_argument("--steps", type=int, default=64)
    args = p.parse_args()
    for name, value in run(args.sequences, args.context, args.chosen, args.steps).items():
        print(f"{name}: {value:.4g}" if isinstance(value, float) else f"{name}: {value}")


if __name__ == "__main__":
    main()
