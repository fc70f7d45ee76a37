"""The attention half of a W4A16 decoder layer, one token per sequence and step:

    x -> RMSNorm + INT4 q/k/v projection -> per-head norm and rotation
      -> quantised append to the paged cache -> attention over it
      -> INT4 output projection -> + x

`AttentionLayer.step` is the composition of the public operators, every one on
the current stream, none of which synchronises: it can be captured in a CUDA
graph.  Run as a module it times such a step, captured and replayed, and each
operator alone in the same graph form:

    python -m cudalab_b200.evaluator.decode_step [--batch 16] [--context 4096] [--bits 8]
        [--prefix 0]

With --prefix the sequences share that many tokens in front of their own.
"""
from __future__ import annotations

import argparse
import json
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[2]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from cudalab_b200.build import build  # noqa: E402
from cudalab_b200.int4gemv_quantize import quantize_w_device  # noqa: E402


def rotary_table(rows: int, rotary: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """fp32 [rows, rotary]: the cosines of every position's angles, then the sines."""
    inverse = base ** (-torch.arange(rotary // 2, dtype=torch.float64) * 2 / rotary)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), 1).float().contiguous().to(device)


class AttentionLayer:
    """Weights, cache and workspace of one layer; up to 16 sequences (the rows that a quantised
    projection takes at once).  Each sequence owns the pages of `context` tokens, `capacity` in
    all; with a prefix the cache holds its pages behind them."""

    def __init__(self, batch: int, hidden: int, q_heads: int, kv_heads: int, head_dim: int,
                 context: int, bits: int = 8, page_size: int = 64, prefix: int = 0, seed: int = 0):
        self.gemv, self.rope = build("int4gemv"), build("qknorm_rope")
        self.cache, self.attention = build("kvcache"), build("kvattention")
        self.batch, self.q_heads, self.kv_heads, self.head_dim = batch, q_heads, kv_heads, head_dim
        self.page_size, self.prefix = page_size, prefix
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def weights(rows: int, cols: int):
            w = torch.randn(rows, cols, device="cuda", generator=g) * cols ** -0.5
            return quantize_w_device(w.half())

        self.w_qkv = weights((q_heads + 2 * kv_heads) * head_dim, hidden)
        self.w_out = weights(hidden, q_heads * head_dim)
        self.norm, self.q_norm, self.k_norm = (
            (1 + 0.1 * torch.randn(n, device="cuda", generator=g)).half()
            for n in (hidden, head_dim, head_dim))
        width, shared = -(-context // page_size), -(-prefix // page_size)
        self.capacity = width * page_size
        self.table = rotary_table(prefix + self.capacity, head_dim)
        self.pages = self.cache.empty(batch * width + shared, kv_heads, head_dim, bits, page_size)
        self.page_table = torch.arange(batch * width, device="cuda",
                                       dtype=torch.int32).view(batch, width)
        self.prefix_pages = torch.arange(batch * width, batch * width + shared, device="cuda",
                                         dtype=torch.int32)
        self._number_slots()
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.workspace = self.attention.workspace("cuda")

    def fill(self, k, v, sequence: int | None) -> None:
        """Appends k, v [tokens, kv_heads, head_dim] (already rotated) to a sequence, or writes
        the shared prefix (None).  Refuses what the pages do not hold."""
        if sequence is None:
            first, most, pages = 0, self.prefix, self.prefix_pages.long()
        else:
            first, most = int(self.lengths[sequence]), self.capacity
            pages = self.page_table[sequence].long()
        if first + k.size(0) > most:
            raise RuntimeError(f"{k.size(0)} tokens after {first} exceed the {most} that the "
                               f"{'prefix' if sequence is None else 'sequence'} holds")
        at = torch.arange(first, first + k.size(0), device=self.pages.device)
        self.cache.write(k, v, self.pages, pages[at // self.page_size] * self.page_size
                         + at % self.page_size)
        if sequence is not None:
            self.lengths[sequence] += k.size(0)

    def _number_slots(self) -> None:
        """The slot of every token of a sequence, and -1 (skipped by the cache) behind them."""
        first = self.page_table.long() * self.page_size
        of_tokens = first[..., None] + torch.arange(self.page_size, device=first.device)
        self.slot_table = torch.nn.functional.pad(of_tokens.flatten(1), (0, 1), value=-1)

    def slots(self) -> torch.Tensor:
        """int64 [batch]: where each sequence's next token goes, -1 for one whose pages are
        full."""
        at = self.lengths.clamp(max=self.capacity).long()
        return self.slot_table.gather(1, at[:, None])[:, 0]

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """x fp16 [batch, hidden] of each sequence's next token -> the layer's output.  A
        sequence past its capacity keeps its cache; its row attends to that without the new
        token, and the device status records the length (7): a captured step has no other way
        to refuse it."""
        qkv = self.gemv.forward_rmsnorm("int4gemv_rmsnorm", *self.w_qkv, x, self.norm)
        slots, positions = self.slots(), self.lengths + self.prefix
        self.lengths += 1
        qkv = qkv.view(self.batch, -1, self.head_dim)
        q, k, v = qkv.split((self.q_heads, self.kv_heads, self.kv_heads), 1)
        q, k = self.rope.forward(q, k, self.q_norm, self.k_norm, self.table, positions)
        self.cache.write(k, v, self.pages, slots)
        if self.prefix:
            o = self.attention.forward_shared(q, self.pages, self.prefix_pages, self.prefix,
                                              self.page_table, self.lengths,
                                              workspace=self.workspace)
        else:
            o = self.attention.forward(q, self.pages, self.page_table, self.lengths,
                                       workspace=self.workspace)
        return x + self.gemv.forward_batched("int4gemv_mma", *self.w_out, o.view(self.batch, -1))


def _graph_us(fn, repeats: int = 20) -> float:
    """Device time of fn() in microseconds: captured ten times over, replayed."""
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            fn()
    graph.replay()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    times = []
    for _ in range(repeats):
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end) * 100)
    return sorted(times)[repeats // 2]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--context", type=int, default=4096)
    ap.add_argument("--bits", type=int, default=8, choices=(8, 4))
    ap.add_argument("--prefix", type=int, default=0)
    a = ap.parse_args()
    hidden, q_heads, kv_heads, dim = 4096, 32, 8, 128
    layer = AttentionLayer(a.batch, hidden, q_heads, kv_heads, dim, a.context + 512, a.bits,
                           prefix=a.prefix)
    for b in [None] * (a.prefix > 0) + list(range(a.batch)):
        n = a.prefix if b is None else a.context
        k, v = torch.randn(2, n, kv_heads, dim, device="cuda").half()
        layer.fill(k, v, b)
    x = torch.randn(a.batch, hidden, device="cuda").half()
    q = torch.randn(a.batch, q_heads, dim, device="cuda").half()
    k = torch.randn(a.batch, kv_heads, dim, device="cuda").half()
    slots, pos = layer.slots(), layer.lengths.long()
    parts = {
        "norm + qkv projection": lambda: layer.gemv.forward_rmsnorm(
            "int4gemv_rmsnorm", *layer.w_qkv, x, layer.norm),
        "head norm + rotation": lambda: layer.rope.forward(q, k, layer.q_norm, layer.k_norm,
                                                           layer.table, pos),
        "cache append": lambda: layer.cache.write(k, k, layer.pages, slots),
        "attention": (lambda: layer.attention.forward_shared(
            q, layer.pages, layer.prefix_pages, a.prefix, layer.page_table, layer.lengths,
            workspace=layer.workspace)) if a.prefix else (lambda: layer.attention.forward(
                q, layer.pages, layer.page_table, layer.lengths, workspace=layer.workspace)),
        "output projection": lambda: layer.gemv.forward_batched(
            "int4gemv_mma", *layer.w_out, q.view(a.batch, -1)),
    }
    us = {name: round(_graph_us(fn), 2) for name, fn in parts.items()}
    lengths = layer.lengths.clone()
    step = _graph_us(lambda: layer.step(x))
    layer.lengths.copy_(lengths)
    print(json.dumps({"batch": a.batch, "context": a.context, "prefix": a.prefix, "bits": a.bits,
                      "step_us": round(step, 2), "parts_us": us}))


if __name__ == "__main__":
    main()
