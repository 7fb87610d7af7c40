"""One attention layer on the library, as a serving program runs it: prompts of different lengths,
then tokens one after another, on quantized projections and an 8-bit cache.

    python examples/attention_layer.py [--tokens 24] [--check]

The layer is x + out(gate_heads(attention(q, k, v))) with q | k | v from one fused w8g64 projection
(ltx25_linear_q), the per-head gate's logits from a dense one, and the output projection quantized
again. A prompt goes through ltx25_attention on the fused projection's output in place; its keys and
values go into the cache (ltx25_kv_append). A token then takes a projection of one row for each
sequence, an append and ltx25_attention_cached, captured into a HIP graph and replayed: lengths and
page tables live on the GPU, so the graph's arguments never change.

A sequence that was set aside resumes with its next prompt part on top of the cache: its prefix is
read back (ltx25_kv_read) next to the new part's keys and values, and ltx25_attention sees both.

--check computes every token's output again from the layer's inputs in one prompt call, without
the cache, and compares: the two differ by the cache's rounding to 8 bits.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from __graft_entry__ import load_package  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM = 2048, 16, 4, 128
PAGE, PAGES = 64, 64


class Layer:
    """The layer's weights, quantized as a checkpoint holds them, and its calls."""

    def __init__(self, pkg, gen):
        self.pkg = pkg
        self.width = (HEADS + 2 * KV_HEADS) * DIM
        self.qkv = self._quantized(gen, self.width, HIDDEN)
        self.out = self._quantized(gen, HIDDEN, HEADS * DIM)
        self.gate = (torch.randn((HEADS, HIDDEN), device="cuda", generator=gen) * 0.02).bfloat16()

    def _quantized(self, gen, n, k):
        w = torch.randn((n, k), device="cuda", generator=gen) * 0.03
        codes = torch.empty((n, k), dtype=torch.uint8, device="cuda")
        scales, zeros = (torch.empty((n, k // 64), dtype=torch.bfloat16, device="cuda")
                         for _ in range(2))
        self.pkg.quantize_affine(w, codes, scales, zeros, n, k, 8, 64)
        return self.pkg.QWeight(codes, scales, zeros, 8, 64)

    def project(self, x):
        """x [T][HIDDEN] -> q, k, v as parts of one tensor, and the gate's logits. The
        no-allocation linear, so that a captured step allocates nothing."""
        y = torch.empty((len(x), self.width), dtype=torch.bfloat16, device="cuda")
        self.pkg.linear_q_noalloc(x, self.qkv, None, y, len(x), HIDDEN, self.width)
        logits = torch.empty((len(x), HEADS), dtype=torch.bfloat16, device="cuda")
        self.pkg.linear(x, self.gate, None, logits, len(x), HIDDEN, HEADS)
        parts = y.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1)
        return [p.unflatten(1, (-1, DIM)) for p in parts], logits

    def finish(self, x, o, logits):
        self.pkg.gate_heads(o, logits, HEADS, len(x), DIM)
        y = torch.empty_like(x)
        self.pkg.linear_q_noalloc(o.flatten(1), self.out, None, y, len(x), HEADS * DIM, HIDDEN)
        return x + y


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def sums(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return int32(out)


def prompt(pkg, layer, cache, table, x, lengths):
    """New prompts, packed; every output, and their keys and values in the cache."""
    (q, k, v), logits = layer.project(x)
    cu = sums(lengths)
    o = torch.empty((len(x), HEADS, DIM), dtype=torch.bfloat16, device="cuda")
    pkg.attention(q, k, v, o, cu, cu, causal=True)
    pkg.kv_append(cache, table, k, v, cu, int32([0] * len(lengths)))
    return layer.finish(x, o, logits)


def resume(pkg, layer, cache, table, x, held):
    """A later part of one sequence's prompt, on top of the `held` tokens of its cache."""
    (q, k, v), logits = layer.project(x)
    n = len(x)
    keys, values = (torch.empty((held + n, KV_HEADS, DIM), dtype=torch.bfloat16, device="cuda")
                    for _ in range(2))
    pkg.kv_read(cache, table, keys[:held], values[:held], sums([held]), int32([0]))
    keys[held:], values[held:] = k, v
    o = torch.empty((n, HEADS, DIM), dtype=torch.bfloat16, device="cuda")
    pkg.attention(q, keys, values, o, causal=True)   # the last query sees the last key
    pkg.kv_append(cache, table, k, v, sums([n]), int32([held]))
    return layer.finish(x, o, logits)


class Decoder:
    """A step of one token for each sequence, captured once."""

    def __init__(self, pkg, layer, cache, table, lens, longest):
        self.pkg, self.layer, self.cache, self.table = pkg, layer, cache, table
        self.lens, self.longest = lens, longest
        batch = len(lens)
        self.x = torch.zeros((batch, HIDDEN), dtype=torch.bfloat16, device="cuda")
        self.cu = int32(list(range(batch + 1)))
        self.workspace = torch.empty(
            pkg.attention_cached_workspace(batch, 1, HEADS, KV_HEADS, DIM, longest),
            dtype=torch.uint8, device="cuda")
        self.graph = None

    def _step(self):
        pkg = self.pkg
        (q, k, v), logits = self.layer.project(self.x)
        o = torch.empty((len(self.x), HEADS, DIM), dtype=torch.bfloat16, device="cuda")
        pkg.kv_append(self.cache, self.table, k, v, self.cu, self.lens)
        self.lens.add_(1)   # the new token is in the cache now
        pkg.attention_cached(self.cache, self.table, self.lens, q, o, 1, self.longest,
                             self.workspace)
        return self.layer.finish(self.x, o, logits)

    def __call__(self, x):
        self.x.copy_(x)
        if self.graph is None:
            y = self._step().clone()   # the first step eagerly: kernels load, memory is found
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.y = self._step()
            return y
        self.graph.replay()
        return self.y.clone()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawTextHelpFormatter)
    ap.add_argument("--tokens", type=int, default=24, help="tokens decoded for each sequence")
    ap.add_argument("--check", action="store_true", help="compare with one prompt call")
    args = ap.parse_args()
    pkg = load_package()
    pkg.load()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    layer = Layer(pkg, gen)
    cache = pkg.KVCache.empty(PAGES, PAGE, KV_HEADS, DIM)

    lengths, part = [300, 1, 77, 513], 150   # prompts, and a later part of the third
    total = [n + (part if b == 2 else 0) + args.tokens for b, n in enumerate(lengths)]
    pages = [-(-n // PAGE) for n in total]
    if sum(pages) > PAGES:
        ap.error(f"{args.tokens} tokens need {sum(pages)} pages, the cache has {PAGES}")
    table = torch.zeros((len(lengths), max(pages)), dtype=torch.int32, device="cuda")
    free = iter(torch.randperm(PAGES, generator=torch.Generator().manual_seed(1)).tolist())
    for b, n in enumerate(pages):
        table[b, :n] = int32([next(free) for _ in range(n)])

    inputs = [torch.randn((n, HIDDEN), device="cuda", generator=gen).bfloat16() for n in total]
    got = [[] for _ in lengths]

    y = prompt(pkg, layer, cache, table, torch.cat([x[:n] for x, n in zip(inputs, lengths)]), lengths)
    for b, p in enumerate(y.split(lengths)):
        got[b].append(p)
    got[2].append(resume(pkg, layer, cache, table[2:3], inputs[2][77:77 + part], 77))
    lengths[2] += part

    lens = int32(lengths)
    decode = Decoder(pkg, layer, cache, table, lens, max(total))
    for i in range(args.tokens):
        y = decode(torch.stack([x[n + i] for x, n in zip(inputs, lengths)]))
        for b in range(len(lengths)):
            got[b].append(y[b:b + 1])
    torch.cuda.synchronize()
    print(f"{len(lengths)} sequences, {sum(lengths)} prompt tokens, {args.tokens} decoded each")

    if args.check:
        worst = 0.0
        for b, x in enumerate(inputs):
            (q, k, v), logits = layer.project(x)
            o = torch.empty((len(x), HEADS, DIM), dtype=torch.bfloat16, device="cuda")
            pkg.attention(q, k, v, o, causal=True)
            worst = max(worst, rel(torch.cat(got[b]) - x, layer.finish(x, o, logits) - x))
        print(f"largest difference from one prompt call: {worst:.2e}")
        if not worst < 2e-2:
            raise SystemExit("the two disagree")


if __name__ == "__main__":
    main()
