"""One transformer block in 4 bits on the library, as a serving program runs it: prompts of different
lengths, then tokens one after another.

    python examples/block_layer.py [--tokens 8] [--check]

    h = norm(x) (1 + scale) + shift                  in 4 bits       block_norm
    q, k, v = h . Wqkv                                               mx4_gemm
    prompts: q, k rotated in place                                   rope, attention, kv_append
    tokens: q rotated, k on its way into the cache                   rope, kv_append_rope,
                                                                     attention_cached
    x = x + gate (o . Wo); h = norm(x) (1 + scale) + shift           linear_mx4, block_norm
    x = x + gate (gelu(h . Wup) . Wdown)                             mx4_gemm, linear_mx4, block_norm

Weights are microscaled 4-bit codes, the stream is f32. A token's step is captured into a HIP graph
and replayed: lengths, positions and page tables live on the GPU.

--check computes every token's step once more eagerly and compares the bits.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from __graft_entry__ import load_package  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, INNER = 2048, 16, 4, 128, 8192
PAGE, PAGES = 64, 64
WIDTHS = [HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM]


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def sums(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


class Block:
    """The block's weights and its calls. `keep` holds what the stages gave, where it is a dict."""

    def __init__(self, pkg, gen):
        self.pkg, self.keep = pkg, None
        self.qkv = self._coded(gen, sum(WIDTHS), HIDDEN)
        self.out = self._coded(gen, HIDDEN, HEADS * DIM)
        self.up = self._coded(gen, INNER, HIDDEN)
        self.down = self._coded(gen, HIDDEN, INNER)
        # shift, scale and gate of the attention and of the feed-forward, one row for all tokens
        self.mod = (torch.randn((1, 6, HIDDEN), device="cuda", generator=gen) * 0.2).bfloat16()
        pairs = torch.arange(DIM // 2, device="cuda")
        self.freqs = (10000.0 ** (-pairs / (DIM // 2)))[None].contiguous()

    def _coded(self, gen, rows, k):
        w = self.pkg.MX4.empty(rows, k)
        self.pkg.mx4_quantize_rows(torch.randn((rows, k), device="cuda", generator=gen) * 0.03, w)
        return w

    def _seen(self, **stages):
        if self.keep is not None:
            self.keep.update({n: t.clone() if isinstance(t, torch.Tensor) else t
                              for n, t in stages.items()})

    def _empty(self, tokens, width, dtype=torch.bfloat16):
        return torch.empty((tokens, width), dtype=dtype, device="cuda")

    def project(self, x):
        """The block's start: q, k and v as parts of one tensor."""
        h = self.pkg.MX4.empty(len(x), HIDDEN)
        self.pkg.block_norm(x, h, shift=self.mod[:, 0], scale=self.mod[:, 1])
        y = self._empty(len(x), sum(WIDTHS))
        self.pkg.mx4_gemm(h, self.qkv, None, y)
        self._seen(h=h, qkv=y)
        return [p.unflatten(1, (-1, DIM)) for p in y.split(WIDTHS, 1)]

    def finish(self, x, o):
        """From the attention's output to the next block's input."""
        pkg, mod, n = self.pkg, self.mod, len(x)
        a, f = self._empty(n, HIDDEN), self._empty(n, HIDDEN)
        pkg.linear_mx4(o.flatten(1), self.out, None, a)
        mid, h = torch.empty_like(x), pkg.MX4.empty(n, HIDDEN)
        pkg.block_norm(x, h, y=a, x_out=mid, gate=mod[:, 2], shift=mod[:, 3], scale=mod[:, 4])
        u = self._empty(n, INNER)
        pkg.mx4_gemm(h, self.up, None, u, pkg.EPI_GELU_TANH)
        pkg.linear_mx4(u, self.down, None, f)
        end = torch.empty_like(x)
        pkg.block_norm(mid, None, y=f, x_out=end, gate=mod[:, 5])
        self._seen(o=o, a=a, mid=mid, h2=h, u=u, f=f, end=end)
        return end

    def prompt(self, x, lengths, cache, table):
        """New prompts, packed: every output, and their keys and values in the cache."""
        pkg = self.pkg
        q, k, v = self.project(x)
        at = int32([i for n in lengths for i in range(n)])[:, None].contiguous()
        cu = int32(sums(lengths))
        pkg.rope(q, k, at, self.freqs)
        self._seen(q=q, k=k)
        o = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda")
        pkg.attention(q, k, v, o, cu, cu, causal=True)
        pkg.kv_append(cache, table, k, v, cu, int32([0] * len(lengths)))
        return self.finish(x, o)

    def token(self, x, cache, table, lens, cu, longest):
        """One token of each sequence; `lens` tokens are in the cache before it."""
        pkg = self.pkg
        q, k, v = self.project(x)
        pkg.rope(q, None, lens[:, None], self.freqs)
        pkg.kv_append_rope(cache, table, k, v, cu, lens, self.freqs)
        o = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda")
        held = lens + 1
        pkg.attention_cached(cache, table, held, q, o, 1, longest, torch.empty(
            pkg.attention_cached_workspace(len(x), 1, HEADS, KV_HEADS, DIM, longest),
            dtype=torch.uint8, device="cuda"))
        self._seen(q=q, k_raw=k, v=v)
        return self.finish(x, o)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawTextHelpFormatter)
    ap.add_argument("--tokens", type=int, default=8, help="tokens decoded for each sequence")
    ap.add_argument("--check", action="store_true", help="compare replayed steps with eager ones")
    args = ap.parse_args()
    pkg = load_package()
    pkg.load()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    block = Block(pkg, gen)
    cache = pkg.KVCache.empty(PAGES, PAGE, KV_HEADS, DIM)
    lengths = [300, 1, 77, 513]
    pages = [-(-(n + args.tokens) // PAGE) for n in lengths]
    if sum(pages) > PAGES:
        ap.error(f"{args.tokens} tokens need {sum(pages)} pages, the cache has {PAGES}")
    table = torch.zeros((len(lengths), max(pages)), dtype=torch.int32, device="cuda")
    for b, (at, n) in enumerate(zip(sums(pages), pages)):
        table[b, :n] = int32(list(range(at, at + n)))
    x = torch.randn((sum(lengths), HIDDEN), device="cuda", generator=gen)
    y = block.prompt(x, lengths, cache, table)
    last = y[[n - 1 for n in sums(lengths)[1:]]].contiguous()

    lens, cu = int32(lengths), int32(list(range(len(lengths) + 1)))
    longest = max(lengths) + args.tokens
    step_in = last.clone()

    def step():
        return block.token(step_in, cache, table, lens, cu, longest)

    def again():
        """The step eagerly, on a cache of its own."""
        own = pkg.KVCache(*(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        return block.token(step_in, own, table, lens, cu, longest)

    again()   # kernels load and memory is found before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step_out = step()
    for i in range(args.tokens):
        step_in.copy_(last)
        want = again() if args.check else None
        graph.replay()
        if args.check and not torch.equal(step_out, want):
            raise SystemExit(f"token {i}: the replayed step differs from the eager one")
        last = step_out.clone()
        lens.add_(1)
    torch.cuda.synchronize()
    print(f"{len(lengths)} sequences, {sum(lengths)} prompt tokens, {args.tokens} decoded each")


if __name__ == "__main__":
    main()
