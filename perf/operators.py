"""Attention next to the quantized linears, and the 8-bit cache that serving keeps: cases that can
be timed and checked.

Paths:
  prompt   attention of packed sequences, queries / keys / values in place in the fused
           projection's output (`attention`)
  append   new keys and values quantized into the paged 8-bit cache (`kv_append`), and the blocks
           that they touch read back as a resumed prompt reads them (`kv_read`)
  cached   attention of the newest tokens over the cache (`attention_cached`)

With `own` false, `run` is the plain form: elementary torch operations in 32 bits, one rounding at
the end. Both forms work on what `prepare` gives, in the layouts that the framework's callers hold.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.getcwd()


def _package():
    name = "vpipe_ltx25_amd"
    if name not in sys.modules:
        # the package directory's name is no Python identifier: it is loaded by its path
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(ROOT, "vpipe-ltx-2.5_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---- cases ------------------------------------------------------------------------------

def _text(lengths):
    return ",".join(str(n) for n in lengths)


def _ints(text):
    return [int(n) for n in text.split(",")]


def _prompt(keys, heads, kv_heads, dim, causal=True, lse=False, queries=None, **name):
    """`keys`, `queries`: each sequence's numbers of tokens (queries None: one for each key)."""
    return dict(name, path="prompt", keys=_text(keys), queries=_text(queries or keys), heads=heads,
                kv_heads=kv_heads, dim=dim, causal=causal, lse=lse)


def _append(start, new, kv_heads, dim, page, **name):
    """`start`: tokens that a sequence's cache holds before the call; `new`: those that it gets."""
    return dict(name, path="append", start=_text(start), new=_text(new), kv_heads=kv_heads,
                dim=dim, page=page)


def _cached(keys, queries, heads, kv_heads, dim, page, lse=False, **name):
    """`keys`: tokens in each sequence's cache, its `queries` newest ones among them."""
    return dict(name, path="cached", keys=_text(keys), queries=queries, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, lse=lse)


def listed():
    return [
        # The audio stream's self-attention in a denoise step: 126 tokens, every token sees all.
        # The smallest prompt call.
        _prompt([126], 16, 16, 128, causal=False, name="audio_self"),
        # A serving step's batch of new prompts, packed, of very different lengths; the statistics
        # are kept to merge with another part's.
        _prompt([1500, 3, 700, 2047, 64, 129, 1, 1024, 333, 17, 480, 95], 32, 8, 128, lse=True,
                name="packed_prompts"),
        # Many short prompts at the narrow head width: most tiles are partly filled.
        _prompt([40 + (37 * i) % 161 for i in range(48)], 16, 4, 64, name="short_prompts"),
        # One long prompt: the largest causal call.
        _prompt([16384], 32, 8, 128, name="long_prompt"),
        # The video stream's self-attention, all tokens of a clip, a head of keys for each head of
        # queries: the largest square call.
        _prompt([8160], 32, 32, 128, causal=False, name="video_self"),
        # A prompt's keys and values going into the cache, four sequences, two of them resumed in
        # the middle of a block.
        _append([0, 1000, 0, 37], [4096, 2500, 1333, 263], 8, 128, 64, name="append_prompt"),
        # A decode step's append: one token for each of 64 sequences.
        _append([100 + 61 * i for i in range(64)], [1] * 64, 8, 128, 32, name="append_token"),
        # The first tokens of an answer, one user: where latency counts most.
        _cached([700], 1, 32, 8, 128, 64, name="decode_first"),
        # A decode step of a full batch at ordinary, uneven lengths.
        _cached([200 + (1013 * i) % 3897 for i in range(64)], 1, 32, 8, 128, 32,
                name="decode_batch"),
        # A decode step over long contexts: about 1 GB of cache, read once.
        _cached([131072, 99991, 120000, 131071], 1, 32, 8, 128, 64, lse=True, name="decode_long"),
        # A draft of five tokens checked at once, a head of keys for each head of queries, small
        # blocks.
        _cached([900 + (617 * i) % 5200 for i in range(24)], 5, 16, 16, 64, 16,
                name="decode_draft"),
    ]


# No drawn case goes over the largest listed one's operations or bytes.
_MOST_FLOPS = 2.2e12
_MOST_BYTES = 1.0e9


def _spread(rng, lo, hi):
    """A whole number, spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        path = rng.choice(["prompt", "prompt", "append", "cached", "cached"])
        dim = rng.choice([64, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16])
        page = rng.choice([16, 32, 64, 64, 128])
        batch = _spread(rng, 1, 64)
        if heads > 64:
            continue
        if path == "prompt":
            longest = _spread(rng, 1, 16384)
            keys = [_spread(rng, max(1, longest // 30), longest) for _ in range(batch)]
            causal, queries = rng.random() < 0.75, None
            if rng.random() < 0.3:
                # a prompt behind a prefix that is there already, or cross-attention
                queries = [_spread(rng, 1, n if causal else longest) for n in keys]
            case = _prompt(keys, heads, kv_heads, dim, causal, rng.random() < 0.3, queries)
        elif path == "append":
            longest = _spread(rng, 1, 8192)
            new = [_spread(rng, 1, longest) for _ in range(batch)]
            start = [rng.choice([0, _spread(rng, 1, 4096)]) for _ in range(batch)]
            case = _append(start, new, kv_heads, dim, page)
        else:
            queries = rng.choice([1, 1, 1, 2, 3, 5, 8, 16])
            longest = max(queries, _spread(rng, 1, 131072))
            keys = [max(queries, _spread(rng, max(1, longest // 30), longest))
                    for _ in range(batch)]
            case = _cached(keys, queries, heads, kv_heads, dim, page, rng.random() < 0.3)
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return case


# ---- inputs -----------------------------------------------------------------------------

def _sums(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _device(numbers):
    return torch.tensor(numbers, dtype=torch.int32, device="cuda")


def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _projection(gen, tokens, *heads, dim):
    """The output of a fused projection, [tokens][sum of heads * dim], and its parts in place."""
    y = _randn(gen, tokens, sum(heads) * dim).to(torch.bfloat16)
    return [p.unflatten(1, (-1, dim)) for p in y.split([h * dim for h in heads], 1)]


def _cache(gen, lengths, kv_heads, dim, page):
    """A cache that serving has filled: codes as normal values of a block give them, a scale of
    the block's and head's own, pages dealt out in no order."""
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + 3
    codes = []
    for shape in ((pages, kv_heads, page, dim), (pages, kv_heads, dim, page)):
        c = torch.empty(shape, dtype=torch.int8, device="cuda")
        for part in c.split(max(1, (1 << 28) // (kv_heads * page * dim))):
            part.copy_(_randn(gen, *part.shape).mul_(36).round_().clamp_(-127, 127))
        codes.append(c)
    scales = [0.02 + 0.03 * torch.rand((pages, kv_heads), device="cuda", generator=gen)
              for _ in range(2)]
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((len(lengths), max(blocks)), dtype=torch.int32, device="cuda")
    for b, (at, n) in enumerate(zip(_sums(blocks), blocks)):
        table[b, :n] = order[at:at + n]
    return dict(k=codes[0], v=codes[1], k_scale=scales[0], v_scale=scales[1], table=table)


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * int(seed) + 29)
    if c["path"] == "prompt":
        keys, queries = _ints(c["keys"]), _ints(c["queries"])
        if keys == queries:
            q, k, v = _projection(gen, sum(keys), c["heads"], c["kv_heads"], c["kv_heads"],
                                  dim=c["dim"])
        else:
            q, = _projection(gen, sum(queries), c["heads"], dim=c["dim"])
            k, v = _projection(gen, sum(keys), c["kv_heads"], c["kv_heads"], dim=c["dim"])
        return dict(q=q, k=k, v=v, cu_q=_device(_sums(queries)), cu_k=_device(_sums(keys)))
    if c["path"] == "append":
        start, new = _ints(c["start"]), _ints(c["new"])
        s = _cache(gen, [a + n for a, n in zip(start, new)], c["kv_heads"], c["dim"], c["page"])
        s["new_k"], s["new_v"] = _projection(gen, sum(new), c["kv_heads"], c["kv_heads"],
                                             dim=c["dim"])
        s["start"], s["cu"] = _device(start), _device(_sums(new))
        return s
    keys = _ints(c["keys"])
    s = _cache(gen, keys, c["kv_heads"], c["dim"], c["page"])
    s["q"], = _projection(gen, len(keys) * c["queries"], c["heads"], dim=c["dim"])
    s["lens"] = _device(keys)
    return s


def _touched(case):
    """Per sequence: the first token of the first block that an append touches, and how many
    tokens there are from it on."""
    page = case["page"]
    first = [a - a % page for a in _ints(case["start"])]
    return first, [a + n - f for a, n, f in zip(_ints(case["start"]), _ints(case["new"]), first)]


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if c["path"] == "append":
        first, count = _touched(c)
        s["first"], s["cu_read"] = _device(first), _device(_sums(count))
        shape = (sum(count), c["kv_heads"], c["dim"])
        s["read_k"] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        s["read_v"] = torch.empty_like(s["read_k"])
    else:
        s["out"] = torch.empty(s["q"].shape, dtype=torch.bfloat16, device="cuda")
        s["lse"] = (torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
                    if c["lse"] else None)
    if own:
        pkg = s["pkg"] = _package()
        pkg.load()
        if c["path"] != "prompt":
            s["cache"] = pkg.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if c["path"] == "cached":
            s["longest"] = max(_ints(c["keys"]))
            s["workspace"] = torch.empty(
                pkg.attention_cached_workspace(len(_ints(c["keys"])), c["queries"], c["heads"],
                                               c["kv_heads"], c["dim"], s["longest"]),
                dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append,
                "cached": _plain_cached}[c["path"]](s, c)
    pkg = s["pkg"]
    if c["path"] == "append":
        pkg.kv_append(s["cache"], s["table"], s["new_k"], s["new_v"], s["cu"], s["start"])
        pkg.kv_read(s["cache"], s["table"], s["read_k"], s["read_v"], s["cu_read"], s["first"])
        return {"k": s["read_k"], "v": s["read_v"], "k_scale": s["k_scale"],
                "v_scale": s["v_scale"]}
    if c["path"] == "prompt":
        pkg.attention(s["q"], s["k"], s["v"], s["out"], s["cu_q"], s["cu_k"], causal=c["causal"],
                      lse=s["lse"])
    else:
        pkg.attention_cached(s["cache"], s["table"], s["lens"], s["q"], s["out"], c["queries"],
                             s["longest"], s["workspace"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]} if c["lse"] else {"out": s["out"]}


def _plain_attend(q, k, v, causal):
    """One sequence: q [Lq][H][D], k and v [G][Lk][D] in 32 bits -> out [Lq][H][D] in 32 bits and
    lse [Lq][H]."""
    lq, heads, dim = q.shape
    groups, lk = k.shape[0], k.shape[1]
    out = torch.empty((lq, heads, dim), dtype=torch.float32, device=q.device)
    lse = torch.empty((lq, heads), dtype=torch.float32, device=q.device)
    step = max(1, min(groups, (1 << 30) // (lq * (heads // groups) * lk)))   # for the memory
    hidden = None
    if causal and lq > 1:
        hidden = (torch.arange(lk, device=q.device)[None, :]
                  > torch.arange(lk - lq, lk, device=q.device)[:, None])
    for g in range(0, groups, step):
        n = min(step, groups - g)
        h = slice(g * (heads // groups), (g + n) * (heads // groups))
        x = q[:, h].float().view(lq, n, -1, dim).permute(1, 2, 0, 3).reshape(n, -1, dim)
        p = (x @ k[g:g + n].transpose(1, 2)).mul_(dim ** -0.5).view(n, -1, lq, lk)
        if hidden is not None:
            p.masked_fill_(hidden, -math.inf)
        top = p.amax(3, keepdim=True)
        top.masked_fill_(top == -math.inf, 0.0)   # a query that sees nothing
        p.sub_(top).exp_()
        total = p.sum(3, keepdim=True)
        o = (p.view(n, -1, lk) @ v[g:g + n]).view(n, -1, lq, dim)
        o = o / total.masked_fill(total == 0, 1.0)
        out[:, h] = o.permute(2, 0, 1, 3).reshape(lq, -1, dim)
        lse[:, h] = (top + total.log()).permute(2, 0, 1, 3).reshape(lq, -1)
    return out, lse


def _plain_store(s, at, out, lse):
    s["out"][at] = out
    if s["lse"] is not None:
        s["lse"][at] = lse


def _plain_outputs(s):
    return {"out": s["out"]} if s["lse"] is None else {"out": s["out"], "lse": s["lse"]}


def _plain_prompt(s, c):
    cu_q, cu_k = _sums(_ints(c["queries"])), _sums(_ints(c["keys"]))
    for b in range(len(cu_q) - 1):
        rows, cols = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        k, v = (s[n][cols].float().transpose(0, 1).contiguous() for n in "kv")
        _plain_store(s, rows, *_plain_attend(s["q"][rows], k, v, c["causal"]))
    return _plain_outputs(s)


def _plain_values(codes, scale):
    return codes.float() * scale[:, :, None, None]


def _plain_cached(s, c):
    for b, n in enumerate(_ints(c["keys"])):
        at = s["table"][b, :-(-n // c["page"])]
        k = _plain_values(s["k"][at], s["k_scale"][at])
        v = _plain_values(s["v"][at], s["v_scale"][at]).transpose(2, 3)
        k, v = (x.transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n] for x in (k, v))
        rows = slice(b * c["queries"], (b + 1) * c["queries"])
        _plain_store(s, rows, *_plain_attend(s["q"][rows], k, v, True))
    return _plain_outputs(s)


def _plain_append(s, c):
    page, dev = c["page"], s["k"].device
    start, new, cu = _ints(c["start"]), _ints(c["new"]), _sums(_ints(c["new"]))
    units = [(b, p) for b, (a, n) in enumerate(zip(start, new))
             for p in range(a // page, (a + n - 1) // page + 1)]
    seq, block = (torch.tensor(x, device=dev) for x in zip(*units))
    at = s["table"][seq, block].long()
    place = block[:, None] * page + torch.arange(page, device=dev)
    first = s["start"].long()[seq][:, None]
    token = place - first + s["cu"].long()[seq][:, None]
    old = place < first
    fresh = (token < s["cu"].long()[seq + 1][:, None]) & ~old
    for codes, scale, x, turned in ((s["k"], s["k_scale"], s["new_k"], False),
                                    (s["v"], s["v_scale"], s["new_v"], True)):
        x = x[token.clamp(0, cu[-1] - 1)].float().masked_fill(~fresh[:, :, None, None], 0.0)
        s0 = scale[at] * old.any(1, keepdim=True)
        s1 = torch.maximum(s0, x.abs().amax((1, 3)) / 127.0)
        over = s1.masked_fill(s1 == 0, 1.0)[:, None, :, None]
        was = codes[at].transpose(2, 3) if turned else codes[at]
        was = was.transpose(1, 2).float()
        again = torch.where(s1 > s0, 1.0, 0.0)[:, None, :, None]
        kept = torch.where(again > 0, (was * s0[:, None, :, None] / over).round(), was)
        put = (x / over).round().clamp(-127.0, 127.0)
        now = torch.where(fresh[:, :, None, None], put,
                          torch.where(old[:, :, None, None], kept, was))
        now = now.to(torch.int8).transpose(1, 2)
        codes[at] = now.transpose(2, 3) if turned else now
        scale[at] = s1
    first, count = _touched(c)
    for b, (lo, n, to) in enumerate(zip(first, count, _sums(count))):
        at = s["table"][b, lo // page:(lo + n - 1) // page + 1]
        k = _plain_values(s["k"][at], s["k_scale"][at]).transpose(1, 2)
        v = _plain_values(s["v"][at], s["v_scale"][at]).permute(0, 3, 1, 2)
        s["read_k"][to:to + n] = k.flatten(0, 1)[:n]
        s["read_v"][to:to + n] = v.flatten(0, 1)[:n]
    return {"k": s["read_k"], "v": s["read_v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ---- what a pass cannot do without --------------------------------------------------------

def _visible(lq, lk, causal):
    """Pairs of a query and a key that it sees."""
    if not causal:
        return lq * lk
    rows = min(lq, lk)   # those that see any key; the last of them sees all
    return rows * lk - rows * (rows - 1) // 2


def work(case):
    c = case
    if c["path"] == "append":
        put, got = (float(sum(n)) * c["kv_heads"] * c["dim"]
                    for n in (_ints(c["new"]), _touched(c)[1]))
        # bf16 keys and values in, codes out; codes in, bf16 out
        return {"bytes": 6.0 * put + 6.0 * got, "flops": 8.0 * put + 2.0 * got}
    keys = _ints(c["keys"])
    queries = [c["queries"]] * len(keys) if c["path"] == "cached" else _ints(c["queries"])
    causal = c["path"] == "cached" or c["causal"]
    pairs = sum(_visible(lq, lk, causal) for lq, lk in zip(queries, keys))
    rows = float(sum(queries)) * c["heads"]
    held = float(sum(keys)) * c["kv_heads"]
    if c["path"] == "cached":
        blocks = sum(-(-n // c["page"]) for n in keys)
        moved = 2.0 * held * c["dim"] + 8.0 * blocks * c["kv_heads"]
    else:
        moved = 4.0 * held * c["dim"]
    return {"bytes": moved + 4.0 * rows * c["dim"] + (4.0 * rows if c["lse"] else 0.0),
            "flops": 4.0 * c["dim"] * c["heads"] * pairs}


# ---- the same in 64 bits -------------------------------------------------------------------

def _exact_attend(q, k, v, causal):
    """q [Lq][D], k and v [Lk][D] of one head, any type -> out and lse in 64 bits."""
    lq, lk = len(q), len(k)
    k, v = k.double(), v.double()
    outs, stats = [], []
    for lo in range(0, lq, 2048):
        x = q[lo:lo + 2048].double() @ k.t() / math.sqrt(k.shape[1])
        if causal:
            last = torch.arange(lo, lo + len(x), device=x.device) + (lk - lq)
            x = x + torch.where(torch.arange(lk, device=x.device) <= last[:, None], 0.0, -math.inf)
        z = torch.logsumexp(x, 1)
        w = (x - z[:, None]).exp_()
        w[z == -math.inf] = 0.0
        outs.append(w @ v)
        stats.append(z)
    return torch.cat(outs), torch.cat(stats)


def _exact_heads(s, c, spans, causal):
    """`spans`: (rows of q, a function from a kv head to its keys and values) per sequence."""
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    share = c["heads"] // c["kv_heads"]
    for rows, held in spans:
        for g in range(c["kv_heads"]):
            k, v = held(g)
            for h in range(g * share, (g + 1) * share):
                out[rows, h], lse[rows, h] = _exact_attend(s["q"][rows, h], k, v, causal)
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def _exact_append(s, c):
    """Page by page, each quotient in 64 bits and then in 32: the definition's own steps (a
    quotient of two 32-bit numbers rounds the same through 64 bits)."""
    page, table = c["page"], s["table"].tolist()
    first, count = _touched(c)
    total = sum(count)
    got = {n: torch.empty((total, c["kv_heads"], c["dim"]), dtype=torch.float64, device="cuda")
           for n in "kv"}
    scales = {n: s[n + "_scale"].double() for n in "kv"}
    f32 = lambda x: x.float().double()  # noqa: E731
    to, cu = _sums(count), _sums(_ints(c["new"]))
    for b, (a, n) in enumerate(zip(_ints(c["start"]), _ints(c["new"]))):
        for p in range(a // page, (a + n - 1) // page + 1):
            lo, hi = max(a, p * page), min(a + n, (p + 1) * page)
            pid, kept = table[b][p], lo - p * page
            for name in "kv":
                x = s["new_" + name][cu[b] + lo - a:cu[b] + hi - a].double()
                was = s[name][pid] if name == "k" else s[name][pid].transpose(1, 2)
                was = was[:, :kept].transpose(0, 1).double()
                s0 = scales[name][pid] if kept else torch.zeros_like(scales[name][pid])
                s1 = torch.maximum(s0, f32(x.abs().amax((0, 2)) / 127))
                per = torch.where(s1 > 0, s1, 1.0)[:, None]
                was = torch.where((s1 > s0)[:, None], f32(f32(was * s0[:, None]) / per).round(), was)
                codes = torch.cat([was, f32(x / per).round().clamp(-127, 127)])
                at = to[b] + p * page - first[b]
                got[name][at:at + len(codes)] = codes * s1[:, None]
                scales[name][pid] = s1
    return {"k": got["k"], "v": got["v"], "k_scale": scales["k"], "v_scale": scales["v"]}


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["path"] == "append":
        return _exact_append(s, c)
    spans, keys = [], _ints(c["keys"])
    if c["path"] == "prompt":
        cu_q, cu_k = _sums(_ints(c["queries"])), _sums(keys)
        for b in range(len(keys)):
            cols = slice(cu_k[b], cu_k[b + 1])
            spans.append((slice(cu_q[b], cu_q[b + 1]),
                          lambda g, cols=cols: (s["k"][cols, g], s["v"][cols, g])))
        return _exact_heads(s, c, spans, c["causal"])
    for b, n in enumerate(keys):
        at = s["table"][b, :-(-n // c["page"])].long()

        def held(g, at=at, n=n):
            k = s["k"][at, g].double() * s["k_scale"][at, g].double()[:, None, None]
            v = s["v"][at, g].double() * s["v_scale"][at, g].double()[:, None, None]
            return k.flatten(0, 1)[:n], v.transpose(1, 2).flatten(0, 1)[:n]

        spans.append((slice(b * c["queries"], (b + 1) * c["queries"]), held))
    return _exact_heads(s, c, spans, True)
