"""What a block does around its linears and its attention, in 4 bits: cases that can be timed and
checked.

Paths:
  codes    a weight's or an activation's rows to microscaled 4-bit codes (`mx4_quantize_rows`) and
           their values back in bf16 (`mx4_dequant`), as a loader checks what it coded
  linear   bf16 activations, 4-bit weights: the activations coded on the way, the product of the
           codes, bias and GELU (`linear_mx4`)
  normed   residual, norm and modulation straight to 4-bit codes (`block_norm`), then their product
           with a weight (`mx4_gemm`)
  norm     the same norms with a bf16 output (`block_norm`)
  rope     positions of one or several axes rotated into queries and keys (`rope`)
  append   keys rotated on their way into the paged 8-bit cache, values with them
           (`kv_append_rope`), and the pages that they touch read back (`kv_read`)

With `own` false, `run` is the plain form: elementary torch operations in 32 bits (angles in 64), one
rounding at the end. Both forms work on what `prepare` gives.
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


def _codes(rows, width, wide, **name):
    """wide: float32 values, as a checkpoint's weight comes; else bf16."""
    return dict(name, path="codes", rows=rows, width=width, wide=wide)


def _linear(tokens, width, out, bias=True, gelu=False, **name):
    return dict(name, path="linear", tokens=tokens, width=width, out=out, bias=bias, gelu=gelu)


def _norm(tokens, width, wide=False, branch=True, after=False, layer=False, modulated=True,
          mod_rows=1, mapped=False, weight=False, alpha=1.0, **name):
    """wide: the residual stream in float32; branch: a block's output is added first, after:
    normed before it is; modulated: gate, scale and shift, `mod_rows` rows of them, `mapped` to the
    tokens by an index or dealt to them evenly."""
    return dict(name, path="norm", tokens=tokens, width=width, wide=wide, branch=branch,
                after=after, layer=layer, modulated=modulated, mod_rows=mod_rows, mapped=mapped,
                weight=weight, alpha=alpha)


def _normed(tokens, width, out, gelu=False, **more):
    return dict(_norm(tokens, width, **more), path="normed", out=out, gelu=gelu)


def _rope(tokens, heads, kv_heads, dim, rotated, axes=1, per_head=False, pairs_side=False,
          **name):
    """rotated: how many of a head's channels; pairs_side: a pair's two channels lie side by side,
    else half of the rotated ones apart; per_head: each head has frequencies of its own."""
    return dict(name, path="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rotated=rotated, axes=axes, per_head=per_head, pairs_side=pairs_side)


def _append(start, new, kv_heads, dim, page, rotated, pairs_side=False, **name):
    return dict(name, path="append", start=_text(start), new=_text(new), kv_heads=kv_heads,
                dim=dim, page=page, rotated=rotated, pairs_side=pairs_side)


def listed():
    return [
        # A feed-forward's weight as it is loaded: float32 in, 4-bit codes, and the values that
        # they stand for.
        _codes(16384, 4096, True, name="weight_codes"),
        # A short clip's audio tokens.
        _codes(126, 2048, False, name="token_codes"),
        # One token through a projection: the weight is read once, latency counts.
        _linear(1, 4096, 4096, name="one_token"),
        # Prompt tokens of no round number, an output of no round width, no bias.
        _linear(333, 2080, 1001, bias=False, name="odd_linear"),
        # The video stream's feed-forward, up: the largest call.
        _linear(8160, 4096, 16384, gelu=True, name="ffn_up"),
        # A serving step's prompts: the branch before it closed, normed, modulated and coded, then
        # the fused projection.
        _normed(1024, 4096, 12288, name="normed_projection"),
        # A block's end on the video stream: gate, residual, norm and modulation with a row for
        # each of the clip's conditioned and free tokens.
        _norm(8160, 4096, mod_rows=17, mapped=True, name="video_norm"),
        # A batch's next tokens, the stream in float32, norms before and after each block with
        # learned weights, the residual scaled.
        _norm(64, 2048, wide=True, after=True, modulated=False, weight=True, alpha=0.7,
              name="token_norm"),
        # The video stream's queries and keys: time, height and width, every head with frequencies
        # of its own.
        _rope(8160, 32, 32, 128, 128, axes=3, per_head=True, name="video_rope"),
        # A decode step's queries and keys, one axis, pairs side by side.
        _rope(64, 32, 8, 128, 128, pairs_side=True, name="token_rope"),
        # Prompts into the cache, two of them resumed in the middle of a page.
        _append([0, 1000, 0, 37], [4096, 2500, 1333, 263], 8, 128, 64, 128,
                name="append_prompt"),
        # One token each of 64 sequences into the cache; half of a head's channels are rotated.
        _append([100 + 61 * i for i in range(64)], [1] * 64, 8, 128, 32, 64, pairs_side=True,
                name="append_token"),
    ]


# No drawn case goes over the largest listed one's operations or bytes.
_MOST_FLOPS = 1.1e12
_MOST_BYTES = 3.7e8


def _spread(rng, lo, hi):
    """A whole number, spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _some(rng, share):
    return rng.random() < share


def _drawn_norm(rng, step):
    tokens, width = _spread(rng, 1, 16384), step * _spread(rng, 1, 16384 // step)
    rows = rng.choice([1, tokens, _spread(rng, 1, tokens)])
    return dict(tokens=tokens, width=width, wide=_some(rng, 0.3), branch=_some(rng, 0.8),
                after=_some(rng, 0.3), layer=_some(rng, 0.3), modulated=_some(rng, 0.7),
                mod_rows=rows, mapped=tokens % rows != 0 or _some(rng, 0.5),
                weight=_some(rng, 0.5), alpha=rng.choice([1.0, 1.0, 0.5, 1.3]))


def draw(rng):
    while True:
        path = rng.choice(["codes", "linear", "linear", "linear", "normed", "norm", "norm", "rope",
                           "rope", "append"])
        if path == "codes":
            case = _codes(_spread(rng, 1, 16384), 32 * _spread(rng, 1, 512), _some(rng, 0.5))
        elif path == "linear":
            case = _linear(_spread(rng, 1, 8192), 32 * _spread(rng, 1, 512),
                           _spread(rng, 1, 16384), _some(rng, 0.6), _some(rng, 0.3))
        elif path == "normed":
            case = _normed(out=_spread(rng, 1, 16384), gelu=_some(rng, 0.3), **_drawn_norm(rng, 32))
        elif path == "norm":
            case = _norm(**_drawn_norm(rng, 8))
        elif path == "rope":
            kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
            heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8])
            dim = rng.choice([32, 64, 80, 128, 128, 256])
            case = _rope(_spread(rng, 1, 16384), heads, kv_heads, dim,
                         dim if _some(rng, 0.6) else 16 * rng.randint(1, dim // 16),
                         rng.choice([1, 2, 3, 3, 4]), heads == kv_heads and _some(rng, 0.5),
                         _some(rng, 0.5))
            if heads > 64:
                continue
        else:
            longest = _spread(rng, 1, 8192)
            batch = _spread(rng, 1, 64)
            dim = rng.choice([64, 128])
            case = _append([rng.choice([0, _spread(rng, 1, 4096)]) for _ in range(batch)],
                           [_spread(rng, 1, longest) for _ in range(batch)],
                           rng.choice([1, 2, 4, 8, 8, 16]), dim, rng.choice([16, 32, 64, 64, 128]),
                           rng.choice([dim, dim, dim // 2]), _some(rng, 0.5))
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


def _activations(gen, tokens, width):
    """Activations as a stream has them: some channels are much larger than others."""
    return _randn(gen, tokens, width) * torch.exp(0.7 * _randn(gen, width))


def _weight(gen, rows, width):
    """A weight as a checkpoint in 4 bits holds it: codes, the low half first, and each block of
    32's exponent with 127 added."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    codes = torch.empty((rows, width // 2), dtype=torch.uint8, device="cuda")
    for part in codes.split(max(1, (1 << 26) // width)):
        v = 2 * _randn(gen, len(part), width // 2, 2)
        half = torch.bucketize(v.abs(), mids).to(torch.uint8) + 8 * (v < 0).to(torch.uint8)
        part.copy_(half[:, :, 0] + 16 * half[:, :, 1])
    spread = torch.randint(0, 3, (rows, width // 32), dtype=torch.uint8, device="cuda",
                           generator=gen)
    return codes, spread + 118


def _pages(gen, lengths, kv_heads, dim, page):
    """A cache that serving has filled, its pages dealt out in no order."""
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + 3
    k, v = (_randn(gen, *shape).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
            for shape in ((pages, kv_heads, page, dim), (pages, kv_heads, dim, page)))
    scales = [0.02 + 0.03 * torch.rand((pages, kv_heads), device="cuda", generator=gen)
              for _ in range(2)]
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((len(lengths), max(blocks)), dtype=torch.int32, device="cuda")
    for b, (at, n) in enumerate(zip(_sums(blocks), blocks)):
        table[b, :n] = order[at:at + n]
    return dict(k=k, v=v, k_scale=scales[0], v_scale=scales[1], table=table)


def _norm_inputs(c, gen):
    tokens, width, rows = c["tokens"], c["width"], c["mod_rows"]
    s = dict(x=_activations(gen, tokens, width).to(torch.float32 if c["wide"] else torch.bfloat16),
             y=None, gate=None, scale=None, shift=None, rows=None, weight=None, after=None)
    if c["branch"]:
        s["y"] = _activations(gen, tokens, width).bfloat16()
        if c["after"]:
            s["after"] = (1 + 0.2 * _randn(gen, width)).bfloat16()
    if c["modulated"]:
        # the parts of one tensor, as a timestep's projection gives them
        six = (0.3 * _randn(gen, rows, 6, width)).bfloat16()
        s["shift"], s["scale"] = six[:, 3], six[:, 4]
        if c["branch"]:
            s["gate"] = six[:, 2]
        if c["mapped"]:
            s["rows"] = torch.randint(0, rows, (tokens,), dtype=torch.int32, device="cuda",
                                      generator=gen)
    if c["weight"]:
        s["weight"] = (1 + 0.2 * _randn(gen, width)).bfloat16()
    return s


def _frequencies(pairs, theta=10000.0):
    return torch.tensor([[theta ** (-i / pairs) for i in range(pairs)]], dtype=torch.float32,
                        device="cuda")


def _rope_inputs(c, gen):
    tokens, heads, kv_heads, dim = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    pairs, axes = c["rotated"] // 2, c["axes"]
    y = _randn(gen, tokens, (heads + 2 * kv_heads) * dim).bfloat16()
    q, k, _ = (p.unflatten(1, (-1, dim)) for p in
               y.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    if axes == 1:
        # text: whole positions, some of them far into a document
        at = torch.randint(0, 1 << 20, (tokens, 1), dtype=torch.int32, device="cuda", generator=gen)
    else:
        # a grid's middles, as shares of its length, from -1 to 1
        at = 2 * torch.rand((tokens, axes), device="cuda", generator=gen) - 1
    if c["per_head"]:
        n = heads * pairs
        steps = max(1, n // axes - 1)
        freqs = torch.tensor([math.pi / 2 * 10000.0 ** min(1.0, (i // axes) / steps)
                              for i in range(n)], device="cuda").view(heads, pairs)
        which = _device([i % axes for i in range(n)]).view(heads, pairs)
    else:
        freqs = _frequencies(pairs) if axes == 1 else math.pi / 2 * 1000 * _frequencies(pairs)
        which = _device([[i * axes // pairs for i in range(pairs)]])
    return dict(q=q, k=k, at=at, freqs=freqs, which=which)


def _append_inputs(c, gen):
    start, new = _ints(c["start"]), _ints(c["new"])
    s = _pages(gen, [a + n for a, n in zip(start, new)], c["kv_heads"], c["dim"], c["page"])
    y = _randn(gen, sum(new), 2 * c["kv_heads"] * c["dim"]).bfloat16()
    s["new_k"], s["new_v"] = (p.unflatten(1, (-1, c["dim"])) for p in y.chunk(2, 1))
    s["start"], s["cu"] = _device(start), _device(_sums(new))
    s["freqs"] = _frequencies(c["rotated"] // 2)
    s["which"] = torch.zeros_like(s["freqs"], dtype=torch.int32)
    return s


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * int(seed) + 41)
    if c["path"] == "codes":
        x = _activations(gen, c["rows"], c["width"])
        return dict(x=x if c["wide"] else x.bfloat16())
    if c["path"] == "rope":
        return _rope_inputs(c, gen)
    if c["path"] == "append":
        return _append_inputs(c, gen)
    if c["path"] == "linear":
        s = dict(x=_activations(gen, c["tokens"], c["width"]).bfloat16(),
                 bias=0.5 * _randn(gen, c["out"]) if c["bias"] else None)
    else:
        s = _norm_inputs(c, gen)
        s["bias"] = None
    if c["path"] != "norm":
        s["codes"], s["exps"] = _weight(gen, c["out"], c["width"])
    return s


def _touched(case):
    """Per sequence: the first token of the first page that an append touches, and how many tokens
    there are from it on."""
    page = case["page"]
    first = [a - a % page for a in _ints(case["start"])]
    return first, [a + n - f for a, n, f in zip(_ints(case["start"]), _ints(case["new"]), first)]


def _empty(shape, like=torch.bfloat16):
    return torch.empty(shape, dtype=like, device="cuda")


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if c["path"] == "codes":
        s["out"] = _empty(s["x"].shape)
    elif c["path"] == "rope":
        s["q_out"] = _empty(s["q"].shape)
        s["k_out"] = _empty(s["k"].shape)
    elif c["path"] == "append":
        first, count = _touched(c)
        s["first"], s["cu_read"] = _device(first), _device(_sums(count))
        s["read_k"] = _empty((sum(count), c["kv_heads"], c["dim"]))
        s["read_v"] = torch.empty_like(s["read_k"])
    else:
        s["out"] = _empty((c["tokens"], c["width" if c["path"] == "norm" else "out"]))
        if c["path"] != "linear":
            s["x_out"] = torch.empty_like(s["x"]) if c["branch"] else None
    if own:
        pkg = s["pkg"] = _package()
        pkg.load()
        if c["path"] == "append":
            s["cache"] = pkg.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if c["path"] == "codes":
            s["coded"] = pkg.MX4.empty(c["rows"], c["width"])
        if "codes" in s:
            s["w"] = pkg.MX4.packed(s["codes"], s["exps"])
        if c["path"] == "normed":
            s["coded"] = pkg.MX4.empty(c["tokens"], c["width"])
        if "out" in c:
            need = pkg.linear_mx4_workspace if c["path"] == "linear" else pkg.mx4_gemm_workspace
            s["workspace"] = torch.empty(need(c["tokens"], c["width"], c["out"]),
                                         dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"codes": _plain_codes, "linear": _plain_linear, "normed": _plain_normed,
                "norm": _plain_norm, "rope": _plain_rope, "append": _plain_append}[c["path"]](s, c)
    pkg = s["pkg"]
    if c["path"] == "codes":
        pkg.mx4_quantize_rows(s["x"], s["coded"])
        pkg.mx4_dequant(s["coded"], s["out"])
        return {"out": s["out"]}
    if c["path"] == "rope":
        pkg.rope(s["q"], s["k"], s["at"], s["freqs"], s["which"], q_out=s["q_out"],
                 k_out=s["k_out"], interleaved=c["pairs_side"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if c["path"] == "append":
        pkg.kv_append_rope(s["cache"], s["table"], s["new_k"], s["new_v"], s["cu"], s["start"],
                           s["freqs"], s["which"], interleaved=c["pairs_side"])
        pkg.kv_read(s["cache"], s["table"], s["read_k"], s["read_v"], s["cu_read"], s["first"])
        return {"k": s["read_k"], "v": s["read_v"], "k_scale": s["k_scale"],
                "v_scale": s["v_scale"]}
    epilogue = pkg.EPI_GELU_TANH if c.get("gelu") else pkg.EPI_NONE
    if c["path"] == "linear":
        pkg.linear_mx4(s["x"], s["w"], s["bias"], s["out"], epilogue, workspace=s["workspace"])
        return {"out": s["out"]}
    pkg.block_norm(s["x"], s["coded"] if c["path"] == "normed" else s["out"], y=s["y"],
                   x_out=s["x_out"], gate=s["gate"], post_weight=s["after"], weight=s["weight"],
                   scale=s["scale"], shift=s["shift"], rows=s["rows"], layer=c["layer"],
                   residual_scale=c["alpha"])
    if c["path"] == "normed":
        pkg.mx4_gemm(s["coded"], s["w"], None, s["out"], epilogue, workspace=s["workspace"])
    return _norm_outputs(s)


def _norm_outputs(s):
    return {"out": s["out"]} if s["x_out"] is None else {"out": s["out"], "x": s["x_out"]}


_MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _plain_mx4(x):
    """Rows' values after 4-bit coding, in 32 bits: a block of 32 is held as the nearest of eight
    magnitudes, ties to the even one, times a power of two two below its largest value's."""
    b = x.float().unflatten(1, (-1, 32))
    top = b.abs().amax(2, keepdim=True)
    # frexp: top = m 2^e with m in [0.5, 1)
    exp = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    v = torch.ldexp(b, -exp)
    mag, idx = v.abs(), torch.zeros_like(v, dtype=torch.int32)
    for i in range(7):
        mid = (_MAGNITUDES[i] + _MAGNITUDES[i + 1]) / 2
        idx += (mag >= mid) if i % 2 else (mag > mid)
    q = torch.tensor(_MAGNITUDES, device=x.device)[idx.long()]
    return torch.ldexp(torch.where(v < 0, -q, q), exp).flatten(1)


def _plain_weight(s):
    """The weight's values in 32 bits from its codes and exponents."""
    values = torch.tensor(_MAGNITUDES + [-m for m in _MAGNITUDES], device=s["codes"].device)
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).flatten(1)
    w = values[codes.int()].unflatten(1, (-1, 32))
    return torch.ldexp(w, (s["exps"].int() - 127)[:, :, None]).flatten(1)


def _plain_codes(s, c):
    s["out"].copy_(_plain_mx4(s["x"]))
    return {"out": s["out"]}


def _plain_product(s, c, x):
    y = x @ _plain_weight(s).t()
    if s["bias"] is not None:
        y += s["bias"]
    if c["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    s["out"].copy_(y)


def _plain_linear(s, c):
    _plain_product(s, c, _plain_mx4(s["x"]))
    return {"out": s["out"]}


_EPS = 1e-6


def _plain_scaled(x, layer):
    if layer:
        x = x - x.mean(1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + _EPS)


def _token_rows(s, c, m):
    """A modulation's row for each token, in 32 bits."""
    m = m.float()
    if s["rows"] is not None:
        return m[s["rows"].long()]
    return m.repeat_interleave(c["tokens"] // c["mod_rows"], 0)


def _plain_normalised(s, c):
    x = s["x"].float()
    if s["y"] is not None:
        u = s["y"].float()
        if s["after"] is not None:
            u = _plain_scaled(u, c["layer"]) * s["after"].float()
        if s["gate"] is not None:
            u = u * _token_rows(s, c, s["gate"])
        x = c["alpha"] * x + u
        s["x_out"].copy_(x)
    h = _plain_scaled(x, c["layer"])
    if s["weight"] is not None:
        h = h * s["weight"].float()
    if s["scale"] is not None:
        h = h * (1 + _token_rows(s, c, s["scale"])) + _token_rows(s, c, s["shift"])
    return h


def _plain_norm(s, c):
    s["out"].copy_(_plain_normalised(s, c))
    return _norm_outputs(s)


def _plain_normed(s, c):
    _plain_product(s, c, _plain_mx4(_plain_normalised(s, c)))
    return _norm_outputs(s)


def _plain_rotate(x, cos, sin, side):
    """x [tokens][heads][dim] in 32 bits; cos, sin [tokens][heads or 1][pairs]."""
    n = cos.shape[2]
    rot, rest = x[:, :, :2 * n], x[:, :, 2 * n:]
    a, b = (rot[:, :, 0::2], rot[:, :, 1::2]) if side else (rot[:, :, :n], rot[:, :, n:])
    a, b = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack([a, b], 3).flatten(2) if side else torch.cat([a, b], 2)
    return torch.cat([rot, rest], 2)


def _plain_turns(at, freqs, which):
    """cos and sin [tokens][heads or 1][pairs]; angles in 64 bits."""
    angle = at.double()[:, which.long()] * freqs.double()
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_rope(s, c):
    cos, sin = _plain_turns(s["at"], s["freqs"], s["which"])
    for n in "qk":
        s[n + "_out"].copy_(_plain_rotate(s[n].float(), cos, sin, c["pairs_side"]))
    return {"q": s["q_out"], "k": s["k_out"]}


def _plain_append(s, c):
    page, dev = c["page"], s["k"].device
    start, new, cu = _ints(c["start"]), _ints(c["new"]), _sums(_ints(c["new"]))
    at = torch.cat([torch.arange(a, a + n, device=dev) for a, n in zip(start, new)])
    cos, sin = _plain_turns(at[:, None], s["freqs"], s["which"])
    # the cache holds codes of the keys that a rotation of their own would have written
    keys = _plain_rotate(s["new_k"].float(), cos, sin, c["pairs_side"]).bfloat16()
    units = [(b, p) for b, (a, n) in enumerate(zip(start, new))
             for p in range(a // page, (a + n - 1) // page + 1)]
    seq, block = (torch.tensor(x, device=dev) for x in zip(*units))
    where = s["table"][seq, block].long()
    place = block[:, None] * page + torch.arange(page, device=dev)
    first = s["start"].long()[seq][:, None]
    token = place - first + s["cu"].long()[seq][:, None]
    old = place < first
    fresh = (token < s["cu"].long()[seq + 1][:, None]) & ~old
    for codes, scale, x, turned in ((s["k"], s["k_scale"], keys, False),
                                    (s["v"], s["v_scale"], s["new_v"], True)):
        x = x[token.clamp(0, cu[-1] - 1)].float().masked_fill(~fresh[:, :, None, None], 0.0)
        s0 = scale[where] * old.any(1, keepdim=True)
        s1 = torch.maximum(s0, x.abs().amax((1, 3)) / 127.0)
        over = s1.masked_fill(s1 == 0, 1.0)[:, None, :, None]
        was = codes[where].transpose(2, 3) if turned else codes[where]
        was = was.transpose(1, 2).float()
        again = (s1 > s0)[:, None, :, None]
        kept = torch.where(again, (was * s0[:, None, :, None] / over).round(), was)
        put = (x / over).round().clamp(-127.0, 127.0)
        now = torch.where(fresh[:, :, None, None], put,
                          torch.where(old[:, :, None, None], kept, was))
        now = now.to(torch.int8).transpose(1, 2)
        codes[where] = now.transpose(2, 3) if turned else now
        scale[where] = s1
    first, count = _touched(c)
    for b, (lo, n, to) in enumerate(zip(first, count, _sums(count))):
        ids = s["table"][b, lo // page:(lo + n - 1) // page + 1].long()
        k = (s["k"][ids].float() * s["k_scale"][ids][:, :, None, None]).transpose(1, 2)
        v = (s["v"][ids].float() * s["v_scale"][ids][:, :, None, None]).permute(0, 3, 1, 2)
        s["read_k"][to:to + n] = k.flatten(0, 1)[:n]
        s["read_v"][to:to + n] = v.flatten(0, 1)[:n]
    return {"k": s["read_k"], "v": s["read_v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ---- what a pass cannot do without --------------------------------------------------------

_MX4_BYTES = 17.0 / 32   # a value's code and its share of the block's exponent


def work(case):
    c = case
    if c["path"] == "codes":
        n = float(c["rows"]) * c["width"]
        return {"bytes": n * ((4 if c["wide"] else 2) + 2 * _MX4_BYTES + 2), "flops": 6.0 * n}
    if c["path"] == "rope":
        heads = float(c["tokens"]) * (c["heads"] + c["kv_heads"])
        tables = 8.0 * c["rotated"] / 2 * (c["heads"] if c["per_head"] else 1)
        return {"bytes": 4.0 * heads * c["dim"] + 4.0 * c["tokens"] * c["axes"] + tables,
                "flops": 3.0 * heads * c["rotated"]}
    if c["path"] == "append":
        put, got = (float(sum(n)) * c["kv_heads"] * c["dim"]
                    for n in (_ints(c["new"]), _touched(c)[1]))
        # bf16 keys and values in, codes out; codes in, bf16 out
        return {"bytes": 6.0 * put + 6.0 * got, "flops": 11.0 * put + 2.0 * got}
    t, w = float(c["tokens"]), float(c["width"])
    moved, flops = 0.0, 0.0
    if c["path"] in ("norm", "normed"):
        stream = 4.0 if c["wide"] else 2.0
        moved = t * w * stream * (2 if c["branch"] else 1) + (2.0 * t * w if c["branch"] else 0.0)
        if c["modulated"]:
            moved += 2.0 * c["mod_rows"] * w * (3 if c["branch"] else 2)
            moved += 4.0 * t if c["mapped"] else 0.0
        flops = t * w * 10.0
        if c["path"] == "norm":
            return {"bytes": moved + 2.0 * t * w, "flops": flops}
    else:
        moved = 2.0 * t * w
    n = float(c["out"])
    return {"bytes": moved + _MX4_BYTES * n * w + 2.0 * t * n, "flops": flops + 2.0 * t * n * w}


# ---- the same in 64 bits -------------------------------------------------------------------

def _exact_mx4(x):
    """Coding as the format defines it: exponent floor(log2 of the largest), steps of a half, one or
    two units by the magnitude's binade."""
    rows, width = x.shape
    b = x.double().reshape(rows, width // 32, 32)
    top = b.abs().max(2, keepdim=True)[0]
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.full_like(top, 2.0 ** -149)))) - 2
    unit = torch.pow(torch.full_like(e, 2.0), e.clamp(-127, 127))
    v = b / unit
    step = 0.5 + 0.5 * (v.abs() >= 2) + 1.0 * (v.abs() >= 4)
    q = torch.round(v / step) * step
    return (q.clamp(-6, 6) * unit).reshape(rows, width)


def _exact_weight(s):
    out = []
    for half in (s["codes"] % 16, s["codes"] // 16):
        sign = 1.0 - 2.0 * (half // 8).double()
        e, m = ((half % 8) // 2).double(), (half % 2).double()
        out.append(sign * torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1), m / 2))
    w = torch.stack(out, -1).reshape(len(s["codes"]), -1)
    return w * torch.pow(2.0, s["exps"].double() - 127).repeat_interleave(32, 1)


def _exact_product(s, c, x):
    y = x @ _exact_weight(s).t()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if c["gelu"]:
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def _exact_norm(s, c):
    def scaled(x):
        if c["layer"]:
            x = x - x.sum(1, keepdim=True) / c["width"]
        return x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / c["width"] + _EPS)

    if s["rows"] is not None:
        row = s["rows"].long()
    else:
        row = torch.arange(c["tokens"], device="cuda") // max(1, c["tokens"] // c["mod_rows"])
    x = s["x"].double()
    if s["y"] is not None:
        u = s["y"].double()
        if s["after"] is not None:
            u = scaled(u) * s["after"].double()
        if s["gate"] is not None:
            u = u * s["gate"].double()[row]
        x = x * c["alpha"] + u
    h = scaled(x)
    if s["weight"] is not None:
        h = h * s["weight"].double()
    if s["scale"] is not None:
        h = h * (s["scale"].double()[row] + 1) + s["shift"].double()[row]
    return h, x


def _exact_rotate(x, at, freqs, which, side):
    """Channel by channel pair, as complex numbers."""
    out = x.double().clone()
    pairs = freqs.shape[1]
    for p in range(pairs):
        i, j = (2 * p, 2 * p + 1) if side else (p, p + pairs)
        angle = at.double()[:, which[:, p].long()] * freqs[:, p].double()
        turn = torch.polar(torch.ones_like(angle), angle)
        z = torch.complex(x[:, :, i].double(), x[:, :, j].double()) * turn
        out[:, :, i], out[:, :, j] = z.real, z.imag
    return out


def _exact_append(s, c):
    """Page by page, each quotient in 64 bits and then in 32: the definition's own steps (a quotient
    of two 32-bit numbers rounds the same through 64 bits)."""
    page, table = c["page"], s["table"].tolist()
    first, count = _touched(c)
    total = sum(count)
    got = {n: torch.empty((total, c["kv_heads"], c["dim"]), dtype=torch.float64, device="cuda")
           for n in "kv"}
    scales = {n: s[n + "_scale"].double() for n in "kv"}
    f32 = lambda x: x.float().double()  # noqa: E731
    to, cu = _sums(count), _sums(_ints(c["new"]))
    for b, (a, n) in enumerate(zip(_ints(c["start"]), _ints(c["new"]))):
        at = torch.arange(a, a + n, device="cuda")[:, None]
        keys = _exact_rotate(s["new_k"][cu[b]:cu[b + 1]], at, s["freqs"], s["which"],
                             c["pairs_side"]).bfloat16()
        for p in range(a // page, (a + n - 1) // page + 1):
            lo, hi = max(a, p * page), min(a + n, (p + 1) * page)
            pid, kept = table[b][p], lo - p * page
            for name in "kv":
                x = (keys if name == "k" else s["new_v"][cu[b]:cu[b + 1]])[lo - a:hi - a].double()
                was = s[name][pid] if name == "k" else s[name][pid].transpose(1, 2)
                was = was[:, :kept].transpose(0, 1).double()
                s0 = scales[name][pid] if kept else torch.zeros_like(scales[name][pid])
                s1 = torch.maximum(s0, f32(x.abs().amax((0, 2)) / 127))
                per = torch.where(s1 > 0, s1, 1.0)[:, None]
                was = torch.where((s1 > s0)[:, None], f32(f32(was * s0[:, None]) / per).round(), was)
                codes = torch.cat([was, f32(x / per).round().clamp(-127, 127)])
                where = to[b] + p * page - first[b]
                got[name][where:where + len(codes)] = codes * s1[:, None]
                scales[name][pid] = s1
    return {"k": got["k"], "v": got["v"], "k_scale": scales["k"], "v_scale": scales["v"]}


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["path"] == "codes":
        return {"out": _exact_mx4(s["x"])}
    if c["path"] == "linear":
        return {"out": _exact_product(s, c, _exact_mx4(s["x"]))}
    if c["path"] == "rope":
        return {n: _exact_rotate(s[n], s["at"], s["freqs"], s["which"], c["pairs_side"])
                for n in "qk"}
    if c["path"] == "append":
        return _exact_append(s, c)
    h, x = _exact_norm(s, c)
    out = h if c["path"] == "norm" else _exact_product(s, c, _exact_mx4(h))
    return {"out": out} if s["y"] is None else {"out": out, "x": x}
