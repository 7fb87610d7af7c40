"""examples/block_layer.py: a block in 4 bits over prompts and captured tokens, and each of its stages
against 64 bits from what the stage before it gave."""
import importlib.util
import os
import runpy
import sys

import numpy as np
import pytest
import torch

import attn_ref
import mx4_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PATH = os.path.join(ROOT, "examples", "block_layer.py")


def test_replayed_steps_are_the_eager_ones(pkg, dev, monkeypatch, capsys):
    say("block layer example")
    monkeypatch.setattr(sys, "argv", ["block_layer.py", "--tokens", "12", "--check"])
    runpy.run_path(PATH, run_name="__main__")
    assert "12 decoded each" in capsys.readouterr().out


def _f64(t):
    return t.double().cpu().numpy()


def _value(q):
    return ref.values(*ref.download(q))


def _codes_close(q, h, mag):
    """Codes of values within f32's roundings of h."""
    codes, scales = ref.download(q)
    near = [ref.code(h + s * ref.F32_SHARE * mag) for s in (-1, 0, 1)]
    sure = (near[0][1] == near[1][1]) & (near[1][1] == near[2][1])
    firm = np.repeat(sure, 32, 1) & (near[0][0] == near[1][0]) & (near[1][0] == near[2][0])
    assert firm.mean() > 0.9 and (codes == near[1][0])[firm].all()


def _norm_of(x, y, mod, gate, shift, scale):
    m = [None if i is None else mod[i:i + 1] for i in (gate, shift, scale)]
    row = np.zeros(len(x), int)
    return ref.block_norm(x, y, None, m[0], None, m[2], m[1], row, False, 1e-6, 1.0)


def _stream(got, want, mag):
    err = np.abs(_f64(got) - want) - (2.0 ** -23 * np.abs(want) + ref.F32_SHARE * mag)
    assert float(err.max()) <= 0, float(err.max())


def _check_block(block, x, k):
    """The stages around the attention."""
    s, mod = block.keep, _f64(block.mod[0])
    h, _, mag, _ = _norm_of(_f64(x), None, mod, None, 0, 1)
    _codes_close(s["h"], h, mag)
    ref.check_product(s["qkv"], _value(s["h"]), _value(block.qkv), None, False, "qkv")
    o = ref.values(*ref.code(_f64(s["o"].flatten(1))))
    ref.check_product(s["a"], o, _value(block.out), None, False, "out")
    h, mid, mag, mag_x = _norm_of(_f64(x), _f64(s["a"]), mod, 2, 3, 4)
    _stream(s["mid"], mid, mag_x)
    _codes_close(s["h2"], h, mag)
    ref.check_product(s["u"], _value(s["h2"]), _value(block.up), None, True, "up")
    u = ref.values(*ref.code(_f64(s["u"])))
    ref.check_product(s["f"], u, _value(block.down), None, False, "down")
    _, end, _, mag_x = _norm_of(_f64(s["mid"]), _f64(s["f"]), mod, 5, None, None)
    _stream(s["end"], end, mag_x)


def test_each_stage(pkg, dev):
    say("block layer stages")
    spec = importlib.util.spec_from_file_location("block_layer", PATH)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    block = ex.Block(pkg, gen)
    cache = pkg.KVCache.empty(8, ex.PAGE, ex.KV_HEADS, ex.DIM)
    lengths = [70, 1, 30]
    table = ex.int32([[0, 1], [2, 3], [4, 5]])
    x = torch.randn((sum(lengths), ex.HIDDEN), device="cuda", generator=gen)
    freqs, axes = block.freqs.cpu().numpy(), np.zeros((1, ex.DIM // 2), int)

    block.keep = {}
    y = block.prompt(x, lengths, cache, table)
    _check_block(block, x, None)
    s = block.keep
    pos = np.concatenate([np.arange(n) for n in lengths])[:, None]
    raw = [p.unflatten(1, (-1, ex.DIM)) for p in s["qkv"].split(ex.WIDTHS, 1)]
    rotated = []
    for name, t in (("q", raw[0]), ("k", raw[1])):
        # (the projection was rotated in place after it was kept)
        want, mag = ref.rotate(_f64(t), pos, freqs, axes, False)
        ref.check_rotated(s[name], want, mag, name)
        rotated.append(s[name])
    at = 0
    for n in lengths:
        rows = slice(at, at + n)
        want = attn_ref.attend(rotated[0][rows], rotated[1][rows], raw[2][rows], ex.DIM ** -0.5, True)
        attn_ref.check(s["o"][rows], None, want, f"prompt of {n}")
        at += n

    # one token more for each, on the cache that the prompts filled
    host = attn_ref.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    last = y[[n - 1 for n in ex.sums(lengths)[1:]]].contiguous()
    block.keep = {}
    block.token(last, cache, table, ex.int32(lengths), ex.int32([0, 1, 2, 3]), max(lengths) + 1)
    _check_block(block, last, None)
    s = block.keep
    pos = np.array(lengths)[:, None]
    raw = [p.unflatten(1, (-1, ex.DIM)) for p in s["qkv"].split(ex.WIDTHS, 1)]
    want, mag = ref.rotate(_f64(raw[0]), pos, freqs, axes, False)
    ref.check_rotated(s["q"], want, mag, "q")
    turned = torch.empty_like(raw[1].contiguous())
    pkg.rope(None, raw[1], ex.int32(lengths)[:, None], block.freqs, k_out=turned)
    host.append(table.cpu().numpy(), turned.float().cpu().numpy(), raw[2].float().cpu().numpy(),
                [0, 1, 2, 3], lengths)
    for b, n in enumerate(lengths):
        held = [torch.from_numpy(host.values(i, table[b].cpu().numpy(), 0, n + 1)) for i in (0, 1)]
        want = attn_ref.attend(s["q"][b:b + 1], *held, ex.DIM ** -0.5, True)
        attn_ref.check(s["o"][b:b + 1], None, want, f"token after {n}")
