"""attention_cached where the cache's value scales are small or far apart, and over contexts whose
parts are many: against 64 bits of the same codes."""
import numpy as np
import pytest
import torch

import attn_ref
from gpu_util import say

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(seed, *shape, std=1.0):
    return (torch.randn(shape, device="cuda", generator=_gen(seed)) * std).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(pkg, seed, pages, page, heads, dim):
    g = _gen(seed)
    c = pkg.KVCache.empty(pages, page, heads, dim)
    for t in (c.k, c.v):
        t.copy_((torch.randn(t.shape, device="cuda", generator=g) * 36).round().clamp(-127, 127))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, device="cuda", generator=g) * 0.03 + 0.005)
    return c


def _table(seed, lens, page):
    n = [-(-x // page) for x in lens]
    order = np.random.default_rng(seed).permutation(sum(n))
    t = np.zeros((len(lens), max(n)), np.int32)
    for b, at in enumerate(np.cumsum([0] + n[:-1])):
        t[b, :n[b]] = order[at:at + n[b]]
    return t, sum(n)


def _attend(pkg, c, table, lens, q, q_len, causal=True):
    need = pkg.attention_cached_workspace(len(lens), q_len, q.shape[1], c.kv_heads, c.head_dim, max(lens))
    ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")   # a NaN in every word
    out = torch.full_like(q, float("nan"))
    z = torch.full(q.shape[:2], float("nan"), device="cuda")
    pkg.attention_cached(c, _i32(table), _i32(lens), q, out, q_len, max(lens), ws, causal=causal, lse=z)
    torch.cuda.synchronize()
    return out, z, need // (len(q) * q.shape[1] * (c.head_dim + 2) * 4)


def _close(c, table, n, q, b, q_len, out, z, heads=None):
    """One sequence within attn_ref's bound and half a unit of bf16's smallest values (2^-133) with as
    much again for f32's own."""
    rows = slice(b * q_len, (b + 1) * q_len)
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    k, v = (torch.from_numpy(ref.values(w, table[b], 0, n)) for w in (0, 1))
    want, zw, mag, size = attn_ref.attend(q[rows], k, v, c.head_dim ** -0.5, True)
    err = (out[rows].cpu().double() - want).abs()
    assert bool((err <= attn_ref.OUT_BOUND * mag + 2.0 ** -133).all()), \
        float((err / (attn_ref.OUT_BOUND * mag + 2.0 ** -133)).max())
    d = (z[rows].cpu().double() - zw).abs() - attn_ref.LSE_BOUND * (1 + size)
    assert float(d.max()) <= 0


# tokens, queries, heads, kv heads, width: one, two and four row tiles, one part and several
FORMS = [(300, 1, 4, 1, 64), (300, 1, 4, 1, 128), (200, 8, 4, 1, 128), (200, 12, 4, 1, 64),
         (5000, 1, 4, 1, 128), (5000, 1, 4, 1, 64)]


@pytest.mark.parametrize("power", [-90, -112, -114, -120, -126, -130, -133])
@pytest.mark.parametrize("n,q_len,heads,kv_heads,dim", FORMS)
def test_small_value_scales(pkg, dev, power, n, q_len, heads, kv_heads, dim):
    """Scales down to those that appending makes of bf16's smallest normal values (2^-126 / 127)."""
    table, pages = _table(1, [n], 64)
    c = _cache(pkg, 2, pages, 64, kv_heads, dim)
    c.v.copy_(c.v.abs())          # means of the values' size
    c.v_scale.fill_(2.0 ** power)
    q = _randn(3, q_len, heads, dim)
    say(f"attention_cached value scales 2^{power}, {n} tokens, q_len {q_len} x {dim}")
    out, z, _ = _attend(pkg, c, table, [n], q, q_len)
    _close(c, table, n, q, 0, q_len, out, z)


@pytest.mark.parametrize("n,q_len,heads,kv_heads,dim", FORMS)
def test_value_scales_at_both_ends_of_the_range(pkg, dev, n, q_len, heads, kv_heads, dim):
    """Zero, denormal, small, ordinary and the largest scales in one sequence; then the blocks that
    the queries look at hold zeros or tiny values and all others count for 2^-100 or less."""
    table, pages = _table(4, [n], 64)
    c = _cache(pkg, 5, pages, 64, kv_heads, dim)
    for p in range(pages):
        c.v_scale[table[0, p]] = (0.0, 2.0 ** -140, 2.0 ** -100, 0.02)[p % 4]
    q = _randn(6, q_len, heads, dim).abs() + 0.1
    say(f"attention_cached scales of all sizes, {n} tokens, q_len {q_len} x {dim}")
    out, z, _ = _attend(pkg, c, table, [n], q, q_len)
    _close(c, table, n, q, 0, q_len, out, z)
    for tiny in (0.0, 2.0 ** -140, 2.0 ** -60):
        for loud in (0, pages - 1):
            c.k.fill_(0)
            c.k[table[0, loud]] = 127        # logits of about 80 there, 0 elsewhere
            c.k_scale.fill_(80.0 / 127.0 / dim ** 0.5)
            c.v_scale.fill_(1.0)
            c.v_scale[table[0, loud]] = tiny
            x = torch.ones_like(q)
            out, z, _ = _attend(pkg, c, table, [n], x, q_len)
            assert bool(torch.isfinite(out).all())
            _close(c, table, n, x, 0, q_len, out, z)


def test_appended_small_values_are_attended_to(pkg, dev):
    """What kv_append makes of small values, kv_read and attention_cached give back alike."""
    n, dim = 130, 128
    table, pages = _table(7, [n], 64)
    c = _cache(pkg, 8, pages, 64, 2, dim)
    k = _randn(9, n, 2, dim)
    v = ((1.0 + torch.rand((n, 2, dim), device="cuda", generator=_gen(10))) * 2.0 ** -125).to(torch.bfloat16)
    pkg.kv_append(c, _i32(table), k, v, _i32([0, n]), _i32([0]))
    q = _randn(11, 1, 4, dim)
    say("attention_cached over appended small values")
    out, z, _ = _attend(pkg, c, table, [n], q, 1)
    _close(c, table, n, q, 0, 1, out, z)
    assert bool((out.float() > 2.0 ** -126).all())


# keys, batch, heads, kv heads, width: both sides of 20 rounds of 256 tokens with every CU's work
# there, and parts beyond a wave's lanes
LONG = [([5120] * 2 + [300] * 62, 8, 8, 64), ([5121] * 2 + [300] * 62, 8, 8, 64),
        ([17000], 2, 1, 128), ([131072], 1, 1, 128), ([131072], 2, 1, 64), ([40000, 131, 9000], 4, 2, 64)]


@pytest.mark.parametrize("lens,heads,kv_heads,dim", LONG)
def test_long_contexts_in_many_parts(pkg, dev, lens, heads, kv_heads, dim):
    page = 64
    table, pages = _table(12, lens, page)
    c = _cache(pkg, 13, pages, page, kv_heads, dim)
    q = _randn(14, len(lens), heads, dim)
    say(f"attention_cached long {lens[:3]} heads {heads}/{kv_heads} x {dim}")
    out, z, parts = _attend(pkg, c, table, lens, q, 1)
    assert parts >= (65 if lens[0] >= 17000 and len(lens) == 1 else 0)
    share = heads // kv_heads
    for b in (0, 1, len(lens) - 1):
        if b >= len(lens):
            continue
        ids = torch.from_numpy(table[b, :-(-lens[b] // page)]).cuda().long()
        k = (c.k[ids].double() * c.k_scale[ids].double()[:, :, None, None]).transpose(1, 2)
        v = (c.v[ids].double() * c.v_scale[ids].double()[:, :, None, None]).permute(0, 3, 1, 2)
        k, v = (x.reshape(-1, kv_heads, dim)[:lens[b]] for x in (k, v))
        for h in range(heads):
            x = k[:, h // share] @ q[b, h].double() * dim ** -0.5
            top = torch.logsumexp(x, 0)
            w = torch.exp(x - top)
            want, mag = w @ v[:, h // share], w @ v[:, h // share].abs()
            err = (out[b, h].double() - want).abs() - attn_ref.OUT_BOUND * mag
            assert float(err.max()) <= 0, (b, h)
            size = (k[:, h // share].abs() @ q[b, h].double().abs()).max() * dim ** -0.5
            assert abs(float(z[b, h] - top)) <= attn_ref.LSE_BOUND * (1 + float(size)), (b, h)
