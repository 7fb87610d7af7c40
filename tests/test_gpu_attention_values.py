"""Prompt attention (ltx25_attention, ltx25_attention_split) at the ends of the values' range:
infinities and NaN that a row sees or does not see, in one part of the keys and in several."""
import pytest
import torch

import attn_ref
from gpu_util import say

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def _randn(seed, *shape, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def _attend(pkg, q, k, v, causal, parts=True, scale=0.0):
    """One sequence. `parts` false: a stream is named, so that the binding does not split."""
    out = torch.full_like(q, NAN)
    z = torch.full(q.shape[:2], NAN, device="cuda")
    stream = None if parts else torch.cuda.current_stream().cuda_stream
    pkg.attention(q, k, v, out, causal=causal, scale=scale, lse=z, stream=stream)
    torch.cuda.synchronize()
    return out, z


def _parts(pkg, q, k):
    need = pkg.attention_workspace(q.shape[1], k.shape[1], q.shape[2], 1, len(q), len(k))
    return need // (q.shape[0] * q.shape[1] * (q.shape[2] + 2) * 4)


def _bits(t):
    return t.contiguous().view(torch.int16)


# keys and heads: 4 to 50 parts at width 128, 6 to 42 at 64 (from 800 keys on), multiples of 8 and
# 16 among them
@pytest.mark.parametrize("n,heads,kv_heads", [(520, 2, 1), (600, 2, 1), (800, 2, 1), (1000, 2, 1),
                                              (1100, 2, 1), (1500, 2, 1), (2000, 2, 1),
                                              (3000, 8, 2), (4000, 8, 2), (16000, 8, 2)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("split", [True, False])
def test_seen_infinities_stay_infinities(pkg, dev, n, heads, kv_heads, dim, split):
    """Every row sees them: their channels hold them with their sign, wherever among the keys they
    lie; both signs, or a NaN, make a NaN; the other channels keep their bits."""
    q, k, v = _randn(1, 5, heads, dim), _randn(2, n, kv_heads, dim), _randn(3, n, kv_heads, dim)
    if split and n >= 800:
        assert _parts(pkg, q, k) >= 2
    clean, _ = _attend(pkg, q, k, v, False, split)
    assert bool(torch.isfinite(clean).all())
    v[n - 1, :, 5], v[n - 1, :, 6], v[0, :, 7], v[n // 2, :, 9] = INF, -INF, INF, -INF
    v[0, :, 11], v[n - 1, :, 11] = INF, -INF
    v[n - 1, :, 13] = NAN
    say(f"attention seen infinities {n} heads {heads}/{kv_heads} x {dim} in {_parts(pkg, q, k)} parts, "
        f"split {split}")
    out, z = _attend(pkg, q, k, v, False, split)
    assert bool(torch.isfinite(z).all())
    for channel, want in ((5, INF), (6, -INF), (7, INF), (9, -INF)):
        assert bool((out[..., channel] == want).all()), channel
    assert bool(torch.isnan(out[..., [11, 13]]).all())
    rest = torch.ones(dim, dtype=torch.bool)
    rest[[5, 6, 7, 9, 11, 13]] = False
    assert torch.equal(_bits(out[..., rest]), _bits(clean[..., rest]))


@pytest.mark.parametrize("dim", [64, 128])
def test_seen_infinity_in_a_part_that_hardly_counts(pkg, dev, dim):
    """A softmax's weights are positive, however small: the infinity of a key whose part's weight
    is too small for f32 beside the others' is the row's."""
    n = 1100
    q = torch.ones(3, 2, dim, dtype=torch.bfloat16, device="cuda")
    k, v = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device="cuda"), _randn(4, n, 1, dim)
    k[:64] = 2.0            # logits 2 * dim and 0 at scale 1: e^-128 or e^-256 of the first ones'
    v[n - 1, :, 5], v[n - 1, :, 6] = INF, -INF
    say(f"attention infinity in a part that hardly counts x {dim}")
    assert _parts(pkg, q, k) >= 2
    out, _ = _attend(pkg, q, k, v, False, True, 1.0)
    assert bool((out[..., 5] == INF).all()) and bool((out[..., 6] == -INF).all())
    assert bool(torch.isfinite(out[..., 7:]).all())


# queries, heads, kv heads, width: the 8-wave form, the 4-wave form, and the keys in parts
COSTS = [(8192, 32, 8, 128), (8192, 32, 8, 64), (2048, 1, 1, 128), (2048, 1, 1, 64)]


@pytest.mark.parametrize("n,heads,kv_heads,dim", COSTS)
def test_a_value_that_rows_do_not_see_costs_them_little(pkg, dev, n, heads, kv_heads, dim):
    """One value that is not finite in the last token of a causal prompt: the rows that share its
    tile and do not see it are right, and the call is not much slower (the rows of one tile of 64
    walk their keys once more; 3 times a clean call and 3 ms leave room for a busy card)."""
    q, k, v = _randn(5, n, heads, dim), _randn(6, n, kv_heads, dim), _randn(7, n, kv_heads, dim)
    clean, zc = _attend(pkg, q, k, v, True)
    assert bool(torch.isfinite(clean).all()) and bool(torch.isfinite(zc).all())

    def took(value):
        times = []
        for _ in range(3):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            pkg.attention(q, k, value, out, causal=True)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    out = torch.empty_like(q)
    before = took(v)
    for bad in (NAN, INF):
        w = v.clone()
        w[n - 1, :, 3] = bad
        say(f"attention one value {bad} in the last of {n} tokens, heads {heads}/{kv_heads} x {dim}")
        after = took(w)
        rest = torch.ones(dim, dtype=torch.bool)
        rest[3] = False
        assert torch.equal(_bits(out[:, :, rest]), _bits(clean[:, :, rest]))
        assert bool(torch.isnan(out[n - 1, :, 3]).all() if bad != bad else (out[n - 1, :, 3] == bad).all())
        for i in (n - 64, n - 33, n - 32, n - 2):
            for h in (0, heads - 1):
                g = h // (heads // kv_heads)
                want = attn_ref.attend(q[i:i + 1, h:h + 1], k[:i + 1, g:g + 1],
                                       w[:i + 1, g:g + 1], dim ** -0.5, False)
                attn_ref.check(out[i:i + 1, h:h + 1], None, want, f"row {i} head {h}")
        assert after < 3.0 * before + 3.0, (after, before)


def _even(seed, *shape):
    """Values from 1 to 2 of one sign, so that a mean of them is of their size."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return 1.0 + torch.rand(shape, device="cuda", generator=g)


def _check_small(q, k, v, out, rows, scale, what):
    """attn_ref's bound for the roundings to 8 bits, and half a unit of bf16's smallest values (2^-133)
    with as much again for f32's own."""
    heads, kv_heads = q.shape[1], k.shape[1]
    for i in rows:
        for h in (0, heads - 1):
            g = h // (heads // kv_heads)
            ref, _, mag, _ = attn_ref.attend(q[i:i + 1, h:h + 1], k[:, g:g + 1], v[:, g:g + 1], scale,
                                             False)
            err = (out[i:i + 1, h:h + 1].cpu().double() - ref).abs()
            assert bool((err <= attn_ref.OUT_BOUND * mag + 2.0 ** -133).all()), (what, i, h)


# queries, keys, heads, kv heads: in parts, the 4-wave form, the 8-wave form
SMALL = [(5, 1500, 2, 1), (300, 300, 2, 1), (4200, 4200, 32, 8)]


@pytest.mark.parametrize("power", [-90, -100, -112, -120, -125])
@pytest.mark.parametrize("nq,nk,heads,kv_heads", SMALL)
@pytest.mark.parametrize("dim", [64, 128])
def test_small_values_keep_their_bits(pkg, dev, power, nq, nk, heads, kv_heads, dim):
    """Values down to the smallest normal ones, under logits that rise so that the maximum lags."""
    q = torch.ones(nq, heads, dim, dtype=torch.bfloat16, device="cuda")
    k = torch.linspace(0, 5, nk, device="cuda")[:, None, None].expand(nk, kv_heads, dim) / dim
    k = k.to(torch.bfloat16)
    v = (_even(8, nk, kv_heads, dim) * 2.0 ** power).to(torch.bfloat16)
    say(f"attention values of 2^{power}, {nq} x {nk} heads {heads}/{kv_heads} x {dim}")
    out, z = _attend(pkg, q, k, v, False, True, 1.0)
    _check_small(q, k, v, out, (0, nq // 2, nq - 1), 1.0, power)


@pytest.mark.parametrize("nq,nk,heads,kv_heads", SMALL)
@pytest.mark.parametrize("dim", [64, 128])
def test_small_values_beside_the_largest_and_beside_unseen_ones(pkg, dev, nq, nk, heads, kv_heads, dim):
    """One row's channels at both ends of the range, and a small channel whose last token holds an
    infinity that only the last query sees."""
    q, k = _randn(9, nq, heads, dim), _randn(10, nk, kv_heads, dim)
    v = _even(11, nk, kv_heads, dim)
    v[..., :8] *= 2.0 ** 126
    v[..., 8:] *= 2.0 ** -122
    v = v.to(torch.bfloat16)
    say(f"attention values at both ends, {nq} x {nk} heads {heads}/{kv_heads} x {dim}")
    out, _ = _attend(pkg, q, k, v, False)
    assert bool(torch.isfinite(out).all())
    _check_small(q, k, v, out, (0, nq // 2, nq - 1), dim ** -0.5, "both ends")
    if nq == nk:
        v[nk - 1, :, 9] = INF
        out, _ = _attend(pkg, q, k, v, True)
        assert bool((out[nq - 1, :, 9] == INF).all()) and bool(torch.isfinite(out[:nq - 1]).all())
        for i in (nq - 40, nq - 2):
            _check_small(q, k[:i + 1], v[:i + 1], out, (i,), dim ** -0.5, "beside an unseen infinity")


@pytest.mark.parametrize("stride", [513, 532, 1 << 23, 0])
def test_one_token_of_any_stride(pkg, dev, stride):
    """A tensor of one token has no next one: what its stride says does not matter."""
    q, k, v = (_randn(s, 1, h, 64).as_strided((1, h, 64), (stride, 64, 1))
               for s, h in ((12, 8), (13, 2), (14, 2)))
    out = torch.full((1, 8, 64), NAN, dtype=torch.bfloat16, device="cuda")
    z = torch.full((1, 8), NAN, device="cuda")
    say(f"attention one token of stride {stride}")
    pkg.attention(q, k, v, out.as_strided((1, 8, 64), (stride, 64, 1)), causal=True, lse=z)
    torch.cuda.synchronize()
    attn_ref.check(out, z, attn_ref.attend(q, k, v, 64 ** -0.5, True))
