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
