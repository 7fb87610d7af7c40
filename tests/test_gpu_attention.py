"""Prompt attention (ltx25_attention) on the GPU against 64 bits, at the sizes, masks and values
where it can go wrong. The bounds are attn_ref's, from the roundings that the definition has."""
import numpy as np
import pytest
import torch

import attn_ref
from gpu_util import say

pytestmark = pytest.mark.gpu


def _randn(seed, *shape, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def _cu(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _run(pkg, q, k, v, lens_q, lens_k, causal, scale=0.0, lse=True, null_cu=False):
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device="cuda")
    z = torch.full(q.shape[:2], float("nan"), device="cuda") if lse else None
    cu = (None, None) if null_cu else (_cu(lens_q), _cu(lens_k))
    pkg.attention(q, k, v, out, *cu, causal=causal, scale=scale, lse=z)
    torch.cuda.synchronize()
    return out, z


def _verify(q, k, v, out, z, lens_q, lens_k, causal, scale=None):
    scale = scale or q.shape[2] ** -0.5
    a = b = 0
    for i, (nq, nk) in enumerate(zip(lens_q, lens_k)):
        want = attn_ref.attend(q[a:a + nq], k[b:b + nk], v[b:b + nk], scale, causal)
        attn_ref.check(out[a:a + nq], None if z is None else z[a:a + nq], want, f"sequence {i}")
        a, b = a + nq, b + nk


SHAPES = [  # queries, keys, heads, kv heads, width, causal
    ([1], [1], 1, 1, 128, True),
    ([1], [1], 1, 1, 64, False),
    ([1], [300], 8, 2, 128, True),
    ([31, 32, 33], [31, 32, 33], 4, 4, 128, True),
    ([63, 64, 65, 1], [63, 64, 65, 1], 6, 2, 64, True),
    ([127, 129], [127, 129], 5, 5, 128, True),
    ([255, 3, 257], [255, 3, 257], 2, 1, 128, True),
    ([130], [130], 7, 1, 64, True),
    ([70, 20], [70, 20], 16, 1, 128, True),
    ([40], [40], 24, 8, 128, True),
    ([50, 10, 5], [7, 10, 40], 4, 2, 128, True),       # queries that see nothing; a prefix
    ([90], [20], 8, 1, 64, True),
    ([20, 0, 5, 1], [0, 9, 5, 0], 4, 2, 128, True),    # sequences without queries, without keys
    ([20, 0, 5, 1], [0, 9, 5, 0], 4, 2, 64, False),
    ([126], [126], 16, 16, 128, False),
    ([100, 33], [17, 200], 3, 3, 128, False),          # as cross-attention
    ([33] * 70, [33] * 70, 1, 1, 64, True),            # more sequences than a wave has lanes
    ([600], [600], 2, 2, 128, True),
    ([300], [700], 8, 2, 64, True),
]


@pytest.mark.parametrize("lens_q,lens_k,heads,kv_heads,dim,causal", SHAPES)
def test_attention_against_64_bits(pkg, dev, lens_q, lens_k, heads, kv_heads, dim, causal):
    say(f"attention {lens_q[:4]} {lens_k[:4]} heads {heads}/{kv_heads} x {dim} causal={causal}")
    q = _randn(1, sum(lens_q), heads, dim)
    k, v = (_randn(s, sum(lens_k), kv_heads, dim) for s in (2, 3))
    out, z = _run(pkg, q, k, v, lens_q, lens_k, causal)
    _verify(q, k, v, out, z, lens_q, lens_k, causal)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_on_a_fused_projections_output(pkg, dev, dim):
    """q, k and v as column ranges of one tensor, out as a range of another; the rest of it
    stays."""
    lens, heads, kv_heads = [37, 90, 1], 8, 2
    y = _randn(4, sum(lens), (heads + 2 * kv_heads) * dim)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in
               y.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    wide = torch.full((sum(lens), heads * dim + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 32:32 + heads * dim].unflatten(1, (-1, dim))
    say(f"attention fused projection x {dim}")
    pkg.attention(q, k, v, out, _cu(lens), _cu(lens), causal=True)
    torch.cuda.synchronize()
    _verify(q, k, v, out, None, lens, lens, True)
    assert bool((wide[:, :32] == 7).all()) and bool((wide[:, 32 + heads * dim:] == 7).all())


def test_attention_without_lengths_is_one_sequence(pkg, dev):
    q, k, v = _randn(5, 77, 4, 128), _randn(6, 140, 4, 128), _randn(7, 140, 4, 128)
    say("attention null lengths")
    out, z = _run(pkg, q, k, v, [77], [140], False, null_cu=True)
    _verify(q, k, v, out, z, [77], [140], False)


@pytest.mark.parametrize("std,scale", [(1.0, 0.5), (8.0, 0.0), (1.0, 1e-3), (0.0, 0.0)])
def test_attention_scales_and_steep_logits(pkg, dev, std, scale):
    """Logits up to hundreds (one key takes all the weight, the running maximum jumps), nearly
    flat ones, and all-zero queries."""
    q, k, v = _randn(8, 150, 4, 128, std=std), _randn(9, 150, 2, 128, std=std), _randn(10, 150, 2, 128)
    say(f"attention std {std} scale {scale}")
    out, z = _run(pkg, q, k, v, [150], [150], True, scale)
    _verify(q, k, v, out, z, [150], [150], True, scale)


def test_attention_maximum_rising_and_falling(pkg, dev):
    """Keys ordered so that the row's maximum rises at every tile, and falls at every tile."""
    for sign in (1.0, -1.0):
        n = 700
        q = torch.ones(40, 2, 64, dtype=torch.bfloat16, device="cuda")
        ramp = sign * torch.arange(n, device="cuda").float() / 16
        k = (ramp[:, None, None] * torch.ones(1, 2, 64, device="cuda") / 64).to(torch.bfloat16)
        v = _randn(11, n, 2, 64)
        say(f"attention ramp {sign}")
        out, z = _run(pkg, q, k, v, [40], [n], False, 1.0)
        _verify(q, k, v, out, z, [40], [n], False, 1.0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_unseen_values_have_no_influence(pkg, dev, bad, dim):
    """A NaN or an infinity in keys and values of a later token, and in a neighbouring sequence:
    the rows that do not see it are what they are without it."""
    lens = [100, 70]
    q, k, v = _randn(12, 170, 4, dim), _randn(13, 170, 2, dim), _randn(14, 170, 2, dim)
    clean, zc = _run(pkg, q, k, v, lens, lens, True)
    k[90, 0], v[90, 0, 3], v[95, 1], v[100:, 1, 5] = bad, bad, bad, bad
    say(f"attention unseen {bad} x {dim}")
    out, z = _run(pkg, q, k, v, lens, lens, True)
    _verify(q[:90], k[:90], v[:90], out[:90], z[:90], [90], [90], True)
    assert bool(torch.isfinite(out[:95, 2:].float()).all())
    assert torch.equal(out[100:, :2].view(torch.int16), clean[100:, :2].view(torch.int16))
    _verify(q[:95, 2:], k[:95, 1:], v[:95, 1:], out[:95, 2:], z[:95, 2:], [95], [95], True)
    # those that do see it show it
    assert not bool(torch.isfinite(out[99, 2].float()).any())
    assert not bool(torch.isfinite(out[100:, 2:, 5].float()).any())
    assert not bool(torch.isfinite(z[90:100, :2]).all()) or bad == -float("inf")


def test_attention_repeats_bit_for_bit_on_its_stream_and_in_a_graph(pkg, dev):
    lens = [200, 5, 64]
    q, k, v = _randn(15, 269, 8, 128), _randn(16, 269, 2, 128), _randn(17, 269, 2, 128)
    cu = _cu(lens)
    want, _ = _run(pkg, q, k, v, lens, lens, True)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    say("attention on a side stream")
    with torch.cuda.stream(side):
        pkg.attention(q, k, v, out, cu, cu, causal=True)
    side.synchronize()
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.attention(q, k, v, out, cu, cu, causal=True)
    for rep in range(3):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        say(f"attention replay {rep}")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_attention_lengths_that_do_not_fit_are_cut(pkg, dev):
    """Cumulative lengths past the tensors, negative or falling: nothing outside is read or
    written, and a sequence within them is still right."""
    guard = torch.full((300, 2, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    out = guard[100:200]
    q, k, v = _randn(18, 100, 2, 128), _randn(19, 100, 2, 128), _randn(20, 100, 2, 128)
    for cu in ([0, 60, 4000], [-7, 60, 100], [0, 60, 30]):
        c = torch.tensor(cu, dtype=torch.int32, device="cuda")
        say(f"attention lengths {cu}")
        pkg.attention(q, k, v, out, c, c, causal=True)
        torch.cuda.synchronize()
        assert bool((guard[:100] == 5).all()) and bool((guard[200:] == 5).all())
        _verify(q, k, v, out, None, [60], [60], True)


def test_attention_far_offsets(pkg, dev):
    """Keys past 2^31 elements from the tensor's start (4.3 GB), queries and outputs too."""
    stride, n = 8192, 270000
    big = torch.empty((n, stride), dtype=torch.bfloat16, device="cuda")
    big[-80:] = _randn(21, 80, stride)
    q = big[:, :256].unflatten(1, (2, 128))
    k = big[:, 256:512].unflatten(1, (2, 128))
    v = big[:, 512:768].unflatten(1, (2, 128))
    out = big[:, 1024:1280].unflatten(1, (2, 128))
    cu = torch.tensor([n - 70, n], dtype=torch.int32, device="cuda")
    say("attention far offsets")
    pkg.attention(q, k, v, out, cu, cu, causal=True)
    torch.cuda.synchronize()
    _verify(q[-70:], k[-70:], v[-70:], out[-70:], None, [70], [70], True)


def test_attention_empty_calls_do_nothing(pkg, dev):
    e = torch.empty((0, 2, 128), dtype=torch.bfloat16, device="cuda")
    k = _randn(22, 3, 2, 128)
    pkg.attention(e, k, k, e, causal=True)
    out = torch.full((2, 2, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    z = torch.zeros((2, 2), device="cuda")
    pkg.attention(k[:2], e, e, out, causal=False, lse=z)     # no keys: zeros, -inf
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((z == -float("inf")).all())


# long enough for the form whose waves take turns (from 2048 keys a sequence and 512 of its
# workgroups on): queries, keys, heads, kv heads, causal
LONG = [
    ([4097], [4097], 32, 8, True),
    ([4200], [4200], 32, 32, False),
    ([2600], [3000], 56, 8, True),                    # 2^3 heads of 7 do not divide: one at a time
    ([1, 2500, 3900], [2100, 2500, 4100], 24, 3, True),
    ([3000, 2000], [1500, 2700], 32, 8, True),        # queries that see nothing
    ([8200], [2048], 16, 16, False),
]


@pytest.mark.parametrize("lens_q,lens_k,heads,kv_heads,causal", LONG)
def test_attention_long_against_64_bits(pkg, dev, lens_q, lens_k, heads, kv_heads, causal):
    """Rows at the ends, on both sides of tile and workgroup edges, and spread between."""
    say(f"attention long {lens_q} {lens_k} heads {heads}/{kv_heads} causal={causal}")
    q = _randn(31, sum(lens_q), heads, 128, std=1.5)
    k, v = (_randn(s, sum(lens_k), kv_heads, 128) for s in (32, 33))
    out, z = _run(pkg, q, k, v, lens_q, lens_k, causal)
    again, _ = _run(pkg, q, k, v, lens_q, lens_k, causal)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    assert not bool(torch.isnan(out).any()) and not bool(torch.isnan(z).any())
    kc, vc = k.cpu(), v.cpu()
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        edges = [0, 1, 31, 32, 63, 64, 65, 255, 256, 1000, n // 2, n - 257, n - 65, n - 2, n - 1]
        for i in sorted({e for e in edges if 0 <= e < n}):
            see = max(0, min(m, i + 1 + m - n)) if causal else m
            row = slice(a + i, a + i + 1)
            want = attn_ref.attend(q[row], kc[b:b + see], vc[b:b + see], 128 ** -0.5, False)
            attn_ref.check(out[row], z[row], want, f"row {i} of {n}")
        a, b = a + n, b + m


def test_attention_long_unseen_values_have_no_influence(pkg, dev):
    n = 4200
    q, k, v = _randn(34, n, 32, 128), _randn(35, n, 8, 128), _randn(36, n, 8, 128)
    clean, _ = _run(pkg, q, k, v, [n], [n], True)
    k[3001, 2], v[3001, 2, 7], v[4150, 5] = float("nan"), float("inf"), float("nan")
    say("attention long unseen")
    out, _ = _run(pkg, q, k, v, [n], [n], True)
    same = torch.ones(n, 32, dtype=torch.bool)
    same[3001:, 8:12], same[4150:, 20:24] = False, False
    # rows beside a bad value in a tile are computed again, one key at a time: within the bounds
    # of the clean ones, not the same bits
    near = torch.zeros_like(same)
    near[2944:3001, 8:12], near[4096:4150, 20:24] = True, True
    bits = (out.view(torch.int16) == clean.view(torch.int16)).all(2).cpu()
    assert bool(bits[same & ~near].all())
    for i, h in ((2990, 8), (3000, 11), (4149, 20), (4097, 23)):
        want = attn_ref.attend(q[i:i + 1, h:h + 1], k[:i + 1, h // 4:h // 4 + 1],
                               v[:i + 1, h // 4:h // 4 + 1], 128 ** -0.5, False)
        attn_ref.check(out[i:i + 1, h:h + 1], None, want, f"row {i} head {h}")
    assert not bool(torch.isfinite(out[3001:, 8:12]).any())
    assert not bool(torch.isfinite(out[4150:, 20:24]).any())


def test_attention_rising_logits_over_many_tiles(pkg, dev):
    """A maximum that rises by more than 2^12 in the weights again and again, in both forms."""
    for n, heads in ((900, 2), (4100, 32)):
        q = torch.ones(n, heads, 128, dtype=torch.bfloat16, device="cuda")
        ramp = torch.arange(n, device="cuda").float() * 0.4
        k = (ramp[:, None, None] * torch.ones(1, 2, 128, device="cuda") / 128).to(torch.bfloat16)
        v = _randn(37, n, 2, 128)
        say(f"attention rising {n}")
        out, z = _run(pkg, q, k, v, [n], [n], True, 1.0)
        for i in (0, 5, 64, 200, 777, n - 1):
            want = attn_ref.attend(q[i:i + 1], k[:i + 1], v[:i + 1], 1.0, False)
            attn_ref.check(out[i:i + 1], z[i:i + 1], want, f"row {i} of {n}")


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_several_hundred_sequences(pkg, dev, dim):
    rng = np.random.default_rng(38)
    lens = [int(n) for n in rng.integers(0, 6, 600)]
    lens[300], lens[577] = 70, 40
    q, k, v = _randn(39, sum(lens), 2, dim), _randn(40, sum(lens), 1, dim), _randn(41, sum(lens), 1, dim)
    say(f"attention of 600 sequences x {dim}")
    out, z = _run(pkg, q, k, v, lens, lens, True)
    _verify(q, k, v, out, z, lens, lens, True)


@pytest.mark.parametrize("n,heads,kv_heads,dim", [(300, 2, 1, 64), (300, 2, 2, 128), (4200, 32, 8, 128)])
def test_attention_values_near_the_end_of_f32(pkg, dev, n, heads, kv_heads, dim):
    """Values up to 2^126 under logits that rise slowly: each row's mean is finite, though its sums
    under a maximum that lags are not."""
    q = torch.ones(n, heads, dim, dtype=torch.bfloat16, device="cuda")
    k = torch.linspace(0, 5, n, device="cuda")[:, None, None].expand(n, kv_heads, dim) / dim
    k, v = k.to(torch.bfloat16), _randn(38, n, kv_heads, dim)
    v[:, 0] = (v[:, 0].float().clamp(-2, 2) * 2.0 ** 125).to(torch.bfloat16)
    say(f"attention large values {n}")
    out, z = _run(pkg, q, k, v, [n], [n], False, 1.0)
    for i in (0, n - 1):
        for h in (0, heads - 1):
            g = h // (heads // kv_heads)
            want = attn_ref.attend(q[i:i + 1, h:h + 1], k[:, g:g + 1], v[:, g:g + 1], 1.0, False)
            attn_ref.check(out[i:i + 1, h:h + 1], z[i:i + 1, h:h + 1], want, f"row {i} head {h}")


@pytest.mark.parametrize("n,heads,kv_heads,dim", [(200, 4, 2, 64), (200, 4, 2, 128), (4200, 32, 8, 128)])
def test_attention_nan_channels_that_are_seen_and_unseen(pkg, dev, n, heads, kv_heads, dim):
    """Channels of the values that are NaN from a seen token, from an unseen one of the same tile, or
    from both: the seen ones show, the others do not, and what is beside them keeps its bits."""
    q, k, v = _randn(39, n, heads, dim), _randn(40, n, kv_heads, dim), _randn(41, n, kv_heads, dim)
    clean, _ = _run(pkg, q, k, v, [n], [n], True)
    nan, at = float("nan"), n - n % 64 - 30     # `at` lies inside a tile
    v[10, :, 3], v[at, :, 3], v[at, :, 5], v[at + 2, 0, 7] = nan, nan, nan, float("inf")
    say(f"attention nan channels {n} x {dim}")
    out, z = _run(pkg, q, k, v, [n], [n], True)
    assert bool(torch.isfinite(z).all())
    bad = torch.isnan(out)
    assert not bool(bad[:10].any()) and bool(bad[10:, :, 3].all())
    assert bool(bad[at:, :, 5].all()) and not bool(bad[:at, :, 5].any())
    share = heads // kv_heads
    assert bool(torch.isinf(out[at + 2:, :share, 7]).all())
    assert bool(torch.isfinite(out[:at + 2, :share, 7]).all())
    untouched = torch.ones(dim, dtype=torch.bool)
    untouched[[3, 5, 7]] = False
    assert torch.equal(out[..., untouched].view(torch.int16), clean[..., untouched].view(torch.int16))
    for i in (at - 1, at):
        want = attn_ref.attend(q[i:i + 1], k[:i + 1], v[:i + 1], dim ** -0.5, False)
        ok = ~torch.isnan(want[0])
        err = (out[i:i + 1].cpu().double() - want[0]).abs()[ok] - attn_ref.OUT_BOUND * want[2][ok]
        assert float(err.max()) <= 0, f"row {i}"


def test_attention_nan_everywhere_ends_soon(pkg, dev):
    """Tensors full of NaN: NaN out, and in about the time of any others."""
    n = 6000
    q, k, v = _randn(42, n, 32, 128), _randn(43, n, 8, 128), _randn(44, n, 8, 128)
    times = []
    for bad in (None, q, v, k):
        t = [x if x is not bad else torch.full_like(x, float("nan")) for x in (q, k, v)]
        out = torch.empty_like(q)
        say("attention full of NaN")
        pkg.attention(*t, out, causal=True)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        pkg.attention(*t, out, causal=True)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
        assert bool(torch.isnan(out).all()) == (bad is not None)
    assert max(times[1:]) < 20 * times[0] + 1.0, times


def _parts(pkg, heads, kv_heads, dim, batch, nq, nk):
    return pkg.attention_workspace(heads, kv_heads, dim, batch, nq, nk) // max(
        nq * heads * (dim + 2) * 4, 1)


SPLIT = [  # queries, keys, heads, kv heads, width, causal
    ([1], [1100], 1, 1, 128, True),
    ([5], [4000], 8, 2, 128, True),
    ([5], [4001], 8, 2, 64, True),
    ([70], [3000], 4, 4, 128, False),
    ([70], [3000], 4, 4, 64, False),
    ([1300], [1300], 1, 1, 128, True),                     # parts past the first rows' last key
    ([1300], [1300], 2, 1, 64, True),
    ([3, 1, 9], [5000, 2, 4000], 4, 1, 128, True),         # a sequence with fewer tiles than parts
    ([40, 0, 7], [3000, 100, 1500], 6, 2, 64, True),
    ([2, 6], [0, 3000], 4, 2, 128, False),                 # queries without keys
    ([20, 5], [10, 3000], 4, 2, 128, True),                # queries that see nothing
]


@pytest.mark.parametrize("lens_q,lens_k,heads,kv_heads,dim,causal", SPLIT)
def test_attention_of_few_rows_in_parts(pkg, dev, lens_q, lens_k, heads, kv_heads, dim, causal):
    nq, nk, batch = sum(lens_q), sum(lens_k), len(lens_q)
    q, k, v = _randn(45, nq, heads, dim), _randn(46, nk, kv_heads, dim), _randn(47, nk, kv_heads, dim)
    need = pkg.attention_workspace(heads, kv_heads, dim, batch, nq, nk)
    assert _parts(pkg, heads, kv_heads, dim, batch, nq, nk) >= 2
    # a byte pattern that is a NaN in every word, and a margin that has to stay
    ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full((nq + 3, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    z = torch.full((nq, heads), float("nan"), device="cuda")
    say(f"attention in parts {lens_q} {lens_k} heads {heads}/{kv_heads} x {dim} causal {causal}")
    pkg.attention(q, k, v, out[:nq], _cu(lens_q), _cu(lens_k), causal=causal, lse=z,
                  workspace=ws[:need])
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xff).all()) and bool((out[nq:] == 7.0).all())
    _verify(q, k, v, out[:nq], z, lens_q, lens_k, causal)
    # the binding's own workspace, no statistics, and again: the same bits
    for _ in range(2):
        again = torch.full_like(out[:nq], float("nan"))
        pkg.attention(q, k, v, again, _cu(lens_q), _cu(lens_k), causal=causal)
        torch.cuda.synchronize()
        assert torch.equal(again.view(torch.int16), out[:nq].view(torch.int16))


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_in_parts_unseen_and_seen_nan(pkg, dev, dim):
    """As without parts: what a row does not see has no influence, what it sees shows."""
    n = 1400
    q, k, v = _randn(48, n, 2, dim), _randn(49, n, 1, dim), _randn(50, n, 1, dim)
    assert _parts(pkg, 2, 1, dim, 1, n, n) >= 2
    clean, _ = _run(pkg, q, k, v, [n], [n], True)
    nan = float("nan")
    v[700, 0, 3], v[1300, 0, 5], k[1390], v[1395, 0, 9] = nan, float("inf"), nan, nan
    say(f"attention in parts, NaN x {dim}")
    out, z = _run(pkg, q, k, v, [n], [n], True)
    assert bool(torch.isfinite(out[:700]).all()) and bool(torch.isfinite(z[:1390]).all())
    assert bool(torch.isnan(out[700:, :, 3]).all())
    assert bool(torch.isfinite(out[700:1300, :, 4:]).all())
    assert not bool(torch.isfinite(out[1300:, :, 5]).any())
    assert bool(torch.isnan(out[1390:]).all()) and bool(torch.isnan(z[1390:]).all())
    rest = torch.ones(dim, dtype=torch.bool)
    rest[[3, 5]] = False
    # a NaN logit makes all rows of its wave take their maxima: beside it other bits
    assert torch.equal(out[:1344][..., rest].view(torch.int16), clean[:1344][..., rest].view(torch.int16))
    for i in (680, 699, 1350, 1380, 1389):
        want = attn_ref.attend(q[i:i + 1], k[:i + 1], v[:i + 1], dim ** -0.5, False)
        err = (out[i:i + 1].cpu().double() - want[0]).abs() - attn_ref.OUT_BOUND * want[2]
        assert float((err if i < 700 else err[..., rest]).max()) <= 0, f"row {i}"


def test_attention_in_parts_rows_of_no_sequence_stay(pkg, dev):
    """Tokens before, between and after the sequences that cu_q names keep what they hold."""
    q, k, v = _randn(51, 20, 4, 128), _randn(52, 4000, 2, 128), _randn(53, 4000, 2, 128)
    out = torch.full_like(q, 7.0)
    z = torch.full((20, 4), 7.0, device="cuda")
    cu_q = torch.tensor([4, 12], dtype=torch.int32, device="cuda")
    cu_k = torch.tensor([100, 3900], dtype=torch.int32, device="cuda")
    say("attention in parts, tokens of no sequence")
    pkg.attention(q, k, v, out, cu_q, cu_k, causal=True, lse=z)
    torch.cuda.synchronize()
    for t in (out, z):
        assert bool((t[:4] == 7.0).all()) and bool((t[12:] == 7.0).all())
    want = attn_ref.attend(q[4:12], k[100:3900], v[100:3900], 128 ** -0.5, True)
    attn_ref.check(out[4:12], z[4:12], want)


def test_attention_in_parts_in_a_graph(pkg, dev):
    q, k, v = _randn(54, 9, 8, 128), _randn(55, 6000, 2, 128), _randn(56, 6000, 2, 128)
    want, _ = _run(pkg, q, k, v, [9], [6000], True, lse=False)
    out, cu_q, cu_k = torch.empty_like(q), _cu([9]), _cu([6000])
    ws = torch.zeros(pkg.attention_workspace(8, 2, 128, 1, 9, 6000), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.attention(q, k, v, out, cu_q, cu_k, causal=True, workspace=ws)
    for rep in range(3):
        out.fill_(float("nan"))
        ws.fill_(0xff)
        torch.cuda.synchronize()
        say(f"attention in parts, replay {rep}")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_attention_in_parts_of_pinned_queries(pkg, dev):
    """Queries in pinned host memory: the workspace of the call's own lies on the GPU."""
    q, k, v = _randn(57, 3, 8, 128), _randn(58, 6000, 2, 128), _randn(59, 6000, 2, 128)
    assert pkg.attention_workspace(8, 2, 128, 1, 3, 6000) > 0
    want, got = torch.empty_like(q), torch.empty_like(q)
    say("attention in parts, pinned queries")
    pkg.attention(q, k, v, want, causal=True)
    pkg.attention(q.cpu().pin_memory(), k, v, got, causal=True)
    assert torch.equal(got, want)
