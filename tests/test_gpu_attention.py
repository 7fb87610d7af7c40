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
