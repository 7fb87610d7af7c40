"""Microscaled 4-bit rows on the GPU: codes and scales exactly, products against 64 bits."""
import numpy as np
import pytest
import torch

import mx4_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

SHAPES = [(1, 32), (1, 512), (3, 64), (15, 480), (16, 512), (17, 544), (33, 1056), (64, 2048),
          (5, 16384), (200, 96)]


def _bits(rng, shape, wide):
    """Values of any bits: denormals, zeros, and here and there an infinity or a NaN."""
    if wide:
        b = rng.integers(0, 1 << 32, shape, dtype=np.uint64).astype(np.uint32)
        x = torch.from_numpy(b.view(np.int32).copy()).view(torch.float32)
    else:
        b = rng.integers(0, 1 << 16, shape).astype(np.uint16)
        x = torch.from_numpy(b.view(np.int16).copy()).view(torch.bfloat16)
    # exponents side by side within a block, and blocks without a value that is not finite
    base = 2.0 ** torch.from_numpy(rng.integers(-130, 120, (shape[0], shape[1] // 32, 1))).double()
    near = torch.from_numpy(rng.standard_normal((shape[0], shape[1] // 32, 32))) * base
    near = near.reshape(shape).to(x.dtype)
    keep = torch.from_numpy(rng.random((shape[0], shape[1] // 32, 1)) < 0.2).expand(
        -1, -1, 32).reshape(shape)
    x = torch.where(keep, x, near)
    x[-1, :32] = 0
    return x


def _strided(x, extra=16):
    """The same rows with a gap between them."""
    wide = torch.empty((len(x), x.shape[1] + extra), dtype=x.dtype, device="cuda")
    wide.fill_(float("nan"))
    wide[:, :x.shape[1]] = x.cuda()
    return wide[:, :x.shape[1]]


def _same_codes(q, want):
    codes, scales = ref.download(q)
    assert (scales == want[1]).all()
    ok = np.repeat(want[1] != 255, 32, 1)
    assert (codes[ok] == want[0][ok]).all()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_codes_and_scales(pkg, dev, shape, wide):
    say(f"mx4 quantize {shape} wide={wide}")
    x = _bits(np.random.default_rng(shape[0] * 7 + shape[1] + wide), shape, wide)
    q = pkg.MX4.empty(*shape)
    q.codes.fill_(0xAA)
    q.scales.fill_(0xAA)
    pkg.mx4_quantize_rows(_strided(x), q)
    want = ref.code(x.double().numpy())
    _same_codes(q, want)
    # bytes of blocks past the row's end are zeros
    for got, tiled, wide_ones in ((q.scales, ref.tiles, 1), (q.codes, ref.code_tiles, 16)):
        whole = -(-want[1].shape[1] // (16 if wide_ones == 1 else 4)) * (16 if wide_ones == 1 else 4)
        there = tiled(np.ones((shape[0], want[1].shape[1] * wide_ones), np.uint8)) == 1
        rows = tiled(np.ones((shape[0], whole * wide_ones), np.uint8)) == 1
        assert (got.cpu().numpy()[rows & ~there] == 0).all()


def test_every_value_of_bf16(pkg, dev):
    """Each of the 65536 patterns as a value beside each of a few largest ones, so that every rounding
    and tie is met at every place of the exponent."""
    say("mx4 every bf16 value")
    allb = np.arange(65536, dtype=np.uint16)
    x = torch.from_numpy(allb.view(np.int16).copy()).view(torch.bfloat16).double().numpy()
    x = np.where(np.isfinite(x), x, 1.0).reshape(-1, 1)
    # the block's largest is the value times 1, 1.3, 3 or 9 where that is finite
    rows = []
    for f in (1.0, 1.3, 3.0, 9.0):
        top = torch.from_numpy(np.clip(np.abs(x) * f, 0, 3e38)).bfloat16().double().numpy()
        rows.append(np.concatenate([x, -x, top, np.repeat(0 * x, 29, 1)], 1))
    x = np.concatenate(rows).reshape(-1, 512)
    q = pkg.MX4.empty(*x.shape)
    pkg.mx4_quantize_rows(torch.from_numpy(x).bfloat16().cuda(), q)
    _same_codes(q, ref.code(x))


@pytest.mark.parametrize("shape", SHAPES)
def test_values_back(pkg, dev, shape):
    say(f"mx4 dequant {shape}")
    rng = np.random.default_rng(shape[1])
    codes = rng.integers(0, 16, shape).astype(np.uint8)
    scales = rng.integers(0, 256, (shape[0], shape[1] // 32)).astype(np.uint8)
    scales[0, 0] = 255
    q = ref.upload(pkg, codes, scales)
    out = _strided(torch.zeros(shape, dtype=torch.bfloat16))
    pkg.mx4_dequant(q, out)
    want = torch.from_numpy(ref.values(codes, scales)).float().bfloat16()
    got = out.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0, posinf=1, neginf=-1),
                       torch.nan_to_num(want, nan=0.0, posinf=1, neginf=-1))
    gap = torch.as_strided(out, (shape[0], 16), (out.stride(0), 1), out.storage_offset() + shape[1])
    assert bool(torch.isnan(gap).all())


@pytest.mark.parametrize("shape", SHAPES)
def test_the_two_orders(pkg, dev, shape):
    say(f"mx4 orders {shape}")
    rng = np.random.default_rng(1)
    codes = rng.integers(0, 16, shape).astype(np.uint8)
    scales = rng.integers(0, 256, (shape[0], shape[1] // 32)).astype(np.uint8)
    rows = [torch.from_numpy(t).cuda() for t in (ref.packed(codes), scales)]
    q = pkg.MX4.packed(*rows)
    pad = 16 * (-(-shape[0] // 16)) - shape[0]
    assert (q.codes.cpu().numpy() == ref.code_tiles(np.pad(ref.packed(codes), ((0, pad), (0, 0))))).all()
    assert (q.scales.cpu().numpy() == ref.tiles(np.pad(scales, ((0, pad), (0, 0))))).all()
    back = q.unpacked()
    assert torch.equal(back[0], rows[0]) and torch.equal(back[1], rows[1])


# sizes around each kernel's rows, columns and steps, and around the changes from one to another
PRODUCTS = [(1, 32, 1), (1, 64, 16), (2, 512, 17), (5, 544, 40), (16, 1024, 64), (17, 1056, 63),
            (31, 96, 100), (33, 2080, 129), (64, 4096, 96), (65, 512, 257), (100, 2048, 1000),
            (127, 160, 130), (129, 4096, 72), (200, 8192, 24), (255, 256, 255), (257, 768, 520),
            (300, 1568, 1001), (520, 2048, 776), (1, 16384, 48), (1000, 288, 1500), (3, 8224, 9)]


def _bias(rng, n, kind):
    if kind is None:
        return None, None
    b = torch.from_numpy(rng.standard_normal(n)).to(kind)
    return b.cuda(), b.double().numpy()


def _guarded(m, n):
    """An output between two stretches that no call may write."""
    flat = torch.full((m * n + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    return flat[2048:2048 + m * n].view(m, n), flat


def _untouched(flat, n):
    assert bool((flat[:2048] == 7).all()) and bool((flat[2048 + n:] == 7).all())


@pytest.mark.parametrize("kind,gelu", [(None, False), (torch.float32, True), (torch.bfloat16, False)])
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(pkg, dev, m, k, n, kind, gelu):
    say(f"mx4 gemm {m}x{k}->{n} bias={kind} gelu={gelu}")
    rng = np.random.default_rng(m * 31 + k + n)
    x, w = ref.random_operand(rng, m, k), ref.random_operand(rng, n, k, low=118)
    bias, b = _bias(rng, n, kind)
    y, flat = _guarded(m, n)
    pkg.mx4_gemm(ref.upload(pkg, *x), ref.upload(pkg, *w), bias, y,
                 pkg.EPI_GELU_TANH if gelu else pkg.EPI_NONE)
    ref.check_product(y, ref.values(*x), ref.values(*w), b, gelu, f"{m}x{k}->{n}")
    _untouched(flat, m * n)


@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_linear_is_coding_and_product(pkg, dev, m, k, n):
    say(f"linear_mx4 {m}x{k}->{n}")
    rng = np.random.default_rng(m + k * 3 + n)
    x = torch.from_numpy(rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k))).bfloat16()
    w = ref.random_operand(rng, n, k, low=118)
    weight = ref.upload(pkg, *w)
    bias, b = _bias(rng, n, torch.float32)
    y, flat = _guarded(m, n)
    need = pkg.linear_mx4_workspace(m, k, n)
    ws = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    pkg.linear_mx4(_strided(x), weight, bias, y, workspace=ws[:need])
    ref.check_product(y, ref.values(*ref.code(x.double().numpy())), ref.values(*w), b, False)
    _untouched(flat, m * n)
    assert bool((ws[need:] == 0xAB).all())
    q = pkg.MX4.empty(m, k)
    pkg.mx4_quantize_rows(x.cuda(), q)
    two = torch.empty_like(y)
    pkg.mx4_gemm(q, weight, bias, two)
    assert torch.equal(y, two)
    pkg.linear_mx4(x.cuda(), weight, bias, two)
    assert torch.equal(y, two)


@pytest.mark.parametrize("m", [1, 3, 4, 5, 15, 16])
@pytest.mark.parametrize("k", [32, 96, 512, 1056, 4128])
def test_few_rows_are_coded_alike(pkg, dev, m, k):
    """Up to 16 rows are coded by the product's own waves: values of any bits, NaN and infinities
    among them, give what the two calls give."""
    say(f"linear_mx4 of any bits {m}x{k}")
    rng = np.random.default_rng(m * k)
    x = _strided(_bits(rng, (m, k), False))
    w = ref.upload(pkg, *ref.random_operand(rng, 40, k, low=118))
    q = pkg.MX4.empty(m, k)
    pkg.mx4_quantize_rows(x, q)
    one, two = (torch.empty((m, 40), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pkg.linear_mx4(x, w, None, one)
    pkg.mx4_gemm(q, w, None, two)
    assert torch.equal(torch.isnan(one), torch.isnan(two))
    assert torch.equal(torch.nan_to_num(one, nan=7.0), torch.nan_to_num(two, nan=7.0))


@pytest.mark.parametrize("m,k,n,ahead", [(16, 4096, 4096, False), (17, 4096, 4096, True), (1, 4128, 4112, False),
                                         (5, 4128, 4112, True), (16, 96, 8208, True), (9, 12320, 40, True),
                                         (4, 12320, 40, False)])
def test_few_rows_that_are_coded_ahead(pkg, dev, m, k, n, ahead):
    """More coding than a launch costs goes into the workspace; the results are the two calls'."""
    say(f"linear_mx4 coded ahead {m}x{k}->{n}")
    need = pkg.linear_mx4_workspace(m, k, n)
    assert (need > 0) == ahead and pkg.linear_mx4_workspace(m + 1, k, n) >= need
    rng = np.random.default_rng(m * k)
    x = _strided(_bits(rng, (m, k), False))
    w = ref.upload(pkg, *ref.random_operand(rng, n, k, low=118))
    q = pkg.MX4.empty(m, k)
    pkg.mx4_quantize_rows(x, q)
    one, two = (torch.empty((m, n), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ws = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    pkg.linear_mx4(x, w, None, one, workspace=ws[:need])
    pkg.mx4_gemm(q, w, None, two)
    assert bool((ws[need:] == 0xAB).all())
    assert torch.equal(torch.isnan(one), torch.isnan(two))
    assert torch.equal(torch.nan_to_num(one, nan=7.0), torch.nan_to_num(two, nan=7.0))


# Outputs of enough tiles for each kind of workgroup in turn, the largest last, with rows, columns
# and K that end inside a tile, spans of K fewer than and around the stages', and more tiles than
# workgroups that walk them.
LARGE = [(20, 512, 3100, True), (100, 2080, 1800, False), (200, 544, 1300, True), (200, 32, 3100, False),
         (200, 1056, 3100, True), (250, 4608, 3101, False), (130, 32, 6151, True), (140, 1568, 6150, False),
         (130, 2592, 6152, False), (300, 64, 6200, False), (290, 1024, 6200, True), (300, 5120, 6199, False),
         (1010, 1056, 6100, True), (600, 544, 12201, False), (2040, 32, 6104, True), (2810, 1568, 12792, True),
         (2100, 4096, 3000, True), (4097, 1056, 4104, False), (1500, 8192, 2049, False),
         (8160, 512, 4096, False), (8160, 96, 4095, True), (5000, 544, 4100, True)]


def _on_gpu(pkg, rows, k, gen):
    codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.randint(118, 122, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=gen)
    lut = torch.tensor(ref.VALUES, device="cuda")
    v = lut[torch.stack([codes & 15, codes >> 4], 2).flatten(1).int()]
    return pkg.MX4.packed(codes, scales), v * (2.0 ** (scales.double() - 127)).repeat_interleave(32, 1)


@pytest.mark.parametrize("m,k,n,gelu", LARGE)
def test_large_products(pkg, dev, m, k, n, gelu):
    """Against torch in 64 bits on the GPU, with the bounds of ref.check_product."""
    say(f"mx4 large {m}x{k}->{n}")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + k)
    (x, xv), (w, wv) = _on_gpu(pkg, m, k, gen), _on_gpu(pkg, n, k, gen)
    bias = torch.randn(n, device="cuda", generator=gen).to(torch.bfloat16 if gelu else torch.float32)
    y, flat = _guarded(m, n)
    pkg.mx4_gemm(x, w, bias, y, pkg.EPI_GELU_TANH if gelu else pkg.EPI_NONE)
    want = xv @ wv.T + bias.double()
    slack = 1.13 * (k + 1) * 2.0 ** -24 * (xv.abs() @ wv.abs().T + bias.double().abs())
    if gelu:
        want = torch.nn.functional.gelu(want, approximate="tanh")
    err = (y.double() - want).abs() - (1.01 * 2.0 ** -8 * want.abs() + slack)
    assert float(err.max()) <= 0, float(err.max())
    _untouched(flat, m * n)
    again = torch.empty_like(y)
    pkg.mx4_gemm(x, w, bias, again, pkg.EPI_GELU_TANH if gelu else pkg.EPI_NONE)
    assert torch.equal(again, y)


def test_sizes_past_32_bits(pkg, dev):
    """Codes beyond 1 GiB go out in two launches, and outputs and activations of more than 2^31
    elements: rows of the whole call against calls on those rows alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    for m, k, n in [(17_000_003, 96, 8), (140_001, 64, 16384)]:
        say(f"mx4 past 32 bits {m}x{k}->{n}")
        w = pkg.MX4.packed(torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen),
                           torch.randint(118, 122, (n, k // 32), dtype=torch.uint8, device="cuda", generator=gen))
        x = torch.randn((m, k), device="cuda", generator=gen).bfloat16()
        y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
        pkg.linear_mx4(x, w, None, y)
        edge = (1 << 30) // 64
        for lo in (0, 130_900, min(edge - 200, m - 600), m - 600):
            part = torch.empty((600, n), dtype=torch.bfloat16, device="cuda")
            pkg.linear_mx4(x[lo:lo + 600], w, None, part)
            # (another kernel may take the smaller call: sums in another order)
            d = (part.float() - y[lo:lo + 600].float()).abs()
            assert float((d - 2.0 ** -7 * part.float().abs()).max()) <= 1e-3
        del x, y
    m, k = 270_001, 8192
    say("mx4 quantize past 32 bits")
    x = torch.randn((1, k), device="cuda", generator=gen).bfloat16().expand(m, k).contiguous()
    x[-5:] = torch.randn((5, k), device="cuda", generator=gen).bfloat16()
    q, part, back = pkg.MX4.empty(m, k), pkg.MX4.empty(5, k), torch.empty_like(x)
    pkg.mx4_quantize_rows(x, q)
    pkg.mx4_dequant(q, back)
    want = torch.empty((5, k), dtype=torch.bfloat16, device="cuda")
    pkg.mx4_quantize_rows(x[-5:], part)
    pkg.mx4_dequant(part, want)
    assert torch.equal(back[-5:], want) and torch.equal(back[m // 2], back[0])


@pytest.mark.parametrize("m,k,n", [(1, 1024, 64), (20, 1024, 64), (300, 1024, 520), (2000, 1024, 4000)])
def test_blocks_of_nan_stay_in_their_rows(pkg, dev, m, k, n):
    say(f"mx4 NaN blocks {m}x{k}->{n}")
    rng = np.random.default_rng(5)
    x, w = ref.random_operand(rng, m, k), ref.random_operand(rng, n, k)
    x[1][m // 2, 7] = 255
    w[1][n // 3, 30] = 255
    # a block of zero codes with a scale of NaN is one of NaN, too
    w[0][n // 3, 960:992] = 0
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    pkg.mx4_gemm(ref.upload(pkg, *x), ref.upload(pkg, *w), None, y)
    bad = torch.isnan(y).cpu().numpy()
    want = np.zeros((m, n), bool)
    want[m // 2], want[:, n // 3] = True, True
    assert (bad == want).all()


def test_scales_at_both_ends(pkg, dev):
    """Exponents far apart in the two operands whose products are ordinary numbers; products beyond
    f32's range are infinite, those below it zero."""
    say("mx4 scales at both ends")
    rng = np.random.default_rng(6)
    m, k, n = 33, 512, 48
    for a, b in [(0, 254), (254, 0), (10, 230), (127, 127), (60, 200)]:
        x, w = ref.random_operand(rng, m, k, 1, a), ref.random_operand(rng, n, k, 1, b)
        y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
        pkg.mx4_gemm(ref.upload(pkg, *x), ref.upload(pkg, *w), None, y)
        ref.check_product(y, ref.values(*x), ref.values(*w), None, False, f"{a} {b}")
    x, w = ref.random_operand(rng, m, k, 1, 254), ref.random_operand(rng, n, k, 1, 254)
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    x = (np.full_like(x[0], 7), x[1])
    w = (np.full_like(w[0], 2), w[1])
    pkg.mx4_gemm(ref.upload(pkg, *x), ref.upload(pkg, *w), None, y)
    assert bool((y == float("inf")).all())
    low = np.zeros_like(x[1])
    pkg.mx4_gemm(ref.upload(pkg, x[0], low), ref.upload(pkg, w[0], np.zeros_like(w[1])), None, y)
    assert bool((y == 0).all())


def test_no_rows_and_no_columns(pkg, dev):
    w = ref.upload(pkg, *ref.random_operand(np.random.default_rng(0), 16, 64))
    none = pkg.MX4(w.codes[:0], w.scales[:0], 0, 64)
    y = torch.empty((0, 16), dtype=torch.bfloat16, device="cuda")
    pkg.mx4_gemm(none, w, None, y)
    pkg.linear_mx4(torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"), w, None, y)
    pkg.mx4_gemm(w, none, None, torch.empty((16, 0), dtype=torch.bfloat16, device="cuda"))
    pkg.mx4_quantize_rows(torch.empty((0, 64), device="cuda"), none)
    pkg.mx4_dequant(none, torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,k,n", [(1, 4096, 512), (24, 2048, 264), (150, 4096, 1000), (1100, 1024, 2048)])
def test_captured_on_a_stream_and_repeated(pkg, dev, m, k, n):
    """Captured with its workspace, replayed with other inputs and other work between, on a side
    stream and twice: the same bits."""
    say(f"mx4 graph {m}x{k}->{n}")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    w = ref.upload(pkg, *ref.random_operand(np.random.default_rng(2), n, k))
    bias = torch.randn(n, device="cuda", generator=gen)
    xs = [torch.randn((m, k), device="cuda", generator=gen).bfloat16() for _ in range(4)]
    want = []
    for x in xs:
        y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
        pkg.linear_mx4(x, w, bias, y)
        want.append(y)
    ws = torch.empty(pkg.linear_mx4_workspace(m, k, n), dtype=torch.uint8, device="cuda")
    x, y = xs[0].clone(), torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.linear_mx4(x, w, bias, y, workspace=ws)
    for i in (1, 0, 3, 2, 1):
        x.copy_(xs[i])
        ws.fill_(0x5A)
        graph.replay()
        assert torch.equal(y, want[i])
        (xs[i].float() @ xs[i].float().T).sum()
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [torch.empty_like(y) for _ in xs]
        for a, o in zip(xs, outs):
            pkg.linear_mx4(a, w, bias, o)
    side.synchronize()
    assert all(torch.equal(o, t) for o, t in zip(outs, want))


def test_orders_on_a_stream_of_the_callers(pkg, dev):
    """Packing and unpacking into the caller's tensors on its stream."""
    say("mx4 orders on a stream")
    rng = np.random.default_rng(11)
    codes, scales = ref.random_operand(rng, 37, 1056)
    rows = [torch.from_numpy(t).cuda() for t in (ref.packed(codes), scales)]
    q, back = pkg.MX4.empty(37, 1056), [torch.zeros_like(t) for t in rows]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert pkg.MX4.packed(*rows, stream=s.cuda_stream, out=q) is q
    q.unpacked(s.cuda_stream, *back)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(rows, back))
    assert all(torch.equal(a, b) for a, b in zip(pkg.MX4.packed(*rows).unpacked(), rows))


def test_results_beside_pinned_memory(pkg, dev):
    """Inputs in pinned host memory: results and workspaces of the calls' own lie on the GPU."""
    say("mx4 pinned")
    rng = np.random.default_rng(12)
    codes, scales = ref.random_operand(rng, 20, 1056)
    rows = [torch.from_numpy(t).pin_memory() for t in (ref.packed(codes), scales)]
    q = pkg.MX4.packed(*rows)
    assert q.codes.is_cuda and q.scales.is_cuda
    there = pkg.MX4(q.codes.cpu().pin_memory(), q.scales.cpu().pin_memory(), 20, 1056)
    for held in (q, there):
        back = held.unpacked()
        assert all(b.is_cuda and torch.equal(b.cpu(), r) for b, r in zip(back, rows))
    x = torch.from_numpy(rng.standard_normal((40, 1056))).bfloat16().cuda()
    y, want = torch.zeros((40, 20), dtype=torch.bfloat16).pin_memory(), torch.empty((40, 20), dtype=torch.bfloat16, device="cuda")
    pkg.linear_mx4(x, q, None, y)
    pkg.linear_mx4(x, q, None, want)
    torch.cuda.synchronize()
    assert torch.equal(y, want.cpu())


@pytest.mark.parametrize("m,k,n,gelu", [(8160, 1056, 4096, False), (8160, 1568, 4095, True)])
def test_tiles_walked_over_several_spans(pkg, dev, m, k, n, gelu):
    """1024 tiles of 256 x 128 for 512 workgroups: stages and rows of x change hands between a
    workgroup's tiles after an odd and an even number of spans."""
    test_large_products(pkg, dev, m, k, n, gelu)
