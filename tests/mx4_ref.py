"""Microscaled 4-bit rows, norms and rotations restated in 64 bits, for the tests."""
import math

import numpy as np
import torch

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def code(x):
    """float64 rows [R][K] (NaN and infinities among them) -> codes u8 [R][K], scales u8 [R][K / 32]."""
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(b).max(2)
    bad = ~np.isfinite(b).all(2)
    top = np.where(bad | (top == 0), 2.0 ** -140, top)
    exp = np.clip(np.frexp(top)[1] - 1 - 2, -127, 127)
    v = np.ldexp(np.where(bad[:, :, None], 0.0, b), -exp[:, :, None])
    mag = np.abs(v)
    step = np.where(mag < 2, 0.5, np.where(mag < 4, 1.0, 2.0))
    q = np.minimum(np.rint(mag / step) * step, 6.0)     # rint: ties to even, as the codes' do
    idx = np.searchsorted(VALUES[:8], q).astype(np.uint8)
    idx = np.where(np.signbit(v), idx + 8, idx).astype(np.uint8)
    return idx.reshape(rows, k), np.where(bad, 255, exp + 127).astype(np.uint8)


def values(codes, scales):
    """Codes [R][K] and scales [R][K / 32] -> float64 values."""
    rows, k = codes.shape
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (VALUES[codes].reshape(rows, k // 32, 32) * s[:, :, None]).reshape(rows, k)


def packed(codes):
    """Two codes a byte, the earlier one in the low half."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpacked(b):
    return np.stack([b & 15, b >> 4], 2).reshape(len(b), -1)


def tiles(scales):
    """Scales [R][K / 32] in the matrix cores' order; bytes that stand for no block are 0."""
    rows, blocks = scales.shape
    spans = -(-blocks // 16)
    out = np.zeros((-(-rows // 16)) * spans * 256, np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[((r // 16) * spans + b // 16) * 256 + ((b % 4) * 16 + r % 16) * 4 + (b // 4) % 4] = scales
    return out


def code_tiles(b):
    """Packed codes [R][K / 2] in the matrix cores' order; bytes that stand for no block are 0."""
    rows, blocks = len(b), b.shape[1] // 16
    slices = -(-blocks // 4)
    out = np.zeros(((-(-rows // 16)) * slices * 64, 16), np.uint8)
    r, k = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[((r // 16) * slices + k // 4) * 64 + (k % 4) * 16 + r % 16] = b.reshape(rows, blocks, 16)
    return out.reshape(-1)


def random_operand(rng, rows, k, spread=3, low=120):
    codes = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    scales = rng.integers(low, low + spread, (rows, k // 32)).astype(np.uint8)
    return codes, scales


def upload(pkg, codes, scales):
    return pkg.MX4(torch.from_numpy(code_tiles(packed(codes))).cuda(),
                   torch.from_numpy(tiles(scales)).cuda(), *codes.shape)


def download(q):
    """An MX4's codes [R][K] and scales [R][K / 32]."""
    codes, scales = q.unpacked()
    return unpacked(codes.cpu().numpy()), scales.cpu().numpy()


def gelu(y):
    with np.errstate(over="ignore"):
        return y / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def check_product(got, x, w, bias, use_gelu, what=""):
    """got bf16 [M][N] against x . w^T in 64 bits. The products are exact; f32 sums of K of them are
    within K 2^-24 of the sum of magnitudes, the bias adds one rounding, GELU's slope is below 1.13
    and its own steps cost 2^-20 of the result, and the output's rounding is 2^-8 of it."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    slack = 1.13 * (x.shape[1] + 1) * 2.0 ** -24 * mag
    if use_gelu:
        y = gelu(y)
    got = got.float().cpu().numpy().astype(np.float64)
    nan = np.isnan(y)
    assert (np.isnan(got) == nan).all(), f"{what}: NaN in other places"
    err = np.abs(got - y) - (2.0 ** -8 * 1.01 * np.abs(y) + slack + 1e-38)
    assert nan.all() or float(err[~nan].max()) <= 0, f"{what}: off by {float(err[~nan].max()):.3e}"


# ---- norms ------------------------------------------------------------------------------


def norm(x, layer, eps, width):
    if layer:
        x = x - x.mean(1, keepdims=True)
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps)


def block_norm(x, y, post, gate, weight, scale, shift, row, layer, eps, alpha):
    """float64 arrays or None -> out, x_out, and the magnitudes that f32's roundings are shares of."""
    w = x.shape[1]
    mag_x = np.abs(x)
    if y is not None:
        u = y
        if post is not None:
            u = norm(u, layer, eps, w) * post
        if gate is not None:
            u = u * gate[row]
        mag_x = np.abs(alpha * x) + np.abs(u)
        if post is not None:
            mag_x = mag_x + np.abs(y).max(1, keepdims=True) / np.sqrt(
                ((y - (y.mean(1, keepdims=True) if layer else 0)) ** 2).mean(1, keepdims=True)
                + eps) * np.abs(post) * (np.abs(gate[row]) if gate is not None else 1)
        x = alpha * x + u
    h = norm(x, layer, eps, w)
    c = x - (x.mean(1, keepdims=True) if layer else 0)
    mag = mag_x.max(1, keepdims=True) / np.sqrt((c * c).mean(1, keepdims=True) + eps) + np.abs(h)
    for f in (weight, None if scale is None else 1 + scale[row]):
        if f is not None:
            h, mag = h * f, mag * np.abs(f)
    if shift is not None:
        h, mag = h + shift[row], mag + np.abs(shift[row])
    return h, x, mag, mag_x


# Each value takes a dozen f32 steps and shares in sums of up to 16384 values that are added in at most
# 64 steps one after another: 2^-17 of the magnitudes is more than all of these.
F32_SHARE = 2.0 ** -17
BF16_SHARE = 2.0 ** -8 * 1.01


# ---- rotations ----------------------------------------------------------------------------


def rotate(x, positions, freqs, axes, interleaved):
    """x float64 [T][H][D]; positions [T][A], freqs and axes [1 or H][P] -> rotated, and for each
    channel |a| + |b| of its pair."""
    out, mag = x.copy(), np.zeros_like(x)
    pairs = freqs.shape[1]
    axes = np.clip(axes, 0, positions.shape[1] - 1)
    ang = positions.astype(np.float64)[:, axes] * freqs.astype(np.float64)     # [T][1 or H][P]
    i = np.arange(pairs)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    cs, sn = np.cos(ang), np.sin(ang)
    out[:, :, a] = x[:, :, a] * cs - x[:, :, b] * sn
    out[:, :, b] = x[:, :, a] * sn + x[:, :, b] * cs
    mag[:, :, a] = mag[:, :, b] = np.abs(x[:, :, a]) + np.abs(x[:, :, b])
    return out, mag


def _inverse_turn(bits):
    """floor(2^bits / (2 pi)), by Machin's formula in whole numbers."""
    one = 1 << (bits + 64)

    def arctan(x):   # of 1 / x
        term = total = one // x
        n = 1
        while term:
            n, term = n + 2, -term // (x * x)
            total += term // n
        return total

    return (one << bits) // (2 * 4 * (4 * arctan(5) - arctan(239)))


def reduced_angles(positions, freqs):
    """Whole or float32 positions [T] times float32 freqs [P], exactly, less whole turns: float64
    [T][P] within half a turn, for products far past what 64 bits hold."""
    bits = 400
    inv = _inverse_turn(bits)
    out = np.empty((len(positions), len(freqs)))
    for i, p in enumerate(positions):
        for j, f in enumerate(freqs):
            (a, b), (c, d) = float(p).as_integer_ratio(), float(f).as_integer_ratio()
            left = (a * c * inv // (b * d)) % (1 << bits)
            left -= (1 << bits) if left >> (bits - 1) else 0
            out[i, j] = 2 * math.pi * (left / (1 << bits))
    return out


def check_rotated(got, want, mag, what=""):
    """One rounding to bf16; sines and cosines to 2^-20, and the products' own roundings."""
    got = got.float().cpu().numpy().astype(np.float64)
    err = np.abs(got - want) - (BF16_SHARE * np.abs(want) + 1.1 * 2.0 ** -20 * mag + 1e-38)
    assert float(err.max()) <= 0, f"{what}: off by {float(err.max()):.3e}"
