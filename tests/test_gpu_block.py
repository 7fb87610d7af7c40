"""Norms, rotations and the rotating append on the GPU against 64 bits."""
import itertools

import numpy as np
import pytest
import torch

import mx4_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _f64(t):
    return None if t is None else t.double().cpu().numpy()


def _t(rng, shape, kind, scale=1.0):
    return (torch.from_numpy(rng.standard_normal(shape)) * scale).to(kind).cuda()


def _strided(t, gap=24):
    """The same rows apart from each other, with NaN between."""
    wide = torch.full((t.shape[0], t.shape[1] + gap), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _gap_is_nan(view, gap=24):
    past = torch.as_strided(view, (view.shape[0], gap), (view.stride(0), 1),
                            view.storage_offset() + view.shape[1])
    assert bool(torch.isnan(past).all())


def _close(got, want, mag, kind, what):
    got = _f64(got)
    share = ref.BF16_SHARE if kind is BF16 else 2.0 ** -24
    err = np.abs(got - want) - (share * np.abs(want) + ref.F32_SHARE * mag + 1e-37)
    assert float(err.max()) <= 0, f"{what}: off by {float(err.max()):.3e}"


WIDTHS = [8, 40, 64, 72, 128, 136, 256, 264, 504, 512, 520, 1024, 1032, 1536, 1544, 2048, 2056, 3080, 4096, 4104,
          6144, 6152, 8192, 8200, 12288, 12296, 16384]
FORMS = [  # kind of x, kind of the modulations, y, post, gate, weight, modulated, layer, alpha
    (BF16, BF16, True, False, True, False, True, False, 1.0),
    (F32, F32, True, True, True, True, True, True, 0.7),
    (BF16, F32, False, False, False, True, False, False, 1.0),
    (F32, BF16, True, False, False, False, False, True, -1.5),
    (BF16, BF16, True, True, True, True, True, False, 0.0),
]


def _norm_case(rng, tokens, width, form, rows):
    kind, mod, y, post, gate, weight, modulated, layer, alpha = form
    c = dict(x=_strided(_t(rng, (tokens, width), kind, 3.0)), layer=layer, residual_scale=alpha)
    c["weight"] = _t(rng, (width,), BF16) if weight else None
    if y:
        c["y"] = _strided(_t(rng, (tokens, width), BF16))
        c["post_weight"] = _t(rng, (width,), BF16) if post else None
    if modulated:
        six = _t(rng, (rows, 3 * width), mod, 0.4)
        parts = dict(zip(("gate", "scale", "shift"), six.split(width, 1)))
        if not (y and gate):
            parts.pop("gate")
        c.update(parts)
    return c


def _want(c, row, eps=1e-6):
    return ref.block_norm(_f64(c["x"]), _f64(c.get("y")), _f64(c.get("post_weight")),
                          _f64(c.get("gate")), _f64(c.get("weight")), _f64(c.get("scale")),
                          _f64(c.get("shift")), row, c["layer"], eps, c["residual_scale"])


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(pkg, dev, width, form):
    tokens = [1, 5, 2, 7, 4][(WIDTHS.index(width) + form) % 5]
    say(f"block_norm {tokens}x{width} form {form}")
    rng = np.random.default_rng(width + form)
    rows = 1 if form % 2 else tokens
    c = _norm_case(rng, tokens, width, FORMS[form], rows)
    row = np.arange(tokens) // (tokens // rows)
    if "y" in c:
        c["x_out"] = _strided(torch.zeros_like(c["x"]))
    out = _strided(torch.zeros((tokens, width), dtype=BF16, device="cuda"))
    pkg.block_norm(out=out, **c)
    h, x, mag, mag_x = _want(c, row)
    _close(out, h, mag, BF16, "out")
    _gap_is_nan(out)
    if "y" in c:
        _close(c["x_out"], x, mag_x, c["x"].dtype, "x_out")
        _gap_is_nan(c["x_out"])
        # in place, and without the next norm
        again = c["x"].clone()
        pkg.block_norm(out=None, **dict(c, x=again, x_out=again))
        assert torch.equal(again, c["x_out"])


@pytest.mark.parametrize("tokens,rows", [(1, 1), (12, 4), (63, 63), (130, 5), (9, 2)])
def test_norm_rows_of_the_modulation(pkg, dev, tokens, rows):
    say(f"block_norm rows {tokens} {rows}")
    rng = np.random.default_rng(tokens)
    c = _norm_case(rng, tokens, 264, FORMS[0], rows)
    c["x_out"] = torch.empty_like(c["x"])
    out = torch.empty((tokens, 264), dtype=BF16, device="cuda")
    given = rng.integers(0, rows, tokens)
    for index in (given, None):
        if index is None and tokens % rows:
            continue
        row = np.arange(tokens) // (tokens // rows) if index is None else index
        c["rows"] = None if index is None else torch.from_numpy(index.astype(np.int32)).cuda()
        pkg.block_norm(out=out, **c)
        h, _, mag, _ = _want(c, row)
        _close(out, h, mag, BF16, "out")
    # rows that there are not are the nearest that there are
    c["rows"] = torch.from_numpy((given - 3 * rows).astype(np.int32)).cuda()
    pkg.block_norm(out=out, **c)
    _close(out, *[_want(c, np.zeros(tokens, int))[i] for i in (0, 2)], BF16, "below")
    c["rows"] = torch.full((tokens,), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    pkg.block_norm(out=out, **c)
    _close(out, *[_want(c, np.full(tokens, rows - 1))[i] for i in (0, 2)], BF16, "above")


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("width", [32, 96, 160, 1024, 1280, 2048, 2400, 4096, 5120, 9600, 16384])
def test_norm_of_values_at_both_ends(pkg, dev, width, layer):
    """Squares beyond f32's range and below it, constant rows, and values that are not finite, which
    stay in their rows."""
    say(f"block_norm ends {width} {layer}")
    rng = np.random.default_rng(width)
    x = _t(rng, (8, width), F32)
    x[0] *= 1e36
    x[1] *= 1e-30
    x[2] = 3e38
    x[3] = 0
    x[4, 3] = 3.2e38
    x[5, -1] = float("inf")
    x[6, 1] = float("nan")
    out = torch.empty((8, width), dtype=BF16, device="cuda")
    pkg.block_norm(x, out, layer=layer)
    fine = [0, 1, 2, 3, 4, 7]
    h, _, mag, _ = ref.block_norm(_f64(x)[fine], None, None, None, None, None, None, None, layer, 1e-6, 1.0)
    if layer:
        # a constant row's mean is its value to f32's rounding, and what is left of the row is shared
        # out by a deviation of the same size: both are noise of the sum
        h, fine_out = np.delete(h, 2, 0), _f64(out[[0, 1, 3, 4, 7]])
        mag = np.delete(mag, 2, 0)
        assert bool(torch.isfinite(out[2].float()).all())
    else:
        fine_out = _f64(out[fine])
    err = np.abs(fine_out - h) - (ref.BF16_SHARE * np.abs(h) + ref.F32_SHARE * mag + 1e-37)
    assert float(err.max()) <= 0, float(err.max())
    assert bool(torch.isnan(out[6]).all())
    assert bool(torch.isnan(out[5, -1])) or layer


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("scale,eps", [(1e19, 3.2e38), (1e19, 1e38), (1e18, 3e37), (1e20, 1e38), (1.0, 1e38)])
def test_norm_of_a_large_eps(pkg, dev, scale, eps, layer):
    """It counts where the squares or their sum with it leave f32's range, too."""
    say(f"block_norm eps {scale} {eps} {layer}")
    x = _t(np.random.default_rng(3), (5, 1024), F32, scale)
    out = torch.empty((5, 1024), dtype=BF16, device="cuda")
    pkg.block_norm(x, out, layer=layer, eps=eps)
    h, _, mag, _ = ref.block_norm(_f64(x), None, None, None, None, None, None, None, layer,
                                  float(np.float32(eps)), 1.0)
    _close(out, h, mag, BF16, "out")


def test_norm_in_place(pkg, dev):
    """out in x (queries normed over all heads in the projection's output), and in y."""
    say("block_norm in place")
    rng = np.random.default_rng(8)
    proj = _t(rng, (37, 3 * 256), BF16)
    w, keep = _t(rng, (256,), BF16), proj.clone()
    want = torch.empty((37, 256), dtype=BF16, device="cuda")
    pkg.block_norm(keep[:, 256:512], want, weight=w)
    pkg.block_norm(proj[:, 256:512], proj[:, 256:512], weight=w)
    assert torch.equal(proj[:, 256:512], want)
    assert torch.equal(proj[:, :256], keep[:, :256]) and torch.equal(proj[:, 512:], keep[:, 512:])
    x, y = _t(rng, (37, 256), F32), _t(rng, (37, 256), BF16)
    xo = torch.empty_like(x)
    pkg.block_norm(x, want, y=y, x_out=xo)
    pkg.block_norm(x, y, y=y, x_out=x)
    assert torch.equal(y, want) and torch.equal(x, xo)


@pytest.mark.parametrize("tokens,width", [(1, 32), (5, 544), (16, 512), (18, 1056), (33, 2048), (40, 64),
                                          (9, 2592), (4, 4128), (17, 8224), (2, 16384), (3, 12800)])
def test_norm_coded(pkg, dev, tokens, width):
    """4-bit output: the codes of values within f32's roundings of the 64-bit ones, so that where no
    tie or largest value is that near they are the same."""
    say(f"block_norm_mx4 {tokens}x{width}")
    rng = np.random.default_rng(width)
    c = _norm_case(rng, tokens, width, FORMS[0], 1)
    c["x_out"] = torch.empty_like(c["x"])
    q = pkg.MX4.empty(tokens, width)
    q.scales.fill_(0xAA)
    q.codes.fill_(0xAA)
    pkg.block_norm(out=q, **c)
    h, _, mag, _ = _want(c, np.zeros(tokens, int))
    codes, scales = ref.download(q)
    near = [ref.code(h + s * ref.F32_SHARE * mag) for s in (-1, 0, 1)]
    sure = (near[0][1] == near[1][1]) & (near[1][1] == near[2][1])
    assert sure.mean() > 0.98 and (scales == near[1][1])[sure].all()
    firm = np.repeat(sure, 32, 1) & (near[0][0] == near[1][0]) & (near[1][0] == near[2][0])
    assert firm.mean() > 0.95 and (codes == near[1][0])[firm].all()
    full = ref.tiles(np.ones((tokens, -(-width // 512) * 16), np.uint8)) == 1
    there = ref.tiles(np.ones((tokens, width // 32), np.uint8)) == 1
    assert (q.scales.cpu().numpy()[full & ~there] == 0).all()
    full = ref.code_tiles(np.ones((tokens, -(-width // 128) * 64), np.uint8)) == 1
    there = ref.code_tiles(np.ones((tokens, width // 2), np.uint8)) == 1
    assert (q.codes.cpu().numpy()[full & ~there] == 0).all()
    out = torch.empty((tokens, width), dtype=BF16, device="cuda")
    xo = c["x_out"].clone()
    pkg.block_norm(out=out, **c)
    assert torch.equal(xo, c["x_out"])


CODED_FORMS = [  # the same, of coded outputs alone
    (BF16, BF16, False, False, False, True, True, False, 1.0),
    (BF16, F32, False, False, False, False, False, True, 1.0),
    (F32, BF16, False, False, False, False, True, False, 1.0),
    *FORMS]


CODED_SIZES = [(515, 64), (1030, 512), (600, 544), (128, 1056), (129, 2048), (200, 2592), (140, 4128),
               (131, 8224), (130, 16384)]


@pytest.mark.parametrize("tokens,width,form", [(*size, (i + j) % len(CODED_FORMS))
                                               for i, size in enumerate(CODED_SIZES) for j in (0, 3, 5)])
def test_norm_coded_of_many_tokens(pkg, dev, tokens, width, form):
    """From 128 workgroups on tokens change places, so that 16 rows are coded on one XCD: every row
    its own, in every form, against the codes of 64 bits as in test_norm_coded."""
    say(f"block_norm_mx4 {tokens}x{width} form {form}")
    rng = np.random.default_rng(width + form)
    c = _norm_case(rng, tokens, width, CODED_FORMS[form], tokens)
    if "y" in c:
        c["x_out"] = torch.empty_like(c["x"])
    q = pkg.MX4.empty(tokens, width)
    pkg.block_norm(out=q, **c)
    h, x, mag, mag_x = _want(c, np.arange(tokens))
    codes, scales = ref.download(q)
    near = [ref.code(h + s * ref.F32_SHARE * mag) for s in (-1, 0, 1)]
    sure = (near[0][1] == near[1][1]) & (near[1][1] == near[2][1])
    assert sure.mean() > 0.98 and (scales == near[1][1])[sure].all()
    firm = np.repeat(sure, 32, 1) & (near[0][0] == near[1][0]) & (near[1][0] == near[2][0])
    assert firm.mean() > 0.95 and (codes == near[1][0])[firm].all()
    if "y" in c:
        _close(c["x_out"], x, mag_x, c["x"].dtype, "x_out")


def test_norm_and_rope_past_32_bits(pkg, dev):
    """Tensors of more than 2^31 elements: their last rows against calls on those alone."""
    say("norm and rope past 32 bits")
    t, w = 140_000, 16384
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    x = torch.randn((1, w), device="cuda", generator=gen).bfloat16().expand(t, w).contiguous()
    x[-40:] = torch.randn((40, w), device="cuda", generator=gen).bfloat16()
    out, q = torch.empty_like(x), pkg.MX4.empty(t, w)
    pkg.block_norm(x, out)
    pkg.block_norm(x, q)
    want, coded, back = torch.empty_like(x[-40:]), pkg.MX4.empty(40, w), torch.empty_like(x)
    pkg.block_norm(x[-40:], want)
    pkg.block_norm(x[-40:], coded)
    assert torch.equal(out[-40:], want) and torch.equal(out[t // 2], out[0])
    values = torch.empty_like(want)
    pkg.mx4_dequant(coded, values)
    pkg.mx4_dequant(q, back)
    assert torch.equal(back[-40:], values) and torch.equal(back[t // 2], back[0])
    heads = x.view(t, 128, 128)
    pos = torch.zeros((t, 2), device="cuda")
    pos[-40:] = torch.randn((40, 2), device="cuda", generator=gen)
    freqs = torch.rand((1, 64), device="cuda", generator=gen)
    which = (torch.arange(64, device="cuda", dtype=torch.int32) % 2)[None].contiguous()
    for side in (False, True):
        pkg.rope(heads, None, pos, freqs, which, q_out=out.view(t, 128, 128), interleaved=side)
        small = torch.empty((40, 128, 128), dtype=BF16, device="cuda")
        pkg.rope(heads[-40:], None, pos[-40:].contiguous(), freqs, which, q_out=small, interleaved=side)
        assert torch.equal(out[-40:].view(40, 128, 128), small) and torch.equal(out[5], x[5])


# ---- rotations ------------------------------------------------------------------------------


def test_rope_of_more_threads_than_a_launch_has(pkg, dev):
    """In place, where a token that two launches turned would be turned twice."""
    say("rope past 2^32 threads")
    tokens, heads, dim = (1 << 27) - 5, 17, 16
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 73 GB")
    gen = torch.Generator(device="cuda").manual_seed(9)
    block = torch.randn((4096, heads, dim), device="cuda", generator=gen).to(BF16)
    q = torch.empty((1 << 27, heads, dim), dtype=BF16, device="cuda")
    q.view(-1, 4096, heads, dim).copy_(block)
    positions = torch.arange(1 << 27, dtype=torch.int32, device="cuda").view(-1, 1)
    freqs = torch.rand((1, dim // 2), device="cuda", generator=gen)
    pkg.rope(q[:tokens], None, positions[:tokens], freqs, interleaved=True)
    edge = ((1 << 32) - 512) // (heads * dim // 8) // 4096 * 4096
    for lo in (0, edge - 4096, edge, edge + 4096, (1 << 27) - 4096):
        n = min(4096, tokens - lo)
        want = block.clone()
        pkg.rope(want[:n], None, positions[lo:lo + n], freqs, interleaved=True)
        assert torch.equal(q[lo:lo + 4096], want), lo
    del q
    torch.cuda.empty_cache()


def _rope_case(rng, tokens, heads, kv, dim, rot, axes, per_head, whole, far=1000):
    proj = _t(rng, (tokens, (heads + 2 * kv) * dim), BF16)
    q, k, _ = (p.unflatten(1, (-1, dim)) for p in
               proj.split([heads * dim, kv * dim, kv * dim], 1))
    pos = (rng.integers(-far, far, (tokens, axes)).astype(np.int32) if whole
           else (rng.standard_normal((tokens, axes)) * far).astype(np.float32))
    fh = heads if per_head else 1
    freqs = (np.exp(rng.uniform(-9, 0.5, (fh, rot // 2)))).astype(np.float32)
    which = rng.integers(0, axes, (fh, rot // 2)).astype(np.int32)
    return proj, q, k, pos, freqs, which


ROPES = [(1, 1, 1, 16, 16, 1, False), (3, 4, 2, 64, 64, 1, False), (130, 8, 8, 128, 128, 3, True),
         (17, 5, 1, 80, 48, 2, False), (9, 3, 3, 256, 224, 4, True), (70, 2, 2, 128, 64, 1, False),
         (2, 64, 64, 128, 128, 3, True), (513, 1, 1, 32, 32, 2, False), (5, 12, 4, 96, 16, 3, False)]


@pytest.mark.parametrize("side,whole", itertools.product([False, True], [False, True]))
@pytest.mark.parametrize("case", ROPES)
def test_rope(pkg, dev, case, side, whole):
    say(f"rope {case} side={side} whole={whole}")
    rng = np.random.default_rng(sum(case))
    proj, q, k, pos, freqs, which = _rope_case(rng, *case, whole)
    up = [torch.from_numpy(a).cuda() for a in (pos, freqs, which)]
    qo = torch.full((case[0], case[1] + 1, case[3]), 7.0, dtype=BF16, device="cuda")
    ko = torch.full((case[0], case[2] + 2, case[3]), 7.0, dtype=BF16, device="cuda")
    pkg.rope(q, k, *up, q_out=qo[:, :case[1]], k_out=ko[:, 2:], interleaved=side)
    for got, x in ((qo[:, :case[1]], q), (ko[:, 2:], k)):
        want, mag = ref.rotate(_f64(x), pos, freqs, which, side)
        ref.check_rotated(got, want, mag, str(case))
        assert torch.equal(got[:, :, case[4]:], x[:, :, case[4]:])
    assert bool((qo[:, case[1]:] == 7).all()) and bool((ko[:, :2] == 7).all())
    # in place, and one of the two alone
    keep = proj.clone()
    pkg.rope(q, None, *up, interleaved=side)
    assert torch.equal(q, qo[:, :case[1]])
    n = case[1] * case[3]
    assert torch.equal(proj[:, n:], keep[:, n:])
    pkg.rope(None, k, *up, interleaved=side)
    assert torch.equal(k, ko[:, 2:])
    # negated frequencies turn back
    pkg.rope(q, k, up[0], -up[1], up[2], interleaved=side)
    was = keep[:, :n].unflatten(1, (-1, case[3]))
    assert float((q - was).abs().max()) <= 0.05 and torch.equal(proj[:, n + case[2] * case[3]:],
                                                               keep[:, n + case[2] * case[3]:])


def test_rope_far_positions(pkg, dev):
    """Angles of 2^30 radians, and positions whose angle is near a whole number of quarter turns, where
    a sine or cosine is small and its absolute error shows."""
    say("rope far positions")
    rng = np.random.default_rng(1)
    for side in (False, True):
        proj, q, k, pos, freqs, which = _rope_case(rng, 600, 2, 1, 64, 64, 1, False, True, 1 << 30)
        freqs[0, :4] = 1.0
        quarter = np.rint(np.arange(600) * np.pi / 2 * 710).astype(np.int32)
        pos[:300, 0] = quarter[:300]
        freqs[0, 4] = np.float32(np.pi / 2)
        pos[0] = 0
        want, mag = ref.rotate(_f64(q), pos, freqs, which, side)
        pkg.rope(q, None, *(torch.from_numpy(a).cuda() for a in (pos, freqs, which)), interleaved=side)
        ref.check_rotated(q, want, mag, "far")


@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("top,whole", [(1 << 20, True), (1 << 24, True), ((1 << 31) - 1, True),
                                       (1 << 24, False), (1 << 36, False)])
def test_rope_angles_past_64_bits(pkg, dev, top, whole, axes, side):
    """Positions and frequencies whose product's own bits go past what 64 bits hold: the angles come
    from whole numbers. A channel pair (1, 0) gives the cosine and the sine themselves, and f32
    products and sums of it have no error; the check's 2^-20 is the sine's."""
    say(f"rope angles {top} {whole} {axes} {side}")
    rng = np.random.default_rng(top % 1000 + axes)
    tokens, pairs = 160, 8
    at = rng.integers(top // 2, top, tokens, endpoint=True) * rng.choice([-1, 1], tokens)
    at = at.astype(np.int32 if whole else np.float32)
    freqs = (15708.0 * np.exp(rng.uniform(-3, 0, (1, pairs)))).astype(np.float32)
    freqs[0, 0], freqs[0, 1] = 1.0, np.float32(np.pi)   # (a whole position is near half a turn)
    ang = ref.reduced_angles(at, freqs[0])
    x = np.zeros((tokens, 1, 16))
    first, second = (slice(0, 16, 2), slice(1, 16, 2)) if side else (slice(0, 8), slice(8, 16))
    x[:, :, first] = 1.0
    want = np.zeros_like(x)
    want[:, 0, first], want[:, 0, second] = np.cos(ang), np.sin(ang)
    pos = np.zeros((tokens, axes), at.dtype)
    pos[:, axes - 1] = at
    which = np.full((1, pairs), axes - 1, np.int32)
    up = [torch.from_numpy(a).cuda() for a in (pos, freqs, which)]
    q = torch.from_numpy(x).to(BF16).cuda()
    pkg.rope(q, None, *up, interleaved=side)
    ref.check_rotated(q, want, np.ones_like(x), "far angles")
    if not whole:
        return
    # the append's keys are turned alike (heads of 64, of which 16 channels turn)
    parts, table, k, v, (cu, st) = _append_case(pkg, rng, ([3], [tokens], 2, 64, 32))
    plain, one = (pkg.KVCache(*(t.clone() for t in parts)) for _ in range(2))
    turned = torch.empty_like(k.contiguous())
    pkg.rope(None, k, *up, k_out=turned, interleaved=side)
    pkg.kv_append(plain, table, turned, v, cu, st)
    pkg.kv_append_rope(one, table, k, v, cu, st, up[1], up[2], up[0], interleaved=side)
    mask = _defined(([3], [tokens], 2, 64, 32), table.cpu().numpy(), one.k.shape, "k")
    assert torch.equal(one.k.cpu()[mask], plain.k.cpu()[mask])
    assert torch.equal(one.k_scale, plain.k_scale)


def test_rope_axes_out_of_range_and_absent(pkg, dev):
    say("rope axes")
    rng = np.random.default_rng(2)
    _, q, k, pos, freqs, which = _rope_case(rng, 20, 3, 1, 64, 64, 2, False, False)
    wild = which.copy()
    wild[0, :10] = [-5, 2, 3, 100, -1, 1 << 30, -(1 << 31), 0, 1, 7]
    want, mag = ref.rotate(_f64(q), pos, freqs, wild, False)
    out = torch.empty_like(q)
    up = [torch.from_numpy(a).cuda() for a in (pos, freqs, wild)]
    pkg.rope(q, None, *up, q_out=out)
    ref.check_rotated(out, want, mag, "axes")
    want, mag = ref.rotate(_f64(q), pos, freqs, 0 * which, False)
    pkg.rope(q, None, up[0], up[1], q_out=out)
    ref.check_rotated(out, want, mag, "no axes")


APPENDS = [([0], [1], 1, 64, 16), ([5, 0, 31], [1, 40, 1], 2, 128, 32), ([100, 7], [3, 300], 4, 128, 64),
           ([0, 0], [0, 129], 3, 64, 128), ([1000, 63, 64], [70, 1, 64], 8, 128, 64)]


def _append_case(pkg, rng, case):
    start, new, heads, dim, page = case
    pages = [-(-(a + n) // page) for a, n in zip(start, new)]
    total = sum(pages) + 2
    k = torch.from_numpy(rng.integers(-127, 128, (total, heads, page, dim)).astype(np.int8)).cuda()
    v = torch.from_numpy(rng.integers(-127, 128, (total, heads, dim, page)).astype(np.int8)).cuda()
    s = [torch.from_numpy((0.001 + 0.03 * rng.random((total, heads))).astype(np.float32)).cuda()
         for _ in range(2)]
    order = rng.permutation(total)
    table = np.full((len(start), max(pages) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    proj = _t(rng, (sum(new), 2 * heads * dim), BF16)
    kk, vv = (p.unflatten(1, (-1, dim)) for p in proj.chunk(2, 1))
    ints = [torch.tensor(a, dtype=torch.int32, device="cuda")
            for a in (np.concatenate([[0], np.cumsum(new)]), start)]
    return (k, v, *s), torch.from_numpy(table).cuda(), kk, vv, ints


@pytest.mark.parametrize("share,per_head,given", [(1, False, False), (2, False, True), (1, True, True),
                                                  (4, True, False)])
@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_is_rope_and_append(pkg, dev, case, side, share, per_head, given):
    say(f"kv_append_rope {APPENDS[case]} side={side} {share} {per_head} {given}")
    rng = np.random.default_rng(case)
    start, new, heads, dim, page = APPENDS[case]
    parts, table, k, v, (cu, st) = _append_case(pkg, rng, APPENDS[case])
    axes = 3 if given else 1
    shape = (heads if per_head else 1, dim // share // 2)
    freqs = torch.from_numpy(np.exp(rng.uniform(-9, 0, shape)).astype(np.float32)).cuda()
    which = torch.from_numpy(rng.integers(0, axes, shape).astype(np.int32)).cuda()
    if given:
        pos = torch.from_numpy(rng.standard_normal((sum(new), 3)).astype(np.float32) * 100).cuda()
    else:
        pos = torch.from_numpy(np.concatenate([np.arange(a, a + n) for a, n in zip(start, new)])
                               .astype(np.int32)[:, None]).cuda()
    plain = pkg.KVCache(*(t.clone() for t in parts))
    turned = torch.empty_like(k.contiguous())
    pkg.rope(None, k, pos, freqs, which, k_out=turned, interleaved=side)
    pkg.kv_append(plain, table, turned, v, cu, st)
    one = pkg.KVCache(*(t.clone() for t in parts))
    pkg.kv_append_rope(one, table, k, v, cu, st, freqs, which, pos if given else None,
                       interleaved=side)
    for name in ("k", "v", "k_scale", "v_scale"):
        a, b = getattr(one, name), getattr(plain, name)
        if name in ("k", "v"):
            # a written page's contents past the last new token are undefined
            mask = _defined(APPENDS[case], table.cpu().numpy(), a.shape, name)
            a, b = a.cpu()[mask], b.cpu()[mask]
        assert torch.equal(a, b), name


def _defined(case, table, shape, name):
    start, new, _, _, page = case
    mask = np.ones(shape, bool)
    for b, (a, n) in enumerate(zip(start, new)):
        if n and (a + n) % page:
            p, t = table[b, (a + n) // page], (a + n) % page
            if name == "k":
                mask[p, :, t:] = False
            else:
                mask[p, :, :, t:] = False
    return torch.from_numpy(mask)


@pytest.mark.parametrize("op", ["norm", "norm_mx4", "rope", "append"])
def test_captured_and_repeated(pkg, dev, op):
    """Captured, replayed on other inputs with other work between, against eager calls."""
    say(f"captured {op}")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    rng = np.random.default_rng(0)
    xs = [torch.randn((24, 1024), device="cuda", generator=gen).bfloat16() for _ in range(4)]
    x, y = xs[0].clone(), torch.randn((24, 1024), device="cuda", generator=gen).bfloat16()
    w = torch.randn(1024, device="cuda", generator=gen)
    out, xo, q = torch.empty_like(x), torch.empty_like(x), pkg.MX4.empty(24, 1024)
    freqs = torch.rand((1, 32), device="cuda", generator=gen)
    pos = torch.arange(24, dtype=torch.int32, device="cuda")[:, None].contiguous()
    parts, table, _, _, _ = _append_case(pkg, rng, ([3], [24], 8, 64, 16))
    fresh = [t.clone() for t in parts]
    cache = pkg.KVCache(*parts)
    cu, start = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, 24], [3]))

    def call():
        if op == "norm":
            pkg.block_norm(x, out, y=y, x_out=xo, weight=w, layer=True)
        elif op == "norm_mx4":
            pkg.block_norm(x, q, y=y, x_out=xo, weight=w)
        elif op == "rope":
            pkg.rope(x.view(24, 16, 64), None, pos, freqs, q_out=out.view(24, 16, 64))
        else:
            pkg.kv_append_rope(cache, table, x[:, :512].unflatten(1, (8, 64)),
                               x[:, 512:].unflatten(1, (8, 64)), cu, start, freqs)

    def results():
        if op == "append":
            return [t.clone() for t in parts[2:]] + [parts[0][table[0, 0]].clone()]
        return [t.clone() for t in ((q.codes, xo) if op == "norm_mx4" else (out, xo) if op == "norm"
                                    else (out,))]

    def reset():
        for t, f in zip(parts, fresh):
            t.copy_(f)

    want = []
    for a in xs:
        reset()
        x.copy_(a)
        call()
        want.append(results())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (2, 0, 3, 1, 1):
        reset()
        x.copy_(xs[i])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(results(), want[i]))
        (xs[i].float() @ xs[i].float().T).sum()
        torch.cuda.synchronize()
