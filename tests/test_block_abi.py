"""What the 4-bit, norm and rotation entry points refuse, on the host: every check comes before any
device use."""
import ctypes

import pytest
import torch

FAKE = 0x10000   # never dereferenced: every call below ends in a check or is empty
BF16, F32 = 1, 2


def _mx4(pkg, rows=4, k=64, codes=FAKE, scales=FAKE):
    return pkg.Mx4C(codes, scales, rows, k)


def _norm(pkg, **kw):
    n = dict(width=64, layer=0, eps=1e-6, residual_scale=1.0, x_dtype=BF16, mod_dtype=BF16,
             weight_dtype=BF16, mod_rows=1, x_stride=64, x_out_stride=64, y_stride=64, mod_stride=64,
             out_stride=64)
    n.update(kw)
    return pkg.NormC(*[n[f] for f, _ in pkg.NormC._fields_])


def _rotation(pkg, **kw):
    r = dict(head_dim=64, rot_dim=0, interleaved=0, n_axes=1, freq_heads=1, pos_dtype=F32, freqs=FAKE,
             axes=None, positions=FAKE)
    r.update(kw)
    return pkg.RotationC(*[r[f] for f, _ in pkg.RotationC._fields_])


def _run_norm(pkg, lib, n=None, coded=False, q=None, tokens=4, **kw):
    a = dict(x=FAKE, y=2 * FAKE, x_out=3 * FAKE, post=FAKE, gate=FAKE, weight=FAKE, scale=FAKE,
             shift=FAKE, rows=None, out=4 * FAKE)
    a.update(kw)
    n = n if n is not None else _norm(pkg)
    args = [None, ctypes.byref(n), *(a[k] for k in ("x", "y", "x_out", "post", "gate", "weight",
                                                    "scale", "shift", "rows"))]
    if coded:
        q = q if q is not None else _mx4(pkg, tokens)
        return lib.ltx25_block_norm_mx4(*args, ctypes.byref(q), tokens)
    return lib.ltx25_block_norm(*args, a["out"], tokens)


def _rope(pkg, lib, r=None, q=FAKE, q_out=FAKE, heads=4, qs=256, qos=256, k=FAKE, k_out=FAKE, kv=2,
          ks=128, kos=128, tokens=3):
    r = r if r is not None else _rotation(pkg)
    return lib.ltx25_rope(None, ctypes.byref(r), q, q_out, heads, qs, qos, k, k_out, kv, ks, kos, tokens)


def _gemm(pkg, lib, x=None, w=None, bias=None, kind=0, y=FAKE, epi=0, ws=None, nbytes=0):
    x, w = x or _mx4(pkg), w or _mx4(pkg, 8)
    return lib.ltx25_mx4_gemm(None, ctypes.byref(x), ctypes.byref(w), bias, kind, y, epi, ws, nbytes)


def _linear(pkg, lib, x=FAKE, stride=64, m=40, w=None, bias=None, kind=0, y=FAKE, epi=0, ws=FAKE,
            nbytes=1 << 20):
    w = w or _mx4(pkg, 8)
    return lib.ltx25_linear_mx4(None, x, stride, m, ctypes.byref(w), bias, kind, y, epi, ws, nbytes)


# ---- 4 bits -----------------------------------------------------------------------------


def test_sizes_of_codes_and_scales(pkg, lib):
    for rows, k in [(1, 32), (16, 512), (17, 544), (1000, 16384)]:
        assert lib.ltx25_mx4_code_bytes(rows, k) == -(-rows // 16) * -(-k // 128) * 1024
        assert lib.ltx25_mx4_scale_bytes(rows, k) == -(-rows // 16) * -(-k // 512) * 256
    for rows, k in [(0, 32), (-1, 32), (4, 0), (4, 48), (4, -32), (1 << 28, 32), (4, 1 << 21)]:
        assert lib.ltx25_mx4_code_bytes(rows, k) == 0 and lib.ltx25_mx4_scale_bytes(rows, k) == 0
        assert lib.ltx25_linear_mx4_workspace(rows, k, 64) == 0
        assert lib.ltx25_mx4_gemm_workspace(rows, k, 64) == 0


BAD_OPERANDS = [dict(k=0), dict(k=48), dict(k=-32), dict(k=1 << 21), dict(rows=-1), dict(rows=1 << 28),
                dict(codes=None), dict(scales=None), dict(codes=FAKE + 8), dict(scales=FAKE + 2)]


@pytest.mark.parametrize("bad", BAD_OPERANDS)
def test_operands_that_are_refused(pkg, lib, bad):
    q = _mx4(pkg, **bad)
    b = ctypes.byref(q)
    assert lib.ltx25_mx4_quantize_rows(None, FAKE, BF16, 1 << 21, b) == pkg.E_INVAL
    assert lib.ltx25_mx4_dequant(None, b, FAKE, 1 << 21) == pkg.E_INVAL
    assert lib.ltx25_mx4_pack(None, FAKE, FAKE, b) == pkg.E_INVAL
    assert lib.ltx25_mx4_unpack(None, b, FAKE, FAKE) == pkg.E_INVAL
    assert _gemm(pkg, lib, x=q) == pkg.E_INVAL and _gemm(pkg, lib, w=q) == pkg.E_INVAL
    assert _linear(pkg, lib, w=q, stride=1 << 21) == pkg.E_INVAL


def test_null_operands(pkg, lib):
    q = ctypes.byref(_mx4(pkg))
    assert lib.ltx25_mx4_quantize_rows(None, FAKE, BF16, 64, None) == pkg.E_INVAL
    assert lib.ltx25_mx4_dequant(None, None, FAKE, 64) == pkg.E_INVAL
    assert lib.ltx25_mx4_pack(None, FAKE, FAKE, None) == pkg.E_INVAL
    assert lib.ltx25_mx4_gemm(None, None, q, None, 0, FAKE, 0, None, 0) == pkg.E_INVAL
    assert lib.ltx25_mx4_gemm(None, q, None, None, 0, FAKE, 0, None, 0) == pkg.E_INVAL
    assert lib.ltx25_linear_mx4(None, FAKE, 64, 4, None, None, 0, FAKE, 0, None, 0) == pkg.E_INVAL
    for p in ((None, FAKE), (FAKE, None), (FAKE + 8, FAKE), (FAKE, FAKE + 8)):
        assert lib.ltx25_mx4_pack(None, *p, q) == pkg.E_INVAL
        assert lib.ltx25_mx4_unpack(None, q, *p) == pkg.E_INVAL


def test_coding_refusals(pkg, lib):
    q = _mx4(pkg)
    b = ctypes.byref(q)
    for x, kind, stride in [(None, BF16, 64), (FAKE + 8, BF16, 64), (FAKE, 0, 64), (FAKE, 3, 64),
                            (FAKE, BF16, 56), (FAKE, BF16, 68), (FAKE, F32, 66), (FAKE, F32, 60),
                            (FAKE, BF16, 1 << 31)]:
        assert lib.ltx25_mx4_quantize_rows(None, x, kind, stride, b) == pkg.E_INVAL, (x, kind, stride)
    for out, stride in [(None, 64), (FAKE + 8, 64), (FAKE, 56), (FAKE, 68), (FAKE, 1 << 31)]:
        assert lib.ltx25_mx4_dequant(None, b, out, stride) == pkg.E_INVAL


def test_product_refusals(pkg, lib):
    bad = [dict(kind=1), dict(kind=2), dict(bias=FAKE), dict(bias=FAKE, kind=3), dict(bias=FAKE, kind=-1),
           dict(epi=2), dict(epi=-1), dict(y=None), dict(y=FAKE + 8), dict(bias=FAKE + 2, kind=2),
           dict(bias=FAKE + 1, kind=1)]
    for b in bad:
        assert _gemm(pkg, lib, **b) == pkg.E_INVAL, b
        assert _linear(pkg, lib, **b) == pkg.E_INVAL, b
    assert _gemm(pkg, lib, x=_mx4(pkg, k=96)) == pkg.E_INVAL          # another K
    huge = _mx4(pkg, 1 << 18, 1 << 14)                                # 2 GiB of codes
    assert _gemm(pkg, lib, x=_mx4(pkg, k=1 << 14), w=huge) == pkg.E_UNSUPPORTED
    assert _linear(pkg, lib, w=huge, stride=1 << 14) == pkg.E_UNSUPPORTED
    for b in [dict(x=None), dict(x=FAKE + 8), dict(stride=56), dict(stride=68), dict(m=-1),
              dict(m=1 << 28), dict(ws=None), dict(ws=FAKE + 8)]:
        assert _linear(pkg, lib, **b) == pkg.E_INVAL, b
    need = lib.ltx25_linear_mx4_workspace(40, 64, 8)
    assert need > 0 and _linear(pkg, lib, nbytes=need - 1) == pkg.E_INVAL
    assert "workspace" in pkg.last_error()


def test_empty_products(pkg, lib):
    none = _mx4(pkg, 0, codes=None, scales=None)
    assert _gemm(pkg, lib, x=none, y=None) == pkg.OK and _gemm(pkg, lib, w=none, y=None) == pkg.OK
    assert _linear(pkg, lib, m=0, x=None, y=None, ws=None) == pkg.OK
    assert _linear(pkg, lib, w=none, x=None, y=None, ws=None) == pkg.OK
    b = ctypes.byref(none)
    assert lib.ltx25_mx4_quantize_rows(None, None, BF16, 64, b) == pkg.OK
    assert lib.ltx25_mx4_dequant(None, b, None, 64) == pkg.OK
    assert lib.ltx25_mx4_pack(None, None, None, b) == pkg.OK


# ---- norms ------------------------------------------------------------------------------

BAD_NORMS = [dict(width=0), dict(width=-8), dict(width=60), dict(width=16392), dict(layer=2), dict(layer=-1),
             dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
             dict(eps=1e-30), dict(residual_scale=float("nan")), dict(residual_scale=float("inf")),
             dict(x_dtype=0), dict(x_dtype=3), dict(mod_dtype=0), dict(weight_dtype=7), dict(mod_rows=0),
             dict(mod_rows=-2), dict(mod_rows=3), dict(x_stride=56), dict(x_stride=68),
             dict(y_stride=60), dict(y_stride=56), dict(x_out_stride=8), dict(mod_stride=56),
             dict(mod_stride=66), dict(x_stride=1 << 31)]


@pytest.mark.parametrize("bad", BAD_NORMS)
def test_norm_sizes_that_are_refused(pkg, lib, bad):
    n = _norm(pkg, **bad)
    assert _run_norm(pkg, lib, n) == pkg.E_INVAL
    q = _mx4(pkg, 4, bad.get("width", 64))
    assert _run_norm(pkg, lib, n, coded=True, q=q) == pkg.E_INVAL


def test_norm_pointers(pkg, lib):
    assert lib.ltx25_block_norm(None, None, *[FAKE] * 8, None, FAKE, 4) == pkg.E_INVAL
    for name in ("x", "y", "x_out", "post", "gate", "weight", "scale", "shift", "out"):
        assert _run_norm(pkg, lib, **{name: FAKE + 8}) == pkg.E_INVAL, name
    assert _run_norm(pkg, lib, rows=FAKE + 2) == pkg.E_INVAL
    assert _run_norm(pkg, lib, x=None) == pkg.E_INVAL
    assert _run_norm(pkg, lib, x_out=None) == pkg.E_INVAL                 # y without it
    none = dict(y=None, x_out=None, post=None, gate=None)
    for name in ("x_out", "post", "gate"):
        assert _run_norm(pkg, lib, **dict(none, **{name: FAKE})) == pkg.E_INVAL
    assert _run_norm(pkg, lib, out=None, **none) == pkg.E_INVAL           # nothing to do
    assert _run_norm(pkg, lib, _norm(pkg, out_stride=56)) == pkg.E_INVAL
    assert _run_norm(pkg, lib, tokens=-1) == pkg.E_INVAL
    assert _run_norm(pkg, lib, tokens=(1 << 27) + 1) == pkg.E_INVAL
    assert _run_norm(pkg, lib, tokens=0, x=None) == pkg.OK


def test_norm_outputs_in_an_inputs_place(pkg, lib):
    """Token for token, or not at all."""
    x, y, xo = FAKE, 2 * FAKE, 3 * FAKE
    alone = dict(y=None, x_out=None, post=None, gate=None)
    for sizes, kw in [(dict(x_out_stride=128), dict(x_out=x)), (dict(out_stride=128), dict(out=y)),
                      (dict(out_stride=128), dict(alone, out=x)),
                      (dict(x_dtype=F32), dict(alone, out=x)), (dict(), dict(out=x)),
                      (dict(), dict(out=xo)), (dict(), dict(x_out=y))]:
        assert _run_norm(pkg, lib, _norm(pkg, **sizes), **kw) == pkg.E_INVAL, (sizes, kw)
        assert " is " in pkg.last_error(), pkg.last_error()


def test_rope_in_place_at_another_stride(pkg, lib):
    for kw in (dict(qos=512), dict(kos=256, q=2 * FAKE), dict(qs=512, kos=128)):
        assert _rope(pkg, lib, **kw) == pkg.E_INVAL
        assert "stride" in pkg.last_error() and "_out is " in pkg.last_error()


def test_norm_coded_output(pkg, lib):
    for q in (_mx4(pkg, 5), _mx4(pkg, 4, 96), _mx4(pkg, codes=None), _mx4(pkg, scales=None),
              _mx4(pkg, codes=FAKE + 4), _mx4(pkg, scales=FAKE + 1)):
        assert _run_norm(pkg, lib, coded=True, q=q) == pkg.E_INVAL
    wide = dict(width=72, x_stride=72, x_out_stride=72, y_stride=72, mod_stride=72)
    assert _run_norm(pkg, lib, _norm(pkg, **wide), coded=True, q=_mx4(pkg, 4, 72)) == pkg.E_INVAL
    assert _run_norm(pkg, lib, coded=True, tokens=0, x=None) == pkg.OK


# ---- rotations --------------------------------------------------------------------------

BAD_ROTATIONS = [dict(rot_dim=8), dict(rot_dim=80), dict(rot_dim=-16), dict(rot_dim=24),
                 dict(interleaved=2), dict(n_axes=0), dict(n_axes=5), dict(freq_heads=3),
                 dict(freq_heads=0), dict(freq_heads=4), dict(pos_dtype=1), dict(pos_dtype=0),
                 dict(freqs=None), dict(freqs=FAKE + 4), dict(axes=FAKE + 8), dict(positions=None),
                 dict(positions=FAKE + 2)]


@pytest.mark.parametrize("bad", BAD_ROTATIONS)
def test_rotations_that_are_refused(pkg, lib, bad):
    assert _rope(pkg, lib, _rotation(pkg, **bad)) == pkg.E_INVAL


@pytest.mark.parametrize("dim", [0, 8, 24, 272, -16])
def test_head_widths_that_are_refused(pkg, lib, dim):
    assert _rope(pkg, lib, _rotation(pkg, head_dim=dim), qs=4096, ks=4096) == pkg.E_UNSUPPORTED


def test_rope_tensors(pkg, lib):
    for name in ("q", "q_out", "k", "k_out"):
        assert _rope(pkg, lib, **{name: None}) == pkg.E_INVAL
        assert _rope(pkg, lib, **{name: FAKE + 8}) == pkg.E_INVAL
    for name in ("qs", "qos", "ks", "kos"):
        assert _rope(pkg, lib, **{name: 120}) == pkg.E_INVAL
        assert _rope(pkg, lib, **{name: 260}) == pkg.E_INVAL
        assert _rope(pkg, lib, **{name: 1 << 31}) == pkg.E_INVAL
    assert _rope(pkg, lib, heads=0) == pkg.E_INVAL                        # q without heads
    assert _rope(pkg, lib, heads=-1) == pkg.E_INVAL
    assert _rope(pkg, lib, heads=0, kv=0, q=None, q_out=None, k=None, k_out=None) == pkg.E_INVAL
    assert _rope(pkg, lib, heads=2000, qs=1 << 20, qos=1 << 20) == pkg.E_INVAL
    assert _rope(pkg, lib, tokens=-1) == pkg.E_INVAL
    assert _rope(pkg, lib, tokens=(1 << 27) + 1) == pkg.E_INVAL
    r = ctypes.byref(_rotation(pkg))
    assert lib.ltx25_rope(None, None, FAKE, FAKE, 4, 256, 256, None, None, 0, 0, 0, 3) == pkg.E_INVAL
    assert lib.ltx25_rope(None, r, None, None, 4, 256, 256, None, None, 0, 0, 0, 0) == pkg.OK


def test_append_refusals(pkg, lib):
    def call(r=None, kv=2, dim=64, k=FAKE, total=3, batch=2, **kw):
        c = pkg.KVCacheC(FAKE, FAKE, FAKE, FAKE, 4, 64, kv, dim)
        r = r if r is not None else _rotation(pkg, **kw)
        return lib.ltx25_kv_append_rope(None, ctypes.byref(c), FAKE, 4, k, FAKE, kv * dim, kv * dim, FAKE,
                                        FAKE, ctypes.byref(r), batch, total)

    for bad in BAD_ROTATIONS:
        if bad not in (dict(positions=None),):
            assert call(**bad) == pkg.E_INVAL, bad
    assert call(dim=128) == pkg.E_INVAL                                   # the cache's heads are wider
    assert call(k=FAKE + 8) == pkg.E_INVAL
    assert call(total=-1) == pkg.E_INVAL
    assert call(total=0, freqs=None) == pkg.OK
    assert call(batch=0, positions=None, pos_dtype=0, freqs=None) == pkg.OK


# ---- the binding ------------------------------------------------------------------------


class OnGpu(torch.Tensor):
    """A tensor that says that it lies in the GPU's memory: what the binding looks at."""

    is_cuda = True


def _gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)


def _coded(pkg, rows=4, k=64, host=False):
    c = torch.zeros(pkg.mx4_code_bytes(rows, k), dtype=torch.uint8)
    s = torch.zeros(pkg.mx4_scale_bytes(rows, k), dtype=torch.uint8)
    return pkg.MX4(*((c, s) if host else (c.as_subclass(OnGpu), s.as_subclass(OnGpu))), rows, k)


def _host(args, name):
    args = dict(args)
    args[name] = args[name].as_subclass(torch.Tensor).clone()
    return args


NORM = dict(x=(4, 64), out=(4, 64), y=(4, 64), x_out=(4, 64), gate=(1, 64), post_weight=(64,), weight=(64,),
            scale=(1, 64), shift=(1, 64))


@pytest.mark.parametrize("name", [*NORM, "rows"])
def test_norm_takes_no_host_memory(pkg, name):
    args = {n: _gpu(*s) for n, s in NORM.items()}
    args["rows"] = _gpu(4, dtype=torch.int32)
    with pytest.raises(ValueError, match=name):
        pkg.block_norm(**_host(args, name))


@pytest.mark.parametrize("name", ["q", "k", "positions", "freqs", "axes", "q_out", "k_out"])
def test_rope_takes_no_host_memory(pkg, name):
    args = dict(q=_gpu(4, 2, 64), k=_gpu(4, 1, 64), positions=_gpu(4, 1, dtype=torch.int32),
                freqs=_gpu(1, 32, dtype=torch.float32), axes=_gpu(1, 32, dtype=torch.int32),
                q_out=_gpu(4, 2, 64), k_out=_gpu(4, 1, 64))
    with pytest.raises(ValueError, match=name):
        pkg.rope(**_host(args, name))


@pytest.mark.parametrize("name", ["freqs", "axes", "positions"])
def test_append_takes_no_host_memory(pkg, name):
    cache = pkg.KVCache(_gpu(4, 2, 64, 64, dtype=torch.int8), _gpu(4, 2, 64, 64, dtype=torch.int8),
                        _gpu(4, 2, dtype=torch.float32), _gpu(4, 2, dtype=torch.float32))
    args = dict(freqs=_gpu(1, 32, dtype=torch.float32), axes=_gpu(1, 32, dtype=torch.int32),
                positions=_gpu(4, 1, dtype=torch.int32))
    x = _gpu(4, 2, 64)
    with pytest.raises(ValueError, match=name):
        pkg.kv_append_rope(cache, _gpu(1, 3, dtype=torch.int32), x, x, _gpu(2, dtype=torch.int32),
                           _gpu(1, dtype=torch.int32), **_host(args, name))


def test_4_bit_calls_take_no_host_memory(pkg):
    q, x, y = _coded(pkg), _gpu(4, 64), _gpu(4, 4)
    host = x.as_subclass(torch.Tensor)
    for call in (lambda: pkg.mx4_quantize_rows(host, q), lambda: pkg.mx4_dequant(q, host),
                 lambda: pkg.mx4_quantize_rows(x, _coded(pkg, host=True)),
                 lambda: pkg.linear_mx4(host, q, None, y, workspace=x),
                 lambda: pkg.linear_mx4(x, q, None, y.as_subclass(torch.Tensor), workspace=x),
                 lambda: pkg.mx4_gemm(q, _coded(pkg, host=True), None, y, workspace=x),
                 lambda: pkg.mx4_gemm(q, q, torch.zeros(4), y, workspace=x),
                 lambda: pkg.MX4.packed(torch.zeros((4, 32), dtype=torch.uint8),
                                        torch.zeros((4, 2), dtype=torch.uint8))):
        with pytest.raises(ValueError, match="GPU's memory"):
            call()


def test_shapes_and_types_that_do_not_fit(pkg):
    q, x, y = _coded(pkg), _gpu(4, 64), _gpu(4, 4)
    wrong = [lambda: pkg.mx4_quantize_rows(_gpu(5, 64), q), lambda: pkg.mx4_quantize_rows(_gpu(4, 32), q),
             lambda: pkg.mx4_quantize_rows(x.t(), q), lambda: pkg.mx4_quantize_rows(_gpu(4, 64, dtype=torch.float16), q),
             lambda: pkg.mx4_dequant(q, _gpu(4, 64, dtype=torch.float32)), lambda: pkg.mx4_dequant(q, _gpu(3, 64)),
             lambda: pkg.linear_mx4(_gpu(4, 32), q, None, y), lambda: pkg.linear_mx4(x, q, None, _gpu(4, 5)),
             lambda: pkg.linear_mx4(x, q, _gpu(5), y), lambda: pkg.linear_mx4(x, q, _gpu(4, dtype=torch.float16), y),
             lambda: pkg.mx4_gemm(q, q, None, _gpu(4, 8)[:, ::2]),
             lambda: pkg.MX4(q.codes, q.scales, 4, 160), lambda: pkg.MX4(q.codes, q.scales, 4, 60),
             lambda: pkg.MX4(q.codes[:-1], q.scales, 4, 64),
             lambda: pkg.MX4.packed(torch.zeros((4, 24), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.uint8)),
             lambda: pkg.block_norm(x, y), lambda: pkg.block_norm(x, x, y=_gpu(4, 64)),
             lambda: pkg.block_norm(x, x, y=_gpu(3, 64), x_out=x), lambda: pkg.block_norm(x, x, weight=_gpu(32)),
             lambda: pkg.block_norm(x, x, scale=_gpu(1, 64), shift=_gpu(2, 64)),
             lambda: pkg.block_norm(x, x, scale=_gpu(1, 64), shift=_gpu(1, 64, dtype=torch.float32)),
             lambda: pkg.block_norm(x, x, weight=_gpu(64), y=x, x_out=x, post_weight=_gpu(64, dtype=torch.float32)),
             lambda: pkg.block_norm(x, x, rows=_gpu(4)), lambda: pkg.block_norm(x, _coded(pkg, 5)),
             lambda: pkg.block_norm(x, _gpu(4, 64, dtype=torch.float32)),
             lambda: pkg.rope(None, None, None, None),
             lambda: pkg.rope(_gpu(4, 2, 64), None, _gpu(3, 1, dtype=torch.int32), _gpu(1, 32, dtype=torch.float32)),
             lambda: pkg.rope(_gpu(4, 2, 64), _gpu(5, 2, 64), _gpu(4, 1, dtype=torch.int32),
                              _gpu(1, 32, dtype=torch.float32)),
             lambda: pkg.rope(_gpu(4, 2, 64), None, _gpu(4, 1, dtype=torch.int64), _gpu(1, 32, dtype=torch.float32)),
             lambda: pkg.rope(_gpu(4, 2, 64), None, _gpu(4, 1, dtype=torch.int32), _gpu(1, 32)),
             lambda: pkg.rope(_gpu(4, 2, 64), None, _gpu(4, 1, dtype=torch.int32), _gpu(1, 32, dtype=torch.float32),
                              _gpu(1, 16, dtype=torch.int32)),
             lambda: pkg.rope(_gpu(4, 2, 64), None, _gpu(4, 1, dtype=torch.int32), _gpu(1, 32, dtype=torch.float32),
                              q_out=_gpu(4, 2, 32)),
             lambda: pkg.rope(None, _gpu(4, 2, 64), _gpu(4, 1, dtype=torch.int32), _gpu(1, 32, dtype=torch.float32),
                              q_out=_gpu(4, 2, 64))]
    for i, call in enumerate(wrong):
        with pytest.raises((TypeError, ValueError)):
            call()
            pytest.fail(f"call {i} was taken")


def test_a_stream_of_the_callers_needs_its_workspace(pkg):
    w, x, y = _coded(pkg, 8), _gpu(40, 64), _gpu(40, 8)
    with pytest.raises(ValueError, match="workspace"):
        pkg.linear_mx4(x, w, None, y, stream=1)


def test_a_stream_of_the_callers_needs_its_results(pkg):
    """What packed() and unpacked() would allocate belongs to torch's current stream: work queued there
    may still read memory that a kernel on another stream then writes."""
    codes, scales = _gpu(4, 32, dtype=torch.uint8), _gpu(4, 2, dtype=torch.uint8)
    q = _coded(pkg)
    for call in (lambda: pkg.MX4.packed(codes, scales, stream=1), lambda: q.unpacked(stream=1),
                 lambda: q.unpacked(stream=1, codes=codes), lambda: q.unpacked(1, scales=scales)):
        with pytest.raises(ValueError, match="the caller's too"):
            call()
    for call in (lambda: pkg.MX4.packed(codes, scales, 1, _coded(pkg, 5)),
                 lambda: pkg.MX4.packed(codes, scales, 1, _coded(pkg, 4, 96)),
                 lambda: pkg.MX4.packed(codes, scales, 1, _coded(pkg, host=True)),
                 lambda: q.unpacked(1, codes, codes), lambda: q.unpacked(1, scales, scales),
                 lambda: q.unpacked(1, codes, scales.as_subclass(torch.Tensor)),
                 lambda: q.unpacked(1, codes.as_subclass(torch.Tensor), scales)):
        with pytest.raises((TypeError, ValueError)) as e:
            call()
        assert "too" not in str(e.value)


class Pinned(torch.Tensor):
    """A tensor that says that it lies in pinned host memory."""

    def is_pinned(self, *args):
        return True


def test_memory_of_a_calls_own_beside_pinned_tensors_lies_on_the_gpu(pkg, monkeypatch):
    """Beside a pinned tensor is pageable host memory, which a kernel may not touch."""
    asked, empty = [], torch.empty

    class Lib:
        def __getattr__(self, name):
            return getattr(lib, name) if name.endswith("_bytes") or "workspace" in name else (
                lambda *args: pkg.OK)

    def recorded(*shape, device=None, **kw):
        asked.append(str(device))
        return empty(*shape, **kw)

    lib = pkg.load()
    codes, scales, x, y = (torch.zeros(s, dtype=t).as_subclass(Pinned) for s, t in (
        ((4, 32), torch.uint8), ((4, 2), torch.uint8), ((40, 64), torch.bfloat16),
        ((40, 4), torch.bfloat16)))
    held = pkg.MX4(*(torch.zeros(n, dtype=torch.uint8).as_subclass(Pinned)
                     for n in (pkg.mx4_code_bytes(4, 64), pkg.mx4_scale_bytes(4, 64))), 4, 64)
    q = torch.zeros((1, 8, 64), dtype=torch.bfloat16).as_subclass(Pinned)
    k = torch.zeros((4096, 8, 64), dtype=torch.bfloat16).as_subclass(Pinned)
    monkeypatch.setattr(torch, "empty", recorded)
    monkeypatch.setattr(pkg, "load", Lib)
    monkeypatch.setattr(pkg, "_on_device", lambda stream, names, tensors: 0)
    monkeypatch.setattr(pkg, "_stream", lambda stream: 0)
    monkeypatch.setattr(pkg, "_reachable", lambda names, *tensors: None)
    for call, times in ((lambda: pkg.MX4.packed(codes, scales), 2), (held.unpacked, 2),
                        (lambda: pkg.linear_mx4(x, held, None, y), 1),
                        (lambda: pkg.attention(q, k, k, q.clone(), causal=False), 1)):
        asked.clear()
        call()
        assert asked == ["cuda"] * times, asked


def test_codes_and_scales_of_which_one_is_pinned(pkg):
    """Calls look for pageable host memory among the codes; the scales lie there only with them."""
    held = [torch.zeros(n, dtype=torch.uint8) for n in (pkg.mx4_code_bytes(4, 64), pkg.mx4_scale_bytes(4, 64))]
    pinned = [t.as_subclass(Pinned) for t in held]
    pkg.MX4(*held, 4, 64)
    pkg.MX4(*pinned, 4, 64)
    for pair in ((pinned[0], held[1]), (held[0], pinned[1])):
        with pytest.raises(ValueError, match="pinned"):
            pkg.MX4(*pair, 4, 64)


@pytest.mark.parametrize("kw,what", [(dict(), "q_out is k_out"), (dict(q=2 * FAKE, k=3 * FAKE), "q_out is k_out"),
                                     (dict(q_out=2 * FAKE, k=2 * FAKE, k_out=3 * FAKE), "q_out is k:"),
                                     (dict(q_out=2 * FAKE, k=3 * FAKE), "k_out is q:")])
def test_rope_of_one_tensor_as_queries_and_keys(pkg, lib, kw, what):
    """Two threads would turn the same channels, or one read what the other writes."""
    assert _rope(pkg, lib, kv=4, ks=256, kos=256, **kw) == pkg.E_INVAL
    assert what in pkg.last_error()


def test_4_bit_outputs_in_an_inputs_place(pkg, lib):
    """What is written where the call still reads: K is N, or the rows and the order have one size."""
    a, b = 4 * FAKE, 5 * FAKE
    q = _mx4(pkg, 16, 128, a, b)
    for codes, scales in ((a, FAKE), (FAKE, b), (b, FAKE), (FAKE, a)):
        assert lib.ltx25_mx4_pack(None, codes, scales, ctypes.byref(q)) == pkg.E_INVAL
        assert "not in place" in pkg.last_error()
        assert lib.ltx25_mx4_unpack(None, ctypes.byref(q), codes, scales) == pkg.E_INVAL
        assert "not in place" in pkg.last_error()
    x, w = _mx4(pkg, 4, 64, 6 * FAKE, 7 * FAKE), _mx4(pkg, 64, 64, a, b)
    for y in (a, b, 6 * FAKE, 7 * FAKE, 8 * FAKE):
        assert _gemm(pkg, lib, x, w, 8 * FAKE, BF16, y) == pkg.E_INVAL
        assert "y is " in pkg.last_error()
    for m in (4, 40):
        for y in (a, b, 6 * FAKE, 7 * FAKE, 8 * FAKE):
            assert _linear(pkg, lib, 6 * FAKE, 64, m, w, 8 * FAKE, BF16, y, ws=7 * FAKE) == pkg.E_INVAL
            assert "y is " in pkg.last_error()


class OnSecond(OnGpu):
    """A tensor of the second GPU."""

    def get_device(self):
        return 1

    @property
    def device(self):
        return torch.device("cuda", 1)


class OnFirst(OnGpu):
    def get_device(self):
        return 0


@pytest.mark.parametrize("name", ["freqs", "axes", "positions", "k", "v", "table", "cu", "start", "cache.k",
                                  "cache.v", "cache.k_scale", "cache.v_scale"])
def test_append_takes_no_other_gpus_memory(pkg, monkeypatch, name):
    """Every tensor must lie on the GPU whose stream the call goes to."""
    int8, f32, i32, bf16 = torch.int8, torch.float32, torch.int32, torch.bfloat16
    shapes = dict(freqs=((1, 32), f32), axes=((1, 32), i32), positions=((4, 1), i32), k=((4, 2, 64), bf16),
                  v=((4, 2, 64), bf16), table=((1, 3), i32), cu=((2,), i32), start=((1,), i32))
    shapes.update({"cache.k": ((4, 2, 64, 64), int8), "cache.v": ((4, 2, 64, 64), int8),
                   "cache.k_scale": ((4, 2), f32), "cache.v_scale": ((4, 2), f32)})
    t = {n: torch.zeros(s, dtype=d).as_subclass(OnSecond if n == name else OnFirst)
         for n, (s, d) in shapes.items()}
    monkeypatch.setattr(pkg, "_device_now", lambda: 0)
    cache = pkg.KVCache(*(t["cache." + n] for n in ("k", "v", "k_scale", "v_scale")))
    # (a cache of two GPUs is refused by itself, at its tensor of the lower one)
    with pytest.raises(ValueError, match="^cache.* lies on" if "cache" in name else f"^{name} lies on"):
        pkg.kv_append_rope(cache, *(t[n] for n in ("table", "k", "v", "cu", "start", "freqs", "axes",
                                                   "positions")))
    if "cache" not in name:
        return
    cache = pkg.KVCache(*(t["cache." + n].as_subclass(OnSecond) for n in ("k", "v", "k_scale", "v_scale")))
    with pytest.raises(ValueError, match="^cache.k lies on"):
        pkg.kv_append_rope(cache, *(t[n] for n in ("table", "k", "v", "cu", "start", "freqs", "axes",
                                                   "positions")))
