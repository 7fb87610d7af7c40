"""Python binding of the ltx25 quantized-linear C ABI (include/ltx25_qlinear.h).

A thin ctypes layer over libltx25_qlinear.so for tests and the benchmark:
device buffers are torch tensors (plumbing only) whose data pointers are
passed through the C ABI, and every call runs on torch's current stream
unless a stream is given. The HIP library is the only compute path; when it
is missing, load() raises instead of falling back to anything else.

The package directory name is not a Python identifier, so callers import it
by path; ``load_package()`` in __graft_entry__.py and tests/conftest.py do
that.
"""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libltx25_qlinear.so")
HEADER_PATH = os.path.join(HERE, "..", "include", "ltx25_qlinear.h")

OK = 0
E_INVAL = 1
E_UNSUPPORTED = 2
E_HIP = 3
E_NODEV = 4
E_DECLINED = 5

DT_NONE = 0
DT_BF16 = 1
DT_F32 = 2
DT_I32 = 3

EPI_NONE = 0
EPI_GELU_TANH = 1

DEQUANT_ONCE_OFF = 0
DEQUANT_ONCE_ON = 1
DEQUANT_ONCE_AUTO = 2

TILE_AUTO = 0
TILE_TALL = 1
TILE_MID = 2
TILE_SKINNY = 3

LORA_AUTO = 0
LORA_NONE = 0
LORA_PAIR = 1
LORA_RFIRST = 2
LORA_FUSED = 3


class QWeightC(ctypes.Structure):
    """ltx25_qweight (mirrors QWeight, src/ltx25-metal-ops.h:45-57)."""

    _fields_ = [
        ("w", ctypes.c_void_p),
        ("codes", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("qbias", ctypes.c_void_p),
        ("bits", ctypes.c_int),
        ("group", ctypes.c_int),
        ("quantized", ctypes.c_int),
    ]


class RouteC(ctypes.Structure):
    """ltx25_route: what a linear runs on (ltx25_linear_route)."""

    _fields_ = [
        ("tile", ctypes.c_int),
        ("i8", ctypes.c_int),
        ("dequant_once", ctypes.c_int),
        ("splits", ctypes.c_int),
        ("slabs", ctypes.c_int),
        ("slab_rows", ctypes.c_int),
        ("scratch_bytes", ctypes.c_size_t),
    ]


class AttnC(ctypes.Structure):
    """ltx25_attn: how an attention call's heads lie in its tensors."""

    _fields_ = [
        ("heads", ctypes.c_int),
        ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("causal", ctypes.c_int),
        ("scale", ctypes.c_float),
        ("q_stride", ctypes.c_int64),
        ("k_stride", ctypes.c_int64),
        ("v_stride", ctypes.c_int64),
        ("out_stride", ctypes.c_int64),
    ]


class KVCacheC(ctypes.Structure):
    """ltx25_kv_cache: a paged cache of 8-bit keys and values."""

    _fields_ = [
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("pages", ctypes.c_int),
        ("page_tokens", ctypes.c_int),
        ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
    ]


class Mx4C(ctypes.Structure):
    """ltx25_mx4: rows in microscaled 4 bits."""

    _fields_ = [
        ("codes", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("rows", ctypes.c_int),
        ("K", ctypes.c_int),
    ]


class NormC(ctypes.Structure):
    """ltx25_norm: sizes and types of a norm's tensors."""

    _fields_ = [
        ("width", ctypes.c_int),
        ("layer", ctypes.c_int),
        ("eps", ctypes.c_float),
        ("residual_scale", ctypes.c_float),
        ("x_dtype", ctypes.c_int),
        ("mod_dtype", ctypes.c_int),
        ("weight_dtype", ctypes.c_int),
        ("mod_rows", ctypes.c_int),
        ("x_stride", ctypes.c_int64),
        ("x_out_stride", ctypes.c_int64),
        ("y_stride", ctypes.c_int64),
        ("mod_stride", ctypes.c_int64),
        ("out_stride", ctypes.c_int64),
    ]


class RotationC(ctypes.Structure):
    """ltx25_rotation: positions of one to four axes and their frequencies."""

    _fields_ = [
        ("head_dim", ctypes.c_int),
        ("rot_dim", ctypes.c_int),
        ("interleaved", ctypes.c_int),
        ("n_axes", ctypes.c_int),
        ("freq_heads", ctypes.c_int),
        ("pos_dtype", ctypes.c_int),
        ("freqs", ctypes.c_void_p),
        ("axes", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
    ]


class Ltx25Error(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"ltx25 error {code}: {msg}")
        self.code = code


_vp = ctypes.c_void_p
_i = ctypes.c_int
_sz = ctypes.c_size_t
_long = ctypes.c_long

# name -> (restype, argtypes)
SIGNATURES = {
    "ltx25_init": (_i, []),
    "ltx25_last_error": (ctypes.c_char_p, []),
    "ltx25_quant_available": (_i, []),
    "ltx25_linear_q": (_i, [_vp, _vp, ctypes.POINTER(QWeightC), _vp, _i, _vp, _i, _i, _i]),
    "ltx25_linear_q_ex": (_i, [_vp, _vp, ctypes.POINTER(QWeightC), _vp, _i, _vp, _i, _i, _i, _i]),
    "ltx25_linear_q_noalloc": (_i, [_vp, _vp, ctypes.POINTER(QWeightC), _vp, _i, _vp, _i, _i, _i,
                                    _i]),
    "ltx25_noalloc_scratch_bytes": (_sz, []),
    "ltx25_linear": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _i, _i, _i]),
    "ltx25_bias_add": (_i, [_vp, _vp, _vp, _i, _i, _i]),
    "ltx25_gelu_tanh": (_i, [_vp, _vp, _vp, _sz]),
    "ltx25_gate_heads": (_i, [_vp, _vp, _vp, _i, _i, _i]),
    "ltx25_probe_read": (_i, [_vp, _vp, _sz, _vp, _i]),
    "ltx25_probe_mfma": (_i, [_vp, _i, _i, _i, _vp]),
    "ltx25_probe_skinny_phases": (_i, [_vp, _vp, ctypes.POINTER(QWeightC), _vp, _i, _vp, _i, _i,
                                       _i, _i, _vp, _sz, ctypes.POINTER(ctypes.c_int)]),
    "ltx25_probe_tall_phases": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _i, _i, _i, _i, _vp, _sz]),
    "ltx25_probe_tall_i8_phases": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _i, _i, _vp,
                                        _sz]),
    "ltx25_dequant": (_i, [_vp, ctypes.POINTER(QWeightC), _vp, _i, _i]),
    "ltx25_set_dequant_once": (_i, [_i]),
    "ltx25_dequant_once_takes": (_i, [_i, _i, _i]),
    "ltx25_lora_add": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i]),
    "ltx25_lora_on_matrix_cores": (_i, [_i, _i, _i, _i]),
    "ltx25_set_lora_matrix_cores": (_i, [_i]),
    "ltx25_set_lora_route": (_i, [_i]),
    "ltx25_lora_route": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, ctypes.POINTER(_i)]),
    "ltx25_linear_q_lora": (_i, [_vp, _vp, ctypes.POINTER(QWeightC), _vp, _i, _vp, _vp, _i, _vp,
                                 _i, _i, _i, _i]),
    "ltx25_lora_fold_takes": (_i, [_i, _i, _i, _i, _i]),
    "ltx25_set_tile": (_i, [_i]),
    "ltx25_linear_route": (_i, [_i, _i, _i, _i, ctypes.POINTER(RouteC)]),
    "ltx25_set_i8_gemm": (_i, [_i]),
    "ltx25_i8_takes": (_i, [_i, _i, _i]),
    "ltx25_i8_quantize_rows": (_i, [_vp, _vp, _vp, _vp, _i, _i]),
    "ltx25_i8_quantize_qweight": (_i, [_vp, ctypes.POINTER(QWeightC), _vp, _vp, _i, _i]),
    "ltx25_i8_gemm": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _i, _i]),
    "ltx25_pack_codes": (_i, [_vp, _vp, _vp, _i, _i, _i]),
    "ltx25_unpack_codes": (_i, [_vp, _vp, _vp, _i, _i, _i]),
    "ltx25_quantize_affine": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i]),
    "ltx25_f16_to_bf16": (_i, [_vp, _vp, _vp, _sz]),
    "ltx25_qweight_infer": (_i, [_i, _long, _long, ctypes.POINTER(_i), ctypes.POINTER(_i)]),
    "ltx25_pack_open": (_i, [ctypes.c_char_p, ctypes.POINTER(_vp)]),
    "ltx25_pack_close": (None, [_vp]),
    "ltx25_pack_tensor": (_i, [_vp, ctypes.c_char_p, ctypes.c_char_p, ctypes.POINTER(_i),
                               ctypes.POINTER(_long)]),
    "ltx25_pack_metadata": (ctypes.c_char_p, [_vp, ctypes.c_char_p]),
    "ltx25_pack_read_bf16": (_i, [_vp, _vp, ctypes.c_char_p, ctypes.POINTER(_vp),
                                  ctypes.POINTER(_sz)]),
    "ltx25_pack_bind_qlinear": (_i, [_vp, _vp, ctypes.c_char_p, _i, ctypes.POINTER(_i),
                                     ctypes.POINTER(QWeightC), ctypes.c_char_p, _sz]),
    "ltx25_pack_quantizable": (_i, [ctypes.c_char_p, ctypes.c_char_p, _i]),
    "ltx25_attention": (_i, [_vp, ctypes.POINTER(AttnC), _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i,
                             _i]),
    "ltx25_attention_split": (_i, [_vp, ctypes.POINTER(AttnC), _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i,
                                   _i, _i, _vp, _sz]),
    "ltx25_attention_workspace": (_sz, [ctypes.POINTER(AttnC), _i, _i, _i]),
    "ltx25_kv_append": (_i, [_vp, ctypes.POINTER(KVCacheC), _vp, _i, _vp, _vp, ctypes.c_int64,
                             ctypes.c_int64, _vp, _vp, _i, _i]),
    "ltx25_kv_read": (_i, [_vp, ctypes.POINTER(KVCacheC), _vp, _i, _vp, _vp, ctypes.c_int64,
                           ctypes.c_int64, _vp, _vp, _i, _i]),
    "ltx25_attention_cached": (_i, [_vp, ctypes.POINTER(AttnC), ctypes.POINTER(KVCacheC), _vp, _i,
                                    _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _sz]),
    "ltx25_attention_cached_workspace": (_sz, [_i, _i, _i, _i, _i, _i]),
    "ltx25_mx4_code_bytes": (_sz, [_i, _i]),
    "ltx25_mx4_scale_bytes": (_sz, [_i, _i]),
    "ltx25_mx4_quantize_rows": (_i, [_vp, _vp, _i, ctypes.c_int64, ctypes.POINTER(Mx4C)]),
    "ltx25_mx4_dequant": (_i, [_vp, ctypes.POINTER(Mx4C), _vp, ctypes.c_int64]),
    "ltx25_mx4_pack": (_i, [_vp, _vp, _vp, ctypes.POINTER(Mx4C)]),
    "ltx25_mx4_unpack": (_i, [_vp, ctypes.POINTER(Mx4C), _vp, _vp]),
    "ltx25_mx4_gemm": (_i, [_vp, ctypes.POINTER(Mx4C), ctypes.POINTER(Mx4C), _vp, _i, _vp, _i, _vp,
                            _sz]),
    "ltx25_mx4_gemm_workspace": (_sz, [_i, _i, _i]),
    "ltx25_linear_mx4": (_i, [_vp, _vp, ctypes.c_int64, _i, ctypes.POINTER(Mx4C), _vp, _i, _vp, _i,
                              _vp, _sz]),
    "ltx25_linear_mx4_workspace": (_sz, [_i, _i, _i]),
    "ltx25_block_norm": (_i, [_vp, ctypes.POINTER(NormC), _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                              _vp, _vp, _i]),
    "ltx25_block_norm_mx4": (_i, [_vp, ctypes.POINTER(NormC), _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                  _vp, _vp, ctypes.POINTER(Mx4C), _i]),
    "ltx25_rope": (_i, [_vp, ctypes.POINTER(RotationC), _vp, _vp, _i, ctypes.c_int64,
                        ctypes.c_int64, _vp, _vp, _i, ctypes.c_int64, ctypes.c_int64, _i]),
    "ltx25_kv_append_rope": (_i, [_vp, ctypes.POINTER(KVCacheC), _vp, _i, _vp, _vp, ctypes.c_int64,
                                  ctypes.c_int64, _vp, _vp, ctypes.POINTER(RotationC), _i, _i]),
}

_lib = None


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load libltx25_qlinear.so once; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(
            f"{path} is missing: build it first (python -c 'import __graft_entry__ as g; g.build()')"
        )
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def last_error() -> str:
    return load().ltx25_last_error().decode()


def check(rc: int) -> None:
    if rc != OK:
        raise Ltx25Error(rc, last_error())


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


_torch = None
_raw_stream = None
_device_now = None


def _import_torch():
    """torch, imported on first use, and how its current stream's handle is read: the accessor
    that returns the handle alone where torch has it (0.07 us; torch.cuda.current_stream() builds
    a Stream object, 2.7 of the 8.2 us that a call took on the host)."""
    global _torch, _raw_stream, _device_now
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _raw_stream = raw if raw is not None else (
        lambda device: torch.cuda.current_stream(device).cuda_stream)
    # where a tensor already lies on a GPU, and torch's CUDA state is there with it (0.14 us less
    # than torch.cuda.current_device())
    _device_now = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    _torch = torch
    return torch


def _current_stream() -> int:
    torch = _torch or _import_torch()
    # current_device() initialises torch's CUDA state, as current_stream() does
    return _raw_stream(torch.cuda.current_device())


def _stream(stream) -> int | None:
    return stream if stream is not None else _current_stream()


def bias_dtype_of(bias) -> int:
    if bias is None:
        return DT_NONE
    torch = _torch or _import_torch()
    if bias.dtype == torch.bfloat16:
        return DT_BF16
    if bias.dtype == torch.float32:
        return DT_F32
    raise TypeError(f"bias must be bf16 or f32, got {bias.dtype}")


class QWeight:
    """A packed linear weight held in torch device tensors.

    codes: uint8 [N][K*bits/8] (the little-endian bytes of the u32 words),
    scales / qbias: bf16 [N][K/group].
    """

    def __init__(self, codes, scales, qbias, bits: int = 8, group: int = 64):
        self.codes, self.scales, self.qbias = codes, scales, qbias
        self.bits, self.group = bits, group

    def c(self) -> QWeightC:
        return QWeightC(None, _ptr(self.codes), _ptr(self.scales), _ptr(self.qbias),
                        self.bits, self.group, 1)


def dense_weight(w) -> QWeightC:
    return QWeightC(_ptr(w), None, None, None, 0, 0, 0)


def linear_q(x, w: QWeight, bias, y, M: int, K: int, N: int, epilogue: int = EPI_NONE,
             stream=None) -> None:
    cw = w.c()
    check(load().ltx25_linear_q_ex(_stream(stream), _ptr(x), ctypes.byref(cw), _ptr(bias),
                                   bias_dtype_of(bias), _ptr(y), M, K, N, epilogue))


def linear_q_noalloc(x, w: QWeight, bias, y, M: int, K: int, N: int, epilogue: int = EPI_NONE,
                     stream=None) -> None:
    """linear_q that allocates nothing: split-K partials in the library's fixed
    per-GPU scratch (noalloc_scratch_bytes()); overlapping calls on one GPU race."""
    cw = w.c()
    check(load().ltx25_linear_q_noalloc(_stream(stream), _ptr(x), ctypes.byref(cw), _ptr(bias),
                                        bias_dtype_of(bias), _ptr(y), M, K, N, epilogue))


def noalloc_scratch_bytes() -> int:
    return int(load().ltx25_noalloc_scratch_bytes())


def linear_q_lora(x, w: QWeight, bias, a, b, rank: int, y, M: int, K: int, N: int,
                  epilogue: int = EPI_NONE, stream=None) -> None:
    """The linear and its adapter (a [rank][K], b [N][rank]) in one call, the
    adapter added before the epilogue; folded into the GEMM where
    lora_fold_takes says so."""
    cw = w.c()
    check(load().ltx25_linear_q_lora(_stream(stream), _ptr(x), ctypes.byref(cw), _ptr(bias),
                                     bias_dtype_of(bias), _ptr(a), _ptr(b), rank, _ptr(y), M, K,
                                     N, epilogue))


def lora_fold_takes(M: int, K: int, N: int, rank: int, bits: int = 8) -> bool:
    return bool(load().ltx25_lora_fold_takes(M, K, N, rank, bits))


def linear(x, w, bias, y, M: int, K: int, N: int, stream=None) -> None:
    check(load().ltx25_linear(_stream(stream), _ptr(x), _ptr(w), _ptr(bias),
                              bias_dtype_of(bias), _ptr(y), M, K, N))


def bias_add(y, bias, M: int, N: int, stream=None) -> None:
    check(load().ltx25_bias_add(_stream(stream), _ptr(y), _ptr(bias), bias_dtype_of(bias), M, N))


def gelu_tanh(x, y, stream=None) -> None:
    check(load().ltx25_gelu_tanh(_stream(stream), _ptr(x), _ptr(y), x.numel()))


def gate_heads(y, logits, heads: int, tokens: int, head_dim: int, stream=None) -> None:
    check(load().ltx25_gate_heads(_stream(stream), _ptr(y), _ptr(logits), heads, tokens,
                                  head_dim))


# ---- attention (include/ltx25_attention.h) ------------------------------------------


def _tokens(name: str, t, shape) -> int:
    """The elements from a token to the next of a bf16 tensor [tokens][heads][head_dim] (its
    `shape`) whose tokens lie in one piece each, as a part of a fused projection's output does.
    A decode step can take as long on the host as on the GPU, hence the one test of what is
    usual."""
    stride = t.stride()
    if (len(shape) == 3 and stride[2] == 1 and stride[1] == shape[2] and shape[0] > 1
            and t.dtype is _torch.bfloat16):
        return stride[0]
    if len(shape) != 3 or t.dtype is not _torch.bfloat16:
        raise TypeError(f"{name} must be bf16 [tokens][heads][head_dim], got {t.dtype} "
                        f"{tuple(shape)}")
    n, heads, dim = shape
    if n > 0 and ((stride[2] != 1 and dim > 1) or (stride[1] != dim and heads > 1)):
        raise ValueError(f"{name}: a token's heads must lie side by side, got strides {stride}")
    return stride[0] if n > 1 else heads * dim   # one token: there is no next one


def _int32(name: str, t, count: int) -> None:
    if t.dtype is not _torch.int32 or t.numel() != count or not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous int32 with {count} elements, got {t.dtype} "
                        f"{tuple(t.shape)}")


def _table(t, batch: int) -> int:
    shape = t.shape
    if (t.dtype is not _torch.int32 or len(shape) != 2 or shape[0] != batch
            or not t.is_contiguous()):
        raise TypeError(f"table must be contiguous int32 [{batch}][pages], got {t.dtype} "
                        f"{tuple(shape)}")
    return shape[1]


def _lse(t, tokens: int, heads: int) -> None:
    if (t.dtype is not _torch.float32 or tuple(t.shape) != (tokens, heads)
            or not t.is_contiguous()):
        raise TypeError(f"lse must be contiguous float32 [{tokens}][{heads}], got {t.dtype} "
                        f"{tuple(t.shape)}")


def _reachable(names: str, *tensors) -> None:
    """Refuse a tensor in host memory, whose address means nothing to the kernels (None, and
    pinned memory, which they do reach, pass). Callers look at is_cuda themselves first: 0.2 us
    less for a call whose tensors all lie there."""
    for i, t in enumerate(tensors):
        if t is not None and not t.is_cuda and not t.is_pinned():
            raise ValueError(f"{names.split()[i]} must lie in the GPU's memory, got a tensor on "
                             f"{t.device}")


def _gpu_of(t):
    """Where memory of a call's own goes: beside t, or on the current GPU where t is pinned host
    memory (beside it would be pageable host memory, which no kernel reaches)."""
    return t.device if t.is_cuda else "cuda"


def attention(q, k, v, out, cu_q=None, cu_k=None, *, causal: bool, scale: float = 0.0, lse=None,
              workspace=None, stream=None) -> None:
    """Attention of packed sequences (ltx25_attention): q, out [total_q][heads][head_dim], k, v
    [total_k][kv_heads][head_dim] bf16, cu_q, cu_k int32 [batch + 1] (both None: one sequence),
    lse float32 [total_q][heads] or None. scale 0 is 1 / sqrt(head_dim).

    Few rows over many keys are split (ltx25_attention_split) in `workspace`, a uint8 tensor of
    attention_workspace() bytes; on torch's current stream one is allocated where none is given."""
    if _torch is None:
        _import_torch()
    q_shape, k_shape = q.shape, k.shape
    qs, ks = _tokens("q", q, q_shape), _tokens("k", k, k_shape)
    vs, os_ = _tokens("v", v, v.shape), _tokens("out", out, out.shape)
    nq, heads, dim = q_shape
    nk, kv_heads, kdim = k_shape
    if k_shape != v.shape or q_shape != out.shape or kdim != dim:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, out "
                         f"{tuple(out.shape)} do not fit each other")
    batch, pq, pk = 1, None, None
    if cu_q is not None or cu_k is not None:
        if cu_q is None or cu_k is None:
            raise ValueError("cu_q and cu_k go together")
        batch = cu_q.numel() - 1
        _int32("cu_q", cu_q, batch + 1)
        _int32("cu_k", cu_k, batch + 1)
        pq, pk = cu_q.data_ptr(), cu_k.data_ptr()
    if lse is not None:
        _lse(lse, nq, heads)
    if not (q.is_cuda and k.is_cuda and v.is_cuda and out.is_cuda
            and (cu_q is None or cu_q.is_cuda and cu_k.is_cuda)
            and (lse is None or lse.is_cuda) and (workspace is None or workspace.is_cuda)):
        _reachable("q k v out cu_q cu_k lse workspace", q, k, v, out, cu_q, cu_k, lse, workspace)
    a = AttnC(heads, kv_heads, dim, 1 if causal else 0, scale, qs, ks, vs, os_)
    # only such sizes can have parts: 8 tiles of 64 keys, 256 workgroups of 128 rows at most
    if nk > 448 * batch and nq * heads <= 65536 and (workspace is not None or stream is None):
        need = load().ltx25_attention_workspace(ctypes.byref(a), batch, nq, nk)
        if need > 0:
            if workspace is None:
                workspace = _torch.empty(need, dtype=_torch.uint8, device=_gpu_of(q))
            check(load().ltx25_attention_split(
                _stream(stream), ctypes.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                out.data_ptr(), _ptr(lse), pq, pk, batch, nq, nk, workspace.data_ptr(),
                workspace.numel() * workspace.element_size()))
            return
    check(load().ltx25_attention(_stream(stream), ctypes.byref(a), q.data_ptr(), k.data_ptr(),
                                 v.data_ptr(), out.data_ptr(), _ptr(lse), pq, pk, batch, nq, nk))


def attention_workspace(heads: int, kv_heads: int, head_dim: int, batch: int, total_q: int,
                        total_k: int) -> int:
    """Bytes of workspace in which attention splits the keys of few rows
    (ltx25_attention_workspace); 0 where it does not."""
    a = AttnC(heads, kv_heads, head_dim, 0, 0.0, 0, 0, 0, 0)
    return int(load().ltx25_attention_workspace(ctypes.byref(a), batch, total_q, total_k))


class KVCache:
    """A paged 8-bit cache held in torch device tensors (ltx25_kv_cache).

    k: int8 [pages][kv_heads][page_tokens][head_dim], v: int8
    [pages][kv_heads][head_dim][page_tokens], k_scale / v_scale: float32 [pages][kv_heads].

    Calls work on the tensors given here, whose contents may change at will; a cache in other
    tensors is another KVCache (assigning to k, v, k_scale or v_scale is refused, since the calls
    would go on with the old ones' memory).
    """

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    def __init__(self, k, v, k_scale, v_scale):
        torch = _torch or _import_torch()
        pages, heads, page, dim = k.shape
        if (k.dtype != torch.int8 or v.dtype != torch.int8
                or tuple(v.shape) != (pages, heads, dim, page)
                or not (k.is_contiguous() and v.is_contiguous())):
            raise TypeError(f"k and v must be contiguous int8 [pages][kv_heads][tokens][width] and "
                            f"[pages][kv_heads][width][tokens], got {k.dtype} {tuple(k.shape)}, "
                            f"{v.dtype} {tuple(v.shape)}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) or not t.is_contiguous():
                raise TypeError(f"{name} must be contiguous float32 [{pages}][{heads}], got "
                                f"{t.dtype} {tuple(t.shape)}")
        self._tensors = (k, v, k_scale, v_scale)
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = pages, heads, page, dim
        self._c = KVCacheC(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), pages, page, heads, dim)
        self.checked = False

    @classmethod
    def empty(cls, pages: int, page_tokens: int, kv_heads: int, head_dim: int, device="cuda"):
        torch = _torch or _import_torch()
        k = torch.empty((pages, kv_heads, page_tokens, head_dim), dtype=torch.int8, device=device)
        v = torch.empty((pages, kv_heads, head_dim, page_tokens), dtype=torch.int8, device=device)
        scales = [torch.empty((pages, kv_heads), dtype=torch.float32, device=device)
                  for _ in range(2)]
        return cls(k, v, *scales)

    def c(self) -> KVCacheC:
        return self._c

    def check(self) -> None:
        """Refuse a cache in host memory or of several GPUs, which may be made but not given to a
        kernel."""
        names = "cache.k cache.v cache.k_scale cache.v_scale"
        _reachable(names, *self._tensors)
        on = [t.get_device() for t in self._tensors]
        for name, t, at in zip(names.split(), self._tensors, on):
            if t.is_cuda and at != max(on):
                raise ValueError(f"{name} lies on {t.device}, others of the cache on cuda:{max(on)}")
        self.checked = True


def _moved(cache: KVCache, table, k, v, cu, start, looked: bool = False):
    """The arguments that appending and reading share; `looked`: the caller looks at where the
    tensors lie."""
    shape = k.shape
    ks, vs = _tokens("k", k, shape), _tokens("v", v, v.shape)
    total, heads, dim = shape
    if shape != v.shape or heads != cache.kv_heads or dim != cache.head_dim:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit the cache's "
                         f"{cache.kv_heads} heads of width {cache.head_dim}")
    batch = start.numel()
    stride = _table(table, batch)
    _int32("cu", cu, batch + 1)
    _int32("start", start, batch)
    if not cache.checked:
        cache.check()
    if not (looked or table.is_cuda and k.is_cuda and v.is_cuda and cu.is_cuda and start.is_cuda):
        _reachable("table k v cu start", table, k, v, cu, start)
    return (ctypes.byref(cache.c()), table.data_ptr(), stride, k.data_ptr(), v.data_ptr(), ks, vs,
            cu.data_ptr(), start.data_ptr(), batch, total)


def kv_append(cache: KVCache, table, k, v, cu, start, stream=None) -> None:
    """Quantize new keys and values [total][kv_heads][head_dim] into the cache
    (ltx25_kv_append): sequence b's tokens cu[b] .. cu[b + 1] - 1 become tokens start[b] ... of
    its pages table[b]."""
    args = _moved(cache, table, k, v, cu, start)
    check(load().ltx25_kv_append(_stream(stream), *args))


def kv_read(cache: KVCache, table, k, v, cu, start, stream=None) -> None:
    """Read tokens start[b] ... of each sequence back into k, v [total][kv_heads][head_dim] at
    cu[b] ... (ltx25_kv_read)."""
    args = _moved(cache, table, k, v, cu, start)
    check(load().ltx25_kv_read(_stream(stream), *args))


def attention_cached_workspace(batch: int, q_len: int, heads: int, kv_heads: int, head_dim: int,
                               max_len: int) -> int:
    """Bytes of workspace that attention_cached needs (ltx25_attention_cached_workspace); not monotone
    in the sizes."""
    return int(load().ltx25_attention_cached_workspace(batch, q_len, heads, kv_heads, head_dim,
                                                       max_len))


def attention_cached(cache: KVCache, table, lens, q, out, q_len: int, max_len: int, workspace=None,
                     *, causal: bool = True, scale: float = 0.0, lse=None, stream=None) -> None:
    """Attention of each sequence's q_len newest tokens over its cache (ltx25_attention_cached):
    q, out [batch * q_len][heads][head_dim] bf16, lens int32 [batch] with the queries' own tokens
    counted, workspace a uint8 tensor of attention_cached_workspace() bytes."""
    shape = q.shape
    qs, os_ = _tokens("q", q, shape), _tokens("out", out, out.shape)
    nq, heads, dim = shape
    batch = lens.numel()
    if shape != out.shape or nq != batch * q_len:
        raise ValueError(f"q {tuple(q.shape)} and out {tuple(out.shape)} are not {batch} x {q_len} "
                         f"tokens")
    pages = _table(table, batch)
    _int32("lens", lens, batch)
    if lse is not None:
        _lse(lse, nq, heads)
    if not cache.checked:
        cache.check()
    if not (table.is_cuda and lens.is_cuda and q.is_cuda and out.is_cuda
            and (workspace is None or workspace.is_cuda) and (lse is None or lse.is_cuda)):
        _reachable("table lens q out workspace lse", table, lens, q, out, workspace, lse)
    a = AttnC(heads, cache.kv_heads, dim, 1 if causal else 0, scale, qs, 0, 0, os_)
    at, held = None, 0
    if workspace is not None:
        at, held = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    check(load().ltx25_attention_cached(_stream(stream), ctypes.byref(a), ctypes.byref(cache.c()),
                                        table.data_ptr(), pages, lens.data_ptr(), q.data_ptr(),
                                        out.data_ptr(), _ptr(lse), batch, q_len, max_len, at,
                                        held))


# ---- microscaled 4 bits (include/ltx25_mx4.h) ------------------------------------------


def _on_device(stream, names: str, tensors) -> int:
    """The stream to launch on: the caller's, or the current one of the current device, where the
    tensors must lie (pinned host memory is reached from any). One look at each tensor; what it
    finds is named afterwards."""
    if stream is not None:
        for t in tensors:
            if t is not None and not t.is_cuda:
                _reachable(names, *tensors)
        return stream
    try:
        device = _device_now()
    except Exception:
        _reachable(names, *tensors)   # without a GPU: a tensor in host memory is what is wrong
        raise
    for t in tensors:
        if t is not None and t.get_device() != device:
            _reachable(names, *tensors)
            for name, u in zip(names.split(), tensors):
                if u is not None and u.is_cuda and u.get_device() != device:
                    raise ValueError(f"{name} lies on {u.device}, the current device is "
                                     f"cuda:{device}")
            break
    return _raw_stream(device)


def _callers(stream, what: str) -> None:
    """Refuse memory of the binding's own on a stream of the caller's: torch's allocator orders it
    after the work of its own current stream alone, which may still read what lay there."""
    if stream is not None:
        raise ValueError(f"on a stream of the caller's, {what} must be the caller's too")


def _float_type(name: str, t) -> int:
    if t.dtype is _torch.bfloat16:
        return DT_BF16
    if t.dtype is _torch.float32:
        return DT_F32
    raise TypeError(f"{name} must be bf16 or f32, got {t.dtype}")


def _rows(name: str, t, width: int | None = None) -> int:
    """The elements from a row to the next of a tensor [rows][width] whose rows lie in one piece
    each."""
    shape = t.shape
    if len(shape) != 2 or (width is not None and shape[1] != width):
        raise ValueError(f"{name} must be [rows][{'width' if width is None else width}], got "
                         f"{tuple(shape)}")
    stride = t.stride()
    if shape[1] > 1 and stride[1] != 1:
        raise ValueError(f"{name}: a row's values must lie side by side, got strides {stride}")
    return stride[0] if shape[0] > 1 else (shape[1] + 7) // 8 * 8   # one row: there is no next


def _alike(name: str, t, shape, dtype) -> int:
    """_rows of a tensor that must have this shape and type."""
    if t.dtype is not dtype or t.shape != shape:
        raise TypeError(f"{name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}: a row's values must lie side by side, got strides {stride}")
    return stride[0] if shape[0] > 1 else (shape[1] + 7) // 8 * 8


class MX4:
    """`rows` rows of K values in microscaled 4 bits, held in torch device tensors (ltx25_mx4): uint8
    `codes` and `scales` in the order of the matrix cores' reads, mx4_code_bytes() and
    mx4_scale_bytes() long.

    Calls work on the tensors given here, whose contents may change at will.
    """

    codes = property(lambda self: self._tensors[0])
    scales = property(lambda self: self._tensors[1])

    def __init__(self, codes, scales, rows: int, K: int):
        torch = _torch or _import_torch()
        if rows < 0 or K <= 0 or K % 32:
            raise ValueError(f"{rows} rows of {K} values: K is a multiple of 32")
        for name, t, need in (("codes", codes, mx4_code_bytes(rows, K)),
                              ("scales", scales, mx4_scale_bytes(rows, K))):
            if t.dtype != torch.uint8 or t.numel() != need or not t.is_contiguous():
                raise TypeError(f"{name} must be contiguous uint8 with {need} elements, got "
                                f"{t.dtype} {tuple(t.shape)}")
        if codes.device != scales.device or codes.is_cuda != scales.is_cuda:
            raise ValueError(f"codes lie on {codes.device}, scales on {scales.device}")
        # (calls look at the codes alone)
        if not codes.is_cuda and codes.is_pinned() != scales.is_pinned():
            raise ValueError("of codes and scales in host memory one is pinned and one is not")
        self._tensors = (codes, scales)
        self.rows, self.K = rows, K
        self._c = Mx4C(_ptr(codes), _ptr(scales), rows, K)
        self.by_reference = ctypes.byref(self._c)

    @classmethod
    def empty(cls, rows: int, K: int, device="cuda"):
        torch = _torch or _import_torch()
        return cls(torch.empty(mx4_code_bytes(rows, K), dtype=torch.uint8, device=device),
                   torch.empty(mx4_scale_bytes(rows, K), dtype=torch.uint8, device=device), rows, K)

    @classmethod
    def packed(cls, codes, scales, stream=None, out=None):
        """From uint8 codes [rows][K / 2], the earlier of a byte's two values in its low half, and
        scales [rows][K / 32], as checkpoints hold them (ltx25_mx4_pack): into `out`, an MX4 of
        their size, or on torch's current stream into a new one."""
        torch = _torch or _import_torch()
        rows, half = codes.shape
        if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or half % 16
                or tuple(scales.shape) != (rows, half // 16)
                or not (codes.is_contiguous() and scales.is_contiguous())):
            raise TypeError(f"codes and scales must be contiguous uint8 [rows][K / 2] and "
                            f"[rows][K / 32], got {codes.dtype} {tuple(codes.shape)}, "
                            f"{scales.dtype} {tuple(scales.shape)}")
        if out is None:
            _callers(stream, "out")
        elif out.rows != rows or out.K != 2 * half:
            raise ValueError(f"out has {out.rows} rows of {out.K}, not {rows} of {2 * half}")
        at = _on_device(stream, "codes scales out.codes",
                        (codes, scales, None if out is None else out.codes))
        q = cls.empty(rows, 2 * half, _gpu_of(codes)) if out is None else out
        check(load().ltx25_mx4_pack(at, _ptr(codes), _ptr(scales), ctypes.byref(q.c())))
        return q

    def unpacked(self, stream=None, codes=None, scales=None):
        """codes [rows][K / 2] and scales [rows][K / 32] as packed() takes them (ltx25_mx4_unpack):
        into those given, or on torch's current stream into new ones."""
        torch = _torch or _import_torch()
        shapes = (self.rows, self.K // 2), (self.rows, self.K // 32)
        for name, t, shape in zip(("codes", "scales"), (codes, scales), shapes):
            if t is None:
                _callers(stream, name)
            elif t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous():
                raise TypeError(f"{name} must be contiguous uint8 {list(shape)}, got {t.dtype} "
                                f"{tuple(t.shape)}")
        at = _on_device(stream, "q.codes codes scales", (self.codes, codes, scales))
        codes, scales = (torch.empty(shape, dtype=torch.uint8, device=_gpu_of(self.codes))
                         if t is None else t for t, shape in zip((codes, scales), shapes))
        check(load().ltx25_mx4_unpack(at, ctypes.byref(self.c()), _ptr(codes), _ptr(scales)))
        return codes, scales

    def c(self) -> Mx4C:
        return self._c


def mx4_code_bytes(rows: int, K: int) -> int:
    return int(load().ltx25_mx4_code_bytes(rows, K))


def mx4_scale_bytes(rows: int, K: int) -> int:
    return int(load().ltx25_mx4_scale_bytes(rows, K))


def mx4_quantize_rows(x, q: MX4, stream=None) -> None:
    """Codes of the rows of x, bf16 or f32 [rows][K] (ltx25_mx4_quantize_rows)."""
    if _torch is None:
        _import_torch()
    kind = _float_type("x", x)
    stride = _rows("x", x, q.K)
    if x.shape[0] != q.rows:
        raise ValueError(f"x {tuple(x.shape)} does not have q's {q.rows} rows")
    check(load().ltx25_mx4_quantize_rows(_on_device(stream, "x q.codes", (x, q.codes)),
                                         x.data_ptr(), kind, stride, q.by_reference))


def mx4_dequant(q: MX4, out, stream=None) -> None:
    """The values as bf16 [rows][K] (ltx25_mx4_dequant)."""
    if _torch is None:
        _import_torch()
    stride = _rows("out", out, q.K)
    if out.dtype is not _torch.bfloat16 or out.shape[0] != q.rows:
        raise TypeError(f"out must be bf16 [{q.rows}][{q.K}], got {out.dtype} {tuple(out.shape)}")
    check(load().ltx25_mx4_dequant(_on_device(stream, "out q.codes", (out, q.codes)),
                                   q.by_reference, out.data_ptr(), stride))


def mx4_gemm_workspace(M: int, K: int, N: int) -> int:
    return int(load().ltx25_mx4_gemm_workspace(M, K, N))


def linear_mx4_workspace(M: int, K: int, N: int) -> int:
    return int(load().ltx25_linear_mx4_workspace(M, K, N))


def _product(y, bias, M: int, K: int, N: int, workspace, need_of, stream):
    """What the two products check alike; the workspace, allocated on torch's current stream
    where none is given (one that is given the library checks)."""
    if y.dtype is not _torch.bfloat16 or y.shape != (M, N) or not y.is_contiguous():
        raise TypeError(f"y must be contiguous bf16 [{M}][{N}], got {y.dtype} {tuple(y.shape)}")
    if bias is not None and (bias.shape != (N,) or not bias.is_contiguous()):
        raise TypeError(f"bias must be contiguous [{N}], got {tuple(bias.shape)}")
    if workspace is None:
        need = need_of(M, K, N)
        if need:
            _callers(stream, f"a workspace of {need} bytes")
            workspace = _torch.empty(need, dtype=_torch.uint8, device=_gpu_of(y))
    return workspace


def _held(workspace) -> tuple:
    if workspace is None:
        return None, 0
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def mx4_gemm(x: MX4, w: MX4, bias, y, epilogue: int = EPI_NONE, workspace=None,
             stream=None) -> None:
    """y [M][N] = epilogue(x . w^T + bias) of two coded operands (ltx25_mx4_gemm)."""
    if _torch is None:
        _import_torch()
    kind = bias_dtype_of(bias)
    workspace = _product(y, bias, x.rows, x.K, w.rows, workspace, mx4_gemm_workspace, stream)
    at = _on_device(stream, "x.codes w.codes y bias workspace",
                    (x.codes, w.codes, y, bias, workspace))
    check(load().ltx25_mx4_gemm(at, x.by_reference, w.by_reference, _ptr(bias), kind, y.data_ptr(),
                                epilogue, *_held(workspace)))


def linear_mx4(x, w: MX4, bias, y, epilogue: int = EPI_NONE, workspace=None, stream=None) -> None:
    """y [M][N] = epilogue(coded x . w^T + bias), x bf16 [M][K] (ltx25_linear_mx4)."""
    if _torch is None:
        _import_torch()
    kind = bias_dtype_of(bias)
    if x.dtype is not _torch.bfloat16:
        raise TypeError(f"x must be bf16, got {x.dtype}")
    stride = _rows("x", x, w.K)
    M, N = x.shape[0], w.rows
    workspace = _product(y, bias, M, w.K, N, workspace, linear_mx4_workspace, stream)
    at = _on_device(stream, "x w.codes y bias workspace", (x, w.codes, y, bias, workspace))
    check(load().ltx25_linear_mx4(at, x.data_ptr(), stride, M, w.by_reference, _ptr(bias), kind,
                                  y.data_ptr(), epilogue, *_held(workspace)))


# ---- around a block's linears and attention (include/ltx25_block.h) -----------------------


def block_norm(x, out, *, y=None, x_out=None, gate=None, post_weight=None, weight=None, scale=None,
               shift=None, rows=None, layer: bool = False, eps: float = 1e-6,
               residual_scale: float = 1.0, stream=None) -> None:
    """The end of one block and the start of the next (ltx25_block_norm):

        u = y, or norm(y) post_weight;  x_out = residual_scale x + gate u
        out = norm(x_out) weight (1 + scale) + shift

    x, x_out bf16 or f32 [tokens][width]; y bf16; weight, post_weight [width]; gate, scale, shift
    [mod_rows][width] of one type and row stride; rows int32 [tokens]. Without y, out is of x. out
    is bf16, an MX4 (ltx25_block_norm_mx4), or None where y is given."""
    if _torch is None:
        _import_torch()
    shape = x.shape
    kind, xs = _float_type("x", x), _rows("x", x)
    tokens, width = shape
    xos = ys = ms = os_ = mod_rows = 0
    mod = weights = DT_BF16
    if y is not None:
        ys = _alike("y", y, shape, _torch.bfloat16)
        if x_out is None:
            raise ValueError("x_out must be given with y (it may be x)")
    if x_out is not None:
        xos = _alike("x_out", x_out, shape, x.dtype)
    if gate is not None or scale is not None or shift is not None:
        first = None
        for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
            if t is None:
                continue
            if first is None:
                first = t
                mod, ms, mod_rows = _float_type(name, t), _rows(name, t, width), t.shape[0]
            elif (t.dtype != first.dtype or t.shape != first.shape
                  or _rows(name, t, width) != ms):
                raise ValueError(f"{name}: gate, scale and shift must be alike in type, rows and "
                                 f"row stride")
    if rows is not None:
        _int32("rows", rows, tokens)
    for name, t in (("post_weight", post_weight), ("weight", weight)):
        if t is None:
            continue
        weights = _float_type(name, t)
        if (t.shape != shape[1:] or not t.is_contiguous()
                or (weight is not None and t.dtype != weight.dtype)):
            raise TypeError(f"{name} must be contiguous [{width}], and of one type with the other "
                            f"weight, got {t.dtype} {tuple(t.shape)}")
    if isinstance(out, MX4):
        if out.rows != tokens or out.K != width:
            raise ValueError(f"out has {out.rows} rows of {out.K}, not {tokens} of {width}")
        held, fn, to = out.codes, load().ltx25_block_norm_mx4, out.by_reference
    else:
        if out is not None:
            os_ = _alike("out", out, shape, _torch.bfloat16)
        held, fn, to = out, load().ltx25_block_norm, _ptr(out)
    tensors = (x, y, x_out, post_weight, gate, weight, scale, shift, rows, held)
    at = _on_device(stream, "x y x_out post_weight gate weight scale shift rows out", tensors)
    n = NormC(width, 1 if layer else 0, eps, residual_scale, kind, mod, weights, mod_rows, xs, xos,
              ys, ms, os_)
    check(fn(at, ctypes.byref(n), *[t if t is None else t.data_ptr() for t in tensors[:9]], to,
             tokens))


def _rotation(head_dim: int, freqs, axes, positions, tokens: int, interleaved: bool) -> RotationC:
    shape = freqs.shape
    if (freqs.dtype is not _torch.float32 or len(shape) != 2 or shape[1] == 0
            or not freqs.is_contiguous()):
        raise TypeError(f"freqs must be contiguous float32 [1 or heads][pairs], got {freqs.dtype} "
                        f"{tuple(shape)}")
    pa = pp = None
    if axes is not None:
        if axes.dtype is not _torch.int32 or axes.shape != shape or not axes.is_contiguous():
            raise TypeError(f"axes must be contiguous int32 {tuple(shape)}, got {axes.dtype} "
                            f"{tuple(axes.shape)}")
        pa = axes.data_ptr()
    kind, n_axes = DT_F32, 1
    if positions is not None:
        ps = positions.shape
        if len(ps) != 2 or ps[0] != tokens or not positions.is_contiguous():
            raise TypeError(f"positions must be contiguous [{tokens}][axes], got {tuple(ps)}")
        if positions.dtype is _torch.int32:
            kind = DT_I32
        elif positions.dtype is not _torch.float32:
            raise TypeError(f"positions must be int32 or float32, got {positions.dtype}")
        n_axes, pp = ps[1], positions.data_ptr()
    return RotationC(head_dim, 2 * shape[1], 1 if interleaved else 0, n_axes, shape[0], kind,
                     freqs.data_ptr(), pa, pp)


def _rotated(name: str, t, to, tokens: int, dim: int) -> tuple:
    """What ltx25_rope takes of a tensor: pointers, heads and strides."""
    if t is None:
        return (None, None, 0, 0, 0)
    shape = t.shape
    stride = _tokens(name, t, shape)
    if shape[0] != tokens or shape[2] != dim:
        raise ValueError(f"{name} {tuple(shape)} is not {tokens} tokens of heads of {dim}")
    if to is None:
        return (t.data_ptr(), t.data_ptr(), shape[1], stride, stride)
    if to.shape != shape:
        raise ValueError(f"{name}_out {tuple(to.shape)} is not {name}'s {tuple(shape)}")
    return (t.data_ptr(), to.data_ptr(), shape[1], stride, _tokens(name + "_out", to, shape))


def rope(q, k, positions, freqs, axes=None, *, q_out=None, k_out=None, interleaved: bool = False,
         stream=None) -> None:
    """Rotates queries and keys, bf16 [tokens][heads][head_dim], by their positions (ltx25_rope), in
    place or into q_out and k_out. Either of q and k may be None.

    positions int32 or float32 [tokens][axes]; freqs float32 [1 or heads][pairs], axes int32 of the
    same shape: pair p turns by positions[token][axes[p]] * freqs[p]. interleaved: pair p is
    channels 2 p and 2 p + 1, else p and p + pairs."""
    if _torch is None:
        _import_torch()
    given = q if q is not None else k
    if given is None or (q is None and q_out is not None) or (k is None and k_out is not None):
        raise ValueError("rope rotates q, k or both, and an output goes with its input")
    tokens, _, dim = given.shape
    args = _rotated("q", q, q_out, tokens, dim) + _rotated("k", k, k_out, tokens, dim)
    r = _rotation(dim, freqs, axes, positions, tokens, interleaved)
    at = _on_device(stream, "q k positions freqs axes q_out k_out",
                    (q, k, positions, freqs, axes, q_out, k_out))
    check(load().ltx25_rope(at, ctypes.byref(r), *args, tokens))


def kv_append_rope(cache: KVCache, table, k, v, cu, start, freqs, axes=None, positions=None, *,
                   interleaved: bool = False, stream=None) -> None:
    """kv_append with the keys rotated on the way (ltx25_kv_append_rope): the bits of rope on k and
    kv_append. positions [total][axes] as for rope, or None: a token's place in its sequence on
    every axis."""
    args = _moved(cache, table, k, v, cu, start, True)
    r = _rotation(cache.head_dim, freqs, axes, positions, k.shape[0], interleaved)
    at = _on_device(stream, "freqs axes positions k v table cu start cache.k",
                    (freqs, axes, positions, k, v, table, cu, start, cache.k))
    check(load().ltx25_kv_append_rope(at, *args[:9], ctypes.byref(r), *args[9:]))


def probe_read(src, nbytes: int, sink, blocks: int, stream=None) -> None:
    """The streaming-read ceiling probe (ltx25_probe_read)."""
    check(load().ltx25_probe_read(_stream(stream), _ptr(src), nbytes, _ptr(sink), blocks))


def probe_mfma(iters: int, random: bool, waves_per_simd: int, out, stream=None) -> None:
    """The MFMA-stream ceiling probe (ltx25_probe_mfma)."""
    check(load().ltx25_probe_mfma(_stream(stream), iters, 1 if random else 0, waves_per_simd,
                                  _ptr(out)))


def probe_skinny_phases(x, w: QWeight, bias, y, M: int, K: int, N: int, k_chunk: int, stamps,
                        stamps_bytes: int, stream=None) -> int:
    """One w8 linear on the M <= 128 kernel's phase-stamp instantiation
    (ltx25_probe_skinny_phases); returns the number of K splits."""
    cw = w.c()
    splits = ctypes.c_int(0)
    check(load().ltx25_probe_skinny_phases(_stream(stream), _ptr(x), ctypes.byref(cw), _ptr(bias),
                                           bias_dtype_of(bias), _ptr(y), M, K, N, k_chunk,
                                           _ptr(stamps), stamps_bytes, ctypes.byref(splits)))
    return splits.value


def probe_tall_phases(x, w_bf16, bias, y, M: int, K: int, N: int, epilogue: int, stamps,
                      stamps_bytes: int, stream=None) -> None:
    """The dense bf16 GEMM on the 256 x 256 tile's phase-stamp instantiation
    (ltx25_probe_tall_phases)."""
    check(load().ltx25_probe_tall_phases(_stream(stream), _ptr(x), _ptr(w_bf16), _ptr(bias),
                                         bias_dtype_of(bias), _ptr(y), M, K, N, epilogue,
                                         _ptr(stamps), stamps_bytes))


def probe_tall_i8_phases(xq, sx, wq, sw, bias, y, M: int, K: int, N: int, stamps,
                         stamps_bytes: int, stream=None) -> None:
    """The int8 GEMM on the 256 x 256 tile's phase-stamp instantiation
    (ltx25_probe_tall_i8_phases)."""
    check(load().ltx25_probe_tall_i8_phases(_stream(stream), _ptr(xq), _ptr(sx), _ptr(wq),
                                            _ptr(sw), _ptr(bias), bias_dtype_of(bias), _ptr(y),
                                            M, K, N, _ptr(stamps), stamps_bytes))


def dequant(w: QWeight, out, N: int, K: int, stream=None) -> None:
    cw = w.c()
    check(load().ltx25_dequant(_stream(stream), ctypes.byref(cw), _ptr(out), N, K))


def quantize_affine(w_f32, codes, scales, qbias, N: int, K: int, bits: int = 8,
                    group: int = 64, stream=None) -> None:
    check(load().ltx25_quantize_affine(_stream(stream), _ptr(w_f32), _ptr(codes), _ptr(scales),
                                       _ptr(qbias), N, K, bits, group))


def pack_codes(q, codes, N: int, K: int, bits: int, stream=None) -> None:
    check(load().ltx25_pack_codes(_stream(stream), _ptr(q), _ptr(codes), N, K, bits))


def unpack_codes(codes, q, N: int, K: int, bits: int, stream=None) -> None:
    check(load().ltx25_unpack_codes(_stream(stream), _ptr(codes), _ptr(q), N, K, bits))


def f16_to_bf16(src, dst, stream=None) -> None:
    check(load().ltx25_f16_to_bf16(_stream(stream), _ptr(src), _ptr(dst), src.numel()))


def set_dequant_once(mode) -> None:
    """DEQUANT_ONCE_OFF / _ON / _AUTO (the default); a bool means OFF / ON."""
    check(load().ltx25_set_dequant_once(int(mode)))


def dequant_once_takes(M: int, K: int, N: int) -> bool:
    return bool(load().ltx25_dequant_once_takes(M, K, N))


def lora_add(x, a, b, y, M: int, K: int, N: int, rank: int, r=None, d=None,
             stream=None) -> None:
    """y += (x . a^T) . b^T in place (MetalOps::lora_add). r: optional caller scratch
    [M][rank] (16-byte aligned) that receives r = bf16(x . a^T) on the r-first route and
    on the GEMM pair when rank % 64 == 0; d is unused."""
    check(load().ltx25_lora_add(_stream(stream), _ptr(x), _ptr(a), _ptr(b), _ptr(y), _ptr(r),
                                _ptr(d), M, K, N, rank))


def lora_on_matrix_cores(M: int, K: int, N: int, rank: int) -> bool:
    return bool(load().ltx25_lora_on_matrix_cores(M, K, N, rank))


def set_lora_matrix_cores(on: bool) -> None:
    check(load().ltx25_set_lora_matrix_cores(1 if on else 0))


def set_lora_route(route: int) -> None:
    """LORA_AUTO / LORA_PAIR / LORA_RFIRST / LORA_FUSED for every later lora_add."""
    check(load().ltx25_set_lora_route(route))


def lora_route(x, a, b, y, M: int, K: int, N: int, rank: int) -> int:
    """The LORA_* route lora_add would take; raises when a forced route cannot."""
    r = ctypes.c_int(-1)
    check(load().ltx25_lora_route(_ptr(x), _ptr(a), _ptr(b), _ptr(y), M, K, N, rank,
                                  ctypes.byref(r)))
    return r.value


def set_tile(tile: int) -> None:
    """TILE_AUTO / TILE_TALL / TILE_MID / TILE_SKINNY for every later linear."""
    check(load().ltx25_set_tile(tile))


def linear_route(M: int, K: int, N: int, bits: int = 8) -> dict:
    """The route a linear takes (bits 4 / 8 codes, 16 dense), as a dict."""
    r = RouteC()
    check(load().ltx25_linear_route(M, K, N, bits, ctypes.byref(r)))
    return {f: getattr(r, f) for f, _ in RouteC._fields_}


def set_i8_gemm(on: bool) -> None:
    check(load().ltx25_set_i8_gemm(1 if on else 0))


def i8_takes(M: int, K: int, N: int) -> bool:
    return bool(load().ltx25_i8_takes(M, K, N))


def i8_quantize_rows(x, q, scale, M: int, K: int, stream=None) -> None:
    check(load().ltx25_i8_quantize_rows(_stream(stream), _ptr(x), _ptr(q), _ptr(scale), M, K))


def i8_quantize_qweight(w: QWeight, wq, sw, N: int, K: int, stream=None) -> None:
    cw = w.c()
    check(load().ltx25_i8_quantize_qweight(_stream(stream), ctypes.byref(cw), _ptr(wq), _ptr(sw),
                                           N, K))


def i8_gemm(xq, sx, wq, sw, bias, y, acc, M: int, K: int, N: int, stream=None) -> None:
    check(load().ltx25_i8_gemm(_stream(stream), _ptr(xq), _ptr(sx), _ptr(wq), _ptr(sw),
                               _ptr(bias), bias_dtype_of(bias), _ptr(y), _ptr(acc), M, K, N))


def qweight_infer(K: int, scales_cols: int, codes_cols: int, group: int = 0) -> tuple[int, int]:
    """(bits, group) from packed shapes; raises Ltx25Error when they do not close."""
    b = ctypes.c_int(0)
    g = ctypes.c_int(group)
    check(load().ltx25_qweight_infer(K, scales_cols, codes_cols, ctypes.byref(b), ctypes.byref(g)))
    return b.value, g.value


def _pack_stream(stream):
    """torch's current stream when a device is visible; NULL otherwise, so
    that host-side validation runs (and fails) without touching a device."""
    if stream is not None:
        return stream
    torch = _torch or _import_torch()
    return _current_stream() if torch.cuda.is_available() else None


class Pack:
    """An open .safetensors pack (ltx25_pack_*). Device tensors it binds stay
    valid until close()."""

    def __init__(self, path: str):
        h = ctypes.c_void_p()
        check(load().ltx25_pack_open(path.encode(), ctypes.byref(h)))
        self._h = h
        self.group = 0   # the checkpoint's group, set by the first quantized bind

    def close(self) -> None:
        if self._h:
            load().ltx25_pack_close(self._h)
            self._h = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def tensor(self, name: str) -> tuple[str, tuple[int, ...]]:
        dt = ctypes.create_string_buffer(16)
        nd = ctypes.c_int(0)
        dims = (ctypes.c_long * 8)()
        check(load().ltx25_pack_tensor(self._h, name.encode(), dt, ctypes.byref(nd), dims))
        return dt.value.decode(), tuple(dims[i] for i in range(nd.value))

    def metadata(self, key: str):
        v = load().ltx25_pack_metadata(self._h, key.encode())
        return None if v is None else v.decode()

    def read_bf16(self, name: str, stream=None) -> tuple[int, int]:
        """(device pointer, element count) of the tensor as bf16."""
        p = ctypes.c_void_p()
        n = ctypes.c_size_t(0)
        check(load().ltx25_pack_read_bf16(self._h, _pack_stream(stream), name.encode(),
                                          ctypes.byref(p), ctypes.byref(n)))
        return p.value, n.value

    def bind_qlinear(self, name: str, K: int, stream=None) -> QWeightC:
        """The C weight descriptor of linear `name` (quantized or dense)."""
        out = QWeightC()
        g = ctypes.c_int(self.group)
        miss = ctypes.create_string_buffer(256)
        rc = load().ltx25_pack_bind_qlinear(self._h, _pack_stream(stream), name.encode(), K,
                                            ctypes.byref(g), ctypes.byref(out), miss, 256)
        if rc != OK:
            raise Ltx25Error(rc, last_error() + (f" (missing {miss.value.decode()})"
                                                 if miss.value else ""))
        self.group = g.value
        return out


def pack_quantizable(name: str, dtype: str, ndim: int) -> bool:
    return bool(load().ltx25_pack_quantizable(name.encode(), dtype.encode(), ndim))


def linear_qc(x, cw: QWeightC, bias, y, M: int, K: int, N: int, epilogue: int = EPI_NONE,
              stream=None) -> None:
    """linear over an already-built C weight descriptor (e.g. from Pack.bind_qlinear)."""
    check(load().ltx25_linear_q_ex(_stream(stream), _ptr(x), ctypes.byref(cw), _ptr(bias),
                                   bias_dtype_of(bias), _ptr(y), M, K, N, epilogue))
