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


def _import_torch():
    """torch, imported on first use, and how its current stream's handle is read: the accessor
    that returns the handle alone where torch has it (0.07 us; torch.cuda.current_stream() builds
    a Stream object, 2.7 of the 8.2 us that a call took on the host)."""
    global _torch, _raw_stream
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _raw_stream = raw if raw is not None else (
        lambda device: torch.cuda.current_stream(device).cuda_stream)
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
                workspace = _torch.empty(need, dtype=_torch.uint8, device=q.device)
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
        """Refuse a cache in host memory, which may be made but not given to a kernel."""
        _reachable("cache.k cache.v cache.k_scale cache.v_scale", *self._tensors)
        self.checked = True


def _moved(cache: KVCache, table, k, v, cu, start):
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
    if not (table.is_cuda and k.is_cuda and v.is_cuda and cu.is_cuda and start.is_cuda):
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
