"""What the attention entry points refuse, on the host: every check comes before any device use."""
import ctypes

import pytest
import torch

FAKE = 0x10000   # never dereferenced: every call below ends in a check or is empty


def _attn(pkg, **kw):
    a = dict(heads=8, kv_heads=2, head_dim=128, causal=1, scale=0.0, q_stride=1024, k_stride=256,
             v_stride=256, out_stride=1024)
    a.update(kw)
    return pkg.AttnC(*[a[n] for n, _ in pkg.AttnC._fields_])


def _cache(pkg, **kw):
    c = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, pages=4, page_tokens=64, kv_heads=2,
             head_dim=128)
    c.update(kw)
    return pkg.KVCacheC(*[c[n] for n, _ in pkg.KVCacheC._fields_])


def _attention(pkg, lib, a=None, q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=None, cu_q=FAKE, cu_k=FAKE,
               batch=1, total_q=4, total_k=4, **kw):
    a = a if a is not None else _attn(pkg, **kw)
    return lib.ltx25_attention(None, ctypes.byref(a), q, k, v, out, lse, cu_q, cu_k, batch, total_q,
                               total_k)


def _cached(pkg, lib, a=None, c=None, table=FAKE, stride=4, lens=FAKE, q=FAKE, out=FAKE, lse=None,
            batch=2, q_len=1, max_len=4000, ws=FAKE, ws_bytes=1 << 30):
    a, c = a or _attn(pkg), c or _cache(pkg)
    return lib.ltx25_attention_cached(None, ctypes.byref(a), ctypes.byref(c), table, stride, lens, q,
                                      out, lse, batch, q_len, max_len, ws, ws_bytes)


def _append(pkg, lib, c=None, table=FAKE, stride=4, k=FAKE, v=FAKE, ks=256, vs=256, cu=FAKE,
            start=FAKE, batch=2, total=3, name="ltx25_kv_append"):
    c = c or _cache(pkg)
    return getattr(lib, name)(None, ctypes.byref(c), table, stride, k, v, ks, vs, cu, start, batch,
                              total)


BAD_SIZES = [("heads", 0), ("heads", 7), ("kv_heads", 0), ("kv_heads", -2), ("q_stride", 1020),
             ("q_stride", 1016), ("out_stride", 8), ("q_stride", 1 << 23), ("scale", -1.0),
             ("scale", float("nan")), ("scale", float("inf"))]


@pytest.mark.parametrize("field,value", BAD_SIZES)
def test_sizes_that_are_refused(pkg, lib, field, value):
    a = _attn(pkg, **{field: value})
    assert _attention(pkg, lib, a) == pkg.E_INVAL
    assert field.split("_")[0] in pkg.last_error()
    assert _cached(pkg, lib, a) == pkg.E_INVAL


@pytest.mark.parametrize("dim", [0, 32, 96, 256])
def test_widths_that_no_kernel_takes(pkg, lib, dim):
    wide = dict(head_dim=dim, q_stride=8192, k_stride=8192, v_stride=8192, out_stride=8192)
    assert _attention(pkg, lib, _attn(pkg, **wide)) == pkg.E_UNSUPPORTED
    assert _append(pkg, lib, _cache(pkg, head_dim=dim)) == pkg.E_UNSUPPORTED
    assert "head_dim" in pkg.last_error()


def test_attention_pointers_and_lengths(pkg, lib):
    for name in ("q", "k", "v", "out"):
        assert _attention(pkg, lib, **{name: None}) == pkg.E_INVAL
        assert _attention(pkg, lib, **{name: FAKE + 8}) == pkg.E_INVAL
    assert _attention(pkg, lib, lse=FAKE + 2) == pkg.E_INVAL
    assert _attention(pkg, lib, cu_q=FAKE + 2) == pkg.E_INVAL
    assert _attention(pkg, lib, cu_q=None) == pkg.E_INVAL              # one without the other
    assert _attention(pkg, lib, cu_q=None, cu_k=None, batch=2) == pkg.E_INVAL
    assert _attention(pkg, lib, batch=-1) == pkg.E_INVAL
    assert _attention(pkg, lib, total_q=-1) == pkg.E_INVAL
    assert _attention(pkg, lib, total_k=(1 << 30) + 1) == pkg.E_INVAL
    assert _attention(pkg, lib, k_stride=248) == pkg.E_INVAL
    assert _attention(pkg, lib, v_stride=260) == pkg.E_INVAL
    assert lib.ltx25_attention(None, None, FAKE, FAKE, FAKE, FAKE, None, None, None, 1, 1,
                               1) == pkg.E_INVAL
    # empty: no device use
    assert _attention(pkg, lib, q=None, k=None, v=None, out=None, total_q=0) == pkg.OK
    assert _attention(pkg, lib, batch=0) == pkg.OK


def test_cache_refusals(pkg, lib):
    for name in ("k", "v", "k_scale", "v_scale"):
        assert _append(pkg, lib, _cache(pkg, **{name: None})) == pkg.E_INVAL
        assert _cached(pkg, lib, c=_cache(pkg, **{name: FAKE + 2})) == pkg.E_INVAL
    for page in (0, 8, 24, 48, 256, -64):
        assert _append(pkg, lib, _cache(pkg, page_tokens=page)) == pkg.E_UNSUPPORTED
    for call in (lambda **k: _append(pkg, lib, **k),
                 lambda **k: _append(pkg, lib, name="ltx25_kv_read", **k)):
        assert call(c=_cache(pkg, pages=0)) == pkg.E_INVAL
        assert call(stride=0) == pkg.E_INVAL
        assert call(table=None) == pkg.E_INVAL
        assert call(k=FAKE + 4) == pkg.E_INVAL
        assert call(v=None) == pkg.E_INVAL
        assert call(ks=128) == pkg.E_INVAL
        assert call(vs=257) == pkg.E_INVAL
        assert call(cu=None) == pkg.E_INVAL
        assert call(start=None) == pkg.E_INVAL
        assert call(batch=-1) == pkg.E_INVAL
        assert call(total=-1) == pkg.E_INVAL
        assert call(total=0, k=None, v=None) == pkg.OK
        assert call(batch=0, table=None) == pkg.OK


def test_cached_refusals(pkg, lib):
    assert _cached(pkg, lib, c=_cache(pkg, kv_heads=4)) == pkg.E_INVAL
    assert _cached(pkg, lib, c=_cache(pkg, head_dim=64)) == pkg.E_INVAL
    assert _cached(pkg, lib, lens=None) == pkg.E_INVAL
    assert _cached(pkg, lib, q=FAKE + 8) == pkg.E_INVAL
    assert _cached(pkg, lib, out=None) == pkg.E_INVAL
    assert _cached(pkg, lib, lse=FAKE + 1) == pkg.E_INVAL
    assert _cached(pkg, lib, q_len=-1) == pkg.E_INVAL
    assert _cached(pkg, lib, max_len=-1) == pkg.E_INVAL
    assert _cached(pkg, lib, max_len=(1 << 30) + 1) == pkg.E_INVAL
    assert _cached(pkg, lib, batch=1 << 16, q_len=1 << 15) == pkg.E_INVAL
    need = pkg.attention_cached_workspace(2, 1, 8, 2, 128, 4000)
    assert need > 0
    assert _cached(pkg, lib, ws=None) == pkg.E_INVAL
    assert _cached(pkg, lib, ws_bytes=need - 1) == pkg.E_INVAL
    assert str(need) in pkg.last_error()
    assert _cached(pkg, lib, ws=FAKE + 8) == pkg.E_INVAL
    assert _cached(pkg, lib, batch=0, table=None, lens=None) == pkg.OK
    assert _cached(pkg, lib, q_len=0) == pkg.OK


def test_workspace_sizes(pkg):
    for bad in ((0, 1, 8, 2, 128, 100), (1, 0, 8, 2, 128, 100), (1, 1, 7, 2, 128, 100),
                (1, 1, 8, 0, 128, 100), (1, 1, 8, 2, 96, 100), (1, 1, 8, 2, 128, 0),
                (1, 1, 8, 2, 128, (1 << 30) + 1)):
        assert pkg.attention_cached_workspace(*bad) == 0
    # one part of each row: no workspace
    assert pkg.attention_cached_workspace(1, 1, 8, 2, 128, 64) == 0
    # a part is a row's sums, its maximum and its sum, in floats
    for batch, q_len, heads, kv, dim, n in ((1, 1, 32, 8, 128, 131072), (64, 1, 32, 8, 128, 4096),
                                            (3, 40, 6, 2, 64, 5000), (1, 1, 1, 1, 64, 1 << 30)):
        ws = pkg.attention_cached_workspace(batch, q_len, heads, kv, dim, n)
        parts, rest = divmod(ws, batch * q_len * heads * (dim + 2) * 4)
        assert rest == 0 and parts * 64 <= n + 64


def test_binding_checks_tensors(pkg):
    def t(*s):
        return torch.zeros(s, dtype=torch.bfloat16)

    q, k = t(4, 8, 128), t(4, 2, 128)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(TypeError):
        pkg.attention(q.float(), k, k, q, causal=True)
    with pytest.raises(ValueError):
        pkg.attention(q, k, t(5, 2, 128), q, causal=True)
    with pytest.raises(ValueError):
        pkg.attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, k, q, causal=True)
    with pytest.raises(ValueError):
        pkg.attention(q, k, k, q, i32(0, 4), None, causal=True)
    with pytest.raises(TypeError):
        pkg.attention(q, k, k, q, torch.tensor([0, 4]), i32(0, 4), causal=True)
    with pytest.raises(TypeError):
        pkg.attention(q, k, k, q, causal=True, lse=torch.zeros(8, 4))
    with pytest.raises(TypeError):
        pkg.KVCache(*[torch.zeros(2, 2, 64, 64, dtype=torch.uint8)] * 2, None, None)
    c = pkg.KVCache.empty(4, 64, 2, 128, device="cpu")
    with pytest.raises(TypeError):
        pkg.KVCache(c.k, c.k, c.k_scale, c.v_scale)
    table = torch.zeros((1, 3), dtype=torch.int32)
    with pytest.raises(ValueError):
        pkg.kv_append(c, table, t(4, 2, 64), t(4, 2, 64), i32(0, 4), i32(0))
    with pytest.raises(TypeError):
        pkg.kv_append(c, table, k, k, i32(0, 4, 4), i32(0))
    with pytest.raises(ValueError):
        pkg.attention_cached(c, table, i32(10), t(3, 8, 128), t(3, 8, 128), 2, 100)


def test_more_packed_tokens_than_a_call_takes(pkg, lib):
    many = (1 << 27) + 1
    assert _attention(pkg, lib, total_q=many) == pkg.E_INVAL
    assert "total_q" in pkg.last_error()
    assert _attention(pkg, lib, total_k=many) == pkg.E_INVAL
    for name in ("ltx25_kv_append", "ltx25_kv_read"):
        assert _append(pkg, lib, total=many, name=name) == pkg.E_INVAL
        assert "total" in pkg.last_error()
    assert _cached(pkg, lib, batch=1 << 14, q_len=(1 << 13) + 1) == pkg.E_INVAL


def test_workspace_of_each_size_is_asked_for(pkg, lib):
    """More sequences may need less workspace: a call is held to its own need."""
    one, few = (pkg.attention_cached_workspace(b, 1, 8, 8, 128, 5120) for b in (64, 60))
    assert one == 0 and few > 0
    c, a = _cache(pkg, kv_heads=8), _attn(pkg, kv_heads=8)
    assert _cached(pkg, lib, a, c, batch=60, max_len=5120, ws_bytes=few - 1) == pkg.E_INVAL


def _split(pkg, lib, a=None, ws=FAKE, ws_bytes=1 << 30, total_q=4, total_k=4000, **kw):
    a = a or _attn(pkg)
    p = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, batch=1)
    p.update(kw)
    return lib.ltx25_attention_split(None, ctypes.byref(a), p["q"], p["k"], p["v"], p["out"], None,
                                     FAKE, FAKE, p["batch"], total_q, total_k, ws, ws_bytes)


def test_split_refusals_and_workspace(pkg, lib):
    need = pkg.attention_workspace(8, 2, 128, 1, 4, 4000)
    assert need > 0 and need % (4 * 8 * (128 + 2) * 4) == 0
    assert _split(pkg, lib, ws=None) == pkg.E_INVAL
    assert _split(pkg, lib, ws=FAKE + 8) == pkg.E_INVAL
    assert _split(pkg, lib, ws_bytes=need - 1) == pkg.E_INVAL
    assert str(need) in pkg.last_error()
    assert _split(pkg, lib, _attn(pkg, heads=7)) == pkg.E_INVAL
    assert _split(pkg, lib, q=None) == pkg.E_INVAL
    assert _split(pkg, lib, total_k=(1 << 27) + 1) == pkg.E_INVAL
    assert _split(pkg, lib, total_q=0, ws=None) == pkg.OK
    assert _split(pkg, lib, batch=0, ws=None) == pkg.OK
    # many rows, short keys, no keys, sizes that are refused: nothing to split
    for sizes in ((32, 8, 128, 1, 16384, 16384), (8, 2, 128, 1, 4, 200), (8, 2, 128, 1, 4, 0),
                  (7, 2, 128, 1, 4, 4000), (8, 2, 96, 1, 4, 4000), (8, 2, 128, 0, 4, 4000),
                  (8, 0, 128, 1, 4, 4000), (8, 2, 128, 1, 4, (1 << 27) + 1)):
        assert pkg.attention_workspace(*sizes) == 0
