"""What the Python binding of attention refuses before it hands an address to the library."""
import pytest
import torch


class OnGpu(torch.Tensor):
    """A tensor that says that it lies in the GPU's memory: what the binding looks at."""

    is_cuda = True


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16).as_subclass(OnGpu)


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32).as_subclass(OnGpu)


def _on_host(args, name):
    """The arguments with one of them in host memory."""
    args = dict(args)
    args[name] = args[name].as_subclass(torch.Tensor).clone()
    return args


def _cache(pkg, host=None):
    parts = dict(k=torch.zeros((4, 2, 64, 128), dtype=torch.int8),
                 v=torch.zeros((4, 2, 128, 64), dtype=torch.int8),
                 k_scale=torch.zeros((4, 2)), v_scale=torch.zeros((4, 2)))
    return pkg.KVCache(**{n: t if n == host else t.as_subclass(OnGpu) for n, t in parts.items()})


@pytest.mark.parametrize("name", ["q", "k", "v", "out", "cu_q", "cu_k", "lse", "workspace"])
def test_attention_takes_no_host_memory(pkg, name):
    args = dict(q=_bf16(4, 8, 128), k=_bf16(4, 2, 128), v=_bf16(4, 2, 128), out=_bf16(4, 8, 128),
                cu_q=_i32(0, 4), cu_k=_i32(0, 4), lse=torch.zeros((4, 8)).as_subclass(OnGpu),
                workspace=torch.zeros(64, dtype=torch.uint8).as_subclass(OnGpu))
    with pytest.raises(ValueError, match=name):
        pkg.attention(**_on_host(args, name), causal=True)


@pytest.mark.parametrize("call", ["kv_append", "kv_read"])
@pytest.mark.parametrize("name", ["table", "k", "v", "cu", "start"])
def test_cache_moves_take_no_host_memory(pkg, call, name):
    args = dict(table=torch.zeros((1, 3), dtype=torch.int32).as_subclass(OnGpu), k=_bf16(4, 2, 128),
                v=_bf16(4, 2, 128), cu=_i32(0, 4), start=_i32(0))
    with pytest.raises(ValueError, match=name):
        getattr(pkg, call)(_cache(pkg), **_on_host(args, name))


@pytest.mark.parametrize("name", ["table", "lens", "q", "out", "workspace", "lse"])
def test_attention_cached_takes_no_host_memory(pkg, name):
    args = dict(table=torch.zeros((1, 3), dtype=torch.int32).as_subclass(OnGpu), lens=_i32(100),
                q=_bf16(1, 8, 128), out=_bf16(1, 8, 128),
                workspace=torch.zeros(64, dtype=torch.uint8).as_subclass(OnGpu),
                lse=torch.zeros((1, 8)).as_subclass(OnGpu))
    with pytest.raises(ValueError, match=name):
        pkg.attention_cached(_cache(pkg), q_len=1, max_len=100, **_on_host(args, name))


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_a_cache_in_host_memory_is_refused_by_every_call(pkg, name):
    c = _cache(pkg, name)
    table, x = torch.zeros((1, 3), dtype=torch.int32).as_subclass(OnGpu), _bf16(4, 2, 128)
    for _ in range(2):
        for call in (pkg.kv_append, pkg.kv_read):
            with pytest.raises(ValueError, match="cache." + name):
                call(c, table, x, x, _i32(0, 4), _i32(0))
        with pytest.raises(ValueError, match="cache." + name):
            pkg.attention_cached(c, table, _i32(4), _bf16(1, 8, 128), _bf16(1, 8, 128), 1, 100)


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_a_caches_tensors_stay_its_own(pkg, name):
    """Calls go to the addresses that the cache was made with: another tensor in their place would
    be ignored, and the old one's memory, freed, written to."""
    c = _cache(pkg)
    old, address = getattr(c, name), bytes(c.c())
    with pytest.raises(AttributeError):
        setattr(c, name, old.clone())
    assert getattr(c, name) is old and bytes(c.c()) == address
