"""The paged 8-bit cache on the GPU: appending and reading back bit for bit against the
definition's steps, attention over it against 64 bits of the same codes."""
import numpy as np
import pytest
import torch

import attn_ref
from gpu_util import say

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(seed, *shape, std=1.0):
    return (torch.randn(shape, device="cuda", generator=_gen(seed)) * std).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(lens):
    return [0] + list(np.cumsum(lens))


def _cache(pkg, seed, pages, page, heads, dim):
    """A cache whose every page holds something: normal codes, scales of its own."""
    g = _gen(seed)
    c = pkg.KVCache.empty(pages, page, heads, dim)
    for t in (c.k, c.v):
        t.copy_((torch.randn(t.shape, device="cuda", generator=g) * 36).round().clamp(-127, 127))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, device="cuda", generator=g) * 0.05 + 0.005)
    return c


def _table(seed, lens, page, spare=0):
    n = [-(-x // page) for x in lens]
    rng = np.random.default_rng(seed)
    order = rng.permutation(sum(n) + spare)
    t = np.zeros((len(lens), max(max(n), 1)), np.int32)
    at = 0
    for b, m in enumerate(n):
        t[b, :m] = order[at:at + m]
        at += m
    return t, sum(n) + spare


def _bits(t):
    return t.view(torch.int16).cpu().numpy()


def _read(pkg, c, table, counts, first):
    total = sum(counts)
    k = torch.full((total, c.kv_heads, c.head_dim), 3.0, dtype=torch.bfloat16, device="cuda")
    v = torch.full_like(k, 3.0)
    pkg.kv_read(c, table, k, v, _i32(_cu(counts)), _i32(first))
    torch.cuda.synchronize()
    return k, v


def _held(pkg, c, ref, table, lens):
    """The cache's first lens[b] tokens are the reference's, through kv_read and in the bytes."""
    k, v = _read(pkg, c, _i32(table), lens, [0] * len(lens))
    for which, got in enumerate((k, v)):
        at = 0
        for b, n in enumerate(lens):
            want = torch.from_numpy(ref.values(which, table[b], 0, n)).to(torch.bfloat16)
            assert np.array_equal(_bits(got[at:at + n]), _bits(want)), (which, b)
            at += n
    now = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    for which in (0, 1):
        for b, n in enumerate(lens):
            for p in range(-(-n // c.page_tokens)):
                pid, m = table[b, p], min(n - p * c.page_tokens, c.page_tokens)
                assert np.array_equal(now.codes[which][pid][:, :m], ref.codes[which][pid][:, :m])
                assert np.array_equal(now.scale[which][pid], ref.scale[which][pid])


APPENDS = [  # tokens held, new tokens, kv heads, width, page
    ([0], [1], 1, 128, 16),
    ([0, 5, 16, 31], [40, 1, 1, 2], 2, 64, 16),
    ([7, 0, 33], [9, 64, 200], 3, 128, 32),
    ([63, 64, 65, 0], [1, 1, 130, 64], 8, 128, 64),
    ([1, 100, 127], [127, 300, 2], 2, 64, 128),
    ([50, 3, 0], [0, 20, 0], 2, 128, 64),
    ([i % 37 for i in range(70)], [1 + i % 3 for i in range(70)], 1, 64, 16),
    ([i % 23 for i in range(300)], [i % 4 for i in range(300)], 1, 64, 16),
]


@pytest.mark.parametrize("start,new,heads,dim,page", APPENDS)
def test_append_and_read_bit_for_bit(pkg, dev, start, new, heads, dim, page):
    """Quiet and loud tokens in turn, so that some blocks keep their scale and some requantize;
    keys and values are column ranges of one tensor."""
    say(f"kv_append {start[:4]} + {new[:4]} heads {heads} x {dim} page {page}")
    lens = [a + n for a, n in zip(start, new)]
    table, pages = _table(31, lens, page, 2)
    c = _cache(pkg, 32, pages, page, heads, dim)
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    y = _randn(33, sum(new), 2 * heads * dim)
    y *= torch.exp2(torch.randint(-6, 6, (sum(new), 1), device="cuda", generator=_gen(34))).to(y.dtype)
    k, v = (t.unflatten(1, (-1, dim)) for t in y.split([heads * dim] * 2, 1))
    other = [t.clone() for t in (c.k, c.v)]
    pkg.kv_append(c, _i32(table), k, v, _i32(_cu(new)), _i32(start))
    torch.cuda.synchronize()
    ref.append(table, k.float().cpu().numpy(), v.float().cpu().numpy(), _cu(new), start)
    _held(pkg, c, ref, table, lens)
    # pages of no sequence are as they were
    used = {int(table[b, p]) for b, n in enumerate(lens) for p in range(-(-n // page))}
    for pid in sorted(set(range(pages)) - used):
        assert torch.equal(c.k[pid], other[0][pid]) and torch.equal(c.v[pid], other[1][pid])
    # and the same call again changes nothing
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    pkg.kv_append(c, _i32(table), k, v, _i32(_cu(new)), _i32(start))
    torch.cuda.synchronize()
    _held(pkg, c, ref, table, lens)
    assert torch.equal(before[2], c.k_scale) and torch.equal(before[3], c.v_scale)


def test_append_token_by_token(pkg, dev):
    """150 single appends into one sequence, each louder or quieter than the last."""
    page, heads, dim, n = 64, 2, 128, 150
    table, pages = _table(35, [n], page)
    c = _cache(pkg, 36, pages, page, heads, dim)
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    x = _randn(37, n, 2, heads, dim)
    x *= torch.exp2(torch.randint(-4, 4, (n, 1, 1, 1), device="cuda", generator=_gen(38))).to(x.dtype)
    say("kv_append token by token")
    for i in range(n):
        pkg.kv_append(c, _i32(table), x[i:i + 1, 0], x[i:i + 1, 1], _i32([0, 1]), _i32([i]))
    torch.cuda.synchronize()
    h = x.float().cpu().numpy()
    for i in range(n):
        ref.append(table, h[i:i + 1, 0], h[i:i + 1, 1], [0, 1], [i])
    _held(pkg, c, ref, table, [n])


def test_append_ties_denormals_and_values_that_are_not_finite(pkg, dev):
    """Half-way quotients go to even; denormal and all-zero blocks; NaN gives 0, infinities the
    end codes, and neither touches the scale."""
    page, heads, dim = 16, 1, 64
    x = np.zeros((5 * page, heads, dim), np.float32)
    x[0, 0, :6] = [127, 0.5, 1.5, -2.5, 126.5, -0.5]            # scale 1: ties
    x[page, 0, :3] = [1e-39, -3e-40, 9.2e-41]                   # denormals
    x[2 * page:3 * page] = 0                                    # scale 0
    x[3 * page, 0, :5] = [np.nan, np.inf, -np.inf, 2.0, -1.0]
    x[4 * page, 0, :2] = [3.0e38, -1.0e38]
    t = torch.from_numpy(x).cuda().to(torch.bfloat16)
    table, pages = _table(39, [5 * page], page)
    c = _cache(pkg, 40, pages, page, heads, dim)
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    say("kv_append ties and odd values")
    pkg.kv_append(c, _i32(table), t, t, _i32([0, 5 * page]), _i32([0]))
    torch.cuda.synchronize()
    h = t.float().cpu().numpy()
    ref.append(table, h, h, [0, 5 * page], [0])
    _held(pkg, c, ref, table, [5 * page])
    p3 = table[0, 3]
    assert c.k[p3, 0, 0, :5].tolist() == [0, 127, -127, 127, -64]
    assert float(c.k_scale[p3, 0]) == float(np.float32(2) / np.float32(127))
    assert float(c.k_scale[table[0, 2], 0]) == 0.0


def test_append_and_read_where_there_is_no_page(pkg, dev):
    """Page ids outside the cache and tokens past the table: dropped, and read as zeros; the
    cache's neighbours in memory stay."""
    page, heads, dim, pages = 16, 2, 64, 4
    kb = torch.full((pages + 2, heads, page, dim), 9, dtype=torch.int8, device="cuda")
    vb = torch.full((pages + 2, heads, dim, page), 9, dtype=torch.int8, device="cuda")
    sb = [torch.full((pages + 2, heads), 0.5, device="cuda") for _ in range(2)]
    c = pkg.KVCache(kb[1:-1], vb[1:-1], sb[0][1:-1], sb[1][1:-1])
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    table = np.array([[2, -1, 0], [pages, 3, 1 << 30]], np.int32)
    start, new = [0, 3], [60, 40]
    x = _randn(41, 100, heads, dim)
    say("kv_append without pages")
    pkg.kv_append(c, _i32(table), x, x, _i32(_cu(new)), _i32(start))
    torch.cuda.synchronize()
    h = x.float().cpu().numpy()
    ref.append(table, h, h, _cu(new), start)
    k, v = _read(pkg, c, _i32(table), [60, 43], [0, 0])
    for which, got in enumerate((k, v)):
        want = np.concatenate([ref.values(which, table[0], 0, 60), ref.values(which, table[1], 0, 43)])
        # page 0 of sequence 1 has no id: zeros; its tokens past the new ones are undefined
        assert np.array_equal(_bits(got), _bits(torch.from_numpy(want).to(torch.bfloat16)))
    for t in (kb, vb):
        assert bool((t[0] == 9).all()) and bool((t[-1] == 9).all())
    for t in sb:
        assert bool((t[0] == 0.5).all()) and bool((t[-1] == 0.5).all())


CACHED = [  # lens, q_len, heads, kv heads, width, page, causal
    ([1], 1, 1, 1, 128, 16, True),
    ([700], 1, 32, 8, 128, 64, True),
    ([0, 1, 15, 16, 17, 63, 64, 65], 1, 8, 2, 64, 16, True),
    ([255, 256, 257, 300], 1, 4, 4, 128, 32, True),
    ([5000, 30, 2049], 1, 8, 1, 128, 64, True),
    ([100, 3, 0, 900], 5, 6, 2, 64, 16, True),        # a draft longer than its cache
    ([90, 511], 16, 4, 1, 128, 128, True),            # 64 rows
    ([200], 33, 10, 2, 128, 64, True),                # three blocks of rows
    ([77], 8, 16, 16, 64, 32, True),
    ([129, 400], 20, 6, 2, 128, 64, False),           # every query sees all
    ([64] * 70, 1, 2, 2, 64, 64, True),
    ([3000], 3, 7, 1, 64, 128, True),
]


def _attend(pkg, c, table, lens, q, q_len, causal, max_len=None, scale=0.0):
    max_len = max(max(lens), 1) if max_len is None else max_len
    batch, heads = len(lens), q.shape[1]
    need = pkg.attention_cached_workspace(batch, q_len, heads, c.kv_heads, c.head_dim, max_len)
    # a byte pattern that is a NaN in every word, and a margin that has to stay
    ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device="cuda")
    z = torch.full(q.shape[:2], float("nan"), device="cuda")
    pkg.attention_cached(c, _i32(table), _i32(lens), q, out, q_len, max_len, ws[:need] if need else None,
                         causal=causal, scale=scale, lse=z)
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xff).all())
    return out, z


def _verify(c, table, lens, q, q_len, causal, out, z, scale=None):
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    scale = scale or c.head_dim ** -0.5
    for b, n in enumerate(lens):
        rows = slice(b * q_len, (b + 1) * q_len)
        pages = [table[b][t // c.page_tokens] for t in range(n)]
        seen = torch.tensor([0 <= p < c.pages for p in pages], dtype=torch.bool)
        k, v = (torch.from_numpy(ref.values(w, table[b], 0, n)) for w in (0, 1))
        want = attn_ref.attend(q[rows], k, v, scale, causal, seen)
        attn_ref.check(out[rows], z[rows], want, f"sequence {b}")


@pytest.mark.parametrize("lens,q_len,heads,kv_heads,dim,page,causal", CACHED)
def test_attention_cached_against_64_bits(pkg, dev, lens, q_len, heads, kv_heads, dim, page, causal):
    say(f"attention_cached {lens[:4]} q_len {q_len} heads {heads}/{kv_heads} x {dim} page {page}")
    table, pages = _table(51, lens, page, 2)
    c = _cache(pkg, 52, pages, page, kv_heads, dim)
    q = _randn(53, len(lens) * q_len, heads, dim)
    out, z = _attend(pkg, c, table, lens, q, q_len, causal)
    _verify(c, table, lens, q, q_len, causal, out, z)


def test_attention_cached_unseen_pages_and_scales(pkg, dev):
    """Pages past a sequence's end with scales that are no numbers; ids outside the cache, whose
    tokens no query sees; two sequences on the same pages; a longer table than is used."""
    page, dim = 16, 128
    c = _cache(pkg, 54, 12, page, 2, dim)
    c.k_scale[9:], c.v_scale[9:] = float("nan"), float("inf")
    table = np.array([[0, 1, 2, 9, 10], [0, 1, 3, 11, 9], [4, -5, 5, 100, 9], [-1, -1, 9, 9, 9]],
                     np.int32)
    lens = [40, 33, 48, 20]
    q = _randn(55, 4, 4, dim)
    say("attention_cached unseen pages")
    out, z = _attend(pkg, c, table, lens, q, 1, True)
    _verify(c, table, lens, q, 1, True, out, z)
    assert bool((out[3] == 0).all()) and bool((z[3] == -float("inf")).all())


def test_attention_cached_lens_past_their_bound_are_cut(pkg, dev):
    page = 32
    table, pages = _table(56, [200, 200], page)
    c = _cache(pkg, 57, pages, page, 2, 64)
    q = _randn(58, 2, 4, 64)
    say("attention_cached lens past max_len and past the table")
    out, z = _attend(pkg, c, table, [1000000, -3], q, 1, True, max_len=150)
    _verify(c, table, [150, 0], q, 1, True, out, z)
    out, z = _attend(pkg, c, table, [1000000, 2 ** 31 - 1], q, 1, True, max_len=1 << 20)
    _verify(c, table, [7 * page, 7 * page], q, 1, True, out, z)


@pytest.mark.parametrize("std,scale", [(8.0, 0.0), (1.0, 0.7), (1.0, 1e-3)])
def test_attention_cached_steep_and_flat_logits(pkg, dev, std, scale):
    lens = [3000, 70]
    table, pages = _table(59, lens, 64)
    c = _cache(pkg, 60, pages, 64, 2, 128)
    q = _randn(61, 2, 8, 128, std=std)
    say(f"attention_cached std {std} scale {scale}")
    out, z = _attend(pkg, c, table, lens, q, 1, True, scale=scale)
    _verify(c, table, lens, q, 1, True, out, z, scale)


def test_attention_cached_block_scales_far_apart(pkg, dev):
    """Blocks whose scales lie 60 powers of two apart: the sums stay in range, and the loud block
    does not drown the others where the queries do not look at it."""
    lens = [256]
    table, pages = _table(62, lens, 64)
    c = _cache(pkg, 63, pages, 64, 1, 64)
    c.v_scale[table[0, 1], 0] = 2.0 ** -30
    c.v_scale[table[0, 2], 0] = 2.0 ** 30
    q = _randn(64, 1, 4, 64)
    say("attention_cached scales apart")
    out, z = _attend(pkg, c, table, lens, q, 1, True)
    _verify(c, table, lens, q, 1, True, out, z)


def _verify_close(c, table, lens, q, q_len, out, z):
    """The weights keep 11 bits for the second product, and what is done in f32 adds at most 2^-12 at
    these logits (130 products of f32 each): beside the output's own rounding to bf16, 2^-8 of it."""
    ref = attn_ref.Cache(c.k, c.v, c.k_scale, c.v_scale)
    for b, n in enumerate(lens):
        rows = slice(b * q_len, (b + 1) * q_len)
        k, v = (torch.from_numpy(ref.values(w, table[b], 0, n)) for w in (0, 1))
        want = attn_ref.attend(q[rows], k, v, c.head_dim ** -0.5, True)
        attn_ref.check(out[rows], z[rows], want, f"sequence {b}")
        exact, mag = want[0], want[2]
        err = (out[rows].cpu().double() - exact).abs()
        err -= 2.0 ** -8 * 1.001 * exact.abs() + (2.0 ** -11 + 2.0 ** -12) * mag
        assert float(err.max()) <= 0, f"sequence {b}: {float(err.max()):.3e} past the bound"


@pytest.mark.parametrize("lens,q_len,heads,kv_heads,dim,page", [
    ([16], 16, 16, 2, 64, 32), ([700], 1, 32, 8, 128, 64), ([1, 2, 3, 2000], 3, 8, 2, 128, 16),
    ([1100], 24, 2, 1, 128, 64), ([5000], 1, 4, 1, 64, 128)])
def test_attention_cached_rounds_the_output_alone(pkg, dev, lens, q_len, heads, kv_heads, dim, page):
    say(f"attention_cached close {lens} q_len {q_len} heads {heads}/{kv_heads} x {dim} page {page}")
    table, pages = _table(68, lens, page)
    c = _cache(pkg, 69, pages, page, kv_heads, dim)
    q = _randn(70, len(lens) * q_len, heads, dim)
    out, z = _attend(pkg, c, table, lens, q, q_len, True)
    _verify_close(c, table, lens, q, q_len, out, z)


@pytest.mark.parametrize("loud", [2.0 ** 10, 2.0 ** 24])
@pytest.mark.parametrize("q_len,heads", [(1, 4), (8, 4), (12, 4)])
def test_attention_cached_loud_blocks_that_no_query_looks_at(pkg, dev, loud, q_len, heads):
    """Blocks of values that are much larger than the others', before and after them, whose keys
    have logits so low that they do not count; a block of zeros that does."""
    lens, page, dim = [640], 64, 64
    table, pages = _table(71, lens, page)
    c = _cache(pkg, 72, pages, page, 1, dim)
    q = _randn(73, q_len, heads, dim).abs()
    for at in (0, 4, 9):
        c.k[table[0, at]] = -127
        c.k_scale[table[0, at], 0] = 0.2
        c.v_scale[table[0, at], 0] *= loud
    c.v_scale[table[0, 2], 0] = 0.0
    say(f"attention_cached loud {loud} q_len {q_len}")
    # the last tokens lie in a loud block: the queries see it, and none of it counts
    out, z = _attend(pkg, c, table, lens, q, q_len, True)
    _verify_close(c, table, lens, q, q_len, out, z)


@pytest.mark.parametrize("n,heads,dim", [(300, 4, 64), (700, 40, 128), (5000, 4, 128), (5000, 4, 64)])
def test_attention_cached_values_near_the_end_of_f32(pkg, dev, n, heads, dim):
    """Values up to 2^126 under flat logits: the means are finite, though the sums are not, in one
    part and in several."""
    table, pages = _table(74, [n], 64)
    c = _cache(pkg, 75, pages, 64, 1, dim)
    c.v_scale.fill_(2.0 ** 119)
    q = _randn(76, 1, heads, dim, std=0.1)
    say(f"attention_cached large values {n}")
    out, z = _attend(pkg, c, table, [n], q, 1, True)
    _verify(c, table, [n], q, 1, True, out, z)


def test_attention_cached_far_pages(pkg, dev):
    """Pages past 2^31 bytes of the cache."""
    page, heads, dim, pages = 64, 8, 128, 33000
    c = pkg.KVCache.empty(pages, page, heads, dim)
    last = _cache(pkg, 65, 4, page, heads, dim)
    ids = [pages - 1, pages - 3, 0, pages - 2]
    for i, p in enumerate(ids):
        c.k[p], c.v[p], c.k_scale[p], c.v_scale[p] = last.k[i], last.v[i], last.k_scale[i], last.v_scale[i]
    lens = [230]
    q = _randn(66, 1, 16, dim)
    say("attention_cached far pages")
    out, z = _attend(pkg, c, np.array([ids], np.int32), lens, q, 1, True)
    _verify(last, np.array([[0, 1, 2, 3]]), lens, q, 1, True, out, z)
    x = _randn(67, 30, heads, dim)
    pkg.kv_append(c, _i32([ids]), x, x, _i32([0, 26]), _i32([230]))
    pkg.kv_append(last, _i32([[0, 1, 2, 3]]), x, x, _i32([0, 26]), _i32([230]))
    torch.cuda.synchronize()
    assert torch.equal(c.k[ids[3]], last.k[3]) and torch.equal(c.v[ids[3]], last.v[3])
    a, b = _read(pkg, c, _i32([ids]), [256], [0])
    d, e = _read(pkg, last, _i32([[0, 1, 2, 3]]), [256], [0])
    assert torch.equal(a.view(torch.int16), d.view(torch.int16))
    assert torch.equal(b.view(torch.int16), e.view(torch.int16))


def test_cache_ops_repeat_bit_for_bit_on_a_stream_and_in_a_graph(pkg, dev):
    """A decode step, append then attend, on a side stream and captured; replays after other
    work has dirtied the workspace."""
    lens, heads, kv_heads, dim, page = [3000, 77, 641], 8, 2, 128, 64
    table, pages = _table(68, lens, page)
    t, n = _i32(table), _i32(lens)
    c = _cache(pkg, 69, pages, page, kv_heads, dim)
    q, x = _randn(70, 3, heads, dim), _randn(71, 3, kv_heads, dim)
    cu, start = _i32([0, 1, 2, 3]), _i32([m - 1 for m in lens])
    need = pkg.attention_cached_workspace(3, 1, heads, kv_heads, dim, max(lens))
    assert need > 0
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)

    def step():
        pkg.kv_append(c, t, x, x, cu, start)
        pkg.attention_cached(c, t, n, q, out, 1, max(lens), ws)

    step()
    torch.cuda.synchronize()
    want = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    say("decode step on a side stream")
    with torch.cuda.stream(side):
        out.zero_()
        step()
    side.synchronize()
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(3):
        out.fill_(float("nan"))
        ws.fill_(0xff)
        torch.cuda.synchronize()
        say(f"decode step replay {rep}")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
