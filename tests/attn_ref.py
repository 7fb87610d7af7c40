"""Attention and its 8-bit cache restated in 64 bits (the cache's codes in the definition's own
32-bit steps), for the tests."""
import numpy as np
import torch


def attend(q, k, v, scale, causal, seen=None):
    """One sequence: q [Lq][H][D], k, v [Lk][G][D] -> out [Lq][H][D], lse [Lq][H], the weighted
    mean of |v| per output and the largest sum of |q_i k_i| scale per row, all float64 on the CPU.
    `seen` [Lk] bool: keys that any query may see."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    lq, heads, dim = q.shape
    lk, groups = k.shape[0], k.shape[1]
    out, mag = torch.zeros(lq, heads, dim).double(), torch.zeros(lq, heads, dim).double()
    lse = torch.full((lq, heads), -np.inf).double()
    size = torch.zeros(lq, heads).double()
    if lk == 0:
        return out, lse, mag, size
    vis = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        vis = torch.arange(lk)[None, :] <= torch.arange(lq)[:, None] + (lk - lq)
    if seen is not None:
        vis = vis & seen[None, :]
    for h in range(heads):
        g = h // (heads // groups)
        for i in range(lq):
            at = vis[i].nonzero()[:, 0]
            if len(at) == 0:
                continue
            kk, vv = k[at, g], v[at, g]
            s = (kk @ q[i, h]) * scale
            z = torch.logsumexp(s, 0)
            w = torch.exp(s - z)
            out[i, h], mag[i, h], lse[i, h] = w @ vv, w @ vv.abs(), z
            size[i, h] = ((kk.abs() @ q[i, h].abs()) * scale).max()
    return out, lse, mag, size


# Each weight is rounded to bf16 for the second product and the output once more: bf16 has 8
# significant bits, so each by at most 2^-8 of itself. What is done in f32 adds parts in 2^20 at the
# logits tested here. So an output is within 2^-7 of the weights' mean of |v|, and a tenth is left
# for the f32 parts.
OUT_BOUND = 1.1 * 2.0 ** -7
# The logits are f32 sums of 64 or 128 products: at most 130 * 2^-24 of the sum of magnitudes.
LSE_BOUND = 2e-5


def check(out, lse, want, what=""):
    ref, zref, mag, size = want
    got = out.detach().cpu().double()
    err = (got - ref).abs() - (OUT_BOUND * mag + 1e-30)
    assert bool((err <= 0).all()), f"{what}: off by {float(err.max()):.3e} past the bound"
    if lse is not None:
        z = lse.detach().cpu().double()
        none = torch.isinf(zref)
        assert bool((z[none] == -np.inf).all()), f"{what}: lse of rows that see nothing"
        d = ((z - zref).abs() - LSE_BOUND * (1 + size))[~none]
        assert d.numel() == 0 or float(d.max()) <= 0, f"{what}: lse off by {float(d.max()):.3e}"


# ---- the cache ------------------------------------------------------------------------


def quantize(x, s):
    """rint(x / s) in float32 steps, within +-127; 0 for s = 0 and for NaN."""
    x = np.asarray(x, np.float32)
    if not s > 0:
        return np.zeros(x.shape, np.int8)
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.rint(x / np.float32(s))
    return np.where(np.isnan(r), 0, np.clip(r, -127, 127)).astype(np.int8)


class Cache:
    """The cache on the host: k codes [pages][heads][tokens][width], v codes turned."""

    def __init__(self, k, v, k_scale, v_scale):
        self.codes = [k.cpu().numpy().copy(), v.cpu().numpy().transpose(0, 1, 3, 2).copy()]
        self.scale = [k_scale.cpu().numpy().copy(), v_scale.cpu().numpy().copy()]
        self.page = self.codes[0].shape[2]

    def append(self, table, k, v, cu, start):
        for b in range(len(start)):
            n = cu[b + 1] - cu[b]
            if n <= 0:
                continue
            for p in range(start[b] // self.page, (start[b] + n - 1) // self.page + 1):
                lo, hi = max(start[b], p * self.page), min(start[b] + n, (p + 1) * self.page)
                if p >= table.shape[1] or not 0 <= table[b, p] < len(self.codes[0]):
                    continue
                for which, x in enumerate((k, v)):
                    self._block(which, table[b, p], lo - p * self.page,
                                x[cu[b] + lo - start[b]:cu[b] + hi - start[b]])

    def _block(self, which, pid, old, x):
        codes, scale = self.codes[which][pid], self.scale[which][pid]
        for g in range(x.shape[1]):
            fin = np.abs(x[:, g][np.isfinite(x[:, g])])
            top = np.float32(fin.max() if fin.size else 0) / np.float32(127)
            s0 = scale[g] if old > 0 else np.float32(0)
            s1 = max(s0, top)
            if old > 0 and s1 > s0:
                codes[g, :old] = quantize(codes[g, :old].astype(np.float32) * s0, s1)
            codes[g, old:old + len(x)] = quantize(x[:, g], s1)
            scale[g] = s1

    def values(self, which, table_row, first, n):
        """Tokens first .. first + n - 1 of a sequence as float32 [n][heads][width]."""
        c = self.codes[which]
        out = np.zeros((n, c.shape[1], c.shape[3]), np.float32)
        for i in range(n):
            p, t = (first + i) // self.page, (first + i) % self.page
            if p < len(table_row) and 0 <= table_row[p] < len(c):
                pid = table_row[p]
                out[i] = c[pid, :, t].astype(np.float32) * self.scale[which][pid][:, None]
        return out
