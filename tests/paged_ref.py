"""Plain 64-bit implementations of the paged-cache operators, and how far a
16-bit implementation with 32-bit sums may be from them.

Half steps: u of the element type (fp16 2^-11, bf16 2^-8), e = 2^-24 of fp32.
"""
import numpy as np

E32 = 2.0 ** -24
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}     # half a step of the smallest subnormal


def to16(x, kind):
    """float array -> float16, or uint16 with bfloat16 bits (round to nearest even)."""
    x = np.asarray(x, np.float32)
    if kind == "f16":
        return x.astype(np.float16)
    b = x.view(np.uint32)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def to64(a):
    if a.dtype == np.uint16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


class Cache:
    """A batch of sequences in shuffled pages, and its new tokens' queries."""

    def __init__(self, rng, kv_lens, q_lens, heads, kv_heads, dim, page, kind="f16", spare=2,
                 wide=None, lead=0, trail=0, q_by=1.5, fill=None):
        self.kind, self.heads, self.kv_heads, self.dim, self.page = kind, heads, kv_heads, dim, page
        self.kv_lens = np.array(kv_lens, np.int32)
        counts = [-(-n // page) for n in kv_lens]
        self.wide = max([1, *counts]) if wide is None else wide
        self.pages = sum(counts) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        # what lies behind a sequence's pages must never be followed
        self.table = np.full((len(kv_lens), self.wide), 2 ** 31 - 1, np.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        self.q_offs = (lead + np.concatenate(([0], np.cumsum(q_lens)))).astype(np.int32)
        self.total = int(self.q_offs[-1]) + trail
        shape = (self.pages, kv_heads, page, dim)
        self.q = to16(rng.standard_normal((self.total, heads, dim)) * q_by, kind)
        k, v = rng.standard_normal(shape), rng.standard_normal(shape)
        if fill is not None:   # everything that no sequence uses
            used = np.zeros((self.pages, page), bool)
            for b, n in enumerate(kv_lens):
                for j in range(n):
                    used[self.table[b, j // page], j % page] = True
            k[~used[:, None].repeat(kv_heads, 1)] = fill
            v[~used[:, None].repeat(kv_heads, 1)] = fill
        self.k, self.v = to16(k, kind), to16(v, kind)
        self.scale = dim ** -0.5

    def rows(self, pages, b, h):
        """The cached rows of sequence b and key head h in 64 bits."""
        n = int(self.kv_lens[b])
        j = np.arange(n)
        return to64(pages[self.table[b, j // self.page], h, j % self.page])

    def hidden(self, b, causal):
        n, m = int(self.kv_lens[b]), int(self.q_offs[b + 1] - self.q_offs[b])
        if not causal:
            return np.zeros((m, n), bool)
        return np.arange(n)[None] > n - m + np.arange(m)[:, None]


def paged_attn(c: Cache, causal=True):
    """(out, lse, bound of out, bound of lse) in 64 bits; rows of no sequence are not-a-number."""
    out = np.full(c.q.shape, np.nan)
    lse = np.full(c.q.shape[:2], np.nan)
    b_out, b_lse = np.zeros(c.q.shape), np.zeros(c.q.shape[:2])
    group, u = c.heads // c.kv_heads, U[c.kind]
    for b in range(len(c.kv_lens)):
        lo, hi = c.q_offs[b], c.q_offs[b + 1]
        n = int(c.kv_lens[b])
        hide = c.hidden(b, causal)
        for h in range(c.heads):
            k, v = c.rows(c.k, b, h // group), c.rows(c.v, b, h // group)
            q = to64(c.q[lo:hi, h])
            with np.errstate(all="ignore"):
                x = np.where(hide, -np.inf, q @ k.T * c.scale)
                top = x.max(1, initial=-np.inf)
                p = np.where(hide, 0.0, np.exp(x - np.where(np.isfinite(top), top, 0.0)[:, None]))
                l = p.sum(1)
                w = np.divide(p, l[:, None], out=np.zeros_like(p), where=l[:, None] != 0)
                vis = np.where(hide.any(0)[:, None] & ~np.isfinite(v), 0.0, v)
                out[lo:hi, h] = w @ vis
                lse[lo:hi, h] = top + np.log(l)
                # a score: dim products summed in fp32, scaled, the maximum
                # taken off; its error is the weight's relative error
                mag = np.where(hide, 0.0, np.abs(q) @ np.abs(k).T * c.scale).max(1, initial=0.0)
                span = np.where(np.isfinite(x), np.abs(x - top[:, None]), 0.0).max(1, initial=0.0)
                ds = (c.dim + 4) * E32 * mag + 4 * E32 * (span + np.abs(np.where(np.isfinite(top), top, 0.0)))
                # weights: the score, the exponential, one rounding to 16 bits;
                # sums of n terms in fp32; the largest weight is at least 1, so
                # the rounding of a subnormal one is at most TINY of the sum
                rel = 2 * ds + 8 * E32 + u + (n + 8) * E32
                b_out[lo:hi, h] = (rel[:, None] * (w @ np.abs(vis)) + TINY[c.kind] * np.abs(vis).sum(0)
                                   + u * np.abs(out[lo:hi, h]) + TINY[c.kind])
                b_lse[lo:hi, h] = ds + (n + 16) * E32 + 4 * E32 * np.abs(np.where(np.isfinite(top), top, 0.0))
    return out, lse, b_out, b_lse


def cache_scores(c: Cache, lse, scores, causal=True):
    """(scores, bound): scores float32 as they were, lse float32 as given."""
    got, bound = scores.astype(np.float64), np.zeros(scores.shape)
    group = c.heads // c.kv_heads
    for b in range(len(c.kv_lens)):
        lo, hi = c.q_offs[b], c.q_offs[b + 1]
        hide = c.hidden(b, causal)
        j = np.arange(int(c.kv_lens[b]))
        for h in range(c.kv_heads):
            k = c.rows(c.k, b, h)
            total, off = np.zeros(len(j)), np.zeros(len(j))
            for g in range(group):
                q, z = to64(c.q[lo:hi, h * group + g]), lse[lo:hi, h * group + g].astype(np.float64)[:, None]
                with np.errstate(all="ignore"):
                    x = q @ k.T * c.scale
                    none = hide | (z == -np.inf)
                    w = np.where(none, 0.0, np.exp(x - z))
                    ds = (c.dim + 4) * E32 * (np.abs(q) @ np.abs(k).T * c.scale) + 4 * E32 * (np.abs(x) + np.abs(z))
                    off += np.where(none, 0.0, w * (ds + 8 * E32)).sum(0)
                total += w.sum(0)
            at = (c.table[b, j // c.page], h, j % c.page)
            terms = (hi - lo) * group
            np.add.at(got, at, total)
            np.add.at(bound, at, off + (terms + 2) * E32 * total)
    return got, bound + 2 * E32 * np.abs(got)


def evict_kept(score, budget, sink, recent):
    """Places that stay of one head's scores (fp32), ascending."""
    n = len(score)
    if n <= budget:
        return np.arange(n)
    forced = (np.arange(n) < sink) | (np.arange(n) >= n - recent)
    free = np.flatnonzero(~forced)
    x = score[free].astype(np.float64)
    x = np.where(np.isnan(x), 0.0, x)
    nan = np.isnan(score[free])
    # highest first, not-a-number last, then the lowest place
    order = np.lexsort((free, -x, nan))
    return np.sort(np.concatenate((np.flatnonzero(forced), free[order[:budget - int(forced.sum())]])))


def cache_evict(c: Cache, scores, budget, sink, recent, dst=None):
    """(kept, new_lens, k, v, scores): the arrays after the call."""
    dst = c.table if dst is None else dst
    B = len(c.kv_lens)
    kept = np.full((B, c.kv_heads, budget), -1, np.int32)
    k, v, s = c.k.copy(), c.v.copy(), scores.copy()
    for b in range(B):
        n = int(c.kv_lens[b])
        j = np.arange(n)
        for h in range(c.kv_heads):
            stay = evict_kept(scores[c.table[b, j // c.page], h, j % c.page], budget, sink, recent)
            i = np.arange(len(stay))
            kept[b, h, :len(stay)] = stay
            a, z = (c.table[b, stay // c.page], h, stay % c.page), (dst[b, i // c.page], h, i % c.page)
            k[z], v[z], s[z] = c.k[a], c.v[a], scores[a]
    return kept, np.minimum(c.kv_lens, budget), k, v, s


def qk_norm_rope(x, gain, cos, sin, positions, halves, norm, eps):
    """(y, bound) of heads x [T, H, D] in 64 bits; gain may be None."""
    kind = "bf16" if x.dtype == np.uint16 else "f16"
    y = to64(x)
    dim, half = y.shape[-1], cos.shape[1]
    if norm:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps)
        if gain is not None:
            y = y * to64(gain)
    c, s = cos[positions].astype(np.float64)[:, None], sin[positions].astype(np.float64)[:, None]
    z, mag = y.copy(), np.abs(y)
    a, b = (slice(0, half), slice(half, 2 * half)) if halves else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    m = np.abs(y[..., a]) * np.abs(c) + np.abs(y[..., b]) * np.abs(s)
    n = np.abs(y[..., b]) * np.abs(c) + np.abs(y[..., a]) * np.abs(s)
    mag[..., a], mag[..., b] = m, n
    # the mean of dim squares has a relative error of dim e and enters by half;
    # a root, two products and the rotation's three operations: 10 e more
    return z, U[kind] * np.abs(z) + TINY[kind] + (dim / 2 + 10) * E32 * (1 + U[kind]) * mag


def turns(count, rot, theta=10000.0):
    a = np.arange(count)[:, None] * theta ** (-np.arange(0, rot, 2) / rot)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
