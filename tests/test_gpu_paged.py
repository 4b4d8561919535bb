"""The paged-cache operators against plain 64-bit implementations: head
layouts, ragged batches, odd pages and lengths, what lies behind a sequence,
bad indices in device memory, streams, graphs, and a run of them together."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu
CODE = {"f16": 0, "bf16": 1}


@pytest.fixture(scope="module")
def dev(hx):
    """Device calls on torch's default stream."""
    import torch
    from hexkernels_b200 import _lib, device
    lib = _lib.load()
    device.bind_stream(0)
    lib.hexcuda_set_timing(0)
    yield device
    torch.cuda.synchronize()
    lib.hexcuda_set_timing(1)
    lib.hexcuda_reset_stream(0)


def up(a):
    """NumPy array on the device (16-bit floats as bit patterns)."""
    import torch
    if a is None:
        return None
    a = np.ascontiguousarray(a)
    if a.dtype in (np.float16, np.uint16):
        a = a.view(np.int16)
    return torch.from_numpy(a.copy()).cuda()


def down(t, like):
    return t.cpu().numpy().view(like.dtype)


def space(device):
    import torch
    return torch.full((device.paged_attn_workspace(0),), 0xFF, dtype=torch.uint8, device="cuda")


class OnDevice:
    """A ref.Cache's arrays on the device and the calls on them."""

    def __init__(self, device, c, causal=True, max_q=None, mark=0x7e5a):
        import torch
        self.d, self.c, self.causal = device, c, causal
        self.q, self.k, self.v = up(c.q), up(c.k), up(c.v)
        self.table, self.lens, self.offs = up(c.table), up(c.kv_lens), up(c.q_offs)
        self.out = torch.full(c.q.shape, mark, dtype=torch.int16, device="cuda")
        self.lse = torch.full(c.q.shape[:2], 123.0, device="cuda")
        self.space = space(device)
        self.max_q = int(np.diff(c.q_offs).max(initial=0)) if max_q is None else max_q

    def dims(self):
        c = self.c
        return (len(c.kv_lens), c.total, self.max_q, c.heads, c.kv_heads, c.dim, c.pages, c.page, c.wide,
                c.scale, int(self.causal))

    def attn(self, lse=True):
        self.d.launch("paged_attn", 0, CODE[self.c.kind], self.q, self.k, self.v, self.table, self.lens, self.offs,
                      self.out, self.lse if lse else None, self.space, self.space.numel(), *self.dims())

    def scores(self, s):
        self.d.launch("cache_scores", 0, CODE[self.c.kind], self.q, self.lse, self.k, self.table, self.lens,
                      self.offs, s, *self.dims())

    def results(self):
        return down(self.out, self.c.q), down(self.lse, np.zeros(0, np.float32))


def near(got, want, bound, what=""):
    got = ref.to64(got) if got.dtype != np.float32 else got.astype(np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(all="ignore"):
        bad = ~same & ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: "
                           f"{got[bad][0]} for {want[bad][0]}, bound {np.broadcast_to(bound, want.shape)[bad][0]}")


def check_attn(o, causal, what=""):
    out, lse = o.results()
    want, z, b_out, b_lse = ref.paged_attn(o.c, causal)
    nobody = np.isnan(z).all(1)
    nobody &= ~np.isin(np.arange(o.c.total), np.concatenate([np.arange(a, b) for a, b in zip(o.c.q_offs, o.c.q_offs[1:])]))
    assert (out.view(np.uint16)[nobody] == 0x7e5a).all() and (lse[nobody] == 123.0).all(), f"{what}: rows of no sequence"
    near(out[~nobody], want[~nobody], b_out[~nobody], what + " out")
    near(lse[~nobody], z[~nobody], b_lse[~nobody], what + " lse")


def attn_case(dev, seed, kv, q, heads, kv_heads, dim, page, kind, causal, **kw):
    c = ref.Cache(np.random.default_rng(seed), kv, q, heads, kv_heads, dim, page, kind, fill=np.nan, **kw)
    o = OnDevice(dev, c, causal)
    o.attn()
    dev.sync(0)
    check_attn(o, causal)
    # the same weights, collected by the cached tokens
    base = np.random.default_rng(seed + 1).random((c.pages, kv_heads, page)).astype(np.float32)
    s = up(base)
    o.scores(s)
    dev.sync(0)
    _, lse = o.results()
    want, bound = ref.cache_scores(c, lse, base, causal)
    near(down(s, base), want, bound, "scores")


DECODE = [
    ([1], [1], 1, 1, 128, 16), ([777], [1], 32, 8, 128, 16), ([127, 128, 129], [1, 1, 1], 8, 1, 128, 16),
    ([64, 1, 500, 0, 33], [1, 1, 1, 1, 1], 4, 4, 64, 16), ([300, 1, 2, 1023, 1024, 1025, 40], [1] * 7, 28, 4, 128, 32),
    ([2049], [1], 8, 8, 64, 64), ([130, 257], [1, 0], 5, 1, 128, 128), ([20011], [1], 8, 2, 128, 16),
    ([700, 33], [1, 1], 16, 1, 64, 256), ([90, 4000], [1, 1], 32, 1, 128, 8), ([100, 1000], [1, 1], 6, 2, 64, 24),
    ([200, 300, 513], [2, 4, 3], 16, 4, 128, 16), ([128, 5], [2, 7], 8, 2, 128, 16),
]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", range(len(DECODE)), ids=lambda n: "-".join(map(str, DECODE[n][2:])) + f"x{len(DECODE[n][0])}")
def test_single_tokens(dev, n, kind):
    attn_case(dev, 10 + n, *DECODE[n], kind, True)


@pytest.mark.parametrize("group", [15, 16, 17, 31, 32, 33, 64, 65, 128, 129])
@pytest.mark.parametrize("most", [1, 2])
def test_many_heads_to_a_key_head(dev, group, most):
    attn_case(dev, 300 + group, [150, 20], [most, 1], 2 * group, 2, 64, 16, "bf16", True)


CHUNK = [
    ([300], [300], 4, 2, 128, 16, True), ([300], [77], 8, 2, 128, 16, True), ([700, 129, 1], [300, 129, 1], 4, 4, 64, 32, True),
    ([1000, 250, 0, 40], [200, 250, 0, 8], 10, 2, 128, 16, True), ([50, 600, 7], [70, 100, 9], 8, 1, 64, 16, True),
    ([1500, 3], [40, 64], 16, 8, 128, 64, False), ([900, 128, 256], [256, 128, 1], 2, 2, 128, 128, False),
    ([515], [513], 7, 1, 64, 8, True), ([2100], [140], 12, 1, 128, 24, True), ([260], [130], 40, 1, 64, 16, True),
    ([5000], [33], 32, 8, 128, 64, True), ([400], [200], 130, 1, 64, 16, True), ([640, 90], [3, 90], 64, 1, 128, 16, True),
]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", range(len(CHUNK)), ids=lambda n: "-".join(map(str, CHUNK[n][2:])) + f"x{len(CHUNK[n][0])}")
def test_chunks(dev, n, kind):
    attn_case(dev, 50 + n, *CHUNK[n][:-1], kind, CHUNK[n][-1])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("kv, q, heads, kv_heads, dim, page", [
    ([500, 1, 129, 0], [1, 1, 1, 1], 8, 2, 128, 16), ([300, 77], [4, 2], 4, 1, 64, 32), ([1000], [7], 4, 1, 128, 64)])
def test_few_tokens_without_the_causal_rule(dev, kv, q, heads, kv_heads, dim, page, kind):
    attn_case(dev, 31, kv, q, heads, kv_heads, dim, page, kind, False)


@pytest.mark.parametrize("most", [1, 40])
def test_many_sequences(dev, most):
    """More sequences than a CTA has threads, most of them short, some empty."""
    rng = np.random.default_rng(37)
    n = 1500 if most == 1 else 500
    kv = rng.integers(0, 300, n) * (rng.random(n) < 0.9)
    q = np.minimum(rng.integers(0, most + 1, n), kv)
    attn_case(dev, 38, kv.tolist(), q.tolist(), 4, 2, 64, 16, "f16", True)


def test_a_cache_of_more_than_4g_elements(dev):
    """A sequence at the far end of pages whose element offsets pass 32 bits."""
    import torch
    kv_heads, dim, page = 8, 128, 16
    pages = 2 ** 32 // (kv_heads * dim * page) + 40
    for q in ([1], [90]):
        c = ref.Cache(np.random.default_rng(41), [500], q, 8, kv_heads, dim, page, "f16")
        o = OnDevice(dev, c)
        s = up(np.zeros(c.k.shape[:3], np.float32))
        o.attn()
        o.scores(s)
        dev.sync(0)
        want = (*o.results(), down(s, np.zeros(0, np.float32)))
        far = pages - c.pages
        big = []
        for small in (o.k, o.v, s):
            t = torch.empty((pages, *small.shape[1:]), dtype=small.dtype, device="cuda")
            t[far:] = small if small is not s else 0
            big.append(t)
        o.k, o.v, s = big
        o.table += far * (o.table < c.pages)
        c.pages = pages
        o.out.zero_()
        o.attn()
        o.scores(s)
        dev.sync(0)
        for a, b in zip((*o.results(), s[far:].cpu().numpy()), want):
            np.testing.assert_array_equal(a, b)
        # cut to 100 tokens there, and append one
        lens, kept = o.lens.clone(), torch.empty(1, kv_heads, 100, dtype=torch.int32, device="cuda")
        k0, v0 = o.k[far:].clone(), o.v[far:].clone()
        dev.launch("cache_evict", 0, o.k, o.v, s, o.table, None, lens, lens, kept, 1, kv_heads, dim, pages, page, c.wide, 0, 100, 4, 10)
        dev.sync(0)
        place = ref.evict_kept(want[2][c.table[0, np.arange(500) // page], 3, np.arange(500) % page], 100, 4, 10)
        np.testing.assert_array_equal(kept[0, 3].cpu().numpy(), place)
        i = torch.arange(100)
        j = torch.from_numpy(place)
        tab = torch.from_numpy(c.table[0]).long()
        for now, was in ((o.k, k0), (o.v, v0)):
            assert torch.equal(now[far:][tab[i // page], 3, i % page], was[tab[j // page], 3, j % page])
        x = torch.randn(3 * kv_heads * dim, device="cuda").to(torch.float16)
        slot = torch.tensor([(pages - 1) * page + 5], dtype=torch.int32, device="cuda")
        out = torch.empty(kv_heads * dim, dtype=torch.float16, device="cuda")
        dev.launch("qk_norm_rope", 0, 0, x, 3 * kv_heads * dim, x[kv_heads * dim:], 3 * kv_heads * dim, x[2 * kv_heads * dim:],
                   3 * kv_heads * dim, None, None, None, None, None, slot, out, o.k, o.v, s, 1, kv_heads, kv_heads, dim, 0, 0, 0, 0,
                   pages, page, 0.0)
        dev.sync(0)
        half = o.k.view(torch.float16)
        assert torch.equal(half[pages - 1, :, 5].flatten(), x[kv_heads * dim:2 * kv_heads * dim])
        assert torch.equal(o.v.view(torch.float16)[pages - 1, :, 5].flatten(), x[2 * kv_heads * dim:])
        del o, s, big, half, k0, v0
        torch.cuda.empty_cache()


def test_two_streams_at_once(dev):
    """Calls in flight on two streams, each with a workspace of its own."""
    import torch
    rng = np.random.default_rng(43)
    cs = [ref.Cache(rng, [3000, 200], [1, 1], 16, 4, 128, 16, "bf16"), ref.Cache(rng, [700, 900], [200, 60], 8, 2, 128, 32, "f16")]
    os = [OnDevice(dev, c) for c in cs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    try:
        for _ in range(5):
            for o, st in zip(os, streams):
                dev.bind_stream(0, st)
                o.attn()
        torch.cuda.synchronize()
        for o in os:
            check_attn(o, True)
    finally:
        dev.bind_stream(0)


OTHER = [([70, 200], [3, 40], 4, 2, 80, 16), ([33], [5], 3, 1, 1, 7), ([150], [1], 2, 2, 256, 16), ([64, 9], [2, 2], 6, 3, 96, 5),
         ([130], [129], 2, 1, 128, 1), ([77], [1], 4, 1, 128, 3), ([40], [6], 2, 1, 33, 4)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", range(len(OTHER)), ids=lambda n: "-".join(map(str, OTHER[n][2:])))
def test_other_head_and_page_sizes(dev, n, kind):
    attn_case(dev, 90 + n, *OTHER[n], kind, True)


@pytest.mark.parametrize("dim, page", [(128, 16), (64, 32), (80, 16)])
@pytest.mark.parametrize("q", [[1, 1, 1], [40, 1, 100]])
def test_rows_of_no_sequence_stay(dev, dim, page, q):
    attn_case(dev, 7, [300, 5, 120], q, 8, 2, dim, page, "f16", True, lead=3, trail=5, wide=40)


@pytest.mark.parametrize("dim, page", [(128, 16), (64, 64), (72, 16)])
def test_unaligned_tensors(dev, dim, page):
    """Tensors that start two bytes into an allocation."""
    import torch
    c = ref.Cache(np.random.default_rng(5), [200, 31], [1, 20], 4, 2, dim, page, "bf16", fill=np.inf)
    for name in ("q", "k", "v", "out"):
        o = OnDevice(dev, c)
        t = getattr(o, name)
        moved = torch.empty(t.numel() + 1, dtype=torch.int16, device="cuda")[1:].view(t.shape)
        moved.copy_(t)
        setattr(o, name, moved)
        o.attn()
        dev.sync(0)
        check_attn(o, True, name)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_peaked_scores(dev, kind):
    """Scores far from one another: the running maximum moves in every tile,
    and most weights vanish."""
    for seed, dim, q in ((1, 128, [1, 1]), (2, 128, [150, 64]), (3, 64, [1, 3]), (4, 64, [200, 5])):
        c = ref.Cache(np.random.default_rng(seed), [1500, 600], q, 8, 2, dim, 16, kind, q_by=12.0, fill=np.nan)
        # keys that grow along the sequence
        k = ref.to64(c.k)
        for b, n in enumerate(c.kv_lens):
            j = np.arange(n)
            at = (c.table[b, j // 16], slice(None), j % 16)
            k[at] *= (0.2 + 3.0 * j / n)[:, None, None]
        c.k = ref.to16(k, kind)
        o = OnDevice(dev, c)
        o.attn()
        dev.sync(0)
        check_attn(o, True, f"dim {dim} q {q}")


def test_all_scores_far_below_zero(dev):
    for q in ([1], [130]):
        c = ref.Cache(np.random.default_rng(9), [400], q, 4, 1, 128, 16, "bf16", fill=np.nan)
        c.q = ref.to16(np.abs(ref.to64(c.q)) * 8, "bf16")
        c.k = ref.to16(-np.abs(ref.to64(c.k)) * 8, "bf16")
        o = OnDevice(dev, c)
        o.attn()
        dev.sync(0)
        check_attn(o, True)


def test_a_non_finite_sequence_leaves_the_others(dev):
    """Not-a-number and infinities among one sequence's keys and values make
    its own rows not-a-number, and nobody else's."""
    for dim, q in ((128, [1, 1, 1]), (128, [40, 70, 90]), (64, [1, 1, 1]), (64, [3, 200, 5])):
        c = ref.Cache(np.random.default_rng(11), [300, 170, 290], q, 4, 2, dim, 16, "f16")
        k, v = ref.to64(c.k), ref.to64(c.v)
        k[c.table[1, 0], 0, 3] = np.nan
        v[c.table[1, 1], 1, 2] = np.nan
        c.k, c.v = ref.to16(k, "f16"), ref.to16(v, "f16")
        o = OnDevice(dev, c)
        o.attn()
        dev.sync(0)
        out, lse = o.results()
        want, z, b_out, b_lse = ref.paged_attn(c, True)
        lo, hi = c.q_offs[1], c.q_offs[2]
        # the rows that see both (tokens 3 and 18 of 170)
        sees = lo + np.flatnonzero(170 - q[1] + np.arange(q[1]) >= 18)
        assert len(sees) and np.isnan(out[sees]).all() and np.isnan(lse[sees, :2]).all()
        rest = np.r_[0:lo, hi:c.total]
        near(out[rest], want[rest], b_out[rest], f"dim {dim} q {q}")
        near(lse[lo:hi, 2:], z[lo:hi, 2:], b_lse[lo:hi, 2:])


LATER = [   # kv, q, heads, kv_heads, dim, page: single tiles and pairs, whole items and cut ones
    ([300] * 40, [4] * 40, 4, 1, 128, 16), ([5000], [3], 10, 2, 128, 16), ([700] * 30, [7, 8] * 15, 4, 1, 64, 16),
    ([90] * 80, [40] * 80, 4, 2, 64, 16), ([4000], [60], 4, 2, 128, 16), ([200] * 90, [200] * 90, 4, 2, 128, 32),
    ([1500], [400], 2, 2, 64, 64), ([33, 20], [33, 50], 4, 1, 80, 16), ([40] * 20, [90] * 20, 2, 1, 128, 16),
]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", range(len(LATER)), ids=lambda n: "-".join(map(str, LATER[n][2:])) + f"x{len(LATER[n][0])}")
def test_later_tokens_that_are_not_finite(dev, n, kind):
    """Rows before a token whose key or values are not finite do not know of it."""
    kv, q, heads, kv_heads, dim, page = LATER[n]
    rng = np.random.default_rng(70 + n)
    c = ref.Cache(rng, kv, q, heads, kv_heads, dim, page, kind, fill=np.nan)
    k, v = ref.to64(c.k), ref.to64(c.v)
    first, second = np.zeros(len(kv), int), np.zeros(len(kv), int)
    for b, (n_kv, n_q) in enumerate(zip(kv, q)):
        new = min(n_q, n_kv)
        first[b], second[b] = sorted(rng.integers(n_kv - new + 1, n_kv, 2)) if new > 2 else (n_kv - 1, n_kv - 1)
        at = lambda j: (c.table[b, j // page], slice(None), j % page)
        v[at(first[b])] = np.where(np.arange(dim) < 5, np.nan, np.where(np.arange(dim) < 8, -np.inf, v[at(first[b])]))
        v[at(second[b])] = np.where(np.arange(dim) % 7 == 3, np.inf, v[at(second[b])])
        k[at(second[b])] = np.nan
    c.k, c.v = ref.to16(k, kind), ref.to16(v, kind)
    o = OnDevice(dev, c)
    o.attn()
    dev.sync(0)
    out, lse = o.results()
    # what no key of a row is, it must not see: the expected values come from finite keys
    c.k = ref.to16(np.where(np.isnan(k), 0.0, k), kind)
    want, z, b_out, b_lse = ref.paged_attn(c)
    got = ref.to64(out)
    for b, (n_kv, n_q) in enumerate(zip(kv, q)):
        rows = np.arange(c.q_offs[b], c.q_offs[b + 1])
        sees = n_kv - n_q + np.arange(n_q)                 # the last token that each sees
        before = rows[sees < first[b]]
        near(out[before], want[before], b_out[before], f"sequence {b} before")
        near(lse[before], z[before], b_lse[before], f"sequence {b} lse before")
        if first[b] < second[b]:
            mid = rows[(sees >= first[b]) & (sees < second[b])]
            assert np.isnan(got[mid][..., :5]).all() and (got[mid][..., 5:8] == -np.inf).all()
            near(out[mid][..., 8:], want[mid][..., 8:], b_out[mid][..., 8:], f"sequence {b} between")
            near(lse[mid], z[mid], b_lse[mid], f"sequence {b} lse between")
        last = rows[sees >= second[b]]
        assert np.isnan(got[last]).all() and np.isnan(lse[last]).all()


@pytest.mark.parametrize("dim", [128, 64, 80])
@pytest.mark.parametrize("q", [[1, 1, 1], [60, 35, 50]])
def test_bad_indices_are_skipped_and_reported(dev, dim, q):
    from hexkernels_b200 import HexcudaError
    rng = np.random.default_rng(13)

    def run(change):
        c = ref.Cache(rng, [300, 200, 250], q, 8, 2, dim, 16, "f16")
        good = OnDevice(dev, c)
        o = OnDevice(dev, c)
        s = up(np.zeros((c.pages, 2, 16), np.float32))
        change(o)
        o.attn()
        with pytest.raises(HexcudaError, match="out of range") as e:
            dev.sync(0)
        assert e.value.code == 1
        o.lse.zero_()
        o.scores(s)
        with pytest.raises(HexcudaError, match="out of range"):
            dev.sync(0)
        dev.sync(0)     # reported once
        good.attn()
        dev.sync(0)
        a, _ = o.results()
        b, _ = good.results()
        return c, a, b

    for page in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        def change(o):
            o.table[1, 3] = page
        c, a, b = run(change)
        for i in (0, 2):
            np.testing.assert_array_equal(a[c.q_offs[i]:c.q_offs[i + 1]], b[c.q_offs[i]:c.q_offs[i + 1]])
    for n in (-5, 10 ** 6, 2 ** 31 - 1):
        def change(o):
            o.lens[0] = n
        c, a, b = run(change)
        np.testing.assert_array_equal(a[c.q_offs[1]:], b[c.q_offs[1]:])
    for i, n in ((1, -3), (1, 10 ** 6), (0, -1), (3, 2 ** 31 - 1), (2, 0)):
        def change(o):
            o.offs[i] = n
        run(change)


def test_no_lse_and_any_max_q(dev):
    rng = np.random.default_rng(17)
    for q in ([1, 1], [90, 3]):
        c = ref.Cache(rng, [300, 77], q, 8, 2, 128, 16, "f16", fill=np.nan)
        for max_q in (0, 1, 5, 90, 100000):
            o = OnDevice(dev, c, max_q=max_q)
            o.attn(lse=False)
            dev.sync(0)
            assert (down(o.lse, np.zeros(0, np.float32)) == 123.0).all()
            o.attn()
            dev.sync(0)
            check_attn(o, True, f"q {q} max_q {max_q}")
            s = up(np.zeros(c.k.shape[:3], np.float32))
            o.scores(s)
            dev.sync(0)
            want, bound = ref.cache_scores(c, o.results()[1], np.zeros(c.k.shape[:3], np.float32), True)
            near(down(s, np.zeros(0, np.float32)), want, bound, f"q {q} max_q {max_q}")


def test_output_must_not_be_the_queries(dev):
    from hexkernels_b200 import HexcudaError
    c = ref.Cache(np.random.default_rng(4), [40], [3], 4, 1, 64, 16)
    o = OnDevice(dev, c)
    o.out = o.q
    with pytest.raises(HexcudaError, match="out is q"):
        o.attn()


def test_workspace_must_be_large_enough(dev):
    from hexkernels_b200 import HexcudaError
    c = ref.Cache(np.random.default_rng(1), [30], [1], 4, 1, 64, 16)
    o = OnDevice(dev, c)
    o.space = o.space[:-16]
    with pytest.raises(HexcudaError, match="workspace"):
        o.attn()
    o.space = space(dev)[1:]
    with pytest.raises(HexcudaError, match="workspace"):
        o.attn()


def test_results_do_not_depend_on_the_run(dev):
    """Twice the same bits, whatever the workspace held."""
    for q in ([1, 1, 1, 1], [130, 1, 64, 200]):
        c = ref.Cache(np.random.default_rng(19), [3000, 10, 700, 2000], q, 16, 4, 128, 16, "bf16")
        got = []
        for fill in (0, 0x7f, 0xff):
            o = OnDevice(dev, c)
            o.space.fill_(fill)
            s = up(np.zeros(c.k.shape[:3], np.float32))
            o.attn()
            o.scores(s)
            dev.sync(0)
            got.append((*o.results(), down(s, np.zeros(0, np.float32))))
        for x in got[1:]:
            for a, b in zip(got[0], x):
                np.testing.assert_array_equal(a, b)


def test_other_stream_and_two_graphs(dev, hx):
    """Work on a side stream, then two captured graphs replayed on two streams
    at once, each with its own workspace."""
    import torch
    rng = np.random.default_rng(23)
    cs = [ref.Cache(rng, [900, 20, 333], [1, 1, 1], 32, 8, 128, 16, "f16"),
          ref.Cache(rng, [500, 260], [300, 7], 8, 2, 64, 32, "bf16")]
    os = [OnDevice(dev, c) for c in cs]
    scores = [up(np.zeros(c.k.shape[:3], np.float32)) for c in cs]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    try:
        for o, s, st in zip(os, scores, side):
            dev.bind_stream(0, st)
            o.attn()
            o.scores(s)
            st.synchronize()
            check_attn(o, True, "side stream")
            s.zero_()
            o.out.zero_()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                o.attn()
                o.scores(s)
            graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(3):
            for o, s in zip(os, scores):
                s.zero_()
                o.out.fill_(0x7e5a)
            torch.cuda.synchronize()
            for g, st in zip(graphs, side):
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for o, s in zip(os, scores):
                check_attn(o, True, "replayed")
                want, bound = ref.cache_scores(o.c, o.results()[1], np.zeros(o.c.k.shape[:3], np.float32), True)
                near(down(s, np.zeros(0, np.float32)), want, bound, "replayed scores")
        # new lengths and tables in the same buffers: the graph reads them anew
        o, c = os[0], cs[0]
        c.kv_lens = np.array([17, 20, 300], np.int32)
        o.lens.copy_(torch.from_numpy(c.kv_lens))
        graphs[0].replay()
        torch.cuda.synchronize()
        check_attn(o, True, "shorter")
    finally:
        del graphs
        dev.bind_stream(0)


def test_shared_pages_collect_from_every_sequence(dev):
    """Two sequences with a common prompt: its scores get both weights."""
    c = ref.Cache(np.random.default_rng(29), [160, 200, 90], [1, 30, 2], 8, 2, 128, 16, "f16")
    c.table[1, :6] = c.table[0, :6]
    c.table[2, :5] = c.table[0, :5]
    o = OnDevice(dev, c)
    o.attn()
    base = np.zeros(c.k.shape[:3], np.float32)
    s = up(base)
    o.scores(s)
    dev.sync(0)
    check_attn(o, True)
    want, bound = ref.cache_scores(c, o.results()[1], base, True)
    near(down(s, base), want, bound)


# ------------------------------------------------------------------ eviction

def evict(dev, c, scores, budget, sink, recent, dst=None, alias=False):
    import torch
    k, v, s = up(c.k), up(c.v), up(scores)
    table, lens = up(c.table), up(c.kv_lens)
    to = up(dst)
    new = lens if alias else torch.full_like(lens, 77)
    kept = torch.full((len(c.kv_lens), c.kv_heads, budget), 99, dtype=torch.int32, device="cuda")
    dev.launch("cache_evict", 0, k, v, s, table, to, lens, new, kept, len(c.kv_lens), c.kv_heads, c.dim, c.pages,
               c.page, c.wide, 0 if dst is None else dst.shape[1], budget, sink, recent)
    dev.sync(0)
    return down(kept, c.table), down(new, c.table), down(k, c.k), down(v, c.v), down(s, scores)


def weights(rng, c, ties=True):
    x = np.exp(1.5 * rng.standard_normal(c.k.shape[:3]))
    return (np.round(x * 8) / 8 if ties else x).astype(np.float32)


def same(got, want):
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.view(np.uint16) if a.dtype == np.float16 else a.view(np.int32) if a.dtype == np.float32 else a,
                                      b.view(np.uint16) if b.dtype == np.float16 else b.view(np.int32) if b.dtype == np.float32 else b)


EVICT = [
    ([40], 1, 128, 16, 10, 2, 3), ([1000, 3, 0, 65, 64], 3, 64, 16, 64, 4, 16), ([5000, 100], 2, 128, 32, 1024, 4, 256),
    ([300, 299], 2, 80, 16, 100, 0, 0), ([129, 700], 1, 33, 7, 50, 50, 0), ([129, 700], 1, 128, 1, 50, 0, 50),
    ([77], 2, 128, 24, 76, 1, 1), ([9000], 1, 64, 64, 1, 0, 0), ([2500], 4, 128, 16, 2048, 1, 2047), ([70000], 1, 64, 128, 3000, 16, 500),
]


@pytest.mark.parametrize("place", ["in place", "same table", "new pages"])
@pytest.mark.parametrize("n", range(len(EVICT)), ids=lambda n: "-".join(map(str, EVICT[n][1:])))
def test_evict(dev, n, place):
    kv, kv_heads, dim, page, budget, sink, recent = EVICT[n]
    rng = np.random.default_rng(100 + n)
    need = [-(-min(x, budget) // page) for x in kv]
    c = ref.Cache(rng, kv, [0] * len(kv), kv_heads, kv_heads, dim, page, "f16" if n % 2 else "bf16", spare=sum(need) + 1)
    s = weights(rng, c)
    dst = None
    if place == "same table":
        dst = np.pad(c.table, ((0, 0), (0, -(-budget // page))), constant_values=-7)
    elif place == "new pages":
        dst = np.full((len(kv), -(-budget // page) + 1), -9, np.int32)
        at = 0
        for b, m in enumerate(need):
            dst[b, :m] = c.free[at:at + m]
            at += m
    same(evict(dev, c, s, budget, sink, recent, dst), ref.cache_evict(c, s, budget, sink, recent, dst))


@pytest.mark.parametrize("what", ["zeros", "equal", "special", "one ulp"])
def test_evict_ties_and_special_scores(dev, what):
    rng = np.random.default_rng(41)
    c = ref.Cache(rng, [3000, 1500, 700], [0] * 3, 2, 2, 64, 16, "f16")
    shape = c.k.shape[:3]
    s = {"zeros": np.where(rng.random(shape) < 0.5, 0.0, -0.0), "equal": np.full(shape, 2.5),
         "special": rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42, -1e-42, 3.4e38, -1.0, 1.0], shape),
         "one ulp": np.nextafter(np.float32(1), np.float32(2), dtype=np.float32) ** rng.integers(0, 2, shape)}[what].astype(np.float32)
    for budget, sink, recent in ((1000, 4, 100), (700, 0, 0), (699, 1, 0)):
        same(evict(dev, c, s, budget, sink, recent), ref.cache_evict(c, s, budget, sink, recent))


@pytest.mark.parametrize("wide", [600, 2000, 30000])
def test_evict_with_wide_tables(dev, wide):
    """Tables that could name far more tokens than there are: more CTAs to a
    sequence, and (480000 tokens) keys that are not kept in shared memory."""
    rng = np.random.default_rng(59)
    c = ref.Cache(rng, [3000, 10, 7777], [0] * 3, 2, 2, 64, 16, "f16", wide=wide)
    s = weights(rng, c)
    for budget, sink, recent in ((1000, 4, 100), (64, 0, 0)):
        same(evict(dev, c, s, budget, sink, recent), ref.cache_evict(c, s, budget, sink, recent))


def test_evict_many_sequences(dev):
    rng = np.random.default_rng(67)
    kv = rng.integers(0, 900, 120)
    c = ref.Cache(rng, kv.tolist(), [0] * 120, 4, 4, 64, 16, "bf16")
    s = weights(rng, c)
    same(evict(dev, c, s, 128, 4, 32), ref.cache_evict(c, s, 128, 4, 32))


def test_evict_lengths_in_the_same_buffer(dev):
    rng = np.random.default_rng(43)
    c = ref.Cache(rng, [500, 64, 0, 65, 2000], [0] * 5, 4, 4, 128, 16, "f16")
    s = weights(rng, c)
    same(evict(dev, c, s, 64, 2, 8, alias=True), ref.cache_evict(c, s, 64, 2, 8))


def test_evict_again_and_again(dev):
    """Cut, then cut what is left: each round from the last one's result."""
    rng = np.random.default_rng(47)
    c = ref.Cache(rng, [4000, 900], [0, 0], 2, 2, 128, 16, "bf16")
    s = weights(rng, c, ties=False)
    for budget in (2000, 1000, 333, 5):
        got, want = evict(dev, c, s, budget, 2, 3), ref.cache_evict(c, s, budget, 2, 3)
        same(got, want)
        _, c.kv_lens, c.k, c.v, s = got


def test_evict_bad_indices(dev):
    from hexkernels_b200 import HexcudaError
    rng = np.random.default_rng(53)
    for where in ("table", "dst", "len", "negative"):
        c = ref.Cache(rng, [500, 300, 400], [0] * 3, 2, 2, 64, 16, "f16", spare=20)
        s = weights(rng, c)
        dst = c.free[:18].reshape(3, 6).copy()
        want = ref.cache_evict(c, s, 90, 1, 5, dst)
        if where == "table":
            c.table[1, 4] = -3
        elif where == "dst":
            dst[1, 2] = c.pages
        else:
            c.kv_lens[1] = 10 ** 8 if where == "len" else -1
        k, v = c.k, c.v
        with pytest.raises(HexcudaError, match="out of range"):
            evict(dev, c, s, 90, 1, 5, dst)
        assert k is c.k and v is c.v
        dev.sync(0)
        # the other sequences are served all the same
        kk, vv, ss = up(c.k), up(c.v), up(s)
        kept = up(np.zeros((3, 2, 90), np.int32))
        new = up(np.zeros(3, np.int32))
        dev.launch("cache_evict", 0, kk, vv, ss, up(c.table), up(dst), up(c.kv_lens), new, kept, 3, 2, 64, c.pages, 16,
                   c.wide, 6, 90, 1, 5)
        with pytest.raises(HexcudaError):
            dev.sync(0)
        for b in (0, 2):
            np.testing.assert_array_equal(down(kept, c.table)[b], want[0][b])
            pages = dst[b]
            np.testing.assert_array_equal(down(kk, c.k)[pages], want[2][pages])
            np.testing.assert_array_equal(down(ss, s)[pages], want[4][pages])


# ----------------------------------------------------- norm, rotation, append

def norm_rope(dev, rng, T, heads, kv_heads, dim, rot, page, kind, halves=True, norm=True, gains=True, values=True,
              scores=True, pad=0, shift=0, inplace=False, eps=1e-6, table=300):
    import torch
    x = ref.to16(rng.standard_normal((T, (heads + 2 * kv_heads) * dim + pad)) * 2, kind)
    q, k, v = (x[:, a * dim:b * dim].reshape(T, b - a, dim) for a, b in
               ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    qg, kg = (ref.to16(1 + 0.2 * rng.standard_normal(dim), kind) if gains else None for _ in range(2))
    cos, sin = ref.turns(table, rot)
    pos = rng.integers(0, table, T).astype(np.int32)
    if T > 1:
        pos[:2] = 0, table - 1
    pages = -(-T // page) + 2
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    skip = rng.random(T) < 0.2 if T > 4 else np.zeros(T, bool)
    slots[skip] = -1
    pos[skip] = 10 ** 9     # never looked at
    kp = ref.to16(rng.standard_normal((pages, kv_heads, page, dim)), kind)
    vp, sc = kp[::-1].copy(), np.ones(kp.shape[:3], np.float32)
    d = up(x).view(-1)
    packed = torch.empty(d.numel() + shift, dtype=torch.int16, device="cuda")[shift:]
    packed.copy_(d)
    wide = x.shape[1]
    if inplace:
        packed = torch.cat([up(q).view(-1), up(k).view(-1), up(v).view(-1)])
        at = [packed, packed[T * heads * dim:], packed[T * (heads + kv_heads) * dim:]]
        stride = [heads * dim, kv_heads * dim, kv_heads * dim]
        out = packed
    else:
        at, stride = [packed, packed[heads * dim:], packed[(heads + kv_heads) * dim:]], [wide] * 3
        out = torch.full((T * heads * dim + shift,), 0x1234, dtype=torch.int16, device="cuda")[shift:]
    dk, dv, ds = up(kp), up(vp), up(sc)
    dev.launch("qk_norm_rope", 0, CODE[kind], at[0], stride[0], at[1], stride[1], at[2] if values else None, stride[2],
               up(qg), up(kg), up(cos), up(sin), up(pos), up(slots), out, dk, dv if values else None,
               ds if scores else None, T, heads, kv_heads, dim, rot, int(halves), int(norm), table, pages, page, eps)
    dev.sync(0)
    live = ~skip
    mark = np.uint16(0x1234)
    got = out[:T * heads * dim].cpu().numpy().view(q.dtype).reshape(T, heads, dim)
    want, bound = ref.qk_norm_rope(q[live], qg, cos, sin, pos[live], halves, norm, eps)
    near(got[live], want, bound, "queries")
    if not inplace:
        assert (got[skip].view(np.uint16) == mark).all()
    want, bound = ref.qk_norm_rope(k[live], kg, cos, sin, pos[live], halves, norm, eps)
    where, off = slots[live] // page, slots[live] % page
    gk, gv, gs = down(dk, kp), down(dv, vp), down(ds, sc)
    near(gk[where, :, off], want, bound, "keys")
    bits = lambda a: a.view(np.uint16)
    untouched = np.ones((pages, page), bool)
    untouched[where, off] = False
    np.testing.assert_array_equal(bits(gk.transpose(0, 2, 1, 3)[untouched]), bits(kp.transpose(0, 2, 1, 3)[untouched]))
    if values:
        np.testing.assert_array_equal(bits(gv[where, :, off]), bits(v[live]))
        np.testing.assert_array_equal(bits(gv.transpose(0, 2, 1, 3)[untouched]), bits(vp.transpose(0, 2, 1, 3)[untouched]))
    else:
        np.testing.assert_array_equal(bits(gv), bits(vp))
    want = sc.copy()
    if scores:
        want[where, :, off] = 0
    np.testing.assert_array_equal(gs, want)


NORM = [(1, 32, 8, 128, 128, 16), (37, 8, 2, 128, 128, 16), (253, 20, 4, 64, 32, 32), (5, 3, 1, 256, 256, 8), (9, 4, 4, 80, 80, 5),
        (11, 2, 1, 33, 32, 3), (70, 7, 7, 128, 64, 64), (6, 1, 1, 2, 2, 4), (8, 5, 1, 64, 0, 16), (13, 4, 2, 96, 48, 16), (21, 4, 2, 128, 6, 16),
        (4, 2, 1, 1, 0, 2), (17, 130, 2, 64, 64, 16), (10, 4, 2, 256, 64, 16), (33, 4, 2, 32, 32, 16), (12, 2, 2, 8, 8, 16), (12, 2, 2, 24, 24, 16)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("n", range(len(NORM)), ids=lambda n: "-".join(map(str, NORM[n])))
def test_norm_rope(dev, n, halves, kind):
    norm_rope(dev, np.random.default_rng(200 + n), *NORM[n], kind, halves=halves)


@pytest.mark.parametrize("kw", [dict(norm=False), dict(gains=False), dict(values=False), dict(scores=False), dict(pad=8), dict(pad=3),
                                dict(shift=1), dict(shift=4), dict(inplace=True), dict(eps=0.0), dict(eps=0.5), dict(table=1)], ids=str)
@pytest.mark.parametrize("dim, halves", [(128, True), (64, False), (72, True)])
def test_norm_rope_forms(dev, dim, halves, kw):
    norm_rope(dev, np.random.default_rng(300), 41, 6, 3, dim, dim // 2, 16, "bf16", halves=halves, **kw)
    norm_rope(dev, np.random.default_rng(301), 2, 6, 3, dim, dim, 16, "f16", halves=halves, **kw)


def test_norm_rope_extreme_rows(dev):
    """Rows of zeros, of the largest values and of the smallest."""
    kind, T, H, D = "f16", 6, 2, 128
    x = np.zeros((T, H, D), np.float16)
    x[1], x[2], x[3, :, 5], x[4] = 65504, 6e-8, 65504, -1
    x[5] = np.random.default_rng(0).choice([65504, 6e-8, 1], (H, D))
    cos, sin = ref.turns(8, D)
    pos = np.arange(T, dtype=np.int32)
    for eps in (1e-6, 1e-12):
        out = up(np.zeros_like(x))
        dev.launch("qk_norm_rope", 0, 0, up(x), H * D, None, 0, None, 0, None, None, up(cos), up(sin), up(pos), None, out,
                   None, None, None, T, H, 0, D, D, 1, 1, 8, 0, 0, eps)
        dev.sync(0)
        want, bound = ref.qk_norm_rope(x, None, cos, sin, pos, True, True, eps)
        near(down(out, x), want, bound, f"eps {eps}")


def test_norm_rope_bad_indices(dev):
    from hexkernels_b200 import HexcudaError
    rng = np.random.default_rng(61)
    T, H, KV, D, page, pages = 8, 4, 2, 128, 16, 3
    x = ref.to16(rng.standard_normal((T, (H + 2 * KV), D)), "f16")
    cos, sin = ref.turns(20, D)
    for dim_bad, at in (("pos", 20), ("pos", -1), ("pos", 2 ** 31 - 1), ("slot", pages * page), ("slot", 2 ** 31 - 1)):
        pos, slots = np.arange(T, dtype=np.int32), np.arange(T, dtype=np.int32)
        (pos if dim_bad == "pos" else slots)[3] = at
        k = up(np.zeros((pages, KV, page, D), np.float16))
        v = k.clone()
        out = up(np.zeros((T, H, D), np.float16))
        packed = up(x).view(-1)
        dev.launch("qk_norm_rope", 0, 0, packed, (H + 2 * KV) * D, packed[H * D:], (H + 2 * KV) * D,
                   packed[(H + KV) * D:], (H + 2 * KV) * D, None, None, up(cos), up(sin), up(pos), up(slots), out, k, v,
                   None, T, H, KV, D, D, 1, 1, 20, pages, page, 1e-6)
        with pytest.raises(HexcudaError, match="out of range"):
            dev.sync(0)
        live = np.arange(T) != 3
        want, bound = ref.qk_norm_rope(x[live][:, :H], None, cos, sin, pos[live], True, True, 1e-6)
        got = down(out, x)
        near(got[live], want, bound)
        assert (got[3] == 0).all()
        assert (down(k, x)[0, :, 3] == 0).all() and (down(v, x)[0, :, 3] == 0).all()


# ------------------------------------------------------------- host entries

@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_host_entries(hx, kind):
    rng = np.random.default_rng(71)
    T, H, KV, D, page = 7, 8, 2, 64, 16
    x = ref.to16(rng.standard_normal((T, H + 2 * KV, D)), kind)
    c = ref.Cache(rng, [100, 40], [4, 3], H, KV, D, page, kind)
    s = np.ones(c.k.shape[:3], np.float32)
    cos, sin = ref.turns(128, D)
    pos = np.array([96, 97, 98, 99, 37, 38, 39], np.int32)
    slots = np.array([c.table[b, j // page] * page + j % page for b, j in zip([0] * 4 + [1] * 3, pos)], np.int32)
    g = ref.to16(1 + 0.1 * rng.standard_normal(D), kind)
    k0 = c.k.copy()
    q = hx.qk_norm_rope(x[:, :H], x[:, H:H + KV], x[:, H + KV:], c.k, c.v, cos, sin, pos, slots, g, g, s)
    near(q, *ref.qk_norm_rope(x[:, :H], g, cos, sin, pos, True, True, 1e-6), "queries")
    near(c.k[slots // page, :, slots % page], *ref.qk_norm_rope(x[:, H:H + KV], g, cos, sin, pos, True, True, 1e-6), "keys")
    np.testing.assert_array_equal(c.v[slots // page, :, slots % page].view(np.uint16), x[:, H + KV:].view(np.uint16))
    assert (s[slots // page, :, slots % page] == 0).all() and s.sum() == s.size - T * KV
    assert (c.k != k0).any()
    c.q = q
    out, lse = hx.paged_attn(q, c.k, c.v, c.table, c.kv_lens, c.q_offs)
    want, z, b_out, b_lse = ref.paged_attn(c)
    near(out, want, b_out, "out")
    near(lse, z, b_lse, "lse")
    base = s.copy()
    hx.cache_scores(q, lse, c.k, c.table, c.kv_lens, c.q_offs, s)
    near(s, *ref.cache_scores(c, lse, base), "scores")
    want = ref.cache_evict(c, s, 32, 1, 4)
    kept, new = hx.cache_evict(c.k, c.v, s, c.table, c.kv_lens, 32, 1, 4)
    same((kept, new, c.k, c.v, s), want)


def test_host_entries_report_bad_indices_and_leave_the_outputs(hx):
    from hexkernels_b200 import HexcudaError
    c = ref.Cache(np.random.default_rng(73), [100, 40], [4, 3], 4, 2, 64, 16)
    c.table[0, 1] = c.pages
    s = np.ones(c.k.shape[:3], np.float32)
    k, v = c.k.copy(), c.v.copy()
    with pytest.raises(HexcudaError, match="out of range"):
        hx.paged_attn(c.q, c.k, c.v, c.table, c.kv_lens, c.q_offs)
    with pytest.raises(HexcudaError, match="out of range"):
        hx.cache_evict(c.k, c.v, s, c.table, c.kv_lens, 32, 1, 4)
    np.testing.assert_array_equal(k, c.k)
    np.testing.assert_array_equal(v, c.v)
    assert (s == 1).all()
    assert hx.paged_attn(c.q[:0], c.k, c.v, c.table[:0], c.kv_lens[:0], np.zeros(1, np.int32))[0].shape == (0, 4, 64)


def test_shims(hx):
    """The candidate_kernel of each operator is its host entry."""
    from pathlib import Path
    shims = Path(__file__).resolve().parent.parent / "hexkernels_b200" / "shims"
    p = lambda a: a.ctypes.data_as(C.c_void_p)
    c = ref.Cache(np.random.default_rng(79), [90, 33], [2, 5], 4, 2, 64, 16)
    B, T, scale = 2, 7, C.c_float(0.125)
    out, lse = np.zeros_like(c.q), np.zeros(c.q.shape[:2], np.float32)
    C.CDLL(str(shims / "libcand_paged_attn.so")).candidate_kernel(
        0, p(c.q), p(c.k), p(c.v), p(c.table), p(c.kv_lens), p(c.q_offs), p(out), p(lse), B, T, 5, 4, 2, 64, c.pages, 16,
        c.wide, scale, 1)
    c.scale = 0.125
    want, z, b_out, b_lse = ref.paged_attn(c)
    near(out, want, b_out)
    near(lse, z, b_lse)
    s = np.zeros(c.k.shape[:3], np.float32)
    C.CDLL(str(shims / "libcand_cache_scores.so")).candidate_kernel(
        0, p(c.q), p(lse), p(c.k), p(c.table), p(c.kv_lens), p(c.q_offs), p(s), B, T, 5, 4, 2, 64, c.pages, 16, c.wide,
        scale, 1)
    near(s, *ref.cache_scores(c, lse, np.zeros_like(s)))
    want = ref.cache_evict(c, s, 32, 1, 2)
    kept, new = np.zeros((2, 2, 32), np.int32), np.zeros(2, np.int32)
    C.CDLL(str(shims / "libcand_cache_evict.so")).candidate_kernel(
        p(c.k), p(c.v), p(s), p(c.table), None, p(c.kv_lens), p(new), p(kept), B, 2, 64, c.pages, 16, c.wide, 0, 32, 1, 2)
    same((kept, new, c.k, c.v, s), want)
    x = ref.to16(np.random.default_rng(1).standard_normal((3, 8, 64)), "f16")
    cos, sin = ref.turns(9, 64)
    pos = slots = np.arange(3, dtype=np.int32)
    q = np.zeros((3, 4, 64), np.float16)
    L = C.c_int64(512)
    C.CDLL(str(shims / "libcand_qk_norm_rope.so")).candidate_kernel(
        0, p(x), L, C.c_void_p(x.ctypes.data + 512), L, C.c_void_p(x.ctypes.data + 768), L, None, None, p(cos), p(sin),
        p(pos), p(slots), p(q), p(c.k), p(c.v), None, 3, 4, 2, 64, 64, 0, 1, 9, c.pages, 16, C.c_float(1e-6))
    near(q, *ref.qk_norm_rope(x[:, :4], None, cos, sin, pos, False, True, 1e-6))
    near(c.k[0, :, :3].transpose(1, 0, 2), *ref.qk_norm_rope(x[:, 4:6], None, cos, sin, pos, False, True, 1e-6))


# ---------------------------------------------------------- a run of them all

@pytest.mark.parametrize("kind, dim", [("f16", 128), ("bf16", 64)])
def test_serving_loop(dev, kind, dim):
    """A prompt in chunks, then single tokens: norm and rotation into the
    cache, attention, collected weight, and a cut whenever a sequence outgrows
    its budget.  Every step's outputs are compared with the 64-bit
    implementations on the state that the step found."""
    import torch
    rng = np.random.default_rng(83)
    H, KV, page, wide, budget = 8, 2, 16, 12, 96
    B = 3
    table = rng.permutation(B * wide).astype(np.int32).reshape(B, wide)
    c = ref.Cache(rng, [0] * B, [0] * B, H, KV, dim, page, kind, wide=wide, spare=B * wide)
    c.table = table
    lens, seen = np.zeros(B, np.int32), np.zeros(B, np.int64)
    gains = [ref.to16(1 + 0.1 * rng.standard_normal(dim), kind) for _ in range(2)]
    cos, sin = ref.turns(4096, dim)
    k, v, s = up(c.k), up(c.v), up(np.full(c.k.shape[:3], 5.0, np.float32))
    work = space(dev)
    f32 = np.zeros(0, np.float32)
    for new in ([50, 1, 90], [40, 70, 20], [1, 1, 1], [1, 1, 1], [60, 1, 1], [1, 1, 1], [1, 0, 1]):
        new = np.array(new, np.int32)
        T = int(new.sum())
        x = ref.to16(rng.standard_normal((T, H + 2 * KV, dim)), kind)
        seq = np.repeat(np.arange(B), new)
        place = np.concatenate([lens[b] + np.arange(n) for b, n in enumerate(new)]).astype(np.int64)
        pos = np.concatenate([seen[b] + np.arange(n) for b, n in enumerate(new)]).astype(np.int32)
        slots = (table[seq, place // page] * page + place % page).astype(np.int32)
        stride = (H + 2 * KV) * dim
        packed, out = up(x).view(-1), torch.zeros(T * H * dim, dtype=torch.int16, device="cuda")
        code = CODE[kind]
        dev.launch("qk_norm_rope", 0, code, packed, stride, packed[H * dim:], stride, packed[(H + KV) * dim:], stride, up(gains[0]),
                   up(gains[1]), up(cos), up(sin), up(pos), up(slots), out, k, v, s, T, H, KV, dim, dim, 1, 1, 4096, c.pages, page, 1e-6)
        lens, seen = lens + new, seen + new
        offs = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        o, lse = torch.zeros_like(out), torch.zeros(T, H, device="cuda")
        dims = (B, T, int(new.max()), H, KV, dim, c.pages, page, wide, dim ** -0.5, 1)
        dt, dl, do = up(table), up(lens), up(offs)
        before = down(s, f32).copy()
        dev.launch("paged_attn", 0, code, out, k, v, dt, dl, do, o, lse, work, work.numel(), *dims)
        dev.launch("cache_scores", 0, code, out, lse, k, dt, dl, do, s, *dims)
        dev.sync(0)
        # norm and rotation
        want, bound = ref.qk_norm_rope(x[:, :H], gains[0], cos, sin, pos, True, True, 1e-6)
        c.q = out.cpu().numpy().view(c.k.dtype).reshape(T, H, dim)
        near(c.q, want, bound, "queries")
        c.k, c.v = down(k, c.k), down(v, c.v)
        want, bound = ref.qk_norm_rope(x[:, H:H + KV], gains[1], cos, sin, pos, True, True, 1e-6)
        near(c.k[slots // page, :, slots % page], want, bound, "keys")
        assert (before[slots // page, :, slots % page] == 0).all()
        # attention and weights
        c.kv_lens, c.q_offs, c.total = lens.copy(), offs, T
        want, z, b_out, b_lse = ref.paged_attn(c)
        near(o.cpu().numpy().view(c.k.dtype).reshape(T, H, dim), want, b_out, "out")
        near(lse.cpu().numpy(), z, b_lse, "lse")
        after, bound = ref.cache_scores(c, lse.cpu().numpy(), before)
        near(down(s, f32), after, bound, "scores")
        if lens.max() > budget:
            now = down(s, f32).copy()
            kept = torch.empty(B, KV, budget, dtype=torch.int32, device="cuda")
            dev.launch("cache_evict", 0, k, v, s, dt, None, dl, dl, kept, B, KV, dim, c.pages, page, wide, 0, budget, 2, 16)
            dev.sync(0)
            want = ref.cache_evict(c, now, budget, 2, 16)
            same((down(kept, table), down(dl, table), down(k, c.k), down(v, c.v), down(s, f32)), want)
            lens = down(dl, table).copy()
    assert lens.max() <= budget < seen.max()
