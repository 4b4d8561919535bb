"""The paged-cache operators on inputs at the edge of what they take: values
that are not finite, rows and pages that do not count, calls without a cache.
Expected values are 64-bit, as in test_gpu_paged."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import CODE, OnDevice, check_attn, dev, down, near, up  # noqa: F401

pytestmark = pytest.mark.gpu
F32 = np.zeros(0, np.float32)


# ------------------------------------------------------------ qk_norm_rope

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dim, rot, shift", [(128, 64, 0), (128, 0, 0), (64, 16, 0), (80, 32, 0), (256, 128, 0), (128, 64, 1), (72, 32, 0)])
def test_columns_that_do_not_turn_keep_to_themselves(dev, dim, rot, shift, norm, halves, kind):
    """An infinity, a not-a-number or a zero of either sign behind the columns
    that turn is nobody else's."""
    import torch
    rng = np.random.default_rng(500 + dim + rot)
    T, H, KV, page, pages = 24, 3, 2, 16, 2
    x = rng.standard_normal((T, H + 2 * KV, dim))
    odd = rng.random(x.shape) < 0.05
    odd[..., :rot] = False
    odd[:4] = False
    x = np.where(odd, rng.choice([np.nan, np.inf, -np.inf], x.shape), x)
    x = np.where(rng.random(x.shape) < 0.2, rng.choice([0.0, -0.0], x.shape), x)
    x = ref.to16(x, kind)
    gain = ref.to16(1 + 0.2 * rng.standard_normal(dim), kind)
    cos, sin = ref.turns(40, rot)
    pos, slots = rng.integers(0, 40, T).astype(np.int32), np.arange(T, dtype=np.int32)
    packed = torch.empty(x.size + shift, dtype=torch.int16, device="cuda")[shift:]
    packed.copy_(up(x).view(-1))
    wide = (H + 2 * KV) * dim
    out = torch.empty(T * H * dim, dtype=torch.int16, device="cuda")
    k, v = (up(np.zeros((pages, KV, page, dim), x.dtype)) for _ in range(2))
    dev.launch("qk_norm_rope", 0, CODE[kind], packed, wide, packed[H * dim:], wide, packed[(H + KV) * dim:], wide, up(gain), up(gain),
               up(cos) if rot else None, up(sin) if rot else None, up(pos), up(slots), out, k, v, None, T, H, KV, dim, rot,
               int(halves), int(norm), 40, pages, page, 1e-6)
    dev.sync(0)
    got_q = out.cpu().numpy().view(x.dtype).reshape(T, H, dim)
    got_k = down(k, x)[slots // page, :, slots % page]
    for got, src in ((got_q, x[:, :H]), (got_k, x[:, H:H + KV])):
        with np.errstate(all="ignore"):
            want, bound = ref.qk_norm_rope(src, gain, cos, sin, pos, halves, norm, 1e-6)
        near(got, want, bound)
        if not norm:    # what does not turn is copied, to the sign of a zero
            kept = ~np.isnan(ref.to64(src))
            kept[..., :rot] = False
            np.testing.assert_array_equal(got.view(np.uint16)[kept], src.view(np.uint16)[kept])
    np.testing.assert_array_equal(down(v, x)[slots // page, :, slots % page].view(np.uint16), x[:, H + KV:].view(np.uint16))


@pytest.mark.parametrize("dim", [128, 72])
@pytest.mark.parametrize("pages, page", [(0, 16), (1, 1), (0, 1)])
def test_queries_alone_take_any_slot(dev, pages, page, dim):
    """Without key heads there is no cache: a slot says only whether the token
    counts, and the cache's sizes say nothing."""
    rng = np.random.default_rng(521)
    T, H = 40, 3
    x = ref.to16(rng.standard_normal((T, H, dim)), "bf16")
    cos, sin = ref.turns(64, dim)
    pos = rng.integers(0, 64, T).astype(np.int32)
    slots = rng.integers(0, 2 ** 31 - 1, T).astype(np.int32)
    slots[:2] = 0, 2 ** 31 - 1
    skip = np.arange(T) % 5 == 2
    slots[skip], pos[skip] = -1, -7
    out = up(np.full(x.shape, 0x1234, np.uint16))
    dev.launch("qk_norm_rope", 0, 1, up(x), H * dim, None, 0, None, 0, None, None, up(cos), up(sin), up(pos), up(slots), out, None,
               None, None, T, H, 0, dim, dim, 1, 1, 64, pages, page, 1e-6)
    dev.sync(0)
    got = down(out, x)
    want, bound = ref.qk_norm_rope(x[~skip], None, cos, sin, pos[~skip], True, True, 1e-6)
    near(got[~skip], want, bound)
    assert (got[skip] == 0x1234).all()


# ------------------------------------------------------------ cache_scores

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads, kv_heads, dim, page, causal", [(8, 2, 128, 16, True), (4, 4, 64, 32, True), (6, 1, 64, 8, False),
                                                                 (8, 2, 80, 16, True), (40, 1, 128, 16, False)])
@pytest.mark.parametrize("q", [[1, 1, 1], [9, 1, 3], [60, 33, 128], [300, 1, 40]])
def test_rows_of_no_weight_add_nothing(dev, q, heads, kv_heads, dim, page, causal, kind):
    """Rows whose lse is minus infinity count for nothing, whatever their query
    holds; the rows beside them count as before, one of plus infinity as zero."""
    rng = np.random.default_rng(531 + sum(q))
    c = ref.Cache(rng, [700, 90, 257], q, heads, kv_heads, dim, page, kind, fill=np.nan)
    o = OnDevice(dev, c, causal)
    o.attn()
    dev.sync(0)
    lse = o.results()[1].copy()
    none = rng.random(lse.shape) < 0.3
    none[0], none[-1] = True, False
    odd = np.where(rng.random(c.q.shape) < 0.5, rng.choice([np.nan, np.inf, -np.inf], c.q.shape), 0.0)
    x = np.where(none[..., None], np.where(odd == 0, ref.to64(c.q), odd), ref.to64(c.q))
    lse[none] = -np.inf
    full = ~none & (rng.random(lse.shape) < 0.05)
    lse[full] = np.inf
    o.q, o.lse = up(ref.to16(x, kind)), up(lse)
    base = rng.random((c.pages, kv_heads, page)).astype(np.float32)
    s = up(base)
    o.scores(s)
    dev.sync(0)
    # (exp(x - inf) is 0 without any rounding, so such a row adds nothing to the bound either)
    near(down(s, base), *ref.cache_scores(c, np.where(full, -np.inf, lse).astype(np.float32), base, causal))
    # all rows without weight, beside keys that are not finite: not a bit changes
    o.k = up(ref.to16(np.where(rng.random(c.k.shape) < 0.1, np.inf, ref.to64(c.k)), kind))
    o.lse.fill_(-np.inf)
    s = up(base)
    o.scores(s)
    dev.sync(0)
    np.testing.assert_array_equal(down(s, base), base)


# --------------------------------------------------------- pages that are not there

PAGES = [
    ([300, 200, 250], [1, 1, 1], 8, 2, 128, 16), ([300, 200, 250], [5, 1, 3], 8, 2, 64, 8), ([300, 200, 250], [60, 35, 50], 8, 2, 128, 16),
    ([900, 200, 250], [60, 35, 250], 4, 1, 64, 24), ([300, 200, 250], [1, 1, 1], 4, 2, 64, 256), ([300, 200, 250], [7, 60, 9], 4, 4, 128, 128),
    ([5000, 16, 33], [1, 1, 1], 16, 2, 64, 16), ([3000, 16, 40], [200, 16, 40], 8, 2, 128, 16), ([300, 200, 250], [5, 40, 3], 8, 2, 80, 16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", range(len(PAGES)), ids=lambda n: "-".join(map(str, PAGES[n][1:])).replace(" ", ""))
def test_a_page_out_of_range_counts_as_zeros(dev, n, causal):
    """Its keys and values are zeros in every kernel, and its tokens collect nothing."""
    from hexkernels_b200 import HexcudaError
    rng = np.random.default_rng(541 + n)
    c = ref.Cache(rng, *PAGES[n], "f16" if n % 2 else "bf16", fill=np.nan, q_by=0.5)
    page = PAGES[n][-1]
    bad = [(b, i) for b, m in enumerate(c.kv_lens) for i in range(-(-int(m) // page)) if b == 1 or rng.random() < 0.3]
    o = OnDevice(dev, c, causal)
    for b, i in bad:
        o.table[b, i] = int(rng.choice([-1, c.pages, 2 ** 31 - 1, -2 ** 31]))
    o.attn()
    with pytest.raises(HexcudaError, match="out of range"):
        dev.sync(0)
    out, lse = o.results()
    gone = [c.table[b, i] for b, i in bad]
    c.k[gone] = c.v[gone] = 0
    want, z, b_out, b_lse = ref.paged_attn(c, causal)
    near(out, want, b_out, "out")
    near(lse, z, b_lse, "lse")
    base = rng.random(c.k.shape[:3]).astype(np.float32)
    s = up(base)
    o.scores(s)
    with pytest.raises(HexcudaError, match="out of range"):
        dev.sync(0)
    want, bound = ref.cache_scores(c, lse, base, causal)
    got = down(s, base)
    np.testing.assert_array_equal(got[gone], base[gone])
    want[gone] = base[gone]
    near(got, want, bound, "scores")


# ------------------------------------------------- values that are not finite

def attn_odd(c, causal):
    """ref.paged_attn where V is not finite: a column of a row that sees such
    values is their sum (weights are positive), the others never meet them."""
    v = ref.to64(c.v)
    keep = c.v
    c.v = ref.to16(np.where(np.isfinite(v), v, 0.0), c.kind)
    want, z, b_out, b_lse = ref.paged_attn(c, causal)
    c.v = keep
    odd = np.where(np.isfinite(v), 0.0, v)
    group = c.heads // c.kv_heads
    for b in range(len(c.kv_lens)):
        seen = ~c.hidden(b, causal)
        j = np.arange(int(c.kv_lens[b]))
        for h in range(c.kv_heads):
            x = odd[c.table[b, j // c.page], h, j % c.page]
            with np.errstate(all="ignore"):
                for t in range(len(seen)):
                    add = x[seen[t]].sum(0)
                    if (add != 0).any():
                        want[c.q_offs[b] + t, h * group:(h + 1) * group] += add
    return want, z, b_out, b_lse


ODD = [     # kv, q, heads, kv_heads, dim, page: whole items and cut ones, one query tile and two
    ([300, 77], [4, 1], 8, 2, 128, 16), ([5000], [3], 10, 2, 128, 16), ([700, 640, 513], [7, 8, 2], 4, 1, 64, 16), ([900, 40], [60, 40], 4, 2, 64, 32),
    ([2500], [300], 8, 2, 128, 16), ([1500, 128], [400, 128], 2, 2, 64, 64), ([600], [200], 16, 1, 128, 16), ([260, 20], [33, 50], 4, 1, 80, 16),
    ([200] * 40, [90] * 40, 8, 2, 128, 32), ([1300], [1300], 4, 1, 64, 16), ([130], [3], 40, 1, 128, 16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("where", ["channel", "scattered", "new tokens"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", range(len(ODD)), ids=lambda n: "-".join(map(str, ODD[n][2:])) + f"x{len(ODD[n][0])}")
def test_values_that_are_not_finite(dev, n, kind, where, causal):
    rng = np.random.default_rng(551 + n)
    c = ref.Cache(rng, *ODD[n], kind, fill=np.nan, q_by=0.7)
    v = ref.to64(c.v)
    if where == "channel":          # one that overflowed from the start
        v[..., 5] = np.inf
        v[..., c.dim - 1] = np.where(np.arange(v.shape[2]) % 2, np.inf, np.nan)
    elif where == "scattered":
        v = np.where(rng.random(v.shape) < 2e-4, rng.choice([np.nan, np.inf, -np.inf], v.shape), v)
    else:
        for b, (n_kv, n_q) in enumerate(zip(c.kv_lens, np.diff(c.q_offs))):
            for j in range(max(0, n_kv - n_q), n_kv):
                at = (c.table[b, j // c.page], slice(None), j % c.page)
                v[at] = np.where(rng.random(v[at].shape) < 0.02, rng.choice([np.nan, np.inf, -np.inf], v[at].shape), v[at])
    c.v = ref.to16(v, kind)
    o = OnDevice(dev, c, causal)
    o.attn()
    dev.sync(0)
    out, lse = o.results()
    want, z, b_out, b_lse = attn_odd(c, causal)
    near(out, want, b_out, "out")
    near(lse, z, b_lse, "lse")


@pytest.mark.parametrize("dim, kv, q", [(128, 6000, 600), (64, 6000, 600), (128, 12000, 7)])
def test_a_channel_of_infinities_costs_little(dev, dim, kv, q):
    """The time of a call is bounded by its sizes, not by what V holds."""
    import torch
    c = ref.Cache(np.random.default_rng(571), [kv], [q], 16, 4, dim, 16, "bf16")
    o = OnDevice(dev, c)

    def time():
        ts = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            o.attn()
            b.record()
            torch.cuda.synchronize()
            ts.append(a.elapsed_time(b))
        return sorted(ts)[2]

    plain = time()
    o.v.view(torch.bfloat16)[..., 3] = float("inf")
    odd = time()
    dev.sync(0)
    print(f"dim {dim} {q} of {kv}: {plain * 1e3:.0f} us, with an infinite channel {odd * 1e3:.0f} us")
    assert odd < 4 * plain + 0.5


def test_a_workspace_of_the_least_alignment(dev):
    """16 bytes, as documented, and not a byte behind its end."""
    import torch
    need = dev.paged_attn_workspace(0)
    for q in ([1, 1], [3, 2], [130, 70]):
        c = ref.Cache(np.random.default_rng(577), [3000, 900], q, 8, 2, 128, 16, "bf16", fill=np.nan)
        o = OnDevice(dev, c)
        whole = torch.full((need + 48,), 0xA5, dtype=torch.uint8, device="cuda")
        assert whole.data_ptr() % 32 == 0
        o.space = whole[16:16 + need]
        o.attn()
        dev.sync(0)
        out, lse = o.results()
        want, z, b_out, b_lse = ref.paged_attn(c)
        near(out, want, b_out)
        near(lse, z, b_lse)
        assert (whole[:16] == 0xA5).all() and (whole[16 + need:] == 0xA5).all()


AGAIN = [   # kv, q, heads, kv_heads, dim, page: items of one query tile, many of them to a CTA, and pairs
    ([5107, 2554], [43, 22], 32, 16, 128, 32), ([130, 250, 70] * 40, [40, 33, 60] * 40, 8, 4, 128, 16), ([100] * 300, [40] * 300, 4, 4, 128, 32),
    ([390] * 60, [50] * 60, 8, 4, 64, 16), ([1000, 600] * 8, [300, 100] * 8, 8, 2, 128, 16), ([3000, 200] * 8, [5, 3] * 8, 16, 4, 128, 16),
    ([700] * 20, [129, 64] * 10, 4, 4, 128, 16), ([900, 129] * 12, [7, 2] * 12, 16, 4, 64, 16),
]


@pytest.mark.parametrize("n", range(len(AGAIN)), ids=lambda n: "-".join(map(str, AGAIN[n][2:])) + f"x{len(AGAIN[n][0])}")
def test_calls_behind_one_another_repeat_bit_for_bit(dev, n):
    """Calls on two batches in turn, none waited for: the same bits each time,
    and the right ones."""
    cs = [ref.Cache(np.random.default_rng(590 + n + i), *AGAIN[n], "f16", fill=np.nan) for i in range(2)]
    os = [OnDevice(dev, c) for c in cs]
    os[1].space = os[0].space
    os[0].attn()
    dev.sync(0)
    check_attn(os[0], True, "first")
    first = [t.clone() for t in (os[0].out, os[0].lse)]
    for _ in range(40):
        os[0].out.fill_(0)
        for o in (os[0], os[1], os[0], os[0], os[1]):
            o.attn()
        for t, f in zip((os[0].out, os[0].lse), first):
            assert bool((t == f).all())
    dev.sync(0)
    check_attn(os[1], True, "second")


def test_captured_calls_take_what_is_there_when_they_are_replayed(dev):
    """A captured step, replayed with values that are not finite, with a page
    that is not there, and again with good ones."""
    import torch
    from hexkernels_b200 import HexcudaError
    c = ref.Cache(np.random.default_rng(601), [700, 90, 300], [40, 3, 70], 8, 2, 128, 16, "bf16", fill=np.nan)
    o = OnDevice(dev, c)
    s = up(np.zeros(c.k.shape[:3], np.float32))
    side = torch.cuda.Stream()
    good_v, good_table = o.v.clone(), o.table.clone()
    g = None
    try:
        dev.bind_stream(0, side)
        with torch.cuda.stream(side):
            o.attn()
            o.scores(s)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o.attn()
            o.scores(s)

        def replay():
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.synchronize()

        for _ in range(2):
            v = ref.to64(c.v)
            keep = c.v
            v[..., 3] = np.inf
            v[c.table[0, 42], :, 5, 9] = np.nan      # token 677 of 700: among the new ones
            c.v = ref.to16(v, "bf16")
            o.v.copy_(up(c.v))
            replay()
            out, lse = o.results()
            want, z, b_out, b_lse = attn_odd(c, True)
            near(out, want, b_out, "not finite")
            near(lse, z, b_lse)
            c.v = keep
            o.v.copy_(good_v)
            o.table[1, 2] = -1
            replay()
            with pytest.raises(HexcudaError, match="out of range"):
                dev.sync(0)
            o.table.copy_(good_table)
            replay()
            dev.sync(0)
            check_attn(o, True, "good again")
    finally:
        del g
        dev.bind_stream(0)


# ----------------------------------------------------------------- errors

def test_a_call_after_one_that_ran_out_of_memory(hx):
    """A refused allocation is that call's error and not the next one's."""
    from hexkernels_b200 import _lib
    lib = _lib.load()
    assert not lib.hexcuda_alloc(0, 1 << 50)
    c = ref.Cache(np.random.default_rng(581), [100, 40], [4, 3], 4, 2, 64, 16)
    out, lse = hx.paged_attn(c.q, c.k, c.v, c.table, c.kv_lens, c.q_offs)
    want, z, b_out, b_lse = ref.paged_attn(c)
    near(out, want, b_out)
    near(lse, z, b_lse)
