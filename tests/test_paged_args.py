"""The paged-cache entries without a GPU: refusals come before any device
work and leave outputs alone, and the 64-bit implementations that the GPU
tests compare with agree with ones written out by hand."""
import numpy as np
import pytest

import paged_ref as ref

P = 4096     # any non-null address: nothing may be read before a refusal


@pytest.fixture(scope="module")
def lib():
    from hexkernels_b200 import _lib
    return _lib.load()


def norm_rope(lib, host=False, **kw):
    a = dict(dtype=0, q=P, q_stride=512, k=P, k_stride=256, v=P, v_stride=256, q_gain=P, k_gain=P, cos=P,
             sin=P, positions=P, slots=P, q_out=P, k_pages=P, v_pages=P, scores=P, tokens=3, heads=4,
             kv_heads=2, dim=128, rot=128, halves=1, norm=1, table=64, pages=8, page=16, eps=1e-6)
    a |= kw
    return lib.hexcuda_qk_norm_rope(0, *a.values())


def attn(lib, **kw):
    a = dict(dtype=0, q=P, k=P, v=P, table=P, lens=P, offs=P, out=P, lse=P, space=P, space_bytes=1 << 30,
             batch=2, total=4, max_q=3, heads=8, kv_heads=2, dim=128, pages=8, page=16, wide=4, scale=0.1,
             causal=1)
    a |= kw
    return lib.hexcuda_paged_attn(0, *a.values())


def scores(lib, **kw):
    a = dict(dtype=0, q=P, lse=P, k=P, table=P, lens=P, offs=P, scores=P, batch=2, total=4, max_q=3, heads=8,
             kv_heads=2, dim=128, pages=8, page=16, wide=4, scale=0.1, causal=1)
    a |= kw
    return lib.hexcuda_cache_scores(0, *a.values())


def evict(lib, **kw):
    a = dict(k=P, v=P, scores=P, table=P, dst=P, lens=P, new=P, kept=P, batch=2, kv_heads=2, dim=128, pages=8,
             page=16, wide=4, dst_wide=4, budget=32, sink=2, recent=4)
    a |= kw
    return lib.hexcuda_cache_evict(0, *a.values())


SHAPE = [dict(dtype=2), dict(dtype=-1), dict(batch=-1), dict(total=-1), dict(max_q=-1), dict(heads=0), dict(kv_heads=0),
         dict(heads=7), dict(dim=0), dict(dim=257), dict(pages=0), dict(page=0), dict(wide=0),
         dict(pages=1 << 20, page=1 << 12), dict(wide=1 << 20, page=1 << 12), dict(scale=0.0), dict(scale=-1.0),
         dict(scale=float("nan")), dict(scale=float("inf")), dict(table=None), dict(lens=None), dict(offs=None),
         dict(q=None), dict(k=None)]


@pytest.mark.parametrize("bad", SHAPE + [dict(v=None), dict(out=None), dict(space=None)], ids=str)
def test_paged_attn_refuses(lib, bad):
    assert attn(lib, **bad) == 1
    assert b"paged_attn" in lib.hexcuda_last_error_string()


@pytest.mark.parametrize("bad", SHAPE + [dict(lse=None), dict(scores=None)], ids=str)
def test_cache_scores_refuses(lib, bad):
    assert scores(lib, **bad) == 1
    assert b"cache_scores" in lib.hexcuda_last_error_string()


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(kv_heads=0), dict(dim=0), dict(dim=257), dict(pages=0), dict(page=0), dict(wide=0),
    dict(budget=0), dict(sink=-1), dict(recent=-1), dict(sink=20, recent=13), dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1),
    dict(dst_wide=1), dict(dst_wide=0), dict(k=None), dict(v=None), dict(scores=None), dict(table=None),
    dict(lens=None), dict(new=None), dict(kept=None)], ids=str)
def test_cache_evict_refuses(lib, bad):
    assert evict(lib, **bad) == 1
    assert b"cache_evict" in lib.hexcuda_last_error_string()


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(tokens=-1), dict(heads=-1), dict(kv_heads=-1), dict(dim=0), dict(dim=257, q_stride=2000),
    dict(rot=-2), dict(rot=130), dict(rot=7), dict(table=0), dict(eps=-1.0), dict(eps=float("nan")), dict(q=None),
    dict(q_out=None), dict(cos=None), dict(sin=None), dict(positions=None), dict(slots=None), dict(k=None),
    dict(k_pages=None), dict(v=None), dict(v_pages=None), dict(q_stride=511), dict(k_stride=255),
    dict(v_stride=255), dict(pages=0), dict(page=0), dict(pages=1 << 20, page=1 << 12)], ids=str)
def test_qk_norm_rope_refuses(lib, bad):
    assert norm_rope(lib, **bad) == 1
    assert b"qk_norm_rope" in lib.hexcuda_last_error_string()


@pytest.mark.parametrize("call, nothing", [(norm_rope, dict(tokens=0)), (norm_rope, dict(heads=0, kv_heads=0)),
                                           (attn, dict(batch=0)), (attn, dict(total=0)), (scores, dict(batch=0)),
                                           (scores, dict(total=0)), (evict, dict(batch=0))])
def test_nothing_to_do_needs_no_device(lib, call, nothing):
    assert call(lib, **nothing) == 0


def test_numpy_level_refusals():
    from hexkernels_b200 import ops
    c = ref.Cache(np.random.default_rng(0), [5], [2], 2, 1, 16, 4)
    with pytest.raises(TypeError):
        ops.paged_attn(c.q, c.k.view(np.uint16), c.v, c.table, c.kv_lens, c.q_offs)
    with pytest.raises(TypeError):
        ops.paged_attn(c.q.astype(np.float32), c.k, c.v, c.table, c.kv_lens, c.q_offs)
    with pytest.raises(TypeError):
        ops.paged_attn(c.q, c.k, c.v, c.table.astype(np.int64), c.kv_lens, c.q_offs)
    s = np.zeros(c.k.shape[:3], np.float32)
    with pytest.raises(ValueError):
        ops.cache_evict(c.k[:, :, ::2], c.v, s, c.table, c.kv_lens, 3)
    with pytest.raises(ValueError):
        ops.cache_scores(c.q, np.zeros((2, 2), np.float32), c.k, c.table, c.kv_lens, c.q_offs, s[:1])
    # scores are written in place: a strided or read-only array is not copied and lost
    strided = np.zeros((*s.shape[:2], 2 * s.shape[2]), np.float32)[..., ::2]
    fixed = s.copy()
    fixed.flags.writeable = False
    x, tab = np.zeros((2, 1, 16), np.float16), np.ones((8, 8), np.float32)
    for bad, error in ((strided, ValueError), (fixed, ValueError), (s.astype(np.float64), TypeError)):
        with pytest.raises(error):
            ops.cache_scores(c.q, np.zeros((2, 2), np.float32), c.k, c.table, c.kv_lens, c.q_offs, bad)
        with pytest.raises(error):
            ops.cache_evict(c.k, c.v, bad, c.table, c.kv_lens, 3)
        with pytest.raises(error):
            ops.qk_norm_rope(c.q, x, x, c.k, c.v, tab, tab, np.zeros(2, np.int32), np.arange(2, dtype=np.int32),
                             scores=bad)


# ------------------------------------------- the 64-bit implementations themselves

def test_bfloat16_rounding():
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -3.1415927, 0.0, np.inf, 1e-40], np.float32)
    import torch
    want = torch.from_numpy(x).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)
    np.testing.assert_array_equal(ref.to16(x, "bf16"), want)
    np.testing.assert_array_equal(ref.to64(want), torch.from_numpy(x).to(torch.bfloat16).double().numpy())


@pytest.mark.parametrize("causal", [True, False])
def test_reference_attention_by_hand(causal):
    c = ref.Cache(np.random.default_rng(1), [5, 0, 3, 2], [2, 1, 3, 4], 4, 2, 8, 2, fill=np.nan)
    out, lse, b_out, b_lse = ref.paged_attn(c, causal)
    s0 = np.zeros(c.k.shape[:3], np.float32)
    got, _ = ref.cache_scores(c, lse.astype(np.float32), s0, causal)
    want = np.zeros(s0.shape)
    for b in range(4):
        n, m = int(c.kv_lens[b]), int(c.q_offs[b + 1] - c.q_offs[b])
        for t in range(m):
            r = c.q_offs[b] + t
            last = n - m + t if causal else n - 1
            for h in range(4):
                w = {}
                for j in range(n):
                    if j <= last:
                        page = c.table[b, j // 2]
                        dot = float((c.q[r, h].astype(np.float64) * c.k[page, h // 2, j % 2].astype(np.float64)).sum())
                        w[j] = np.exp(dot * c.scale)
                z = sum(w.values())
                if not w:
                    assert (out[r, h] == 0).all() and lse[r, h] == -np.inf
                    continue
                o = sum(w[j] / z * c.v[c.table[b, j // 2], h // 2, j % 2].astype(np.float64) for j in w)
                np.testing.assert_allclose(out[r, h], o, rtol=1e-12, atol=1e-14)
                np.testing.assert_allclose(lse[r, h], np.log(z), rtol=1e-12)
                for j in w:
                    want[c.table[b, j // 2], h // 2, j % 2] += w[j] / z
    np.testing.assert_allclose(got, want, rtol=1e-6)
    # each row gives a weight of one
    rows = sum(1 for r in range(c.total) if lse[r, 0] > -np.inf)
    np.testing.assert_allclose(got.sum(), rows * 4, rtol=1e-6)


def test_reference_eviction_by_hand():
    x = np.array([0.5, 9, 3, 3, np.nan, 3, -np.inf, 0.0, -0.0, 7, 1], np.float32)
    np.testing.assert_array_equal(ref.evict_kept(x, 5, 1, 1), [0, 1, 2, 9, 10])
    np.testing.assert_array_equal(ref.evict_kept(x, 6, 1, 1), [0, 1, 2, 3, 9, 10])
    np.testing.assert_array_equal(ref.evict_kept(x, 8, 1, 1), [0, 1, 2, 3, 5, 7, 9, 10])
    np.testing.assert_array_equal(ref.evict_kept(x, 10, 1, 1), [0, 1, 2, 3, 5, 6, 7, 8, 9, 10])
    np.testing.assert_array_equal(ref.evict_kept(x, 2, 2, 0), [0, 1])
    np.testing.assert_array_equal(ref.evict_kept(x, 2, 0, 2), [9, 10])
    np.testing.assert_array_equal(ref.evict_kept(x, 11, 0, 0), np.arange(11))


def test_reference_rotation_keeps_lengths():
    rng = np.random.default_rng(3)
    x = ref.to16(rng.standard_normal((6, 3, 32)), "f16")
    cos, sin = ref.turns(50, 16)
    pos = np.array([0, 1, 49, 7, 7, 20])
    for halves in (True, False):
        z, _ = ref.qk_norm_rope(x, None, cos, sin, pos, halves, True, 0.0)
        np.testing.assert_allclose((z ** 2).mean(-1), 1.0, rtol=1e-6)
        np.testing.assert_allclose(z[0], ref.to64(x)[0] / np.sqrt((ref.to64(x)[0] ** 2).mean(-1, keepdims=True)), rtol=1e-6)
