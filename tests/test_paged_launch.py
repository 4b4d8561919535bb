"""What the paged-cache entries do when a kernel launch is refused, and which
overlapping arrays they refuse, on the CPU with a CUDA runtime that launches
nothing (fakes/refused_launch.cpp)."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

TESTS = Path(__file__).resolve().parent
CSRC = TESTS.parent / "hexkernels_b200" / "csrc"
P = 4096
Q, K, V, OUT = (n << 32 for n in range(1, 5))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    objects = [f"_build/{n}.o" for n in ("paged_attn", "paged_dec", "paged_pre", "cache_scores", "scores_tc", "cache_evict", "qk_norm_rope")]
    subprocess.run(["make", "-s", "-j4", "-C", str(CSRC), *objects], check=True)
    out = tmp_path_factory.mktemp("fake") / "librefused.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-I{CSRC}", f"-I{TESTS.parent / 'include'}",
                    "-I/usr/local/cuda/include", str(TESTS / "fakes" / "refused_launch.cpp"), *[str(CSRC / o) for o in objects],
                    "-o", str(out)], check=True)
    from hexkernels_b200._lib import SIGNATURES
    lib = C.CDLL(str(out))
    for name in ("paged_attn", "cache_scores", "cache_evict", "qk_norm_rope"):
        getattr(lib, "hexcuda_" + name).argtypes = SIGNATURES["hexcuda_" + name][1]
    return lib


def attn(lib, max_q, dim, q=Q, k=K, v=V, out=OUT):
    return lib.hexcuda_paged_attn(0, 0, q, k, v, P, P, P, out, P, P, 1 << 30, 2, 500, max_q, 8, 2, dim, 8, 16, 4, 0.1, 1)


def scores(lib, max_q, dim):
    return lib.hexcuda_cache_scores(0, 0, Q, P, K, P, P, P, P, 2, 500, max_q, 8, 2, dim, 8, 16, 4, 0.1, 1)


def evict(lib, max_q, dim, k=K, v=V):
    return lib.hexcuda_cache_evict(0, k, v, P, P, None, P, P, P, 2, 2, dim, 8, 16, 4, 0, 32, 2, 4)


def norm_rope(lib, tokens=5, q=Q, q_stride=1536, k=Q + 2048, v=Q + 2560, out=OUT, k_pages=K, v_pages=V):
    """8 query heads and 2 key heads of 128, columns of one array unless said otherwise."""
    return lib.hexcuda_qk_norm_rope(0, 0, q, q_stride, k, 1536, v, 1536, None, None, P, P, P, P, out, k_pages, v_pages, P, tokens, 8, 2, 128,
                                    128, 1, 1, 64, 8, 16, 1e-6)


@pytest.mark.parametrize("call, most, count", [(attn, 1, 2), (attn, 8, 2), (attn, 200, 2), (scores, 1, 1), (scores, 200, 1), (evict, 1, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_nothing_follows_a_refused_launch(lib, call, most, count, dim):
    """Its records would be whatever the workspace holds."""
    lib.refuse(0)
    assert call(lib, most, dim) == 0 and lib.launches() == count
    for nth in range(1, count + 1):
        lib.refuse(nth)
        assert call(lib, most, dim) == 2
        assert lib.launches() == nth


ROWS, PAGES = 500 * 8 * 64 * 2, 8 * 2 * 16 * 64 * 2      # bytes of attn's q and out and of the pages, dim 64


@pytest.mark.parametrize("call, bad", [
    (attn, dict(out=Q)), (attn, dict(out=Q + ROWS - 16)), (attn, dict(out=Q - ROWS + 16)), (attn, dict(out=K + PAGES - 16)),
    (attn, dict(out=V - ROWS + 16)), (evict, dict(v=K)), (evict, dict(v=K + PAGES - 16)), (evict, dict(k=V + 16))], ids=str)
def test_overlapping_arrays_are_refused(lib, call, bad):
    lib.refuse(0)
    assert call(lib, 3, 64, **bad) == 1 and lib.launches() == 0


@pytest.mark.parametrize("fine", [dict(out=Q + ROWS), dict(out=Q - ROWS), dict(k=V, v=V), dict(out=K + PAGES)], ids=str)
def test_neighbours_are_not(lib, fine):
    lib.refuse(0)
    assert attn(lib, 3, 64, **fine) == 0 and lib.launches() == 2


ROW = 2 * (8 + 2 + 2) * 128      # bytes of a token
LAST = 4 * ROW                  # from the first to the fifth


@pytest.mark.parametrize("bad", [
    dict(out=Q), dict(out=Q + LAST + 2032), dict(out=Q + LAST + 2048), dict(out=Q + LAST + 3056), dict(out=Q - 5 * 2048 + 16),
    dict(k_pages=V), dict(v_pages=K + 8 * 2 * 16 * 128 * 2 - 16), dict(tokens=1, out=Q + 16),
    dict(q_stride=1024, k=K + (1 << 30), v=V + (1 << 30), out=Q + 16)], ids=str)
def test_queries_over_what_is_still_read(lib, bad):
    """In place only where a token's row is its own: another one's would be written before it is read."""
    lib.refuse(0)
    assert norm_rope(lib, **bad) == 1 and lib.launches() == 0


@pytest.mark.parametrize("fine", [
    dict(), dict(tokens=1, out=Q), dict(q_stride=1024, k=K + (1 << 30), v=V + (1 << 30), out=Q), dict(out=Q + LAST + ROW),
    dict(out=Q - 5 * 2048)], ids=str)
def test_queries_in_place_or_beside(lib, fine):
    lib.refuse(0)
    assert norm_rope(lib, **fine) == 0 and lib.launches() == 1
