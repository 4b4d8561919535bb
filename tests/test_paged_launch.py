"""What the paged-cache entries do when a kernel launch is refused, on the CPU
with a CUDA runtime that refuses it (fakes/refused_launch.cpp)."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

TESTS = Path(__file__).resolve().parent
CSRC = TESTS.parent / "hexkernels_b200" / "csrc"
P = 4096


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    objects = [f"_build/{n}.o" for n in ("paged_attn", "paged_dec", "paged_pre", "cache_scores", "scores_tc", "cache_evict")]
    subprocess.run(["make", "-s", "-j4", "-C", str(CSRC), *objects], check=True)
    out = tmp_path_factory.mktemp("fake") / "librefused.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-I{CSRC}", f"-I{TESTS.parent / 'include'}",
                    "-I/usr/local/cuda/include", str(TESTS / "fakes" / "refused_launch.cpp"), *[str(CSRC / o) for o in objects],
                    "-o", str(out)], check=True)
    from hexkernels_b200._lib import SIGNATURES
    lib = C.CDLL(str(out))
    for name in ("paged_attn", "cache_scores", "cache_evict"):
        getattr(lib, "hexcuda_" + name).argtypes = SIGNATURES["hexcuda_" + name][1]
    return lib


def attn(lib, max_q, dim):
    return lib.hexcuda_paged_attn(0, 0, P, 2 * P, 3 * P, P, P, P, 4 * P, P, P, 1 << 30, 2, 500, max_q, 8, 2, dim, 8, 16, 4, 0.1, 1)


def scores(lib, max_q, dim):
    return lib.hexcuda_cache_scores(0, 0, P, P, 2 * P, P, P, P, P, 2, 500, max_q, 8, 2, dim, 8, 16, 4, 0.1, 1)


def evict(lib, max_q, dim):
    return lib.hexcuda_cache_evict(0, P, P, P, P, None, P, P, P, 2, 2, dim, 8, 16, 4, 0, 32, 2, 4)


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
