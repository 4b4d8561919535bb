"""Refusals of the paged-cache entries that come before any device work: counts
that the kernels' 32-bit steps would pass."""
import pytest

from test_paged_args import attn, evict, lib, scores  # noqa: F401

MOST = 2 ** 31 - 2 ** 16


@pytest.mark.parametrize("call", [attn, scores])
@pytest.mark.parametrize("over", [dict(total=MOST + 1), dict(total=2 ** 31 - 1), dict(page=1, wide=MOST + 1), dict(page=1, wide=2 ** 31 - 1),
                                  dict(page=2 ** 15, wide=2 ** 16 - 1)], ids=str)
def test_more_tokens_than_the_kernels_step_through(lib, call, over):  # noqa: F811
    """A loop from 0 in steps of 32 up to 2^31 - 1 has no end."""
    assert call(lib, **over) == 1
    assert call(lib, **over | {"total": MOST, "wide": 1, "page": 16}) != 1      # (no device: another error)


@pytest.mark.parametrize("over", [dict(budget=MOST + 1), dict(budget=2 ** 31 - 1), dict(page=1, wide=MOST + 1), dict(page=1, dst_wide=2 ** 31 - 1)],
                         ids=str)
def test_a_budget_beyond_the_kernels_steps(lib, over):  # noqa: F811
    assert evict(lib, **({} if "dst_wide" in over else {"dst": None}) | over) == 1
    assert b"cache_evict" in lib.hexcuda_last_error_string()
    assert evict(lib, dst=None, budget=MOST) != 1


@pytest.mark.parametrize("call", [attn, scores])
def test_a_scale_whose_product_with_log2_e_is_infinite(lib, call):  # noqa: F811
    """2^(scale log2(e) x) of a zero score would be not-a-number."""
    assert call(lib, scale=3e38) == 1
    assert b"scale" in lib.hexcuda_last_error_string()
    assert call(lib, scale=2e38) != 1
