"""Attention over pages where index arithmetic, page masks and the choice of a
kernel have their edges. Inputs, the float64 reference and its tolerance are
those of test_paged_gpu.py."""
import pytest
import torch

from test_paged_gpu import BF16, E4M3, E5M2, F16, build, check, nat  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, E4M3)])
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 256), (4, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 4, 1)])
@pytest.mark.parametrize("new,kv", [([9, 30, 1], [4, 27, 1]), ([150, 3], [140, 200])])
def test_largest_window_with_rows_before_the_first_key(nat, x, cache, hq, hk, d, window, sinks, new, kv):  # noqa: F811
    """More new tokens than the length says: the first rows lie before position 0, the others see all keys."""
    got = check(nat, build(new, kv, hq, hk, d, 16, x, cache, seed=d + new[0]), window=window, sinks=sinks, max_new=max(new))
    assert bool((got[new[0] - 1] != 0).any())
