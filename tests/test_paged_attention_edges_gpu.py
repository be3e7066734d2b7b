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


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E5M2)])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("page", [1, 2, 6, 7, 16, 200])
def test_page_masks_of_many_rows(nat, x, cache, hq, hk, d, page):  # noqa: F811
    """Table entries outside the pool at every third page, and in runs: with pages of odd or twice odd slots a key
    tile's mask has more than one word. More than 64 rows a request, tiles before, on and behind the diagonal."""
    new, kv = [90, 300, 2], [700, 300, 40]
    s = build(new, kv, hq, hk, d, page, x, cache, seed=page)
    t = s["table"]
    bad = torch.tensor([-1, s["k"].shape[0], 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    cols = torch.arange(t.shape[1], device="cuda")
    hit = (cols % 3 == 1) | ((cols >= 40) & (cols < 75)) | (cols % 97 > 90)
    t[:2, hit] = bad[cols[hit] % 4]
    check(nat, s, max_new=300)
    check(nat, s, window=100, sinks=9, max_new=300)
    t[1] = -1
    got = check(nat, s, max_new=300)
    assert int((got[90:390] != 0).sum()) == 0


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (BF16, E5M2), (F16, E5M2)])
@pytest.mark.parametrize("hq,hk,d,new", [(8, 1, 64, 5), (8, 1, 64, 6), (8, 1, 64, 7), (8, 1, 64, 8), (14, 2, 48, 5), (14, 2, 48, 9),
                                         (5, 5, 16, 37), (5, 5, 32, 64), (32, 8, 128, 9), (28, 4, 128, 7), (32, 8, 128, 16), (8, 1, 112, 8)])
def test_33_to_64_rows_a_request(nat, x, cache, hq, hk, d, new):  # noqa: F811
    """The widest few-row variants (head sizes up to 64), and the general kernel at the same rows (sizes up to 128)."""
    s = build([new, 1, new, 2], [new + 1500, 65, new, 300], hq, hk, d, 16, x, cache, seed=new + d)
    check(nat, s, max_new=new)
    check(nat, s, window=70, sinks=3, max_new=new)


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, E4M3), (BF16, E5M2)])
@pytest.mark.parametrize("hq,hk,d", [(16, 1, 128), (12, 1, 64), (9, 1, 128), (22, 2, 64), (8, 2, 128), (5, 5, 64)])
def test_short_requests_beside_chunks(nat, x, cache, hq, hk, d):  # noqa: F811
    """Decodes and requests of about 16 rows (either kernel's side of the limit) in one call with chunks."""
    g = hq // hk
    new = [100, 1, 1, 16 // g or 1, 16 // g + 1, 1, 0, 130, 2]
    kv = [160, 1, 700, 300, 90, 2000, 50, 130, 64]
    s = build(new, kv, hq, hk, d, 24, x, cache, seed=hq + d, pad=3)
    check(nat, s, max_new=130)
    check(nat, s, window=90, sinks=5)
