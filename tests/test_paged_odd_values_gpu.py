"""Infinities and NaN in the cache, at keys that a query sees and at keys that
are hidden from it, against float64 (inputs, reference and tolerance of
test_paged_gpu.py): what a query sees is its result, what it does not see has
no effect. Every kernel, segments whole and split."""
import math

import pytest
import torch

from test_paged_gpu import BF16, E4M3, E5M2, F16, build, check, nat, run  # noqa: F401

pytestmark = pytest.mark.gpu
TYPES = [(BF16, BF16), (F16, F16), (BF16, E5M2), (BF16, E4M3), (F16, E4M3)]


@pytest.fixture(autouse=True)
def no_wait_ran_out(device):
    from fp4_fp8_for_torch_mps import _lib
    _lib.paged_status(reset=True)
    yield
    assert _lib.paged_status() == 0


def put(s, which, r, key, head, dim, value):
    page = s[which].shape[1]
    s[which][s["table"][r, key // page].item(), key % page, head, dim] = torch.tensor(value).to(s[which].dtype)


def values(cache):
    return (math.nan,) if cache == E4M3 else (math.nan, math.inf, -math.inf)


# rows a request x group, head size: the kernels for few rows, for more, for chunks, and for wide heads
SHAPES = [([1, 1], [900, 70], 8, 2, 128), ([5, 1], [3000, 70], 8, 1, 64), ([11, 3], [500, 64], 4, 1, 128), ([40, 1], [700, 90], 2, 2, 64),
          ([300, 40], [900, 40], 4, 1, 128), ([130, 2], [4000, 300], 8, 2, 64), ([70, 9], [70, 900], 3, 1, 128), ([2, 1], [600, 50], 4, 1, 256), ([90, 20], [400, 20], 2, 1, 256)]


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("new,kv,hq,hk,d", SHAPES)
def test_seen_and_hidden(nat, x, cache, new, kv, hq, hk, d):  # noqa: F811
    """In V: early, in the middle, among the request's own new tokens and at its last; whole rows of it, both signs."""
    s = build(new, kv, hq, hk, d, 16, x, cache, seed=d + new[0], scales=0)
    v = values(cache)
    n, m = new[0], kv[0]
    put(s, "v", 0, m // 2, 0, 3, v[0])
    check(nat, s, max_new=max(new))
    put(s, "v", 0, m - 1, 0, 5, v[-1])                     # hidden from all but the last query
    put(s, "v", 0, m - 1 - n // 2, hk - 1, 9, v[len(v) // 2])
    check(nat, s, max_new=max(new))
    for dim in range(d):                                   # a whole row: NaN in every dim from here on
        put(s, "v", 0, m - 1 - n // 3, 0, dim, v[dim % len(v)])
    check(nat, s, max_new=max(new))
    put(s, "v", 0, 1, 0, 3, v[-1])
    put(s, "v", 0, 2, 0, 11, v[-1])
    put(s, "v", 0, m // 3, 0, 11, v[len(v) // 2])
    put(s, "v", 1, 0, 0, 2, v[len(v) // 2])
    check(nat, s, max_new=max(new))
    check(nat, s, window=40, sinks=2, max_new=max(new))
    check(nat, s, window=max(n // 2, 7), max_new=max(new))


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("new,kv,hq,hk,d", SHAPES)
def test_hidden_in_k_and_v_of_one_token(nat, x, cache, new, kv, hq, hk, d):  # noqa: F811
    """A token whose K and V are all NaN or infinite: the queries before it keep their results, those after it are NaN."""
    s = build(new, kv, hq, hk, d, 16, x, cache, seed=d + new[0] + 1, scales=0)
    at = kv[0] - 1 - new[0] // 2
    for dim in range(d):
        put(s, "v", 0, at, 0, dim, values(cache)[dim % len(values(cache))])
        put(s, "k", 0, at, 0, dim, math.nan)
    got = check(nat, s, max_new=max(new))
    first = at - (kv[0] - new[0])                          # the first row that sees it
    heads = hq // hk
    assert bool(torch.isfinite(got[:max(first, 0), :heads]).all()) and bool(torch.isnan(got[max(first, 0):new[0], :heads]).all())


@pytest.mark.parametrize("cache", [F16, E5M2])
@pytest.mark.parametrize("new,kv,hq,hk,d", SHAPES)
def test_infinite_scores(nat, cache, new, kv, hq, hk, d):  # noqa: F811
    """K of -inf under positive queries: no weight, unless nothing else is seen; of +inf: NaN."""
    s = build(new, kv, hq, hk, d, 16, F16, cache, seed=d + new[0] + 2, scales=0)
    s["q"] = s["q"].abs() + 0.1
    at = kv[0] // 2
    put(s, "k", 0, at, 0, 4, -50000.0)
    far = check(nat, s, max_new=max(new))
    put(s, "k", 0, at, 0, 4, -math.inf)
    got = check(nat, s, max_new=max(new))
    assert torch.equal(got, far)                           # a score some thousands below the others has no weight either
    put(s, "v", 0, at + 1, 0, 6, math.inf)                 # a seen infinity elsewhere
    put(s, "v", 0, kv[0] - 1, 0, 7, -math.inf)
    check(nat, s, max_new=max(new))
    put(s, "k", 0, at, 0, 4, math.inf)
    got = check(nat, s, max_new=max(new))
    if kv[0] - new[0] > at:
        assert bool(torch.isnan(got[:new[0], 0]).all())


@pytest.mark.parametrize("cache", [BF16, E5M2])
@pytest.mark.parametrize("v_scale", [-0.5, 2.0])
def test_scaled_infinities(nat, cache, v_scale):  # noqa: F811
    """The sign of the output's infinity is that of value times scale; one token, a chunk and split segments."""
    for new, kv, d in (([1, 1], [5000, 9], 128), ([200, 1], [900, 70], 64), ([20, 3], [90, 700], 256)):
        s = build(new, kv, 4, 1, d, 32, BF16, cache, seed=d, scales=1 if cache == E5M2 else 0)
        if cache == E5M2:
            s["vs"].fill_(v_scale)
        put(s, "v", 0, 3, 0, 1, math.inf)
        put(s, "v", 0, kv[0] // 2, 0, 2, -math.inf)
        got = check(nat, s, max_new=max(new))
        sign = v_scale if cache == E5M2 else 1.0
        assert bool((got[new[0] - 1, :, 1] == math.copysign(math.inf, sign)).all()) and bool((got[new[0] - 1, :, 2] == math.copysign(math.inf, -sign)).all())


def test_largest_values(nat):  # noqa: F811
    """bf16 values near the type's largest: sums of weights times values beyond float32 are recomputed, not infinite."""
    for new, kv, d in (([1, 1], [300, 9], 128), ([100, 1], [200, 70], 64), ([20, 3], [90, 70], 256)):
        s = build(new, kv, 4, 1, d, 32, BF16, BF16, seed=d)
        s["v"].mul_(2.0 ** 119)
        got = check(nat, s, max_new=max(new))
        assert bool(torch.isfinite(got).all())


def test_repeats_and_other_rows_keep_their_bits(nat):  # noqa: F811
    """Rows that meet no odd value are the same bits with and without one elsewhere; equal calls give equal bits."""
    for new, kv, d in (([3, 1], [900, 70], 128), ([300, 7], [600, 200], 128), ([300, 7], [600, 200], 64), ([50, 7], [600, 200], 256)):
        s = build(new, kv, 4, 2, d, 16, BF16, BF16, seed=d + 3)
        clean = run(nat, s, max_new=max(new))
        put(s, "v", 0, kv[0] - 1, 0, 5, math.nan)
        got = run(nat, s, max_new=max(new))
        assert torch.equal(got[:, 2:], clean[:, 2:]) and torch.equal(got[new[0]:], clean[new[0]:])
        again = run(nat, s, max_new=max(new))
        assert torch.equal(got.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (BF16, E4M3)])
@pytest.mark.parametrize("new,kv,hq,hk,d", [([600], [16000], 8, 2, 128), ([1] * 16, [16000] * 16, 8, 2, 128), ([300], [9000], 8, 1, 256), ([40], [20000], 8, 2, 64)])
def test_a_seen_value_costs_a_pass_over_v(nat, x, cache, new, kv, hq, hk, d):  # noqa: F811
    """A NaN that every row sees costs about one more reading of V (2 to 6 times the call where this was written), not a
    recomputation of every row; bounded far above that."""
    s = build(new, kv, hq, hk, d, 64, x, cache, seed=d)

    def took():
        run(nat, s, max_new=new[0])
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(5):
            run(nat, s, max_new=new[0])
        b.record()
        b.synchronize()
        return a.elapsed_time(b)
    clean = took()
    put(s, "v", 0, 100, 0, 5, math.nan)
    assert took() < 50 * clean
