"""A thread's first call on the GPU: the kernels that build a tensor map on the
host need the device's context current in the calling thread, which no call
before has seen to there."""
import threading

import pytest
import torch

from test_paged_gpu import BF16, E4M3, build, nat, run  # noqa: F401

pytestmark = pytest.mark.gpu


def in_new_thread(fn):
    out = []

    def target():
        try:
            out.append(fn())
        except BaseException as e:  # noqa: BLE001
            out.append(e)
    t = threading.Thread(target=target)
    t.start()
    t.join()
    if isinstance(out[0], BaseException):
        raise out[0]
    return out[0]


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_paged_attention(nat, cache):  # noqa: F811
    s = build([100, 3], [150, 70], 4, 1, 128, 16, BF16, cache, seed=1)
    want = run(nat, s, max_new=100)
    assert torch.equal(in_new_thread(lambda: run(nat, s, max_new=100)), want)


@pytest.mark.parametrize("m", [16, 128, 512])
def test_products(nat, m):  # noqa: F811
    g = torch.Generator().manual_seed(m)
    a = torch.randn(m, 512, generator=g).to(E4M3).cuda()
    b = torch.randn(256, 512, generator=g).to(E4M3).cuda()
    x = torch.randn(m, 512, generator=g).to(BF16).cuda()
    one, rows = torch.ones(1, device="cuda"), torch.ones(256, 1, device="cuda")
    a4, b4 = (torch.randint(0, 256, (n, 256), dtype=torch.uint8, generator=g).cuda() for n in (m, 256))
    for fn in (lambda: nat.scaled_mm(a, b, one, one, out_dtype=BF16), lambda: nat.fp8_linear(x, b, rows),
               lambda: nat.fp4_scaled_mm(a4, b4, one, one, out_dtype=BF16)):
        want = fn()
        assert torch.equal(in_new_thread(fn), want)
