"""Calls of the paged operators at their least: nothing cached, no pages, no
table columns, no requests, and a process whose first call is captured."""
import os
import subprocess
import sys

import pytest
import torch

from test_paged_gpu import BF16, E4M3, build, check, i32, nat, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("new", [[3, 1], [90, 200]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_no_columns_no_pages_no_requests(nat, cache, new, d):  # noqa: F811
    s = build(new, [n + 50 for n in new], 4, 2, d, 16, BF16, cache, seed=d)
    check(nat, s, max_new=max(new))
    zero = torch.zeros_like(s["q"])
    t = dict(s, table=s["table"][:, :0])
    assert torch.equal(run(nat, t, max_new=max(new)), zero)
    t = dict(s, k=s["k"][:0], v=s["v"][:0])
    assert torch.equal(run(nat, t, max_new=max(new)), zero)
    t = dict(s, table=s["table"][:0], cu=i32([0]), kv=i32([]))
    assert torch.equal(run(nat, t, max_new=max(new)), zero)
    t = dict(s, cu=i32([0, 0, 0]))                         # rows, and none of a request
    assert torch.equal(run(nat, t, max_new=max(new)), zero)
    t = dict(s, kv=i32([0, -5]))
    assert torch.equal(run(nat, t, max_new=max(new)), zero)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("page", [512, 4096])
def test_pages_longer_than_a_request(nat, cache, page):  # noqa: F811
    for new, kv in (([1, 4], [700, 30]), ([100, 300], [700, 300])):
        for hk, d in ((1, 64), (2, 128), (1, 256)):
            check(nat, build(new, kv, 4, hk, d, page, BF16, cache, seed=page), max_new=max(new))


def test_one_page_one_head_one_slot(nat):  # noqa: F811
    """Dimensions of one, whose strides mean nothing: expanded or of any size."""
    for d in (64, 128, 256):
        for new in (1, 100):
            s = build([new], [new], 1, 1, d, 1, BF16, BF16, seed=d)
            s["k"], s["v"] = (c[:, :, :, None].expand(-1, -1, -1, 1, -1)[:, :, :, 0] for c in (s["k"], s["v"]))
            check(nat, s, max_new=new)
            one = dict(s, k=s["k"][s["table"][0, :1].long()], v=s["v"][s["table"][0, :1].long()], table=i32([[0]]), kv=i32([1]),
                       cu=i32([0, 1]), q=s["q"][:1])
            check(nat, one)


def test_nothing_to_write(nat):  # noqa: F811
    k, v = (torch.ones(2, 4, 1, 16, device="cuda", dtype=BF16) for _ in range(2))
    tab = torch.ones(0, 8, device="cuda")
    q = nat.rope_write_paged(torch.ones(0, 64, device="cuda", dtype=BF16), tab, tab, i32([]), torch.empty(0, dtype=torch.int64, device="cuda"), k, v, 2)
    assert q.shape == (0, 2, 16) and bool((k == 1).all())
    q = nat.rope_write_paged(torch.ones(3, 64, device="cuda", dtype=BF16), torch.ones(1, 8, device="cuda"), torch.ones(1, 8, device="cuda"),
                             i32([0, 0, 0]), torch.full((3,), -1, dtype=torch.int64, device="cuda"), k[:0], v[:0], 2)
    assert q.shape == (3, 2, 16) and bool((q[:, :, 8:] == 2).all()) and bool((q[:, :, :8] == 0).all())


FIRST_CALL = """
import sys, torch
sys.path[:0] = {path!r}
from test_paged_gpu import BF16, E4M3, build, i32, run
from fp4_fp8_for_torch_mps import fp8_mps_native as nat
s = build({new}, {kv}, 8, 2, 128, 16, BF16, {cache}, seed=3)
torch.cuda.synchronize()
side = torch.cuda.Stream()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=side):
    o = run(nat, s, max_new={most})
g.replay()
torch.cuda.synchronize()
assert torch.equal(o, run(nat, s, max_new={most}))
print("replayed")
"""


@pytest.mark.parametrize("new,kv", [([1, 1], [300, 40]), ([200, 1], [400, 30])])
@pytest.mark.parametrize("cache", ["BF16", "E4M3"])
def test_the_first_call_of_a_process_is_captured(device, new, kv, cache):
    here = os.path.dirname(os.path.abspath(__file__))
    path = [here, os.path.dirname(here), os.path.join(os.path.dirname(here), "mps-fp8-for-torch-and-comfyui-python-package_b200")]
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(path=path, new=new, kv=kv, cache=cache, most=max(new))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "replayed" in r.stdout, r.stderr[-2000:]
