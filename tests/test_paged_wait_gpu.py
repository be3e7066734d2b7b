"""A wait of the tensor-memory attention kernel that nothing satisfies: the
producers are told to bring no tile in, the limit is 50 ms."""
import threading

import pytest
import torch

from test_paged_gpu import BF16, E4M3, F16, build, check, nat, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (BF16, E4M3), (F16, F16)])
@pytest.mark.parametrize("d", [64, 128])
def test_wait_runs_out_and_the_context_survives(nat, x, cache, d):  # noqa: F811
    from fp4_fp8_for_torch_mps import _lib
    s = build([100, 300], [150, 700], 4, 1, d, 16, x, cache, seed=d)
    nat.paged_status(reset=True)
    try:
        _lib.lib().fp8b200_debug_paged(1, 50_000_000)
        run(nat, s, max_new=300)
        status = nat.paged_status(reset=True)
    finally:
        _lib.lib().fp8b200_debug_paged(0, 0)
    assert status & 0x80000000, hex(status)
    check(nat, s, max_new=300)
    assert nat.paged_status() == 0


def test_the_hook_is_per_thread_and_a_short_limit_harms_nothing(nat):  # noqa: F811
    """Calls of another thread do not see the hook; a call whose tiles do arrive keeps a limit of 20 ms, odd rows included."""
    from fp4_fp8_for_torch_mps import _lib
    s = build([100, 300], [150, 9000], 4, 1, 128, 16, BF16, BF16, seed=1)
    nat.paged_status(reset=True)
    try:
        _lib.lib().fp8b200_debug_paged(1, 50_000_000)
        failed = []

        def other():
            try:
                check(nat, s, max_new=300)
            except BaseException as e:  # noqa: BLE001
                failed.append(e)
        t = threading.Thread(target=other)
        t.start()
        t.join()
        assert not failed
        _lib.lib().fp8b200_debug_paged(0, 20_000_000)
        s["v"][s["table"][1, 8999 // 16].item(), 8999 % 16, 0, 5] = float("nan")  # hidden from all rows but the last
        check(nat, s, max_new=300)
    finally:
        _lib.lib().fp8b200_debug_paged(0, 0)
    assert nat.paged_status() == 0
