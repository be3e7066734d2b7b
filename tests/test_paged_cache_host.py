"""Refusals of the step that keeps account of a cache's pages (the C entry
behind PagedKVCache.step), and of the cache's own call, on the CPU."""
import re

import pytest
import torch

P = 4096  # an aligned address that no check reads
STEP = dict(cached=P, new=P, held=P, requests=2, table=P, table_ld=4, cols=4, free=P, n_free=2, head=None, page=16, tokens=2,
            cu=P, kv=P, pos=P, slots=P, held_out=2 * P, head_out=P, stream=None)


@pytest.mark.parametrize("kw,match", [
    (dict(held=None), "null"), (dict(held_out=None), "null"), (dict(held_out=P), "overlap"), (dict(requests=-1), "negative"),
    (dict(requests=16385), "at most"), (dict(page=0), "page_size"), (dict(tokens=2 ** 31), "2\\^31"), (dict(table_ld=3), "overlap"),
])
def test_step_c_refusals(kw, match):
    from fp4_fp8_for_torch_mps import _lib
    rc = _lib.lib().fp8b200_paged_step(*dict(STEP, **kw).values())
    msg = _lib.lib().fp8b200_last_error().decode()
    assert rc == -1 and re.search(match, msg) and msg.startswith("paged_step"), (rc, msg)


@pytest.mark.parametrize("new,rows,match", [
    (torch.zeros(2, dtype=torch.int64), 2, "new_lens must be"), (torch.zeros(3, dtype=torch.int32), 2, "new_lens and"),
    (torch.zeros(2, dtype=torch.int32), -1, "num_tokens=-1"), (torch.zeros(2, dtype=torch.int32), 2, "CUDA device"),
])
def test_cache_step_refusals(new, rows, match):
    from fp4_fp8_for_torch_mps import paged
    c = paged.PagedKVCache(1, 4, 4, 1, 16, 2, 8, torch.bfloat16, "cpu")
    with pytest.raises(RuntimeError, match=match):
        c.step(new, rows)
    assert c.held.tolist() == [0, 0]
