"""Serving from a paged key/value cache: host launchers.

One step of a batch of requests, each with tokens already cached and new
tokens to add (one when it decodes, many when it is prefilled):

    step = paged_slots(cached_lens, new_lens, block_table, free_pages, page_size, num_tokens)
    q = rope_write_paged(qkv, cos, sin, step.positions, step.slots, k_cache, v_cache, n_q_heads)
    a = paged_attention(q, k_cache, v_cache, block_table, step.cu_new, step.kv_lens)

`paged_slots` runs once a step, the other two once a layer. Everything that
depends on the lengths stays on the device, so a step can be captured in a
CUDA graph and replayed with other lengths. A cache is a (pages, page_size,
kv_heads, head_dim) tensor of the activations' type or of a float8 type; k and
v caches have the same strides (two tensors, or two views of one).

No counterpart in the reference, which has no cache and no attention.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L

_FP8 = (torch.float8_e4m3fn, torch.float8_e5m2)
_16BIT = (torch.bfloat16, torch.float16)
MAX_REQUESTS = 16384
_INT_MAX = 2 ** 31 - 1


class PagedStep(NamedTuple):
    """What `paged_slots` lays out for one step."""
    cu_new: torch.Tensor      # (requests + 1,) int32: first row of each request's new tokens
    kv_lens: torch.Tensor     # (requests,) int32: cached + new tokens
    positions: torch.Tensor   # (num_tokens,) int32
    slots: torch.Tensor       # (num_tokens,) int64: page * page_size + offset, -1 for none
    free_head: torch.Tensor   # (1,) int32: first free page not taken


_workspace_bytes: dict[tuple[int, int, int], int] = {}


# A call's arguments are looked over in one expression (every attribute of a
# tensor costs 0.1 us and a call of a helper more: a small step is bound by
# them); only what does not pass goes through the checks that say why.
def _check(t: torch.Tensor, name: str, what: str, dtype: torch.dtype, dim: int, dev: torch.device) -> None:
    if t.dtype != dtype or t.dim() != dim:
        raise RuntimeError(f"{what}: {name} must be a {dim}-D {dtype} tensor, got {t.dim()}-D {t.dtype}")
    if t.device != dev:
        raise RuntimeError(f"{what}: {name} is on {t.device}, expected {dev}")
    if dim == 1 and not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be contiguous")


def _check_table(table: torch.Tensor, what: str, dev: torch.device) -> int:
    """The row stride of a (requests, columns) block table."""
    _check(table, "block_table", what, torch.int32, 2, dev)
    n, cols = table.shape
    ld = table.stride(0) if n > 1 else cols
    if (n and cols > 1 and table.stride(1) != 1) or ld < cols:
        raise RuntimeError(f"{what}: block_table rows must be contiguous and not overlap, got strides {table.stride()}")
    return ld


def _check_caches(k: torch.Tensor, v: torch.Tensor, x: torch.Tensor, what: str) -> tuple[int, ...]:
    """(pages, page_size, kv_heads, head_dim) of two caches that go with x."""
    if k.dim() != 4 or v.shape != k.shape:
        raise RuntimeError(f"{what}: k_cache and v_cache must be (pages, page_size, kv_heads, head_dim) tensors of one "
                           f"shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if x.dtype not in _16BIT:
        raise RuntimeError(f"{what}: activations must be bfloat16 or float16, got {x.dtype}")
    if v.dtype != k.dtype or (k.dtype != x.dtype and k.dtype not in _FP8):
        raise RuntimeError(f"{what}: the caches must both be {x.dtype} or both one float8 type, got {k.dtype} and {v.dtype}")
    if k.device != x.device or v.device != x.device:
        raise RuntimeError(f"{what}: the caches are on {k.device} and {v.device}, expected {x.device}")
    if v.stride() != k.stride() or (k.numel() and k.stride(3) != 1):
        raise RuntimeError(f"{what}: the caches must have the same strides and contiguous heads, got {k.stride()} and {v.stride()}")
    return tuple(k.shape)


def _check_scale(s: torch.Tensor | None, name: str, what: str, cache: torch.Tensor) -> tuple[int | None, int]:
    """(pointer, step) of a cache scale: one value or one per key/value head."""
    if s is None:
        return None, 0
    if cache.dtype not in _FP8:
        raise RuntimeError(f"{what}: {name} goes with a float8 cache only")
    if s.dtype != torch.float32 or s.device != cache.device or s.numel() not in (1, cache.shape[2]) or not s.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be 1 or {cache.shape[2]} contiguous float32 values on {cache.device}")
    return s.data_ptr(), 0 if s.numel() == 1 else 1


def _launch(dev: torch.device, fn, what: str, *args) -> None:
    """fn(*args, current stream) on `dev`. The stream's handle comes without a
    torch.cuda.Stream object, which takes 2 us."""
    index = dev.index
    if dev.type != "cuda":
        raise RuntimeError(f"{what}: tensors must be on a CUDA device, got {dev}")
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            L.check(rc, what)
    else:
        with torch.cuda.device(dev):
            L.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)), what)


def slots_outputs(requests: int, num_tokens: int, dev: torch.device) -> PagedStep:
    """The tensors of a step, the int32 ones in one allocation."""
    cu, kv, pos, head = torch.empty(2 * requests + 2 + num_tokens, dtype=torch.int32, device=dev).split_with_sizes(
        [requests + 1, requests, num_tokens, 1])
    return PagedStep(cu, kv, pos, torch.empty(num_tokens, dtype=torch.int64, device=dev), head)


def _check_slots(cached_lens, new_lens, block_table, free_pages, page_size, num_tokens, free_head) -> None:
    what = "paged_slots"
    dev = cached_lens.device
    _check(cached_lens, "cached_lens", what, torch.int32, 1, dev)
    _check(new_lens, "new_lens", what, torch.int32, 1, dev)
    _check(free_pages, "free_pages", what, torch.int32, 1, dev)
    _check_table(block_table, what, dev)
    n = cached_lens.numel()
    if new_lens.numel() != n or block_table.shape[0] != n:
        raise RuntimeError(f"{what}: {n} cached_lens, {new_lens.numel()} new_lens and {block_table.shape[0]} block_table rows")
    if n > MAX_REQUESTS:
        raise RuntimeError(f"{what}: {n} requests, at most {MAX_REQUESTS}")
    if page_size < 1 or num_tokens < 0:
        raise RuntimeError(f"{what}: page_size={page_size} must be positive and num_tokens={num_tokens} not negative")
    if free_head is not None and (free_head.dtype != torch.int32 or free_head.numel() != 1 or free_head.device != dev):
        raise RuntimeError(f"{what}: free_head must be one int32 value on {dev}")


def _slots_table_ld(cached_lens, new_lens, block_table, free_pages, page_size, num_tokens, free_head) -> int:
    """The row stride of the block table, once the arguments have passed."""
    dev, n = cached_lens.device, cached_lens.numel()
    rows, cols = block_table.shape if block_table.dim() == 2 else (-1, 0)
    ld = block_table.stride(0) if n > 1 and rows == n else cols
    if not (cached_lens.dtype is new_lens.dtype is block_table.dtype is free_pages.dtype is torch.int32
            and cached_lens.dim() == new_lens.dim() == free_pages.dim() == 1 and new_lens.numel() == n == rows
            and cached_lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous()
            and (cols <= 1 or block_table.stride(1) == 1) and ld >= cols and n <= MAX_REQUESTS
            and new_lens.device == block_table.device == free_pages.device == dev and page_size >= 1 and num_tokens >= 0
            and (free_head is None
                 or (free_head.dtype is torch.int32 and free_head.numel() == 1 and free_head.device == dev))):
        _check_slots(cached_lens, new_lens, block_table, free_pages, page_size, num_tokens, free_head)
    return ld


def paged_slots(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                page_size: int, num_tokens: int, free_head: torch.Tensor | None = None,
                outputs=slots_outputs) -> PagedStep:
    """Page allotment and token placement of one step, one launch, no host sync.

    cached_lens, new_lens: (requests,) int32, tokens each request holds and
    adds (0: it pauses). block_table: (requests, columns) int32, row r listing
    r's pages in order; the new pages' entries are written in place.
    free_pages: int32 ids of free pages, taken in order of the requests from
    `free_head` (int32, one value on the device; None: 0) on. num_tokens: rows
    of the step, at least the sum of new_lens (more in a padded batch: those
    rows get position 0 and slot -1; fewer: the tokens behind them are not
    placed, nor the pages that they open). outputs(requests, num_tokens,
    device) allocates the results.

    Returns a PagedStep. Once the list of free pages is used up, the requests
    after it get table entries of -1 and slots of -1 (`rope_write_paged` skips
    them); the returned free_head is then beyond free_pages.numel(). A token
    beyond the table's columns also gets slot -1. free_head counts every page
    that the lengths ask for: those for columns that the table lacks and those
    that only tokens without a row open are passed over, and no row holds them
    (PagedKVCache.step takes neither). Lengths below zero count as zero; sums of
    lengths stay below 2^31."""
    dev, n = cached_lens.device, cached_lens.numel()
    ld = _slots_table_ld(cached_lens, new_lens, block_table, free_pages, page_size, num_tokens, free_head)
    step = outputs(n, num_tokens, dev)
    _launch(dev, L.lib().fp8b200_paged_slots, "paged_slots", cached_lens.data_ptr(), new_lens.data_ptr(), n,
            block_table.data_ptr(), ld, block_table.shape[1], free_pages.data_ptr(), free_pages.numel(),
            None if free_head is None else free_head.data_ptr(), page_size, num_tokens, step.cu_new.data_ptr(),
            step.kv_lens.data_ptr(), step.positions.data_ptr(), step.slots.data_ptr(), step.free_head.data_ptr())
    return step


def _step_slots(cache: PagedKVCache, new_lens: torch.Tensor, num_tokens: int) -> tuple[PagedStep, torch.Tensor]:
    """(step, held) of a cache's step: paged_slots with its account of the pages."""
    lens, table, free = cache.lens, cache.block_table, cache.free_pages
    ld = _slots_table_ld(lens, new_lens, table, free, cache.page_size, num_tokens, cache.free_head)
    n, dev = lens.numel(), lens.device
    step, held = slots_outputs(n, num_tokens, dev), torch.empty_like(cache.held)
    _launch(dev, L.lib().fp8b200_paged_step, "paged_slots", lens.data_ptr(), new_lens.data_ptr(), cache.held.data_ptr(), n,
            table.data_ptr(), ld, table.shape[1], free.data_ptr(), free.numel(), cache.free_head.data_ptr(),
            cache.page_size, num_tokens, step.cu_new.data_ptr(), step.kv_lens.data_ptr(), step.positions.data_ptr(),
            step.slots.data_ptr(), held.data_ptr(), step.free_head.data_ptr())
    return step, held


def _check_write(qkv, cos, sin, positions, slots, k_cache, v_cache, n_q_heads) -> None:
    what = "rope_write_paged"
    dev = qkv.device
    _, _, hk, d = _check_caches(k_cache, v_cache, qkv, what)
    width = (n_q_heads + 2 * hk) * d
    if qkv.dim() != 2 or n_q_heads < 0 or qkv.shape[1] < width:
        raise RuntimeError(f"{what}: qkv must be (tokens, at least {width}), got {tuple(qkv.shape)}")
    t = qkv.shape[0]
    ld = qkv.stride(0) if t > 1 else width
    if (t and qkv.stride(1) != 1) or ld < width:
        raise RuntimeError(f"{what}: qkv rows must be contiguous and not overlap, got strides {qkv.stride()}")
    _check(cos, "cos", what, torch.float32, 2, dev)
    _check(sin, "sin", what, torch.float32, 2, dev)
    if cos.shape != sin.shape or cos.shape[1] * 2 != d or not cos.is_contiguous() or not sin.is_contiguous():
        raise RuntimeError(f"{what}: cos and sin must be contiguous (positions, {d // 2}) tables, got {tuple(cos.shape)} and "
                           f"{tuple(sin.shape)}")
    _check(positions, "positions", what, torch.int32, 1, dev)
    _check(slots, "slots", what, torch.int64, 1, dev)
    if positions.numel() != t or slots.numel() != t:
        raise RuntimeError(f"{what}: {t} rows, {positions.numel()} positions and {slots.numel()} slots")


def rope_write_paged(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                     slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, n_q_heads: int,
                     k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary embedding of a step's q and k, and its k and v into the paged
    cache, in one pass over the fused projection.

    qkv: (tokens, ld) bfloat16 or float16, row t holding n_q_heads q heads and
    then the k and the v heads (a column slice of a wider tensor is fine).
    cos, sin: (positions, head_dim / 2) float32 tables, read at positions[t]
    (int32; outside the tables: NaN). The head's halves (a, b) become
    (a cos - b sin, b cos + a sin), computed in float32 and rounded once.
    slots: (tokens,) int64 from paged_slots; a token whose slot is outside the
    pool is not kept. Slots must differ: of two tokens with one slot either
    may stay, value by value.
    k_cache, v_cache: written in place, in qkv's type or as float8 codes of
    value / scale (k_scale, v_scale: one float32 value or one per head; None:
    1), saturated at the format's largest finite value; NaN stays NaN.
    Returns q, (tokens, n_q_heads, head_dim)."""
    dev, dt, cdt = qkv.device, qkv.dtype, k_cache.dtype
    shape, strides, t = k_cache.shape, k_cache.stride(), positions.numel()
    pages, page, hk, d = shape if len(shape) == 4 else (0, 0, 0, 0)
    width = (n_q_heads + 2 * hk) * d
    ld = qkv.stride(0) if t > 1 and qkv.dim() == 2 else width
    if not (dt in _16BIT and (cdt is dt or cdt in _FP8) and v_cache.dtype is cdt and v_cache.shape == shape and len(shape) == 4
            and v_cache.stride() == strides and strides[3] == 1 and qkv.dim() == 2 and qkv.shape[0] == t and qkv.shape[1] >= width
            and ld >= width and n_q_heads >= 0 and (t == 0 or qkv.stride(1) == 1)
            and cos.dtype is sin.dtype is torch.float32 and cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] * 2 == d
            and cos.is_contiguous() and sin.is_contiguous() and positions.dtype is torch.int32 and positions.dim() == 1
            and positions.is_contiguous() and slots.dtype is torch.int64 and slots.shape == (t,) and slots.is_contiguous()
            and k_cache.device == v_cache.device == cos.device == sin.device == positions.device == slots.device == dev):
        _check_write(qkv, cos, sin, positions, slots, k_cache, v_cache, n_q_heads)
    ks, ks_step = (None, 0) if k_scale is None else _check_scale(k_scale, "k_scale", "rope_write_paged", k_cache)
    vs, vs_step = (None, 0) if v_scale is None else _check_scale(v_scale, "v_scale", "rope_write_paged", v_cache)
    q = qkv.new_empty((t, n_q_heads, d))
    sp, ss, sh, _ = strides
    _launch(dev, L.lib().fp8b200_rope_write_paged, "rope_write_paged", qkv.data_ptr(), L.dtype_code(dt), t, ld, n_q_heads, hk, d,
            cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), slots.data_ptr(), q.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), L.dtype_code(cdt), pages, page, sp, ss, sh, ks, ks_step, vs, vs_step)
    return q


def _check_attention(q, k_cache, v_cache, block_table, cu_new, kv_lens, window, sinks, max_new) -> None:
    what = "paged_attention"
    dev = q.device
    _, _, hk, d = _check_caches(k_cache, v_cache, q, what)
    if q.dim() != 3 or q.shape[2] != d or (q.numel() and q.stride(2) != 1):
        raise RuntimeError(f"{what}: q must be (tokens, q_heads, {d}) with contiguous heads, got {tuple(q.shape)}")
    hq = q.shape[1]
    if hq < 1 or hk < 1 or hq % hk:
        raise RuntimeError(f"{what}: {hq} query heads over {hk} key/value heads")
    _check_table(block_table, what, dev)
    _check(cu_new, "cu_new", what, torch.int32, 1, dev)
    _check(kv_lens, "kv_lens", what, torch.int32, 1, dev)
    n = block_table.shape[0]
    if cu_new.numel() != n + 1 or kv_lens.numel() != n:
        raise RuntimeError(f"{what}: {n} block_table rows need {n + 1} cu_new and {n} kv_lens, got {cu_new.numel()} and "
                           f"{kv_lens.numel()}")
    if not (0 <= window <= _INT_MAX and 0 <= sinks <= _INT_MAX):
        raise RuntimeError(f"{what}: window={window} and sinks={sinks} must not be negative or 2^31 and more")
    if max_new is not None and max_new < 1:
        raise RuntimeError(f"{what}: max_new={max_new} must be positive")


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    cu_new: torch.Tensor, kv_lens: torch.Tensor, *, scale: float | None = None, window: int = 0,
                    sinks: int = 0, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    max_new: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each request's new tokens over its pages.

    q: (tokens, q_heads, head_dim) bfloat16 or float16; rows cu_new[r] to
    cu_new[r + 1] are request r's, the last at position kv_lens[r] - 1 (cu_new,
    kv_lens: int32, from paged_slots; the step's k and v already in the
    caches). A query at position p sees key j where j <= p and, with window >
    0, p - j < window or j < sinks: a sliding window whose first tokens stay
    visible. Query head h reads key/value head h // (q_heads // kv_heads).
    scale: of the scores, default head_dim ** -0.5. k_scale, v_scale: as in
    rope_write_paged. head_dim: a multiple of 16 up to 256.

    max_new: the largest number of new tokens of one request, where the host
    knows it (it picks the kernels; a wrong value costs time, not results).
    Without it, more than 64 rows (tokens x group) in all launch the kernels for
    chunks too, with their workspace: give 1 for a step that only decodes.
    Scores, maxima, sums and outputs are float32, rounded once to q's type;
    see the kernels for the weights' type. A query that sees no key gives 0; a
    table entry outside the pool hides its keys; hidden keys' values, NaN
    included, have no effect. Rows that belong to no request are left as they
    were in a given `out` (of q's shape and type, any 16-byte aligned rows, no
    overlap with q) and 0 in a new one."""
    what = "paged_attention"
    dev, dt, cdt = q.device, q.dtype, k_cache.dtype
    shape, strides, qshape = k_cache.shape, k_cache.stride(), q.shape
    pages, page, hk, d = shape if len(shape) == 4 else (0, 0, 0, 0)
    t, hq, qd = qshape if len(qshape) == 3 else (0, 0, 0)
    n, cols = block_table.shape if block_table.dim() == 2 else (0, 0)
    ld = block_table.stride(0) if n > 1 else cols
    if not (dt in _16BIT and (cdt is dt or cdt in _FP8) and v_cache.dtype is cdt and v_cache.shape == shape and len(shape) == 4
            and v_cache.stride() == strides and strides[3] == 1 and len(qshape) == 3 and qd == d and q.stride(2) == 1
            and hk >= 1 and hq >= 1 and hq % hk == 0 and block_table.dtype is cu_new.dtype is kv_lens.dtype is torch.int32
            and block_table.dim() == 2 and (cols <= 1 or block_table.stride(1) == 1) and ld >= cols
            and cu_new.shape == (n + 1,) and kv_lens.shape == (n,) and cu_new.is_contiguous() and kv_lens.is_contiguous()
            and 0 <= window <= _INT_MAX and 0 <= sinks <= _INT_MAX and (max_new is None or max_new >= 1)
            and k_cache.device == v_cache.device == block_table.device == cu_new.device == kv_lens.device == dev):
        _check_attention(q, k_cache, v_cache, block_table, cu_new, kv_lens, window, sinks, max_new)
    ks, ks_step = (None, 0) if k_scale is None else _check_scale(k_scale, "k_scale", what, k_cache)
    vs, vs_step = (None, 0) if v_scale is None else _check_scale(v_scale, "v_scale", what, v_cache)
    new_out = out is None
    if new_out:
        out = q.new_empty(qshape)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or (out.numel() and out.stride(2) != 1):
        raise RuntimeError(f"{what}: `out` must be a {q.dtype} tensor of q's shape on {dev} with contiguous heads")
    elif out.data_ptr() == q.data_ptr() and t:
        raise RuntimeError(f"{what}: `out` must not overlap q")
    max_rows = min(t if max_new is None else max_new, t) * (hq // hk)
    size = _workspace_bytes.get((dev.index, d, max_rows), 0)
    if size == 0 and dev.type == "cuda":
        with torch.cuda.device(dev):
            size = L.lib().fp8b200_paged_attention_workspace(d, max_rows)
        if size < 0:
            L.check(size, what)
        _workspace_bytes[dev.index, d, max_rows] = size
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    sp, ss, sh, _ = strides
    q_tok, q_head, _ = q.stride()
    o_tok, o_head, _ = out.stride()
    _launch(dev, L.lib().fp8b200_paged_attention, what, q.data_ptr(), L.dtype_code(q.dtype), q_tok, q_head, t, hq, hk, d,
            k_cache.data_ptr(), v_cache.data_ptr(), L.dtype_code(k_cache.dtype), pages, page, sp, ss, sh,
            block_table.data_ptr(), ld, cols, cu_new.data_ptr(), kv_lens.data_ptr(), n, d ** -0.5 if scale is None else scale,
            ks, ks_step, vs, vs_step, window, sinks, max_new or 0, out.data_ptr(), o_tok, o_head, 1 if new_out else 0,
            ws.data_ptr(), size)
    return out


class PagedKVCache:
    """The pool of pages of a model's layers and the bookkeeping of a batch of
    requests over it, all on the device.

        cache = PagedKVCache(layers, pages, page_size, kv_heads, head_dim, requests, max_len, dtype, device)
        step = cache.step(new_lens, num_tokens)          # once a step
        k, v = cache.k[layer], cache.v[layer]            # for rope_write_paged and paged_attention

    `dtype`: the activations' type or a float8 type; k_scale, v_scale: float8
    caches' scales, one value or one per head (None: 1). All layers share the
    pages' numbering. Slots hold nothing until they are written; the operators
    never read such a slot. `step` only launches kernels, so it can be part of
    a captured step.

    lens may be lowered in place between steps (drafted tokens that were not
    taken): the pages stay with their request and serve the tokens that come
    instead. A request beyond max_len (rounded up to whole pages) takes no more
    pages; its further tokens get slot -1."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, requests: int, max_len: int,
                 dtype: torch.dtype, device, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        if dtype not in _FP8 + _16BIT:
            raise RuntimeError(f"PagedKVCache: dtype must be bfloat16, float16 or a float8 type, got {dtype}")
        if min(layers, pages, page_size, kv_heads, head_dim, requests, max_len) < 1 or requests > MAX_REQUESTS:
            raise RuntimeError(f"PagedKVCache: sizes must be positive, and at most {MAX_REQUESTS} requests")
        self.page_size = page_size
        pool = torch.empty(layers, 2, pages, page_size, kv_heads, head_dim, dtype=dtype, device=device)
        self.k = [pool[i, 0] for i in range(layers)]
        self.v = [pool[i, 1] for i in range(layers)]
        self.k_scale, self.v_scale = k_scale, v_scale
        self.block_table = torch.full((requests, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.held = torch.zeros(requests, dtype=torch.int32, device=device)  # leading columns of each row that have had a page
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_head = torch.zeros(1, dtype=torch.int32, device=device)

    def step(self, new_lens: torch.Tensor, num_tokens: int) -> PagedStep:
        """Pages and slots for new_lens (requests,) int32 more tokens; the lengths
        move on. Tokens that do not fit into num_tokens rows are not added. See
        paged_slots, also for a pool that runs short: a token that found no
        page is lost for good."""
        s, held = _step_slots(self, new_lens, num_tokens)
        torch._foreach_copy_([self.lens, self.held, self.free_head], [s.kv_lens, held, s.free_head])
        return s

    def release(self, request: int) -> None:
        """Ends a request: its pages are free again, its row starts anew. Waits
        for the device."""
        total = self.free_pages.numel()
        head = min(int(self.free_head), total)
        row = self.block_table[request]
        ids = row[row >= 0]
        n = ids.numel()
        if n > head:
            raise RuntimeError(f"PagedKVCache: request {request} holds {n} pages, {head} are taken")
        self.free_pages[head - n:] = torch.cat([self.free_pages[head:], ids])
        self.free_head.fill_(head - n)
        row.fill_(-1)
        self.lens[request] = 0
        self.held[request] = 0
