"""The paged key/value-cache operators against plain implementations: page
slots against a loop over requests, the rotary cache write against float32
arithmetic bit for bit and against float64, attention against float64.

Attention's tolerance, per output element, from the arithmetic:
  u_out |o|                    the output's rounding (half a step)
  + (u_w + 2 ds + 2^-17) A     A = sum_j w_j |v_j| / sum_j w_j in float64
where u_w is the half step of the weights' type (bf16 2^-8 for a bf16 cache,
f16 2^-11 otherwise), ds bounds the error of a score: (d + 8) 2^-24 of
scale sum |q||k| for the float32 sums, plus, for bf16 queries of a float8
cache, 2^-24 of the row's largest |q| times scale sum |k| (values far below
the row's largest, held in f16); it enters the numerator and the denominator.
2^-17 covers exp2 and the float32 sums over the keys (up to 2^7 joins).
f16 weights have an absolute step too: at most 2^-25 is lost of each (half of
the least subnormal) while the weight of the key that set the row's base is
2^7 and part of the sum, so n keys lose at most n 2^-32 max |v| of the output
(seen where the key with nearly all the weight holds a 0 in that place)."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3, E5M2, BF16, F16 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def nat(device):
    from fp4_fp8_for_torch_mps import fp8_mps_native
    return fp8_mps_native


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def half_step(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------ slots
def plain_slots(cached, new, table, free, page, tokens, head):
    table = [list(r) for r in table]
    cu, kv, pos, slots = [0], [], [], []
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        have, need = -(-c // page), -(-(c + n) // page)
        for col in range(have, need):
            page_id = free[head] if 0 <= head < len(free) else -1
            head += 1
            if col < len(table[r]):
                table[r][col] = page_id
        for p in range(c, c + n):
            col = p // page
            page_id = table[r][col] if col < len(table[r]) else -1
            pos.append(p)
            slots.append(page_id * page + p % page if page_id >= 0 else -1)
        cu.append(cu[-1] + n)
        kv.append(c + n)
    pad = max(0, tokens - len(pos))
    return cu, kv, (pos + [0] * pad)[:tokens], (slots + [-1] * pad)[:tokens], table, head


def check_slots(nat, cached, new, page, cols, n_free, pad=0, head=None, table=None):
    g = torch.Generator().manual_seed(len(cached) * 7 + page)
    n = len(cached)
    if table is None:
        table = torch.randint(0, 1000, (n, cols), generator=g).tolist()
    free = (torch.randperm(max(n_free, 1), generator=g)[:n_free] + 5000).tolist()
    tokens = sum(max(x, 0) for x in new) + pad
    t_dev = i32(table).reshape(n, cols)
    step = nat.paged_slots(i32(cached), i32(new), t_dev, i32(free), page, tokens, None if head is None else i32([head]))
    cu, kv, pos, slots, want, want_head = plain_slots(cached, new, table, free, page, tokens, head or 0)
    assert step.cu_new.tolist() == cu
    assert step.kv_lens.tolist() == kv
    assert step.positions.tolist() == pos
    assert step.slots.tolist() == slots
    assert step.free_head.tolist() == [want_head]
    assert t_dev.tolist() == want


@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("requests", [1, 5, 511, 512, 513, 1700])
def test_slots(nat, requests, page):
    g = torch.Generator().manual_seed(requests + page)
    cached = torch.randint(0, 100, (requests,), generator=g).tolist()
    new = torch.randint(0, 9, (requests,), generator=g).tolist()
    new[requests // 2] = 130
    check_slots(nat, cached, new, page, 240, 4 * sum(new) + 10, pad=3)


@pytest.mark.parametrize("cached,new,page,cols,free,pad,head", [
    ([0], [1], 16, 1, 1, 0, None), ([15], [1], 16, 1, 0, 0, None), ([16], [1], 16, 2, 1, 0, None),
    ([0, 0, 0], [0, 0, 0], 16, 4, 3, 0, None),            # nothing to place
    ([0, 5, 0], [0, 0, 7], 4, 4, 9, 600, 2),              # empty requests around one, padding, a head
    ([3, 8, 1], [9, 9, 9], 4, 8, 3, 0, None),             # the pool runs short
    ([3, 8, 1], [9, 9, 9], 4, 2, 20, 0, None),            # the table runs short
    ([-4, 2], [3, -7], 4, 4, 8, 1, None),                 # lengths below zero count as zero
    ([5], [3], 4, 4, 8, 0, -3), ([5], [30], 4, 9, 8, 0, 2 ** 31 - 2), ([7], [2], 2 ** 30, 1, 0, 0, None),
])
def test_slots_edges(nat, cached, new, page, cols, free, pad, head):
    if head is not None and head > 10 ** 6:               # the head wraps like int32; only the entries matter
        t = i32([[9] * cols])
        step = nat.paged_slots(i32(cached), i32(new), t, i32(list(range(free))), page, 30, i32([head]))
        assert t.tolist() == [[9, 9] + [-1] * 7] and step.slots.tolist() == [9 * 4 + 1, 9 * 4 + 2, 9 * 4 + 3] + [-1] * 27
        return
    check_slots(nat, cached, new, page, cols, free, pad, head)


def test_slots_fewer_rows_than_tokens(nat):
    """Rows behind num_tokens are neither placed nor written."""
    t = i32([[1, -7, -7], [2, -7, -7]])
    step = nat.paged_slots(i32([3, 4]), i32([4, 4]), t, i32([10, 11, 12]), 4, 2)
    assert step.positions.tolist() == [3, 4] and step.slots.tolist() == [7, 40]
    assert t.tolist() == [[1, 10, -7], [2, -7, -7]] and step.cu_new.tolist() == [0, 4, 8]
    assert step.free_head.tolist() == [2]


def test_slots_no_requests(nat):
    step = nat.paged_slots(i32([]), i32([]), torch.empty(0, 3, dtype=torch.int32, device="cuda"), i32([1]), 16, 3)
    assert step.cu_new.tolist() == [0] and step.slots.tolist() == [-1] * 3 and step.free_head.tolist() == [0]


def test_slots_most_requests_and_strided_table(nat):
    n = 16384
    wide = torch.zeros(n, 5, dtype=torch.int32, device="cuda")
    cached = torch.full((n,), 16, dtype=torch.int32, device="cuda")
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    step = nat.paged_slots(cached, new, wide[:, 1:3], torch.arange(n, dtype=torch.int32, device="cuda"), 16, n)
    assert torch.equal(wide[:, 2], torch.arange(n, dtype=torch.int32, device="cuda"))
    assert int(wide[:, [0, 1, 3, 4]].abs().sum()) == 0
    assert torch.equal(step.slots, torch.arange(n, device="cuda") * 16)
    assert torch.equal(step.cu_new, torch.arange(n + 1, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------ rope + write
def saturated(x, dt):
    if dt in (E4M3, E5M2):
        m = torch.finfo(dt).max
        x = x.clamp(-m, m)
    return x.to(dt)


def bits(t):
    return t.view(torch.uint8 if t.element_size() == 1 else torch.int16)


def same(a, b):
    """Equal bit for bit, any NaN standing for any other."""
    nan = torch.isnan(a.float()) & torch.isnan(b.float())
    return bool(((bits(a) == bits(b)) | nan).all())


def rope_f32(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def make_write(t, hq, hk, d, x, cache, page, seed, scales):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(t, (hq + 2 * hk) * d, generator=g, device="cuda") * 2).to(x)
    ang = torch.rand(97, d // 2, generator=g, device="cuda") * 100
    pos = torch.randint(0, 97, (t,), generator=g, device="cuda").int()
    pages = -(-t // page) + 3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].contiguous()
    k = torch.randn(pages, page, hk, d, generator=g, device="cuda").to(cache)
    v = torch.randn(pages, page, hk, d, generator=g, device="cuda").to(cache)
    ks = vs = None
    if cache in (E4M3, E5M2) and scales:
        ks = torch.rand(hk if scales > 1 else 1, generator=g, device="cuda") * 0.1 + 0.01
        vs = torch.rand(hk if scales > 1 else 1, generator=g, device="cuda") * 0.1 + 0.01
    return qkv, ang.cos(), ang.sin(), pos, slots, k, v, ks, vs


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (BF16, E5M2), (F16, E5M2)])
@pytest.mark.parametrize("t,hq,hk,d,page,scales", [(1, 1, 1, 16, 1, 0), (7, 4, 2, 64, 16, 1), (33, 7, 1, 128, 24, 2),
                                                   (129, 12, 12, 80, 64, 2), (5, 0, 3, 256, 16, 2), (1000, 32, 8, 128, 16, 2), (4100, 32, 8, 128, 64, 2)])
def test_write(nat, x, cache, t, hq, hk, d, page, scales):
    """Every value of q and of both caches, the slots no token has included."""
    qkv, cos, sin, pos, slots, k, v, ks, vs = make_write(t, hq, hk, d, x, cache, page, t + d, scales)
    k0, v0 = k.clone(), v.clone()
    q = nat.rope_write_paged(qkv, cos, sin, pos, slots, k, v, hq, ks, vs)
    xs = qkv.view(t, -1, d)
    y = rope_f32(xs[:, :hq + hk], cos[pos.long()][:, None], sin[pos.long()][:, None])
    one = torch.ones(1, device="cuda")
    bits(k0).view(-1, hk, d)[slots] = bits(saturated(y[:, hq:] / (one if ks is None else ks)[:, None], cache))
    bits(v0).view(-1, hk, d)[slots] = bits(saturated(xs[:, hq + hk:].float() / (one if vs is None else vs)[:, None], cache))
    assert same(q, y[:, :hq].to(x)) and same(k, k0) and same(v, v0)
    # and the float32 arithmetic is right: float64, half a step of the type plus three float32 roundings of the products
    a, b = xs[:, :hq].double().chunk(2, -1)
    c, s = cos[pos.long()][:, None].double(), sin[pos.long()][:, None].double()
    ref, mag = torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([(a * c).abs() + (b * s).abs()] * 2, -1)
    mag[..., d // 2:] = (b * c).abs() + (a * s).abs()
    assert bool(((q.double() - ref).abs() <= half_step(x) * ref.abs() + 2.0 ** -22 * mag + 2.0 ** -25).all())


@pytest.mark.parametrize("cache", [BF16, E4M3, E5M2])
def test_write_odd_values_slots_and_positions(nat, cache):
    """Infinities and NaN, saturation, tokens without a slot (left as it was), positions outside the tables (NaN)."""
    t, hq, hk, d, page = 9, 2, 2, 32, 4
    qkv, cos, sin, pos, slots, k, v, _, _ = make_write(t, hq, hk, d, BF16, cache, page, 3, 0)
    qkv[0], qkv[1], qkv[2] = 1e38, math.inf, -math.inf
    qkv[3, ::3] = math.nan
    qkv[4] = -70000.0
    slots[5], slots[6], slots[7] = -1, k.shape[0] * page, 2 ** 40
    pos[7], pos[8] = -1, 97
    k0, v0 = k.clone(), v.clone()
    q = nat.rope_write_paged(qkv, cos, sin, pos, slots, k, v, hq)
    xs = qkv.view(t, -1, d)
    inside = (pos >= 0) & (pos < 97)
    c = torch.where(inside[:, None], cos[pos.clamp(0, 96).long()], math.nan)[:, None]
    s = torch.where(inside[:, None], sin[pos.clamp(0, 96).long()], math.nan)[:, None]
    y = rope_f32(xs[:, :hq + hk], c, s)
    keep = (slots >= 0) & (slots < k.shape[0] * page)
    bits(k0).view(-1, hk, d)[slots[keep]] = bits(saturated(y[keep, hq:], cache))
    bits(v0).view(-1, hk, d)[slots[keep]] = bits(saturated(xs[keep, hq + hk:].float(), cache))
    assert same(q, y[:, :hq].to(BF16)) and same(k, k0) and same(v, v0)
    assert bool(torch.isnan(q[7:]).all())


def test_write_strides(nat):
    """qkv a column slice of a wider tensor, the caches two views of one tensor with the heads before the slots."""
    t, hq, hk, d, page, pages = 21, 4, 2, 64, 8, 5
    qkv, cos, sin, pos, slots, _, _, ks, vs = make_write(t, hq, hk, d, BF16, E4M3, page, 9, 2)
    wide = torch.zeros(t, qkv.shape[1] + 48, dtype=BF16, device="cuda")
    wide[:, 16:16 + qkv.shape[1]] = qkv
    both = torch.zeros(pages, 2, hk, page, d, dtype=torch.uint8, device="cuda").view(E4M3)
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    slots = torch.arange(t, device="cuda")
    q = nat.rope_write_paged(wide[:, 16:16 + qkv.shape[1]], cos, sin, pos, slots, kc, vc, hq, ks, vs)
    k2 = torch.zeros(pages, page, hk, d, dtype=torch.uint8, device="cuda").view(E4M3)
    v2 = torch.zeros_like(k2)
    q2 = nat.rope_write_paged(qkv, cos, sin, pos, slots, k2, v2, hq, ks, vs)
    assert torch.equal(q, q2)
    assert torch.equal(bits(kc.contiguous()), bits(k2)) and torch.equal(bits(vc.contiguous()), bits(v2))


# ------------------------------------------------------------------ attention
def build(new, kv, hq, hk, d, page, x, cache, seed, scales=2, pad=0, spread=1.5, layout="plain"):
    """Inputs whose unused slots, unused pages and padding rows hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = len(new)
    need = [max(0, -(-b // page)) for b in kv]
    pages = sum(need) + 3
    cols = max(need + [0]) + 2
    table = torch.full((n, cols), -5, dtype=torch.int32, device="cuda")
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    at = 0
    for r in range(n):
        table[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]

    def cache_of():
        c = torch.full((pages, page, hk, d), math.nan, device="cuda")
        for r in range(n):
            if kv[r] > 0:
                flat = torch.full((need[r] * page, hk, d), math.nan, device="cuda")
                flat[:kv[r]] = torch.randn(kv[r], hk, d, generator=g, device="cuda")
                c[table[r, :need[r]].long()] = flat.view(need[r], page, hk, d)
        return c
    kf, vf = cache_of(), cache_of()
    ks = vs = None
    if cache in (E4M3, E5M2):
        if scales:
            ks = torch.rand(hk if scales > 1 else 1, generator=g, device="cuda") * 0.02 + 0.02
            vs = torch.rand(hk if scales > 1 else 1, generator=g, device="cuda") * 0.02 + 0.02
            kf, vf = kf / ks[:, None], vf / vs[:, None]
    k, v = kf.to(cache), vf.to(cache)
    if layout == "heads first":        # (pages, 2, heads, slots, d) storage
        both = torch.stack([bits(k).transpose(1, 2), bits(v).transpose(1, 2)], 1).contiguous().view(cache)
        k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    t = sum(new) + pad
    q = (torch.randn(t, hq, d, generator=g, device="cuda") * spread).to(x)
    if pad:
        q[sum(new):] = math.nan
    cu = i32([0, *itertools.accumulate(new)])
    return dict(q=q, k=k, v=v, table=table, cu=cu, kv=i32(kv), ks=ks, vs=vs)


def reference(s, window=0, sinks=0, scale=None):
    """(out, tolerance) in float64, one request and head at a time."""
    q, k, v = s["q"], s["k"], s["v"]
    pages, page, hk, d = k.shape
    hq = q.shape[1]
    scale = d ** -0.5 if scale is None else scale
    fp8 = k.dtype in (E4M3, E5M2)
    u_w, u_out = half_step(F16 if fp8 else q.dtype), half_step(q.dtype)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    cu, kv = s["cu"].tolist(), s["kv"].tolist()
    for r in range(len(kv)):
        a, b = cu[r], cu[r + 1]
        n, m = b - a, max(kv[r], 0)
        if n == 0 or m == 0:
            continue
        j = torch.arange(m, device="cuda")
        col = j // page
        ids = torch.where(col < s["table"].shape[1], s["table"][r].long()[col.clamp(max=s["table"].shape[1] - 1)], -1)
        ok = (ids >= 0) & (ids < pages)
        pos = torch.arange(m - n, m, device="cuda")[:, None]
        seen = (j <= pos) & ok
        if window:
            seen &= (pos - j < window) | (j < sinks)
        raw = [bits(c.contiguous()).view(-1, hk, d)[ids.clamp(0, pages - 1) * page + j % page].view(c.dtype).double() for c in (k, v)]
        for h in range(hq):
            kh = h // (hq // hk)
            kk, vv = raw[0][:, kh], raw[1][:, kh]
            if s["ks"] is not None:
                kk = kk * s["ks"].double()[kh if s["ks"].numel() > 1 else 0]
                vv = vv * s["vs"].double()[kh if s["vs"].numel() > 1 else 0]
            kk = torch.where(seen.any(0)[:, None], kk, 0.0)
            qq = q[a:b, h].double()
            sc = torch.where(seen, qq @ kk.t() * scale, -math.inf)
            any_seen = seen.any(1, keepdim=True)
            w = torch.where(any_seen, torch.exp(sc - torch.where(any_seen, sc.amax(1, keepdim=True), 0.0)), 0.0)
            w = torch.where(seen, w, 0.0)
            l = w.sum(1, keepdim=True).clamp(min=1e-300)
            hidden = ~seen.any(0)
            vv = torch.where(hidden[:, None], 0.0, vv)
            if not bool(torch.isfinite(vv).all()):     # a key that some rows see and others do not
                vz = torch.where(torch.isfinite(vv), vv, 0.0)
                o = w @ vz
                for jj in torch.nonzero(~torch.isfinite(vv).all(1)).flatten().tolist():
                    o = o + torch.where(seen[:, jj:jj + 1], w[:, jj:jj + 1] * torch.where(torch.isfinite(vv[jj]), 0.0, vv[jj]), 0.0)
                vv_abs = vz.abs()
            else:
                o, vv_abs = w @ vv, vv.abs()
            out[a:b, h] = o / l
            big = w @ vv_abs / l
            mag = torch.where(seen, qq.abs() @ kk.abs().t(), 0.0).amax(1, keepdim=True) * abs(scale)
            ds = (d + 8) * 2.0 ** -24 * mag
            if fp8 and q.dtype == BF16:
                ds = ds + 2.0 ** -24 * qq.abs().amax(1, keepdim=True) * torch.where(seen, kk.abs().sum(1)[None], 0.0).amax(1, keepdim=True) * abs(scale)
            lost = m * 2.0 ** -32 * vv_abs.max() if u_w == half_step(F16) else 0.0
            tol[a:b, h] = u_out * out[a:b, h].abs() + (u_w + 2 * ds + 2.0 ** -17) * big + lost + 1e-30
    return out, tol


def run(nat, s, window=0, sinks=0, scale=None, **kw):
    return nat.paged_attention(s["q"], s["k"], s["v"], s["table"], s["cu"], s["kv"], scale=scale, window=window, sinks=sinks,
                               k_scale=s["ks"], v_scale=s["vs"], **kw)


def check(nat, s, window=0, sinks=0, scale=None, **kw):
    got = run(nat, s, window, sinks, scale, **kw)
    ref, tol = reference(s, window, sinks, scale)
    off = (got.double() - ref).abs()
    same_odd = (torch.isnan(ref) & torch.isnan(got)) | (ref == got.double())
    good = torch.where(torch.isfinite(ref), off <= tol, same_odd)
    assert bool(good.all()), (torch.nonzero(~good)[:5].tolist(), float((off / tol)[~good].nan_to_num(9e9).max()))
    return got


TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (BF16, E5M2), (F16, E5M2)]
LENS = {
    "decode": ([1] * 9, [1, 2, 63, 64, 65, 128, 1000, 17, 333]),
    "verify": ([5, 2, 7, 1, 3], [5, 100, 64, 700, 3]),
    "prefill": ([1, 64, 65, 130, 31], [1, 64, 65, 130, 31]),
    "chunk": ([100, 3, 1, 257, 40], [400, 900, 77, 258, 2000]),
}


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("hq,hk,d,page", [(8, 2, 128, 16), (4, 4, 64, 24)])
def test_attention(nat, x, cache, kind, hq, hk, d, page):
    new, kv = LENS[kind]
    check(nat, build(new, kv, hq, hk, d, page, x, cache, seed=d + len(kv)), max_new=max(new))


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, E4M3)])
@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("hq,hk,d,page", [(1, 1, 16, 1), (7, 1, 128, 64), (6, 2, 80, 40), (12, 4, 96, 16), (16, 1, 256, 16),
                                          (5, 5, 256, 128), (3, 1, 208, 7), (40, 2, 64, 16)])
def test_attention_heads(nat, x, cache, kind, hq, hk, d, page):
    new, kv = LENS[kind]
    check(nat, build(new, kv, hq, hk, d, page, x, cache, seed=hq + d))


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("new,window", [(2, 0), (3, 70), (4, 0), (5, 0), (8, 100), (9, 0), (16, 0), (17, 60), (33, 0)])
def test_attention_wide_heads_by_rows(nat, x, cache, new, window):
    """Head sizes above 128, eight heads a group: 16, 24, 32, 40, 64, 72, 128, 136 and 264 rows a request."""
    s = build([new, 1, new], [new + 700, 65, new], 8, 1, 256, 24, x, cache, seed=new)
    check(nat, s, window=window, sinks=3 if window else 0, max_new=new)


@pytest.mark.parametrize("new", [3, 8, 17])
def test_attention_wide_heads_many_requests(nat, new):
    """More requests than the block that looks for its share has threads."""
    n = 300
    s = build([new] * n, [new + r % 70 for r in range(n)], 8, 1, 256, 16, BF16, E4M3, seed=new)
    check(nat, s, max_new=new)


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (BF16, E4M3)])
@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (64, 0), (100, 64), (100, 130), (63, 1), (1500, 4), (10 ** 9, 7), (300, 10 ** 9)])
def test_attention_window(nat, x, cache, kind, window, sinks):
    new, kv = LENS[kind]
    check(nat, build(new, kv, 8, 2, 128, 16, x, cache, seed=window % 1000 + sinks % 1000), window, sinks, max_new=max(new))


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, E5M2)])
def test_attention_rows_that_see_nothing(nat, x, cache):
    """More new tokens than the length says, no tokens at all, a request with nothing cached: zeros."""
    s = build([4, 0, 3, 70, 1], [2, 50, 0, 10, 0], 4, 2, 64, 16, x, cache, seed=1)
    got = check(nat, s)
    assert int((got[:2] != 0).sum()) == 0 and int((got[4:7] != 0).sum()) == 0
    assert bool((got[2:4] != 0).any())


@pytest.mark.parametrize("max_new", [None, 1, 40, 10 ** 6])
def test_attention_hint_and_padding(nat, max_new):
    """Any max_new gives right results; rows behind the last request stay (given out) or are 0 (new out)."""
    s = build([40, 1, 20], [90, 200, 20], 8, 2, 64, 16, BF16, E4M3, seed=4, pad=13)
    got = check(nat, s, max_new=max_new)
    assert int((got[61:] != 0).sum()) == 0
    out = torch.full_like(s["q"], 7.0)
    again = run(nat, s, max_new=max_new, out=out)
    assert again is out and torch.equal(out[:61], got[:61]) and bool((out[61:] == 7.0).all())


def test_attention_offsets_outside_the_rows(nat):
    """cu_new beyond q's rows is clipped; requests of no rows and no requests give zeros."""
    s = build([3, 2], [30, 20], 4, 2, 64, 16, BF16, BF16, seed=5)
    whole = run(nat, s)
    s["cu"] = i32([0, 3, 900])
    s["kv"] = i32([30, 20])
    assert torch.equal(run(nat, s)[:3], whole[:3])
    none = nat.paged_attention(s["q"], s["k"], s["v"], s["table"][:0], i32([0]), i32([]))
    assert int((none != 0).sum()) == 0
    empty = nat.paged_attention(s["q"][:0], s["k"], s["v"], s["table"], i32([0, 0, 0]), s["kv"])
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("new,kv", [([1, 1], [300, 40]), ([90, 2], [200, 40])])
def test_attention_bad_pages_hide_their_keys(nat, new, kv):
    s = build(new, kv, 4, 2, 64, 16, BF16, E4M3, seed=6)
    s["table"][0, 3], s["table"][0, 4], s["table"][0, 7] = -1, s["k"].shape[0], 2 ** 31 - 1
    s["table"][1, 0] = -2 ** 31
    check(nat, s)
    s["table"][1, :] = -1
    got = check(nat, s)
    assert int((got[new[0]:] != 0).sum()) == 0
    s["table"] = s["table"][:, :2].contiguous()           # the table is shorter than the lengths say
    check(nat, s)


@pytest.mark.parametrize("x,cache", [(BF16, BF16), (F16, F16), (BF16, E5M2), (BF16, E4M3)])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (4, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("new,kv", [([70, 1], [150, 64]), ([300], [300]), ([2, 1], [128, 65])])
def test_attention_infinities_and_nan_at_hidden_keys(nat, x, cache, hq, hk, d, new, kv):
    """A later token's infinity or NaN does not reach the queries before it, and does reach those that see it."""
    s = build(new, kv, hq, hk, d, 16, x, cache, seed=8, scales=0)
    page = s["table"][0, (kv[0] - 1) // 16].item()
    slot = (kv[0] - 1) % 16
    bad = math.nan if cache == E4M3 else math.inf
    s["v"][page, slot, 0, 5] = torch.tensor(bad).to(cache)
    s["k"][page, slot, 0, 9] = torch.tensor(math.nan).to(cache)
    got = check(nat, s)
    assert bool(torch.isfinite(got[:new[0] - 1]).all())
    s["k"][page, slot, 0, 9] = torch.tensor(0.5).to(cache)
    got = check(nat, s)
    assert bool(torch.isfinite(got[:new[0] - 1]).all()) and not bool(torch.isfinite(got[new[0] - 1, 0, 5]))
    s["v"][page, slot, 0, 5] = torch.tensor(0.5).to(cache)  # and past a window
    first = s["table"][0, 0].item()
    s["v"][first, 2, 0, 7] = torch.tensor(bad).to(cache)
    check(nat, s, window=20, sinks=0)
    check(nat, s, window=20, sinks=2)


def test_attention_scores_far_apart(nat):
    """Scores of a few hundred, and one key far above the rest: no overflow, no lost weights."""
    for cache in (BF16, E4M3):
        s = build([1, 30, 100], [700, 90, 300], 4, 1, 128, 16, BF16, cache, seed=10, spread=60.0)
        check(nat, s)
        check(nat, s, scale=0.0)
        check(nat, s, scale=-0.3)


def test_attention_large_and_small_queries(nat):
    """bf16 queries beyond f16's range, and far below it, over a float8 cache."""
    for factor in (2.0 ** 100, 2.0 ** -100):
        s = build([1, 5, 80], [200, 300, 100], 4, 2, 64, 16, BF16, E4M3, seed=11)
        s["q"] = (s["q"].double() * factor).to(BF16)
        check(nat, s, scale=0.125 / factor)


def test_attention_strides(nat):
    """q and out column slices of wider tensors, the caches two views of one tensor with the heads before the slots."""
    for cache in (BF16, E4M3):
        new, kv = LENS["chunk"]
        s = build(new, kv, 8, 2, 64, 16, BF16, cache, seed=12)
        want = check(nat, s)
        h = build(new, kv, 8, 2, 64, 16, BF16, cache, seed=12, layout="heads first")
        wide = torch.zeros(s["q"].shape[0], 12, 80, dtype=BF16, device="cuda")
        wide[:, 1:9, 8:72] = s["q"]
        h["q"] = wide[:, 1:9, 8:72]
        res = torch.full((s["q"].shape[0], 10, 72), 3.0, dtype=BF16, device="cuda")
        run(nat, h, out=res[:, 2:, 8:])
        assert torch.equal(res[:, 2:, 8:], want) and bool((res[:, :2] == 3.0).all()) and bool((res[:, :, :8] == 3.0).all())


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attention_offsets_past_32_bits(nat, cache):
    """A pool of more than 2^32 values whose far pages are used."""
    hk, d, page = 8, 128, 64
    pages = 2 ** 32 // (hk * d * page) + 40
    s = build([1, 100], [500, 700], 16, hk, d, page, BF16, cache, seed=13)
    small = s["k"].shape[0]
    want = run(nat, s)
    big = []
    for c in (s["k"], s["v"]):
        b = torch.empty((pages, page, hk, d), dtype=cache, device="cuda")
        bits(b)[-small:] = bits(c)
        big.append(b)
    s["k"], s["v"] = big
    s["table"] = torch.where(s["table"] >= 0, s["table"] + pages - small, s["table"])
    assert torch.equal(run(nat, s), want)


def test_attention_repeats_bit_for_bit(nat):
    for kind, (new, kv) in LENS.items():
        s = build(new, kv, 8, 2, 128, 16, BF16, E4M3, seed=14)
        a = run(nat, s)
        for _ in range(3):
            assert torch.equal(run(nat, s), a)


def test_attention_many_requests(nat):
    """More requests than one scan of the block holds, most of them idle."""
    new = [1 if r % 3 else 0 for r in range(700)]
    kv = [(r * 7) % 150 + (1 if r % 3 else 0) for r in range(700)]
    check(nat, build(new, kv, 2, 1, 64, 16, BF16, BF16, seed=15))
    new = [0] * 400 + [50] + [0] * 300
    check(nat, build(new, [50] * 701, 2, 1, 64, 16, BF16, BF16, seed=16))
    new = [0] * 20000                                     # more than the kernel for chunks plans for
    new[3], new[19999] = 130, 1
    kv = [0] * 20000
    kv[3], kv[19999] = 140, 70
    check(nat, build(new, kv, 2, 1, 64, 16, BF16, E4M3, seed=19))
    new = [0] * 400 + [50] + [0] * 300
    check(nat, build(new, [50] * 701, 2, 1, 64, 16, BF16, BF16, seed=16))


def test_two_streams_and_two_graphs(nat):
    """Calls that overlap on two streams, and graphs captured with other lengths in the same tensors: each its own result."""
    new, kv = LENS["chunk"]
    a, b = (build(new, kv, 8, 2, 128, 16, BF16, E4M3, seed=s) for s in (17, 18))
    want = [run(nat, a), run(nat, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(nat, s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(nat, s))
        graphs.append(g)
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            for _ in range(5):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    a["kv"].copy_(i32([300, 500, 50, 257, 1000]))         # other lengths through the same graph
    graphs[0].replay()
    assert torch.equal(outs[0], run(nat, a)) and not torch.equal(outs[0], want[0])


# ------------------------------------------------------------------ the three together
@pytest.mark.parametrize("cache", [BF16, E4M3, E5M2])
def test_steps_of_a_batch(nat, cache):
    """Prefill, mixed and decode steps of three requests through slots, write
    and attention, each step's result against float64 over everything that
    was cached so far (as the cache holds it)."""
    hq, hk, d, page = 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(20)
    k = torch.zeros(40, page, hk, d, dtype=torch.uint8 if cache != BF16 else BF16, device="cuda")
    k = k.view(cache)
    v = torch.zeros_like(k)
    ks = torch.full((hk,), 0.02, device="cuda") if cache != BF16 else None
    vs = torch.full((1,), 0.03, device="cuda") if cache != BF16 else None
    ang = torch.rand(300, d // 2, generator=g, device="cuda") * 50
    cos, sin = ang.cos(), ang.sin()
    table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(40, generator=g, device="cuda").int()
    head = i32([0])
    cached = i32([0, 0, 0])
    for new in ([50, 0, 7], [1, 90, 1], [1, 1, 1], [1, 0, 1], [1, 1, 1], [3, 3, 3]):
        t = sum(new) + 2
        step = nat.paged_slots(cached, i32(new), table, free, page, t, head)
        qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g, device="cuda").to(BF16)
        q = nat.rope_write_paged(qkv, cos, sin, step.positions, step.slots, k, v, hq, ks, vs)
        s = dict(q=q, k=k, v=v, table=table, cu=step.cu_new, kv=step.kv_lens, ks=ks, vs=vs)
        check(nat, s, max_new=max(new))
        check(nat, s, window=30, sinks=2)
        cached, head = step.kv_lens, step.free_head
    used = table[table >= 0]
    assert int(head) == used.numel() == used.unique().numel()
    # the custom ops are the same calls
    t2 = table.clone()
    got = torch.ops.fp8_mps.paged_slots(cached, i32([1, 1, 1]), t2, free, page, 3, head)
    want = nat.paged_slots(cached, i32([1, 1, 1]), table, free, page, 3, head)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(t2, table)
    assert torch.equal(torch.ops.fp8_mps.paged_attention(q, k, v, table, step.cu_new, step.kv_lens, k_scale=ks, v_scale=vs),
                       nat.paged_attention(q, k, v, table, step.cu_new, step.kv_lens, k_scale=ks, v_scale=vs))
    k2, v2 = k.clone(), v.clone()
    assert torch.equal(torch.ops.fp8_mps.rope_write_paged(qkv, cos, sin, step.positions, step.slots, k2, v2, hq, ks, vs), q)
    assert torch.equal(bits(k2), bits(k)) and torch.equal(bits(v2), bits(v))
