"""Measured cases of the paged key/value-cache operators of an FP8 inference stack.

Three operators, in the order in which one decoding or prefill step calls them:

  slots      page allotment and token placement of one step: request lengths ->
             offsets, positions, cache slots, grown block tables
  write      rotary embedding of q and k, k and v rounded into the paged cache
             (16-bit or float8 with a scale per head)
  attention  causal attention of each request's new tokens over its pages, with
             an optional sliding window whose first tokens stay visible

`own` selects what run() computes with: False, the plain form in elementary
torch operations; True, the package's operators.
"""
import itertools
import math
import os
import random
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_SIZE = {"bf16": 2, "f16": 2, "e4m3": 1, "e5m2": 1}
_FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
_HEADS = ((32, 8, 128), (32, 32, 128), (28, 4, 128), (16, 2, 64), (12, 12, 64), (24, 8, 80), (8, 1, 256), (7, 1, 128))
_PAGES = (16, 32, 64, 128, 24)


def listed():
    llama = {"hq": 32, "hk": 8, "d": 128}
    return [
        # one request decodes one token: pure launch latency
        {"name": "slots 1 request", "op": "slots", "requests": 1, "cached": 2047, "new": 1, "ragged": False, "page": 16, "pad": 0},
        # a full prefill step of ragged prompts, padded to the captured size
        {"name": "slots 300 prompts", "op": "slots", "requests": 300, "cached": 4000, "new": 830, "ragged": True, "page": 64, "pad": 1021},
        # a decode step of 16 requests into a float8 cache
        {"name": "write 16 tokens e4m3", "op": "write", "tokens": 16, **llama, "x": "bf16", "cache": "e4m3", "page": 16, "positions": 32768},
        # the prefill of batch 8 x 2048, 16-bit cache
        {"name": "write 8x2048 bf16", "op": "write", "tokens": 16384, **llama, "x": "bf16", "cache": "bf16", "page": 64, "positions": 2048},
        # an odd number of tokens, other head layout, pages that are no power of two
        {"name": "write 5001 tokens e5m2", "op": "write", "tokens": 5001, "hq": 16, "hk": 2, "d": 64, "x": "f16", "cache": "e5m2", "page": 24, "positions": 131072},
        # one request, one token: the smallest attention call of a chat
        {"name": "decode 1 x 2048", "op": "attention", "requests": 1, "cached": 2047, "new": 1, "ragged": False, **llama, "x": "bf16", "cache": "bf16", "page": 16, "window": 0, "sinks": 0},
        # a batch of decodes of very different lengths over a float8 cache: the cache is what is read
        {"name": "decode 64 ragged e4m3", "op": "attention", "requests": 64, "cached": 32767, "new": 1, "ragged": True, **llama, "x": "bf16", "cache": "e4m3", "page": 64, "window": 0, "sinks": 0},
        # five drafted tokens a request are verified at once
        {"name": "verify 24 x 5 e5m2", "op": "attention", "requests": 24, "cached": 8000, "new": 5, "ragged": True, "hq": 16, "hk": 2, "d": 64, "x": "f16", "cache": "e5m2", "page": 16, "window": 0, "sinks": 0},
        # the prefill of batch 8 x 2048: compute bound
        {"name": "prefill 8x2048", "op": "attention", "requests": 8, "cached": 0, "new": 2048, "ragged": False, **llama, "x": "bf16", "cache": "bf16", "page": 64, "window": 0, "sinks": 0},
        # one chunk of a long prompt over what is cached in float8
        {"name": "chunk 2048 over 14000 e4m3", "op": "attention", "requests": 1, "cached": 14001, "new": 2048, "ragged": False, **llama, "x": "bf16", "cache": "e4m3", "page": 64, "window": 0, "sinks": 0},
        # the same with a sliding window whose first tokens stay visible
        {"name": "window 1500 over 20000", "op": "attention", "requests": 1, "cached": 20003, "new": 1500, "ragged": False, **llama, "x": "bf16", "cache": "bf16", "page": 32, "window": 4096, "sinks": 4},
        # a mixed step: one chunk among decoding requests
        {"name": "mixed 12 f16", "op": "attention", "requests": 12, "cached": 6000, "new": 700, "ragged": True, "mixed": True, "hq": 28, "hk": 4, "d": 128, "x": "f16", "cache": "f16", "page": 16, "window": 0, "sinks": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("slots", "write", "write", "attention", "attention", "attention", "attention"))
    page = rng.choice(_PAGES)
    if op == "slots":
        requests = _log(rng, 1, 2000)
        return {"op": op, "requests": requests, "cached": _log(rng, 1, 40000), "new": _log(rng, 1, max(1, min(4000, 240000 // requests))),
                "ragged": rng.random() < 0.7, "page": page, "pad": rng.choice((0, 1, rng.randint(2, 500)))}
    hq, hk, d = rng.choice(_HEADS)
    x = rng.choice(("bf16", "bf16", "f16"))
    cache = rng.choice((x, x, "e4m3", "e4m3", "e5m2"))
    heads = {"hq": hq, "hk": hk, "d": d, "x": x, "cache": cache, "page": page}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 16000), **heads, "positions": rng.choice((2048, 32768, 131072))}
    kind = rng.choice(("decode", "verify", "chunk", "mixed"))
    window, sinks = rng.choice(((0, 0), (0, 0), (rng.randint(1, 6000), 0), (rng.randint(100, 6000), rng.randint(1, 130))))
    if kind == "decode":
        requests, new = _log(rng, 1, 96), 1
    elif kind == "verify":
        requests, new = _log(rng, 1, 32), rng.randint(2, 12)
    elif kind == "chunk":
        requests, new = _log(rng, 1, 6), _log(rng, 13, 1500)
    else:
        requests, new = _log(rng, 2, 16), _log(rng, 13, 700)
    # the plain form holds all scores of the padded batch: bound them, and the cache's size
    most = int(min(32000, 1.0e9 / (requests * new * hq), 6.0e8 / (requests * hk * d)))
    case = {"op": op, "requests": requests, "cached": _log(rng, 1, max(2, most - new)), "new": new, "ragged": rng.random() < 0.7, **heads, "window": window, "sinks": sinks}
    if kind == "mixed":
        case["mixed"] = True
    return case


# ------------------------------------------------------------------ lengths and inputs
def _lengths(c):
    """(cached, new) tokens of each request: part of the case, not of its seed."""
    r = random.Random("%(requests)d %(cached)d %(new)d %(page)d" % c)
    n = c["requests"]
    if c.get("mixed"):
        new = [1] * n
        new[r.randrange(n)] = c["new"]
        cached = [r.randint(0, c["cached"]) for _ in range(n)]
    elif c["ragged"]:
        new = [1] * n if c["new"] == 1 else [r.randint(1, c["new"]) for _ in range(n)]
        cached = [r.randint(0, c["cached"]) for _ in range(n)]
        new[r.randrange(n)], cached[r.randrange(n)] = c["new"], c["cached"]
    else:
        new, cached = [c["new"]] * n, [c["cached"]] * n
    return cached, new


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _random_cache(g, shape, scale, dtype):
    """N(0, 1) values held as `dtype` codes of value / scale, a part of the pool at a time."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // max(1, out[0].numel()))
    for i in range(0, shape[0], step):
        v = torch.randn(out[i:i + step].shape, generator=g, device="cuda")
        _bits(out)[i:i + step] = _bits(_round(v / scale.view(1, 1, -1, 1), dtype))
    return out


def _bits(t):
    return t.view(torch.uint8 if t.dtype.itemsize == 1 else torch.int16)


def _round(v, dtype):
    """One rounding of float32 values to `dtype`; float8 saturates at its largest finite value."""
    if dtype.itemsize == 1:
        m = torch.finfo(dtype).max
        v = v.clamp(-m, m)
    return v.to(dtype)


def _scales(g, c):
    if c["cache"] not in _FMAX:
        return None, None
    s = (0.5 + torch.rand(2, c["hk"], generator=g, device="cuda")) * (8.0 / _FMAX[c["cache"]])
    return s[0].contiguous(), s[1].contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "slots":
        cached, new = _lengths(c)
        have = [-(-a // c["page"]) for a in cached]
        need = [-(-(a + b) // c["page"]) for a, b in zip(cached, new)]
        pool = torch.randperm(sum(need) + 64, generator=g, device="cuda").to(torch.int32)
        width = max(need) + 3
        table = torch.full((c["requests"], width), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(width, device="cuda")[None] < _i32(have)[:, None]
        table[held] = pool[: sum(have)]
        return {"case": c, "cached": _i32(cached), "new": _i32(new), "table": table, "free": pool[sum(have):].contiguous(),
                "tokens": sum(new) + c["pad"], "page": c["page"]}
    if c["op"] == "write":
        t, hq, hk, d, page = c["tokens"], c["hq"], c["hk"], c["d"], c["page"]
        pages = -(-t // page) + 2
        ks, vs = _scales(g, c)
        one = torch.ones(hk, device="cuda")
        angle = torch.arange(c["positions"], device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))[None]
        start = torch.randint(0, max(1, c["positions"] - t), (1,), generator=g, device="cuda")
        pos = ((start + torch.arange(t, device="cuda")) % c["positions"]).to(torch.int32)
        if t <= 512:  # decoding requests, each at a place of its own
            pos = torch.randint(0, c["positions"], (t,), generator=g, device="cuda").to(torch.int32)
            slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].contiguous()
        else:         # prompts: runs of slots in pages of any order
            order = torch.randperm(pages, generator=g, device="cuda")
            at = torch.arange(t, device="cuda")
            slots = order[at // page] * page + at % page
        return {"case": c, "qkv": torch.randn(t, (hq + 2 * hk) * d, generator=g, device="cuda").to(_DT[c["x"]]),
                "cos": angle.cos().float(), "sin": angle.sin().float(), "pos": pos, "slots": slots,
                "k": _random_cache(g, (pages, page, hk, d), one if ks is None else ks, _DT[c["cache"]]),
                "v": _random_cache(g, (pages, page, hk, d), one if vs is None else vs, _DT[c["cache"]]), "ks": ks, "vs": vs}
    cached, new = _lengths(c)
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    kv = [a + b for a, b in zip(cached, new)]
    need = [-(-a // page) for a in kv]
    pages, width = sum(need) + 2, max(need) + 1
    table = torch.zeros((c["requests"], width), dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None] < _i32(need)[:, None]] = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[: sum(need)]
    ks, vs = _scales(g, c)
    one = torch.ones(hk, device="cuda")
    cu = [0, *itertools.accumulate(new)]
    return {"case": c, "q": torch.randn(sum(new), hq, d, generator=g, device="cuda").mul_(1.5).to(_DT[c["x"]]),
            "k": _random_cache(g, (pages, page, hk, d), one if ks is None else ks, _DT[c["cache"]]),
            "v": _random_cache(g, (pages, page, hk, d), one if vs is None else vs, _DT[c["cache"]]),
            "ks": ks, "vs": vs, "table": table, "cu": _i32(cu), "kv": _i32(kv), "most_new": max(new), "most_kv": max(kv)}


# ------------------------------------------------------------------ the plain forms
def _plain_slots(s):
    cached, new, table, free, page = s["cached"].long(), s["new"].long(), s["table"], s["free"], s["page"]
    have, kv = (cached + page - 1) // page, cached + new
    add = (kv + page - 1) // page - have
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), new.cumsum(0)])
    base = add.cumsum(0) - add
    col = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (col >= have[:, None]) & (col < (have + add)[:, None])
    take = (base[:, None] + col - have[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[take], table))
    t = torch.arange(s["tokens"], device="cuda")
    r = torch.searchsorted(cu, t, right=True) - 1
    in_batch = r < new.numel()
    r = r.clamp(max=new.numel() - 1)
    pos = torch.where(in_batch, cached[r] + t - cu[r], 0)
    slot = torch.where(in_batch, table[r, pos // page].long() * page + pos % page, -1)
    return cu.int(), kv.int(), pos.int(), slot, table, add.sum().int().reshape(1)


def _plain_write(s):
    c = s["case"]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    x = s["qkv"].float().view(-1, hq + 2 * hk, d)
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    a, b = x[:, : hq + hk, : d // 2], x[:, : hq + hk, d // 2:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    k, v = y[:, hq:], x[:, hq + hk:]
    if s["ks"] is not None:
        k, v = k / s["ks"][:, None], v / s["vs"][:, None]
    _bits(s["k"]).view(-1, hk, d)[s["slots"]] = _bits(_round(k, s["k"].dtype))
    _bits(s["v"]).view(-1, hk, d)[s["slots"]] = _bits(_round(v, s["v"].dtype))
    return y[:, :hq].to(s["qkv"].dtype), s["k"], s["v"]


def _gathered(cache, scale, table, most, dtype):
    """(requests, kv heads, most, head size) values of the requests' pages."""
    page = cache.shape[1]
    at = torch.arange(most, device="cuda")
    v = _bits(cache)[table[:, at // page].long(), at % page].view(cache.dtype).to(dtype)
    if scale is not None:
        v = v * scale[:, None].to(dtype)
    return v.transpose(1, 2)


def _plain_attention(s):
    c = s["case"]
    hq, hk, d, n, kv = c["hq"], c["hk"], c["d"], s["most_new"], s["kv"].long()
    cu, group = s["cu"].long(), c["hq"] // c["hk"]
    new = cu[1:] - cu[:-1]
    i = torch.arange(n, device="cuda")
    rows = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(-1, n, hk, group, d).permute(0, 2, 1, 3, 4).reshape(-1, hk, n * group, d)
    k = _gathered(s["k"], s["ks"], s["table"], s["most_kv"], torch.float32)
    p = (q @ k.transpose(2, 3)).mul_(d ** -0.5).view(-1, hk, n, group, s["most_kv"])
    at = torch.arange(s["most_kv"], device="cuda")
    pos = (kv - new)[:, None] + i
    seen = at <= pos[..., None]
    if c["window"]:
        seen &= (pos[..., None] - at < c["window"]) | (at < c["sinks"])
    seen = seen[:, None, :, None]
    p.masked_fill_(~seen, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_().masked_fill_(~seen, 0.0)
    total = p.sum(-1, keepdim=True)
    v = _gathered(s["v"], s["vs"], s["table"], s["most_kv"], torch.float32)
    o = (p.view(-1, hk, n * group, s["most_kv"]) @ v).view(-1, hk, n, group, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(-1, n, hq, d)
    return o[i[None] < new[:, None]].to(s["q"].dtype)


# ------------------------------------------------------------------ the framework's operators
_nat = None


def _native():
    global _nat
    if _nat is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mps-fp8-for-torch-and-comfyui-python-package_b200"))
        from fp4_fp8_for_torch_mps import fp8_mps_native
        _nat = fp8_mps_native
    return _nat


def _own(s):
    nat, c = _native(), s["case"]
    if c["op"] == "slots":
        step = nat.paged_slots(s["cached"], s["new"], s["table"], s["free"], s["page"], s["tokens"])
        return step.cu_new, step.kv_lens, step.positions, step.slots, s["table"], step.free_head
    if c["op"] == "write":
        q = nat.rope_write_paged(s["qkv"], s["cos"], s["sin"], s["pos"], s["slots"], s["k"], s["v"], c["hq"], k_scale=s["ks"], v_scale=s["vs"])
        return q, s["k"], s["v"]
    return nat.paged_attention(s["q"], s["k"], s["v"], s["table"], s["cu"], s["kv"], window=c["window"], sinks=c["sinks"],
                               k_scale=s["ks"], v_scale=s["vs"], max_new=s["most_new"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_slots(state) if op == "slots" else _plain_write(state) if op == "write" else _plain_attention(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "slots":
        cached, new = _lengths(c)
        t, fresh = sum(new), sum(-(-(a + b) // c["page"]) - -(-a // c["page"]) for a, b in zip(cached, new))
        started = sum(a % c["page"] > 0 for a in cached)
        return {"bytes": 8 * c["requests"] + 4 * started + 8 * fresh + 8 * c["requests"] + 8 + 12 * (t + c["pad"]), "flops": 0}
    hq, hk, d = c["hq"], c["hk"], c["d"]
    if c["op"] == "write":
        t, e = c["tokens"], _SIZE[c["cache"]]
        return {"bytes": t * ((2 * hq + 2 * hk) * d * 2 + 2 * hk * d * e + 12) + min(t, c["positions"]) * d * 4, "flops": t * (hq + hk) * d * 3}
    cached, new = _lengths(c)
    w, sinks, pairs, keys = c["window"], c["sinks"], 0, 0
    for a, b in zip(cached, new):
        if not w:
            pairs += b * a + b * (b + 1) // 2
            keys += a + b
        else:
            first = max(0, a + 1 - w)                      # the oldest key in the first query's window
            keys += a + b - first + min(sinks, first)
            pairs += sum(min(p + 1, w) + min(sinks, max(0, p + 1 - w)) for p in range(a, a + b))
    return {"bytes": 2 * sum(new) * hq * d * 2 + keys * 2 * hk * d * _SIZE[c["cache"]], "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ the definition in 64 bits
def _held(x, name):
    """float64 values at the nearest value of a float8 format (ties to even, saturated), in arithmetic on its grid."""
    digits, least = {"e4m3": (3, -6), "e5m2": (2, -14)}[name]
    step = torch.exp2(((x.abs().frexp().exponent - 1).clamp(min=least) - digits).double())
    return ((x / step).round() * step).clamp(-_FMAX[name], _FMAX[name])


def exact(case, seed):
    c = case
    if c["op"] == "slots":
        return None                                        # whole numbers
    s = prepare(case, seed)
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    group = hq // hk
    if c["op"] == "write":
        x = s["qkv"].double().reshape(c["tokens"], -1, d)
        z = torch.complex(x[..., : d // 2], x[..., d // 2:])
        turn = torch.complex(s["cos"].double(), s["sin"].double()).index_select(0, s["pos"].long())
        z = torch.cat([z[:, : hq + hk] * turn.unsqueeze(1), z[:, hq + hk:]], 1)
        y = torch.cat([z.real, z.imag], -1)
        out = [y[:, :hq]]
        for cache, scale, part in ((s["k"], s["ks"], y[:, hq:hq + hk]), (s["v"], s["vs"], y[:, hq + hk:])):
            if scale is not None:
                part = _held(part / scale.double().view(1, -1, 1), c["cache"])
            flat = cache.double().reshape(-1, hk, d)
            flat.index_copy_(0, s["slots"], part)
            out.append(flat.view(cache.shape))
        return tuple(out)
    cached, new = _lengths(c)
    out, row = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for r, (a, b) in enumerate(zip(cached, new)):
        pages = s["table"][r, : -(-(a + b) // page)].long()
        wide = []
        for cache, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            flat = _bits(cache)[pages].view(cache.dtype).double()
            flat = flat.reshape(-1, hk, d)[: a + b]
            wide.append(flat if scale is None else flat * scale.double().view(1, hk, 1))
        age = torch.arange(a, a + b, device="cuda").view(-1, 1) - torch.arange(a + b, device="cuda").view(1, -1)
        hidden = age < 0
        if c["window"]:
            hidden |= (age >= c["window"]) & (torch.arange(a + b, device="cuda") >= c["sinks"]).view(1, -1)
        for h in range(hq):
            score = s["q"][row:row + b, h].double() @ wide[0][:, h // group].t() / math.sqrt(d)
            score = score.masked_fill_(hidden, -math.inf).softmax(-1)
            out[row:row + b, h] = score @ wide[1][:, h // group]
        row += b
    return out
