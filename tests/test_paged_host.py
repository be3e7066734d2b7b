"""Refusals of the paged key/value-cache operators: the launchers' argument
checks and the C entries' own, none of which needs a GPU, and the fake
implementations of the custom ops."""
import ctypes

import pytest
import torch

E4M3, BF16, F16 = torch.float8_e4m3fn, torch.bfloat16, torch.float16


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def slots_args(**kw):
    a = dict(cached_lens=i32(3, 4), new_lens=i32(1, 1), block_table=torch.zeros(2, 4, dtype=torch.int32),
             free_pages=i32(7, 8), page_size=16, num_tokens=2)
    a.update(kw)
    return a


def write_args(**kw):
    k = torch.zeros(4, 16, 2, 64, dtype=BF16)
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=BF16), cos=torch.zeros(10, 32), sin=torch.zeros(10, 32), positions=i32(0, 1, 2),
             slots=torch.zeros(3, dtype=torch.int64), k_cache=k, v_cache=k.clone(), n_q_heads=4)
    a.update(kw)
    return a


def attention_args(**kw):
    k = torch.zeros(4, 16, 2, 64, dtype=BF16)
    a = dict(q=torch.zeros(3, 4, 64, dtype=BF16), k_cache=k, v_cache=k.clone(), block_table=torch.zeros(2, 4, dtype=torch.int32),
             cu_new=i32(0, 1, 3), kv_lens=i32(5, 6))
    a.update(kw)
    return a


WIDE = torch.zeros(4, 16, 2, 128, dtype=BF16)
SLOTS = [
    (dict(cached_lens=torch.zeros(2, dtype=torch.int64)), "cached_lens must be"),
    (dict(new_lens=i32(1)), "new_lens and"),
    (dict(new_lens=i32(1, 9, 1, 9)[::2]), "contiguous"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), "block_table rows"),
    (dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()), "rows must be contiguous"),
    (dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), "not overlap"),
    (dict(free_pages=torch.zeros(2, 2, dtype=torch.int32)), "free_pages must be"),
    (dict(page_size=0), "page_size=0"),
    (dict(num_tokens=-1), "num_tokens=-1"),
    (dict(free_head=i32(1, 2)), "free_head must be"),
    (dict(free_head=torch.zeros(1)), "free_head must be"),
    (dict(cached_lens=torch.zeros(16385, dtype=torch.int32), new_lens=torch.zeros(16385, dtype=torch.int32),
          block_table=torch.zeros(16385, 1, dtype=torch.int32)), "at most 16384"),
    ({}, "CUDA device"),
]
WRITE = [
    (dict(qkv=torch.zeros(3, 512)), "bfloat16 or float16"),
    (dict(qkv=torch.zeros((), dtype=BF16)), "qkv must be"),
    (dict(qkv=torch.zeros(3, 512, dtype=F16)), "the caches must both be"),
    (dict(v_cache=torch.zeros(4, 16, 2, 64, dtype=BF16).to(E4M3)), "the caches must both be"),
    (dict(v_cache=WIDE), "of one shape"),
    (dict(k_cache=torch.zeros(4, 16, 128, dtype=BF16), v_cache=torch.zeros(4, 16, 128, dtype=BF16)), "of one shape"),
    (dict(k_cache=WIDE[..., ::2], v_cache=WIDE[..., ::2]), "contiguous heads"),
    (dict(v_cache=WIDE[..., :64]), "same strides"),
    (dict(n_q_heads=5), "at least 576"),
    (dict(n_q_heads=-1), "qkv must be"),
    (dict(qkv=torch.zeros(512, 3, dtype=BF16).t()), "rows must be contiguous"),
    (dict(qkv=torch.zeros(1, 512, dtype=BF16).expand(3, 512)), "not overlap"),
    (dict(cos=torch.zeros(10, 32, dtype=BF16)), "cos must be"),
    (dict(sin=torch.zeros(9, 32)), "tables"),
    (dict(cos=torch.zeros(10, 31), sin=torch.zeros(10, 31)), "tables"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions must be"),
    (dict(positions=i32(0, 1)), "3 rows, 2 positions"),
    (dict(slots=i32(0, 1, 2)), "slots must be"),
    (dict(k_scale=torch.ones(1)), "float8 cache only"),
    ({}, "CUDA device"),
]
FP8_CACHES = dict(k_cache=torch.zeros(4, 16, 2, 64).to(E4M3), v_cache=torch.zeros(4, 16, 2, 64).to(E4M3))
WRITE += [(dict(FP8_CACHES, k_scale=s), "k_scale must be") for s in
          (torch.ones(3), torch.ones(2, dtype=BF16), torch.ones(4)[::2])] + [(FP8_CACHES, "CUDA device")]
SAME = torch.zeros(3, 4, 64, dtype=BF16)
ATTENTION = [
    (dict(q=torch.zeros(3, 4, 64)), "bfloat16 or float16"),
    (dict(q=torch.zeros(3, 4, 32, dtype=BF16)), "q must be"),
    (dict(q=torch.zeros(3, 256, dtype=BF16)), "q must be"),
    (dict(q=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2)), "contiguous heads"),
    (dict(q=torch.zeros(3, 5, 64, dtype=BF16)), "5 query heads over 2"),
    (dict(q=torch.zeros(3, 0, 64, dtype=BF16)), "0 query heads"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), "block_table must be"),
    (dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), "not overlap"),
    (dict(cu_new=i32(0, 3)), "need 3 cu_new"),
    (dict(kv_lens=i32(5)), "2 kv_lens"),
    (dict(kv_lens=torch.zeros(2, dtype=torch.int64)), "kv_lens must be"),
    (dict(window=-1), "window=-1"),
    (dict(sinks=-1), "sinks=-1"),
    (dict(window=2 ** 32), "2\\^31"),
    (dict(sinks=2 ** 31), "2\\^31"),
    (dict(max_new=0), "max_new=0"),
    (dict(v_scale=torch.ones(1)), "float8 cache only"),
    (dict(FP8_CACHES, v_scale=torch.ones(3)), "v_scale must be"),
    (dict(out=torch.zeros(3, 4, 64)), "`out` must be"),
    (dict(out=torch.zeros(3, 4, 128, dtype=BF16)[..., ::2]), "`out` must be"),
    (dict(out=torch.zeros(2, 4, 64, dtype=BF16)), "`out` must be"),
    (dict(q=SAME, out=SAME), "overlap"),
    ({}, "CUDA device"),
]


@pytest.mark.parametrize("kw,match", SLOTS)
def test_slots_refusals(kw, match):
    from fp4_fp8_for_torch_mps import fp8_mps_native as nat
    with pytest.raises(RuntimeError, match=match):
        nat.paged_slots(**slots_args(**kw))


@pytest.mark.parametrize("kw,match", WRITE)
def test_write_refusals(kw, match):
    from fp4_fp8_for_torch_mps import fp8_mps_native as nat
    with pytest.raises(RuntimeError, match=match):
        nat.rope_write_paged(**write_args(**kw))


@pytest.mark.parametrize("kw,match", ATTENTION)
def test_attention_refusals(kw, match):
    from fp4_fp8_for_torch_mps import fp8_mps_native as nat
    with pytest.raises(RuntimeError, match=match):
        nat.paged_attention(**attention_args(**kw))


def c_call(name, base, **kw):
    """The C entry with arguments that pass its checks up to the device, but for `kw`: (status, message)."""
    from fp4_fp8_for_torch_mps import _lib
    a = dict(base, **kw)
    rc = getattr(_lib.lib(), name)(*a.values())
    return rc, _lib.lib().fp8b200_last_error().decode()


P = 4096  # an aligned address that no check reads
C_SLOTS = dict(cached=P, new=P, requests=2, table=P, table_ld=4, cols=4, free=P, n_free=2, head=None, page=16, tokens=2, cu=P,
               kv=P, pos=P, slots=P, head_out=P, stream=None)
C_WRITE = dict(qkv=P, dt=1, tokens=3, ld=512, nq=4, nkv=2, hd=64, cos=P, sin=P, rows=10, pos=P, slots=P, q=P, k=P, v=P, cdt=1,
               pages=4, page=16, sp=2048, ss=128, sh=64, ks=None, kst=0, vs=None, vst=0, stream=None)
C_ATT = dict(q=P, dt=1, qt=256, qh=64, tokens=3, hq=4, hk=2, hd=64, k=P, v=P, cdt=1, pages=4, page=16, sp=2048, ss=128, sh=64,
             table=P, ld=4, cols=4, cu=P, kv=P, requests=2, scale=0.125, ks=None, kst=0, vs=None, vst=0, window=0, sinks=0,
             max_new=0, out=P, ot=256, oh=64, rest=0, ws=P, wsb=1 << 40, stream=None)


@pytest.mark.parametrize("name,base,kw,match", [
    ("fp8b200_paged_slots", C_SLOTS, dict(requests=-1), "negative"),
    ("fp8b200_paged_slots", C_SLOTS, dict(requests=16385), "at most"),
    ("fp8b200_paged_slots", C_SLOTS, dict(page=0), "page_size"),
    ("fp8b200_paged_slots", C_SLOTS, dict(tokens=2 ** 31), "2\\^31"),
    ("fp8b200_paged_slots", C_SLOTS, dict(table_ld=3), "overlap"),
    ("fp8b200_paged_slots", C_SLOTS, dict(slots=None), "null"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(dt=0), "bf16 or f16"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(cdt=2), "qkv's type"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(hd=24), "head_dim"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(ld=504), "row stride"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(ld=516), "row stride"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(pages=2 ** 30, page=16), "slots"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(sh=60), "strides"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(qkv=P + 2), "aligned"),
    ("fp8b200_rope_write_paged", C_WRITE, dict(cos=None), "null"),
    ("fp8b200_paged_attention", C_ATT, dict(dt=3), "bf16 or f16"),
    ("fp8b200_paged_attention", C_ATT, dict(cdt=2), "q's type"),
    ("fp8b200_paged_attention", C_ATT, dict(hq=5), "heads over"),
    ("fp8b200_paged_attention", C_ATT, dict(hd=272), "head_dim"),
    ("fp8b200_paged_attention", C_ATT, dict(hd=40), "head_dim"),
    ("fp8b200_paged_attention", C_ATT, dict(page=0), "page_size"),
    ("fp8b200_paged_attention", C_ATT, dict(tokens=2 ** 30), "2\\^31"),
    ("fp8b200_paged_attention", C_ATT, dict(window=-1), "window"),
    ("fp8b200_paged_attention", C_ATT, dict(qh=60), "strides"),
    ("fp8b200_paged_attention", C_ATT, dict(cdt=3, ss=120), "16 bytes"),
    ("fp8b200_paged_attention", C_ATT, dict(ld=2), "overlap"),
    ("fp8b200_paged_attention", C_ATT, dict(k=P + 8), "aligned"),
    ("fp8b200_paged_attention", C_ATT, dict(ws=None), "null"),
])
def test_c_refusals(name, base, kw, match):
    import re
    rc, msg = c_call(name, base, **kw)
    assert rc == -1 and re.search(match, msg), (rc, msg)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on the addresses of the refusal tests")
@pytest.mark.parametrize("name,base", [("fp8b200_paged_slots", C_SLOTS), ("fp8b200_rope_write_paged", C_WRITE),
                                       ("fp8b200_paged_attention", C_ATT)])
def test_c_without_device(name, base):
    assert c_call(name, base)[0] == -3
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_fakes():
    """Shapes and types of the custom ops on meta tensors."""
    import fp4_fp8_for_torch_mps  # noqa: F401
    m = lambda d: {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in d.items()}  # noqa: E731
    cu, kv, pos, slots, head = torch.ops.fp8_mps.paged_slots(**m(slots_args(num_tokens=5)))
    assert (cu.shape, kv.shape, pos.shape, slots.shape, head.shape) == ((3,), (2,), (5,), (5,), (1,))
    assert slots.dtype == torch.int64 and {t.dtype for t in (cu, kv, pos, head)} == {torch.int32}
    q = torch.ops.fp8_mps.rope_write_paged(**m(write_args()))
    assert q.shape == (3, 4, 64) and q.dtype == BF16
    assert torch.ops.fp8_mps.paged_attention(**m(attention_args())).shape == (3, 4, 64)


def test_cache_release_on_the_host():
    """Which pages are free after requests end, in any order, and the refusals."""
    from fp4_fp8_for_torch_mps import paged
    c = paged.PagedKVCache(2, 6, 4, 1, 16, 3, 16, E4M3, "cpu")
    assert len(c.k) == 2 and c.k[0].shape == (6, 4, 1, 16) and c.k[1].stride() == c.v[1].stride()
    c.block_table[0, :2], c.block_table[2, :3] = i32(0, 1), i32(2, 3, 4)     # as two prompts would leave it
    c.free_head.fill_(5)
    c.lens.copy_(i32(7, 0, 12))
    c.release(0)
    assert c.free_pages[3:].tolist() == [5, 0, 1] and int(c.free_head) == 3 and c.lens.tolist() == [0, 0, 12]
    c.release(1)                                                             # holds nothing
    c.release(2)
    assert sorted(c.free_pages.tolist()) == list(range(6)) and int(c.free_head) == 0
    assert int((c.block_table >= 0).sum()) == 0
    c.block_table[1, 0] = 3
    with pytest.raises(RuntimeError, match="0 are taken"):
        c.release(1)
    for bad in (dict(layers=0), dict(requests=16385), dict(dtype=torch.float32)):
        a = dict(layers=1, pages=2, page_size=4, kv_heads=1, head_dim=16, requests=1, max_len=4, dtype=BF16, device="cpu")
        with pytest.raises(RuntimeError, match="PagedKVCache"):
            paged.PagedKVCache(**{**a, **bad})
