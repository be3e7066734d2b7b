"""The FP8 Llama-shaped stack over a paged cache against the same layers in
float32 from the dequantised weights, with the bound of the dense path's test
(tests/test_llama_gpu.py): the error of a layer's update relative to the
update stays below 10 %. A float8 cache adds one e4m3 rounding (half a step
2^-4, 2.6 % of a value in the root mean square) of k and v to the four of the
activations that the bound covers."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def float32_layer(W, layer, x, cos, sin, window=0, sinks=0):
    """One layer over one request's tokens from position 0, in float32."""
    c = W.LLAMA
    h, hd, nkv, nh = c["hidden"], c["head_dim"], c["kv_heads"], c["heads"]
    t = x.shape[0]
    deq = lambda w, s: w.float() * s.float().reshape(-1, 1)  # noqa: E731
    r = F.rms_norm(x, (h,), None, c["eps"])
    q, k, v = (r @ deq(layer.w_qkv, layer.s_qkv).t()).split([h, nkv * hd, nkv * hd], dim=1)
    cf, sf = cos[:t, None], sin[:t, None]
    q, k = W._rope(q.view(t, nh, hd), cf, sf).transpose(0, 1), W._rope(k.view(t, nkv, hd), cf, sf).transpose(0, 1)
    v = v.view(t, nkv, hd).transpose(0, 1)
    i = torch.arange(t, device=x.device)
    seen = i[None] <= i[:, None]
    if window:
        seen &= (i[:, None] - i[None] < window) | (i[None] < sinks)
    s = q @ k.repeat_interleave(nh // nkv, 0).transpose(1, 2) * hd ** -0.5
    a = s.masked_fill(~seen, float("-inf")).softmax(-1) @ v.repeat_interleave(nh // nkv, 0)
    x1 = x + a.transpose(0, 1).reshape(t, h) @ deq(layer.w_o, layer.s_o).t()
    g, u = (F.rms_norm(x1, (h,), None, c["eps"]) @ deq(layer.w_gu, layer.s_gu).t()).chunk(2, dim=1)
    return x1 + (F.silu(g) * u) @ deq(layer.w_d, layer.s_d).t()


@pytest.mark.parametrize("dtype,window,sinks", [(torch.bfloat16, 0, 0), (torch.float8_e4m3fn, 0, 0), (torch.float8_e4m3fn, 64, 4)])
def test_prompts_and_decoded_tokens(device, dtype, window, sinks):
    """Two requests: prompts of 150 and 9 tokens, then chunks and single
    tokens, padded rows among them. Every row against the float32 layer."""
    from fp4_fp8_for_torch_mps import _lib, workloads as W
    stack = W.Fp8LlamaStack(torch.device("cuda"), layers=1, seed=0)
    cos, sin = W.paged_rope_tables(256, "cuda")
    scale = torch.full((1,), 0.05, device="cuda") if dtype != torch.bfloat16 else None
    cache = stack.paged_cache(2, 256, 40, page_size=16, dtype=dtype, k_scale=scale, v_scale=scale)
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(220, W.LLAMA["hidden"], generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    got, done = [[], []], [0, 0]
    for new in ((150, 9), (1, 70), (1, 1), (1, 1), (40, 1)):
        rows = torch.cat([x[r][done[r]:done[r] + new[r]] for r in range(2)] + [torch.zeros_like(x[0][:3])])
        y = stack.forward_paged(rows, cache, torch.tensor(new, dtype=torch.int32, device="cuda"), cos, sin, max_new=max(new),
                                window=window, sinks=sinks)
        assert bool(torch.isfinite(y).all())
        for r, part in enumerate(y[:sum(new)].split(list(new))):
            got[r].append(part)
            done[r] += new[r]
    assert cache.lens.tolist() == done
    for r in range(2):
        xf = x[r][:done[r]].float()
        ref = float32_layer(W, stack.layers[0], xf, cos, sin, window, sinks)
        rel = ((torch.cat(got[r]).float() - ref).norm() / (ref - xf).norm()).item()
        assert rel < 0.10, (r, rel)
    assert _lib.paged_status() == 0


def test_captured_decode_steps(device):
    """A decode step of two layers, bookkeeping included, captured once and
    replayed for several tokens gives the eager steps' bits."""
    from fp4_fp8_for_torch_mps import workloads as W
    stack = W.Fp8LlamaStack(torch.device("cuda"), layers=2, seed=0)
    cos, sin = W.paged_rope_tables(256, "cuda")
    g = torch.Generator().manual_seed(2)
    prompt = torch.randn(45, W.LLAMA["hidden"], generator=g).to(torch.bfloat16).cuda()
    tokens = torch.randn(20, 3, W.LLAMA["hidden"], generator=g).to(torch.bfloat16).cuda()
    first = torch.tensor([30, 0, 15], dtype=torch.int32, device="cuda")
    one = torch.ones(3, dtype=torch.int32, device="cuda")

    def new_cache():
        c = stack.paged_cache(3, 256, 30, page_size=16)
        stack.forward_paged(prompt, c, first, cos, sin)
        return c
    eager_cache, graph_cache = new_cache(), new_cache()
    eager = [stack.forward_paged(t, eager_cache, one, cos, sin, max_new=1).clone() for t in tokens]
    x = tokens[0].clone()
    keep = [t.clone() for t in (graph_cache.lens, graph_cache.free_head, graph_cache.block_table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = stack.forward_paged(x, graph_cache, one, cos, sin, max_new=1)
    for t, old in zip((graph_cache.lens, graph_cache.free_head, graph_cache.block_table), keep):
        assert torch.equal(t, old)                        # capturing ran nothing
    for t, want in zip(tokens, eager):
        x.copy_(t)
        graph.replay()
        assert torch.equal(y, want)
    assert graph_cache.lens.tolist() == eager_cache.lens.tolist() == [50, 20, 35]
    assert torch.equal(graph_cache.block_table, eager_cache.block_table)


def test_released_pages_are_used_again(device):
    from fp4_fp8_for_torch_mps import paged
    c = paged.PagedKVCache(1, 6, 4, 1, 16, 3, 16, torch.bfloat16, "cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c.step(i32(9, 4, 5), 18)
    assert int(c.free_head) == 6 and c.block_table[:, :3].tolist() == [[0, 1, 2], [3, -1, -1], [4, 5, -1]]
    c.release(0)
    assert int(c.free_head) == 3 and c.lens.tolist() == [0, 4, 5]
    s = c.step(i32(1, 1, 4), 6)
    assert c.block_table[:, :3].tolist() == [[0, -1, -1], [3, 1, -1], [4, 5, 2]]
    assert s.slots.tolist() == [0, 4, 21, 22, 23, 8]
