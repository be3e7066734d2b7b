// Shared pieces of the paged attention kernels.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace fp8b200 {
namespace paged {

// A segment that was cut, for the merge: written by the block that begins it.
struct alignas(16) PartDesc {
  int rows;                   // of the row tile; 0: this block began no such segment
  int row0, h;                // the tile's first row in its request, the key/value head
  int start;                  // the request's first row of q
  int parts, step;            // the parts: the second of this block, the first of the blocks step, 2 * step, ... behind it
};
static_assert(sizeof(PartDesc) == 32, "two 16-byte words");

// One call. Element strides throughout; the two caches share their strides.
struct AttnParams {
  const uint16_t *q;
  int64_t q_tok, q_head;
  uint16_t *out;
  int64_t o_tok, o_head;
  const uint8_t *k, *v;
  int64_t s_page, s_slot, s_head;
  int64_t pages;
  int page;
  const int32_t *table;
  int64_t table_ld;
  int table_cols;
  const int32_t *cu, *kv;
  int requests;
  int tokens;                 // rows of q
  int hq, hk, group, d;
  float scale_log2;           // softmax scale times log2(e)
  const float *ks, *vs;
  int ks_step, vs_step;       // 0: one scale, 1: one per head
  int window, sinks;          // window 0: none
  int zero_rest;              // zero the rows of out that belong to no request
  int rows_over, rows_upto;   // requests whose query rows (tokens x group) lie in (rows_over, rows_upto] are taken
  // split segments: partial results and which block continues what
  float *part;
  PartDesc *desc;
  int blocks;                 // for the merge: how many descriptors there are
  int line_heads;             // key/value heads that a line of units holds: all, or one (a line a head)
};

// The new tokens of request r: rows [start, start + n) of q, the last at
// position kv - 1. Offsets outside q's rows are clipped, so no row is read or
// written behind it.
struct Request {
  int start, n, first;        // first: position of row `start`, negative where kv < n
};
__device__ __forceinline__ Request load_request(const AttnParams &p, int r) {
  Request q;
  const int a = min(max(__ldg(p.cu + r), 0), p.tokens), b = min(max(__ldg(p.cu + r + 1), a), p.tokens);
  const int kv = max(__ldg(p.kv + r), 0);
  q.start = a;
  q.n = b - a;
  q.first = kv - q.n;
  return q;
}
__device__ __forceinline__ bool takes(const AttnParams &p, int n) {
  const int64_t rows = (int64_t)n * p.group;
  return rows > p.rows_over && rows <= p.rows_upto;
}

// Zeros to the rows of out that no request has (a padded batch), by blocks
// [block, blocks) of the launch.
__device__ __forceinline__ void zero_rest(const AttnParams &p, int block, int blocks) {
  const int a = min(max(__ldg(p.cu), 0), p.tokens);
  const int b = p.requests > 0 ? min(max(__ldg(p.cu + p.requests), a), p.tokens) : a;
  const int rest = a + p.tokens - b, units = p.hq * (p.d / 8);
  for (int i = block; i < rest; i += blocks) {
    const int row = i < a ? i : b + i - a;
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      const int head = u / (p.d / 8), c = u - head * (p.d / 8);
      *reinterpret_cast<uint4 *>(p.out + (int64_t)row * p.o_tok + (int64_t)head * p.o_head + c * 8) = make_uint4(0, 0, 0, 0);
    }
  }
}

// Key tiles that any query at positions [lo, hi] can see: the tiles of the
// sinks, [0, sinks), and those of the windows, [from, to).
template <int BN>
struct Tiles {
  int sinks, from, to;
  __device__ __forceinline__ int count() const { return sinks + to - from; }
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : from + i - sinks; }
};
template <int BN>
__device__ __forceinline__ Tiles<BN> visible_tiles(const AttnParams &p, int lo, int hi) {
  Tiles<BN> t;
  // keys behind the last table column have no page
  const int64_t cap = (int64_t)p.table_cols * p.page;
  const int end = hi < 0 ? 0 : (int)min((int64_t)hi + 1, cap);
  t.to = (int)(((int64_t)end + BN - 1) / BN);
  t.from = 0;
  t.sinks = 0;
  if (p.window > 0 && end > 0) {
    const int64_t first = (int64_t)max(lo, 0) - p.window + 1;
    if (first > 0) t.from = min((int)(first / BN), t.to);
    t.sinks = (int)min(((int64_t)p.sinks + BN - 1) / BN, (int64_t)t.from);
  }
  return t;
}
__device__ __forceinline__ bool visible(const AttnParams &p, int key, int pos) {
  return key <= pos && (p.window <= 0 || pos - key < p.window || key < p.sinks);
}

// Element offset of key j's slot in the pool, -1 where it has no page: a
// table entry outside the pool hides its keys.
__device__ __forceinline__ int64_t slot_offset(const AttnParams &p, int r, int j) {
  const uint32_t col = (uint32_t)j / (uint32_t)p.page;
  if (col >= (uint32_t)p.table_cols) return -1;
  const int page = __ldg(p.table + (int64_t)r * p.table_ld + col);
  if (page < 0 || page >= p.pages) return -1;
  return (int64_t)page * p.s_page + (int64_t)((uint32_t)j - col * (uint32_t)p.page) * p.s_slot;
}

__device__ __forceinline__ uint32_t saddr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ float to_f32(uint16_t v) {
  if constexpr (F16) return __half2float(__ushort_as_half(v));
  else return u2f((uint32_t)v << 16);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}
// Two float8 codes (low 16 bits) to a half pair: exact, infinities and NaN kept.
template <int KV>
__device__ __forceinline__ uint32_t fp8x2_to_f16x2(uint32_t two) {
  uint32_t h;
  const uint16_t in = (uint16_t)two;
  if constexpr (KV == FP8B200_E4M3) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(in));
  else asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(in));
  return h;
}
// One cached value as float (KV: E4M3, E5M2, or the 16-bit type).
template <bool F16, int KV>
__device__ __forceinline__ float cache_value(const uint8_t *base, int64_t elem) {
  if constexpr (KV == FP8B200_E4M3 || KV == FP8B200_E5M2)
    return __half2float(__ushort_as_half((uint16_t)fp8x2_to_f16x2<KV>(__ldg(base + elem))));
  else
    return to_f32<F16>(__ldg(reinterpret_cast<const uint16_t *>(base) + elem));
}

// The kernel for many query rows (paged_attention_tc.cu): head sizes up to
// 128, caches that a tensor map can describe, at most 16384 requests (tc_takes).
bool tc_takes(const AttnParams &p);
int64_t tc_workspace(int dp, int sms);
int launch_tc(const AttnParams &params, bool f16, int cache_dtype, int dp, int sms, uint8_t *workspace, cudaStream_t st);

// One query row over the keys of tiles [t0, t1) of `tiles`, value by value:
// the way out where a hidden key's infinity or NaN met a zero weight in a
// matrix product (0 * inf). Hidden keys are not touched here. The warp's
// lanes hold dims lane, lane + 32, ...; returns the running maximum (log2
// units) and sum, and the unnormalised output in o.
template <bool F16, int KV, int DMAX, int BN>
__device__ __noinline__ void careful_row(const AttnParams &p, int r, int tok, int head, int pos, const Tiles<BN> tiles,
                                         int t0, int t1, float &m_out, float &l_out, float (&o)[DMAX / 32]) {
  const int lane = threadIdx.x & 31;
  const int kh = head / p.group;
  const uint16_t *q = p.q + (int64_t)tok * p.q_tok + (int64_t)head * p.q_head;
  const float s2 = p.scale_log2 * (p.ks ? __ldg(p.ks + p.ks_step * kh) : 1.0f);
  float qv[DMAX / 32];
#pragma unroll
  for (int i = 0; i < DMAX / 32; i++) {
    qv[i] = lane + 32 * i < p.d ? to_f32<F16>(__ldg(q + lane + 32 * i)) : 0.0f;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t = t0; t < t1; t++) {
    const int k0 = tiles.at(t) * BN;
    for (int j = k0; j < k0 + BN; j++) {
      if (!visible(p, j, pos)) continue;
      const int64_t off = slot_offset(p, r, j);
      if (off < 0) continue;
      const int64_t e = off + (int64_t)kh * p.s_head;
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < DMAX / 32; i++)
        if (lane + 32 * i < p.d) s += qv[i] * cache_value<F16, KV>(p.k, e + lane + 32 * i);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      s *= s2;
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;
      const float keep = exp2f(m - base), w = exp2f(s - base);
      m = mn;
      l = l * keep + w;
      if (l != l) {            // a score is NaN, or +inf: so is every output
#pragma unroll
        for (int i = 0; i < DMAX / 32; i++) o[i] = l;
        m_out = m;
        l_out = l;
        return;
      }
#pragma unroll
      for (int i = 0; i < DMAX / 32; i++)
        if (lane + 32 * i < p.d) o[i] = o[i] * keep + w * cache_value<F16, KV>(p.v, e + lane + 32 * i);
    }
  }
  m_out = m;
  l_out = l;
}

// Joins the parts of the segments that were cut: block c the one that began
// in block c of the attention kernel (its second part), with the first parts
// of the blocks that went on with it, in their order. A warp a row: its lanes fetch the
// parts' bases and sums together, then the rows' values, whose loads do not
// wait for one another. MR: rows a part has room for. A block an SM (times
// the row groups) goes through the descriptors: so few fit beside the
// attention kernel's blocks and are there when it ends.
constexpr int MERGE_THREADS = 256;
template <bool F16, int DP, int MR>
__device__ __forceinline__ void merge_segment(const AttnParams &p, int64_t c, const PartDesc &d) {
  const int lane = threadIdx.x & 31;
  const int n = d.parts;
  constexpr int64_t SLOT = MR * (DP + 2);
  const float *parts = p.part + (c * 2 + 1) * SLOT;         // the first; part k > 0 is the first of block c + k * step
  auto part_at = [&](int k) { return parts + (k == 0 ? 0 : (2 * (int64_t)k * d.step - 1) * SLOT); };
  const float vs = p.vs ? __ldg(p.vs + p.vs_step * d.h) : 1.0f;
  constexpr int V = DP / 4;                                 // float4 a row
  constexpr int SPLIT = V < 32 ? 32 / V : 1, PASS = V > 32 ? V / 32 : 1;  // parts side by side, float4 a lane
  for (int row = blockIdx.y * (MERGE_THREADS / 32) + (threadIdx.x >> 5); row < d.rows; row += gridDim.y * (MERGE_THREADS / 32)) {
    // AT parts at a time: their values, bases and sums in flight together. A
    // few rows' segment has many parts, a block of 256 rows two or three.
    constexpr int AT = MR >= 128 ? 4 : 16 / PASS, N = AT / SPLIT;
    float base = -INFINITY, l = 0.0f;
    float4 acc[PASS];
#pragma unroll
    for (int q = 0; q < PASS; q++) acc[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int k0 = 0; k0 < n; k0 += AT) {
      float4 v[N][PASS];
      const int side = SPLIT > 1 ? lane / V : 0;
#pragma unroll
      for (int j = 0; j < N; j++)
#pragma unroll
        for (int q = 0; q < PASS; q++) {
          v[j][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (k0 + j * SPLIT + side < n)
            v[j][q] = *reinterpret_cast<const float4 *>(part_at(k0 + j * SPLIT + side) + row * DP + ((SPLIT > 1 ? lane % V : lane) + 32 * q) * 4);
        }
      float b = -INFINITY, bl = 0.0f;
      if (lane < AT && k0 + lane < n) {
        const float *part = part_at(k0 + lane) + MR * DP + row;
        b = part[0];
        bl = part[MR];
      }
      float nb = fmaxf(base, b);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) nb = fmaxf(nb, __shfl_xor_sync(~0u, nb, x));
      const float ref = nb == -INFINITY ? 0.0f : nb, f = ex2(base - ref), w = ex2(b - ref);
      base = nb;
      l = l * f + w * bl;
#pragma unroll
      for (int q = 0; q < PASS; q++) acc[q].x *= f, acc[q].y *= f, acc[q].z *= f, acc[q].w *= f;
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float wj = __shfl_sync(~0u, w, j * SPLIT + side);
        if (k0 + j * SPLIT + side < n)
#pragma unroll
          for (int q = 0; q < PASS; q++)
            acc[q].x += wj * v[j][q].x, acc[q].y += wj * v[j][q].y, acc[q].z += wj * v[j][q].z, acc[q].w += wj * v[j][q].w;
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(~0u, l, x);
    if constexpr (SPLIT > 1) {
#pragma unroll
      for (int x = V; x < 32; x <<= 1) {
        acc[0].x += __shfl_xor_sync(~0u, acc[0].x, x);
        acc[0].y += __shfl_xor_sync(~0u, acc[0].y, x);
        acc[0].z += __shfl_xor_sync(~0u, acc[0].z, x);
        acc[0].w += __shfl_xor_sync(~0u, acc[0].w, x);
      }
    }
    const float inv = l == 0.0f ? 0.0f : vs / l;
    const int qr = d.row0 + row, tok = d.start + qr / p.group, head = d.h * p.group + qr % p.group;
#pragma unroll
    for (int q = 0; q < PASS; q++) {
      const int d4 = ((SPLIT > 1 ? lane % V : lane) + 32 * q) * 4;
      if (lane < V && d4 < p.d) {
        uint16_t *out = p.out + (int64_t)tok * p.o_tok + (int64_t)head * p.o_head + d4;
        *reinterpret_cast<uint2 *>(out) =
            make_uint2(pack2<F16>(acc[q].x * inv, acc[q].y * inv), pack2<F16>(acc[q].z * inv, acc[q].w * inv));
      }
    }
  }
}

template <bool F16, int DP, int MR>
__global__ void __launch_bounds__(MERGE_THREADS) paged_merge_kernel(const AttnParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int c = blockIdx.x; c < p.blocks; c += gridDim.x) {
    const PartDesc d = p.desc[c];
    if (d.rows) merge_segment<F16, DP, MR>(p, c, d);
  }
}

// Launch with programmatic stream serialization: the kernel's prologue may
// overlap the previous kernel's end (griddepcontrol.wait before the first
// global access).
template <typename... Params, typename... Args>
inline void launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t st, const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}
// Dynamic shared memory above 48 KB, and all of the SM's memory as shared:
// without it an SM that has just run a kernel without shared memory may split
// its memory for one block.
int launch_attributes(const void *kernel, int smem);

}  // namespace paged
}  // namespace fp8b200
