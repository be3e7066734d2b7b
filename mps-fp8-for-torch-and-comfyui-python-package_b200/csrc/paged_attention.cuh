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
  // the tensor-memory kernel: its waits run out that long after the last progress; test hook: no tile of K and V arrives
  uint64_t wait_ns;
  int no_tiles;
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

__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
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

// ---- rows whose product came out not finite
//
// A hidden key's weight is 0, but 0 times its V's infinity or NaN is NaN and
// takes a whole output with it. odd_rows puts such rows right at a segment's
// end, a warp's rows at a time, in two steps:
//   1. one pass over V alone finds the keys that hold infinities or NaN. What a
//      row sees of them is its result in that dim, whatever the other keys add
//      (weights of visible keys are above 0): NaN, or both infinities: NaN; else
//      the infinity. Rows whose every odd dim is settled so need nothing more.
//   2. the others (a hidden key's value in the way) are recomputed from their
//      visible keys alone, CAREFUL rows at a time (careful_rows). Those are at
//      most the rows whose tiles hold the key and that do not see it.
// 2048 rows of 32 / 8 heads of 128 over 16049 keys in bf16 (0.50 ms): 1.7 ms with
// a NaN that all rows of one head see, 2.9 ms with one in each head; 78 ms with
// one in the last key, hidden from 252 rows of a head.
constexpr int CAREFUL = 4;

// An infinity or NaN among the 16 bytes of cached values.
template <bool F16, int KV>
__device__ __forceinline__ bool odd16(const uint4 &v) {
  constexpr bool BYTES = KV == FP8B200_E4M3 || KV == FP8B200_E5M2;
  constexpr uint32_t ONES = KV == FP8B200_E4M3 ? 0x7F7F7F7Fu : KV == FP8B200_E5M2 ? 0x7C7C7C7Cu : F16 ? 0x7C007C00u : 0x7F807F80u;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t hit = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) hit |= BYTES ? __vcmpeq4(w[i] & ONES, ONES) : __vcmpeq2(w[i] & ONES, ONES);
  return hit != 0;
}
// 16 values from element `elem` (at 16 bytes' alignment) as floats.
template <bool F16, int KV>
__device__ __forceinline__ void load16(const void *base, int64_t elem, float (&f)[16]) {
  if constexpr (KV == FP8B200_E4M3 || KV == FP8B200_E5M2) {
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(base) + elem));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t h = fp8x2_to_f16x2<KV>((w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
      f[2 * i] = to_f32<true>((uint16_t)h);
      f[2 * i + 1] = to_f32<true>((uint16_t)(h >> 16));
    }
  } else {
    const uint4 *at = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + elem);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const uint4 v = __ldg(at + k);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f[8 * k + 2 * i] = to_f32<F16>((uint16_t)w[i]);
        f[8 * k + 2 * i + 1] = to_f32<F16>((uint16_t)(w[i] >> 16));
      }
    }
  }
}

// A segment: request r with rows from `start` of q and positions from `first`,
// key/value head h, rows of the request from row0 on, key tiles [t0, t1).
template <int BN>
struct SegmentRows {
  int r, start, first, h, row0;
  Tiles<BN> tiles;
  int t0, t1;
};

// Rows `row` of a segment (-1: none) over their visible keys, 32 keys at a
// time: a lane has a key's scores, then dims lane, lane + 32, ... of the outputs.
// Gives the maxima (log2 units), the sums, and the unnormalised outputs. The
// `deadline` of the other roles' waits, if any, moves on at every tile.
template <bool F16, int KV, int DMAX, int BN>
__device__ __noinline__ void careful_rows(const AttnParams &params, const SegmentRows<BN> &segment, const int (&row)[CAREFUL],
                                          volatile uint64_t *deadline, float (&m)[CAREFUL], float (&l)[CAREFUL],
                                          float (&o)[CAREFUL][DMAX / 32]) {
  const AttnParams p = params;                            // in registers
  const SegmentRows<BN> sg = segment;
  constexpr int N = DMAX / 32, AT = N > 4 ? 4 : 8;        // keys whose V is in flight
  const int lane = threadIdx.x & 31;
  const float s2 = p.scale_log2 * (p.ks ? __ldg(p.ks + p.ks_step * sg.h) : 1.0f);
  int64_t q_at[CAREFUL];
  int pos[CAREFUL];
  uint32_t dead = 0;                                      // rows with a score of NaN or +inf: every output is NaN
#pragma unroll
  for (int x = 0; x < CAREFUL; x++) {
    const int qr = sg.row0 + max(row[x], 0), tok = qr / p.group;
    q_at[x] = (int64_t)(sg.start + tok) * p.q_tok + (int64_t)(sg.h * p.group + qr - tok * p.group) * p.q_head;
    pos[x] = row[x] < 0 ? -1 : sg.first + tok;
    m[x] = -INFINITY;
    l[x] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) o[x][i] = 0.0f;
  }
#pragma unroll 1
  for (int t = sg.t0; t < sg.t1; t++) {
    if (deadline && lane == 0) *deadline = now_ns() + p.wait_ns;
#pragma unroll 1
    for (int j0 = 0; j0 < BN; j0 += 32) {
      const int j = sg.tiles.at(t) * BN + j0 + lane;
      bool see[CAREFUL], any = false;
#pragma unroll
      for (int x = 0; x < CAREFUL; x++) any |= see[x] = visible(p, j, pos[x]);
      const int64_t off = any ? slot_offset(p, sg.r, j) : -1, e = off + (int64_t)sg.h * p.s_head;
      const uint32_t there = __ballot_sync(~0u, off >= 0);
      if (!there) continue;
      float s[CAREFUL] = {};
      if (off >= 0) {
#pragma unroll 2
        for (int d = 0; d < p.d; d += 16) {
          float k[16];
          load16<F16, KV>(p.k, e + d, k);
#pragma unroll
          for (int x = 0; x < CAREFUL; x++) {
            float y[16];
            load16<F16, F16 ? FP8B200_F16 : FP8B200_BF16>(p.q, q_at[x] + d, y);
#pragma unroll
            for (int i = 0; i < 16; i++) s[x] = fmaf(y[i], k[i], s[x]);
          }
        }
      }
      float w[CAREFUL];
      uint32_t sees[CAREFUL];
#pragma unroll
      for (int x = 0; x < CAREFUL; x++) {
        see[x] = see[x] && off >= 0;
        sees[x] = __ballot_sync(~0u, see[x]);
        s[x] = see[x] ? s[x] * s2 : -INFINITY;
        if (__any_sync(~0u, !(s[x] < INFINITY))) dead |= 1u << x;
        float top = fmaxf(m[x], s[x]);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const float base = top == -INFINITY ? 0.0f : top, keep = exp2f(m[x] - base);
        w[x] = see[x] ? exp2f(s[x] - base) : 0.0f;
        m[x] = top;
        float sum = w[x];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        l[x] = l[x] * keep + sum;
#pragma unroll
        for (int i = 0; i < N; i++) o[x][i] *= keep;
      }
#pragma unroll 1
      for (int k0 = 0; k0 < 32; k0 += AT) {
        if (!((there >> k0) & ((1u << AT) - 1u))) continue;
        float v[AT][N];
#pragma unroll
        for (int k = 0; k < AT; k++) {
          const int64_t ek = __shfl_sync(~0u, e, k0 + k);
#pragma unroll
          for (int i = 0; i < N; i++) {
            v[k][i] = 0.0f;
            if (((there >> (k0 + k)) & 1u) && lane + 32 * i < p.d) v[k][i] = cache_value<F16, KV>(p.v, ek + lane + 32 * i);
          }
        }
#pragma unroll
        for (int k = 0; k < AT; k++)
#pragma unroll
          for (int x = 0; x < CAREFUL; x++) {
            const float wk = __shfl_sync(~0u, w[x], k0 + k);
            if ((sees[x] >> (k0 + k)) & 1u)               // a value that the row does not see is not touched
#pragma unroll
              for (int i = 0; i < N; i++) o[x][i] = fmaf(wk, v[k][i], o[x][i]);
          }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < CAREFUL; x++)
    if ((dead >> x) & 1u) {
      l[x] = u2f(0x7FC00000u);
#pragma unroll
      for (int i = 0; i < N; i++) o[x][i] = u2f(0x7FC00000u);
    }
}

// The rows of a warp's lanes, `row` of the segment: `odd` for the rows to be
// looked at, l their sum of weights. The rows' results lie in p.out (whole) or
// in the segment's part of mr rows; other lanes' stores of them are ordered
// before the call.
template <bool F16, int KV, int DP, int BN>
__device__ __noinline__ void odd_rows(const AttnParams &params, const SegmentRows<BN> &segment, int row, bool odd, float l, bool whole,
                                      float *part, int mr, volatile uint64_t *deadline) {
  const AttnParams p = params;                            // in registers
  const SegmentRows<BN> sg = segment;
  constexpr int N = DP / 32, AT = 8;
  constexpr int ESZ = KV == FP8B200_E4M3 || KV == FP8B200_E5M2 ? 1 : 2;
  const int lane = threadIdx.x & 31;
  odd = odd && l == l;                                    // a NaN among the visible scores: so is every output, and stays it
  const uint32_t rows = __ballot_sync(~0u, odd);
  if (!rows) return;
  const int tok = (sg.row0 + row) / p.group, pos = odd ? sg.first + tok : -1;
  int last = pos;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) last = max(last, __shfl_xor_sync(~0u, last, d));
  // a row whose weights are all 0 saw nothing, or scores of -inf alone: value by value
  uint32_t redo = __ballot_sync(~0u, odd && l == 0.0f);
  // bit q: in the row of lane q, a visible key holds NaN, +inf, -inf in this lane's dim i
  uint32_t nan[N], up[N], down[N];
#pragma unroll
  for (int i = 0; i < N; i++) nan[i] = up[i] = down[i] = 0u;
  const int upr = p.d * ESZ / 16;                         // 16-byte units of a key's row
  const int key_first = lane / upr, cu_first = lane % upr, key_step = 32 / upr, cu_step = 32 % upr;
  bool done = false;
#pragma unroll 1
  for (int t = sg.t0; t < sg.t1 && !done; t++) {
    if (deadline && lane == 0) *deadline = now_ns() + p.wait_ns;
#pragma unroll 1
    for (int j0 = 0; j0 < BN && !done; j0 += 32) {
      const int j = sg.tiles.at(t) * BN + j0 + lane;
      const int64_t off = j <= last ? slot_offset(p, sg.r, j) : -1, e = off + (int64_t)sg.h * p.s_head;
      const uint32_t there = __ballot_sync(~0u, off >= 0);
      if (!there) continue;
      // units lane, lane + 32, ... of the 32 keys' rows
      uint32_t found = 0;
      int key = key_first, cu = cu_first;
#pragma unroll 1
      for (int k0 = 0; k0 < upr; k0 += AT) {
        uint4 v[AT];
        int keys[AT];
#pragma unroll
        for (int k = 0; k < AT; k++) {
          keys[k] = key;
          const int64_t ek = __shfl_sync(~0u, e, key & 31);
          v[k] = make_uint4(0, 0, 0, 0);
          if (k0 + k < upr && ((there >> (key & 31)) & 1u)) v[k] = __ldg(reinterpret_cast<const uint4 *>(p.v + ek * ESZ) + cu);
          key += key_step;
          cu += cu_step;
          if (cu >= upr) cu -= upr, key++;
        }
#pragma unroll
        for (int k = 0; k < AT; k++)
          if (odd16<F16, KV>(v[k])) found |= 1u << (keys[k] & 31);
      }
      found = __reduce_or_sync(~0u, found);
      for (; found; found &= found - 1) {
        const int src = __ffs(found) - 1, jk = __shfl_sync(~0u, j, src);
        const int64_t ek = __shfl_sync(~0u, e, src);
        const uint32_t see = __ballot_sync(~0u, odd && visible(p, jk, pos));
        if (!see) continue;
        bool k_odd = false;                               // then the score may be -inf and the weight 0: value by value
        float v[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
          v[i] = 0.0f;
          if (lane + 32 * i < p.d) {
            v[i] = cache_value<F16, KV>(p.v, ek + lane + 32 * i);
            k_odd |= !(fabsf(cache_value<F16, KV>(p.k, ek + lane + 32 * i)) < INFINITY);
          }
        }
        if (__any_sync(~0u, k_odd)) {
          redo |= see;
          continue;
        }
        bool all = true;                                  // NaN in every dim of every row: nothing changes that
#pragma unroll
        for (int i = 0; i < N; i++) {
          if (v[i] != v[i]) nan[i] |= see;
          else if (v[i] == INFINITY) up[i] |= see;
          else if (v[i] == -INFINITY) down[i] |= see;
          all &= lane + 32 * i >= p.d || (nan[i] & rows) == rows;
        }
        done = __all_sync(~0u, all);
        if (done) break;
      }
    }
  }
  const float vs = ESZ == 1 && p.vs ? __ldg(p.vs + p.vs_step * sg.h) : 1.0f;
  auto out_at = [&](int row_s) {
    const int qr = sg.row0 + row_s, t = qr / p.group;
    return p.out + (int64_t)(sg.start + t) * p.o_tok + (int64_t)(sg.h * p.group + qr - t * p.group) * p.o_head;
  };
  // The row of lane src: its dims that are settled get their value; true if it has others that are not finite.
  auto settled = [&](int src, int i) { return !((redo >> src) & 1u) && (((nan[i] | up[i] | down[i]) >> src) & 1u); };
  auto value = [&](int src, int i) {
    const bool n = (nan[i] >> src) & 1u, u = (up[i] >> src) & 1u, b = (down[i] >> src) & 1u;
    return n || (u && b) ? u2f(0x7FC00000u) : u ? INFINITY : -INFINITY;
  };
  uint32_t again = 0;
#pragma unroll 1
  for (uint32_t rest = rows; rest; rest &= rest - 1) {
    const int src = __ffs(rest) - 1, row_s = __shfl_sync(~0u, row, src);
    const float l_s = __shfl_sync(~0u, l, src), inv = l_s == 0.0f ? 0.0f : vs / l_s;
    uint16_t *os = out_at(row_s);
    bool left = false;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int d = lane + 32 * i;
      if (d >= p.d || fabsf(whole ? to_f32<F16>(os[d]) : part[row_s * DP + d]) < INFINITY) continue;
      if (!settled(src, i)) left = true;
      else if (whole) os[d] = (uint16_t)pack2<F16>(value(src, i) * inv, 0.0f);
      else part[row_s * DP + d] = value(src, i);
    }
    if (__any_sync(~0u, left)) again |= 1u << src;
  }
#pragma unroll 1
  while (again) {
    int src[CAREFUL], row_s[CAREFUL];
    float m[CAREFUL], ls[CAREFUL], o[CAREFUL][N];
#pragma unroll
    for (int x = 0; x < CAREFUL; x++) {
      src[x] = __ffs(again) - 1;
      row_s[x] = src[x] < 0 ? -1 : __shfl_sync(~0u, row, src[x]);
      again &= again - 1;
    }
    careful_rows<F16, KV, DP, BN>(params, segment, row_s, deadline, m, ls, o);
#pragma unroll
    for (int x = 0; x < CAREFUL; x++) {
      if (src[x] < 0) continue;
      const float inv = ls[x] == 0.0f ? 0.0f : vs / ls[x];
      uint16_t *os = out_at(row_s[x]);
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int d = lane + 32 * i;
        const float y = settled(src[x], i) ? value(src[x], i) : o[x][i];
        if (!whole) part[row_s[x] * DP + d] = y;
        else if (d < p.d) os[d] = (uint16_t)pack2<F16>(y * inv, 0.0f);
      }
      if (!whole && lane == 0) {
        part[mr * DP + row_s[x]] = m[x];
        part[mr * DP + mr + row_s[x]] = ls[x];
      }
    }
  }
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
