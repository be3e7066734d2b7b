// The bookkeeping and the writing side of a paged key/value cache.
//
// A cache is a pool of pages, each `page_size` slots of kv_heads x head_dim
// values (16-bit, or float8 codes with a float32 scale per head); a request's
// tokens fill the pages its block-table row lists, in order.
//
//   slots_kernel        one step's page allotment and token placement from the
//                       request lengths, by itself or with the account that a
//                       cache keeps of its pages (HELD)
//   rope_write_kernel   rotary embedding of q and k, and k and v rounded into
//                       the cache
//
// No counterpart in the reference, which has no cache of any kind.
#include "paged_attention.cuh"

#include <algorithm>
#include <atomic>

namespace fp8b200 {
namespace paged {
namespace {

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------ slots
//
// With have_r = ceil(cached_r / P), add_r = ceil((cached_r + new_r) / P) - have_r
// and their exclusive prefix sums (cu over new, base over add):
//   table[r][have_r + i] = free[head + base_r + i]            i < add_r
//   token t of request r: position cached_r + t - cu_r, slot page * P + position % P
// Every CTA scans all requests into its own shared memory and then places its
// share of the tokens, so one launch does without a grid-wide wait. A token
// that opens a page writes that page's table entry (each new page holds one);
// entries before have_r are only read, entries from have_r on only written.
// Bound by latency: 2.4 us for one request, 4.8 us for 300 prompts with 124468
// rows (in a graph), of which the scan over 300 lengths and the launch are most.
//
// HELD is the form for a cache that keeps account of its pages from step to
// step (PagedKVCache): held_r is the number of leading columns of row r that
// have had a page, and
//   new_r  = what of the new tokens still fits into `tokens` rows
//   have_r = min(max(held_r, ceil(cached_r / P)), columns)
//   add_r  = max(min(ceil((cached_r + new_r) / P), columns) - have_r, 0)
// so a page is only taken for a column that exists and a token that is placed,
// and one that the row still holds (lengths were taken back) serves again. Every
// new column then begins with a placed token, which writes its entry. new_r
// needs the tokens' running sum, so the pages are summed in a second scan.
constexpr int SL_THREADS = 512;
constexpr int SL_MAX_REQUESTS = 16384;  // two int32 a request in shared memory

struct SlotsParams {
  const int32_t *cached, *fresh;
  int requests;
  int32_t *table;
  int64_t table_ld;
  int table_cols;
  const int32_t *free_pages;
  int64_t n_free;
  const int32_t *free_head;
  int page;
  int tokens;
  int32_t *cu, *kv, *positions;
  int64_t *slots;
  int32_t *head_out;
  const int32_t *held;                    // HELD
  int32_t *held_out;
};

__device__ __forceinline__ int pages_for(int64_t n, int page) { return (int)((n + page - 1) / page); }

// Inclusive sum over the block's threads; s has a place a warp.
__device__ __forceinline__ int block_sum(int v, int *s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += a;
  }
  if (lane == 31) s[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; w++) v += s[w];
  return v;
}

template <bool HELD>
__global__ void __launch_bounds__(SL_THREADS) slots_kernel(const SlotsParams p) {
  extern __shared__ int s_mem[];
  int *s_cu = s_mem;                      // [requests + 1] first token of each request
  int *s_base = s_mem + p.requests + 1;   // [requests] first new page of each request
  __shared__ int s_tok[SL_THREADS / 32], s_pg[SL_THREADS / 32];
  launch_dependents();
  wait_prior();
  const int tid = threadIdx.x;
  const int head = p.free_head ? *p.free_head : 0;
  // columns of request r that have a page already, of c cached and n new tokens
  auto columns = [&](int r, int c, int n, int &have) {
    have = pages_for(c, p.page);
    int need = pages_for((int64_t)c + n, p.page);
    if constexpr (HELD) {
      have = min(max(have, p.held[r]), p.table_cols);
      need = max(min(need, p.table_cols), have);
    }
    return need - have;
  };
  // each thread a contiguous run of requests; lengths below zero count as zero
  const int run = (p.requests + SL_THREADS - 1) / SL_THREADS;
  const int r0 = min(tid * run, p.requests), r1 = min(r0 + run, p.requests);
  int tok = 0, pg = 0, have;
  for (int r = r0; r < r1; r++) {
    const int c = max(p.cached[r], 0), n = max(p.fresh[r], 0);
    tok += n;
    if constexpr (!HELD) pg += columns(r, c, n, have);
  }
  int ctok = block_sum(tok, s_tok) - tok;
  auto placed = [&](int n) { return HELD ? min(n, max(p.tokens - ctok, 0)) : n; };  // of n tokens from row ctok on
  if constexpr (HELD) {
    const int first = ctok;
    for (int r = r0; r < r1; r++) {
      const int c = max(p.cached[r], 0), n = max(p.fresh[r], 0);
      pg += columns(r, c, placed(n), have);
      ctok += n;
    }
    ctok = first;
  }
  int cpg = block_sum(pg, s_pg) - pg;
  auto offset = [&]() { return HELD ? min(ctok, p.tokens) : ctok; };
  const bool writer = blockIdx.x == 0;
  for (int r = r0; r < r1; r++) {
    const int c = max(p.cached[r], 0), n = max(p.fresh[r], 0), add = columns(r, c, placed(n), have);
    s_cu[r] = offset();
    s_base[r] = cpg;
    if (writer) {
      p.cu[r] = offset();
      p.kv[r] = c + placed(n);
      if constexpr (HELD) {               // once the list is used up, columns get no page
        const int64_t left = p.n_free - ((int64_t)head + cpg);
        p.held_out[r] = have + (int)min((int64_t)add, max(left, (int64_t)0));
      }
    }
    ctok += n;
    cpg += add;
  }
  if (tid == SL_THREADS - 1) {            // its run ends with the last request
    s_cu[p.requests] = offset();
    if (writer) {
      p.cu[p.requests] = offset();
      *p.head_out = head + cpg;
    }
  }
  __syncthreads();
  const int total = s_cu[p.requests];
  for (int64_t t64 = (int64_t)blockIdx.x * SL_THREADS + tid; t64 < p.tokens; t64 += (int64_t)gridDim.x * SL_THREADS) {
    const int t = (int)t64;
    int pos = 0;
    int64_t slot = -1;
    if (t < total) {
      int lo = 0, hi = p.requests;        // the last request with cu <= t (empty ones before it are passed over)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int c = max(p.cached[lo], 0);
      pos = c + (t - s_cu[lo]);
      const int col = pos / p.page, off = pos - col * p.page;
      int have;
      columns(lo, c, 0, have);
      int page = -1;
      if (col >= 0 && col < p.table_cols) {
        int32_t *e = p.table + (int64_t)lo * p.table_ld + col;
        if (col < have) {
          page = *e;
        } else {
          const int64_t f = (int64_t)head + s_base[lo] + (col - have);
          if (f >= 0 && f < p.n_free) page = p.free_pages[f];
          if (off == 0) *e = page;
        }
      }
      if (page >= 0) slot = (int64_t)page * p.page + off;
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// ------------------------------------------------------------------ rope + write
//
// Row t of qkv holds n_q q heads, then n_kv k heads, then n_kv v heads.
//   q, k:  (a, b) -> (a cos - b sin, b cos + a sin), a and b the head's halves
//   q out: rounded to qkv's type
//   k, v:  cache[slots[t]] = round(value / scale)
// All in float32 with separately rounded products (as elementary torch
// operations compute it) and one rounding at the end; a float8 cache
// saturates at the format's largest finite value, so one outlier cannot put
// a NaN where every later query reads it. NaN stays NaN.
// A thread takes 8 + 8 values (a 16-byte unit of each half) of up to HG heads
// of one token, so the units' cos / sin are read once for HG heads. HBM bound:
// 16384 tokens of 32 / 8 / 8 heads of 128, 16-bit cache, in 66.6 us (6.06 TB/s)
// with HG = 4 and 69.2 us with 2. With few tokens the loads' latency counts,
// and more threads hide it: 16 tokens into e4m3 in 3.0 us with HG = 2 and 4.7
// with 4, 5001 tokens of 16 / 2 / 2 heads of 64 into e5m2 in 8.7 and 10.8 us (in
// a graph). So HG = 4 where that fills the GPU (RW_FULL blocks an SM) and else 2.
constexpr int RW_THREADS = 128;
constexpr int RW_FULL = 16;

struct WriteParams {
  const uint16_t *qkv;
  int64_t ld;
  int64_t tokens;
  int nq, nkv, hd;
  const float *cos_t, *sin_t;
  int64_t table_rows;
  const int32_t *positions;
  const int64_t *slots;
  uint16_t *q;
  void *k_cache, *v_cache;
  int64_t pages, s_page, s_slot, s_head;  // strides in elements, the same for both caches
  int page;
  const float *ks, *vs;
  int ks_step, vs_step;                   // 0: one scale, 1: one per head
};

template <bool F16>
__device__ __forceinline__ void unpack8(const uint4 &v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (F16) {
      const __half2 h = *reinterpret_cast<const __half2 *>(&w[i]);
      f[2 * i] = __low2float(h);
      f[2 * i + 1] = __high2float(h);
    } else {
      f[2 * i] = u2f(w[i] << 16);
      f[2 * i + 1] = u2f(w[i] & 0xFFFF0000u);
    }
  }
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (F16) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&f)[8]) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint16_t r;
    if constexpr (FMT == FP8B200_E4M3)
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
    else
      asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
    h[i] = r;
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// Eight values into the cache at element offset `off` (a multiple of 8).
template <bool F16, int CACHE>
__device__ __forceinline__ void store8(void *cache, int64_t off, float (&f)[8], float scale) {
  if constexpr (CACHE == FP8B200_E4M3 || CACHE == FP8B200_E5M2) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __fdiv_rn(f[i], scale);
    *reinterpret_cast<uint2 *>(reinterpret_cast<uint8_t *>(cache) + off) = encode8<CACHE>(f);
  } else {
    *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(cache) + off) = pack8<F16>(f);
  }
}

// CACHE: E4M3, E5M2, or anything else for qkv's own type.
template <bool F16, int CACHE, int HG>
__global__ void __launch_bounds__(RW_THREADS, HG == 4 ? 5 : 6) rope_write_kernel(const WriteParams p) {
  launch_dependents();
  wait_prior();
  const int half = p.hd / 2, units = half / 8;
  const int heads = p.nq + 2 * p.nkv, groups = (heads + HG - 1) / HG;
  const int per_token = groups * units;
  const int64_t total = p.tokens * per_token;
  for (int64_t w = (int64_t)blockIdx.x * RW_THREADS + threadIdx.x; w < total; w += (int64_t)gridDim.x * RW_THREADS) {
    const int64_t t = total < (1ll << 31) ? (int64_t)((uint32_t)w / (uint32_t)per_token) : w / per_token;
    const int in = (int)(w - t * per_token);
    const int g = in / units, u = in - g * units;
    const int h0 = g * HG;
    const uint16_t *x = p.qkv + t * p.ld + (int64_t)h0 * p.hd + u * 8;
    uint4 lo[HG], hi[HG];
#pragma unroll
    for (int i = 0; i < HG; i++)
      if (h0 + i < heads) {
        lo[i] = *reinterpret_cast<const uint4 *>(x + (int64_t)i * p.hd);
        hi[i] = *reinterpret_cast<const uint4 *>(x + (int64_t)i * p.hd + half);
      }
    float c[8], s[8];
    if (h0 < p.nq + p.nkv) {
      const int pos = p.positions[t];
      if (pos >= 0 && pos < p.table_rows) {
        const float4 *cp = reinterpret_cast<const float4 *>(p.cos_t + (int64_t)pos * half + u * 8);
        const float4 *sp = reinterpret_cast<const float4 *>(p.sin_t + (int64_t)pos * half + u * 8);
        const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
        c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
        s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
      } else {                            // a position outside the tables gives NaN, never a read behind them
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = s[i] = u2f(0x7FC00000u);
      }
    }
    int64_t slot_off = -1;                // element offset of the token's slot; -1: the token is not kept
    if (h0 + HG > p.nq) {
      const int64_t slot = p.slots[t];
      if (slot >= 0 && slot < p.pages * p.page) {
        const uint32_t page = (uint32_t)slot / (uint32_t)p.page;
        slot_off = (int64_t)page * p.s_page + (int64_t)((uint32_t)slot - page * (uint32_t)p.page) * p.s_slot + u * 8;
      }
    }
#pragma unroll
    for (int i = 0; i < HG; i++) {
      const int h = h0 + i;
      if (h >= heads) break;
      float a[8], b[8];
      unpack8<F16>(lo[i], a);
      unpack8<F16>(hi[i], b);
      if (h < p.nq + p.nkv) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float ra = __fsub_rn(__fmul_rn(a[j], c[j]), __fmul_rn(b[j], s[j]));
          b[j] = __fadd_rn(__fmul_rn(b[j], c[j]), __fmul_rn(a[j], s[j]));
          a[j] = ra;
        }
      }
      if (h < p.nq) {
        uint16_t *o = p.q + ((int64_t)t * p.nq + h) * p.hd + u * 8;
        *reinterpret_cast<uint4 *>(o) = pack8<F16>(a);
        *reinterpret_cast<uint4 *>(o + half) = pack8<F16>(b);
      } else if (slot_off >= 0) {
        const bool is_k = h < p.nq + p.nkv;
        const int kh = is_k ? h - p.nq : h - p.nq - p.nkv;
        const float *sc = is_k ? p.ks : p.vs;
        const float scale = sc ? __ldg(sc + (is_k ? p.ks_step : p.vs_step) * kh) : 1.0f;
        void *cache = is_k ? p.k_cache : p.v_cache;
        const int64_t off = slot_off + (int64_t)kh * p.s_head;
        store8<F16, CACHE>(cache, off, a, scale);
        store8<F16, CACHE>(cache, off + half, b, scale);
      }
    }
  }
}

template <bool F16, int CACHE>
auto rope_write(bool full) {
  return full ? rope_write_kernel<F16, CACHE, 4> : rope_write_kernel<F16, CACHE, 2>;
}

}  // namespace
}  // namespace paged
}  // namespace fp8b200

namespace fp8b200 {
namespace paged {
namespace {

// `what` names the entry in messages; HELD: with held and held_out.
template <bool HELD>
int launch_slots(const char *what, const int32_t *cached_lens, const int32_t *new_lens, const int32_t *held, int64_t requests,
                 int32_t *block_table, int64_t table_ld, int64_t table_cols, const int32_t *free_pages, int64_t n_free,
                 const int32_t *free_head, int64_t page_size, int64_t tokens, int32_t *cu_new, int32_t *kv_lens,
                 int32_t *positions, int64_t *slots, int32_t *held_out, int32_t *free_head_out, void *stream) {
  if (requests < 0 || table_cols < 0 || n_free < 0 || tokens < 0) return set_error(FP8B200_EINVAL, "%s: negative size", what);
  if (requests > SL_MAX_REQUESTS)
    return set_error(FP8B200_EINVAL, "%s: %lld requests, at most %d", what, (long long)requests, SL_MAX_REQUESTS);
  if (page_size < 1 || page_size > (1 << 30)) return set_error(FP8B200_EINVAL, "%s: page_size must be in 1 .. 2^30", what);
  if (tokens > INT32_MAX || table_cols > INT32_MAX)
    return set_error(FP8B200_EINVAL, "%s: more than 2^31 - 1 tokens or table columns", what);
  if (table_ld < table_cols) return set_error(FP8B200_EINVAL, "%s: block-table rows overlap", what);
  if (!cu_new || !free_head_out ||
      (requests && (!cached_lens || !new_lens || !kv_lens || (table_cols && !block_table) || (HELD && (!held || !held_out)))) ||
      (tokens && (!positions || !slots)) || (n_free && !free_pages))
    return set_error(FP8B200_EINVAL, "%s: null pointer", what);
  int dev;
  if (int rc = check_device(&dev)) return rc;
  const int smem = (int)(2 * requests + 1) * 4;
  static std::atomic<uint64_t> raised{0};
  if (smem > 47 * 1024 && !((raised.load() >> dev) & 1)) {
    if (cudaFuncSetAttribute(slots_kernel<HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * SL_MAX_REQUESTS + 1) * 4) !=
        cudaSuccess)
      return check_launch(what);
    raised.fetch_or(1ull << dev);
  }
  SlotsParams p{cached_lens, new_lens, (int)requests, block_table, table_ld, (int)table_cols, free_pages, n_free,
                free_head, (int)page_size, (int)tokens, cu_new, kv_lens, positions, slots, free_head_out, held, held_out};
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((tokens + SL_THREADS - 1) / SL_THREADS, current_sm_count()));
  launch_dependent(slots_kernel<HELD>, dim3((unsigned)grid), SL_THREADS, smem, (cudaStream_t)stream, p);
  count_launch();
  return check_launch(what);
}

}  // namespace
}  // namespace paged
}  // namespace fp8b200

extern "C" int fp8b200_paged_slots(const int32_t *cached_lens, const int32_t *new_lens, int64_t requests,
                                   int32_t *block_table, int64_t table_ld, int64_t table_cols,
                                   const int32_t *free_pages, int64_t n_free, const int32_t *free_head, int64_t page_size,
                                   int64_t tokens, int32_t *cu_new, int32_t *kv_lens, int32_t *positions,
                                   int64_t *slots, int32_t *free_head_out, void *stream) {
  return fp8b200::paged::launch_slots<false>("paged_slots", cached_lens, new_lens, nullptr, requests, block_table, table_ld,
                                             table_cols, free_pages, n_free, free_head, page_size, tokens, cu_new, kv_lens,
                                             positions, slots, nullptr, free_head_out, stream);
}

extern "C" int fp8b200_paged_step(const int32_t *cached_lens, const int32_t *new_lens, const int32_t *held, int64_t requests,
                                  int32_t *block_table, int64_t table_ld, int64_t table_cols, const int32_t *free_pages,
                                  int64_t n_free, const int32_t *free_head, int64_t page_size, int64_t tokens, int32_t *cu_new,
                                  int32_t *kv_lens, int32_t *positions, int64_t *slots, int32_t *held_out,
                                  int32_t *free_head_out, void *stream) {
  if (held && held == held_out) return fp8b200::set_error(FP8B200_EINVAL, "paged_step: held and held_out must not overlap");
  return fp8b200::paged::launch_slots<true>("paged_step", cached_lens, new_lens, held, requests, block_table, table_ld,
                                            table_cols, free_pages, n_free, free_head, page_size, tokens, cu_new, kv_lens,
                                            positions, slots, held_out, free_head_out, stream);
}

extern "C" int fp8b200_rope_write_paged(const void *qkv, int dtype, int64_t tokens, int64_t ld, int n_q_heads,
                                        int n_kv_heads, int head_dim, const float *cos_table, const float *sin_table,
                                        int64_t table_rows, const int32_t *positions, const int64_t *slots, void *q_out,
                                        void *k_cache, void *v_cache, int cache_dtype, int64_t pages, int64_t page_size,
                                        int64_t stride_page, int64_t stride_slot, int64_t stride_head,
                                        const float *k_scale, int k_scale_step, const float *v_scale, int v_scale_step,
                                        void *stream) {
  using namespace fp8b200;
  using namespace fp8b200::paged;
  if (dtype != FP8B200_BF16 && dtype != FP8B200_F16)
    return set_error(FP8B200_EINVAL, "rope_write_paged: qkv must be bf16 or f16");
  const bool fp8 = cache_dtype == FP8B200_E4M3 || cache_dtype == FP8B200_E5M2;
  if (!fp8 && cache_dtype != dtype)
    return set_error(FP8B200_EINVAL, "rope_write_paged: the cache must be float8 or of qkv's type");
  if (tokens < 0 || n_q_heads < 0 || n_kv_heads < 1 || table_rows < 0 || pages < 0)
    return set_error(FP8B200_EINVAL, "rope_write_paged: bad size");
  if (head_dim <= 0 || head_dim % 16 || head_dim > 65536)
    return set_error(FP8B200_EINVAL, "rope_write_paged: head_dim=%d must be a positive multiple of 16", head_dim);
  if ((int64_t)n_q_heads + 2ll * n_kv_heads > (1 << 20))
    return set_error(FP8B200_EINVAL, "rope_write_paged: too many heads");
  if (page_size < 1 || pages * (__int128)page_size > INT32_MAX)
    return set_error(FP8B200_EINVAL, "rope_write_paged: a pool holds 1 .. 2^31 - 1 slots");
  const int64_t unit = 8;  // 16-byte (8-byte float8) vector accesses of 8 elements
  if (ld < (int64_t)(n_q_heads + 2 * n_kv_heads) * head_dim || ld % unit)
    return set_error(FP8B200_EINVAL, "rope_write_paged: row stride must cover the heads and be a multiple of 8");
  if (stride_page % unit || stride_slot % unit || stride_head % unit)
    return set_error(FP8B200_EINVAL, "rope_write_paged: cache strides must be multiples of 8 elements");
  if (tokens == 0) return FP8B200_OK;
  const uintptr_t calign = fp8 ? 7u : 15u;
  if (!qkv || !cos_table || !sin_table || !positions || !slots || (n_q_heads && !q_out) ||
      (pages && (!k_cache || !v_cache)))
    return set_error(FP8B200_EINVAL, "rope_write_paged: null pointer");
  if (!aligned16(qkv) || !aligned16(cos_table) || !aligned16(sin_table) || !aligned16(q_out) ||
      ((uintptr_t)k_cache & calign) || ((uintptr_t)v_cache & calign))
    return set_error(FP8B200_EINVAL, "rope_write_paged: tensors must be 16-byte aligned (a float8 cache: 8)");
  int dev;
  if (int rc = check_device(&dev)) return rc;
  WriteParams p{(const uint16_t *)qkv, ld, tokens, n_q_heads, n_kv_heads, head_dim, cos_table, sin_table, table_rows,
                positions, slots, (uint16_t *)q_out, k_cache, v_cache, pages, stride_page, stride_slot, stride_head,
                (int)page_size, fp8 ? k_scale : nullptr, fp8 ? v_scale : nullptr, k_scale_step, v_scale_step};
  const int64_t heads = (int64_t)n_q_heads + 2 * n_kv_heads;
  const int64_t work4 = tokens * ((heads + 3) / 4) * (head_dim / 16), work2 = tokens * ((heads + 1) / 2) * (head_dim / 16);
  const bool full = work4 >= (int64_t)RW_THREADS * RW_FULL * current_sm_count();
  const int grid = grid_for(full ? work4 : work2, RW_THREADS, RW_FULL);
  const bool f16 = dtype == FP8B200_F16;
  void (*kernel)(WriteParams);
  if (cache_dtype == FP8B200_E4M3) kernel = f16 ? rope_write<true, FP8B200_E4M3>(full) : rope_write<false, FP8B200_E4M3>(full);
  else if (cache_dtype == FP8B200_E5M2) kernel = f16 ? rope_write<true, FP8B200_E5M2>(full) : rope_write<false, FP8B200_E5M2>(full);
  else kernel = f16 ? rope_write<true, FP8B200_F16>(full) : rope_write<false, FP8B200_BF16>(full);
  launch_dependent(kernel, dim3((unsigned)grid), RW_THREADS, 0, (cudaStream_t)stream, p);
  count_launch();
  return check_launch("rope_write_paged");
}
