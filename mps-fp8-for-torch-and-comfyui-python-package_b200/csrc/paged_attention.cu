// Causal attention of each request's new tokens over its pages of a
// key/value cache, on warp-level matrix instructions.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j   over the keys j <= p_i with
//         p_i - j < window or j < sinks            (no window: all j <= p_i)
//
// Two kernels, for few query rows a request (paged_few_kernel, blocks of four
// warps) and for more (paged_attention_kernel, four warps, eight at head sizes
// above 128); chunks and prompts go to paged_attention_tc.cu where it serves. The query heads that share a
// key/value head are rows of one tile: row token * group + g.
//
// Work: a segment is one row tile of one request under one key/value head;
// its units are its tiles of 64 keys. The segments' units form a line, which
// is cut into equal shares, one a block (found from the lengths on the GPU:
// the host need not know them, and one long request among short ones is
// spread over all SMs). A block that holds only part of a segment leaves its
// partial result and base in the workspace; the merge kernel joins them in the
// order of the keys. Nothing depends on the order in which blocks run.
//
// K and V come through cp.async into rings of stages (any page size, any
// stride that is a multiple of 16 bytes); float8 codes stay float8 in shared
// memory and become half pairs in registers (cvt, exact), so a float8 cache
// moves half the bytes all the way. Bound by the cache's bytes where a request
// has few rows (decoding), else by the matrix instructions.
//
// Rounding: the weights are rounded to the matrix instruction's 16-bit type
// (bf16 for a bf16 cache, f16 for f16 and float8 ones). In f16 they are scaled
// by 2^7 (few rows: the base may lag the maximum by 2^8) or 2^15, so that
// weights down to 2^-31 or 2^-39 of the base's keep a place; sums, bases and
// outputs are float32. bf16 queries of a float8 cache become f16 after an
// exact power-of-two scaling of the row (the largest value in [1, 2): an
// element loses bits only below 2^-14 of it).
//
// No counterpart in the reference, which has no attention.
#include "paged_attention.cuh"

#include <algorithm>
#include <atomic>

namespace fp8b200 {
namespace paged {
namespace {

constexpr int BN = 64;        // keys a tile
constexpr int THREADS = 128;  // four warps

template <int KV>
constexpr bool is_fp8 = KV == FP8B200_E4M3 || KV == FP8B200_E5M2;

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where 16-byte unit c of key row r sits in its tile. 16-bit K and V and
// float8 V are read eight rows of one unit at a time (ldmatrix), float8 K two
// rows of four units: each pattern meets every bank once.
template <int ROWB, bool KTILE8>
__device__ __forceinline__ uint32_t unit_at(int r, int c) {
  constexpr int CPR = ROWB / 16;
  int x;
  if constexpr (KTILE8) x = CPR >= 8 ? ((r & 1) << 2) : 0;
  else x = CPR >= 8 ? (r & 7) : ((r >> 1) & 3);
  return (uint32_t)(r * ROWB + ((c ^ x) << 4));
}

// Units (key tiles x row tiles, x heads unless each head has blocks of its own)
// of request r; 0 if this launch leaves it to another. A request whose mask leaves nothing still has one, which
// writes its zeros.
template <int MR>
__device__ __forceinline__ long long units_of(const AttnParams &p, int r, int &tiles) {
  const Request q = load_request(p, r);
  tiles = 0;
  if (q.n == 0 || !takes(p, q.n)) return 0;
  tiles = max(1, visible_tiles<BN>(p, q.first, q.first + q.n - 1).count());
  const long long row_tiles = ((long long)q.n * p.group + MR - 1) / MR;
  return row_tiles * p.line_heads * tiles;
}

// a / b and the rest, in 32 bits where they fit (a 64-bit division is a call of
// some hundred cycles, and these stand in front of the first load).
__device__ __forceinline__ long long quotient(long long a, long long b, long long &rest) {
  if (((a | b) >> 32) == 0) {
    const uint32_t q = (uint32_t)a / (uint32_t)b;
    rest = (uint32_t)a - q * (uint32_t)b;
    return q;
  }
  const long long q = a / b;
  rest = a - q * b;
  return q;
}

// A block's share [u, u_end) of the line of units, found by all its threads:
// the request that u falls into and the units before that request. The first
// `extra` blocks have `each` + 1 units, the others `each`. With few units every
// one has its block: with two a block as the least, blocks whose two units lie in
// different segments went through two prologues and ends (12 rows of 3 requests
// over 700 keys 20.9 us, now 18.4; 64 rows of 4 over 300 30.9, now 20.6), which
// outweighs the join of segments of two units (16 decodes over 100 keys 12.5 us,
// now 14.5; in graphs).
struct Share {
  long long u, u_end, before, each, extra;
  int r;  // -1: nothing for this block
  // the block that has unit x
  __device__ __forceinline__ int block_of(long long x) const {
    long long rest;
    const long long front = extra * (each + 1);
    return (int)(x < front ? quotient(x, each + 1, rest) : extra + quotient(x - front, each, rest));
  }
};
template <int MR, int NW = 4>  // NW: the block's warps
__device__ __forceinline__ Share find_share(const AttnParams &p, long long *s_scan, long long c, long long most) {  // block c of at most `most`
  constexpr int THREADS = NW * 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Share sh;
  int tiles;
  // inclusive scan over up to THREADS requests; with more, their sum first
  auto scan = [&](long long mine, long long &total) {
    long long inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long a = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += a;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      if (w < warp) inc += s_scan[w];
      total += s_scan[w];
    }
    return inc;
  };
  const long long first = tid < p.requests ? units_of<MR>(p, tid, tiles) : 0;
  long long total, inc = scan(first, total);
  if (p.requests > THREADS) {
    long long more = 0, sum;
    for (int r = tid + THREADS; r < p.requests; r += THREADS) more += units_of<MR>(p, r, tiles);
    __syncthreads();
    scan(more, sum);
    total += sum;
  }
  if (tid == 0) p.desc[blockIdx.x].rows = 0;
  const long long blocks = min(most, total);
  sh.r = -1;
  sh.u = sh.u_end = sh.before = sh.each = sh.extra = 0;
  if (c >= blocks) return sh;
  sh.each = quotient(total, blocks, sh.extra);
  sh.u = c * sh.each + min(c, sh.extra);
  sh.u_end = sh.u + sh.each + (c < sh.extra);
  long long before = 0, mine = first;
  for (int r0 = 0; r0 < p.requests; r0 += THREADS) {
    const int r = r0 + tid;
    long long all = total;
    if (p.requests > THREADS) {
      mine = r < p.requests ? units_of<MR>(p, r, tiles) : 0;
      __syncthreads();
      inc = scan(mine, all);
    }
    if (before + inc > sh.u && before + inc - mine <= sh.u) {
      s_scan[NW] = r;
      s_scan[NW + 1] = before + inc - mine;
    }
    before += all;
    if (before > sh.u) break;
  }
  __syncthreads();
  sh.r = (int)s_scan[NW];
  sh.before = s_scan[NW + 1];
  return sh;
}

// bf16 rows of s_q to f16 with the largest value in [1, 2); `flip` changes the
// signs (a negative scale: the maximum of the products is then that of the
// scores). Rows are shared by the block's warps.
template <bool TO_F16, int DP, int NW = 4>
__device__ __forceinline__ void normalise_rows(uint8_t *s_q, int qrow, int rows, float *s_qscale, uint32_t flip) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int row = warp; row < rows; row += NW) {
    uint32_t *w = reinterpret_cast<uint32_t *>(s_q + row * qrow);
    if constexpr (TO_F16) {
      float a = 0.0f;
      for (int i = lane; i < DP / 2; i += 32) a = fmaxf(a, fmaxf(fabsf(u2f(w[i] << 16)), fabsf(u2f(w[i] & 0xFFFF0000u))));
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) a = fmaxf(a, __shfl_xor_sync(~0u, a, d));
      uint32_t eb = f2u(a) >> 23;
      eb = (eb == 255u || a == 0.0f) ? 127u : min(max(eb, 1u), 253u);
      const float mul = u2f((254u - eb) << 23);
      for (int i = lane; i < DP / 2; i += 32)
        w[i] = pack2<true>(u2f(w[i] << 16) * mul, u2f(w[i] & 0xFFFF0000u) * mul) ^ flip;
      if (lane == 0) s_qscale[row] = u2f(eb << 23);
    } else if (flip) {
      for (int i = lane; i < DP / 2; i += 32) w[i] ^= flip;
    }
  }
}

// ------------------------------------------------------------------ few rows
//
// Up to 8 * NG query rows a request (decoding, a few drafted tokens). The
// products are turned around: S^T = K Q^T and O^T = V^T P^T, so that keys and
// dims fill the MMA's 16 rows and the query rows its 8 columns: half the MMAs
// and exponentials of 16-row tiles where a decode has 8 rows or fewer. P^T
// becomes the second product's operand by an 8 x 8 transpose (movmatrix).
// The four warps of a block share nothing but the queries: each takes 16 of a
// tile's 64 keys, brings them into a ring of its own and multiplies them with
// all rows, so there is no block barrier between a segment's ends, a key's
// codes are converted once whatever the number of rows, and the SM's warps
// drift apart and cover one another's latencies. O is rescaled only when a
// row's maximum has grown by more than 2^8 (see paged_attention_tc.cu).
//
// Measured, 64 decodes of up to 32768 cached tokens, 32 / 8 heads of 128, e4m3
// (1.90 GB of cache, 290 us at the measured copy rate): 572 us with one block
// barrier a tile and 16-row tiles, 470 us with a ring a warp, 424 us turned
// around, 402 us with a line of work a head, 389 us (338 us in a graph) since the
// segment's end no longer holds a row's recomputation; before
// the kernels' shared-memory carve-out was fixed an SM could take one block of
// three after a kernel without shared memory (672 us). 24 requests of 5 tokens,
// 16 / 2 heads of 64, e5m2, up to 8000 cached: 35 us, of which about 16 are the
// fixed costs of finding the share, the first loads and the join.
template <bool F16, int KV, int DP, int NG>
struct Few {
  static constexpr bool FP8 = is_fp8<KV>;
  static constexpr bool MF16 = F16 || FP8;
  static constexpr int ROWB = DP * (FP8 ? 1 : 2), CPR = ROWB / 16;
  static constexpr int WK = 16;                           // keys a warp takes of a tile
  static constexpr int HALF = WK * ROWB;                  // K or V of them
  static constexpr int ST = DP == 256 && !FP8 ? 2 : DP == 64 ? 4 : 3;
  static constexpr int RING = ST * 2 * HALF;              // a warp's
  static constexpr int MR = 8 * NG;
  static constexpr int QROW = DP * 2 + 16;
  static constexpr int SO = DP + 4;                       // floats a row of the warps' outputs (padded: no bank conflicts)
  static constexpr int OFF_Q = 4 * RING;
  static constexpr int OFF_SCALE = OFF_Q + MR * QROW;     // [MR] query scales, [4][MR] bases, [4][MR] sums
  static constexpr int OFF_SCAN = OFF_SCALE + 9 * MR * 4;
  static constexpr int SMEM = OFF_SCAN + 64;
  static constexpr float SHIFT = MF16 ? 7.0f : 0.0f;
  static constexpr bool QREG = NG * DP <= 128;            // query fragments stay in registers
  // blocks an SM: what the registers (outputs: NG * DP / 4 a thread) and the rings leave
  static constexpr int PER_SM = DP == 256 ? (FP8 ? 2 : 1)
                                : DP == 128 ? (FP8 ? (NG == 1 ? 4 : NG == 2 ? 3 : 2) : 2)
                                            : (NG <= 2 ? (FP8 ? 4 : 3) : NG == 4 ? 3 : 2);
  static_assert(4 * 16 * SO * 4 <= 4 * RING, "the warps' outputs of 16 rows fit the drained rings");
  static_assert(PER_SM * (SMEM + 1024) <= 233472, "blocks an SM");
};

template <bool F16, int KV, int DP, int NG>
__global__ void __launch_bounds__(THREADS, (Few<F16, KV, DP, NG>::PER_SM)) paged_few_kernel(const AttnParams p) {
  using C = Few<F16, KV, DP, NG>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *s_q = smem + C::OFF_Q;
  float *s_qscale = reinterpret_cast<float *>(smem + C::OFF_SCALE), *s_base = s_qscale + C::MR, *s_sum = s_base + 4 * C::MR;
  long long *s_scan = reinterpret_cast<long long *>(smem + C::OFF_SCAN);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tg = lane & 3;
  uint8_t *ring = smem + warp * C::RING;
  const uint32_t ring_a = saddr(ring);
  const uint8_t *none = reinterpret_cast<const uint8_t *>(p.q);  // where nothing is read from
  const int used = (p.d * (C::FP8 ? 1 : 2)) / 16;          // 16-byte units of a key's row that hold values
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // line_heads 1: as many lines as heads, their blocks side by side, so that the
  // heads of a key (neighbours in memory) are read at about the same time
  const long long c = blockIdx.x;
  const int lines = p.line_heads == 1 ? p.hk : 1, line = (int)(c % lines);
  const Share sh = find_share<C::MR>(p, s_scan, c / lines, gridDim.x / lines);
  long long u = sh.u, before = sh.before;
  int r = sh.r;
  while (r >= 0 && u < sh.u_end) {
    // ---- the segment that unit u belongs to
    const Request rq = load_request(p, r);
    int tiles_n;
    const long long n_units = units_of<C::MR>(p, r, tiles_n);
    if (u >= before + n_units) {
      before += n_units;
      r++;
      continue;
    }
    long long in_tiles, in_heads;
    const int qt = (int)quotient(quotient(u - before, tiles_n, in_tiles), p.line_heads, in_heads), h = line + (int)in_heads;
    const int t_begin = (int)in_tiles, t_end = (int)min((long long)tiles_n, t_begin + (sh.u_end - u));
    const long long seg_start = u - t_begin;
    u += t_end - t_begin;
    const Tiles<BN> tl = visible_tiles<BN>(p, rq.first, rq.first + rq.n - 1);
    const int row0 = qt * C::MR;
    const int rows = (int)min((long long)C::MR, (long long)rq.n * p.group - row0);
    const int pos_lo = rq.first + row0 / p.group, pos_hi = rq.first + (row0 + rows - 1) / p.group;
    const float scale = p.scale_log2 * (C::FP8 && p.ks ? __ldg(p.ks + p.ks_step * h) : 1.0f);

    // this warp's keys of list entry i: lane < 16 finds the slot of key `lane`
    auto find = [&](int i) -> long long {
      if (i >= t_end || lane >= C::WK) return -1;
      const int j = tl.at(i) * BN + warp * C::WK + lane;
      return j <= pos_hi ? slot_offset(p, r, j) : -2;      // -2: no key, -1: a key without a page
    };
    unsigned long long hidden = 0;                          // keys without a page, 16 bits a tile, newest last
    auto issue = [&](int stage, long long off) {            // of the tile whose offsets the lanes hold
      hidden = (hidden << 16) | (__ballot_sync(~0u, off == -1) & 0xFFFFu);
      constexpr int STEP = 32 / C::CPR > 0 ? 32 / C::CPR : 1, PASS = C::CPR > 32 ? C::CPR / 32 : 1;
#pragma unroll
      for (int k = 0; k < C::WK / STEP; k++) {
        const int row = k * STEP + (C::CPR < 32 ? lane / C::CPR : 0);
        const long long o = __shfl_sync(~0u, off, row);
#pragma unroll
        for (int q = 0; q < PASS; q++) {
          const int cu = C::CPR < 32 ? lane % C::CPR : lane + 32 * q;
          if (cu < used) {
            const bool valid = o >= 0;
            const long long byte = valid ? (o + (long long)h * p.s_head) * (C::FP8 ? 1 : 2) + cu * 16 : 0;
            const uint32_t at = ring_a + stage * 2 * C::HALF;
            cp16(at + (C::FP8 ? unit_at<C::ROWB, true>(row, cu) : unit_at<C::ROWB, false>(row, cu)), valid ? p.k + byte : none, valid);
            cp16(at + C::HALF + unit_at<C::ROWB, false>(row, cu), valid ? p.v + byte : none, valid);
          }
        }
      }
    };

    __syncthreads();  // the previous segment's readers of shared memory are done
    if (used < C::CPR) {  // units without values are zero while the segment lasts (its end uses the ring for something else)
      for (int i = lane; i < C::RING / 16; i += 32) {
        const int half = i / (C::HALF / 16), row = (i % (C::HALF / 16)) / C::CPR, cu = i % C::CPR;
        if (cu >= used) {
          const uint32_t at = (C::FP8 && half % 2 == 0) ? unit_at<C::ROWB, true>(row, cu) : unit_at<C::ROWB, false>(row, cu);
          *reinterpret_cast<uint4 *>(ring + half * C::HALF + at) = make_uint4(0, 0, 0, 0);
        }
      }
      __syncwarp();
    }
    long long off[C::ST];
#pragma unroll
    for (int k = 0; k < C::ST; k++) off[k] = find(t_begin + k);  // all table reads in flight at once
    constexpr int QU = C::MR * (DP / 8), QN = (QU + THREADS - 1) / THREADS;  // 16-byte units of the queries, a thread's
    uint4 qv[QN];
#pragma unroll
    for (int k = 0; k < QN; k++) {
      const int row = (tid + k * THREADS) / (DP / 8), cu = (tid + k * THREADS) % (DP / 8);
      qv[k] = make_uint4(0, 0, 0, 0);
      if (row < rows && cu * 8 < p.d) {
        const int qr = row0 + row, tok = qr / p.group, head = h * p.group + qr - tok * p.group;
        qv[k] = __ldg(reinterpret_cast<const uint4 *>(p.q + (int64_t)(rq.start + tok) * p.q_tok + (int64_t)head * p.q_head + cu * 8));
      }
    }
#pragma unroll
    for (int k = 0; k < C::ST - 1; k++) {
      issue(k, off[k]);
      cp_commit();
    }
#pragma unroll
    for (int k = 0; k < QN; k++)
      if (tid + k * THREADS < QU)
        *reinterpret_cast<uint4 *>(s_q + (tid + k * THREADS) / (DP / 8) * C::QROW + (tid + k * THREADS) % (DP / 8) * 16) = qv[k];
    long long ahead = off[C::ST - 1];                       // offsets of the next tile to load
    __syncthreads();
    if ((C::FP8 && !F16) || scale < 0.0f) {
      normalise_rows<C::FP8 && !F16, DP>(s_q, C::QROW, C::MR, s_qscale, scale < 0.0f ? 0x80008000u : 0u);
      __syncthreads();
    }
    // the queries as the first product's B: row ng * 8 + g, values of K step ks
    auto load_q = [&](int ng, int ks, uint32_t (&q)[2]) {
      const uint8_t *q0 = s_q + (ng * 8 + g) * C::QROW;
      if constexpr (C::FP8) {                               // k order of a 64-value block: lane tg holds values 16 tg .. 16 tg + 15
        const uint2 x = *reinterpret_cast<const uint2 *>(q0 + ((ks >> 2) * 64 + tg * 16 + (ks & 3) * 4) * 2);
        q[0] = x.x, q[1] = x.y;
      } else {
        const int at = (ks * 16 + tg * 2) * 2;
        q[0] = *reinterpret_cast<const uint32_t *>(q0 + at);
        q[1] = *reinterpret_cast<const uint32_t *>(q0 + at + 16);
      }
    };
    uint32_t qf[C::QREG ? NG : 1][C::QREG ? DP / 16 : 1][2];
    if constexpr (C::QREG) {
#pragma unroll
      for (int ng = 0; ng < NG; ng++)
#pragma unroll
        for (int ks = 0; ks < DP / 16; ks++) load_q(ng, ks, qf[ng][ks]);
    }
    // a thread's rows: ng * 8 + 2 tg and the next; its keys of a tile: g and g + 8
    float sc[NG][2];                                        // above 0, see paged_attention_tc.cu
    int pos[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ng++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = ng * 8 + 2 * tg + e;
        sc[ng][e] = fabsf(scale) * ((C::FP8 && !F16) ? s_qscale[row] : 1.0f);
        if (sc[ng][e] == 0.0f) sc[ng][e] = 1e-30f;
        pos[ng][e] = rq.first + min(row0 + row, row0 + rows - 1) / p.group;
      }
    float o[NG][DP / 16][4], base[NG][2], sum[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ng++) {
#pragma unroll
      for (int i = 0; i < DP / 16; i++) o[ng][i][0] = o[ng][i][1] = o[ng][i][2] = o[ng][i][3] = 0.0f;
      base[ng][0] = base[ng][1] = -INFINITY;
      sum[ng][0] = sum[ng][1] = 0.0f;
    }

    int stage = 0;
#pragma unroll 1
    for (int i = t_begin; i < t_end; i++) {
      cp_wait<C::ST - 2>();
      __syncwarp();
      {
        int st = stage + C::ST - 1;
        if (st >= C::ST) st -= C::ST;
        issue(st, ahead);                                   // behind the last tile: copies nothing that is read
        cp_commit();
        ahead = find(i + C::ST);
      }
      const uint32_t kt = ring_a + stage * 2 * C::HALF, vt = kt + C::HALF;
      if (++stage == C::ST) stage = 0;
      float s[NG][4];                                       // [keys g, g + 8][rows 2 tg, 2 tg + 1]
#pragma unroll
      for (int ng = 0; ng < NG; ng++) s[ng][0] = s[ng][1] = s[ng][2] = s[ng][3] = 0.0f;
      auto first_product = [&](int ks, const uint32_t (&a)[4]) {
#pragma unroll
        for (int ng = 0; ng < NG; ng++) {
          if constexpr (C::QREG) {
            mma<C::MF16>(s[ng], a, qf[ng][ks][0], qf[ng][ks][1]);
          } else {
            uint32_t q[2];
            load_q(ng, ks, q);
            mma<C::MF16>(s[ng], a, q[0], q[1]);
          }
        }
      };
      if constexpr (C::FP8) {
#pragma unroll
        for (int b = 0; b < DP / 64; b++) {
          uint32_t w[2][4];                                 // 16 codes of keys g and g + 8
#pragma unroll
          for (int e = 0; e < 2; e++)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[e][0]), "=r"(w[e][1]), "=r"(w[e][2]), "=r"(w[e][3])
                         : "r"(kt + unit_at<C::ROWB, true>(e * 8 + g, b * 4 + tg)));
#pragma unroll
          for (int ks = 0; ks < 4; ks++) {
            const uint32_t a[4] = {fp8x2_to_f16x2<KV>(w[0][ks] & 0xFFFFu), fp8x2_to_f16x2<KV>(w[1][ks] & 0xFFFFu),
                                   fp8x2_to_f16x2<KV>(w[0][ks] >> 16), fp8x2_to_f16x2<KV>(w[1][ks] >> 16)};
            first_product(b * 4 + ks, a);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ks++) {
          uint32_t a[4];
          ldsm4(kt + unit_at<C::ROWB, false>((((lane >> 3) & 1) << 3) + (lane & 7), ks * 2 + (lane >> 4)), a);
          first_product(ks, a);
        }
      }
      const int k0 = tl.at(i) * BN + warp * C::WK;
      const uint32_t hide = (uint32_t)(hidden >> (16 * (C::ST - 1))) & 0xFFFFu;
      if (k0 + C::WK - 1 > pos_lo || hide || (p.window > 0 && pos_hi - k0 >= p.window && k0 + C::WK - 1 >= p.sinks)) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int kk = g + 8 * e;
          const bool gone = (hide >> kk) & 1u;
#pragma unroll
          for (int ng = 0; ng < NG; ng++)
#pragma unroll
            for (int x = 0; x < 2; x++)
              if (gone || !visible(p, k0 + kk, pos[ng][x])) s[ng][2 * e + x] = -INFINITY;
        }
      }
      float top[NG][2];
      bool grow = false;
#pragma unroll
      for (int ng = 0; ng < NG; ng++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          float m = fmaxf(s[ng][x], s[ng][2 + x]);
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
          top[ng][x] = m * sc[ng][x];
          grow |= top[ng][x] > base[ng][x] + 8.0f;          // also a row's first key
        }
      if (__any_sync(~0u, grow)) {
#pragma unroll
        for (int ng = 0; ng < NG; ng++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const float nb = fmaxf(base[ng][x], top[ng][x]);
            const float f = base[ng][x] == -INFINITY ? 0.0f : ex2(base[ng][x] - nb);
            base[ng][x] = nb;
            sum[ng][x] *= f;
#pragma unroll
            for (int j = 0; j < DP / 16; j++) o[ng][j][x] *= f, o[ng][j][2 + x] *= f;
          }
      }
      uint32_t pb[NG][2];                                   // the weights as the second product's B
#pragma unroll
      for (int ng = 0; ng < NG; ng++) {
        const float o0 = C::SHIFT - (base[ng][0] == -INFINITY ? 0.0f : base[ng][0]);
        const float o1 = C::SHIFT - (base[ng][1] == -INFINITY ? 0.0f : base[ng][1]);
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float e0 = ex2(fmaf(s[ng][2 * e], sc[ng][0], o0)), e1 = ex2(fmaf(s[ng][2 * e + 1], sc[ng][1], o1));
          sum[ng][0] += e0;
          sum[ng][1] += e1;
          const uint32_t w = pack2<C::MF16>(e0, e1);
          asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[ng][e]) : "r"(w));
        }
      }
      if constexpr (C::FP8) {
        const int key = (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
        for (int cp = 0; cp < DP / 32; cp++) {
          uint32_t w[4];
          ldsm4t(vt + unit_at<C::ROWB, false>(key, cp * 2 + (lane >> 4)), w);
#pragma unroll
          for (int e = 0; e < 2; e++) {                     // unit cp * 2 + e: rows g its even dims, rows g + 8 its odd dims
            uint32_t x, y;
            asm("prmt.b32 %0, %1, 0, 0x3120;" : "=r"(x) : "r"(w[2 * e]));
            asm("prmt.b32 %0, %1, 0, 0x3120;" : "=r"(y) : "r"(w[2 * e + 1]));
            const uint32_t a[4] = {fp8x2_to_f16x2<KV>(x & 0xFFFFu), fp8x2_to_f16x2<KV>(x >> 16), fp8x2_to_f16x2<KV>(y & 0xFFFFu),
                                   fp8x2_to_f16x2<KV>(y >> 16)};
#pragma unroll
            for (int ng = 0; ng < NG; ng++) mma<true>(o[ng][cp * 2 + e], a, pb[ng][0], pb[ng][1]);
          }
        }
      } else {
#pragma unroll
        for (int dp = 0; dp < DP / 16; dp++) {
          uint32_t a[4];
          ldsm4t(vt + unit_at<C::ROWB, false>(((lane >> 4) << 3) + (lane & 7), dp * 2 + ((lane >> 3) & 1)), a);
#pragma unroll
          for (int ng = 0; ng < NG; ng++) mma<C::MF16>(o[ng][dp], a, pb[ng][0], pb[ng][1]);
        }
      }
    }
    cp_wait<0>();

    // ---- the segment's end: the warps' results, a row group at a time, through the drained rings
    bool odd = false;                                       // infinities or NaN: see odd_rows
#pragma unroll
    for (int ng = 0; ng < NG; ng++) {
#pragma unroll
      for (int j = 0; j < DP / 16; j++)
#pragma unroll
        for (int x = 0; x < 4; x++) odd |= !(fabsf(o[ng][j][x]) < INFINITY);
#pragma unroll
      for (int x = 0; x < 2; x++) {
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) sum[ng][x] += __shfl_xor_sync(~0u, sum[ng][x], d);
        if (g == 0) {
          s_base[warp * C::MR + ng * 8 + 2 * tg + x] = base[ng][x] - C::SHIFT;
          s_sum[warp * C::MR + ng * 8 + 2 * tg + x] = sum[ng][x];
        }
      }
    }
    const bool careful = __syncthreads_or(odd);
    const bool begins = t_begin == 0, ends = t_end == tiles_n;
    const float vs = C::FP8 && p.vs ? __ldg(p.vs + p.vs_step * h) : 1.0f;
    float *part = p.part + (c * 2 + (begins ? 1 : 0)) * (int64_t)(C::MR * (DP + 2));
    if (tid == 0 && begins && !ends)
      p.desc[c] = PartDesc{rows, row0, h, rq.start, sh.block_of(seg_start + tiles_n - 1) - (int)(c / lines) + 1, lines};
    float *s_o = reinterpret_cast<float *>(smem);           // [4 warps][16 rows][SO]
#pragma unroll
    for (int mg = 0; mg < (NG + 1) / 2; mg++) {
      if (mg * 16 < rows) {
        if (mg) __syncthreads();
#pragma unroll
        for (int half = 0; half < (NG > 1 ? 2 : 1); half++) {
          const int ng = mg * 2 + half;
          if (ng >= NG) continue;
          float *x0 = s_o + (warp * 16 + half * 8 + 2 * tg) * C::SO, *x1 = x0 + C::SO;
#pragma unroll
          for (int j = 0; j < DP / 16; j++) {
            const float(&v)[4] = o[ng][j];
            if constexpr (C::FP8) {
              *reinterpret_cast<float2 *>(x0 + j * 16 + 2 * g) = make_float2(v[0], v[2]);
              *reinterpret_cast<float2 *>(x1 + j * 16 + 2 * g) = make_float2(v[1], v[3]);
            } else {
              x0[j * 16 + g] = v[0], x0[j * 16 + g + 8] = v[2];
              x1[j * 16 + g] = v[1], x1[j * 16 + g + 8] = v[3];
            }
          }
        }
        __syncthreads();
        const int group_rows = min(16, rows - mg * 16);
        for (int i = tid; i < group_rows * (DP / 4); i += THREADS) {
          const int row = i / (DP / 4), d4 = (i % (DP / 4)) * 4, at = mg * 16 + row;
          float b = fmaxf(fmaxf(s_base[at], s_base[C::MR + at]), fmaxf(s_base[2 * C::MR + at], s_base[3 * C::MR + at]));
          const float ref = b == -INFINITY ? 0.0f : b;
          float l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const float f = ex2(s_base[w * C::MR + at] - ref);
            const float4 v = *reinterpret_cast<const float4 *>(s_o + (w * 16 + row) * C::SO + d4);
            l += f * s_sum[w * C::MR + at];
            x[0] += f * v.x, x[1] += f * v.y, x[2] += f * v.z, x[3] += f * v.w;
          }
          if (careful && d4 == 0) s_qscale[at] = l;
          if (begins && ends) {
            if (d4 < p.d) {
              const float inv = l == 0.0f ? 0.0f : vs / l;
              const int qr = row0 + at, tok = rq.start + qr / p.group, head = h * p.group + qr % p.group;
              uint16_t *out = p.out + (int64_t)tok * p.o_tok + (int64_t)head * p.o_head + d4;
              *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<F16>(x[0] * inv, x[1] * inv), pack2<F16>(x[2] * inv, x[3] * inv));
            }
          } else {
            *reinterpret_cast<float4 *>(part + at * DP + d4) = make_float4(x[0], x[1], x[2], x[3]);
            if (d4 == 0) {
              part[C::MR * DP + at] = b;
              part[C::MR * DP + C::MR + at] = l;
            }
          }
        }
      }
    }
    if (careful) {                                          // each warp looks through its share of the rows
      __syncthreads();
      const int row = warp + 4 * lane;
      const bool mine = lane < C::MR / 4 && row < rows;
      const SegmentRows<BN> seg_rows{r, rq.start, rq.first, h, row0, tl, t_begin, t_end};
      odd_rows<F16, KV, DP, BN>(p, seg_rows, row, mine, mine ? s_qscale[row] : 0.0f, begins && ends, part, C::MR, nullptr);
    }
  }
  if (p.zero_rest) zero_rest(p, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------ more rows
//
// Where the tensor-memory kernel does not serve (head sizes above 128, caches
// that no tensor map describes, a few dozen rows): each of the block's NW warps
// takes 16 rows; with fewer than 16 NW rows NW / RW warps share the tile's keys.
// Head sizes up to 128: four warps, two blocks an SM. Above, where one block
// fills the SM: eight warps, since four, one a scheduler, wait on each
// instruction: 1073 rows of 8 heads over up to 2408 keys 182 -> 138 us in e4m3
// (127 now, 105 in bf16); 88 rows a request, 10 over 19531 keys in f16 183 -> 142 us. A
// tile of 128 rows by 64 keys takes 5 to 6 us: 2 us of warp-level MMA, as much
// of shared-memory reads (each warp reads all of K and V), little overlapped.
template <bool F16, int KV, int DP, int RW, int NW>
struct Cfg {
  static constexpr int THREADS = NW * 32;
  static constexpr bool FP8 = is_fp8<KV>;
  static constexpr bool MF16 = F16 || FP8;              // operand type of the matrix instructions
  static constexpr int ROWB = DP * (FP8 ? 1 : 2);       // bytes of a key's row in shared memory
  static constexpr int CPR = ROWB / 16;                 // 16-byte units of it
  static constexpr int TILE = BN * ROWB;                // K or V
  // two blocks an SM (head size 256: one), the more bytes in flight the better
  static constexpr int STAGES = FP8 ? (DP == 64 ? 8 : DP == 128 ? 5 : 4)
                                    : (DP == 64 ? 6 : 2);
  static constexpr int MR = 16 * RW;                    // rows a block
  static constexpr int KW = NW / RW;                    // warps that share a tile's keys
  static constexpr int WN = BN / KW;                    // keys a warp
  static constexpr int QROW = DP * 2 + 16;              // bytes of a query row (padded: no bank conflicts)
  static constexpr int RING = STAGES * 2 * TILE;
  static constexpr int OFFS = STAGES + 1;               // slot offsets are found one tile further ahead
  static constexpr int SMEM = RING + MR * QROW + OFFS * BN * 8 + OFFS * 2 * 4 + MR * 4 + NW * 16 * 2 * 4 + NW * 8 + 32;
  static constexpr float SHIFT = MF16 ? 15.0f : 0.0f;   // weights are scaled by 2^SHIFT
  static_assert(MR <= NW * 32, "a lane a row");
  static_assert(NW * 16 * DP * 4 <= RING, "the warps' outputs fit the drained ring");
};

template <bool F16, int KV, int DP, int RW, int NW>
__global__ void __launch_bounds__(NW * 32, DP == 256 ? 1 : 2) paged_attention_kernel(const AttnParams p) {
  using C = Cfg<F16, KV, DP, RW, NW>;
  constexpr int THREADS = C::THREADS;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *ring = smem;
  uint8_t *s_q = ring + C::RING;
  long long *s_off = reinterpret_cast<long long *>(s_q + C::MR * C::QROW);
  int *s_bad = reinterpret_cast<int *>(s_off + C::OFFS * BN);   // [OFFS][2]
  float *s_qscale = reinterpret_cast<float *>(s_bad + C::OFFS * 2);
  float *s_base = s_qscale + C::MR;                             // [NW warps][16 rows]
  float *s_sum = s_base + NW * 16;
  long long *s_scan = reinterpret_cast<long long *>(s_sum + NW * 16);  // NW warps' totals, then found request and its prefix
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tg = lane & 3;
  const int rw = warp / C::KW, kw = warp % C::KW;
  const uint32_t ring_a = saddr(ring), q_a = saddr(s_q);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint8_t *none = reinterpret_cast<const uint8_t *>(p.q);  // where nothing is read from
  const int used = (p.d * (C::FP8 ? 1 : 2)) / 16;  // 16-byte units of a key's row that hold values
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this block's share of the line of units
  const Share sh = find_share<C::MR, NW>(p, s_scan, blockIdx.x, gridDim.x);
  if (p.zero_rest) zero_rest(p, blockIdx.x, gridDim.x);
  if (sh.r < 0) return;
  const long long c = blockIdx.x, u_end = sh.u_end;
  long long u = sh.u, before = sh.before;
  int r = sh.r;
  while (u < u_end) {
    // ---- the segment that unit u belongs to
    const Request rq = load_request(p, r);
    int tiles_n;
    const long long n_units = units_of<C::MR>(p, r, tiles_n);
    if (u >= before + n_units) {
      before += n_units;
      r++;
      continue;
    }
    const long long local = u - before;
    const long long seg = local / tiles_n;
    const int t_begin = (int)(local - seg * tiles_n);
    const int t_end = (int)min((long long)tiles_n, t_begin + (u_end - u));
    const int h = (int)(seg % p.hk), qt = (int)(seg / p.hk);
    const long long seg_start = u - t_begin;
    u += t_end - t_begin;
    const Tiles<BN> tl = visible_tiles<BN>(p, rq.first, rq.first + rq.n - 1);
    const int row0 = qt * C::MR;
    const int rows = (int)min((long long)C::MR, (long long)rq.n * p.group - row0);
    const int pos_lo = rq.first + row0 / p.group, pos_hi = rq.first + (row0 + rows - 1) / p.group;
    // of the request's tiles, those that this row tile sees
    const int live_from = p.window > 0 ? (int)(max((long long)pos_lo - p.window + 1, 0ll) / BN) : 0;
    const int live_sinks = p.window > 0 ? (int)(((long long)p.sinks + BN - 1) / BN) : 0;
    auto live = [&](int i) {
      const int t = tl.at(i);
      return t * BN <= pos_hi && (t >= live_from || t < live_sinks);
    };
    auto next_live = [&](int i) {
      while (i < t_end && !live(i)) i++;
      return i;
    };

    // slot offset of this thread's key (threads 0 .. 63) of list entry i; bad: a key that should have a page has none
    auto find_offset = [&](int i, long long &off, bool &bad) {
      off = -1;
      bad = false;
      if (i < t_end && tid < BN) {
        const int j = tl.at(i) * BN + tid;
        if (j <= pos_hi) {
          off = slot_offset(p, r, j);
          bad = off < 0;
        }
      }
    };
    auto put_offset = [&](int slot, long long off, bool bad) {
      if (tid < BN) {
        s_off[slot * BN + tid] = off;
        const bool any = __any_sync(~0u, bad);
        if (lane == 0) s_bad[slot * 2 + warp] = any;
      }
    };
    auto issue = [&](int stage, int slot) {
      const int cunit = tid % C::CPR;
      if (cunit < used) {
#pragma unroll
        for (int row = tid / C::CPR; row < BN; row += THREADS / C::CPR) {
          const long long off = s_off[slot * BN + row];
          const long long byte = (off < 0 ? 0 : (off + (long long)h * p.s_head) * (C::FP8 ? 1 : 2)) + cunit * 16;
          const bool valid = off >= 0;
          const uint32_t kd = ring_a + stage * 2 * C::TILE + (C::FP8 ? unit_at<C::ROWB, true>(row, cunit) : unit_at<C::ROWB, false>(row, cunit));
          const uint32_t vd = ring_a + (stage * 2 + 1) * C::TILE + unit_at<C::ROWB, false>(row, cunit);
          cp16(kd, valid ? p.k + byte : none, valid);
          cp16(vd, valid ? p.v + byte : none, valid);
        }
      }
    };

    __syncthreads();  // the previous segment's readers of shared memory are done
    if (used < C::CPR) {  // the others are zero while the segment lasts (its end uses the ring for something else)
      for (int i = tid; i < C::RING / 16; i += THREADS) {
        const int tile = i / (C::TILE / 16), row = (i % (C::TILE / 16)) / C::CPR, cu = i % C::CPR;
        if (cu >= used) {
          const uint32_t at = (C::FP8 && tile % 2 == 0) ? unit_at<C::ROWB, true>(row, cu) : unit_at<C::ROWB, false>(row, cu);
          *reinterpret_cast<uint4 *>(ring + tile * C::TILE + at) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    // ---- prologue: offsets of the first STAGES tiles, loads of the first STAGES - 1
    int ahead = next_live(t_begin);           // list entry of the next tile to find offsets for
    const int first_tile = ahead;
    int n_ahead = 0;                          // tiles whose offsets are known
    {
      long long offs[C::STAGES];              // all table reads in flight at once
      bool bads[C::STAGES];
#pragma unroll
      for (int s = 0; s < C::STAGES; s++) {
        find_offset(ahead, offs[s], bads[s]);
        if (ahead < t_end) {
          n_ahead++;
          ahead = next_live(ahead + 1);
        }
      }
#pragma unroll
      for (int s = 0; s < C::STAGES; s++) put_offset(s, offs[s], bads[s]);
    }
    // query rows, four units a thread in flight
    constexpr int QU = C::MR * (DP / 8), QN = 4;
    static_assert(QU % (THREADS * QN) == 0, "whole rounds");
#pragma unroll 1
    for (int i0 = tid; i0 < QU; i0 += THREADS * QN) {
      uint4 v[QN];
#pragma unroll
      for (int k = 0; k < QN; k++) {
        const int i = i0 + k * THREADS, row = i / (DP / 8), cu = i % (DP / 8);
        v[k] = make_uint4(0, 0, 0, 0);
        if (row < rows && cu * 8 < p.d) {
          const int qr = row0 + row, tok = qr / p.group, head = h * p.group + qr - tok * p.group;
          v[k] = __ldg(reinterpret_cast<const uint4 *>(p.q + (int64_t)(rq.start + tok) * p.q_tok + (int64_t)head * p.q_head + cu * 8));
        }
      }
#pragma unroll
      for (int k = 0; k < QN; k++) {
        const int i = i0 + k * THREADS;
        *reinterpret_cast<uint4 *>(s_q + i / (DP / 8) * C::QROW + i % (DP / 8) * 16) = v[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; s++) {
      if (s < n_ahead) issue(s, s);
      cp_commit();
    }
    if constexpr (C::FP8 && !F16) {           // bf16 rows to f16, the largest value in [1, 2)
      normalise_rows<true, DP, NW>(s_q, C::QROW, C::MR, s_qscale, 0u);
      __syncthreads();
    }
    const int wr = rw * 16;                   // this warp's first row in the tile
    float qs0 = 1.0f, qs1 = 1.0f;
    if constexpr (C::FP8 && !F16) {
      qs0 = s_qscale[wr + g];
      qs1 = s_qscale[wr + g + 8];
    }
    const float sc = p.scale_log2 * (C::FP8 && p.ks ? __ldg(p.ks + p.ks_step * h) : 1.0f);
    const float sc0 = sc * qs0, sc1 = sc * qs1;
    const int pos0 = rq.first + min(row0 + wr + g, row0 + rows - 1) / p.group;
    const int pos1 = rq.first + min(row0 + wr + g + 8, row0 + rows - 1) / p.group;

    auto load_q = [&](int ks, uint32_t (&a)[4]) {
      const uint8_t *q0 = s_q + (wr + g) * C::QROW, *q1 = q0 + 8 * C::QROW;
      if constexpr (C::FP8) {                 // k order of a 64-value block: lane tg holds values 16 tg .. 16 tg + 15
        const int at = ((ks >> 2) * 64 + tg * 16 + (ks & 3) * 4) * 2;
        const uint2 x = *reinterpret_cast<const uint2 *>(q0 + at), y = *reinterpret_cast<const uint2 *>(q1 + at);
        a[0] = x.x, a[1] = y.x, a[2] = x.y, a[3] = y.y;
      } else {
        const int at = (ks * 16 + tg * 2) * 2;
        a[0] = *reinterpret_cast<const uint32_t *>(q0 + at);
        a[1] = *reinterpret_cast<const uint32_t *>(q1 + at);
        a[2] = *reinterpret_cast<const uint32_t *>(q0 + at + 16);
        a[3] = *reinterpret_cast<const uint32_t *>(q1 + at + 16);
      }
    };
    constexpr bool QREG = DP <= 128;          // query fragments stay in registers
    uint32_t qf[QREG ? DP / 16 : 1][4];
    if constexpr (QREG) {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ks++) load_q(ks, qf[ks]);
    }

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    int cur = first_tile;                     // list entry of the tile being computed
    int stage = 0, slot = 0;
    for (int it = 0; cur < t_end; it++) {
      cp_wait<C::STAGES - 2>();
      __syncthreads();
      // loads of tile it + STAGES - 1 (its offsets were published by the barrier), offsets of the one after it
      if (it + C::STAGES - 1 < n_ahead) {
        int st = stage + C::STAGES - 1, sl = slot + C::STAGES - 1;
        if (st >= C::STAGES) st -= C::STAGES;
        if (sl >= C::OFFS) sl -= C::OFFS;
        issue(st, sl);
      }
      cp_commit();
      long long next_off;
      bool next_bad;
      find_offset(ahead, next_off, next_bad);

      const uint32_t kt = ring_a + stage * 2 * C::TILE, vt = kt + C::TILE;
      const int key0 = kw * C::WN;            // this warp's first key in the tile
      float s[C::WN / 8][4];
#pragma unroll
      for (int i = 0; i < C::WN / 8; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
      if constexpr (C::FP8) {
#pragma unroll
        for (int b = 0; b < DP / 64; b++)
#pragma unroll
          for (int nt = 0; nt < C::WN / 8; nt++) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(kt + unit_at<C::ROWB, true>(key0 + nt * 8 + g, b * 4 + tg)));
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
              const uint32_t b0 = fp8x2_to_f16x2<KV>(w[ks] & 0xFFFFu), b1 = fp8x2_to_f16x2<KV>(w[ks] >> 16);
              if constexpr (QREG) {
                mma<true>(s[nt], qf[b * 4 + ks], b0, b1);
              } else {
                uint32_t a[4];
                load_q(b * 4 + ks, a);
                mma<true>(s[nt], a, b0, b1);
              }
            }
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ks++) {
          uint32_t a[4];
          if constexpr (QREG) a[0] = qf[ks][0], a[1] = qf[ks][1], a[2] = qf[ks][2], a[3] = qf[ks][3];
          else load_q(ks, a);
#pragma unroll
          for (int np = 0; np < C::WN / 16; np++) {
            uint32_t b[4];
            ldsm4(kt + unit_at<C::ROWB, false>(key0 + np * 16 + ((lane >> 4) << 3) + (lane & 7), ks * 2 + ((lane >> 3) & 1)), b);
            mma<C::MF16>(s[2 * np], a, b[0], b[1]);
            mma<C::MF16>(s[2 * np + 1], a, b[2], b[3]);
          }
        }
      }
      // scores in log2 units; hidden keys to -inf
      const int k0 = tl.at(cur) * BN;
      const bool bad = s_bad[slot * 2] | s_bad[slot * 2 + 1];
      const bool whole = k0 + BN - 1 <= pos_lo && !bad &&
                         (p.window <= 0 || pos_hi - k0 < p.window || k0 + BN - 1 < p.sinks);
#pragma unroll
      for (int i = 0; i < C::WN / 8; i++) {
        s[i][0] *= sc0, s[i][1] *= sc0, s[i][2] *= sc1, s[i][3] *= sc1;
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < C::WN / 8; i++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const int kk = key0 + i * 8 + tg * 2 + x;
            const bool has = !bad || s_off[slot * BN + kk] >= 0;
            if (!(has && visible(p, k0 + kk, pos0))) s[i][x] = -INFINITY;
            if (!(has && visible(p, k0 + kk, pos1))) s[i][2 + x] = -INFINITY;
          }
      }
      float n0 = m0, n1 = m1;
#pragma unroll
      for (int i = 0; i < C::WN / 8; i++) {
        n0 = fmaxf(n0, fmaxf(s[i][0], s[i][1]));
        n1 = fmaxf(n1, fmaxf(s[i][2], s[i][3]));
      }
      n0 = fmaxf(n0, __shfl_xor_sync(~0u, n0, 1));
      n0 = fmaxf(n0, __shfl_xor_sync(~0u, n0, 2));
      n1 = fmaxf(n1, __shfl_xor_sync(~0u, n1, 1));
      n1 = fmaxf(n1, __shfl_xor_sync(~0u, n1, 2));
      const float b0 = n0 == -INFINITY ? 0.0f : n0 - C::SHIFT, b1 = n1 == -INFINITY ? 0.0f : n1 - C::SHIFT;
      const float a0 = ex2(m0 - C::SHIFT - b0), a1 = ex2(m1 - C::SHIFT - b1);
      m0 = n0;
      m1 = n1;
      l0 *= a0;
      l1 *= a1;
#pragma unroll
      for (int i = 0; i < DP / 8; i++) {
        o[i][0] *= a0, o[i][1] *= a0, o[i][2] *= a1, o[i][3] *= a1;
      }
#pragma unroll
      for (int i = 0; i < C::WN / 8; i++) {
        s[i][0] = ex2(s[i][0] - b0);
        s[i][1] = ex2(s[i][1] - b0);
        s[i][2] = ex2(s[i][2] - b1);
        s[i][3] = ex2(s[i][3] - b1);
        l0 += s[i][0] + s[i][1];
        l1 += s[i][2] + s[i][3];
      }
#pragma unroll
      for (int kk = 0; kk < C::WN / 16; kk++) {
        const uint32_t a[4] = {pack2<C::MF16>(s[2 * kk][0], s[2 * kk][1]), pack2<C::MF16>(s[2 * kk][2], s[2 * kk][3]),
                               pack2<C::MF16>(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                               pack2<C::MF16>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        const int key = key0 + kk * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
        if constexpr (C::FP8) {
#pragma unroll
          for (int cp = 0; cp < DP / 32; cp++) {
            uint32_t w[4];
            ldsm4t(vt + unit_at<C::ROWB, false>(key, cp * 2 + (lane >> 4)), w);
#pragma unroll
            for (int e = 0; e < 2; e++) {     // unit cp * 2 + e: its even dims, then its odd dims
              uint32_t x, y;
              asm("prmt.b32 %0, %1, 0, 0x3120;" : "=r"(x) : "r"(w[2 * e]));
              asm("prmt.b32 %0, %1, 0, 0x3120;" : "=r"(y) : "r"(w[2 * e + 1]));
              mma<true>(o[cp * 4 + e * 2], a, fp8x2_to_f16x2<KV>(x & 0xFFFFu), fp8x2_to_f16x2<KV>(y & 0xFFFFu));
              mma<true>(o[cp * 4 + e * 2 + 1], a, fp8x2_to_f16x2<KV>(x >> 16), fp8x2_to_f16x2<KV>(y >> 16));
            }
          }
        } else {
#pragma unroll
          for (int dp = 0; dp < DP / 16; dp++) {
            uint32_t b[4];
            ldsm4t(vt + unit_at<C::ROWB, false>(key, dp * 2 + (lane >> 4)), b);
            mma<C::MF16>(o[2 * dp], a, b[0], b[1]);
            mma<C::MF16>(o[2 * dp + 1], a, b[2], b[3]);
          }
        }
      }
      {
        int sl = slot + C::STAGES;
        if (sl >= C::OFFS) sl -= C::OFFS;
        put_offset(sl, next_off, next_bad);
        if (ahead < t_end) {
          n_ahead++;
          ahead = next_live(ahead + 1);
        }
      }
      cur = next_live(cur + 1);
      if (++stage == C::STAGES) stage = 0;
      if (++slot == C::OFFS) slot = 0;
    }
    cp_wait<0>();

    // ---- end of the segment: the warps' results through shared memory
    l0 += __shfl_xor_sync(~0u, l0, 1);
    l0 += __shfl_xor_sync(~0u, l0, 2);
    l1 += __shfl_xor_sync(~0u, l1, 1);
    l1 += __shfl_xor_sync(~0u, l1, 2);
    bool odd = false;                         // infinities or NaN: see odd_rows
#pragma unroll
    for (int i = 0; i < DP / 8; i++)
#pragma unroll
      for (int x = 0; x < 4; x++) odd |= !(fabsf(o[i][x]) < INFINITY);
    const bool careful = __syncthreads_or(odd);
    float *s_o = reinterpret_cast<float *>(ring);  // [NW warps][16 rows][DP]
    float *o0 = s_o + (warp * 16 + g) * DP, *o1 = o0 + 8 * DP;
    if constexpr (C::FP8) {
#pragma unroll
      for (int u2 = 0; u2 < DP / 16; u2++) {
        *reinterpret_cast<float4 *>(o0 + u2 * 16 + tg * 4) = make_float4(o[2 * u2][0], o[2 * u2 + 1][0], o[2 * u2][1], o[2 * u2 + 1][1]);
        *reinterpret_cast<float4 *>(o1 + u2 * 16 + tg * 4) = make_float4(o[2 * u2][2], o[2 * u2 + 1][2], o[2 * u2][3], o[2 * u2 + 1][3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < DP / 8; j++) {
        *reinterpret_cast<float2 *>(o0 + j * 8 + tg * 2) = make_float2(o[j][0], o[j][1]);
        *reinterpret_cast<float2 *>(o1 + j * 8 + tg * 2) = make_float2(o[j][2], o[j][3]);
      }
    }
    if (tg == 0) {
      s_base[warp * 16 + g] = m0 - C::SHIFT;
      s_base[warp * 16 + g + 8] = m1 - C::SHIFT;
      s_sum[warp * 16 + g] = l0;
      s_sum[warp * 16 + g + 8] = l1;
    }
    __syncthreads();
    const bool begins = t_begin == 0, ends = t_end == tiles_n;
    const float vs = C::FP8 && p.vs ? __ldg(p.vs + p.vs_step * h) : 1.0f;
    float *part = p.part + (c * 2 + (begins ? 1 : 0)) * (int64_t)(C::MR * (DP + 2));
    if (tid == 0 && begins && !ends)
      p.desc[c] = PartDesc{rows, row0, h, rq.start, sh.block_of(seg_start + tiles_n - 1) - (int)c + 1, 1};
    for (int i = tid; i < rows * (DP / 4); i += THREADS) {
      const int row = i / (DP / 4), d4 = (i % (DP / 4)) * 4;
      const int at = (row >> 4) * C::KW * 16 + (row & 15);
      float base = s_base[at];
#pragma unroll
      for (int w = 1; w < C::KW; w++) base = fmaxf(base, s_base[at + w * 16]);
      const float ref = base == -INFINITY ? 0.0f : base;
      float l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < C::KW; w++) {
        const float f = ex2(s_base[at + w * 16] - ref);
        const float4 v = *reinterpret_cast<const float4 *>(s_o + (at + w * 16) * DP + d4);
        l += f * s_sum[at + w * 16];
        x[0] += f * v.x, x[1] += f * v.y, x[2] += f * v.z, x[3] += f * v.w;
      }
      if (careful && d4 == 0) s_qscale[row] = l;
      if (begins && ends) {
        if (d4 < p.d) {
          const float inv = l == 0.0f ? 0.0f : vs / l;
          const int qr = row0 + row, tok = rq.start + qr / p.group, head = h * p.group + qr % p.group;
          uint16_t *out = p.out + (int64_t)tok * p.o_tok + (int64_t)head * p.o_head + d4;
          *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<F16>(x[0] * inv, x[1] * inv), pack2<F16>(x[2] * inv, x[3] * inv));
        }
      } else {
        *reinterpret_cast<float4 *>(part + row * DP + d4) = make_float4(x[0], x[1], x[2], x[3]);
        if (d4 == 0) {
          part[C::MR * DP + row] = base;
          part[C::MR * DP + C::MR + row] = l;
        }
      }
    }
    if (careful) {                            // each warp looks through its share of the rows
      __syncthreads();
      const int row = warp + NW * lane;
      const bool mine = lane < C::MR / NW && row < rows;
      const SegmentRows<BN> seg_rows{r, rq.start, rq.first, h, row0, tl, t_begin, t_end};
      odd_rows<F16, KV, DP, BN>(p, seg_rows, row, mine, mine ? s_qscale[row] : 0.0f, begins && ends, part, C::MR, nullptr);
    }
  }
}

struct Variant {
  void (*main)(AttnParams);
  void (*merge)(AttnParams);
  int threads, smem, per_sm, rows;
  bool few;
};
template <bool F16, int KV, int DP, int NG>
Variant few() {
  using C = Few<F16, KV, DP, NG>;
  return {paged_few_kernel<F16, KV, DP, NG>, paged_merge_kernel<F16, DP, C::MR>, THREADS, C::SMEM, C::PER_SM, C::MR, true};
}
template <bool F16, int KV, int DP, int RW = 4, int NW = 4>
Variant many() {
  using C = Cfg<F16, KV, DP, RW, NW>;
  return {paged_attention_kernel<F16, KV, DP, RW, NW>, paged_merge_kernel<F16, DP, C::MR>, C::THREADS, C::SMEM, DP == 256 ? 1 : 2, C::MR, false};
}
// `rows`: query rows of the longest request (a request with more is served in several row tiles).
template <bool F16, int KV>
Variant pick(int dp, int64_t rows) {
  if (dp == 64)
    return rows <= 8    ? few<F16, KV, 64, 1>()
           : rows <= 16 ? few<F16, KV, 64, 2>()
           : rows <= 32 ? few<F16, KV, 64, 4>()
           : rows <= 48 ? few<F16, KV, 64, 6>()
           : rows <= 64 ? few<F16, KV, 64, 8>()
                        : many<F16, KV, 64>();
  if (dp == 128)
    return rows <= 8    ? few<F16, KV, 128, 1>()
           : rows <= 16 ? few<F16, KV, 128, 2>()
           : rows <= 32 ? few<F16, KV, 128, 4>()
                        : many<F16, KV, 128>();
  return rows <= 8    ? few<F16, KV, 256, 1>()
         : rows <= 16 ? few<F16, KV, 256, 2>()
         : rows <= 32 ? many<F16, KV, 256, 2, 8>()
         : rows <= 64 ? many<F16, KV, 256, 4, 8>()
                      : many<F16, KV, 256, 8, 8>();
}
Variant variant_for(bool f16, int cache_dtype, int dp, int64_t rows) {
  if (cache_dtype == FP8B200_E4M3) return f16 ? pick<true, FP8B200_E4M3>(dp, rows) : pick<false, FP8B200_E4M3>(dp, rows);
  if (cache_dtype == FP8B200_E5M2) return f16 ? pick<true, FP8B200_E5M2>(dp, rows) : pick<false, FP8B200_E5M2>(dp, rows);
  return f16 ? pick<true, FP8B200_F16>(dp, rows) : pick<false, FP8B200_BF16>(dp, rows);
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

}  // namespace
}  // namespace paged
}  // namespace fp8b200

// Requests with more query rows than TC_OVER (tokens x group) go to the
// tensor-memory kernel when the longest has more than TC_FROM and the head
// size is at most 128. Both sides, in graphs, this file's kernel -> that one:
//   96 rows, 24 requests x 24 tokens over 4000 keys, 32 / 8 heads of 128, bf16: 247 -> 115 us
//   64 rows, 24 x 16: 141 -> 113 us; 1 x 16 over 2000: 25.9 -> 20.6 us
//   36 rows, 24 x 9: 130 -> 110 us; 20 rows, 24 x 5 in e4m3: 94 -> 117 us
//   96 rows, 24 x 12, 16 / 2 heads of 64: 53 -> 36 us; 1 x 12 over 30000: 33.5 -> 49.3 us
//   48 rows, 24 x 6, 16 / 2 heads of 64: 39.2 -> 35.0 us; 1 x 6 over 2000: 18.0 -> 18.5 us
// so 64 suits the small head sizes; at 128 the limit lies near 32.
// Beside a chunk of 512 rows over 2000 keys, short requests there:
//   32 rows, 16 x 8 over 4000, 32 / 8 heads of 128, bf16: 229 -> 113 us, e4m3 172 -> 129 us
//   16 rows, 16 x 4: bf16 145 -> 112 us, e4m3 130 -> 129 us; 40 x 4 over 2000 in e4m3 143 -> 157 us
static constexpr int64_t TC_FROM = 64, TC_OVER = 16;
// Two parts a block (64 rows by two blocks an SM, 16 by four, ...: at most 128 rows an SM) and a descriptor.
static int64_t paged_generic_workspace(int dp, int sms) { return (int64_t)sms * (2 * 128 * (int64_t)(dp + 2) * 4 + 4 * (int64_t)sizeof(fp8b200::paged::PartDesc)); }

extern "C" int64_t fp8b200_paged_attention_workspace(int head_dim, int64_t max_rows) {
  using namespace fp8b200;
  using namespace fp8b200::paged;
  int dev;
  if (int rc = check_device(&dev)) return rc;
  if (head_dim < 16 || head_dim > 256) return set_error(FP8B200_EINVAL, "paged_attention: head_dim must be in 16 .. 256");
  const int dp = padded_dim(head_dim), sms = current_sm_count();
  return paged_generic_workspace(dp, sms) + (dp <= 128 && max_rows > TC_FROM ? tc_workspace(dp, sms) : 0);
}

extern "C" int fp8b200_paged_attention(const void *q, int dtype, int64_t q_stride_token, int64_t q_stride_head,
                                       int64_t tokens, int n_q_heads, int n_kv_heads, int head_dim, const void *k_cache,
                                       const void *v_cache, int cache_dtype, int64_t pages, int64_t page_size,
                                       int64_t stride_page, int64_t stride_slot, int64_t stride_head,
                                       const int32_t *block_table, int64_t table_ld, int64_t table_cols,
                                       const int32_t *cu_new, const int32_t *kv_lens, int64_t requests, float scale,
                                       const float *k_scale, int k_scale_step, const float *v_scale, int v_scale_step,
                                       int window, int sinks, int64_t max_new, void *out, int64_t out_stride_token,
                                       int64_t out_stride_head, int zero_rest, void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace fp8b200;
  using namespace fp8b200::paged;
  if (dtype != FP8B200_BF16 && dtype != FP8B200_F16)
    return set_error(FP8B200_EINVAL, "paged_attention: q must be bf16 or f16");
  const bool fp8 = cache_dtype == FP8B200_E4M3 || cache_dtype == FP8B200_E5M2;
  if (!fp8 && cache_dtype != dtype)
    return set_error(FP8B200_EINVAL, "paged_attention: the cache must be float8 or of q's type");
  if (tokens < 0 || requests < 0 || pages < 0 || table_cols < 0 || max_new < 0)
    return set_error(FP8B200_EINVAL, "paged_attention: negative size");
  if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads)
    return set_error(FP8B200_EINVAL, "paged_attention: %d query heads over %d key/value heads", n_q_heads, n_kv_heads);
  if (head_dim < 16 || head_dim > 256 || head_dim % 16)
    return set_error(FP8B200_EINVAL, "paged_attention: head_dim=%d must be a multiple of 16 up to 256", head_dim);
  if (page_size < 1 || page_size > INT32_MAX || requests > INT32_MAX || table_cols > INT32_MAX ||
      tokens * (__int128)n_q_heads > INT32_MAX)
    return set_error(FP8B200_EINVAL, "paged_attention: page_size below 1, or a size of 2^31 or more");
  if (table_ld < table_cols) return set_error(FP8B200_EINVAL, "paged_attention: block-table rows overlap");
  if (window < 0 || sinks < 0) return set_error(FP8B200_EINVAL, "paged_attention: window and sinks must not be negative");
  const int64_t cunit = fp8 ? 16 : 8;
  if (q_stride_token % 8 || q_stride_head % 8 || out_stride_token % 8 || out_stride_head % 8)
    return set_error(FP8B200_EINVAL, "paged_attention: q and out strides must be multiples of 8 elements");
  if (stride_page % cunit || stride_slot % cunit || stride_head % cunit)
    return set_error(FP8B200_EINVAL, "paged_attention: cache strides must be multiples of 16 bytes");
  if (tokens == 0) return FP8B200_OK;
  if (!q || !out || !cu_new || !workspace || (pages && (!k_cache || !v_cache)) ||
      (requests && (!kv_lens || (table_cols && !block_table))))
    return set_error(FP8B200_EINVAL, "paged_attention: null pointer");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
    return set_error(FP8B200_EINVAL, "paged_attention: tensors must be 16-byte aligned");
  const int64_t group = n_q_heads / n_kv_heads;
  const int64_t most = std::min(max_new > 0 ? max_new : tokens, tokens) * group;  // query rows of the longest request
  const int64_t need = fp8b200_paged_attention_workspace(head_dim, most);
  if (need < 0) return (int)need;
  if (workspace_bytes < need)
    return set_error(FP8B200_EINVAL, "paged_attention: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes,
                     (long long)need);
  int dev;
  if (int rc = check_device(&dev)) return rc;
  const int blocks_max = 4 * current_sm_count();
  AttnParams p{};
  p.q = (const uint16_t *)q;
  p.q_tok = q_stride_token, p.q_head = q_stride_head;
  p.out = (uint16_t *)out;
  p.o_tok = out_stride_token, p.o_head = out_stride_head;
  p.k = (const uint8_t *)k_cache, p.v = (const uint8_t *)v_cache;
  p.s_page = stride_page, p.s_slot = stride_slot, p.s_head = stride_head;
  p.pages = pages;
  p.page = (int)page_size;
  p.table = block_table;
  p.table_ld = table_ld;
  p.table_cols = pages ? (int)table_cols : 0;
  p.cu = cu_new, p.kv = kv_lens;
  p.requests = (int)requests;
  p.tokens = (int)tokens;
  p.hq = n_q_heads, p.hk = n_kv_heads, p.group = n_q_heads / n_kv_heads, p.d = head_dim;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.ks = fp8 ? k_scale : nullptr, p.vs = fp8 ? v_scale : nullptr;
  p.ks_step = k_scale_step, p.vs_step = v_scale_step;
  p.window = window, p.sinks = sinks;
  p.zero_rest = zero_rest;
  p.rows_over = 0;
  p.rows_upto = INT32_MAX;
  p.desc = (PartDesc *)workspace;
  p.part = (float *)((uint8_t *)workspace + (int64_t)blocks_max * sizeof(PartDesc));
  const int dp = padded_dim(head_dim);
  const bool f16 = dtype == FP8B200_F16;
  if (dp <= 128 && most > TC_FROM && requests > 0 && tc_takes(p)) {
    // all requests alike: one launch; else the short ones (decoding among chunks) keep the kernel made for them
    const bool alike = max_new > 0 && max_new * requests == tokens;
    AttnParams t = p;
    if (!alike) {
      t.rows_over = TC_OVER;
      p.rows_upto = TC_OVER;
    }
    if (int rc = launch_tc(t, f16, cache_dtype, dp, current_sm_count(), (uint8_t *)workspace + paged_generic_workspace(dp, current_sm_count()),
                           (cudaStream_t)stream))
      return rc;
    if (alike) return FP8B200_OK;
    p.zero_rest = 0;
  }
  // beside chunks nearly all short requests decode one token: their rows are the group
  const int64_t rows = p.rows_upto == TC_OVER ? std::min<int64_t>(p.group <= 8 ? 8 : 16, TC_OVER) : most;
  const Variant v = variant_for(f16, cache_dtype, dp, rows);
  if (int rc = launch_attributes((const void *)v.main, v.smem)) return rc;
  if (int rc = launch_attributes((const void *)v.merge, 0)) return rc;
  const int grid = current_sm_count() * v.per_sm;
  // A line a head against one for all heads, in graphs: one decode of 30000 keys, 32 / 8 heads of 128, bf16 35 and 43 us, 64 of
  // 4000 in e4m3 133 and 137 us; 32 heads of 128, one decode 87 and 91 us, 16 of 100 keys 26.8 and 25.1 us; 64 heads of 64, 64 of
  // 4000 in e4m3 651 and 970 us, in bf16 1066 and 927 us. More heads than a quarter of the grid leave a line under four blocks.
  p.line_heads = v.few && n_kv_heads <= grid / 4 ? 1 : n_kv_heads;
  launch_dependent(v.main, dim3((unsigned)grid), v.threads, v.smem, (cudaStream_t)stream, p);
  p.blocks = grid;
  launch_dependent(v.merge, dim3((unsigned)current_sm_count(), (unsigned)std::max(1, v.rows / 16)), MERGE_THREADS, 0, (cudaStream_t)stream, p);
  count_launch(2);
  return check_launch("paged_attention");
}
