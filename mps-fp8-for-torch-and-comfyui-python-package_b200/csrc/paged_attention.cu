// Causal attention of each request's new tokens over its pages of a
// key/value cache, on warp-level matrix instructions.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j   over the keys j <= p_i with
//         p_i - j < window or j < sinks            (no window: all j <= p_i)
//
// The query heads that share a key/value head are rows of one tile: row
// token * group + g. A block of four warps holds 16 * RW rows and walks tiles
// of 64 keys; the warps split the rows RW ways and each tile's keys 4 / RW
// ways, with a running maximum, sum and output a warp (float32), joined once
// at the end of a segment.
//
// Work: a segment is one row tile of one request under one key/value head;
// its units are its key tiles. All segments' units form one line, which is
// cut into equal shares, one a block (found from the lengths on the GPU: the
// host need not know them, and one long request among short ones is spread
// over all SMs). A block that holds only part of a segment leaves its partial
// result and maximum in the workspace; the merge kernel joins them in the
// order of the keys. Nothing depends on the order in which blocks run.
//
// K and V tiles come through cp.async into a ring of stages (any page size,
// any stride that is a multiple of 16 bytes); float8 codes stay float8 in
// shared memory and become half pairs in registers (cvt, exact), so a float8
// cache moves half the bytes all the way. Bound by the cache's bytes where a
// request has few rows (decoding), else by the matrix instructions.
//
// Rounding: the weights of a tile are rounded to the matrix instruction's
// 16-bit type (bf16 for a bf16 cache, f16 for f16 and float8 ones), scaled by
// 2^15 in f16 so that weights down to 2^-39 of the largest keep their
// precision; sums, maxima and outputs are float32. bf16 queries of a float8
// cache become f16 after an exact power-of-two scaling of the row (the
// largest value in [1, 2): an element loses bits only below 2^-14 of it).
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

template <bool F16, int KV, int DP, int RW>
struct Cfg {
  static constexpr bool FP8 = is_fp8<KV>;
  static constexpr bool MF16 = F16 || FP8;              // operand type of the matrix instructions
  static constexpr int ROWB = DP * (FP8 ? 1 : 2);       // bytes of a key's row in shared memory
  static constexpr int CPR = ROWB / 16;                 // 16-byte units of it
  static constexpr int TILE = BN * ROWB;                // K or V
  // two blocks an SM (head size 256: one), the more bytes in flight the better
  static constexpr int STAGES = FP8 ? (DP == 64 ? 8 : DP == 128 ? (RW == 4 ? 5 : 6) : 3)
                                    : (DP == 64 ? 6 : DP == 128 ? (RW == 4 ? 2 : 3) : 2);
  static constexpr int MR = 16 * RW;                    // rows a block
  static constexpr int KW = 4 / RW;                     // warps that share a tile's keys
  static constexpr int WN = BN / KW;                    // keys a warp
  static constexpr int QROW = DP * 2 + 16;              // bytes of a query row (padded: no bank conflicts)
  static constexpr int RING = STAGES * 2 * TILE;
  static constexpr int OFFS = STAGES + 1;               // slot offsets are found one tile further ahead
  static constexpr int SMEM = RING + MR * QROW + OFFS * BN * 8 + OFFS * 2 * 4 + MR * 4 + 64 * 2 * 4 + 64;
  static constexpr float SHIFT = MF16 ? 15.0f : 0.0f;   // weights are scaled by 2^SHIFT
  static_assert(64 * DP * 4 <= RING, "the warps' outputs fit the drained ring");
};

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

// Units (key tiles x row tiles x heads) of request r; 0 if this launch leaves
// it to another. A request whose mask leaves nothing still has one, which
// writes its zeros.
template <int MR>
__device__ __forceinline__ long long units_of(const AttnParams &p, int r, int &tiles) {
  const Request q = load_request(p, r);
  tiles = 0;
  if (q.n == 0 || !takes(p, q.n)) return 0;
  tiles = max(1, visible_tiles<BN>(p, q.first, q.first + q.n - 1).count());
  const long long row_tiles = ((long long)q.n * p.group + MR - 1) / MR;
  return row_tiles * p.hk * tiles;
}

template <bool F16, int KV, int DP, int RW>
__global__ void __launch_bounds__(THREADS, DP == 256 ? 1 : 2) paged_attention_kernel(const AttnParams p) {
  using C = Cfg<F16, KV, DP, RW>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *ring = smem;
  uint8_t *s_q = ring + C::RING;
  long long *s_off = reinterpret_cast<long long *>(s_q + C::MR * C::QROW);
  int *s_bad = reinterpret_cast<int *>(s_off + C::OFFS * BN);   // [OFFS][2]
  float *s_qscale = reinterpret_cast<float *>(s_bad + C::OFFS * 2);
  float *s_base = s_qscale + C::MR;                             // [4 warps][16 rows]
  float *s_sum = s_base + 64;
  long long *s_scan = reinterpret_cast<long long *>(s_sum + 64);  // 4 warps' totals, then found request and its prefix
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tg = lane & 3;
  const int rw = warp / C::KW, kw = warp % C::KW;
  const uint32_t ring_a = saddr(ring), q_a = saddr(s_q);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int used = (p.d * (C::FP8 ? 1 : 2)) / 16;  // 16-byte units of a key's row that hold values
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this block's share of the line of units
  long long total = 0;
  int tiles_r = 0;
  for (int r = tid; r < p.requests; r += THREADS) total += units_of<C::MR>(p, r, tiles_r);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
  if (lane == 0) s_scan[warp] = total;
  __syncthreads();
  total = s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3];
  __syncthreads();
  if (p.zero_rest) zero_rest(p, blockIdx.x, gridDim.x);
  const long long blocks = min((long long)gridDim.x, total);  // no block is left without a unit between two others
  const long long c = blockIdx.x;
  if (tid == 0) p.desc[c] = make_int4(-1, 0, 0, 0);
  if (c >= blocks) return;
  long long u = c * total / blocks;
  const long long u_end = (c + 1) * total / blocks;
  long long before = 0;                                       // units before the requests looked at
  for (int r0 = 0; r0 < p.requests; r0 += THREADS) {
    const int r = r0 + tid;
    const long long mine = r < p.requests ? units_of<C::MR>(p, r, tiles_r) : 0;
    long long inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long a = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += a;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long base = before;
    for (int w = 0; w < warp; w++) base += s_scan[w];
    const long long all = before + s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3];
    if (base + inc > u && base + inc - mine <= u) {
      s_scan[4] = r;
      s_scan[5] = base + inc - mine;
    }
    __syncthreads();
    before = all;
    if (before > u) break;
  }
  int r = (int)s_scan[4];
  before = s_scan[5];

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
    const int live_from = p.window > 0 ? max(0, pos_lo - p.window + 1) / BN : 0;
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
          cp16(kd, valid ? p.k + byte : p.k, valid);
          cp16(vd, valid ? p.v + byte : p.v, valid);
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
    // query rows
    for (int i = tid; i < C::MR * (DP / 8); i += THREADS) {
      const int row = i / (DP / 8), cu = i % (DP / 8);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < rows && cu * 8 < p.d) {
        const int qr = row0 + row, tok = rq.start + qr / p.group, head = h * p.group + qr % p.group;
        v = __ldg(reinterpret_cast<const uint4 *>(p.q + (int64_t)tok * p.q_tok + (int64_t)head * p.q_head + cu * 8));
      }
      *reinterpret_cast<uint4 *>(s_q + row * C::QROW + cu * 16) = v;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; s++) {
      if (s < n_ahead) issue(s, s);
      cp_commit();
    }
    if constexpr (C::FP8 && !F16) {           // bf16 rows to f16, the largest value in [1, 2)
      for (int row = warp; row < C::MR; row += 4) {
        uint32_t *w = reinterpret_cast<uint32_t *>(s_q + row * C::QROW);
        float a = 0.0f;
        for (int i = lane; i < DP / 2; i += 32)
          a = fmaxf(a, fmaxf(fabsf(u2f(w[i] << 16)), fabsf(u2f(w[i] & 0xFFFF0000u))));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) a = fmaxf(a, __shfl_xor_sync(~0u, a, d));
        uint32_t eb = f2u(a) >> 23;
        eb = (eb == 255u || a == 0.0f) ? 127u : min(max(eb, 1u), 253u);
        const float mul = u2f((254u - eb) << 23);
        for (int i = lane; i < DP / 2; i += 32) w[i] = pack2<true>(u2f(w[i] << 16) * mul, u2f(w[i] & 0xFFFF0000u) * mul);
        if (lane == 0) s_qscale[row] = u2f(eb << 23);
      }
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
    bool odd = false;                         // infinities or NaN: see careful_row
#pragma unroll
    for (int i = 0; i < DP / 8; i++)
#pragma unroll
      for (int x = 0; x < 4; x++) odd |= !(fabsf(o[i][x]) < INFINITY);
    const bool careful = __syncthreads_or(odd);
    float *s_o = reinterpret_cast<float *>(ring);  // [4 warps][16 rows][DP]
    if (!careful) {
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
    } else {
      for (int row = warp; row < rows; row += 4) {
        const int qr = row0 + row, tok = qr / p.group;
        float m, l, ov[DP / 32];
        careful_row<F16, KV, DP, BN>(p, r, rq.start + tok, h * p.group + qr % p.group, rq.first + tok, tl, t_begin, t_end, m, l, ov);
        const int at = (row >> 4) * C::KW * 16 + (row & 15);  // the row's place in its first key warp
#pragma unroll
        for (int i = 0; i < DP / 32; i++) s_o[at * DP + lane + 32 * i] = ov[i];
        if (lane == 0) {
          for (int w = 0; w < C::KW; w++) {
            s_base[at + w * 16] = w == 0 ? m : -INFINITY;
            s_sum[at + w * 16] = w == 0 ? l : 0.0f;
          }
        }
        for (int w = 1; w < C::KW; w++)
          for (int i = lane; i < DP; i += 32) s_o[(at + w * 16) * DP + i] = 0.0f;
      }
    }
    __syncthreads();
    const bool begins = t_begin == 0, ends = t_end == tiles_n;
    const float vs = C::FP8 && p.vs ? __ldg(p.vs + p.vs_step * h) : 1.0f;
    float *part = p.part + (c * 2 + (begins ? 1 : 0)) * (int64_t)(C::MR * (DP + 2));
    if (tid == 0 && begins && !ends)
      p.desc[c] = make_int4(r, qt, h, (int)(((seg_start + tiles_n) * blocks - 1) / total));
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
  }
}

// Joins the parts of the segments that were cut: block c the one that began
// in block c of the attention kernel (its second part), with the first parts
// of the blocks after it, in their order.
template <bool F16, int DP, int MR>
__global__ void __launch_bounds__(THREADS) paged_merge_kernel(const AttnParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long c = blockIdx.x;
  const int4 d = p.desc[c];
  if (d.x < 0) return;
  const Request rq = load_request(p, d.x);
  const int row0 = d.y * MR, h = d.z;
  const int rows = (int)min((long long)MR, (long long)rq.n * p.group - row0);
  const float vs = p.vs ? __ldg(p.vs + p.vs_step * h) : 1.0f;
  constexpr int64_t SLOT = MR * (DP + 2);
  for (int i = threadIdx.x; i < rows * (DP / 4); i += THREADS) {
    const int row = i / (DP / 4), d4 = (i % (DP / 4)) * 4;
    if (d4 >= p.d) continue;
    float base = -INFINITY, l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (long long b = c; b <= d.w; b++) {
      const float *part = p.part + (b * 2 + (b == c ? 1 : 0)) * SLOT;
      const float bb = part[MR * DP + row], bl = part[MR * DP + MR + row];
      const float4 v = *reinterpret_cast<const float4 *>(part + row * DP + d4);
      const float nb = fmaxf(base, bb), ref = nb == -INFINITY ? 0.0f : nb;
      const float f = ex2(base - ref), e = ex2(bb - ref);
      base = nb;
      l = l * f + bl * e;
      x[0] = x[0] * f + v.x * e, x[1] = x[1] * f + v.y * e, x[2] = x[2] * f + v.z * e, x[3] = x[3] * f + v.w * e;
    }
    const float inv = l == 0.0f ? 0.0f : vs / l;
    const int qr = row0 + row, tok = rq.start + qr / p.group, head = h * p.group + qr % p.group;
    uint16_t *out = p.out + (int64_t)tok * p.o_tok + (int64_t)head * p.o_head + d4;
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<F16>(x[0] * inv, x[1] * inv), pack2<F16>(x[2] * inv, x[3] * inv));
  }
}

template <typename P>
cudaError_t launch_pdl(void (*kernel)(P), int grid, int threads, int smem, cudaStream_t st, const P &p) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

struct Variant {
  void (*main)(AttnParams);
  void (*merge)(AttnParams);
  int smem, per_sm;
};
template <bool F16, int KV, int DP, int RW>
Variant variant() {
  return {paged_attention_kernel<F16, KV, DP, RW>, paged_merge_kernel<F16, DP, 16 * RW>, Cfg<F16, KV, DP, RW>::SMEM,
          DP == 256 ? 1 : 2};
}
template <bool F16, int KV>
Variant pick(int dp, int rw) {
  if (dp == 64) return rw == 1 ? variant<F16, KV, 64, 1>() : rw == 2 ? variant<F16, KV, 64, 2>() : variant<F16, KV, 64, 4>();
  if (dp == 128) return rw == 1 ? variant<F16, KV, 128, 1>() : rw == 2 ? variant<F16, KV, 128, 2>() : variant<F16, KV, 128, 4>();
  return rw == 1 ? variant<F16, KV, 256, 1>() : rw == 2 ? variant<F16, KV, 256, 2>() : variant<F16, KV, 256, 4>();
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

}  // namespace
}  // namespace paged
}  // namespace fp8b200

// Requests with more query rows than TC_OVER (tokens x group) go to the
// tensor-memory kernel when the longest has more than TC_FROM and the head
// size is at most 128.
static constexpr int64_t TC_FROM = 64, TC_OVER = 16;
static int64_t paged_generic_workspace(int dp, int sms) { return 2 * (int64_t)sms * (2 * 64 * (int64_t)(dp + 2) * 4 + 16); }

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
  const int blocks_max = 2 * current_sm_count();
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
  p.desc = (int4 *)workspace;
  p.part = (float *)((uint8_t *)workspace + (int64_t)blocks_max * 16);
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
  const int rw = p.rows_upto <= 16 || most <= 16 ? 1 : most <= 32 ? 2 : 4;
  Variant v;
  if (cache_dtype == FP8B200_E4M3) v = f16 ? pick<true, FP8B200_E4M3>(dp, rw) : pick<false, FP8B200_E4M3>(dp, rw);
  else if (cache_dtype == FP8B200_E5M2) v = f16 ? pick<true, FP8B200_E5M2>(dp, rw) : pick<false, FP8B200_E5M2>(dp, rw);
  else v = f16 ? pick<true, FP8B200_F16>(dp, rw) : pick<false, FP8B200_BF16>(dp, rw);
  cudaError_t e = cudaFuncSetAttribute(v.main, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem);
  if (e != cudaSuccess) return check_launch("paged_attention");
  const int grid = current_sm_count() * v.per_sm;
  launch_pdl(v.main, grid, THREADS, v.smem, (cudaStream_t)stream, p);
  launch_pdl(v.merge, grid, THREADS, 0, (cudaStream_t)stream, p);
  count_launch(2);
  return check_launch("paged_attention");
}
