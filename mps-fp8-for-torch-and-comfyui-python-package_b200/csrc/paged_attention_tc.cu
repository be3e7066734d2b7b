// Attention over the pages of a key/value cache for requests with many query
// rows (chunks and prompts), on the 5th-generation tensor cores.
//
// The mathematics, the masks and the segments are those of paged_attention.cu;
// a block of rows is 256 (two tiles of 128: one row per tensor-memory lane),
// a key tile 128. One persistent CTA an SM; its warps:
//   0-7      two softmax groups, one per row tile, a thread a row: S from
//            tensor memory, weights back to it as the second product's A
//            operand, running maximum and sum in registers
//   8-11     float8 caches only: turn the raw codes of a tile into f16 (exact)
// and a warpgroup for control:
//   MMA      issues S = Q K^T and O += P V (a uniform warp, one lane's
//            instructions: the descriptors stay in uniform registers)
//   segments walks the CTA's share of the work and hands its segments on; with a
//            16-bit cache and a group that divides 128 it also brings their rows
//            of Q by TMA boxes (397 -> 364 us at 8 x 2048), else the groups do
//   2 x TMA  in turn bring K and V tiles in, boxes of as many slots as divide
//            both the page and the tile (16 for pages of 16 or 48 slots); boxes
//            without a key are out of the map's bounds and arrive as zeros, a
//            box that runs past the request's last key goes slot by slot, so
//            that what an unwritten slot holds is never multiplied. (Gathering
//            four rows a copy, tile::gather4, for all pages alike took 53
//            cycles a copy: half the speed at 8 x 2048.)
// While one group computes its weights the tensor core works for the other.
// Tensor memory: S of either tile (128 columns each, P over its first 64) and
// O of either tile.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since its
// base was set (the weights stay below 2^8, or 2^15 with the f16 scaling, so
// nothing overflows and the quotient is the same): after the first tiles that
// is rare, and the O accumulator stays in tensor memory.
//
// Work: the units (key tiles, and SEG_COST more for its start and end) of all
// segments in one line, cut into one share a CTA; a cut within a sixteenth of a
// share of a segment's edge moves there, so with many segments none is split,
// and with few all SMs still work.
//
// Bound by the chain S -> weights -> P V -> next S of a row tile, against the
// other's: 256 x 128 scores cost 2048 cycles of MMA at head size 128 and 2048
// cycles of ex2 (16 a cycle), and take about 4100 (tensor pipe busy 49 % of the
// time at 2048 rows over 14001 keys). Measured, 32 / 8 heads of 128: 2048 tokens
// over 14001 cached in e4m3 519 us (972 TFLOP/s), prompts of 8 x 2048 in bf16
// 355 us (775 TFLOP/s; short segments, so their starts and ends count; 309 in a
// graph), 1500 tokens with a window of 4096 and 4 sinks 144 us. SEG_COST of 2 gave
// 351 us on the prompts, 3 gave 364. Slower when they were tried, on the kernel
// whose MMAs still took 100 cycles to issue (540 us for the chunk then), and not
// tried since: two score buffers of 64 keys a row tile (570 us), part of the
// exponentials as a polynomial on the multiply-add pipes (596 us). Dropped for
// good: two threads a row (the registers spill; the float8 forms here spill 272
// to 296 bytes a thread themselves), K and V through cp.async (a proxy fence waits
// for all of a thread's copies), four-row gathers. The time depends on the layout
// of the code: variants of the page masks' few lines that do the same work took
// 304 to 358 us on the prompts in a graph.
//
// No counterpart in the reference.
#include "paged_attention.cuh"

#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>

namespace fp8b200 {
namespace paged {
namespace {

constexpr int KT = 128;          // keys a tile
constexpr int QT = 128;          // rows a tile
constexpr int QB = 2 * QT;       // rows a block
constexpr int SEG_COST = 2;       // what a segment's start and end cost, in key tiles
constexpr int MAX_REQUESTS = 16384;  // their first rows pass through shared memory
constexpr int SEGS = 4;           // segments in the ring
constexpr int HIDE_RING = 8;     // tiles whose page masks are kept: more than the producers run ahead of the softmax

__device__ uint32_t g_paged_status;  // 0, or the site of a wait that ran out

// Tensor maps of the caches, 4-D (head_dim, heads, slots of a page, pages):
// boxes of 2^box_log slots, and of one.
// And of q (head_dim, heads, tokens), boxes of 128 rows of the group's heads.
struct TcMaps {
  CUtensorMap box[2], one[2];  // K, V
  CUtensorMap q;
};

template <bool F16, int KV, int DP>
struct Tc {
  static constexpr bool FP8 = KV == FP8B200_E4M3 || KV == FP8B200_E5M2;
  static constexpr bool MF16 = F16 || FP8;
  static constexpr int TILE = KT * DP * 2;                // K or V tile, Q tile (16-bit)
  static constexpr int CTRL = FP8 ? 12 : 8;               // first warp of the control group
  static constexpr int THREADS = (CTRL + 4) * 32;
  // registers a thread: 128 (168) at launch, moved to the softmax by warpgroup: 2 x 184 + 72 + 72 = 4 x 128
  // (float8), 2 x 216 + 72 = 3 x 168
  static constexpr int REGS_SOFTMAX = FP8 ? 184 : 216, REGS_OTHER = 72;
  static constexpr int SLOTS = DP == 128 ? (FP8 ? 4 : 5) : 8;
  static constexpr int RAWS = FP8 ? (DP == 128 ? 2 : 4) : 0;  // float8: raw tiles on their way
  static constexpr int RAW = KT * 128;                    // rows of 128 bytes: a copy's target must be 128-byte aligned
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_RAW = OFF_KV + SLOTS * TILE;
  static constexpr int OFF_PLAN = OFF_RAW + RAWS * RAW;   // the plan's scratch
  static constexpr int OFF_HIDE = OFF_PLAN + 256;         // page masks, 128 bits a tile
  static constexpr int OFF_BARS = OFF_HIDE + HIDE_RING * 16;
  static constexpr int BARS = 2 * SLOTS + 2 * RAWS + 11 + 2 * SEGS;
  static constexpr int OFF_SEGS = (OFF_BARS + BARS * 8 + 15) / 16 * 16;
  static constexpr int SMEM = OFF_SEGS + SEGS * 48 + 16;
  static constexpr float SHIFT = MF16 ? 7.0f : 0.0f;      // weights are scaled by 2^SHIFT and stay below 2^(SHIFT + 8)
  static constexpr uint32_t FMT = MF16 ? 0u : 1u;
  // f32 accumulator, A and B of one type, M = 128; S: N = 128 keys, B K-major; O: N = DP, B (V) MN-major
  static constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(KT >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t IDESC_O =
      (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((128u >> 4) << 24);
  static_assert(OFF_PLAN >= (MAX_REQUESTS + 1) * 4, "the requests' first rows fit in front of it");
  static_assert(OFF_KV % 1024 == 0 && TILE % 1024 == 0 && OFF_RAW % 1024 == 0 && OFF_PLAN % 16 == 0 && OFF_HIDE % 16 == 0 &&
                    OFF_BARS % 8 == 0 && OFF_SEGS % 16 == 0,
                "swizzled tiles, vector accesses and barriers are aligned");
  static_assert(SMEM <= 232448, "shared memory of one CTA");
};

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded: a wait runs out at the CTA's deadline (behind s_failed), which moves on
// with every key tile of the first softmax group, and with every tile where odd_rows
// keeps the other roles waiting (a wait with a clock of its own takes more code at
// each of its places: 8 x 2048 324 us against 307). It then records its site, tells
// the other roles (s_failed) and holds its thread for 200 us so that copies and MMAs issued
// before it have landed when the CTA tears down.
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t *s_failed, uint32_t site) {
  for (uint32_t n = 1;; n++) {
    if (bar_test(bar, parity)) return true;
    if ((n & 31u) == 0) {
      const bool late = now_ns() > *reinterpret_cast<volatile uint64_t *>(s_failed + 1);
      if (late || *s_failed) {
        if (late) {
          *s_failed = 1;
          atomicCAS(&g_paged_status, 0u, 0x80000000u | site);
        }
        const uint64_t t1 = now_ns();
        while (now_ns() - t1 < 200000ull) __nanosleep(1000);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *s_failed, uint32_t site) {
  if (bar_test(bar, parity)) return true;
  return bar_wait_slow(bar, parity, s_failed, site);
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// MMAs and commits are issued by one thread of a warp that runs the code as a
// whole, elected in the same statement: with any other predicate each MMA took
// 100 cycles to issue, more than an MMA of 128 x 128 x 16 takes to run (64).
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
// Four K steps of 16 along a 128-byte swizzled row: A and B advance by 32 bytes.
__device__ __forceinline__ void mma_ss4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, q;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "add.u64 a1, %1, 2;\n\tadd.u64 b1, %2, 2;\n\t"
      "add.u64 a2, %1, 4;\n\tadd.u64 b2, %2, 4;\n\t"
      "add.u64 a3, %1, 6;\n\tadd.u64 b3, %2, 6;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Four K steps of 16 keys: A (tensor memory) advances by 8 columns, B by 16 rows of 128 bytes.
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, q;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u64 b1, %2, 128;\n\t"
      "add.u32 a2, %1, 16;\n\tadd.u64 b2, %2, 256;\n\t"
      "add.u32 a3, %1, 24;\n\tadd.u64 b3, %2, 384;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
#define PAGED_R32(r)                                                                                                   \
  "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),          \
      "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),           \
      "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),          \
      "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
__device__ __forceinline__ void tld32(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Waits for the loads issued before it; r is an operand so that no use of it moves ahead.
__device__ __forceinline__ void tld_wait(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : PAGED_R32(r) : : "memory");
}
__device__ __forceinline__ void tst32(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tst16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tst_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptors, 128-byte swizzle. K-major (Q, K): rows of
// 64 values, 8-row groups 1024 bytes apart. MN-major (V): 8 keys x 64 dims an
// atom, 8-key groups 1024 bytes apart (stride), 64-dim blocks `lead` apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t a, uint32_t lead) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box of the pool: columns x .., key/value head h, slots off .. of one page.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int x, int h, int off, int page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(h), "r"(off), "r"(page), "r"(bar)
      : "memory");
}
// Columns x .. of the group's heads from h on, of the tokens from tok on.
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap *map, int x, int h, int tok, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(h), "r"(tok), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t *>(&d))
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t *>(&d))
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
  return d;
}

// ---- the line of units
// Blocks of rows have places x: request r's from place(r) on, where place(r)
// = floor(rows before r / 256) + r leaves room for its last, partial block
// (some places stay empty). A place's segments, one a key/value head, follow
// one another; a segment's units are the key tiles its 256 rows can see, and
// SEG_COST behind them.
__device__ __forceinline__ int place(const AttnParams &p, int start, int r) {
  return (int)((int64_t)start * p.group / QB) + r;
}
struct Block {
  Request rq;
  Tiles<KT> tl;
  int qt, tiles;  // 0 tiles: the place is empty
  __device__ __forceinline__ int units() const { return tiles ? tiles + SEG_COST : 0; }
};
__device__ __forceinline__ Block block_at(const AttnParams &p, const Request &rq, int qt) {
  Block b;
  b.rq = rq;
  b.qt = qt;
  const int64_t rows = (int64_t)rq.n * p.group;
  b.tiles = 0;
  b.tl = Tiles<KT>{0, 0, 0};
  if (rq.n == 0 || !takes(p, rq.n) || (int64_t)qt * QB >= rows) return b;
  const int last = (int)(min(rows, (int64_t)(qt + 1) * QB) - 1);
  b.tl = visible_tiles<KT>(p, rq.first + qt * QB / p.group, rq.first + last / p.group);
  b.tiles = max(1, b.tl.count());
  return b;
}
// Within a request the last blocks, which see the most keys, come first.
__device__ __forceinline__ Block block_of_place(const AttnParams &p, int r, int x) {
  const Request rq = load_request(p, r);
  const int64_t n = ((int64_t)rq.n * p.group + QB - 1) / QB;
  const int i = x - place(p, rq.start, r);
  if (i < 0 || i >= n) {
    Block b;
    b.rq = rq, b.qt = 0, b.tiles = 0;
    b.tl = Tiles<KT>{0, 0, 0};
    return b;
  }
  return block_at(p, rq, (int)(n - 1) - i);
}

// A segment, or the part of it that falls into this CTA's share.
struct alignas(16) Segment {
  int r, h, qt;                // request (-1: no more segments), key/value head, block of rows
  int start, n, first;         // the request's new tokens (see Request)
  int t_begin, t_end, units;   // key tiles [t_begin, t_end) of `units` tiles
  int sinks, from;             // list entry i is key tile i < sinks ? i : from + i - sinks
  int last;                    // if the part begins the segment and does not end it: the CTA that ends it
  __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : from + i - sinks; }
  __device__ __forceinline__ Tiles<KT> tiles() const { return Tiles<KT>{sinks, from, 0}; }
};
static_assert(sizeof(Segment) == 48, "SEGS * 48 bytes");

template <bool F16, int KV, int DP>
__global__ void __launch_bounds__((Tc<F16, KV, DP>::THREADS), 1)
    paged_attention_tc_kernel(const AttnParams p, const __grid_constant__ TcMaps maps, const int box_log,
                              const int q_boxes) {
  using C = Tc<F16, KV, DP>;
  constexpr int TC_THREADS = C::THREADS;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base_a = saddr(smem);
  const uint32_t kv_a = base_a + C::OFF_KV, raw_a = base_a + C::OFF_RAW;
  uint32_t *s_hide = reinterpret_cast<uint32_t *>(smem + C::OFF_HIDE);    // [HIDE_RING][4]
  const uint32_t bars = base_a + C::OFF_BARS;
  Segment *s_seg = reinterpret_cast<Segment *>(smem + C::OFF_SEGS);
  uint32_t *s_misc = reinterpret_cast<uint32_t *>(smem + C::OFF_SEGS + SEGS * 48);  // tensor memory base, failed flag, deadline (64 bits)
  volatile uint32_t *s_failed = s_misc + 1;
  volatile uint64_t *s_deadline = reinterpret_cast<volatile uint64_t *>(s_misc + 2);
  auto kv_full = [&](int s) { return bars + 8u * s; };
  auto kv_empty = [&](int s) { return bars + 8u * (C::SLOTS + s); };
  auto raw_full = [&](int s) { return bars + 8u * (2 * C::SLOTS + s); };
  auto raw_empty = [&](int s) { return bars + 8u * (2 * C::SLOTS + C::RAWS + s); };
  const uint32_t q_full = bars + 8u * (2 * C::SLOTS + 2 * C::RAWS), s_full = q_full + 16, p_full = q_full + 32, pv_done = q_full + 48;
  const uint32_t p_half = q_full + 64, q_free = q_full + 80, seg_full = q_full + 88, seg_empty = seg_full + 8 * SEGS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (base_a & 1023u) {  // the swizzled tiles need it; the same for every CTA
    if (tid == 0) atomicCAS(&g_paged_status, 0u, 0x80000000u | 99u);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < C::SLOTS; s++) {
      bar_init(kv_full(s), C::FP8 ? 128 : 1);
      bar_init(kv_empty(s), 1);
    }
    for (int s = 0; s < C::RAWS; s++) {
      bar_init(raw_full(s), 1);
      bar_init(raw_empty(s), 128);
    }
    for (int g = 0; g < 2; g++) {
      bar_init(q_full + 8 * g, q_boxes ? 1 : QT);
      bar_init(s_full + 8 * g, 1);
      bar_init(p_half + 8 * g, QT);
      bar_init(p_full + 8 * g, QT);
      bar_init(pv_done + 8 * g, 1);
    }
    bar_init(q_free, 1);
    for (int i = 0; i < SEGS; i++) {
      bar_init(seg_full + 8 * i, 1);
      bar_init(seg_empty + 8 * i, C::FP8 ? 15 : 11);  // the warps that read it: softmax, converting, MMA, TMA
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *s_failed = 0;
  }
  if (warp == C::CTRL) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(s_misc)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this CTA's share; the requests' first rows in shared memory that Q and K take over later
  int *s_start = reinterpret_cast<int *>(smem);  // [requests + 1]
  long long *s_sum = reinterpret_cast<long long *>(smem + C::OFF_PLAN);                 // [warps]
  long long(*s_found)[4] = reinterpret_cast<long long(*)[4]>(s_sum + TC_THREADS / 32);  // cut, place, units before it, request
  for (int r = tid; r <= p.requests; r += TC_THREADS) {
    s_start[r] = r < p.requests ? load_request(p, r).start : p.tokens;
    fence_async();  // Q and K arrive over it through TMA
  }
  if (tid < 2) s_found[tid][0] = -1;
  if (tid == 0) *s_deadline = now_ns() + p.wait_ns;
  __syncthreads();
  const int places = p.requests == 0 ? 0 : place(p, min(max(__ldg(p.cu + p.requests), 0), p.tokens), p.requests);
  auto request_of = [&](int x) {
    int lo = 0, hi = p.requests;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (place(p, s_start[mid], mid) <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  long long total = 0;
  for (int x = tid; x < places; x += TC_THREADS) total += (long long)block_of_place(p, request_of(x), x).units() * p.hk;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  total = 0;
  for (int i = 0; i < TC_THREADS / 32; i++) total += s_sum[i];
  __syncthreads();
  if (p.zero_rest) zero_rest(p, blockIdx.x, gridDim.x);
  const long long ctas = min((long long)gridDim.x, total), c = blockIdx.x;
  if (tid == 0) p.desc[c].rows = 0;
  const long long slack = ctas > 0 ? total / ctas / 16 : 0;
  long long u = 0, u_end = 0, u_before = 0;      // the share, and the units before place x
  int u_x = 0, u_r = 0;
  if (c < ctas) {
    const long long raw[2] = {c * total / ctas, (c + 1) * total / ctas};
    long long before = 0;
    for (int x0 = 0; x0 < places; x0 += TC_THREADS) {
      const int x = x0 + tid;
      const int r = x < places ? request_of(x) : 0;
      Block blk;
      blk.tiles = 0;
      if (x < places) blk = block_of_place(p, r, x);
      const int units = blk.units();
      const long long mine = (long long)units * p.hk;
      long long inc = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long a = __shfl_up_sync(~0u, inc, d);
        if (lane >= d) inc += a;
      }
      if (lane == 31) s_sum[warp] = inc;
      __syncthreads();
      long long b = before + inc - mine, all = before;
      for (int w = 0; w < TC_THREADS / 32; w++) {
        if (w < warp) b += s_sum[w];
        all += s_sum[w];
      }
#pragma unroll
      for (int k = 0; k < 2; k++)
        if (raw[k] >= b && raw[k] < b + mine) {
          const long long in = (raw[k] - b) % units;  // of the segment that the cut falls into
          long long cut = raw[k];
          if (in <= slack) cut -= in;
          else if (in >= blk.tiles - slack) cut += units - in;
          s_found[k][0] = cut, s_found[k][1] = x, s_found[k][2] = b, s_found[k][3] = r;
        }
      __syncthreads();
      before = all;
      if (before > raw[1]) break;
    }
    u = s_found[0][0];
    u_end = raw[1] >= total ? total : s_found[1][0];
    u_x = (int)s_found[0][1];
    u_before = s_found[0][2];
    u_r = (int)s_found[0][3];
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(s_misc);
  // tensor memory columns: S (P) of tile g at 128 g, O of tile g at 256 + DP g

  // The segment in ring place n % SEGS once it is there; 0 if the wait ran out.
  auto seg_at = [&](uint32_t n, uint32_t site) -> const Segment * {
    if (!bar_wait(seg_full + 8 * (n % SEGS), (n / SEGS) & 1, s_failed, site)) return nullptr;
    return s_seg + n % SEGS;
  };
  if (warp >= C::CTRL) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHER));
    if (warp == C::CTRL + 1) {
      // ================================================= the share's segments
      if (lane == 0) {
        uint32_t n = 0;
        bool more = true;
        while (more) {
          Segment sg;
          sg.r = -1;
          while (u < u_end && u_r < p.requests) {
            const Block b = block_of_place(p, u_r, u_x);
            const int units = b.units();
            const long long all = (long long)units * p.hk;
            if (u < u_before + all) {
              const int local = (int)(u - u_before);       // units of one place: below 2^31
              sg.r = u_r, sg.h = local / units, sg.qt = b.qt;
              sg.start = b.rq.start, sg.n = b.rq.n, sg.first = b.rq.first;
              sg.t_begin = local - sg.h * units;
              sg.t_end = (int)min((long long)b.tiles, sg.t_begin + (u_end - u));
              sg.units = b.tiles, sg.sinks = b.tl.sinks, sg.from = b.tl.from;
              const long long tiles_end = u - sg.t_begin + b.tiles;
              sg.last = 0;
              if (sg.t_begin == 0 && sg.t_end < b.tiles) {
                long long last = c + 1;                    // the CTA whose share reaches the segment's end
                while (last + 1 < ctas && (last + 1) * total / ctas < tiles_end - slack) last++;
                sg.last = (int)last;
              }
              u = sg.t_end == b.tiles ? tiles_end + SEG_COST : u + (sg.t_end - sg.t_begin);
              break;
            }
            u_before += all;
            u_x++;
            while (u_r + 1 < p.requests && u_x >= place(p, load_request(p, u_r + 1).start, u_r + 1)) u_r++;
            // behind the last request's places nothing is left (only if the offsets make no sense)
            if (u_r + 1 == p.requests && b.tiles == 0 &&
                (long long)(u_x - place(p, b.rq.start, u_r)) * QB > (long long)b.rq.n * p.group + QB)
              break;
          }
          if (n >= SEGS && !bar_wait(seg_empty + 8 * (n % SEGS), ((n / SEGS) & 1) ^ 1, s_failed, 50)) break;
          s_seg[n % SEGS] = sg;
          bar_arrive(seg_full + 8 * (n % SEGS));
          if (!C::FP8 && q_boxes && sg.r >= 0) {           // its rows of Q, once the last S of the segment before has read those
            if (n > 0 && !bar_wait(q_free, (n - 1) & 1, s_failed, 56)) break;
            for (int g = 0; g < 2; g++) {
              const int tok = sg.start + (sg.qt * QB + g * QT) / p.group;
              bar_expect(q_full + 8 * g, C::TILE);
              for (int b = 0; b < DP / 64; b++)
                load_rows(base_a + g * C::TILE + b * (QT * 128), &maps.q, b * 64, sg.h * p.group, tok, q_full + 8 * g);
            }
          }
          more = sg.r >= 0;
          n++;
        }
      }
      __syncwarp();
    } else if (warp == C::CTRL) {
      // ================================================= MMA issue
      int slot = 0;
      uint32_t phase = 0, segs = 0, tiles = 0;
      bool ok = true;
      auto step = [&]() {
        if (++slot == C::SLOTS) slot = 0, phase ^= 1;
      };
      auto issue_s = [&](int g, int s) {
        const uint64_t qd = desc_k(base_a + g * C::TILE), kd = desc_k(kv_a + s * C::TILE);
#pragma unroll
        for (int k = 0; k < DP / 64; k++)
          mma_ss4(tmem + 128 * g, qd + k * (KT * 128 / 16), kd + k * (KT * 128 / 16), C::IDESC_S, k > 0);
        commit(s_full + 8 * g);
      };
      while (ok) {
        const Segment *sg = seg_at(segs, 51);
        if (!__all_sync(~0u, sg != nullptr) || sg->r < 0) break;
        const int n = sg->t_end - sg->t_begin;
        __syncwarp();
        if (lane == 0) bar_arrive(seg_empty + 8 * (segs % SEGS));
        ok = bar_wait(q_full, segs & 1, s_failed, 1) && bar_wait(q_full + 8, segs & 1, s_failed, 2) &&
             bar_wait(kv_full(slot), phase, s_failed, 3);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        fence_after();
        issue_s(0, slot);
        issue_s(1, slot);
        commit(kv_empty(slot));
        if (n == 1) commit(q_free);
        step();
        for (int j = 0; j < n && ok; j++) {
          const bool more = j + 1 < n;
          const int ks = slot;
          if (more) {
            ok = bar_wait(kv_full(ks), phase, s_failed, 4);
            step();
          }
          const int vs = slot;
          ok = ok && bar_wait(kv_full(vs), phase, s_failed, 5);
          step();
#pragma unroll 1
          for (int g = 0; g < 2; g++) {
            ok = ok && bar_wait(p_half + 8 * g, tiles & 1, s_failed, 6 + g);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            fence_after();
            const uint64_t vd = desc_mn(kv_a + vs * C::TILE, KT * 128);
            mma_ts4(tmem + 256 + DP * g, tmem + 128 * g, vd, C::IDESC_O, j > 0);
            ok = bar_wait(p_full + 8 * g, tiles & 1, s_failed, 8 + g);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            fence_after();
            mma_ts4(tmem + 256 + DP * g, tmem + 128 * g + 32, vd + 512, C::IDESC_O, 1);
            commit(pv_done + 8 * g);
            if (more) issue_s(g, ks);
          }
          if (!ok) break;
          commit(kv_empty(vs));
          if (more) commit(kv_empty(ks));
          if (j + 2 == n) commit(q_free);                  // the segment's last S is issued
          tiles++;
        }
        segs++;
      }
    } else {
      // ================================================= K and V tiles, in turn: K 0, K 1, V 0, K 2, V 1, ...
      const uint32_t turn = warp - (C::CTRL + 2);
      // float8 tiles go to the raw ring, 16-bit ones straight to the operands' ring
      constexpr int RING = C::FP8 ? C::RAWS : C::SLOTS;
      uint32_t filled = 0, tiles = 0;
      bool ok = !p.no_tiles;
      for (uint32_t segs = 0; ok; segs++) {
        const Segment *sg = seg_at(segs, 52);
        if (!__all_sync(~0u, sg != nullptr) || sg->r < 0) break;
        const int r = sg->r, h = sg->h, n = sg->t_end - sg->t_begin;
        const int last = sg->first + sg->n - 1;           // the request's last key
        const int B = 1 << box_log, boxes = KT >> box_log;
#pragma unroll 1
        for (int i = 0; i < 2 * n; i++, filled++) {
          const bool keys = i == 0 || ((i & 1) && i < 2 * n - 1);
          const uint32_t number = tiles;
          tiles += keys;
          if ((filled & 1u) != turn) continue;
          const int t = sg->t_begin + (keys ? (i + 1) / 2 : i == 2 * n - 1 ? n - 1 : i / 2 - 1);
          const int k0 = sg->tile(t) * KT;
          const uint32_t at = filled % RING, turns = filled / RING;
          const uint32_t bar = C::FP8 ? raw_full(at) : kv_full(at);
          const uint32_t dst = C::FP8 ? raw_a + at * C::RAW : kv_a + at * C::TILE;
          const CUtensorMap *map = &maps.box[keys ? 0 : 1], *one = &maps.one[keys ? 0 : 1];
          constexpr uint32_t row_bytes = 128;
#pragma unroll 1
          for (int b0 = 0; b0 < boxes; b0 += 32) {        // once, unless a page's slots are odd or twice odd
            const int b = b0 + lane, j = k0 + (b << box_log);
            int page = -1, off = 0;
            if (b < boxes && j <= last) {
              const uint32_t col = (uint32_t)j / (uint32_t)p.page;
              off = (int)((uint32_t)j - col * (uint32_t)p.page);
              if (col < (uint32_t)p.table_cols) page = __ldg(p.table + (int64_t)r * p.table_ld + col);
              if (page >= p.pages) page = -1;
            }
            const uint32_t hide = __ballot_sync(~0u, b < boxes && j <= last && page < 0);
            if (b0 == 0) {
              if (filled >= RING) ok = bar_wait(C::FP8 ? raw_empty(at) : kv_empty(at), (turns & 1) ^ 1, s_failed, 10);
              ok = __all_sync(~0u, ok);
              if (!ok) break;
              if (lane == 0 && keys) {
#pragma unroll
                for (int e = 1; e < 4; e++) s_hide[(number % HIDE_RING) * 4 + e] = 0;
              }
            }
            if (lane == 0 && keys) s_hide[(number % HIDE_RING) * 4 + (b0 >> 5)] = hide;  // bit b: box b
            __syncwarp();
            if (b < boxes) {
              const uint32_t to = dst + (uint32_t)(b << box_log) * row_bytes;
              const int pg = page < 0 ? (int)p.pages : page;  // behind the last page: zeros
              if (page < 0 || j + B - 1 <= last) {
                load_box(to, map, 0, h, off, pg, bar);
                if constexpr (!C::FP8 && DP == 128) load_box(to + KT * 128, map, 64, h, off, pg, bar);
              } else {
                for (int e = 0; e < B; e++) {
                  const int pe = j + e <= last ? page : (int)p.pages;
                  load_box(to + e * row_bytes, one, 0, h, off + e, pe, bar);
                  if constexpr (!C::FP8 && DP == 128) load_box(to + e * row_bytes + KT * 128, one, 64, h, off + e, pe, bar);
                }
              }
            }
          }
          if (!ok) break;
          // The bytes may arrive before they are expected; the mask's words all stand before this arrival, which the
          // softmax's wait goes back to.
          if (lane == 0) bar_expect(bar, C::FP8 ? C::RAW : C::TILE);
        }
        __syncwarp();
        if (lane == 0) bar_arrive(seg_empty + 8 * (segs % SEGS));
      }
    }
  } else if (C::FP8 && warp >= 8) {
    // =================================================== float8 codes to f16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHER));
    if constexpr (C::FP8) {
      const int pt = tid - 8 * 32;
      constexpr int CPR = DP / 16, STEP = 128 / CPR, UNITS = KT / STEP;  // a thread's units lie STEP rows apart
      static_assert(STEP % 8 == 0, "a thread's rows share their place in the swizzle");
      const int cu = pt % CPR, row0 = pt / CPR, x = row0 & 7;
      // the halves' order alternates between the column blocks, so that the eight lanes of a row meet eight bank groups
      const int swap = cu >> 2, u0 = (cu & 3) * 2 + swap, u1 = (cu & 3) * 2 + 1 - swap;
      const uint32_t at8 = (uint32_t)((cu >> 2) * (KT * 128) + row0 * 128);
      uint32_t done = 0;
      bool ok = true;
      for (uint32_t segs = 0; ok; segs++) {
        const Segment *sg = seg_at(segs, 54);
        if (!__all_sync(~0u, sg != nullptr) || sg->r < 0) break;
        const int n = 2 * (sg->t_end - sg->t_begin);
#pragma unroll 1
        for (int i = 0; i < n && ok; i++, done++) {
          const uint32_t rs = done % C::RAWS, ks = done % C::SLOTS;
          ok = bar_wait(raw_full(rs), (done / C::RAWS) & 1, s_failed, 11);
          if (done >= C::SLOTS) ok = ok && bar_wait(kv_empty(ks), ((done / C::SLOTS) & 1) ^ 1, s_failed, 12);
          if (!ok) break;
          const uint32_t raw = raw_a + rs * C::RAW + row0 * 128 + cu * 16, dst = kv_a + ks * C::TILE + at8;
#pragma unroll
          for (int k = 0; k < UNITS; k++) {
            uint32_t q[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(raw + k * (STEP * 128)));
            const uint32_t a0 = swap ? q[2] : q[0], a1 = swap ? q[3] : q[1], b0 = swap ? q[0] : q[2], b1 = swap ? q[1] : q[3];
            sts16(dst + k * (STEP * 128) + ((u0 ^ x) << 4), fp8x2_to_f16x2<KV>(a0 & 0xFFFFu), fp8x2_to_f16x2<KV>(a0 >> 16),
                  fp8x2_to_f16x2<KV>(a1 & 0xFFFFu), fp8x2_to_f16x2<KV>(a1 >> 16));
            sts16(dst + k * (STEP * 128) + ((u1 ^ x) << 4), fp8x2_to_f16x2<KV>(b0 & 0xFFFFu), fp8x2_to_f16x2<KV>(b0 >> 16),
                  fp8x2_to_f16x2<KV>(b1 & 0xFFFFu), fp8x2_to_f16x2<KV>(b1 >> 16));
          }
          bar_arrive(raw_empty(rs));
          fence_async();
          bar_arrive(kv_full(ks));
        }
        __syncwarp();
        if (lane == 0) bar_arrive(seg_empty + 8 * (segs % SEGS));
      }
    }
  } else {
    // =================================================== softmax, one row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    const int g = warp >> 2;
    const int my = (warp & 3) * 32 + lane;                 // row of the tile
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + 128 * g, t_o = tmem + lanes + 256 + DP * g;
    const uint32_t q_a = base_a + g * C::TILE;
    uint32_t tiles = 0;
    bool ok = true;
    // The group's rows of Q for a segment, where they do not come by boxes
    // (float8 caches, groups that do not divide 128, negative scales). A row takes DP / 8 lanes, so that a
    // warp reads whole rows; the owner of row r gets its scale from them.
    float qscale = 1.0f;
    auto load_q = [&](const Segment *sg) {
      constexpr int LPR = DP / 8, RPI = 32 / LPR;          // lanes a row, rows an instruction
      const int cu = lane % LPR, sub = lane / LPR;
      const int all_rows = sg->n * p.group, row0 = sg->qt * QB + g * QT + (warp & 3) * 32;
      const int own = min(row0 + lane, all_rows - 1), own_tok = own / p.group;
      const int64_t own_at = (int64_t)(sg->start + own_tok) * p.q_tok + (int64_t)(sg->h * p.group + own - own_tok * p.group) * p.q_head;
      // its sign takes that of the scale, so that the maximum of the products is the maximum of the scores
      const uint32_t flip = p.scale_log2 * (C::FP8 && p.ks ? __ldg(p.ks + p.ks_step * sg->h) : 1.0f) < 0.0f ? 0x80008000u : 0u;
      constexpr int BATCH = C::FP8 ? 4 : DP == 64 ? 8 : 16;  // loads in flight
#pragma unroll 1
      for (int i0 = 0; i0 < 32 / RPI; i0 += BATCH) {
        uint4 v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
          const int row = (i0 + k) * RPI + sub;
          const int64_t at = __shfl_sync(~0u, own_at, row);
          v[k] = make_uint4(0, 0, 0, 0);
          if (row0 + row < all_rows && cu * 8 < p.d) v[k] = __ldg(reinterpret_cast<const uint4 *>(p.q + at) + cu);
        }
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
          const int row = (i0 + k) * RPI + sub, my_row = (warp & 3) * 32 + row;
          uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          if constexpr (C::FP8 && !F16) {                  // bf16 to f16, the largest value in [1, 2)
            float a = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) a = fmaxf(a, fmaxf(fabsf(u2f(x[e] << 16)), fabsf(u2f(x[e] & 0xFFFF0000u))));
#pragma unroll
            for (int d = LPR / 2; d > 0; d >>= 1) a = fmaxf(a, __shfl_xor_sync(~0u, a, d));
            uint32_t eb = f2u(a) >> 23;
            eb = (eb == 255u || a == 0.0f) ? 127u : min(max(eb, 1u), 253u);
            const float mul = u2f((254u - eb) << 23);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = pack2<true>(u2f(x[e] << 16) * mul, u2f(x[e] & 0xFFFF0000u) * mul);
            const float qs = __shfl_sync(~0u, u2f(eb << 23), (lane % RPI) * LPR);  // of row (i0 + k) * RPI + lane % RPI
            if (lane / RPI == i0 + k) qscale = qs;
          }
          sts16(q_a + (cu >> 3) * (QT * 128) + my_row * 128 + (((cu & 7) ^ (my_row & 7)) << 4), x[0] ^ flip, x[1] ^ flip,
                x[2] ^ flip, x[3] ^ flip);
        }
      }
      fence_async();
      bar_arrive(q_full + 8 * g);
    };
    // Its rows into L2, a segment ahead.
    auto prefetch_q = [&](const Segment *sg) {
      const int row = sg->qt * QB + g * QT + my;
      if (row < sg->n * p.group) {
        const int tok = row / p.group;
        const uint16_t *at = p.q + (int64_t)(sg->start + tok) * p.q_tok + (int64_t)(sg->h * p.group + row - tok * p.group) * p.q_head;
        for (int d = 0; d < p.d; d += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + d));
      }
    };
    const Segment *sg = seg_at(0, 53);
    if (!__all_sync(~0u, sg != nullptr)) ok = false;
    if (ok && sg->r >= 0 && !q_boxes) load_q(sg);
    for (uint32_t segs = 0; ok && sg->r >= 0; segs++) {
      const int h = sg->h, first = sg->first, t_begin = sg->t_begin, t_end = sg->t_end;
      const int all_rows = sg->n * p.group;                // below 2^31: tokens x query heads are
      const int row0 = sg->qt * QB + g * QT;               // the tile's first row; it may lie behind the request's last
      const bool mine = row0 + my < all_rows;
      const int clipped = min(row0 + my, all_rows - 1);
      const int tok = clipped / p.group, head = h * p.group + clipped - tok * p.group;
      const int pos = first + tok;
      const int pos_lo = first + min(row0, all_rows - 1) / p.group;
      const int pos_hi = first + (min(row0 + QT, all_rows) - 1) / p.group;
      // a scale of 0 weighs all keys alike; kept above 0 so that a hidden key's -inf stays one
      float sc = fabsf(p.scale_log2 * (C::FP8 && p.ks ? __ldg(p.ks + p.ks_step * h) : 1.0f)) * qscale;
      if (sc == 0.0f) sc = 1e-30f;
      const Segment *next = seg_at(segs + 1, 55);
      if (!__all_sync(~0u, next != nullptr)) {
        ok = false;
        break;
      }
      if (next->r >= 0 && !q_boxes) prefetch_q(next);
      float base = -INFINITY, sum = 0.0f;                  // of this row: weights are 2^(score - base + SHIFT)
      for (int t = t_begin; t < t_end; t++) {
        const int k0 = sg->tile(t) * KT;
        ok = bar_wait(s_full + 8 * g, tiles & 1, s_failed, 20 + g);
        if (!__all_sync(~0u, ok)) {
          ok = false;
          break;
        }
        fence_after();
        uint32_t s[128];
#pragma unroll
        for (int i = 0; i < 4; i++) tld32(t_s + 32 * i, s + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; i++) tld_wait(s + 32 * i);
        const uint4 hide = *reinterpret_cast<const uint4 *>(s_hide + (tiles % HIDE_RING) * 4);
        const bool any_hide = (hide.x | hide.y | hide.z | hide.w) != 0u;
        if (k0 + KT - 1 > pos_lo) {                          // keys behind the query
          const int lim = pos - k0;
#pragma unroll
          for (int i = 0; i < 128; i++) s[i] = i > lim ? 0xFF800000u : s[i];
        }
        if (p.window > 0 && pos_hi - k0 >= p.window && k0 + KT - 1 >= p.sinks) {  // before its window, behind the sinks
          const int wlo = (int)max((int64_t)pos - p.window - k0, (int64_t)-1);
          const int sk = (int)min(max((int64_t)p.sinks - k0, (int64_t)0), (int64_t)KT);
#pragma unroll
          for (int i = 0; i < 128; i++) s[i] = i <= wlo && i >= sk ? 0xFF800000u : s[i];
        }
        if (any_hide) {                                      // without a page
#pragma unroll
          for (int i = 0; i < 128; i++) {
            const int b = i >> box_log;
            const uint32_t word = b < 32 ? hide.x : b < 64 ? hide.y : b < 96 ? hide.z : hide.w;
            if ((word >> (b & 31)) & 1u) s[i] = 0xFF800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int k = 0; k < 4; k++) mx[k] = fmaxf(u2f(s[k]), u2f(s[4 + k]));
#pragma unroll
        for (int i = 8; i < 128; i += 8)
#pragma unroll
          for (int k = 0; k < 4; k++) mx[k] = fmaxf(mx[k], fmaxf(u2f(s[i + k]), u2f(s[i + 4 + k])));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        const bool grow = top > base + 8.0f;               // also the first key of the row (base -inf)
        if (__any_sync(~0u, grow)) {
          const float nb = grow ? top : base;
          const float f = base == -INFINITY ? 0.0f : ex2(base - nb);
          sum *= f;
          base = nb;
          if (t > t_begin) {                               // O holds the tiles before: wait for the last one, rescale
            ok = bar_wait(pv_done + 8 * g, (tiles - 1) & 1, s_failed, 30 + g);
            if (!__all_sync(~0u, ok)) {
              ok = false;
              break;
            }
            fence_after();
#pragma unroll 1
            for (int i = 0; i < DP / 32; i++) {
              uint32_t o[32];
              tld32(t_o + 32 * i, o);
              tld_wait(o);
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = f2u(u2f(o[e]) * f);
              tst32(t_o + 32 * i, o);
            }
          }
        }
        const float off = C::SHIFT - (base == -INFINITY ? 0.0f : base);
        const float2 sc2 = make_float2(sc, sc), off2 = make_float2(off, off);
        float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int c4 = 0; c4 < 4; c4++) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            float2 e = fma2(make_float2(u2f(s[c4 * 32 + 2 * i]), u2f(s[c4 * 32 + 2 * i + 1])), sc2, off2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            acc[i & 1] = add2(acc[i & 1], e);
            pk[i] = pack2<C::MF16>(e.x, e.y);
          }
          tst16(t_s + 16 * c4, pk);
          if (c4 == 1) {                                   // the second product can begin with half of the keys
            tst_wait();
            fence_before();
            bar_arrive(p_half + 8 * g);
          }
        }
        tst_wait();
        fence_before();
        bar_arrive(p_full + 8 * g);
        if (tid == 0) *s_deadline = now_ns() + p.wait_ns;
        const float2 a2 = add2(acc[0], acc[1]);
        sum += a2.x + a2.y;
        tiles++;
      }
      if (!__all_sync(~0u, ok)) {
        ok = false;
        break;
      }
      // ---- the next segment's rows of Q: the last S, for which all have waited, was the last reader of these
      if (next->r >= 0 && !q_boxes) load_q(next);
      // ---- the segment's end
      ok = bar_wait(pv_done + 8 * g, (tiles - 1) & 1, s_failed, 40 + g);
      if (!__all_sync(~0u, ok)) {
        ok = false;
        break;
      }
      fence_after();
      const bool begins = t_begin == 0, whole = begins && t_end == sg->units;
      if (tid == 0 && begins && !whole)
        p.desc[c] = PartDesc{min(QB, all_rows - sg->qt * QB), sg->qt * QB, h, sg->start, sg->last - (int)c + 1, 1};
      const float vs = C::FP8 && p.vs ? __ldg(p.vs + p.vs_step * h) : 1.0f;
      const float inv = sum == 0.0f ? 0.0f : vs / sum;
      const float mine_base = base - C::SHIFT;
      float *part = p.part + (c * 2 + (begins ? 1 : 0)) * (int64_t)(QB * (DP + 2));
      const int brow = g * QT + my;
      const int64_t out_at = (int64_t)(sg->start + tok) * p.o_tok + (int64_t)head * p.o_head;
      int64_t to[4];                                       // of the rows that this lane stores, -1 for none
#pragma unroll
      for (int q = 0; q < 4; q++) to[q] = __shfl_sync(~0u, mine ? out_at : (int64_t)-1, (lane & ~3) + q);
      bool odd = false;
#pragma unroll 1
      for (int i = 0; i < DP / 32; i++) {
        uint32_t o[32];
        __syncwarp();
        tld32(t_o + 32 * i, o);
        tld_wait(o);
        if (mine) {
#pragma unroll
          for (int e = 0; e < 32; e++) odd |= !(fabsf(u2f(o[e])) < INFINITY);
        }
        if (whole) {
          // 16-byte units through a transpose among four lanes: a store then covers 64 bytes of each of eight rows
          uint4 x[4];
#pragma unroll
          for (int q = 0; q < 4; q++) {
            x[q].x = pack2<F16>(u2f(o[q * 8]) * inv, u2f(o[q * 8 + 1]) * inv);
            x[q].y = pack2<F16>(u2f(o[q * 8 + 2]) * inv, u2f(o[q * 8 + 3]) * inv);
            x[q].z = pack2<F16>(u2f(o[q * 8 + 4]) * inv, u2f(o[q * 8 + 5]) * inv);
            x[q].w = pack2<F16>(u2f(o[q * 8 + 6]) * inv, u2f(o[q * 8 + 7]) * inv);
          }
#pragma unroll
          for (int d = 1; d <= 2; d <<= 1) {               // lane l gives away its units whose bit d differs from l's
            const bool up = lane & d;
#pragma unroll
            for (int q = 0; q < 4; q++)
              if (!(q & d)) {
                uint4 &lo = x[q], &hi = x[q | d];
                uint4 out4 = up ? lo : hi;
                out4.x = __shfl_xor_sync(~0u, out4.x, d);
                out4.y = __shfl_xor_sync(~0u, out4.y, d);
                out4.z = __shfl_xor_sync(~0u, out4.z, d);
                out4.w = __shfl_xor_sync(~0u, out4.w, d);
                if (up) lo = out4;
                else hi = out4;
              }
          }
          const int col = i * 32 + (lane & 3) * 8;
#pragma unroll
          for (int q = 0; q < 4; q++)                      // x[q]: unit lane % 4 of the row of lane (lane & ~3) + q
            if (to[q] >= 0 && col < p.d) *reinterpret_cast<uint4 *>(p.out + to[q] + col) = x[q];
        } else if (mine) {
#pragma unroll
          for (int q = 0; q < 8; q++)
            *reinterpret_cast<uint4 *>(part + brow * DP + i * 32 + q * 4) = make_uint4(o[q * 4], o[q * 4 + 1], o[q * 4 + 2], o[q * 4 + 3]);
        }
      }
      fence_before();
      if (mine && !whole) {
        part[QB * DP + brow] = mine_base;
        part[QB * DP + QB + brow] = sum;
      }
      if (__any_sync(~0u, odd)) {
        __syncwarp();                                      // the rows' stores, by other lanes too
        const SegmentRows<KT> rows{sg->r, sg->start, first, h, sg->qt * QB, sg->tiles(), t_begin, t_end};
        odd_rows<F16, KV, DP, KT>(p, rows, brow, odd, sum, whole, part, QB, s_deadline);
      }
      __syncwarp();
      if (lane == 0) bar_arrive(seg_empty + 8 * (segs % SEGS));
      sg = next;
    }
  }
  // ---- teardown, reached by every role whether or not a wait ran out
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == C::CTRL) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

using TcKernel = void (*)(AttnParams, TcMaps, int, int);
struct TcVariant {
  TcKernel main;
  void (*merge)(AttnParams);
  int smem, threads;
};
template <bool F16, int KV, int DP>
TcVariant tc_variant() {
  return {paged_attention_tc_kernel<F16, KV, DP>, paged_merge_kernel<F16, DP, QB>, Tc<F16, KV, DP>::SMEM, Tc<F16, KV, DP>::THREADS};
}
template <bool F16, int KV>
TcVariant pick_tc(int dp) {
  return dp == 64 ? tc_variant<F16, KV, 64>() : tc_variant<F16, KV, 128>();
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static std::once_flag once;
  static EncodeTiled fn = nullptr;
  std::call_once(once, [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(ptr);
  });
  return fn;
}

}  // namespace

constexpr uint64_t WAIT_NS = 10000000000ull;
thread_local uint64_t g_wait_ns = WAIT_NS;
thread_local int g_no_tiles = 0;

// The attributes last as long as the process: set once a kernel and device.
int launch_attributes(const void *kernel, int smem) {
  static std::mutex m;
  static const void *done[256];
  static int devices[256], n = 0;
  int dev;
  if (int rc = check_device(&dev)) return rc;
  std::lock_guard<std::mutex> lock(m);
  for (int i = 0; i < n; i++)
    if (done[i] == kernel && devices[i] == dev) return FP8B200_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
    return check_launch("paged_attention");
  if (n < 256) {
    done[n] = kernel;
    devices[n++] = dev;
  }
  return FP8B200_OK;
}

int64_t tc_workspace(int dp, int sms) { return (int64_t)sms * (2 * QB * (int64_t)(dp + 2) * 4 + (int64_t)sizeof(PartDesc)); }

// What a tensor map can describe: strides above 0 (below 2^40 bytes), extents
// below 2^31; and as many requests as the plan holds.
bool tc_takes(const AttnParams &p) {
  const int64_t most = (int64_t)1 << 38;
  auto fits = [&](int64_t n, int64_t stride) { return n == 1 || (stride > 0 && stride < most); };
  return p.requests <= MAX_REQUESTS && p.pages > 0 && p.pages < INT32_MAX && fits(p.hk, p.s_head) && fits(p.page, p.s_slot) && fits(p.pages, p.s_page);
}

int launch_tc(const AttnParams &params, bool f16, int cache_dtype, int dp, int sms, uint8_t *workspace, cudaStream_t st) {
  AttnParams p = params;
  p.desc = (PartDesc *)workspace;
  p.part = (float *)(workspace + (int64_t)sms * sizeof(PartDesc));
  p.blocks = sms;
  p.wait_ns = g_wait_ns;
  p.no_tiles = g_no_tiles;
  const bool fp8 = cache_dtype == FP8B200_E4M3 || cache_dtype == FP8B200_E5M2;
  TcVariant v;
  if (cache_dtype == FP8B200_E4M3) v = f16 ? pick_tc<true, FP8B200_E4M3>(dp) : pick_tc<false, FP8B200_E4M3>(dp);
  else if (cache_dtype == FP8B200_E5M2) v = f16 ? pick_tc<true, FP8B200_E5M2>(dp) : pick_tc<false, FP8B200_E5M2>(dp);
  else v = f16 ? pick_tc<true, FP8B200_F16>(dp) : pick_tc<false, FP8B200_BF16>(dp);
  EncodeTiled encode = encode_tiled();
  if (!encode) return set_error(FP8B200_ELAUNCH, "paged_attention: cuTensorMapEncodeTiled not available");
  int box_log = 0;  // slots a box: the largest power of two that divides the page and the tile
  while (box_log < 7 && !((p.page >> box_log) & 1)) box_log++;
  TcMaps maps;
  for (int i = 0; i < 4; i++) {
    // 64 16-bit values (one swizzled 128-byte row) or a head's float8 codes wide
    const int64_t esz = fp8 ? 1 : 2, any = (int64_t)p.d * esz;
    const cuuint64_t dims[4] = {(cuuint64_t)p.d, (cuuint64_t)p.hk, (cuuint64_t)p.page, (cuuint64_t)p.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)(p.hk > 1 ? p.s_head * esz : any), (cuuint64_t)(p.page > 1 ? p.s_slot * esz : any),
                                   (cuuint64_t)(p.pages > 1 ? p.s_page * esz : any)};
    const cuuint32_t box[4] = {fp8 ? 128u : 64u, 1, i < 2 ? 1u << box_log : 1u, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(i < 2 ? &maps.box[i] : &maps.one[i - 2], fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                              4, const_cast<uint8_t *>(i & 1 ? p.v : p.k), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              fp8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(FP8B200_ELAUNCH, "paged_attention: tensor map encode failed (%d)", (int)r);
  }
  const auto above0 = [](int64_t n, int64_t stride) { return n == 1 || (stride > 0 && stride < (int64_t)1 << 38); };
  int q_boxes = !fp8 && QT % p.group == 0 && !(p.scale_log2 < 0.0f) && above0(p.hq, p.q_head) && above0(p.tokens, p.q_tok);
  maps.q = maps.box[0];
  if (q_boxes) {
    const cuuint64_t dims[3] = {(cuuint64_t)p.d, (cuuint64_t)p.hq, (cuuint64_t)p.tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)(p.hq > 1 ? p.q_head : p.d) * 2, (cuuint64_t)(p.tokens > 1 ? p.q_tok : p.d) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(QT / p.group)}, step[3] = {1, 1, 1};
    q_boxes = encode(&maps.q, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<uint16_t *>(p.q), dims, strides, box, step,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
  if (int rc = launch_attributes((const void *)v.main, v.smem)) return rc;
  if (int rc = launch_attributes((const void *)v.merge, 0)) return rc;
  launch_dependent(v.main, dim3((unsigned)sms), v.threads, v.smem, st, p, maps, box_log, q_boxes);
  launch_dependent(v.merge, dim3((unsigned)sms, 8), MERGE_THREADS, 0, st, p);
  count_launch(2);
  return check_launch("paged_attention");
}

}  // namespace paged
}  // namespace fp8b200

extern "C" int fp8b200_paged_status(uint32_t *status_out, int reset) {
  using namespace fp8b200;
  int dev;
  if (int rc = check_device(&dev)) return rc;
  uint32_t s = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&s, paged::g_paged_status, sizeof(s));
  if (e == cudaSuccess && reset && s) {
    const uint32_t zero = 0;
    e = cudaMemcpyToSymbol(paged::g_paged_status, &zero, sizeof(zero));
  }
  if (e != cudaSuccess) return set_error(FP8B200_ELAUNCH, "paged_status: %s", cudaGetErrorString(e));
  if (status_out) *status_out = s;
  return s ? set_error(FP8B200_ETIMEOUT, "paged_attention: a wait ran out (site %u)", s & 0x7FFFFFFFu) : FP8B200_OK;
}

extern "C" int fp8b200_debug_paged(int no_tiles, unsigned long long wait_timeout_ns) {
  using namespace fp8b200::paged;
  g_no_tiles = no_tiles ? 1 : 0;
  g_wait_ns = wait_timeout_ns ? wait_timeout_ns : WAIT_NS;
  return FP8B200_OK;
}
