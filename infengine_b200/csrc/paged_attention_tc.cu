// Paged attention of chunks of tokens on the 5th-generation tensor cores
// (tcgen05 + TMEM + TMA): the kernel of ie_paged_attention for more rows than
// the few-rows kernel takes.
//
// A piece is up to 256 (token, head) rows of one KV head, as two
// lanes of up to 128 rows (one TMEM lane a row; whole tokens, so 126 rows in
// groups of 3), over a range of 64-key blocks. Both lanes use a key or value
// block from shared memory once it is there, so L2 sees half the traffic of
// 128-row tiles. Where a piece has at most 32 rows (a decoding sequence in a
// batch with a chunk), both lanes serve the same rows, each half of the blocks,
// and lane 0 adds lane 1's outputs to its own: 24 single tokens over up to 8000
// rows beside a chunk of 512 tokens over 3000 took 131 us with lane 1 idle and
// take 107.
//
//   S = Q K^T  (fp32, TMEM)  ->  p = 2^(s c - m), c = scale log2 e  ->  O += P V
//
// The running maximum m is lazy: O is rescaled only when a row's maximum rises
// by more than 2^8 over the reference it uses, and after the first blocks nearly
// no row needs it. p then stays below 2^8, which bf16 and the fp32 sums do not
// notice; of fp16 the reference's p is 2^7, so that the largest is 2^15 at most
// and 2^7 at least (paged_attention.cuh says why). p is rounded to the storage
// type for the product, the sum takes the unrounded values.
//
// What bounds it: 128 x 128 scores cost 1024 cycles of tensor work (D = 128)
// and 1024 cycles of exponentials on the special-function unit (16 a cycle and
// SM). Each lane has two 64-key score buffers, so its next scores are ready
// when its softmax is done with the last, and neither the tensor cores nor the
// softmax wait for the other's latency: with one 128-key buffer a lane the
// chain scores -> softmax -> product took 4900 cycles a 128-key block. A share
// of the exponentials runs as a polynomial on the FMA pipes instead.
//
// TMEM columns: lane i's scores [128 i, 128 i + 64) and [128 i + 64, 128 i +
// 128), O_i [256 + 128 i, + D); P overwrites the first 32 columns of the scores
// it came from. Shared memory: the two Q tiles, a ring of key / value blocks.
// Operands are 64-dimension halves of 128-byte rows, 128-byte swizzle: Q and K
// K-major, V MN-major as it arrives.
//
// One CTA an SM takes pieces from a queue (in batches of up to 32 sequences the
// longest come first, see Finder) until none is left, and every role runs ahead
// of the next as far as its buffers allow: a CTA for each piece spent 10 us of a
// 30 us piece on finding it, the first copies and the epilogue; a fixed share of
// the pieces for each CTA left a ragged batch of 10 to 800 tokens over up to
// 5000 rows at 297 us for 194.
//
// Warp roles: 0 finds the pieces and copies queries and keys, 2 values (TMA
// boxes of up to 64 rows of one page; the lanes hold the next table entries),
// 1 and 3 issue the two lanes' MMAs, 4-7 and 8-11 are the lanes' softmax and
// epilogue. A barrier wait costs an issuing warp about 110 cycles even when it
// is over, a TMA or MMA some tens: with one warp for all copies a step of 64
// keys took 1900 cycles (2700 with pages of 16), with one for all MMAs 2600.
// Value rows that no row of the tile sees (range edges inside a block; what the
// page holds there may be NaN) are zeroed by the MMA warps before the product.
// Every mbarrier wait is bounded: on expiry IE_ERR_TIMEOUT is recorded, all
// roles leave their loops, and MMAs and copies in flight are waited for before
// TMEM is freed.
#include <cstdio>
#include <type_traits>
#include "ie_common.cuh"
#include "paged_attention.cuh"
#include "paged_ops.cuh"
#include "norm.cuh"
#include "tc_ptx.cuh"

namespace ie {

__device__ int g_paged_tc_status = 0;
__device__ unsigned long long g_paged_tc_wait_ns = kDefaultWaitNs;

namespace pa {
namespace {

using namespace tc;

constexpr int kKB = 64;              // keys of a block
constexpr int kThreads = 384;
constexpr int kSharedRows = 32, kSharedBlocks = 8;  // at most, at least: a piece that both lanes serve
// log2 of the growth of a row's maximum that O tolerates (4 would keep 16 times
// more of an fp16 tail; the rescaling it brings took a mixed batch of wide
// scores from 152 to 165 us), and of the reference's p
constexpr float kLazy = 8.0f;
template <typename T>
constexpr float kRefLog2 = DT<T>::id == IE_DTYPE_F16 ? kLargestLog2F16 - kLazy : 0.f;

template <int D>
struct Cfg {
  static constexpr int kQTile = 128 * D * 2;      // a lane's queries
  static constexpr int kQHalf = 128 * 128;        // their 64-dimension halves
  static constexpr int kTile = kKB * D * 2;       // a key or value block
  static constexpr int kHalf = kKB * 128;
  static constexpr int kDepth = 4;                // blocks of keys, and of values, in the ring
  static constexpr int kOut = 32 * 64 * 2;        // a softmax warp's staging: 32 rows of 64 outputs
  static constexpr int kOffRing = 2 * kQTile;
  static constexpr int kOffOut = kOffRing + 2 * kDepth * kTile;
  static constexpr int kTiles = kOffOut + 8 * kOut;
  // Of 8 pairs of exponentials, those on the FMA pipes: 2 and 3 took 103.1 and
  // 105.5 us over windows of 1024 (D = 64), 161.3 and 162.3 for a mixed batch
  // (D = 128); 0, 2, 4 and 8 took 1970, 1880, 1990 and 2590 cycles a step at D = 64.
  static constexpr int kPoly = 2;
};

// A piece of work, as the roles need it.
struct Item {
  int n;                            // blocks; -1: no more pieces
  int j0;                           // the first of them
  Keys keys;
  int seq, head, row_first, tokens; // sequence, KV head, first row of q, tokens of the tile
  int pos0, rows;                   // position of the first token; rows of the tile
  int slot, split, piece, pieces;
  int shared;                       // both lanes serve the same rows, each half of the blocks (copied in turn)
};

// What the roles share, before the tiles in shared memory (which begin on a
// multiple of 1024 bytes).
struct Control {
  uint64_t bars[56];
  Item items[2];
  int abort, issued[2], queries;
  uint32_t tmem;
  float2 ml[32];                    // lane 1's maxima and sums of a shared piece
};
constexpr int kControl = 1024;
static_assert(sizeof(Control) <= kControl && kControl + Cfg<128>::kTiles <= 227 * 1024, "shared memory per CTA");

// ---- two fp32 values at a time
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// (2^a, 2^b) on the FMA pipes, for values up to 2^22: the nearest integer n by
// adding 1.5 * 2^23, 2^f for the rest f in [-1/2, 1/2] by the polynomial of
// degree 5 of least relative error (2^-22.1 as evaluated: like ex2.approx's
// 2^-22, so that a column's accuracy does not depend on which of the two it
// gets; degree 4, 2^-18.5, was 0.6 % faster over windows), n added to the
// exponent field. Values below -126 count as -126.
__device__ __forceinline__ void ex2_poly2(float& a, float& b) {
  const uint64_t x = pair(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
  const float big = 12582912.0f;
  const uint64_t r = add2(x, pair(big, big));
  const uint64_t f = fma2(add2(r, pair(-big, -big)), pair(-1.0f, -1.0f), x);
  auto c = [](float v) { return pair(v, v); };
  uint64_t p = fma2(c(1.3276472e-3f), f, c(9.675541e-3f));
  p = fma2(p, f, c(5.550713e-2f));
  p = fma2(p, f, c(2.4022120e-1f));
  p = fma2(p, f, c(6.9314694e-1f));
  p = fma2(p, f, c(1.0000001f));
  float r0, r1, p0, p1;
  split(r, r0, r1);
  split(p, p0, p1);
  a = __int_as_float(__float_as_int(p0) + (__float_as_int(r0) << 23));
  b = __int_as_float(__float_as_int(p1) + (__float_as_int(r1) << 23));
}
// One lane of a converged warp, the same one each time. The MMA warp runs its
// loop as a whole and elects only for the instructions: their operands then
// stay in uniform registers (with `if (lane == 0)` around the loop an MMA took
// about 150 cycles to issue, longer than it takes to run).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
// the n lowest bits (none for n <= 0, all from 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
}
// NaN if any operand is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// D (TMEM) (+)= A (TMEM) . B (shared memory descriptor)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(
          d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
// N consecutive columns of this warp's 32 lanes; tmem_ld_wait() before the values are used.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31"
      "}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// 64 columns, waited for in the same statement.
__device__ __forceinline__ void tmem_ld64_wait(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,"
      "%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
// Waits for the loads above. The values pass through the statements, so that
// no use of them can move before it.
template <int N>
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_wait(bar, parity, abort_flag, &g_paged_tc_status, &g_paged_tc_wait_ns);
}
// (the bounded loop stays out of the roles' code, which is long enough to be felt in the instruction cache)
template <bool kPolled>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if constexpr (kPolled) return mbar_poll(bar, parity, abort_flag, &g_paged_tc_status, &g_paged_tc_wait_ns);
  else return mbar_try(bar, parity) || wait_long(bar, parity, abort_flag);
}

// kPolled: for wait limits that a suspended wait would outlast.
template <typename T, int D, bool kPolled>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const __grid_constant__ Args a) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Control& ctl = *reinterpret_cast<Control*>(smem_raw);
  uint8_t* smem = smem_raw + kControl;
  volatile int* abort_flag = &ctl.abort;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kDepth = C::kDepth;
  const uint32_t bars = smem_u32(ctl.bars);
  auto full_bar = [&](int s) { return bars + 8 * s; };                     // keys 0 .., values kDepth ..
  auto empty_bar = [&](int s) { return bars + 8 * (2 * kDepth + s); };
  constexpr int kB = 4 * kDepth;
  const uint32_t q_full = bars + 8 * kB, q_empty = bars + 8 * (kB + 1);
  auto item_full = [&](int t) { return bars + 8 * (kB + 2 + (t & 1)); };
  auto item_empty = [&](int t) { return bars + 8 * (kB + 4 + (t & 1)); };
  auto s_full = [&](int i, int b) { return bars + 8 * (kB + 6 + 2 * i + b); };  // scores of lane i, buffer b
  auto p_full = [&](int i, int b) { return bars + 8 * (kB + 10 + 2 * i + b); };
  // by buffer too: two products may be done before the issuing warp asks for the first
  auto pv_done = [&](int i, int b) { return bars + 8 * (kB + 14 + 2 * i + b); };
  auto o_full = [&](int i) { return bars + 8 * (kB + 18 + i); };
  auto o_empty = [&](int i) { return bars + 8 * (kB + 20 + i); };
  auto drain_bar = [&](int i) { return bars + 8 * (kB + 22 + i); };
  // lane 1's part of a shared piece
  const uint32_t part_full = bars + 8 * (kB + 24), part_empty = bars + 8 * (kB + 25);
  static_assert(kB + 26 <= 56, "barriers");

  if (threadIdx.x == 32) {
    for (int s = 0; s < 2 * kDepth; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 2);  // both lanes' MMAs
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    mbar_init(part_full, 1);
    mbar_init(part_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(item_full(i), 1);
      mbar_init(item_empty(i), 11);  // every warp but the finding one
      mbar_init(o_full(i), 1);
      mbar_init(o_empty(i), 4);
      mbar_init(drain_bar(i), 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(s_full(i, b), 1);
        mbar_init(pv_done(i, b), 1);
        mbar_init(p_full(i, b), 4);
      }
    }
    ctl.abort = 0;
    ctl.issued[0] = ctl.issued[1] = ctl.queries = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&a.tmQ);
    prefetch_map(&a.tmK);
    prefetch_map(&a.tmV);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)),
                 "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ctl.tmem;

  // Blocks are counted over all pieces, by the copies and by each lane: block
  // g of the copies lies in stage g % kDepth, scores of block g of a lane in
  // buffer g & 1.
  auto phase = [&](int g) { return (uint32_t)((g / kDepth) & 1); };
  auto over = [&](uint32_t bar, uint32_t parity) {
    return __all_sync(0xffffffffu, wait<kPolled>(bar, parity, abort_flag)) != 0;
  };
  // piece t's description; the slot is free for the next but one once every warp has its copy
  auto take = [&](int t, Item& it) {
    if (!over(item_full(t), (uint32_t)((t >> 1) & 1))) return false;
    it = ctl.items[t & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(item_empty(t));
    return it.n >= 0;
  };

  // Registers: 384 x 168 at launch; the softmax warps take 216 each, the
  // others give up down to 72.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------- copies of queries and keys (0) or values (2)
      const int v = warp >> 1;
      const CUtensorMap* map = v ? &a.tmV : &a.tmK;
      // rows of a copy, copies of a block's half, blocks whose table entries the warp holds
      const int box_log2 = min(a.l.page_log2, 6), box = 1 << box_log2, boxes_log2 = 6 - box_log2;
      const int held_log2 = 5 - boxes_log2, held = 1 << held_log2;
      int g = 0, queries = 0;  // blocks and query tiles copied so far
      int index = blockIdx.x;   // of the piece; the ones after the first come from the queue
      auto claim = [&] {
        if (lane == 0) index = (int)gridDim.x + atomicAdd(a.queue, 1);
      };
      // the copies of one piece; false when a wait gave up
      auto copy_as = [&](const Item& it, auto is_shared) {
        constexpr bool shared = decltype(is_shared)::value;
        const int n = __shfl_sync(0xffffffffu, it.n, 0), head = __shfl_sync(0xffffffffu, it.head, 0);
        if (n == 0) {
          if (v == 0) claim();
          return true;
        }
        const bool two = it.rows > a.lane_rows;
        const int* table = a.b.page_table + (int64_t)it.seq * a.b.ld_table;
        // copy j's block: of a shared piece the two halves in turn
        auto first_key = [&](int j) {
          return it.keys.block(it.j0 + (!shared ? j : (j >> 1) + (j & 1 ? n - (n >> 1) : 0))) * kKB;
        };
        auto load_entries = [&](int first) {
          const int j = first + (lane >> boxes_log2);
          if (j >= n) return -1;
          const int kb = first_key(j) + (lane & ((1 << boxes_log2) - 1)) * box;
          if (!(kb < it.keys.hi && (kb + box > it.keys.lo || kb < it.keys.sink_end))) return -1;
          const int page = table[kb >> a.l.page_log2];
          if (page < 0 || page >= a.l.num_pages) {
            atomicExch(&g_paged_tc_status, IE_ERR_INVALID_ARG);
            return a.l.num_pages;  // outside the tensor map: zeros
          }
          return page;
        };
        int entries = load_entries(0), next = load_entries(held);
        if (v == 0) {
          // the last piece's scores are done with its queries
          if (!over(q_empty, (uint32_t)((queries & 1) ^ 1))) return false;
          if (elect_one()) {
            mbar_expect_tx(q_full, (two ? 2 : 1) * a.lane_rows * D * 2);
            for (int i = 0; i < (two ? 2 : 1); ++i)
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                tma_load_3d(smem_u32(smem + i * C::kQTile + h * C::kQHalf), &a.tmQ, q_full, 64 * h, head * a.group,
                            it.row_first + i * (a.lane_rows / a.group));
          }
          ++queries;
        }
        for (int j = 0; j < n; ++j, ++g) {
          const int at = j & (held - 1);
          if (j > 0 && at == 0) {
            entries = next;
            next = load_entries(j + held);
          }
          const int s = v * kDepth + g % kDepth;
          const uint32_t full = full_bar(s), dst = smem_u32(smem + C::kOffRing + s * C::kTile);
          const int r0 = first_key(j) & (a.l.page_size - 1);
          int page[4], copies = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            page[x] = __shfl_sync(0xffffffffu, entries, ((at << boxes_log2) + x) & 31);
            if (x >> boxes_log2) page[x] = -1;
            copies += page[x] >= 0;
          }
          if (!over(empty_bar(s), phase(g) ^ 1u)) return false;
          // the next piece is asked for when this one's last keys are: the ring's blocks cover the answer's way
          if (v == 0 && j == n - 1) claim();
          if (elect_one()) {
            mbar_expect_tx(full, copies * box * D * 2);
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (page[x] >= 0) {
                const int r = (r0 + x * box) & (a.l.page_size - 1);
#pragma unroll
                for (int h = 0; h < D / 64; ++h)
                  tma_load_4d(dst + h * C::kHalf + x * box * 128, map, full, 64 * h, a.swap_rc ? head : r,
                              a.swap_rc ? r : head, page[x]);
              }
          }
        }
        return true;
      };
      auto copy = [&](const Item& it) {
        return __shfl_sync(0xffffffffu, it.shared, 0) ? copy_as(it, std::true_type{}) : copy_as(it, std::false_type{});
      };
      Item it;
      if (v == 1) {
        for (int t = 0; take(t, it) && copy(it); ++t) {
        }
      } else {
        Finder<kKB> finder(a, &g_paged_tc_status);
        if (blockIdx.x == 0 && lane == 0) *a.n_split = min(finder.splits, a.split_cap);
        for (int t = 0;; ++t) {
          if (!over(item_empty(t), (uint32_t)(((t >> 1) & 1) ^ 1))) break;
          index = __shfl_sync(0xffffffffu, index, 0);
          bool more = index < finder.total;
          if (more) {
            Piece p;
            const bool mine = finder.find(index, p, &g_paged_tc_status);
            more = __any_sync(0xffffffffu, mine);
            if (mine) {
              const Seq& sq = finder.s;
              const int row0 = p.tile * a.tile_rows, per = a.tile_rows / a.group, tok0 = p.tile * per;
              Item x;
              x.rows = min(a.tile_rows, sq.tokens * a.group - row0);
              x.tokens = min(per, sq.tokens - tok0);
              x.keys = tile_keys<kKB>(a, sq, tok0, tok0 + x.tokens - 1);
              piece_range(x.keys.blocks(), p.pieces, p.piece, x.j0, x.n);
              x.seq = p.b;
              x.head = p.head;
              x.row_first = sq.start + tok0;
              x.pos0 = sq.pos0 + tok0;
              x.slot = p.slot;
              x.split = p.split;
              x.piece = p.piece;
              x.pieces = p.pieces;
              x.shared = x.rows <= kSharedRows && x.n >= kSharedBlocks;
              ctl.items[t & 1] = x;
            }
          }
          if (!more && lane == 0) ctl.items[t & 1].n = -1;
          __syncwarp();
          it = ctl.items[t & 1];
          __syncwarp();
          if (lane == 0) mbar_arrive(item_full(t));
          if (!more || !copy(it)) break;
        }
        if (lane == 0) ctl.queries = queries;
      }
      if (lane == 0) ctl.issued[v] = g;
    } else {
      // ---------------------------------------------- MMAs of lane i
      const int i = warp >> 1;
      const uint32_t id_qk = idesc_f16<T>(128, kKB, 0), id_pv = idesc_f16<T>(128, D, 1);
      const uint32_t ring = smem_u32(smem + C::kOffRing);
      const uint64_t qs = sw128_desc(smem_u32(smem) + i * C::kQTile);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0) + 128 * i;
      int gc = 0, g = 0, tiles = 0, queries = 0;  // blocks of the copies and of this lane, its tiles, query tiles
      Item it;
      bool ok = true;
      for (int t = 0; ok && take(t, it); ++t) {
        const int n = __shfl_sync(0xffffffffu, it.n, 0);
        if (n == 0) continue;
        const bool two = __shfl_sync(0xffffffffu, it.rows, 0) > a.lane_rows;
        const bool shared = __shfl_sync(0xffffffffu, it.shared, 0) != 0;
        if (i == 1 && !two && !shared) {
          // nothing for this lane: it only passes everything on (no phase may
          // go by unseen, the next wait could not tell it from its own)
          ok = over(q_full, (uint32_t)(queries++ & 1));
          if (ok && lane == 0) mbar_arrive(q_empty);
          for (int j = 0; ok && j < n; ++j, ++gc)
            for (int v = 0; ok && v < 2; ++v) {
              const int s = v * kDepth + gc % kDepth;
              ok = over(full_bar(s), phase(gc));
              if (ok && lane == 0) mbar_arrive(empty_bar(s));
            }
          continue;
        }
        // (compiled apart: with a shared piece's index arithmetic a step of the others took 2 % longer)
        auto serve = [&](auto is_shared) {
          constexpr bool shared = decltype(is_shared)::value;
          // of a shared piece's copies every other one is this lane's; it passes the others on
          constexpr int step = shared ? 2 : 1;
          const int first = shared ? i : 0, own = (n - first + step - 1) / step;
          const uint64_t qt = qs - (shared ? i * (C::kQTile >> 4) : 0);
          const int j0 = it.j0 + (first ? n - own : 0);
          auto block = [&](int j) { return gc + first + j * step; };
          // waits for keys (v = 0) or values (kDepth) of this lane's block j; those before it that are not its own
          auto there = [&](int j, int v) {
            const int at = block(j);
            if (shared && at > gc) {
              if (!over(full_bar(v + (at - 1) % kDepth), phase(at - 1))) return false;
              if (lane == 0) mbar_arrive(empty_bar(v + (at - 1) % kDepth));
            }
            return over(full_bar(v + at % kDepth), phase(at));
          };
          auto k_there = [&](int j) { return there(j, 0); };
          auto qk = [&](int j) {  // scores of block j, into the buffer of block g + j - 2; its keys are there
            const int s = block(j) % kDepth, b = (g + j) & 1;
            const uint64_t sk = sw128_desc(ring + (uint32_t)s * C::kTile);
            if (g + j >= 2 && !over(pv_done(i, b), (uint32_t)(((g + j - 2) >> 1) & 1))) return false;
            fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < D / 16; ++k)
                mma_f16(tm + 64 * b, qt + (k >> 2) * (C::kQHalf >> 4) + 2 * (k & 3),
                        sk + (k >> 2) * (C::kHalf >> 4) + 2 * (k & 3), id_qk, k != 0 ? 1u : 0u);
              mma_commit(s_full(i, b));
              mma_commit(empty_bar(s));
              if (j == own - 1) mma_commit(q_empty);
            }
            return true;
          };
          bool ok = over(q_full, (uint32_t)(queries & 1));
          ++queries;
          for (int j = 0; ok && j < min(own, 2); ++j) ok = k_there(j) && qk(j);
          // the epilogue has read the last tile's outputs
          if (ok && tiles > 0) ok = over(o_empty(i), (uint32_t)((tiles - 1) & 1));
          for (int j = 0; ok && j < own; ++j) {
            // what can be waited for before P is: this block's values, the keys of the next but one
            const int s = kDepth + block(j) % kDepth, b = (g + j) & 1;
            const int kb = it.keys.block(j0 + j) * kKB;
            if (!(ok = there(j, kDepth))) break;
            if (kb + kKB > it.keys.hi || (kb < it.keys.lo && kb + kKB > it.keys.sink_end)) {
              // rows that no row of the tile sees (both lanes' warps write the same zeros)
              uint8_t* v = smem + C::kOffRing + s * C::kTile;
              for (int r = lane; r < kKB; r += 32) {
                const int key = kb + r;
                if (!(key < it.keys.hi && (key >= it.keys.lo || key < it.keys.sink_end)))
#pragma unroll
                  for (int c = 0; c < D / 8; ++c)
                    *reinterpret_cast<uint4*>(v + (c >> 3) * C::kHalf + r * 128 + ((c & 7) << 4)) =
                        make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
            if (j + 2 < own && !(ok = k_there(j + 2))) break;
            const uint64_t sv = sw128_desc_mn(ring + (uint32_t)s * C::kTile, C::kHalf);
            if (!(ok = over(p_full(i, b), (uint32_t)(((g + j) >> 1) & 1)))) break;
            fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kKB / 16; ++k)
                mma_ts(tm + 256, tm + 64 * b + 8 * k, sv + k * (16 * 128 >> 4), id_pv, (j | k) != 0 ? 1u : 0u);
              mma_commit(pv_done(i, b));
              if (j == own - 1) mma_commit(o_full(i));
              mma_commit(empty_bar(s));
            }
            // the scores of block j + 2 go where P_j was; those of j + 1 keep the softmax busy meanwhile
            if (j + 2 < own) ok = qk(j + 2);
          }
          if (shared && block(own - 1) < gc + n - 1)  // the last block is the other lane's
            for (int v = 0; ok && v <= kDepth; v += kDepth) {
              const int s = v + (gc + n - 1) % kDepth;
              ok = over(full_bar(s), phase(gc + n - 1));
              if (ok && lane == 0) mbar_arrive(empty_bar(s));
            }
          g += own;
          return ok;
        };
        ok = shared ? serve(std::true_type{}) : serve(std::false_type{});
        gc += n;
        ++tiles;
      }
      // every MMA issued is done before TMEM is released, whoever gave up
      __syncwarp();
      if (elect_one()) mma_commit(drain_bar(i));
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(drain_bar(i), 0) && globaltimer() - t0 < kDrainWaitNs) {
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------ softmax and epilogue
    const int i = (warp - 4) >> 2, quad = warp & 3;  // TMEM lane quarter = warp & 3
    const int r = 32 * quad + lane;                  // row of the lane
    const uint32_t tl = (uint32_t)(32 * quad) << 16;
    const uint32_t to = tmem + tl + 256 + 128 * i;
    // a scale of 0 weighs all seen keys alike: scores 0, so that masked ones can stay infinite
    const bool flat = a.scale_log2 == 0.f;
    const float c = flat ? 1.0f : a.scale_log2;
    int g = 0, tiles = 0, parts = 0;  // this lane's blocks and tiles, the shared pieces so far
    Item it;
    bool ok = true;
    for (int t = 0; ok && take(t, it); ++t) {
      const bool shared = it.shared != 0;
      if (i == 1 && it.rows <= a.lane_rows && !shared) continue;
      const int half = it.n >> 1, n = !shared ? it.n : i == 0 ? it.n - half : half;
      const int j0 = it.j0 + (shared && i == 1 ? it.n - half : 0);
      const int lane_of_rows = shared ? 0 : i;
      const int row = r < a.lane_rows ? lane_of_rows * a.lane_rows + r : INT_MAX;  // row of the tile
      const bool valid = row < it.rows;
      const bool idle = lane_of_rows * a.lane_rows + 32 * quad >= it.rows;  // no row is this warp's
      const int pos = valid ? it.pos0 + (row * a.group_magic >> 16) : -1;
      const int pos_min = it.pos0 + lane_of_rows * (a.lane_rows / a.group);
      const int pos_max = it.pos0 + min(it.tokens, (lane_of_rows + 1) * (a.lane_rows / a.group)) - 1;
      float m = -INFINITY, l = 0.f;  // m: the reference, in log2 units
      if (idle)  // (what its rows of P hold stays in its rows of O)
        for (int j = 0; ok && j < n; ++j) {
          ok = over(s_full(i, (g + j) & 1), (uint32_t)(((g + j) >> 1) & 1));
          if (ok && lane == 0) mbar_arrive(p_full(i, (g + j) & 1));
        }
      for (int j = idle ? n : 0; j < n; ++j) {
        const int kb = it.keys.block(j0 + j) * kKB, b = (g + j) & 1;
        const uint32_t ts = tmem + tl + 128 * i + 64 * b;
        ok = over(s_full(i, b), (uint32_t)(((g + j) >> 1) & 1));
        if (!ok) break;
        fence_after();
        float v[kKB];
        {
          uint32_t w[kKB];
          tmem_ld64_wait(ts, w);
#pragma unroll
          for (int x = 0; x < kKB; ++x) v[x] = __uint_as_float(w[x]);
        }
        const bool masked = kb + kKB - 1 > pos_min || (a.window && (int64_t)pos_max - kb >= a.window);
        if (flat) {
#pragma unroll
          for (int x = 0; x < kKB; ++x) v[x] = 0.f;
        }
        if (masked) {
          // the columns the row sees, as bits
          const float hidden = c > 0.f ? -INFINITY : INFINITY;
          const int hi = pos - kb + 1;  // columns below hi
          uint32_t see[2] = {low_bits(hi), low_bits(hi - 32)};
          if (a.window) {
            const int64_t lo64 = (int64_t)pos - a.window - kb + 1;
            const int lo = (int)(lo64 < 0 ? 0 : lo64), sk = a.sinks - kb;  // but not those below lo, unless below sk
            see[0] &= ~low_bits(lo) | low_bits(sk);
            see[1] &= ~low_bits(lo - 32) | low_bits(sk - 32);
          }
#pragma unroll
          for (int x = 0; x < kKB; ++x) v[x] = see[x >> 5] >> (x & 31) & 1 ? v[x] : hidden;
        }
        // the row's largest scaled score
        float top;
        {
          if (c > 0.f) {
            float t4[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) t4[x] = v[x];
#pragma unroll
            for (int x = 4; x + 8 <= kKB; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y) t4[y] = max3(t4[y], v[x + 2 * y], v[x + 2 * y + 1]);
#pragma unroll
            for (int y = 0; y < 2; ++y) t4[y] = max3(t4[y], v[kKB - 4 + 2 * y], v[kKB - 3 + 2 * y]);
            top = max3(max3(t4[0], t4[1], t4[2]), t4[3], t4[3]) * c;
          } else {
            top = v[0] * c;
#pragma unroll
            for (int x = 1; x < kKB; ++x) top = max3(top, v[x] * c, top);
          }
        }
        // (a NaN or infinite score turns the row's reference, and with it the row, into NaN)
        const bool rise = valid && !(top <= m + kLazy);
        if (__any_sync(0xffffffffu, rise)) {
          const float to_m = !rise ? m : top < INFINITY ? top : __int_as_float(0x7fffffff);
          const float f = rise ? ex2(m - to_m) : 1.0f;
          if (j > 0) {
            // every product before this block's
            ok = over(pv_done(i, b ^ 1), (uint32_t)(((g + j - 1) >> 1) & 1));
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
              uint32_t o[32];
              tmem_ld(to + 32 * x, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
              tmem_st(to + 32 * x, o);
            }
          }
          l *= f;
          m = to_m;
        }
        const float mb = kRefLog2<T> - (m == -INFINITY ? 0.f : m);
        const uint64_t c2 = pair(c, c), mb2 = pair(mb, mb);
        uint64_t l2 = pair(0.f, 0.f);
        uint32_t pk[kKB / 2];
        // the polynomial has no 0 for a masked score: such blocks do without
        auto exps = [&](auto poly) {
#pragma unroll
          for (int y = 0; y < kKB / 2; ++y) {
            float e0, e1;
            split(fma2(pair(v[2 * y], v[2 * y + 1]), c2, mb2), e0, e1);
            if (y % 8 < decltype(poly)::value) {
              ex2_poly2(e0, e1);
            } else {
              e0 = ex2(e0);
              e1 = ex2(e1);
            }
            l2 = add2(l2, pair(e0, e1));
            pk[y] = pack2<T>(e0, e1);
          }
        };
        if (masked) exps(std::integral_constant<int, 0>{});
        else exps(std::integral_constant<int, C::kPoly>{});
        tmem_st(ts, pk);
        {
          float l0, l1;
          split(l2, l0, l1);
          l += l0 + l1;
        }
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(i, b));
      }
      // ---- epilogue
      if (ok && n > 0) ok = over(o_full(i), (uint32_t)(tiles & 1));
      if (!ok) break;
      fence_after();
      const bool cut = it.slot >= 0;
      if (shared && !idle) {
        // lane 1's outputs, maxima and sums reach lane 0 through lane 1's staging
        float4* part = reinterpret_cast<float4*>(smem + C::kOffOut + 4 * C::kOut) + lane;
        if (i == 0) {
          ok = over(part_full, (uint32_t)(parts & 1));
          if (!ok) break;
        }
        const float2 other = i == 0 ? ctl.ml[lane] : make_float2(m, l);
        const float top = fmaxf(m, other.x), ref = top == -INFINITY ? 0.f : top;
        const float f0 = ex2(m - ref), f1 = ex2(other.x - ref);
#pragma unroll 1
        for (int x = 0; x < D / 32; ++x) {
          uint32_t w[32];
          tmem_ld(to + 32 * x, w);
          tmem_ld_wait(w);
          if (i == 1) {
#pragma unroll
            for (int y = 0; y < 8; ++y)
              part[(8 * x + y) * 32] = make_float4(__uint_as_float(w[4 * y]), __uint_as_float(w[4 * y + 1]),
                                                   __uint_as_float(w[4 * y + 2]), __uint_as_float(w[4 * y + 3]));
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const float4 u = part[(8 * x + y) * 32];
              w[4 * y] = __float_as_uint(__uint_as_float(w[4 * y]) * f0 + u.x * f1);
              w[4 * y + 1] = __float_as_uint(__uint_as_float(w[4 * y + 1]) * f0 + u.y * f1);
              w[4 * y + 2] = __float_as_uint(__uint_as_float(w[4 * y + 2]) * f0 + u.z * f1);
              w[4 * y + 3] = __float_as_uint(__uint_as_float(w[4 * y + 3]) * f0 + u.w * f1);
            }
            tmem_st(to + 32 * x, w);
          }
        }
        if (i == 1) {
          ctl.ml[lane] = make_float2(m, l);
        } else {
          tmem_st_wait();
          l = l * f0 + other.y * f1;
          m = top;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(i == 1 ? part_full : part_empty);
      }
      // (every warp of lane 1: the staging is theirs too, and no phase of the barrier may go by unseen)
      if (shared && i == 1) ok = over(part_empty, (uint32_t)(parts & 1));
      if (shared) ++parts;
      if (!ok) break;
      if (idle || (shared && i == 1)) {
        // nothing to write
      } else if (cut && (it.slot >= a.slot_cap || it.split >= a.split_cap)) {
        // cannot be: the pieces were chosen to fit
      } else if (cut) {
        // row-interleaved 16-byte pieces, so that a warp's stores are contiguous
        float4* po =
            reinterpret_cast<float4*>(a.part_o) + ((int64_t)it.slot * 8 + 4 * i + quad) * (D / 4) * 32 + lane;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          uint32_t w[32];
          tmem_ld(to + 32 * x, w);
          tmem_ld_wait(w);
          if (n == 0) {
#pragma unroll
            for (int y = 0; y < 32; ++y) w[y] = 0u;
          }
#pragma unroll
          for (int y = 0; y < 8; ++y)
            po[(8 * x + y) * 32] = make_float4(__uint_as_float(w[4 * y]), __uint_as_float(w[4 * y + 1]),
                                               __uint_as_float(w[4 * y + 2]), __uint_as_float(w[4 * y + 3]));
        }
        a.part_ml[(int64_t)it.slot * kRowsChunk + 128 * i + r] = make_float2(m, l);
        if (it.piece == 0 && i == 0 && r == 0) {
          Split sp = {};
          sp.slot0 = it.slot;
          sp.pieces = it.pieces;
          sp.token0 = it.row_first;
          sp.rows = it.rows;
          sp.head0 = it.head * a.group;
          a.splits[it.split] = sp;
        }
      } else {
        // through the warp's staging, 64 outputs at a time: swizzled rows in, 8 lanes a row out
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        uint8_t* st = smem + C::kOffOut + (4 * i + quad) * C::kOut;
#pragma unroll 1
        for (int h = 0; h < D / 64; ++h) {
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            uint32_t w[32];
            tmem_ld(to + 64 * h + 32 * z, w);
            tmem_ld_wait(w);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              uint4 u = make_uint4(0, 0, 0, 0);
              if (n > 0) {
                u.x = pack2<T>(__uint_as_float(w[8 * y]) * inv, __uint_as_float(w[8 * y + 1]) * inv);
                u.y = pack2<T>(__uint_as_float(w[8 * y + 2]) * inv, __uint_as_float(w[8 * y + 3]) * inv);
                u.z = pack2<T>(__uint_as_float(w[8 * y + 4]) * inv, __uint_as_float(w[8 * y + 5]) * inv);
                u.w = pack2<T>(__uint_as_float(w[8 * y + 6]) * inv, __uint_as_float(w[8 * y + 7]) * inv);
              }
              *reinterpret_cast<uint4*>(st + lane * 128 + (((4 * z + y) ^ (lane & 7)) << 4)) = u;
            }
          }
          __syncwarp();
          T* out = static_cast<T*>(a.out) + (int64_t)it.row_first * a.ld_out + (int64_t)it.head * a.group * D +
                   64 * h + 8 * (lane & 7);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int q = 4 * x + (lane >> 3), rr = 32 * quad + q, gr = i * a.lane_rows + rr;
            if (rr < a.lane_rows && gr < it.rows) {
              const int tok = gr * a.group_magic >> 16;
              *reinterpret_cast<uint4*>(out + (int64_t)tok * a.ld_out + (gr - tok * a.group) * D) =
                  *reinterpret_cast<const uint4*>(st + q * 128 + (((lane & 7) ^ (q & 7)) << 4));
            }
          }
          __syncwarp();
        }
      }
      if (n > 0) {
        // the outputs are read: the next tile's first product may overwrite them
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty(i));
        ++tiles;
        g += n;
      }
    }
  }

  // ---------------------------------------------------------- teardown
  fence_before();
  __syncthreads();
  fence_after();
  if (*abort_flag && threadIdx.x == 0) {
    atomicExch(a.n_split, 0);  // nothing to join
    // copies still in flight land before the CTA exits: the last queries, and
    // the last kDepth blocks of keys and values (an earlier one's stage was reused)
    auto landed = [&](uint32_t bar, uint32_t parity) {
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(bar, parity) && globaltimer() - t0 < kDrainWaitNs / 4) {
      }
    };
    if (ctl.queries > 0) landed(q_full, (uint32_t)((ctl.queries - 1) & 1));
    for (int v = 0; v < 2; ++v)
      for (int g = max(0, ctl.issued[v] - kDepth); g < ctl.issued[v]; ++g)
        landed(full_bar(v * kDepth + g % kDepth), phase(g));
  }
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

// Joins the cut tiles' pieces. An item is 32 rows of a tile (one warp's of the
// chunk kernel) and `wide` of their 16-byte columns, as the chunk kernel stored
// them; the CTA's warps share an item's columns and, where these are fewer than
// the warps, its pieces, whose parts then meet in shared memory in a fixed
// order. What bounds it is latency: a few tiles in many pieces are the common
// case, so the items are as narrow as leaves each CTA one (a chunk of 64 tokens
// over 8192 rows, 8 tiles in 18 pieces, took 48 us with a CTA for 32 whole rows
// and 26 so), all of a thread's loads go out at once, and so do the descriptions
// of a CTA's items, most of which have no rows where sequences bring few.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) join_chunks_kernel(const __grid_constant__ Args a) {
  constexpr int kCols = D / 4;
  __shared__ float4 part_s[8][32];
  __shared__ float2 ml_s[8][32];
  __shared__ __align__(16) uint2 rows_s[32][9];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.queue = 0;
  const int n = min(*a.n_split, a.split_cap);
  int wide_log2 = 3;
  while (wide_log2 > 0 && n * 8 * (kCols >> wide_log2) * 2 <= (int)gridDim.x) --wide_log2;
  const int wide = 1 << wide_log2, parts = kCols >> wide_log2, ways = 8 >> wide_log2;
  const int way = warp >> wide_log2, items = n * 8 * parts;
  const int64_t step = a.l.n_kv_heads;
  for (int base = blockIdx.x; base < items; base += 32 * gridDim.x) {
    // this lane's item of the CTA's next 32
    const int mine = base + lane * (int)gridDim.x;
    Split sp = {};
    if (mine < items) sp = a.splits[mine % n];
    const int my_group = mine / n / parts, my_r0 = 32 * (my_group & 3);
    // a chunk kernel that gave up may have left a description unwritten: nothing is taken on trust
    const bool sound = sp.pieces >= 1 && sp.pieces <= a.slot_cap && sp.slot0 >= 0 &&
                       sp.slot0 + (sp.pieces - 1) * step < a.slot_cap && sp.rows >= 1 && sp.rows <= a.tile_rows &&
                       sp.token0 >= 0 && sp.token0 + (int64_t)((sp.rows - 1) / a.group) < a.b.T && sp.head0 >= 0 &&
                       sp.head0 <= (a.l.n_kv_heads - 1) * a.group;
    unsigned todo = __ballot_sync(0xffffffffu, mine < items && sound && my_r0 < a.lane_rows &&
                                                   (my_group >> 2) * a.lane_rows + my_r0 < sp.rows);
    for (; todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1, at = (base + src * (int)gridDim.x) / n;
      const int group = at / parts, part = at - group * parts;
      const int slot0 = __shfl_sync(0xffffffffu, sp.slot0, src), pieces = __shfl_sync(0xffffffffu, sp.pieces, src);
      const int col = (part << wide_log2) + (warp & (wide - 1));
      const float2* ml = a.part_ml + (int64_t)slot0 * kRowsChunk + 32 * group + lane;
      const float4* po =
          reinterpret_cast<const float4*>(a.part_o) + (((int64_t)slot0 * 8 + group) * kCols + col) * 32 + lane;
      float m = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      // (m2, l2, u): maximum, sum and outputs to be added
      auto add = [&](float m2, float l2, const float4& u) {
        const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
        const float f = ex2(m - ref), f2 = ex2(m2 - ref);
        m = top;
        l = l * f + l2 * f2;
        o.x = o.x * f + u.x * f2;
        o.y = o.y * f + u.y * f2;
        o.z = o.z * f + u.z * f2;
        o.w = o.w * f + u.w * f2;
      };
      constexpr int kAhead = 4;
      for (int s0 = way; s0 < pieces; s0 += kAhead * ways) {
        float2 x[kAhead];
        float4 u[kAhead];
#pragma unroll
        for (int y = 0; y < kAhead; ++y) {
          const int64_t s = (s0 + y * ways) * step;
          if (s0 + y * ways < pieces) {
            x[y] = __ldcg(ml + s * kRowsChunk);
            u[y] = __ldcg(po + s * 8 * kCols * 32);
          }
        }
#pragma unroll
        for (int y = 0; y < kAhead; ++y)
          if (s0 + y * ways < pieces) add(x[y].x, x[y].y, u[y]);
      }
      if (ways > 1) {
        part_s[warp][lane] = o;
        ml_s[warp][lane] = make_float2(m, l);
        __syncthreads();
        if (way == 0)
          for (int w = warp + wide; w < 8; w += wide) add(ml_s[w][lane].x, ml_s[w][lane].y, part_s[w][lane]);
      }
      // out through shared memory: `wide` threads a row, 8 bytes each
      if (way == 0) {
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        rows_s[lane][warp] = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
      }
      __syncthreads();
      const int token0 = __shfl_sync(0xffffffffu, sp.token0, src), rows = __shfl_sync(0xffffffffu, sp.rows, src),
                head0 = __shfl_sync(0xffffffffu, sp.head0, src);
      const int q = threadIdx.x >> wide_log2, c = threadIdx.x & (wide - 1);
      const int r = 32 * (group & 3) + q, g = (group >> 2) * a.lane_rows + r;
      if (q < 32 && r < a.lane_rows && g < rows) {
        const int tok = g * a.group_magic >> 16;
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(token0 + tok) * a.ld_out +
                                  (int64_t)(head0 + g - tok * a.group) * D + 4 * ((part << wide_log2) + c)) =
            rows_s[q][c];
      }
      __syncthreads();
    }
  }
}

template <typename T, int D, bool kPolled = false>
int launch(Args& a, int64_t most_tiles, cudaStream_t st) {
  if (!kPolled && a.polled) return launch<T, D, true>(a, most_tiles, st);
  auto kernel = chunk_kernel<T, D, kPolled>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return IE_ERR_LAUNCH;
  static bool configured[64] = {};
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kControl + Cfg<D>::kTiles) !=
        cudaSuccess)
      return IE_ERR_LAUNCH;
    configured[dev] = true;
  }
  if (most_tiles + a.slot_cap > INT_MAX) return IE_ERR_UNSUPPORTED;
  const int64_t most = most_tiles + a.slot_cap, grid = most < a.wave ? most : a.wave;
  kernel<<<(unsigned)grid, kThreads, kControl + Cfg<D>::kTiles, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) {
    const int64_t items = 8 * (D / 4) * (most_tiles < a.target ? most_tiles : a.target);  // at most
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items < kSMs * 4 ? items : kSMs * 4));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_launch_enabled() ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, join_chunks_kernel<T, D>, a);
  }
  if (e != cudaSuccess) {
    std::fprintf(stderr, "infengine_b200: paged attention launch failed: %s\n", cudaGetErrorString(e));
    return IE_ERR_LAUNCH;
  }
  return IE_OK;
}

}  // namespace

int launch_chunks(ie_dtype dt, int D, Args& a, int64_t most_tiles, cudaStream_t st) {
  if (dt == IE_DTYPE_F16)
    return D == 128 ? launch<__half, 128>(a, most_tiles, st) : launch<__half, 64>(a, most_tiles, st);
  return D == 128 ? launch<__nv_bfloat16, 128>(a, most_tiles, st) : launch<__nv_bfloat16, 64>(a, most_tiles, st);
}

}  // namespace pa

int read_paged_tc_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_paged_tc_status, sizeof(int)) != cudaSuccess) return IE_ERR_LAUNCH;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_paged_tc_status, &z, sizeof(int));
  }
  return v;
}

cudaError_t set_paged_tc_wait_ns(unsigned long long ns) {
  return cudaMemcpyToSymbol(g_paged_tc_wait_ns, &ns, sizeof(ns));
}

}  // namespace ie
