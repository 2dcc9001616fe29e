// Paged attention of chunks of tokens on the 5th-generation tensor cores
// (tcgen05 + TMEM + TMA): the kernel of ie_paged_attention for more rows than
// the few-rows kernel takes.
//
// One CTA serves a piece: up to 256 (token, head) rows of one KV head, as two
// lanes of 128 rows (one TMEM lane a row), over a range of 128-key blocks.
// Both lanes use a key or value block from shared memory once it is there, so
// L2 sees half the traffic of 128-row tiles, and while one lane's softmax runs
// on its warps the tensor cores work for the other.
//
//   S = Q K^T  (fp32, TMEM)  ->  p = 2^(s c - m), c = scale log2 e  ->  O += P V
//
// The running maximum m is lazy: O is rescaled only when a row's maximum rises
// by more than 2^8 over the reference it uses; p then stays below 2^8, which
// neither type's rounding nor the fp32 sums notice, and after the first blocks
// nearly no row needs it. p is rounded to the storage type for the product, the
// sum takes the unrounded values.
//
// What bounds it: 128 x 128 scores cost 1024 cycles of tensor work (D = 128)
// and 1024 cycles of exponentials (16 a cycle and SM), so the two are balanced
// at best and the softmax chain has to stay off the tensor cores' path.
//
// TMEM columns: S0 [0, 128), S1 [128, 256), O0 [256, 256 + D), O1 [384, 384 +
// D); P overwrites the first 64 columns of the S it came from. Shared memory:
// the two Q tiles, a ring of 5 key / value blocks (10 of D = 64). Operands are
// 64-dimension halves of 128-byte rows, 128-byte swizzle: Q and K K-major, V
// MN-major as it arrives.
//
// Warp roles: 0 copies (TMA boxes of up to 128 rows of one page; the lanes
// hold the next table entries), 1 issues MMAs, 2 zeroes value rows that no row
// of the tile sees (range edges inside a block; what the page holds there may
// be NaN), 4-7 and 8-11 the lanes' softmax and epilogue. Every mbarrier wait is
// bounded: on expiry IE_ERR_TIMEOUT is recorded, all roles leave their loops,
// and MMAs and copies in flight are waited for before TMEM is freed.
#include <cstdio>
#include "ie_common.cuh"
#include "paged_attention.cuh"
#include "paged_ops.cuh"
#include "tc_ptx.cuh"

namespace ie {

__device__ int g_paged_tc_status = 0;
__device__ unsigned long long g_paged_tc_wait_ns = kDefaultWaitNs;

namespace pa {
namespace {

using namespace tc;

constexpr int kKB = 128;             // keys of a block
constexpr int kMT = kRowsChunk;      // rows of a tile: two lanes of 128
constexpr int kThreads = 384;
constexpr float kLazy = 8.0f;        // log2 of the growth of a row's maximum that O tolerates

template <int D>
struct Cfg {
  static constexpr int kTile = kKB * D * 2;                   // one Q lane, key or value block
  static constexpr int kHalf = kKB * 128;                     // its 64-dimension halves
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kOffRing = 2 * kTile;
  static constexpr int kOffBars = kOffRing + kStages * kTile;
  static constexpr int kSmem = kOffBars + 512 + 1024;         // + alignment slack
};
static_assert(Cfg<128>::kSmem <= 227 * 1024 - 1024, "shared memory per CTA");

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT<T>::id == IE_DTYPE_BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// D (TMEM) (+)= A (TMEM) . B (shared memory descriptor)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
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
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,"
      "%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];"
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
// 16 columns, as above
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_wait(bar, parity, abort_flag, &g_paged_tc_status, &g_paged_tc_wait_ns);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const __grid_constant__ Args a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
  __shared__ Scan scan;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_s, issued_s;
  volatile int* abort_flag = &abort_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + C::kStages + s); };
  constexpr int kB = 2 * C::kStages;
  const uint32_t q_full = smem_u32(bars + kB);
  auto s_full = [&](int i) { return smem_u32(bars + kB + 1 + i); };
  auto p_full = [&](int i) { return smem_u32(bars + kB + 3 + i); };
  auto pv_done = [&](int i) { return smem_u32(bars + kB + 5 + i); };
  const uint32_t drain_bar = smem_u32(bars + kB + 7);
  auto fixed_bar = [&](int s) { return smem_u32(bars + kB + 8 + s); };
  static_assert((kB + 8 + C::kStages) * 8 <= 512, "barriers");

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
      mbar_init(fixed_bar(s), 1);
    }
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_full(i), 4);
      mbar_init(pv_done(i), 1);
    }
    mbar_init(drain_bar, 1);
    abort_s = 0;
    issued_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!find_piece<kMT, kKB, kThreads>(a, blockIdx.x, scan, &g_paged_tc_status)) return;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)),
                 "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_holder;

  const Piece pc = scan.p;
  const Seq sq = sequence(a, pc.b);
  const int row0 = pc.tile * kMT, nrows = min(kMT, sq.tokens * a.group - row0);
  const int tok0 = row0 / a.group, tok1 = (row0 + nrows - 1) / a.group;
  const Keys ks = tile_keys<kKB>(a, sq, tok0, tok1);
  const int all = ks.blocks();
  const int j0 = (int)((int64_t)all * pc.piece / pc.pieces);
  const int n = (int)((int64_t)all * (pc.piece + 1) / pc.pieces) - j0;  // blocks of this piece
  const bool two = nrows > 128;

  // Registers: 384 x 168 at launch; the softmax warps take 216 each, the
  // others give up down to 56.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ------------------------------------------------ copies: K_0 V_0 K_1 V_1 ..
      const int box = min(a.l.page_size, kKB), boxes = kKB / box;  // 1 .. 8
      const int per_batch = 32 / boxes;
      const int* table = a.b.page_table + (int64_t)pc.b * a.b.ld_table;
      auto load_entries = [&](int it0) {
        const int it = it0 + lane / boxes;
        if (it >= n) return -1;
        const int kb = ks.block(j0 + it) * kKB + (lane % boxes) * box;
        if (!(kb < ks.hi && (kb + box > ks.lo || kb < ks.sink_end))) return -1;
        const int page = table[kb >> a.l.page_log2];
        if (page < 0 || page >= a.l.num_pages) {
          atomicExch(&g_paged_tc_status, IE_ERR_INVALID_ARG);
          return a.l.num_pages;  // outside the tensor map: zeros
        }
        return page;
      };
      int entries = load_entries(0), next = load_entries(per_batch), batch = 0, issued = 0;
      for (int t = 0; t < 2 * n; ++t) {
        const int it = t >> 1, s = t % C::kStages;
        if (it >= batch + per_batch) {
          batch += per_batch;
          entries = next;
          next = load_entries(batch + per_batch);
        }
        if (!__all_sync(0xffffffffu, wait(empty_bar(s), (uint32_t)(((t / C::kStages) & 1) ^ 1), abort_flag))) break;
        // lane x * (D / 64) + h copies half h of box x
        const int x = lane / (D / 64), h = lane % (D / 64);
        const int page = __shfl_sync(0xffffffffu, entries, (it - batch) * boxes + min(x, boxes - 1));
        const bool mine = x < boxes && page >= 0;
        const int copies = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) mbar_expect_tx(full_bar(s), copies * box * 128);
        __syncwarp();
        if (mine) {
          const int kb = ks.block(j0 + it) * kKB + x * box, r = kb & (a.l.page_size - 1);
          tma_load_4d(smem_u32(smem + C::kOffRing + s * C::kTile) + h * C::kHalf + x * box * 128,
                      (t & 1) ? &a.tmV : &a.tmK, full_bar(s), 64 * h, a.swap_rc ? pc.head : r, a.swap_rc ? r : pc.head,
                      page);
        }
        issued = t + 1;
      }
      if (lane == 0) issued_s = issued;
    } else if (warp == 1) {
      if (lane == 0) {
        // ---------------------------------------------- MMAs
        const uint32_t id_qk = idesc_f16<T>(128, kKB, 0), id_pv = idesc_f16<T>(128, D, 1);
        const uint32_t ring = smem_u32(smem + C::kOffRing);
        bool any = false;
        auto qk = [&](int i, int it) {  // S_i = Q_i K_it^T (copy 2 it)
          if (it > 0 && !wait(pv_done(i), (uint32_t)((it - 1) & 1), abort_flag)) return false;
          fence_after();
          const uint32_t sk = ring + (uint32_t)((2 * it) % C::kStages) * C::kTile;
          const uint32_t sq_ = smem_u32(smem) + i * C::kTile;
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_f16(tmem + 128 * i, sw128_desc(sq_ + (uint32_t)(k >> 2) * C::kHalf) + 2 * (k & 3),
                    sw128_desc(sk + (uint32_t)(k >> 2) * C::kHalf) + 2 * (k & 3), id_qk, k != 0 ? 1u : 0u);
          mma_commit(s_full(i));
          any = true;
          return true;
        };
        auto pv = [&](int i, int it) {  // O_i += P_i V_it (copy 2 it + 1)
          if (!wait(p_full(i), (uint32_t)(it & 1), abort_flag)) return false;
          fence_after();
          const uint32_t sv = ring + (uint32_t)((2 * it + 1) % C::kStages) * C::kTile;
#pragma unroll
          for (int k = 0; k < kKB / 16; ++k)
            mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * k, sw128_desc_mn(sv + (uint32_t)k * 16 * 128, C::kHalf),
                   id_pv, (it | k) != 0 ? 1u : 0u);
          mma_commit(pv_done(i));
          any = true;
          return true;
        };
        auto arrived = [&](int t) {
          return wait(full_bar(t % C::kStages), (uint32_t)((t / C::kStages) & 1), abort_flag);
        };
        auto release = [&](int t) { mma_commit(empty_bar(t % C::kStages)); };
        bool ok = wait(q_full, 0, abort_flag);
        fence_after();
        if (ok && n > 0) {
          ok = arrived(0) && qk(0, 0) && (!two || qk(1, 0));
          if (ok) release(0);
          for (int it = 0; ok && it < n; ++it) {
            // P_0 V_it, S_0 of the next block, P_1 V_it, S_1 of the next block
            ok = arrived(2 * it + 1) && wait(fixed_bar(it % C::kStages), (uint32_t)((it / C::kStages) & 1), abort_flag);
            const bool more = it + 1 < n;
            ok = ok && pv(0, it);
            if (!two && ok) release(2 * it + 1);
            if (ok && more) ok = arrived(2 * it + 2) && qk(0, it + 1);
            if (!two && ok && more) release(2 * it + 2);
            if (two) {
              ok = ok && pv(1, it);
              if (ok) release(2 * it + 1);
              if (ok && more) ok = qk(1, it + 1);
              if (ok && more) release(2 * it + 2);
            }
          }
        }
        if (*abort_flag && any) {
          mma_commit(drain_bar);
          const unsigned long long t0 = globaltimer();
          while (!mbar_try(drain_bar, 0) && globaltimer() - t0 < kDrainWaitNs) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // ------------------------------------------------ value rows nobody sees
      // (it passes every value block on, so that it never falls a ring behind)
      for (int it = 0; it < n; ++it) {
        const int kb = ks.block(j0 + it) * kKB;
        const int t = 2 * it + 1, s = t % C::kStages;
        if (!__all_sync(0xffffffffu, wait(full_bar(s), (uint32_t)((t / C::kStages) & 1), abort_flag))) break;
        if (kb + kKB > ks.hi || (kb < ks.lo && kb + kKB > ks.sink_end)) {
          uint8_t* v = smem + C::kOffRing + s * C::kTile;
          for (int r = lane; r < kKB; r += 32) {
            const int j = kb + r;
            if (!(j < ks.hi && (j >= ks.lo || j < ks.sink_end)))
#pragma unroll
              for (int c = 0; c < D / 8; ++c)
                *reinterpret_cast<uint4*>(v + (c >> 3) * C::kHalf + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(fixed_bar(it % C::kStages));  // by value block: keys use the stages too
      }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------ softmax and epilogue
    const int i = (warp - 4) >> 2, quad = warp & 3;  // TMEM lane quarter = warp & 3
    const int r = 32 * quad + lane, row = 128 * i + r;
    const uint32_t tl = (uint32_t)(32 * quad) << 16;
    const uint32_t ts = tmem + tl + 128 * i, to = tmem + tl + 256 + 128 * i;
    {
      // this warp's 32 rows of Q, D / 8 lanes a row
      constexpr int kChunks = D / 8, kRows = 32 / kChunks;
      uint8_t* qs = smem + i * C::kTile;
#pragma unroll 4
      for (int x = 0; x < 32 / kRows; ++x) {
        const int rr = 32 * quad + x * kRows + lane / kChunks, c = lane % kChunks, g = row0 + 128 * i + rr;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (128 * i + rr < nrows)
          w = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(sq.start + g / a.group) * a.ldq +
                                              (int64_t)(pc.head * a.group + g % a.group) * a.hsq + 8 * c);
        *reinterpret_cast<uint4*>(qs + (c >> 3) * C::kHalf + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = w;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const int tok = (row0 + row) / a.group;
    const int pos = row < nrows ? sq.pos0 + tok : -1;
    const int pos_min = sq.pos0 + (row0 + 128 * i) / a.group;
    const int pos_max = sq.pos0 + (row0 + min(nrows, 128 * i + 128) - 1) / a.group;
    // a scale of 0 weighs all seen keys alike: scores 0, so that masked ones can stay infinite
    const bool flat = a.scale_log2 == 0.f;
    const float c = flat ? 1.0f : a.scale_log2;
    const float hidden = c > 0.f ? -INFINITY : INFINITY;
    float m = -INFINITY, l = 0.f;  // m: the reference, in log2 units
    bool ok = true;
    if (i == 0 || two) {
      for (int it = 0; it < n; ++it) {
        const int kb = ks.block(j0 + it) * kKB;
        if (!wait(s_full(i), (uint32_t)(it & 1), abort_flag)) { ok = false; break; }
        fence_after();
        float v[128];
        {
          uint32_t r0[64], r1[64];
          tmem_ld(ts, r0);
          tmem_ld(ts + 64, r1);
          tmem_ld_wait(r0);
          tmem_ld_wait(r1);
#pragma unroll
          for (int x = 0; x < 64; ++x) {
            v[x] = __uint_as_float(r0[x]);
            v[64 + x] = __uint_as_float(r1[x]);
          }
        }
        if (flat) {
#pragma unroll
          for (int x = 0; x < 128; ++x) v[x] = 0.f;
        }
        if (kb + kKB - 1 > pos_min || (a.window && (int64_t)pos_max - kb >= a.window)) {
          const int hi = pos - kb;  // columns <= hi
          if (!a.window) {
#pragma unroll
            for (int x = 0; x < 128; ++x) v[x] = x <= hi ? v[x] : hidden;
          } else {
            const int64_t lo64 = (int64_t)pos - a.window - kb;
            const int lo = (int)(lo64 < -1 ? -1 : lo64), sk = a.sinks - kb;  // columns > lo or < sk
#pragma unroll
            for (int x = 0; x < 128; ++x)
              v[x] = x <= hi && (x > lo || x < sk) ? v[x] : hidden;
          }
        }
        // the row's largest scaled score
        float t[4] = {v[0], v[1], v[2], v[3]};
        if (c > 0.f) {
#pragma unroll
          for (int x = 4; x < 128; ++x) t[x & 3] = fmaxf(t[x & 3], v[x]);
          t[0] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        } else {
#pragma unroll
          for (int x = 4; x < 128; ++x) t[x & 3] = fminf(t[x & 3], v[x]);
          t[0] = fminf(fminf(t[0], t[1]), fminf(t[2], t[3]));
        }
        const float top = t[0] * c;
        const bool rise = top > m + kLazy;
        if (__any_sync(0xffffffffu, rise)) {
          const float to_m = rise ? top : m;
          const float f = rise ? ex2(m - to_m) : 1.0f;
          if (it > 0) {
            if (!wait(pv_done(i), (uint32_t)((it - 1) & 1), abort_flag)) { ok = false; break; }
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
        const float mb = m == -INFINITY ? 0.f : -m;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t pk[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const float e0 = ex2(fmaf(v[32 * x + 2 * y], c, mb)), e1 = ex2(fmaf(v[32 * x + 2 * y + 1], c, mb));
            l0 += e0;
            l1 += e1;
            pk[y] = pack2<T>(e0, e1);
          }
          tmem_st(ts + 16 * x, pk);
        }
        l += l0 + l1;
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(i));
      }
    }
    // ---- epilogue: one row a thread
    const bool cut = pc.slot >= 0;
    if (ok && n > 0 && (i == 0 || two)) ok = wait(pv_done(i), (uint32_t)((n - 1) & 1), abort_flag);
    if (ok && !*abort_flag && 128 * i < nrows && (!cut || (pc.slot < a.slot_cap && pc.split < a.split_cap))) {
      fence_after();
      const float inv = l > 0.f ? 1.0f / l : 0.f;
      const int g = row0 + row;
      T* dst = static_cast<T*>(a.out) + (int64_t)(sq.start + g / a.group) * a.ld_out +
               (int64_t)(pc.head * a.group + g % a.group) * D;
      float* po = a.part_o + ((int64_t)pc.slot * kMT + row) * D;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        float o[32];
        if (n > 0) {
          uint32_t w[32];
          tmem_ld(to + 32 * x, w);
          tmem_ld_wait(w);
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __uint_as_float(w[y]);
        } else {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = 0.f;
        }
        if (row < nrows) {
          if (cut) {
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              *reinterpret_cast<float4*>(po + 32 * x + y) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          } else {
#pragma unroll
            for (int y = 0; y < 32; y += 8) {
              uint4 w;
              w.x = pack2<T>(o[y] * inv, o[y + 1] * inv);
              w.y = pack2<T>(o[y + 2] * inv, o[y + 3] * inv);
              w.z = pack2<T>(o[y + 4] * inv, o[y + 5] * inv);
              w.w = pack2<T>(o[y + 6] * inv, o[y + 7] * inv);
              *reinterpret_cast<uint4*>(dst + 32 * x + y) = w;
            }
          }
        }
      }
      if (cut && row < nrows) a.part_ml[(int64_t)pc.slot * kMT + row] = make_float2(m, l);
      if (cut && pc.piece == 0 && row == 0) {
        Split s = {};
        s.slot0 = pc.slot;
        s.pieces = pc.pieces;
        s.token0 = sq.start;
        s.rows = nrows;
        s.head0 = pc.head * a.group;
        s.row0 = row0;
        a.splits[pc.split] = s;
      }
    }
  }

  // ---------------------------------------------------------- teardown
  fence_before();
  __syncthreads();
  fence_after();
  if (*abort_flag && threadIdx.x == 0) {
    // copies still in flight land before the CTA exits: the last kStages
    for (int t = max(0, issued_s - C::kStages); t < issued_s; ++t) {
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(full_bar(t % C::kStages), (uint32_t)((t / C::kStages) & 1)) &&
             globaltimer() - t0 < kDrainWaitNs / 4) {
      }
    }
  }
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

template <typename T, int D>
int launch(Args& a, int64_t grid, cudaStream_t st) {
  auto kernel = chunk_kernel<T, D>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return IE_ERR_LAUNCH;
  static bool configured[64] = {};
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem) != cudaSuccess)
      return IE_ERR_LAUNCH;
    configured[dev] = true;
  }
  kernel<<<(unsigned)grid, kThreads, Cfg<D>::kSmem, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    std::fprintf(stderr, "infengine_b200: paged attention launch failed: %s\n", cudaGetErrorString(e));
    return IE_ERR_LAUNCH;
  }
  return IE_OK;
}

}  // namespace

int launch_chunks(ie_dtype dt, int D, Args& a, int64_t grid, cudaStream_t st) {
  if (dt == IE_DTYPE_F16) return D == 128 ? launch<__half, 128>(a, grid, st) : launch<__half, 64>(a, grid, st);
  return D == 128 ? launch<__nv_bfloat16, 128>(a, grid, st) : launch<__nv_bfloat16, 64>(a, grid, st);
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
