// Attention of new tokens over a paged cache: entry point and the kernel for
// few rows.
//
//   x_j = scale * q . k_j        keys j <= position with (position - j < window or j < sinks)
//   o   = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m)       zeros where no key is seen
//
// in one pass with a running maximum m (base 2, scale * log2 e folded into one
// factor), fp32 throughout; p_j is rounded to the storage type for the tensor
// cores (fp16 with the maximum at 2^15, see paged_attention.cuh) and the sum
// takes the rounded values, so a rounding of p moves weight between keys but not
// the total.
//
// few_rows_kernel (at most 16 (token, head) rows a tile: decode, verification
// of a few draft tokens). What bounds it: a cache row of 512 bytes costs
// 16 flop a byte, far below the tensor cores, so the cache's bytes over HBM do,
// and for short contexts the latency of one chain (page entry, copy, scores,
// softmax, values, join). A warp works alone on its own range of keys, 32 at a
// time: its lane 0 keeps copies of the next key and value blocks in flight
// into the warp's ring (TMA boxes of up to 32 rows of one page x 64
// dimensions, 128-byte swizzle, conflict-free for ldmatrix), the products run
// as m16n8k16 with the rows as M, and no barrier is shared between warps until
// the four warps' outputs meet at the end. 96 KB of ring a CTA, two CTAs an SM:
// 192 KB of copies in flight an SM, above the ~50 KB that HBM latency needs.
// The CTA that finishes a cut tile's last piece joins the pieces in their order:
// with M = max_s m_s the output is sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s
// (a joining kernel in its place cost a decode step of one row 3 us more).
//
// A block's box is copied only if some row of the tile sees one of its keys, so
// table entries outside the visible range are never followed; visible range's
// edges inside a box are zeroed in shared memory before the product, so what a
// page holds there (NaN included) does not reach a sum.
#include <atomic>
#include <cstdio>
#include <cstring>
#include "ie_common.cuh"
#include "paged_attention.cuh"
#include "paged_ops.cuh"
#include "norm.cuh"
#include "tc_ptx.cuh"

namespace ie {

__device__ int g_paged_attn_status = 0;
__device__ unsigned long long g_paged_attn_wait_ns = kDefaultWaitNs;

namespace pa {
namespace {

using namespace tc;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kKB = 32;           // keys of a warp's block
constexpr int kMT = kRowsFew;
constexpr int kRingBytes = 24576;  // a warp's ring

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT<T>::id == IE_DTYPE_F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t r) {
  if constexpr (DT<T>::id == IE_DTYPE_BF16)
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&r));
}

// The bounded loop of a wait, out of line: this kernel's code is run through
// about once, and its fetches are a fifth of a short call's time.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_wait(bar, parity, abort_flag, &g_paged_attn_status, &g_paged_attn_wait_ns);
}

// kPolled: for wait limits that a suspended wait would outlast (compiled apart,
// since the choice at each wait took the chunk kernel 4 to 6 % longer).
template <typename T, int D, bool kPolled>
__global__ void __launch_bounds__(kThreads, 2) few_rows_kernel(const __grid_constant__ Args a) {
  constexpr int kSlotBytes = kKB * D * 2;         // a key or value block: D / 64 halves of 32 rows x 128 bytes
  constexpr int kSlots = kRingBytes / kSlotBytes;  // 3 (D = 128) or 6
  constexpr int kHalf = kKB * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[kWarps * kSlots];
  __shared__ Scan scan;
  __shared__ float sm_m[kWarps][kMT], sm_l[kWarps][kMT];
  __shared__ int abort_s, last_s;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 32) {
    for (int i = 0; i < kWarps * kSlots; ++i) mbar_init(smem_u32(bars + i), 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&a.tmK);
    prefetch_map(&a.tmV);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!find_piece<kKB, kThreads>(a, blockIdx.x, scan, &g_paged_attn_status)) return;
  const Piece pc = scan.p;
  const Seq sq = scan.seq;
  const int rows = sq.tokens * a.group;
  const int row0 = pc.tile * kMT, nrows = min(kMT, rows - row0);
  const int tok0 = row0 / a.group, tok1 = (row0 + nrows - 1) / a.group;
  const Keys ks = tile_keys<kKB>(a, sq, tok0, tok1);
  const int nb = ks.blocks();
  int p0, np, j0, n;  // the piece's blocks, this warp's
  piece_range(nb, pc.pieces, pc.piece, p0, np);
  piece_range(np, kWarps, warp, j0, n);
  j0 += p0;

  uint8_t* ring = smem + warp * kRingBytes;
  const uint32_t ring_u = smem_u32(ring), bar_u = smem_u32(bars + warp * kSlots);
  volatile int* abort_flag = &abort_s;
  const int* table = a.b.page_table + (int64_t)pc.b * a.b.ld_table;
  const int box = min(a.l.page_size, kKB), boxes = kKB / box;  // rows of a copy, copies of a block's half
  const int per_batch = 32 / boxes;                            // blocks whose table entries a warp holds

  auto box_seen = [&](int kb) { return kb < ks.hi && (kb + box > ks.lo || kb < ks.sink_end); };
  // entry `lane` of the batch of blocks it0 ..: its page, -1 where no copy is made
  auto load_entries = [&](int it0) {
    const int it = it0 + lane / boxes;
    if (it >= n) return -1;
    const int kb = ks.block(j0 + it) * kKB + (lane % boxes) * box;
    if (!box_seen(kb)) return -1;
    const int page = table[kb >> a.l.page_log2];
    if (page < 0 || page >= a.l.num_pages) {
      atomicExch(&g_paged_attn_status, IE_ERR_INVALID_ARG);
      return a.l.num_pages;  // outside the tensor map: zeros
    }
    return page;
  };
  int entries = load_entries(0), entries_next = load_entries(per_batch), batch = 0;
  // copy i: keys of block i / 2 (even) or values (odd)
  auto issue = [&](int i) {
    const int it = i >> 1;
    if (it >= n) return;
    if (it >= batch + per_batch) {
      batch += per_batch;
      entries = entries_next;
      entries_next = load_entries(batch + per_batch);
    }
    const int slot = i % kSlots;
    const uint32_t dst = ring_u + slot * kSlotBytes, bar = bar_u + 8 * slot;
    const int kb = ks.block(j0 + it) * kKB;
    const CUtensorMap* map = (i & 1) ? &a.tmV : &a.tmK;
    int pages[2];
    pages[0] = __shfl_sync(0xffffffffu, entries, (it - batch) * boxes);
    pages[1] = boxes == 2 ? __shfl_sync(0xffffffffu, entries, (it - batch) * boxes + 1) : -1;
    if (lane == 0) {
      mbar_expect_tx(bar, ((pages[0] >= 0) + (pages[1] >= 0)) * box * D * 2);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (pages[x] >= 0) {
          const int r = (kb + x * box) & (a.l.page_size - 1);
#pragma unroll
          for (int h = 0; h < D / 64; ++h)
            tma_load_4d(dst + h * kHalf + x * box * 128, map, bar, 64 * h, a.swap_rc ? pc.head : r,
                        a.swap_rc ? r : pc.head, pages[x]);
        }
    }
  };

  // Q as A operands (rows lane / 4 and lane / 4 + 8)
  const int g = lane >> 2, tq = lane & 3;
  uint32_t qa[D / 16][4];
  int pos[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = g + 8 * x;
    const int tok = (row0 + r) / a.group;
    pos[x] = sq.pos0 + tok;
    const T* qr = static_cast<const T*>(a.q) + (int64_t)(sq.start + tok) * a.ldq +
                  (int64_t)(pc.head * a.group + (row0 + r) % a.group) * a.hsq;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qa[k][x] = r < nrows ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 2 * tq) : 0u;
      qa[k][x + 2] = r < nrows ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 8 + 2 * tq) : 0u;
    }
  }
  __syncthreads();  // the barriers are initialised
#pragma unroll 1
  for (int i = 0; i < kSlots; ++i) issue(i);

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  constexpr float kTop = DT<T>::id == IE_DTYPE_F16 ? kLargestLog2F16 : 0.f;  // log2 of the largest p
  const int pos_min = sq.pos0 + tok0, pos_max = sq.pos0 + tok1;
  auto wait = [&](int i) {
    const uint32_t bar = bar_u + 8 * (i % kSlots), parity = (uint32_t)((i / kSlots) & 1);
    if constexpr (kPolled) return mbar_poll(bar, parity, abort_flag, &g_paged_attn_status, &g_paged_attn_wait_ns);
    else return mbar_try(bar, parity) || wait_long(bar, parity, abort_flag);
  };
  int done = 0;  // copies waited for
  bool ok = true;
  for (int it = 0; it < n; ++it) {
    const int kb = ks.block(j0 + it) * kKB;
    // ---- scores
    ok = __all_sync(0xffffffffu, wait(2 * it));
    if (!ok) break;
    float s[kKB / 8][4];
#pragma unroll
    for (int i = 0; i < kKB / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    {
      const uint32_t base = ring_u + (2 * it % kSlots) * kSlotBytes;
      const int key = ((lane >> 4) & 1) * 8 + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int y = 0; y < kKB / 16; ++y) {
          uint32_t b[4];
          const int row = y * 16 + key, c16 = 2 * k + c;
          ldsm4(base + (c16 >> 3) * kHalf + row * 128 + (((c16 & 7) ^ (row & 7)) << 4), b);
          mma16816<T>(s[2 * y], qa[k], b[0], b[1]);
          mma16816<T>(s[2 * y + 1], qa[k], b[2], b[3]);
        }
    }
    __syncwarp();
    issue(2 * it + kSlots);
    done = 2 * it + 1;
    // ---- softmax over the block: columns 8i + 2 tq + {0, 1}, rows g and g + 8
#pragma unroll
    for (int i = 0; i < kKB / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] *= a.scale_log2;
    if (kb + kKB - 1 > pos_min || (a.window && (int64_t)pos_max - kb >= a.window)) {
#pragma unroll
      for (int i = 0; i < kKB / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = kb + 8 * i + 2 * tq + (e & 1), p = pos[e >> 1];
          const bool seen = j <= p && j < ks.hi && (!a.window || p - j < a.window || j < a.sinks);
          s[i][e] = seen ? s[i][e] : -INFINITY;
        }
    }
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int i = 0; i < kKB / 8; ++i) {
      mx[0] = fmaxf(mx[0], fmaxf(s[i][0], s[i][1]));
      mx[1] = fmaxf(mx[1], fmaxf(s[i][2], s[i][3]));
    }
    float base[2];
    bool moved = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
      base[x] = mx[x] == -INFINITY ? 0.f : mx[x];
      moved = moved || mx[x] != m[x];
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f = ex2(m[x] - base[x]);
        l[x] *= f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][2 * x] *= f;
          o[i][2 * x + 1] *= f;
        }
        m[x] = mx[x];
      }
    }
    const float one[2] = {base[0] - kTop, base[1] - kTop};  // the score whose p is 1
    uint32_t pa[kKB / 16][4];
#pragma unroll
    for (int i = 0; i < kKB / 8; ++i) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t w = pack2<T>(ex2(s[i][2 * x] - one[x]), ex2(s[i][2 * x + 1] - one[x]));
        const float2 r = unpack2<T>(w);
        l[x] += r.x + r.y;
        pa[i >> 1][2 * (i & 1) + x] = w;
      }
    }
    // ---- values
    ok = __all_sync(0xffffffffu, wait(2 * it + 1));
    if (!ok) break;
    uint8_t* vb = ring + ((2 * it + 1) % kSlots) * kSlotBytes;
    if (kb + kKB > ks.hi || (kb < ks.lo && kb + kKB > ks.sink_end)) {
      const int j = kb + lane;  // one row a lane
      if (!(j < ks.hi && (j >= ks.lo || j < ks.sink_end))) {
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4*>(vb + (c >> 3) * kHalf + lane * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into this slot
      __syncwarp();
    }
    {
      const uint32_t vu = smem_u32(vb);
      const int key = ((lane >> 3) & 1) * 8 + (lane & 7), c = lane >> 4;
#pragma unroll
      for (int y = 0; y < kKB / 16; ++y)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t b[4];
          const int row = y * 16 + key, c16 = 2 * k + c;
          ldsm4_t(vu + (c16 >> 3) * kHalf + row * 128 + (((c16 & 7) ^ (row & 7)) << 4), b);
          mma16816<T>(o[2 * k], pa[y], b[0], b[1]);
          mma16816<T>(o[2 * k + 1], pa[y], b[2], b[3]);
        }
    }
    __syncwarp();
    issue(2 * it + 1 + kSlots);
    done = 2 * it + 2;
  }
  if (!ok) {
    // copies in flight land before the CTA leaves (bounded; they always end)
    const int issued = min(2 * n, done + kSlots);
    for (int i = done; i < issued; ++i) {
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(bar_u + 8 * (i % kSlots), (uint32_t)((i / kSlots) & 1)) && globaltimer() - t0 < kDrainWaitNs) {
      }
    }
  }

  // ---- the four warps meet: scale to the common maximum, add in warp order
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    if (tq == 0) {
      sm_m[warp][g + 8 * x] = m[x];
      sm_l[warp][g + 8 * x] = l[x];
    }
  }
  __syncthreads();
  const bool cut = pc.slot >= 0 && pc.slot < a.slot_cap && pc.split < a.split_cap;
  bool good = !abort_s && (cut || pc.slot < 0);
  float* acc = reinterpret_cast<float*>(ring);  // [16][D], this warp's
  // 16-byte columns of the rows a quad writes together are spread over the banks
  auto at = [&](int r, int d) { return r * D + (d ^ (8 * (r & 3))); };
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (8 * x < nrows) {
      const int r = g + 8 * x;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(acc + at(r, 8 * i + 2 * tq)) = make_float2(o[i][2 * x], o[i][2 * x + 1]);
    }
  __syncthreads();
  constexpr int kPer = kMT * D / kThreads;  // consecutive outputs of a thread
  const int r = tid / (D / kPer), d0 = (tid % (D / kPer)) * kPer;
  float v[kPer], top = sm_m[0][r], sum = 0.f;
  // the warps' parts of this thread's outputs at their common maximum, in warp order
  auto add_up = [&] {
    top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = 0.f;
#pragma unroll 1
    for (int w = 0; w < kWarps; ++w) {
      const float f = top == -INFINITY ? 0.f : ex2(sm_m[w][r] - top);
      sum += f * sm_l[w][r];
      const float* p = reinterpret_cast<const float*>(smem + w * kRingBytes);
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const float4 u = *reinterpret_cast<const float4*>(p + at(r, d0 + i));
        v[i] += f * u.x;
        v[i + 1] += f * u.y;
        v[i + 2] += f * u.z;
        v[i + 3] += f * u.w;
      }
    }
  };
  if (good && r < nrows) add_up();
  if (cut) {
    if (good && r < nrows) {
      float* po = a.part_o + ((int64_t)pc.slot * kMT + r) * D + d0;
#pragma unroll
      for (int i = 0; i < kPer; i += 4)
        __stcg(reinterpret_cast<float4*>(po + i), make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
      if (d0 == 0) __stcg(a.part_ml + (int64_t)pc.slot * kMT + r, make_float2(top, sum));
    }
    // (a piece that gave up arrives too, so that the count ends at 0 whatever happens)
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const int before = atomicAdd(a.arrived + pc.split, 1);
      last_s = before == pc.pieces - 1;
      if (last_s) a.arrived[pc.split] = 0;
      __threadfence();
    }
    __syncthreads();
    if (!last_s) return;
    // ---- join: warp w takes every fourth piece, four rows at a time, lane l
    // the outputs from D / 32 * l on; each warp at its own pieces' maximum
    constexpr int kV = D / 32;
    const int64_t stride = (int64_t)a.l.n_kv_heads * kMT, first = (int64_t)pc.slot * kMT - pc.piece * stride;
    const float2* ml = a.part_ml + first + min(lane, kMT - 1);
    float most = -INFINITY, total = 0.f;
#pragma unroll 4
    for (int s = warp; s < pc.pieces; s += kWarps) most = fmaxf(most, __ldcg(ml + s * stride).x);
#pragma unroll 1
    for (int q0 = 0; q0 < nrows; q0 += 4) {
      float part[4][kV] = {};
      total = 0.f;
#pragma unroll 4
      for (int s = warp; s < pc.pieces; s += kWarps) {
        const float2 x = __ldcg(ml + s * stride);
        const float f = x.x == -INFINITY ? 0.f : ex2(x.x - most);
        total += f * x.y;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int q = min(q0 + y, nrows - 1);
          const float fq = __shfl_sync(0xffffffffu, f, q);
          const float* po = a.part_o + (first + s * stride + q) * D + lane * kV;
          if constexpr (kV == 4) {
            const float4 u = __ldcg(reinterpret_cast<const float4*>(po));
            part[y][0] += fq * u.x;
            part[y][1] += fq * u.y;
            part[y][2] += fq * u.z;
            part[y][3] += fq * u.w;
          } else {
            const float2 u = __ldcg(reinterpret_cast<const float2*>(po));
            part[y][0] += fq * u.x;
            part[y][1] += fq * u.y;
          }
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (q0 + y < nrows)
#pragma unroll
          for (int i = 0; i < kV; i += 2)
            *reinterpret_cast<float2*>(acc + at(q0 + y, lane * kV + i)) = make_float2(part[y][i], part[y][i + 1]);
    }
    if (lane < kMT) {
      sm_m[warp][lane] = most;
      sm_l[warp][lane] = total;
    }
    __syncthreads();
    if (r < nrows) add_up();
    good = true;
  }
  if (good && r < nrows) {
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    const int tok = (row0 + r) / a.group;
    T* dst = static_cast<T*>(a.out) + (int64_t)(sq.start + tok) * a.ld_out +
             (int64_t)(pc.head * a.group + (row0 + r) % a.group) * D + d0;
#pragma unroll
    for (int i = 0; i < kPer; i += 8) {
      uint4 w;
      w.x = pack2<T>(v[i] * inv, v[i + 1] * inv);
      w.y = pack2<T>(v[i + 2] * inv, v[i + 3] * inv);
      w.z = pack2<T>(v[i + 4] * inv, v[i + 5] * inv);
      w.w = pack2<T>(v[i + 6] * inv, v[i + 7] * inv);
      *reinterpret_cast<uint4*>(dst + i) = w;
    }
  }
}

// A page's rows as boxes of 64 dimensions x `box` rows of one head and page,
// zeros outside. The map lists row and head in the order of their strides.
bool make_map(CUtensorMap* map, ie_dtype dt, const void* base, int D, const PagedLayout& l, int box, bool swap) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)(swap ? l.n_kv_heads : l.page_size),
                        (cuuint64_t)(swap ? l.page_size : l.n_kv_heads), (cuuint64_t)l.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)(swap ? l.head_stride : l.row_stride) * 2,
                           (cuuint64_t)(swap ? l.row_stride : l.head_stride) * 2, (cuuint64_t)l.page_stride * 2};
  cuuint32_t boxes[4] = {64, (cuuint32_t)(swap ? 1 : box), (cuuint32_t)(swap ? box : 1), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t =
      dt == IE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, t, 4, const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// The queries as boxes of 64 dimensions x the heads of a group x `tokens`.
bool make_q_map(CUtensorMap* map, ie_dtype dt, const void* q, int D, int T, int heads, int64_t ld, int64_t hs,
                int group, int tokens) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)(T > 1 ? ld : D) * 2};
  cuuint32_t boxes[3] = {64, (cuuint32_t)group, (cuuint32_t)tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType t =
      dt == IE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, t, 3, const_cast<void*>(q), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

template <typename K>
int launch(K kernel, dim3 grid, int threads, size_t smem, bool pdl, cudaStream_t st, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), args);
  if (e != cudaSuccess) {
    std::fprintf(stderr, "infengine_b200: paged attention launch failed: %s\n", cudaGetErrorString(e));
    return IE_ERR_LAUNCH;
  }
  return IE_OK;
}

template <typename T, int D, bool kPolled>
int launch_few(Args& a, int64_t grid, cudaStream_t st) {
  if (!kPolled && a.polled) return launch_few<T, D, true>(a, grid, st);
  constexpr size_t kSmem = kWarps * kRingBytes + 1024;
  auto kernel = few_rows_kernel<T, D, kPolled>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return IE_ERR_LAUNCH;
  static bool configured[64] = {};
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess)
      return IE_ERR_LAUNCH;
    configured[dev] = true;
  }
  void* args[] = {&a};
  return launch(kernel, dim3((unsigned)grid), kThreads, kSmem, pdl_launch_enabled() && a.b.T <= pdl_max_rows(), st,
                args);
}

// workspace: pieces done of each tile (few rows) and handed out (chunks), zeroed by the caller once |
// number of cut tiles | their descriptions (chunks) | (maximum, sum) | outputs
constexpr int kCapSplits = kTargetFew > kTargetChunk ? kTargetFew : kTargetChunk;
constexpr int64_t kSlotRowsFew = (int64_t)2 * kTargetFew * kRowsFew;
constexpr int64_t kSlotRowsChunk = (int64_t)2 * kTargetChunk * kRowsChunk;
constexpr int64_t kSlotRows = kSlotRowsFew > kSlotRowsChunk ? kSlotRowsFew : kSlotRowsChunk;
constexpr size_t kOffCount = 65536, kOffQueue = kOffCount - 64;
static_assert(kCapSplits * sizeof(int) <= kOffQueue, "counters");
constexpr size_t kOffSplits = kOffCount + 64;
constexpr size_t kOffMl = kOffSplits + kCapSplits * sizeof(Split);
constexpr size_t kOffO = kOffMl + kSlotRows * sizeof(float2);
constexpr size_t kWorkspace = kOffO + kSlotRows * 128 * sizeof(float);
static_assert(kOffSplits % 16 == 0 && kOffMl % 16 == 0 && kOffO % 16 == 0, "alignment of the workspace's parts");

}  // namespace
}  // namespace pa

int read_paged_attn_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_paged_attn_status, sizeof(int)) != cudaSuccess) return IE_ERR_LAUNCH;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_paged_attn_status, &z, sizeof(int));
  }
  return v;
}

namespace {
// By device: whether its waits' limit is one that a suspended wait could outlast.
constexpr unsigned long long kPolledBelowNs = 1000000;
std::atomic<bool> limit_is_short[64];
}  // namespace

cudaError_t set_paged_attn_wait_ns(unsigned long long ns) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64) limit_is_short[dev].store(ns < kPolledBelowNs, std::memory_order_relaxed);
  return cudaMemcpyToSymbol(g_paged_attn_wait_ns, &ns, sizeof(ns));
}

}  // namespace ie

using namespace ie;

extern "C" size_t ie_paged_attention_workspace_size(void) { return pa::kWorkspace; }

extern "C" int ie_paged_attention(ie_dtype dt, int B, int T, int max_q, int n_q_heads, const void* q, int64_t ldq,
                                  int64_t q_head_stride, const ie_paged_cache* cache, const int* page_table,
                                  int64_t ld_table, int max_pages, const int* q_start, const int* kv_len, int window,
                                  int sinks, float scale, void* out, int64_t ld_out, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace pa;
  if ((dt != IE_DTYPE_F16 && dt != IE_DTYPE_BF16) || n_q_heads <= 0 || max_q < 0 || window < 0 || sinks < 0)
    return IE_ERR_INVALID_ARG;
  int s = check_paged(cache, B, T, page_table, ld_table, max_pages, q_start, kv_len);
  if (s) return s;
  if (n_q_heads % cache->n_kv_heads) return IE_ERR_UNSUPPORTED;
  const int D = cache->head_dim, group = n_q_heads / cache->n_kv_heads;
  if (group > kRowsFew) return IE_ERR_UNSUPPORTED;
  if (!(scale > -INFINITY && scale < INFINITY)) return IE_ERR_INVALID_ARG;
  if (sinks && !window) return IE_ERR_INVALID_ARG;
  if (B == 0 || T == 0 || max_q == 0) return IE_OK;
  if (!q || !out || q_head_stride < D || (T > 1 ? ldq < D : ldq < 0) || ld_out < (int64_t)n_q_heads * D)
    return IE_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(out) || ldq % 8 || q_head_stride % 8 || ld_out % 8) return IE_ERR_ALIGNMENT;
  if ((int64_t)max_q * group > INT_MAX - kRowsChunk || (int64_t)T * group > INT_MAX - kRowsChunk)
    return IE_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < kWorkspace) return IE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return IE_ERR_ALIGNMENT;

  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return IE_ERR_LAUNCH;
  Args a = {};
  a.polled = limit_is_short[dev].load(std::memory_order_relaxed);
  a.b = {q_start, kv_len, page_table, ld_table, B, T, max_pages};
  a.l = paged_layout(cache);
  a.q = q; a.ldq = ldq; a.hsq = q_head_stride;
  a.out = out; a.ld_out = ld_out;
  a.group = group; a.max_q = max_q; a.window = window; a.sinks = sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.swap_rc = cache->row_stride > cache->head_stride && cache->n_kv_heads > 1;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.splits = reinterpret_cast<Split*>(ws + kOffSplits);
  a.part_ml = reinterpret_cast<float2*>(ws + kOffMl);
  a.part_o = reinterpret_cast<float*>(ws + kOffO);
  a.split_cap = kCapSplits;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);

  // most tiles a batch of these extents can have
  auto tiles = [&](int rows) {
    const int64_t by_seq = (int64_t)B * (((int64_t)max_q * group + rows - 1) / rows);
    const int64_t by_rows = (int64_t)T * group / rows + B;
    return cache->n_kv_heads * (by_seq < by_rows ? by_seq : by_rows);
  };
  // Up to 16 rows a sequence and head the few-rows kernel; 17 to 32, which it
  // takes as two tiles, only for fewer than 32 sequences: with 20 rows it needs
  // 12 us where the chunk kernel needs 16 (8 sequences of 300 cached rows) and 28
  // where that needs 31 (8 of 2000), both need 61 (32 of 2048), and then it needs
  // 76 against 69 (64 of 1000) and 369 against 351 (128 of 4000).
  const bool few = (int64_t)max_q * group <= (B < 32 ? 2 * kRowsFew : kRowsFew);
  const int keys = few ? kKB : 64, box = a.l.page_size < keys ? a.l.page_size : keys;
  if (!make_map(&a.tmK, dt, cache->k, D, a.l, box, a.swap_rc) ||
      !make_map(&a.tmV, dt, cache->v, D, a.l, box, a.swap_rc))
    return IE_ERR_UNSUPPORTED;
  if (!few) {
    a.n_split = reinterpret_cast<int*>(ws + kOffCount);
    a.wave = kSMs;
    a.whole = 4;
    a.cut = 6;
    a.join = 6;
    a.queue = reinterpret_cast<int*>(ws + kOffQueue);
    a.max_pieces = INT_MAX;
    a.group_magic = 65536 / group + 1;
    a.lane_rows = kRowsChunk / 2 / group * group;
    a.tile_rows = 2 * a.lane_rows;
    a.target = kTargetChunk;
    a.min_blocks = 4;
    a.slot_cap = 2 * kTargetChunk;
    if (!make_q_map(&a.tmQ, dt, q, D, T, n_q_heads, ldq, q_head_stride, group, kRowsChunk / 2 / group))
      return IE_ERR_UNSUPPORTED;
    return launch_chunks(dt, D, a, tiles(a.tile_rows), st);
  }
  a.arrived = reinterpret_cast<int*>(ws);
  a.tile_rows = kRowsFew;
  a.target = kTargetFew;
  a.wave = 2 * kSMs;
  a.whole = 5;
  a.cut = 20;
  a.min_blocks = 4;
  a.slot_cap = 2 * kTargetFew;
  const int64_t grid = tiles(kRowsFew) + (B <= 32 ? a.wave : a.target);
  if (grid > INT_MAX) return IE_ERR_UNSUPPORTED;
  a.max_pieces = (int)grid;
  if (dt == IE_DTYPE_F16)
    s = D == 128 ? launch_few<__half, 128, false>(a, grid, st) : launch_few<__half, 64, false>(a, grid, st);
  else
    s = D == 128 ? launch_few<__nv_bfloat16, 128, false>(a, grid, st)
                 : launch_few<__nv_bfloat16, 64, false>(a, grid, st);
  return s;
}
