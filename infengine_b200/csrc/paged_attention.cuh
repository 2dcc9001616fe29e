// Shared by the two paged-attention kernels (paged_attention.cu: few rows,
// paged_attention_tc.cu: chunks): the arguments, the division of the work and
// the partial results in the workspace.
//
// Work. A tile is up to tile_rows rows of one sequence and KV head, a row one
// (token, query head of the group) pair in that order, so that rows which
// share a cache row share its load. The keys some row of the tile sees are covered by
// blocks of KB keys (aligned; sink rows first). A tile with many blocks is cut
// into S pieces of at most C blocks each, where C is chosen from the whole
// batch so that the pieces fill the GPU; the pieces' unnormalised outputs,
// maxima and sums meet in the workspace and are joined in piece order (by the
// tile's last CTA or by a second kernel). All of it is computed on the device from the lengths, so a
// captured graph follows them.
//
// Probabilities p = 2^(x - m) meet the values in the storage type. fp16 has no
// normal number below 2^-14 and none at all below 2^-25, so with the maximum at
// 1 a long tail of small p vanished: 131070 keys 17.5 nats below one of value 0
// gave 0 for 0.0033. Its range above 1 is free: both kernels hold p of fp16 as
// p 2^k, k such that the largest is 2^15 (65504 is the type's), in the product
// and in the sum, where it cancels; half a subnormal step is then 2^-32 of the
// largest p or less. bf16 has the range of fp32 and needs none (k = 0).
#pragma once
#include <cuda.h>
#include "paged.cuh"

namespace ie {
namespace pa {

constexpr float kLargestLog2F16 = 15.0f;  // of a p in fp16

struct Split {     // one tile that was cut, for the joining kernel
  int slot0, pieces, token0, rows, head0, row0, pad0, pad1;
};

struct Args {
  CUtensorMap tmK, tmV;  // (dim, row, head, page), or head before row where rows lie further apart
  CUtensorMap tmQ;       // (dim, head, token); chunk kernel
  PagedBatch b;
  PagedLayout l;
  const void* q;
  int64_t ldq, hsq;
  void* out;
  int64_t ld_out;
  int group, max_q, window, sinks, swap_rc;
  int tile_rows;  // rows of a tile
  int lane_rows;  // chunk kernel: rows of its lane, whole tokens (a tile is two lanes)
  int group_magic;  // r / group = r * group_magic >> 16 for r < 512
  float scale_log2;
  int target;     // pieces to aim at in a batch of more than 32 sequences
  int wave;       // CTAs that run at once
  int max_pieces; // few rows: CTAs of the launch (a CTA without a piece costs its start)
  int whole, cut; // start and end of a piece, in blocks
  int join;       // chunks: the joining kernel's time, in blocks
  int min_blocks; // smallest piece
  int slot_cap, split_cap;
  bool polled;    // the waits' limit is short: the kernels that look at their barriers without suspending
  int* arrived;   // few rows: pieces done of each cut tile, 0 between calls
  int* queue;     // chunks: pieces handed out behind the first of each CTA, 0 between calls
  int* n_split;   // chunks: number of cut tiles, and what the joining kernel needs of each
  Split* splits;
  float2* part_ml;  // [slot][row] (maximum in log2 units, sum)
  float* part_o;    // few rows: [slot][16][D]; chunks: [slot][8 warps][D / 4][32 rows][4]
};

constexpr int kSMs = 148;  // what the work is cut for; more or fewer serve it too

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT<T>::id == IE_DTYPE_BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// One sequence's extents after clamping to what the call was given.
struct Seq {
  int start, tokens, kv, pos0;  // first row of q, rows served, cache rows, position of the first row
  bool bad;
};
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.start = a.b.q_start[b];
  const int64_t n = (int64_t)a.b.q_start[b + 1] - s.start;
  const int kv = a.b.kv_len[b];
  const int64_t cap = (int64_t)a.b.max_pages << a.l.page_log2;
  s.bad = n < 0 || n > a.max_q || kv < 0 || kv > cap || s.start < 0 || (n > 0 && s.start + n > a.b.T);
  s.kv = kv < 0 ? 0 : kv > cap ? (int)cap : kv;
  int64_t serve = n < a.max_q ? n : a.max_q;
  if (s.start < 0 || s.start >= a.b.T) serve = 0;
  else if (s.start + serve > a.b.T) serve = a.b.T - s.start;
  s.tokens = serve < 0 ? 0 : (int)serve;
  const int64_t p = (int64_t)s.kv - (n < 0 ? 0 : n);
  s.pos0 = (int)(p < -INT_MAX ? -INT_MAX : p);
  return s;
}
__device__ __forceinline__ int tile_count(const Args& a, const Seq& s) {
  return (s.tokens * a.group + a.tile_rows - 1) / a.tile_rows;  // the host checked the range
}
// Most blocks any tile of the sequence can have.
template <int KB>
__device__ __forceinline__ int most_blocks(const Args& a, const Seq& s) {
  const int all = s.kv / KB + (s.kv % KB != 0);
  if (!a.window) return all;
  const int span = min(s.tokens, a.tile_rows / a.group + 2);  // tokens of a tile
  const int64_t w = ((int64_t)a.window + span) / KB + 2 + ((int64_t)a.sinks + KB - 1) / KB;
  return (int)(w < all ? w : all);
}

// The keys of one tile: [lo, hi) and the sinks [0, sink_end), in blocks
// 0 .. n_sink - 1 and first .. first + n_main - 1.
struct Keys {
  int lo, hi, sink_end, first, n_sink, n_main;
  __device__ __forceinline__ int blocks() const { return n_sink + n_main; }
  __device__ __forceinline__ int block(int j) const { return j < n_sink ? j : first + j - n_sink; }
};
template <int KB>
__device__ __forceinline__ Keys tile_keys(const Args& a, const Seq& s, int tok0, int tok1) {  // tokens tok0 .. tok1
  Keys k;
  const int64_t hi = (int64_t)s.pos0 + tok1 + 1;
  k.hi = (int)(hi < 0 ? 0 : hi < s.kv ? hi : s.kv);
  k.lo = 0;
  if (a.window) {
    const int64_t lo = (int64_t)s.pos0 + tok0 - a.window + 1;
    k.lo = (int)(lo < 0 ? 0 : lo < k.hi ? lo : k.hi);
  }
  k.sink_end = min(a.sinks, k.lo);
  k.first = k.lo / KB;
  k.n_main = k.hi > k.lo ? (k.hi + KB - 1) / KB - k.first : 0;
  k.n_sink = min((k.sink_end + KB - 1) / KB, k.first);
  if (k.n_main == 0) k.n_sink = 0;
  return k;
}

// Blocks of piece p of P: first and number.
__device__ __forceinline__ void piece_range(int blocks, int P, int p, int& first, int& n) {
  const int each = P > 1 ? blocks / P : blocks, more = blocks - each * P;
  first = p * each + min(p, more);
  n = each + (p < more);
}

struct Piece {
  int b, head, tile, pieces, piece, slot, split;  // slot, split < 0: the tile is whole
};

// Scratch of find_piece.
struct Scan {
  long long w[3][32];
  Piece p;
  Seq seq;
  int found;
};

// Sum over the block / exclusive scan of three counts over the block.
template <int THREADS>
__device__ __forceinline__ void block_scan3(long long (&v)[3], long long (&total)[3], Scan& sc) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x[3] = {v[0], v[1], v[2]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const long long u = __shfl_up_sync(0xffffffffu, x[j], o);
      if (lane >= o) x[j] += u;
    }
  if (lane == 31)
#pragma unroll
    for (int j = 0; j < 3; ++j) sc.w[j][warp] = x[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    long long before = 0;
    total[j] = 0;
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += sc.w[j][i];
      total[j] += sc.w[j][i];
    }
    v[j] = before + x[j] - v[j];
  }
  __syncthreads();
}

// Blocks of a piece, for u blocks in the batch (each tile counted at its
// sequence's most).
__device__ __forceinline__ int piece_blocks(const Args& a, long long u) {
  long long c = u <= INT_MAX ? ((int)u - 1) / a.target + 1 : (u - 1) / a.target + 1;
  if (c < a.min_blocks) c = a.min_blocks;
  return c > INT_MAX / 2 ? INT_MAX / 2 : (int)c;
}

// Piece `at` of a sequence of `tiles` tiles in S pieces each: the last
// (longest) tiles first, the heads of a piece next to one another.
__device__ __forceinline__ Piece piece_at(const Args& a, int b, int tiles, int S, int at, int slots, int splits) {
  const int nkv = a.l.n_kv_heads, r = at / nkv;
  Piece p;
  p.b = b;
  p.head = at - r * nkv;
  p.tile = tiles - 1 - (S > 1 ? r / S : r);
  p.pieces = S;
  p.piece = S > 1 ? r % S : 0;
  p.slot = S > 1 ? slots + (p.tile * S + p.piece) * nkv + p.head : -1;
  p.split = S > 1 ? splits + p.tile * nkv + p.head : -1;
  return p;
}

// Pieces of a tile of n blocks, about C = 1 / per each. (No integer division: a
// wave of CTAs counts them for 32 sequences and 32 lengths before it starts.)
__device__ __forceinline__ int pieces_of(int n, int C, float per) {
  return n > C ? (int)((float)(n - 1) * per) + 1 : 1;
}

// Blocks of a piece where whole waves of a.wave CTAs count: lane k - 1 weighs
// cutting the longest tile into k pieces of C = most / k blocks. With P pieces
// of A blocks on average, W = ceil(P / wave) waves cost W (A + o) + C - A
// blocks, o the start and end of a piece in blocks (a.whole; a.cut with the
// partial results' way through memory). tiles_heads, most: sequence `lane`'s.
__device__ __forceinline__ int piece_blocks_by_waves(const Args& a, int tiles_heads, int most) {
  const int lane = threadIdx.x & 31;
  const int longest = __reduce_max_sync(0xffffffffu, most), all = __reduce_add_sync(0xffffffffu, tiles_heads);
  // (the last lanes: as many pieces as just fill one wave, and two)
  const int k = lane < 30 ? lane + 1 : max((lane - 29) * a.wave / max(all, 1), 1);
  const int C = max((longest - 1) / k + 1, 1);
  const float per = 1.0f / (float)C;
  float pieces = 0.f, cut = 0.f, blocks = 0.f;
#pragma unroll 4
  for (int b = 0; b < a.b.B; ++b) {
    const int t = __shfl_sync(0xffffffffu, tiles_heads, b), n = __shfl_sync(0xffffffffu, most, b);
    const float p = (float)t * (float)pieces_of(n, C, per);
    pieces += p;
    cut += n > C ? p : 0.f;
    blocks += (float)t * (float)n;
  }
  const float avg = pieces > 0.f ? blocks / pieces : 0.f;
  const float waves = ceilf(pieces / (float)a.wave);
  float cost = waves * (avg + (cut > 0.f ? a.cut : a.whole)) + (float)C - avg;
  if (cut > (float)a.slot_cap || pieces > (float)a.max_pieces || (k > 1 && C < a.min_blocks)) cost = INFINITY;
  float least = cost;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  const int who = __ffs(__ballot_sync(0xffffffffu, cost == least)) - 1;
  return __shfl_sync(0xffffffffu, C, max(who, 0));
}

// The same for pieces that a.wave CTAs take from a queue, sequences in
// descending order of their most blocks. A sequence's last piece ends at about
// the work up to there divided by the CTAs, and half a piece (the first one's
// pieces: in whole waves); the joining kernel adds a.join blocks and 1 / 25 a
// partial result.
__device__ __forceinline__ int piece_blocks_by_ends(const Args& a, int tiles_heads, int most) {
  const int lane = threadIdx.x & 31;
  const int longest = __shfl_sync(0xffffffffu, most, 0), all = __reduce_add_sync(0xffffffffu, tiles_heads);
  const int k = lane < 30 ? lane + 1 : max((lane - 29) * a.wave / max(all, 1), 1);
  const int C = max((longest - 1) / k + 1, 1);
  const float per = 1.0f / (float)C, each = 1.0f / (float)a.wave;
  float slots = 0.f, work = 0.f, cost = 0.f;
#pragma unroll 4
  for (int b = 0; b < a.b.B; ++b) {
    const int t = __shfl_sync(0xffffffffu, tiles_heads, b), n = __shfl_sync(0xffffffffu, most, b);
    const int S = pieces_of(n, C, per);
    const float pieces = (float)t * (float)S;
    const float size = __fdividef((float)n, (float)S) + (float)(n > C ? a.cut : a.whole);
    slots += n > C ? pieces : 0.f;
    work += pieces * size;
    const float end = b == 0 ? ceilf(pieces * each) * size : work * each + 0.5f * size;
    cost = t ? fmaxf(cost, end) : cost;
  }
  if (slots > 0.f) cost += (float)a.join + 0.04f * slots;
  if (slots > (float)a.slot_cap || (k > 1 && C < a.min_blocks)) cost = INFINITY;
  float least = cost;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  const int who = __ffs(__ballot_sync(0xffffffffu, cost == least)) - 1;
  return __shfl_sync(0xffffffffu, C, max(who, 0));
}

// Finds pieces for one warp, in increasing order of their index: sequences are
// taken 32 at a time, one a lane. Up to 32 sequences are read once, come in
// descending order of their most blocks, and the pieces' length is chosen by
// where the pieces end; more are read twice, come in the batch's order, and a
// piece has an even share of the batch's blocks (a chunk of 512 tokens over 3000
// rows beside 63 single tokens takes 213 to 217 us wherever it stands; one over
// 30000 rows 464 first and 483 last).
template <int KB>
struct Finder {
  const Args& a;
  int C, total, splits;  // blocks of a piece; pieces and cut tiles of the batch
  int b0;                // first sequence of the held ones
  Seq s;
  int tiles, S, mine, x, y, z;  // this lane's; x, y, z inclusive sums of pieces, slots, cut tiles
  int rx, ry, rz;               // of the sequences before b0
  int seq;                      // this lane's sequence

  __device__ __forceinline__ explicit Finder(const Args& args, int* status) : a(args) {
    const bool tell = blockIdx.x == 0;
    if (a.b.B <= 32) {
      read(0, tell, status);
      if (a.b.B > 1) longest_first();
      C = piece_blocks_by_ends(a, tiles * a.l.n_kv_heads, most);
    } else {
      long long u = 0;
      for (int b = 0; b < a.b.B; b += 32) {
        read(b, tell, status);
        u += (long long)tiles * a.l.n_kv_heads * most;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      C = piece_blocks(a, u);
    }
    // the batch's totals: pieces here, cut tiles for the one CTA that reports them
    rx = ry = rz = 0;
    if (a.b.B <= 32) {
      scan();
    } else {
      for (int b = 0; b < a.b.B; b += 32) {
        read(b, false, status);
        scan();
        if (b + 32 < a.b.B) skip();
      }
    }
    total = rx + __shfl_sync(0xffffffffu, x, 31);
    splits = rz + __shfl_sync(0xffffffffu, z, 31);
    if (a.b.B > 32) {
      rx = ry = rz = 0;
      read(0, false, status);
      scan();
    }
  }
  // Piece `index` (at least the last one asked for); true in the lane that has it.
  __device__ __forceinline__ bool find(int index, Piece& p, int* status) {
    while (index >= rx + __shfl_sync(0xffffffffu, x, 31) && b0 + 32 < a.b.B) {
      skip();
      read(b0 + 32, false, status);
      scan();
    }
    const int at = index - rx - (x - mine);
    if (at < 0 || at >= mine) return false;
    const int nkv = a.l.n_kv_heads;
    p = piece_at(a, seq, tiles, S, at, ry + y - (S > 1 ? mine : 0),
                 rz + z - (S > 1 ? tiles * nkv : 0));
    return true;
  }

 private:
  int most;
  __device__ __forceinline__ void read(int first, bool tell, int* status) {
    b0 = first;
    s = {};
    tiles = most = 0;
    const int b = first + (threadIdx.x & 31);
    seq = b;
    if (b < a.b.B) {
      s = sequence(a, b);
      tiles = tile_count(a, s);
      most = tiles ? most_blocks<KB>(a, s) : 0;
      if (s.bad && tell) atomicExch(status, IE_ERR_INVALID_ARG);
    }
  }
  // Sequences in descending order of their most blocks, so that the last pieces
  // handed out are short.
  __device__ __forceinline__ void longest_first() {
    const int lane = threadIdx.x & 31;
    int rank = 0, from = 0;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
      const int n = __shfl_sync(0xffffffffu, most, i);
      rank += n > most || (n == most && i < lane);
    }
#pragma unroll 8
    for (int i = 0; i < 32; ++i)
      if (__shfl_sync(0xffffffffu, rank, i) == lane) from = i;
    s.start = __shfl_sync(0xffffffffu, s.start, from);
    s.tokens = __shfl_sync(0xffffffffu, s.tokens, from);
    s.kv = __shfl_sync(0xffffffffu, s.kv, from);
    s.pos0 = __shfl_sync(0xffffffffu, s.pos0, from);
    tiles = __shfl_sync(0xffffffffu, tiles, from);
    most = __shfl_sync(0xffffffffu, most, from);
    seq = from;
  }
  __device__ __forceinline__ void scan() {
    const int lane = threadIdx.x & 31, nkv = a.l.n_kv_heads;
    S = pieces_of(most, C, 1.0f / (float)C);
    // a count past the range cannot be asked for: the host bounds the pieces
    mine = (int)min((long long)tiles * S * nkv, 1LL << 25);
    x = mine;
    y = S > 1 ? mine : 0;
    z = S > 1 ? tiles * nkv : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ux = __shfl_up_sync(0xffffffffu, x, o), uy = __shfl_up_sync(0xffffffffu, y, o),
                uz = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) {
        x += ux;
        y += uy;
        z += uz;
      }
    }
  }
  __device__ __forceinline__ void skip() {
    rx += __shfl_sync(0xffffffffu, x, 31);
    ry += __shfl_sync(0xffffffffu, y, 31);
    rz += __shfl_sync(0xffffffffu, z, 31);
  }
};

// The piece a CTA serves and its sequence, in sc; false when there are fewer
// pieces. Called by the whole block (few-rows kernel).
template <int KB, int THREADS>
__device__ __forceinline__ bool find_piece(const Args& a, int index, Scan& sc, int* status) {
  const int tid = threadIdx.x, nkv = a.l.n_kv_heads;
  if (a.b.B <= 32) {
    // one warp, one sequence a lane, one round trip to the lengths
    if (tid < 32) {
      Seq s = {};
      int tiles = 0, most = 0;
      if (tid < a.b.B) {
        s = sequence(a, tid);
        tiles = tile_count(a, s);
        most = tiles ? most_blocks<KB>(a, s) : 0;
        if (s.bad && index == 0) atomicExch(status, IE_ERR_INVALID_ARG);
      }
      const int C = piece_blocks_by_waves(a, tiles * nkv, most);
      const int S = pieces_of(most, C, 1.0f / (float)C);
      // a count past the grid's range cannot be asked for: the host bounds the pieces
      const int mine = (int)min((long long)tiles * S * nkv, 1LL << 25);
      int x = mine, y = S > 1 ? mine : 0, z = S > 1 ? tiles * nkv : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int ux = __shfl_up_sync(0xffffffffu, x, o), uy = __shfl_up_sync(0xffffffffu, y, o),
                  uz = __shfl_up_sync(0xffffffffu, z, o);
        if (tid >= o) {
          x += ux;
          y += uy;
          z += uz;
        }
      }
      const bool hit = index >= x - mine && index < x;
      if (hit) {
        sc.p = piece_at(a, tid, tiles, S, index - (x - mine), y - (S > 1 ? mine : 0), z - (S > 1 ? tiles * nkv : 0));
        sc.seq = s;
      }
      const unsigned any = __ballot_sync(0xffffffffu, hit);
      if (tid == 0) sc.found = any != 0;
    }
    __syncthreads();
    return sc.found != 0;
  }
  long long u[3] = {0, 0, 0}, sums[3];  // blocks, tiles
  for (int b = tid; b < a.b.B; b += THREADS) {
    const Seq s = sequence(a, b);
    const long long t = (long long)tile_count(a, s) * nkv;
    u[0] += t * most_blocks<KB>(a, s);
    u[1] += t;
    if (s.bad && index == 0) atomicExch(status, IE_ERR_INVALID_ARG);
  }
  if (tid == 0) sc.found = 0;
  block_scan3<THREADS>(u, sums, sc);
  // lengths that contradict T could ask for more pieces than were launched:
  // then no tile is cut, since a cut one needs all of its pieces
  const int C = sums[1] + a.target > a.max_pieces ? INT_MAX / 2 : piece_blocks(a, sums[0]);
  long long run[3] = {0, 0, 0};  // pieces, slots, cut tiles so far
  for (int b0 = 0; b0 < a.b.B; b0 += THREADS) {
    const int b = b0 + tid;
    long long v[3] = {0, 0, 0}, total[3];
    int tiles = 0, S = 1;
    Seq s = {};
    if (b < a.b.B) {
      s = sequence(a, b);
      const int most = most_blocks<KB>(a, s);
      tiles = tile_count(a, s);
      S = pieces_of(most, C, 1.0f / (float)C);
      v[0] = (long long)tiles * S * nkv;
      v[1] = S > 1 ? v[0] : 0;
      v[2] = S > 1 ? (long long)tiles * nkv : 0;
    }
    const long long mine = v[0];
    block_scan3<THREADS>(v, total, sc);
    const long long at = index - (run[0] + v[0]);
    if (at >= 0 && at < mine) {
      sc.p = piece_at(a, b, tiles, S, (int)at, (int)(run[1] + v[1]), (int)(run[2] + v[2]));
      sc.seq = s;
      sc.found = 1;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) run[j] += total[j];
    if (run[0] > index) break;
  }
  __syncthreads();
  return sc.found != 0;
}

// Chunks of tokens on tcgen05 (paged_attention_tc.cu), with the joining of
// their pieces. most_tiles: an upper bound of the batch's tiles.
int launch_chunks(ie_dtype dt, int D, Args& a, int64_t most_tiles, cudaStream_t st);

constexpr int kRowsFew = 16;         // tile_rows of the few-rows kernel
constexpr int kTargetFew = kSMs * 4;  // its pieces
constexpr int kRowsChunk = 256;      // tile_rows of the chunk kernel, at most
constexpr int kTargetChunk = kSMs;

}  // namespace pa
}  // namespace ie
