// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// A row's tokens in descending order of their logits (equal logits: lowest id
// first), w = exp((x - max) / T):
//   top-k  keeps the first k;
//   top-p  keeps those whose mass before them is below p * (mass of the top k);
//   min-p  keeps those with w >= min_p;
// each cut keeps a prefix of the order, so the kept set is its first L tokens
// (L >= 1), Z their mass, and the sample is the first whose running mass
// exceeds u * Z.
//
// The result turns on which side of a border a running mass falls, so masses
// are 64-bit. Sorting is not needed: a 16-bit logit has one of 65536 values,
// so counting the row's tokens by value gives the whole order, exactly and
// whatever the order of the counting atomics; exp is evaluated once for each
// value that occurs (a few thousand) instead of once a token, and the mass of
// a value is count * w. A token is found from its rank by a last pass over
// the logits that looks for the n-th occurrence of its value.
//
// What bounds it: the row is read twice (the second time from L2) and counted
// with one shared-memory atomic a token (about 7 cycles a warp of them); the
// rest is latency. One cluster of N CTAs serves a row: each counts its N-th of
// the row into its own 65536 16-bit counters (128 KB of shared memory; a slice
// is kept to 65535 tokens so that none overflows), then sums the N counts of its
// N-th of the values and their masses, 32 values to a group. Rank 0 gathers and
// scans the 2048 groups, its first warp makes the cuts by searching the scanned
// groups and then one group's 32 values, and the CTA whose slice holds the
// token looks for it.
#include <atomic>
#include <cooperative_groups.h>
#include "ie_common.cuh"

namespace ie {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kKeys = 65536;
constexpr int kGroups = kKeys / 32;                // 2 a thread
constexpr int kMaxSlice = 65535;
constexpr int kHistBytes = kKeys * 2;
// shared memory: counters | group masses | group counts
constexpr int kOffMass = kHistBytes;
constexpr int kOffCount = kOffMass + kGroups * 8;
constexpr int kSmem = kOffCount + kGroups * 4;
static_assert(kSmem <= 227 * 1024 - 2048, "shared memory per CTA");

struct SampleArgs {
  const void* logits;
  int64_t ld;
  int V;
  const float *temperature, *top_p, *min_p, *u;
  const int* top_k;
  int* idx;
  float* logprob;
};

// Position of a value in the descending order of the 65536 16-bit values, -1
// for what is never sampled (NaN, -infinity). -0 counts as +0.
template <typename T>
__device__ __forceinline__ int key_of(unsigned b) {
  constexpr unsigned kInf = DT<T>::id == IE_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  if ((b & 0x7FFFu) > kInf || b == (0x8000u | kInf)) return -1;
  if (b == 0x8000u) b = 0u;
  const unsigned up = (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
  return (int)(0xFFFFu - up);
}
__device__ __forceinline__ unsigned bits_of(int key) {
  const unsigned up = 0xFFFFu - (unsigned)key;
  return (up & 0x8000u) ? (up & 0x7FFFu) : (~up & 0xFFFFu);
}
template <typename T>
__device__ __forceinline__ double value_of(int key) {
  const unsigned short b = (unsigned short)bits_of(key);
  T v;
  memcpy(&v, &b, 2);
  return (double)DT<T>::to_f(v);
}

// Distance from a value of this 16-bit pattern to its neighbours (the 8 aligned
// values around it are equally spaced).
template <typename T>
__device__ __forceinline__ double spacing_of(int key) {
  const unsigned up = 0xFFFFu - (unsigned)key, b = (up & 0x8000u) ? up & 0x7FFFu : ~up & 0x7FFFu;
  constexpr int kMant = DT<T>::id == IE_DTYPE_BF16 ? 7 : 10, kBias = DT<T>::id == IE_DTYPE_BF16 ? 127 : 15;
  const int e = max((int)(b >> kMant), 1) - kBias - kMant;
  return __hiloint2double((1023 + e) << 20, 0);
}

// K of the 16-byte chunks c, c + step .. (0xFFFF, a NaN in both types, from
// `end` on), all loads in flight at once.
template <int K>
__device__ __forceinline__ void load_chunks(const uint4* p, int c, int step, int end, uint4 (&x)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i)
    x[i] = c + i * step < end ? __ldg(p + c + i * step)
                              : make_uint4(0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu);
}

// 2^x for x <= 0 in 64 bits: the nearest integer and a polynomial of degree 10
// for the rest, fitted for the least relative error on [-1/2, 1/2] (2.8e-16 with
// the coefficients as stored, before the roundings of its evaluation). About a
// third of the library exponential's instructions, and the 64-bit pipe is what
// masses wait for.
__device__ __forceinline__ double exp2_neg(double x) {
  if (!(x > -1000.0)) return 0.0;
  const double big = 6755399441055744.0;  // 1.5 * 2^52
  const double r = x + big;
  const double f = x - (r - big);
  double p = 7.037279530582804e-09;
  p = fma(p, f, 1.0208537904552164e-07);
  p = fma(p, f, 1.3215662831846104e-06);
  p = fma(p, f, 1.5252658116561384e-05);
  p = fma(p, f, 1.5403529961135955e-04);
  p = fma(p, f, 1.3333558228561476e-03);
  p = fma(p, f, 9.61812910803459e-03);
  p = fma(p, f, 5.550410866445883e-02);
  p = fma(p, f, 2.4022650695908768e-01);
  p = fma(p, f, 6.931471805599497e-01);
  p = fma(p, f, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(r) << 20), __double2loint(p));
}

// What rank 0 tells the others: the value and which of a slice's tokens of it.
struct Pick {
  int key, slice, rank;
  int greedy;
  double share;
};

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned* hist = reinterpret_cast<unsigned*>(smem);  // two counters a word
  double* mass = reinterpret_cast<double*>(smem + kOffMass);
  int* count = reinterpret_cast<int*>(smem + kOffCount);
  __shared__ int best_key;   // this CTA's smallest key (largest logit)
  __shared__ int above_min;  // its tokens with w >= min_p
  __shared__ double wsum[kWarps];
  __shared__ int csum[kWarps];
  __shared__ int hits[8][kWarps];
  __shared__ Pick pick;

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = N == 1 ? 0 : (int)cluster.block_rank();
  const int row = blockIdx.x / N, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  // (also for a cluster of one: with __syncthreads in its place the one-warp
  // part ran four times slower)
  auto sync_row = [&] { cluster.sync(); };
  auto peer = [&](auto* p, int r) {
    if constexpr (N == 1) return p;
    else return cluster.map_shared_rank(p, r);
  };

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const unsigned short* base = static_cast<const unsigned short*>(a.logits) + (int64_t)row * a.ld;
  // The row as up to 7 tokens before the first 16-byte boundary (slice 0's),
  // chunks of 8, of which this slice has c0 .. c1 - 1, and up to 7 tokens
  // behind them (the last slice's).
  const int head = min((int)((0u - (unsigned)reinterpret_cast<uintptr_t>(base)) & 15u) >> 1, a.V);
  const int chunks = (a.V - head) >> 3, tail0 = head + 8 * chunks;
  const uint4* body = reinterpret_cast<const uint4*>(base + head);
  const int c0 = (int)((int64_t)chunks * rank / N), c1 = (int)((int64_t)chunks * (rank + 1) / N);
  // the first chunks are on their way while the counters are cleared
  constexpr int kAhead = 2;
  uint4 x[kAhead];
  load_chunks(body, c0 + t, kThreads, c1, x);
  for (int i = t; i < kHistBytes / 16; i += kThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (t == 0) {
    best_key = kKeys;
    above_min = 0;
  }
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const bool greedy = !(temp > 0.f);
  const double per = 1.4426950408889634 / (greedy ? 1.0 : (double)temp);  // log2 e / T
  const double low = a.min_p ? (double)a.min_p[row] : 0.0;
  __syncthreads();

  // ---- count this slice's tokens by value
  int best = kKeys;
  auto take = [&](unsigned bits) {
    const int key = key_of<T>(bits);
    if (key >= 0) {
      best = min(best, key);
      atomicAdd(hist + (key >> 1), 1u << (16 * (key & 1)));
    }
  };
  if (rank == 0 && t < head) take(__ldg(base + t));
  if (rank == N - 1 && t < a.V - tail0) take(__ldg(base + tail0 + t));
  for (int c = c0 + t; c < c1;) {
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const unsigned w[4] = {x[y].x, x[y].y, x[y].z, x[y].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) take((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
    }
    c += kAhead * kThreads;
    load_chunks(body, c, kThreads, c1, x);
  }
  best = __reduce_min_sync(0xffffffffu, best);
  if (lane == 0) atomicMin(&best_key, best);
  sync_row();
#pragma unroll
  for (int r = 0; r < N; ++r) best = min(best, *peer(&best_key, r));
  const double top = best < kKeys ? value_of<T>(best) : 0.0;
  // weight of a value that occurs; an infinite largest logit takes it all
  auto weight = [&](int key) -> double {
    if (key == best) return 1.0;
    const double d = value_of<T>(key) - top;
    return d < -1e300 ? 0.0 : exp2_neg(d * per);
  };

  // ---- counts and masses of this CTA's N-th of the values: 8 a thread and
  // step, 4 threads a group
  constexpr int kMine = kKeys / N;
  int above = 0;
#pragma unroll 1
  for (int i = 0; i < kMine / (8 * kThreads); ++i) {
    const int key = rank * kMine + 8 * (i * kThreads + t);
    uint4 x[N];
#pragma unroll
    for (int r = 0; r < N; ++r) x[r] = *reinterpret_cast<const uint4*>(peer(hist, r) + (key >> 1));
    int n[8] = {};
    int cnt = 0;
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const unsigned w[4] = {x[r].x, x[r].y, x[r].z, x[r].w};
#pragma unroll
      for (int y = 0; y < 8; ++y) n[y] += (w[y >> 1] >> (16 * (y & 1))) & 0xFFFF;
    }
#pragma unroll
    for (int y = 0; y < 8; ++y) cnt += n[y];
    double m = 0.0;
    if (__any_sync(0xffffffffu, cnt != 0)) {
      if (cnt) {
        // equally spaced values: each weight is the last one times r
        const double r = exp2_neg(-spacing_of<T>(key) * per);
        double w = best >= key && best < key + 8 ? 0.0 : weight(key);
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          if (key + y == best) w = 1.0;
          // n as a double: its bits below 2^52, without the slow conversion
          const double dn = __hiloint2double(0x43300000, n[y]) - 4503599627370496.0;
          m += n[y] ? dn * w : 0.0;
          if (low > 0.0) above += n[y] && w >= low ? n[y] : 0;
          w *= r;
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        m += __shfl_xor_sync(0xffffffffu, m, o);
        cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
      }
    }
    if ((lane & 3) == 0) {
      mass[key >> 5] = m;
      count[key >> 5] = cnt;
    }
  }
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0 && above) atomicAdd(&above_min, above);
  sync_row();

  if (rank == 0) {
    // ---- scan the groups, thread t groups 2t and 2t + 1: mass[g] and count[g]
    // become what lies before group g
    double m0, m1;
    int n0, n1;
    {
      const int r = (2 * t) / (kGroups / N);
      const double2 pm = *reinterpret_cast<const double2*>(peer(mass, r) + 2 * t);
      const int2 pn = *reinterpret_cast<const int2*>(peer(count, r) + 2 * t);
      m0 = pm.x; m1 = pm.y;
      n0 = pn.x; n1 = pn.y;
    }
    double sm = m0 + m1;
    int sn = n0 + n1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double um = __shfl_up_sync(0xffffffffu, sm, o);
      const int un = __shfl_up_sync(0xffffffffu, sn, o);
      if (lane >= o) { sm += um; sn += un; }
    }
    if (lane == 31) { wsum[warp] = sm; csum[warp] = sn; }
    __syncthreads();
    // every warp scans the 32 warps' sums
    double bm = wsum[lane];
    int bn = csum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double um = __shfl_up_sync(0xffffffffu, bm, o);
      const int un = __shfl_up_sync(0xffffffffu, bn, o);
      if (lane >= o) { bm += um; bn += un; }
    }
    const double all_m = __shfl_sync(0xffffffffu, bm, 31);
    const int all_n = __shfl_sync(0xffffffffu, bn, 31);
    bm = __shfl_sync(0xffffffffu, bm, max(warp - 1, 0));
    bn = __shfl_sync(0xffffffffu, bn, max(warp - 1, 0));
    if (warp == 0) { bm = 0.0; bn = 0; }
    *reinterpret_cast<double2*>(mass + 2 * t) = make_double2(bm + (sm - (m0 + m1)), bm + (sm - m1));
    *reinterpret_cast<int2*>(count + 2 * t) = make_int2(bn + sn - n0 - n1, bn + sn - n1);
    __syncthreads();

    if (warp == 0) {
      // The values of one group, one a lane: tokens, weight, what lies before.
      struct Lane {
        int key, n, before_n;
        double w, before_m;
      };
      auto tokens = [&](int key) {
        int n = 0;
#pragma unroll
        for (int r = 0; r < N; ++r) n += (peer(hist, r)[key >> 1] >> (16 * (key & 1))) & 0xFFFF;
        return n;
      };
      auto values = [&](int g) {
        Lane v;
        v.key = 32 * g + lane;
        v.n = tokens(v.key);
        v.w = v.n ? weight(v.key) : 0.0;
        double m = v.n * v.w;
        int c = v.n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double um = __shfl_up_sync(0xffffffffu, m, o);
          const int uc = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) { m += um; c += uc; }
        }
        v.before_m = mass[g] + (m - v.n * v.w);
        v.before_n = count[g] + c - v.n;
        return v;
      };
      // first group whose end passes the border; ends(g) is what lies before g
      auto group_of = [&](auto passes) {
        const int s = __ffs(__ballot_sync(0xffffffffu, passes(64 * (lane + 1)))) - 1;
        if (s < 0) return kGroups - 1;
        const unsigned odd = __ballot_sync(0xffffffffu, passes(64 * s + 2 * lane + 1));
        const unsigned even = __ballot_sync(0xffffffffu, passes(64 * s + 2 * lane + 2));
        const int f = __ffs(even) - 1;
        return 64 * s + 2 * f + ((odd >> f) & 1 ? 0 : 1);
      };
      auto count_at = [&](int g) { return g < kGroups ? count[g] : all_n; };
      auto mass_at = [&](int g) { return g < kGroups ? mass[g] : all_m; };
      // mass of the first n tokens, 1 <= n <= all_n
      auto mass_of_first = [&](int n) {
        if (n >= all_n) return all_m;
        const Lane v = values(group_of([&](int g) { return count_at(g) >= n; }));
        const int who = __ffs(__ballot_sync(0xffffffffu, v.before_n + v.n >= n)) - 1;
        return __shfl_sync(0xffffffffu, v.before_m + (double)(n - v.before_n) * v.w, max(who, 0));
      };
      Pick out = {-1, 0, 0, greedy, 0.0};
      if (all_n > 0) {
        int L = all_n;
        double Z = all_m;
        if (greedy) {
          L = 1;
          Z = 1.0;
        } else {
          const double p = a.top_p ? (double)a.top_p[row] : 1.0;
          const int k = a.top_k ? a.top_k[row] : 0;
          if (k > 0 && k < L) {
            L = k;
            Z = mass_of_first(L);
          }
          if (!(p >= 1.0)) {
            // a token is kept while the mass before it is below the border
            const double border = p * Z;
            const Lane v = values(group_of([&](int g) { return mass_at(g) >= border; }));
            const unsigned over = __ballot_sync(0xffffffffu, v.n && v.before_m + v.n * v.w >= border);
            const int who = over ? __ffs(over) - 1 : 31;  // none by a rounding: the border is the group's end
            int n = v.n;
            if (over && v.w > 0.0) {
              n = (int)ceil(fmin(fmax((border - v.before_m) / v.w, 0.0), (double)v.n));
              while (n > 0 && v.before_m + (double)(n - 1) * v.w >= border) --n;
              while (n < v.n && v.before_m + (double)n * v.w < border) ++n;
            }
            const int kept = max(__shfl_sync(0xffffffffu, v.before_n + n, who), 1);
            const double mk = __shfl_sync(0xffffffffu, v.before_m + (double)n * v.w, who);
            if (p != p) {
              L = 1;
              Z = 1.0;
            } else if (kept < L) {
              L = kept;
              Z = kept == 1 ? 1.0 : mk;
            }
          }
          int m = 0;
          if (low > 0.0 || low != low) {
#pragma unroll
            for (int r = 0; r < N; ++r) m += *peer(&above_min, r);
            if (m < 1) m = 1;
            if (m < L) {
              L = m;
              Z = mass_of_first(L);
            }
          }
        }
        const float u = a.u[row];
        const double border = greedy || u < 0.f ? 0.0 : (double)u * Z;
        Lane v = values(group_of([&](int g) { return mass_at(g) > border; }));
        const unsigned any = __ballot_sync(0xffffffffu, v.n != 0);
        const unsigned over = __ballot_sync(0xffffffffu, v.n && v.before_m + v.n * v.w > border);
        // none by a rounding: the group's last token
        int who = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
        int n = (int)fmin(fmax((border - v.before_m) / v.w, 0.0), (double)max(v.n - 1, 0));
        if (v.w > 0.0) {
          while (n > 0 && v.before_m + (double)n * v.w > border) --n;
          while (n < v.n - 1 && v.before_m + (double)(n + 1) * v.w <= border) ++n;
        }
        if (__shfl_sync(0xffffffffu, v.n == 0 || !(border < Z) || v.before_n + n >= L, who)) {
          // u * Z reached the end of the kept mass: the last kept token
          v = values(group_of([&](int g) { return count_at(g) >= L; }));
          who = __ffs(__ballot_sync(0xffffffffu, v.before_n + v.n >= L)) - 1;
          n = L - 1 - v.before_n;
        }
        out.key = __shfl_sync(0xffffffffu, v.key, who);
        out.rank = __shfl_sync(0xffffffffu, n, who);
        out.share = __shfl_sync(0xffffffffu, v.w, who) / Z;
        // the slice that holds that one of the value's tokens
#pragma unroll
        for (int r = 0; r < N - 1; ++r) {
          const int c = (peer(hist, r)[out.key >> 1] >> (16 * (out.key & 1))) & 0xFFFF;
          if (out.slice == r && out.rank >= c) {
            out.rank -= c;
            ++out.slice;
          }
        }
      }
      if (lane < N) *peer(&pick, lane) = out;
    }
  }
  sync_row();

  // ---- that token of the slice, in index order: chunks go by (step, thread)
  const Pick out = pick;
  if (out.key < 0) {
    if (rank == 0 && t == 0) {
      a.idx[row] = -1;
      if (a.logprob) a.logprob[row] = __int_as_float(0xff800000);
    }
    return;
  }
  if (rank != out.slice) return;
  // tokens of the value in a chunk: equal bits, or either zero
  const unsigned bits = bits_of(out.key), both = bits | bits << 16;
  const unsigned care = bits == 0u ? 0x7FFF7FFFu : 0xFFFFFFFFu;
  auto matches = [&](const uint4& x) -> unsigned {
    const unsigned w[4] = {(x.x ^ both) & care, (x.y ^ both) & care, (x.z ^ both) & care, (x.w ^ both) & care};
    unsigned any = 0;  // never 0 when a half word is
#pragma unroll
    for (int y = 0; y < 4; ++y) any |= (w[y] - 0x00010001u) & ~w[y];
    unsigned h = 0;
    if (any & 0x80008000u)
#pragma unroll
      for (int y = 0; y < 8; ++y)
        if (((w[y >> 1] >> (16 * (y & 1))) & 0xFFFFu) == 0u) h |= 1u << y;
    return h;
  };
  auto write = [&](int id) {
    a.idx[row] = id;
    if (a.logprob) a.logprob[row] = out.greedy ? 0.f : (float)log(out.share);
  };
  unsigned found[8];  // a slice has at most 8 kThreads chunks
  {
    uint4 y[8];
    load_chunks(body, c0 + t, kThreads, c1, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) found[i] = c0 + i * kThreads < c1 ? matches(y[i]) : 0u;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = __reduce_add_sync(0xffffffffu, __popc(found[i]));
    if (lane == 0) hits[i][warp] = n;
  }
  __syncthreads();
  if (warp == 0) {
    // lane l scans the 8 entries 8 l .. of the 256 (step, warp) counts
    int mine[8], sum = 0;
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      mine[y] = hits[lane >> 2][8 * (lane & 3) + y];
      sum += mine[y];
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    const int all = __shfl_sync(0xffffffffu, before, 31);
    before -= sum;
    // the tokens outside the chunks, one a lane: those before and those behind
    const int i0 = min(lane, a.V - 1), i1 = min(tail0 + lane, a.V - 1);
    const unsigned first =
        __ballot_sync(0xffffffffu, rank == 0 && lane < head && key_of<T>(__ldg(base + i0)) == out.key);
    const unsigned last =
        __ballot_sync(0xffffffffu, rank == N - 1 && tail0 + lane < a.V && key_of<T>(__ldg(base + i1)) == out.key);
    int left = out.rank;
    auto nth = [](unsigned m, int n) {
      for (; n > 0; --n) m &= m - 1;
      return __ffs(m) - 1;
    };
    if (lane == 0) csum[1] = -1;
    __syncwarp();
    if (left < __popc(first)) {
      if (lane == 0) write(nth(first, left));
    } else if ((left -= __popc(first)) >= all) {
      if (lane == 0) write(tail0 + nth(last, left - all));
    } else if (left >= before && left < before + sum) {
      left -= before;
      int y = 0;
#pragma unroll
      for (int z = 0; z < 7; ++z)
        if (y == z && left >= mine[z]) {
          left -= mine[z];
          y = z + 1;
        }
      csum[0] = lane >> 2;           // the step
      csum[1] = 8 * (lane & 3) + y;  // the warp
      csum[2] = left;
    }
  }
  __syncthreads();
  if (warp == csum[1]) {
    unsigned h = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i == csum[0]) h = found[i];
    const int n = __popc(h);
    int before = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    int skip = csum[2] - (before - n);
    if (skip >= 0 && skip < n) {
      for (; skip > 0; --skip) h &= h - 1;
      write(head + 8 * (c0 + csum[0] * kThreads + t) + __ffs(h) - 1);
    }
  }
}

// A launch of M rows on clusters of N CTAs.
struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  Launch(int M, int N, cudaStream_t st) {
    cfg.gridDim = dim3((unsigned)M * N);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = N;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
};

// Clusters of N CTAs that run at once on the current device (asked once), 0 on
// failure. A CTA takes an SM and a cluster lies in one GPC, so there are fewer
// than SMs / N: 15 of 8 and 33 of 4 on a B200 of 148 SMs, where that would be
// 18 and 37.
template <typename T, int N>
int at_once() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  static std::atomic<int> known[64];
  int n = known[dev].load(std::memory_order_relaxed);
  if (n) return n;
  auto kernel = sample_kernel<T, N>;
  const Launch l(1, N, nullptr);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &l.cfg) != cudaSuccess || n < 1)
    return 0;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int N>
int launch(const SampleArgs& a, int M, cudaStream_t st) {
  if (!at_once<T, N>()) return IE_ERR_LAUNCH;
  const Launch l(M, N, st);
  return cudaLaunchKernelEx(&l.cfg, sample_kernel<T, N>, a) == cudaSuccess ? IE_OK : IE_ERR_LAUNCH;
}

template <typename T>
int dispatch(const SampleArgs& a, int M, cudaStream_t st) {
  // As many CTAs a row as let all rows run at once, at least as many as the
  // 16-bit counters need. Both sides of the borders, of 128256 logits: 16 rows
  // take 32.9 us with 8 CTAs each and 18.2 with 4, 15 take 19.7 with 8; 34 rows
  // take 31.7 with 4 and 21.5 with 2, 32 take 18.9 with 4.
  auto fits = [&](int n) { return (int64_t)a.V / 8 / n + 1 <= (kMaxSlice - 14) / 8; };
  if (!fits(8)) return IE_ERR_UNSUPPORTED;
  if (!fits(4) || M <= at_once<T, 8>()) return launch<T, 8>(a, M, st);
  if (!fits(2) || M <= at_once<T, 4>()) return launch<T, 4>(a, M, st);
  if (!fits(1) || M <= at_once<T, 2>()) return launch<T, 2>(a, M, st);
  return launch<T, 1>(a, M, st);
}

}  // namespace
}  // namespace ie

using namespace ie;

extern "C" int ie_sample(ie_dtype dt, int M, int V, const void* logits, int64_t ld, const float* temperature,
                         const int* top_k, const float* top_p, const float* min_p, const float* u, int* idx_out,
                         float* logprob_out, void* stream) {
  if ((dt != IE_DTYPE_F16 && dt != IE_DTYPE_BF16) || M < 0 || V < 0 || ld < V) return IE_ERR_INVALID_ARG;
  if (M == 0) return IE_OK;
  if (V == 0 || !logits || !u || !idx_out) return IE_ERR_INVALID_ARG;
  if (M > (1 << 24)) return IE_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(logits) & 1u) return IE_ERR_ALIGNMENT;
  for (const void* p : {(const void*)temperature, (const void*)top_k, (const void*)top_p, (const void*)min_p,
                        (const void*)u, (const void*)idx_out, (const void*)logprob_out})
    if (reinterpret_cast<uintptr_t>(p) & 3u) return IE_ERR_ALIGNMENT;
  SampleArgs a = {logits, ld, V, temperature, top_p, min_p, u, top_k, idx_out, logprob_out};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dt == IE_DTYPE_F16 ? dispatch<__half>(a, M, st) : dispatch<__nv_bfloat16>(a, M, st);
}
