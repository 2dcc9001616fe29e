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
// with one shared-memory atomic a token; the rest is latency. One cluster of
// N CTAs serves a row: each counts its N-th of the row into its own 65536
// 16-bit counters (128 KB of shared memory; a slice is kept to 65535 tokens so
// that none overflows), then sums the N counts of its N-th of the values and
// their masses, 32 values to a group; rank 0 gathers the 2048 groups, scans
// them and cuts.
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
template <typename T>
__device__ __forceinline__ double value_of(int key) {
  const unsigned up = 0xFFFFu - (unsigned)key;
  const unsigned short b = (unsigned short)((up & 0x8000u) ? (up & 0x7FFFu) : (~up & 0xFFFFu));
  T v;
  memcpy(&v, &b, 2);
  return (double)DT<T>::to_f(v);
}

// The row cut into 16-byte aligned chunks of 8: chunk c holds tokens
// 8c - lead .. 8c - lead + 7, of which the first and last chunk may lack some.
struct Row {
  const unsigned short* first;  // address of chunk 0 (not read below the row)
  int lead, V, chunks;
  __device__ __forceinline__ uint4 load(int c) const {
    const int i0 = 8 * c - lead;
    if (i0 >= 0 && i0 + 8 <= V) return __ldg(reinterpret_cast<const uint4*>(first) + c);
    unsigned short e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i0 + i >= 0 && i0 + i < V ? __ldg(first + 8 * c + i) : (unsigned short)0xFFFFu;
    uint4 r;  // 0xFFFF is a NaN in both types: skipped
    memcpy(&r, e, 16);
    return r;
  }
};

struct Found {
  int key, rank;    // value and rank among its tokens
  double w, before;  // its weight, the mass before the value
};

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned* hist = reinterpret_cast<unsigned*>(smem);  // two counters a word
  double* mass = reinterpret_cast<double*>(smem + kOffMass);
  int* count = reinterpret_cast<int*>(smem + kOffCount);
  __shared__ int best_key;            // this CTA's smallest key (largest logit)
  __shared__ long long above_min;     // its tokens with w >= min_p
  __shared__ double wsum[kWarps];
  __shared__ int csum[kWarps];
  __shared__ int hit_group;
  __shared__ long long hit_count;
  __shared__ double hit_mass;
  __shared__ Found found;
  __shared__ long long kept;

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = N == 1 ? 0 : (int)cluster.block_rank();
  const int row = blockIdx.x / N, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  auto sync_row = [&] {
    if constexpr (N == 1) __syncthreads();
    else cluster.sync();
  };
  auto peer = [&](auto* p, int r) {
    if constexpr (N == 1) return p;
    else return cluster.map_shared_rank(p, r);
  };

  for (int i = t; i < kHistBytes / 16; i += kThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (t == 0) {
    best_key = kKeys;
    above_min = 0;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const unsigned short* base = static_cast<const unsigned short*>(a.logits) + (int64_t)row * a.ld;
  Row in;
  in.lead = (int)((reinterpret_cast<uintptr_t>(base) & 15u) >> 1);
  in.first = base - in.lead;
  in.V = a.V;
  in.chunks = (in.lead + a.V + 7) >> 3;
  const int c0 = (int)((int64_t)in.chunks * rank / N), c1 = (int)((int64_t)in.chunks * (rank + 1) / N);
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const bool greedy = !(temp > 0.f);
  const double T64 = greedy ? 1.0 : (double)temp;
  const double low = a.min_p ? (double)a.min_p[row] : 0.0;
  const double p = a.top_p ? (double)a.top_p[row] : 1.0;
  const int k = a.top_k ? a.top_k[row] : 0;
  __syncthreads();

  // ---- count this slice's tokens by value
  int best = kKeys;
  for (int c = c0 + t; c < c1; c += kThreads) {
    const uint4 x = in.load(c);
    const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = key_of<T>((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
      if (key >= 0) {
        best = min(best, key);
        atomicAdd(hist + (key >> 1), 1u << (16 * (key & 1)));
      }
    }
  }
  best = __reduce_min_sync(0xffffffffu, best);
  if (lane == 0) atomicMin(&best_key, best);
  sync_row();
  for (int r = 0; r < N; ++r) best = min(best, *peer(&best_key, r));
  const double top = best < kKeys ? value_of<T>(best) : 0.0;
  // weight of a value that occurs; +infinity as the largest logit takes it all
  auto weight = [&](int key) -> double {
    if (key == best) return 1.0;
    const double d = value_of<T>(key) - top;
    return d < -1e300 ? 0.0 : exp(d / T64);
  };
  auto tokens = [&](int key) -> int {
    int n = 0;
#pragma unroll
    for (int r = 0; r < N; ++r)
      n += (peer(hist, r)[key >> 1] >> (16 * (key & 1))) & 0xFFFF;
    return n;
  };

  // ---- masses of this CTA's N-th of the values, 32 values (a warp) at a time
  constexpr int kMine = kKeys / N;
  long long above = 0;
  for (int i = 0; i < kMine / kThreads; ++i) {
    const int key = rank * kMine + i * kThreads + t;
    const int n = tokens(key);
    const unsigned any = __ballot_sync(0xffffffffu, n != 0);
    double m = 0.0;
    int cnt = 0;
    if (any) {
      cnt = __reduce_add_sync(0xffffffffu, n);
      if (n) {
        const double w = weight(key);
        m = n * w;
        if (w >= low) above += n;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    }
    if (lane == 0) {
      mass[key >> 5] = m;
      count[key >> 5] = cnt;
    }
  }
  if (above) atomicAdd(reinterpret_cast<unsigned long long*>(&above_min), (unsigned long long)above);
  sync_row();

  if (rank == 0) {
    // ---- scan the groups: thread t holds groups 2t and 2t + 1
    double m0, m1;
    int n0, n1;
    {
      const int r = (2 * t) / (kGroups / N);
      const double* pm = peer(mass, r) + 2 * t;
      const int* pc = peer(count, r) + 2 * t;
      m0 = pm[0]; m1 = pm[1];
      n0 = pc[0]; n1 = pc[1];
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
    double bm = 0.0, all_m = 0.0;
    long long bn = 0, all_n = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) { bm += wsum[i]; bn += csum[i]; }
      all_m += wsum[i];
      all_n += csum[i];
    }
    // mass and tokens before each of the two groups, and after the second
    const double e0 = bm + (sm - (m0 + m1)), e1 = bm + (sm - m1), e2 = bm + sm;
    const long long f0 = bn + sn - n0 - n1, f1 = f0 + n0, f2 = f1 + n1;

    // Each search below leaves one thread's group in shared memory and lets
    // warp 0 find the value in it. `in0`, `in1`: the border lies in the group.
    auto search = [&](bool in0, bool in1, auto inside) {
      if (t == 0) hit_group = -1;
      __syncthreads();
      // the first group that holds the border (rounding may let two claim it)
      if (in0) atomicMax(&hit_group, kGroups - 2 * t);
      else if (in1) atomicMax(&hit_group, kGroups - 2 * t - 1);
      __syncthreads();
      const int g = kGroups - hit_group;
      if (hit_group > 0 && (g >> 1) == t) {
        hit_mass = (g & 1) ? e1 : e0;
        hit_count = (g & 1) ? f1 : f0;
      }
      __syncthreads();
      if (warp == 0 && hit_group > 0) {
        const int key = 32 * g + lane;
        const int n = tokens(key);
        const double w = n ? weight(key) : 0.0, mass_before = hit_mass;
        const long long count_before = hit_count;
        double m = n * w;
        int c = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double um = __shfl_up_sync(0xffffffffu, m, o);
          const int uc = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) { m += um; c += uc; }
        }
        inside(key, n, w, mass_before + (m - n * w), count_before + c - n);
      }
      __syncthreads();
      return hit_group > 0;
    };
    // mass of the first n tokens, 1 <= n < all_n (all threads)
    auto mass_of_first = [&](long long n) -> double {
      search(f0 < n && n <= f1, f1 < n && n <= f2, [&](int, int c, double w, double before, long long cb) {
        if (c && cb < n && n <= cb + c) hit_mass = before + (double)(n - cb) * w;
      });
      return hit_mass;
    };

    if (all_n == 0) {
      if (t == 0) {
        a.idx[row] = -1;
        if (a.logprob) a.logprob[row] = __int_as_float(0xff800000);
      }
    } else {
      long long L = all_n;
      double Z = all_m;
      if (greedy) {
        L = 1;
      } else {
        if (k > 0 && k < L) {
          L = k;
          if (p < 1.0) Z = mass_of_first(L);
        }
        if (!(p >= 1.0)) {
          // the first value that holds a token with mass >= target before it
          // or right after its last one: its tokens before the target are kept
          const double target = p * Z;
          if (t == 0) kept = L;
          const bool some = search(m0 > 0.0 && e1 >= target, m1 > 0.0 && e2 >= target,
                                   [&](int, int c, double w, double before, long long cb) {
            const bool over = c && before + c * w >= target;
            const unsigned who = __ballot_sync(0xffffffffu, over);
            if (!who && lane == 31) kept = cb + c;  // by a rounding: the border is the group's end
            if (who && lane == __ffs(who) - 1) {
              long long n = w > 0.0 ? (long long)ceil(fmin(fmax((target - before) / w, 0.0), (double)c)) : c;
              while (n > 0 && before + (double)(n - 1) * w >= target) --n;
              while (n < c && before + (double)n * w < target) ++n;
              kept = cb + n;
            }
          });
          if (some && kept < L) L = kept;
          if (p != p) L = 1;
        }
        long long m = 0;
        for (int r = 0; r < N; ++r) m += *peer(&above_min, r);
        if (m < L) L = m;
        if (L < 1) L = 1;
      }
      Z = L < all_n ? mass_of_first(L) : all_m;
      const double target = (greedy ? 0.0 : (double)a.u[row]) * Z;
      if (t == 0) found.key = -1;
      search(n0 && e1 > target, n1 && e2 > target, [&](int key, int c, double w, double before, long long cb) {
        const bool over = c && before + c * w > target;
        const unsigned who = __ballot_sync(0xffffffffu, over), any = __ballot_sync(0xffffffffu, c != 0);
        // by a rounding none may pass it: then the group's last token does
        if (any && lane == (who ? __ffs(who) - 1 : 31 - __clz(any))) {
          long long n = (long long)fmin(fmax((target - before) / w, 0.0), (double)(c - 1));
          while (n > 0 && before + (double)n * w > target) --n;
          while (n < c - 1 && before + (double)(n + 1) * w <= target) ++n;
          if (cb + n < L) {
            found.key = key;
            found.rank = (int)n;
            found.w = w;
          }
        }
      });
      // u * Z reached the end of the kept mass (u >= 1, or rounding): the last kept token
      if (found.key < 0) {
        __syncthreads();
        search(f0 < L && L <= f1, f1 < L && L <= f2, [&](int key, int c, double w, double, long long cb) {
          if (c && cb < L && L <= cb + c) {
            found.key = key;
            found.rank = (int)(L - cb - 1);
            found.w = w;
          }
        });
      }
      // ---- the found.rank-th token of that value in index order
      const int key = found.key;
      int left = found.rank, slice = 0;
      for (; slice < N - 1; ++slice) {
        const int n = (peer(hist, slice)[key >> 1] >> (16 * (key & 1))) & 0xFFFF;
        if (left < n) break;
        left -= n;
      }
      const int s0 = (int)((int64_t)in.chunks * slice / N), s1 = (int)((int64_t)in.chunks * (slice + 1) / N);
      const int each = (s1 - s0 + kThreads - 1) / kThreads;
      const int b0 = s0 + t * each, b1 = min(b0 + each, s1);
      int mine = 0;
      auto matches = [&](const uint4& x) {
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
        unsigned hits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key_of<T>((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) == key) hits |= 1u << i;
        return hits;
      };
      for (int c = b0; c < b1; ++c) mine += __popc(matches(in.load(c)));
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
      }
      if (lane == 31) csum[warp] = sum;
      __syncthreads();
      for (int i = 0; i < warp; ++i) sum += csum[i];
      int skip = left - (sum - mine);  // this thread's matches to pass over
      if (skip >= 0 && skip < mine) {
        for (int c = b0; c < b1; ++c) {
          unsigned h = matches(in.load(c));
          const int n = __popc(h);
          if (skip >= n) {
            skip -= n;
            continue;
          }
          for (; skip > 0; --skip) h &= h - 1;
          a.idx[row] = 8 * c - in.lead + __ffs(h) - 1;
          if (a.logprob) a.logprob[row] = greedy ? 0.f : (float)log(found.w / Z);
          break;
        }
      }
    }
  }
  // the peers' shared memory stays until rank 0 has read it
  if constexpr (N > 1) cluster.sync();
}

template <typename T, int N>
int launch(const SampleArgs& a, int M, cudaStream_t st) {
  auto kernel = sample_kernel<T, N>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return IE_ERR_LAUNCH;
  static bool configured[64] = {};
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return IE_ERR_LAUNCH;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)M * N);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = N;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? IE_OK : IE_ERR_LAUNCH;
}

template <typename T>
int dispatch(const SampleArgs& a, int M, cudaStream_t st) {
  // As many CTAs a row as keep the rows within one wave of the 148 SMs, at
  // least as many as the 16-bit counters need.
  auto fits = [&](int n) { return ((int64_t)a.V + 14) / 8 / n + 1 <= kMaxSlice / 8; };
  if (!fits(8)) return IE_ERR_UNSUPPORTED;
  if (M * 8 <= 148 || !fits(4)) return launch<T, 8>(a, M, st);
  if (M * 4 <= 148 || !fits(2)) return launch<T, 4>(a, M, st);
  if (M * 2 <= 148 || !fits(1)) return launch<T, 2>(a, M, st);
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
  SampleArgs a = {logits, ld, V, temperature, top_p, min_p, u, top_k, idx_out, logprob_out};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dt == IE_DTYPE_F16 ? dispatch<__half>(a, M, st) : dispatch<__nv_bfloat16>(a, M, st);
}
