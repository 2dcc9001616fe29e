// Per-head RMSNorm of the new tokens' queries and keys, rotation, and the
// write of keys and values to their rows of a paged cache, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (over the head's dimensions, fp32; skipped without weights)
//   z[d]        = y[d] cos[p][d] - y[d + D/2] sin[p][d]
//   z[d + D/2]  = y[d + D/2] cos[p][d] + y[d] sin[p][d]      d < D/2, p the token's position
//
// everything in fp32 with one rounding when z is stored; values are copied.
// What bounds it: each query, key and value is read once and written once, so
// a large batch is HBM-bound and a decode step is one launch's latency.
//
// Layout: D/16 lanes serve a head (8 for D = 128, 4 for 64). A lane loads the
// 16 bytes at dimension 8i and the 16 bytes at D/2 + 8i, so both members of
// every rotated pair are in its registers and the norm needs 3 (or 2)
// shuffles. A warp serves one token: it issues the loads of kHeads rounds of
// 32 / (D/16) heads, finds the token's sequence (a 32-ary search over q_start)
// and page meanwhile, and holds the position's cosines and sines in registers
// for all its heads.
#include "ie_common.cuh"
#include "norm.cuh"
#include "paged.cuh"
#include "paged_ops.cuh"

namespace ie {

__device__ int g_paged_norm_status = 0;

namespace {

constexpr int kMaxThreads = 256;

struct NormArgs {
  PagedBatch b;
  PagedLayout l;
  const void *q, *k, *v, *qw, *kw;
  int64_t ldq, hsq, ldk, hsk, ldv, hsv, ldo, hso;
  void *q_out, *kc, *vc;
  const float *cos, *sin;
  int rope_rows, n_q;
  float eps;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& r, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = DT<T>::to_f(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = DT<T>::from_f(f[i]);
  return r;
}
// coherent (q_out may alias q) and past L1, which no row visits twice: 53.2 -> 52.4 us at 11204 tokens
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

template <typename T, int D, int kHeads>
__global__ void __launch_bounds__(kMaxThreads) qk_norm_rope_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kLanes = D / 16;          // lanes of one head
  constexpr int kPerRound = 32 / kLanes;  // heads of one round
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x;
  const int d = 8 * (lane % kLanes);  // this lane's dimensions: d .. d + 7 and D/2 + d ..
  const int heads = a.n_q + 2 * a.l.n_kv_heads;
  const int h0 = ((int)blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kHeads * kPerRound + lane / kLanes;

  // the rows are on their way while the token's place is found
  uint4 lo[kHeads], hi[kHeads];
#pragma unroll
  for (int r = 0; r < kHeads; ++r) {
    const int h = h0 + r * kPerRound;
    if (h < heads) {
      const T* src;
      if (h < a.n_q)
        src = static_cast<const T*>(a.q) + t * a.ldq + h * a.hsq;
      else if (h < a.n_q + a.l.n_kv_heads)
        src = static_cast<const T*>(a.k) + t * a.ldk + (h - a.n_q) * a.hsk;
      else
        src = static_cast<const T*>(a.v) + t * a.ldv + (h - a.n_q - a.l.n_kv_heads) * a.hsv;
      lo[r] = ld16(src + d);
      hi[r] = ld16(src + D / 2 + d);
    }
  }
  const int seq = paged_owner(a.b.q_start, a.b.B, (int)t);
  if (seq < 0 || seq >= a.b.B) return;  // a row no sequence owns is left as it is
  const int start = a.b.q_start[seq];
  const int64_t pos64 = (int64_t)a.b.kv_len[seq] - ((int64_t)a.b.q_start[seq + 1] - start) + (t - start);
  bool bad = pos64 < 0 || pos64 >= ((int64_t)a.b.max_pages << a.l.page_log2) || (a.cos && pos64 >= a.rope_rows);
  const int pos = bad ? 0 : (int)pos64;
  int page = 0;
  if (!bad) page = a.b.page_table[(int64_t)seq * a.b.ld_table + (pos >> a.l.page_log2)];
  bad = bad || page < 0 || page >= a.l.num_pages;
  if (bad) {
    if (lane == 0) atomicExch(&g_paged_norm_status, IE_ERR_INVALID_ARG);
    return;
  }
  const int64_t row = (int64_t)page * a.l.page_stride + (int64_t)(pos & (a.l.page_size - 1)) * a.l.row_stride;
  float c[8], s[8];
  if (a.cos) {
    const float4* cp = reinterpret_cast<const float4*>(a.cos + (int64_t)pos * (D / 2) + d);
    const float4* sp = reinterpret_cast<const float4*>(a.sin + (int64_t)pos * (D / 2) + d);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 x = __ldg(cp + i), y = __ldg(sp + i);
      c[4 * i] = x.x; c[4 * i + 1] = x.y; c[4 * i + 2] = x.z; c[4 * i + 3] = x.w;
      s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
    }
  }
#pragma unroll
  for (int r = 0; r < kHeads; ++r) {
    const int h = h0 + r * kPerRound;
    const bool is_v = h >= a.n_q + a.l.n_kv_heads;
    float x[8], y[8];
    unpack8<T>(lo[r], x);
    unpack8<T>(hi[r], y);
    // every lane of the warp takes part in the shuffles, rows past the last head included
    const void* wt = h < a.n_q ? a.qw : a.kw;
    float ss = 0.f;
    if (h < heads && !is_v && wt) {
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (h >= heads) continue;
    T* dst;
    if (is_v) {
      dst = static_cast<T*>(a.vc) + row + (h - a.n_q - a.l.n_kv_heads) * a.l.head_stride;
    } else {
      if (wt) {
        const float scale = rsqrtf(ss * (1.0f / D) + a.eps);
        float u[8], v[8];
        unpack8<T>(ld_act_v4(static_cast<const T*>(wt) + d), u);
        unpack8<T>(ld_act_v4(static_cast<const T*>(wt) + D / 2 + d), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * scale * u[i];
          y[i] = y[i] * scale * v[i];
        }
      }
      if (a.cos) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = x[i], q = y[i];
          x[i] = p * c[i] - q * s[i];
          y[i] = q * c[i] + p * s[i];
        }
      }
      lo[r] = pack8<T>(x);
      hi[r] = pack8<T>(y);
      dst = h < a.n_q ? static_cast<T*>(a.q_out) + t * a.ldo + h * a.hso
                      : static_cast<T*>(a.kc) + row + (h - a.n_q) * a.l.head_stride;
    }
    *reinterpret_cast<uint4*>(dst + d) = lo[r];
    *reinterpret_cast<uint4*>(dst + D / 2 + d) = hi[r];
  }
}

template <typename T, int D, int kHeads>
int launch_heads(NormArgs& a, cudaStream_t st) {
  constexpr int kPerRound = 32 / (D / 16);
  const int warps = ceil_div(a.n_q + 2 * a.l.n_kv_heads, kPerRound * kHeads);
  const int blocks = ceil_div(warps, kMaxThreads / 32);  // of a token, evenly filled
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.b.T, (unsigned)blocks);
  cfg.blockDim = dim3(32u * ceil_div(warps, blocks));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_enabled() && a.b.T <= pdl_max_rows() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<T, D, kHeads>, a) == cudaSuccess ? IE_OK : IE_ERR_LAUNCH;
}

template <typename T, int D>
int launch_norm(NormArgs& a, cudaStream_t st) {
  // One round of heads a warp while that leaves the GPU's warp slots unfilled
  // (a decode step), else three: with 11204 tokens of 32 + 8 + 8 heads one,
  // two, three, four and six rounds took 78, 65, 55, 56 and 65 us.
  constexpr int kPerRound = 32 / (D / 16);
  const int64_t warps = (int64_t)a.b.T * ceil_div(a.n_q + 2 * a.l.n_kv_heads, kPerRound);
  return warps <= 148 * 32 ? launch_heads<T, D, 1>(a, st) : launch_heads<T, D, 3>(a, st);
}

// rows of `heads` heads of D elements at the given strides
int check_rows(const void* p, int64_t ld, int64_t hs, int D) {
  if (!p || ld < 0 || hs < D || ld > (INT64_C(1) << 40) || hs > (INT64_C(1) << 40)) return IE_ERR_INVALID_ARG;
  if (!aligned16(p) || ld % 8 || hs % 8) return IE_ERR_ALIGNMENT;
  return IE_OK;
}

}  // namespace

int read_paged_norm_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_paged_norm_status, sizeof(int)) != cudaSuccess) return IE_ERR_LAUNCH;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_paged_norm_status, &z, sizeof(int));
  }
  return v;
}

}  // namespace ie

using namespace ie;

extern "C" int ie_qk_norm_rope_paged(ie_dtype dt, int B, int T, int n_q_heads, const void* q, int64_t ldq,
                                     int64_t q_head_stride, const void* k, int64_t ldk, int64_t k_head_stride,
                                     const void* v, int64_t ldv, int64_t v_head_stride, const void* q_weight,
                                     const void* k_weight, float eps, const float* rope_cos, const float* rope_sin,
                                     int rope_rows, const ie_paged_cache* cache, const int* page_table,
                                     int64_t ld_table, int max_pages, const int* q_start, const int* kv_len,
                                     void* q_out, int64_t ldo, int64_t o_head_stride, void* stream) {
  if ((dt != IE_DTYPE_F16 && dt != IE_DTYPE_BF16) || n_q_heads <= 0) return IE_ERR_INVALID_ARG;
  int s = check_paged(cache, B, T, page_table, ld_table, max_pages, q_start, kv_len);
  if (s) return s;
  if ((rope_cos == nullptr) != (rope_sin == nullptr) || (rope_cos && rope_rows <= 0)) return IE_ERR_INVALID_ARG;
  if (!(eps >= 0.f)) return IE_ERR_INVALID_ARG;
  if (n_q_heads > 65536 || cache->n_kv_heads > 65536) return IE_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return IE_OK;
  const int D = cache->head_dim;
  if ((s = check_rows(q, ldq, q_head_stride, D)) || (s = check_rows(k, ldk, k_head_stride, D)) ||
      (s = check_rows(v, ldv, v_head_stride, D)) || (s = check_rows(q_out, ldo, o_head_stride, D)))
    return s;
  // output rows must not overlap: tokens outside heads or heads outside tokens
  if (T > 1 && !(ldo >= (n_q_heads - 1) * o_head_stride + D ||
                 (ldo >= D && (n_q_heads == 1 || o_head_stride >= (T - 1) * ldo + D))))
    return IE_ERR_INVALID_ARG;
  if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight)) ||
      (rope_cos && (!aligned16(rope_cos) || !aligned16(rope_sin))))
    return IE_ERR_ALIGNMENT;
  NormArgs a = {};
  a.b = {q_start, kv_len, page_table, ld_table, B, T, max_pages};
  a.l = paged_layout(cache);
  a.q = q; a.ldq = ldq; a.hsq = q_head_stride;
  a.k = k; a.ldk = ldk; a.hsk = k_head_stride;
  a.v = v; a.ldv = ldv; a.hsv = v_head_stride;
  a.qw = q_weight; a.kw = k_weight; a.eps = eps;
  a.q_out = q_out; a.ldo = ldo; a.hso = o_head_stride;
  a.kc = cache->k; a.vc = cache->v;
  a.cos = rope_cos; a.sin = rope_sin; a.rope_rows = rope_rows;
  a.n_q = n_q_heads;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dt == IE_DTYPE_F16) return D == 128 ? launch_norm<__half, 128>(a, st) : launch_norm<__half, 64>(a, st);
  return D == 128 ? launch_norm<__nv_bfloat16, 128>(a, st) : launch_norm<__nv_bfloat16, 64>(a, st);
}
