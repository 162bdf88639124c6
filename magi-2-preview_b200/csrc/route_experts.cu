// Expert routing with groups, masks and a backward pass.
//
// Forward, one warp per row (h, s) of logits l[0..E):
//   score = softmax(l) or sigmoid(l); an expert is masked where l or its bias is -inf
//   key   = score + bias, or l itself without a bias (both scores are monotone in l)
//   group score = sum of the two largest unmasked (score + bias) of a group; the `keep` best
//   groups stay; the K largest keys among them are chosen, equal keys to the lower id
//   w = scale * score / max(sum of the chosen scores, eps)  (or scale * score)
// The selection is that of 64-bit keys: it does not depend on how 32-bit scores round.
//
// Backward, from the weights' gradient g (times scale) and the chosen scores p:
//   norm:  ds = g / d - [n > eps] (sum g p) / d^2,  n = sum p, d = max(n, eps);  else ds = g
//   sigmoid: dl[idx] = ds p (1 - p)
//   softmax: dl = -score (sum ds p) + [chosen] ds p; with the norm the sum is 0 for n > eps
#include <cfloat>

#include "mxfp4.cuh"

namespace mhmoe {

namespace {

constexpr int RE_WARPS = 4;
constexpr unsigned FULL = 0xffffffffu;

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
// Larger value first, then the lower index; index -1 loses against everything.
__device__ __forceinline__ void warp_best(double& v, int& i) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(FULL, v, o);
    const int oi = __shfl_xor_sync(FULL, i, o);
    if (oi >= 0 && (i < 0 || ov > v || (ov == v && oi < i))) {
      v = ov;
      i = oi;
    }
  }
}

// Row selection in 64 bits.  key: shared [E], value: shared [E] (score + bias; may alias key
// when there are no groups).  Masked experts hold -inf, NaN holds -DBL_MAX (below every
// number, above the masked).  Lane k returns the id of the k-th choice (-1: none left).
__device__ int select64(double* key, double* value, double* gscore, int E, int K, int G, int keep, int lane) {
  if (G > 1) {
    const int per = E / G;
    for (int g = lane; g < G; g += 32) {
      double b1 = -INFINITY, b2 = -INFINITY;
      for (int j = 0; j < per; ++j) {
        const double v = value[g * per + j];
        if (v > b1) {
          b2 = b1;
          b1 = v;
        } else if (v > b2) {
          b2 = v;
        }
      }
      const double s = b2 == -INFINITY ? b1 : b1 + b2;
      gscore[g] = b1 == -INFINITY ? -INFINITY : fmax(s, -DBL_MAX);
    }
    __syncwarp();
    unsigned long long chosen = 0;
    for (int t = 0; t < keep; ++t) {
      double v = 0;
      int i = -1;
      for (int g = lane; g < G; g += 32)
        if (!(chosen >> g & 1ull) && gscore[g] != -INFINITY && (i < 0 || gscore[g] > v)) {
          v = gscore[g];
          i = g;
        }
      warp_best(v, i);
      if (i < 0) break;
      chosen |= 1ull << i;
    }
    for (int e = lane; e < E; e += 32)
      if (!(chosen >> (e / per) & 1ull)) key[e] = -INFINITY;
    __syncwarp();
  }
  int mine = -1;
  for (int k = 0; k < K; ++k) {
    double v = 0;
    int i = -1;
    for (int e = lane; e < E; e += 32)
      if (key[e] != -INFINITY && (i < 0 || key[e] > v)) {
        v = key[e];
        i = e;
      }
    warp_best(v, i);
    if (i < 0) break;
    if (lane == k) mine = i;
    if ((i & 31) == lane) key[i] = -INFINITY;
    __syncwarp();
  }
  return mine;
}

template <int DT>
__global__ void __launch_bounds__(RE_WARPS * 32)
    route_experts_kernel(const RouteArgs a, float* __restrict__ weights, int64_t* __restrict__ idx,
                         float* __restrict__ saved) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  extern __shared__ double smd[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * RE_WARPS + warp;
  if (row >= (int64_t)a.H * a.S) return;
  const int64_t h = row / a.S, s = row % a.S;
  const int E = a.E, K = a.K;
  double* key = smd + (size_t)warp * (2 * E + 64);
  double* value = key + E;
  double* gscore = value + E;
  const T* lg = static_cast<const T*>(a.logits) + h * a.stride_h + s * a.stride_s;
  const float* bias = a.bias ? a.bias + h * E : nullptr;
  int mine = -1;
  float m = -INFINITY, sum = 0.f;
  const bool routed = !a.token_mask || a.token_mask[h * a.mask_stride_h + s];
  if (routed) {
    if (a.score_func == 0) {
      bool nan = false;
      for (int e = lane; e < E; e += 32) {
        const float x = mx_to_f32(lg[e]);
        nan |= x != x;
        m = fmaxf(m, x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      if (__any_sync(FULL, nan)) m = NAN;
      double sum64 = 0;
      if (m != -INFINITY) {
        for (int e = lane; e < E; e += 32) {
          const float x = mx_to_f32(lg[e]);
          sum += expf(x - m);
          sum64 += exp((double)x - (double)m);
        }
        sum = warp_sum(sum);
        sum64 = warp_sum(sum64);
      }
      for (int e = lane; e < E; e += 32) value[e] = exp((double)mx_to_f32(lg[e]) - (double)m) / sum64;
    } else {
      for (int e = lane; e < E; e += 32) value[e] = 1.0 / (1.0 + exp(-(double)mx_to_f32(lg[e])));
    }
    for (int e = lane; e < E; e += 32) {
      const float x = mx_to_f32(lg[e]);
      const float b = bias ? bias[e] : 0.f;
      const bool masked = x == -INFINITY || b == -INFINITY;
      double v = value[e] + (double)b;
      if (v != v) v = -DBL_MAX;
      double kx = bias ? v : (x != x ? -DBL_MAX : (double)x);
      value[e] = masked ? -INFINITY : v;
      key[e] = masked ? -INFINITY : kx;
    }
    __syncwarp();
    mine = select64(key, value, gscore, E, K, a.groups, a.keep, lane);
  }
  float p = 0.f, keep_for_bwd = 0.f;
  if (mine >= 0) {
    const float x = mx_to_f32(lg[mine]);
    p = a.score_func == 0 ? __fdiv_rn(expf(x - m), sum) : __fdiv_rn(1.f, 1.f + expf(-x));
    keep_for_bwd = a.score_func == 0 ? p : x;
  }
  float w = p;
  if (a.route_norm) {
    const float n = warp_sum(p);
    w = __fdiv_rn(p, n != n ? n : fmaxf(n, a.norm_eps));
  }
  if (lane < K) {
    weights[row * K + lane] = w * a.route_scale;
    idx[row * K + lane] = mine;
    if (saved) saved[row * K + lane] = keep_for_bwd;
  }
}

// One warp per row; the row's gradient is built in shared memory and stored in order.
template <int DT>
__global__ void __launch_bounds__(RE_WARPS * 32)
    route_experts_bwd_kernel(const RouteArgs a, const float* __restrict__ grad_w, int64_t gs_h, int64_t gs_s,
                             const int64_t* __restrict__ idx, const float* __restrict__ saved,
                             typename MxType<DT>::T* __restrict__ dl) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  extern __shared__ float smf[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * RE_WARPS + warp;
  if (row >= (int64_t)a.H * a.S) return;
  const int64_t h = row / a.S, s = row % a.S;
  const int E = a.E, K = a.K;
  float* d = smf + (size_t)warp * E;
  const int64_t id = lane < K ? idx[row * K + lane] : -1;
  const bool has = id >= 0 && id < E;
  float p = 0.f, q = 0.f, g = 0.f;
  if (has) {
    p = saved[row * K + lane];
    g = grad_w[h * gs_h + s * gs_s + lane] * a.route_scale;
    if (a.score_func == 1) {
      q = __fdiv_rn(1.f, 1.f + expf(p));
      p = __fdiv_rn(1.f, 1.f + expf(-p));
    }
  }
  float ds = g;
  bool zero_dot = false;
  if (a.route_norm) {
    const float n = warp_sum(p);
    const float gp = warp_sum(g * p);
    const float den = n != n ? n : fmaxf(n, a.norm_eps);
    zero_dot = n > a.norm_eps;
    ds = __fdiv_rn(g, den);
    if (zero_dot) ds = __fdiv_rn(g - __fdiv_rn(gp, den), den);
  }
  for (int e = lane; e < E; e += 32) d[e] = 0.f;
  if (a.score_func == 0 && !zero_dot) {
    const float dot = warp_sum(has ? ds * p : 0.f);
    const T* lg = static_cast<const T*>(a.logits) + h * a.stride_h + s * a.stride_s;
    if (__any_sync(FULL, has)) {
      float m = -INFINITY, sum = 0.f;
      for (int e = lane; e < E; e += 32) m = fmaxf(m, mx_to_f32(lg[e]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      for (int e = lane; e < E; e += 32) {
        const float v = expf(mx_to_f32(lg[e]) - m);
        d[e] = v;
        sum += v;
      }
      sum = warp_sum(sum);
      for (int e = lane; e < E; e += 32) d[e] = d[e] == 0.f ? 0.f : -__fdiv_rn(d[e], sum) * dot;
    }
  }
  __syncwarp();
  if (has) d[id] += a.score_func == 0 ? ds * p : ds * p * q;
  __syncwarp();
  for (int e = lane; e < E; e += 32) mx_store(dl + row * E + e, d[e]);
}

}  // namespace

cudaError_t launch_route_experts(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st) {
  const int64_t rows = (int64_t)a.H * a.S;
  const unsigned grid = (unsigned)((rows + RE_WARPS - 1) / RE_WARPS);
  const size_t smem = (size_t)RE_WARPS * (2 * a.E + 64) * sizeof(double);
#define MX_R(DT)                                                                                                 \
  do {                                                                                                           \
    if (smem > 48 * 1024) {                                                                                      \
      const cudaError_t e = cudaFuncSetAttribute(route_experts_kernel<DT>,                                       \
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);        \
      if (e != cudaSuccess) return e;                                                                            \
    }                                                                                                            \
    MHMOE_LAUNCH_PDL(route_experts_kernel<DT>, grid, RE_WARPS * 32, smem, st, a, weights, idx, saved);           \
  } while (0)
  if (a.dtype == DT_F32) MX_R(DT_F32);
  else if (a.dtype == DT_BF16) MX_R(DT_BF16);
  else MX_R(DT_F16);
#undef MX_R
  return cudaGetLastError();
}

cudaError_t launch_route_experts_bwd(const RouteArgs& a, const float* grad_w, int64_t gs_h, int64_t gs_s,
                                     const int64_t* idx, const float* saved, void* dl, cudaStream_t st) {
  const int64_t rows = (int64_t)a.H * a.S;
  const unsigned grid = (unsigned)((rows + RE_WARPS - 1) / RE_WARPS);
  const size_t smem = (size_t)RE_WARPS * a.E * sizeof(float);
#define MX_R(DT)                                                                                          \
  MHMOE_LAUNCH_PDL(route_experts_bwd_kernel<DT>, grid, RE_WARPS * 32, smem, st, a, grad_w, gs_h, gs_s, idx, \
                   saved, static_cast<MxType<DT>::T*>(dl))
  if (a.dtype == DT_F32) MX_R(DT_F32);
  else if (a.dtype == DT_BF16) MX_R(DT_BF16);
  else MX_R(DT_F16);
#undef MX_R
  return cudaGetLastError();
}

}  // namespace mhmoe
