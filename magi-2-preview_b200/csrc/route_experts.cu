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
#include <type_traits>

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

// Experts e0 .. e0 + NPL of a row as fp32; those behind E read as `pad`.  vec: E is a multiple of
// NPL and every chunk is aligned to its size (16 B at most).
template <typename T, int NPL>
__device__ __forceinline__ void load_chunk(const T* p, int e0, int E, bool vec, float pad, float (&x)[NPL]) {
  constexpr int BYTES = NPL * (int)sizeof(T);
  if (vec && e0 + NPL <= E) {
    struct alignas(BYTES < 16 ? BYTES : 16) Chunk {
      T v[NPL];
    };
    const Chunk c = *reinterpret_cast<const Chunk*>(p + e0);
#pragma unroll
    for (int j = 0; j < NPL; ++j) x[j] = mx_to_f32(c.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) x[j] = e0 + j < E ? mx_to_f32(p[e0 + j]) : pad;
  }
}

// Order-preserving map of a number to an unsigned key >= 2; NaN gives 1, masked entries use 0.
__device__ __forceinline__ unsigned order_key(float v) {
  v += 0.f;                                       // -0 -> +0
  const unsigned b = __float_as_uint(v);
  return v != v ? 1u : b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// A row's selection with 64-bit keys (shared memory: key[E], value[E], gscore[64]).
template <typename T>
__device__ __noinline__ int select_row64(const RouteArgs& a, const T* lg, const float* bias, double* key, int lane) {
  const int E = a.E;
  double* value = key + E;
  double* gscore = value + E;
  if (a.score_func == 0) {
    float m = -INFINITY;
    bool nan = false;
    for (int e = lane; e < E; e += 32) {
      const float x = mx_to_f32(lg[e]);
      nan |= x != x;
      m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
    if (__any_sync(FULL, nan)) m = NAN;
    double sum = 0;
    for (int e = lane; e < E; e += 32) sum += exp((double)mx_to_f32(lg[e]) - (double)m);
    sum = warp_sum(sum);
    for (int e = lane; e < E; e += 32) value[e] = exp((double)mx_to_f32(lg[e]) - (double)m) / sum;
  } else {
    for (int e = lane; e < E; e += 32) value[e] = 1.0 / (1.0 + exp(-(double)mx_to_f32(lg[e])));
  }
  for (int e = lane; e < E; e += 32) {
    const float x = mx_to_f32(lg[e]);
    const float b = bias ? bias[e] : 0.f;
    const bool masked = x == -INFINITY || b == -INFINITY;
    double v = value[e] + (double)b;
    if (v != v) v = -DBL_MAX;
    const double kx = bias ? v : (x != x ? -DBL_MAX : (double)x);
    value[e] = masked ? -INFINITY : v;
    key[e] = masked ? -INFINITY : kx;
  }
  __syncwarp();
  return select64(key, value, gscore, E, a.K, a.groups, a.keep, lane);
}

// Lane l holds experts [l * NPL, (l + 1) * NPL) in registers.  Keys are fp32; where two candidates
// whose order matters are closer than the keys' error (and are not the same logit and bias),
// the row's selection is done again in 64 bits.  Bounds of that error: a softmax score is off by
// less than 2^-18 of the row's largest score (sum, exponent argument and exponential), a
// sigmoid by less than 2^-21, the sum with the bias by half a unit of 2^-23; a difference of two is
// off by twice that, of two group sums by four times.
template <int DT, int NPL>
__global__ void __launch_bounds__(RE_WARPS * 32)
    route_experts_kernel(const RouteArgs a, bool vec, unsigned per_magic, float* __restrict__ weights,
                         int64_t* __restrict__ idx, float* __restrict__ saved) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  extern __shared__ double smd[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned row = blockIdx.x * RE_WARPS + warp;
  if (row >= (unsigned)(a.H * a.S)) return;
  const unsigned h = row / (unsigned)a.S, s = row - h * (unsigned)a.S;
  const int E = a.E, K = a.K, e0 = lane * NPL;
  const T* lg = static_cast<const T*>(a.logits) + h * a.stride_h + s * a.stride_s;
  const float* bias = a.bias ? a.bias + (int64_t)h * E : nullptr;
  double* scratch = smd + (size_t)warp * (2 * E + 64);
  int mine = -1;
  float m = 0.f, sum = 1.f;
  if (!a.token_mask || a.token_mask[h * a.mask_stride_h + s]) {
    float x[NPL];
    load_chunk<T, NPL>(lg, e0, E, vec, -INFINITY, x);
    float smax = 1.f;
    if (a.score_func == 0) {
      m = x[0];
      bool nan = x[0] != x[0];
#pragma unroll
      for (int j = 1; j < NPL; ++j) {
        nan |= x[j] != x[j];
        m = fmaxf(m, x[j]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      if (__any_sync(FULL, nan)) m = NAN;
    }
    unsigned key[NPL];
    if (a.score_func == 0 && m == -INFINITY) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) key[j] = 0;                   // no expert is left
    } else {
      const bool need_v = bias || a.groups > 1;
      float v[NPL];
      if (a.score_func == 0) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          v[j] = __expf(x[j] - m);
          sum += v[j];
        }
        sum = warp_sum(sum);
        smax = __fdiv_rn(1.f, sum);
#pragma unroll
        for (int j = 0; j < NPL; ++j) v[j] *= smax;
      } else if (need_v) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) v[j] = __fdividef(1.f, 1.f + __expf(-x[j]));
      }
      bool gone[NPL];
#pragma unroll
      for (int j = 0; j < NPL; ++j) gone[j] = x[j] == -INFINITY;
      if (bias) {
        float b[NPL];
        load_chunk<float, NPL>(bias, e0, E, vec, -INFINITY, b);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          gone[j] |= b[j] == -INFINITY;
          v[j] += b[j];
        }
      }
#pragma unroll
      for (int j = 0; j < NPL; ++j) key[j] = gone[j] ? 0u : order_key(bias ? v[j] : x[j]);
      const float tol0 = a.score_func == 0 ? smax * 0x1p-17f : 0x1p-20f;
      bool close = false;                                         // warp-uniform
      if (a.groups > 1 && a.keep < a.groups) {
        // two best of every group: 32 / G lanes (a power of two) walk a group in shared memory
        const int G = a.groups, per = E / G;
        unsigned* sv = reinterpret_cast<unsigned*>(scratch);
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (e0 + j < E) sv[e0 + j] = gone[j] ? 0u : order_key(v[j]);
        __syncwarp();
        const int lanes = G > 16 ? 1 : G > 8 ? 2 : G > 4 ? 4 : G > 2 ? 8 : 16;
        unsigned gk[2];
        float mag = 0.f;                                          // bounds the roundings of v: sums may cancel
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int g = lane / lanes + 32 * half;
          unsigned b1 = 0, b2 = 0;
          if (g < G)
            for (int i = lane & (lanes - 1); i < per; i += lanes) {
              const unsigned k = sv[g * per + i];
              b2 = max(b2, min(b1, k));
              b1 = max(b1, k);
            }
          for (int o = 1; o < lanes; o <<= 1) {
            const unsigned o1 = __shfl_xor_sync(FULL, b1, o), o2 = __shfl_xor_sync(FULL, b2, o);
            b2 = max(max(b2, o2), min(b1, o1));
            b1 = max(b1, o1);
          }
          close |= b1 == 1u || b2 == 1u;                          // a NaN among the two best
          if (b1 > 1u) mag = fmaxf(mag, fabsf(key_value(b1)) + (b2 > 1u ? fabsf(key_value(b2)) : 0.f));
          const float total = b2 ? key_value(b1) + key_value(b2) : key_value(b1);
          gk[half] = b1 == 0 || (lane & (lanes - 1)) ? 0u : order_key(total);
          if (G <= 32) {
            gk[1] = 0;
            break;
          }
        }
        close = __any_sync(FULL, close);
        mag = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(mag)));
        unsigned long long kept = 0;
        unsigned last = 0;
        for (int t = 0; t <= a.keep; ++t) {
          const unsigned best = __reduce_max_sync(FULL, max(gk[0], gk[1]));
          if (best == 0) break;
          if (t == a.keep) {
            const float lv = key_value(last);
            close |= !(lv - key_value(best) > 4.f * tol0 + 0x1p-21f * mag);
            break;
          }
          const unsigned in0 = __ballot_sync(FULL, gk[0] == best), in1 = __ballot_sync(FULL, gk[1] == best);
          const int owner = __ffs(in0 ? in0 : in1) - 1;
          kept |= 1ull << (in0 ? owner / lanes : owner + 32);
          if (lane == owner) gk[in0 ? 0 : 1] = 0;
          last = best;
        }
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (!(kept >> ((((e0 + j) * per_magic) >> 20) & 63u) & 1ull)) key[j] = 0;
      }
      // K rounds: the best lane wins, the lower lane (and expert) among equals; one more round
      // shows how close the first one left out is
      unsigned top = 0, next = 0;
      int tj = 0, mine_next = -1;
      auto local_best = [&] {
        top = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (key[j] > top) {
            top = key[j];
            tj = j;
          }
      };
      local_best();
      unsigned mine_key = 0;
      const int rounds = bias ? K + 1 : K;
      for (int k = 0; k < rounds; ++k) {
        const unsigned best = __reduce_max_sync(FULL, top);
        if (best == 0) break;
        const int owner = __ffs(__ballot_sync(FULL, top == best)) - 1;
        const int id = owner * NPL + __shfl_sync(FULL, tj, owner);
        if (lane == k && k < K) {
          mine = id;
          mine_key = best;
        }
        if (lane == k - 1) {
          mine_next = id;
          next = best;
        }
        if (lane == owner) {
#pragma unroll
          for (int j = 0; j < NPL; ++j)
            if (j == tj) key[j] = 0;
          local_best();
        }
      }
      if (bias) {
        bool mine_close = false;
        if (mine >= 0 && mine_next >= 0) {
          const float v0 = key_value(mine_key), v1 = key_value(next);
          if (!(v0 - v1 > tol0 + 0x1p-22f * fabsf(v0)) || next == 1u)
            mine_close = mx_to_f32(lg[mine]) != mx_to_f32(lg[mine_next]) || bias[mine] != bias[mine_next];
        }
        close |= __any_sync(FULL, mine_close);
      }
      if (close) {
        __syncwarp();
        mine = select_row64<T>(a, lg, bias, scratch, lane);
      }
    }
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
    const int64_t o = (int64_t)row * K + lane;
    weights[o] = w * a.route_scale;
    idx[o] = mine;
    if (saved) saved[o] = keep_for_bwd;
  }
}

// One warp per row; the row's gradient is put together in shared memory (most of it zero) and
// stored in order, NPL experts a lane.
template <int DT, int NPL>
__global__ void __launch_bounds__(RE_WARPS * 32)
    route_experts_bwd_kernel(const RouteArgs a, bool vec, bool vec_out, const float* __restrict__ grad_w, int64_t gs_h,
                             int64_t gs_s, const int64_t* __restrict__ idx, const float* __restrict__ saved,
                             typename MxType<DT>::T* __restrict__ dl) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  extern __shared__ float smf[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned row = blockIdx.x * RE_WARPS + warp;
  if (row >= (unsigned)(a.H * a.S)) return;
  const unsigned h = row / (unsigned)a.S, s = row - h * (unsigned)a.S;
  const int E = a.E, K = a.K, e0 = lane * NPL;
  float* d = smf + (size_t)warp * (32 * NPL);
  const int64_t id = lane < K ? idx[(int64_t)row * K + lane] : -1;
  const bool has = id >= 0 && id < E;
  float p = 0.f, q = 0.f, g = 0.f;
  if (has) {
    p = saved[(int64_t)row * K + lane];
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
  float o[NPL];
#pragma unroll
  for (int j = 0; j < NPL; ++j) o[j] = 0.f;
  if (a.score_func == 0 && !zero_dot && __any_sync(FULL, has)) {
    const float dot = warp_sum(has ? ds * p : 0.f);
    const T* lg = static_cast<const T*>(a.logits) + h * a.stride_h + s * a.stride_s;
    load_chunk<T, NPL>(lg, e0, E, vec, -INFINITY, o);
    float m = o[0], sum = 0.f;
#pragma unroll
    for (int j = 1; j < NPL; ++j) m = fmaxf(m, o[j]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, k));
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      o[j] = o[j] == -INFINITY ? 0.f : expf(o[j] - m);
      sum += o[j];
    }
    const float f = -__fdiv_rn(dot, warp_sum(sum));
#pragma unroll
    for (int j = 0; j < NPL; ++j) o[j] = o[j] == 0.f ? 0.f : o[j] * f;
  }
#pragma unroll
  for (int j = 0; j < NPL; ++j) d[j * 32 + lane] = o[j];          // expert e at (e % NPL) * 32 + e / NPL
  __syncwarp();
  if (has) d[(int)(id % NPL) * 32 + (int)(id / NPL)] += a.score_func == 0 ? ds * p : ds * p * q;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < NPL; ++j) o[j] = d[j * 32 + lane];
  T* out = dl + (int64_t)row * E + e0;
  if (vec_out && e0 + NPL <= E) {
    constexpr int BYTES = NPL * (int)sizeof(T);
    struct alignas(BYTES < 16 ? BYTES : 16) Chunk {
      T v[NPL];
    } c;
#pragma unroll
    for (int j = 0; j < NPL; ++j) mx_store(&c.v[j], o[j]);
    *reinterpret_cast<Chunk*>(out) = c;
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (e0 + j < E) mx_store(out + j, o[j]);
  }
}

// Experts a lane: the smallest power of two that covers E with 32 lanes.
int experts_per_lane(int E) {
  int n = 1;
  while (32 * n < E) n *= 2;
  return n;
}

// Chunks of npl elements start on multiples of their size (16 B at most) in every row.
bool chunks_aligned(const void* p, int64_t stride_h, int64_t stride_s, int E, int esz, int npl) {
  const int64_t unit = std::min(16, esz * npl);
  return E % npl == 0 && reinterpret_cast<uintptr_t>(p) % unit == 0 && stride_h * esz % unit == 0 &&
         stride_s * esz % unit == 0;
}

template <int DT, int NPL>
cudaError_t run_fwd(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)a.H * a.S + RE_WARPS - 1) / RE_WARPS);
  const size_t smem = (size_t)RE_WARPS * (2 * a.E + 64) * sizeof(double);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(route_experts_kernel<DT, NPL>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const bool vec = chunks_aligned(a.logits, a.stride_h, a.stride_s, a.E, DT == DT_F32 ? 4 : 2, NPL) &&
                   (!a.bias || chunks_aligned(a.bias, a.E, 0, a.E, 4, NPL));
  // e / per = e * ceil(2^20 / per) >> 20 for e < 1024
  const unsigned per = (unsigned)(a.E / a.groups), magic = ((1u << 20) + per - 1) / per;
  MHMOE_LAUNCH_PDL((route_experts_kernel<DT, NPL>), grid, RE_WARPS * 32, smem, st, a, vec, magic, weights, idx, saved);
  return cudaGetLastError();
}

template <int DT, int NPL>
cudaError_t run_bwd(const RouteArgs& a, const float* grad_w, int64_t gs_h, int64_t gs_s, const int64_t* idx,
                    const float* saved, void* dl, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)a.H * a.S + RE_WARPS - 1) / RE_WARPS);
  constexpr int esz = DT == DT_F32 ? 4 : 2;
  const bool vec = a.logits && chunks_aligned(a.logits, a.stride_h, a.stride_s, a.E, esz, NPL);
  const bool vec_out = chunks_aligned(dl, 0, a.E, a.E, esz, NPL);
  MHMOE_LAUNCH_PDL((route_experts_bwd_kernel<DT, NPL>), grid, RE_WARPS * 32, (size_t)RE_WARPS * 32 * NPL * 4, st, a, vec,
                   vec_out, grad_w, gs_h, gs_s, idx, saved, static_cast<typename MxType<DT>::T*>(dl));
  return cudaGetLastError();
}

template <int DT, class F>
cudaError_t by_width(int E, F&& f) {
  switch (experts_per_lane(E)) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 8: return f(std::integral_constant<int, 8>{});
    case 16: return f(std::integral_constant<int, 16>{});
    default: return f(std::integral_constant<int, 32>{});
  }
}

}  // namespace

cudaError_t launch_route_experts(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st) {
  auto go = [&](auto dt) {
    return by_width<dt>(a.E, [&](auto npl) { return run_fwd<dt, npl>(a, weights, idx, saved, st); });
  };
  if (a.dtype == DT_F32) return go(std::integral_constant<int, DT_F32>{});
  if (a.dtype == DT_BF16) return go(std::integral_constant<int, DT_BF16>{});
  return go(std::integral_constant<int, DT_F16>{});
}

cudaError_t launch_route_experts_bwd(const RouteArgs& a, const float* grad_w, int64_t gs_h, int64_t gs_s,
                                     const int64_t* idx, const float* saved, void* dl, cudaStream_t st) {
  auto go = [&](auto dt) {
    return by_width<dt>(a.E, [&](auto npl) { return run_bwd<dt, npl>(a, grad_w, gs_h, gs_s, idx, saved, dl, st); });
  };
  if (a.dtype == DT_F32) return go(std::integral_constant<int, DT_F32>{});
  if (a.dtype == DT_BF16) return go(std::integral_constant<int, DT_BF16>{});
  return go(std::integral_constant<int, DT_F16>{});
}

}  // namespace mhmoe
