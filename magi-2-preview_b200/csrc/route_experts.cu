// Expert routing with groups, masks and a backward pass.
//
// Forward, one warp per row (h, s) of logits l[0..E):
//   score = softmax(l) or sigmoid(l); an expert is masked where l or its bias is -inf
//   key   = score + bias, or l itself without a bias (both scores are monotone in l)
//   group score = sum of the two largest unmasked (score + bias) of a group; the `keep` best
//   groups stay; the K largest keys among them are chosen, equal keys to the lower id
//   w = scale * score / max(sum of the chosen scores, eps)  (or scale * score); 0 without an expert
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

// A row's selection with 64-bit keys, in shared memory val[E] and gscore[64].  Masked experts hold
// -inf, NaN holds -DBL_MAX (below every number, above the masked).  Lane k returns the id of the
// k-th choice (-1: none left).
template <typename T>
__device__ __noinline__ int select_row64(const RouteArgs& a, const T* lg, const float* bias, double* val, int lane) {
  const int E = a.E, G = a.groups;
  double* gscore = val + E;
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
    for (int e = lane; e < E; e += 32) val[e] = exp((double)mx_to_f32(lg[e]) - (double)m) / sum;
  } else {
    for (int e = lane; e < E; e += 32) val[e] = 1.0 / (1.0 + exp(-(double)mx_to_f32(lg[e])));
  }
  for (int e = lane; e < E; e += 32) {
    const float b = bias ? bias[e] : 0.f;
    const double v = val[e] + (double)b;
    val[e] = mx_to_f32(lg[e]) == -INFINITY || b == -INFINITY ? -INFINITY : (v != v ? -DBL_MAX : v);
  }
  __syncwarp();
  unsigned long long kept = ~0ull;
  const int per = E / G;
  if (a.keep < G) {
    for (int g = lane; g < G; g += 32) {
      double b1 = -INFINITY, b2 = -INFINITY;
      for (int j = 0; j < per; ++j) {
        const double v = val[g * per + j];
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
    kept = 0;
    for (int t = 0; t < a.keep; ++t) {
      double v = 0;
      int i = -1;
      for (int g = lane; g < G; g += 32)
        if (!(kept >> g & 1ull) && gscore[g] != -INFINITY && (i < 0 || gscore[g] > v)) {
          v = gscore[g];
          i = g;
        }
      warp_best(v, i);
      if (i < 0) break;
      kept |= 1ull << i;
    }
  }
  // the keys: score + bias, or the logits
  for (int e = lane; e < E; e += 32) {
    const float x = mx_to_f32(lg[e]);
    if (!bias && val[e] != -INFINITY) val[e] = x != x ? -DBL_MAX : (double)x;
    if (!(kept >> (e / per) & 1ull)) val[e] = -INFINITY;
  }
  __syncwarp();
  int mine = -1;
  for (int k = 0; k < a.K; ++k) {
    double v = 0;
    int i = -1;
    for (int e = lane; e < E; e += 32)
      if (val[e] != -INFINITY && (i < 0 || val[e] > v)) {
        v = val[e];
        i = e;
      }
    warp_best(v, i);
    if (i < 0) break;
    if (lane == k) mine = i;
    if ((i & 31) == lane) val[i] = -INFINITY;
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

// Order-preserving map of a number to an unsigned key; a masked entry is 0, below all of them.
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned b = __float_as_uint(v);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Descending sort of a thread's keys: Batcher's odd-even merge network (Batcher 1968).
template <int N>
__device__ __forceinline__ void sort_keys(unsigned (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j < N - q; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const unsigned hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
            k[i + j] = hi;
            k[i + j + q] = lo;
          }
}

// Bytes of shared memory a warp needs: the lanes' sorted keys of its rows (NPL and a 0 behind them),
// over which a row that is done again puts its 64-bit keys and group scores; and a row's keys by
// expert, to walk groups in.
__host__ __device__ constexpr int fwd_scratch_bytes(int E, int npl, int rpw, bool grouped) {
  const int lists = rpw * (npl + 1) * 128, again = 8 * E + 512;
  return (lists > again ? lists : again) + (grouped ? (4 * E + 7) / 8 * 8 : 0);
}

// A warp takes RPW consecutive rows: scores, keys and sorting one row after another, the selection's
// rounds for all of them together (a round is a chain of a warp-wide maximum and a load, which one
// row alone leaves waiting), and what follows (scores of the chosen, normalisation, stores) for all
// at once, 32 / RPW >= K lanes a row.
//
// Lane l holds experts [l * NPL, (l + 1) * NPL) of the row in registers.  A key is the order-preserving map of
// the candidate's fp32 value with its low bits replaced by the complement of the expert's id:
// keys are unique, equal values rank by id, and one warp-wide integer maximum gives the best
// value and its id.  Each lane sorts its keys once and offers its largest.
//
// The bits given up and fp32 scores can put close candidates in the wrong order.  So the chosen
// ones are compared once more by their full fp32 values, and the last of them with the largest
// value the first one left out can have; where a gap is not above the values' error (and the
// two are not the same logit and bias) the row is selected again in 64 bits.  Bounds of the
// error: a softmax score is off by less than 2^-18 of the row's largest score (sum, exponent
// argument and exponential), a sigmoid by less than 2^-21, the sum with the bias by half a unit
// of 2^-23; a difference of two by twice that, of two group sums by four times.  Logits
// themselves (no bias) are exact: 16-bit ones fit above the id bits, so their keys are too.
//
// Bound by instructions and the latency of the K dependent maxima, not by the 2 or 4 B a logit read: that is
// why up to four rows share a warp's reductions, and why kernels of four rows have the score function and
// the presence of a bias (SCORE, BIAS; -1: read from the arguments) as constants.  196608 rows of 256 fp32
// logits, top-6 of sigmoid + bias: 88 us, 2.4 TB/s (108 with the two read from the arguments and a block
// more a SM; 222 with a row a warp and the ids reduced beside the values); 16381 rows of 128, softmax
// top-8: 16 us (19); 16396 rows of 160 in 8 groups: 30 us (35).  A full fp32 count of the row's
// candidates before the 64-bit selection saved none of it (109 against 108 us).
template <int DT, int NPL, int RPW, bool GROUPED, int SCORE, int BIAS>
__global__ void __launch_bounds__(RE_WARPS * 32, NPL <= 8 ? (SCORE < 0 ? 9 : 8) : NPL <= 16 ? 6 : 4)
    route_experts_kernel(const __grid_constant__ RouteArgs a, bool vec, unsigned per_magic, float* __restrict__ weights,
                         int64_t* __restrict__ idx, float* __restrict__ saved) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  constexpr unsigned ID = 32 * NPL - 1;                           // id bits of a key
  constexpr float LOG2E = 1.44269504f;
  extern __shared__ double smd[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int SEG = 32 / RPW;
  const unsigned rows = (unsigned)(a.H * a.S), row0 = (blockIdx.x * RE_WARPS + warp) * RPW;
  if (row0 >= rows) return;
  const int n_rows = (int)min((unsigned)RPW, rows - row0), mine_r = lane / SEG, rank = lane % SEG;
  const bool softmax = SCORE < 0 ? a.score_func == 0 : SCORE == 0, biased = BIAS < 0 ? a.bias != nullptr : BIAS == 1;
  const int E = a.E, K = a.K, e0 = lane * NPL, G = a.groups;
  const bool exact = DT != DT_F32 && !biased;
  const int bytes = fwd_scratch_bytes(E, NPL, RPW, GROUPED);
  double* scratch = smd + (size_t)warp * (bytes / 8);
  unsigned* lists = reinterpret_cast<unsigned*>(scratch);         // [RPW][NPL + 1][32]
  unsigned* words = lists + bytes / 4 - (E + 1) / 2 * 2;          // [E], with groups
  float b[NPL];                                                   // the head's biases
  bool b_odd = false;                                             // one of them is no number
  // of this lane's choice (row row0 + mine_r, the rank-th)
  unsigned mine_key = 0, extra = 0;
  float m_l = 0.f, sum_l = 1.f, tol_l = 0x1p-20f;
  bool close = false;
  unsigned h = row0 / (unsigned)a.S, s = row0 - h * (unsigned)a.S;
  // a row's logits are loaded while the row before is worked on
  float ahead[NPL];
  auto fetch = [&](unsigned fh, unsigned fs) {
    load_chunk<T, NPL>(static_cast<const T*>(a.logits) + fh * a.stride_h + fs * a.stride_s, e0, E, vec, -INFINITY, ahead);
  };
  fetch(h, s);
  for (int r = 0; r < n_rows; ++r, ++s) {
    if (s == (unsigned)a.S) {
      s = 0;
      ++h;
    }
    if (biased && (r == 0 || s == 0)) {
      load_chunk<float, NPL>(a.bias + (int64_t)h * E, e0, E, vec, 0.f, b);
      float probe = 0.f;
#pragma unroll
      for (int j = 0; j < NPL; ++j) probe = fmaf(b[j], 0.f, probe);
      b_odd = !(probe == 0.f);
    }
    float x[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) x[j] = ahead[j];
    if (r + 1 < n_rows) fetch(s + 1 == (unsigned)a.S ? h + 1 : h, s + 1 == (unsigned)a.S ? 0u : s + 1);
    unsigned* list = lists + r * (NPL + 1) * 32 + lane;
    list[0] = 0;                                                  // for a row without a choice
    if (a.token_mask && !a.token_mask[h * a.mask_stride_h + s]) continue;
    const bool mine_row = mine_r == r;
    // infinities and NaN make a product with 0 that is not 0; lanes that reach over E count too
    float probe = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) probe = fmaf(x[j], 0.f, probe);
    const bool special = e0 < E && !(probe == 0.f);
    float m = 0.f, tol0 = 0x1p-20f;
    if (softmax) {
      m = x[0];
#pragma unroll
      for (int j = 1; j < NPL; ++j) m = fmaxf(m, x[j]);
      bool nan = false;
      if (special) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) nan |= x[j] != x[j];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      if (__any_sync(FULL, nan)) m = NAN;
      if (m == -INFINITY) continue;                               // no expert is left
    }
    unsigned key[NPL];
    if (biased || GROUPED || softmax) {
      float v[NPL];
      if (softmax) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          v[j] = ex2_approx((x[j] - m) * LOG2E);
          sum += v[j];
        }
        sum = warp_sum(sum);
        const float smax = __fdividef(1.f, sum);
        if (mine_row) {
          m_l = m;
          sum_l = sum;
        }
        tol0 = smax * 0x1p-17f;
        if (biased || GROUPED) {
#pragma unroll
          for (int j = 0; j < NPL; ++j) v[j] *= smax;
        }
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) v[j] = rcp_approx(1.f + ex2_approx(x[j] * -LOG2E));
      }
      if (biased || GROUPED) {
        if (biased) {
#pragma unroll
          for (int j = 0; j < NPL; ++j) v[j] += b[j];
        }
#pragma unroll
        for (int j = 0; j < NPL; ++j) key[j] = order_key(v[j]);
        // experts without a number: masked ones (a bias may be -inf too) and NaN
        if (special || b_odd) {
#pragma unroll
          for (int j = 0; j < NPL; ++j) {
            if (v[j] != v[j]) key[j] = order_key(-FLT_MAX);
            if (x[j] == -INFINITY || (biased && b[j] == -INFINITY)) key[j] = 0;
          }
        }
      }
    }
    unsigned long long kept = ~0ull;
    if constexpr (GROUPED) {
      // two best of every group: 32 / G lanes (a power of two) walk a group in shared memory
      const int per = E / G;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (e0 + j < E) words[e0 + j] = key[j];
      __syncwarp();
      const int lanes = G > 16 ? 1 : G > 8 ? 2 : G > 4 ? 4 : G > 2 ? 8 : 16;
      unsigned gk[2];
      float mag = 0.f;                                            // bounds the roundings of v: sums may cancel
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int g = lane / lanes + 32 * half;
        unsigned b1 = 0, b2 = 0;
        if (g < G)
          for (int i = lane & (lanes - 1); i < per; i += lanes) {
            const unsigned k = words[g * per + i];
            b2 = max(b2, min(b1, k));
            b1 = max(b1, k);
          }
        for (int o = 1; o < lanes; o <<= 1) {
          const unsigned o1 = __shfl_xor_sync(FULL, b1, o), o2 = __shfl_xor_sync(FULL, b2, o);
          b2 = max(max(b2, o2), min(b1, o1));
          b1 = max(b1, o1);
        }
        const float v1 = key_value(b1), v2 = b2 ? key_value(b2) : 0.f;
        if (b1) mag = fmaxf(mag, fabsf(v1) + fabsf(v2));
        // unique keys again: the group's id in the low six bits
        gk[half] = b1 == 0 || (lane & (lanes - 1)) ? 0u : (order_key(v1 + v2) & ~63u) | (63u - g);
        if (G <= 32) {
          gk[1] = 0;
          break;
        }
      }
      mag = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(mag)));
      kept = 0;
      unsigned last = 0, best = __reduce_max_sync(FULL, max(gk[0], gk[1]));
      for (int t = 0; t < a.keep && best; ++t) {
        kept |= 1ull << (63u - (best & 63u));
        gk[0] = gk[0] == best ? 0u : gk[0];
        gk[1] = gk[1] == best ? 0u : gk[1];
        last = best;
        best = __reduce_max_sync(FULL, max(gk[0], gk[1]));
      }
      if (best) close |= mine_row && !(key_value(last & ~63u) - key_value(best | 63u) > 4.f * tol0 + 0x1p-21f * mag);
      __syncwarp();
    }
    if (!biased) {
      if (special) {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          key[j] = x[j] == -INFINITY ? 0u : order_key(x[j] != x[j] ? -FLT_MAX : x[j] + 0.f);
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) key[j] = order_key(x[j] + 0.f);        // -0 ranks as 0
      }
    }
    if constexpr (GROUPED) {
      const int g0 = (int)((e0 * per_magic) >> 20), per = E / G;
      if (per >= NPL) {                                           // a lane's experts lie in two groups at most
        const bool in0 = kept >> (g0 & 63) & 1ull, in1 = kept >> ((g0 + 1) & 63) & 1ull;
        const int edge = (g0 + 1) * per - e0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) key[j] = (j < edge ? in0 : in1) ? key[j] : 0u;
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (!(kept >> ((((e0 + j) * per_magic) >> 20) & 63u) & 1ull)) key[j] = 0;
      }
    }
    const unsigned high = e0 < E ? ~ID : 0u;
#pragma unroll
    for (int j = 0; j < NPL; ++j) key[j] = (key[j] & high) | (ID - e0 - j);
    sort_keys(key);
#pragma unroll
    for (int j = 0; j < NPL; ++j) list[j * 32] = key[j];
    list[NPL * 32] = 0;
    if (mine_row) tol_l = tol0;
  }

  // K rounds, and one more that shows the first one left out; what is left when nothing is, are bare
  // ids, and 0 behind them, which is not taken off
  unsigned at[RPW], top[RPW];
#pragma unroll
  for (int r = 0; r < RPW; ++r) {
    at[r] = r * (NPL + 1) * 32 + lane;
    top[r] = r < n_rows ? lists[at[r]] : 0u;
  }
#pragma unroll(RPW == 1 ? 4 : 2)
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
      const unsigned best = __reduce_max_sync(FULL, top[r]);
      mine_key = lane == r * SEG + k ? best : mine_key;
      at[r] += top[r] == best && best ? 32 : 0;
      top[r] = r < n_rows ? lists[at[r]] : 0u;
    }
  }
  if (!exact) {
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
      const unsigned best = __reduce_max_sync(FULL, top[r]);
      extra = mine_r == r && best > ID ? best : extra;
    }
  }

  // each lane its own choice
  const unsigned row = row0 + mine_r;
  const bool live = mine_r < n_rows && rank < K;
  h = row / (unsigned)a.S;
  s = row - h * (unsigned)a.S;
  const T* lg = static_cast<const T*>(a.logits) + h * a.stride_h + s * a.stride_s;
  const float* bias = biased ? a.bias + (int64_t)h * E : nullptr;
  int mine = mine_key > ID ? (int)(ID - (mine_key & ID)) : -1;
  float x = 0.f, p = 0.f, b_mine = 0.f;
  auto score = [&] {
    p = 0.f;
    if (mine >= 0) {
      x = mx_to_f32(lg[mine]);
      p = softmax ? __fdividef(expf(x - m_l), sum_l) : __fdividef(1.f, 1.f + expf(-x));
    }
  };
  score();
  if (!exact) {
    if (biased && mine >= 0) b_mine = bias[mine];
    const float v = biased ? p + b_mine : x;
    const float tol = biased ? tol_l + 0x1p-22f * fabsf(v) : 0.f;
    const float v1 = __shfl_down_sync(FULL, v, 1), x1 = __shfl_down_sync(FULL, x, 1), b1 = __shfl_down_sync(FULL, b_mine, 1);
    const bool next = __shfl_down_sync(FULL, mine, 1) >= 0;
    if (mine >= 0) {
      if (rank + 1 < K) {
        if (next) close |= !(v - v1 > tol) && !(x == x1 && b_mine == b1);
      } else if (extra) {
        close |= !(v - key_value(extra | ID) > tol);
      }
    }
  }
  for (unsigned again = __ballot_sync(FULL, close && live); again;) {
    const int r = (__ffs(again) - 1) / SEG;
    again &= SEG == 32 ? 0u : ~(((1u << (SEG & 31)) - 1u) << (r * SEG));
    __syncwarp();
    const unsigned rr = row0 + r, hr = rr / (unsigned)a.S;
    const int id = select_row64<T>(a, static_cast<const T*>(a.logits) + hr * a.stride_h + (rr - hr * a.S) * a.stride_s,
                                   a.bias ? a.bias + (int64_t)hr * E : nullptr, scratch, lane);
    const int got = __shfl_sync(FULL, id, rank);
    if (mine_r == r) {
      mine = got;
      score();
    }
  }
  float w = p;
  if (a.route_norm) {
    float n = p;
    #pragma unroll
    for (int o = SEG / 2; o > 0; o >>= 1) n += __shfl_xor_sync(FULL, n, o);
    // a slot without an expert weighs 0 whatever the divisor is, and so does all of a sum of 0 without an eps
    const float d = n != n ? n : fmaxf(n, a.norm_eps);
    w = mine >= 0 && d != 0.f ? __fdividef(p, d) : 0.f;
  }
  if (live) {
    const int64_t o = (int64_t)row * K + rank;
    weights[o] = w * a.route_scale;
    idx[o] = mine;
    if (saved) saved[o] = softmax ? p : x;
  }
}

// `rpw` rows a warp, seg = 32 / rpw >= K lanes a row for the chosen experts.  A row's gradient is zero
// but for the chosen ones (sigmoid, or softmax with the norm): rows are cleared with wide stores
// and the chosen entries stored over them.  The other rows (softmax where the norm does not
// cancel the common term) are written by the whole warp, dl = -score (sum ds p), and the chosen
// entries, p (ds - sum ds p), over them.  Bound by latency at the sizes of a training step: 6 to 7 us
// for 16 k rows.
template <int DT, int NPL>
__global__ void __launch_bounds__(RE_WARPS * 32)
    route_experts_bwd_kernel(const __grid_constant__ RouteArgs a, bool vec, bool vec_out, int rpw,
                             const float* __restrict__ grad_w, int64_t gs_h, int64_t gs_s,
                             const int64_t* __restrict__ idx, const float* __restrict__ saved,
                             typename MxType<DT>::T* __restrict__ dl) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rows = (unsigned)(a.H * a.S), row0 = (blockIdx.x * RE_WARPS + warp) * (unsigned)rpw;
  if (row0 >= rows) return;
  const int n_rows = (int)min((unsigned)rpw, rows - row0), seg = 32 / rpw;
  const int E = a.E, K = a.K, rank = lane % seg;
  const unsigned row = row0 + lane / seg;
  const bool live = lane / seg < n_rows && rank < K;
  const unsigned h = row / (unsigned)a.S, s = row - h * (unsigned)a.S;
  const int64_t id = live ? idx[(int64_t)row * K + rank] : -1;
  const bool has = id >= 0 && id < E;
  float p = 0.f, q = 0.f, g = 0.f;
  if (has) {
    p = saved[(int64_t)row * K + rank];
    g = grad_w[h * gs_h + s * gs_s + rank] * a.route_scale;
    if (a.score_func == 1) {
      q = __fdiv_rn(1.f, 1.f + expf(p));
      p = __fdiv_rn(1.f, 1.f + expf(-p));
    }
  }
  auto seg_sum = [&](float v) {
    for (int o = seg / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
  };
  float ds = g, unscale = 1.f;
  bool cancels = false;                                           // the softmax's common term is 0
  if (a.route_norm) {
    const float n = seg_sum(p);
    float den = n != n ? n : fmaxf(n, a.norm_eps);
    cancels = n > a.norm_eps;
    if (den < 0x1p-64f) {           // g / den alone could overflow: p and den times 2^64, ds over it
      unscale = 0x1p-64f;
      p *= 0x1p64f;
      den = den < FLT_MIN ? 0.f : den * 0x1p64f;                  // scores below FLT_MIN counted as 0
    }
    const float gp = seg_sum(g * p);
    ds = __fdiv_rn(g, den);
    if (cancels) ds = __fdiv_rn(g - __fdiv_rn(gp, den), den);
    if (den == 0.f) ds = 0.f;                                     // the weights were 0
  }
  const bool dense_row = a.score_func == 0 && !cancels;
  const float dot = seg_sum(has && dense_row ? ds * p : 0.f);
  const unsigned dense = a.score_func == 0 ? __ballot_sync(FULL, dense_row && has) : 0u;
  const unsigned sparse = __ballot_sync(FULL, live && !dense_row) | __ballot_sync(FULL, live && !has);
  T* out = dl + (int64_t)row0 * E;
  if (sparse) {
    const int64_t n = (int64_t)n_rows * E;
    constexpr int W = 16 / (int)sizeof(T);
    const int64_t wide = vec_out ? n / W : 0;
    for (int64_t i = lane; i < wide; i += 32) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
    for (int64_t i = wide * W + lane; i < n; i += 32) mx_store(out + i, 0.f);
  }
  __syncwarp();
  for (unsigned todo = dense; todo;) {
    const int r = (__ffs(todo) - 1) / seg;
    todo &= seg == 32 ? 0u : ~(((1u << seg) - 1u) << (r * seg));
    const unsigned rr = row0 + r, hr = rr / (unsigned)a.S;
    const T* lg = static_cast<const T*>(a.logits) + hr * a.stride_h + (rr - hr * a.S) * a.stride_s;
    const float row_dot = __shfl_sync(FULL, dot, r * seg);
    const int e0 = lane * NPL;
    float o[NPL];
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
    const float f = -__fdiv_rn(row_dot, warp_sum(sum));
    T* dst = out + (int64_t)r * E + e0;
    constexpr int BYTES = NPL * (int)sizeof(T);
    struct alignas(BYTES < 16 ? BYTES : 16) Chunk {
      T v[NPL];
    } c;
#pragma unroll
    for (int j = 0; j < NPL; ++j) mx_store(&c.v[j], o[j] == 0.f ? 0.f : o[j] * f);
    if (vec && e0 + NPL <= E) {
      *reinterpret_cast<Chunk*>(dst) = c;
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (e0 + j < E) dst[j] = c.v[j];
    }
  }
  __syncwarp();
  if (has) mx_store(dl + (int64_t)row * E + id, a.score_func == 1 ? ds * p * q : p * (ds - dot * unscale));
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

// Rows a warp takes, up to 4: as many as have K lanes each, while 16 warps a SM are left.
int rows_per_warp(int64_t rows, int K) {
  int rpw = 1;
  while (2 * rpw * K <= 32 && rpw < 4 && rows >= (int64_t)num_sms() * 16 * rpw * 2) rpw *= 2;
  return rpw;
}

template <int DT, int NPL, int RPW, bool GROUPED, int SCORE = -1, int BIAS = -1>
cudaError_t run_fwd(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st) {
  const int64_t rows = (int64_t)a.H * a.S;
  const unsigned grid = (unsigned)((rows + RE_WARPS * RPW - 1) / (RE_WARPS * RPW));
  const size_t smem = (size_t)RE_WARPS * fwd_scratch_bytes(a.E, NPL, RPW, GROUPED);
  auto kernel = route_experts_kernel<DT, NPL, RPW, GROUPED, SCORE, BIAS>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const bool vec = chunks_aligned(a.logits, a.stride_h, a.stride_s, a.E, DT == DT_F32 ? 4 : 2, NPL) &&
                   (!a.bias || chunks_aligned(a.bias, a.E, 0, a.E, 4, NPL));
  // e / per = e * ceil(2^20 / per) >> 20 for e < 1024
  const unsigned per = (unsigned)(a.E / a.groups), magic = ((1u << 20) + per - 1) / per;
  MHMOE_LAUNCH_PDL((route_experts_kernel<DT, NPL, RPW, GROUPED, SCORE, BIAS>), grid, RE_WARPS * 32, smem, st, a, vec,
                   magic, weights, idx, saved);
  return cudaGetLastError();
}

template <int DT, int NPL, bool GROUPED>
cudaError_t run_fwd(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st) {
  if constexpr (NPL <= 8) {
    const int rpw = rows_per_warp((int64_t)a.H * a.S, a.K);
    if (rpw == 4) {                                               // many rows: one kernel a score and bias
      if (a.score_func == 0)
        return a.bias ? run_fwd<DT, NPL, 4, GROUPED, 0, 1>(a, weights, idx, saved, st)
                      : run_fwd<DT, NPL, 4, GROUPED, 0, 0>(a, weights, idx, saved, st);
      return a.bias ? run_fwd<DT, NPL, 4, GROUPED, 1, 1>(a, weights, idx, saved, st)
                    : run_fwd<DT, NPL, 4, GROUPED, 1, 0>(a, weights, idx, saved, st);
    }
    if (rpw == 2) return run_fwd<DT, NPL, 2, GROUPED>(a, weights, idx, saved, st);
  }
  return run_fwd<DT, NPL, 1, GROUPED>(a, weights, idx, saved, st);
}

template <int DT, int NPL>
cudaError_t run_fwd(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st) {
  return a.keep < a.groups ? run_fwd<DT, NPL, true>(a, weights, idx, saved, st)
                           : run_fwd<DT, NPL, false>(a, weights, idx, saved, st);
}

template <int DT, int NPL>
cudaError_t run_bwd(const RouteArgs& a, const float* grad_w, int64_t gs_h, int64_t gs_s, const int64_t* idx,
                    const float* saved, void* dl, cudaStream_t st) {
  const int64_t rows = (int64_t)a.H * a.S;
  const int rpw = rows_per_warp(rows, a.K);
  const unsigned grid = (unsigned)((rows + RE_WARPS * rpw - 1) / (RE_WARPS * rpw));
  constexpr int esz = DT == DT_F32 ? 4 : 2;
  // dense rows: logits and gradient in the same chunks; cleared rows: 16-B stores from the warp's first
  const bool vec = a.logits && chunks_aligned(a.logits, a.stride_h, a.stride_s, a.E, esz, NPL) &&
                   chunks_aligned(dl, 0, a.E, a.E, esz, NPL);
  const bool vec_out = reinterpret_cast<uintptr_t>(dl) % 16 == 0 && (int64_t)rpw * a.E * esz % 16 == 0;
  MHMOE_LAUNCH_PDL((route_experts_bwd_kernel<DT, NPL>), grid, RE_WARPS * 32, 0, st, a, vec, vec_out, rpw, grad_w, gs_h,
                   gs_s, idx, saved, static_cast<typename MxType<DT>::T*>(dl));
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
