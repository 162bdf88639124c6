// MXFP4 helpers: E2M1 values with one power-of-two E8M0 scale per 32 elements along K.
//
// A matrix [rows, cols] is held as packed bytes [rows, cols_p/2] (low nibble = even column)
// and scale bytes in 512-byte atoms of 128 rows x 128 columns (4 scales a row): scale
// (row, block c) sits in atom (row/128) * (cols_p/128) + c/4 at byte (row%32)*16 +
// (row%128/32)*4 + c%4, the layout the block-scaled tensor-core instructions read.  cols_p is
// cols rounded up to 128; the columns behind cols hold zeros with scale byte 0.  A scale byte b
// stands for 2^(b-127), 255 for NaN.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "kernels.cuh"

namespace mhmoe {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

constexpr int MX_BLOCK = 32;

__host__ __device__ constexpr int64_t mx_padded_cols(int64_t cols) { return (cols + 127) / 128 * 128; }

__host__ __device__ __forceinline__ uint64_t mx_sf_offset(uint64_t row, uint32_t c, uint32_t katoms) {
  const uint32_t m = (uint32_t)(row & 127u);
  return ((row >> 7) * katoms + (c >> 2)) * 512u + (m & 31u) * 16u + (m >> 5) * 4u + (c & 3u);
}

template <int DT>
struct MxType;
template <>
struct MxType<DT_F32> {
  using T = float;
};
template <>
struct MxType<DT_BF16> {
  using T = __nv_bfloat16;
};
template <>
struct MxType<DT_F16> {
  using T = __half;
};

__device__ __forceinline__ float mx_to_f32(float v) { return v; }
__device__ __forceinline__ float mx_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float mx_to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void mx_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void mx_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void mx_store(__half* p, float v) { *p = __float2half_rn(v); }

// Sixteen consecutive elements as raw words (fp32: one a word, else two).  vec: p is 16-B aligned
// and all sixteen exist; otherwise the first `avail` are read and the rest are zero.
template <typename T>
struct MxRaw16 {
  static constexpr int WORDS = 16 * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p, bool vec, int avail) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = 0;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < avail) w[i] = __float_as_uint(reinterpret_cast<const float*>(p)[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < avail) w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
      }
    }
  }
  // fp32 bits of the largest magnitude (NaN above infinity): magnitudes order like their bits
  __device__ __forceinline__ uint32_t amax_bits() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t a = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) a = max(a, w[i] & 0x7fffffffu);
      return a;
    } else {
      uint32_t a = 0;
#pragma unroll
      for (int i = 0; i < 8; i += 2) a = __vimax3_u16x2(a, w[i] & 0x7fff7fffu, w[i + 1] & 0x7fff7fffu);
      a = max(a & 0xffffu, a >> 16);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return a << 16;
      else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)a)));
    }
  }
  __device__ __forceinline__ void values(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
};

// Scale byte of a block whose largest magnitude has the fp32 bits `abits` (sign cleared):
// floor: 2^floor(log2 amax) / 4, ceil: the smallest power of two s with amax <= 6 s.  The
// exponent field gives floor(log2) + 127 (0 for subnormals, whose scale is the smallest), and
// amax > 1.5 * 2^floor(log2) is mantissa > 0.5.  NaN or Inf anywhere makes the block NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t abits, bool ceil) {
  if (abits >= 0x7f800000u) return 255u;
  const int f = (int)(abits >> 23);
  const int b = f - 2 + (ceil && (abits & 0x7fffffu) > 0x400000u ? 1 : 0);
  return (uint32_t)max(b, 0);
}

// 2^(127 - b), the exact factor that takes a block's values to the E2M1 grid (b <= 253).
__device__ __forceinline__ float mx_inv_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// 2^(b - 127); 255 gives NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t b) {
  if (b == 0) return __uint_as_float(0x00400000u);
  return __uint_as_float(b == 255u ? 0x7fc00000u : b << 23);
}

// Quantise a thread's 16 elements: two neighbouring threads hold a block of 32, eight (sub = 0..7,
// all in `mask`) an atom column of 128.  code: the 16 packed values; returns the atom column's
// four scale bytes, the same word in all eight.
template <typename T>
__device__ __forceinline__ uint32_t mx_quantize16(const MxRaw16<T>& x, bool ceil, int sub, uint32_t mask,
                                                  uint2& code) {
  uint32_t a = x.amax_bits();
  a = max(a, __shfl_xor_sync(mask, a, 1));
  const uint32_t s = mx_scale_byte(a, ceil);
  const float f = s == 255u ? 0.f : mx_inv_scale(s);
  float v[16];
  x.values(v);
  const uint64_t f2 = f2_pack(f, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f2_unpack(f2_mul(f2_pack(v[2 * i], v[2 * i + 1]), f2), v[2 * i], v[2 * i + 1]);
  code.x = cvt_e2m1x8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
  code.y = cvt_e2m1x8(v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]);
  if (s == 255u) code = make_uint2(0, 0);
  uint32_t sw = s << (8 * (sub >> 1));
  sw |= __shfl_xor_sync(mask, sw, 2);
  sw |= __shfl_xor_sync(mask, sw, 4);
  return sw;
}

// Division by a fixed d >= 1 of numbers below 2^31: (mulhi(n, mul) + n) >> shift with
// 2^shift >= d and mul = floor(2^32 (2^shift - d) / d) + 1 (Granlund and Montgomery 1994).
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(uint32_t d_) : d(d_), mul(0), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// Eight E2M1 values of a packed word (nibble i = value i) as fp32.
__device__ __forceinline__ void mx_decode8(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// SwiGLU7: min(g, 7) * sigmoid(1.702 min(g, 7)) * (clamp(u, -7, 7) + 1); NaN goes through.  2^x and
// 1/x are the special-function unit's, each off by two units of 2^-23 at most; where they flush
// to 0 or overflow, |g sigmoid| is below 2^-100.
__device__ __forceinline__ float mx_min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float mx_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float mx_swiglu7(float g, float u) {
  g = mx_min_nan(g, 7.f);
  u = mx_max_nan(mx_min_nan(u, 7.f), -7.f);
  return g * rcp_approx(1.f + ex2_approx(g * (-1.702f * 1.44269504f))) * (u + 1.f);
}

// mxfp4.cu
cudaError_t launch_mx_quantize(const void* x, int dtype, int64_t stride_n, int64_t stride_row, int64_t n,
                               int64_t rows, int64_t cols, bool ceil, uint8_t* data, uint8_t* sf, cudaStream_t st);
cudaError_t launch_mx_dequantize(const uint8_t* data, const uint8_t* sf, int64_t n, int64_t rows, int64_t cols,
                                 int dtype, void* out, cudaStream_t st);

// mxfp4_gemm.cu
struct MxProduct {
  const void* x;              // activations [x_rows, cols], or null with xq / xsf
  int x_dtype;
  int64_t x_stride, x_rows;
  bool ceil;
  const uint8_t* xq;          // activations already in MXFP4
  const uint8_t* xsf;
  const uint8_t* w_data;      // n matrices [N, cols]
  const uint8_t* w_sf;
  int n, N, cols;
  const int64_t* offsets;     // null: dense (n == 1, R == x_rows)
  const int32_t* gather_ids;
  int64_t R;
  const float* row_weights;
  const float* bias;          // [n, N] or null
  int act;                    // 0 none, 1 swiglu7
  void* y;
  int y_dtype;
  int64_t y_stride;
  bool zero_tail;             // clear the rows behind the last expert's
  int* status;
  uint64_t timeout_ns;
};
size_t mx_product_workspace_bytes(int64_t x_rows, int64_t R, int n, int N, int cols, bool grouped);
int mx_product(const MxProduct& p, void* workspace, cudaStream_t st, cudaError_t* cerr);

// route_experts.cu
struct RouteArgs {
  const void* logits;
  int dtype;
  int64_t stride_h, stride_s;
  const float* bias;
  const uint8_t* token_mask;
  int64_t mask_stride_h;
  int H, S, E, K, score_func, groups, keep, route_norm;
  float norm_eps, route_scale;
};
cudaError_t launch_route_experts(const RouteArgs& a, float* weights, int64_t* idx, float* saved, cudaStream_t st);
cudaError_t launch_route_experts_bwd(const RouteArgs& a, const float* grad_w, int64_t grad_stride_h,
                                     int64_t grad_stride_s, const int64_t* idx, const float* saved, void* grad_logits,
                                     cudaStream_t st);

}  // namespace mhmoe
