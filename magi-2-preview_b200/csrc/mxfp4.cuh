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

// Eight consecutive elements as fp32; vec: p is 16-B aligned and all eight exist, otherwise
// only the first `avail` are read and the rest are zero.
__device__ __forceinline__ void mx_load8(const float* p, bool vec, int avail, float (&v)[8]) {
  if (vec) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < avail ? p[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void mx_load8(const T* p, bool vec, int avail, float (&v)[8]) {
  if (vec) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx_to_f32(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < avail ? mx_to_f32(p[i]) : 0.f;
  }
}

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

// Quantise the 8 values of a thread: four neighbouring threads hold a block of 32, sixteen (sub =
// 0..15, all in `mask`) an atom column of 128.  Returns the packed codes; sw is the atom
// column's four scale bytes, the same word in all sixteen.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&v)[8], bool ceil, int sub, uint32_t mask, uint32_t& sw) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
  a = max(a, __shfl_xor_sync(mask, a, 1));
  a = max(a, __shfl_xor_sync(mask, a, 2));
  const uint32_t s = mx_scale_byte(a, ceil);
  uint32_t w = 0;
  if (s != 255u) {
    const float f = mx_inv_scale(s);
    w = cvt_e2m1x8(v[0] * f, v[1] * f, v[2] * f, v[3] * f, v[4] * f, v[5] * f, v[6] * f, v[7] * f);
  }
  sw = s << (8 * (sub >> 2));
  sw |= __shfl_xor_sync(mask, sw, 4);
  sw |= __shfl_xor_sync(mask, sw, 8);
  return w;
}

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

// SwiGLU7: min(g, 7) * sigmoid(1.702 min(g, 7)) * (clamp(u, -7, 7) + 1); NaN goes through.
__device__ __forceinline__ float mx_swiglu7(float g, float u) {
  g = g > 7.f ? 7.f : g;
  u = u > 7.f ? 7.f : (u < -7.f ? -7.f : u);
  return __fdividef(g, 1.f + __expf(-1.702f * g)) * (u + 1.f);
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
