// MXFP4 quantisation and its inverse.
//
// quantise: per row and per 32 columns, a = max |x|, e from mx_scale_byte, values
// E2M1(x * 2^-e) rounded to nearest even and saturated at 6.  x * 2^-e is exact in fp32 (a power
// of two; results below the E2M1 range round to 0 either way), so the codes are the
// definition's for every input type.
//
// Both kernels are bound by HBM: 2 or 4 bytes an element one way, 17/32 of a byte the other.
// 268 M elements (n = 16): fp32 quantised in 170 us (7.1 TB/s, codes partly still in L2), to bf16 in
// 124 us (5.5 TB/s).  A few tokens are bound by the launch: 3.3 and 3.5 us.
#include "mxfp4.cuh"

namespace mhmoe {

constexpr int MXQ_THREADS = 256;

// Eight threads take one atom column (128 columns of a row), 16 columns each: 8 B of codes a
// thread, one 4-B word of scales from four shuffled bytes (a scale needs two threads' maxima).  Items are (matrix, row, atom column) with the rows of each
// matrix counted to a multiple of 128, so that every scale byte is written.
template <int DT>
__global__ void __launch_bounds__(MXQ_THREADS)
    mx_quantize_kernel(const typename MxType<DT>::T* __restrict__ x, int64_t stride_n, int64_t stride_row,
                       uint32_t rows, uint32_t cols, FastDiv katoms, FastDiv rows_p, uint32_t items, bool ceil,
                       bool vec_ok, uint8_t* __restrict__ data, uint8_t* __restrict__ sf) {
  pdl_wait();
  pdl_trigger();
  const int sub = threadIdx.x & 7;
  const uint32_t mask = 0xffu << (threadIdx.x & 24);
  for (uint32_t it = blockIdx.x * (MXQ_THREADS / 8) + (threadIdx.x >> 3); it < items;
       it += gridDim.x * (MXQ_THREADS / 8)) {
    const uint32_t rr = katoms.div(it), ka = it - rr * katoms.d;
    const uint32_t b = rows_p.div(rr), row = rr - b * rows_p.d;
    const uint32_t c0 = ka * 128 + sub * 16;
    MxRaw16<typename MxType<DT>::T> v;
    const bool live = row < rows && c0 < cols;
    v.load(x + b * stride_n + row * stride_row + c0, live && vec_ok && c0 + 16 <= cols,
           live ? (int)min(16u, cols - c0) : 0);
    uint2 code;
    const uint32_t sw = mx_quantize16(v, ceil, sub, mask, code);
    if (row < rows)
      *reinterpret_cast<uint2*>(data + ((uint64_t)b * rows + row) * katoms.d * 64 + ka * 64 + sub * 8) = code;
    if (sub == 0)
      *reinterpret_cast<uint32_t*>(sf + (uint64_t)b * (rows_p.d >> 7) * katoms.d * 512 +
                                   mx_sf_offset(row, ka * 4, katoms.d)) = sw;
  }
}

// Sixteen threads take one atom column, 8 columns each (a 16-B store in a 2-byte type), and MXD_UN
// items a grid apart, so that as many loads of 5 B are in flight a thread (268 M elements to bf16:
// 138 us with one, 4.9 TB/s, 124 with four).
constexpr int MXD_UN = 4;
template <int DT>
__global__ void __launch_bounds__(MXQ_THREADS)
    mx_dequantize_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ sf, FastDiv rows,
                         uint32_t rows_p, uint32_t cols, FastDiv katoms, uint32_t items, bool vec_ok,
                         typename MxType<DT>::T* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  using T = typename MxType<DT>::T;
  const int sub = threadIdx.x & 15;
  const uint32_t hop = gridDim.x * (MXQ_THREADS / 16);
  for (uint32_t it0 = blockIdx.x * (MXQ_THREADS / 16) + (threadIdx.x >> 4); it0 < items; it0 += hop * MXD_UN) {
    uint32_t w[MXD_UN], sb[MXD_UN], c0[MXD_UN];
    T* o[MXD_UN];
#pragma unroll
    for (int u = 0; u < MXD_UN; ++u) {
      const uint32_t it = it0 + u * hop;
      const uint32_t rr = katoms.div(it), ka = it - rr * katoms.d;
      const uint32_t b = rows.div(rr), row = rr - b * rows.d;
      c0[u] = it < items ? ka * 128 + sub * 8 : cols;
      o[u] = out + (uint64_t)rr * cols + c0[u];
      w[u] = 0;
      sb[u] = 0;
      if (c0[u] < cols) {
        w[u] = __ldg(reinterpret_cast<const uint32_t*>(data + (uint64_t)it * 64 + sub * 4));
        sb[u] = __ldg(sf + (uint64_t)b * (rows_p >> 7) * katoms.d * 512 +
                      mx_sf_offset(row, ka * 4 + (sub >> 2), katoms.d));
      }
    }
#pragma unroll
    for (int u = 0; u < MXD_UN; ++u) {
      if (c0[u] >= cols) continue;
      const float s = mx_scale_value(sb[u]);
      float v[8];
      mx_decode8(w[u], v);
      if (vec_ok && c0[u] + 8 <= cols) {
        __align__(16) T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx_store(&t[i], v[i] * s);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
          reinterpret_cast<uint4*>(o[u])[i] = reinterpret_cast<const uint4*>(t)[i];
      } else {
        for (uint32_t i = 0; i < min(8u, cols - c0[u]); ++i) mx_store(o[u] + i, v[i] * s);
      }
    }
  }
}

// Blocks of `per_block` items each, at most 16 rounds of 8 resident blocks a SM.
static unsigned mx_grid(int64_t items, int per_block) {
  return (unsigned)std::min<int64_t>((items + per_block - 1) / per_block, (int64_t)num_sms() * 128);
}

cudaError_t launch_mx_quantize(const void* x, int dtype, int64_t stride_n, int64_t stride_row, int64_t n,
                               int64_t rows, int64_t cols, bool ceil, uint8_t* data, uint8_t* sf, cudaStream_t st) {
  const int64_t rows_p = (rows + 127) / 128 * 128, katoms = mx_padded_cols(cols) / 128;
  const int64_t items = n * rows_p * katoms;
  if (items == 0) return cudaSuccess;
  if (items >= (int64_t)1 << 31) return cudaErrorInvalidValue;      // above 2^38 elements
  const int64_t esz = dtype == DT_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && stride_n * esz % 16 == 0 && stride_row * esz % 16 == 0;
  const unsigned grid = mx_grid(items, MXQ_THREADS / 8);
#define MX_Q(DT)                                                                                                 \
  MHMOE_LAUNCH_PDL(mx_quantize_kernel<DT>, grid, MXQ_THREADS, 0, st, static_cast<const MxType<DT>::T*>(x),       \
                   stride_n, stride_row, (uint32_t)rows, (uint32_t)cols, FastDiv((uint32_t)katoms),              \
                   FastDiv((uint32_t)rows_p), (uint32_t)items, ceil, vec, data, sf)
  if (dtype == DT_F32) MX_Q(DT_F32);
  else if (dtype == DT_BF16) MX_Q(DT_BF16);
  else MX_Q(DT_F16);
#undef MX_Q
  return cudaGetLastError();
}

cudaError_t launch_mx_dequantize(const uint8_t* data, const uint8_t* sf, int64_t n, int64_t rows, int64_t cols,
                                 int dtype, void* out, cudaStream_t st) {
  const int64_t rows_p = (rows + 127) / 128 * 128, katoms = mx_padded_cols(cols) / 128;
  const int64_t items = n * rows * katoms;
  if (items == 0) return cudaSuccess;
  if (items >= (int64_t)1 << 30) return cudaErrorInvalidValue;      // above 2^37 elements (an item number stays below 2^31)
  const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && cols * (dtype == DT_F32 ? 4 : 2) % 16 == 0;
  const unsigned grid = mx_grid(items, MXQ_THREADS / 16 * MXD_UN);
#define MX_D(DT)                                                                                                 \
  MHMOE_LAUNCH_PDL(mx_dequantize_kernel<DT>, grid, MXQ_THREADS, 0, st, data, sf, FastDiv((uint32_t)rows),        \
                   (uint32_t)rows_p, (uint32_t)cols, FastDiv((uint32_t)katoms), (uint32_t)items, vec,            \
                   static_cast<MxType<DT>::T*>(out))
  if (dtype == DT_F32) MX_D(DT_F32);
  else if (dtype == DT_BF16) MX_D(DT_BF16);
  else MX_D(DT_F16);
#undef MX_D
  return cudaGetLastError();
}

}  // namespace mhmoe
