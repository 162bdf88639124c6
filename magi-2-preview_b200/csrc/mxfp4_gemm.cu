// Products with MXFP4 weights: y = act(Q(x) W^T + bias), dense or per expert over sorted rows.
//
// Every product of two E2M1 values and of two scales is exact in fp32, so the result is the
// fp32 sum of exact terms, plus the epilogue's roundings: one to the output's type.
#include "mxfp4.cuh"

namespace mhmoe {

namespace {

constexpr int SG_BM = 64, SG_BN = 64, SG_BK = 32;

struct SimpleArgs {
  const uint8_t* xq;
  const uint8_t* xsf;
  const uint8_t* w;
  const uint8_t* wsf;
  int n, N;
  uint32_t katoms;
  const int64_t* offsets;
  const int32_t* gather;
  int64_t R, x_rows;
  const float* row_weights;
  const float* bias;
  int act;
  int64_t y_stride;
  bool zero_tail;
  int* status;
};

__device__ __forceinline__ int64_t clip(int64_t v, int64_t hi) { return v < 0 ? 0 : (v > hi ? hi : v); }

// 64 x 64 outputs per CTA, 256 threads of 4 x 4, one scale block of K at a time.
template <int DT>
__global__ void __launch_bounds__(256) mx_product_simple_kernel(const SimpleArgs p, typename MxType<DT>::T* y) {
  pdl_wait();
  pdl_trigger();
  __shared__ float xs[SG_BK][SG_BM + 1], ws[SG_BK][SG_BN + 1];
  const int n0 = blockIdx.x * SG_BN;
  const int64_t t = blockIdx.y;
  int e = 0;
  int64_t row0 = t * SG_BM, row1 = p.R;
  if (p.offsets) {
    int lo = 0, hi = p.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (clip(p.offsets[mid], p.R) / SG_BM + mid <= t) lo = mid;
      else hi = mid - 1;
    }
    e = lo;
    const int64_t a = clip(p.offsets[e], p.R);
    row1 = clip(p.offsets[e + 1], p.R);
    row0 = a + (t - (a / SG_BM + e)) * SG_BM;
    if (t == 0 && blockIdx.x == 0) {
      for (int i = threadIdx.x; i <= p.n; i += 256) {
        const int64_t o = p.offsets[i];
        if (o < 0 || o > p.R || (i > 0 && o < p.offsets[i - 1])) record_error(p.status, MHMOE_ERR_ARGS);
      }
    }
    if (p.zero_tail && t == 0) {
      const int cols = p.act ? p.N / 2 : p.N, c0 = p.act ? n0 / 2 : n0, nc = min(p.act ? SG_BN / 2 : SG_BN, cols - c0);
      for (int64_t r = clip(p.offsets[p.n], p.R); r < p.R; ++r)
        for (int c = threadIdx.x; c < nc; c += 256) mx_store(y + r * p.y_stride + c0 + c, 0.f);
    }
  }
  if (row0 >= row1) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (uint32_t kb = 0; kb < p.katoms * 4; ++kb) {
    for (int i = threadIdx.x; i < 2 * 64 * 4; i += 256) {
      const int which = i >> 8, r = (i >> 2) & 63, q = i & 3;
      float v[8] = {};
      if (which == 0) {
        const int64_t row = row0 + r;
        int64_t src = row;
        bool ok = row < row1;
        if (ok && p.gather) {
          src = p.gather[row];
          ok = src >= 0 && src < p.x_rows;
          if (!ok && kb == 0) record_error(p.status, MHMOE_ERR_ARGS);
        }
        if (ok) {
          mx_decode8(*reinterpret_cast<const uint32_t*>(p.xq + src * p.katoms * 64 + kb * 16 + q * 4), v);
          const float s = mx_scale_value(p.xsf[mx_sf_offset(src, kb, p.katoms)]);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= s;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) xs[q * 8 + j][r] = v[j];
      } else {
        const int64_t row = n0 + r;
        if (row < p.N) {
          const uint64_t base = (uint64_t)e * ((p.N + 127) / 128) * p.katoms * 512;
          mx_decode8(*reinterpret_cast<const uint32_t*>(p.w + ((int64_t)e * p.N + row) * p.katoms * 64 + kb * 16 + q * 4), v);
          const float s = mx_scale_value(p.wsf[base + mx_sf_offset(row, kb, p.katoms)]);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= s;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ws[q * 8 + j][r] = v[j];
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < SG_BK; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = xs[k][ty * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = ws[k][tx * 4 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + ty * 4 + i;
    if (row >= row1) break;
    const float rw = p.row_weights ? p.row_weights[row] : 1.f;
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = n0 + tx * 4 + j;
      o[j] = acc[i][j] + (p.bias && c < p.N ? p.bias[(int64_t)e * p.N + c] : 0.f);
    }
    if (p.act) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = (n0 + tx * 4) / 2 + j;
        if (2 * c < p.N) mx_store(y + row * p.y_stride + c, mx_swiglu7(o[2 * j], o[2 * j + 1]) * rw);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = n0 + tx * 4 + j;
        if (c < p.N) mx_store(y + row * p.y_stride + c, o[j] * rw);
      }
    }
  }
}

}  // namespace

size_t mx_product_workspace_bytes(int64_t x_rows, int64_t R, int n, int N, int cols, bool grouped) {
  const int64_t katoms = mx_padded_cols(cols) / 128;
  return (size_t)((x_rows * katoms * 64 + 255) / 256 * 256 + (x_rows + 127) / 128 * katoms * 512);
}

int mx_product(const MxProduct& p, void* workspace, cudaStream_t st, cudaError_t* cerr) {
  const int64_t katoms = mx_padded_cols(p.cols) / 128;
  const uint8_t* xq = p.xq;
  const uint8_t* xsf = p.xsf;
  if (!xq) {
    uint8_t* d = static_cast<uint8_t*>(workspace);
    uint8_t* s = d + (p.x_rows * katoms * 64 + 255) / 256 * 256;
    *cerr = launch_mx_quantize(p.x, p.x_dtype, 0, p.x_stride, 1, p.x_rows, p.cols, p.ceil, d, s, st);
    if (*cerr != cudaSuccess) return MHMOE_ERR_LAUNCH;
    xq = d;
    xsf = s;
  }
  SimpleArgs a{xq, xsf, p.w_data, p.w_sf, p.n, p.N, (uint32_t)katoms, p.offsets, p.gather_ids, p.R, p.x_rows,
               p.row_weights, p.bias, p.act, p.y_stride, p.zero_tail, p.status};
  const int64_t slots = p.offsets ? p.R / SG_BM + p.n : (p.R + SG_BM - 1) / SG_BM;
  const dim3 grid((p.N + SG_BN - 1) / SG_BN, (unsigned)slots);
  if (p.y_dtype == DT_F32)
    *cerr = launch_pdl(mx_product_simple_kernel<DT_F32>, grid, dim3(256), 0, st, a, static_cast<float*>(p.y));
  else if (p.y_dtype == DT_BF16)
    *cerr = launch_pdl(mx_product_simple_kernel<DT_BF16>, grid, dim3(256), 0, st, a, static_cast<__nv_bfloat16*>(p.y));
  else
    *cerr = launch_pdl(mx_product_simple_kernel<DT_F16>, grid, dim3(256), 0, st, a, static_cast<__half*>(p.y));
  return *cerr == cudaSuccess ? MHMOE_OK : MHMOE_ERR_LAUNCH;
}

}  // namespace mhmoe
