// Products with MXFP4 weights: y = act(Q(x) W^T + bias), dense or per expert over sorted rows.
//
// Every product of two E2M1 values and of two scales is exact in fp32, so the result is the
// fp32 sum of exact terms, plus the epilogue's roundings: one to the output's type.
//
// Two launches.  The first quantises the activations (mx_quantize_kernel, or mx_group_kernel
// for expert rows: gather, quantise, scale atoms per token tile, and in one extra block the list
// of token tiles).  The second, mx_gemm_kernel, multiplies on the tensor cores
// (tcgen05.mma kind::mxf4, fp32 accumulators in TMEM).
//
// A work item is (token tile, weight tile), in one of two kernels:
//   wide   128 tokens x 256 weight rows: the most math per operand byte
//   flat   128 weight rows x 16..128 tokens: with a few tokens the instruction's 128 lanes are
//          filled by the weights, which is what a decode step streams.  A cluster may share an
//          item along the columns.
// Warp roles: 0 TMA producer, 1 TMEM owner and issuer of the scale copies into TMEM and the MMAs (the
// tensor pipe keeps their order; a warp of its own for the copies, as the NVFP4 kernel has for its
// twice as many, measured 2 % slower here), then the epilogue warps.
#include "mxfp4.cuh"

namespace mhmoe {

namespace {

constexpr int MG_BM = 128;                  // rows of operand A a CTA
constexpr int MG_BK = 256;                  // columns of a stage: 128 B a row
constexpr int MG_A_BYTES = MG_BM * MG_BK / 2;
constexpr int MG_SF_BYTES = 2 * 512;        // scales of 128 rows x 256 columns: two atoms
constexpr int MG_STG_WIDE = 32, MG_STG_FLAT = 64;   // bytes of a row of an epilogue warp's store staging, 32 rows
constexpr int MG_MISC_BYTES = 512;          // barriers, TMEM slot
constexpr int MG_TMEM_COLS = 512;

struct WideShape {
  static constexpr int SLOT = 128, BN = 256;                    // tokens and weight rows of a tile
  static constexpr int B_BYTES = BN * MG_BK / 2;
  static constexpr int STAGE = MG_A_BYTES + B_BYTES + 3 * MG_SF_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int EPW = 16;                                // epilogue warps: 64 columns each
  static constexpr int THREADS = 32 * (2 + EPW);
  static constexpr int SMEM = STAGES * STAGE + EPW * 32 * MG_STG_WIDE + MG_MISC_BYTES + 1024;
  static constexpr int SF_COLS = 24, SF_COL0 = 256;             // TMEM: accumulator, then the stages' scales
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(SF_COL0 + STAGES * SF_COLS <= MG_TMEM_COLS, "TMEM");
};

template <int BN>
struct FlatShape {
  static constexpr int SLOT = BN;                               // tokens of a tile
  static constexpr int B_BYTES = BN * MG_BK / 2;
  static constexpr int STAGE = MG_A_BYTES + B_BYTES + 2 * MG_SF_BYTES;
  static constexpr int EPW = BN >= 64 ? 8 : 4;
  static constexpr int STAGES = BN <= 16 ? 9 : BN <= 32 ? 8 : BN <= 64 ? 7 : 5;
  static constexpr int THREADS = 32 * (2 + EPW);
  static constexpr int SMEM = STAGES * STAGE + EPW * 32 * MG_STG_FLAT + MG_MISC_BYTES + 1024;
  static constexpr int NACC = 2;                                // accumulators in TMEM
  static constexpr int SF_COLS = 16, SF_COL0 = NACC * BN;
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(SF_COL0 + STAGES * SF_COLS <= MG_TMEM_COLS, "TMEM");
};

struct MgParams {
  const void* x;              // rows that the flat kernel quantises itself
  int64_t x_stride;
  int cols;
  bool ceil, x_vec;
  const uint8_t* sf_tok;      // scale atoms of the token tiles, a 128-row block per slot
  const uint8_t* sf_w;
  const int4* tiles;          // grouped: {expert, first row, rows, slot}; null: dense
  const int* n_tiles;         // grouped: their number (device)
  int max_tiles;
  int64_t R;
  int N, n_wt;
  uint32_t katoms;
  const float* row_weights;
  const float* bias;
  int act;
  void* y;
  int y_dtype;
  int64_t y_stride;
  bool y_vec, y_vec32;        // 16-B, 32-B stores are possible
  int* status;
  uint64_t timeout_ns;
};

struct MgTile {
  int e, rows;
  int64_t row0, slot;
};

// A tile's entry is fetched a tile ahead and taken apart only when it is used, so that nothing waits
// for the load in between.
__device__ __forceinline__ int4 mg_fetch(const MgParams& p, int tt) {
  return p.tiles ? __ldg(p.tiles + tt) : make_int4(0, 0, tt, 0);
}
template <int SLOT>
__device__ __forceinline__ MgTile mg_tile(const MgParams& p, const int4& v) {
  MgTile t;
  if (p.tiles) {
    t.e = v.x;
    t.row0 = v.y;
    t.rows = v.z;
    t.slot = v.w;
  } else {
    t.e = 0;
    t.row0 = (int64_t)v.z * SLOT;
    t.rows = (int)min((int64_t)SLOT, p.R - t.row0);
    t.slot = v.z;
  }
  return t;
}

// Bounded wait of one role.  A role that gives up tells the others of its CTA through `gave_up` in shared
// memory and the host through the status word.  What that word held before ends no wait: it is kept
// from call to call, and an earlier launch's error is not this one's.
__device__ __forceinline__ bool mg_wait(uint32_t bar, uint32_t parity, uint32_t gave_up, int* status,
                                        uint64_t timeout_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      int left;
      asm volatile("ld.volatile.shared::cta.s32 %0, [%1];" : "=r"(left) : "r"(gave_up) : "memory");
      if (left) return false;
      if (globaltimer_ns() - t0 > timeout_ns) {
        asm volatile("st.volatile.shared::cta.s32 [%0], %1;" ::"r"(gave_up), "r"(1) : "memory");
        record_gave_up(status, MHMOE_ERR_TIMEOUT);
        return false;
      }
    }
  }
}

template <int OUT>
__device__ __forceinline__ uint32_t mg_pack16(float a, float b) {
  if constexpr (OUT == DT_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ void mg_store(void* y, int dtype, int64_t at, float v) {
  if (dtype == DT_F32) static_cast<float*>(y)[at] = v;
  else if (dtype == DT_BF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(y)[at] = __float2half_rn(v);
}

// Byte offset of 16-B chunk k of a staging row of ROWB bytes, so that eight threads' chunks (the same
// k of eight rows, or all of neighbouring rows) lie in different banks.
template <int ROWB>
__device__ __forceinline__ int mg_stg(int row, int k) {
  return row * ROWB + ((k ^ (ROWB == 32 ? (row >> 2) & 1 : (row >> 1) & 3)) << 4);
}

// 32 rows x ROWB bytes of the warp's staging to the rows row0 + 0.. of y, `rows` of them, from output
// column c0; `width` outputs a row are valid.
template <int ESZ, int ROWB>
__device__ __forceinline__ void mg_store_rows(const MgParams& p, const uint8_t* stg, int64_t row0, int rows, int c0,
                                              int width, int lane) {
  uint8_t* y = static_cast<uint8_t*>(p.y);
  constexpr int K = ROWB / 16, P16 = 16 / ESZ;
  if (p.y_vec) {
    const int k = lane % K;
    uint8_t* dst = y + ((row0 + lane / K) * p.y_stride + c0 + k * P16) * ESZ;
    const int64_t hop = (int64_t)(32 / K) * p.y_stride * ESZ;
#pragma unroll
    for (int i = 0; i < K; ++i, dst += hop) {
      const int row = i * (32 / K) + lane / K;
      if (row < rows && k * P16 < width)
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(stg + mg_stg<ROWB>(row, k));
    }
  } else {
    constexpr int PER = ROWB / ESZ;                 // one output a lane
    const int col = lane % PER;
    for (int row = lane / PER; row < rows; row += 32 / PER) {
      if (col >= width) break;
      const uint8_t* src = stg + mg_stg<ROWB>(row, col * ESZ >> 4) + (col * ESZ & 15);
      uint8_t* dst = y + ((row0 + row) * p.y_stride + c0 + col) * ESZ;
      if constexpr (ESZ == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
      else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
    }
  }
}

// Wide epilogue: 32 token rows (one a thread) x 64 accumulator columns from weight row col0.  A thread
// stores its row's outputs as whole sectors of 32 B, or, where y's rows do not start on those, through
// the staging.
template <int OUT, bool SWIGLU>
__device__ __forceinline__ void mg_wide_epilogue(const MgParams& p, const MgTile& t, uint32_t (&r)[64], int col0,
                                                 int m0, int lane, uint8_t* stg) {
  constexpr int ESZ = OUT == DT_F32 ? 4 : 2;
  constexpr int PER = 32 / ESZ;                     // outputs of a sector, or of a staging row
  constexpr int ACC = SWIGLU ? 2 * PER : PER;       // accumulator columns behind them
  static_assert(MG_STG_WIDE == 32, "a sector a row");
  const int n_out = SWIGLU ? p.N / 2 : p.N;
  if (p.bias) {
    const float* bias = p.bias + (int64_t)t.e * p.N + col0;
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (col0 + i < p.N) r[i] = __float_as_uint(__uint_as_float(r[i]) + __ldg(bias + i));
  }
  const bool live = m0 + lane < t.rows;
  float rw = 1.f;
  if (p.row_weights && live) rw = __ldg(p.row_weights + t.row0 + m0 + lane);
  const int o0 = SWIGLU ? col0 / 2 : col0;
  uint8_t* dst = static_cast<uint8_t*>(p.y) + ((t.row0 + m0 + lane) * p.y_stride + o0) * ESZ;
#pragma unroll
  for (int c = 0; c < 64 / ACC; ++c) {
    float v[PER];
    const uint32_t* rc = r + c * ACC;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if constexpr (SWIGLU) v[i] = mx_swiglu7(__uint_as_float(rc[2 * i]), __uint_as_float(rc[2 * i + 1]));
      else v[i] = __uint_as_float(rc[i]);
    }
    if (p.row_weights) {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] *= rw;
    }
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (OUT == DT_F32) w[j] = __float_as_uint(v[j]);
      else w[j] = mg_pack16<OUT>(v[2 * j], v[2 * j + 1]);
    }
    if (p.y_vec32) {
      if (live && o0 + c * PER < n_out) st_global_32(dst + c * 32, w);
    } else {
      __syncwarp();                                 // the chunk before has left the staging
      *reinterpret_cast<uint4*>(stg + mg_stg<MG_STG_WIDE>(lane, 0)) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(stg + mg_stg<MG_STG_WIDE>(lane, 1)) = make_uint4(w[4], w[5], w[6], w[7]);
      __syncwarp();
      mg_store_rows<ESZ, MG_STG_WIDE>(p, stg, t.row0 + m0, min(32, t.rows - m0), o0 + c * PER, n_out - o0 - c * PER,
                                      lane);
    }
  }
}

// Flat epilogue: one weight row n a thread (32 of the warp's from n0) x NC token columns from j0.
// The transposed outputs go through the staging in passes of 64 B a token row.
template <int NC, int OUT>
__device__ __forceinline__ void mg_flat_epilogue(const MgParams& p, const MgTile& t, const uint32_t (&r)[NC], int j0,
                                                 int n0, float b, int lane, uint8_t* stg) {
  using U = typename std::conditional<OUT == DT_F32, float, uint16_t>::type;
  constexpr int ESZ = OUT == DT_F32 ? 4 : 2, PER = MG_STG_FLAT / ESZ;
  const int rows = min(NC, t.rows - j0);
  // a row's weight, from the lane that holds it
  float rw = 1.f;
  if (p.row_weights && lane < rows) rw = __ldg(p.row_weights + t.row0 + j0 + lane);
  float v[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    v[j] = __uint_as_float(r[j]) + b;
    if (p.act) v[j] = mx_swiglu7(v[j], __shfl_down_sync(0xffffffffu, v[j], 1));     // even lanes: (gate, up)
    if (p.row_weights) v[j] *= __shfl_sync(0xffffffffu, rw, j);
  }
  const int n_out = p.act ? p.N / 2 : p.N, o0 = p.act ? n0 / 2 : n0;
  const int width = p.act ? 16 : 32;                // outputs of the warp a token row
#pragma unroll
  for (int c = 0; c < 32 / PER; ++c) {              // fp32 without activation: two passes of 16 outputs
    if (c * PER >= width) break;
    const int at = (p.act ? lane >> 1 : lane) - c * PER;
    __syncwarp();
    if (at >= 0 && at < PER && !(p.act && (lane & 1))) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        U* dst = reinterpret_cast<U*>(stg + mg_stg<MG_STG_FLAT>(j, at * ESZ >> 4) + (at * ESZ & 15));
        if constexpr (OUT == DT_F32) *dst = v[j];
        else *dst = (uint16_t)mg_pack16<OUT>(v[j], 0.f);
      }
    }
    __syncwarp();
    mg_store_rows<ESZ, MG_STG_FLAT>(p, stg, t.row0 + j0, rows, o0 + c * PER, min(width - c * PER, n_out - o0 - c * PER),
                                    lane);
  }
}

// The producer and MMA warps share their schedulers with busy epilogue warps, so every
// instruction of theirs between two asynchronous operations costs tensor time (8192^2 x 4096: a
// loop over the stages with descriptors made on the way 120 us, this form 110; and 91 since
// the scale copies come from the MMA warp and the outputs leave from registers).
// Hence: the stages are unrolled, so that barriers, descriptors and TMEM columns are constants
// plus a base; the elected lane and the role are warp-uniform values; all 512 TMEM columns are
// allocated, so addresses start at 0; and each role reads its next tile's entry a tile ahead.
//
// role(t, kb, s, phase): one stage of item t in ring slot s.  Items t0, t0 + step, ... below total, stages
// kb0 .. kb1 of each; ends where a call returns false.  UNROLL: slots are constants (the flat
// kernel, whose 5 to 9 slots of four roles would not fit the instruction cache, streams weights
// and does without: 27 against 34 us for 32 tokens over 128 experts).
template <int STAGES, bool UNROLL, class Stage>
__device__ __forceinline__ void mg_for_stages(int t0, int total, int step, int kb0, int kb1, Stage&& role) {
  int t = t0, kb = kb0;
  uint32_t phase = 0;
  while (t < total) {
#pragma unroll(UNROLL ? STAGES : 1)
    for (int s = 0; s < STAGES; ++s) {
      if (!role(t, kb, s, phase)) return;
      if (++kb == kb1) {
        kb = kb0;
        t += step;
        if (t >= total) return;
      }
    }
    phase ^= 1;
  }
}

// Wide kernel.  tmT: token rows [R, cols_p/2], box 128 B x 128; tmW: weight rows [n * N, cols_p/2], box
// 128 B x 256.
//
// 8192^2 x 4096 with SwiGLU: 91 us, 6.0 PFLOP/s, bound by the MMAs and the waits between a stage's scale copies
// and its MMAs.  131072 expert rows x 2048 x 1024 with SwiGLU: 146 us, 3.8 PFLOP/s, 4900 clocks a tile at
// 1965 MHz.  The MMAs and loads of its four stages alone take 107 us (3600 clocks), the two
// special-function operations an output 2048 clocks; the rest is the part of the epilogue that runs beside
// no MMA.
//
// One accumulator: its 256 columns leave for registers in about 400 clocks, once the warps have finished the tile
// before, and only then do the next tile's MMAs run under the epilogue.  Measured and slower (those expert
// rows; then 8192^2 x 4096): two accumulators sharing 48 columns, the scales in two slots, 187 against
// 165 us, 112 against 109;
// pairs of CTAs on one tile (cta_group::2) 252 against 199 with the grouping, 135 against 126 with the quantiser;
// 8 epilogue warps of 128 columns 213 against 203; SwiGLU in packed pairs 214 against 156.
template <int OUT, bool SWIGLU>
__global__ void __launch_bounds__(WideShape::THREADS, 1)
    mx_wide_kernel(const __grid_constant__ CUtensorMap tmT, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ MgParams p) {
  pdl_wait();
  pdl_trigger();
  using S = WideShape;
  constexpr int STAGES = S::STAGES, EPW = S::EPW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * MG_A_BYTES;
  uint8_t* sSFA = sB + STAGES * S::B_BYTES;
  uint8_t* sSFB = sSFA + STAGES * MG_SF_BYTES;
  uint8_t* sSTG = sSFB + STAGES * 2 * MG_SF_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sSTG + EPW * 32 * MG_STG_WIDE);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 1;
  uint64_t* drain_bar = tempty_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  const uint32_t gave_up = smem_u32(tmem_slot + 1);
  static_assert((2 * STAGES + 3) * 8 + 8 <= MG_MISC_BYTES, "barriers");

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);   // known to be uniform
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    mbar_init(smem_u32(tfull_bar), 1);
    mbar_init(smem_u32(tempty_bar), EPW);
    mbar_init(smem_u32(drain_bar), 1);
    tmem_slot[1] = 0;                              // gave_up
    fence_mbar_init();
    tma_prefetch_desc(&tmT);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), MG_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const int n_tiles = p.n_tiles ? min(*p.n_tiles, p.max_tiles) : p.max_tiles;
  const int total = n_tiles * p.n_wt;
  const int n_kblk = (int)((p.katoms + 1) / 2);
  const int t0 = blockIdx.x, step = gridDim.x;
  const uint64_t timeout = p.timeout_ns ? p.timeout_ns : 2000000000ull;

  if (warp == 0) {
    // ───────── producer ─────────
    const bool one = elect_one();
    int64_t issued = 0;
    const uint32_t wblk = (uint32_t)((p.N + 127) / 128);
    int4 next = mg_fetch(p, t0 < total ? t0 / p.n_wt : 0);
    int trow = 0, wrow = 0;
    const uint8_t *sf_t = nullptr, *sf_w = nullptr;
    bool second = false;                                            // the weight tile's second atom block exists
    mg_for_stages<STAGES, true>(t0, total, step, 0, n_kblk, [&](int t, int kb, int s, uint32_t phase) {
      if (kb == 0) {
        const int wt = t % p.n_wt;
        const MgTile tile = mg_tile<S::SLOT>(p, next);
        trow = (int)tile.row0;
        wrow = tile.e * p.N + wt * S::BN;
        sf_t = p.sf_tok + (uint64_t)tile.slot * p.katoms * 512;
        sf_w = p.sf_w + ((uint64_t)tile.e * wblk + wt * 2) * p.katoms * 512;
        second = wt * 2 + 1 < (int)wblk;
        if (t + step < total) next = mg_fetch(p, (t + step) / p.n_wt);
      }
      if (!mg_wait(smem_u32(&empty_bar[s]), phase ^ 1, gave_up, p.status, timeout)) return false;
      if (one) {
        const uint32_t fb = smem_u32(&full_bar[s]);
        const uint32_t sfn = min(2u, p.katoms - 2 * kb) * 512;      // atoms of this stage
        mbar_arrive_expect_tx(fb, MG_A_BYTES + S::B_BYTES + sfn * (2 + (second ? 1 : 0)));
        tma_load_2d(smem_u32(sA + s * MG_A_BYTES), &tmT, fb, kb * (MG_BK / 2), trow);
        tma_load_2d(smem_u32(sB + s * S::B_BYTES), &tmW, fb, kb * (MG_BK / 2), wrow);
        const uint32_t sb = smem_u32(sSFB + s * 2 * MG_SF_BYTES);
        bulk_load(smem_u32(sSFA + s * MG_SF_BYTES), sf_t + kb * 1024, sfn, fb);
        bulk_load(sb, sf_w + kb * 1024, sfn, fb);
        if (second) bulk_load(sb + MG_SF_BYTES, sf_w + (uint64_t)p.katoms * 512 + kb * 1024, sfn, fb);
      }
      __syncwarp();
      ++issued;
      return true;
    });
    // every copy lands before the CTA can exit (returns at once unless a consumer gave up)
    for (int64_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
      mbar_wait(smem_u32(&full_bar[i % STAGES]), (uint32_t)((i / STAGES) & 1), nullptr, 0, MHMOE_DRAIN_NS);
  } else if (warp == 1) {
    // ───────── MMA issuer ─────────
    const bool one = elect_one();
    uint32_t acc_phase = 0;
    constexpr uint32_t idesc[2] = {idesc_mxf4(MG_BM, S::BN, 0), idesc_mxf4(MG_BM, S::BN, 2)};
    const uint64_t a0 = sdesc_kmajor_sw128(smem_u32(sA)), b0 = sdesc_kmajor_sw128(smem_u32(sB));
    const uint64_t sa0 = sdesc_sf_chunk(smem_u32(sSFA)), sb0 = sdesc_sf_chunk(smem_u32(sSFB));
    // A stage's scale slot in TMEM is free when the stage is: both wait for the MMAs of the round before.
    mg_for_stages<STAGES, true>(t0, total, step, 0, n_kblk, [&](int, int kb, int s, uint32_t phase) {
      if (kb == 0 && !mg_wait(smem_u32(tempty_bar), acc_phase ^ 1, gave_up, p.status, timeout)) return false;
      if (!mg_wait(smem_u32(&full_bar[s]), phase, gave_up, p.status, timeout)) return false;
      tc_fence_after();
      const uint64_t a_d = a0 + s * (MG_A_BYTES >> 4), b_d = b0 + s * (S::B_BYTES >> 4);
      const uint32_t tsfa = S::SF_COL0 + s * S::SF_COLS, tsfb = tsfa + 8;
      const uint64_t sa = sa0 + s * (MG_SF_BYTES >> 4), sb = sb0 + s * (2 * MG_SF_BYTES >> 4);
      if (one) {
        const bool whole = 2 * kb + 1 < (int)p.katoms;
        tc_cp_32x128b_warpx4(tsfa, sa);
        tc_cp_32x128b_warpx4(tsfb, sb);
        tc_cp_32x128b_warpx4(tsfb + 4, sb + (MG_SF_BYTES >> 4));
        if (whole) {
          tc_cp_32x128b_warpx4(tsfa + 4, sa + 32);
          tc_cp_32x128b_warpx4(tsfb + 8, sb + 32);
          tc_cp_32x128b_warpx4(tsfb + 12, sb + (MG_SF_BYTES >> 4) + 32);
        }
        mma_mxf4(0, a_d, b_d, idesc[0], tsfa, tsfb, kb != 0 ? 1u : 0u);
        mma_mxf4(0, a_d + 2, b_d + 2, idesc[1], tsfa, tsfb, 1u);
        if (whole) {
          mma_mxf4(0, a_d + 4, b_d + 4, idesc[0], tsfa + 4, tsfb + 8, 1u);
          mma_mxf4(0, a_d + 6, b_d + 6, idesc[1], tsfa + 4, tsfb + 8, 1u);
        }
        tc_commit(smem_u32(&empty_bar[s]));
        if (kb + 1 == n_kblk) tc_commit(smem_u32(tfull_bar));
      }
      __syncwarp();
      if (kb + 1 == n_kblk) acc_phase ^= 1;
      return true;
    });
  } else {
    // ───────── epilogue ─────────
    const int q = warp & 3;                        // TMEM lane quarter of this warp
    const int slice = (warp - 2) >> 2;             // accumulator columns [64 * slice, +64)
    uint8_t* stg = sSTG + (warp - 2) * 32 * MG_STG_WIDE;
    uint32_t acc_phase = 0;
    int4 next = mg_fetch(p, t0 < total ? t0 / p.n_wt : 0);
    for (int t = t0; t < total; t += step) {
      const int wt = t % p.n_wt;
      const MgTile tile = mg_tile<S::SLOT>(p, next);
      if (t + step < total) next = mg_fetch(p, (t + step) / p.n_wt);
      if (!mg_wait(smem_u32(tfull_bar), acc_phase, gave_up, p.status, timeout)) break;
      acc_phase ^= 1;
      tc_fence_after();
      uint32_t r[64];
      const uint32_t taddr = ((uint32_t)(q * 32) << 16) + (uint32_t)(slice * 64);
      MHMOE_TMEM_LD_32x32b_X32(taddr, (r + 0));
      MHMOE_TMEM_LD_32x32b_X32(taddr + 32, (r + 32));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(tempty_bar));
      if (q * 32 < tile.rows)
        mg_wide_epilogue<OUT, SWIGLU>(p, tile, r, wt * S::BN + slice * 64, q * 32, lane, stg);
    }
  }

  // Retire every tcgen05 op that was issued before TMEM is released (a formality unless a wait gave up).
  if (warp == 1 && lane == 0) {
    tc_commit(smem_u32(drain_bar));
    mbar_wait(smem_u32(drain_bar), 0, nullptr, 0, MHMOE_DRAIN_NS);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, MG_TMEM_COLS);
  }
}

// Flat kernel.  tmT: token rows [R, cols_p/2], box 128 B x BN; tmW: weight rows [n * N, cols_p/2], box
// 128 B x 128.  SPLIT: a cluster of CTAs shares one work item along the columns; their partial
// accumulators meet in distributed shared memory and are summed in the order of the ranks.
//
// XQ (with SPLIT, where a CTA has one item): the type of the up to BN rows of x that the epilogue warps
// quantise into operand B's stages themselves, before they have outputs to write, instead of a
// kernel ahead of this one (one token x 4096 x 2048: 8.1 us, 11.3 with the two kernels).
//
// Bound by the weights' bytes where there are many (256 rows over 128 experts of 2048 x 1024: 24.5 us, 5.8 TB/s),
// by latency where there are few: launch, TMEM allocation, the cluster's join and the stores.
template <int BN, bool SPLIT, int OUT, int XQ>
__global__ void __launch_bounds__(FlatShape<BN>::THREADS, 1)
    mx_flat_kernel(const __grid_constant__ CUtensorMap tmT, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ MgParams p) {
  pdl_wait();
  pdl_trigger();
  using S = FlatShape<BN>;
  constexpr int STAGES = S::STAGES, EPW = S::EPW, NACC = S::NACC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * MG_A_BYTES;
  uint8_t* sSFA = sB + STAGES * S::B_BYTES;
  uint8_t* sSFB = sSFA + STAGES * MG_SF_BYTES;
  uint8_t* sSTG = sSFB + STAGES * MG_SF_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sSTG + EPW * 32 * MG_STG_FLAT);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;    // [NACC]
  uint64_t* tempty_bar = tfull_bar + NACC;     // [NACC]
  uint64_t* drain_bar = tempty_bar + NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  const uint32_t gave_up = smem_u32(tmem_slot + 1);
  static_assert((2 * STAGES + 2 * NACC + 1) * 8 + 8 <= MG_MISC_BYTES, "barriers");
  static_assert(XQ < 0 || (SPLIT && BN <= 32 && EPW == 4), "a stage of rows is quantised by 128 threads");
  static_assert(!SPLIT || BN * 128 * 4 <= STAGES * MG_A_BYTES, "partial sums lie over operand A's stages");

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);   // known to be uniform
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), XQ >= 0 ? 1 + EPW : 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < NACC; ++a) {
      mbar_init(smem_u32(&tfull_bar[a]), 1);
      mbar_init(smem_u32(&tempty_bar[a]), EPW);
    }
    mbar_init(smem_u32(drain_bar), 1);
    tmem_slot[1] = 0;                              // gave_up
    fence_mbar_init();
    if (XQ < 0) tma_prefetch_desc(&tmT);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), MG_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const int n_tiles = p.n_tiles ? min(*p.n_tiles, p.max_tiles) : p.max_tiles;
  const int total = n_tiles * p.n_wt;
  const int n_kblk = (int)((p.katoms + 1) / 2);
  int t0 = blockIdx.x, step = gridDim.x, kb0 = 0, kb1 = n_kblk, rank = 0, csize = 1;
  if constexpr (SPLIT) {
    rank = (int)cluster_ctarank();
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
    t0 = blockIdx.x / csize;
    step = 1 << 30;                            // one item per cluster
    kb0 = n_kblk * rank / csize;
    kb1 = n_kblk * (rank + 1) / csize;
  }
  const uint64_t timeout = p.timeout_ns ? p.timeout_ns : 2000000000ull;

  if (warp == 0) {
    // ───────── producer ─────────
    const bool one = elect_one();
    int64_t issued = 0;
    const uint32_t wblk = (uint32_t)((p.N + 127) / 128);
    int4 next = mg_fetch(p, t0 < total ? t0 / p.n_wt : 0);
    int trow = 0, wrow = 0;
    const uint8_t *sf_t = nullptr, *sf_w = nullptr;
    mg_for_stages<STAGES, false>(t0, total, step, kb0, kb1, [&](int t, int kb, int s, uint32_t phase) {
      if (kb == kb0) {
        const int wt = t % p.n_wt;
        const MgTile tile = mg_tile<S::SLOT>(p, next);
        trow = (int)tile.row0;
        wrow = tile.e * p.N + wt * 128;
        sf_t = p.sf_tok + (uint64_t)tile.slot * p.katoms * 512;
        sf_w = p.sf_w + ((uint64_t)tile.e * wblk + wt) * p.katoms * 512;
        if (t + step < total) next = mg_fetch(p, (t + step) / p.n_wt);
      }
      if (!mg_wait(smem_u32(&empty_bar[s]), phase ^ 1, gave_up, p.status, timeout)) return false;
      if (one) {
        const uint32_t fb = smem_u32(&full_bar[s]);
        const uint32_t sfn = min(2u, p.katoms - 2 * kb) * 512;      // atoms of this stage
        mbar_arrive_expect_tx(fb, MG_A_BYTES + sfn + (XQ < 0 ? S::B_BYTES + sfn : 0));
        tma_load_2d(smem_u32(sA + s * MG_A_BYTES), &tmW, fb, kb * (MG_BK / 2), wrow);
        bulk_load(smem_u32(sSFA + s * MG_SF_BYTES), sf_w + kb * 1024, sfn, fb);
        if constexpr (XQ < 0) {
          tma_load_2d(smem_u32(sB + s * S::B_BYTES), &tmT, fb, kb * (MG_BK / 2), trow);
          bulk_load(smem_u32(sSFB + s * MG_SF_BYTES), sf_t + kb * 1024, sfn, fb);
        }
      }
      __syncwarp();
      ++issued;
      return true;
    });
    // every copy lands before the CTA can exit (returns at once unless a consumer gave up)
    for (int64_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
      mbar_wait(smem_u32(&full_bar[i % STAGES]), (uint32_t)((i / STAGES) & 1), nullptr, 0, MHMOE_DRAIN_NS);
  } else if (warp == 1) {
    // ───────── MMA issuer ─────────
    const bool one = elect_one();
    uint32_t acc = 0, acc_phase = 0;
    constexpr uint32_t idesc[2] = {idesc_mxf4(MG_BM, BN, 0), idesc_mxf4(MG_BM, BN, 2)};
    const uint64_t a0 = sdesc_kmajor_sw128(smem_u32(sA)), b0 = sdesc_kmajor_sw128(smem_u32(sB));
    const uint64_t sa0 = sdesc_sf_chunk(smem_u32(sSFA)), sb0 = sdesc_sf_chunk(smem_u32(sSFB));
    // A stage's scale slot in TMEM is free when the stage is: both wait for the MMAs of the round before.
    mg_for_stages<STAGES, false>(t0, total, step, kb0, kb1, [&](int, int kb, int s, uint32_t phase) {
      if (kb == kb0 && !mg_wait(smem_u32(&tempty_bar[acc]), acc_phase ^ 1, gave_up, p.status, timeout))
        return false;
      if (!mg_wait(smem_u32(&full_bar[s]), phase, gave_up, p.status, timeout)) return false;
      tc_fence_after();
      const uint64_t a_d = a0 + s * (MG_A_BYTES >> 4), b_d = b0 + s * (S::B_BYTES >> 4);
      const uint32_t tsfa = S::SF_COL0 + s * S::SF_COLS, tsfb = tsfa + 8, d = acc * BN;
      const uint64_t sa = sa0 + s * (MG_SF_BYTES >> 4), sb = sb0 + s * (MG_SF_BYTES >> 4);
      if (one) {
        const bool whole = 2 * kb + 1 < (int)p.katoms;
        tc_cp_32x128b_warpx4(tsfa, sa);
        tc_cp_32x128b_warpx4(tsfb, sb);
        if (whole) {
          tc_cp_32x128b_warpx4(tsfa + 4, sa + 32);
          tc_cp_32x128b_warpx4(tsfb + 4, sb + 32);
        }
        mma_mxf4(d, a_d, b_d, idesc[0], tsfa, tsfb, kb != kb0 ? 1u : 0u);
        mma_mxf4(d, a_d + 2, b_d + 2, idesc[1], tsfa, tsfb, 1u);
        if (whole) {
          mma_mxf4(d, a_d + 4, b_d + 4, idesc[0], tsfa + 4, tsfb + 4, 1u);
          mma_mxf4(d, a_d + 6, b_d + 6, idesc[1], tsfa + 4, tsfb + 4, 1u);
        }
        tc_commit(smem_u32(&empty_bar[s]));
        if (kb + 1 == kb1) tc_commit(smem_u32(&tfull_bar[acc]));
      }
      __syncwarp();
      if (kb + 1 == kb1 && ++acc == NACC) {
        acc = 0;
        acc_phase ^= 1;
      }
      return true;
    });
  } else {
    // ───────── epilogue ─────────
    const int q = warp & 3;                    // TMEM lane quarter of this warp
    const int part = (warp - 2) >> 2;          // with 8 warps: every other chunk of columns
    constexpr int NC = BN < 32 ? BN : 32;
    uint8_t* stg = sSTG + (warp - 2) * 32 * MG_STG_FLAT;
    if constexpr (XQ >= 0) {
      // 16 threads a row, 16 columns each; rows behind the last hold what was there: their columns of
      // the accumulator are not stored
      using T = typename MxType<XQ < 0 ? 0 : XQ>::T;
      const int tid = threadIdx.x - 64, chunk = tid & 15;
      const uint32_t mask = 0xffu << (lane & 24);
      mg_for_stages<STAGES, false>(t0, total, step, kb0, kb1, [&](int, int kb, int s, uint32_t phase) {
        if (!mg_wait(smem_u32(&empty_bar[s]), phase ^ 1, gave_up, p.status, timeout)) return false;
        const int c0 = kb * MG_BK + chunk * 16;
#pragma unroll
        for (int row = tid >> 4; row < BN; row += 8) {
          if (row >= (int)p.R) break;              // the same for the 16 threads of a row
          MxRaw16<T> v;
          const bool live = c0 < p.cols;
          v.load(static_cast<const T*>(p.x) + row * p.x_stride + c0, live && p.x_vec && c0 + 16 <= p.cols,
                 live ? min(16, p.cols - c0) : 0);
          uint2 code;
          const uint32_t sw = mx_quantize16(v, p.ceil, chunk & 7, mask, code);
          // 128-B swizzle: 16-B chunk k of row r sits at chunk k ^ (r & 7)
          *reinterpret_cast<uint2*>(sB + s * S::B_BYTES + row * 128 + (((chunk >> 1) ^ (row & 7)) << 4) +
                                    (chunk & 1) * 8) = code;
          if ((chunk & 7) == 0)
            *reinterpret_cast<uint32_t*>(sSFB + s * MG_SF_BYTES + (chunk >> 3) * 512 + row * 16) = sw;
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full_bar[s]));
        return true;
      });
    }
    int acc = 0;
    uint32_t acc_phase = 0;
    int4 next = mg_fetch(p, t0 < total ? t0 / p.n_wt : 0);
    for (int t = t0; t < total; t += step) {
      const int wt = t % p.n_wt;
      const MgTile tile = mg_tile<S::SLOT>(p, next);
      if (t + step < total) next = mg_fetch(p, (t + step) / p.n_wt);
      const int n0 = wt * 128 + q * 32;
      const float b = p.bias && n0 + lane < p.N ? __ldg(p.bias + (int64_t)tile.e * p.N + n0 + lane) : 0.f;
      if (!mg_wait(smem_u32(&tfull_bar[acc]), acc_phase, gave_up, p.status, timeout)) break;
      tc_fence_after();
      const uint32_t taddr = ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN);
      for (int j0 = part * NC; j0 < BN && j0 < tile.rows; j0 += NC * (EPW / 4)) {
        uint32_t r[NC];
        if constexpr (NC == 16) MHMOE_TMEM_LD_32x32b_X16(taddr + j0, r);
        else MHMOE_TMEM_LD_32x32b_X32(taddr + j0, r);
        tmem_wait_ld();
        if constexpr (SPLIT) {
          // partial sums [token][weight row] over the stages' memory, all of it consumed by now
          float* red = reinterpret_cast<float*>(smem);
#pragma unroll
          for (int j = 0; j < NC; ++j) red[(j0 + j) * 128 + q * 32 + lane] = __uint_as_float(r[j]);
        } else {
          if (n0 < p.N) mg_flat_epilogue<NC, OUT>(p, tile, r, j0, n0, b, lane, stg);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[acc]));
      if (++acc == NACC) { acc = 0; acc_phase ^= 1; }
    }
  }

  // Retire every tcgen05 op that was issued before TMEM is released (a formality unless a wait gave up).
  if (warp == 1 && lane == 0) {
    tc_commit(smem_u32(drain_bar));
    mbar_wait(smem_u32(drain_bar), 0, nullptr, 0, MHMOE_DRAIN_NS);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, MG_TMEM_COLS);
  }
  if constexpr (SPLIT) {
    cluster_sync();
    if (t0 < total) {
      const int tt = t0 / p.n_wt, wt = t0 % p.n_wt;
      const MgTile tile = mg_tile<S::SLOT>(p, mg_fetch(p, tt));
      const uint32_t red = smem_u32(smem);
      uint32_t peer[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) peer[c] = mapa_shared(red, (uint32_t)min(c, csize - 1));
      auto sum = [&](int at) {                 // partial sums of one output in the order of the ranks
        float z = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          float v = 0.f;
          if (c < csize)
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer[c] + at * 4) : "memory");
          z += v;
        }
        return z;
      };
      const float* bias = p.bias ? p.bias + (int64_t)tile.e * p.N : nullptr;
      const int per_row = p.act ? 64 : 128;    // outputs of a token in this tile
      for (int i = threadIdx.x + blockDim.x * rank; i < tile.rows * per_row; i += blockDim.x * csize) {
        const int j = i / per_row, c = i % per_row;
        const int64_t row = tile.row0 + j;
        const float rw = p.row_weights ? __ldg(p.row_weights + row) : 1.f;
        if (p.act) {
          const int n = wt * 128 + 2 * c;
          if (n < p.N) {
            float g = sum(j * 128 + 2 * c), u = sum(j * 128 + 2 * c + 1);
            if (bias) {
              g += __ldg(bias + n);
              u += __ldg(bias + n + 1);
            }
            mg_store(p.y, p.y_dtype, row * p.y_stride + n / 2, mx_swiglu7(g, u) * rw);
          }
        } else {
          const int n = wt * 128 + c;
          if (n < p.N) {
            float z = sum(j * 128 + c);
            if (bias) z += __ldg(bias + n);
            mg_store(p.y, p.y_dtype, row * p.y_stride + n, z * rw);
          }
        }
      }
    }
    cluster_sync();                            // no CTA leaves while others read its memory
  }
}

// ───────────────────────────── expert rows ─────────────────────────────

__device__ __forceinline__ int64_t clip(int64_t v, int64_t hi) { return v < 0 ? 0 : (v > hi ? hi : v); }

struct MgGroup {
  const void* x;              // activations, or with xq the tokens already in MXFP4
  int64_t x_stride, x_rows, R;
  const uint8_t* xq;
  const uint8_t* xsf;
  uint32_t cols, katoms;
  bool ceil, vec;
  const int64_t* offsets;
  int n, slot_rows, max_tiles;
  const int32_t* gather;
  uint8_t* data;              // [R, katoms * 64]
  uint8_t* sf;                // slots of katoms atoms
  int4* tiles;
  int* n_tiles;
  uint8_t* y;                 // rows without an expert are cleared
  int64_t y_row_bytes, y_pitch;
  bool zero_tail;
  int* status;
};

// The list of token tiles, by one block of 256 threads.  Expert e's tiles take the scale slots
// offsets[e] / slot_rows + e + 0, 1, ...: the sum of the rounded-up tile counts before e is at most
// that, so that the blocks that fill the slots need no prefix sum.
__device__ __forceinline__ void mg_list_tiles(const MgGroup& p) {
  __shared__ int wsum[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  bool bad = false;
  for (int e0 = 0; e0 < p.n; e0 += 256) {
    const int e = e0 + threadIdx.x;
    int64_t a = 0;
    int rows = 0;
    if (e < p.n) {
      const int64_t lo = p.offsets[e], hi = p.offsets[e + 1];
      bad |= lo < 0 || lo > p.R || hi < lo || hi > p.R;
      a = clip(lo, p.R);
      rows = (int)max((int64_t)0, clip(hi, p.R) - a);
    }
    const int cnt = (rows + p.slot_rows - 1) / p.slot_rows;
    int inc = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < 8; ++w) {
      before += w < warp ? wsum[w] : 0;
      all += wsum[w];
    }
    const int64_t at = (int64_t)base + before + inc - cnt;
    const int slot0 = (int)(a / p.slot_rows) + e;
    for (int j = 0; j < cnt && at + j < p.max_tiles; ++j)
      p.tiles[at + j] = make_int4(e, (int)a + j * p.slot_rows, min(p.slot_rows, rows - j * p.slot_rows), slot0 + j);
    // Offsets that decrease can count the rows many times over: such a sum is above max_tiles in this round
    // (256 experts of up to 2^23 tiles, every other one, fit 31 bits) and stays there.
    base = (int)min((int64_t)base + all, (int64_t)p.max_tiles);
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.n_tiles = base;
  if (bad) record_error(p.status, MHMOE_ERR_ARGS);
}

// Where sorted row r goes and comes from.
struct MgRow {
  int64_t src;                // row of x, -1: a row of zeros (its id is outside x)
  uint64_t sf;                // byte of its first scale word in MgGroup::sf
  bool none;                  // no expert
};
__device__ __forceinline__ MgRow mg_row(const MgGroup& p, int64_t r, int e) {
  MgRow w;
  const int64_t a = clip(p.offsets[e], p.R);
  w.none = a > r || clip(p.offsets[e + 1], p.R) <= r;       // before the first, behind the last (or offsets that decrease)
  const int64_t tile = w.none ? 0 : (r - a) / p.slot_rows;
  const int m = w.none ? 0 : (int)(r - a - tile * p.slot_rows);
  w.sf = (uint64_t)(a / p.slot_rows + e + tile) * p.katoms * 512 + (m & 31) * 16 + (m >> 5) * 4;
  w.src = w.none ? -1 : (p.gather ? p.gather[r] : r);
  if (!w.none && (w.src < 0 || w.src >= p.x_rows)) {
    record_error(p.status, MHMOE_ERR_ARGS);
    w.src = -1;
  }
  return w;
}

__device__ __forceinline__ void mg_clear_row(const MgGroup& p, int64_t r, int lane) {
  uint8_t* o = p.y + r * p.y_pitch;              // elements of 2 or 4 bytes
  for (int64_t i = lane * 2; i < p.y_row_bytes; i += 64) *reinterpret_cast<uint16_t*>(o + i) = 0;
}

// Block 0 lists the token tiles; every other warp quantises one sorted row.
template <int DT>
__global__ void __launch_bounds__(256) mx_group_kernel(const __grid_constant__ MgGroup p) {
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0) return mg_list_tiles(p);
  using T = typename MxType<DT>::T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = (int64_t)(blockIdx.x - 1) * 8 + warp;
  if (r >= p.R) return;
  // the last expert whose first row is at or before r, 32 candidates a step
  int e = 0, len = p.n;
  while (len > 1) {
    const int step = (len + 31) / 32, i = e + lane * step;
    const bool le = lane * step < len && clip(p.offsets[i], p.R) <= r;
    const int k = max(__popc(__ballot_sync(0xffffffffu, le)), 1) - 1;
    e += k * step;
    len = min(step, len - k * step);
  }
  const MgRow w = mg_row(p, r, e);
  if (w.none) {
    if (p.zero_tail) mg_clear_row(p, r, lane);
    return;
  }
  const bool ok = w.src >= 0;
  const T* xr = static_cast<const T*>(p.x) + (ok ? w.src : 0) * p.x_stride;
  uint8_t* d = p.data + r * (int64_t)p.katoms * 64;
  uint8_t* s = p.sf + w.sf;
#pragma unroll 2
  for (uint32_t c0 = lane * 16; c0 < (p.katoms + 3) / 4 * 512; c0 += 512) {
    MxRaw16<T> v;
    const bool live = ok && c0 < p.cols;
    v.load(xr + c0, live && p.vec && c0 + 16 <= p.cols, live ? (int)min(16u, p.cols - c0) : 0);
    uint2 code;
    const uint32_t sw = mx_quantize16(v, p.ceil, lane & 7, 0xffffffffu, code);
    if (c0 < p.katoms * 128) {
      *reinterpret_cast<uint2*>(d + c0 / 2) = code;
      if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(s + (c0 / 128) * 512) = sw;
    }
  }
}

// The same from tokens that are quantised already (once a token instead of once a row): every other
// warp copies MG_COPY_ROWS sorted rows, all their loads in flight together.
constexpr int MG_COPY_ROWS = 8;
__global__ void __launch_bounds__(256) mx_group_copy_kernel(const __grid_constant__ MgGroup p, const FastDiv katoms) {
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0) return mg_list_tiles(p);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = ((int64_t)(blockIdx.x - 1) * 8 + warp) * MG_COPY_ROWS;
  if (r0 >= p.R) return;
  const int rows = (int)min((int64_t)MG_COPY_ROWS, p.R - r0);
  // one lane a row: the last expert whose first row is at or before it
  MgRow w{-1, 0, true};
  if (lane < rows) {
    int e = 0, hi = p.n - 1;
    while (e < hi) {
      const int mid = (e + hi + 1) >> 1;
      if (clip(p.offsets[mid], p.R) <= r0 + lane) e = mid;
      else hi = mid - 1;
    }
    w = mg_row(p, r0 + lane, e);
  }
  const uint32_t n16 = katoms.d * 4;               // 16-B chunks of a row
  for (uint32_t i = lane; i < (n16 + 31) / 32 * 32; i += 32) {
    uint4 v[MG_COPY_ROWS];
#pragma unroll
    for (int k = 0; k < MG_COPY_ROWS; ++k) {
      const int64_t src = __shfl_sync(0xffffffffu, w.src, k);
      v[k] = src >= 0 && i < n16 ? __ldg(reinterpret_cast<const uint4*>(p.xq + src * katoms.d * 64) + i)
                                 : make_uint4(0, 0, 0, 0);
    }
    const unsigned none = __ballot_sync(0xffffffffu, w.none);
#pragma unroll
    for (int k = 0; k < MG_COPY_ROWS; ++k)
      if (!(none >> k & 1) && i < n16) reinterpret_cast<uint4*>(p.data + (r0 + k) * (int64_t)katoms.d * 64)[i] = v[k];
  }
  // scale words: row k, atom a
  for (uint32_t i = lane; i < (MG_COPY_ROWS * katoms.d + 31) / 32 * 32; i += 32) {
    const uint32_t k = katoms.div(i), a = i - k * katoms.d;
    const int from = (int)min(k, (uint32_t)MG_COPY_ROWS - 1);
    const int64_t src = __shfl_sync(0xffffffffu, w.src, from);
    const uint64_t at = __shfl_sync(0xffffffffu, w.sf, from);
    const bool none = __shfl_sync(0xffffffffu, (int)w.none, from) != 0;
    if (k < MG_COPY_ROWS && !none)
      *reinterpret_cast<uint32_t*>(p.sf + at + a * 512) =
          src >= 0 ? __ldg(reinterpret_cast<const uint32_t*>(p.xsf + mx_sf_offset(src, a * 4, katoms.d))) : 0u;
  }
  if (p.zero_tail)
    for (unsigned none = __ballot_sync(0xffffffffu, w.none && lane < rows); none; none &= none - 1)
      mg_clear_row(p, r0 + __ffs(none) - 1, lane);
}

// ───────────────────────────── launch ─────────────────────────────

struct MgPlan {
  bool flat;
  int bn, slot_rows, split;
  int64_t tiles, slots;       // token tiles at most; scale slots
  int n_wt;
  bool once;                  // quantise the tokens first, then copy their rows
  bool own;                   // the flat kernel quantises x itself
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Orientation, tile and split by the sizes alone.
MgPlan mg_plan(int64_t x_rows, int64_t R, int n, int N, int64_t katoms, bool grouped) {
  const int sms = num_sms();
  MgPlan g;
  const int64_t avg = grouped ? ceil_div(R, n) : R;
  auto tiles_of = [&](int64_t slot) { return grouped ? R / slot + std::min<int64_t>(n, R) : ceil_div(R, slot); };
  if (grouped ? avg <= 16 : R <= 128) {
    // a few rows per matrix: one flat tile holds them
    const int64_t want = grouped ? avg + avg / 2 : avg;
    g.flat = true;
    g.bn = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : 128;
  } else {
    // Above that the wide tile, however few of its 128 rows an expert fills: its 256 weight rows
    // stream past faster than HBM delivers them (128 experts of 2048 x 1024, 4096 rows: 34 us wide, 45
    // and 57 flat with 128 and 64 columns, grouping included).  Flat where the wide tiles
    // would not reach every SM.
    g.flat = tiles_of(128) * ceil_div(N, 256) < sms;
    g.bn = 128;
  }
  g.slot_rows = g.bn;
  g.tiles = tiles_of(g.slot_rows);
  g.slots = grouped ? R / g.slot_rows + n + 1 : g.tiles;
  g.n_wt = (int)ceil_div(N, g.flat ? 128 : 256);
  // Copying a row costs a third of quantising it, a launch more about 2 us (top-8 of 128 experts, 1024
  // columns: 8192 rows 16.1 us quantised each, 17.7 copied; 32768 rows 38.3 and 30.8).
  g.once = grouped && R >= 2 * x_rows && R >= 16384;
  g.own = !grouped && R <= 16 && g.n_wt <= sms;     // one item a CTA
  g.split = 1;
  const int64_t n_kblk = ceil_div(katoms, 2);
  while (g.flat && g.split < 8 && g.tiles * g.n_wt * g.split * 2 <= sms && g.split * 2 <= n_kblk) g.split *= 2;
  return g;
}

struct MgScratch {
  size_t data, sf, tiles, count, tok, tok_sf, bytes;
};
MgScratch mg_scratch(const MgPlan& g, int64_t x_rows, int64_t R, int64_t katoms, bool grouped) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  MgScratch s;
  s.data = 0;
  s.sf = up((size_t)R * katoms * 64);
  s.tiles = s.sf + up((size_t)(grouped ? g.slots : ceil_div(R, 128)) * katoms * 512);
  s.count = s.tiles + (grouped ? up((size_t)g.tiles * sizeof(int4)) : 0);
  s.tok = s.count + (grouped ? 256 : 0);
  s.tok_sf = s.tok + (g.once ? up((size_t)x_rows * katoms * 64) : 0);
  s.bytes = s.tok_sf + (g.once ? (size_t)ceil_div(x_rows, 128) * katoms * 512 : 0);
  return s;
}

template <int OUT, bool SWIGLU>
cudaError_t launch_wide(const CUtensorMap& tt, const CUtensorMap& tw, const MgParams& p, const MgPlan& g,
                        cudaStream_t st) {
  using S = WideShape;
  auto kernel = mx_wide_kernel<OUT, SWIGLU>;
  static PerDeviceOnce once;
  const cudaError_t attr = once.run(
      [&](int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
  if (attr != cudaSuccess) return attr;
  return launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(num_sms(), g.tiles * g.n_wt)), dim3(S::THREADS), S::SMEM, st,
                    tt, tw, p);
}

template <int BN, bool SPLIT, int OUT, int XQ = -1>
cudaError_t launch_flat(const CUtensorMap& tt, const CUtensorMap& tw, const MgParams& p, const MgPlan& g,
                        cudaStream_t st) {
  using S = FlatShape<BN>;
  auto kernel = mx_flat_kernel<BN, SPLIT, OUT, XQ>;
  static PerDeviceOnce once;
  const cudaError_t attr = once.run(
      [&](int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
  if (attr != cudaSuccess) return attr;
  const int64_t items = g.tiles * g.n_wt;
  if constexpr (!SPLIT) {
    return launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(num_sms(), items)), dim3(S::THREADS), S::SMEM, st, tt, tw,
                      p);
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * g.split));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = (unsigned)g.split;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, tt, tw, p);
  }
}

template <int BN>
cudaError_t launch_flat(const CUtensorMap& tt, const CUtensorMap& tw, const MgParams& p, const MgPlan& g,
                        cudaStream_t st) {
  if (g.split > 1) return launch_flat<BN, true, DT_F32, -1>(tt, tw, p, g, st);      // stores by p.y_dtype
  return p.y_dtype == DT_F32    ? launch_flat<BN, false, DT_F32, -1>(tt, tw, p, g, st)
         : p.y_dtype == DT_BF16 ? launch_flat<BN, false, DT_BF16, -1>(tt, tw, p, g, st)
                                : launch_flat<BN, false, DT_F16, -1>(tt, tw, p, g, st);
}

template <int OUT>
cudaError_t launch_wide(const CUtensorMap& tt, const CUtensorMap& tw, const MgParams& p, const MgPlan& g,
                        cudaStream_t st) {
  return p.act ? launch_wide<OUT, true>(tt, tw, p, g, st) : launch_wide<OUT, false>(tt, tw, p, g, st);
}

}  // namespace

size_t mx_product_workspace_bytes(int64_t x_rows, int64_t R, int n, int N, int cols, bool grouped) {
  const int64_t katoms = mx_padded_cols(cols) / 128;
  if (R == 0) return 0;
  const MgPlan g = mg_plan(x_rows, R, n, N, katoms, grouped);
  return g.own ? 0 : mg_scratch(g, x_rows, R, katoms, grouped).bytes;
}

int mx_product(const MxProduct& p, void* workspace, cudaStream_t st, cudaError_t* cerr) {
  const int64_t katoms = mx_padded_cols(p.cols) / 128;
  const bool grouped = p.offsets != nullptr;
  const MgPlan g = mg_plan(p.x_rows, p.R, p.n, p.N, katoms, grouped);
  if (g.tiles * g.n_wt >= (int64_t)1 << 30) return MHMOE_ERR_CAPACITY;
  const bool own = g.own && !p.xq;
  const MgScratch ws = mg_scratch(g, p.x_rows, p.R, katoms, grouped);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  const int64_t y_esz = p.y_dtype == DT_F32 ? 4 : 2, n_out = p.act ? p.N / 2 : p.N;
  const uint8_t* data = p.xq;
  MgParams a{};
  a.sf_tok = p.xsf;
  if (grouped) {
    const int64_t esz = p.x_dtype == DT_F32 ? 4 : 2;
    MgGroup q{};
    q.x_stride = p.x_stride;
    q.x_rows = p.x_rows;
    q.R = p.R;
    q.cols = (uint32_t)p.cols;
    q.katoms = (uint32_t)katoms;
    q.ceil = p.ceil;
    q.vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.x_stride * esz % 16 == 0;
    q.offsets = p.offsets;
    q.n = p.n;
    q.slot_rows = g.slot_rows;
    q.max_tiles = (int)g.tiles;
    q.gather = p.gather_ids;
    q.data = base + ws.data;
    q.sf = base + ws.sf;
    q.tiles = reinterpret_cast<int4*>(base + ws.tiles);
    q.n_tiles = reinterpret_cast<int*>(base + ws.count);
    q.y = static_cast<uint8_t*>(p.y);
    q.y_row_bytes = n_out * y_esz;
    q.y_pitch = p.y_stride * y_esz;
    q.zero_tail = p.zero_tail;
    q.status = p.status;
    q.x = p.x;
    if (g.once) {
      q.xq = base + ws.tok;
      q.xsf = base + ws.tok_sf;
      *cerr = launch_mx_quantize(p.x, p.x_dtype, 0, p.x_stride, 1, p.x_rows, p.cols, p.ceil, base + ws.tok,
                                 base + ws.tok_sf, st);
      if (*cerr == cudaSuccess)
        *cerr = launch_pdl(mx_group_copy_kernel, dim3((unsigned)(1 + ceil_div(p.R, 8 * MG_COPY_ROWS))), dim3(256), 0, st,
                           q, FastDiv((uint32_t)katoms));
    } else {
      const dim3 grid((unsigned)(1 + ceil_div(p.R, 8)));
      *cerr = p.x_dtype == DT_F32    ? launch_pdl(mx_group_kernel<DT_F32>, grid, dim3(256), 0, st, q)
              : p.x_dtype == DT_BF16 ? launch_pdl(mx_group_kernel<DT_BF16>, grid, dim3(256), 0, st, q)
                                     : launch_pdl(mx_group_kernel<DT_F16>, grid, dim3(256), 0, st, q);
    }
    data = q.data;
    a.sf_tok = q.sf;
    a.tiles = q.tiles;
    a.n_tiles = q.n_tiles;
  } else if (!p.xq && !own) {
    *cerr = launch_mx_quantize(p.x, p.x_dtype, 0, p.x_stride, 1, p.R, p.cols, p.ceil, base + ws.data, base + ws.sf, st);
    data = base + ws.data;
    a.sf_tok = base + ws.sf;
  }
  if (*cerr != cudaSuccess) return MHMOE_ERR_LAUNCH;
  a.sf_w = p.w_sf;
  a.max_tiles = (int)g.tiles;
  a.R = p.R;
  a.N = p.N;
  a.n_wt = g.n_wt;
  a.katoms = (uint32_t)katoms;
  a.row_weights = p.row_weights;
  a.bias = p.bias;
  a.act = p.act;
  a.y = p.y;
  a.y_dtype = p.y_dtype;
  a.y_stride = p.y_stride;
  a.y_vec = (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && p.y_stride * y_esz % 16 == 0 && n_out * y_esz % 16 == 0;
  a.y_vec32 = (reinterpret_cast<uintptr_t>(p.y) & 31) == 0 && p.y_stride * y_esz % 32 == 0 && n_out * y_esz % 32 == 0;
  a.status = p.status;
  a.timeout_ns = p.timeout_ns;
  CUtensorMap tt{}, tw;
  if ((!own && encode_tmap_2d_u8(&tt, data, (uint64_t)katoms * 64, (uint64_t)p.R, 128, (uint32_t)g.slot_rows) !=
                   cudaSuccess) ||
      encode_tmap_2d_u8(&tw, p.w_data, (uint64_t)katoms * 64, (uint64_t)p.n * p.N, 128, g.flat ? 128 : 256) != cudaSuccess)
    return MHMOE_ERR_DRIVER;
  if (own) {
    a.x = p.x;
    a.x_stride = p.x_stride;
    a.cols = p.cols;
    a.ceil = p.ceil;
    a.x_vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.x_stride * (p.x_dtype == DT_F32 ? 4 : 2) % 16 == 0;
    *cerr = p.x_dtype == DT_F32    ? launch_flat<16, true, DT_F32, DT_F32>(tt, tw, a, g, st)
            : p.x_dtype == DT_BF16 ? launch_flat<16, true, DT_F32, DT_BF16>(tt, tw, a, g, st)
                                   : launch_flat<16, true, DT_F32, DT_F16>(tt, tw, a, g, st);
  } else if (g.flat)
    *cerr = g.bn == 16   ? launch_flat<16>(tt, tw, a, g, st)
            : g.bn == 32 ? launch_flat<32>(tt, tw, a, g, st)
            : g.bn == 64 ? launch_flat<64>(tt, tw, a, g, st)
                         : launch_flat<128>(tt, tw, a, g, st);
  else
    *cerr = p.y_dtype == DT_F32    ? launch_wide<DT_F32>(tt, tw, a, g, st)
            : p.y_dtype == DT_BF16 ? launch_wide<DT_BF16>(tt, tw, a, g, st)
                                   : launch_wide<DT_F16>(tt, tw, a, g, st);
  return *cerr == cudaSuccess ? MHMOE_OK : MHMOE_ERR_LAUNCH;
}

}  // namespace mhmoe
