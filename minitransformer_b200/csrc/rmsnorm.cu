// Residual addition + root-mean-square norm, with the MXFP8 copy of the result, and its gradient.
//
//   h = bf16(x + r)                     (h = x without a residual)
//   rstd = 1 / sqrt(mean_k h_k^2 + eps) fp32, from the rounded h: what the next layer adds to and
//                                       what the backward pass reads again
//   y = bf16(h * rstd * gamma)          products in fp32, rounded once
//   copy: E4M3 codes and E8M0 scales of y in 1x32 blocks, bit for bit what mt_quantize_mxfp8 makes of y
//
// Both directions move every element once and do a few operations on it: they are bound by HBM. 8192 x 4096 with a
// residual: h and y 48 us (268 MB, 5.6 TB/s), with row-wise codes 57 us (303 MB, 5.3 TB/s), with both copies 66 us
// (340 MB, 5.2 TB/s); 8192 x 8192 with both copies 147 us. Gradient of 8192 x 8192 with a residual: 84 us (537 MB,
// 6.4 TB/s). A plain copy reaches 6.46 TB/s. One token of 4096 columns: 2.4 us, a launch.
#include "tile_quant.cuh"

namespace mt {

constexpr int RN_MAX_COLS = 32768;

struct RmsNormArgs {
  const __nv_bfloat16 *x, *r;
  int64_t x_stride, r_stride;
  const void* gamma;
  int gamma_f32;
  int64_t rows, cols;
  float eps;
  __nv_bfloat16* h;
  float* rstd;
  __nv_bfloat16* y;
  float* amax;
  int cluster;         // CTAs per panel (rmsnorm_panel_kernel)
  int run;             // consecutive panels that a cluster takes at a time: 1 or 4
  int* status;
  MxTileOut out;
};

// Order in which both forward kernels add the squares of a row, so that a row's result does not depend
// on which of them ran: of eight columns the even and the odd ones in turn; the eight such sums of a
// 64-column segment by a tree over lanes 4, 2, 1 apart; the eight segments of a 512-column group in
// turn; the groups in turn.
__device__ __forceinline__ float sum_squares8(const uint4& w) {
  f32x2_t v = bf16x2_to_f32x2(w.x), s = mul2(v, v);
  v = bf16x2_to_f32x2(w.y); s = fma2(v, v, s);
  v = bf16x2_to_f32x2(w.z); s = fma2(v, v, s);
  v = bf16x2_to_f32x2(w.w); s = fma2(v, v, s);
  float lo, hi;
  unpack2(s, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ float rstd_of(float sum, int64_t cols, float eps) {
  return __frsqrt_rn(__fdiv_rn(sum, (float)cols) + eps);
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {   // the exact sums, rounded once
  uint32_t d;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint4 add_bf16x8(const uint4& a, const uint4& b) {
  return make_uint4(add_bf16x2(a.x, b.x), add_bf16x2(a.y, b.y), add_bf16x2(a.z, b.z), add_bf16x2(a.w, b.w));
}
__device__ __forceinline__ void scale_row8(const uint4& w, float rstd, const float (&g)[8], uint32_t (&y)[4]) {
  const f32x2_t r2 = pack2(rstd, rstd);
  y[0] = f32x2_to_bf16x2(mul2(mul2(bf16x2_to_f32x2(w.x), r2), pack2(g[0], g[1])));
  y[1] = f32x2_to_bf16x2(mul2(mul2(bf16x2_to_f32x2(w.y), r2), pack2(g[2], g[3])));
  y[2] = f32x2_to_bf16x2(mul2(mul2(bf16x2_to_f32x2(w.z), r2), pack2(g[4], g[5])));
  y[3] = f32x2_to_bf16x2(mul2(mul2(bf16x2_to_f32x2(w.w), r2), pack2(g[6], g[7])));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the CTA, the same value (and the same order of additions) in every thread. `slot` holds
// 32 floats; callers that reduce twice alternate between two of them.
__device__ __forceinline__ float block_sum(float v, float* slot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? slot[lane] : 0.0f);
}

// Eight consecutive gammas as fp32.
__device__ __forceinline__ void load_gamma8(const void* gamma, int is_f32, int64_t col, float (&g)[8]) {
  if (is_f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(gamma) + col);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w; g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(gamma) + col));
    g[0] = bf16_lo(a.x); g[1] = bf16_hi(a.x); g[2] = bf16_lo(a.y); g[3] = bf16_hi(a.y);
    g[4] = bf16_lo(a.z); g[5] = bf16_hi(a.z); g[6] = bf16_lo(a.w); g[7] = bf16_hi(a.w);
  }
}

// Sum of squares of the row that the CTA holds, the same in every thread; one barrier. `seg4` belongs to this row until
// the barrier of the next one.
template <int V>
__device__ __forceinline__ float rmsnorm_row_sum(const uint4 (&w)[V], float4* seg4) {
  float* seg = reinterpret_cast<float*>(seg4);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float ss = sum_squares8(w[i]);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    if ((threadIdx.x & 7) == 0) seg[(i * blockDim.x + threadIdx.x) >> 3] = ss;   // zeros beyond the row
  }
  __syncthreads();
  const int groups = (int)(V * blockDim.x) >> 6;   // blockDim is a multiple of 64
  float total = 0.0f;
#pragma unroll 4
  for (int j = 0; j < groups; ++j) {
    const float4 p = seg4[2 * j], u = seg4[2 * j + 1];
    total += ((((((p.x + p.y) + p.z) + p.w) + u.x) + u.y) + u.z) + u.w;
  }
  return total;
}
// Scales of rows that the GEMM layout pads to 128.
__device__ __forceinline__ void rmsnorm_pad_row(const MxTileOut& o, int64_t row) {
  uint8_t* cell = o.s_swz + (row >> 7) * o.kc_row * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
  for (int64_t c = threadIdx.x; c < o.kc_row; c += blockDim.x) *reinterpret_cast<uint32_t*>(cell + c * 512) = 0u;
}

// A row in registers, its rstd known: y, codes, scales, and the row's abs-max into am.
template <int V>
__device__ __forceinline__ void rmsnorm_finish_row(const RmsNormArgs& a, const uint4 (&w)[V], int64_t row, float rstd, bool row_words,
                                                   uint32_t& am) {
  const MxTileOut& o = a.out;
  const int tid = threadIdx.x, nvec = (int)(a.cols >> 3);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + tid;
    const bool on = v < nvec;
    float g[8];
    uint32_t yw[4] = {0, 0, 0, 0};
    if (on) {
      load_gamma8(a.gamma, a.gamma_f32, (int64_t)v * 8, g);
      scale_row8(w[i], rstd, g, yw);
      if (a.y != nullptr)
        *reinterpret_cast<uint4*>(a.y + row * a.cols + (int64_t)v * 8) = make_uint4(yw[0], yw[1], yw[2], yw[3]);
    }
    uint32_t m = absmax2(absmax2(yw[0], yw[1]), absmax2(yw[2], yw[3]));
    am = absmax2(am, m);
    if (o.q != nullptr) {
      m = absmax2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = absmax2(m, __shfl_xor_sync(0xffffffffu, m, 2));
      uint32_t f;
      uint32_t word = mx_scale(mx_amax_bits(m), f) << (8 * ((tid >> 2) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);      // the four blocks of sixteen lanes
      if (on) {
        const float enc = __uint_as_float(f << 16);
        const f32x2_t enc2 = pack2(enc, enc);
        *reinterpret_cast<uint2*>(o.q + row * a.cols + (int64_t)v * 8) =
            make_uint2(e4m3x4_from_words(yw[0], yw[1], enc2), e4m3x4_from_words(yw[2], yw[3], enc2));
        if ((v & 15) == 0) {
          const int kb = v >> 2, n = min(4, (nvec >> 2) - kb);
          mx_store_scale_word(word, n, n == 4 && row_words, o.s + row * o.s_stride + kb, o.s_swz, (uint32_t)row, kb, (uint32_t)o.kc_row);
        }
      }
    }
  }
  if (o.s_swz != nullptr)   // blocks beyond the row, up to the padded chunk count
    for (int64_t kb = (a.cols >> 5) + tid; kb < o.kc_row * 4; kb += blockDim.x)
      o.s_swz[((row >> 7) * o.kc_row + (kb >> 2)) * 512 + sf_chunk_offset((int)(row & 127), (int)kb)] = 0;
}
__device__ __forceinline__ void rmsnorm_publish_amax(const RmsNormArgs& a, uint32_t am) {
  if (a.amax != nullptr) {
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(absmax2_to_float(am)));
    if ((threadIdx.x & 31) == 0 && bits != 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), bits);
  }
}

// Rows without a transposed copy. One CTA per row, V vectors of 8 columns per thread (vector
// i * blockDim + thread). The row stays in registers between the sum and the scaling. A 1x32 block is
// four adjacent lanes. CTAs beyond the last row fill the padding of the GEMM-layout scales with zeros.
template <int V, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) rmsnorm_rows_kernel(const RmsNormArgs a) {
  __shared__ float4 seg4[RN_MAX_COLS / 256];   // sums of 64-column segments, a group being two of these
  const MxTileOut& o = a.out;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, nvec = (int)(a.cols >> 3);
  pdl_trigger();
  pdl_wait();
  if (row >= a.rows) {
    rmsnorm_pad_row(o, row);
    return;
  }
  uint4 w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + tid;
    w[i] = make_uint4(0, 0, 0, 0);
    if (v < nvec) {
      w[i] = *reinterpret_cast<const uint4*>(a.x + row * a.x_stride + (int64_t)v * 8);
      if (a.r != nullptr) w[i] = add_bf16x8(w[i], *reinterpret_cast<const uint4*>(a.r + row * a.r_stride + (int64_t)v * 8));
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + tid;
    if (a.h != nullptr && v < nvec) *reinterpret_cast<uint4*>(a.h + row * a.cols + (int64_t)v * 8) = w[i];
  }
  const float rstd = rstd_of(rmsnorm_row_sum<V>(w, seg4), a.cols, a.eps);
  if (tid == 0 && a.rstd != nullptr) a.rstd[row] = rstd;
  uint32_t am = 0;
  rmsnorm_finish_row<V>(a, w, row, rstd, mx_word_aligned(o.s, o.s_stride), am);
  rmsnorm_publish_amax(a, am);
}

// With a transposed copy. A cluster of C CTAs owns a panel of 32 rows, each CTA 64 columns per warp of it, each
// warp one 32 x 64 tile (layout of tile_quant.cuh). x is read once: the sums of squares of 512-column groups go to
// every CTA of the cluster through distributed shared memory, then the tiles are scaled and quantized both
// ways in registers. The clusters are persistent: a warp asks for its tiles of the next panel (TMA, one mbarrier
// per warp) as soon as it holds the present ones, so that they arrive while it waits for its cluster,
// quantizes and stores. The sums travel by st.async onto an mbarrier of the receiving CTA: a cluster barrier's
// release would wait for the stores of h, y and the copies as well (81 us instead of 69 on 8192 x 4096). h is stored
// before the exchange, y and the copies after it. Three CTAs per SM at 80 registers: 77 us instead of 66. Two sets of sums and barriers alternate: a
// CTA that has received all sums of panel n + 1 knows that everybody has read those of panel n.
// Panels beyond the last row (up to 128 rows) and the last panel write the scales' padding.
constexpr int RN_PANEL_MAX_COLS = 8192;
constexpr int RN_PANEL_WARPS = 8, RN_PANEL_RANKS = RN_PANEL_MAX_COLS / (64 * RN_PANEL_WARPS);

// Bounded wait for data that other CTAs of the cluster send onto a barrier of this one.
__device__ __forceinline__ void cluster_data_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
  const uint64_t t0 = global_timer_ns();
  uint32_t spins = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return;
    if ((++spins & 255u) == 0) {
      if (*abort_flag != 0) return;
      if (global_timer_ns() - t0 > 2000000000ull) {
        *abort_flag = 1;
        atomicOr(status, DS_QUANT_WAIT);
        return;
      }
    }
  }
}

template <bool kRagged>
__global__ void __launch_bounds__(32 * RN_PANEL_WARPS, 2)
    rmsnorm_panel_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_r, const RmsNormArgs a) {
  constexpr int WARPS = RN_PANEL_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  __shared__ float seg[WARPS][32];                         // this CTA's segments
  __shared__ float grp[2][RN_PANEL_RANKS][32];             // the panel's groups, one per CTA; panels alternate
  __shared__ __align__(16) uint8_t s_row[32][WARPS * 2];
  __shared__ uint64_t bars[WARPS], empty[WARPS], xbar[2];
  __shared__ int abort_flag;
  const MxTileOut& o = a.out;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int cg = lane & 7, rg = lane >> 3;
  const int rank = (int)cluster_ctarank(), ranks = a.cluster;
  const int clusters = gridDim.x / ranks, panels = (int)((a.rows + 127) / 128 * 4);
  const int64_t cta_col0 = (int64_t)rank * warps * 64, col0 = cta_col0 + warp * 64, c = col0 + cg * 8;
  const bool w_ok = col0 < a.cols;                         // uniform for the warp
  uint8_t* buf = smem + warp * 2 * MX_TILE_BYTES;
  const bool row_words = mx_word_aligned(o.s, o.s_stride), col_words = mx_word_aligned(o.s_t, o.s_t_stride);
  const bool pad_cols = rank == ranks - 1 && (a.cols & 511) != 0;   // GEMM-layout scales go beyond the last column
  if (tid == 0) {
    abort_flag = 0;
    mbar_init(&xbar[0], 1);
    mbar_init(&xbar[1], 1);
  }
  if (lane == 0) {
    mbar_init(&bars[warp], 1);
    mbar_init(&empty[warp], 32);
  }
  mbar_fence_init();
  __syncthreads();
  if (ranks > 1) {   // every CTA's barriers exist before anything is sent to it
    cluster_arrive();
    cluster_wait();
  }
  pdl_wait();
  auto fetch = [&](int panel) {
    mbar_expect_tx(&bars[warp], (a.r != nullptr ? 2 : 1) * MX_TILE_BYTES);
    tma_load_2d(buf, &map_x, &bars[warp], (int32_t)col0, panel * 32);
    if (a.r != nullptr) tma_load_2d(buf + MX_TILE_BYTES, &map_r, &bars[warp], (int32_t)col0, panel * 32);
  };
  // panels are a multiple of four: a run is whole
  auto after = [&](int panel) { return (panel + 1) % a.run != 0 ? panel + 1 : panel + 1 + (clusters - 1) * a.run; };
  const int first = (int)blockIdx.x / ranks * a.run;
  if (lane == 0 && w_ok && first < panels) fetch(first);
  uint32_t turn = 0, col_word[2] = {0, 0};
  for (int panel = first; panel < panels; panel = after(panel), ++turn) {
    const int64_t row0 = (int64_t)panel * 32, r0 = row0 + rg * 8;
    const int nrow = c < a.cols ? mx_valid_rows(a.rows, r0) : 0;
    uint4 w[8];
    if (w_ok) {
      // on expiry the status word tells; the warp goes on with what is there, so that nobody waits for it
      mbar_wait_bounded(&bars[warp], turn & 1, &abort_flag, a.status, DS_QUANT_WAIT);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = mx_tile_row(buf, i);
      if (a.r != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = add_bf16x8(w[i], mx_tile_row(buf + MX_TILE_BYTES, i));
      }
      mx_release_tile(&empty[warp], turn & 1, &abort_flag, a.status);
      if (lane == 0 && after(panel) < panels) fetch(after(panel));
      if (a.h != nullptr) {
        __nv_bfloat16* p = a.h + r0 * a.cols + c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < nrow) *reinterpret_cast<uint4*>(p) = w[i];
          p += a.cols;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = sum_squares8(w[i]);
    // eight row sums over eight lanes: every exchange halves the rows a lane still carries
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float send = (cg & 4) ? v[i] : v[i + 4], keep = (cg & 4) ? v[i + 4] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 4);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float send = (cg & 2) ? v[i] : v[i + 2], keep = (cg & 2) ? v[i + 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 2);
    }
    {
      const float send = (cg & 1) ? v[0] : v[1], keep = (cg & 1) ? v[1] : v[0];
      v[0] = keep + __shfl_xor_sync(0xffffffffu, send, 1);
    }
    seg[warp][lane] = v[0];       // lane l: row l of the panel
    __syncthreads();
    {
      float sum = seg[0][lane];
#pragma unroll
      for (int j = 1; j < WARPS; ++j)
        if (j < warps) sum += seg[j][lane];
      float* mine = &grp[turn & 1][rank][lane];
      if (ranks == 1) {
        if (warp == 0) *mine = sum;
      } else {   // the warps share the receivers
        if (tid == 0) mbar_expect_tx(&xbar[turn & 1], (uint32_t)ranks * 128);
        for (int r = warp; r < ranks; r += warps)
          asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
                       ::"r"(map_to_cta(smem_u32(mine), (uint32_t)r)), "r"(__float_as_uint(sum)),
                         "r"(map_to_cta(smem_u32(&xbar[turn & 1]), (uint32_t)r)) : "memory");
      }
    }
    if (ranks > 1) cluster_data_wait(&xbar[turn & 1], (turn >> 1) & 1, &abort_flag, a.status);
    else __syncthreads();
    float total = 0.0f;
#pragma unroll 4
    for (int j = 0; j < ranks; ++j) total += grp[turn & 1][j][lane];
    const bool live = row0 + lane < a.rows;
    const float rstd_l = live ? rstd_of(total, a.cols, a.eps) : 0.0f;
    if (rank == 0 && warp == 0 && a.rstd != nullptr && live) a.rstd[row0 + lane] = rstd_l;
    if (w_ok) {
      float g[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = 0.0f;
      if (c < a.cols) load_gamma8(a.gamma, a.gamma_f32, c, g);
      uint32_t yw[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i)    // (rows beyond the last are zeros)
        scale_row8(w[i], __shfl_sync(0xffffffffu, rstd_l, rg * 8 + i), g, yw[i]);
      if (a.y != nullptr) {
        __nv_bfloat16* p = a.y + r0 * a.cols + c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < nrow) *reinterpret_cast<uint4*>(p) = make_uint4(yw[i][0], yw[i][1], yw[i][2], yw[i][3]);
          p += a.cols;
        }
      }
      if (a.amax != nullptr) {
        uint32_t am = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) am = absmax2(am, absmax2(absmax2(yw[i][0], yw[i][1]), absmax2(yw[i][2], yw[i][3])));
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(absmax2_to_float(am)));
        if (lane == 0 && bits != 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), bits);
      }
      const MxTileScales sc = mx_tile_store<kRagged>(o, yw, row0, col0, a.cols);
      const uint32_t f0 = (uint32_t)col0 + cg * 8 + rg * 2;    // two adjacent features: both inside or both outside
#pragma unroll
      for (int j = 0; j < 2; ++j)
        s_row[rg * 8 + (lane & 3) * 2 + j][warp * 2 + (cg >> 2)] = static_cast<uint8_t>(sc.row[j]);
      if (f0 < a.cols && a.run == 4) {
        // a lane has the same features in every panel: four scales of each make a word
#pragma unroll
        for (int j = 0; j < 2; ++j) col_word[j] = __funnelshift_r(col_word[j], sc.col[j], 8);
        if ((panel & 3) == 3) {
          const uint32_t b0 = (uint32_t)panel - 3;
          const int n = (int)min((int64_t)4, ((o.rows + 31) >> 5) - b0);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mx_store_scale_word(col_word[j], n, n == 4 && col_words, o.s_t + ((f0 + j) * o.s_t_stride + b0), nullptr, f0 + j, b0, 0);
            if (o.s_t_swz != nullptr)   // (panels without a row: zeros)
              *reinterpret_cast<uint32_t*>(o.s_t_swz + mx_swz_offset(f0 + j, b0, (uint32_t)o.kc_col)) = col_word[j];
          }
        }
      } else if (f0 < a.cols) {
        if (row0 < o.rows) {
          uint8_t* lin = o.s_t + (f0 * o.s_t_stride + panel);
          lin[0] = static_cast<uint8_t>(sc.col[0]);
          lin[o.s_t_stride] = static_cast<uint8_t>(sc.col[1]);
        }
        if (o.s_t_swz != nullptr) {
          uint8_t* swz = o.s_t_swz + mx_swz_offset(f0, panel, (uint32_t)o.kc_col);
          swz[0] = static_cast<uint8_t>(sc.col[0]);
          swz[16] = static_cast<uint8_t>(sc.col[1]);
        }
      }
    }
    __syncthreads();
    if (warp * 2 < warps) {
      // row scales: a word (four blocks) per row and pair of warps
      const uint32_t r = (uint32_t)row0 + lane, b0 = (uint32_t)(cta_col0 >> 5) + warp * 4;
      const int n = min(min(4, warps * 2 - warp * 4), (int)(a.cols >> 5) - (int)b0);
      if (n > 0)
        mx_store_scale_word(*reinterpret_cast<const uint32_t*>(&s_row[lane][warp * 4]), n, n == 4 && row_words,
                            live ? o.s + (r * o.s_stride + b0) : nullptr, o.s_swz, r, b0, (uint32_t)o.kc_row);
    }
    if (pad_cols) {
      mx_pad_row_scales(o, row0, 32, tid, blockDim.x);
      mx_pad_col_features(o, panel, tid, blockDim.x);
    }
    if (panel == panels - 1) {
      const int64_t c0 = min(cta_col0, a.cols), c1 = min(c0 + (int64_t)warps * 64, a.cols);
      if (c1 > c0) mx_pad_col_blocks(o, panel + 1, c0, c1, tid, blockDim.x);
      if (pad_cols) mx_pad_col_blocks(o, panel + 1, a.cols, (a.cols + 127) / 128 * 128, tid, blockDim.x);
    }
  }
  if (ranks > 1) {   // nobody leaves while something may still be on its way to it
    cluster_arrive();
    cluster_wait();
  }
  // only now: with clusters of the next kernel taking their places earlier, calls in a row took 104 us instead of 81
  pdl_trigger();
}

// Four panels in a row where that evens out over the clusters as well as single ones: the transposed scales then leave
// as words instead of bytes (a sector each). 8192 x 4096, y and both copies: 57 -> 51 us without a residual, 70 -> 69 with.
static int rn_panel_run(int64_t panels, int64_t clusters) {
  const int64_t apart = (panels + clusters - 1) / clusters, runs = (panels / 4 + clusters - 1) / clusters * 4;
  return runs * 20 <= apart * 21 ? 4 : 1;
}

// 512 columns (8 warps) per CTA, up to 16 CTAs per panel, two CTAs per SM. (Rows beyond 4096 columns by 1024-column CTAs,
// one per SM, in clusters of up to 8: 156 us instead of 147 on 8192 x 8192, 89 / 75 on 8192 x 4608, 100 / 104 on 8192 x 6144.)
template <bool kRagged>
static int rmsnorm_panel(RmsNormArgs& a, cudaStream_t st) {
  a.status = device_status_ptr();
  if (!a.status) return fail(MT_ERR_CUDA, "device status word not reachable");
  const int ranks = (int)((a.cols + 511) / 512), warps = ranks > 1 ? RN_PANEL_WARPS : (int)((a.cols + 63) / 64);
  CUtensorMap mx, mr;
  int rc = mx_tile_map(&mx, a.x, a.rows, a.cols, a.x_stride);
  if (rc == MT_OK) rc = a.r ? mx_tile_map(&mr, a.r, a.rows, a.cols, a.r_stride) : (mr = mx, MT_OK);
  if (rc != MT_OK) return rc;
  auto kern = rmsnorm_panel_kernel<kRagged>;
  const size_t smem = (size_t)warps * 2 * MX_TILE_BYTES + 128;
  static int max_clusters_dev[MT_MAX_DEVICES][RN_PANEL_RANKS + 1] = {};   // by cluster size, for the full number of warps
  int& max_clusters = max_clusters_dev[current_device_slot()][ranks];
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  if (max_clusters <= 0) {
    const size_t most = (size_t)RN_PANEL_WARPS * 2 * MX_TILE_BYTES + 128;
    MT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    MT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cfg.gridDim = dim3(ranks * 1024);
    cfg.blockDim = dim3(32 * RN_PANEL_WARPS);
    cfg.dynamicSmemBytes = most;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) { cudaGetLastError(); n = mx_sm_count() / ranks; }
    max_clusters = n > 0 ? n : 1;
  }
  const int64_t panels = (a.rows + 127) / 128 * 4;
  a.cluster = ranks;
  a.run = rn_panel_run(panels, max_clusters);
  const int64_t runs = panels / a.run;
  cfg.gridDim = dim3((unsigned)((runs < max_clusters ? runs : max_clusters) * ranks));
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const RmsNormArgs& ca = a;
  MT_CUDA(cudaLaunchKernelEx(&cfg, kern, mx, mr, ca));
  return MT_OK;
}

// ---- gradient ----
//   a = dy * gamma, xhat = h * rstd
//   dx = rstd * (a - xhat * mean_k(a * xhat)) (+ dres),   dgamma = sum_rows dy * xhat
constexpr int RN_RING_STAGES = 8;
constexpr int RN_RING_MAX_COLS = 16384;
constexpr int RN_RING_BYTES = 200 * 1024;   // shared memory per SM that the rings share

struct RmsNormGradArgs {
  const __nv_bfloat16 *dy, *h, *dres;
  int64_t dy_stride, h_stride, dres_stride;
  const void* gamma;
  int gamma_f32;
  const float* rstd;
  int64_t rows, cols;
  __nv_bfloat16* dx;
  float* partial;   // [gridDim.x, cols]
  int stages;       // of the ring
  int* status;
};

// Persistent CTAs over rows; a thread keeps the same columns for every row, so the column sums
// of dgamma stay in its registers and are written once per CTA. The partial sums are then added
// in a fixed order (rmsnorm_dgamma_kernel): the result does not depend on scheduling.
template <int V>
__global__ void __launch_bounds__(1024) rmsnorm_grad_kernel(const RmsNormGradArgs a) {
  __shared__ float slot[2][32];
  const int tid = threadIdx.x, nvec = (int)(a.cols >> 3);
  pdl_trigger();
  pdl_wait();
  float acc[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    uint4 dy[V], h[V];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = i * blockDim.x + tid;
      dy[i] = h[i] = make_uint4(0, 0, 0, 0);
      if (v < nvec) {
        dy[i] = *reinterpret_cast<const uint4*>(a.dy + row * a.dy_stride + (int64_t)v * 8);
        h[i] = *reinterpret_cast<const uint4*>(a.h + row * a.h_stride + (int64_t)v * 8);
      }
    }
    const float rstd = a.rstd[row];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = i * blockDim.x + tid;
      if (v >= nvec) continue;
      float g[8];
      load_gamma8(a.gamma, a.gamma_f32, (int64_t)v * 8, g);
      const uint32_t d[4] = {dy[i].x, dy[i].y, dy[i].z, dy[i].w}, x[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dot = fmaf(bf16_lo(d[j]) * g[2 * j], bf16_lo(x[j]), dot);
        dot = fmaf(bf16_hi(d[j]) * g[2 * j + 1], bf16_hi(x[j]), dot);
      }
    }
    dot = block_sum(dot, slot[turn]);
    // xhat * mean(a * xhat) = h * rstd * (rstd * dot / cols)
    const float c = rstd * rstd * __fdiv_rn(dot, (float)a.cols);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = i * blockDim.x + tid;
      if (v >= nvec) continue;
      float g[8];
      load_gamma8(a.gamma, a.gamma_f32, (int64_t)v * 8, g);
      uint4 rs = make_uint4(0, 0, 0, 0);
      if (a.dres != nullptr) rs = *reinterpret_cast<const uint4*>(a.dres + row * a.dres_stride + (int64_t)v * 8);
      const uint32_t d[4] = {dy[i].x, dy[i].y, dy[i].z, dy[i].w}, x[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
      const uint32_t r[4] = {rs.x, rs.y, rs.z, rs.w};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d0 = bf16_lo(d[j]), d1 = bf16_hi(d[j]), x0 = bf16_lo(x[j]), x1 = bf16_hi(x[j]);
        const float o0 = fmaf(rstd, fmaf(d0, g[2 * j], -x0 * c), bf16_lo(r[j]));
        const float o1 = fmaf(rstd, fmaf(d1, g[2 * j + 1], -x1 * c), bf16_hi(r[j]));
        o[j] = f32x2_to_bf16x2(pack2(o0, o1));
        acc[i][2 * j] = fmaf(d0, x0 * rstd, acc[i][2 * j]);
        acc[i][2 * j + 1] = fmaf(d1, x1 * rstd, acc[i][2 * j + 1]);
      }
      *reinterpret_cast<uint4*>(a.dx + row * a.cols + (int64_t)v * 8) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + tid;
    if (v >= nvec) continue;
    float4* p = reinterpret_cast<float4*>(a.partial + (int64_t)blockIdx.x * a.cols + (int64_t)v * 8);
    p[0] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    p[1] = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
  }
}

// The same with the rows on their way ahead of time (138 -> 84 us on 8192 x 8192 with a residual): a ring of shared-memory stages, each one row of dy, h and dres
// fetched by bulk copies (one mbarrier per stage). A row needs one barrier (inside the sum); once a thread
// has passed the one of row n + 1, everybody is done with row n, and its stage is filled again.
template <int V, int kMaxThreads, int kMinCtas>
__global__ void __launch_bounds__(kMaxThreads, kMinCtas) rmsnorm_grad_ring_kernel(const RmsNormGradArgs a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float slot[2][32];
  __shared__ uint64_t full[RN_RING_STAGES];
  __shared__ int abort_flag;
  const int tid = threadIdx.x, nvec = (int)(a.cols >> 3), stages = a.stages;
  const uint32_t row_bytes = (uint32_t)a.cols * 2, stage_bytes = row_bytes * (a.dres != nullptr ? 3 : 2);
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  auto fetch = [&](int64_t row, int s) {
    uint8_t* p = ring + s * stage_bytes;
    mbar_expect_tx(&full[s], stage_bytes);
    bulk_load_1d(p, a.dy + row * a.dy_stride, row_bytes, &full[s]);
    bulk_load_1d(p + row_bytes, a.h + row * a.h_stride, row_bytes, &full[s]);
    if (a.dres != nullptr) bulk_load_1d(p + 2 * row_bytes, a.dres + row * a.dres_stride, row_bytes, &full[s]);
  };
  if (tid == 0)
    for (int i = 0; i < stages; ++i) {
      const int64_t row = blockIdx.x + (int64_t)i * gridDim.x;
      if (row < a.rows) fetch(row, i);
    }
  float g[V][8], acc[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[i][j] = acc[i][j] = 0.0f;
    if (i * (int)blockDim.x + tid < nvec) load_gamma8(a.gamma, a.gamma_f32, (int64_t)(i * blockDim.x + tid) * 8, g[i]);
  }
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  int s = 0, turn = 0, last = 0;
  uint32_t ph = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const uint8_t* p = ring + s * stage_bytes;
    const float rstd = a.rstd[row];
    // on expiry the status word tells; the CTA goes on with what is there
    mbar_wait_bounded(&full[s], ph, &abort_flag, a.status, DS_QUANT_WAIT);
    f32x2_t dot2 = pack2(0.0f, 0.0f);
    uint4 dy[V], h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = i * blockDim.x + tid;
      dy[i] = h[i] = make_uint4(0, 0, 0, 0);
      if (v < nvec) {
        dy[i] = *reinterpret_cast<const uint4*>(p + v * 16);
        h[i] = *reinterpret_cast<const uint4*>(p + row_bytes + v * 16);
      }
      const uint32_t d[4] = {dy[i].x, dy[i].y, dy[i].z, dy[i].w}, x[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        dot2 = fma2(mul2(bf16x2_to_f32x2(d[j]), pack2(g[i][2 * j], g[i][2 * j + 1])), bf16x2_to_f32x2(x[j]), dot2);
    }
    float d0, d1;
    unpack2(dot2, d0, d1);
    fence_proxy_async_smem();                // this thread's reads of the row before come ahead of the copies into its stage
    const float dot = block_sum(d0 + d1, slot[turn]);
    if (tid == 0 && row != blockIdx.x) {     // the row before this one is done with
      const int64_t next = row + (int64_t)(stages - 1) * gridDim.x;
      if (next < a.rows) fetch(next, last);
    }
    const float c = -rstd * rstd * (dot * inv);
    const f32x2_t c2 = pack2(c, c), r2 = pack2(rstd, rstd);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = i * blockDim.x + tid;
      if (v < nvec) {
        uint4 rs = make_uint4(0, 0, 0, 0);
        if (a.dres != nullptr) rs = *reinterpret_cast<const uint4*>(p + 2 * row_bytes + v * 16);
        const uint32_t d[4] = {dy[i].x, dy[i].y, dy[i].z, dy[i].w}, x[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
        const uint32_t r[4] = {rs.x, rs.y, rs.z, rs.w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x2_t dv = bf16x2_to_f32x2(d[j]), xv = bf16x2_to_f32x2(x[j]), gv = pack2(g[i][2 * j], g[i][2 * j + 1]);
          o[j] = f32x2_to_bf16x2(fma2(r2, fma2(dv, gv, mul2(xv, c2)), bf16x2_to_f32x2(r[j])));
          const f32x2_t sum = fma2(dv, mul2(xv, r2), pack2(acc[i][2 * j], acc[i][2 * j + 1]));
          unpack2(sum, acc[i][2 * j], acc[i][2 * j + 1]);
        }
        *reinterpret_cast<uint4*>(a.dx + row * a.cols + (int64_t)v * 8) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    last = s;
    if (++s == stages) { s = 0; ph ^= 1; }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + tid;
    if (v >= nvec) continue;
    float4* q = reinterpret_cast<float4*>(a.partial + (int64_t)blockIdx.x * a.cols + (int64_t)v * 8);
    q[0] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    q[1] = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
  }
  pdl_trigger();
}

// dgamma[k] = sum of `parts` partial rows, in a fixed order. 32 columns per CTA, one row group per warp.
constexpr int RN_SUM_GROUPS = 16;
__global__ void __launch_bounds__(32 * RN_SUM_GROUPS) rmsnorm_dgamma_kernel(const float* partial, int parts, int64_t cols,
                                                                           float* dgamma) {
  __shared__ float sum[RN_SUM_GROUPS][32];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + lane;
  pdl_trigger();
  pdl_wait();
  float v = 0.0f;
  if (col < cols)
#pragma unroll 4
    for (int p = grp; p < parts; p += RN_SUM_GROUPS) v += partial[(int64_t)p * cols + col];
  sum[grp][lane] = v;
  __syncthreads();
  if (grp == 0 && col < cols) {
#pragma unroll
    for (int i = 1; i < RN_SUM_GROUPS; ++i) v += sum[i][lane];
    dgamma[col] = v;
  }
}

// Threads per row for V vectors per thread (a multiple of 64: whole groups of four segments).
static int rn_threads(int64_t cols, int V) { return (int)(((cols / 8 + V - 1) / V + 63) / 64 * 64); }

// CTAs per SM that share its memory for their rings, one vector of 8 columns per thread: two CTAs of 512 threads on
// 4096 columns, one of 1024 on 8192. With two vectors per thread (two CTAs of 512) the gradient of 8192 x 8192 took
// 119 us instead of 84. Beyond 8192 columns four vectors per thread of one CTA of 512: 4096 x 16384 takes 118 us with a
// residual and 89 without (4.5 TB/s), though 124 bytes of it spill; 126 and 110 us with two vectors per thread of 1024, which
// leave it 64 registers.
static int rn_ring_ctas_per_sm(int64_t cols) { return cols <= 2048 ? 4 : cols <= 4096 ? 2 : 1; }
static int rn_ring_stages(int64_t cols, int64_t stage) {
  const int64_t n = RN_RING_BYTES / rn_ring_ctas_per_sm(cols) / stage;
  return (int)(n < RN_RING_STAGES ? n : RN_RING_STAGES);
}
static int rn_grad_ctas(int64_t rows, int64_t cols) {
  const int64_t most = (int64_t)rn_ring_ctas_per_sm(cols) * mx_sm_count();
  return (int)(rows < most ? rows : most);
}
template <int V, int kMaxThreads, int kMinCtas>
static int launch_grad_ring(RmsNormGradArgs& a, int ctas, cudaStream_t st) {
  auto kern = rmsnorm_grad_ring_kernel<V, kMaxThreads, kMinCtas>;
  static bool attr_set[MT_MAX_DEVICES] = {};
  const int slot = current_device_slot();
  if (!attr_set[slot]) {
    MT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RN_RING_BYTES));
    attr_set[slot] = true;
  }
  const int64_t stage = a.cols * (a.dres ? 6 : 4);
  a.stages = rn_ring_stages(a.cols, stage);
  a.status = device_status_ptr();
  if (!a.status) return fail(MT_ERR_CUDA, "device status word not reachable");
  MT_CUDA(launch_pdl(kern, dim3(ctas), dim3(rn_threads(a.cols, V)), (size_t)(a.stages * stage), st, a));
  return MT_OK;
}
static bool row_aligned(const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; }

}  // namespace mt

extern "C" int mt_rmsnorm_forward(const void* x, int64_t x_stride, const void* residual, int64_t r_stride, const void* gamma,
                                  int gamma_dtype, int64_t rows, int64_t cols, float eps, void* h, float* rstd, void* y,
                                  float* amax, uint8_t* q, uint8_t* s, int64_t s_stride, uint8_t* s_swz, uint8_t* q_t,
                                  uint8_t* s_t, int64_t s_t_stride, uint8_t* s_t_swz, mt_stream_t stream) {
  using namespace mt;
  const char* name = "mt_rmsnorm_forward";
  MT_REQUIRE(rows >= 0 && cols > 0 && cols <= RN_MAX_COLS, "%s: cols (%lld) must be within [1, %d]", name, (long long)cols, RN_MAX_COLS);
  MT_REQUIRE(cols % 8 == 0, "%s: cols (%lld) must be a multiple of 8", name, (long long)cols);
  MT_REQUIRE(gamma_dtype == MT_BF16 || gamma_dtype == MT_F32, "%s: gamma dtype %d not supported", name, gamma_dtype);
  MT_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", name);
  MT_REQUIRE(rows < (int64_t)1 << 30, "%s: too many rows", name);
  if (rows == 0) return MT_OK;
  MT_REQUIRE(x && gamma, "%s: null x / gamma", name);
  MT_REQUIRE(x_stride >= cols && row_aligned(x, x_stride), "%s: x needs 16-byte aligned rows", name);
  MT_REQUIRE(!residual || (r_stride >= cols && row_aligned(residual, r_stride)), "%s: residual needs 16-byte aligned rows", name);
  MT_REQUIRE(!residual || h, "%s: a residual needs an output for the sum", name);
  MT_REQUIRE(residual || !h, "%s: without a residual there is no sum to write", name);
  MT_REQUIRE(!h || ((h != x || x_stride == cols) && (h != residual || r_stride == cols)),
             "%s: h in the place of an input needs that input's row stride to be cols", name);
  MT_REQUIRE(aligned16(gamma) && aligned16(h) && aligned16(y), "%s: pointers must be 16-byte aligned", name);
  int rc = mx_outputs_ok(name, rows, cols, q, s, s_stride, s_swz, q_t, s_t, s_t_stride, s_t_swz);
  if (rc != MT_OK) return rc;
  if (q_t && cols > RN_PANEL_MAX_COLS)
    return fail(MT_ERR_UNSUPPORTED, "%s: a transposed copy of more than %d columns: quantize y instead", name, RN_PANEL_MAX_COLS);
  RmsNormArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x); a.x_stride = x_stride;
  a.r = static_cast<const __nv_bfloat16*>(residual); a.r_stride = r_stride;
  a.gamma = gamma; a.gamma_f32 = gamma_dtype == MT_F32;
  a.rows = rows; a.cols = cols; a.eps = eps;
  a.h = static_cast<__nv_bfloat16*>(h); a.rstd = rstd; a.y = static_cast<__nv_bfloat16*>(y); a.amax = amax;
  a.out = {q, s, s_swz, q_t, s_t, s_t_swz, rows, cols, s_stride, s_t_stride, mx_padded_chunks(cols / 32),
           mx_padded_chunks((rows + 31) / 32)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t padded = (rows + 127) / 128 * 128;
  if (q_t) return rows % 8 ? rmsnorm_panel<true>(a, st) : rmsnorm_panel<false>(a, st);
  const dim3 grid((unsigned)(s_swz ? padded : rows));
  // Few rows: one vector per thread, the shortest way through a row. Many rows: four vectors per thread, so that more
  // rows (and bytes) are in flight per SM. 8192 x 4096 with one vector / with four / with a ring of rows in shared
  // memory as in the gradient: h and y 54 / 48 / 53 us, y alone 47 / 26 / 46 us, h, y and codes 65 / 57 / 64 us.
  const bool many = rows >= 4 * mx_sm_count();
  if (cols <= 8192 && !many) MT_CUDA(launch_pdl(rmsnorm_rows_kernel<1, 1024>, grid, dim3(rn_threads(cols, 1)), 0, st, a));
  else if (cols <= 8192) MT_CUDA(launch_pdl(rmsnorm_rows_kernel<4, 256>, grid, dim3(rn_threads(cols, 4)), 0, st, a));
  else MT_CUDA(launch_pdl(rmsnorm_rows_kernel<4, 1024>, grid, dim3(rn_threads(cols, 4)), 0, st, a));
  return MT_OK;
}

extern "C" int64_t mt_rmsnorm_backward_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (int64_t)mt::rn_grad_ctas(rows, cols) * cols * 4;
}

extern "C" int mt_rmsnorm_backward(const void* dy, int64_t dy_stride, const void* h, int64_t h_stride, const void* gamma,
                                   int gamma_dtype, const float* rstd, const void* dres, int64_t dres_stride, int64_t rows,
                                   int64_t cols, void* dx, float* dgamma, void* workspace, int64_t workspace_bytes,
                                   mt_stream_t stream) {
  using namespace mt;
  const char* name = "mt_rmsnorm_backward";
  MT_REQUIRE(rows >= 0 && cols > 0 && cols <= RN_MAX_COLS, "%s: cols (%lld) must be within [1, %d]", name, (long long)cols, RN_MAX_COLS);
  MT_REQUIRE(cols % 8 == 0, "%s: cols (%lld) must be a multiple of 8", name, (long long)cols);
  MT_REQUIRE(gamma_dtype == MT_BF16 || gamma_dtype == MT_F32, "%s: gamma dtype %d not supported", name, gamma_dtype);
  MT_REQUIRE(dgamma && aligned16(dgamma), "%s: dgamma must be given, 16-byte aligned", name);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {   // no rows: the sum over them is zero
    MT_CUDA(cudaMemsetAsync(dgamma, 0, (size_t)cols * 4, st));
    return MT_OK;
  }
  MT_REQUIRE(dy && h && gamma && rstd && dx, "%s: null pointer", name);
  MT_REQUIRE(dy_stride >= cols && row_aligned(dy, dy_stride) && h_stride >= cols && row_aligned(h, h_stride),
             "%s: dy and h need 16-byte aligned rows", name);
  MT_REQUIRE(!dres || (dres_stride >= cols && row_aligned(dres, dres_stride)), "%s: dres needs 16-byte aligned rows", name);
  MT_REQUIRE(dx != dres || dres_stride == cols, "%s: dx in the place of dres needs a row stride of cols", name);
  MT_REQUIRE(aligned16(gamma) && aligned16(dx), "%s: pointers must be 16-byte aligned", name);
  MT_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= mt_rmsnorm_backward_workspace(rows, cols),
             "%s: workspace of %lld bytes is too small (mt_rmsnorm_backward_workspace)", name, (long long)workspace_bytes);
  RmsNormGradArgs a{};
  a.dy = static_cast<const __nv_bfloat16*>(dy); a.dy_stride = dy_stride;
  a.h = static_cast<const __nv_bfloat16*>(h); a.h_stride = h_stride;
  a.dres = static_cast<const __nv_bfloat16*>(dres); a.dres_stride = dres_stride;
  a.gamma = gamma; a.gamma_f32 = gamma_dtype == MT_F32; a.rstd = rstd;
  a.rows = rows; a.cols = cols;
  a.dx = static_cast<__nv_bfloat16*>(dx); a.partial = static_cast<float*>(workspace);
  const int ctas = rn_grad_ctas(rows, cols);
  int rc = MT_OK;
  if (cols <= 4096) rc = launch_grad_ring<1, 512, 2>(a, ctas, st);
  else if (cols <= 8192) rc = launch_grad_ring<1, 1024, 1>(a, ctas, st);
  else if (cols <= RN_RING_MAX_COLS) rc = launch_grad_ring<4, 512, 1>(a, ctas, st);
  else MT_CUDA(launch_pdl(rmsnorm_grad_kernel<4>, dim3(ctas), dim3(rn_threads(cols, 4)), 0, st, a));   // two rows do not fit
  if (rc != MT_OK) return rc;
  MT_CUDA(launch_pdl(rmsnorm_dgamma_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(32 * RN_SUM_GROUPS), 0, st,
                     static_cast<const float*>(workspace), ctas, cols, dgamma));
  return MT_OK;
}
