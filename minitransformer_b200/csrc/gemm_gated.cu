// Gated projection for sm_100a: h = act(x Wg^T) * (x Wu^T) from block-scaled operands (MXFP8 or
// NVFP4, K-major), both products, the activation and the product of the two in one kernel.
//
//   [g | u] = alpha * x W^T, W = [Wg; Wu] of 2F rows          fp32 in tensor memory
//   h = bf16(act(g) * u)                                      from the fp32 accumulators
//   on request: bf16 [g | u] (what the backward pass reads), E4M3 codes + E8M0 scales of h by rows
//   (bit for bit mt_quantize_mxfp8 of h), max |h|
//
// Two kernels, by the number of rows M of x:
//
// gemm_gated_rows_kernel (decoding, short prompts): the weights dominate, so they take the 128-row side of the
// MMA and the tokens the column side (32 to 128 of them): the tensor time shrinks with the tokens and the pipeline
// holds almost only weight bytes. A CTA owns 128 features; its accumulators [128 features x tokens] put one
// feature in each lane, so a warp owns one 1x32 block of h for every token. Bound by reading the weights: one
// token on 14336 x 4096 takes 20.9 us (MXFP8; 121 MB, 18.8 us at the measured copy rate) or 13.1 us (NVFP4; 66 MB,
// 10.2 us).
//
// gemm_gated_pair_kernel (the rest): a CTA pair (cta_group::2) per 256 rows x 128 features. The B tile of
// 256 rows is [128 rows of Wg; 128 rows of Wu], one half loaded by either CTA, so g and u of a feature end up 128
// accumulator columns apart in the same lane. Bound by the tensor pipe (82 % busy in the NVFP4 form, 74 % when it writes
// [g | u] as well, 89 % in the MXFP8 form) and by power: 8192 x 4096 x 14336 takes 342 us (NVFP4, 5.6 PFLOP/s) or 645 us
// (MXFP8, 3.0) for h alone, 392 and 681 with [g | u]; twenty in a row, at the power cap, 350, 750, 410 and 770 us each.
//
// Every wait on an mbarrier is bounded, as in the plain GEMM kernels.
#include <algorithm>

#include "gated_act.cuh"
#include "gemm_common.cuh"
#include "tile_quant.cuh"

namespace mt {

struct GatedArgs {
  const uint8_t *sa, *sb_gate, *sb_up;   // scale factors, chunk layout
  int64_t kc;                            // chunks per 128-row block (all operands share K)
  int64_t M, F, K_bytes;
  const float *amax_a, *amax_b;
  int* status;
  int act;
  // outputs, each optional
  __nv_bfloat16 *h, *gu;
  float* amax;
  uint8_t *q, *s, *s_swz;
  int64_t s_stride, kc_h;                // kc_h: chunks per 128-row block of s_swz
  int tiles_m, tiles_n, num_tiles;
  int band;                              // pair kernel: row blocks per band of the tile order
};

__device__ __forceinline__ float gated_alpha(const GatedArgs& a) {
  return a.amax_a != nullptr ? __fdiv_rn(__fmul_rn(*a.amax_a, *a.amax_b), 6.0f * 6.0f * 448.0f * 448.0f) : 1.0f;
}

// ------------------------------------------------------------------------------------------
// few tokens
// ------------------------------------------------------------------------------------------
// 32 lanes x 8 consecutive 32-bit columns of tensor memory.
__device__ __forceinline__ void tc_ld_32x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr) : "memory");
}

// An epilogue warp takes 32 features of 8 tokens at a time, four warps share the tokens of 32 features. It is a CTA's only
// one, so nothing hides it: with one warp for all tokens, 32 at a time, one token on 14336 x 4096 (MXFP8) took 22.5 us
// instead of 20.9, 128 tokens 30.6 instead of 26.5; with 16 at a time 21.6 and 26.8.
constexpr int GR_TOKENS = 8, GR_SHARE = 4;
constexpr int GR_THREADS = 64 + 128 * GR_SHARE;

template <int kFormat, int BT, int STAGES>
struct GatedRowsCfg {
  static constexpr int CH = (kFormat == FMT_NVFP4) ? 4 : 1;
  static constexpr int W_BYTES = 128 * G_BLOCK_KB;       // one projection's rows of a stage
  static constexpr int T_BYTES = BT * G_BLOCK_KB;        // tokens of a stage
  static constexpr int SF_BYTES = CH * 512;
  static constexpr int STAGE_BYTES = 2 * W_BYTES + T_BYTES + 3 * SF_BYTES;
  static constexpr int OFF_G = 0;
  static constexpr int OFF_U = STAGES * W_BYTES;
  static constexpr int OFF_T = 2 * STAGES * W_BYTES;
  static constexpr int OFF_SF = OFF_T + STAGES * T_BYTES;   // [gate | up | tokens] chunks per stage
  static constexpr int OFF_BAR = OFF_SF + STAGES * 3 * SF_BYTES;
  static constexpr int NUM_BARS = 2 * STAGES + 1;
  static constexpr int SMEM_ALLOC = OFF_BAR + NUM_BARS * 8 + 16 + 1024;
  static constexpr int TMEM_G = 0, TMEM_U = BT;
  static constexpr int TMEM_SF = 2 * BT;                 // gate, up, tokens: 4 * CH columns each
  static constexpr int TMEM_COLS = (2 * BT + 12 * CH <= 128) ? 128 : (2 * BT + 12 * CH <= 256) ? 256 : 512;
  static_assert(2 * BT + 12 * CH <= 512, "tensor memory over-subscribed");
  static_assert(SMEM_ALLOC <= 227 * 1024, "shared memory over-subscribed");
};

// One CTA per 128 features and BT tokens (blockIdx.y): TMA producer warp, MMA warp, epilogue warps.
template <int kFormat, int BT, int STAGES>
__global__ void __launch_bounds__(GR_THREADS, 1)
    gemm_gated_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_g,
                           const __grid_constant__ CUtensorMap map_u, const GatedArgs a) {
  using Cfg = GatedRowsCfg<kFormat, BT, STAGES>;
  constexpr int CH = Cfg::CH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + STAGES;
  uint64_t* acc_full = bars + 2 * STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NUM_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x, m0 = (int)blockIdx.y * BT;
  const int64_t f0 = (int64_t)tile * 128;
  const int num_k = (int)((a.K_bytes + G_BLOCK_KB - 1) / G_BLOCK_KB);

  pdl_trigger();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], 1); }
    mbar_init(acc_full, 1);
    mbar_fence_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_g);
    prefetch_tensormap(&map_u);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      for (int k = 0; k < num_k; ++k) {
        if (!mbar_wait_bounded(&empty_bar[s], ph ^ 1, abort_flag, a.status, DS_EMPTY_WAIT)) break;
        mbar_expect_tx(&full_bar[s], Cfg::STAGE_BYTES);
        tma_load_2d(smem + Cfg::OFF_G + s * Cfg::W_BYTES, &map_g, &full_bar[s], k * G_BLOCK_KB, (int32_t)f0);
        tma_load_2d(smem + Cfg::OFF_U + s * Cfg::W_BYTES, &map_u, &full_bar[s], k * G_BLOCK_KB, (int32_t)f0);
        tma_load_2d(smem + Cfg::OFF_T + s * Cfg::T_BYTES, &map_x, &full_bar[s], k * G_BLOCK_KB, m0);
        uint8_t* sf = smem + Cfg::OFF_SF + s * 3 * Cfg::SF_BYTES;
        const int64_t chunk = (int64_t)tile * a.kc + (int64_t)k * CH;
        bulk_load_1d(sf, a.sb_gate + chunk * 512, Cfg::SF_BYTES, &full_bar[s]);
        bulk_load_1d(sf + Cfg::SF_BYTES, a.sb_up + chunk * 512, Cfg::SF_BYTES, &full_bar[s]);
        bulk_load_1d(sf + 2 * Cfg::SF_BYTES, a.sa + ((m0 >> 7) * a.kc + (int64_t)k * CH) * 512, Cfg::SF_BYTES, &full_bar[s]);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool alive = true;
      const uint32_t sm = smem_u32(smem);
      for (int k = 0; k < num_k; ++k) {
        if (!mbar_wait_bounded(&full_bar[s], ph, abort_flag, a.status, DS_TMA_WAIT)) { alive = false; break; }
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 3 * CH; ++i)
          tc_copy_sf(tmem_base + Cfg::TMEM_SF + 4 * i, umma_desc_sf(sm + Cfg::OFF_SF + s * 3 * Cfg::SF_BYTES + i * 512));
        const uint64_t gdesc = umma_desc_sw128(sm + Cfg::OFF_G + s * Cfg::W_BYTES);
        const uint64_t udesc = umma_desc_sw128(sm + Cfg::OFF_U + s * Cfg::W_BYTES);
        const uint64_t tdesc = umma_desc_sw128(sm + Cfg::OFF_T + s * Cfg::T_BYTES);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t idesc = make_idesc(kFormat, BT, j);
          const uint32_t sf = tmem_base + Cfg::TMEM_SF + (kFormat == FMT_NVFP4 ? 4 * j : 0);
          const uint32_t sft = sf + 8 * CH + ((m0 >> 5) & 3);   // 32 rows of a chunk per column
          const uint32_t acc = (k > 0 || j > 0) ? 1u : 0u;
          issue_mma<kFormat>(tmem_base + Cfg::TMEM_G, gdesc + 2 * j, tdesc + 2 * j, idesc, sf, sft, acc);
          issue_mma<kFormat>(tmem_base + Cfg::TMEM_U, udesc + 2 * j, tdesc + 2 * j, idesc, sf + 4 * CH, sft, acc);
        }
        tc_commit(&empty_bar[s]);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (alive) tc_commit(acc_full);
    }
    __syncwarp();
  } else {
    // epilogue: lane <-> feature, warp <-> one 1x32 block of h per token
    const int qd = warp & 3, part = (warp - 2) >> 2;
    const float alpha = gated_alpha(a);
    const bool silu = a.act == MT_ACT_SILU;
    const int64_t f = f0 + qd * 32 + lane;
    const bool f_ok = f < a.F;
    const int kb = (int)(f0 >> 5) + qd;
    AmaxAcc am;
    if (mbar_wait_bounded(acc_full, 0, abort_flag, a.status, DS_ACC_FULL_WAIT)) {
      tc_fence_after();
      const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(qd * 32) << 16);
      uint8_t* chunk = a.s_swz + ((m0 >> 7) * a.kc_h + tile) * 512;   // tokens of one 128-row block, blocks 4 tile ..
      const int M = (int)min((int64_t)BT, a.M - m0);                  // of this CTA
#pragma unroll 1
      for (int c = part * GR_TOKENS; c < M; c += GR_SHARE * GR_TOKENS) {
        uint32_t g[GR_TOKENS], u[GR_TOKENS];
        tc_ld_32x8(lane_base + Cfg::TMEM_G + c, g);
        tc_ld_32x8(lane_base + Cfg::TMEM_U + c, u);
        tc_wait_ld();
        const int n = min(GR_TOKENS, M - c);     // (columns beyond the last token hold zeros: their rows of x are not there)
        if (a.gu != nullptr && f_ok) {
          __nv_bfloat16* p = a.gu + (int64_t)(m0 + c) * 2 * a.F + f;
#pragma unroll
          for (int i = 0; i < GR_TOKENS; ++i) {
            if (i < n) {
              p[0] = __float2bfloat16_rn(alpha * __uint_as_float(g[i]));
              p[a.F] = __float2bfloat16_rn(alpha * __uint_as_float(u[i]));
            }
            p += 2 * a.F;
          }
        }
        // h of the tokens, all independent of one another; bf16 bits in the upper half of the word
#pragma unroll
        for (int i = 0; i < GR_TOKENS; ++i) {
          const float v = alpha * __uint_as_float(g[i]);
          const float h = (silu ? gated_act<MT_ACT_SILU>(v) : gated_act<MT_ACT_GELU>(v)) * (alpha * __uint_as_float(u[i]));
          g[i] = f_ok ? static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(h))) << 16 : 0u;
        }
        if (a.h != nullptr && f_ok) {
          __nv_bfloat16* p = a.h + (int64_t)(m0 + c) * a.F + f;
#pragma unroll
          for (int i = 0; i < GR_TOKENS; ++i) {
            if (i < n) *p = __ushort_as_bfloat16(static_cast<unsigned short>(g[i] >> 16));
            p += a.F;
          }
        }
        if (a.amax != nullptr) {
#pragma unroll
          for (int i = 0; i < GR_TOKENS; ++i)
            if (i < n) am.f = fmaxf(am.f, fabsf(__uint_as_float(g[i])));
        }
        if (a.q != nullptr) {
          // lane i ends up with token i's abs-max over the block (bit patterns of magnitudes order like integers; a
          // NaN is dropped as in mt_quantize_mxfp8) and computes its scale once
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < GR_TOKENS; ++i) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(__uint_as_float(g[i])), 0.0f)));
            if (lane == i) top = m;
          }
          uint32_t enc;
          const uint32_t sb = mx_scale(top >> 16, enc);
          uint8_t* p = a.q + (int64_t)(m0 + c) * a.F + f;
#pragma unroll
          for (int i = 0; i < GR_TOKENS; ++i) {
            const float e = __uint_as_float(__shfl_sync(0xffffffffu, enc, i) << 16);
            if (i < n && f_ok) *p = __nv_cvt_float_to_fp8(__uint_as_float(g[i]) * e, __NV_SATFINITE, __NV_E4M3);
            p += a.F;
          }
          const int t = m0 + c + lane;
          if (lane < n) {
            const bool in = (int64_t)kb * 32 < a.F;
            if (in && a.s != nullptr) a.s[t * a.s_stride + kb] = static_cast<uint8_t>(sb);
            if (a.s_swz != nullptr) chunk[sf_chunk_offset(t, kb)] = in ? static_cast<uint8_t>(sb) : 0;
          }
        }
      }
      if (a.s_swz != nullptr) {   // rows without a token, and the chunks up to the padded count
        if (blockIdx.y == gridDim.y - 1)
          for (int t = m0 + M + part * 32 + lane; t < ((m0 >> 7) + 1) * 128; t += GR_SHARE * 32) chunk[sf_chunk_offset(t, kb)] = 0;
        if (tile == a.tiles_n - 1 && (m0 & 127) == 0)
          for (int64_t i = 32 + (warp - 2) * 32 + lane; i < (a.kc_h - tile) * 32; i += 128 * GR_SHARE)
            *reinterpret_cast<uint4*>(chunk + i * 16) = make_uint4(0, 0, 0, 0);
      }
      if (a.amax != nullptr) amax_publish(a.amax, am, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------
// many tokens
// ------------------------------------------------------------------------------------------
// 16 row blocks (4096 rows) per band: at 8192 x 4096 x 14336 with both bf16 outputs, bands of 1 / 4 / 8 / 16 / 32 took
// 474 / 442 / 422 / 412 / 411 us (NVFP4) and 870 / 741 / 715 / 702 / 704 us (MXFP8, whose weight alone fills L2).
constexpr int GP_BAND = 16;
constexpr int GP_EPI_WARPS = 8;
constexpr int GP_THREADS = 64 + 32 * GP_EPI_WARPS;

template <int kFormat, int STAGES>
struct GatedPairCfg {
  static constexpr int CH = (kFormat == FMT_NVFP4) ? 4 : 1;
  static constexpr int A_BYTES = 128 * G_BLOCK_KB;
  static constexpr int B_BYTES = 128 * G_BLOCK_KB;       // this CTA's projection: gate (rank 0) or up (rank 1)
  static constexpr int SF_BYTES = CH * 512;              // x rows of this CTA; gate and up: both CTAs load both
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 3 * SF_BYTES;
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = STAGES * A_BYTES;
  static constexpr int OFF_SF = OFF_B + STAGES * B_BYTES;   // [x | gate | up] per stage
  static constexpr int OFF_BAR = OFF_SF + STAGES * 3 * SF_BYTES;
  static constexpr int NUM_BARS = 2 * STAGES + 2;
  static constexpr int SMEM_ALLOC = OFF_BAR + NUM_BARS * 8 + 16 + 1024;
  static constexpr int TMEM_SFA = 256;
  static constexpr int TMEM_SFB = TMEM_SFA + 4 * CH;
  static_assert(TMEM_SFB + 8 * CH <= G_TMEM_COLS, "tensor memory over-subscribed");
  static_assert(SMEM_ALLOC <= 227 * 1024, "shared memory over-subscribed");
};

// Hands tensor memory back to the issuer in the leader CTA. Relaxed: the accumulator is in registers (tcgen05.wait::ld
// has returned), and a release would wait for this lane's global stores of the tile before as well (8192 x 4096 x
// 14336, NVFP4: 412 -> 392 us with the saved projections, 367 -> 342 us without).
__device__ __forceinline__ void arrive_acc_empty(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Tile order of the pair kernel: bands of row blocks, the row block fastest inside a band. The weight tiles are read
// once per band and the band's rows of x stay in L2 meanwhile.
__device__ __forceinline__ void gated_tile(const GatedArgs& a, int tile, int& mb, int& nb) {
  const int per_band = a.band * a.tiles_n, b = tile / per_band, r = tile - b * per_band;
  const int rows = min(a.band, a.tiles_m - b * a.band);
  nb = r / rows;
  mb = b * a.band + (r - nb * rows);
}

// 32 features of one row: bf16 h (and bf16 g, u) -> global memory, codes and scale byte.
template <int kAct>
__device__ __forceinline__ void gated_store_block(const GatedArgs& a, const uint32_t (&g)[32], const uint32_t (&u)[32],
                                                  float alpha, int64_t row, int64_t f, bool row_ok, AmaxAcc& am) {
  const bool ok = row_ok && f < a.F;    // F is a multiple of 32: a block is whole or absent
  uint32_t hw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float g0 = alpha * __uint_as_float(g[2 * i]), g1 = alpha * __uint_as_float(g[2 * i + 1]);
    const float u0 = alpha * __uint_as_float(u[2 * i]), u1 = alpha * __uint_as_float(u[2 * i + 1]);
    hw[i] = f32x2_to_bf16x2(pack2(gated_act<kAct>(g0) * u0, gated_act<kAct>(g1) * u1));
  }
  if (ok && a.gu != nullptr) {
    __nv_bfloat16* pg = a.gu + row * 2 * a.F + f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t wg[8], wu[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = 16 * half + 2 * i;
        wg[i] = f32x2_to_bf16x2(pack2(alpha * __uint_as_float(g[c]), alpha * __uint_as_float(g[c + 1])));
        wu[i] = f32x2_to_bf16x2(pack2(alpha * __uint_as_float(u[c]), alpha * __uint_as_float(u[c + 1])));
      }
      st_global_v8(pg + 16 * half, wg);
      st_global_v8(pg + a.F + 16 * half, wu);
    }
  }
  if (ok && a.h != nullptr) {
    __nv_bfloat16* ph = a.h + row * a.F + f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t w[8] = {hw[8 * half], hw[8 * half + 1], hw[8 * half + 2], hw[8 * half + 3],
                             hw[8 * half + 4], hw[8 * half + 5], hw[8 * half + 6], hw[8 * half + 7]};
      st_global_v8(ph + 16 * half, w);
    }
  }
  if (a.amax == nullptr && a.q == nullptr) return;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = absmax2(m, hw[i]);
  if (ok) amax_bf16x2(am, m);
  if (a.q == nullptr) return;
  const int e = e8m0_exponent(absmax2_to_float(m));
  const float enc = exp2_neg(e);
  const f32x2_t enc2 = pack2(enc, enc);
  uint32_t cw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cw[i] = e4m3x4_from_words(hw[2 * i], hw[2 * i + 1], enc2);
  if (ok) st_global_v8(a.q + row * a.F + f, cw);
  const uint8_t sb = ok ? static_cast<uint8_t>(e + 127) : 0;
  const int64_t kb = f >> 5;
  if (ok && a.s != nullptr) a.s[row * a.s_stride + kb] = sb;
  if (a.s_swz != nullptr && (row >> 7) < (a.M + 127) / 128)
    a.s_swz[((row >> 7) * a.kc_h + (kb >> 2)) * 512 + sf_chunk_offset((int)(row & 127), (int)kb)] = sb;
}

template <int kFormat, int STAGES, int kAct>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GP_THREADS, 1)
    gemm_gated_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_g,
                           const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_sx,
                           const __grid_constant__ CUtensorMap map_sg, const __grid_constant__ CUtensorMap map_su,
                           const GatedArgs a) {
  using Cfg = GatedPairCfg<kFormat, STAGES>;
  constexpr int CH = Cfg::CH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* full_bar = bars;                  // leader only, signalled by both CTAs' loads
  uint64_t* empty_bar = bars + STAGES;        // per CTA, signalled by the leader's commit
  uint64_t* acc_full = bars + 2 * STAGES;     // per CTA, signalled by the leader's commit
  uint64_t* acc_empty = bars + 2 * STAGES + 1;   // leader only: 2 x GP_EPI_WARPS arrivals
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NUM_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int num_k = (int)((a.K_bytes + G_BLOCK_KB - 1) / G_BLOCK_KB);

  pdl_trigger();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], 1); }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * GP_EPI_WARPS);
    mbar_fence_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(rank == 0 ? &map_g : &map_u);
    prefetch_tensormap(&map_sx);
    prefetch_tensormap(&map_sg);
    prefetch_tensormap(&map_su);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, G_TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();      // both CTAs' barriers exist before either signals the other
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool alive = true;
      const CUtensorMap* map_w = rank == 0 ? &map_g : &map_u;
      for (int tile = pair; tile < a.num_tiles && alive; tile += num_pairs) {
        int mb, nb;
        gated_tile(a, tile, mb, nb);
        const int32_t x_row = mb * 256 + (int)rank * 128, w_row = nb * 128;
        const int32_t sx_chunk = (int32_t)((2 * mb + (int)rank) * a.kc), sw_chunk = (int32_t)(nb * a.kc);
        for (int k = 0; k < num_k; ++k) {
          if (!mbar_wait_bounded(&empty_bar[s], ph ^ 1, abort_flag, a.status, DS_EMPTY_WAIT)) { alive = false; break; }
          if (leader) mbar_expect_tx(&full_bar[s], 2 * Cfg::STAGE_BYTES);
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[s]), 0);
          tma_load_2d_pair(smem + Cfg::OFF_A + s * Cfg::A_BYTES, &map_x, bar, k * G_BLOCK_KB, x_row);
          tma_load_2d_pair(smem + Cfg::OFF_B + s * Cfg::B_BYTES, map_w, bar, k * G_BLOCK_KB, w_row);
          uint8_t* sf = smem + Cfg::OFF_SF + s * 3 * Cfg::SF_BYTES;
          tma_load_2d_pair(sf, &map_sx, bar, 0, sx_chunk + k * CH);
          tma_load_2d_pair(sf + Cfg::SF_BYTES, &map_sg, bar, 0, sw_chunk + k * CH);
          tma_load_2d_pair(sf + 2 * Cfg::SF_BYTES, &map_su, bar, 0, sw_chunk + k * CH);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader && elect_one()) {
      int s = 0;
      uint32_t ph = 0, tile_it = 0;
      bool alive = true;
      const uint32_t sm = smem_u32(smem);
      for (int tile = pair; tile < a.num_tiles && alive; tile += num_pairs, ++tile_it) {
        if (!mbar_wait_bounded(acc_empty, (tile_it & 1) ^ 1, abort_flag, a.status, DS_ACC_EMPTY_WAIT)) { alive = false; break; }
        tc_fence_after();
        for (int k = 0; k < num_k; ++k) {
          if (!mbar_wait_bounded(&full_bar[s], ph, abort_flag, a.status, DS_TMA_WAIT)) { alive = false; break; }
          tc_fence_after();
          const uint32_t sf = sm + Cfg::OFF_SF + s * 3 * Cfg::SF_BYTES;
#pragma unroll
          for (int c = 0; c < CH; ++c) tc_copy_sf_pair(tmem_base + Cfg::TMEM_SFA + 4 * c, umma_desc_sf(sf + c * 512));
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int c = 0; c < CH; ++c)
              tc_copy_sf_pair(tmem_base + Cfg::TMEM_SFB + 4 * (2 * c + p), umma_desc_sf(sf + ((1 + p) * CH + c) * 512));
          const uint64_t adesc = umma_desc_sw128(sm + Cfg::OFF_A + s * Cfg::A_BYTES);
          const uint64_t bdesc = umma_desc_sw128(sm + Cfg::OFF_B + s * Cfg::B_BYTES);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t idesc = make_idesc_pair(kFormat, 256, j);
            issue_mma_pair<kFormat>(tmem_base, adesc + 2 * j, bdesc + 2 * j, idesc,
                                    tmem_base + Cfg::TMEM_SFA + (kFormat == FMT_NVFP4 ? 4 * j : 0),
                                    tmem_base + Cfg::TMEM_SFB + (kFormat == FMT_NVFP4 ? 8 * j : 0), (k > 0 || j > 0) ? 1u : 0u);
          }
          tc_commit_pair(&empty_bar[s], 3);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        if (alive) tc_commit_pair(acc_full, 3);
      }
    }
    __syncwarp();
  } else {
    // epilogue: a warp reads the lane quarter warp % 4 and 64 of the 128 features
    const int e = warp - 2, qd = warp & 3, half = (e >> 2) & 1;
    const float alpha = gated_alpha(a);
    const uint32_t acc_empty_leader = map_to_cta(smem_u32(acc_empty), 0);
    uint32_t tile_it = 0;
    AmaxAcc am;
    for (int tile = pair; tile < a.num_tiles; tile += num_pairs, ++tile_it) {
      int mb, nb;
      gated_tile(a, tile, mb, nb);
      if (!mbar_wait_bounded(acc_full, tile_it & 1, abort_flag, a.status, DS_ACC_FULL_WAIT)) break;
      tc_fence_after();
      const uint32_t tm = tmem_base + (static_cast<uint32_t>(qd * 32) << 16) + half * 64;
      // the whole block goes to registers and tensor memory back to the MMA issuer at once
      uint32_t g[2][32], u[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tc_ld_32x32(tm + c * 32, g[c]);
        tc_ld_32x32(tm + 128 + c * 32, u[c]);
      }
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_acc_empty(acc_empty_leader);
      const int64_t row = (int64_t)mb * 256 + rank * 128 + qd * 32 + lane;
      const int64_t f = (int64_t)nb * 128 + half * 64;
#pragma unroll
      for (int c = 0; c < 2; ++c) gated_store_block<kAct>(a, g[c], u[c], alpha, row, f + c * 32, row < a.M, am);
      if (a.s_swz != nullptr && nb == a.tiles_n - 1 && half == 0 && (row >> 7) < (a.M + 127) / 128) {
        // this row's words in the chunks up to the padded count
        uint8_t* cell = a.s_swz + (row >> 7) * a.kc_h * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
        for (int64_t c = a.tiles_n; c < a.kc_h; ++c) *reinterpret_cast<uint32_t*>(cell + c * 512) = 0u;
      }
    }
    if (a.amax != nullptr) amax_publish(a.amax, am, lane);
  }
  tc_fence_before();
  __syncthreads();
  // neither CTA may exit (or free tensor memory) while its peer can still touch it
  cluster_arrive();
  cluster_wait();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, G_TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
template <int kFormat, int BT, int STAGES>
static int launch_gated_rows(const CUtensorMap& mx, const CUtensorMap& mg, const CUtensorMap& mu, const GatedArgs& a,
                             cudaStream_t st) {
  using Cfg = GatedRowsCfg<kFormat, BT, STAGES>;
  auto kern = gemm_gated_rows_kernel<kFormat, BT, STAGES>;
  static bool attr_set[MT_MAX_DEVICES] = {};
  const int slot = current_device_slot();
  if (!attr_set[slot]) {
    MT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_ALLOC));
    attr_set[slot] = true;
  }
  MT_CUDA(launch_pdl(kern, dim3(a.tiles_n, (unsigned)((a.M + BT - 1) / BT)), dim3(GR_THREADS), (size_t)Cfg::SMEM_ALLOC, st, mx, mg, mu, a));
  return MT_OK;
}

template <int kFormat, int STAGES, int kAct>
static int launch_gated_pair(const CUtensorMap (&m)[6], const GatedArgs& a, cudaStream_t st) {
  using Cfg = GatedPairCfg<kFormat, STAGES>;
  auto kern = gemm_gated_pair_kernel<kFormat, STAGES, kAct>;
  static int max_pairs_dev[MT_MAX_DEVICES] = {};   // 0 = not yet queried on that device
  int& max_pairs = max_pairs_dev[current_device_slot()];
  if (max_pairs <= 0) {
    MT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_ALLOC));
    int dev = 0, sms = 0;
    MT_CUDA(cudaGetDevice(&dev));
    MT_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms / 2 * 2);
    cfg.blockDim = dim3(GP_THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_ALLOC;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) { cudaGetLastError(); n = sms / 2; }
    max_pairs = n;
  }
  const int pairs = std::min(a.num_tiles, max_pairs);
  MT_CUDA(launch_pdl(kern, dim3(2 * pairs), dim3(GP_THREADS), (size_t)Cfg::SMEM_ALLOC, st, m[0], m[1], m[2], m[3], m[4], m[5], a));
  return MT_OK;
}

template <int kFormat>
static int launch_gated(const uint8_t* x, const uint8_t* wg, const uint8_t* wu, GatedArgs& a, cudaStream_t st) {
  CUtensorMap m[6];
  const uint64_t ld = (uint64_t)a.K_bytes;
  constexpr uint32_t CH = kFormat == FMT_NVFP4 ? 4 : 1;
  a.tiles_n = (int)((a.F + 127) / 128);
  // Blocks of 64 tokens where one wave holds them all: the fewer tokens a CTA has, the sooner it is done. 1000 tokens on
  // 768 x 2048: 7.9 us in 64-token blocks, 9.4 us in 256-row pairs; 128 on 4096 x 1024: 5.7 us in two blocks, 7.5 us in one.
  const bool spread = a.M > 64 && (a.M + 63) / 64 * a.tiles_n <= mx_sm_count();
  const bool small = spread || a.M <= 128;
  const uint32_t bt = spread ? 64u : small ? (uint32_t)((a.M + 31) / 32 * 32) : 128u;
  int rc = make_tensor_map_2d(&m[0], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, ld, (uint64_t)a.M, ld, G_BLOCK_KB, bt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == MT_OK) rc = make_tensor_map_2d(&m[1], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wg, ld, (uint64_t)a.F, ld, G_BLOCK_KB, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == MT_OK) rc = make_tensor_map_2d(&m[2], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wu, ld, (uint64_t)a.F, ld, G_BLOCK_KB, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != MT_OK) return rc;
  if (small) {
    // As many stages as shared memory holds: with 2 / 3 / 4 / 5 one token on 14336 x 4096 (MXFP8) took 30.3 / 24.6 / 23.6 /
    // 22.7 us, 64 tokens with 4 / 5 24.2 / 23.4. A variant with 16 tokens on the column side and 6 stages was no faster.
    if (bt == 32) return launch_gated_rows<kFormat, 32, 5>(m[0], m[1], m[2], a, st);
    if (bt == 64) return launch_gated_rows<kFormat, 64, kFormat == FMT_NVFP4 ? 4 : 5>(m[0], m[1], m[2], a, st);
    if (bt == 96) return launch_gated_rows<kFormat, 96, 4>(m[0], m[1], m[2], a, st);
    return launch_gated_rows<kFormat, 128, 4>(m[0], m[1], m[2], a, st);
  }
  const uint64_t rb_x = (uint64_t)((a.M + 127) / 128), rb_w = (uint64_t)((a.F + 127) / 128);
  rc = make_tensor_map_2d(&m[3], CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.sa, 128, rb_x * a.kc, 512, 128, CH, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc == MT_OK) rc = make_tensor_map_2d(&m[4], CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.sb_gate, 128, rb_w * a.kc, 512, 128, CH, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc == MT_OK) rc = make_tensor_map_2d(&m[5], CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.sb_up, 128, rb_w * a.kc, 512, 128, CH, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc != MT_OK) return rc;
  a.tiles_m = (int)((a.M + 255) / 256);
  a.num_tiles = a.tiles_m * a.tiles_n;
  a.band = GP_BAND;
  constexpr int ST = kFormat == FMT_NVFP4 ? 5 : 6;
  return a.act == MT_ACT_SILU ? launch_gated_pair<kFormat, ST, MT_ACT_SILU>(m, a, st)
                              : launch_gated_pair<kFormat, ST, MT_ACT_GELU>(m, a, st);
}

static int gemm_gated(int format, const uint8_t* x, const uint8_t* sx, const float* amax_x, const uint8_t* w,
                      const uint8_t* sw, const uint8_t* sw_up, const float* amax_w, int64_t M, int64_t F, int64_t K,
                      const mt_gated_outputs* out, int act, cudaStream_t st) {
  const char* name = format == FMT_NVFP4 ? "mt_gemm_gated_nvfp4" : "mt_gemm_gated_mxfp8";
  MT_REQUIRE(M >= 0 && F >= 0 && K >= 0, "%s: negative shape", name);
  MT_REQUIRE(M < (int64_t)1 << 30 && F < (int64_t)1 << 28 && K < (int64_t)1 << 30, "%s: shape out of range", name);
  MT_REQUIRE(gated_act_known(act), "%s: activation %d not supported", name, act);
  MT_REQUIRE(out != nullptr, "%s: null outputs", name);
  MT_REQUIRE(K > 0 && K % 32 == 0, "%s: K (%lld) must be a positive multiple of 32", name, (long long)K);
  MT_REQUIRE(F % 32 == 0, "%s: F (%lld) must be a multiple of 32", name, (long long)F);
  if (M == 0 || F == 0) return MT_OK;
  MT_REQUIRE(x && sx && w && sw, "%s: null pointer", name);
  MT_REQUIRE(sw_up || F % 128 == 0, "%s: with F (%lld) not a multiple of 128 the scales of the second projection must be "
             "given apart, in a layout of their own", name, (long long)F);
  MT_REQUIRE(aligned16(x) && aligned16(sx) && aligned16(w) && aligned16(sw) && aligned16(sw_up),
             "%s: operands must be 16-byte aligned", name);
  if (format == FMT_NVFP4) MT_REQUIRE(amax_x && amax_w, "%s: per-tensor abs-max pointers are required", name);
  MT_REQUIRE(out->h || out->gu || out->q, "%s: no output requested", name);
  const uintptr_t align = reinterpret_cast<uintptr_t>(out->h) | reinterpret_cast<uintptr_t>(out->gu) | reinterpret_cast<uintptr_t>(out->q);
  MT_REQUIRE((align & 31) == 0, "%s: outputs must be 32-byte aligned", name);
  MT_REQUIRE(aligned16(out->s_swz), "%s: swizzled scale buffer must be 16-byte aligned", name);
  MT_REQUIRE(!out->q || (out->s && out->s_stride >= F / 32), "%s: codes need s with a stride of at least F / 32", name);
  MT_REQUIRE(out->q || (!out->s && !out->s_swz), "%s: scales without codes", name);
  const int64_t block = format == FMT_NVFP4 ? 16 : 32;
  GatedArgs a{};
  a.M = M; a.F = F;
  a.K_bytes = format == FMT_NVFP4 ? K / 2 : K;
  a.kc = ((K / block + 3) / 4 + 3) / 4 * 4;
  a.sa = sx; a.sb_gate = sw; a.sb_up = sw_up ? sw_up : sw + F / 128 * a.kc * 512;
  a.amax_a = format == FMT_NVFP4 ? amax_x : nullptr;
  a.amax_b = format == FMT_NVFP4 ? amax_w : nullptr;
  a.act = act;
  a.h = static_cast<__nv_bfloat16*>(out->h); a.gu = static_cast<__nv_bfloat16*>(out->gu); a.amax = out->amax;
  a.q = out->q; a.s = out->s; a.s_swz = out->s_swz; a.s_stride = out->s_stride;
  a.kc_h = ((F / 32 + 3) / 4 + 3) / 4 * 4;
  a.status = device_status_ptr();
  if (!a.status) return fail(MT_ERR_CUDA, "device status word not reachable");
  const uint8_t* wu = w + F * a.K_bytes;
  return format == FMT_NVFP4 ? launch_gated<FMT_NVFP4>(x, w, wu, a, st) : launch_gated<FMT_MXFP8>(x, w, wu, a, st);
}

}  // namespace mt

extern "C" int mt_gemm_gated_mxfp8(const uint8_t* x, const uint8_t* sx_swz, const uint8_t* w, const uint8_t* sw_swz,
                                   const uint8_t* sw_up_swz, int64_t M, int64_t F, int64_t K, int activation,
                                   const mt_gated_outputs* out, mt_stream_t stream) {
  return mt::gemm_gated(mt::FMT_MXFP8, x, sx_swz, nullptr, w, sw_swz, sw_up_swz, nullptr, M, F, K, out, activation,
                        static_cast<cudaStream_t>(stream));
}

extern "C" int mt_gemm_gated_nvfp4(const uint8_t* x, const uint8_t* sx_swz, const float* amax_x, const uint8_t* w,
                                   const uint8_t* sw_swz, const uint8_t* sw_up_swz, const float* amax_w, int64_t M,
                                   int64_t F, int64_t K, int activation, const mt_gated_outputs* out, mt_stream_t stream) {
  return mt::gemm_gated(mt::FMT_NVFP4, x, sx_swz, amax_x, w, sw_swz, sw_up_swz, amax_w, M, F, K, out, activation,
                        static_cast<cudaStream_t>(stream));
}
