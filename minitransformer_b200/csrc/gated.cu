// Gradient of the gated activation: from dh and the saved projections [g | u],
//   du = bf16(dh * act(g)),   dg = bf16(dh * u * act'(g))
// and, from the same registers, the MXFP8 copies of [dg | du] that the dgrad and wgrad GEMMs read (row-wise and
// transposed). 6 bytes read and 4 written per (row, feature): bound by HBM. 8192 x 14336 with both copies takes 236 us (silu)
// or 233 us (gelu) (1204 MB, 5.1 - 5.2 TB/s), the bf16 gradient and its abs-max 207 or 212 us (1174 MB, 5.5 - 5.7 TB/s; without
// the abs-max and the arithmetic 203 us, without the stores 101 us). 1021 x 1376: 12.2 / 12.5 us (1024 x 1376: 9.3 / 9.4 us).
#include "gated_act.cuh"
#include "tile_quant.cuh"

namespace mt {

struct GatedGradArgs {
  int64_t rows, F;
  int tiles_x, tiles;
  int* status;
  __nv_bfloat16* dgu;
  float* amax;
  MxTileOut out;       // out.q null: no copies
};

// Persistent CTAs, two per SM; a CTA takes 128 rows x 128 features at a time: four warps of 32 rows side by side in
// each of two 64-column halves, so that row-wise codes leave in whole 128-byte lines and transposed codes in
// 128-byte runs of one feature. Every warp fetches its own 32 x 64 tiles of dh, g and u by TMA (12 KB, one
// mbarrier per warp) and asks for the next ones as soon as it has computed dg and du into registers: they arrive
// while the warp quantizes and stores. Scale bytes are collected in shared memory and leave as words. Measured and
// left out: an L2 hint that lets the inputs go first (301 us instead of 241 on 8192 x 14336), warps that store by
// themselves (slower, their scales leave as bytes), dg and du in CTAs of their own for few tiles (1024 x 1376: 8.8 us), scale chunks
// written as whole lines (no change).
constexpr int GG_SMEM = 8 * 3 * MX_TILE_BYTES + 128;

// kDgu: the bf16 gradient or its abs-max is asked for; kCopies: the MXFP8 copies are. Spills cost more here than their
// number says, since they queue behind the stores: one kernel for all of it, without the two __syncwarp that keep the
// loads of a tile from being moved ahead all at once, spilled 22 registers and took 116 us instead of 110 on 4096 x
// 14336 (copies), 226 instead of 204 on 8192 x 14336 (dgu alone). Copies and gradient together still spill (28 registers).
template <int kAct, bool kRagged, bool kDgu, bool kCopies>
__global__ void __launch_bounds__(256, 2)
    gated_grad_kernel(const __grid_constant__ CUtensorMap map_dh, const __grid_constant__ CUtensorMap map_gu, const GatedGradArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  __shared__ __align__(16) uint8_t s_rows[2][2][128][4], s_cols[2][2][128][4];   // [turn][dg, du][row / feature][block]
  __shared__ uint64_t bars[8], empty[8];
  __shared__ int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wr = warp & 3, wc = warp >> 2;
  uint8_t* buf = smem + warp * 3 * MX_TILE_BYTES;
  const MxTileOut& o = a.out;
  const bool row_words = mx_word_aligned(o.s, o.s_stride), col_words = mx_word_aligned(o.s_t, o.s_t_stride);
  if (tid == 0) abort_flag = 0;
  if (lane == 0) {
    mbar_init(&bars[warp], 1);
    mbar_init(&empty[warp], 32);
  }
  mbar_fence_init();
  __syncthreads();
  pdl_wait();

  auto fetch = [&](int tile) {
    const int y = tile / a.tiles_x, x = tile - y * a.tiles_x;
    const int32_t r = y * 128 + wr * 32, c = x * 128 + wc * 64;
    mbar_expect_tx(&bars[warp], 3 * MX_TILE_BYTES);
    tma_load_2d(buf, &map_gu, &bars[warp], c, r);
    tma_load_2d(buf + MX_TILE_BYTES, &map_dh, &bars[warp], c, r);
    tma_load_2d(buf + 2 * MX_TILE_BYTES, &map_gu, &bars[warp], (int32_t)a.F + c, r);
  };
  if (lane == 0 && (int)blockIdx.x < a.tiles) fetch(blockIdx.x);
  uint32_t ph = 0;
  for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ph ^= 1) {
    const int ty = tile / a.tiles_x, tx = tile - ty * a.tiles_x;
    const int64_t m0 = (int64_t)ty * 128, f0 = (int64_t)tx * 128;
    const int64_t row0 = m0 + wr * 32, c0 = f0 + wc * 64;
    uint8_t (&s_row)[2][128][4] = s_rows[ph], (&s_col)[2][128][4] = s_cols[ph];   // turns alternate: one barrier each
    // on expiry the status word tells; the warp goes on with what is there, so that nobody waits for it
    mbar_wait_bounded(&bars[warp], ph, &abort_flag, a.status, DS_QUANT_WAIT);
    uint32_t wg[8][4], wu[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 g4 = mx_tile_row(buf, i), d4 = mx_tile_row(buf + MX_TILE_BYTES, i), u4 = mx_tile_row(buf + 2 * MX_TILE_BYTES, i);
      const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x2_t act, grad;
        gated_act_grad2<kAct>(bf16x2_to_f32x2(g[j]), act, grad);
        const f32x2_t d2 = bf16x2_to_f32x2(d[j]);
        wu[i][j] = f32x2_to_bf16x2(mul2(d2, act));
        wg[i][j] = f32x2_to_bf16x2(mul2(mul2(d2, bf16x2_to_f32x2(u[j])), grad));
      }
      if (kCopies ? i % 4 == 3 : i % 3 == 2) __syncwarp();   // (where nothing spills)
    }
    mx_release_tile(&empty[warp], ph, &abort_flag, a.status);
    if (lane == 0 && tile + (int)gridDim.x < a.tiles) fetch(tile + gridDim.x);
    if (kDgu && a.dgu != nullptr) {
      const int64_t row = row0 + (lane >> 3) * 8, f = c0 + (lane & 7) * 8;
      const int nrow = f < a.F ? mx_valid_rows(a.rows, row) : 0;
      __nv_bfloat16* pg = a.dgu + row * 2 * a.F + f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i < nrow) {
          *reinterpret_cast<uint4*>(pg) = make_uint4(wg[i][0], wg[i][1], wg[i][2], wg[i][3]);
          *reinterpret_cast<uint4*>(pg + a.F) = make_uint4(wu[i][0], wu[i][1], wu[i][2], wu[i][3]);
        }
        pg += 2 * a.F;
      }
    }
    if (kDgu && a.amax != nullptr) {
      const bool in = c0 + (lane & 7) * 8 < a.F;   // a tile across the border holds the first columns of u as g
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) am = absmax2(am, absmax2(wu[i][j], wg[i][j]));
      const uint32_t bits = __reduce_max_sync(0xffffffffu, in ? __float_as_uint(absmax2_to_float(am)) : 0u);
      if (lane == 0 && bits != 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), bits);
    }
    if (!kCopies) continue;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const MxTileScales sc = p ? mx_tile_store<kRagged>(o, wu, row0, a.F + c0, 2 * a.F)
                                : mx_tile_store<kRagged>(o, wg, row0, c0, a.F);
      const int r = wr * 32 + (lane >> 3) * 8 + (lane & 3) * 2, kb = wc * 2 + ((lane & 7) >> 2);
      const int c = wc * 64 + (lane & 7) * 8 + (lane >> 3) * 2;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s_row[p][r + j][kb] = static_cast<uint8_t>(sc.row[j]);
        s_col[p][c + j][wr] = static_cast<uint8_t>(sc.col[j]);
      }
    }
    __syncthreads();
    const uint32_t t = tid & 127;
    if (tid < 128) {
      const uint32_t r = (uint32_t)m0 + t;
      const int n = (int)min((int64_t)4, (a.F - f0) >> 5);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t b0 = (uint32_t)((p ? a.F + f0 : f0) >> 5);
        mx_store_scale_word(*reinterpret_cast<const uint32_t*>(s_row[p][t]), n, n == 4 && (b0 & 3) == 0 && row_words,
                            r < o.rows ? o.s + (r * o.s_stride + b0) : nullptr, o.s_swz, r, b0, (uint32_t)o.kc_row);
      }
    } else if (o.q_t != nullptr && f0 + t < a.F) {
      const uint32_t b0 = (uint32_t)(m0 >> 5);
      const int n = (int)min((int64_t)4, ((o.rows + 31) >> 5) - b0);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t c = (uint32_t)((p ? a.F : 0) + f0) + t, word = *reinterpret_cast<const uint32_t*>(s_col[p][t]);
        mx_store_scale_word(word, n, n == 4 && col_words, o.s_t + (c * o.s_t_stride + b0), nullptr, c, b0, 0);
        // (token blocks without a row: zeros)
        if (o.s_t_swz != nullptr) *reinterpret_cast<uint32_t*>(o.s_t_swz + mx_swz_offset(c, b0, (uint32_t)o.kc_col)) = word;
      }
    }
    // padding of the GEMM-layout scales: beyond the last feature, and token blocks up to the padded count
    const int64_t mb0 = m0 >> 5, f1 = min(f0 + 128, a.F);
    const bool last_x = tx == a.tiles_x - 1, last_y = (ty + 1) * a.tiles_x >= a.tiles;
    if (last_x) {
      mx_pad_row_scales(o, m0, 128, tid, 256);
      for (int i = 0; i < 4; ++i) mx_pad_col_features(o, mb0 + i, tid, 256);
    }
    if (last_y) {
      mx_pad_col_blocks(o, mb0 + 4, f0, f1, tid, 256);
      mx_pad_col_blocks(o, mb0 + 4, a.F + f0, a.F + f1, tid, 256);
      if (last_x) mx_pad_col_blocks(o, mb0 + 4, 2 * a.F, (2 * a.F + 127) / 128 * 128, tid, 256);
    }
  }
  pdl_trigger();
}

template <int kAct, bool kRagged, bool kDgu, bool kCopies>
static int launch_gated_grad(const CUtensorMap& mdh, const CUtensorMap& mgu, const GatedGradArgs& a, cudaStream_t st) {
  auto kern = gated_grad_kernel<kAct, kRagged, kDgu, kCopies>;
  static bool attr_set[MT_MAX_DEVICES] = {};
  const int slot = current_device_slot();
  if (!attr_set[slot]) {
    MT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GG_SMEM));
    attr_set[slot] = true;
  }
  const int grid = a.tiles < 2 * mx_sm_count() ? a.tiles : 2 * mx_sm_count();
  MT_CUDA(launch_pdl(kern, dim3(grid), dim3(256), (size_t)GG_SMEM, st, mdh, mgu, a));
  return MT_OK;
}
template <int kAct>
static int gated_grad(const CUtensorMap& mdh, const CUtensorMap& mgu, const GatedGradArgs& a, cudaStream_t st) {
  const bool dgu = a.dgu != nullptr || a.amax != nullptr;
  if (a.out.q == nullptr) return launch_gated_grad<kAct, false, true, false>(mdh, mgu, a, st);
  if (a.rows % 8 != 0)
    return dgu ? launch_gated_grad<kAct, true, true, true>(mdh, mgu, a, st) : launch_gated_grad<kAct, true, false, true>(mdh, mgu, a, st);
  return dgu ? launch_gated_grad<kAct, false, true, true>(mdh, mgu, a, st) : launch_gated_grad<kAct, false, false, true>(mdh, mgu, a, st);
}

}  // namespace mt

extern "C" int mt_gated_backward(const void* dh, int64_t dh_stride, int64_t dh_rows, const void* gu, int64_t rows, int64_t F,
                                 int activation, void* dgu, float* amax, uint8_t* q, uint8_t* s, int64_t s_stride, uint8_t* s_swz, uint8_t* q_t,
                                 uint8_t* s_t, int64_t s_t_stride, uint8_t* s_t_swz, mt_stream_t stream) {
  using namespace mt;
  const char* name = "mt_gated_backward";
  MT_REQUIRE(rows >= 0 && F >= 0, "%s: negative shape", name);
  MT_REQUIRE(rows < (int64_t)1 << 30 && F < (int64_t)1 << 29, "%s: shape out of range", name);
  MT_REQUIRE(gated_act_known(activation), "%s: activation %d not supported", name, activation);
  MT_REQUIRE(F % 32 == 0, "%s: F (%lld) must be a multiple of 32", name, (long long)F);
  if (rows == 0 || F == 0) return MT_OK;
  MT_REQUIRE(dh && gu, "%s: null pointer", name);
  MT_REQUIRE(dgu || q, "%s: no output requested", name);
  MT_REQUIRE(aligned16(dh) && aligned16(gu) && aligned16(dgu), "%s: pointers must be 16-byte aligned", name);
  MT_REQUIRE(dh_stride >= F && dh_stride % 8 == 0, "%s: dh needs 16-byte aligned rows", name);
  MT_REQUIRE(dh_rows > 0 && dh_rows <= rows, "%s: dh has %lld rows for %lld of gu", name, (long long)dh_rows, (long long)rows);
  int rc = mx_outputs_ok(name, rows, 2 * F, q, s, s_stride, s_swz, q_t, s_t, s_t_stride, s_t_swz);
  if (rc != MT_OK) return rc;
  GatedGradArgs a{};
  a.rows = rows; a.F = F;
  a.dgu = static_cast<__nv_bfloat16*>(dgu); a.amax = amax;
  a.out = {q, s, s_swz, q_t, s_t, s_t_swz, rows, 2 * F, s_stride, s_t_stride, mx_padded_chunks(2 * F / 32),
           mx_padded_chunks((rows + 31) / 32)};
  const int64_t tiles_x = (F + 127) / 128, tiles = tiles_x * ((rows + 127) / 128);
  MT_REQUIRE(tiles < (int64_t)1 << 30, "%s: shape out of range", name);
  a.tiles_x = (int)tiles_x; a.tiles = (int)tiles;
  a.status = device_status_ptr();
  if (!a.status) return fail(MT_ERR_CUDA, "device status word not reachable");
  CUtensorMap mdh, mgu;
  rc = mx_tile_map(&mdh, dh, dh_rows, F, dh_stride);   // (rows beyond its own read as zeros)
  if (rc == MT_OK) rc = mx_tile_map(&mgu, gu, rows, 2 * F, 2 * F);
  if (rc != MT_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return activation == MT_ACT_SILU ? gated_grad<MT_ACT_SILU>(mdh, mgu, a, st) : gated_grad<MT_ACT_GELU>(mdh, mgu, a, st);
}
