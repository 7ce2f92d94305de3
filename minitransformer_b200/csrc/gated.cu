// Gradient of the gated activation: from dh and the saved projections [g | u],
//   du = bf16(dh * act(g)),   dg = bf16(dh * u * act'(g))
// and, from the same registers, the MXFP8 copies of [dg | du] that the dgrad and wgrad GEMMs read (row-wise and
// transposed). 2 + 4 bytes read and 4 written per (row, feature): bound by HBM.
#include "gated_act.cuh"
#include "tile_quant.cuh"

namespace mt {

struct GatedGradArgs {
  const __nv_bfloat16 *dh, *gu;
  int64_t dh_stride, rows, F;
  __nv_bfloat16* dgu;
  float* amax;
  MxTileOut out;       // out.q null: no copies
};

// A CTA covers 128 rows x 128 features: four warps of 32 rows side by side in each of two 64-column halves, so that
// row-wise codes leave in whole 128-byte lines and transposed codes in 128-byte runs of one feature. All loads of
// a thread (24 of 16 bytes) are issued before the first is used: the two CTAs of an SM then keep 196 KB in flight,
// and one computes while the other waits. Scale bytes are collected in shared memory and leave as words.
template <int kAct>
__global__ void __launch_bounds__(256, 2) gated_grad_kernel(const GatedGradArgs a) {
  __shared__ __align__(16) uint8_t s_row[2][128][4], s_col[2][128][4];   // [dg, du][row / feature][block]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m0 = (int64_t)blockIdx.y * 128, f0 = (int64_t)blockIdx.x * 128;
  const int wr = warp & 3, wc = warp >> 2;
  const int64_t row0 = m0 + wr * 32, c0 = f0 + wc * 64;
  const int64_t row = row0 + (lane >> 3) * 8, f = c0 + (lane & 7) * 8;
  const bool f_ok = f < a.F;
  pdl_trigger();
  pdl_wait();
  uint4 d4[8], g4[8], u4[8];
  const __nv_bfloat16* pd = a.dh + row * a.dh_stride + f;
  const __nv_bfloat16* pg = a.gu + row * 2 * a.F + f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    d4[i] = g4[i] = u4[i] = make_uint4(0, 0, 0, 0);
    if (f_ok && row + i < a.rows) {
      g4[i] = *reinterpret_cast<const uint4*>(pg + i * 2 * a.F);
      d4[i] = *reinterpret_cast<const uint4*>(pd + i * a.dh_stride);
      u4[i] = *reinterpret_cast<const uint4*>(pg + i * 2 * a.F + a.F);
    }
  }
  uint32_t wg[8][4], wu[8][4], am = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t d[4] = {d4[i].x, d4[i].y, d4[i].z, d4[i].w}, g[4] = {g4[i].x, g4[i].y, g4[i].z, g4[i].w};
    const uint32_t u[4] = {u4[i].x, u4[i].y, u4[i].z, u4[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x2_t act, grad;
      gated_act_grad2<kAct>(bf16x2_to_f32x2(g[j]), act, grad);
      const f32x2_t d2 = bf16x2_to_f32x2(d[j]);
      wu[i][j] = f32x2_to_bf16x2(mul2(d2, act));
      wg[i][j] = f32x2_to_bf16x2(mul2(mul2(d2, bf16x2_to_f32x2(u[j])), grad));
    }
    if (a.dgu != nullptr && f_ok && row + i < a.rows) {
      *reinterpret_cast<uint4*>(a.dgu + (row + i) * 2 * a.F + f) = make_uint4(wg[i][0], wg[i][1], wg[i][2], wg[i][3]);
      *reinterpret_cast<uint4*>(a.dgu + (row + i) * 2 * a.F + a.F + f) = make_uint4(wu[i][0], wu[i][1], wu[i][2], wu[i][3]);
    }
  }
  if (a.amax != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) am = absmax2(am, absmax2(wu[i][j], wg[i][j]));
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(absmax2_to_float(am)));
    if (lane == 0 && bits != 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), bits);
  }
  const MxTileOut& o = a.out;
  if (o.q == nullptr) return;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const MxTileScales sc = p ? mx_tile_store(o, wu, row0, a.F + c0, 2 * a.F) : mx_tile_store(o, wg, row0, c0, a.F);
    const int r = wr * 32 + (lane >> 3) * 8 + (lane & 3) * 2, kb = wc * 2 + ((lane & 7) >> 2);
    const int c = wc * 64 + (lane & 7) * 8 + (lane >> 3) * 2;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s_row[p][r + j][kb] = static_cast<uint8_t>(sc.row[j]);
      s_col[p][c + j][wr] = static_cast<uint8_t>(sc.col[j]);
    }
  }
  __syncthreads();
  const int t = tid & 127;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (tid < 128) {
      const int64_t b0 = (p ? a.F + f0 : f0) >> 5;
      const int n = (int)min((int64_t)4, (a.F - f0) >> 5);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(s_row[p][t]);
      mx_store_scale_word(word, n, m0 + t < o.rows ? o.s + (m0 + t) * o.s_stride + b0 : nullptr, o.s_swz, m0 + t, b0, o.kc_row);
    } else if (o.q_t != nullptr && f0 + t < a.F) {
      const int64_t c = (p ? a.F : 0) + f0 + t, b0 = m0 >> 5;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(s_col[p][t]);
      const int n = (int)min((int64_t)4, ((o.rows + 31) >> 5) - b0);
      mx_store_scale_word(word, n, o.s_t + c * o.s_t_stride + b0, nullptr, c, b0, o.kc_col);
      mx_store_scale_word(word, 4, nullptr, o.s_t_swz, c, b0, o.kc_col);   // token blocks without a row: zeros
    }
  }
  // padding of the GEMM-layout scales: beyond the last feature, and token blocks up to the padded count
  const int64_t mb0 = m0 >> 5, f1 = min(f0 + 128, a.F);
  const bool last_x = blockIdx.x == gridDim.x - 1, last_y = blockIdx.y == gridDim.y - 1;
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

}  // namespace mt

extern "C" int mt_gated_backward(const void* dh, int64_t dh_stride, const void* gu, int64_t rows, int64_t F, int activation,
                                 void* dgu, float* amax, uint8_t* q, uint8_t* s, int64_t s_stride, uint8_t* s_swz, uint8_t* q_t,
                                 uint8_t* s_t, int64_t s_t_stride, uint8_t* s_t_swz, mt_stream_t stream) {
  using namespace mt;
  const char* name = "mt_gated_backward";
  MT_REQUIRE(rows >= 0 && F >= 0, "%s: negative shape", name);
  MT_REQUIRE(rows < (int64_t)1 << 23 && F < (int64_t)1 << 30, "%s: shape out of range", name);   // grid.y <= 65535
  MT_REQUIRE(gated_act_known(activation), "%s: activation %d not supported", name, activation);
  MT_REQUIRE(F % 32 == 0, "%s: F (%lld) must be a multiple of 32", name, (long long)F);
  if (rows == 0 || F == 0) return MT_OK;
  MT_REQUIRE(dh && gu, "%s: null pointer", name);
  MT_REQUIRE(dgu || q, "%s: no output requested", name);
  MT_REQUIRE(aligned16(dh) && aligned16(gu) && aligned16(dgu), "%s: pointers must be 16-byte aligned", name);
  MT_REQUIRE(dh_stride >= F && dh_stride % 8 == 0, "%s: dh needs 16-byte aligned rows", name);
  int rc = mx_outputs_ok(name, rows, 2 * F, q, s, s_stride, s_swz, q_t, s_t, s_t_stride, s_t_swz);
  if (rc != MT_OK) return rc;
  GatedGradArgs a{};
  a.dh = static_cast<const __nv_bfloat16*>(dh); a.gu = static_cast<const __nv_bfloat16*>(gu);
  a.dh_stride = dh_stride; a.rows = rows; a.F = F;
  a.dgu = static_cast<__nv_bfloat16*>(dgu); a.amax = amax;
  a.out = {q, s, s_swz, q_t, s_t, s_t_swz, rows, 2 * F, s_stride, s_t_stride, mx_padded_chunks(2 * F / 32),
           mx_padded_chunks((rows + 31) / 32)};
  const dim3 grid((unsigned)((F + 127) / 128), (unsigned)((rows + 127) / 128));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (activation == MT_ACT_SILU) MT_CUDA(launch_pdl(gated_grad_kernel<MT_ACT_SILU>, grid, dim3(256), 0, st, a));
  else MT_CUDA(launch_pdl(gated_grad_kernel<MT_ACT_GELU>, grid, dim3(256), 0, st, a));
  return MT_OK;
}
