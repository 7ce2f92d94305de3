// Gradient of the gated activation: from dh and the saved projections [g | u],
//   du = bf16(dh * act(g)),   dg = bf16(dh * u * act'(g))
// Elementwise; 2 + 4 bytes read per (row, feature) and 4 written: bound by HBM.
#include "gated_act.cuh"
#include "quantize_common.cuh"

namespace mt {

struct GatedGradArgs {
  const __nv_bfloat16 *dh, *gu;
  int64_t dh_stride, rows, F;
  __nv_bfloat16* dgu;
  float* amax;
};

// 8 features per thread.
template <int kAct>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GatedGradArgs a) {
  pdl_trigger();
  pdl_wait();
  const int64_t per_row = a.F >> 3, n = a.rows * per_row;
  uint32_t am = 0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per_row, f = (i - row * per_row) * 8;
    const uint4 d4 = *reinterpret_cast<const uint4*>(a.dh + row * a.dh_stride + f);
    const uint4 g4 = *reinterpret_cast<const uint4*>(a.gu + row * 2 * a.F + f);
    const uint4 u4 = *reinterpret_cast<const uint4*>(a.gu + row * 2 * a.F + a.F + f);
    const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a0, a1, p0, p1;
      gated_act_grad<kAct>(bf16_lo(g[j]), a0, p0);
      gated_act_grad<kAct>(bf16_hi(g[j]), a1, p1);
      const float d0 = bf16_lo(d[j]), d1 = bf16_hi(d[j]);
      ou[j] = f32x2_to_bf16x2(pack2(d0 * a0, d1 * a1));
      og[j] = f32x2_to_bf16x2(pack2(d0 * bf16_lo(u[j]) * p0, d1 * bf16_hi(u[j]) * p1));
      am = absmax2(am, absmax2(ou[j], og[j]));
    }
    *reinterpret_cast<uint4*>(a.dgu + row * 2 * a.F + f) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(a.dgu + row * 2 * a.F + a.F + f) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
  if (a.amax != nullptr) {
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(absmax2_to_float(am)));
    if ((threadIdx.x & 31) == 0 && bits != 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), bits);
  }
}

}  // namespace mt

extern "C" int mt_gated_backward(const void* dh, int64_t dh_stride, const void* gu, int64_t rows, int64_t F, int activation,
                                 void* dgu, float* amax, mt_stream_t stream) {
  using namespace mt;
  const char* name = "mt_gated_backward";
  MT_REQUIRE(rows >= 0 && F >= 0, "%s: negative shape", name);
  MT_REQUIRE(rows < (int64_t)1 << 31 && F < (int64_t)1 << 30, "%s: shape out of range", name);
  MT_REQUIRE(gated_act_known(activation), "%s: activation %d not supported", name, activation);
  MT_REQUIRE(F % 32 == 0, "%s: F (%lld) must be a multiple of 32", name, (long long)F);
  if (rows == 0 || F == 0) return MT_OK;
  MT_REQUIRE(dh && gu && dgu, "%s: null pointer", name);
  MT_REQUIRE(aligned16(dh) && aligned16(gu) && aligned16(dgu), "%s: pointers must be 16-byte aligned", name);
  MT_REQUIRE(dh_stride >= F && dh_stride % 8 == 0, "%s: dh needs 16-byte aligned rows", name);
  GatedGradArgs a{static_cast<const __nv_bfloat16*>(dh), static_cast<const __nv_bfloat16*>(gu), dh_stride, rows, F,
                  static_cast<__nv_bfloat16*>(dgu), amax};
  const int64_t n = rows * (F / 8);
  const unsigned grid = (unsigned)((n + 255) / 256 < 148 * 16 ? (n + 255) / 256 : 148 * 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (activation == MT_ACT_SILU) MT_CUDA(launch_pdl(gated_grad_kernel<MT_ACT_SILU>, dim3(grid), dim3(256), 0, st, a));
  else MT_CUDA(launch_pdl(gated_grad_kernel<MT_ACT_GELU>, dim3(grid), dim3(256), 0, st, a));
  return MT_OK;
}
