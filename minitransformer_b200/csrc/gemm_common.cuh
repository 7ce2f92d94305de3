// Device helpers shared by the block-scaled GEMM kernels: operand formats, MMA instruction
// descriptors and issue (one CTA and CTA pair), abs-max tracking, sector-wide stores.
#pragma once

#include "mt_common.cuh"

namespace mt {

constexpr int G_BLOCK_M = 128;
constexpr int G_BLOCK_KB = 128;  // bytes of K per row per stage (256 FP4 or 128 FP8 elements)
constexpr int G_THREADS = 192;
constexpr int G_TMEM_COLS = 512;

enum GemmFormat : int { FMT_NVFP4 = 0, FMT_MXFP8 = 1 };

#if defined(__CUDACC__)

__device__ __forceinline__ uint32_t make_idesc(int format, int block_n, int sf_id) {
  uint32_t d = 0;
  if (format == FMT_NVFP4) {
    d |= 1u << 7;   // A: E2M1
    d |= 1u << 10;  // B: E2M1
    // scale format UE4M3 = 0 at bit 23
  } else {
    // A, B: E4M3 = 0
    d |= 1u << 23;                             // scale format UE8M0
    d |= static_cast<uint32_t>(sf_id) << 4;    // B scale-factor byte inside the 32-bit column
    d |= static_cast<uint32_t>(sf_id) << 29;   // A scale-factor byte
  }
  d |= static_cast<uint32_t>(block_n >> 3) << 17;
  d |= static_cast<uint32_t>(G_BLOCK_M >> 4) << 24;
  return d;
}

template <int kFormat>
__device__ __forceinline__ void issue_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if (kFormat == FMT_NVFP4) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  }
}

template <int kFormat>
__device__ __forceinline__ void issue_mma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if (kFormat == FMT_NVFP4) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  }
}

__device__ __forceinline__ uint32_t make_idesc_pair(int format, int block_n, int sf_id) {
  uint32_t d = 0;
  if (format == FMT_NVFP4) {
    d |= 1u << 7;
    d |= 1u << 10;
  } else {
    d |= 1u << 23;
    d |= static_cast<uint32_t>(sf_id) << 4;
    d |= static_cast<uint32_t>(sf_id) << 29;
  }
  d |= static_cast<uint32_t>(block_n >> 3) << 17;
  d |= static_cast<uint32_t>(256 >> 4) << 24;  // M = 256 across the pair
  return d;
}

// Running abs-max of what a thread stores: bf16 outputs are tracked two per word with the packed
// bf16 instruction (sign bits are garbage until amax_finish strips them), fp32 outputs as fp32.
struct AmaxAcc {
  uint32_t packed = 0;
  float f = 0.0f;
};
__device__ __forceinline__ void amax_bf16x2(AmaxAcc& m, uint32_t w) {
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m.packed) : "r"(m.packed), "r"(w));
}
__device__ __forceinline__ float amax_finish(const AmaxAcc& m) {
  const uint32_t p = m.packed & 0x7FFF7FFFu;
  return fmaxf(m.f, fmaxf(__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u)));
}
// Warp-wide maximum of the threads' abs-max values -> one atomic max on the fp32 scalar (values
// are non-negative, so their bit patterns order like unsigned integers).
__device__ __forceinline__ void amax_publish(float* d_amax, const AmaxAcc& m, int lane) {
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(amax_finish(m)));
  if (lane == 0 && bits != 0) atomicMax(reinterpret_cast<unsigned int*>(d_amax), bits);
}

__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

#endif  // __CUDACC__

}  // namespace mt
