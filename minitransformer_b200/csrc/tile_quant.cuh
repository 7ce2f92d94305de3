// MXFP8 quantization of a 32-row x 64-column tile held in the registers of one warp, row-wise and
// transposed, for kernels that have just computed the tile (norm, gated gradient): the bf16 result
// does not pass through memory.
//
// Lane l holds rows 8 (l / 8) .. +7 of columns 8 (l % 8) .. +7 as packed bf16x2, w[row][column pair].
// A 1x32 block along a row is four lanes (l xor 1, 2), a block along a column four lanes (l xor 8,
// 16). Row-wise stores are 8 bytes per lane in 64-byte runs, transposed stores 8 bytes per lane in
// runs of whole 32-byte sectors; where the row count is not a multiple of 8 these runs start anywhere and leave as aligned
// words (gated gradient, 3511 / 3512 x 4800: 76 / 50 us). Codes, scales and padding are bit for bit those of
// mt_quantize_mxfp8.
#pragma once

#include "quantize_common.cuh"

namespace mt {

struct MxTileOut {
  uint8_t *q, *s, *s_swz, *q_t, *s_t, *s_t_swz;   // q_t null: no transposed copy; *_swz may be null
  int64_t rows, cols, s_stride, s_t_stride;
  int64_t kc_row, kc_col;                         // chunks per 128-row block of s_swz / s_t_swz
};

static inline int64_t mx_padded_chunks(int64_t blocks) { return ((blocks + 3) / 4 + 3) / 4 * 4; }

// Checks of the MXFP8 output arguments of a [rows, cols] tensor (q null: none of them may be given).
static inline int mx_outputs_ok(const char* name, int64_t rows, int64_t cols, const uint8_t* q, const uint8_t* s, int64_t s_stride,
                                const uint8_t* s_swz, const uint8_t* q_t, const uint8_t* s_t, int64_t s_t_stride,
                                const uint8_t* s_t_swz) {
  if (q == nullptr) {
    MT_REQUIRE(!s && !s_swz && !q_t && !s_t && !s_t_swz, "%s: scales or transposed codes without codes", name);
    return MT_OK;
  }
  MT_REQUIRE(cols % 32 == 0, "%s: cols (%lld) must be a multiple of 32 for the MXFP8 copies", name, (long long)cols);
  MT_REQUIRE(s && s_stride >= cols / 32, "%s: codes need s with a stride of at least cols / 32", name);
  MT_REQUIRE(q_t || (!s_t && !s_t_swz), "%s: transposed scales without transposed codes", name);
  MT_REQUIRE(!q_t || (s_t && s_t_stride >= (rows + 31) / 32), "%s: transposed codes need s_t with a stride of at least rows / 32", name);
  MT_REQUIRE(aligned16(q) && aligned16(s_swz) && aligned16(q_t) && aligned16(s_t_swz), "%s: codes and swizzled scales must be 16-byte aligned", name);
  return MT_OK;
}

constexpr int MX_TILE_BYTES = 32 * 128;
// Tensor map of a bf16 matrix read in 32 x 64 tiles (zeros beyond its bounds).
static inline int mx_tile_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t stride) {
  return make_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, (uint64_t)cols, (uint64_t)rows, (uint64_t)stride * 2, 64,
                            32, CU_TENSOR_MAP_SWIZZLE_NONE);
}
// Streaming multiprocessors of the current device.
static inline int mx_sm_count() {
  static int n[MT_MAX_DEVICES] = {};
  const int slot = current_device_slot();
  if (n[slot] == 0) {
    int dev = 0, c = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
    n[slot] = c > 0 ? c : 148;
  }
  return n[slot];
}

#if defined(__CUDACC__)

// Scale of a block from the bits of its abs-max as bf16 (sign cleared): E8M0 byte and the factor 2^-e that the
// elements are multiplied by, as bf16 bits. e = ceil(log2(amax / 448)) clamped to [-127, 127], as e8m0_exponent():
// 448 = 1.75 * 2^8, so with amax = m 2^x it is x - 8, plus one if m > 1.75; adding 0x1F to the seven mantissa bits
// carries into the exponent exactly then. Infinity keeps its byte of 254.
__device__ __forceinline__ uint32_t mx_scale(uint32_t bits, uint32_t& enc) {
  const uint32_t E = max((bits + 0x1Fu) >> 7, 8u);
  const bool inf = bits == 0x7F80u;
  enc = inf ? (__float_as_uint(exp2_neg(127)) >> 16) : (262u - E) << 7;
  return inf ? 254u : E - 8u;
}
// (absmax2 with zero: a block of nothing but NaN counts as zero, as in mt_quantize_mxfp8)
__device__ __forceinline__ uint32_t mx_amax_bits(uint32_t m) {
  m = absmax2(m, 0u);
  return max(m & 0x7FFFu, (m >> 16) & 0x7FFFu);
}

// Both halves times a power of two: exact, or so small that E4M3 rounds it to zero.
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Four E4M3 bytes from four fp32 values (round to nearest even, saturating).
__device__ __forceinline__ uint32_t e4m3x4_rn(float a, float b, float c, float d) {
  uint32_t out;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(out) : "f"(a), "f"(b), "f"(c), "f"(d));
  return out;
}

// Scale bytes of a tile that this lane is to store: rows 8 (l / 8) + 2 (l % 4) + {0, 1} of the 32-column block
// (l % 8) / 4, and columns 8 (l % 8) + 2 (l / 8) + {0, 1} of the tile's one 32-row block.
struct MxTileScales {
  uint32_t row[2], col[2];
};

// A warp's 32 x 64 bf16 tile as TMA leaves it (rows of 128 bytes): this lane's 16 bytes of row i.
__device__ __forceinline__ uint4 mx_tile_row(const uint8_t* tile, int i) {
  const int lane = threadIdx.x & 31;
  uint4 v;   // volatile: stays ahead of the buffer's release
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(smem_u32(tile) + ((lane >> 3) * 8 + i) * 128 + (lane & 7) * 16) : "memory");
  return v;
}

// Gives a warp's tile buffer back before the next TMA load into it: every lane puts its reads (generic proxy) before the
// copy engine's writes (async proxy) with the proxy fence and arrives on `empty` (32 arrivals); lane 0, the one that
// loads, waits for the phase. A __syncwarp, and the arrivals without the fence, let the engine overtake the
// last reads: some rows of one in ten to one in two calls came out wrong.
__device__ __forceinline__ void mx_release_tile(uint64_t* empty, uint32_t parity, volatile int* abort_flag, int* status) {
  fence_proxy_async_smem();
  mbar_arrive(empty);
  if ((threadIdx.x & 31) == 0) mbar_wait_bounded(empty, parity, abort_flag, status, DS_EMPTY_WAIT);
  __syncwarp();
}

// Rows of [row, row + 8) below `rows`.
__device__ __forceinline__ int mx_valid_rows(int64_t rows, int64_t row) {
  return (int)max((int64_t)0, min((int64_t)8, rows - row));
}
// The first n of eight bytes, anywhere.
__device__ __forceinline__ void mx_store_bytes(uint8_t* dst, uint2 v, int n) {
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    dst[i] = static_cast<uint8_t>(v.x);
    v.x = __funnelshift_r(v.x, v.y, 8);
    v.y >>= 8;
  }
}

// Eight consecutive bytes per lane, the four lanes of a column making a run of 32 that starts anywhere: as aligned
// words, each taking the bytes it lacks from the lane before; the run's first and last bytes one by one.
__device__ __forceinline__ void mx_store_run(uint8_t* dst, uint2 v, bool ok) {
  const int rg = (threadIdx.x & 31) >> 3;
  const uint32_t a = reinterpret_cast<uintptr_t>(dst) & 3;
  const uint32_t before = __shfl_up_sync(0xffffffffu, v.y, 8);
  if (!ok) return;
  uint32_t* word = reinterpret_cast<uint32_t*>(dst - a);
  if (a == 0 || rg > 0) word[0] = __funnelshift_l(before, v.x, 8 * a);
  word[1] = __funnelshift_l(v.x, v.y, 8 * a);
  if (a != 0 && (rg == 0 || rg == 3)) {
    const uint32_t n = rg == 0 ? 4 - a : a;
    uint8_t* p = rg == 0 ? dst : dst + 8 - a;
    uint32_t b = rg == 0 ? v.x : v.y >> (8 * (4 - a));
#pragma unroll
    for (uint32_t k = 0; k < 3; ++k, b >>= 8)
      if (k < n) p[k] = static_cast<uint8_t>(b);
  }
}

// Codes of the tile -> global memory. row0 / col0: its first row and column (multiples of 32). Columns from
// `limit` on are not stored; rows beyond o.rows hold zeros. A column block is whole or absent (limit % 32 == 0).
// The abs-max of a block is reduced over its four lanes so that every exchange halves the number of rows (or
// column pairs) a lane still carries; the lane that ends up with a row computes its scale, and the factors
// travel back two to a word.
// kRagged: the row count is not a multiple of 8, so the transposed rows start anywhere.
template <bool kRagged>
__device__ __forceinline__ MxTileScales mx_tile_store(const MxTileOut& o, const uint32_t (&w)[8][4], int64_t row0, int64_t col0,
                                                      int64_t limit) {
  const int lane = threadIdx.x & 31, cg = lane & 7, rg = lane >> 3;
  const int64_t row = row0 + rg * 8, col = col0 + cg * 8;
  const bool col_ok = col < limit;
  const int nrow = col_ok ? mx_valid_rows(o.rows, row) : 0;   // rows of this lane that are stored
  MxTileScales sc;
  // ---- rows ----
  {
    uint32_t m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = absmax2(absmax2(w[i][0], w[i][1]), absmax2(w[i][2], w[i][3]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t send = (cg & 2) ? m[i] : m[i + 4], keep = (cg & 2) ? m[i + 4] : m[i];
      m[i] = absmax2(keep, __shfl_xor_sync(0xffffffffu, send, 2));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t send = (cg & 1) ? m[i] : m[i + 2], keep = (cg & 1) ? m[i + 2] : m[i];
      m[i] = absmax2(keep, __shfl_xor_sync(0xffffffffu, send, 1));
    }
    uint32_t e0, e1;
    sc.row[0] = mx_scale(mx_amax_bits(m[0]), e0);
    sc.row[1] = mx_scale(mx_amax_bits(m[1]), e1);
    const uint32_t pair = e0 | (e1 << 16);
    uint8_t* dst = o.q + row * o.cols + col;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t enc = __shfl_sync(0xffffffffu, pair, (lane & ~3) + j);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = 2 * j + h;
        const uint32_t f = h ? __byte_perm(enc, 0, 0x3232) : __byte_perm(enc, 0, 0x1010);
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = mul_bf16x2(w[i][k], f);
        if (i < nrow)
          *reinterpret_cast<uint2*>(dst) = make_uint2(e4m3x4_rn(bf16_lo(v[0]), bf16_hi(v[0]), bf16_lo(v[1]), bf16_hi(v[1])),
                                                      e4m3x4_rn(bf16_lo(v[2]), bf16_hi(v[2]), bf16_lo(v[3]), bf16_hi(v[3])));
        dst += o.cols;
      }
    }
  }
  if (o.q_t == nullptr) return sc;
  // ---- columns ----
  uint32_t m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = w[0][j];
#pragma unroll
    for (int i = 1; i < 8; ++i) m[j] = absmax2(m[j], w[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t send = (rg & 2) ? m[j] : m[j + 2], keep = (rg & 2) ? m[j + 2] : m[j];
    m[j] = absmax2(keep, __shfl_xor_sync(0xffffffffu, send, 16));
  }
  {
    const uint32_t send = (rg & 1) ? m[0] : m[1], keep = (rg & 1) ? m[1] : m[0];
    m[0] = absmax2(absmax2(keep, __shfl_xor_sync(0xffffffffu, send, 8)), 0u);
  }
  uint32_t e0, e1;
  sc.col[0] = mx_scale(m[0] & 0x7FFFu, e0);
  sc.col[1] = mx_scale((m[0] >> 16) & 0x7FFFu, e1);
  const uint32_t pair = e0 | (e1 << 16);
  uint8_t* dst = o.q_t + col * o.rows + row;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t f = __shfl_sync(0xffffffffu, pair, j * 8 + cg);
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mul_bf16x2(w[i][j], f);
    const uint2 lo = make_uint2(e4m3x4_rn(bf16_lo(v[0]), bf16_lo(v[1]), bf16_lo(v[2]), bf16_lo(v[3])),
                                e4m3x4_rn(bf16_lo(v[4]), bf16_lo(v[5]), bf16_lo(v[6]), bf16_lo(v[7])));
    const uint2 hi = make_uint2(e4m3x4_rn(bf16_hi(v[0]), bf16_hi(v[1]), bf16_hi(v[2]), bf16_hi(v[3])),
                                e4m3x4_rn(bf16_hi(v[4]), bf16_hi(v[5]), bf16_hi(v[6]), bf16_hi(v[7])));
    if (!kRagged) {                  // a lane has all of its rows or none
      if (nrow > 0) *reinterpret_cast<uint2*>(dst) = lo;
      dst += o.rows;
      if (nrow > 0) *reinterpret_cast<uint2*>(dst) = hi;
    } else if (row0 + 32 <= o.rows) {
      mx_store_run(dst, lo, col_ok);
      dst += o.rows;
      mx_store_run(dst, hi, col_ok);
    } else {
      mx_store_bytes(dst, lo, nrow);
      dst += o.rows;
      mx_store_bytes(dst, hi, nrow);
    }
    dst += o.rows;
  }
  return sc;
}

// Byte offset of the scale of (row, block) in a GEMM layout of kc chunks per 128 rows. (Its padding lets it pass 32
// bits where the tensor's own scales would not.)
__device__ __forceinline__ uint64_t mx_swz_offset(uint32_t row, uint32_t block, uint32_t kc) {
  return ((uint64_t)(row >> 7) * kc + (block >> 2)) * 512 + sf_chunk_offset((int)(row & 127), (int)(block & 3));
}
// The first n scale bytes of `word` (blocks b0 .. of one row) to their places in a row-major row (lin, null: none)
// and in the GEMM layout (swz, null: none); `whole`: n == 4, b0 % 4 == 0 and lin 4-byte aligned (uniform).
__device__ __forceinline__ void mx_store_scale_word(uint32_t word, int n, bool whole, uint8_t* lin, uint8_t* swz, uint32_t row,
                                                    uint32_t b0, uint32_t kc) {
  if (whole) {
    if (lin != nullptr) *reinterpret_cast<uint32_t*>(lin) = word;
    if (swz != nullptr) *reinterpret_cast<uint32_t*>(swz + mx_swz_offset(row, b0, kc)) = word;
  } else {
#pragma unroll 1
    for (int i = 0; i < n; ++i, word >>= 8) {
      if (lin != nullptr) lin[i] = static_cast<uint8_t>(word);
      if (swz != nullptr) swz[mx_swz_offset(row, b0 + i, kc)] = static_cast<uint8_t>(word);
    }
  }
}
__device__ __forceinline__ bool mx_word_aligned(const void* p, int64_t stride) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)stride) & 3) == 0;
}

// Zeros of the GEMM-layout scales that no tile covers: blocks beyond the last column (for `nrows` rows from
// row0, a multiple of 32 inside one 128-row block), called by `nthreads` threads.
__device__ __forceinline__ void mx_pad_row_scales(const MxTileOut& o, int64_t row0, int nrows, int tid, int nthreads) {
  if (o.s_swz == nullptr) return;
  const int64_t kb0 = o.cols >> 5, n = o.kc_row * 4 - kb0;
  for (int64_t i = tid; i < n * nrows; i += nthreads) {
    const int64_t r = row0 + i % nrows, kb = kb0 + i / nrows;
    o.s_swz[((r >> 7) * o.kc_row + (kb >> 2)) * 512 + sf_chunk_offset((int)(r & 127), (int)(kb & 3))] = 0;
  }
}
// The same for the transposed scales: feature rows beyond the last column, for token block mb.
__device__ __forceinline__ void mx_pad_col_features(const MxTileOut& o, int64_t mb, int tid, int nthreads) {
  if (o.q_t == nullptr || o.s_t_swz == nullptr || mb >= o.kc_col * 4) return;
  for (int64_t c = o.cols + tid; c < (o.cols + 127) / 128 * 128; c += nthreads)
    o.s_t_swz[((c >> 7) * o.kc_col + (mb >> 2)) * 512 + sf_chunk_offset((int)(c & 127), (int)(mb & 3))] = 0;
}
// And token blocks from mb0 (a multiple of 4) up to the padded count, for features [c0, c1).
__device__ __forceinline__ void mx_pad_col_blocks(const MxTileOut& o, int64_t mb0, int64_t c0, int64_t c1, int tid, int nthreads) {
  if (o.q_t == nullptr || o.s_t_swz == nullptr) return;
  const int64_t k0 = mb0 >> 2, n = o.kc_col - k0;
  for (int64_t i = tid; i < n * (c1 - c0); i += nthreads) {
    const int64_t c = c0 + i % (c1 - c0), k = k0 + i / (c1 - c0);
    *reinterpret_cast<uint32_t*>(o.s_t_swz + ((c >> 7) * o.kc_col + k) * 512 + sf_chunk_offset((int)(c & 127), 0)) = 0u;
  }
}

#endif  // __CUDACC__

}  // namespace mt
