// Block-scaled 4-bit floating point: element and scale conversions, the scale layout, and the tcgen05 forms
// that multiply such operands.
//
// A code is an e2m1 value: +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}. Two formats (include/foidfinder_b200.h):
//   FF_FP4_NV  16 columns share a UE4M3 scale S; a row has an f32 scale s, a power of two
//   FF_FP4_MX  32 columns share a UE8M0 scale, a power of two; no row scale
//
// Scales are stored as the tensor cores read them: 512-byte chunks of 128 rows x 4 scales along the columns
// (64 columns of FF_FP4_NV, 128 of FF_FP4_MX), row r's four scales at byte (r % 32) * 16 + (r / 32) * 4. The
// chunks of one 128-row tile are contiguous along the columns, padded to whole 256-column steps with zero
// scales, so that a step's chunks are one 2048-byte (NV) or 1024-byte (MX) copy.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace ff {

constexpr int kFp4Step = 256;      // columns per 128-byte row of codes: one stage of the product's K loop
constexpr int kSfChunk = 512;      // bytes of one scale chunk

__host__ __device__ constexpr int fp4_block(bool mx) { return mx ? 32 : 16; }
__host__ __device__ constexpr int sf_chunks_per_step(bool mx) { return mx ? 2 : 4; }
// Byte pitch of a row of codes: columns padded to 32 so that every row starts 16-byte aligned.
__host__ __device__ constexpr int64_t fp4_row_bytes(int cols) { return static_cast<int64_t>((cols + 31) / 32) * 16; }
__host__ __device__ constexpr int64_t sf_tile_bytes(int cols, bool mx) {
  return static_cast<int64_t>((cols + kFp4Step - 1) / kFp4Step) * sf_chunks_per_step(mx) * kSfChunk;
}
// Byte of row `row`'s scale of column block `blk`.
__host__ __device__ constexpr int64_t sf_offset(int row, int blk, int64_t tile_bytes) {
  return static_cast<int64_t>(row >> 7) * tile_bytes + static_cast<int64_t>(blk >> 2) * kSfChunk + (row & 31) * 16 +
         ((row >> 5) & 3) * 4 + (blk & 3);
}

// ---------------------------------------------------------------- conversions
// Eight f32 -> eight e2m1 codes, element i in bits [4i, 4i + 4): round to nearest even, saturating at +-6.
__device__ __forceinline__ uint32_t e2m1x8(const float2* y) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(y[0].x), "f"(y[0].y), "f"(y[1].x), "f"(y[1].y), "f"(y[2].x), "f"(y[2].y), "f"(y[3].x), "f"(y[3].y));
  return r;
}
// Eight e2m1 codes -> four half2 (exact).
__device__ __forceinline__ void e2m1x8_to_half2(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}
// f32 >= 0 -> e4m3 byte, nearest even, saturating at 448.
__device__ __forceinline__ uint32_t e4m3_byte(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(byte)));
  return unpack_half2(h).x;
}
// 2^(byte - 127); byte 0 is the f32 subnormal 2^-127, 255 is NaN.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// 16-bit storage types by template.
template <class T>
struct Pair16;
template <>
struct Pair16<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return unpack_half2(v); }
};
template <>
struct Pair16<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

// Arrive on another CTA's barrier (a shared::cluster address) without release: for an arrival that hands over
// TMEM which this thread has finished reading (tcgen05.wait::ld), so that there are no writes to publish. The
// releasing form waited for every outstanding write of the CTA, 1.5-2 us under the epilogue's stores.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// ---------------------------------------------------------------- tcgen05
// Instruction descriptor of the block-scaled 4-bit MMAs, both operands e2m1 and K-major.
// Bits: [4,6) B scale id, [7,10) A format, [10,12) B format (1 = e2m1), [17,23) N>>3, 23 scale type
// (0 UE4M3, 1 UE8M0), [24,29) M>>4, [29,31) A scale id. The scale ids pick the byte (of the four that one
// 32-bit TMEM column holds per row) where an MMA's scales start.
__host__ __device__ constexpr uint32_t idesc_fp4(int m, int n, bool mx) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (mx ? 1u << 23 : 0u) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
__host__ __device__ constexpr uint32_t idesc_sf_id(uint32_t id) { return (id << 4) | (id << 29); }

// Shared-memory descriptor of one scale chunk (32 rows x 16 bytes, no swizzle: 8-row groups 128 bytes apart).
__device__ __forceinline__ uint64_t sdesc_sf(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 32;  // stride byte offset
  d |= static_cast<uint64_t>(1u) << 46;         // descriptor version for sm_100
  return d;
}
// One chunk into four TMEM columns, repeated in all four lane quarters. Issued by the thread that issues the
// MMAs: tcgen05.cp and tcgen05.mma of one thread execute in order.
template <bool PAIR>
__device__ __forceinline__ void tc_cp_sf(uint32_t taddr, uint64_t sdesc) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

// D (+)= (A scaled) * (B scaled)^T over 64 columns.
template <bool PAIR, bool MX>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define FF_MMA_FP4(GROUP, KIND, VEC)                                                                             \
  asm volatile("{\n\t.reg .pred p;\n\t"                                                                          \
               "setp.ne.b32 p, %6, 0;\n\t"                                                                       \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND ".block_scale.scale_vec::" VEC                     \
               " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),                                         \
               "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                         \
               : "memory")
  if constexpr (PAIR) {
    if constexpr (MX)
      FF_MMA_FP4("2", "mxf4", "2X");
    else
      FF_MMA_FP4("2", "mxf4nvf4", "4X");
  } else {
    if constexpr (MX)
      FF_MMA_FP4("1", "mxf4", "2X");
    else
      FF_MMA_FP4("1", "mxf4nvf4", "4X");
  }
#undef FF_MMA_FP4
}

}  // namespace ff
