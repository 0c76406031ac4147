// Block-scaled 4-bit quantisation (with an optional LayerNorm in front) and its inverse.
//
//   x [rows, cols] -> (LayerNorm over the row, f32 statistics) -> v
//   FF_FP4_NV: s = smallest power of two (>= 2^-110) with amax(row) <= 2688 s (2688 = 6 * 448)
//              S = e4m3(amax(block of 16) / (6 s)),  code = e2m1(v / (S s))
//   FF_FP4_MX: scale = 2^(floor(log2 amax(block of 32)) - 2),  code = e2m1(v / scale)
//
// The power-of-two row scale costs no accuracy that the e4m3 block scale would have kept, and makes v / s and
// S * s exact, so the codes are the correctly rounded quotients: amax / 6 is rounded correctly (sixth()), and v / S
// is a product with the reciprocal whose last bits are snapped off for 16-bit inputs, and corrected by its remainder
// for f32 (quotient2(); 5460 x 1024 6.9 us, 10.3 with IEEE divisions).
// A row (NV) or block (MX) that holds an infinity or NaN gets a NaN scale, so that it shows in every result.
//
// Bound by HBM: 2 bytes read and 0.56 (NV) or 0.53 (MX) written per value. The whole row stays in registers,
// 16 consecutive columns per lane, so a 16-column block never leaves its lane and a 32-column block is a pair
// of lanes. Without a norm a warp takes rows of 16-bit values up to 5120 columns wide, packed as loaded; with one,
// and for f32, a row's values are f32 in as many warps as leave each lane 32 or 48 of them. CTAs are persistent.
//
// Measured, 65600 rows of 1024 fp16 (171 MB moved): NV 27.5 us, 95% of the copy rate, MX 26.7. 65600 x 2730 bf16: MX
// 72 us where rows start at 16-byte boundaries and 84 where they do not (shifting them into place doubles the
// instructions); NV 71 and 85. With LayerNorm 38 us and 126 (2730): bound by the shared-memory pipe (88% busy at 1024
// columns), which delivers 8 bytes of gamma and beta per value. What did not help: two rows at a time for the same gamma
// and beta (38.9 us and 140: half the warps), half a row per warp with two rows (43 and 172: barriers), the next row read
// ahead into shared memory (50 and 148), 32-byte loads (37.6 and 148), gamma and beta in registers (73) or TMEM (78).
// Dequantisation, 65600 x 1024 fp16 30 us (5.7 TB/s), 32000 x 4096 f32 102 us; 65600 x 2730 bf16 89 us aligned, 105 not.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kQuantThreads = 256;

// 16 consecutive values of a row, as loaded. Rows may start anywhere: whole aligned 16-byte granules are read, those
// that hold at least one byte of the row, and shifted into place afterwards.
template <class T, bool ALIGNED>
struct Raw {
  static constexpr int W = sizeof(T) * 4;  // words of 16 values
  uint32_t t[ALIGNED ? W : W + 4];
};

template <class T, bool ALIGNED>
__device__ __forceinline__ void load_raw(const T* __restrict__ xr, int col, int cols, Raw<T, ALIGNED>& r) {
  constexpr int E = 16 / sizeof(T);  // values per granule
  constexpr int N = Raw<T, ALIGNED>::W / 4 + (ALIGNED ? 0 : 1);
  // values between the granule's start and the row's (the same for all columns)
  const int mis = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(xr) & 15u) / static_cast<int>(sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(xr + col - mis);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (col < cols && col + E * j - mis < cols) u = __ldg(base + j);
    r.t[4 * j] = u.x;
    r.t[4 * j + 1] = u.y;
    r.t[4 * j + 2] = u.z;
    r.t[4 * j + 3] = u.w;
  }
}

// The loaded words shifted into place, values at or past the row's end zero.
template <class T, bool ALIGNED, bool WHOLE = false>
__device__ __forceinline__ void realign(const T* xr, int col, int cols, Raw<T, ALIGNED>& r) {
  constexpr int W = Raw<T, ALIGNED>::W;
  if constexpr (!ALIGNED) {
    const uint32_t mis = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(xr)) & 15u;  // the same for all columns
    const uint32_t sh = (mis & 2u) * 8u;  // 0 or 16 bits
    auto shift = [&](auto words) {
      constexpr int K = decltype(words)::value;
#pragma unroll
      for (int i = 0; i < W; ++i) r.t[i] = sizeof(T) == 4 ? r.t[i + K] : __funnelshift_r(r.t[i + K], r.t[i + K + 1], sh);
    };
    switch (mis >> 2) {  // one move per word, where shifting by 8, 4 and 2 bytes in turn took three
      case 0: shift(std::integral_constant<int, 0>{}); break;
      case 1: shift(std::integral_constant<int, 1>{}); break;
      case 2: shift(std::integral_constant<int, 2>{}); break;
      default: shift(std::integral_constant<int, 3>{});
    }
  }
  if (!WHOLE && col + 16 > cols) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) {
        if (col + i >= cols) r.t[i] = 0;
      } else {
        if (col + 2 * i >= cols)
          r.t[i] = 0;
        else if (col + 2 * i + 1 >= cols)
          r.t[i] &= 0xffffu;
      }
    }
  }
}

template <class T>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (sizeof(T) == 2)
    return Pair16<T>::unpack(w);
  else
    return make_float2(0.f, 0.f);
}
template <class T, bool ALIGNED>
__device__ __forceinline__ void to_f32(const Raw<T, ALIGNED>& r, float2 (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    v[e] = sizeof(T) == 4 ? make_float2(__uint_as_float(r.t[sizeof(T) == 4 ? 2 * e : 0]), __uint_as_float(r.t[sizeof(T) == 4 ? 2 * e + 1 : 0]))
                          : unpack16<T>(r.t[e]);
}

template <class T>
__device__ __forceinline__ void load16(const T* __restrict__ xr, int col, int cols, float2 (&v)[8]) {
  Raw<T, false> r;
  load_raw<T, false>(xr, col, cols, r);
  realign<T, false>(xr, col, cols, r);
  to_f32<T, false>(r, v);
}

// Maximum of magnitudes that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b, float c = 0.f) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float amax16(const float2 (&v)[8]) {
  float m[2] = {0.f, 0.f};  // two chains
#pragma unroll
  for (int e = 0; e < 8; ++e) m[e & 1] = max_nan(m[e & 1], v[e].x, v[e].y);
  return max_nan(m[0], m[1]);
}
// The same on 16-bit pairs as loaded (the running maximum's sign is not meaningful until the end).
template <class T>
__device__ __forceinline__ float amax_pairs(const uint32_t* w) {
  uint32_t m[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (std::is_same<T, __half>::value)
      asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m[e & 1]) : "r"(w[e]));
    else
      asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m[e & 1]) : "r"(w[e]));
  }
  const float2 a = Pair16<T>::unpack(m[0]), b = Pair16<T>::unpack(m[1]);
  return max_nan(max_nan(a.x, a.y, b.x), b.y);
}
__device__ __forceinline__ bool not_finite(float amax) { return !(amax <= 3.402823466e38f); }

// FF_FP4_NV row scale s = 2^e: e = floor(log2 amax) - 11, one more when amax's mantissa is above 2688's
// (1.3125), and -110 at least.
__device__ __forceinline__ float nv_row_scale(float amax) {
  const int biased = static_cast<int>((__float_as_uint(amax) + (0x7fffffu - 0x280000u)) >> 23) - 11;
  return __uint_as_float(static_cast<uint32_t>(max(biased, 127 - 110)) << 23);
}
__device__ __forceinline__ float inv_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// v / (S s) for the code, r about 1 / (S s). A code's ties are T = 0.25, 0.75, 1.25, 1.75, 2.5, 3.5 and 5; T S s has
// at most seven significant bits (three of T, four of S), and a quotient is a tie only if v is T S s.
// kExact16: v came from a 16-bit type and has at most 11 significant bits, so v and T S s differ by 2^-11 of themselves or
//   not at all: a quotient that is no tie is at least 2^-11 T, that is 2^-13, away from one, while v * r is within 2^-20 of the quotient. Rounding v * r + 192 (one
//   FMA, to multiples of 2^-16) puts true ties exactly on the tie and moves no other across (r within 2^-22 of 1 / (S s) is
//   enough).
// kExact32: v from f32 and already divided by s (exact, or far below any tie), r the reciprocal of scale = S. The quotient
//   v * r is corrected by its remainder, which is exact in an FMA (P. Markstein, Computation of elementary functions on the
//   IBM RISC System/6000 processor, IBM J. Res. Dev. 34, 1990): before its rounding the result is within 2^-45 of the true
//   quotient Q. With Q = T it rounds to T. Otherwise |Q - T| is at least u / S, u the unit in the last place of T S. Let a and
//   b be the significands of T and S, in [1, 2), and h half the unit in the last place of T (a <= 1.75). Above T,
//   u / S = 2 h / b where a b < 2 and 4 h / b where not: for a = 1 (T = 0.25) at least 2 h / 1.875 = 1.067 h, for a = 1.25
//   (b <= 1.5) 1.33 h, for 1.5 (b <= 1.25) 1.6 h, for 1.75 (b <= 1.125) 1.78 h. Below T it is the same, but for T = 0.25,
//   where h is half as large, and T S a power of two (a = b = 1), where both are: 2 h at least. Always more than h, so the
//   result rounds to T's neighbour or beyond.
// kPlain: v is itself rounded (after a LayerNorm) or r a power of two.
enum QuotientKind { kPlain, kExact16, kExact32 };
template <int KIND>
__device__ __forceinline__ float2 quotient2(float2 v, float r, float scale) {
  if constexpr (KIND == kExact32) {
    const float2 r2 = make_float2(r, r), q = mul2(v, r2);
    return fma2(fma2(q, make_float2(-scale, -scale), v), r2, q);
  } else if constexpr (KIND == kExact16) {
    return add2(fma2(v, make_float2(r, r), make_float2(192.f, 192.f)), make_float2(-192.f, -192.f));
  } else {
    return mul2(v, make_float2(r, r));
  }
}

template <int KIND>
__device__ __forceinline__ uint2 codes16(const float2 (&v)[8], float r, float scale) {
  float2 q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = quotient2<KIND>(v[e], r, scale);
  return make_uint2(e2m1x8(q), e2m1x8(q + 4));
}

// amax / 6, its product with 1 / 6 corrected by the remainder in the same way. Ties of e4m3 have five significant bits: a
// quotient that is one comes out as it is. Any other is u / 6 away at least, u the unit in the last place of 6 T:
// 4/3 of half the unit in the last place of T (significand below 4/3) or 8/3 (above), and does not move onto it.
__device__ __forceinline__ float sixth(float a) {
  const float q = a * (1.f / 6.f);
  return fmaf(fmaf(-6.f, q, a), 1.f / 6.f, q);
}
// One 16-column piece of an NV row with row scale s: its scale byte and codes.
template <int KIND>
__device__ __forceinline__ uint32_t nv_piece(const float2 (&v)[8], float amax, float s, bool bad, uint2* codes) {
  const float is = inv_pow2(s);
  const float t = sixth(amax * is);
  const uint32_t byte = bad ? 0u : e4m3_byte(t);
  const float S = e4m3_value(byte);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(S));
  r = fmaf(r, fmaf(-S, r, 1.f), r);  // one step of Newton's method
  if constexpr (KIND == kExact32) {
    float2 u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = mul2(v[e], make_float2(is, is));
    *codes = bad ? make_uint2(0, 0) : codes16<KIND>(u, byte ? r : 0.f, S);
  } else {
    *codes = bad ? make_uint2(0, 0) : codes16<KIND>(v, byte ? r * is : 0.f, S * s);
  }
  return byte;
}
// One 16-column piece of an MX block whose 32 columns have maximum amax. Scaling by a power of two is exact.
__device__ __forceinline__ uint32_t mx_piece(const float2 (&v)[8], float amax, uint2* codes) {
  if (not_finite(amax)) {
    *codes = make_uint2(0, 0);
    return 255u;
  }
  const int byte = max(static_cast<int>(__float_as_uint(amax) >> 23) - 2, 0);
  *codes = codes16<kPlain>(v, __uint_as_float(static_cast<uint32_t>(254 - byte) << 23), 0.f);
  return static_cast<uint32_t>(byte);
}

template <class T, bool NORM>
__device__ constexpr int quotient_kind() {
  return NORM ? kPlain : sizeof(T) == 4 ? kExact32 : kExact16;
}

struct QuantArgs {
  const void* x;
  int64_t ldx;
  const float *gamma, *beta;
  float eps;
  int rows, cols;
  uint8_t *codes, *scales;
  float* row_scale;
};

__device__ __forceinline__ void affine16(float2 (&v)[8], float mean, float rstd, const QuantArgs& a, int col) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = col + 2 * e;
    v[e].x = c < a.cols ? fmaf(v[e].x - mean, rstd * __ldg(a.gamma + c), __ldg(a.beta + c)) : 0.f;
    v[e].y = c + 1 < a.cols ? fmaf(v[e].y - mean, rstd * __ldg(a.gamma + c + 1), __ldg(a.beta + c + 1)) : 0.f;
  }
}

// Where a row's codes and scales go.
struct RowOut {
  uint8_t *codes, *scales;
  int pitch;
};
template <bool MX>
__device__ __forceinline__ RowOut row_out(const QuantArgs& a, int row) {
  const int64_t pitch = fp4_row_bytes(a.cols);
  return {a.codes + row * pitch, a.scales + sf_offset(row, 0, sf_tile_bytes(a.cols, MX)), static_cast<int>(pitch)};
}
// Codes and scale byte of the piece at 16-column index c. Lanes hold consecutive c: the warp's byte stores fall into
// whole 4-byte groups of the scale chunks.
template <bool MX>
__device__ __forceinline__ void store_piece(const RowOut& o, int c, int pieces, uint2 codes, uint32_t byte) {
  if (c >= pieces) return;
  if (8 * c < o.pitch) *reinterpret_cast<uint2*>(o.codes + 8 * c) = codes;
  if (MX) {
    if ((c & 1) == 0) o.scales[(c >> 3) * kSfChunk + ((c >> 1) & 3)] = static_cast<uint8_t>(byte);
  } else {
    o.scales[(c >> 2) * kSfChunk + (c & 3)] = static_cast<uint8_t>(byte);
  }
}

// gamma and beta in shared memory, zero past the row's end: columns 4 j .. 4 j + 3 of the 16-column piece c are the
// float4 at plane j of P pieces (beta: plane 4 + j), so that lanes with consecutive pieces read consecutive float4.
__device__ __forceinline__ void fill_norm(float4* norm_s, const QuantArgs& a, int P) {
  for (int i = threadIdx.x; i < P * 4; i += blockDim.x) {
    const int c = i >> 2, j = i & 3;
    float g[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int col = 16 * c + 4 * j + e;
      g[e] = col < a.cols ? __ldg(a.gamma + col) : 0.f;
      b[e] = col < a.cols ? __ldg(a.beta + col) : 0.f;
    }
    norm_s[j * P + c] = make_float4(g[0], g[1], g[2], g[3]);
    norm_s[(4 + j) * P + c] = make_float4(b[0], b[1], b[2], b[3]);
  }
}

// Largest magnitude over the warp, NaN if there is one.
__device__ __forceinline__ float warp_amax(float v) {
  float r;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// FF_FP4_NV rows of 16-bit values without a norm, one warp per row: the row stays in registers as loaded (8 words per 16
// values), its maxima are taken on pairs, and it is unpacked once, for the codes. No barriers and few registers:
// NW pieces of 16 columns per lane, rows of up to 512 * NW columns.
template <int NW>
__host__ __device__ constexpr int row_ctas() {  // CTAs of 256 threads per SM that the registers are held to
  return NW <= 3 ? 4 : NW <= 6 ? 3 : 2;
}
template <class T, bool ALIGNED, bool WHOLE, int NW>
__global__ void __launch_bounds__(kQuantThreads, row_ctas<NW>()) quantize_fp4_rows_kernel(const QuantArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int WARPS = kQuantThreads / 32;
  const int pieces = (a.cols + kFp4Step - 1) / kFp4Step * (kFp4Step / 16);
  pdl_wait();
  pdl_trigger();
  for (int row = static_cast<int>(blockIdx.x) * WARPS + warp; row < a.rows; row += static_cast<int>(gridDim.x) * WARPS) {
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const RowOut o = row_out<false>(a, row);
    Raw<T, ALIGNED> raw[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) load_raw<T, ALIGNED>(xr, (i * 32 + lane) * 16, a.cols, raw[i]);
    float amax[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      realign<T, ALIGNED, WHOLE>(xr, (i * 32 + lane) * 16, a.cols, raw[i]);
      amax[i] = amax_pairs<T>(raw[i].t);
    }
    float m = amax[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) m = max_nan(m, amax[i]);
    m = warp_amax(m);
    const bool bad = not_finite(m);
    const float s = nv_row_scale(bad ? 0.f : m);
    if (lane == 0) a.row_scale[row] = bad ? __uint_as_float(0x7fffffffu) : s;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      float2 v[8];
      to_f32<T, ALIGNED>(raw[i], v);
      uint2 codes;
      const uint32_t byte = nv_piece<kExact16>(v, amax[i], s, bad, &codes);
      store_piece<false>(o, i * 32 + lane, pieces, codes, byte);
    }
  }
}

// FF_FP4_MX without a norm: blocks stand alone, so a warp takes 32 * NW pieces of a row at a time, of rows of any width.
template <class T>
__host__ __device__ constexpr int mx_ctas() {
  return sizeof(T) == 4 ? 4 : 5;
}
template <class T>
__host__ __device__ constexpr int mx_pieces() {
  return sizeof(T) == 4 ? 1 : 2;
}
template <class T, bool ALIGNED, bool WHOLE>
__global__ void __launch_bounds__(kQuantThreads, mx_ctas<T>()) quantize_fp4_mx_kernel(const QuantArgs a) {
  constexpr int NW = mx_pieces<T>();
  constexpr int WARPS = kQuantThreads / 32;
  const int lane = threadIdx.x & 31;
  const int pieces = (a.cols + kFp4Step - 1) / kFp4Step * (kFp4Step / 16);
  const int c0 = static_cast<int>(blockIdx.x) * 32 * NW + lane;
  pdl_wait();
  pdl_trigger();
  for (int row = static_cast<int>(blockIdx.y) * WARPS + (threadIdx.x >> 5); row < a.rows; row += static_cast<int>(gridDim.y) * WARPS) {
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const RowOut o = row_out<true>(a, row);
    Raw<T, ALIGNED> raw[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) load_raw<T, ALIGNED>(xr, (c0 + 32 * i) * 16, a.cols, raw[i]);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      realign<T, ALIGNED, WHOLE>(xr, (c0 + 32 * i) * 16, a.cols, raw[i]);
      float2 v[8];
      to_f32<T, ALIGNED>(raw[i], v);
      float amax;
      if constexpr (sizeof(T) == 2)
        amax = amax_pairs<T>(raw[i].t);
      else
        amax = amax16(v);
      uint2 codes;
      const uint32_t byte = mx_piece(v, max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1)), &codes);
      store_piece<true>(o, c0 + 32 * i, pieces, codes, byte);
    }
  }
}

// wpr warps per row (WPR where it is not 0: then the compiler knows all offsets), NC pieces of 16 columns per lane:
// rows of up to 512 * wpr * NC columns.
template <class T, bool MX, bool NORM, bool ALIGNED, bool WHOLE, int NC, int WPR>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 4 ? 2 : NC == 2 ? 4 : 3) quantize_fp4_kernel(const QuantArgs a, const int wpr_any) {
  const int wpr = WPR > 0 ? WPR : wpr_any;
  const int P = 32 * NC * wpr;  // pieces that the lanes of a row hold
  extern __shared__ float4 norm_s[];  // gamma, then beta
  __shared__ float red[2][3][kQuantThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rpc = static_cast<int>(blockDim.x >> 5) / wpr;  // rows per CTA
  const int grp = warp / wpr, wr = warp - grp * wpr;
  const int pieces = (a.cols + kFp4Step - 1) / kFp4Step * (kFp4Step / 16);
  int parity = 0;
  auto row_all = [&](float v, int slot, auto op) {  // over the warps of the row, after a warp reduction
    if (wpr > 1) {
      if (lane == 0) red[parity][slot][warp] = v;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "r"(32 * wpr) : "memory");
      v = red[parity][slot][grp * wpr];
      for (int i = 1; i < wpr; ++i) v = op(v, red[parity][slot][grp * wpr + i]);
    }
    return v;
  };
  auto plus = [](float p, float q) { return p + q; };
  pdl_wait();
  pdl_trigger();
  if constexpr (NORM) {
    fill_norm(norm_s, a, P);
    __syncthreads();
  }
  const float inv_n = 1.f / static_cast<float>(a.cols);
  const int step = static_cast<int>(gridDim.x) * rpc;
  int row = static_cast<int>(blockIdx.x) * rpc + grp;
  for (; row < a.rows; row += step, parity ^= 1) {
    const RowOut o = row_out<MX>(a, row);
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    Raw<T, ALIGNED> raw[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) load_raw<T, ALIGNED>(xr, ((i * wpr + wr) * 32 + lane) * 16, a.cols, raw[i]);
    float2 v[NC][8];
    float amax[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      realign<T, ALIGNED, WHOLE>(xr, ((i * wpr + wr) * 32 + lane) * 16, a.cols, raw[i]);
      to_f32<T, ALIGNED>(raw[i], v[i]);
    }
    if constexpr (NORM) {
      float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s2 = add2(s2, v[i][e]);
      const float mean = row_all(warp_sum(s2.x + s2.y), 0, plus) * inv_n;
      float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        // columns past the row's end stay out of the variance
        const int left = a.cols - ((i * wpr + wr) * 32 + lane) * 16;
        const float m = left > 0 ? -mean : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = add2(v[i][e], make_float2(m, m));
        if (!WHOLE && left > 0 && left < 16) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (2 * e >= left) v[i][e].x = 0.f;
            if (2 * e + 1 >= left) v[i][e].y = 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) q2 = fma2(v[i][e], v[i][e], q2);
      }
      const float rstd = rsqrtf(row_all(warp_sum(q2.x + q2.y), 1, plus) * inv_n + a.eps);
      const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const float4* const ns = norm_s + (i * wpr + wr) * 32 + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 g = ns[j * P], b = ns[(4 + j) * P];
          v[i][2 * j] = fma2(v[i][2 * j], mul2(r2, make_float2(g.x, g.y)), make_float2(b.x, b.y));
          v[i][2 * j + 1] = fma2(v[i][2 * j + 1], mul2(r2, make_float2(g.z, g.w)), make_float2(b.z, b.w));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) amax[i] = amax16(v[i]);
    float s = 1.f;
    bool bad = false;
    if constexpr (!MX) {
      float m = amax[0];
#pragma unroll
      for (int i = 1; i < NC; ++i) m = max_nan(m, amax[i]);
      m = row_all(warp_amax(m), 2, [](float p, float q) { return max_nan(p, q); });
      bad = not_finite(m);
      s = nv_row_scale(bad ? 0.f : m);
      if (lane == 0 && wr == 0) a.row_scale[row] = bad ? __uint_as_float(0x7fffffffu) : s;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * wpr + wr) * 32 + lane;
      uint2 codes;
      uint32_t byte;
      if constexpr (MX)
        byte = mx_piece(v[i], max_nan(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], 1)), &codes);
      else
        byte = nv_piece<quotient_kind<T, NORM>()>(v[i], amax[i], s, bad, &codes);
      store_piece<MX>(o, c, pieces, codes, byte);
    }
  }
}

// Rows too wide for registers: one CTA per row, the row read again for each step (mean, variance, maximum,
// codes); the later reads hit L2.
template <class T, bool MX, bool NORM>
__global__ void __launch_bounds__(kQuantThreads) quantize_fp4_wide_kernel(const QuantArgs a) {
  __shared__ float red[kQuantThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x;
  const RowOut o = row_out<MX>(a, row);
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  auto cta_all = [&](float v, auto op) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < kQuantThreads / 32; ++i) v = op(v, red[i]);
    return v;
  };
  auto plus = [](float p, float q) { return p + q; };
  pdl_wait();
  pdl_trigger();
  const int pieces = (a.cols + kFp4Step - 1) / kFp4Step * (kFp4Step / 16);
  float mean = 0.f, rstd = 1.f;
  float2 v[8];
  if constexpr (NORM) {
    float s = 0.f;
    for (int c = threadIdx.x; c * 16 < a.cols; c += kQuantThreads) {
      load16<T>(xr, c * 16, a.cols, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e].x + v[e].y;
    }
    mean = cta_all(s, plus) / static_cast<float>(a.cols);
    float q = 0.f;
    for (int c = threadIdx.x; c * 16 < a.cols; c += kQuantThreads) {
      load16<T>(xr, c * 16, a.cols, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d0 = c * 16 + 2 * e < a.cols ? v[e].x - mean : 0.f, d1 = c * 16 + 2 * e + 1 < a.cols ? v[e].y - mean : 0.f;
        q = fmaf(d0, d0, fmaf(d1, d1, q));
      }
    }
    rstd = rsqrtf(cta_all(q, plus) / static_cast<float>(a.cols) + a.eps);
  }
  float s = 1.f;
  bool bad = false;
  if constexpr (!MX) {
    float m = 0.f;
    for (int c = threadIdx.x; c * 16 < a.cols; c += kQuantThreads) {
      load16<T>(xr, c * 16, a.cols, v);
      if constexpr (NORM) affine16(v, mean, rstd, a, c * 16);
      m = max_nan(m, amax16(v));
    }
    m = cta_all(m, [](float p, float q) { return max_nan(p, q); });
    bad = not_finite(m);
    s = nv_row_scale(bad ? 0.f : m);
    if (threadIdx.x == 0) a.row_scale[row] = bad ? __uint_as_float(0x7fffffffu) : s;
  }
  for (int c0 = warp * 32; c0 < pieces; c0 += kQuantThreads) {  // whole warps: the stores join lanes' bytes
    const int c = c0 + lane;
    load16<T>(xr, c * 16, a.cols, v);
    if constexpr (NORM) affine16(v, mean, rstd, a, c * 16);
    uint2 codes;
    uint32_t byte;
    if constexpr (MX) {
      float m = amax16(v);
      m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
      byte = mx_piece(v, m, &codes);
    } else {
      byte = nv_piece<quotient_kind<T, NORM>()>(v, amax16(v), s, bad, &codes);
    }
    store_piece<MX>(o, c, pieces, codes, byte);
  }
}

// A CTA per segment of the rows (x) and, up to what the GPU holds, group of rows (y).
dim3 segment_grid(int segs, int groups, int per_sm) {
  const int most = std::max(per_sm * sm_count() / segs, 1);
  return dim3(segs, std::min(groups, most));
}

template <class T, bool ALIGNED, bool WHOLE, int NW>
int launch_rows(const QuantArgs& a, cudaStream_t stream) {
  const int want = (a.rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32), full = row_ctas<NW>() * sm_count();
  launch(quantize_fp4_rows_kernel<T, ALIGNED, WHOLE, NW>, dim3(want < full ? want : full), dim3(kQuantThreads), 0, stream, a);
  return check_launch("quantize_fp4_rows_kernel");
}

template <class T, bool ALIGNED, bool WHOLE>
int launch_mx(const QuantArgs& a, int cols, cudaStream_t stream) {
  constexpr int span = 512 * mx_pieces<T>();
  const dim3 grid = segment_grid((cols + span - 1) / span, (a.rows - 1) / (kQuantThreads / 32) + 1, mx_ctas<T>());
  launch(quantize_fp4_mx_kernel<T, ALIGNED, WHOLE>, grid, dim3(kQuantThreads), 0, stream, a);
  return check_launch("quantize_fp4_mx_kernel");
}

template <class T, bool MX, bool NORM, bool ALIGNED, bool WHOLE, int NC, int WPR>
int launch_joined(const QuantArgs& a, int wpr, cudaStream_t stream) {
  constexpr int WARPS = kQuantThreads / 32;
  if (wpr > WARPS) {
    launch(quantize_fp4_wide_kernel<T, MX, NORM>, dim3(a.rows), dim3(kQuantThreads), 0, stream, a);
    return check_launch("quantize_fp4_wide_kernel");
  }
  const int rpc = WARPS / wpr, threads = 32 * wpr * rpc;
  auto kernel = quantize_fp4_kernel<T, MX, NORM, ALIGNED, WHOLE, NC, WPR>;
  const size_t smem = NORM ? static_cast<size_t>(512) * NC * wpr * 8 : 0;
  static int per_sm[64][WARPS] = {};  // resident CTAs per device and wpr, 0 = not configured yet
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  int most = known ? per_sm[dev][wpr - 1] : 0;
  if (most == 0) {
    constexpr int widest = 512 * NC * WARPS * 8;  // gamma and beta of the widest rows
    if ((NORM && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, widest) != cudaSuccess) ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kernel, threads, smem) != cudaSuccess || most < 1)
      return check_launch("quantize_fp4: configuration");
    if (known) per_sm[dev][wpr - 1] = most;
  }
  const int want = (a.rows + rpc - 1) / rpc, full = most * sm_count();
  launch(kernel, dim3(want < full ? want : full), dim3(threads), smem, stream, a, wpr);
  return check_launch("quantize_fp4_kernel");
}

template <class T, bool MX, bool NORM, bool ALIGNED, bool WHOLE>
int dispatch_quant(const QuantArgs& a, cudaStream_t stream) {
  const int cols = (a.cols + kFp4Step - 1) / kFp4Step * kFp4Step;  // the padded scales are written too
  if constexpr (MX && !NORM) return launch_mx<T, ALIGNED, WHOLE>(a, cols, stream);
  if constexpr (sizeof(T) == 2 && !MX && !NORM) {
    // The fewest pieces of 1, 2, 3, 4, 6, 8 and 10 per lane that hold the row: a piece too many is work for nothing (65600 x 512
    // 18.2 us with one piece, 20.4 with two; 1600 43.4 with four, 52.4 with six; 4096 103.8 with eight, 104.6 with ten; no gain
    // from five: 2560 66.1, 65.9 with six).
    const int nw = (cols + 511) / 512;
    if (nw <= 1) return launch_rows<T, ALIGNED, WHOLE, 1>(a, stream);
    if (nw <= 2) return launch_rows<T, ALIGNED, WHOLE, 2>(a, stream);
    if (nw <= 3) return launch_rows<T, ALIGNED, WHOLE, 3>(a, stream);
    if (nw <= 4) return launch_rows<T, ALIGNED, WHOLE, 4>(a, stream);
    if (nw <= 6) return launch_rows<T, ALIGNED, WHOLE, 6>(a, stream);
    if (nw <= 8) return launch_rows<T, ALIGNED, WHOLE, 8>(a, stream);
    if (nw <= 10) return launch_rows<T, ALIGNED, WHOLE, 10>(a, stream);
  }
  if constexpr (!MX || NORM) {
    const int wpr2 = (cols + 1023) / 1024, wpr3 = (cols + 1535) / 1536;
    // two or three pieces per lane, whichever leaves fewer lanes idle; three where that is even (fewer warps to join) and
    // where two need more warps than a CTA has (8000 x 9500 fp16 behind a LayerNorm 108 us, 618 as a row too wide for
    // registers; f32 without one 72 and 111)
    const bool three = 3 * wpr3 <= 2 * wpr2 || wpr2 > kQuantThreads / 32;
    const int wpr = three ? wpr3 : wpr2;
    if constexpr (sizeof(T) == 2 && NORM) {
      if (wpr == 1)
        return three ? launch_joined<T, MX, NORM, ALIGNED, WHOLE, 3, 1>(a, wpr, stream)
                     : launch_joined<T, MX, NORM, ALIGNED, WHOLE, 2, 1>(a, wpr, stream);
      if (wpr == 2)
        return three ? launch_joined<T, MX, NORM, ALIGNED, WHOLE, 3, 2>(a, wpr, stream)
                     : launch_joined<T, MX, NORM, ALIGNED, WHOLE, 2, 2>(a, wpr, stream);
    }
    return three ? launch_joined<T, MX, NORM, ALIGNED, WHOLE, 3, 0>(a, wpr, stream)
                 : launch_joined<T, MX, NORM, ALIGNED, WHOLE, 2, 0>(a, wpr, stream);
  }
}

template <class T, bool MX, bool NORM>
int dispatch_quant_align(const QuantArgs& a, cudaStream_t stream) {
  const bool aligned = aligned16(a.x) && a.ldx * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  // aligned rows of whole 16-column pieces (the usual widths) do without shifts and masks
  return aligned && a.cols % 16 == 0 ? dispatch_quant<T, MX, NORM, true, true>(a, stream)
         : aligned                   ? dispatch_quant<T, MX, NORM, true, false>(a, stream)
                                     : dispatch_quant<T, MX, NORM, false, false>(a, stream);
}

template <class T>
int dispatch_quant_t(const QuantArgs& a, bool mx, cudaStream_t stream) {
  if (a.gamma != nullptr) return mx ? dispatch_quant_align<T, true, true>(a, stream) : dispatch_quant_align<T, false, true>(a, stream);
  return mx ? dispatch_quant_align<T, true, false>(a, stream) : dispatch_quant_align<T, false, false>(a, stream);
}

// ---------------------------------------------------------------- dequantisation
template <class T>
__device__ __forceinline__ void store_one(T* p, float v) {
  if constexpr (sizeof(T) == 4)
    *p = v;
  else if constexpr (std::is_same<T, __half>::value)
    *p = __float2half_rn(v);
  else
    *p = __float2bfloat16_rn(v);
}

template <class T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(Pair16<T>::pack(v[0], v[1]), Pair16<T>::pack(v[2], v[3]), Pair16<T>::pack(v[4], v[5]),
                      Pair16<T>::pack(v[6], v[7]));
}

// A warp takes 256 columns, 8 per lane, of rows r, r + 32, r + 64 and r + 96 of a 128-row scale tile: the scales of four
// blocks of these four rows are 16 neighbouring bytes. All loads of a lane are independent of each other.
// Rows that lie 32 apart are equally far from a 16-byte boundary, whatever the pitch. Rows that do not start on one
// (!ALIGNED) have their lanes' columns moved down to the boundary before: a lane's columns then lie in two words of
// codes and up to two blocks. Stores are whole 16-byte granules; those that stick out of the row are written by value.
template <class T, bool MX, bool ALIGNED>
__global__ void __launch_bounds__(256)
    dequantize_fp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                          const float* __restrict__ row_scale, int rows, int cols, T* __restrict__ out, int64_t ldo) {
  constexpr int B = MX ? 32 : 16;
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x, seg = static_cast<int>(blockIdx.x * blockDim.y + threadIdx.y);
  pdl_wait();
  pdl_trigger();
  const int64_t pitch = fp4_row_bytes(cols), tile = sf_tile_bytes(cols, MX);
  const int quads = (rows + 127) / 128 * 32;
  for (int quad = static_cast<int>(blockIdx.y * blockDim.z + threadIdx.z); quad < quads; quad += static_cast<int>(gridDim.y * blockDim.z)) {
    const int row0 = (quad >> 5) * 128 + (quad & 31);
    const int off = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(out + row0 * ldo) & 15) / static_cast<int>(sizeof(T));
    const int c = (seg * 32 + lane) * 8 - off;  // the lane's first column, may be negative
    if (row0 >= rows || c >= cols) continue;
    // the (at most two) blocks that the columns touch
    const int blk = ALIGNED ? c / B : max(c, 0) / B, blk1 = ALIGNED ? blk : min(c + 7, cols - 1) / B;
    const uint8_t* const sq = scales + (quad >> 5) * tile + (quad & 31) * 16;
    const uint4 sw = __ldg(reinterpret_cast<const uint4*>(sq + static_cast<int64_t>(blk >> 2) * kSfChunk));
    uint4 sw1 = sw;
    if constexpr (!ALIGNED) sw1 = __ldg(reinterpret_cast<const uint4*>(sq + static_cast<int64_t>(blk1 >> 2) * kSfChunk));
    const uint32_t sb[4] = {sw.x, sw.y, sw.z, sw.w}, sb1[4] = {sw1.x, sw1.y, sw1.z, sw1.w};
    uint32_t w[4], w1[4];
    float rs[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + 32 * j, k = c >> 3;
      const uint32_t* const p = reinterpret_cast<const uint32_t*>(codes + row * pitch) + k;
      w[j] = row < rows && (ALIGNED || k >= 0) ? __ldg(p) : 0u;
      w1[j] = !ALIGNED && row < rows && 8 * (k + 1) < cols ? __ldg(p + 1) : 0u;
      rs[j] = !MX && row < rows ? __ldg(row_scale + row) : 1.f;
    }
    const int cut = ALIGNED ? 8 : (blk + 1) * B - c;  // columns of the first block
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + 32 * j;
      if (row >= rows) break;
      auto scale = [&](uint32_t bytes, int b) {
        const uint32_t byte = (bytes >> (8 * (b & 3))) & 0xffu;
        return MX ? e8m0_value(byte) : e4m3_value(byte) * rs[j];
      };
      const float sc = scale(sb[j], blk), sc1 = ALIGNED ? sc : scale(sb1[j], blk1);
      uint32_t h[4];
      e2m1x8_to_half2(ALIGNED ? w[j] : __funnelshift_r(w[j], w1[j], 4 * (c & 7)), h);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 f = mul2(unpack_half2(h[e / 2]), make_float2(e < cut ? sc : sc1, e + 1 < cut ? sc : sc1));
        v[e] = f.x;
        v[e + 1] = f.y;
      }
      T* const o = out + row * ldo + c;
      const bool whole = (ALIGNED || c >= 0) && c + 8 <= cols;
      const bool wide = sizeof(T) == 4 && (reinterpret_cast<uintptr_t>(o) & 31) == 0;
#pragma unroll
      for (int g = 0; g < 8; g += E) {
        if (whole || ((ALIGNED || c + g >= 0) && c + g + E <= cols)) {
          if (sizeof(T) == 4 && whole && wide) {  // one store of 32 bytes: two of 16 would each write half sectors
            if (g == 0)
              asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                           "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                           : "memory");
          } else {
            __stcs(reinterpret_cast<uint4*>(o + g), pack16<T>(v + g));
          }
        } else {
#pragma unroll
          for (int e = g; e < g + E; ++e)
            if ((ALIGNED || c + e >= 0) && c + e < cols) store_one(o + e, v[e]);
        }
      }
    }
  }
}

template <class T, bool MX>
int launch_dequant(const uint8_t* codes, const uint8_t* scales, const float* rs, int rows, int cols, void* out, int64_t ldo,
                   cudaStream_t stream) {
  T* const o = static_cast<T*>(out);
  const bool aligned = aligned16(out) && (rows == 1 || ldo * static_cast<int64_t>(sizeof(T)) % 16 == 0);
  const int segs = (cols + (aligned ? 0 : 16 / static_cast<int>(sizeof(T)) - 1) + 255) / 256;
  // Warps of a CTA side by side in a row where they divide its segments (32000 x 4096 f32 146 us, 158 below one another;
  // 65600 x 2730, 11 segments, 104 us below one another, 117 with 12 warps for them).
  int wx = 8;
  while (segs % wx != 0) --wx;
  const int wy = 8 / wx;
  const dim3 block(32, wx, wy), grid = segment_grid(segs / wx, ((rows + 127) / 128 * 32 + wy - 1) / wy, 64 / (wx * wy));
  if (aligned)
    launch(dequantize_fp4_kernel<T, MX, true>, grid, block, 0, stream, codes, scales, rs, rows, cols, o, ldo);
  else
    launch(dequantize_fp4_kernel<T, MX, false>, grid, block, 0, stream, codes, scales, rs, rows, cols, o, ldo);
  return check_launch("dequantize_fp4_kernel");
}

}  // namespace

int quantize_fp4(const void* x, int dtype, int64_t ldx, const float* gamma, const float* beta, float eps, int rows,
                 int cols, int fmt, uint8_t* codes, uint8_t* scales, float* row_scale, cudaStream_t stream) {
  FF_REQUIRE(fmt == FF_FP4_NV || fmt == FF_FP4_MX, "ff_quantize_fp4: unknown format %d", fmt);
  FF_REQUIRE(dtype == FF_F16 || dtype == FF_BF16 || dtype == FF_F32, "ff_quantize_fp4: unknown type %d", dtype);
  FF_REQUIRE(rows >= 0 && rows <= (1 << 30) && cols >= 1 && cols <= (1 << 24) && ldx >= cols, "ff_quantize_fp4: bad shape [%d, %d], row stride %lld", rows,
             cols, static_cast<long long>(ldx));
  if (rows == 0) return FF_OK;
  FF_REQUIRE(x && codes && scales, "ff_quantize_fp4: NULL pointer");
  FF_REQUIRE(fmt == FF_FP4_MX || row_scale, "ff_quantize_fp4: FF_FP4_NV needs row_scale");
  FF_REQUIRE((gamma == nullptr) == (beta == nullptr), "ff_quantize_fp4: give both gamma and beta or neither");
  FF_REQUIRE(reinterpret_cast<uintptr_t>(x) % (dtype == FF_F32 ? 4 : 2) == 0, "ff_quantize_fp4: x is not aligned to its type");
  FF_REQUIRE(aligned16(codes) && aligned16(scales), "ff_quantize_fp4: codes and scales must be 16-byte aligned");
  const QuantArgs a{x, ldx, gamma, beta, eps, rows, cols, codes, scales, row_scale};
  const bool mx = fmt == FF_FP4_MX;
  switch (dtype) {
    case FF_F16: return dispatch_quant_t<__half>(a, mx, stream);
    case FF_BF16: return dispatch_quant_t<__nv_bfloat16>(a, mx, stream);
    default: return dispatch_quant_t<float>(a, mx, stream);
  }
}

}  // namespace ff

using namespace ff;

extern "C" int64_t ff_fp4_code_bytes(int rows, int cols) {
  return rows < 0 || cols < 1 ? 0 : static_cast<int64_t>(rows) * fp4_row_bytes(cols);
}

extern "C" int64_t ff_fp4_scale_bytes(int rows, int cols, int fmt) {
  if (rows < 0 || cols < 1 || (fmt != FF_FP4_NV && fmt != FF_FP4_MX)) return 0;
  return static_cast<int64_t>((rows + 127) / 128) * sf_tile_bytes(cols, fmt == FF_FP4_MX);
}

extern "C" int ff_quantize_fp4(const void* x, int dtype, int64_t ldx, const float* gamma, const float* beta, float eps,
                               int rows, int cols, int fmt, uint8_t* codes, uint8_t* scales, float* row_scale,
                               void* stream) {
  return quantize_fp4(x, dtype, ldx, gamma, beta, eps, rows, cols, fmt, codes, scales, row_scale,
                      static_cast<cudaStream_t>(stream));
}

extern "C" int ff_dequantize_fp4(const uint8_t* codes, const uint8_t* scales, const float* row_scale, int rows, int cols,
                                 int fmt, void* out, int dtype, int64_t ldo, void* stream) {
  FF_REQUIRE(fmt == FF_FP4_NV || fmt == FF_FP4_MX, "ff_dequantize_fp4: unknown format %d", fmt);
  FF_REQUIRE(dtype == FF_F16 || dtype == FF_BF16 || dtype == FF_F32, "ff_dequantize_fp4: unknown type %d", dtype);
  FF_REQUIRE(rows >= 0 && rows <= (1 << 30) && cols >= 1 && cols <= (1 << 24) && ldo >= cols, "ff_dequantize_fp4: bad shape [%d, %d], row stride %lld", rows,
             cols, static_cast<long long>(ldo));
  if (rows == 0) return FF_OK;
  FF_REQUIRE(codes && scales && out, "ff_dequantize_fp4: NULL pointer");
  FF_REQUIRE(fmt == FF_FP4_MX || row_scale, "ff_dequantize_fp4: FF_FP4_NV needs row_scale");
  FF_REQUIRE(reinterpret_cast<uintptr_t>(out) % (dtype == FF_F32 ? 4 : 2) == 0, "ff_dequantize_fp4: out is not aligned to its type");
  FF_REQUIRE(aligned16(codes) && aligned16(scales), "ff_dequantize_fp4: codes and scales must be 16-byte aligned");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool mx = fmt == FF_FP4_MX;
  switch (dtype) {
    case FF_F16:
      return mx ? launch_dequant<__half, true>(codes, scales, row_scale, rows, cols, out, ldo, st)
                : launch_dequant<__half, false>(codes, scales, row_scale, rows, cols, out, ldo, st);
    case FF_BF16:
      return mx ? launch_dequant<__nv_bfloat16, true>(codes, scales, row_scale, rows, cols, out, ldo, st)
                : launch_dequant<__nv_bfloat16, false>(codes, scales, row_scale, rows, cols, out, ldo, st);
    default:
      return mx ? launch_dequant<float, true>(codes, scales, row_scale, rows, cols, out, ldo, st)
                : launch_dequant<float, false>(codes, scales, row_scale, rows, cols, out, ldo, st);
  }
}
