// The end of a block and the norm before the next one, in one pass over the rows:
//   out    = alpha x + scale * act(gate) * post(y)
//   normed = pre(out), from the 32-bit values of out before they are rounded
// post and pre: nothing, RMS (v / sqrt(mean(v^2) + eps) * w + b) or LAYER ((v - mean) / sqrt(var + eps) * w + b, the variance
// from centred values).
//
// Bound by HBM: x and y are read and out and normed written once. A row stays in the registers of its threads: a warp takes
// rows of up to 1024 columns (32 values per lane), wider rows are shared by more warps, whose sums meet in shared memory.
// All sums, statistics and products are f32; each output is rounded once.
//
// Measured: 65600 x 1024 bf16, two RMS norms, gate per image and scale (537 MB) 106 us, 5.1 TB/s, and without gate and scale 87 us,
// 6.2 TB/s (at 1965 MHz; 92 at 1755, under the power limit), with two LayerNorms 122 us; 16400 x 2730 bf16, gate per element
// 78 us, 4.6 TB/s (2736 columns: 62 us, 5.8 TB/s); 8200 x 768 f32 with a bf16 branch, two LayerNorms and a scale 17.7 us,
// 4.3 TB/s; one row of 1024 3.3 us with its call. What is short of HBM's rate waits:
// a row's sums need all of it, and its registers are not free for the next before. (Sums of warps merged around their own
// means, one barrier less: 121 -> 130 us with two LayerNorms, for the instructions more. Persistent CTAs with the
// parameters in registers: 160.)
//
// Four ways to deal out the columns. FULL: 16-byte chunks (8 columns of 16 bits) that divide the rows of every matrix. SHIFTED:
// the same, where a row is equally far off 16 bytes in every matrix: its chunks begin before it, and the first and last are
// dealt with by 4-byte words. PAIRS: neighbouring pairs of columns to neighbouring lanes, where all rows and the width are
// whole pairs; parameters then come in whole 8-byte words, and a warp's pairs still fill cache lines. SINGLES: columns one by
// one, for any alignment and width.
#include <algorithm>

#include "common.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kChunk = 8;
constexpr int kNrThreads = 128;    // of a CTA whose warps take rows of their own
constexpr int kNrMaxCols = 16384;  // 16 warps x 32 lanes x 4 chunks of 8

enum class Deal { kFull, kShifted, kPairs, kSingles };

struct NrArgs {
  ff_norm_residual_args p;
  int lanes;  // per row: 4, 8, 16 or 32, or 32 times the row's warps
};

// Conversions of 8 values between memory and f32 pairs.
template <class T>
struct Raw {
  uint4 w[sizeof(T) == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& u = w[i >> 2];
    return (i & 3) == 0 ? u.x : (i & 3) == 1 ? u.y : (i & 3) == 2 ? u.z : u.w;
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
    else
      return Pair16<T>::unpack(word(i));
  }
  __device__ __forceinline__ void set_word(int i, uint32_t x) {
    uint4& u = w[i >> 2];
    ((i & 3) == 0 ? u.x : (i & 3) == 1 ? u.y : (i & 3) == 2 ? u.z : u.w) = x;
  }
  __device__ __forceinline__ void set(const float2 (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
      w[0] = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
      w[sizeof(w) / 16 - 1] = make_uint4(__float_as_uint(v[2].x), __float_as_uint(v[2].y), __float_as_uint(v[3].x), __float_as_uint(v[3].y));
    } else {
      w[0] = make_uint4(Pair16<T>::pack(v[0].x, v[0].y), Pair16<T>::pack(v[1].x, v[1].y), Pair16<T>::pack(v[2].x, v[2].y),
                        Pair16<T>::pack(v[3].x, v[3].y));
    }
  }
};

__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_f32(float v) { return v; }

// The columns of one thread: chunk k, value e of its eight.
template <Deal D>
struct Columns {
  static constexpr int kUnit = D == Deal::kFull || D == Deal::kShifted ? kChunk : D == Deal::kPairs ? 2 : 1;  // neighbouring columns of a lane
  int cols, first, step;  // of unit 0, and between units
  Columns() = default;
  __device__ __forceinline__ Columns(int cols, int lane, int lanes) : cols(cols), first(lane * kUnit), step(lanes * kUnit) {}
  __device__ __forceinline__ int at(int k, int e) const { return first + (k * kChunk + e) / kUnit * step + e % kUnit; }

  __device__ __forceinline__ bool within(int k, int e) const {
    return D == Deal::kShifted ? static_cast<uint32_t>(at(k, e)) < static_cast<uint32_t>(cols) : at(k, e) < cols;
  }
  __device__ __forceinline__ bool whole(int k) const { return at(k, 0) >= 0 && at(k, kChunk - 1) < cols; }

  template <class T>
  __device__ __forceinline__ void load(const T* row, int k, Raw<T>& r) const {
    if constexpr (D == Deal::kFull) {
      r.clear();
      if (at(k, 0) < cols) r.load(row + at(k, 0));
    } else if constexpr (D == Deal::kShifted) {
      if (whole(k)) {
        r.load(row + at(k, 0));
      } else {
#pragma unroll
        for (int e = 0; e < kChunk; e += 2) r.set_word(e / 2, within(k, e) ? *reinterpret_cast<const uint32_t*>(row + at(k, e)) : 0u);
      }
    } else if constexpr (D == Deal::kPairs) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool there = at(k, 2 * e) < cols;
        if constexpr (sizeof(T) == 4) {
          const uint2 w = there ? *reinterpret_cast<const uint2*>(row + at(k, 2 * e)) : make_uint2(0, 0);
          r.set_word(2 * e, w.x);
          r.set_word(2 * e + 1, w.y);
        } else {
          r.set_word(e, there ? *reinterpret_cast<const uint32_t*>(row + at(k, 2 * e)) : 0u);
        }
      }
    } else {
      using B = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
      const B* const p = reinterpret_cast<const B*>(row);
      B w[kChunk];
#pragma unroll
      for (int e = 0; e < kChunk; ++e) w[e] = at(k, e) < cols ? p[at(k, e)] : B(0);
#pragma unroll
      for (int i = 0; i < (sizeof(T) == 4 ? 8 : 4); ++i)
        r.set_word(i, sizeof(T) == 4 ? w[i] : w[2 * i & 7] | static_cast<uint32_t>(w[(2 * i + 1) & 7]) << 16);
    }
  }
  template <class T>
  __device__ __forceinline__ void store(T* row, int k, const float2 (&v)[4]) const {
    Raw<T> r;
    r.set(v);
    if constexpr (D == Deal::kFull) {
      if (at(k, 0) < cols) r.store(row + at(k, 0));
    } else if constexpr (D == Deal::kShifted) {
      if (whole(k)) {
        r.store(row + at(k, 0));
      } else {
#pragma unroll
        for (int e = 0; e < kChunk; e += 2)
          if (within(k, e)) *reinterpret_cast<uint32_t*>(row + at(k, e)) = r.word(e / 2);
      }
    } else if constexpr (D == Deal::kPairs) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at(k, 2 * e) < cols) {
          if constexpr (sizeof(T) == 4)
            *reinterpret_cast<uint2*>(row + at(k, 2 * e)) = make_uint2(r.word(2 * e), r.word(2 * e + 1));
          else
            *reinterpret_cast<uint32_t*>(row + at(k, 2 * e)) = r.word(e);
        }
    } else {
      using B = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
      B* const p = reinterpret_cast<B*>(row);
#pragma unroll
      for (int e = 0; e < kChunk; ++e)
        if (at(k, e) < cols) p[at(k, e)] = static_cast<B>(sizeof(T) == 4 ? r.word(e) : r.word(e / 2) >> (16 * (e & 1)));
    }
  }
  // f32 parameters of chunk k's columns (0 where there is none).
  __device__ __forceinline__ void parameters(const float* p, int k, float2 (&v)[4]) const {
    if constexpr (D == Deal::kFull) {
      const bool there = at(k, 0) < cols;
      const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 a = there ? __ldg(reinterpret_cast<const float4*>(p + at(k, 0))) : z, b = there ? __ldg(reinterpret_cast<const float4*>(p + at(k, 0)) + 1) : z;
      v[0] = make_float2(a.x, a.y);
      v[1] = make_float2(a.z, a.w);
      v[2] = make_float2(b.x, b.y);
      v[3] = make_float2(b.z, b.w);
    } else if constexpr (D == Deal::kShifted) {
      if (whole(k) && reinterpret_cast<uintptr_t>(p + at(k, 0)) % 8 == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __ldg(reinterpret_cast<const float2*>(p + at(k, 2 * e)));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = make_float2(within(k, 2 * e) ? __ldg(p + at(k, 2 * e)) : 0.f, within(k, 2 * e + 1) ? __ldg(p + at(k, 2 * e + 1)) : 0.f);
      }
    } else {
      Raw<float> r;
      load(p, k, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = r.pair(e);
    }
  }
  // Values outside the row to 0.
  template <int K>
  __device__ __forceinline__ void trim(float2 (&v)[K][4]) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!within(k, 2 * e)) v[k][e].x = 0.f;
        if (!within(k, 2 * e + 1)) v[k][e].y = 0.f;
      }
  }
};

// Sums over the threads of a row, of R rows. Sums of several warps go through `part` (32 R words per call).
template <bool MULTI, int R>
__device__ __forceinline__ void row_sums(float (&v)[R], int lanes, float (*part)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if constexpr (MULTI) {
      v[r] = warp_sum(v[r]);
      if (lane == 0) part[r][warp] = v[r];
    } else {
#pragma unroll
      for (int o = 16; o; o >>= 1)
        if (o < lanes) v[r] += __shfl_xor_sync(0xffffffffu, v[r], o);
    }
  }
  if constexpr (MULTI) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = warp_sum(lane * 32 < lanes ? part[r][lane] : 0.f);
  }
}

// v (0 past the row) -> its norm, in place, for R rows.
template <Deal D, int R, int K, bool MULTI>
__device__ __forceinline__ void norm(float2 (&v)[R][K][4], const Columns<D> (&c)[R], int kind, const float* w, const float* b, float eps, int lanes,
                                     float (*part)[32]) {
  const float inv = 1.f / static_cast<float>(c[0].cols);
  float sum[R];
  if (kind == FF_NORM_LAYER) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e & 1] = add2(s[e & 1], v[r][k][e]);
      s[0] = add2(s[0], s[1]);
      sum[r] = s[0].x + s[0].y;
    }
    row_sums<MULTI>(sum, lanes, part);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mean = sum[r] * inv;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][k][e] = sub2(v[r][k][e], make_float2(mean, mean));
      c[r].trim(v[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float2 q[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e & 1] = fma2(v[r][k][e], v[r][k][e], q[e & 1]);
    q[0] = add2(q[0], q[1]);
    sum[r] = q[0].x + q[0].y;
  }
  row_sums<MULTI>(sum, lanes, part + R);
  float2 r2[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float rstd = rsqrtf(sum[r] * inv + eps);
    r2[r] = make_float2(rstd, rstd);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float2 wk[4];
    if (w != nullptr) {
      c[0].parameters(w, k, wk);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][k][e] = mul2(v[r][k][e], mul2(wk[e], r2[r]));
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][k][e] = mul2(v[r][k][e], r2[r]);
    }
    if (b != nullptr) {
      c[0].parameters(b, k, wk);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][k][e] = add2(v[r][k][e], wk[e]);
    }
  }
}

// e^x within a few 2^-24 of itself: 2^t of the rounded t = x log2(e), corrected by what the product and the constant lost.
__device__ __forceinline__ float exp_close(float x) {
  constexpr float kLog2e = 1.44269504f, kBelow = static_cast<float>(1.4426950408889634 - static_cast<double>(kLog2e));
  const float t = x * kLog2e;
  const float lost = fmaf(x, kLog2e, -t) + x * kBelow;
  const float y = ex2_approx(t);
  return fabsf(t) < 126.f ? fmaf(y, lost * 0.693147181f, y) : y;
}
__device__ __forceinline__ float reciprocal(float v) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
  return y;
}
// 1 / (1 + e^-g), and for tanh 1 - 2 / (1 + e^2|g|), but its series g (1 - g^2 / 3 + 2 g^4 / 15 - 17 g^6 / 315 + 62 g^8 / 2835 -
// 1382 g^10 / 155925) below 0.35 (the next term is 2^-25 of it there). CLOSE (32-bit results): within 2^-20 of the
// value; else, for results that are rounded to 12 bits at most, within 2^-19, but sigmoids of g below -22 within 2^-18 and
// below -44 within 2^-17 (half a unit of t = g log2(e) is that much of 2^t). Below -87.3 a sigmoid is less than f32's
// smallest normal number, and 0 here.
template <bool CLOSE>
__device__ __forceinline__ float activate(float g, int act) {
  auto exponential = [](float x) { return CLOSE ? exp_close(x) : ex2_approx(x * 1.44269504f); };
  if (act == FF_GATE_SIGMOID) return reciprocal(1.f + exponential(-g));
  if (act == FF_GATE_TANH) {
    const float a = fabsf(g), q = g * g;
    float s = fmaf(q, -8.863235530e-3f, 2.186948854e-2f);
    s = fmaf(q, s, -5.396825397e-2f);
    s = fmaf(q, s, 1.333333333e-1f);
    s = fmaf(q, s, -3.333333333e-1f);
    const float far = 1.f - 2.f * reciprocal(1.f + exponential(2.f * a));
    return a < 0.35f ? fmaf(g * q, s, g) : g != g ? g : copysignf(far, g);
  }
  return g;
}

// R rows at a time by the same threads, which then read the parameters once for all of them.
template <class TX, class TY, int R, int K, Deal D, bool MULTI>
__global__ void __launch_bounds__(MULTI ? (R * K == 1 ? 1024 : 512) : kNrThreads, MULTI ? 1 : R * K <= 2 ? 8 : sizeof(TX) == 2 && D == Deal::kFull ? 5 : 4)
    norm_residual_kernel(const __grid_constant__ NrArgs a) {
  __shared__ float part[MULTI ? 4 * R : 1][32];
  const ff_norm_residual_args& p = a.p;
  const int lanes = a.lanes;  // a power of two unless MULTI
  const int in_row = MULTI ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) & (lanes - 1);
  const int group = MULTI ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * (kNrThreads / lanes) + static_cast<int>(threadIdx.x) / lanes;
  pdl_wait();
  pdl_trigger();
  Columns<D> c[R];
  int64_t row[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t n = static_cast<int64_t>(group) * R + r;
    const bool real = (MULTI && R == 1) || n < p.rows;  // lanes without a row go along, on nothing
    row[r] = real ? n : 0;
    c[r] = Columns<D>(p.cols, in_row, lanes);
    if constexpr (D == Deal::kShifted)  // the row's columns before its first whole 16 bytes
      c[r].first -= static_cast<int>(reinterpret_cast<uintptr_t>(static_cast<const TY*>(p.y) + row[r] * p.ldy) % 16 / sizeof(TY));
    if (!real) c[r].first = p.cols;
  }
  Raw<TY> raw[R][K];
  Raw<TX> xr[R][K];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < K; ++k) c[r].load(static_cast<const TY*>(p.y) + row[r] * p.ldy, k, raw[r][k]);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < K; ++k) c[r].load(static_cast<const TX*>(p.x) + row[r] * p.ldx, k, xr[r][k]);
  float2 v[R][K][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[r][k][e] = raw[r][k].pair(e);
  int64_t gate_at[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    gate_at[r] = p.gate != nullptr ? static_cast<int64_t>(static_cast<uint32_t>(row[r]) / static_cast<uint32_t>(p.gate_rows)) * p.ldg : 0;
  const bool narrow = p.gate != nullptr && p.gate_cols > 1 && p.gate_type != FF_F32;  // a gate of 16 bits per column
  if (narrow || (sizeof(TY) == 4 && p.gate != nullptr && p.gate_cols > 1)) {  // under way during the norm
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < K; ++k) c[r].load(static_cast<const TY*>(p.gate) + gate_at[r], k, raw[r][k]);
  }
  if (p.post != FF_NORM_NONE) norm<D, R, K, MULTI>(v, c, p.post, p.post_w, p.post_b, p.post_eps, lanes, part);
  if (p.gate != nullptr) {
    if (p.gate_cols == 1) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float g = activate<true>(
            p.gate_type == FF_F32 ? static_cast<const float*>(p.gate)[gate_at[r]] : as_f32(static_cast<const TY*>(p.gate)[gate_at[r]]), p.gate_act);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[r][k][e] = mul2(v[r][k][e], make_float2(g, g));
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 g[4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (narrow || sizeof(TY) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = raw[r][k].pair(e);
          } else if (r == 0 || gate_at[r] != gate_at[r - 1]) {
            c[r].parameters(static_cast<const float*>(p.gate) + gate_at[r], k, g);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[r][k][e] = mul2(v[r][k][e], g[e]);
            continue;
          }
          if (p.gate_act != FF_GATE_PLAIN) {
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = make_float2(activate<sizeof(TX) == 4>(g[e].x, p.gate_act), activate<sizeof(TX) == 4>(g[e].y, p.gate_act));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[r][k][e] = mul2(v[r][k][e], g[e]);
        }
      }
    }
  }
  if (p.scale != nullptr) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 s[4];
      c[0].parameters(p.scale, k, s);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][k][e] = mul2(v[r][k][e], s[e]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[r][k][e] = fma2(make_float2(p.alpha, p.alpha), xr[r][k].pair(e), v[r][k][e]);
      c[r].store(static_cast<TX*>(p.out) + row[r] * p.ldo, k, v[r][k]);
    }
  if (p.normed == nullptr) return;
#pragma unroll
  for (int r = 0; r < R; ++r) c[r].trim(v[r]);  // statistics, biases, gates and infinities can have left others than 0 there
  norm<D, R, K, MULTI>(v, c, p.pre, p.pre_w, p.pre_b, p.pre_eps, lanes, part + (MULTI ? 2 * R : 0));
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < K; ++k) c[r].store(static_cast<TY*>(p.normed) + row[r] * p.ldn, k, v[r][k]);
}

template <class TX, class TY, int R, int K, Deal D, bool MULTI>
void launch_nr(const NrArgs& a, cudaStream_t s) {
  const int rows = (a.p.rows + R - 1) / R, per = kNrThreads / a.lanes;
  launch(norm_residual_kernel<TX, TY, R, K, D, MULTI>, dim3(MULTI ? rows : (rows + per - 1) / per), dim3(MULTI ? a.lanes : kNrThreads), 0, s, a);
}

template <class TX, class TY, Deal D>
void launch_nr_deal(NrArgs& a, int vectors, int chunks, cudaStream_t s) {
  const int wide = (chunks + 31) / 32;  // warps with a chunk per lane
  const ff_norm_residual_args& p = a.p;
  const int lanes = chunks <= 4 ? 4 : chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32;  // of a row within a warp
  const bool sums = p.post != FF_NORM_NONE || p.normed != nullptr, few = static_cast<int64_t>(p.rows) * wide * lanes <= 512LL * sm_count();
  if constexpr (D != Deal::kShifted) {
    if (wide == 1) {
      a.lanes = lanes;
      if constexpr (sizeof(TX) == 2) {
        if (!few && vectors >= 2) return launch_nr<TX, TY, 2, 1, D, false>(a, s);
      }
      return launch_nr<TX, TY, 1, 1, D, false>(a, s);
    }
  }
  if (wide <= 32 && (few || D == Deal::kSingles)) {
    a.lanes = 32 * wide;
    return launch_nr<TX, TY, 1, 1, D, true>(a, s);
  }
  if constexpr (D != Deal::kSingles) {
    if constexpr (D != Deal::kShifted) {
      if (wide <= 8 && sums && vectors >= 3) {
        a.lanes = 32 * wide;
        return launch_nr<TX, TY, 2, 1, D, true>(a, s);
      }
    }
    if (wide <= 4 && (wide == 2 || !sums)) {
      a.lanes = 32;
      return wide == 2 ? launch_nr<TX, TY, 1, 2, D, false>(a, s) : launch_nr<TX, TY, 1, 4, D, false>(a, s);
    }
    if (wide <= 32) {
      a.lanes = 32 * ((wide + 1) / 2);
      return launch_nr<TX, TY, 1, 2, D, true>(a, s);
    }
  }
  a.lanes = 32 * ((wide + 3) / 4);
  launch_nr<TX, TY, 1, 4, D, true>(a, s);
}

template <class TX, class TY>
void launch_nr_types(NrArgs& a, cudaStream_t s) {
  const ff_norm_residual_args& p = a.p;
  bool full = p.cols % kChunk == 0, pairs = p.cols % 2 == 0;
  auto look = [&](const void* q, int64_t ld, int64_t size, int64_t rows) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(q) | static_cast<uint64_t>(rows > 1 ? ld * size : 0);
    full = full && bits % 16 == 0;
    pairs = pairs && bits % (2 * size) == 0;
  };
  look(p.y, p.ldy, sizeof(TY), p.rows);
  look(p.x, p.ldx, sizeof(TX), p.rows);
  look(p.out, p.ldo, sizeof(TX), p.rows);
  look(p.normed, p.ldn, sizeof(TY), p.rows);
  for (const float* q : {p.post_w, p.post_b, p.pre_w, p.pre_b, p.scale}) look(q, 0, 4, 1);
  if (p.gate != nullptr && p.gate_cols > 1) look(p.gate, p.ldg, p.gate_type == FF_F32 ? 4 : 2, p.rows <= p.gate_rows ? 1 : p.rows);
  // Lanes, chunks and rows per lane. Two chunks of a row (65600 x 1024 bf16 with two RMS norms: 87 us, four chunks of it with gate and
  // scale 146 against 117), or one chunk of two rows where at least three vectors of parameters are then read once for
  // both (with gate and scale 117 -> 105 us; without 89), or two where a warp has all of a row of 16 bits (60000 x 256: 26.5 ->
  // 23.8; f32 24.7 -> 26.6), but not in more than 8 warps (16400 x 2736: 85 -> 102). One chunk of one row where rows are few (less than 16 warps per SM even
  // so), for the shortest way through a row, or columns come one by one (16400 x 2731: 126 us, 151 with two), and four where no
  // sum holds a row together (58 us, 69 with two).
  int vectors = p.scale != nullptr;  // of parameters
  for (const float* q : {p.post_w, p.post_b, p.pre_w, p.pre_b}) vectors += q != nullptr;
  vectors += p.gate != nullptr && p.gate_cols > 1 && p.gate_type == FF_F32 && p.gate_rows > 1;
  const int chunks = (p.cols + kChunk - 1) / kChunk;
  if (full) return launch_nr_deal<TX, TY, Deal::kFull>(a, vectors, chunks, s);
  // SHIFTED: for 16 bits, rows that a warp has not all of, and either one vector of parameters (these are off their 16 bytes; 16400 x
  // 770, gate per element: 32 -> 26 us, but 35 -> 38 at 902 columns with three) or more than 2048 columns (2050 with three:
  // 102 -> 84, 2730 with a gate per element 98 -> 78). f32: 16400 x 1030 57, and 66 so.
  if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2) {
    bool alike = p.cols % 2 == 0;
    auto like_y = [&](const void* q, int64_t ld) {  // every row as far off 16 bytes as y's
      const uint64_t from = reinterpret_cast<uintptr_t>(q), y = reinterpret_cast<uintptr_t>(p.y);
      alike = alike && from % 4 == 0 && from % 16 == y % 16 && (p.rows == 1 || (2 * ld % 4 == 0 && 2 * ld % 16 == 2 * p.ldy % 16));
    };
    like_y(p.y, p.ldy);
    like_y(p.x, p.ldx);
    like_y(p.out, p.ldo);
    if (p.normed != nullptr) like_y(p.normed, p.ldn);
    if (p.gate != nullptr && p.gate_cols > 1 && p.gate_type != FF_F32) {
      alike = alike && (p.gate_rows == 1 || p.rows == 1);
      like_y(p.gate, p.ldg);
    }
    const int shifted = (p.cols + 2 * kChunk - 2) / kChunk;  // the first can begin before the row
    if (alike && shifted <= kNrMaxCols / kChunk && chunks > 32 && (vectors <= 1 || chunks > 256))
      return launch_nr_deal<TX, TY, Deal::kShifted>(a, vectors, shifted, s);
  }
  if (pairs)
    launch_nr_deal<TX, TY, Deal::kPairs>(a, vectors, chunks, s);
  else
    launch_nr_deal<TX, TY, Deal::kSingles>(a, vectors, chunks, s);
}

}  // namespace

}  // namespace ff

using namespace ff;

extern "C" int ff_norm_residual(const ff_norm_residual_args* args, void* stream) {
  FF_REQUIRE(args != nullptr, "ff_norm_residual: NULL arguments");
  NrArgs a{};
  a.p = *args;
  const ff_norm_residual_args& p = a.p;
  auto type = [](int t) { return t == FF_F16 || t == FF_BF16 || t == FF_F32; };
  FF_REQUIRE(type(p.x_type) && type(p.y_type) && (p.x_type == p.y_type || p.x_type == FF_F32),
             "ff_norm_residual: y of type %d beside x of type %d (alike, or x in f32)", p.y_type, p.x_type);
  FF_REQUIRE(p.rows >= 0 && p.rows <= (1 << 30) && p.cols >= 0 && p.cols <= kNrMaxCols, "ff_norm_residual: bad shape rows=%d cols=%d (at most %d)",
             p.rows, p.cols, kNrMaxCols);
  auto kind = [](int n) { return n == FF_NORM_NONE || n == FF_NORM_RMS || n == FF_NORM_LAYER; };
  FF_REQUIRE(kind(p.post) && kind(p.pre), "ff_norm_residual: unknown norm %d or %d", p.post, p.pre);
  FF_REQUIRE(p.rows <= 1 || (p.ldx >= p.cols && p.ldy >= p.cols && p.ldo >= p.cols && (p.normed == nullptr || p.ldn >= p.cols)),
             "ff_norm_residual: row strides must hold %d columns", p.cols);
  if (p.rows == 0 || p.cols == 0) return FF_OK;
  FF_REQUIRE((p.pre != FF_NORM_NONE) == (p.normed != nullptr), "ff_norm_residual: the pre norm and its output come together");
  FF_REQUIRE(p.x && p.y && p.out, "ff_norm_residual: NULL pointer");
  if (p.gate != nullptr) {
    FF_REQUIRE(p.gate_type == FF_F32 || p.gate_type == p.y_type, "ff_norm_residual: a gate of type %d (f32, or as y)", p.gate_type);
    FF_REQUIRE(p.gate_cols == 1 || p.gate_cols == p.cols, "ff_norm_residual: a gate of %d columns (1 or %d)", p.gate_cols, p.cols);
    FF_REQUIRE(p.gate_rows >= 1 && p.ldg >= 0, "ff_norm_residual: a gate of %d rows each, row stride %lld", p.gate_rows, static_cast<long long>(p.ldg));
    FF_REQUIRE(p.gate_act == FF_GATE_PLAIN || p.gate_act == FF_GATE_SIGMOID || p.gate_act == FF_GATE_TANH, "ff_norm_residual: unknown gate %d",
               p.gate_act);
  }
  auto aligned = [](const void* q, int t) { return reinterpret_cast<uintptr_t>(q) % (t == FF_F32 ? 4 : 2) == 0; };
  FF_REQUIRE(aligned(p.x, p.x_type) && aligned(p.out, p.x_type) && aligned(p.y, p.y_type) && aligned(p.normed, p.y_type) &&
                 aligned(p.gate, p.gate_type) && aligned(p.post_w, FF_F32) && aligned(p.post_b, FF_F32) && aligned(p.pre_w, FF_F32) &&
                 aligned(p.pre_b, FF_F32) && aligned(p.scale, FF_F32),
             "ff_norm_residual: misaligned pointer");
  FF_REQUIRE((p.out != p.x || p.ldo == p.ldx || p.rows == 1) && (p.normed == nullptr || p.normed != p.y || p.ldn == p.ldy || p.rows == 1),
             "ff_norm_residual: in place needs equal row strides");
  FF_REQUIRE(p.normed == nullptr || p.normed != p.out, "ff_norm_residual: out and normed are one tensor");
  FF_REQUIRE((p.normed == nullptr || p.normed != p.x) && p.out != p.y, "ff_norm_residual: only out may be x, and only normed y");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.x_type == FF_F32) {
    if (p.y_type == FF_F32)
      launch_nr_types<float, float>(a, s);
    else if (p.y_type == FF_F16)
      launch_nr_types<float, __half>(a, s);
    else
      launch_nr_types<float, __nv_bfloat16>(a, s);
  } else if (p.x_type == FF_F16) {
    launch_nr_types<__half, __half>(a, s);
  } else {
    launch_nr_types<__nv_bfloat16, __nv_bfloat16>(a, s);
  }
  return check_launch("norm_residual_kernel");
}
