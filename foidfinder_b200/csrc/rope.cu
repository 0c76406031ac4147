// Rotation of heads by positions given per row.
//   t = position * frequency;  (y0, y1) -> scale * (y0 cos t - y1 sin t, y0 sin t + y1 cos t)
// for the rotary / 2 pairs of every head's columns [start, start + rotary): neighbours (FF_ROPE_PAIRS) or a half apart
// (FF_ROPE_HALVES). The other columns are copied (or stay, in place). Rows may have several positions (axes), whose shares
// of the pairs are equal and in order.
//
// Angles: position * frequency and its part of a whole turn in 64 bits (at position 2^20 an angle in 32 bits is off by up
// to 0.06), the sine and cosine of that part in 32 bits, the rotation in 32 bits, one rounding at the end.
//
// Bound by HBM: every value is read and written once. A CTA takes rows whose chunks (16 bytes of a head, or two a half
// apart) make up to kUnits per thread; their loads are issued before the angles of these rows are worked out into shared
// memory, once for all heads. Chunks get narrower (8, 4 bytes, single values) where a size, stride or address asks for it.
#include <algorithm>

#include "common.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeUnits = 4;       // per thread, whose loads are issued together
constexpr int kRopeAngles = 2048;   // per CTA, in shared memory

// n / d for n < 2^31 by a multiplication: m = ceil(2^(31 + l) / d), l = ceil(log2 d), so m d - 2^(31 + l) < d <= 2^l and the
// quotient is exact.
struct Divisor {
  uint32_t d = 1, shift = 0;
  uint64_t m = 0;
  Divisor() = default;
  explicit Divisor(uint32_t v) : d(v) {
    while ((1ull << shift) < v) ++shift;
    m = ((1ull << (31 + shift)) + v - 1) / v;
  }
  __device__ __forceinline__ void operator()(uint32_t n, uint32_t& q, uint32_t& r) const {
    q = static_cast<uint32_t>((n * m) >> (31 + shift));
    r = n - q * d;
  }
};

struct RopeArgs {
  const void* x;
  int64_t ldx;
  void* out;
  int64_t ldo;
  int rows, rows_per_cta, head_dim, start, rotary, axes;
  uint32_t turn_units;  // of a head that turn; those after them copy
  Divisor row_units, head_units;
  const void* positions;
  const void* frequencies;
  bool wide_positions, wide_frequencies;
  float scale;
};

template <int BYTES>
struct Word;
template <>
struct Word<2> { using type = uint16_t; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

// N values of T that are read and written whole, or (ALIGNED false) one by one.
template <class T, int N, bool ALIGNED>
struct Chunk {
  T v[N];
  __device__ __forceinline__ void load(const T* p) {
    using W = typename Word<N * sizeof(T)>::type;
    if constexpr (ALIGNED) {
      const W w = *reinterpret_cast<const W*>(p);
      __builtin_memcpy(v, &w, sizeof v);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    using W = typename Word<N * sizeof(T)>::type;
    if constexpr (ALIGNED) {
      W w;
      __builtin_memcpy(&w, v, sizeof v);
      *reinterpret_cast<W*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = v[i];
    }
  }
};

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// A unit: N values that hold N / 2 neighbouring pairs, or N values and their partners a half further (HALVES). Units past
// turn_units copy N values (one, if not ALIGNED) of the columns outside [start, start + rotary).
template <class T, int N, bool HALVES, bool ALIGNED>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int U = kRopeUnits, COPY = ALIGNED ? N : 1;
  extern __shared__ float2 angle[];  // [rows of the CTA][rotary / 2] (cos, sin), times scale
  pdl_wait();
  pdl_trigger();
  const int row0 = static_cast<int>(blockIdx.x) * a.rows_per_cta, half = a.rotary / 2;
  const uint32_t rows = static_cast<uint32_t>(min(a.rows_per_cta, a.rows - row0)), units = rows * a.row_units.d;
  const T* const x = static_cast<const T*>(a.x) + row0 * a.ldx;
  T* const out = static_cast<T*>(a.out) + row0 * a.ldo;
  for (uint32_t base = 0; base < units; base += kRopeThreads * U) {
    Chunk<T, N, ALIGNED> u[U], v[HALVES ? U : 1];
    uint32_t row[U], col[U], k[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t at = base + i * kRopeThreads + threadIdx.x;
      if (at >= units) break;
      uint32_t c, head;
      a.row_units(at, row[i], c);
      a.head_units(c, head, k[i]);
      const T* const p = x + row[i] * a.ldx;
      col[i] = head * a.head_dim;
      if (k[i] < a.turn_units) {
        col[i] += a.start + k[i] * N;
        u[i].load(p + col[i]);
        if constexpr (HALVES) v[i].load(p + col[i] + half);
      } else {
        const uint32_t o = (k[i] - a.turn_units) * COPY;
        col[i] += o < a.start ? o : o + a.rotary;
        if constexpr (ALIGNED)
          u[i].load(p + col[i]);
        else
          u[i].v[0] = p[col[i]];
      }
    }
    if (base == 0) {
      const int share = half / a.axes;
      for (int i = threadIdx.x; i < static_cast<int>(rows) * half; i += kRopeThreads) {
        const int r = i / half, j = i - r * half;
        const int64_t at = static_cast<int64_t>(row0 + r) * a.axes + j / share;
        const double position = a.wide_positions ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                                                 : static_cast<double>(static_cast<const int*>(a.positions)[at]);
        const double frequency = a.wide_frequencies ? static_cast<const double*>(a.frequencies)[j]
                                                    : static_cast<double>(static_cast<const float*>(a.frequencies)[j]);
        const double turns = position * frequency * 0.15915494309189533577;  // 1 / (2 pi)
        float s, c;
        sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
        angle[i] = make_float2(c * a.scale, s * a.scale);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (base + i * kRopeThreads + threadIdx.x >= units) break;
      T* const p = out + row[i] * a.ldo + col[i];
      if (k[i] >= a.turn_units) {
        if constexpr (ALIGNED)
          u[i].store(p);
        else
          *p = u[i].v[0];
        continue;
      }
      const float2* const t = angle + row[i] * half + k[i] * (HALVES ? N : N / 2);
      if constexpr (HALVES) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 w = t[e];
          const float y0 = to_f32(u[i].v[e]), y1 = to_f32(v[i].v[e]);
          u[i].v[e] = from_f32<T>(y0 * w.x - y1 * w.y);
          v[i].v[e] = from_f32<T>(y0 * w.y + y1 * w.x);
        }
        u[i].store(p);
        v[i].store(p + half);
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 w = t[e / 2];
          const float y0 = to_f32(u[i].v[e]), y1 = to_f32(u[i].v[e + 1]);
          u[i].v[e] = from_f32<T>(y0 * w.x - y1 * w.y);
          u[i].v[e + 1] = from_f32<T>(y0 * w.y + y1 * w.x);
        }
        u[i].store(p);
      }
    }
  }
}

template <class T, int N, bool HALVES, bool ALIGNED>
void launch_rope(RopeArgs& a, int heads, cudaStream_t s) {
  const uint32_t copies = a.x == a.out ? 0 : static_cast<uint32_t>(a.head_dim - a.rotary) / (ALIGNED ? N : 1);
  a.turn_units = static_cast<uint32_t>(a.rotary) / (HALVES ? 2 * N : N);
  a.head_units = Divisor(a.turn_units + copies);
  a.row_units = Divisor(static_cast<uint32_t>(heads) * a.head_units.d);
  const int half = a.rotary / 2;
  // Rows of a CTA: all its threads' units in one go and at most kRopeAngles angles, but fewer while SMs would have nothing
  a.rows_per_cta = std::max(1, std::min<int>(kRopeThreads * kRopeUnits / a.row_units.d, kRopeAngles / half));
  a.rows_per_cta = std::max(1, std::min(a.rows_per_cta, (a.rows + sm_count() - 1) / sm_count()));
  launch(rope_kernel<T, N, HALVES, ALIGNED>, dim3((a.rows + a.rows_per_cta - 1) / a.rows_per_cta), dim3(kRopeThreads),
         sizeof(float2) * a.rows_per_cta * half, s, a);
}

template <class T, bool HALVES>
void launch_rope_width(RopeArgs& a, int heads, cudaStream_t s) {
  // The widest chunk that divides every offset: of a head, of the turning columns and their halves, of rows and addresses.
  const uint64_t bytes = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out);
  uint64_t all = static_cast<uint64_t>(a.head_dim) | a.start | (HALVES ? a.rotary / 2 : a.rotary) | 16 / sizeof(T);
  if (a.rows > 1) all |= static_cast<uint64_t>(a.ldx) | static_cast<uint64_t>(a.ldo);
  all |= bytes / sizeof(T);  // a multiple of sizeof(T)
  const int n = static_cast<int>(all & (~all + 1));
  if constexpr (sizeof(T) == 2)
    if (n >= 8) return launch_rope<T, 8, HALVES, true>(a, heads, s);
  if (n >= 4) return launch_rope<T, 4, HALVES, true>(a, heads, s);
  if (n == 2) return launch_rope<T, 2, HALVES, true>(a, heads, s);
  if constexpr (HALVES)
    launch_rope<T, 1, true, true>(a, heads, s);
  else
    launch_rope<T, 2, false, false>(a, heads, s);
}

template <class T>
void launch_rope_type(RopeArgs& a, int heads, int pairing, cudaStream_t s) {
  if (pairing == FF_ROPE_HALVES)
    launch_rope_width<T, true>(a, heads, s);
  else
    launch_rope_width<T, false>(a, heads, s);
}

}  // namespace

}  // namespace ff

using namespace ff;

extern "C" int ff_rope(const void* x, int dtype, int64_t ldx, void* out, int64_t ldo, int rows, int heads, int head_dim,
                       int start, int rotary, int pairing, const void* positions, int position_bytes, int axes,
                       const void* frequencies, int frequency_bytes, float scale, void* stream) {
  FF_REQUIRE(dtype == FF_F16 || dtype == FF_BF16 || dtype == FF_F32, "ff_rope: unknown type %d", dtype);
  FF_REQUIRE(pairing == FF_ROPE_PAIRS || pairing == FF_ROPE_HALVES, "ff_rope: unknown pairing %d", pairing);
  FF_REQUIRE(rows >= 0 && rows <= (1 << 30) && heads >= 0 && heads <= (1 << 16) && head_dim >= 1 && head_dim <= 1024,
             "ff_rope: bad shape rows=%d heads=%d head_dim=%d", rows, heads, head_dim);
  FF_REQUIRE(rotary >= 2 && rotary % 2 == 0 && start >= 0 && start <= head_dim - rotary,
             "ff_rope: columns %d to %d + %d of a head of %d, in pairs", start, start, rotary, head_dim);
  FF_REQUIRE(axes >= 1 && (rotary / 2) % axes == 0, "ff_rope: %d pairs do not divide into %d axes", rotary / 2, axes);
  FF_REQUIRE((position_bytes == 4 || position_bytes == 8) && (frequency_bytes == 4 || frequency_bytes == 8),
             "ff_rope: positions and frequencies have 4 or 8 bytes, not %d and %d", position_bytes, frequency_bytes);
  const int64_t cols = static_cast<int64_t>(heads) * head_dim;
  FF_REQUIRE(rows <= 1 || (ldx >= cols && ldo >= cols), "ff_rope: row strides %lld and %lld must hold %lld columns",
             static_cast<long long>(ldx), static_cast<long long>(ldo), static_cast<long long>(cols));
  if (rows == 0 || cols == 0) return FF_OK;
  FF_REQUIRE(x && out && positions && frequencies, "ff_rope: NULL pointer");
  const uintptr_t size = dtype == FF_F32 ? 4 : 2;
  FF_REQUIRE(reinterpret_cast<uintptr_t>(x) % size == 0 && reinterpret_cast<uintptr_t>(out) % size == 0 &&
                 reinterpret_cast<uintptr_t>(positions) % position_bytes == 0 &&
                 reinterpret_cast<uintptr_t>(frequencies) % frequency_bytes == 0,
             "ff_rope: misaligned pointer");
  FF_REQUIRE(x != out || ldx == ldo || rows == 1, "ff_rope: in place needs equal row strides");
  RopeArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.out = out;
  a.ldo = ldo;
  a.rows = rows;
  a.head_dim = head_dim;
  a.start = start;
  a.rotary = rotary;
  a.axes = axes;
  a.positions = positions;
  a.frequencies = frequencies;
  a.wide_positions = position_bytes == 8;
  a.wide_frequencies = frequency_bytes == 8;
  a.scale = scale;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FF_F16)
    launch_rope_type<__half>(a, heads, pairing, s);
  else if (dtype == FF_BF16)
    launch_rope_type<__nv_bfloat16>(a, heads, pairing, s);
  else
    launch_rope_type<float>(a, heads, pairing, s);
  return check_launch("rope_kernel");
}
