// Rotation of heads by positions given per row.
//   t = position * frequency;  (y0, y1) -> scale * (y0 cos t - y1 sin t, y0 sin t + y1 cos t)
// for the rotary / 2 pairs of every head's columns [start, start + rotary): neighbours (FF_ROPE_PAIRS) or a half apart
// (FF_ROPE_HALVES). The other columns are copied (or stay, in place). Rows may have several positions (axes), whose shares
// of the pairs are equal and in order.
//
// Angles: position * frequency and its part of a whole turn in 64 bits (at position 2^20 an angle in 32 bits is off by up
// to 0.06), the sine and cosine of that part in 32 bits, the rotation in 32 bits, one rounding at the end.
//
// Measured: 65600 rows of 32 heads of 64, fp16 (537 MB): pairs 91 us, 5.9 TB/s (at 1965 MHz; 94 at 1840, under the power limit);
// halves 87 us, 6.1 TB/s (91 at 1810 MHz). 32001 rows of 8 heads of 128, bf16, 64 columns turning: halves 23.0 us, 5.7 TB/s.
//
// Bound by HBM: every value is read and written once. A CTA takes rows whose turning units (32 bytes of a head, or twice 16 a
// half apart) make up to kTurning per thread; their loads are issued before the angles of the rows are worked out into
// shared memory, once for all heads, and the columns that do not turn are copied. Units get narrower, down to single
// values, where a size, stride or address asks for it.
#include <algorithm>

#include "common.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kTurning = 2;         // units per thread whose loads are issued together
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
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return static_cast<uint32_t>((n * m) >> (31 + shift)); }
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
  Divisor turn_row, turn_head, copy_row, copy_head;  // units of a row and of a head that turn, and that are copied
  Divisor angles, share;                            // of a row, and of an axis
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
template <>
struct Word<32> { using type = struct { uint4 a, b; }; };

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

// Values as pairs of f32, and back.
template <class T, int N>
__device__ __forceinline__ void widen(const T (&v)[N], float (&f)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = v[e];
  } else if constexpr (N == 1) {
    uint16_t h;
    __builtin_memcpy(&h, v, 2);
    f[0] = Pair16<T>::unpack(h).x;
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      uint32_t w;
      __builtin_memcpy(&w, v + e, 4);
      const float2 p = Pair16<T>::unpack(w);
      f[e] = p.x;
      f[e + 1] = p.y;
    }
  }
}
template <class T, int N>
__device__ __forceinline__ void narrow(const float (&f)[N], T (&v)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = f[e];
  } else if constexpr (N == 1) {
    const uint32_t w = Pair16<T>::pack(f[0], 0.f);
    __builtin_memcpy(v, &w, 2);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const uint32_t w = Pair16<T>::pack(f[e], f[e + 1]);
      __builtin_memcpy(v + e, &w, 4);
    }
  }
}
// N neighbouring f32 values of shared memory that start at a multiple of N.
template <int N>
__device__ __forceinline__ void read(const float* p, float (&f)[N]) {
  constexpr int W = N >= 4 ? 4 : N;
#pragma unroll
  for (int i = 0; i < N; i += W) __builtin_memcpy(f + i, __builtin_assume_aligned(p + i, 4 * W), 4 * W);
}

// A unit: N values that hold N / 2 neighbouring pairs, or N values and their partners a half further (HALVES). Columns outside
// [start, start + rotary) are copied N at a time (one, if not ALIGNED).
template <class T, int N, bool HALVES, bool ALIGNED>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int U = kTurning, COPY = ALIGNED ? N : 1, COPIES = N * sizeof(T) > 16 ? 2 : 4, PAIRS = HALVES ? N : N / 2;
  extern __shared__ __align__(16) float table[];  // [rows of the CTA][rotary / 2] cosines, then sines, both times scale
  pdl_wait();
  pdl_trigger();
  const int row0 = static_cast<int>(blockIdx.x) * a.rows_per_cta, half = a.rotary / 2;
  const uint32_t rows = static_cast<uint32_t>(min(a.rows_per_cta, a.rows - row0)), units = rows * a.turn_row.d;
  float* const sines = table + a.rows_per_cta * half;
  const T* const x = static_cast<const T*>(a.x) + row0 * a.ldx;
  T* const out = static_cast<T*>(a.out) + row0 * a.ldo;
  for (uint32_t base = 0; base < units; base += kRopeThreads * U) {
    Chunk<T, N, ALIGNED> u[U], v[HALVES ? U : 1];
    // Row, column and number within its head of a unit (worked out twice: kept, they take the registers of a CTA per SM).
    auto locate = [&](uint32_t at, uint32_t& row, uint32_t& col, uint32_t& k) {
      uint32_t c, head;
      a.turn_row(at, row, c);
      a.turn_head(c, head, k);
      col = head * a.head_dim + a.start + k * N;
    };
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t at = base + i * kRopeThreads + threadIdx.x;
      if (at >= units) break;
      uint32_t row, col, k;
      locate(at, row, col, k);
      const T* const p = x + row * a.ldx + col;
      u[i].load(p);
      if constexpr (HALVES) v[i].load(p + half);
    }
    if (base == 0) {
      for (uint32_t i = threadIdx.x; i < rows * half; i += kRopeThreads) {
        uint32_t r, j;
        a.angles(i, r, j);
        const int64_t at = static_cast<int64_t>(row0 + r) * a.axes + (a.axes == 1 ? 0u : a.share(j));
        const double position = a.wide_positions ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                                                 : static_cast<double>(static_cast<const int*>(a.positions)[at]);
        const double frequency = a.wide_frequencies ? static_cast<const double*>(a.frequencies)[j]
                                                    : static_cast<double>(static_cast<const float*>(a.frequencies)[j]);
        const double turns = position * frequency * 0.15915494309189533577;  // 1 / (2 pi)
        float s, c;
        sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
        table[i] = c * a.scale;
        sines[i] = s * a.scale;
      }
      if (a.x != a.out) {
        const uint32_t copies = rows * a.copy_row.d;
        for (uint32_t first = threadIdx.x; first < copies; first += kRopeThreads * COPIES) {
          Chunk<T, COPY, ALIGNED> w[COPIES];
          uint32_t to_row[COPIES], to[COPIES];
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            const uint32_t at = first + i * kRopeThreads;
            if (at >= copies) break;
            uint32_t c, head, o;
            a.copy_row(at, to_row[i], c);
            a.copy_head(c, head, o);
            o *= COPY;
            to[i] = head * a.head_dim + (o < static_cast<uint32_t>(a.start) ? o : o + a.rotary);
            w[i].load(x + to_row[i] * a.ldx + to[i]);
          }
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            if (first + i * kRopeThreads >= copies) break;
            w[i].store(out + to_row[i] * a.ldo + to[i]);
          }
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      uint32_t at = base + i * kRopeThreads + threadIdx.x;
      if (at >= units) break;
      asm volatile("" : "+r"(at));  // not the values from above
      uint32_t row, col, k;
      locate(at, row, col, k);
      T* const p = out + row * a.ldo + col;
      float c[PAIRS], s[PAIRS], y0[N];
      read(table + row * half + k * PAIRS, c);
      read(sines + row * half + k * PAIRS, s);
      widen(u[i].v, y0);
      if constexpr (HALVES) {
        float y1[N];
        widen(v[i].v, y1);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float r = y0[e] * c[e] - y1[e] * s[e];
          y1[e] = y0[e] * s[e] + y1[e] * c[e];
          y0[e] = r;
        }
        narrow(y0, u[i].v);
        narrow(y1, v[i].v);
        u[i].store(p);
        v[i].store(p + half);
      } else {
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          const float r = y0[2 * e] * c[e] - y0[2 * e + 1] * s[e];
          y0[2 * e + 1] = y0[2 * e] * s[e] + y0[2 * e + 1] * c[e];
          y0[2 * e] = r;
        }
        narrow(y0, u[i].v);
        u[i].store(p);
      }
    }
  }
}

template <class T, int N, bool HALVES, bool ALIGNED>
void launch_rope(RopeArgs& a, int heads, cudaStream_t s) {
  const int copies = (a.head_dim - a.rotary) / (ALIGNED ? N : 1), half = a.rotary / 2, turning = a.rotary / (HALVES ? 2 * N : N);
  a.turn_head = Divisor(turning);
  a.turn_row = Divisor(static_cast<uint32_t>(heads) * turning);
  if (copies > 0 && a.x != a.out) {
    a.copy_head = Divisor(copies);
    a.copy_row = Divisor(static_cast<uint32_t>(heads) * copies);
  } else {
    a.copy_row.d = 0;  // nothing to copy
  }
  a.angles = Divisor(half);
  a.share = Divisor(half / a.axes);
  // Rows of a CTA: their units in one go and at most kRopeAngles angles, but fewer while SMs would have nothing
  a.rows_per_cta = std::max(1, std::min<int>(kRopeThreads * kTurning / a.turn_row.d, kRopeAngles / half));
  a.rows_per_cta = std::max(1, std::min(a.rows_per_cta, (a.rows + sm_count() - 1) / sm_count()));
  launch(rope_kernel<T, N, HALVES, ALIGNED>, dim3((a.rows + a.rows_per_cta - 1) / a.rows_per_cta), dim3(kRopeThreads),
         2 * sizeof(float) * a.rows_per_cta * half, s, a);
}

template <class T, bool HALVES>
void launch_rope_width(RopeArgs& a, int heads, cudaStream_t s) {
  // The widest chunk that divides every offset: of a head, of the turning columns and their halves, of rows and addresses.
  const uint64_t bytes = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out);
  uint64_t all = static_cast<uint64_t>(a.head_dim) | a.start | (HALVES ? a.rotary / 2 : a.rotary) | (HALVES ? 16 : 32) / sizeof(T);
  if (a.rows > 1) all |= static_cast<uint64_t>(a.ldx) | static_cast<uint64_t>(a.ldo);
  all |= bytes / sizeof(T);  // a multiple of sizeof(T)
  const int n = static_cast<int>(all & (~all + 1));
  if constexpr (!HALVES)
    if (n >= static_cast<int>(32 / sizeof(T))) return launch_rope<T, 32 / sizeof(T), HALVES, true>(a, heads, s);
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
