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
// Three ways to deal out the columns: FULL, 16-byte chunks (8 columns) that divide the row; SHIFTED, the same when rows start
// off a chunk but all matrices by the same amount, so that only a row's first and last chunk are taken apart; STRIDED, for
// all else, neighbouring columns to neighbouring lanes, one by one.
#include <algorithm>

#include "common.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kChunk = 8;
constexpr int kNrThreads = 128;    // of a CTA whose warps take rows of their own
constexpr int kNrMaxCols = 16376;  // 16 warps x 32 lanes x 4 chunks, less a shift of up to 7

enum class Deal { kFull, kShifted, kStrided };

struct NrArgs {
  ff_norm_residual_args p;
  int lanes;         // per row: 4, 8, 16 or 32, or 32 times the row's warps
  bool gate_chunks;  // a 16-bit gate for every element, dealt out as y is
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
  __device__ __forceinline__ T& at(int i) { return reinterpret_cast<T*>(w)[i]; }
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

// The columns of one thread: chunk k, value e.
template <Deal D>
struct Columns {
  int cols, first, step;  // FULL and SHIFTED: column of chunk 0's value 0, and between chunks; STRIDED: of value 0 and values
  int shift;
  __device__ __forceinline__ Columns(int cols, int lane, int threads, int shift) : cols(cols), shift(shift) {
    first = D == Deal::kStrided ? lane : lane * kChunk - shift;
    step = D == Deal::kStrided ? threads : threads * kChunk;
  }
  __device__ __forceinline__ int at(int k, int e) const {
    return D == Deal::kStrided ? first + (k * kChunk + e) * step : first + k * step + e;
  }
  __device__ __forceinline__ bool holds(int k, int e) const {
    const int c = at(k, e);
    return c < cols && (D != Deal::kShifted || c >= 0);
  }
  // Whether all of chunk k is there (FULL: all or nothing).
  __device__ __forceinline__ bool whole(int k) const {
    if (D == Deal::kStrided) return false;
    const int c = first + k * step;
    return c + kChunk <= cols && (D == Deal::kFull || c >= 0);
  }

  template <class T>
  __device__ __forceinline__ void load(const T* row, int k, Raw<T>& r) const {
    r.clear();
    if (whole(k)) {
      r.load(row + at(k, 0));
    } else if constexpr (D != Deal::kFull) {
#pragma unroll
      for (int e = 0; e < kChunk; ++e)
        if (holds(k, e)) r.at(e) = row[at(k, e)];
    }
  }
  template <class T>
  __device__ __forceinline__ void store(T* row, int k, const float2 (&v)[4]) const {
    Raw<T> r;
    r.set(v);
    if (whole(k)) {
      r.store(row + at(k, 0));
    } else if constexpr (D != Deal::kFull) {
#pragma unroll
      for (int e = 0; e < kChunk; ++e)
        if (holds(k, e)) row[at(k, e)] = r.at(e);
    }
  }
  // f32 parameters of chunk k's columns (0 where there is none), 16-byte aligned but for STRIDED.
  __device__ __forceinline__ void parameters(const float* p, int k, float2 (&v)[4]) const {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (D == Deal::kFull || (D == Deal::kShifted && (shift & 3) == 0 && whole(k))) {
      if (whole(k)) {
        const float4* const q = reinterpret_cast<const float4*>(p + at(k, 0));
        a = __ldg(q);
        b = __ldg(q + 1);
      }
      v[0] = make_float2(a.x, a.y);
      v[1] = make_float2(a.z, a.w);
      v[2] = make_float2(b.x, b.y);
      v[3] = make_float2(b.z, b.w);
    } else if (D == Deal::kShifted && (shift & 1) == 0 && whole(k)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __ldg(reinterpret_cast<const float2*>(p + at(k, 2 * e)));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = make_float2(holds(k, 2 * e) ? __ldg(p + at(k, 2 * e)) : 0.f, holds(k, 2 * e + 1) ? __ldg(p + at(k, 2 * e + 1)) : 0.f);
    }
  }
  // Values past the row to 0.
  template <int K>
  __device__ __forceinline__ void trim(float2 (&v)[K][4]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (whole(k)) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (D == Deal::kFull || !holds(k, 2 * e)) v[k][e].x = 0.f;
        if (D == Deal::kFull || !holds(k, 2 * e + 1)) v[k][e].y = 0.f;
      }
    }
  }
};

// Sum over the threads of a row. Sums of several warps go through `part` (a slot of 32 per call).
template <bool MULTI>
__device__ __forceinline__ float row_sum(float v, int lanes, float* part) {
  if constexpr (MULTI) {
    v = warp_sum(v);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    return warp_sum(lane * 32 < lanes ? part[lane] : 0.f);
  } else {
#pragma unroll
    for (int o = 16; o; o >>= 1)
      if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
}

// v (0 past the row) -> its norm, in place.
template <Deal D, int K, bool MULTI>
__device__ __forceinline__ void norm(float2 (&v)[K][4], const Columns<D>& c, int kind, const float* w, const float* b, float eps, int lanes,
                                     float (*part)[32]) {
  const float inv = 1.f / static_cast<float>(c.cols);
  if (kind == FF_NORM_LAYER) {
    float2 s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e & 1] = add2(s[e & 1], v[k][e]);
    s[0] = add2(s[0], s[1]);
    const float mean = row_sum<MULTI>(s[0].x + s[0].y, lanes, part[0]) * inv;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = sub2(v[k][e], make_float2(mean, mean));
    c.trim(v);
  }
  float2 q[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e & 1] = fma2(v[k][e], v[k][e], q[e & 1]);
  q[0] = add2(q[0], q[1]);
  const float rstd = rsqrtf(row_sum<MULTI>(q[0].x + q[0].y, lanes, part[1]) * inv + eps);
  const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float2 wk[4];
    if (w != nullptr) {
      c.parameters(w, k, wk);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = mul2(v[k][e], mul2(wk[e], r2));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = mul2(v[k][e], r2);
    }
    if (b != nullptr) {
      c.parameters(b, k, wk);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = add2(v[k][e], wk[e]);
    }
  }
}

// e^x within a few 2^-24 of itself: 2^t of the rounded t = x log2(e), corrected by what the product and the constant lost.
__device__ __forceinline__ float exp_close(float x) {
  const float t = x * 1.44269504f;
  const float lost = fmaf(x, 1.44269504f, -t) + x * 1.925963033e-8f;  // log2(e) = 1.44269504 + 1.926e-8
  const float y = ex2_approx(t);
  return fabsf(t) < 126.f ? fmaf(y, lost * 0.693147181f, y) : y;
}
// Within a few 2^-24 of the value: 1 / (1 + e^-g), and for tanh 1 - 2 / (1 + e^2|g|), but its series
// g (1 - g^2 / 3 + 2 g^4 / 15 - 17 g^6 / 315 + 62 g^8 / 2835 - 1382 g^10 / 155925) below 0.35 (the next term is 2^-25 of it there).
__device__ __forceinline__ float activate(float g, int act) {
  if (act == FF_GATE_SIGMOID) return __fdividef(1.f, 1.f + exp_close(fminf(-g, 87.f)));
  if (act == FF_GATE_TANH) {
    const float a = fabsf(g), q = g * g;
    float s = fmaf(q, -8.863235530e-3f, 2.186948854e-2f);
    s = fmaf(q, s, -5.396825397e-2f);
    s = fmaf(q, s, 1.333333333e-1f);
    s = fmaf(q, s, -3.333333333e-1f);
    const float far = 1.f - __fdividef(2.f, 1.f + exp_close(fminf(2.f * a, 87.f)));
    return a < 0.35f ? fmaf(g * q, s, g) : g != g ? g : copysignf(far, g);
  }
  return g;
}

template <class TX, class TY, int K, Deal D, bool MULTI>
__global__ void __launch_bounds__(MULTI ? (K == 1 ? 1024 : 512) : kNrThreads, MULTI ? 1 : K <= 2 ? 8 : sizeof(TX) == 2 && D == Deal::kFull ? 5 : 4) norm_residual_kernel(const __grid_constant__ NrArgs a) {
  __shared__ float part[MULTI ? 4 : 1][32];
  const ff_norm_residual_args& p = a.p;
  const int lanes = a.lanes;  // a power of two unless MULTI
  const int in_row = MULTI ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) & (lanes - 1);
  const int row = MULTI ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * (kNrThreads / lanes) + static_cast<int>(threadIdx.x) / lanes;
  pdl_wait();
  pdl_trigger();
  const bool real = MULTI || row < p.rows;  // lanes without a row go along (their warp's others have one), on nothing
  const int64_t r = real ? row : 0;
  const TY* const y = static_cast<const TY*>(p.y) + r * p.ldy;
  const TX* const x = static_cast<const TX*>(p.x) + r * p.ldx;
  const int shift = D == Deal::kShifted ? static_cast<int>(reinterpret_cast<uintptr_t>(y) / sizeof(TY) % kChunk) : 0;
  Columns<D> c(p.cols, in_row, lanes, shift);
  if (!real) c.first = p.cols;
  Raw<TY> raw[K];
  Raw<TX> xr[K];
#pragma unroll
  for (int k = 0; k < K; ++k) c.load(y, k, raw[k]);
#pragma unroll
  for (int k = 0; k < K; ++k) c.load(x, k, xr[k]);
  float2 v[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = raw[k].pair(e);
  const int64_t gate_at = p.gate != nullptr ? r / p.gate_rows * p.ldg : 0;
  if (a.gate_chunks) {  // under way during the norm
#pragma unroll
    for (int k = 0; k < K; ++k) c.load(static_cast<const TY*>(p.gate) + gate_at, k, raw[k]);
  }
  if (p.post != FF_NORM_NONE) norm<D, K, MULTI>(v, c, p.post, p.post_w, p.post_b, p.post_eps, lanes, part);
  if (p.gate != nullptr) {
    if (p.gate_cols == 1) {
      const float g = activate(p.gate_type == FF_F32 ? static_cast<const float*>(p.gate)[gate_at] : as_f32(static_cast<const TY*>(p.gate)[gate_at]),
                               p.gate_act);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = mul2(v[k][e], make_float2(g, g));
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 g[4];
        if (a.gate_chunks) {
#pragma unroll
          for (int e = 0; e < 4; ++e) g[e] = raw[k].pair(e);
        } else if (p.gate_type == FF_F32) {
          c.parameters(static_cast<const float*>(p.gate) + gate_at, k, g);
        } else {
          const TY* const q = static_cast<const TY*>(p.gate) + gate_at;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            g[e] = make_float2(c.holds(k, 2 * e) ? as_f32(q[c.at(k, 2 * e)]) : 0.f, c.holds(k, 2 * e + 1) ? as_f32(q[c.at(k, 2 * e + 1)]) : 0.f);
        }
        if (p.gate_act != FF_GATE_PLAIN) {
#pragma unroll
          for (int e = 0; e < 4; ++e) g[e] = make_float2(activate(g[e].x, p.gate_act), activate(g[e].y, p.gate_act));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = mul2(v[k][e], g[e]);
      }
    }
  }
  if (p.scale != nullptr) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 s[4];
      c.parameters(p.scale, k, s);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = mul2(v[k][e], s[e]);
    }
  }
  TX* const out = static_cast<TX*>(p.out) + r * p.ldo;
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = fma2(make_float2(p.alpha, p.alpha), xr[k].pair(e), v[k][e]);
    c.store(out, k, v[k]);
  }
  if (p.normed == nullptr) return;
  c.trim(v);  // statistics, biases, gates and infinities can have left others than 0 there
  norm<D, K, MULTI>(v, c, p.pre, p.pre_w, p.pre_b, p.pre_eps, lanes, part + (MULTI ? 2 : 0));
  TY* const normed = static_cast<TY*>(p.normed) + r * p.ldn;
#pragma unroll
  for (int k = 0; k < K; ++k) c.store(normed, k, v[k]);
}

template <class TX, class TY, int K, bool MULTI>
void launch_nr_deal(const NrArgs& a, Deal deal, cudaStream_t s) {
  const int rows = a.p.rows, per = kNrThreads / a.lanes;
  const dim3 grid(MULTI ? rows : (rows + per - 1) / per), block(MULTI ? a.lanes : kNrThreads);
  switch (deal) {
    case Deal::kFull: launch(norm_residual_kernel<TX, TY, K, Deal::kFull, MULTI>, grid, block, 0, s, a); break;
    case Deal::kShifted: launch(norm_residual_kernel<TX, TY, K, Deal::kShifted, MULTI>, grid, block, 0, s, a); break;
    case Deal::kStrided: launch(norm_residual_kernel<TX, TY, K, Deal::kStrided, MULTI>, grid, block, 0, s, a); break;
  }
}

template <class TX, class TY>
void launch_nr(NrArgs& a, cudaStream_t s) {
  const ff_norm_residual_args& p = a.p;
  // How far a matrix's rows start off a chunk, row 0 and from row to row.
  bool same = true, full = p.cols % kChunk == 0;
  int64_t base = -1, pitch = -1;
  auto look = [&](const void* q, int64_t ld, size_t size) {
    const int64_t b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(q) / size % kChunk), l = p.rows > 1 ? (ld % kChunk + kChunk) % kChunk : 0;
    if (base < 0) base = b, pitch = l;
    same = same && b == base && l == pitch;
    full = full && b == 0 && l == 0;
  };
  look(p.y, p.ldy, sizeof(TY));
  look(p.x, p.ldx, sizeof(TX));
  look(p.out, p.ldo, sizeof(TX));
  if (p.normed != nullptr) look(p.normed, p.ldn, sizeof(TY));
  for (const void* q : {static_cast<const void*>(p.post_w), static_cast<const void*>(p.post_b), static_cast<const void*>(p.pre_w),
                        static_cast<const void*>(p.pre_b), static_cast<const void*>(p.scale)})
    full = full && aligned16(q), same = same && aligned16(q);
  if (p.gate != nullptr && p.gate_cols > 1) {
    const bool one = p.rows <= p.gate_rows;  // a single gate row
    if (p.gate_type == FF_F32) {
      const bool fits = aligned16(p.gate) && (one || p.ldg % 4 == 0);
      full = full && fits;
      same = same && fits;
    } else {
      const int64_t b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p.gate) / sizeof(TY) % kChunk), l = one ? 0 : p.ldg % kChunk;
      a.gate_chunks = full ? b == 0 && l == 0 : same && p.gate_rows == 1 && b == base && l == pitch;
    }
  }
  const Deal deal = full ? Deal::kFull : same ? Deal::kShifted : Deal::kStrided;
  if (deal == Deal::kStrided) a.gate_chunks = false;
  // Lanes and chunks per row. Many rows: as few warps as hold the row in 4 chunks per lane. Few rows (less than 16 warps
  // per SM even so): one chunk per lane, for the shortest way through one row.
  const int chunks = (p.cols + (deal == Deal::kShifted ? kChunk - 1 : 0) + kChunk - 1) / kChunk;
  const int wide = (chunks + 31) / 32;
  if (wide > 1 && wide <= 32 && static_cast<int64_t>(p.rows) * wide <= 16LL * sm_count()) {
    a.lanes = 32 * wide;
    return launch_nr_deal<TX, TY, 1, true>(a, deal, s);
  }
  if (wide > 4) {
    a.lanes = 32 * ((wide + 3) / 4);
    return launch_nr_deal<TX, TY, 4, true>(a, deal, s);
  }
  a.lanes = chunks <= 4 ? 4 : chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32;
  switch (wide) {
    case 1: return launch_nr_deal<TX, TY, 1, false>(a, deal, s);
    case 2: return launch_nr_deal<TX, TY, 2, false>(a, deal, s);
    case 3: return launch_nr_deal<TX, TY, 3, false>(a, deal, s);
    default: return launch_nr_deal<TX, TY, 4, false>(a, deal, s);
  }
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
      launch_nr<float, float>(a, s);
    else if (p.y_type == FF_F16)
      launch_nr<float, __half>(a, s);
    else
      launch_nr<float, __nv_bfloat16>(a, s);
  } else if (p.x_type == FF_F16) {
    launch_nr<__half, __half>(a, s);
  } else {
    launch_nr<__nv_bfloat16, __nv_bfloat16>(a, s);
  }
  return check_launch("norm_residual_kernel");
}
