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
constexpr int kNrWarps = 4;       // rows (warps) of a CTA, when a warp takes a row
constexpr int kNrMaxCols = 16376;  // 16 warps x 32 lanes x 4 chunks, less a shift of up to 7

enum class Deal { kFull, kShifted, kStrided };

struct NrArgs {
  ff_norm_residual_args p;
  int warps;  // per row
  bool gate_chunks;  // a 16-bit gate for every element, dealt out as y is
};

// 8 values of one row as they were loaded.
template <class T>
struct Raw {
  uint4 w[sizeof(T) == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void set(int i, T v) { reinterpret_cast<T*>(w)[i] = v; }
  __device__ __forceinline__ T get(int i) const { return reinterpret_cast<const T*>(w)[i]; }
};

__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ void round_to(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void round_to(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void round_to(float v, float& o) { o = v; }

// The columns of one thread: chunk k, value e.
template <Deal D, int K>
struct Columns {
  int cols, first, step;  // FULL and SHIFTED: column of chunk 0's value 0, and between chunks; STRIDED: of value 0 and values
  __device__ __forceinline__ Columns(int cols, int lane, int threads, int shift) : cols(cols) {
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
    if (whole(k)) {
      r.load(row + at(k, 0));
      return;
    }
    r.clear();
    if constexpr (D != Deal::kFull) {
#pragma unroll
      for (int e = 0; e < kChunk; ++e)
        if (holds(k, e)) r.set(e, row[at(k, e)]);
    }
  }
  template <class T>
  __device__ __forceinline__ void store(T* row, int k, const float* v) const {
    if (whole(k)) {
      Raw<T> r;
#pragma unroll
      for (int e = 0; e < kChunk; ++e) {
        T t;
        round_to(v[e], t);
        r.set(e, t);
      }
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(r.w) / 16); ++i) reinterpret_cast<uint4*>(row + at(k, 0))[i] = r.w[i];
      return;
    }
    if constexpr (D != Deal::kFull) {
#pragma unroll
      for (int e = 0; e < kChunk; ++e)
        if (holds(k, e)) round_to(v[e], row[at(k, e)]);
    }
  }
  // f32 parameters of chunk k's columns (0 where there is none).
  __device__ __forceinline__ void parameters(const float* p, int k, float (&v)[kChunk]) const {
    const bool vec = D == Deal::kFull && (reinterpret_cast<uintptr_t>(p) & 15) == 0;  // uniform
    if (vec) {
      const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 a = whole(k) ? __ldg(reinterpret_cast<const float4*>(p + at(k, 0))) : z;
      const float4 b = whole(k) ? __ldg(reinterpret_cast<const float4*>(p + at(k, 0)) + 1) : z;
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < kChunk; ++e) v[e] = holds(k, e) ? __ldg(p + at(k, e)) : 0.f;
    }
  }
};

// Sum over the threads of a row. Sums of several warps go through `part` (one slot of 32 per call).
__device__ __forceinline__ float row_sum(float v, int warps, float* part) {
  v = warp_sum(v);
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) part[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? part[lane] : 0.f);
}

// v -> its norm, in place. `part`: two slots.
template <Deal D, int K>
__device__ __forceinline__ void norm(float (&v)[K][kChunk], const Columns<D, K>& c, int kind, const float* w, const float* b, float eps,
                                     int warps, float* part) {
  const float inv = 1.f / static_cast<float>(c.cols);
  float mean = 0.f;
  if (kind == FF_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < kChunk; ++e) s += v[k][e];  // 0 past the row
    mean = row_sum(s, warps, part) * inv;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool all = D == Deal::kFull && c.whole(k);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) {
      const float d = v[k][e] - mean;
      if (D == Deal::kFull ? all : c.holds(k, e)) {
        v[k][e] = d;
        q = fmaf(d, d, q);
      }
    }
  }
  const float rstd = rsqrtf(row_sum(q, warps, part + 32) * inv + eps);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float wk[kChunk];
    if (w != nullptr) c.parameters(w, k, wk);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) v[k][e] *= w != nullptr ? rstd * wk[e] : rstd;
    if (b != nullptr) {
      c.parameters(b, k, wk);
#pragma unroll
      for (int e = 0; e < kChunk; ++e) v[k][e] += wk[e];
    }
  }
}

__device__ __forceinline__ float activate(float g, int act) {
  if (act == FF_GATE_SIGMOID) return 1.f / (1.f + expf(-g));
  if (act == FF_GATE_TANH) return tanhf(g);
  return g;
}

template <class TX, class TY, int K, Deal D>
__global__ void __launch_bounds__(K == 1 ? 1024 : 512) norm_residual_kernel(const __grid_constant__ NrArgs a) {
  __shared__ float part[4][32];
  const ff_norm_residual_args& p = a.p;
  const int lane = threadIdx.x & 31;
  const int row = a.warps == 1 ? static_cast<int>(blockIdx.x) * kNrWarps + (threadIdx.x >> 5) : static_cast<int>(blockIdx.x);
  const int in_row = a.warps == 1 ? lane : static_cast<int>(threadIdx.x);
  pdl_wait();
  pdl_trigger();
  if (row >= p.rows) return;  // a whole warp, and only where warps do not meet
  const TY* const y = static_cast<const TY*>(p.y) + row * p.ldy;
  const TX* const x = static_cast<const TX*>(p.x) + row * p.ldx;
  const int shift = D == Deal::kShifted ? static_cast<int>(reinterpret_cast<uintptr_t>(y) / sizeof(TY) % kChunk) : 0;
  const Columns<D, K> c(p.cols, in_row, a.warps * 32, shift);
  Raw<TY> yr[K];
  Raw<TX> xr[K];
#pragma unroll
  for (int k = 0; k < K; ++k) c.load(y, k, yr[k]);
#pragma unroll
  for (int k = 0; k < K; ++k) c.load(x, k, xr[k]);
  float v[K][kChunk];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < kChunk; ++e) v[k][e] = as_f32(yr[k].get(e));
  if (p.post != FF_NORM_NONE)
    norm<D, K>(v, c, p.post, p.post_w, p.post_b, p.post_eps, a.warps, part[0]);
  if (p.gate != nullptr) {
    const int64_t at = static_cast<int64_t>(row / p.gate_rows) * p.ldg;
    if (p.gate_cols == 1) {
      const float g = activate(p.gate_type == FF_F32 ? static_cast<const float*>(p.gate)[at] : as_f32(static_cast<const TY*>(p.gate)[at]),
                               p.gate_act);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < kChunk; ++e) v[k][e] *= g;
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float g[kChunk];
        if (p.gate_type == FF_F32) {
          c.parameters(static_cast<const float*>(p.gate) + at, k, g);
        } else if (a.gate_chunks) {
          Raw<TY> r;
          c.load(static_cast<const TY*>(p.gate) + at, k, r);
#pragma unroll
          for (int e = 0; e < kChunk; ++e) g[e] = as_f32(r.get(e));
        } else {
#pragma unroll
          for (int e = 0; e < kChunk; ++e) g[e] = c.holds(k, e) ? as_f32(static_cast<const TY*>(p.gate)[at + c.at(k, e)]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < kChunk; ++e) v[k][e] *= activate(g[e], p.gate_act);
      }
    }
  }
  if (p.scale != nullptr) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s[kChunk];
      c.parameters(p.scale, k, s);
#pragma unroll
      for (int e = 0; e < kChunk; ++e) v[k][e] *= s[e];
    }
  }
  TX* const out = static_cast<TX*>(p.out) + row * p.ldo;
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int e = 0; e < kChunk; ++e) v[k][e] = fmaf(p.alpha, as_f32(xr[k].get(e)), v[k][e]);
    c.store(out, k, v[k]);
  }
  if (p.normed == nullptr) return;
  if (D != Deal::kFull) {  // past the row: sums take zeros (biases, gates and infinite alphas can leave others there)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < kChunk; ++e)
        if (!c.holds(k, e)) v[k][e] = 0.f;
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (!c.whole(k))
#pragma unroll
        for (int e = 0; e < kChunk; ++e) v[k][e] = 0.f;
  }
  norm<D, K>(v, c, p.pre, p.pre_w, p.pre_b, p.pre_eps, a.warps, part[2]);
  TY* const normed = static_cast<TY*>(p.normed) + row * p.ldn;
#pragma unroll
  for (int k = 0; k < K; ++k) c.store(normed, k, v[k]);
}

template <class TX, class TY, int K>
void launch_nr_deal(const NrArgs& a, Deal deal, cudaStream_t s) {
  const int rows = a.p.rows;
  const dim3 grid(a.warps == 1 ? (rows + kNrWarps - 1) / kNrWarps : rows), block(a.warps == 1 ? 32 * kNrWarps : 32 * a.warps);
  switch (deal) {
    case Deal::kFull: launch(norm_residual_kernel<TX, TY, K, Deal::kFull>, grid, block, 0, s, a); break;
    case Deal::kShifted: launch(norm_residual_kernel<TX, TY, K, Deal::kShifted>, grid, block, 0, s, a); break;
    case Deal::kStrided: launch(norm_residual_kernel<TX, TY, K, Deal::kStrided>, grid, block, 0, s, a); break;
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
  const bool before = same, before_full = full;
  a.gate_chunks = false;
  if (p.gate != nullptr && p.gate_cols > 1 && p.gate_type != FF_F32) {
    const int64_t b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p.gate) / sizeof(TY) % kChunk), l = p.ldg % kChunk;
    a.gate_chunks = before_full ? b == 0 && l == 0 : before && p.gate_rows == 1 && b == base && (p.rows == 1 || l == pitch);
  }
  const Deal deal = full ? Deal::kFull : same ? Deal::kShifted : Deal::kStrided;
  if (deal == Deal::kStrided) a.gate_chunks = false;
  // Warps and chunks per row. Many rows: as few warps as hold the row in 4 chunks per lane. Few rows (less than 16 warps
  // per SM even so): one chunk per lane, for the shortest way through one row.
  const int chunks = (p.cols + (deal == Deal::kShifted ? kChunk - 1 : 0) + kChunk - 1) / kChunk;
  const int wide = (chunks + 31) / 32;
  int k = wide <= 32 && static_cast<int64_t>(p.rows) * wide <= 16LL * sm_count() ? 1 : std::min(4, wide);
  a.warps = (wide + k - 1) / k;
  k = (chunks + 32 * a.warps - 1) / (32 * a.warps);
  switch (k) {
    case 1: return launch_nr_deal<TX, TY, 1>(a, deal, s);
    case 2: return launch_nr_deal<TX, TY, 2>(a, deal, s);
    case 3: return launch_nr_deal<TX, TY, 3>(a, deal, s);
    default: return launch_nr_deal<TX, TY, 4>(a, deal, s);
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
