// Per-head norm of queries and keys with the rotary position rotation in the same pass.
//   n = RMS:   x / sqrt(mean(x^2) + eps) * w          LAYER: (x - mean) / sqrt(var + eps) * w + b
//   (y0, y1) -> (y0 cos - y1 sin, y0 sin + y1 cos) for every pair, f32 throughout, one rounding at the end.
//
// Bound by HBM: every value is read and written once (4 bytes). One warp per row: 8 values (16 bytes) per lane,
// D / 8 lanes per head, so the norm is a sum over D / 8 lanes and a pair of FF_ROPE_PAIRS stays in its lane. Warps
// are persistent and keep the weights in registers, a row's angles serve all its heads, and the loads of four steps
// are issued before the first is worked on. A CTA takes 8 neighbouring rows, whose angles share cache sectors of the
// angle-major tables.
//
// Measured, 65600 rows of 32 heads of 64 fp16 (537 MB moved): FF_ROPE_PAIRS RMS norm 91 us (5.9 TB/s, 90% of the copy rate),
// LayerNorm 98; FF_ROPE_HALVES 99 and 136. 32000 rows of 32 heads of 128: 90 and 97, 96 and 136. LayerNorm with halves does
// not fit its registers (twice the angles, and biases; 132 bytes per thread spilled). With a warp per row that ends with it,
// weights read for every row and fewer loads in flight, pairs took 101 and 114.
#include <algorithm>

#include "common.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kQkWarps = 8;
constexpr int kQkCtas = 3;  // per SM
constexpr int kQkSteps = 4;  // of 256 columns, whose loads are issued together

struct QkArgs {
  const void* x;
  int64_t ldx;
  void* out;
  int64_t ldo;
  int rows, q_heads, k_heads;
  const float *q_w, *q_b, *k_w, *k_b;
  float eps;
  const float *cos, *sin;
  int tokens;
};

template <class T, int D, bool LAYER, bool HALVES, bool SHARED>
__global__ void __launch_bounds__(32 * kQkWarps, kQkCtas) qk_norm_rope_kernel(const QkArgs a) {
  constexpr int G = D / 8;       // lanes per head
  constexpr int HPW = 32 / G;    // heads per warp and step
  constexpr int NA = HALVES ? 8 : 4;  // angles per lane
  constexpr int U = kQkSteps;
  const int lane = threadIdx.x & 31, l = lane % G, hl = lane / G;
  pdl_wait();
  pdl_trigger();
  float wq[8], wk[8], bq[LAYER ? 8 : 1], bk[LAYER ? 8 : 1];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    wq[i] = a.q_w != nullptr ? __ldg(a.q_w + l * 8 + i) : 0.f;
    wk[i] = a.k_w != nullptr ? __ldg(a.k_w + l * 8 + i) : 0.f;
    if constexpr (LAYER) {
      bq[i] = a.q_b != nullptr ? __ldg(a.q_b + l * 8 + i) : 0.f;
      bk[i] = a.k_b != nullptr ? __ldg(a.k_b + l * 8 + i) : 0.f;
    }
  }
  // A row's heads in chunks of CH, q then k. SHARED: several warps (blockIdx.y) take turns with them.
  constexpr int CH = U * HPW;
  const int warps = SHARED ? gridDim.y : 1, turn = SHARED ? blockIdx.y : 0;
  const int stride = warps * CH, q_first = turn * CH;
  const int k_first = (turn + warps - (a.q_heads + CH - 1) / CH % warps) % warps * CH;
  const int step = static_cast<int>(gridDim.x) * kQkWarps;
  for (int row = static_cast<int>(blockIdx.x) * kQkWarps + (threadIdx.x >> 5); row < a.rows; row += step) {
    const int pos = row % a.tokens;
    float c[NA], s[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = HALVES ? (l % (G / 2)) * 8 + i : l * 4 + i;
      c[i] = __ldg(a.cos + static_cast<int64_t>(j) * a.tokens + pos);
      s[i] = __ldg(a.sin + static_cast<int64_t>(j) * a.tokens + pos);
    }
    // The first CH of `count` heads of one kind (q or k), which start at column `col` of the row.
    auto heads = [&](int64_t col, int count, const float(&w)[8], const float(&b)[LAYER ? 8 : 1]) {
      const T* const xr = static_cast<const T*>(a.x) + row * a.ldx + col + l * 8;
      T* const orow = static_cast<T*>(a.out) + row * a.ldo + col + l * 8;
      uint4 u[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        u[k] = hl + k * HPW < count ? *reinterpret_cast<const uint4*>(xr + (hl + k * HPW) * D) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (k * HPW >= count) break;  // the whole warp
        float2 y[4] = {Pair16<T>::unpack(u[k].x), Pair16<T>::unpack(u[k].y), Pair16<T>::unpack(u[k].z),
                       Pair16<T>::unpack(u[k].w)};
        if constexpr (LAYER) {
          const float2 t = add2(add2(y[0], y[1]), add2(y[2], y[3]));
          float m = t.x + t.y;
#pragma unroll
          for (int o = G / 2; o; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
          m *= -1.f / D;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = add2(y[i], make_float2(m, m));
        }
        float2 q = mul2(y[0], y[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) q = fma2(y[i], y[i], q);
        float ss = q.x + q.y;
#pragma unroll
        for (int o = G / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rstd = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 wr = mul2(make_float2(rstd, rstd), make_float2(w[2 * i], w[2 * i + 1]));
          if constexpr (LAYER)
            y[i] = fma2(y[i], wr, make_float2(b[2 * i], b[2 * i + 1]));
          else
            y[i] = mul2(y[i], wr);
        }
        if constexpr (HALVES) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, y[i].x, G / 2),
                                             __shfl_xor_sync(0xffffffffu, y[i].y, G / 2));
            const float sx = l < G / 2 ? -s[2 * i] : s[2 * i], sy = l < G / 2 ? -s[2 * i + 1] : s[2 * i + 1];
            y[i] = make_float2(y[i].x * c[2 * i] + other.x * sx, y[i].y * c[2 * i + 1] + other.y * sy);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = make_float2(y[i].x * c[i] - y[i].y * s[i], y[i].x * s[i] + y[i].y * c[i]);
        }
        if (hl + k * HPW < count)
          *reinterpret_cast<uint4*>(orow + (hl + k * HPW) * D) =
              make_uint4(Pair16<T>::pack(y[0].x, y[0].y), Pair16<T>::pack(y[1].x, y[1].y),
                         Pair16<T>::pack(y[2].x, y[2].y), Pair16<T>::pack(y[3].x, y[3].y));
      }
    };
    for (int h = q_first; h < a.q_heads; h += stride) heads(static_cast<int64_t>(h) * D, a.q_heads - h, wq, bq);
    for (int h = k_first; h < a.k_heads; h += stride) heads((static_cast<int64_t>(a.q_heads) + h) * D, a.k_heads - h, wk, bk);
  }
}

template <class T, int D, bool LAYER, bool HALVES>
void launch_qk(const QkArgs& a, cudaStream_t s) {
  const int want = (a.rows + kQkWarps - 1) / kQkWarps, most = sm_count() * kQkCtas;
  constexpr int CH = kQkSteps * 256 / D;
  const int chunks = (a.q_heads + CH - 1) / CH + (a.k_heads + CH - 1) / CH;
  // Fewer rows than four rounds of the GPU's warps: several warps per row, down to the heads that a warp works on at once
  // (50 rows of 64 heads of 128: 12.8 us with one warp per row, 3.3 so).
  const int share = std::min(chunks, 4 * most / want);
  const dim3 block(32 * kQkWarps);
  if (share > 1)
    launch(qk_norm_rope_kernel<T, D, LAYER, HALVES, true>, dim3(want, share), block, 0, s, a);
  else
    launch(qk_norm_rope_kernel<T, D, LAYER, HALVES, false>, dim3(std::min(want, most)), block, 0, s, a);
}

template <class T, int D>
void launch_qk_norm(const QkArgs& a, int norm, int pairing, cudaStream_t s) {
  const bool halves = pairing == FF_ROPE_HALVES;
  if (norm == FF_NORM_LAYER)
    halves ? launch_qk<T, D, true, true>(a, s) : launch_qk<T, D, true, false>(a, s);
  else
    halves ? launch_qk<T, D, false, true>(a, s) : launch_qk<T, D, false, false>(a, s);
}

template <class T>
void launch_qk_dim(const QkArgs& a, int dim, int norm, int pairing, cudaStream_t s) {
  switch (dim) {
    case 32: return launch_qk_norm<T, 32>(a, norm, pairing, s);
    case 64: return launch_qk_norm<T, 64>(a, norm, pairing, s);
    case 128: return launch_qk_norm<T, 128>(a, norm, pairing, s);
    default: return launch_qk_norm<T, 256>(a, norm, pairing, s);
  }
}

}  // namespace

}  // namespace ff

using namespace ff;

extern "C" int ff_qk_norm_rope(const void* x, int dtype, int64_t ldx, void* out, int64_t ldo, int rows, int q_heads,
                               int k_heads, int head_dim, int norm, const float* q_w, const float* q_b,
                               const float* k_w, const float* k_b, float eps, const float* rope_cos,
                               const float* rope_sin, int tokens, int pairing, void* stream) {
  FF_REQUIRE(dtype == FF_F16 || dtype == FF_BF16, "ff_qk_norm_rope: type %d is not fp16 or bf16", dtype);
  FF_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256,
             "ff_qk_norm_rope: head_dim %d is not 32, 64, 128 or 256", head_dim);
  FF_REQUIRE(norm == FF_NORM_RMS || norm == FF_NORM_LAYER, "ff_qk_norm_rope: unknown norm %d", norm);
  FF_REQUIRE(pairing == FF_ROPE_PAIRS || pairing == FF_ROPE_HALVES, "ff_qk_norm_rope: unknown pairing %d", pairing);
  FF_REQUIRE(rows >= 0 && rows <= (1 << 30) && q_heads >= 0 && k_heads >= 0 && q_heads <= (1 << 16) && k_heads <= (1 << 16) && tokens >= 1,
             "ff_qk_norm_rope: bad shape rows=%d heads=%d+%d tokens=%d", rows, q_heads, k_heads, tokens);
  const int64_t cols = static_cast<int64_t>(q_heads + k_heads) * head_dim;
  FF_REQUIRE(ldx >= cols && ldo >= cols && (rows <= 1 || (ldx % 8 == 0 && ldo % 8 == 0)),  // a single row is never stepped over
             "ff_qk_norm_rope: row strides %lld and %lld must hold %lld columns and be multiples of 8",
             static_cast<long long>(ldx), static_cast<long long>(ldo), static_cast<long long>(cols));
  if (rows == 0 || cols == 0) return FF_OK;
  FF_REQUIRE(x && out && rope_cos && rope_sin && (q_w || q_heads == 0) && (k_w || k_heads == 0), "ff_qk_norm_rope: NULL pointer");
  FF_REQUIRE(aligned16(x) && aligned16(out), "ff_qk_norm_rope: x and out must be 16-byte aligned");
  FF_REQUIRE(x != out || ldx == ldo || rows == 1, "ff_qk_norm_rope: in place needs equal row strides");
  const QkArgs a{x, ldx, out, ldo, rows, q_heads, k_heads, q_w, q_b, k_w, k_b, eps, rope_cos, rope_sin, tokens};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FF_F16)
    launch_qk_dim<__half>(a, head_dim, norm, pairing, s);
  else
    launch_qk_dim<__nv_bfloat16>(a, head_dim, norm, pairing, s);
  return check_launch("qk_norm_rope_kernel");
}
