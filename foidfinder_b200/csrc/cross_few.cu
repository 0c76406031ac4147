// Attention of few queries per sequence to its keys and values (one decoder token, some learned queries).
//   out = softmax(scale q k^T) v, head by head, keys that do not take part left out
//
// Bound by HBM: keys and values are read once, 4 bytes per key, head and column, for a few multiply-adds each. A CTA takes
// one part of one sequence's keys and one key head, and all query rows that read it (the group's heads of every query,
// 16 * RG rows at a time). Key and value tiles of 64 keys come through a ring of asynchronous 16-byte copies, which fill a
// key that does not take part with zeros instead of reading it (so that whatever it holds, its value counts 0 * 0). RG
// warps divide the rows, 4 / RG warps the keys of a tile; each keeps a running maximum, sum and output of its keys in
// registers (mma.sync: the products are far from what bounds this kernel, and 16 rows are what there is). The warps' parts
// are joined through shared memory in a fixed order. Up to 8 parts of a sequence are a cluster of CTAs, which read one
// another's shared memory (no second launch: one token over 1025 keys 9.6 -> 7.4 us, over 4096 keys no gain); more of them go through the workspace
// and a second kernel.
//
// Measured (fp16, at 1965 MHz): 32 queries over 1025 keys of 64 images, 16 heads of 64: 63 us, 4.4 TB/s, where half of the issue
// slots go to the warps' chains of products and exponentials; one query 50.2 us, 5.4 TB/s; one query over 24600 keys of 4
// sequences, 16 heads over 4 of 128: 39 us, 5.2 TB/s; one query over 1025 keys of one image 7.3 us, over 32800 keys of one
// head of 128 13.1.
//
// P is rounded to 16 bits for its product with V, as 2^((s - max) scale + 14) in fp16, where it would else lose bits below 2^-14, and
// with -20 in bf16, so that sums over 2^20 values next to the type's largest stay in f32's range; sums of P are taken
// before that rounding, in f32.
#include <algorithm>

#include "common.h"
#include "cross.h"
#include "fp4.cuh"

namespace ff {

namespace {

constexpr int kKeys = 64;        // of a tile
constexpr int kFewThreads = 128;
constexpr int kCluster = 8;      // CTAs of a cluster, at most
constexpr int kClusterTiles = 40;  // of a sequence, beyond which a second launch costs less than having 8 parts only
__host__ __device__ constexpr int few_stages(int atoms) { return atoms == 1 ? 3 : 2; }
__host__ __device__ constexpr int few_ctas(int atoms) { return atoms == 1 ? 4 : 3; }  // per SM
__host__ __device__ constexpr int few_tile(int atoms) { return atoms * kKeys * 128; }  // bytes of a K or V tile
__host__ __device__ constexpr int few_smem(int atoms) { return few_stages(atoms) * 2 * few_tile(atoms); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define FF_MMA(TYPE)                                                                                              \
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                             \
               ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                             \
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                   \
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
  if constexpr (std::is_same<T, __half>::value)
    FF_MMA("f16");
  else
    FF_MMA("bf16");
#undef FF_MMA
}

// Byte of 16-byte chunk c (of 8 * atoms) of a tile's row: 128-byte rows per atom, chunks permuted by the row so that
// neither eight rows of a chunk nor eight chunks of a row meet in a bank.
__device__ __forceinline__ uint32_t tile_byte(int row, int c) {
  return static_cast<uint32_t>((c >> 3) * (kKeys * 128) + row * 128 + (((c ^ row) & 7) << 4));
}

__device__ __forceinline__ float4 read_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 read_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
// What scores are relative to: the largest, or nothing (where it is -inf, nothing but NaN can be there, and counts all the same).
__device__ __forceinline__ float reference(float top) { return top == -INFINITY ? 0.f : top; }
// Weight of a part whose largest score is m.
__device__ __forceinline__ float part_weight(float m, float ref, float scale_log2) { return ex2_approx((m - ref) * scale_log2); }

struct FewArgs {
  CrossArgs p;
  int passes, splits;
  bool cluster;    // the splits of a sequence are a cluster
  float* part_o;   // [splits][q_rows * heads][dim]
  float2* part_ml;  // [splits][q_rows * heads]: largest score and sum
};

// SHORT: sequences of about a tile of keys, whose products leave out groups of 16 keys that there are not.
template <class T, int ATOMS, int RG, bool SHORT>
__global__ void __launch_bounds__(kFewThreads, few_ctas(ATOMS)) cross_few_kernel(const __grid_constant__ FewArgs a) {
  constexpr int STAGES = few_stages(ATOMS), TILE = few_tile(ATOMS), KG = 4 / RG, KW = kKeys / KG;
  constexpr int ROWS = 16 * RG, STEPS = ATOMS * 4;
  constexpr float kShift = std::is_same<T, __half>::value ? 14.f : -20.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t taken[STAGES];  // bits: keys of a tile that take part
  __shared__ float part_m[KG][ROWS], part_l[KG][ROWS];
  __shared__ __align__(8) float2 joined[ROWS];
  const CrossArgs& p = a.p;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rg = warp % RG, kg = warp / RG;
  const int group = p.heads / p.kv_heads, dim = p.dim, chunks = dim / 8;
  int at = static_cast<int>(blockIdx.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int pass0 = at % a.passes;
  at /= a.passes;
  const int kvh = at % p.kv_heads, b = at / p.kv_heads;
  pdl_wait();
  pdl_trigger();
  const Piece qs = query_piece(p, b), ks = key_piece(p, b);
  const int total_rows = qs.n * group;
  const int all_tiles = (ks.n + kKeys - 1) / kKeys, per = (all_tiles + a.splits - 1) / a.splits;
  const int first = split * per, tiles = max(0, min(per, all_tiles - first));
  const T* const kp = static_cast<const T*>(p.k) + (ks.at + static_cast<int64_t>(first) * kKeys) * p.ldk + static_cast<int64_t>(kvh) * dim;
  const T* const vp = static_cast<const T*>(p.v) + (ks.at + static_cast<int64_t>(first) * kKeys) * p.ldv + static_cast<int64_t>(kvh) * dim;
  const uint8_t* const mask = p.mask != nullptr ? p.mask + ks.at + static_cast<int64_t>(first) * kKeys : nullptr;
  const int keys = max(0, min(tiles * kKeys, ks.n - first * kKeys));
  const uint32_t base = smem_u32(smem);
  const int quads = dim / 4, at_once = 32 / quads, lane_row = lane / quads, c = lane % quads * 4;  // when parts are joined

  // Mask bytes of tile i's keys lane and lane + 32 (1 without a mask), 0 past the end.
  uint32_t ahead[2];
  auto fetch = [&](int i) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int key = i * kKeys + 32 * c + lane;
      ahead[c] = key < keys ? (mask != nullptr ? __ldg(mask + key) : 1u) : 0u;
    }
  };
  auto ahead_bits = [&]() -> uint64_t {  // the keys that take part
    const uint64_t l = __ballot_sync(0xffffffffu, ahead[0] != 0), h = __ballot_sync(0xffffffffu, ahead[1] != 0);
    return l | h << 32;
  };
  // This thread copies chunk t % 8 (of an atom) of the rows t / 8 + 16 n, whose swizzle is the same.
  const int64_t k16 = 16 * p.ldk, v16 = 16 * p.ldv;
  const T* const k_own = kp + (t >> 3) * p.ldk + (t & 7) * 8;
  const T* const v_own = vp + (t >> 3) * p.ldv + (t & 7) * 8;
  const uint32_t own = tile_byte(t >> 3, t & 7);
  auto load = [&](int i, uint64_t bits) {
    const int st = i % STAGES;
    if (t == 0) taken[st] = bits;
    const uint32_t d = base + st * 2 * TILE + own;
    const T* ks = k_own + 4 * i * k16;
    const T* vs = v_own + 4 * i * v16;
    if (bits == ~0ull) {
#pragma unroll
      for (int n = 0; n < 4; ++n, ks += k16, vs += v16)
#pragma unroll
        for (int c = 0; c < ATOMS; ++c)
          if (c * 8 + (t & 7) < chunks) {
            copy16(d + c * (kKeys * 128) + n * 2048, ks + c * 64, true);
            copy16(d + TILE + c * (kKeys * 128) + n * 2048, vs + c * 64, true);
          }
      return;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n, ks += k16, vs += v16) {
      const bool take = bits >> (16 * n + (t >> 3)) & 1;  // a key left out is not read
#pragma unroll
      for (int c = 0; c < ATOMS; ++c)
        if (c * 8 + (t & 7) < chunks) {
          copy16(d + c * (kKeys * 128) + n * 2048, take ? ks + c * 64 : kp, take);
          copy16(d + TILE + c * (kKeys * 128) + n * 2048, take ? vs + c * 64 : vp, take);
        }
    }
  };

  for (int pass = pass0; pass * ROWS < total_rows; pass += a.passes) {
    fetch(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      const uint64_t bits = ahead_bits();
      fetch(i + 1);
      if (i < tiles) load(i, bits);
      copies_commit();
    }
    // Rows of this lane: lane / 4 and 8 further, of the warp's 16.
    uint32_t qf[STEPS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = pass * ROWS + rg * 16 + h * 8 + (lane >> 2);
      const T* qp = static_cast<const T*>(p.q);
      if (row < total_rows) qp += static_cast<int64_t>(qs.at + row / group) * p.ldq + static_cast<int64_t>(kvh * group + row % group) * dim;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          qf[s][2 * c + h] = row < total_rows && s * 16 < dim ? *reinterpret_cast<const uint32_t*>(qp + s * 16 + c * 8 + (lane & 3) * 2) : 0;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2 * STEPS][4];
#pragma unroll
    for (int n = 0; n < 2 * STEPS; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    for (int i = 0; i < tiles; ++i) {
      copies_wait<STAGES - 2>();
      __syncthreads();  // tile i has landed for all, and all are done with tile i - 1, whose place is next
      const uint64_t next = ahead_bits();
      if (i + STAGES - 1 < tiles) load(i + STAGES - 1, next);
      copies_commit();
      fetch(i + STAGES);
      const uint32_t kt = base + (i % STAGES) * 2 * TILE, vt = kt + TILE;
      const uint64_t bits = taken[i % STAGES] >> (kg * KW);  // of this warp's keys
      const int groups = SHORT ? (min(KW, keys - i * kKeys - kg * KW) + 15) >> 4 : KW / 16;  // of 16 keys (none: 0 or less)
      float s[KW / 8][4];
#pragma unroll
      for (int n = 0; n < KW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        if (k * 16 >= dim) break;
#pragma unroll
        for (int n = 0; n < KW / 16; ++n) {
          if (SHORT && n >= groups) break;
          uint32_t f[4];
          ldmatrix4(kt + tile_byte(kg * KW + n * 16 + (lane >> 4) * 8 + (lane & 7), k * 2 + (lane >> 3 & 1)), f);
          mma16816<T>(s[2 * n], qf[k], f[0], f[1]);
          mma16816<T>(s[2 * n + 1], qf[k], f[2], f[3]);
        }
      }
      // Keys that do not take part are -inf (also where their products are NaN).
      const uint64_t all = KW == 64 ? ~0ull : (1ull << (KW & 63)) - 1;
      float mx[2] = {-INFINITY, -INFINITY};
      if ((bits & all) != all) {
#pragma unroll
        for (int n = 0; n < KW / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(bits >> (n * 8 + (lane & 3) * 2 + (e & 1)) & 1)) s[n][e] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < KW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
      float ref[2];  // subtracted from the scores themselves, however large: times scale their difference would be lost
      bool grew = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float now = fmaxf(m[h], mx[h]);
        grew |= now > m[h];
        mx[h] = m[h];  // the old one
        m[h] = now;
        ref[h] = reference(now);
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float corr = ex2_approx((mx[h] - ref[h]) * p.scale_log2);
          l[h] *= corr;
#pragma unroll
          for (int n = 0; n < 2 * STEPS; ++n) {
            o[n][2 * h] *= corr;
            o[n][2 * h + 1] *= corr;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) {
        if (SHORT && n >= 2 * groups) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 x = fma2(sub2(make_float2(s[n][2 * h], s[n][2 * h + 1]), make_float2(ref[h], ref[h])), make_float2(p.scale_log2, p.scale_log2),
                                make_float2(kShift, kShift));
          s[n][2 * h] = ex2_approx(x.x);
          s[n][2 * h + 1] = ex2_approx(x.y);
          l[h] += s[n][2 * h];
          l[h] += s[n][2 * h + 1];
        }
      }
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        if (SHORT && n >= groups) break;
        const uint32_t pf[4] = {Pair16<T>::pack(s[2 * n][0], s[2 * n][1]), Pair16<T>::pack(s[2 * n][2], s[2 * n][3]),
                                Pair16<T>::pack(s[2 * n + 1][0], s[2 * n + 1][1]), Pair16<T>::pack(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
          if (c * 16 >= dim) break;
          uint32_t f[4];
          ldmatrix4_trans(vt + tile_byte(kg * KW + n * 16 + (lane & 15), c * 2 + (lane >> 4)), f);
          mma16816<T>(o[2 * c], pf, f[0], f[1]);
          mma16816<T>(o[2 * c + 1], pf, f[2], f[3]);
        }
      }
    }
    copies_wait<0>();
    __syncthreads();  // the ring is free: the warps' parts meet there, [KG][ROWS][dim] f32
    float* const parts = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int row = rg * 16 + h * 8 + (lane >> 2);
      if ((lane & 3) == 0) {
        part_m[kg][row] = m[h];
        part_l[kg][row] = l[h];
      }
      float* const dst = parts + (kg * ROWS + row) * dim + (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < 2 * STEPS; ++n)
        if (n * 8 < dim) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
    __syncthreads();
    // A row of `dim / 4` lanes, as many rows at a time as a warp has of them.
    for (int r = warp * at_once + lane_row; r < ROWS; r += 4 * at_once) {
      const int row = pass * ROWS + r;
      if (lane_row >= at_once || row >= total_rows) break;
      float top = part_m[0][r];
#pragma unroll
      for (int g = 1; g < KG; ++g) top = fmaxf(top, part_m[g][r]);
      const float ref = reference(top);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const float w = part_weight(part_m[g][r], ref, p.scale_log2);
        const float4 v = *reinterpret_cast<const float4*>(parts + (g * ROWS + r) * dim + c);
        sum = fmaf(part_l[g][r], w, sum);
        acc.x = fmaf(v.x, w, acc.x);
        acc.y = fmaf(v.y, w, acc.y);
        acc.z = fmaf(v.z, w, acc.z);
        acc.w = fmaf(v.w, w, acc.w);
      }
      const int64_t q_row = qs.at + row / group;
      const int head = kvh * group + row % group;
      if (a.splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key: zeros
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + q_row * p.ldo + static_cast<int64_t>(head) * dim + c) =
            make_uint2(Pair16<T>::pack(acc.x * inv, acc.y * inv), Pair16<T>::pack(acc.z * inv, acc.w * inv));
      } else if (a.cluster) {
        *reinterpret_cast<float4*>(parts + r * dim + c) = acc;  // in the place of the first group's, which no one else reads
        if (c == 0) joined[r] = make_float2(top, sum);
      } else {
        const int64_t at_row = (static_cast<int64_t>(split) * p.q_rows + q_row) * p.heads + head;
        *reinterpret_cast<float4*>(a.part_o + at_row * dim + c) = acc;
        if (c == 0) a.part_ml[at_row] = make_float2(top, sum);
      }
    }
    if (a.cluster) {
      __syncwarp();
      cluster_sync();  // every CTA's part of these rows is there
      for (int r = (split * 4 + warp) * at_once + lane_row; r < ROWS; r += a.splits * 4 * at_once) {
        const int row = pass * ROWS + r;
        if (lane_row >= at_once || row >= total_rows) break;
        float2 ml[kCluster];
        float4 v[kCluster];
#pragma unroll
        for (int g = 0; g < kCluster; ++g) {
          ml[g] = make_float2(-INFINITY, 0.f);
          v[g] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (g < a.splits) {
            ml[g] = read_cluster2(mapa_shared(smem_u32(&joined[r]), g));
            v[g] = read_cluster(mapa_shared(smem_u32(parts + r * dim + c), g));
          }
        }
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int g = 0; g < kCluster; ++g) top = fmaxf(top, ml[g].x);
        const float ref = reference(top);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < kCluster; ++g) {
          const float w = part_weight(ml[g].x, ref, p.scale_log2);
          sum = fmaf(ml[g].y, w, sum);
          acc.x = fmaf(v[g].x, w, acc.x);
          acc.y = fmaf(v[g].y, w, acc.y);
          acc.z = fmaf(v[g].z, w, acc.z);
          acc.w = fmaf(v[g].w, w, acc.w);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + static_cast<int64_t>(qs.at + row / group) * p.ldo + static_cast<int64_t>(kvh * group + row % group) * dim + c) =
            make_uint2(Pair16<T>::pack(acc.x * inv, acc.y * inv), Pair16<T>::pack(acc.z * inv, acc.w * inv));
      }
      __syncwarp();
      cluster_sync();  // and has been read
    } else {
      __syncthreads();  // before the next pass fills the ring
    }
  }
}

// out = the splits' parts, joined in order: a CTA per query row and head, a warp for every kJoinWarps-th part.
constexpr int kJoinWarps = 8;
template <class T>
__global__ void __launch_bounds__(32 * kJoinWarps) cross_join_kernel(const __grid_constant__ FewArgs a) {
  __shared__ float sums[kJoinWarps];
  __shared__ float4 accs[kJoinWarps][32];
  const CrossArgs& p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t at = blockIdx.x, rows = static_cast<int64_t>(p.q_rows) * p.heads;
  pdl_wait();
  pdl_trigger();
  const int q_row = static_cast<int>(at / p.heads), head = static_cast<int>(at % p.heads);
  if (p.q_start != nullptr && (q_row < __ldg(p.q_start) || q_row >= __ldg(p.q_start + p.sequences))) return;  // of no sequence
  float top = -INFINITY;
  for (int i = lane; i < a.splits; i += 32) top = fmaxf(top, a.part_ml[i * rows + at].x);
  top = reference(warp_max(top));
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int c = lane * 4;
#pragma unroll 4
  for (int i = warp; i < a.splits; i += kJoinWarps) {
    const float2 ml = a.part_ml[i * rows + at];
    const float w = part_weight(ml.x, top, p.scale_log2);
    sum = fmaf(ml.y, w, sum);
    if (c < p.dim) {
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + (i * rows + at) * p.dim + c);
      acc.x = fmaf(v.x, w, acc.x);
      acc.y = fmaf(v.y, w, acc.y);
      acc.z = fmaf(v.z, w, acc.z);
      acc.w = fmaf(v.w, w, acc.w);
    }
  }
  accs[warp][lane] = acc;
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (warp != 0 || c >= p.dim) return;
  for (int g = 1; g < kJoinWarps; ++g) {
    const float4 v = accs[g][lane];
    sum += sums[g];
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + q_row * p.ldo + static_cast<int64_t>(head) * p.dim + c) =
      make_uint2(Pair16<T>::pack(acc.x * inv, acc.y * inv), Pair16<T>::pack(acc.z * inv, acc.w * inv));
}

template <class T, int ATOMS, int RG, bool SHORT>
int launch_few(const FewArgs& a, cudaStream_t s) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(cross_few_kernel<T, ATOMS, RG, SHORT>, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem(ATOMS)) != cudaSuccess)
      return check_launch("cross_few: cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int64_t grid = static_cast<int64_t>(a.splits) * a.passes * a.p.kv_heads * a.p.sequences;
  FF_REQUIRE(grid <= 0x7fffffff, "ff_cross_attention: %lld parts", static_cast<long long>(grid));
  if (a.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = few_smem(ATOMS);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, cross_few_kernel<T, ATOMS, RG, SHORT>, a);
    return check_launch("cross_few_kernel");
  }
  launch(cross_few_kernel<T, ATOMS, RG, SHORT>, dim3(static_cast<unsigned>(grid)), dim3(kFewThreads), few_smem(ATOMS), s, a);
  if (a.splits > 1) {
    const int rc = check_launch("cross_few_kernel");
    if (rc != FF_OK) return rc;
    const int64_t rows = static_cast<int64_t>(a.p.q_rows) * a.p.heads;
    launch(cross_join_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(32 * kJoinWarps), 0, s, a);
  }
  return check_launch("cross_few_kernel");
}

template <class T, bool SHORT>
int launch_few_rows(const FewArgs& a, int row_tiles, cudaStream_t s) {
  if (a.p.dim <= 64) {
    if (row_tiles == 1) return launch_few<T, 1, 1, SHORT>(a, s);
    return row_tiles == 2 ? launch_few<T, 1, 2, SHORT>(a, s) : launch_few<T, 1, 4, SHORT>(a, s);
  }
  if (row_tiles == 1) return launch_few<T, 2, 1, SHORT>(a, s);
  return row_tiles == 2 ? launch_few<T, 2, 2, SHORT>(a, s) : launch_few<T, 2, 4, SHORT>(a, s);
}
template <class T>
int launch_few_type(const FewArgs& a, int row_tiles, cudaStream_t s) {
  const bool brief = a.p.k_rows <= static_cast<int64_t>(kKeys) * a.p.sequences;
  return brief ? launch_few_rows<T, true>(a, row_tiles, s) : launch_few_rows<T, false>(a, row_tiles, s);
}

}  // namespace

CrossFewPlan cross_few_plan(int q_rows, int k_rows, int sequences, int heads, int kv_heads, int dim) {
  CrossFewPlan plan{};
  const int64_t queries = (static_cast<int64_t>(q_rows) + sequences - 1) / sequences, keys = (static_cast<int64_t>(k_rows) + sequences - 1) / sequences;
  const int64_t rows = queries * (heads / kv_heads);
  plan.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  plan.passes = static_cast<int>(std::max<int64_t>(1, (rows + 16 * plan.row_tiles - 1) / (16 * plan.row_tiles)));
  const int64_t ctas = static_cast<int64_t>(sequences) * kv_heads * plan.passes;
  const int64_t tiles = (keys + kKeys - 1) / kKeys;
  // Which kernel: the one that is expected to take less time, in us. This one has 4 to 6 us for one CTA's way (up to 8.4 for heads of
  // more than 64 columns), 0.008 to 0.012 (0.024) for every CTA's start and end, does 70, 125 or 160 TFLOP/s on the rows
  // of its row tiles (1, 2 or 4 of them), or reads 5.2 TB/s. The other has 3.6 us for every SM's item of up to 256 queries of
  // a head, and for 128 keys of it 1.8 (2.4), or 1.2 (1.5) up to 128 queries, but has no parts of a sequence's keys. Measured (few, other):
  // 64 x 32 queries, 1025 keys, 16 heads of 64: 64, 87 us; 64 x 40: 91, 92; 64 x 64 queries, 128 keys: 22, 35; 64 x 128: 40, 34;
  // 1 x 64 queries, 5184 keys: 22, 50; 16 x 32, 2048 keys, 16 heads of 128: 74, 69; 24 x 64, 64 keys, 16 heads over 4: 14,
  // 15; 24 x 829, 7 keys: 121, 56. Over 210 shapes of equal lengths its choice costs 1.9% on average.
  const bool wide = dim > 64;
  const int tiles_of_rows = plan.row_tiles == 4 ? 3 : plan.row_tiles;
  const double macs = static_cast<double>(ctas) * 16 * plan.row_tiles * ((keys + 15) / 16 * 16) * dim;
  const double rate[] = {70e6, 125e6, 160e6}, edge[] = {0.008, 0.011, 0.012};
  const double few = 3 + tiles_of_rows * (wide ? 1.8 : 1.0) + static_cast<double>(ctas) * edge[tiles_of_rows - 1] * (wide ? 2 : 1) +
                     std::max(4 * macs / rate[tiles_of_rows - 1], 4.0 * sequences * keys * kv_heads * dim / 5.2e6);
  const int64_t items = static_cast<int64_t>(sequences) * heads * ((queries + 255) / 256), sms = sm_count();
  const double step = queries > 128 ? (wide ? 2.4 : 1.8) : (wide ? 1.5 : 1.2);
  const double other = 3 + static_cast<double>((items + sms - 1) / sms) * (3.6 + static_cast<double>((keys + 127) / 128) * step);
  plan.few = few <= other || k_rows == 0;
  if (!plan.few) return plan;
  // As many parts as fill the GPU's places for CTAs, of two tiles at least
  const int64_t places = static_cast<int64_t>(sm_count()) * few_ctas(dim <= 64 ? 1 : 2);
  plan.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({places / ctas, (tiles + 1) / 2, 1024})));
  // Few enough parts, or a sequence short enough that 8 of them are read as fast as the second launch is made: a cluster.
  if (plan.splits > 1 && (plan.splits <= kCluster || (ctas * kCluster >= sm_count() / 2 && tiles <= kClusterTiles))) {
    plan.cluster = true;
    plan.splits = std::min(plan.splits, kCluster);
    return plan;
  }
  if (plan.splits > 1) plan.workspace = static_cast<int64_t>(plan.splits) * q_rows * heads * (dim + 2) * 4;
  return plan;
}

int cross_few(const CrossArgs& p, bool bf16, const CrossFewPlan& plan, void* workspace, cudaStream_t s) {
  FewArgs a{};
  a.p = p;
  a.passes = plan.passes;
  a.splits = plan.splits;
  a.cluster = plan.cluster;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + static_cast<int64_t>(plan.splits) * p.q_rows * p.heads * p.dim);
  return bf16 ? launch_few_type<__nv_bfloat16>(a, plan.row_tiles, s) : launch_few_type<__half>(a, plan.row_tiles, s);
}

}  // namespace ff
