// What the two tensor-core kernels of cross attention share (cross_tc.cu: heads of more than 64 columns; cross_tc64.cu: up to 64).
#pragma once
#include <type_traits>

#include "common.h"
#include "cross.h"
#include "fp4.cuh"

namespace ff {

constexpr int kBQ = 128;          // queries of a tile
constexpr int kAtom = 128 * 128;  // bytes: 128 rows of 64 columns, 128-byte swizzle
constexpr int kTable = 16;        // items of a CTA that are looked up ahead, all at once
constexpr float kGrowth = 8.f;    // powers of two by which the maximum may grow before O is rescaled
// P = 2^(x + kUp), at most 2^8 more. In fp16 up to 2^15, so that weights far below the largest are still normal numbers; in bf16 up to
// 2^-20, so that sums over 2^20 values next to the type's largest stay in f32's range.
template <class T>
constexpr float kUp = std::is_same<T, __half>::value ? 7.f : -28.f;

struct TcArgs {
  CrossArgs p;
  int tiles_per_seq;  // equal pieces: items of 256 queries per sequence and head; 0: by q_start
  int64_t items;
  bool by_cost;  // an item per CTA, by item_by_cost
  int* err;
};

// Up to 256 queries [q, q + nq) of a head against the keys [k, k + nk).
struct Item {
  int q, nq, k, nk;
};

// Tensor maps of q, k and v: boxes of 64 columns and 128 queries or key_rows keys.
int cross_maps(const CrossArgs& p, bool bf16, int key_rows, CUtensorMap (&maps)[3]);
int cross_tc64(const TcArgs& a, bool bf16, int grid, cudaStream_t s);

// Value tile as MN-major operand: key rows of 128 bytes (64 columns), 8-row groups 1024 bytes apart, the next 64 columns an atom
// further.
__device__ __forceinline__ uint64_t sdesc_v(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(kAtom >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Item `n` of this CTA (nq == 0: none). Head fastest, then the 256-query tiles of a sequence. By q_start, tile t of
// sequence b is slot q_start[b] / 256 + b + t: slots of sequences do not overlap, and the one that holds a slot is found by halving.
static __device__ Item item_at(const TcArgs& a, int64_t it) {
  const CrossArgs& p = a.p;
  const int slot = static_cast<int>(it / p.heads);
  int b, tile;
  if (a.tiles_per_seq > 0) {
    b = slot / a.tiles_per_seq;
    tile = slot - b * a.tiles_per_seq;
  } else {
    auto first = [&](int i) { return min(max(__ldg(p.q_start + i), 0), p.q_rows) / 256 + i; };
    int lo = 0, hi = p.sequences - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first(mid) <= slot) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    tile = slot - first(b);
  }
  const Piece q = query_piece(p, b);
  Item r{0, 0, 0, 0};
  if (tile < 0 || static_cast<int64_t>(tile) * 256 >= q.n) return r;
  r.q = q.at + tile * 256;
  r.nq = min(256, q.n - tile * 256);
  const Piece k = key_piece(p, b);
  r.k = k.at;
  r.nk = k.n;
  return r;
}

// The item of a CTA that has one, or none: sequences in falling order of their keys (half of these for up to 128 queries), so
// that no long item starts when the others are about to end. By all threads, for at most one sequence each; `cost` has
// room for all sequences and is left to the asynchronous copies.
static __device__ Item item_by_cost(const TcArgs& a, int2* cost, Item* found) {
  const int i = threadIdx.x, n = a.p.sequences;
  Piece q{0, 0}, k{0, 0};
  int2 mine = make_int2(0, 0);  // cost, items
  if (i < n) {
    q = query_piece(a.p, i);
    k = key_piece(a.p, i);
    mine = make_int2(q.n > kBQ ? k.n : (k.n + 1) / 2, (q.n + 255) / 256);
    cost[i] = mine;
  }
  if (i == 0) *found = Item{0, 0, 0, 0};
  __syncthreads();
  if (i < n) {
    int tile = static_cast<int>(blockIdx.x / static_cast<uint32_t>(a.p.heads));
    for (int j = 0; j < n; ++j) {
      const int2 other = cost[j];
      if (other.x > mine.x || (other.x == mine.x && j < i)) tile -= other.y;
    }
    if (tile >= 0 && tile < mine.y) *found = Item{q.at + tile * 256, min(256, q.n - tile * 256), k.at, k.n};
  }
  fence_async_smem();
  __syncthreads();
  return *found;
}

// 2^-n of a whole n >= 0, exactly (0 where f32 has no normal number for it).
__device__ __forceinline__ float power_below(float n) { return n < 127.f ? __uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(n)) << 23) : 0.f; }

// What a query's weights are relative to: P = 2^((s - ref) scale + shift). ref is 0 and shift a whole number, but for scores
// beyond 2^20 powers of two: their fractions would be lost in a shift of that size, so ref is the score itself. The usual
// way through the scores knows no ref: its shift is then such that they all seem to have grown (kSeemsGrown), and what looks
// into that takes ref off them. Where a weight is NaN, so is the result, whatever the maximum: nothing is looked into again.
constexpr float kFarScore = 1048576.f, kSeemsGrown = 3e38f;
struct Maximum {
  float ref, shift;
  bool set;  // there has been a key
};
// Whether `top` calls for raising the maximum.
template <class T>
__device__ __forceinline__ bool below(const Maximum& m, float top, float scale_log2) {
  return top > -INFINITY && (!m.set || fmaf(top - m.ref, scale_log2, m.shift) > kUp<T> + kGrowth);
}
// `top` (a score above -inf) becomes the maximum, up to a power of two. -> What all before has to be scaled by: a whole
// power of two, or nothing of it is left (2^-512 of P is no number of 32 bits; without a maximum there was no key).
template <class T>
__device__ __forceinline__ float raise(Maximum& m, float top, float scale_log2) {
  const float x = fmaf(top - m.ref, scale_log2, m.shift), up = floorf(x - kUp<T>), at = top * scale_log2;
  const bool far = !(fabsf(at) < kFarScore);
  if (m.set && up < 512.f) {
    m.shift = far ? x - up : m.shift - up;
    if (far) m.ref = top;
    return power_below(up);
  }
  m = {far ? top : 0.f, far ? kUp<T> : kUp<T> - floorf(at), true};
  return 0.f;
}
// Powers of two by which a's maximum is above b's.
__device__ __forceinline__ float above(const Maximum& a, const Maximum& b, float scale_log2) {
  return fmaf(a.ref - b.ref, scale_log2, b.shift - a.shift);
}
template <int N>
__device__ __forceinline__ float largest(const uint32_t (&s)[N]) {
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < N; e += 2) top[(e >> 1) & 1] = max3(top[(e >> 1) & 1], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
  return fmaxf(top[0], top[1]);
}

// O (dim TMEM columns from `to`) scaled by corr; out of line, it is rare.
static __device__ __noinline__ void rescale(uint32_t to, int dim, float corr) {
  for (int c = 0; c < dim; c += 16) {
    uint32_t o[16];
    tmem_ld16(to + c, o);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
    tmem_st16(to + c, o);
  }
}

// 16 columns of a row of the result. One store of 32 bytes, where they start at one: two of 16 would each write half a sector.
static __device__ __forceinline__ void store_columns(void* out, const uint32_t (&w)[8]) {
  if ((reinterpret_cast<uintptr_t>(out) & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    static_cast<uint4*>(out)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(out)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Walks the items of a CTA. next(): the next one with queries (and, WORK, with keys).
struct Items {
  const TcArgs& a;
  const Item* table;
  int n = -1, head = 0;
  template <bool WORK>
  __device__ __forceinline__ bool next(Item& item) {
    for (++n;; ++n) {
      const int64_t it = blockIdx.x + static_cast<int64_t>(n) * gridDim.x;
      if (it >= a.items) return false;
      item = n < kTable ? table[n] : item_at(a, it);
      head = static_cast<int>(it % a.p.heads);
      if (item.nq > 0 && (!WORK || item.nk > 0)) return true;
    }
  }
};

}  // namespace ff
