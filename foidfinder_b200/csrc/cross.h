// What the two kernels of ff_cross_attention share (cross_few.cu: few queries per sequence, bound by reading keys and
// values; cross_tc.cu: many, on the 5th-generation tensor cores).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "foidfinder_b200.h"

namespace ff {

struct CrossArgs {
  const void* q;
  int64_t ldq;
  const void* k;
  int64_t ldk;
  const void* v;
  int64_t ldv;
  void* out;
  int64_t ldo;
  int q_rows, k_rows, sequences;
  const int *q_start, *k_start, *k_len;
  const uint8_t* mask;
  int heads, kv_heads, dim;
  float scale_log2;  // scale * log2(e): the softmax is taken in powers of two
};

#ifdef __CUDACC__
// Rows [at, at + n) of a sequence, whatever the starts hold: always rows that there are.
struct Piece {
  int at, n;
};
__device__ __forceinline__ Piece piece(const int* start, int rows, int sequences, int b) {
  if (start == nullptr) {
    const int n = rows / sequences;
    return {b * n, n};
  }
  const int s = min(max(__ldg(start + b), 0), rows);
  return {s, min(max(__ldg(start + b + 1), s), rows) - s};
}
__device__ __forceinline__ Piece query_piece(const CrossArgs& a, int b) { return piece(a.q_start, a.q_rows, a.sequences, b); }
__device__ __forceinline__ Piece key_piece(const CrossArgs& a, int b) {
  Piece p = piece(a.k_start, a.k_rows, a.sequences, b);
  if (a.k_len != nullptr) p.n = min(p.n, max(__ldg(a.k_len + b), 0));
  return p;
}
#endif

// Few queries per sequence. splits: parts of every sequence's keys that CTAs of their own work on (their results are
// joined within a cluster, or by a second kernel through the workspace).
struct CrossFewPlan {
  bool few;  // whether this kernel takes the call
  bool cluster;  // the splits of a sequence are a cluster
  int row_tiles, passes, splits;
  int64_t workspace;
};
CrossFewPlan cross_few_plan(int q_rows, int k_rows, int sequences, int heads, int kv_heads, int dim);
int cross_few(const CrossArgs& a, bool bf16, const CrossFewPlan& plan, void* workspace, cudaStream_t s);

// Many queries per sequence.
int cross_tc(const CrossArgs& a, bool bf16, cudaStream_t s);

}  // namespace ff
