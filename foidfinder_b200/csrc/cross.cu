// ff_cross_attention: checks, and which kernel takes the call.
#include "common.h"
#include "cross.h"

using namespace ff;

extern "C" int64_t ff_cross_attention_workspace_bytes(int q_rows, int k_rows, int sequences, int heads, int kv_heads, int head_dim) {
  if (q_rows < 1 || k_rows < 0 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || head_dim < 1) return 0;
  return cross_few_plan(q_rows, k_rows, sequences, heads, kv_heads, head_dim).workspace;
}

extern "C" int ff_cross_attention(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* out,
                                  int64_t ldo, int dtype, int q_rows, int k_rows, int sequences, const int32_t* q_start,
                                  const int32_t* k_start, const int32_t* k_len, const uint8_t* mask, int heads, int kv_heads,
                                  int head_dim, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  FF_REQUIRE(dtype == FF_F16 || dtype == FF_BF16, "ff_cross_attention: type %d is not fp16 or bf16", dtype);
  FF_REQUIRE(heads >= 1 && heads <= 1024 && kv_heads >= 1 && heads % kv_heads == 0,
             "ff_cross_attention: %d query heads do not divide into %d key heads", heads, kv_heads);
  FF_REQUIRE(head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0, "ff_cross_attention: head_dim %d is not a multiple of 16 up to 128",
             head_dim);
  FF_REQUIRE(q_rows >= 0 && q_rows <= (1 << 30) && k_rows >= 0 && k_rows <= (1 << 30) && sequences >= 0 && sequences <= (1 << 24),
             "ff_cross_attention: bad shape q_rows=%d k_rows=%d sequences=%d", q_rows, k_rows, sequences);
  FF_REQUIRE(static_cast<int64_t>(q_rows) * (heads / kv_heads) <= (1 << 30), "ff_cross_attention: %d queries of %d heads for each key head", q_rows,
             heads / kv_heads);
  FF_REQUIRE(scale > 0.f && scale <= 1e30f, "ff_cross_attention: scale must be positive");
  if (q_rows == 0 || sequences == 0) return FF_OK;
  FF_REQUIRE(q_start != nullptr || q_rows % sequences == 0, "ff_cross_attention: %d queries are not %d equal pieces", q_rows, sequences);
  FF_REQUIRE(k_start != nullptr || k_rows % sequences == 0, "ff_cross_attention: %d keys are not %d equal pieces", k_rows, sequences);
  FF_REQUIRE(q && out && (k_rows == 0 || (k && v)), "ff_cross_attention: NULL pointer");
  FF_REQUIRE(out != q && out != k && out != v, "ff_cross_attention: out must not be an input");
  FF_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "ff_cross_attention: q, k, v and out must be 16-byte aligned");
  auto words = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; };
  FF_REQUIRE(words(q_start) && words(k_start) && words(k_len), "ff_cross_attention: misaligned starts or lengths");
  const int64_t qc = static_cast<int64_t>(heads) * head_dim, kc = static_cast<int64_t>(kv_heads) * head_dim;
  auto stride = [](int64_t ld, int64_t cols, int rows) { return rows <= 1 || (ld >= cols && ld % 8 == 0); };
  FF_REQUIRE(stride(ldq, qc, q_rows) && stride(ldo, qc, q_rows) && stride(ldk, kc, k_rows) && stride(ldv, kc, k_rows),
             "ff_cross_attention: row strides %lld, %lld, %lld and %lld must hold %lld and %lld columns and be multiples of 8",
             static_cast<long long>(ldq), static_cast<long long>(ldk), static_cast<long long>(ldv), static_cast<long long>(ldo),
             static_cast<long long>(qc), static_cast<long long>(kc));
  const CrossFewPlan plan = cross_few_plan(q_rows, k_rows, sequences, heads, kv_heads, head_dim);
  FF_REQUIRE(plan.workspace == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= plan.workspace),
             "ff_cross_attention: a workspace of %lld bytes, 16-byte aligned, is needed", static_cast<long long>(plan.workspace));
  const CrossArgs a{q,       ldq,     k,     ldk,  v,     ldv,      out,      ldo, q_rows, k_rows, sequences, q_start,
                    k_start, k_len,   mask,  heads, kv_heads, head_dim, scale * 1.4426950408889634f};
  if (!plan.few) return cross_tc(a, dtype == FF_BF16, static_cast<cudaStream_t>(stream));
  return cross_few(a, dtype == FF_BF16, plan, workspace, static_cast<cudaStream_t>(stream));
}
