// What the two attention kernels over the 4-bit cache share: how the keys of a position are split.
#pragma once

#include <algorithm>

#include "q4_cache.hpp"

// length class of a position, and keys per CTA of a class
__host__ __device__ constexpr int qa_class(int64_t pos) {
  return pos < 1024 ? 0 : (pos < 4096 ? 1 : (pos < 131072 ? 2 : 3));
}
__host__ __device__ constexpr int64_t qa_class_end(int cl) {
  return cl == 0 ? 1024 : (cl == 1 ? 4096 : (cl == 2 ? 131072 : (1ll << 40)));
}
__host__ __device__ constexpr int qa_cta_keys(int cl) { return cl == 0 ? 128 : (cl == 1 ? 256 : (cl == 2 ? 1024 : 4096)); }
// The classes from QA_TC_CLASS on are the tensor-core kernel's where the call has more than QA_FEW_ROWS rows
// (tokens times query heads) a kv head.
constexpr int QA_TC_CLASS = 2;
constexpr int QA_FEW_ROWS = 64;
// partial results of one row for lengths up to bound
inline int qa_slots(int64_t bound) {
  int n = 1;
  for (int cl = 0; cl < 4; ++cl) {
    const int64_t end = std::min(bound, qa_class_end(cl));
    n = std::max<int64_t>(n, (end + qa_cta_keys(cl) - 1) / qa_cta_keys(cl));
    if (bound <= qa_class_end(cl)) break;
  }
  return n;
}

// A row's sums are taken relative to 2^m; m moves up only when a score passes it by more than this (in
// powers of two), as moving it costs a product per output. Sums in fp32 and probabilities in bf16 keep
// their relative accuracy below 2^8.
constexpr float QA_SLACK = 8.f;

// 2^x to two units in the last place, 0 below 2^-126
__device__ __forceinline__ float qa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// whether one of the bf16 scales of a pair is NaN (scales are at most 2^120: only a NaN's exponent
// carries into the sign bit)
__device__ __forceinline__ uint32_t qa_scales_nan(uint32_t s2) { return (s2 + 0x00800080u) & 0x80008000u; }

// The classes from QA_TC_CLASS on, bf16 queries, head_dim 128: partial results of tc tokens from t0 on, prows
// rows a head in the workspace.
int launch_q4_attn_tc(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, int grp, int t0, int tc, int prows,
                      float scale_log2, int nslots, int q_vec, float* part_o, float2* part_s, cudaStream_t st, bool pdl);
