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
// Positions from QA_TC_BEGIN on are the tensor-core kernel's where the call has more than QA_FEW_ROWS rows (tokens
// times query heads) a kv head.  It has classes of its own, with a slot of keys per CTA: with 2,048 keys instead
// of 1,024, 16 rows of 13 tokens at up to 16,384 keys took 220 us instead of 196, but 1,024 tokens behind 32,768
// keys (64 / 8 heads) 2,076 instead of 2,640 (with probabilities in one bf16 part).
constexpr int QA_FEW_ROWS = 64;
constexpr int QA_TC_BEGIN = 4096;
// Which kernel takes them: as the call's rows say, or one of the two whatever the rows.
enum class QaLong { BY_ROWS, ROW_TILES, TENSOR_CORE };
constexpr int QA_TC_CLASSES = 3;
__host__ __device__ constexpr int qa_tc_class(int64_t pos) { return pos < 16384 ? 0 : (pos < 65536 ? 1 : 2); }
__host__ __device__ constexpr int qa_tc_class_begin(int cl) { return cl == 0 ? QA_TC_BEGIN : (cl == 1 ? 16384 : 65536); }
__host__ __device__ constexpr int64_t qa_tc_class_end(int cl) {
  return cl == 0 ? 16384 : (cl == 1 ? 65536 : (1ll << 40));
}
__host__ __device__ constexpr int qa_tc_keys(int cl) { return cl == 0 ? 1024 : (cl == 1 ? 2048 : 4096); }
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

inline int qa_tc_slots(int64_t bound) {
  int n = qa_slots(std::min<int64_t>(bound, QA_TC_BEGIN));
  for (int cl = 0; cl < QA_TC_CLASSES && bound > qa_tc_class_begin(cl); ++cl)
    n = std::max<int64_t>(n, (std::min(bound, qa_tc_class_end(cl)) + qa_tc_keys(cl) - 1) / qa_tc_keys(cl));
  return n;
}

// Online softmax (Milakov and Gimelshein, 2018): a row's sums are taken relative to 2^m; m moves up only when a
// score passes it by more than this (in powers of two), as moving it costs a product per output.  Sums in fp32 and
// probabilities in two bf16 parts keep their relative accuracy below 2^8.
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

// The positions from QA_TC_BEGIN on, bf16 queries, head_dim 128: partial results of tc tokens from t0 on, prows
// rows a head in the workspace.
int launch_q4_attn_tc(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, int grp, int t0, int tc, int prows,
                      float scale_log2, int nslots, int q_vec, float* part_o, float2* part_s, cudaStream_t st, bool pdl);
