// Causal attention of new tokens over the paged 4-bit KV cache, grouped heads, rows of different
// lengths: out = softmax(scale q . K) V over the keys 0 .. P of a token at position P.
//
// Split-KV. A warp takes a unit of consecutive keys for a tile of 16 query rows (a row is one token
// of one query head of the kv head) and runs an online softmax over it; the four units of a CTA are
// folded in order, and a second kernel folds the CTAs' partial results in order.  The unit's length
// depends on the row's own position alone (32 keys below 1,024, 64 below 4,096, 256 below 131,072, else
// 1,024), so a token's result does not depend on what else is in the call: verify blocks and single
// steps agree bit for bit.  (Calls of more than 64 rows a kv head, and a model's prompts, leave positions from
// 4,096 on to q4_attention_tc.cu, where a token's result does not depend on the others either.)  Short units give
// few keys to many CTAs; from 131,072 keys on there are enough of them, and longer ones spare partial
// results (440 us instead of 479 at 262,144 keys, then).
//
// Keys and values are decoded in the registers that the products read them from, with no rounding
// between codes and product.  What it takes: 1,116 warp instructions per 32 keys and row tile (384 the
// decode, 96 products), 0.52 issued a clock and scheduler: three warps a scheduler (168 registers) wait for their own
// products, exponentials and loads.  bf16, 32 heads of 128, 13 tokens: 144 us at 65,536 keys (2.1 TB/s of codes and
// scales; floor 46 us), 477 us at 262,144 (2.5 TB/s).
#include <math_constants.h>

#include <algorithm>
#include <cmath>

#include "internal.hpp"
#include "q4.cuh"
#include "q4_attention.hpp"

namespace {

constexpr int QA_WARPS = 4;
constexpr int QA_THREADS = 32 * QA_WARPS;
constexpr int QA_ROWS = 16;
constexpr int QA_CLUSTER = 8;  // slots that one cluster folds: contexts of up to 2,048 keys
constexpr int NS = 2;           // 16-key chunks per online-softmax step of a warp
constexpr int QA_STEP = 16 * NS;

template <int NW>
__device__ __forceinline__ void ld_words(uint32_t (&w)[NW], const uint8_t* p) {
  if constexpr (NW == 4) {
    const uint4 v = q4_ld<uint4>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (NW == 2) {
    const uint2 v = q4_ld<uint2>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = q4_ld<uint32_t>(p);
  }
}

constexpr int qa_parts_q(size_t elem) { return elem == 2 ? 1 : 3; }  // bf16 parts of a query value
// ... and of a probability.  Two for bf16 queries: a key's weight is then off by at most 2^-18 of itself (two
// roundings to the nearest bf16, 2^-9 of what each is given), as in the attention over the bf16 cache.  One part
// would be off by 2^-9, beside outputs that are rounded by as much once more, and take 130 us instead of 145 at
// 65,536 keys (13 tokens, 32 heads of 128) and 414 instead of 477 at 262,144.
constexpr int qa_parts_p(size_t elem) { return elem == 2 ? 2 : 3; }

// The K codes and scales of 32 keys, as one thread multiplies them: per 16-key chunk two 8-key tiles,
// of which it holds key 4 (g / 2) + g % 2 + 2 u, features c DH / 4 .. + DH / 4 - 1.
template <int DH>
struct KTile {
  uint32_t w[NS][2][DH / 32];
  uint32_t s[NS][2];
};
// The V codes and scales: per 16-key chunk the keys 4 c .. 4 c + 3, features g DH / 8 .. + DH / 8 - 1.
template <int DH>
struct VTile {
  static constexpr int NW = DH / 64 > 0 ? DH / 64 : 1;
  uint32_t w[NS][4][NW];
  uint32_t s[NS][2];
};

// floats of the staged queries
template <typename T, int DH>
__host__ __device__ constexpr int qa_q_floats() {
  return qa_parts_q(sizeof(T)) * 2 * (DH / 32) * 32 * 4;
}

// One CTA's keys for one tile of 16 rows.  FUSED: each row's result goes into the shared memory of the CTA
// of the cluster that folds it, else to the CTA's slot of the workspace.  Classes above top are another kernel's.
template <typename T, int DH, bool FUSED>
__device__ __forceinline__ void attn_tile(float* qa_sm, const Q4CacheDev& cache, const Q4RowsDev& rows, const Q4Tensor& q,
                                          int grp, int t0, int tc, int tiles, float scale_log2, int nslots, bool q_vec,
                                          int top, float* __restrict__ part_o, float2* __restrict__ part_s) {
  constexpr int NQ = qa_parts_q(sizeof(T)), NP = qa_parts_p(sizeof(T));
  constexpr int KW = DH / 32;  // code words per thread and key (K)
  constexpr int VN = DH / 8;   // 8-feature tiles of the output
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.y / tiles, tile = blockIdx.y % tiles, b = blockIdx.z;
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
    return;
  }
  const int first = t0 + tile * QA_ROWS / grp;
  const int last = min(min(t0 + (tile * QA_ROWS + QA_ROWS - 1) / grp, t0 + tc - 1), count - 1);
  if (first > last) return;
  const int pmin = len + first, pmax = len + last;
  const int cl0 = qa_class(pmin), cl1 = min(qa_class(pmax), top);
  if (cl1 < cl0 || static_cast<int64_t>(blockIdx.x) * qa_cta_keys(cl0) > pmax) return;

  // Queries as product operands: step 2 w covers the feature pairs (0,4) (1,5) of the word 8 w ..,
  // step 2 w + 1 the pairs (2,6) (3,7), as q4_word decodes the keys; qs[part][step][lane].
  uint4* qs = reinterpret_cast<uint4*>(qa_sm);
  if (threadIdx.x < 32 * KW) {
    uint32_t e[2][8][3];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = tile * QA_ROWS + g + 8 * h, t = t0 + r / grp;
      float qv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) qv[j] = 0.f;
      if (r < tc * grp && t < count)
        q4_load8<T>(qv,
                    static_cast<const T*>(q.p) + b * q.sb + t * q.st + (kvh * grp + r % grp) * q.sh + c * (DH / 4) + 8 * warp,
                    q_vec);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (NQ == 1)
          e[h][j][0] = __float_as_uint(qv[j]) >> 16;
        else
          q4_parts(qv[j], e[h][j]);
      }
    }
#pragma unroll
    for (int p = 0; p < NQ; ++p)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        qs[(p * 2 * KW + 2 * warp + s) * 32 + lane] =
            make_uint4(e[0][2 * s][p] | e[0][2 * s + 4][p] << 16, e[1][2 * s][p] | e[1][2 * s + 4][p] << 16,
                       e[0][2 * s + 1][p] | e[0][2 * s + 5][p] << 16, e[1][2 * s + 1][p] | e[1][2 * s + 5][p] << 16);
  }
  __syncthreads();

  const int32_t* table = rows.table + b * rows.table_stride;
  const int P = cache.P;
  // byte offsets inside a block: this thread's K features and scale group, V features and scale group
  const uint32_t k_off = c * (DH / 8) + (4 * (g >> 1) + (g & 1)) * (DH / 2);
  const uint32_t ks_off = P * DH + 2 * ((c * (DH / 4) / 32) * P + 4 * (g >> 1) + (g & 1));
  const uint32_t v_off = P * (DH / 2) + g * (DH / 16) + 4 * c * (DH / 2);
  const uint32_t vs_off = P * DH + P * (DH / 16) + 2 * ((g * (DH / 8) / 32) * P + 4 * c);
  const uint8_t* head_base = cache.block(0, kvh);
  const size_t page_bytes = static_cast<size_t>(cache.G) * cache.block_bytes;

  for (int cl = cl0; cl <= cl1; ++cl) {
    const int kall = static_cast<int>(min(static_cast<int64_t>(pmax), qa_class_end(cl) - 1)) + 1;  // keys of the class
    const int unit = qa_cta_keys(cl) / QA_WARPS;
    if (static_cast<int64_t>(blockIdx.x) * qa_cta_keys(cl) >= kall) continue;
    const int kbeg = blockIdx.x * qa_cta_keys(cl) + warp * unit, kend = min(kall, kbeg + unit);
    // keys that every row of the class sees need no mask; rows of no token (or another class) take
    // part unmasked, their results are dropped
    const int clear = max(pmin, cl == 0 ? 0 : static_cast<int>(qa_class_end(cl - 1))) + 1;
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = tile * QA_ROWS + g + 8 * i, t = t0 + r / grp;
      lim[i] = r < tc * grp && t < count && qa_class(len + t) == cl ? len + t : INT32_MAX;
    }

    float o[VN][4], m[2], l[2];
#pragma unroll
    for (int n = 0; n < VN; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) m[i] = -CUDART_INF_F, l[i] = 0.f;

    // Pages: lane i holds the page id of the 16-key chunk 32 j + i of the unit (j: the last load);
    // the slot of a chunk inside its page goes along.
    int page_of = -1;
    auto load_pages = [&](int key) {
      const int kk = key + 16 * lane;
      page_of = kk < kend ? table[kk / P] : -1;
    };
    auto page_at = [&](int key, int sub) { return __shfl_sync(0xffffffffu, page_of, (((key - kbeg) >> 4) + sub) & 31); };
    KTile<DH> kt;
    VTile<DH> vt;
    bool bad = false;
    // pages of the step that the next V load reads, and of the step after
    int vpage[NS], kpage[NS], slot[NS];
    auto next_slot = [&](int s) { return s + 16 == P ? 0 : s + 16; };
    auto load_k = [&](int key) {
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) {
        const int id = kpage[sub];
        const bool in = key + 16 * sub < kend;
        if (in && static_cast<uint32_t>(id) < static_cast<uint32_t>(cache.pages)) {
          const uint8_t* blk = head_base + id * page_bytes;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            ld_words<KW>(kt.w[sub][u], blk + (k_off + (slot[sub] + 2 * u) * (DH / 2)));
            kt.s[sub][u] = q4_ld<uint16_t>(blk + (ks_off + 2 * (slot[sub] + 2 * u)));
          }
        } else {
          bad |= in;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int w = 0; w < KW; ++w) kt.w[sub][u][w] = 0u;
            kt.s[sub][u] = 0x7FC0u;  // keys without a page: a NaN score for whoever sees them
          }
        }
      }
    };
    auto load_v = [&](int key) {
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) {
        const int id = vpage[sub];
        if (key + 16 * sub < kend && static_cast<uint32_t>(id) < static_cast<uint32_t>(cache.pages)) {
          const uint8_t* blk = head_base + id * page_bytes;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint8_t* p = blk + (v_off + (slot[sub] + j) * (DH / 2));
            if constexpr (DH == 32)
              vt.w[sub][j][0] = q4_ld<uint16_t>(p);
            else
              ld_words<VTile<DH>::NW>(vt.w[sub][j], p);
          }
          const uint2 s = q4_ld<uint2>(blk + (vs_off + 2 * slot[sub]));
          vt.s[sub][0] = s.x, vt.s[sub][1] = s.y;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int w = 0; w < VTile<DH>::NW; ++w) vt.w[sub][j][w] = 0u;
          vt.s[sub][0] = vt.s[sub][1] = 0u;
        }
      }
    };

    if (kbeg < kend) {
      load_pages(kbeg);
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) {
        slot[sub] = sub == 0 ? kbeg % P : next_slot(slot[sub - 1]);
        kpage[sub] = page_at(kbeg, sub);
      }
      load_k(kbeg);
    }
    for (int key = kbeg; key < kend; key += QA_STEP) {
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) vpage[sub] = kpage[sub];
      load_v(key);
      float s[NS][2][4];
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[sub][u][0] = s[sub][u][1] = s[sub][u][2] = s[sub][u][3] = 0.f;
      Q4Scale ks[NS][2];
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int u = 0; u < 2; ++u) ks[sub][u] = q4_scale(kt.s[sub][u] | kt.s[sub][u] << 16);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        uint32_t kv[NS][2][4];
#pragma unroll
        for (int sub = 0; sub < NS; ++sub)
#pragma unroll
          for (int u = 0; u < 2; ++u) q4_word(kt.w[sub][u][w], ks[sub][u], kv[sub][u]);
#pragma unroll
        for (int p = NQ - 1; p >= 0; --p)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 a = qs[(p * 2 * KW + 2 * w + h) * 32 + lane];
#pragma unroll
            for (int sub = 0; sub < NS; ++sub)
#pragma unroll
              for (int u = 0; u < 2; ++u)
                q4_mma(s[sub][u], a.x, a.y, a.z, a.w, kv[sub][u][2 * h], kv[sub][u][2 * h + 1]);
          }
      }
      const int next = key + QA_STEP;
      if (next < kend) {
        if (((next - kbeg) & 511) == 0) load_pages(next);
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) {
          slot[sub] = next_slot(slot[sub == 0 ? NS - 1 : sub - 1]);
          kpage[sub] = page_at(next, sub);
        }
        load_k(next);
      }
      const bool masked = key + QA_STEP > clear;
      if (masked) {  // thread's keys of a chunk are 4 c + 2 u + (0, 1)
#pragma unroll
        for (int sub = 0; sub < NS; ++sub)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key + 16 * sub + 4 * c + 2 * u + (e & 1) > lim[e >> 1]) s[sub][u][e] = -CUDART_INF_F;
      }
      float mx[2], a[2] = {1.f, 1.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) mx[i] = m[i];
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[sub][u][e]);
      bool moved = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        const float grow = (mx[i] - m[i]) * scale_log2;  // NaN while nothing is visible
        if (grow > QA_SLACK) {
          moved = true;
          a[i] = qa_ex2(-grow);
          m[i] = mx[i];
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[i] *= a[i];
#pragma unroll
          for (int n = 0; n < VN; ++n) {
            o[n][2 * i] *= a[i];
            o[n][2 * i + 1] *= a[i];
          }
        }
      }
      float mu[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) mu[i] = m[i] == -CUDART_INF_F ? 0.f : -m[i] * scale_log2;
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) {
        // probabilities as bf16 parts: keys (4 c, 4 c + 1) of rows g, g + 8, then (4 c + 2, 4 c + 3)
        uint32_t pa[NP][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = qa_ex2(fmaf(s[sub][u][2 * i], scale_log2, mu[i]));
            const float p1 = qa_ex2(fmaf(s[sub][u][2 * i + 1], scale_log2, mu[i]));
            l[i] += p0 + p1;
            float r0 = p0, r1 = p1;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(r0, r1);
              pa[p][2 * u + i] = *reinterpret_cast<const uint32_t*>(&h);
              if (p + 1 < NP) {
                r0 -= __low2float(h);
                r1 -= __high2float(h);
              }
            }
          }
        uint32_t vs[2] = {vt.s[sub][0], vt.s[sub][1]};
        if (masked) {
          // keys behind the last visible one hold whatever the page held: their scale becomes 0
          const int k4 = key + 16 * sub + 4 * c;
          if (k4 >= kend) vs[0] &= 0xFFFF0000u;
          if (k4 + 1 >= kend) vs[0] &= 0x0000FFFFu;
          if (k4 + 2 >= kend) vs[1] &= 0xFFFF0000u;
          if (k4 + 3 >= kend) vs[1] &= 0x0000FFFFu;
        }
        const uint32_t nan0 = qa_scales_nan(vs[0]), nan1 = qa_scales_nan(vs[1]);
        if (__any_sync(0xffffffffu, (nan0 | nan1) != 0u)) {
          // a group held as NaN must not reach rows that do not see its key (0 NaN is NaN): take it
          // out of the product and set the outputs of the rows that see it
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int grp_of = (2 * c + e) * (DH / 8) / 32;
            for (int kk = 0; kk < 16; ++kk) {
              const int src = (kk >> 2) + 4 * ((grp_of * 32) / (DH / 8));  // a lane that holds the group's scale of kk
              const uint32_t w = __shfl_sync(0xffffffffu, vs[0], src), x = __shfl_sync(0xffffffffu, vs[1], src);
              const uint32_t pair = (kk & 2) ? x : w;
              const uint32_t sb = (kk & 1) ? pair >> 16 : pair & 0xFFFFu;
              if ((sb & 0x7F80u) == 0x7F80u) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  if (key + 16 * sub + kk <= lim[i])
#pragma unroll
                    for (int n = 0; n < VN; ++n) o[n][2 * i + e] = CUDART_NAN_F;
              }
            }
          }
          if (nan0 & 0x00008000u) vs[0] &= 0xFFFF0000u;
          if (nan0 & 0x80000000u) vs[0] &= 0x0000FFFFu;
          if (nan1 & 0x00008000u) vs[1] &= 0xFFFF0000u;
          if (nan1 & 0x80000000u) vs[1] &= 0x0000FFFFu;
        }
        const Q4Scale s01 = q4_scale(vs[0]), s23 = q4_scale(vs[1]);
#pragma unroll
        for (int n4 = 0; n4 < VN / 4; ++n4) {
          const int w = n4 >> 1;
          const uint32_t sel = (n4 & 1) ? 0x7632u : 0x5410u;
          uint32_t b01[4], b23[4];
          q4_word(__byte_perm(vt.w[sub][0][w], vt.w[sub][1][w], sel), s01, b01);
          q4_word(__byte_perm(vt.w[sub][2][w], vt.w[sub][3][w], sel), s23, b23);
          // the parts of one output tile apart from each other: a product takes 20 cycles to follow itself
#pragma unroll
          for (int p = NP - 1; p >= 0; --p)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              q4_mma(o[4 * n4 + j], pa[p][0], pa[p][1], pa[p][2], pa[p][3], b01[j], b23[j]);
        }
      }
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // the four units folded in order
    constexpr int LD = DH + 2;
    float* res = qa_sm + qa_q_floats<T, DH>();
    float* mine = res + warp * QA_ROWS * LD;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* row = mine + (g + 8 * i) * LD;
#pragma unroll
      for (int n = 0; n < VN; n += 2) {
        *reinterpret_cast<float2*>(row + 2 * c * VN + n) = make_float2(o[n][2 * i], o[n + 1][2 * i]);
        *reinterpret_cast<float2*>(row + (2 * c + 1) * VN + n) = make_float2(o[n][2 * i + 1], o[n + 1][2 * i + 1]);
      }
      if (c == 0) *reinterpret_cast<float2*>(row + DH) = make_float2(m[i] * scale_log2, l[i]);
    }
    __syncthreads();
    for (int r = warp; r < QA_ROWS; r += QA_WARPS) {
      const int R = tile * QA_ROWS + r, t = t0 + R / grp;
      if (R >= tc * grp || t >= count || qa_class(len + t) != cl) continue;
      float mw[QA_WARPS], big = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < QA_WARPS; ++w) {
        mw[w] = res[(w * QA_ROWS + r) * LD + DH];
        big = fmaxf(big, mw[w]);
      }
      float sum = 0.f, f[QA_WARPS];
#pragma unroll
      for (int w = 0; w < QA_WARPS; ++w) {
        f[w] = mw[w] == -CUDART_INF_F ? 0.f : qa_ex2(mw[w] - big);
        sum = fmaf(res[(w * QA_ROWS + r) * LD + DH + 1], f[w], sum);
      }
      if constexpr (FUSED) {
        // to the CTA that folds the row: [slot][row / nslots] of its shared memory
        const uint32_t at = smem_u32(res + QA_WARPS * QA_ROWS * LD) +
                            4 * ((blockIdx.x * ((QA_ROWS + nslots - 1) / nslots) + r / nslots) * LD);
        uint32_t dst;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(at), "r"(r % nslots));
        if (lane == 0)
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst + 4 * DH), "f"(big), "f"(sum) : "memory");
#pragma unroll
        for (int d = 0; d < DH; d += 32) {
          float acc = 0.f;
#pragma unroll
          for (int w = 0; w < QA_WARPS; ++w) acc = fmaf(res[(w * QA_ROWS + r) * LD + d + lane], f[w], acc);
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4 * (d + lane)), "f"(acc) : "memory");
        }
      } else {
        const size_t prow =
            ((static_cast<size_t>(b) * cache.G + kvh) * (static_cast<size_t>(tc) * grp) + R) * nslots + blockIdx.x;
        if (lane == 0) part_s[prow] = make_float2(big, sum);
#pragma unroll
        for (int d = 0; d < DH; d += 32) {
          float acc = 0.f;
#pragma unroll
          for (int w = 0; w < QA_WARPS; ++w) acc = fmaf(res[(w * QA_ROWS + r) * LD + d + lane], f[w], acc);
          part_o[prow * DH + d + lane] = acc;
        }
      }
    }
    __syncthreads();
  }
}

// whether row b's token t is a token, and its position; a row that cannot be read (bad lengths, or beyond
// the launch's slots) is set to NaN
template <typename T, int DH>
__device__ __forceinline__ bool fold_row(const Q4CacheDev& cache, const Q4RowsDev& rows, int b, int t, int nslots,
                                         bool tcore, T* dst, int* n) {
  const int lane = threadIdx.x & 31;
  int len, count;
  const bool ok = q4_row(rows, b, &len, &count, cache.P);
  if (t >= (ok ? count : min(max(count, 0), rows.T))) return false;
  if (ok) {
    const int pos = len + t;
    *n = pos / (tcore && pos >= QA_TC_BEGIN ? qa_tc_keys(qa_tc_class(pos)) : qa_cta_keys(qa_class(pos))) + 1;
  }
  if (ok && *n <= nslots) return true;
  for (int d = lane; d < DH; d += 32) dst[d] = from_f32<T>(CUDART_NAN_F);
  if (ok && lane == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
  return false;
}

template <typename T, int DH>
__global__ void __launch_bounds__(QA_THREADS, sizeof(T) == 2 ? 3 : 2)
    q4_attn_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor q, int grp, int t0, int tc, int tiles, float scale_log2,
                   int nslots, int q_vec, int top, float* __restrict__ part_o, float2* __restrict__ part_s) {
  pdl_trigger();
  extern __shared__ __align__(16) float qa_sm[];  // the queries, then [warp][16][DH + 2] results
  pdl_wait();
  attn_tile<T, DH, false>(qa_sm, cache, rows, q, grp, t0, tc, tiles, scale_log2, nslots, q_vec != 0, top, part_o, part_s);
}

// rows that the CTAs of a cluster of nslots hold for folding: [slot][row / nslots], at most
constexpr int QA_FOLD_ROWS = QA_ROWS + QA_CLUSTER - 1;

// Short contexts: the CTAs of a tile are one cluster and fold their results through its shared memory,
// with the combine kernel's arithmetic and without its launch and the workspace.  Row r is folded by CTA
// r % nslots, into whose shared memory the others push their results: one cluster barrier on the way.
template <typename T, int DH>
__global__ void __launch_bounds__(QA_THREADS, sizeof(T) == 2 ? 3 : 2)
    q4_attn_fused_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor q, Q4Tensor out, int grp, int tiles,
                         float scale_log2, int q_vec) {
  cluster_arrive_relaxed();
  pdl_trigger();
  extern __shared__ __align__(16) float qa_sm[];  // the queries, [warp][16][DH + 2] results, the rows to fold
  pdl_wait();
  cluster_wait();  // every CTA of the cluster has started
  const int nslots = gridDim.x;
  attn_tile<T, DH, true>(qa_sm, cache, rows, q, grp, 0, rows.T, tiles, scale_log2, nslots, q_vec != 0, 3,
                         nullptr, nullptr);
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y / tiles, tile = blockIdx.y % tiles, b = blockIdx.z;
  const int per = (QA_ROWS + nslots - 1) / nslots;
  const float* fin = qa_sm + qa_q_floats<T, DH>() + QA_WARPS * QA_ROWS * (DH + 2);
  for (int r = warp * nslots + blockIdx.x; r < QA_ROWS; r += QA_WARPS * nslots) {
    const int R = tile * QA_ROWS + r, t = R / grp;
    if (R >= rows.T * grp) break;
    T* dst = static_cast<T*>(out.p) + b * out.sb + t * out.st + (kvh * grp + R % grp) * out.sh;
    int n;
    if (!fold_row<T, DH>(cache, rows, b, t, nslots, false, dst, &n)) continue;
    const float* row = fin + r / nslots * (DH + 2);
    float v[QA_CLUSTER][DH / 32], mx[QA_CLUSTER], sm[QA_CLUSTER], big = -CUDART_INF_F;
#pragma unroll
    for (int x = 0; x < QA_CLUSTER; ++x)
      if (x < n) {
        const float* a = row + x * per * (DH + 2);
        mx[x] = a[DH], sm[x] = a[DH + 1];
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) v[x][d] = a[32 * d + lane];
        big = fmaxf(big, mx[x]);
      }
    float acc[DH / 32], sum = 0.f;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d) acc[d] = 0.f;
#pragma unroll
    for (int w = 0; w < QA_WARPS; ++w) {
      float part[DH / 32], ps = 0.f;
#pragma unroll
      for (int d = 0; d < DH / 32; ++d) part[d] = 0.f;
#pragma unroll
      for (int x = w; x < QA_CLUSTER; x += QA_WARPS)
        if (x < n) {
          const float f = mx[x] == -CUDART_INF_F ? 0.f : qa_ex2(mx[x] - big);
          ps = fmaf(sm[x], f, ps);
#pragma unroll
          for (int d = 0; d < DH / 32; ++d) part[d] = fmaf(v[x][d], f, part[d]);
        }
      sum += ps;
#pragma unroll
      for (int d = 0; d < DH / 32; ++d) acc[d] += part[d];
    }
#pragma unroll
    for (int d = 0; d < DH / 32; ++d) dst[32 * d + lane] = from_f32<T>(acc[d] / sum);
  }
}

// One CTA per output row: warp w folds the slots w, w + 4, ... in order, then the four sums in order.
template <typename T, int DH>
__global__ void __launch_bounds__(QA_THREADS)
    q4_combine_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor out, int grp, int t0, int prows, int nslots,
                      int tcore, const float* part_o, const float2* part_s) {
  __shared__ float fold[QA_WARPS][DH + 1];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.z, kvh = blockIdx.y, R = blockIdx.x;
  const int t = t0 + R / grp;
  T* dst = static_cast<T*>(out.p) + b * out.sb + t * out.st + (kvh * grp + R % grp) * out.sh;
  int n;
  if (!fold_row<T, DH>(cache, rows, b, t, nslots, tcore != 0, dst, &n)) return;  // the same for the whole CTA
  const size_t prow = ((static_cast<size_t>(b) * cache.G + kvh) * static_cast<size_t>(prows) + R) * nslots;
  float big = -CUDART_INF_F;
  for (int x = lane; x < n; x += 32) big = fmaxf(big, part_s[prow + x].x);
  big = warp_max(big);
  float acc[DH / 32], sum = 0.f;
#pragma unroll
  for (int d = 0; d < DH / 32; ++d) acc[d] = 0.f;
#pragma unroll 8
  for (int x = warp; x < n; x += QA_WARPS) {
    const float2 st = part_s[prow + x];
    const float f = st.x == -CUDART_INF_F ? 0.f : qa_ex2(st.x - big);
    sum = fmaf(st.y, f, sum);
#pragma unroll
    for (int d = 0; d < DH / 32; ++d) acc[d] = fmaf(part_o[(prow + x) * DH + 32 * d + lane], f, acc[d]);
  }
#pragma unroll
  for (int d = 0; d < DH / 32; ++d) fold[warp][32 * d + lane] = acc[d];
  if (lane == 0) fold[warp][DH] = sum;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= DH) return;
  float v = fold[0][d], w = fold[0][DH];
#pragma unroll
  for (int i = 1; i < QA_WARPS; ++i) v += fold[i][d], w += fold[i][DH];
  dst[d] = from_f32<T>(v / w);
}

inline int64_t padded_rows(int64_t rows) { return (rows + QA_ROWS - 1) / QA_ROWS * QA_ROWS; }

// one cluster per tile, no workspace
inline bool fused_fits(int nslots, int64_t T, int grp, int G) {
  return nslots <= QA_CLUSTER && padded_rows(T * grp) / QA_ROWS * G <= 65535;
}

template <typename T, int DH>
int launch_attn(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, const Q4Tensor& out, int H, float scale,
                int64_t bound, QaLong longs, float* ws, int64_t ws_floats, cudaStream_t st, bool pdl) {
  const int grp = H / c.G;
  const float scale_log2 = scale * 1.4426950408889634f;
  const int q_vec = q4_vec(q, sizeof(T));
  if (fused_fits(qa_slots(bound), r.T, grp, c.G)) {
    const int nslots = qa_slots(bound);
    auto* kern = q4_attn_fused_kernel<T, DH>;
    const int smem = (qa_q_floats<T, DH>() + (QA_WARPS * QA_ROWS + QA_FOLD_ROWS) * (DH + 2)) * 4;
    static std::atomic<unsigned long long> done{0};
    EVS_TRY(smem_attr_once(done, reinterpret_cast<const void*>(kern), smem));
    const int tiles = static_cast<int>(padded_rows(static_cast<int64_t>(r.T) * grp) / QA_ROWS);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(nslots, c.G * tiles, r.B);
    cfg.blockDim = dim3(QA_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nslots;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    EVS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, c, r, q, out, grp, tiles, scale_log2, q_vec));
    evs_count_launch(1);
    return EVS_OK;
  }
  auto* kern = q4_attn_kernel<T, DH>;
  const int smem = (qa_q_floats<T, DH>() + QA_WARPS * QA_ROWS * (DH + 2)) * 4;
  static std::atomic<unsigned long long> done{0};
  EVS_TRY(smem_attr_once(done, reinterpret_cast<const void*>(kern), smem));
  // From 65 rows a kv head on the tensor-core kernel takes the long positions.  It wins from 17 rows, two of the
  // other's tiles, on (65,536 keys, 32 kv heads: 245 us instead of 259 at 20 rows, 246 instead of 264 at 32, 266
  // instead of 505 at 64, but 244 instead of 145 at 13), but blocks of up to 64 tokens keep the sums of single
  // steps.  A model says which kernel, as its rule must not depend on a call's tokens.
  const bool many =
      longs == QaLong::BY_ROWS ? static_cast<int64_t>(r.T) * grp > QA_FEW_ROWS : longs == QaLong::TENSOR_CORE;
  const bool tcore = sizeof(T) == 2 && DH == 128 && many && bound > QA_TC_BEGIN;
  const int nslots = tcore ? qa_tc_slots(bound) : qa_slots(bound);
  // tokens per pass: as many as the workspace holds partial results for
  const int64_t per_row = static_cast<int64_t>(r.B) * c.G * nslots * (DH + 2);
  const int64_t fit = std::min<int64_t>(ws_floats / per_row, 65535 / c.G * QA_ROWS);  // rows a kv head
  int tokens = static_cast<int>(std::min<int64_t>(r.T, fit / grp));
  EVS_CHECK_RANGE(tokens >= 1, "q4 attention: the workspace is too small");
  if (tokens < r.T && grp <= 128) {  // passes of the same length, in whole tiles of the tensor-core kernel
    const int passes = (r.T + tokens - 1) / tokens, tile = 128 / grp, even = (r.T + passes - 1) / passes;
    tokens = std::min(tokens, (even + tile - 1) / tile * tile);
  }
  for (int t0 = 0; t0 < r.T; t0 += tokens) {
    const int tc = std::min(tokens, r.T - t0);
    const int prows = tc * grp, tiles = (prows + QA_ROWS - 1) / QA_ROWS;
    float* po = ws;
    float2* ps = reinterpret_cast<float2*>(ws + static_cast<int64_t>(r.B) * c.G * prows * nslots * DH);
    EVS_CUDA_TRY(evs_launch(kern, dim3(tcore ? qa_slots(QA_TC_BEGIN) : nslots, c.G * tiles, r.B),
                            dim3(QA_THREADS), smem, st, pdl, c, r, q, grp, t0, tc, tiles, scale_log2, nslots, q_vec,
                            tcore ? qa_class(QA_TC_BEGIN - 1) : 3, po, ps));
    evs_count_launch(1);
    if (tcore) EVS_TRY(launch_q4_attn_tc(c, r, q, grp, t0, tc, prows, scale_log2, nslots, q_vec, po, ps, st, true));
    // the combine may start while the last tiles run (it waits for them before it reads)
    EVS_CUDA_TRY(evs_launch(q4_combine_kernel<T, DH>, dim3(tc * grp, c.G, r.B), dim3(QA_THREADS), 0, st, true, c, r,
                            out, grp, t0, prows, nslots, tcore ? 1 : 0,
                            static_cast<const float*>(po), static_cast<const float2*>(ps)));
    evs_count_launch(1);
  }
  return EVS_OK;
}

int64_t bound_of(const evs_q4_cache* c, const evs_q4_rows* r, int max_length) {
  const int64_t table = static_cast<int64_t>(r->max_pages) * c->page_size;
  return max_length > 0 ? std::min<int64_t>(max_length, table) : table;
}

}  // namespace

int launch_q4_attention(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, const Q4Tensor& out, int H,
                        float scale, int64_t bound, QaLong longs, void* ws, int64_t ws_bytes, int dtype, cudaStream_t st,
                        bool pdl) {
#define QA_GO(T, DH) \
  return launch_attn<T, DH>(c, r, q, out, H, scale, bound, longs, static_cast<float*>(ws), ws_bytes / 4, st, pdl)
  if (dtype == EVS_DTYPE_BF16) {
    if (c.D == 32) QA_GO(__nv_bfloat16, 32);
    if (c.D == 64) QA_GO(__nv_bfloat16, 64);
    QA_GO(__nv_bfloat16, 128);
  }
  if (c.D == 32) QA_GO(float, 32);
  if (c.D == 64) QA_GO(float, 64);
  QA_GO(float, 128);
#undef QA_GO
}

int64_t q4_attention_ws(int B, int T, int G, int D, int H, int64_t bound) {
  // every row in one pass where that takes at most 256 MiB, else as many as fit (a token at least); tiles are
  // whole, their partial results are those of the rows alone
  const int grp = H / G;
  if (fused_fits(qa_slots(bound), T, grp, G)) return 0;
  const int64_t per_row = static_cast<int64_t>(B) * G * qa_slots(bound) * (D + 2) * 4;
  const int64_t fit = (256ll << 20) / per_row;
  return std::min(static_cast<int64_t>(T) * grp, std::max<int64_t>(grp, fit)) * per_row;
}

namespace {
// qkv projection: partial sums [splits][M][3d] -> data dtype [M][3d]
template <typename TD>
__global__ void __launch_bounds__(256) qkv_collect_kernel(const float* ws, int splits, size_t n, TD* out) {
  pdl_trigger();
  pdl_wait();
  const size_t i = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  split_sum4<false>(a, ws + i, n, splits);
  out[i] = from_f32<TD>(a.x);
  out[i + 1] = from_f32<TD>(a.y);
  out[i + 2] = from_f32<TD>(a.z);
  out[i + 3] = from_f32<TD>(a.w);
}

Q4CacheDev state_cache(const evs_state* s, int layer) {
  const int D = s->m->cfg.head_dim;
  return {static_cast<uint8_t*>(s->kv[layer]), s->d_err, static_cast<int64_t>(s->max_batch) * s->kv_pages, Q4_STATE_PAGE,
          s->m->Hl, D, Q4_STATE_PAGE * D + Q4_STATE_PAGE * D / 8};
}
}  // namespace

int launch_attention_q4(const evs_model* m, evs_state* s, int layer, int B, int T, int splits, int bound, bool prefill,
                        cudaStream_t st) {
  const int d = m->dl, H = m->Hl, D = m->cfg.head_dim, dtype = m->cfg.dtype;
  const bool pdl = s->use_pdl();
  const size_t el = m->elem(), n = static_cast<size_t>(B) * T * 3 * d;
  const dim3 grid(static_cast<unsigned>((n / 4 + 255) / 256));
  if (dtype == EVS_DTYPE_BF16)
    EVS_CUDA_TRY(evs_launch(qkv_collect_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, pdl,
                            static_cast<const float*>(s->ws), splits, n, static_cast<__nv_bfloat16*>(s->qkv)));
  else
    EVS_CUDA_TRY(evs_launch(qkv_collect_kernel<float>, grid, dim3(256), 0, st, pdl, static_cast<const float*>(s->ws),
                            splits, n, static_cast<float*>(s->qkv)));
  evs_count_launch(1);
  const Q4CacheDev c = state_cache(s, layer);
  const Q4RowsDev r{s->d_table, s->d_len, nullptr, s->kv_pages, s->kv_pages, B, T};
  char* qkv = static_cast<char*>(s->qkv);
  const int64_t row = 3ll * d;
  const Q4Tensor q{qkv, T * row, row, D}, k{qkv + d * el, T * row, row, D}, v{qkv + 2 * d * el, T * row, row, D};
  const Q4Tensor qr{s->qrot, static_cast<int64_t>(T) * d, d, D};
  const Q4Tensor out{s->act, static_cast<int64_t>(T) * s->ld_act, s->ld_act, D};
  EVS_TRY(launch_q4_append(c, r, q, k, v, qr, H, dtype, m->cfg.rope_base, st, pdl));
  return launch_q4_attention(c, r, qr, out, H, 1.f / std::sqrt(static_cast<float>(D)), bound,
                             prefill ? QaLong::TENSOR_CORE : QaLong::ROW_TILES, s->attn_part,
                             static_cast<int64_t>(s->attn_part_bytes), dtype, st, pdl);
}

int launch_q4_state_read(const evs_state* s, int layer, int row, int width, void* dst, cudaStream_t st) {
  if (width == 0) return EVS_OK;
  const int H = s->m->Hl, D = s->m->cfg.head_dim;
  const int64_t t = 2ll * H * D;
  const Q4RowsDev r{s->d_table + static_cast<size_t>(row) * s->kv_pages, s->d_zero, nullptr, s->kv_pages, s->kv_pages, 1,
                    width};
  const Q4Tensor k{dst, width * t, t, D}, v{static_cast<char*>(dst) + H * D * s->m->elem(), width * t, t, D};
  return launch_q4_read(state_cache(s, layer), r, k, v, s->m->cfg.dtype, st);
}

extern "C" {

int64_t evs_q4_attention_workspace(const evs_q4_cache* cache, const evs_q4_rows* rows, int n_heads, int max_length) {
  if (q4_check_cache(cache) != EVS_OK || q4_check_rows(cache, rows) != EVS_OK || n_heads < cache->kv_heads ||
      n_heads % cache->kv_heads != 0 || max_length < 0)
    return -1;
  return q4_attention_ws(rows->batch, rows->tokens, cache->kv_heads, cache->head_dim, n_heads,
                         bound_of(cache, rows, max_length));
}

int evs_q4_attention(const evs_q4_cache* cache, const evs_q4_rows* rows, const void* q, const int64_t* q_strides,
                     int n_heads, float scale, int max_length, void* out, const int64_t* out_strides, int dtype,
                     void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  EVS_TRY(q4_check_cache(cache));
  EVS_TRY(q4_check_rows(cache, rows));
  EVS_CHECK_ARG(q && out && q_strides && out_strides && (workspace || workspace_bytes == 0), "null argument");
  EVS_CHECK_ARG(dtype == EVS_DTYPE_BF16 || dtype == EVS_DTYPE_FP32, "q4 attention: q must be fp32 or bf16");
  EVS_CHECK_ARG(n_heads >= cache->kv_heads && n_heads % cache->kv_heads == 0,
                "q4 attention: n_heads must be a multiple of kv_heads");
  EVS_CHECK_ARG(scale > 0.f && scale <= 1e38f, "q4 attention: scale must be positive and at most 1e38");
  EVS_CHECK_ARG(max_length >= 0, "q4 attention: max_length must not be negative");
  EVS_CHECK_ARG(cache->kv_heads <= 65535 && rows->batch <= 65535, "q4 attention: too many heads or rows");
  EVS_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "q4 attention: the workspace must be 16-byte aligned");
  const Q4Tensor tq{const_cast<void*>(q), q_strides[0], q_strides[1], q_strides[2]};
  const Q4Tensor to{out, out_strides[0], out_strides[1], out_strides[2]};
  const int B = rows->batch, T = rows->tokens, D = cache->head_dim;
  const bool in_place = q == out && tq.sb == to.sb && tq.st == to.st && tq.sh == to.sh;
  EVS_CHECK_ARG(q4_distinct(to, B, T, n_heads, D), "q4 attention: elements of out overlap");
  EVS_CHECK_ARG(in_place || !q4_share(to, n_heads, tq, n_heads, B, T, D, dtype == EVS_DTYPE_BF16 ? 2 : 4),
                "q4 attention: out overlaps q");
  return launch_q4_attention(q4_cache_dev(cache), q4_rows_dev(rows), tq, to, n_heads, scale,
                             bound_of(cache, rows, max_length), QaLong::BY_ROWS, workspace, workspace_bytes, dtype, st,
                             true);
}

}  // extern "C"
