// Causal attention of new tokens over the paged 4-bit KV cache, grouped heads, rows of different
// lengths: out = softmax(scale q . K) V over the keys 0 .. P of a token at position P.
//
// Split-KV. A warp takes a unit of consecutive keys for a tile of 16 query rows (a row is one token
// of one query head of the kv head) and runs an online softmax over it; the four units of a CTA are
// folded in order, and a second kernel folds the CTAs' partial results in order.  The unit's length
// depends on the row's own position alone (64 keys below 4096, 256 below 65536, else 1024), so a
// token's result does not depend on what else is in the call: verify blocks and single steps agree
// bit for bit.
#include <math_constants.h>

#include <algorithm>

#include "internal.hpp"
#include "q4.cuh"
#include "q4_cache.hpp"

namespace {

constexpr int QA_WARPS = 4;
constexpr int QA_THREADS = 32 * QA_WARPS;
constexpr int QA_ROWS = 16;
constexpr int QA_STEP = 32;  // keys per online-softmax step of a warp

// length class of a position, and keys per CTA of a class
__host__ __device__ constexpr int qa_class(int64_t pos) { return pos < 4096 ? 0 : (pos < 65536 ? 1 : 2); }
__host__ __device__ constexpr int64_t qa_class_end(int cl) { return cl == 0 ? 4096 : (cl == 1 ? 65536 : (1ll << 40)); }
__host__ __device__ constexpr int qa_cta_keys(int cl) { return 256 << (2 * cl); }
// partial results of one row for lengths up to bound
inline int qa_slots(int64_t bound) {
  int n = 1;
  for (int cl = 0; cl < 3; ++cl) {
    const int64_t end = std::min(bound, qa_class_end(cl));
    n = std::max<int64_t>(n, (end + qa_cta_keys(cl) - 1) / qa_cta_keys(cl));
    if (bound <= qa_class_end(cl)) break;
  }
  return n;
}

template <int DH>
struct KTile {  // 32 keys: per 16-key chunk two 8-key tiles, features c DH / 4 .. of one key each
  uint32_t w[2][2][DH / 32];
  uint32_t s[2][2];
};
template <int DH>
struct VTile {  // 32 keys: per 16-key chunk the features g DH / 8 .. of the keys 4 c .. 4 c + 3
  static constexpr int NW = DH / 64 > 0 ? DH / 64 : 1;
  uint32_t w[2][4][NW];
  uint32_t s[2][2];
};

template <int NW>
__device__ __forceinline__ void ld_words(uint32_t (&w)[NW], const uint8_t* p) {
  if constexpr (NW == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (NW == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// whether one of the bf16 scales of a pair is NaN (scales are at most 2^120: only a NaN's exponent
// carries into the sign bit)
__device__ __forceinline__ uint32_t scales_nan(uint32_t s2) { return (s2 + 0x00800080u) & 0x80008000u; }

template <typename T, int DH>
__global__ void __launch_bounds__(QA_THREADS)
    q4_attn_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor q, int grp, int t0, int tc, int tiles, float scale_log2,
                   int nslots, float* __restrict__ part_o, float2* __restrict__ part_s) {
  constexpr int NQ = sizeof(T) == 2 ? 1 : 3;  // bf16 parts of a query value
  constexpr int NP = sizeof(T) == 2 ? 2 : 3;  // bf16 parts of a probability
  constexpr int KW = DH / 32;                 // code words per thread and key (K)
  constexpr int VN = DH / 8;                  // 8-feature tiles of the output
  pdl_trigger();
  extern __shared__ __align__(16) float qa_sm[];  // [warp][16][DH + 2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.y / tiles, tile = blockIdx.y % tiles, b = blockIdx.z;
  pdl_wait();
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
    return;
  }
  const int first = t0 + tile * QA_ROWS / grp;
  const int last = min(min(t0 + (tile * QA_ROWS + QA_ROWS - 1) / grp, t0 + tc - 1), count - 1);
  if (first > last) return;
  const int64_t pmax = static_cast<int64_t>(len) + last;
  const int cl0 = qa_class(static_cast<int64_t>(len) + first), cl1 = qa_class(pmax);
  if (static_cast<int64_t>(blockIdx.x) * qa_cta_keys(cl0) > pmax) return;

  // this thread's two rows: tokens and positions (-1: no token)
  int tok[2], pos[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = tile * QA_ROWS + g + 8 * i;
    tok[i] = t0 + r / grp;
    pos[i] = r < tc * grp && tok[i] < count ? len + tok[i] : -1;
  }
  // queries as product operands: step 2 w covers the feature pairs (0,4) (1,5) of the word 8 w ..,
  // step 2 w + 1 the pairs (2,6) (3,7), as q4_word decodes the keys
  uint32_t qa[NQ][2 * KW][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = tile * QA_ROWS + g + 8 * i;
    const T* src = static_cast<const T*>(q.p) + b * q.sb + tok[i] * q.st + (kvh * grp + r % grp) * q.sh + c * (DH / 4);
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      uint32_t e[8][3];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (NQ == 1)
          e[j][0] = pos[i] >= 0 ? __bfloat16_as_ushort(src[8 * w + j]) : 0u;
        else
          q4_parts(pos[i] >= 0 ? to_f32<T>(src[8 * w + j]) : 0.f, e[j]);
      }
#pragma unroll
      for (int p = 0; p < NQ; ++p) {
        qa[p][2 * w][i] = e[0][p] | e[4][p] << 16;
        qa[p][2 * w][2 + i] = e[1][p] | e[5][p] << 16;
        qa[p][2 * w + 1][i] = e[2][p] | e[6][p] << 16;
        qa[p][2 * w + 1][2 + i] = e[3][p] | e[7][p] << 16;
      }
    }
  }
  const int64_t trow = b * rows.table_stride;
  const int k_scales = cache.P * DH, v_codes = cache.P * (DH / 2), v_scales = k_scales + cache.P * (DH / 16);
  const int kg = c * (DH / 4) / 32, vg = g * (DH / 8) / 32;  // this thread's scale groups

  for (int cl = cl0; cl <= cl1; ++cl) {
    const int64_t kend64 = min(pmax, qa_class_end(cl) - 1) + 1;  // keys seen by some row of the class
    const int unit = qa_cta_keys(cl) / QA_WARPS;
    const int64_t kbeg64 = static_cast<int64_t>(blockIdx.x) * qa_cta_keys(cl) + warp * unit;
    if (static_cast<int64_t>(blockIdx.x) * qa_cta_keys(cl) >= kend64) continue;
    const int kbeg = static_cast<int>(kbeg64), kend = static_cast<int>(min(kend64, kbeg64 + unit));
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) lim[i] = pos[i] >= 0 && qa_class(pos[i]) == cl ? pos[i] : -1;

    float o[VN][4], m[2], l[2];
#pragma unroll
    for (int n = 0; n < VN; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;

    int page_of = -1;  // lane's page id of the 16-key chunk (step & ~15) * 2 + lane
    auto load_pages = [&](int key) {
      const int kk = key + 16 * lane;
      page_of = -1;
      if (kk < kend) page_of = __ldg(rows.table + trow + kk / cache.P);
    };
    // the block of the 16-key chunk starting at key, or null (no keys there, or a bad page)
    auto chunk_of = [&](int key, int sub) -> const uint8_t* {
      const int idx = ((key - kbeg) >> 4) + sub;
      const int id = __shfl_sync(0xffffffffu, page_of, idx & 31);
      if (key + 16 * sub >= kend || id < 0 || id >= cache.pages) return nullptr;
      return cache.block(id, kvh);
    };
    KTile<DH> kt;
    auto load_k = [&](int key) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint8_t* blk = chunk_of(key, sub);
        const int slot0 = (key + 16 * sub) % cache.P;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int slot = slot0 + 4 * (g >> 1) + (g & 1) + 2 * u;
          if (blk != nullptr) {
            ld_words<KW>(kt.w[sub][u], blk + slot * (DH / 2) + c * (DH / 8));
            kt.s[sub][u] = __ldg(reinterpret_cast<const uint16_t*>(blk + k_scales) + kg * cache.P + slot);
          } else {
#pragma unroll
            for (int w = 0; w < KW; ++w) kt.w[sub][u][w] = 0u;
            kt.s[sub][u] = 0x7FC0u;  // keys without a page: a NaN score for whoever sees them
          }
        }
      }
    };
    VTile<DH> vt;
    auto load_v = [&](int key) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint8_t* blk = chunk_of(key, sub);
        const int slot = (key + 16 * sub) % cache.P + 4 * c;
        if (blk != nullptr) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint8_t* p = blk + v_codes + (slot + j) * (DH / 2) + g * (DH / 16);
            if constexpr (DH == 32)
              vt.w[sub][j][0] = __ldg(reinterpret_cast<const uint16_t*>(p));
            else
              ld_words<VTile<DH>::NW>(vt.w[sub][j], p);
          }
          const uint2 s = __ldg(reinterpret_cast<const uint2*>(blk + v_scales + 2 * (vg * cache.P + slot)));
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
      load_k(kbeg);
    }
    for (int key = kbeg; key < kend; key += QA_STEP) {
      load_v(key);
      float s[2][2][4];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[sub][u][0] = s[sub][u][1] = s[sub][u][2] = s[sub][u][3] = 0.f;
          const Q4Scale ks = q4_scale(kt.s[sub][u] | kt.s[sub][u] << 16);
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            uint32_t kv[4];
            q4_word(kt.w[sub][u][w], ks, kv);
#pragma unroll
            for (int p = NQ - 1; p >= 0; --p) {
              q4_mma(s[sub][u], qa[p][2 * w][0], qa[p][2 * w][1], qa[p][2 * w][2], qa[p][2 * w][3], kv[0], kv[1]);
              q4_mma(s[sub][u], qa[p][2 * w + 1][0], qa[p][2 * w + 1][1], qa[p][2 * w + 1][2], qa[p][2 * w + 1][3],
                     kv[2], kv[3]);
            }
          }
        }
      const int next = key + QA_STEP;
      const VTile<DH> vc = vt;
      bool bad_page = false;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
        bad_page |= key + 16 * sub < kend && chunk_of(key, sub) == nullptr;
      if (bad_page && lane == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
      if (next < kend) {
        if (((next - kbeg) & 511) == 0) load_pages(next);
        load_k(next);
      }
      // scores to probabilities: thread's keys of a chunk are 4 c + 2 u + (0, 1)
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kk = key + 16 * sub + 4 * c + 2 * u + (e & 1);
            const float v = kk <= lim[e >> 1] ? s[sub][u][e] * scale_log2 : -CUDART_INF_F;
            s[sub][u][e] = v;
            mx[e >> 1] = fmaxf(mx[e >> 1], v);
          }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] != m[0] || mx[1] != m[1])) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a = mx[i] == m[i] ? 1.f : exp2f(m[i] - mx[i]);
          m[i] = mx[i];
          l[i] *= a;
#pragma unroll
          for (int n = 0; n < VN; ++n) {
            o[n][2 * i] *= a;
            o[n][2 * i + 1] *= a;
          }
        }
      }
      const float mu[2] = {m[0] == -CUDART_INF_F ? 0.f : m[0], m[1] == -CUDART_INF_F ? 0.f : m[1]};
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        // probabilities as bf16 parts: a[p] = keys (4 c, 4 c + 1) of rows g, g + 8, then (4 c + 2, 4 c + 3)
        uint32_t pa[NP][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = exp2f(s[sub][u][2 * i] - mu[i]), p1 = exp2f(s[sub][u][2 * i + 1] - mu[i]);
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
        uint32_t vs[2] = {vc.s[sub][0], vc.s[sub][1]};
        // keys behind the last visible one hold whatever the page held: their scale becomes 0
        const int k4 = key + 16 * sub + 4 * c;
        if (k4 + 4 > kend) {
          if (k4 >= kend) vs[0] &= 0xFFFF0000u;
          if (k4 + 1 >= kend) vs[0] &= 0x0000FFFFu;
          if (k4 + 2 >= kend) vs[1] &= 0xFFFF0000u;
          if (k4 + 3 >= kend) vs[1] &= 0x0000FFFFu;
        }
        const uint32_t nan0 = scales_nan(vs[0]), nan1 = scales_nan(vs[1]);
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
          const uint32_t t01 = __byte_perm(vc.w[sub][0][w], vc.w[sub][1][w], sel);
          const uint32_t t23 = __byte_perm(vc.w[sub][2][w], vc.w[sub][3][w], sel);
          uint32_t b01[4], b23[4];
          q4_word(t01, s01, b01);
          q4_word(t23, s23, b23);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
              q4_mma(o[4 * n4 + j], pa[p][0], pa[p][1], pa[p][2], pa[p][3], b01[j], b23[j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // the four units folded in order
    constexpr int LD = DH + 2;
    float* mine = qa_sm + warp * QA_ROWS * LD;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* row = mine + (g + 8 * i) * LD;
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        row[2 * c * VN + n] = o[n][2 * i];
        row[(2 * c + 1) * VN + n] = o[n][2 * i + 1];
      }
      if (c == 0) {
        row[DH] = m[i];
        row[DH + 1] = l[i];
      }
    }
    __syncthreads();
    for (int r = warp; r < QA_ROWS; r += QA_WARPS) {
      const int R = tile * QA_ROWS + r, t = t0 + R / grp;
      if (R >= tc * grp || t >= count || qa_class(static_cast<int64_t>(len) + t) != cl) continue;
      float mw[QA_WARPS], big = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < QA_WARPS; ++w) {
        mw[w] = qa_sm[(w * QA_ROWS + r) * LD + DH];
        big = fmaxf(big, mw[w]);
      }
      float sum = 0.f, f[QA_WARPS];
#pragma unroll
      for (int w = 0; w < QA_WARPS; ++w) {
        f[w] = mw[w] == -CUDART_INF_F ? 0.f : exp2f(mw[w] - big);
        sum += qa_sm[(w * QA_ROWS + r) * LD + DH + 1] * f[w];
      }
      const size_t prow =
          ((static_cast<size_t>(b) * cache.G + kvh) * (static_cast<size_t>(tiles) * QA_ROWS) + R) * nslots + blockIdx.x;
      for (int d = lane; d < DH; d += 32) {
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < QA_WARPS; ++w) acc += qa_sm[(w * QA_ROWS + r) * LD + d] * f[w];
        part_o[prow * DH + d] = acc;
      }
      if (lane == 0) part_s[prow] = make_float2(big, sum);
    }
    __syncthreads();
  }
}

// One warp per output row: the CTAs' partial results folded in order.
template <typename T, int DH>
__global__ void __launch_bounds__(QA_THREADS)
    q4_combine_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor out, int grp, int t0, int tc, int tiles, int nslots,
                      const float* __restrict__ part_o, const float2* __restrict__ part_s) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, b = blockIdx.z, kvh = blockIdx.y;
  const int R = blockIdx.x * QA_WARPS + (threadIdx.x >> 5);
  if (R >= tc * grp) return;
  const int t = t0 + R / grp;
  int len, count;
  const bool ok = q4_row(rows, b, &len, &count, cache.P);
  if (t >= (ok ? count : min(max(count, 0), rows.T))) return;
  T* dst = static_cast<T*>(out.p) + b * out.sb + t * out.st + (kvh * grp + R % grp) * out.sh;
  if (!ok) {
    for (int d = lane; d < DH; d += 32) dst[d] = from_f32<T>(CUDART_NAN_F);
    return;
  }
  const int64_t pos = static_cast<int64_t>(len) + t;
  const int n = static_cast<int>(pos / qa_cta_keys(qa_class(pos))) + 1;
  const size_t prow = ((static_cast<size_t>(b) * cache.G + kvh) * (static_cast<size_t>(tiles) * QA_ROWS) + R) * nslots;
  if (n > nslots) {  // max_length was below this row's length
    for (int d = lane; d < DH; d += 32) dst[d] = from_f32<T>(CUDART_NAN_F);
    if (lane == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
    return;
  }
  float big = -CUDART_INF_F;
  for (int x = lane; x < n; x += 32) big = fmaxf(big, part_s[prow + x].x);
  big = warp_max(big);
  float acc[DH / 32], sum = 0.f;
#pragma unroll
  for (int d = 0; d < DH / 32; ++d) acc[d] = 0.f;
#pragma unroll 4
  for (int x = 0; x < n; ++x) {
    const float2 st = part_s[prow + x];
    const float f = st.x == -CUDART_INF_F ? 0.f : exp2f(st.x - big);
    sum += st.y * f;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d) acc[d] += part_o[(prow + x) * DH + 32 * d + lane] * f;
  }
#pragma unroll
  for (int d = 0; d < DH / 32; ++d) dst[32 * d + lane] = from_f32<T>(acc[d] / sum);
}

template <typename T, int DH>
int launch_attn(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, const Q4Tensor& out, int H, float scale,
                int64_t bound, float* ws, int64_t ws_floats, cudaStream_t st, bool pdl) {
  const int grp = H / c.G, nslots = qa_slots(bound);
  auto* kern = q4_attn_kernel<T, DH>;
  const int smem = QA_WARPS * QA_ROWS * (DH + 2) * 4;
  static std::atomic<unsigned long long> done{0};
  EVS_TRY(smem_attr_once(done, reinterpret_cast<const void*>(kern), smem));
  // tokens per pass: as many as the workspace holds partial results for
  const int64_t per_tile = static_cast<int64_t>(r.B) * c.G * QA_ROWS * nslots * (DH + 2);
  const int64_t fit = std::min<int64_t>(ws_floats / per_tile, 65535 / c.G);  // row tiles per pass
  int tokens = static_cast<int>(std::min<int64_t>(r.T, fit * QA_ROWS / grp));
  EVS_CHECK_RANGE(fit >= 1 && tokens >= 1, "q4 attention: the workspace is too small");
  for (int t0 = 0; t0 < r.T; t0 += tokens) {
    const int tc = std::min(tokens, r.T - t0);
    const int tiles = (tc * grp + QA_ROWS - 1) / QA_ROWS;
    float* po = ws;
    float2* ps = reinterpret_cast<float2*>(ws + static_cast<int64_t>(r.B) * c.G * tiles * QA_ROWS * nslots * DH);
    EVS_CUDA_TRY(evs_launch(kern, dim3(nslots, c.G * tiles, r.B), dim3(QA_THREADS), smem, st, pdl, c, r, q, grp, t0, tc,
                            tiles, scale * 1.4426950408889634f, nslots, po, ps));
    EVS_CUDA_TRY(evs_launch(q4_combine_kernel<T, DH>, dim3((tc * grp + QA_WARPS - 1) / QA_WARPS, c.G, r.B),
                            dim3(QA_THREADS), 0, st, pdl, c, r, out, grp, t0, tc, tiles, nslots,
                            static_cast<const float*>(po), static_cast<const float2*>(ps)));
    evs_count_launch(2);
  }
  return EVS_OK;
}

int64_t bound_of(const evs_q4_cache* c, const evs_q4_rows* r, int max_length) {
  const int64_t table = static_cast<int64_t>(r->max_pages) * c->page_size;
  return max_length > 0 ? std::min<int64_t>(max_length, table) : table;
}

}  // namespace

int launch_q4_attention(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, const Q4Tensor& out, int H,
                        float scale, int64_t bound, void* ws, int64_t ws_bytes, int dtype, cudaStream_t st, bool pdl) {
#define QA_GO(T, DH) \
  return launch_attn<T, DH>(c, r, q, out, H, scale, bound, static_cast<float*>(ws), ws_bytes / 4, st, pdl)
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
  // all row tiles in one pass where that takes at most 256 MiB, else as many as fit
  const int grp = H / G;
  const int64_t per_tile = static_cast<int64_t>(B) * G * QA_ROWS * qa_slots(bound) * (D + 2) * 4;
  const int64_t least = (std::max(grp, 1) + QA_ROWS - 1) / QA_ROWS;  // one token
  const int64_t all = (static_cast<int64_t>(T) * grp + QA_ROWS - 1) / QA_ROWS;
  const int64_t want = std::min(all, std::max<int64_t>(least, (256ll << 20) / per_tile));
  return want * per_tile;
}

extern "C" {

int64_t evs_q4_attention_workspace(const evs_q4_cache* cache, const evs_q4_rows* rows, int n_heads, int max_length) {
  if (q4_check_cache(cache) != EVS_OK || q4_check_rows(cache, rows) != EVS_OK || n_heads < cache->kv_heads ||
      n_heads % cache->kv_heads != 0 || max_length < 0)
    return 0;
  return q4_attention_ws(rows->batch, rows->tokens, cache->kv_heads, cache->head_dim, n_heads,
                         bound_of(cache, rows, max_length));
}

int evs_q4_attention(const evs_q4_cache* cache, const evs_q4_rows* rows, const void* q, const int64_t* q_strides,
                     int n_heads, float scale, int max_length, void* out, const int64_t* out_strides, int dtype,
                     void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  EVS_TRY(q4_check_cache(cache));
  EVS_TRY(q4_check_rows(cache, rows));
  EVS_CHECK_ARG(q && out && q_strides && out_strides && workspace, "null argument");
  EVS_CHECK_ARG(dtype == EVS_DTYPE_BF16 || dtype == EVS_DTYPE_FP32, "q4 attention: q must be fp32 or bf16");
  EVS_CHECK_ARG(n_heads >= cache->kv_heads && n_heads % cache->kv_heads == 0,
                "q4 attention: n_heads must be a multiple of kv_heads");
  EVS_CHECK_ARG(max_length >= 0, "q4 attention: max_length must not be negative");
  EVS_CHECK_ARG(cache->kv_heads <= 65535 && rows->batch <= 65535, "q4 attention: too many heads or rows");
  EVS_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "q4 attention: the workspace must be 16-byte aligned");
  const Q4Tensor tq{const_cast<void*>(q), q_strides[0], q_strides[1], q_strides[2]};
  const Q4Tensor to{out, out_strides[0], out_strides[1], out_strides[2]};
  return launch_q4_attention(q4_cache_dev(cache), q4_rows_dev(rows), tq, to, n_heads, scale,
                             bound_of(cache, rows, max_length), workspace, workspace_bytes, dtype, st, false);
}

}  // extern "C"
