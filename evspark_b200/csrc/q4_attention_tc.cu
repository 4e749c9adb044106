// Attention over the paged 4-bit KV cache on the 5th-generation tensor cores: the partial results of
// positions from 4,096 on in calls with many rows a kv head (bf16 queries, head_dim 128), in the split and the
// form of q4_attention.cu, whose combine kernel folds them.
//
// One CTA takes up to 128 query rows (a row is one token of one query head of the kv head) over its slot of
// keys, 64 keys a step: S = Q K^T (128 x 64 x 128) and O += P V (128 x 128 x 64).  Four warps decode keys and
// values into shared memory once for all rows; one warp issues whatever product is ready first; four warps run
// the online softmax, one row a thread, with S, then P (two bf16 parts) in S's place, and O in tensor memory.
// Two stages of everything, so that a step's scores are there while the one before is still worked on; two CTAs
// an SM.
//
// Measured beside the 16-row mma.sync kernel, which decodes the keys once per 16 rows: 16 rows of 13 tokens,
// 64 / 8 heads, up to 16,384 keys 209 us instead of 332; 1,024 tokens, 32 heads, behind 16,384 keys 703
// instead of 2,072; but 13 tokens of 32 heads at 65,536 keys 244 instead of 145: a step takes nearly the same
// time for 1 row as for 128.  What it takes: a step's 64 keys about 1,900 clocks an SM, of which shared memory
// (keys stored and read once, values stored once and read for both parts of the probabilities, the queries read
// once a step) is busy for 900 and the tensor pipe for a third; 0.45 instructions issued a clock and scheduler, the
// decoding warps (2,200 clocks a step) and the softmax warps waiting for barriers and tensor memory.
// Tried and no faster (with one part): one CTA an SM with four stages and 8 or 16 decoding warps; the queries in
// tensor memory with one stage of scores; a barrier each for decoded keys and values.
#include <math_constants.h>

#include <algorithm>

#include "internal.hpp"
#include "q4.cuh"
#include "q4_attention.hpp"

namespace {

constexpr int DH = 128;
constexpr int TC_ROWS = 128;
constexpr int TC_KEYS = 64;  // keys a step
constexpr int STAGES = 2;    // of K, V, S and P
constexpr int SOFT_WARPS = 4, DEC_WARPS = 4;
constexpr int TC_THREADS = 32 * (SOFT_WARPS + DEC_WARPS + 1);
constexpr int Q_BYTES = TC_ROWS * DH * 2;   // decoded operands: 128-byte columns of 64 values
constexpr int KV_BYTES = TC_KEYS * DH * 2;  // one stage of K, or of V^T
constexpr int TC_SMEM = Q_BYTES + 2 * STAGES * KV_BYTES + 1024 + 256;  // Q, the stages of K and V; alignment; barriers
constexpr uint32_t TMEM_COLS = 256;  // the stages of S (then P), O
constexpr uint32_t TMEM_O = STAGES * TC_KEYS;

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[smem desc, or tmem: a row a lane, two values a column] * B[smem desc], issued by the one lane
// with on != 0 of a warp that stays together, so that operands live in uniform registers; descriptors as their low
// words beside the high one that they share
template <bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 e, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 x, {%2, %4};\n\tmov.b64 y, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%1], x, y, %5, p;\n\t}"
      ::"r"(on), "r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "n"(ACC ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 y;\n\t"
      "setp.ne.b32 e, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 y, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], y, %5, p;\n\t}"
      ::"r"(on), "r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t on, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %0, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}"
      ::"r"(on), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16-byte unit u of row r of an operand of ROWS rows, 128-byte swizzle
template <int ROWS>
__device__ __forceinline__ uint32_t tile_at(int r, int u) {
  return (u >> 3) * (ROWS * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4);
}

// One step of the online softmax of a row (its thread's lane): the scores at tm -> probabilities in their
// place (the upper parts, then the lower ones), the outputs so far (at to) moved to a new reference once complete() says that they are complete.  Keys
// from seen on are masked.
template <bool MASKED, typename F>
__device__ __forceinline__ void softmax_step(uint32_t tm, uint32_t to, float scale_log2, int seen, float& m, float& l,
                                             F&& complete) {
  float s[TC_KEYS / 16][16];
#pragma unroll
  for (int c = 0; c < TC_KEYS / 16; ++c) tmem_ld_32x32b_x16(tm + 16 * c, s[c]);
  tmem_ld_wait();
  float x[4] = {m, m, m, m};
#pragma unroll
  for (int j = 0; j < TC_KEYS; ++j) {
    float& v = s[j >> 4][j & 15];
    if (MASKED && j >= seen) v = -CUDART_INF_F;
    x[j & 3] = fmaxf(x[j & 3], v);
  }
  const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  const float grow = (mx - m) * scale_log2;  // NaN while nothing is visible
  const bool moved = grow > QA_SLACK;
  float a = 1.f;
  if (moved) {
    a = qa_ex2(-grow);
    m = mx;
    l *= a;
  }
  if (__any_sync(0xffffffffu, moved) && complete()) {
#pragma unroll 1
    for (int c0 = 0; c0 < DH; c0 += 16) {
      float o[16];
      uint32_t w[16];
      tmem_ld_32x32b_x16(to + c0, o);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(o[j] * a);
      tmem_st_32x32b_x16(to + c0, w);
    }
  }
  const float mu = m == -CUDART_INF_F ? 0.f : -m * scale_log2;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c0 = 0; c0 < TC_KEYS; c0 += 16) {
    uint32_t w[8], low[8];  // a weight in two bf16 parts: off by at most 2^-18 of itself
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float p0 = qa_ex2(fmaf(s[c0 >> 4][j], scale_log2, mu));
      const float p1 = qa_ex2(fmaf(s[c0 >> 4][j + 1], scale_log2, mu));
      sum[j & 2] += p0;
      sum[(j & 2) + 1] += p1;
      const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
      w[j >> 1] = *reinterpret_cast<const uint32_t*>(&h);
      const __nv_bfloat162 r = __floats2bfloat162_rn(p0 - __low2float(h), p1 - __high2float(h));
      low[j >> 1] = *reinterpret_cast<const uint32_t*>(&r);
    }
    tmem_st_32x32b_x8(tm + c0 / 2, w);
    tmem_st_32x32b_x8(tm + TC_KEYS / 2 + c0 / 2, low);
  }
  l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  tmem_st_wait();
}

__global__ void __launch_bounds__(TC_THREADS, 2)
    q4_attn_tc_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor q, int grp, int t0, int tc, int tiles, int prows,
                      float scale_log2, int nslots, int q_vec, float* __restrict__ part_o,
                      float2* __restrict__ part_s) {
  extern __shared__ uint8_t tc_raw[];
  __shared__ int nan_from[QA_TC_CLASSES][4];  // per class and 32-feature group: the first key whose values are NaN
  pdl_wait();
  const int kvh = blockIdx.y / tiles, tile = blockIdx.y % tiles, b = blockIdx.z;
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
    return;
  }
  const int first = t0 + tile * TC_ROWS / grp;
  const int last = min(min(t0 + (tile * TC_ROWS + TC_ROWS - 1) / grp, t0 + tc - 1), count - 1);
  if (first > last) return;
  const int pmin = len + first, pmax = len + last;
  const int cl0 = qa_tc_class(pmin), cl1 = qa_tc_class(pmax);
  if (pmax < QA_TC_BEGIN || static_cast<int64_t>(blockIdx.x) * qa_tc_keys(cl0) > pmax) return;

  uint8_t* smem = tc_raw + ((1024 - (smem_u32(tc_raw) & 1023)) & 1023);
  uint8_t *qs = smem, *ks = smem + Q_BYTES, *vs = ks + STAGES * KV_BYTES;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(vs + STAGES * KV_BYTES);  // one of each a stage
  uint64_t *s_full = kv_full + STAGES, *p_full = s_full + STAGES, *pv_done = p_full + STAGES, *done = pv_done + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile uint32_t* gave_up = tmem_slot + 1;  // a wait ran out: the results are NaN
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(kv_full + i, DEC_WARPS);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, SOFT_WARPS);
      mbar_init(pv_done + i, 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
    *gave_up = 0;
  }
  if (threadIdx.x < 4 * QA_TC_CLASSES) nan_from[threadIdx.x >> 2][threadIdx.x & 3] = INT32_MAX;
  if (warp == SOFT_WARPS + DEC_WARPS) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  // the queries: 16-byte units of eight features in the order in which q4_word decodes them
  for (int i = threadIdx.x; i < TC_ROWS * 16; i += TC_THREADS) {
    const int r = i >> 4, u = i & 15, R = tile * TC_ROWS + r, t = t0 + R / grp;
    Q4Raw8<__nv_bfloat16> raw;
    if (R < tc * grp && t < count)
      raw.load(static_cast<const __nv_bfloat16*>(q.p) + b * q.sb + t * q.st + (kvh * grp + R % grp) * q.sh + 8 * u,
               q_vec != 0);
    const uint4 v = raw.w[0];
    *reinterpret_cast<uint4*>(qs + tile_at<TC_ROWS>(r, u)) =
        make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                   __byte_perm(v.y, v.w, 0x7632));
  }
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_o = tmem + TMEM_O;
  // behind the allocation: a later kernel's CTA cannot take the tensor memory that this one waits for
  pdl_trigger();
  // a warp waits until the bars' phase of step n is over (n < 0: none to wait for); false: gave up
  auto wait = [&](uint64_t* bars, int n) {
    if (n < 0) return true;
    uint64_t* bar = bars + n % STAGES;
    const uint32_t parity = n / STAGES & 1;
    for (int i = 0; i < 64; ++i)
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const bool over = *gave_up == 0 && mbar_wait_bounded(bar, parity, cache.err, EVS_K_Q4_ATTN, b);
    if (!over) *gave_up = 1;
    return __all_sync(0xffffffffu, over) != 0;
  };

  bool ok = true;
  int it = 0;  // steps so far
  for (int cl = cl0; cl <= cl1; ++cl) {
    const int kall = static_cast<int>(min(static_cast<int64_t>(pmax), qa_tc_class_end(cl) - 1)) + 1;
    if (static_cast<int64_t>(blockIdx.x) * qa_tc_keys(cl) >= kall) continue;
    const int kbeg = blockIdx.x * qa_tc_keys(cl), kend = min(kall, kbeg + qa_tc_keys(cl));
    const int steps = (kend - kbeg + TC_KEYS - 1) / TC_KEYS;

    if (warp < SOFT_WARPS) {
      const int R = tile * TC_ROWS + threadIdx.x, t = t0 + R / grp;
      const bool mine = R < tc * grp && t < count && len + t >= QA_TC_BEGIN && qa_tc_class(len + t) == cl;
      const int lim = mine ? len + t : INT32_MAX - 1;
      const bool any = __any_sync(0xffffffffu, mine);
      // keys that every row of the class sees need no mask
      const int clear = max(pmin, qa_tc_class_begin(cl)) + 1;
      const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
      float m = -CUDART_INF_F, l = 0.f;
      for (int i = 0; i < steps && ok; ++i) {
        const int key = kbeg + i * TC_KEYS, n = it + i;
        ok = wait(s_full, n);
        if (!ok) break;
        tc_fence_after();
        if (any) {
          const uint32_t tm = tmem + lanes + n % STAGES * TC_KEYS;
          auto complete = [&]() {  // the outputs of the class so far
            if (i == 0) return false;
            ok = wait(pv_done, n - 1);
            tc_fence_after();
            return ok;
          };
          if (key + TC_KEYS > clear)
            softmax_step<true>(tm, tmem_o + lanes, scale_log2, max(0, min(TC_KEYS, lim - key + 1)), m, l, complete);
          else
            softmax_step<false>(tm, tmem_o + lanes, scale_log2, TC_KEYS, m, l, complete);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + n % STAGES);
      }
      it += steps;
      if (ok) ok = wait(pv_done, it - 1);
      tc_fence_after();
      if (any) {
        const size_t prow = ((static_cast<size_t>(b) * cache.G + kvh) * prows + R) * nslots + blockIdx.x;
        if (mine) part_s[prow] = make_float2(m * scale_log2, ok ? l : CUDART_NAN_F);
#pragma unroll
        for (int c0 = 0; c0 < DH; c0 += 16) {
          float o[16];
          tmem_ld_32x32b_x16(tmem_o + lanes + c0, o);
          tmem_ld_wait();
          if (mine) {
            const bool bad = !ok || nan_from[cl][c0 / 32] <= lim;
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(part_o + prow * DH + c0 + j) =
                  bad ? make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F)
                      : make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
        tc_fence_before();
      }
    } else if (warp < SOFT_WARPS + DEC_WARPS) {
      const int dw = warp - SOFT_WARPS, P = cache.P;
      const int32_t* table = rows.table + b * rows.table_stride;
      const uint8_t* head_base = cache.block(0, kvh);
      const size_t page_bytes = static_cast<size_t>(cache.G) * cache.block_bytes;
      // lane i: page id and slot of chunk i (16 keys) of a run of 512 keys; the next run's are on their way while
      // one is used
      int page = -1, slot = 0, page_next = -1, slot_next = 0;
      bool bad = false;
      auto load_pages = [&](int key) {
        const int kk = key + 16 * lane;
        page_next = -1;
        if (kk < kend) {
          const int n = kk / P;
          slot_next = kk - n * P;
          page_next = table[n];
        }
      };
      // chunk sub of step i: whether its page is one of the pool, and its slot
      auto chunk_of = [&](int i, int sub, int* sl) {
        const int at = (4 * i + sub) & 31, id = __shfl_sync(0xffffffffu, page, at);
        *sl = __shfl_sync(0xffffffffu, slot, at);
        const bool in = kbeg + i * TC_KEYS + 16 * sub < kend;
        const bool known = static_cast<uint32_t>(id) < static_cast<uint32_t>(cache.pages);
        bad |= in && !known;
        return in && known ? id : -1;
      };
      // keys: a thread takes 32 features c of key 32 p + 8 dw + lane % 8 (p: two passes); values: eight
      // features f8 of the eight keys from k8 on
      const int c = lane >> 3, f8 = 4 * dw + (lane >> 3), k8 = 8 * (lane & 7);
      struct Raw {
        uint4 kw[2];
        uint32_t ksc[2];
        uint32_t vw[8];
        uint4 vsc;
      } raw[2];
      auto load = [&](Raw& x, int i) {
        if ((i & 7) == 0) {
          page = page_next, slot = slot_next;
          load_pages(kbeg + (i + 8) * TC_KEYS);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          int sl;
          const int id = chunk_of(i, 2 * p + (dw >> 1), &sl);
          sl += (dw & 1) * 8 + (lane & 7);
          x.kw[p] = make_uint4(0u, 0u, 0u, 0u);
          x.ksc[p] = 0x7FC0u;  // keys without a page: a NaN score for whoever sees them
          if (id >= 0) {
            const uint8_t* blk = head_base + id * page_bytes;
            x.kw[p] = q4_ld<uint4>(blk + sl * (DH / 2) + c * 16);
            x.ksc[p] = q4_ld<uint16_t>(blk + P * DH + 2 * (c * P + sl));
          }
        }
        int sl;
        const int id = chunk_of(i, k8 >> 4, &sl);
        sl += k8 & 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) x.vw[j] = 0u;
        x.vsc = make_uint4(0u, 0u, 0u, 0u);
        if (id >= 0) {
          const uint8_t* blk = head_base + id * page_bytes;
          const uint8_t* at = blk + P * (DH / 2) + sl * (DH / 2) + f8 * 4;
#pragma unroll
          for (int j = 0; j < 8; ++j) x.vw[j] = q4_ld<uint32_t>(at + j * (DH / 2));
          x.vsc = q4_ld<uint4>(blk + P * DH + P * (DH / 16) + 2 * ((f8 >> 2) * P + sl));
        }
      };
      auto decode = [&](Raw& x, int i) {
        const int key = kbeg + i * TC_KEYS, n = it + i;
        // the last keys and values of this stage are multiplied
        ok = wait(pv_done, n - STAGES);
        if (!ok) return;
        uint8_t* kst = ks + n % STAGES * KV_BYTES;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const Q4Scale s = q4_scale(x.ksc[p] | x.ksc[p] << 16);
          const int r = 32 * p + 8 * dw + (lane & 7);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t v[4];
            q4_word((&x.kw[p].x)[w], s, v);
            *reinterpret_cast<uint4*>(kst + tile_at<TC_KEYS>(r, 4 * c + w)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        if (key + TC_KEYS > kend) {
          // keys behind the last visible one hold whatever the page held: their scale becomes 0
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (key + k8 + e >= kend) (&x.vsc.x)[e >> 1] &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
        }
        if ((qa_scales_nan(x.vsc.x) | qa_scales_nan(x.vsc.y) | qa_scales_nan(x.vsc.z) | qa_scales_nan(x.vsc.w)) != 0u) {
          // a group held as NaN must not reach rows that do not see its key (0 NaN is NaN): it leaves the
          // product, and the outputs of the rows that see it are set at the end
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t& w = (&x.vsc.x)[e >> 1];
            if (((e & 1 ? w >> 16 : w) & 0x7F80u) == 0x7F80u) {
              atomicMin(&nan_from[cl][f8 >> 2], key + k8 + e);
              w &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
            }
          }
        }
        uint8_t* vst = vs + n % STAGES * KV_BYTES;
        const Q4Scale sp[4] = {q4_scale(x.vsc.x), q4_scale(x.vsc.y), q4_scale(x.vsc.z), q4_scale(x.vsc.w)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // four features of the eight keys: rows of V^T
          uint32_t o[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t v[4];
            q4_word(__byte_perm(x.vw[2 * j], x.vw[2 * j + 1], h ? 0x7632u : 0x5410u), sp[j], v);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e][j] = v[e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(vst + tile_at<DH>(8 * f8 + 4 * h + e, k8 >> 3)) =
                make_uint4(o[e][0], o[e][1], o[e][2], o[e][3]);
        }
        fence_async_smem();  // the stores before the products
        __syncwarp();
        if (lane == 0) mbar_arrive(kv_full + n % STAGES);
        load(x, i + 2);
      };
      load_pages(kbeg);
      load(raw[0], 0);
      load(raw[1], 1);
      for (int i = 0; i < steps && ok; i += 2) {
        decode(raw[0], i);
        if (ok && i + 1 < steps) decode(raw[1], i + 1);
      }
      it += steps;
      if (__any_sync(0xffffffffu, bad) && lane == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_ATTN, b);
    } else {
      const uint32_t on = lane == 0;
      const uint64_t qd = umma_desc_sw128(smem_u32(qs));
      const uint32_t high = static_cast<uint32_t>(qd >> 32), q0 = static_cast<uint32_t>(qd);
      const uint32_t k0 = static_cast<uint32_t>(umma_desc_sw128(smem_u32(ks)));
      const uint32_t v0 = static_cast<uint32_t>(umma_desc_sw128(smem_u32(vs)));
      constexpr uint32_t S_DESC = umma_idesc_bf16(TC_ROWS, TC_KEYS), O_DESC = umma_idesc_bf16(TC_ROWS, DH);
      // whatever is ready first: a step's scores (its keys are decoded, so the P in S's place is multiplied, too)
      // or the outputs of the one before
      auto ready = [&](uint64_t* bars, int n) {
        return __all_sync(0xffffffffu, mbar_try_wait(bars + n % STAGES, n / STAGES & 1)) != 0;
      };
      uint64_t idle_since = 0;
      for (int qk = 0, pv = 0, idle = 0; pv < steps;) {
        if (qk < steps && qk < pv + STAGES && ready(kv_full, it + qk)) {
          tc_fence_after();
          const uint32_t st = (it + qk) % STAGES, d = tmem + st * TC_KEYS, k = k0 + st * (KV_BYTES >> 4);
#pragma unroll
          for (int j = 0; j < DH / 16; ++j) {
            const uint32_t qa = q0 + (((j >> 2) * (TC_ROWS * 128) + (j & 3) * 32) >> 4);
            const uint32_t kb = k + (((j >> 2) * (TC_KEYS * 128) + (j & 3) * 32) >> 4);
            if (j == 0)
              mma_ss<false>(on, d, qa, kb, high, S_DESC);
            else
              mma_ss<true>(on, d, qa, kb, high, S_DESC);
          }
          mma_commit(on, smem_u32(s_full) + 8 * st);
          ++qk, idle = 0;
        } else if (pv < qk && ready(p_full, it + pv)) {
          tc_fence_after();
          const uint32_t st = (it + pv) % STAGES, p = tmem + st * TC_KEYS, v = v0 + st * (KV_BYTES >> 4);
#pragma unroll
          for (int j = 0; j < TC_KEYS / 16; ++j) {
            mma_ts(on, tmem_o, p + TC_KEYS / 2 + 8 * j, v + 2 * j, high, O_DESC, pv != 0 || j != 0);
            mma_ts(on, tmem_o, p + 8 * j, v + 2 * j, high, O_DESC, 1);
          }
          mma_commit(on, smem_u32(pv_done) + 8 * st);
          ++pv, idle = 0;
        } else if ((++idle & 255) == 0) {
          const uint64_t now = __shfl_sync(0xffffffffu, globaltimer_ns(), 0);
          if (idle == 256) idle_since = now;
          if (*gave_up != 0 || now - idle_since > EVS_WAIT_LIMIT_NS) {
            evs_record_error(cache.err, EVS_ETIMEOUT, EVS_K_Q4_ATTN, b);
            *gave_up = 1;
            break;
          }
        }
        __syncwarp();
      }
      it += steps;
    }
  }
  if (warp == SOFT_WARPS + DEC_WARPS) {
    mma_commit(lane == 0, smem_u32(done));  // no product in flight when the memory goes back
    mbar_wait_bounded(done, 0, cache.err, EVS_K_Q4_ATTN, b);
    __syncwarp();
  }
  __syncthreads();
  if (warp == SOFT_WARPS + DEC_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace

int launch_q4_attn_tc(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, int grp, int t0, int tc, int prows,
                      float scale_log2, int nslots, int q_vec, float* part_o, float2* part_s, cudaStream_t st,
                      bool pdl) {
  static std::atomic<unsigned long long> done{0};
  EVS_TRY(smem_attr_once(done, reinterpret_cast<const void*>(q4_attn_tc_kernel), TC_SMEM));
  const int tiles = (tc * grp + TC_ROWS - 1) / TC_ROWS;
  EVS_CUDA_TRY(evs_launch(q4_attn_tc_kernel, dim3(nslots, c.G * tiles, r.B), dim3(TC_THREADS), TC_SMEM, st, pdl, c, r,
                          q, grp, t0, tc, tiles, prows, scale_log2, nslots, q_vec, part_o, part_s));
  evs_count_launch(1);
  return EVS_OK;
}
