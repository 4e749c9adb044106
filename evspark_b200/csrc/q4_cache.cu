// Paged KV cache in the 4-bit format: append (position rotation, quantisation and the page write in
// one pass) and read-back.
//
//   pool  uint8 [num_pages][kv_heads][block], a block holding P = page_size tokens of one head:
//         K codes [P][D / 2] | V codes [P][D / 2] | K scales bf16 [D / 32][P] | V scales the same
//   row b's position p lives in page page_table[b][p / P], slot p % P.
//
// Every token's codes and scales are whole bytes of their own, so rows and tokens never share a
// read-modify-write.  Page ids and lengths are checked before any access: a bad one is recorded in
// the cache's error word and the token is skipped.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "internal.hpp"
#include "q4.cuh"
#include "q4_cache.hpp"

namespace {

constexpr int APP_THREADS = 256;
constexpr int FEW_TOKENS = 296;  // two CTAs an SM
constexpr int FREQ_MAX = 64;  // head_dim / 2 at most

struct RopeFreq {
  double f[FREQ_MAX];
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], bool vec) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = from_f32<T>(v[j]);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v);
    *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(v + 4);
  }
}

// Scale and codes of a group are decided in fp32 wherever that cannot differ from 64 bits, else in 64
// bits.  Scale: t = absmax / 7 in fp32 is within 2^-22 of the exact quotient, so its five-bit rounding
// is the exact one unless the dropped 19 bits lie within 4 units of a half (one group in 2^15).
// Codes: the quotient x / s, corrected once by its remainder, is within 2^-21 of the exact one (half an
// ulp at 4 .. 8 is 2^-22, and the correction is off by less than that); |x / s| <= 7 (1 + 1/32) < 7.5, so
// its rounding needs no clamp.  It is a half exactly where x is, and its rounding is the exact one unless
// it lies within 2^-15 of a half.  Keys, rotated in 64 bits, are looked at again
// there.  Values are x themselves and may sit on a half.  Those of bf16 need no look at all: x = a 2^e
// and s = b 2^f with a < 2^8 and b < 2^5, so a quotient above 0.49 that is not a half is at least
// 1 / (2 max(b, a / 0.49)) > 2^-11 away from one.
__device__ __forceinline__ bool scale_clear(float absmax) {
  const float t = absmax * (1.f / 7.f);
  return (__float_as_uint(t) & 0x7FFFFu) - 0x3FFFCu > 8u && t >= 2.f * Q4_TINY && t <= 0.5f * Q4_HUGE;
}
__device__ __forceinline__ uint32_t scale_bits_fast(float absmax) {
  return (__float_as_uint(absmax * (1.f / 7.f)) + 0x40000u) >> 19 << 3;  // five significant bits, as bf16 bits
}
// Codes of eight values under scale s (inv = 1 / s to 2^-22), value j's at bit 4 j, and the largest
// distance from a code's value so far.  Adding 1.5 2^23 leaves the rounded quotient in the low bits;
// the sum's other bits add up to one constant.
enum Look { LOOK_NONE, LOOK_VALUES, LOOK_ALL };  // distances: none, but exact halves, every one
template <Look LOOK>
__device__ __forceinline__ uint32_t codes_fast(const float (&x)[8], float s, float inv, float& far) {
  constexpr float SHIFT = 12582912.f;
  uint32_t w = 0;
#pragma unroll
  for (int j = 7; j >= 0; --j) {
    float q = x[j] * inv;
    q = fmaf(fmaf(-q, s, x[j]), inv, q);
    const float y = q + SHIFT;
    if constexpr (LOOK != LOOK_NONE) {
      const float d = fabsf(q - (y - SHIFT));
      far = LOOK == LOOK_VALUES && d == 0.5f ? far : fmaxf(far, d);
    }
    w = w * 16u + __float_as_uint(y);
  }
  return w - (0x4B400000u - 8u) * 0x11111111u;
}

// One CTA per token (and block of head rows, where the call has few tokens).  D / 16 threads per head
// row, each holding the features 8 i .. 8 i + 7 of the row's lower half and of its upper half (the
// pairs that the rotation turns).  Rows 0 .. H - 1 are queries, then G keys, then G values.  Angles
// and rotation in 64 bits (2 of the 64 fma a clock that an SM has per value: not what bounds this), so
// that a key's codes are those of its exact rotation.  The next head row's loads are in flight while one
// is worked on (69.5 us instead of 78.1 for eight rows of up to 1,024 tokens, 32 heads of 128, bf16; about
// 2.3 TB/s): instructions bound it, 0.69 issued a clock and scheduler, 30 per value.  13 tokens: 6.3 us, a
// chain of latencies.
template <typename T>
__global__ void __launch_bounds__(APP_THREADS, 4)
    q4_append_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor q, Q4Tensor k, Q4Tensor v, Q4Tensor q_out, int H,
                     int vec, const __grid_constant__ RopeFreq freq) {
  pdl_trigger();
  __shared__ double2 turn[8][FREQ_MAX / 8];  // cos, sin of feature 8 i + j at [j][i]
  pdl_wait();
  const int b = blockIdx.x / rows.T, t = blockIdx.x - b * rows.T;
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
    return;
  }
  if (t >= count) return;
  const int D = cache.D, half = D / 2, G = cache.G;
  const int pos = len + t;
  const int tpr_log = D == 128 ? 3 : (D == 64 ? 2 : 1), per = APP_THREADS >> tpr_log;
  const int total = H + 2 * G;
  const int i = threadIdx.x & ((1 << tpr_log) - 1);
  int r = blockIdx.y * per + (threadIdx.x >> tpr_log);
  const T* q_at = static_cast<const T*>(q.p) + b * q.sb + t * q.st + 8 * i;
  const T* k_at = static_cast<const T*>(k.p) + b * k.sb + t * k.st + 8 * i;
  const T* v_at = static_cast<const T*>(v.p) + b * v.sb + t * v.st + 8 * i;
  Q4Raw8<T> next_lo, next_hi;
  auto load = [&](int row) {
    if (row >= total) return;
    const T* p = row < H ? q_at + row * q.sh : (row < H + G ? k_at + (row - H) * k.sh : v_at + (row - H - G) * v.sh);
    next_lo.load(p, vec != 0);
    next_hi.load(p + half, vec != 0);
  };
  load(r);  // on its way while the angles are computed, as is the page
  const int64_t page = q4_page(cache, rows, b, pos);
  const int slot = pos % cache.P;
  if (threadIdx.x < half && static_cast<int>(blockIdx.y) * per < H + G) {
    double s, c;
    sincos(static_cast<double>(pos) * freq.f[threadIdx.x], &s, &c);
    turn[threadIdx.x & 7][threadIdx.x >> 3] = make_double2(c, s);
  }
  __syncthreads();
  if (page < 0 && threadIdx.x == 0 && blockIdx.y == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
  // rows of one pass share the count of passes, so that whole warps meet the shuffles below
  for (int r0 = blockIdx.y * per; r0 < total; r0 += gridDim.y * per, r += gridDim.y * per) {
    const bool live = r < total, is_q = r < H, is_k = !is_q && r < H + G;
    const int head = is_q ? r : (is_k ? r - H : r - H - G);
    float lo[8], hi[8];
    next_lo.get(lo);
    next_hi.get(hi);
    load(r + gridDim.y * per);  // on its way while this row is worked on
    if (is_q || is_k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double2 cs = turn[j][i];
        const double a = lo[j], d = hi[j];
        lo[j] = static_cast<float>(a * cs.x - d * cs.y);
        hi[j] = static_cast<float>(d * cs.x + a * cs.y);
      }
    }
    // the values in 64 bits (keys: read and rotated again, where fp32 does not decide)
    auto exact = [&](int j, double& l, double& h) {
      l = lo[j];
      h = hi[j];
      if (!is_k) return;
      const double a = to_f32<T>(k_at[head * k.sh + j]), d = to_f32<T>(k_at[head * k.sh + half + j]);
      const double2 cs = turn[j][i];
      l = a * cs.x - d * cs.y;
      h = d * cs.x + a * cs.y;
    };
    if (live && is_q) {
      T* o = static_cast<T*>(q_out.p) + b * q_out.sb + t * q_out.st + head * q_out.sh + 8 * i;
      store8<T>(o, lo, vec != 0);
      store8<T>(o + half, hi, vec != 0);
    }
    const bool put = live && !is_q && page >= 0;
    if (!__any_sync(0xffffffffu, put)) continue;  // a warp of queries
    // groups of 32 features: four threads of one half (D = 64, 128), or both halves of two threads (D = 32)
    auto group_max = [&](auto& ml, auto& mh, auto larger) {
      if (D == 32) ml = mh = larger(ml, mh);
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        if (D == 32 && o == 2) break;
        ml = larger(ml, __shfl_xor_sync(0xffffffffu, ml, o));
        mh = larger(mh, __shfl_xor_sync(0xffffffffu, mh, o));
      }
    };
    // magnitudes as integers: the same order, with NaN on top (x 0 is one for a NaN and an infinity)
    float xl = 0.f, xh = 0.f, zl = 0.f, zh = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xl = fmaxf(xl, fabsf(lo[j]));
      xh = fmaxf(xh, fabsf(hi[j]));
      zl = fmaf(lo[j], 0.f, zl);
      zh = fmaf(hi[j], 0.f, zh);
    }
    uint32_t bl = zl == 0.f ? __float_as_uint(xl) : 0x7FC00000u, bh = zh == 0.f ? __float_as_uint(xh) : 0x7FC00000u;
    group_max(bl, bh, [](uint32_t a, uint32_t o) { return max(a, o); });
    const float ml = __uint_as_float(bl), mh = __uint_as_float(bh);
    uint32_t sl = scale_bits_fast(ml), sh = scale_bits_fast(mh);
    if (__any_sync(0xffffffffu, put && !(scale_clear(ml) && scale_clear(mh)))) {
      double el = 0.0, eh = 0.0;
      auto larger = [](double a, double o) { return (a != a || a >= o) ? a : o; };  // a NaN wins
      if (put) {
        for (int j = 0; j < 8; ++j) {
          double l, h;
          exact(j, l, h);
          el = larger(el, fabs(l));
          eh = larger(eh, fabs(h));
        }
      }
      group_max(el, eh, larger);
      sl = q4_scale_bits(el);
      sh = q4_scale_bits(eh);
    }
    if (put) {
      const float fl = __uint_as_float(sl << 16), fh = __uint_as_float(sh << 16);
      float il, ih;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(il) : "f"(fl));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ih) : "f"(fh));
      uint32_t cl, ch;
      float far = 0.f;
      if (is_k) {
        cl = codes_fast<LOOK_ALL>(lo, fl, il, far);
        ch = codes_fast<LOOK_ALL>(hi, fh, ih, far);
      } else {
        constexpr Look LOOK = sizeof(T) == 2 ? LOOK_NONE : LOOK_VALUES;
        cl = codes_fast<LOOK>(lo, fl, il, far);
        ch = codes_fast<LOOK>(hi, fh, ih, far);
      }
      // a scale of 0 or NaN makes every quotient infinite or NaN: the codes are 8
      const bool odd = !(ml <= FLT_MAX) || !(mh <= FLT_MAX) || sl == 0u || sh == 0u || sl == 0x7FC0u || sh == 0x7FC0u;
      if (far >= 0.5f - 0x1p-15f || odd) {
        cl = ch = 0;
        for (int j = 0; j < 8; ++j) {
          double l, h;
          exact(j, l, h);
          cl |= q4_code(l, sl) << (4 * j);
          ch |= q4_code(h, sh) << (4 * j);
        }
      }
      uint8_t* block = cache.block(page, head);
      uint8_t* codes = block + (is_k ? 0 : cache.P * (D / 2)) + slot * (D / 2);
      *reinterpret_cast<uint32_t*>(codes + 4 * i) = cl;
      *reinterpret_cast<uint32_t*>(codes + half / 2 + 4 * i) = ch;
      uint16_t* scales = reinterpret_cast<uint16_t*>(block + cache.P * D) + (is_k ? 0 : cache.P * (D / 32)) + slot;
      if (D == 32) {
        if (i == 0) scales[0] = static_cast<uint16_t>(sl);
      } else if (i % 4 == 0) {
        scales[(i / 4) * cache.P] = static_cast<uint16_t>(sl);
        scales[(i / 4 + D / 64) * cache.P] = static_cast<uint16_t>(sh);
      }
    }
  }
}

// One thread per eight values of K or V: the values that the cache holds at lengths[b] + t.  A CTA takes TOK
// tokens of a row, with four loads of each on their way per thread.  Eight rows of up to 1,024 tokens, 32
// heads of 128: 27 us with two tokens a CTA, 31.6 with one (a CTA waits for length, page and codes in turn, then stores).
template <typename T, int TOK>
__global__ void __launch_bounds__(APP_THREADS)
    q4_read_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor k, Q4Tensor v, int vec) {
  pdl_trigger();
  pdl_wait();
  const int runs = (rows.T + TOK - 1) / TOK, b = blockIdx.x / runs, t0 = (blockIdx.x - b * runs) * TOK;
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
    return;
  }
  if (t0 >= count) return;
  const int D = cache.D, G = cache.G, log8 = D == 128 ? 4 : (D == 64 ? 3 : 2);
  int64_t page[TOK];
  int slot[TOK];
#pragma unroll
  for (int x = 0; x < TOK; ++x) {
    const int pos = len + t0 + x;
    page[x] = t0 + x < count ? q4_page(cache, rows, b, pos) : -1;
    slot[x] = pos % cache.P;
    if (page[x] < 0 && t0 + x < count && threadIdx.x == 0)
      evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
  }
  const int units = 2 * G << log8;
  constexpr int BATCH = 4;
  for (int i0 = blockIdx.y * APP_THREADS * BATCH + threadIdx.x; i0 < units; i0 += gridDim.y * APP_THREADS * BATCH) {
    uint32_t codes[TOK][BATCH], sb[TOK][BATCH];
#pragma unroll
    for (int x = 0; x < TOK; ++x)
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + u * APP_THREADS, row = i >> log8, w = i & ((1 << log8) - 1);
        if (i >= units || page[x] < 0) continue;
        const bool is_v = row >= G;
        const uint8_t* block = cache.block(page[x], is_v ? row - G : row);
        codes[x][u] = q4_ld<uint32_t>(block + (is_v ? cache.P * (D / 2) : 0) + slot[x] * (D / 2) + 4 * w);
        sb[x][u] = q4_ld<uint16_t>(block + cache.P * D +
                                   2 * ((is_v ? cache.P * (D / 32) : 0) + (w >> 2) * cache.P + slot[x]));
      }
#pragma unroll
    for (int x = 0; x < TOK; ++x)
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + u * APP_THREADS, row = i >> log8, w = i & ((1 << log8) - 1);
        if (i >= units || page[x] < 0) continue;
        const float s = __uint_as_float(sb[x][u] << 16);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (static_cast<int>((codes[x][u] >> (4 * j)) & 15u) - 8) * s;
        const Q4Tensor& dst = row >= G ? v : k;
        store8<T>(static_cast<T*>(dst.p) + b * dst.sb + (t0 + x) * dst.st + (row >= G ? row - G : row) * dst.sh + 8 * w,
                  y, vec != 0);
      }
  }
}

}  // namespace

namespace {
struct Dim {
  int64_t stride, x, y;  // sizes in the two tensors
};
// whether off = sum of t_k stride_k + r with -(y_k - 1) <= t_k <= x_k - 1 and |r| < D: an element of the first
// tensor that is one of the second, off elements behind it.  dim: largest strides first.
bool meet(int64_t off, const Dim* dim, int n, int D) {
  if (n == 0) return off > -D && off < D;
  int64_t low = -(D - 1), high = D - 1;  // of the dimensions behind this one
  for (int i = 1; i < n; ++i) low -= (dim[i].y - 1) * dim[i].stride, high += (dim[i].x - 1) * dim[i].stride;
  auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); };
  const int64_t first = std::max(-(dim[0].y - 1), -floor_div(high - off, dim[0].stride));
  const int64_t last = std::min(dim[0].x - 1, floor_div(off - low, dim[0].stride));
  if (last - first >= 8) return true;  // interleaved beyond what is worth telling apart
  for (int64_t t = first; t <= last; ++t)
    if (meet(off - t * dim[0].stride, dim + 1, n - 1, D)) return true;
  return false;
}
}  // namespace

bool q4_distinct(const Q4Tensor& x, int B, int T, int heads, int D) {
  Dim dim[3] = {{x.sb, B, 1}, {x.st, T, 1}, {x.sh, heads, 1}};
  std::sort(dim, dim + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  int64_t least = D;
  for (const Dim& d : dim) {
    if (d.x <= 1) continue;
    if (d.stride < least) return false;
    least = d.stride * d.x;
  }
  return true;
}

bool q4_share(const Q4Tensor& x, int x_heads, const Q4Tensor& y, int y_heads, int B, int T, int D, size_t el) {
  const int64_t e = static_cast<int64_t>(el), px = reinterpret_cast<intptr_t>(x.p), py = reinterpret_cast<intptr_t>(y.p);
  auto reach = [&](const Q4Tensor& t, int heads, int64_t p, int64_t* lo, int64_t* hi) {
    *lo = p, *hi = p + D * e;
    const int64_t last[3] = {(B - 1) * t.sb * e, (T - 1) * t.st * e, (heads - 1) * t.sh * e};
    for (int64_t d : last) (d < 0 ? *lo : *hi) += d;
  };
  int64_t x0, x1, y0, y1;
  reach(x, x_heads, px, &x0, &x1);
  reach(y, y_heads, py, &y0, &y1);
  if (x1 <= y0 || y1 <= x0) return false;
  // spans that meet: views of one buffer are told apart where their strides are the same
  const int64_t all[3][4] = {{x.sb, y.sb, B, B}, {x.st, y.st, T, T}, {x.sh, y.sh, x_heads, y_heads}};
  Dim dim[3];
  int n = 0;
  for (const auto& d : all) {
    if (d[2] <= 1 && d[3] <= 1) continue;
    if (d[2] > 1 && d[3] > 1 && d[0] != d[1]) return true;
    dim[n++] = {d[2] > 1 ? d[0] : d[1], d[2], d[3]};
    if (dim[n - 1].stride <= 0) return true;
  }
  if ((py - px) % e != 0) return true;
  std::sort(dim, dim + n, [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
  return meet((py - px) / e, dim, n, D);
}

int q4_check_cache(const evs_q4_cache* c) {
  EVS_CHECK_ARG(c != nullptr && c->pool != nullptr, "null argument");
  EVS_CHECK_ARG(c->head_dim == 32 || c->head_dim == 64 || c->head_dim == 128, "q4 cache: head_dim must be 32, 64 or 128");
  EVS_CHECK_ARG(c->page_size >= 16 && c->page_size <= 4096 && c->page_size % 16 == 0,
                "q4 cache: page_size must be a multiple of 16 in [16, 4096]");
  EVS_CHECK_ARG(c->kv_heads >= 1 && c->num_pages >= 1 && c->num_pages <= INT32_MAX,
                "q4 cache: needs kv_heads >= 1 and num_pages in [1, 2^31)");
  EVS_CHECK_ARG(reinterpret_cast<uintptr_t>(c->pool) % 16 == 0, "q4 cache: the pool must be 16-byte aligned");
  return EVS_OK;
}

int q4_check_rows(const evs_q4_cache* c, const evs_q4_rows* r) {
  EVS_CHECK_ARG(r != nullptr && r->page_table != nullptr && r->lengths != nullptr, "null argument");
  EVS_CHECK_ARG(r->batch >= 1 && r->tokens >= 1 && r->max_pages >= 1 && r->table_stride >= r->max_pages,
                "q4 cache: needs batch, tokens and max_pages >= 1 and table_stride >= max_pages");
  EVS_CHECK_ARG(static_cast<int64_t>(r->batch) * r->tokens <= INT32_MAX, "q4 cache: too many tokens in one call");
  EVS_CHECK_RANGE(static_cast<int64_t>(r->max_pages) * c->page_size <= (1ll << 30),
                  "q4 cache: a page table holds at most 2^30 positions");
  return EVS_OK;
}

Q4CacheDev q4_cache_dev(const evs_q4_cache* c) {
  Q4CacheDev d;
  d.pool = static_cast<uint8_t*>(c->pool);
  d.err = reinterpret_cast<EvsDevErr*>(c->err);
  d.pages = c->num_pages;
  d.P = c->page_size;
  d.G = c->kv_heads;
  d.D = c->head_dim;
  d.block_bytes = c->page_size * c->head_dim + c->page_size * c->head_dim / 8;
  return d;
}

Q4RowsDev q4_rows_dev(const evs_q4_rows* r) {
  return {r->page_table, r->lengths, r->counts, r->table_stride, r->max_pages, r->batch, r->tokens};
}

int launch_q4_append(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, const Q4Tensor& k, const Q4Tensor& v,
                     const Q4Tensor& q_out, int H, int dtype, double rope_base, cudaStream_t st, bool pdl) {
  const size_t el = dtype == EVS_DTYPE_BF16 ? 2 : 4;
  const int vec = q4_vec(k, el) && q4_vec(v, el) && q4_vec(q, el) && q4_vec(q_out, el);
  // the frequencies of the last (base, head size), which a caller rarely changes: 64 powers take 2.5 us
  thread_local double f_base = 0.0;
  thread_local int f_dim = 0;
  thread_local RopeFreq f;
  if (f_base != rope_base || f_dim != c.D) {
    for (int j = 0; j < c.D / 2; ++j) f.f[j] = std::pow(rope_base, -2.0 * j / c.D);
    f_base = rope_base;
    f_dim = c.D;
  }
  const int per = APP_THREADS / (c.D / 16);
  // few tokens: their head rows over several CTAs; many: one CTA a token, so that the angles of a token are computed
  // once (32 / 32 heads of 128: 13 tokens 6.9 us instead of 8.0, 208 8.8 instead of 10.5, 312 10.5 instead of 12.3,
  // but 832 19.0 instead of 17.5; 64 / 8 heads: 208 8.3 instead of 8.7, 416 11.8 instead of 10.6)
  const int tokens = r.B * r.T;
  dim3 grid(tokens, tokens >= FEW_TOKENS ? 1 : (H + 2 * c.G + per - 1) / per);
  EVS_CHECK_ARG(grid.y <= 65535, "q4 append: too many heads");
  auto* kern = dtype == EVS_DTYPE_BF16 ? q4_append_kernel<__nv_bfloat16> : q4_append_kernel<float>;
  EVS_CUDA_TRY(evs_launch(kern, grid, dim3(APP_THREADS), 0, st, pdl, c, r, q, k, v, q_out, H, vec, f));
  evs_count_launch(1);
  return EVS_OK;
}

int launch_q4_read(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& k, const Q4Tensor& v, int dtype,
                   cudaStream_t st) {
  const size_t el = dtype == EVS_DTYPE_BF16 ? 2 : 4;
  const int vec = q4_vec(k, el) && q4_vec(v, el);
  const bool few = static_cast<int64_t>(r.B) * r.T < 4 * FEW_TOKENS;
  const int runs = few ? r.T : (r.T + 1) / 2;
  const dim3 grid(r.B * runs, few ? (2 * c.G * (c.D / 8) + 4 * APP_THREADS - 1) / (4 * APP_THREADS) : 1);
  EVS_CHECK_ARG(grid.y <= 65535, "q4 read: too many heads");
  auto* kern = dtype == EVS_DTYPE_BF16 ? (few ? q4_read_kernel<__nv_bfloat16, 1> : q4_read_kernel<__nv_bfloat16, 2>)
                                       : (few ? q4_read_kernel<float, 1> : q4_read_kernel<float, 2>);
  EVS_CUDA_TRY(evs_launch(kern, grid, dim3(APP_THREADS), 0, st, true, c, r, k, v, vec));
  evs_count_launch(1);
  return EVS_OK;
}

namespace {
Q4Tensor tensor_of(void* p, const int64_t* s) { return {p, s[0], s[1], s[2]}; }
Q4Tensor tensor_of(const void* p, const int64_t* s) { return {const_cast<void*>(p), s[0], s[1], s[2]}; }
}  // namespace

extern "C" {

int evs_q4_kv_append(const evs_q4_cache* cache, const evs_q4_rows* rows, const void* k, const int64_t* k_strides,
                     const void* v, const int64_t* v_strides, const void* q, const int64_t* q_strides, void* q_out,
                     const int64_t* q_out_strides, int n_heads, int dtype, double rope_base, cudaStream_t st) {
  EVS_TRY(q4_check_cache(cache));
  EVS_TRY(q4_check_rows(cache, rows));
  EVS_CHECK_ARG(k && v && k_strides && v_strides, "null argument");
  EVS_CHECK_ARG(dtype == EVS_DTYPE_BF16 || dtype == EVS_DTYPE_FP32, "q4 append: k, v and q must be fp32 or bf16");
  EVS_CHECK_ARG((q != nullptr) == (q_out != nullptr), "q4 append: q and q_out come together");
  EVS_CHECK_ARG(q == nullptr || (q_strides && q_out_strides && n_heads >= 1), "q4 append: q needs strides and heads");
  EVS_CHECK_ARG(rope_base > 0.0 && std::isfinite(rope_base), "q4 append: rope_base must be positive");
  const Q4Tensor tk = tensor_of(k, k_strides), tv = tensor_of(v, v_strides);
  const Q4Tensor tq = q != nullptr ? tensor_of(q, q_strides) : tk, to = q != nullptr ? tensor_of(q_out, q_out_strides) : tk;
  if (q != nullptr) {
    const int B = rows->batch, T = rows->tokens, G = cache->kv_heads, D = cache->head_dim;
    const size_t el = dtype == EVS_DTYPE_BF16 ? 2 : 4;
    const bool in_place = q == q_out && tq.sb == to.sb && tq.st == to.st && tq.sh == to.sh;
    EVS_CHECK_ARG(q4_distinct(to, B, T, n_heads, D), "q4 append: elements of q_out overlap");
    EVS_CHECK_ARG((in_place || !q4_share(to, n_heads, tq, n_heads, B, T, D, el)) &&
                      !q4_share(to, n_heads, tk, G, B, T, D, el) && !q4_share(to, n_heads, tv, G, B, T, D, el),
                  "q4 append: q_out overlaps another tensor of the call");
  }
  return launch_q4_append(q4_cache_dev(cache), q4_rows_dev(rows), tq, tk, tv, to, q != nullptr ? n_heads : 0, dtype,
                          rope_base, st, true);
}

int evs_q4_kv_read(const evs_q4_cache* cache, const evs_q4_rows* rows, void* k, const int64_t* k_strides, void* v,
                   const int64_t* v_strides, int dtype, cudaStream_t st) {
  EVS_TRY(q4_check_cache(cache));
  EVS_TRY(q4_check_rows(cache, rows));
  EVS_CHECK_ARG(k && v && k_strides && v_strides, "null argument");
  EVS_CHECK_ARG(dtype == EVS_DTYPE_BF16 || dtype == EVS_DTYPE_FP32, "q4 read: k and v must be fp32 or bf16");
  const Q4Tensor tk = tensor_of(k, k_strides), tv = tensor_of(v, v_strides);
  const int B = rows->batch, T = rows->tokens, G = cache->kv_heads, D = cache->head_dim;
  EVS_CHECK_ARG(q4_distinct(tk, B, T, G, D) && q4_distinct(tv, B, T, G, D) &&
                    !q4_share(tk, G, tv, G, B, T, D, dtype == EVS_DTYPE_BF16 ? 2 : 4),
                "q4 read: elements of k and v overlap");
  return launch_q4_read(q4_cache_dev(cache), q4_rows_dev(rows), tk, tv, dtype, st);
}

}  // extern "C"
