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
#include <cmath>

#include "internal.hpp"
#include "q4.cuh"
#include "q4_cache.hpp"

namespace {

constexpr int APP_THREADS = 256;
constexpr int FREQ_MAX = 64;  // head_dim / 2 at most

struct RopeFreq {
  double f[FREQ_MAX];
};

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, bool vec) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(p[j]);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = (&r.x)[j];
      v[2 * j] = __uint_as_float(w << 16);
      v[2 * j + 1] = __uint_as_float(w & 0xFFFF0000u);
    }
  } else {
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(p + 4);
  }
}
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

// One CTA per (token, block of head rows).  D / 16 threads per head row, each holding the features
// 8 i .. 8 i + 7 of the row's lower half and of its upper half (the pairs that the rotation turns).
// Rows 0 .. H - 1 are queries, then G keys, then G values.
template <typename T>
__global__ void __launch_bounds__(APP_THREADS)
    q4_append_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor q, Q4Tensor k, Q4Tensor v, Q4Tensor q_out, int H,
                     int vec, const __grid_constant__ RopeFreq freq) {
  pdl_trigger();
  __shared__ double cs[FREQ_MAX], sn[FREQ_MAX];
  pdl_wait();
  const int b = blockIdx.x / rows.T, t = blockIdx.x % rows.T;
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
    return;
  }
  if (t >= count) return;
  const int D = cache.D, half = D / 2, G = cache.G;
  const int64_t pos = static_cast<int64_t>(len) + t;
  if (threadIdx.x < half) sincos(static_cast<double>(pos) * freq.f[threadIdx.x], &sn[threadIdx.x], &cs[threadIdx.x]);
  __syncthreads();
  const int64_t page = q4_page(cache, rows, b, pos);
  const int tpr = D / 16, per = APP_THREADS / tpr;
  const int r = blockIdx.y * per + threadIdx.x / tpr, i = threadIdx.x % tpr;
  const bool live = r < H + 2 * G;
  if (page < 0 && threadIdx.x == 0 && blockIdx.y == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
  float lo[8], hi[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) lo[j] = hi[j] = 0.f;
  const bool is_q = r < H, is_k = !is_q && r < H + G;
  const int head = is_q ? r : (is_k ? r - H : r - H - G);
  if (live) {
    const Q4Tensor& src = is_q ? q : (is_k ? k : v);
    const T* p = static_cast<const T*>(src.p) + b * src.sb + t * src.st + head * src.sh + 8 * i;
    load8<T>(lo, p, vec != 0);
    load8<T>(hi, p + half, vec != 0);
  }
  double xl[8], xh[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    xl[j] = lo[j];
    xh[j] = hi[j];
    if (is_q || is_k) {
      const double c = cs[8 * i + j], s = sn[8 * i + j];
      const double a = xl[j] * c - xh[j] * s, d = xh[j] * c + xl[j] * s;
      xl[j] = a;
      xh[j] = d;
    }
  }
  if (live && is_q) {
    T* o = static_cast<T*>(q_out.p) + b * q_out.sb + t * q_out.st + head * q_out.sh + 8 * i;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = static_cast<float>(xl[j]);
      hi[j] = static_cast<float>(xh[j]);
    }
    store8<T>(o, lo, vec != 0);
    store8<T>(o + half, hi, vec != 0);
  }
  // groups of 32 features: four threads of one half (D = 64, 128), or both halves of two threads (D = 32)
  double ml = 0.0, mh = 0.0;
  auto larger = [](double a, double o) { return (a != a || a >= o) ? a : o; };  // a NaN wins
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    ml = larger(ml, fabs(xl[j]));
    mh = larger(mh, fabs(xh[j]));
  }
  if (D == 32) ml = mh = larger(ml, mh);
  const int width = D == 32 ? 2 : 4;
  for (int o = 1; o < width; o <<= 1) {
    ml = larger(ml, __shfl_xor_sync(0xffffffffu, ml, o));
    mh = larger(mh, __shfl_xor_sync(0xffffffffu, mh, o));
  }
  if (!live || is_q || page < 0) return;
  const uint32_t sl = q4_scale_bits(ml), sh = q4_scale_bits(mh);
  uint32_t cl = 0, ch = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    cl |= q4_code(xl[j], sl) << (4 * j);
    ch |= q4_code(xh[j], sh) << (4 * j);
  }
  const int slot = static_cast<int>(pos % cache.P);
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

// One thread per eight values of K or V: the values that the cache holds at lengths[b] + t.
template <typename T>
__global__ void __launch_bounds__(APP_THREADS)
    q4_read_kernel(Q4CacheDev cache, Q4RowsDev rows, Q4Tensor k, Q4Tensor v, int vec) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / rows.T, t = blockIdx.x % rows.T;
  int len, count;
  if (!q4_row(rows, b, &len, &count, cache.P)) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
    return;
  }
  if (t >= count) return;
  const int D = cache.D, G = cache.G, per = D / 8;
  const int64_t pos = static_cast<int64_t>(len) + t;
  const int64_t page = q4_page(cache, rows, b, pos);
  if (page < 0) {
    if (threadIdx.x == 0) evs_record_error(cache.err, EVS_ERANGE, EVS_K_Q4_CACHE, b);
    return;
  }
  const int slot = static_cast<int>(pos % cache.P);
  for (int i = threadIdx.x; i < 2 * G * per; i += APP_THREADS) {
    const bool is_k = i < G * per;
    const int head = (is_k ? i : i - G * per) / per, w = i % per;
    const uint8_t* block = cache.block(page, head);
    const uint32_t codes =
        *reinterpret_cast<const uint32_t*>(block + (is_k ? 0 : cache.P * (D / 2)) + slot * (D / 2) + 4 * w);
    const uint16_t sb = (reinterpret_cast<const uint16_t*>(block + cache.P * D))[(is_k ? 0 : cache.P * (D / 32)) +
                                                                                 (w / 4) * cache.P + slot];
    const float s = __uint_as_float(static_cast<uint32_t>(sb) << 16);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (static_cast<int>((codes >> (4 * j)) & 15u) - 8) * s;
    const Q4Tensor& dst = is_k ? k : v;
    store8<T>(static_cast<T*>(dst.p) + b * dst.sb + t * dst.st + head * dst.sh + 8 * w, x, vec != 0);
  }
}

bool vec_ok(const Q4Tensor& x, size_t el) {
  return reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && (x.sb * el) % 16 == 0 && (x.st * el) % 16 == 0 &&
         (x.sh * el) % 16 == 0;
}

}  // namespace

int q4_check_cache(const evs_q4_cache* c) {
  EVS_CHECK_ARG(c != nullptr && c->pool != nullptr, "null argument");
  EVS_CHECK_ARG(c->head_dim == 32 || c->head_dim == 64 || c->head_dim == 128, "q4 cache: head_dim must be 32, 64 or 128");
  EVS_CHECK_ARG(c->page_size >= 16 && c->page_size <= 4096 && c->page_size % 16 == 0,
                "q4 cache: page_size must be a multiple of 16 in [16, 4096]");
  EVS_CHECK_ARG(c->kv_heads >= 1 && c->num_pages >= 1, "q4 cache: needs kv_heads >= 1 and num_pages >= 1");
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
  const Q4CacheDev c = q4_cache_dev(cache);
  const size_t el = dtype == EVS_DTYPE_BF16 ? 2 : 4;
  const int H = q != nullptr ? n_heads : 0;
  const Q4Tensor tk = tensor_of(k, k_strides), tv = tensor_of(v, v_strides);
  const Q4Tensor tq = q != nullptr ? tensor_of(q, q_strides) : tk, to = q != nullptr ? tensor_of(q_out, q_out_strides) : tk;
  const int vec = vec_ok(tk, el) && vec_ok(tv, el) && vec_ok(tq, el) && vec_ok(to, el);
  RopeFreq f;
  for (int j = 0; j < c.D / 2; ++j) f.f[j] = std::pow(rope_base, -2.0 * j / c.D);
  const int per = APP_THREADS / (c.D / 16);
  dim3 grid(rows->batch * rows->tokens, (H + 2 * c.G + per - 1) / per);
  EVS_CHECK_ARG(grid.y <= 65535, "q4 append: too many heads");
  if (dtype == EVS_DTYPE_BF16)
    q4_append_kernel<__nv_bfloat16><<<grid, APP_THREADS, 0, st>>>(c, q4_rows_dev(rows), tq, tk, tv, to, H, vec, f);
  else
    q4_append_kernel<float><<<grid, APP_THREADS, 0, st>>>(c, q4_rows_dev(rows), tq, tk, tv, to, H, vec, f);
  EVS_CUDA_TRY(cudaGetLastError());
  evs_count_launch(1);
  return EVS_OK;
}

int evs_q4_kv_read(const evs_q4_cache* cache, const evs_q4_rows* rows, void* k, const int64_t* k_strides, void* v,
                   const int64_t* v_strides, int dtype, cudaStream_t st) {
  EVS_TRY(q4_check_cache(cache));
  EVS_TRY(q4_check_rows(cache, rows));
  EVS_CHECK_ARG(k && v && k_strides && v_strides, "null argument");
  EVS_CHECK_ARG(dtype == EVS_DTYPE_BF16 || dtype == EVS_DTYPE_FP32, "q4 read: k and v must be fp32 or bf16");
  const Q4CacheDev c = q4_cache_dev(cache);
  const size_t el = dtype == EVS_DTYPE_BF16 ? 2 : 4;
  const Q4Tensor tk = tensor_of(k, k_strides), tv = tensor_of(v, v_strides);
  const int vec = vec_ok(tk, el) && vec_ok(tv, el);
  const int grid = rows->batch * rows->tokens;
  if (dtype == EVS_DTYPE_BF16)
    q4_read_kernel<__nv_bfloat16><<<grid, APP_THREADS, 0, st>>>(c, q4_rows_dev(rows), tk, tv, vec);
  else
    q4_read_kernel<float><<<grid, APP_THREADS, 0, st>>>(c, q4_rows_dev(rows), tk, tv, vec);
  EVS_CUDA_TRY(cudaGetLastError());
  evs_count_launch(1);
  return EVS_OK;
}

}  // extern "C"
