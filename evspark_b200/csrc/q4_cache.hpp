// Device views of the paged 4-bit KV cache, shared by q4_cache.cu and q4_attention.cu.
#pragma once

#include <cstring>

#include "common.cuh"

struct Q4CacheDev {
  uint8_t* pool;
  EvsDevErr* err;
  int64_t pages;
  int P, G, D;
  int block_bytes;  // one page of one head
  __host__ __device__ uint8_t* block(int64_t page, int head) const {
    return pool + (static_cast<size_t>(page) * G + head) * block_bytes;
  }
};

struct Q4RowsDev {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* counts;  // null: every row has T new tokens
  int64_t table_stride;
  int max_pages, B, T;
};

// a [B, T, heads, D] tensor: strides in elements, D contiguous
struct Q4Tensor {
  void* p;
  int64_t sb, st, sh;
};

// whether eight values at a time can be moved as 16-byte words
inline bool q4_vec(const Q4Tensor& x, size_t el) {
  return reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && (x.sb * el) % 16 == 0 && (x.st * el) % 16 == 0 &&
         (x.sh * el) % 16 == 0;
}
// eight values as they lie in memory
template <typename T>
struct Q4Raw8 {
  uint4 w[sizeof(T) / 2] = {};
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = p[j];
      memcpy(w, e, sizeof(w));
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = (&w[0].x)[j];
        v[2 * j] = __uint_as_float(x << 16);
        v[2 * j + 1] = __uint_as_float(x & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float((&w[j / 4].x)[j % 4]);
    }
  }
};
template <typename T>
__device__ __forceinline__ void q4_load8(float (&v)[8], const T* p, bool vec) {
  Q4Raw8<T> r;
  r.load(p, vec);
  r.get(v);
}

// row b's length and its new tokens; false when they lie outside the page table's positions or T
__device__ __forceinline__ bool q4_row(const Q4RowsDev& r, int b, int* len, int* count, int P) {
  *len = r.lengths[b];
  *count = r.counts != nullptr ? r.counts[b] : r.T;
  return *len >= 0 && *count >= 0 && *count <= r.T &&
         static_cast<int64_t>(*len) + *count <= static_cast<int64_t>(r.max_pages) * P;
}

// page of position pos (inside the table), or -1 when the table's entry is no page of the pool
__device__ __forceinline__ int64_t q4_page(const Q4CacheDev& c, const Q4RowsDev& r, int b, int64_t pos) {
  const int32_t id = r.table[b * r.table_stride + pos / c.P];
  return id >= 0 && id < c.pages ? id : -1;
}

// [B, T, heads, D] tensors (D contiguous): whether an output's elements are distinct, and whether two tensors may
// share one (views of one buffer with the same strides, as q, k and v of a fused projection are, are told apart).
bool q4_distinct(const Q4Tensor& x, int B, int T, int heads, int D);
bool q4_share(const Q4Tensor& x, int x_heads, const Q4Tensor& y, int y_heads, int B, int T, int D, size_t el);
int q4_check_cache(const evs_q4_cache* c);
int q4_check_rows(const evs_q4_cache* c, const evs_q4_rows* r);
Q4CacheDev q4_cache_dev(const evs_q4_cache* c);
Q4RowsDev q4_rows_dev(const evs_q4_rows* r);
int launch_q4_append(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& q, const Q4Tensor& k, const Q4Tensor& v,
                     const Q4Tensor& q_out, int H, int dtype, double rope_base, cudaStream_t st, bool pdl);
int launch_q4_read(const Q4CacheDev& c, const Q4RowsDev& r, const Q4Tensor& k, const Q4Tensor& v, int dtype,
                   cudaStream_t st);
