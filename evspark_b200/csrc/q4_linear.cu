// Tokens times a weight held in 4 bits: y[m][n] = sum_k x[m][k] (c[n][k] - 8) s[k / group][n].
//
//   codes  uint8 [N][Kp / 2], two input features per byte (even one in the low half), Kp = K rounded
//          up to 128 with codes of 8 (zeros) behind K
//   scales bf16 [Kp / group][N]
#include <algorithm>
#include <cstring>

#include "internal.hpp"
#include "q4.cuh"

namespace {

constexpr int LIN_WARPS = 8;
constexpr int LIN_THREADS = 32 * LIN_WARPS;
// CTAs an SM: two wherever registers and shared memory allow it, so that the grid is resident at once
template <typename TX, int NT>
constexpr int lin_per_sm() {
  return NT * (sizeof(TX) == 2 ? 1 : 3) <= 6 ? 2 : 1;
}
constexpr int LIN_CLUSTER = 8;    // CTAs of one output tile at most (splits of K)
// rows of a tile that one CTA of the cluster adds up
__host__ __device__ constexpr int lin_own_rows(int rows, int splits) { return ((rows + splits - 1) / splits + 7) / 8 * 8; }

// x staged in shared memory in the order in which the products read it: per (K block, 8-token
// tile, part) four words of 16 bytes per lane; lane (n, c) word w holds features 32 c + 8 w .. + 7 of
// token n as pairs (0,4) (1,5) (2,6) (3,7), the order in which q4_word decodes a weight word.  Word w
// of lane l sits at l ^ 2 w, so that the eight lanes of one store phase (two c, four w) meet eight
// different 16-byte bank groups; reads stay a permutation of 32 lanes.
__device__ __forceinline__ uint4 pair_up(uint4 v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

template <typename TX, int NT>
__device__ __forceinline__ void stage_x(uint4* xs, const TX* x, int64_t ldx, int M, int K, int m0, int kb0,
                                        int nkb, bool vec) {
  constexpr int NP = sizeof(TX) == 2 ? 1 : 3, NR = NP == 1 ? 1 : 2;
  constexpr int TPB = LIN_THREADS / 16;                   // tokens that the CTA loads at once
  constexpr int KSTEP = TPB > 8 * NT ? TPB / (8 * NT) : 1;  // ... or K blocks
  constexpr int BATCH = NP == 1 ? 4 : 2;                  // loads of a thread in flight
  const int u = threadIdx.x & 15, c = u >> 2, w = u & 3, row = threadIdx.x >> 4;
  for (int n = row % (8 * NT); n < 8 * NT; n += TPB) {
    const bool live = m0 + n < M;
    const TX* src = x + static_cast<int64_t>(m0 + n) * ldx + 8 * u;
    uint4* dst = xs + ((n >> 3) * NP * 4 + w) * 32 + (((n & 7) * 4 + c) ^ (2 * w));
    for (int kb = row / (8 * NT); kb < nkb; kb += BATCH * KSTEP) {
      uint4 raw[BATCH][NR];
#pragma unroll
      for (int r = 0; r < BATCH; ++r) {
        const int k0 = (kb0 + kb + r * KSTEP) * Q4_KBLOCK, k = k0 + 8 * u;
#pragma unroll
        for (int h = 0; h < NR; ++h) raw[r][h] = make_uint4(0u, 0u, 0u, 0u);
        if (kb + r * KSTEP >= nkb || !live) continue;
        if (vec && k + 8 <= K) {
#pragma unroll
          for (int h = 0; h < NR; ++h) raw[r][h] = reinterpret_cast<const uint4*>(src + k0)[h];
        } else if (k < K) {
          TX e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = k + j < K ? src[k0 + j] : from_f32<TX>(0.f);
          memcpy(raw[r], e, sizeof(e));
        }
      }
#pragma unroll
      for (int r = 0; r < BATCH; ++r) {
        if (kb + r * KSTEP >= nkb) break;
        uint4* d = dst + (kb + r * KSTEP) * (NT * NP * 4 * 32);
        if constexpr (NP == 1) {
          *d = pair_up(raw[r][0]);
        } else {
          uint32_t p[8][3];
#pragma unroll
          for (int j = 0; j < 8; ++j) q4_parts(__uint_as_float((&raw[r][j >> 2].x)[j & 3]), p[j]);
#pragma unroll
          for (int q = 0; q < 3; ++q)
            d[q * 4 * 32] = make_uint4(p[0][q] | p[4][q] << 16, p[1][q] | p[5][q] << 16, p[2][q] | p[6][q] << 16,
                                       p[3][q] | p[7][q] << 16);
        }
      }
    }
  }
}

struct LinTile {  // one warp's share of a K block: 32 rows x 128 features
  uint4 w[4];     // rows g, g + 8, g + 16, g + 24, features 32 c .. 32 c + 31
  uint32_t s[4];
};

// the weight streams through once: no space in L1 (volatile, so that it stays behind the wait)
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// Weight rows are the product's 16-row operand and tokens its 8-column one: a warp takes 32 rows x 128
// features a step against every token of the tile, so the codes are decoded once, in the registers that
// the product reads.  What it takes: 420 warp instructions per 4,096 codes (192 of them shifts,
// masks and fma of the decode), 0.44 issued a clock and scheduler: 16 warps an SM wait for their codes, products and
// decode.  13 x 22016 x 4096, group 64: 19.8 us, 2.4 TB/s of codes and scales (floor 7.5 us at 6.5 TB/s);
// 13 x 8192 x 22528: 34.3 us; 1 x 4096 x 4096: 6.3 us (5.6 with the weight in L2); 32 x 4096 x 4096: 12.3 us.
// bf16 rows add all product steps of a warp's K blocks to one fp32 accumulator, which the product cuts instead of
// rounding: 6.7e-7 of the result at 13 x 8192 x 22528.  A sum of its own for each block, as fp32 rows have, brings
// 1.0e-7 but costs 2 to 7 % at up to 16 tokens and 11 to 22 % beyond (its registers spill), so it is left out.
// grid (K splits = cluster, row tiles, token tiles).  Registers hold the next two K blocks' codes
// while one is multiplied; the first ones are on their way before x is staged.
template <typename TX, typename TO, int NT, int KW>
__global__ void __launch_bounds__(LIN_THREADS, lin_per_sm<TX, NT>())
    q4_linear_kernel(const TX* x, int64_t ldx, int M, const uint8_t* codes, const uint16_t* scales, int N, int K,
                     int group_shift, TO* out, int64_t ldo, int chunk_kb, int vec, int wait_first, uint32_t red_offset) {
  constexpr int NP = sizeof(TX) == 2 ? 1 : 3;
  constexpr int LIN_ROWS = 32 * LIN_WARPS / KW, LIN_KW = KW;
  extern __shared__ __align__(16) unsigned char lin_sm[];
  cluster_arrive_relaxed();
  pdl_trigger();
  if (wait_first != 0) pdl_wait();  // the weight itself may be an earlier kernel's
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int wr = warp % (LIN_WARPS / KW), wk = warp / (LIN_WARPS / KW);
  const int S = gridDim.x, rank = blockIdx.x;
  const int n0 = blockIdx.y * LIN_ROWS, m0 = blockIdx.z * 8 * NT;
  const int KB = (K + Q4_KBLOCK - 1) / Q4_KBLOCK;
  const int kb_begin = static_cast<int>(static_cast<int64_t>(KB) * rank / S);
  const int kb_end = static_cast<int>(static_cast<int64_t>(KB) * (rank + 1) / S);
  const size_t row_bytes = static_cast<size_t>(KB) * (Q4_KBLOCK / 2);
  // 32-bit offsets from the row tile's uniform base (its rows span less than 2^32 bytes)
  const uint8_t* base = codes + static_cast<size_t>(n0) * row_bytes;
  const uint8_t* sbase = reinterpret_cast<const uint8_t*>(scales + n0);
  uint32_t off[4], soff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t r = min(32 * wr + g + 8 * i, N - 1 - n0);
    off[i] = r * static_cast<uint32_t>(row_bytes) + 16 * c;
    soff[i] = 2 * r;
  }
  auto load = [&](LinTile& t, int kb) {
    if (kb >= kb_end) return;
    const uint32_t so = static_cast<uint32_t>((kb * Q4_KBLOCK + 32 * c) >> group_shift) * (2u * N);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.w[i] = ld_stream(base + (off[i] + static_cast<uint32_t>(kb) * (Q4_KBLOCK / 2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) t.s[i] = q4_ld<uint16_t>(sbase + (soff[i] + so));
  };

  float acc[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;

  LinTile t0, t1;
  load(t0, kb_begin + wk);
  load(t1, kb_begin + wk + LIN_KW);
  uint4* xs = reinterpret_cast<uint4*>(lin_sm);
  pdl_wait();
  for (int kc = kb_begin; kc < kb_end; kc += chunk_kb) {
    const int nkb = min(chunk_kb, kb_end - kc);
    if (kc != kb_begin) __syncthreads();
    stage_x<TX, NT>(xs, x, ldx, M, K, m0, kc, nkb, vec != 0);
    __syncthreads();
    auto multiply = [&](const LinTile& t, int kb) {
      Q4Scale s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = q4_scale(t.s[i] | t.s[i] << 16);
      const uint4* xb = xs + kb * NT * NP * 4 * 32;
      // three-part fp32 rows: a block's 24 product steps are summed apart, as each step truncates
      float part[2][NT][4];
      if constexpr (NP > 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[i][j][e] = 0.f;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q4_word((&t.w[i].x)[w], s[i], a[i]);
        // products of one sum apart from each other: a product takes 20 cycles to follow itself
        constexpr int JB = NT < 2 ? NT : 2;
#pragma unroll
        for (int j0 = 0; j0 < NT; j0 += JB)
#pragma unroll
          for (int q = NP - 1; q >= 0; --q) {
            uint4 b[JB];
#pragma unroll
            for (int j = 0; j < JB; ++j) b[j] = xb[(((j0 + j) * NP + q) * 4 + w) * 32 + (lane ^ (2 * w))];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < JB; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float(&d)[4] = NP > 1 ? part[i][j0 + j] : acc[i][j0 + j];
                  q4_mma(d, a[2 * i][2 * h], a[2 * i + 1][2 * h], a[2 * i][2 * h + 1], a[2 * i + 1][2 * h + 1],
                         h ? b[j].z : b[j].x, h ? b[j].w : b[j].y);
                }
          }
      }
      if constexpr (NP > 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] += part[i][j][e];
      }
    };
    // a tile's registers are loaded again as soon as it is multiplied (no copies: a move of a
    // register that a load still fills would wait for it); chunks hold an even number of tiles a warp
    for (int kb = wk; kb < nkb; kb += 2 * LIN_KW) {
      multiply(t0, kb);
      load(t0, kc + kb + 2 * LIN_KW);
      if (kb + LIN_KW < nkb) {
        multiply(t1, kb + LIN_KW);
        load(t1, kc + kb + 3 * LIN_KW);
      }
    }
  }
  // Sums over the K warps and the cluster's splits, in that order.  Rank r owns RC rows of the output
  // tile; every CTA pushes its sums into the owner's [split][K warp][row][token] slots, which alias
  // nothing that a slower CTA still reads, so one cluster barrier is enough.  A thread's tokens of a row
  // lie side by side there (place c 2 NT + 2 j + e holds token 8 j + 2 c + e), so that remote stores are
  // wide: 13 x 4096 x 4096 takes 7.3 us, 8.1 with stores of 4 bytes.
  constexpr int TOK = 8 * NT;
  const int RC = lin_own_rows(LIN_ROWS, S);
  const uint32_t red = smem_u32(lin_sm) + red_offset;
  cluster_wait();  // every CTA of the cluster has started
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 32 * wr + 16 * i + 8 * h, owner = r / RC;  // RC is a multiple of 8
      uint32_t a;
      asm("mapa.shared::cluster.u32 %0, %1, %2;"
          : "=r"(a)
          : "r"(red + 4 * (((rank * KW + wk) * RC + r - owner * RC + g) * TOK + c * 2 * NT)), "r"(owner));
      if constexpr (NT == 1) {
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(acc[i][0][2 * h]), "f"(acc[i][0][2 * h + 1])
                     : "memory");
      } else {
#pragma unroll
        for (int j = 0; j < NT; j += 2)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a + 8 * j), "f"(acc[i][j][2 * h]),
                       "f"(acc[i][j][2 * h + 1]), "f"(acc[i][j + 1][2 * h]), "f"(acc[i][j + 1][2 * h + 1])
                       : "memory");
      }
    }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const float4* mine = reinterpret_cast<const float4*>(lin_sm + red_offset);
  constexpr int UNITS = TOK / 4;  // of a row
  const int tokens = min(TOK, M - m0), first = rank * RC, own_rows = min(RC, min(LIN_ROWS, N - n0) - first);
  for (int i = threadIdx.x; i < own_rows * UNITS; i += LIN_THREADS) {
    const int r = i / UNITS, u = i % UNITS;
    float4 v[LIN_CLUSTER][KW];
#pragma unroll
    for (int p = 0; p < LIN_CLUSTER; ++p)
#pragma unroll
      for (int q = 0; q < KW; ++q)
        v[p][q] = p < S ? mine[((p * KW + q) * RC + r) * UNITS + u] : make_float4(0.f, 0.f, 0.f, 0.f);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < LIN_CLUSTER; ++p)
      if (p < S) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float part = (&v[p][0].x)[e];
#pragma unroll
          for (int q = 1; q < KW; ++q) part += (&v[p][q].x)[e];
          sum[e] += part;
        }
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = 4 * u + e, tok = at % (2 * NT) / 2 * 8 + at / (2 * NT) * 2 + (at & 1);
      if (tok < tokens) out[static_cast<int64_t>(m0 + tok) * ldo + n0 + first + r] = from_f32<TO>(sum[e]);
    }
  }
}

template <typename TX, typename TO, int NT, int KW>
int launch_linear_kw(const void* x, int64_t ldx, int M, const void* codes, const void* scales, int N, int K, int group,
                     void* out, int64_t ldo, int S, cudaStream_t st, bool pdl, bool wait_first) {
  constexpr int NP = sizeof(TX) == 2 ? 1 : 3, ROWS = 32 * LIN_WARPS / KW;
  const int tiles = (N + ROWS - 1) / ROWS, KB = (K + Q4_KBLOCK - 1) / Q4_KBLOCK;
  const int block_bytes = NT * NP * 2048;  // staged x of one K block
  const int slice = (KB + S - 1) / S;
  // a multiple of 2 KW blocks: whichever the chunk, a K warp takes the same blocks in the same registers
  const int red_bytes = S * KW * 8 * NT * lin_own_rows(ROWS, S) * 4;
  const int room = (lin_per_sm<TX, NT>() == 2 ? 96 * 1024 : 200 * 1024) - red_bytes;  // some L1 left for the scales
  int chunk = std::max(2 * KW, room / block_bytes / (2 * KW) * (2 * KW));
  chunk = std::min(chunk, slice);
  const int red_offset = chunk * block_bytes, smem = red_offset + red_bytes;
  auto* kern = q4_linear_kernel<TX, TO, NT, KW>;
  static std::atomic<unsigned long long> done{0};
  EVS_TRY(smem_attr_once(done, reinterpret_cast<const void*>(kern), 227 * 1024));
  const int vec = (reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * sizeof(TX)) % 16 == 0) ? 1 : 0;
  const int ztiles = (M + 8 * NT - 1) / (8 * NT);
  EVS_CHECK_ARG(tiles <= 65535 && ztiles <= 65535, "q4 linear: too many rows or tokens");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, tiles, ztiles);
  cfg.blockDim = dim3(LIN_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  EVS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<const TX*>(x), ldx, M, static_cast<const uint8_t*>(codes),
                                  static_cast<const uint16_t*>(scales), N, K, group == 32 ? 5 : (group == 64 ? 6 : 7),
                                  static_cast<TO*>(out), ldo, chunk, vec, wait_first ? 1 : 0,
                                  static_cast<uint32_t>(red_offset)));
  evs_count_launch(1);
  return EVS_OK;
}

template <typename TX, typename TO, int NT>
int launch_linear_nt(const void* x, int64_t ldx, int M, const void* codes, const void* scales, int N, int K, int group,
                     void* out, int64_t ldo, cudaStream_t st, bool pdl, bool wait_first) {
  const int KB = (K + Q4_KBLOCK - 1) / Q4_KBLOCK;
  // From N and K alone, so that a token's sums do not depend on the other tokens: 256 rows per CTA
  // where that leaves enough CTAs (13 x N x 4096: 9.4 us instead of 10.1 with 128 at N = 7,168, 13.7 instead of
  // 16.3 at 12,288, 19.8 instead of 29.9 at 22,016; but 9.5 instead of 9.3 at 6,144, 9.1 instead of 7.6 at 4,096 and
  // 18.7 instead of 13.0 at 13 x 4096 x 11008), and as many splits of K as keep every cluster resident at once: two
  // CTAs an SM, of whose 296 places clusters of up to eight fill 256 to 258 at the sizes above.
  const int KW = N >= 6400 ? 1 : 2;
  const int tiles = (N + 256 / KW - 1) / (256 / KW);
  const int S = std::max(1, std::min({LIN_CLUSTER, 264 / tiles, KB / KW}));
  if (KW == 1)
    return launch_linear_kw<TX, TO, NT, 1>(x, ldx, M, codes, scales, N, K, group, out, ldo, S, st, pdl, wait_first);
  return launch_linear_kw<TX, TO, NT, 2>(x, ldx, M, codes, scales, N, K, group, out, ldo, S, st, pdl, wait_first);
}

template <typename TX, typename TO>
int launch_linear_t(const void* x, int64_t ldx, int M, const void* codes, const void* scales, int N, int K, int group,
                    void* out, int64_t ldo, cudaStream_t st, bool pdl, bool wait_first) {
  if (M <= 8) return launch_linear_nt<TX, TO, 1>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl, wait_first);
  if (M <= 16) return launch_linear_nt<TX, TO, 2>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl, wait_first);
  // tokens beyond one tile's read the weight again: tiles of 64 would leave one CTA an SM (64 tokens x 4096 x
  // 4096 then take 35 us, and 64 x 8192 x 22528 145, instead of 22 and 109)
  return launch_linear_nt<TX, TO, 4>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl, wait_first);
}

// one warp per (row, group): codes and scale of the group's features (K padded with zeros)
template <typename TW>
__global__ void q4_quantize_kernel(const TW* __restrict__ w, int64_t ldw, int N, int K, int group,
                                   uint8_t* __restrict__ codes, uint16_t* __restrict__ scales) {
  const int groups = (K + Q4_KBLOCK - 1) / Q4_KBLOCK * Q4_KBLOCK / group;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  if (i >= static_cast<int64_t>(N) * groups) return;
  const int n = static_cast<int>(i / groups), gi = static_cast<int>(i % groups), lane = threadIdx.x & 31;
  const int per = group / 32;  // 1, 2 or 4 features a lane
  float v[4];
  float m = 0.f;
  bool bad = false;
  for (int j = 0; j < per; ++j) {
    const int k = gi * group + lane * per + j;
    v[j] = k < K ? to_f32<TW>(w[static_cast<int64_t>(n) * ldw + k]) : 0.f;
    bad |= !(fabsf(v[j]) <= 3.4e38f);
    m = fmaxf(m, fabsf(v[j]));
  }
  m = warp_max(m);
  const uint32_t s = __any_sync(0xffffffffu, bad) ? 0x7FC0u : q4_scale_bits(static_cast<double>(m));
  uint32_t c[4];
  for (int j = 0; j < per; ++j) c[j] = q4_code(static_cast<double>(v[j]), s);
  uint8_t* dst = codes + static_cast<size_t>(n) * (groups * static_cast<size_t>(group) / 2) +
                 static_cast<size_t>(gi) * (group / 2);
  if (per == 1) {
    const uint32_t other = __shfl_down_sync(0xffffffffu, c[0], 1);
    if ((lane & 1) == 0) dst[lane / 2] = static_cast<uint8_t>(c[0] | other << 4);
  } else {
    for (int j = 0; j < per; j += 2) dst[(lane * per + j) / 2] = static_cast<uint8_t>(c[j] | c[j + 1] << 4);
  }
  if (lane == 0) scales[static_cast<size_t>(gi) * N + n] = static_cast<uint16_t>(s);
}

// one thread per 16 codes of a row: 16 values
template <typename TO>
__global__ void __launch_bounds__(256)
    q4_decode_kernel(const uint8_t* codes, const uint16_t* scales, int N, int K, int group_shift, TO* out,
                     int64_t ldo, int vec) {
  pdl_trigger();
  pdl_wait();
  const int units = (K + 15) / 16;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(N) * units) return;
  const int n = static_cast<int>(i / units), k = static_cast<int>(i - static_cast<int64_t>(n) * units) * 16;
  const size_t row_bytes = static_cast<size_t>((K + Q4_KBLOCK - 1) / Q4_KBLOCK) * (Q4_KBLOCK / 2);
  const uint2 w = q4_ld<uint2>(codes + n * row_bytes + k / 2);
  const float s = __uint_as_float(static_cast<uint32_t>(scales[static_cast<size_t>(k >> group_shift) * N + n]) << 16);
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = (static_cast<int>(((j < 8 ? w.x : w.y) >> (4 * (j & 7))) & 15u) - 8) * s;
  TO* dst = out + n * ldo + k;
  if (vec && k + 16 <= K) {
    TO t[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = from_f32<TO>(v[j]);
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(t) / 16); ++j)
      reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(t)[j];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (k + j < K) dst[j] = from_f32<TO>(v[j]);
  }
}

}  // namespace

int q4_check_weight(const void* codes, const void* scales, int N, int K, int group) {
  EVS_CHECK_ARG(codes && scales, "null argument");
  EVS_CHECK_ARG(N >= 1 && K >= 1 && K <= (1 << 24), "q4 weight: N and K must be at least 1 (K at most 2^24)");
  EVS_CHECK_ARG(static_cast<int64_t>(N) * K <= (1ll << 35), "q4 weight: at most 2^35 values");
  EVS_CHECK_ARG(group == 32 || group == 64 || group == 128, "q4 weight: group must be 32, 64 or 128");
  EVS_CHECK_ARG(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "q4 weight: codes must be 16-byte aligned");
  EVS_CHECK_ARG(reinterpret_cast<uintptr_t>(scales) % 2 == 0, "q4 weight: scales must be 2-byte aligned");
  return EVS_OK;
}

int launch_q4_linear(const void* x, int x_dtype, int64_t ldx, int M, const void* codes, const void* scales, int N, int K,
                     int group, void* out, int out_dtype, int64_t ldo, cudaStream_t st, bool pdl, bool wait_first) {
  if (x_dtype == EVS_DTYPE_BF16) {
    if (out_dtype == EVS_DTYPE_BF16)
      return launch_linear_t<__nv_bfloat16, __nv_bfloat16>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl,
                                                           wait_first);
    return launch_linear_t<__nv_bfloat16, float>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl, wait_first);
  }
  if (out_dtype == EVS_DTYPE_BF16)
    return launch_linear_t<float, __nv_bfloat16>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl, wait_first);
  return launch_linear_t<float, float>(x, ldx, M, codes, scales, N, K, group, out, ldo, st, pdl, wait_first);
}

int launch_q4_decode(const void* codes, const void* scales, int N, int K, int group, void* out, int out_dtype,
                     int64_t ldo, cudaStream_t st, bool pdl) {
  const int64_t blocks = (static_cast<int64_t>(N) * ((K + 15) / 16) + 255) / 256;
  EVS_CHECK_ARG(blocks <= INT32_MAX, "q4 dequantize: too many values");
  const int shift = group == 32 ? 5 : (group == 64 ? 6 : 7);
  const size_t el = out_dtype == EVS_DTYPE_BF16 ? 2 : 4;
  const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldo * el) % 16 == 0;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (out_dtype == EVS_DTYPE_BF16)
    EVS_CUDA_TRY(evs_launch(q4_decode_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, pdl,
                            static_cast<const uint8_t*>(codes), static_cast<const uint16_t*>(scales), N, K, shift,
                            static_cast<__nv_bfloat16*>(out), ldo, vec));
  else
    EVS_CUDA_TRY(evs_launch(q4_decode_kernel<float>, grid, dim3(256), 0, st, pdl, static_cast<const uint8_t*>(codes),
                            static_cast<const uint16_t*>(scales), N, K, shift, static_cast<float*>(out), ldo, vec));
  evs_count_launch(1);
  return EVS_OK;
}

extern "C" {

int evs_q4_linear(const void* x, int x_dtype, int64_t ldx, int M, const void* codes, const void* scales, int N, int K,
                  int group, void* out, int out_dtype, int64_t ldo, cudaStream_t st) {
  EVS_CHECK_ARG(x && out, "null argument");
  EVS_TRY(q4_check_weight(codes, scales, N, K, group));
  EVS_CHECK_ARG(x_dtype == EVS_DTYPE_BF16 || x_dtype == EVS_DTYPE_FP32, "q4 linear: x must be fp32 or bf16");
  EVS_CHECK_ARG(out_dtype == EVS_DTYPE_BF16 || out_dtype == EVS_DTYPE_FP32, "q4 linear: out must be fp32 or bf16");
  EVS_CHECK_ARG(M >= 1 && ldx >= K && ldo >= N, "q4 linear: needs M >= 1, ldx >= K and ldo >= N");
  const size_t xa = x_dtype == EVS_DTYPE_BF16 ? 2 : 4, oa = out_dtype == EVS_DTYPE_BF16 ? 2 : 4;
  EVS_CHECK_ARG(reinterpret_cast<uintptr_t>(x) % xa == 0 && reinterpret_cast<uintptr_t>(out) % oa == 0,
                "q4 linear: misaligned pointer");
  const char *x0 = static_cast<const char*>(x), *o0 = static_cast<const char*>(out);
  EVS_CHECK_ARG(x0 + ((M - 1) * ldx + K) * xa <= o0 || o0 + ((M - 1) * ldo + N) * oa <= x0, "q4 linear: out overlaps x");
  // launched while the kernel before it ends (it waits for that one before it reads anything): calls behind each
  // other take 20.1 us instead of 22.5 at 13 x 22016 x 4096
  return launch_q4_linear(x, x_dtype, ldx, M, codes, scales, N, K, group, out, out_dtype, ldo, st, true, true);
}

int evs_q4_quantize(const void* w, int dtype, int64_t ldw, int N, int K, int group, void* codes, void* scales,
                    cudaStream_t st) {
  EVS_CHECK_ARG(w != nullptr, "null argument");
  EVS_TRY(q4_check_weight(codes, scales, N, K, group));
  EVS_CHECK_ARG(dtype == EVS_DTYPE_BF16 || dtype == EVS_DTYPE_FP32, "q4 quantize: w must be fp32 or bf16");
  EVS_CHECK_ARG(ldw >= K, "q4 quantize: needs ldw >= K");
  const int64_t groups = static_cast<int64_t>(N) * ((K + Q4_KBLOCK - 1) / Q4_KBLOCK * Q4_KBLOCK / group);
  const int64_t blocks = (groups + 7) / 8;
  EVS_CHECK_ARG(blocks <= INT32_MAX, "q4 quantize: too many groups");
  if (dtype == EVS_DTYPE_BF16)
    q4_quantize_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), 256, 0, st>>>(
        static_cast<const __nv_bfloat16*>(w), ldw, N, K, group, static_cast<uint8_t*>(codes), static_cast<uint16_t*>(scales));
  else
    q4_quantize_kernel<float><<<static_cast<unsigned>(blocks), 256, 0, st>>>(
        static_cast<const float*>(w), ldw, N, K, group, static_cast<uint8_t*>(codes), static_cast<uint16_t*>(scales));
  EVS_CUDA_TRY(cudaGetLastError());
  evs_count_launch(1);
  return EVS_OK;
}

int evs_q4_dequantize(const void* codes, const void* scales, int N, int K, int group, void* out, int out_dtype,
                      int64_t ldo, cudaStream_t st) {
  EVS_CHECK_ARG(out != nullptr, "null argument");
  EVS_TRY(q4_check_weight(codes, scales, N, K, group));
  EVS_CHECK_ARG(out_dtype == EVS_DTYPE_BF16 || out_dtype == EVS_DTYPE_FP32, "q4 dequantize: out must be fp32 or bf16");
  EVS_CHECK_ARG(ldo >= K, "q4 dequantize: needs ldo >= K");
  return launch_q4_decode(codes, scales, N, K, group, out, out_dtype, ldo, st, false);
}

}  // extern "C"
