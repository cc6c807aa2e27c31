// Products of activations and weights in 8-bit integers.
//
//   s_t = max(|x_t|, 1e-10) / 127       c_tk = rint(x_tk / s_t), halves to even
//   y_tn = s_t s_n sum_k c_tk q_nk + b_n            gated: silu(y_tn) y_t,n+F, n < F
//
// The sums are whole numbers below 2^31 (K <= 133144), so their order changes nothing; scales and bias are applied in fp32 and the result is rounded once.
//
// int8_rows_kernel      rows of activations into codes and scales
// int8_few_kernel       up to 64 rows: weight bytes bound it; weights go from memory straight into the fragments of warp-level products
// int8_tile_kernel      more rows: tiles of 256 x 256 on CTA pairs, tcgen05 kind::i8
#include "cta_pair.cuh"
#include "gemm_common.cuh"
#include "once_per_device.h"

namespace inv {

// What the entry is given; sizes in elements.
struct Int8Call {
  const void* x;             // [T, K] bf16 or fp32, ldx apart; null: codes and sx are given
  const int8_t* q;           // [N, K], ldw apart: rows on 16-byte boundaries
  const float* sw;           // [N]
  const void* bias;          // [N] bf16 or fp32, or null
  void* out;                 // [T, N] or gated [T, N / 2], bf16 or fp32, ldo apart
  int8_t* codes;             // [T, K], ldc apart: rows on 16-byte boundaries
  float* sx;                 // [T]
  int* status;
  void* stream;
  int64_t T, N, K, ldx, ldw, ldo, ldc, x_f32, out_f32, bias_f32, gated;
};

// ---------------------------------------------------------------------------------------------- rows into codes
constexpr float INT8_LEAST = 1e-10f;

// rint(x / s), halves to even, |x| <= 127 s: the quotient's whole part is near x * inv, and x against the border s (n + 1/2) is one rounded product-sum, whose
// sign is exact.
__device__ __forceinline__ int int8_code(float x, float s, float inv) {
  const float n = floorf(x * inv);
  const float d = fmaf(-s, n + 0.5f, x);
  const int i = (int)n;
  return d > 0.f || (d == 0.f && (i & 1)) ? i + 1 : i;
}

template <typename T>
__device__ __forceinline__ float int8_as_float(T v);
template <>
__device__ __forceinline__ float int8_as_float(float v) { return v; }
template <>
__device__ __forceinline__ float int8_as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// A CTA takes a row; VEC: rows on 16-byte boundaries. A row with a value that is not finite gets NaN for its scale.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) int8_rows_kernel(const T* __restrict__ x, long ldx, int K, int8_t* __restrict__ codes, long ldc, float* __restrict__ sx) {
  constexpr int PER = 16 / sizeof(T);
  __shared__ uint32_t sh[8];
  release_next();
  const T* row = x + (long)blockIdx.x * ldx;
  int8_t* to = codes + (long)blockIdx.x * ldc;
  const int tid = threadIdx.x, vecs = VEC ? K / PER : 0;
  uint32_t top = 0;                                       // bits of the largest |x|: not a number is above infinity is above the rest
  for (int i = tid; i < vecs; i += 256) {
    const uint4 v = reinterpret_cast<const uint4*>(row)[i];
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int j = 0; j < PER; ++j) top = max(top, __float_as_uint(int8_as_float(e[j])) & 0x7fffffffu);
  }
  for (int i = vecs * PER + tid; i < K; i += 256) top = max(top, __float_as_uint(int8_as_float(row[i])) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) sh[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, sh[i]);
  const bool finite = top < 0x7f800000u;
  const float s = finite ? __fdiv_rn(fmaxf(__uint_as_float(top), INT8_LEAST), 127.f) : __uint_as_float(0x7fc00000u);
  const float inv = finite ? __frcp_rn(s) : 0.f;
  if (tid == 0) sx[blockIdx.x] = s;
  for (int i = tid; i < vecs; i += 256) {
    const uint4 v = reinterpret_cast<const uint4*>(row)[i];
    const T* e = reinterpret_cast<const T*>(&v);
    uint32_t w[PER / 4];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t c = finite ? (uint32_t)int8_code(int8_as_float(e[j]), s, inv) & 255u : 0u;
      w[j / 4] = j % 4 ? w[j / 4] | c << (8 * (j % 4)) : c;
    }
    if constexpr (PER == 8) reinterpret_cast<uint2*>(to)[i] = make_uint2(w[0], w[1]);
    else reinterpret_cast<uint32_t*>(to)[i] = w[0];
  }
  for (int i = vecs * PER + tid; i < K; i += 256) to[i] = finite ? (int8_t)int8_code(int8_as_float(row[i]), s, inv) : (int8_t)0;
}

static int launch_int8_rows(const Int8Call& c, cudaStream_t st) {
  const int size = c.x_f32 ? 4 : 2;
  const bool vec = ((uintptr_t)c.x | (uintptr_t)(c.T > 1 ? c.ldx * size : 0)) % 16 == 0;
#define INV_ROWS(E, V) int8_rows_kernel<E, V><<<(unsigned)c.T, 256, 0, st>>>((const E*)c.x, c.ldx, (int)c.K, c.codes, c.ldc, c.sx)
  if (c.x_f32) {
    if (vec) INV_ROWS(float, true);
    else INV_ROWS(float, false);
  } else {
    if (vec) INV_ROWS(__nv_bfloat16, true);
    else INV_ROWS(__nv_bfloat16, false);
  }
#undef INV_ROWS
  return -(int)cudaGetLastError();
}

__device__ __forceinline__ float int8_silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }

// ---------------------------------------------------------------------------------------------- up to 64 rows
struct Int8Few {
  const int8_t *codes, *q;
  const float *sx, *sw;
  const void* bias;
  void* out;
  long ldc, ldw, ldo;
  int T, N, K, cols, tiles;        // cols: output columns
  int bias_f32, out_f32;
};

__device__ __forceinline__ void int8_mma(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 int8_stream(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// Sixteen codes of which only the first n exist.
__device__ __forceinline__ uint4 int8_mask(uint4 v, int n) {
  uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = n - 4 * j;
    u[j] = b >= 4 ? u[j] : b <= 0 ? 0u : u[j] & (0xffffffffu >> (8 * (4 - b)));
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ float int8_bias(const void* b, int f32, int i) {
  return b == nullptr ? 0.f : f32 ? static_cast<const float*>(b)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(b)[i]);
}

// A CTA takes 32 weight rows at a time (gated: 16 of the gate and their 16 of the up product) as the 16-row operand, NT x 8 activations as the other. Its eight
// warps take every eighth slice of K, 128 bytes of a row, and meet in shared memory. Both operands read a lane's 32 consecutive bytes in the same order, which
// a sum over k does not notice.
constexpr int FEW_WARPS = 8, FEW_SLICE = 128, FEW_PL = 36;

template <int NT, bool GATED>
__global__ void __launch_bounds__(FEW_WARPS * 32, NT <= 2 ? 2 : 1) int8_few_kernel(const Int8Few p) {
  constexpr int UN = NT <= 2 ? 2 : 4;                      // slices of a warp on their way
  extern __shared__ int few_part[];                        // [FEW_WARPS][8 NT][FEW_PL]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
  const int slices = (p.K + FEW_SLICE - 1) / FEW_SLICE;
  release_next();
  uint4 ring[UN][4][2];
  auto fetch = [&](int tile, int s, uint4 (&r)[4][2]) {
    const int at = s * FEW_SLICE + tig * 32;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = GATED ? min(tile * 16 + (t & 1) * 8 + g, p.cols - 1) + (t >> 1) * p.cols : min(tile * 32 + t * 8 + g, p.N - 1);
      const int8_t* from = p.q + (long)row * p.ldw + at;
#pragma unroll
      for (int i = 0; i < 2; ++i) r[t][i] = at + 16 * i < p.K ? int8_stream(from + 16 * i) : make_uint4(0, 0, 0, 0);
    }
  };
  int tile = blockIdx.x;
#pragma unroll
  for (int u = 0; u < UN; ++u)
    if (warp + u * FEW_WARPS < slices) fetch(tile, warp + u * FEW_WARPS, ring[u]);
  wait_previous();                                         // codes and scales of the activations
  const int8_t* xp[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xp[n] = p.codes + (long)min(n * 8 + g, p.T - 1) * p.ldc + tig * 32;
  for (; tile < p.tiles; tile += gridDim.x) {
    int acc[NT][2][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[n][i / 4][i % 4] = 0;
    for (int s0 = warp; s0 < slices; s0 += UN * FEW_WARPS) {
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int s = s0 + u * FEW_WARPS;
        if (s >= slices) break;
        const int left = p.K - s * FEW_SLICE - tig * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint4 b = make_uint4(0, 0, 0, 0);
            if (left > 16 * i) {
              b = *reinterpret_cast<const uint4*>(xp[n] + s * FEW_SLICE + 16 * i);
              if (left < 16 * i + 16) b = int8_mask(b, left - 16 * i);
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const uint4 lo = ring[u][2 * m][i], hi = ring[u][2 * m + 1][i];
              int8_mma(acc[n][m], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
              int8_mma(acc[n][m], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
            }
          }
        }
        const int next = s + UN * FEW_WARPS;
        if (next < slices) fetch(tile, next, ring[u]);
        else if (tile + (int)gridDim.x < p.tiles && warp + u * FEW_WARPS < slices) fetch(tile + gridDim.x, warp + u * FEW_WARPS, ring[u]);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        int* to = few_part + ((warp * NT + n) * 8 + 2 * tig) * FEW_PL + m * 16 + g;
        to[0] = acc[n][m][0];
        to[FEW_PL] = acc[n][m][1];
        to[8] = acc[n][m][2];
        to[FEW_PL + 8] = acc[n][m][3];
      }
    __syncthreads();
    constexpr int COLS = GATED ? 16 : 32;
    for (int i = tid; i < p.T * COLS; i += FEW_WARPS * 32) {
      const int t = i / COLS, c = i % COLS, col = tile * COLS + c;
      if (col >= p.cols) continue;
      int a = 0, b = 0;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) {
        a += few_part[(w * NT * 8 + t) * FEW_PL + c];
        if (GATED) b += few_part[(w * NT * 8 + t) * FEW_PL + 16 + c];
      }
      const float s = p.sx[t];
      float y = fmaf((float)a * s, p.sw[col], int8_bias(p.bias, p.bias_f32, col));
      if (GATED) y = int8_silu(y) * fmaf((float)b * s, p.sw[p.cols + col], int8_bias(p.bias, p.bias_f32, p.cols + col));
      if (p.out_f32) static_cast<float*>(p.out)[t * p.ldo + col] = y;
      else static_cast<__nv_bfloat16*>(p.out)[t * p.ldo + col] = __float2bfloat16_rn(y);
    }
    __syncthreads();
  }
}

template <int NT, bool GATED>
static int launch_int8_few(const Int8Few& p, bool early, int device, cudaStream_t st) {
  constexpr int bytes = FEW_WARPS * NT * 8 * FEW_PL * 4, ctas = 148 * (NT <= 2 ? 2 : 1);
  static OncePerDevice once;
  if (const int e = once.ask(device, [] { return (int)cudaFuncSetAttribute(int8_few_kernel<NT, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }))
    return -e;
  launch_step(early, int8_few_kernel<NT, GATED>, dim3(p.tiles < ctas ? p.tiles : ctas), FEW_WARPS * 32, bytes, st, p);
  return -(int)cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------- tiles
namespace i8t {
constexpr int BM = 256, BN = 256, BK = 128, STAGES = 5;    // BK in bytes: a swizzled row
constexpr int A_STAGE = 128 * BK, B_STAGE = 128 * BK;      // of one CTA
constexpr int THREADS = 320;                               // warp 0 loads, warp 1 products, warps 2 to 9 results
constexpr int STAGING = 8 * 4096;                          // a box of 32 rows x 128 bytes a warp
constexpr int TABLE = 8 * 2 * 128 * 4;                     // scales and biases of a warp's 128 columns of a tile
constexpr int SMEM_BYTES = STAGES * (A_STAGE + B_STAGE) + STAGING + TABLE + 1024 + 256;
constexpr int TMEM_COLS = 512;
// 8-bit signed operands, 32-bit whole sums, both operands K-major
constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((BN >> 3) << 17) | ((BM >> 4) << 24);
}  // namespace i8t

__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct Int8Tiles {
  const float *sx, *sw;
  const void* bias;
  void* out;
  long ldo;
  int T, K, cols, m_tiles, n_tiles;
  int bias_f32, boxes;         // boxes: results leave through TMA stores
  int* status;
};

// The pair protocol of the bf16 product (csrc/gemm_tcgen05_2cta.cu). GATED: the leader's half of the weights' rows are of the gate, the other CTA's of the up
// product, so a CTA finds both in its tensor memory.
template <bool GATED, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(i8t::THREADS, 1)
    int8_tile_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_c,
                     const __grid_constant__ Int8Tiles p) {
  using namespace i8t;
  constexpr int TN = GATED ? BN / 2 : BN;     // output columns of a tile
  constexpr int CW = TN / 2;                  // of a warp
  constexpr int STEP = F32 ? 32 : 64;         // of a box
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_STAGE;
  uint8_t* sStage = smem + STAGES * (A_STAGE + B_STAGE);
  float* table = reinterpret_cast<float*>(sStage + STAGING);               // [warp][scales, biases][128]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sStage + STAGING + TABLE);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  const bool leader = cta == 0;
  const int pair = (int)blockIdx.x >> 1, npairs = (int)gridDim.x >> 1;
  const int kb_total = (p.K + BK - 1) / BK, total = p.m_tiles * p.n_tiles;

  release_next();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 16);          // eight result warps in each CTA
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    if (p.boxes) tma_prefetch_desc(&tmap_c);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_previous();

  if (warp == 0) {
    if (elect_one_sync()) {
      int it = 0;
      bool ok = true;
      for (int w = pair; ok && w < total; w += npairs) {
        const int m0 = w / p.n_tiles * BM + (int)cta * 128, n = w % p.n_tiles * TN;
        const int n0 = GATED ? n + (int)cta * p.cols : n + (int)cta * 128;
        for (int kb = 0; kb < kb_total; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_EMPTY)) { ok = false; break; }
          const uint32_t leader_full = mapa_shared(smem_u32(&full_bar[s]), 0);
          if (leader) mbar_expect_tx(&full_bar[s], 2 * (A_STAGE + B_STAGE));
          tma_load_2d_pair(sA + s * A_STAGE, &tmap_a, leader_full, kb * BK, m0);
          tma_load_2d_pair(sB + s * B_STAGE, &tmap_b, leader_full, kb * BK, n0);
        }
      }
    }
  } else if (warp == 1) {
    if (leader && elect_one_sync()) {
      const uint64_t da0 = make_smem_desc(smem_u32(sA), 16, 1024, 2), db0 = make_smem_desc(smem_u32(sB), 16, 1024, 2);
      const uint32_t e0 = mapa_shared(smem_u32(&empty_bar[0]), 0), e1 = mapa_shared(smem_u32(&empty_bar[0]), 1);
      int s = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int w = pair; ok && w < total; w += npairs, ++i) {
        const int acc = i & 1;
        if (!mbar_wait(&tmem_empty[acc], ((i >> 1) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY)) break;
        tc_fence_after();
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!mbar_wait(&full_bar[s], ph, abort_flag, p.status, ERR_WAIT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint64_t da = da0 + (uint64_t)(s * (A_STAGE >> 4)), db = db0 + (uint64_t)(s * (B_STAGE >> 4));
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_i8_pair(tmem_base + acc * BN, da + 2 * k, db + 2 * k, IDESC, kb > 0 || k > 0 ? 1u : 0u);
          umma_commit_pair(e0 + s * 8);
          umma_commit_pair(e1 + s * 8);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        const uint32_t f = smem_u32(&tmem_full[acc]);
        umma_commit_pair(mapa_shared(f, 0));
        umma_commit_pair(mapa_shared(f, 1));
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* sc = sStage + (warp - 2) * 4096;
    float* scale = table + (warp - 2) * 256;
    float* bias = scale + 128;
    int i = 0;
    for (int w = pair; w < total; w += npairs, ++i) {
      const int m0 = w / p.n_tiles * BM + (int)cta * 128 + q * 32, n0 = w % p.n_tiles * TN, acc = i & 1;
      __syncwarp();
#pragma unroll
      for (int x = 0; x < 128; x += 32) {     // gated: CW columns of the gate, then those of the up product
        const int c = n0 + half * CW + (GATED ? (x & 32) : x) + lane, at = GATED && x >= 64 ? p.cols + c : c;
        scale[x + lane] = c < p.cols ? p.sw[at] : 0.f;
        bias[x + lane] = c < p.cols ? int8_bias(p.bias, p.bias_f32, at) : 0.f;
      }
      const float sx = m0 + lane < p.T ? p.sx[m0 + lane] : 0.f;
      __syncwarp();
      if (!mbar_wait_warp(&tmem_full[acc], (i >> 1) & 1, abort_flag, p.status, ERR_WAIT_TMEM_FULL)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + acc * BN + half * CW + (uint32_t(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < CW; c += STEP) {
        const int col0 = n0 + half * CW + c;
        if (col0 >= p.cols) break;
        if (p.boxes) {
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < STEP; x += 32) {
          uint32_t r[32], r2[GATED ? 32 : 1];
          tmem_ld_32x32(t_row + c + x, r);
          if constexpr (GATED) tmem_ld_32x32(t_row + 128 + c + x, r2);
          tmem_ld_wait();
          float y[32];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(scale + c + x + j), b4 = *reinterpret_cast<const float4*>(bias + c + x + j);
            y[j] = fmaf((float)(int)r[j] * sx, s4.x, b4.x);
            y[j + 1] = fmaf((float)(int)r[j + 1] * sx, s4.y, b4.y);
            y[j + 2] = fmaf((float)(int)r[j + 2] * sx, s4.z, b4.z);
            y[j + 3] = fmaf((float)(int)r[j + 3] * sx, s4.w, b4.w);
            if constexpr (GATED) {
              const float4 s5 = *reinterpret_cast<const float4*>(scale + 64 + c + x + j), b5 = *reinterpret_cast<const float4*>(bias + 64 + c + x + j);
              y[j] = int8_silu(y[j]) * fmaf((float)(int)r2[j] * sx, s5.x, b5.x);
              y[j + 1] = int8_silu(y[j + 1]) * fmaf((float)(int)r2[j + 1] * sx, s5.y, b5.y);
              y[j + 2] = int8_silu(y[j + 2]) * fmaf((float)(int)r2[j + 2] * sx, s5.z, b5.z);
              y[j + 3] = int8_silu(y[j + 3]) * fmaf((float)(int)r2[j + 3] * sx, s5.w, b5.w);
            }
          }
          if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(sc + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint4*>(sc + lane * 128 + (((x / 8 + j) ^ (lane & 7)) << 4)) =
                  make_uint4(pack_bf16x2(y[8 * j], y[8 * j + 1]), pack_bf16x2(y[8 * j + 2], y[8 * j + 3]), pack_bf16x2(y[8 * j + 4], y[8 * j + 5]),
                             pack_bf16x2(y[8 * j + 6], y[8 * j + 7]));
          }
        }
        if (p.boxes) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmap_c, sc, col0, m0);
            tma_store_commit();
          }
        } else {                              // rows off 16-byte boundaries: a row of the box at a time
          __syncwarp();
          const int rows = min(32, p.T - m0), c2 = F32 ? lane : 2 * lane;
          for (int rr = 0; rr < rows; ++rr) {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(sc + rr * 128 + (((lane >> 2) ^ (rr & 7)) << 4) + (lane & 3) * 4);
            const long at = (long)(m0 + rr) * p.ldo + col0 + c2;
            if constexpr (F32) {
              if (col0 + c2 < p.cols) static_cast<float*>(p.out)[at] = __uint_as_float(v);
            } else {
              uint16_t* o = static_cast<uint16_t*>(p.out) + at;
              if (col0 + c2 < p.cols) o[0] = (uint16_t)v;
              if (col0 + c2 + 1 < p.cols) o[1] = (uint16_t)(v >> 16);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&tmem_empty[acc]), 0));
    }
    if (lane == 0) tma_store_wait_all();
  }

  __syncthreads();
  if (*abort_flag) {                          // let the products that are under way end before the memory they read is given up
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

template <bool GATED, bool F32>
static int launch_int8_tiles(const Int8Call& c, bool early, int device, cudaStream_t st) {
  using namespace i8t;
  static OncePerDevice once;
  if (const int e = once.ask(device, [] { return (int)cudaFuncSetAttribute(int8_tile_kernel<GATED, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES); }))
    return -e;
  const int cols = (int)(GATED ? c.N / 2 : c.N), size = F32 ? 4 : 2;
  Int8Tiles p;
  p.sx = c.sx; p.sw = c.sw; p.bias = c.bias; p.out = c.out; p.ldo = c.ldo; p.T = (int)c.T; p.K = (int)c.K; p.cols = cols;
  p.m_tiles = (int)((c.T + BM - 1) / BM); p.n_tiles = (cols + (GATED ? 127 : 255)) / (GATED ? 128 : 256);
  p.bias_f32 = (int)c.bias_f32; p.status = c.status;
  p.boxes = ((uintptr_t)c.out | (uintptr_t)(c.ldo * size)) % 16 == 0;
  CUtensorMap ta, tb, tc;
  int rc = make_tmap_2d_u8(&ta, c.codes, (uint64_t)c.K, (uint64_t)c.T, (uint64_t)c.ldc, BK, 128);
  if (rc == 0) rc = make_tmap_2d_u8(&tb, c.q, (uint64_t)c.K, (uint64_t)c.N, (uint64_t)c.ldw, BK, 128);
  tc = ta;
  if (rc == 0 && p.boxes) rc = F32 ? make_tmap_2d_f32(&tc, c.out, (uint64_t)cols, (uint64_t)c.T, (uint64_t)c.ldo, 32, 32)
                                   : make_tmap_2d_bf16(&tc, c.out, (uint64_t)cols, (uint64_t)c.T, (uint64_t)c.ldo, 64, 32);
  if (rc) return rc;
  const long total = (long)p.m_tiles * p.n_tiles;
  const int pairs = (int)(total < 74 ? total : 74);
  launch_step(early, int8_tile_kernel<GATED, F32>, dim3(2 * pairs), THREADS, SMEM_BYTES, st, ta, tb, tc, p);
  return -(int)cudaGetLastError();
}

}  // namespace inv

using namespace inv;

extern "C" int inv_int8_rows(const void* call) {
  const Int8Call& c = *static_cast<const Int8Call*>(call);
  if (c.T <= 0 || c.K <= 0) return 0;
  return launch_int8_rows(c, (cudaStream_t)c.stream);
}

// Codes first where x is given, then the product, which starts while they are made: the kernel of the codes is launched plainly, so everything in front of it is
// complete when the product's first weights are read.
extern "C" int inv_int8_linear(const void* call) {
  const Int8Call& c = *static_cast<const Int8Call*>(call);
  if (c.T <= 0 || c.N <= 0 || c.K <= 0) return 0;
  if (c.K > 133144 || c.ldw % 16 || c.ldc % 16 || (((uintptr_t)c.q | (uintptr_t)c.codes) & 15) || (c.gated && c.N % 2)) return -ERR_BAD_ARG;
  cudaStream_t st = (cudaStream_t)c.stream;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device)) return -(int)e;
  const bool early = c.x != nullptr;
  if (early)
    if (const int e = launch_int8_rows(c, st)) return e;
  if (c.T <= 64) {
    const int cols = (int)(c.gated ? c.N / 2 : c.N), per = c.gated ? 16 : 32;
    const Int8Few p = {c.codes, c.q, c.sx, c.sw, c.bias, c.out, c.ldc, c.ldw, c.ldo, (int)c.T, (int)c.N, (int)c.K, cols, (cols + per - 1) / per, (int)c.bias_f32,
                       (int)c.out_f32};
#define INV_FEW(NT) (c.gated ? launch_int8_few<NT, true>(p, early, device, st) : launch_int8_few<NT, false>(p, early, device, st))
    return c.T <= 8 ? INV_FEW(1) : c.T <= 16 ? INV_FEW(2) : c.T <= 32 ? INV_FEW(4) : INV_FEW(8);
#undef INV_FEW
  }
  if (c.gated) return c.out_f32 ? launch_int8_tiles<true, true>(c, early, device, st) : launch_int8_tiles<true, false>(c, early, device, st);
  return c.out_f32 ? launch_int8_tiles<false, true>(c, early, device, st) : launch_int8_tiles<false, false>(c, early, device, st);
}
