// Products of activations and weights in 8-bit integers.
//
//   s_t = max(|x_t|, 1e-10) / 127       c_tk = rint(x_tk / s_t), halves to even
//   y_tn = s_t s_n sum_k c_tk q_nk + b_n            gated: silu(y_tn) y_t,n+F, n < F
//
// The sums are whole numbers below 2^31 (K <= 131071, codes from -128), so their order changes nothing; scales and bias are applied in fp32 and the result is rounded
// once.
//
// int8_rows_kernel      rows of activations into codes and scales
// int8_few_kernel       one row, or two and weights of up to 32 MB: codes and product in one launch
// int8_few_mma_kernel   three or four rows, likewise
// int8_split_kernel     up to 128 rows, or results of few tiles: tcgen05 kind::i8, clusters that share K
// int8_tile_kernel      the rest: tiles of 256 x 256 on CTA pairs, tcgen05 kind::i8
#include "cta_pair.cuh"
#include "gemm_common.cuh"
#include "once_per_device.h"
#include <type_traits>

namespace inv {

constexpr long INT8_MOST_K = 131071;      // 128 * 128 K < 2^31
constexpr long INT8_MOST = (1l << 31) - 1024;  // rows, columns and values of a row that is made into codes: counted in 32 bits

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

// ---------------------------------------------------------------------------------------------- plans
constexpr int FEW_WARPS = 8, FEW_ROWS = 4, FEW_SLICE = 512, FEW_RING = 4, FEW_CODES = 88 * 1024, FEW_WIDEST = 512;
constexpr int MMA_SLICE = 128, MMA_PL = 36, MMA_RING = 2;
static long few_room(long T, long K) { return T > 2 ? T * ((K + MMA_SLICE - 1) / MMA_SLICE * MMA_SLICE + 16) : T * ((K + FEW_SLICE - 1) / FEW_SLICE * FEW_SLICE); }

namespace i8s {
constexpr int THREADS = 192, BK = 128, A_STAGE = 128 * BK;  // warp 0 loads, warp 1 products, warps 2 to 5 sums
constexpr int MAX_STAGES = 12, REST = 1024 + 256;
constexpr int stages(int tb, int ctas) { return (227 * 1024 / ctas - 1024 * (ctas - 1) - REST - 4 * tb) / (A_STAGE + tb * BK); }    // with so many CTAs an SM
// At least 48 KB: a CTA of fewer would fit on an SM beside one of a pair that holds all tensor memory (int8_tile_kernel leaves 25 KB, other pairs less). On two streams
// a cluster could then hold what the pair's other CTA wants, and the pair what the cluster's.
constexpr int LEAST = 48 * 1024;
constexpr int smem_bytes(int tb, int n) {
  const int bytes = n * (A_STAGE + tb * BK) + REST + 4 * tb;
  return bytes < LEAST ? LEAST : bytes;
}
}  // namespace i8s
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

// How a product is cut and launched, from its sizes alone.
enum Int8Route { INT8_FEW, INT8_SPLIT, INT8_TILES };
struct Int8Plan {
  int route, cols, grid, cluster, threads, smem;
  int tiles, t_tiles, tb, per, kb, parts, stages;   // tiles in all and along the rows; rows and columns of one; steps of K, parts of it, stages of a ring
};
static Int8Route int8_route(long T, long N, long K, bool gated) {
  if (T <= FEW_ROWS && (T == 1 || N * K <= (32l << 20)) && few_room(T, K) <= FEW_CODES) return INT8_FEW;
  const long tiles = (T + 127) / 128 * ((gated ? N / 2 + 63 : N + 127) / (gated ? 64 : 128));
  return T <= 128 || tiles <= 148 ? INT8_SPLIT : INT8_TILES;
}
static Int8Plan int8_plan(long T, long N, long K, bool gated) {
  Int8Plan n = {};
  n.route = int8_route(T, N, K, gated);
  n.cols = (int)(gated ? N / 2 : N);
  n.cluster = n.parts = 1;
  if (n.route == INT8_FEW) {
    const int least = (T > 2 ? 32 : 4) / (gated ? 2 : 1), most = T > 2 ? least : FEW_WIDEST / (gated ? 2 : 1), even = (n.cols + 295) / 296;
    n.tb = (int)T;
    n.per = even < least ? least : even > most ? most : even;
    n.t_tiles = 1;
    n.tiles = (n.cols + n.per - 1) / n.per;
    n.grid = n.tiles < 296 ? n.tiles : 296;
    n.threads = FEW_WARPS * 32;
    n.smem = (int)few_room(T, K);
  } else if (n.route == INT8_SPLIT) {
    using namespace i8s;
    n.per = gated ? 64 : 128;
    const int col_tiles = (n.cols + n.per - 1) / n.per;
    n.tb = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
    if (T > 64)
      while (n.tb > 32 && (T + n.tb - 1) / n.tb * col_tiles < 100) n.tb /= 2;
    n.kb = (int)((K + BK - 1) / BK);
    n.t_tiles = (int)((T + n.tb - 1) / n.tb);
    n.tiles = col_tiles * n.t_tiles;
    auto fit = [&](int ctas) { const int k = ctas / n.tiles; return k < 1 ? 1 : k > 4 ? 4 : k; };
    int parts = fit(128);
    if (parts * n.tiles < 112) parts = fit(256);
    n.parts = n.cluster = parts > n.kb ? n.kb : parts;
    const int per_sm = n.tiles * n.parts <= 128 ? 1 : 2, most = stages(n.tb, per_sm), steps = (n.kb + n.parts - 1) / n.parts, stage = A_STAGE + n.tb * BK;
    n.stages = most < steps ? most : steps;
    if (n.stages > MAX_STAGES) n.stages = MAX_STAGES;
    if (n.stages * stage < n.tb * 512) n.stages = (n.tb * 512 + stage - 1) / stage;   // the sums take their place
    n.grid = n.tiles * n.parts;
    n.threads = THREADS;
    n.smem = smem_bytes(n.tb, n.stages);
  } else {
    using namespace i8t;
    n.tb = BM;
    n.per = gated ? BN / 2 : BN;
    n.kb = (int)((K + BK - 1) / BK);
    n.t_tiles = (int)((T + BM - 1) / BM);
    n.tiles = (n.cols + n.per - 1) / n.per * n.t_tiles;
    n.stages = STAGES;
    n.cluster = 2;
    n.grid = 2 * (n.tiles < 74 ? n.tiles : 74);
    n.threads = THREADS;
    n.smem = SMEM_BYTES;
  }
  return n;
}

// ---------------------------------------------------------------------------------------------- rows into codes
constexpr float INT8_LEAST = 1e-10f;

// rint(x / s), halves to even, |x| <= 127 s, in the low byte of the result. n is a whole number at or one below x * inv (from the rounding of an addition: conversions
// have a sixteenth of the rate); x against the border s (n + 1/2) is one rounded product-sum, whose sign is exact.
__device__ __forceinline__ uint32_t int8_code(float x, float s, float inv) {
  constexpr float MAGIC = 12582912.f;                     // 1.5 * 2^23: a number near it has its whole part in its lowest bits
  const float m = fmaf(x, inv, -0.5f) + MAGIC;
  const float d = fmaf(-s, (m - MAGIC) + 0.5f, x);
  const uint32_t i = __float_as_uint(m);
  return i + (d > 0.f || (d == 0.f && (i & 1u)) ? 1u : 0u);
}
__device__ __forceinline__ uint64_t int8_two(float2 v) { return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ uint64_t int8_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// The scale of a row from the bits of its largest |x|: not a number is above infinity is above the rest. False where it is not finite.
__device__ __forceinline__ bool int8_scale(uint32_t top, float& s, float& inv) {
  const bool finite = top < 0x7f800000u;
  // a / 127 rounded to the nearest: a quotient corrected by its exact remainder (one step of Newton's method in rounded products and sums)
  constexpr float PART = 1.f / 127.f;
  const float a = finite ? fmaxf(__uint_as_float(top), INT8_LEAST) : 1.f, q = a * PART;
  s = finite ? fmaf(fmaf(-127.f, q, a), PART, q) : __uint_as_float(0x7fc00000u);
  inv = __fdividef(1.f, s);                                // within two units of the last place
  return finite;
}
// Codes of eight values. x * inv is off by under 5e-5 from the quotient, so the sum with MAGIC rounds as the quotient does unless that is as near to a half: there, one
// time in some thousands, the border decides. Packed arithmetic, two values an instruction: instructions bound the kernel of many rows.
__device__ __forceinline__ uint2 int8_pack(const float2* v, float s, float inv) {
  constexpr float MAGIC = 12582912.f;
  const uint64_t inv2 = int8_two(make_float2(inv, inv)), magic = int8_two(make_float2(MAGIC, MAGIC)), minus = int8_two(make_float2(-1.f, -1.f));
  uint32_t u[8];
  float far = 0.f;                                         // from the nearest whole number
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t x = int8_two(v[j]), m = int8_fma2(x, inv2, magic), r = int8_fma2(x, inv2, int8_fma2(m, minus, magic));
    u[2 * j] = (uint32_t)m;
    u[2 * j + 1] = (uint32_t)(m >> 32);
    far = fmaxf(fmaxf(far, fabsf(__uint_as_float((uint32_t)r))), fabsf(__uint_as_float((uint32_t)(r >> 32))));
  }
  if (far > 0.4999f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[2 * j] = int8_code(v[j].x, s, inv);
      u[2 * j + 1] = int8_code(v[j].y, s, inv);
    }
  }
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

// Eight values of a row, of which n exist, as they are in memory. VEC: all of them, on a 16-byte boundary.
template <typename T, bool VEC>
struct Int8Eight {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ void load(const T* row, int n) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) *reinterpret_cast<uint4*>(w + 4 * j) = reinterpret_cast<const uint4*>(row)[j];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = j < n ? __float_as_uint(row[j]) : 0u;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (2 * j < n ? (uint32_t)h[2 * j] : 0u) | (2 * j + 1 < n ? (uint32_t)h[2 * j + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void values(float2* v) const {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = sizeof(T) == 4 ? make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]))
                            : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  }
  // the larger of `top` and the bits of every |x|
  __device__ __forceinline__ uint32_t largest(uint32_t top) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, w[j] & 0x7fffffffu);
    } else {                                               // pairs; not a number stays one
      __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
      for (int j = 1; j < 4; ++j) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])));
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
      top = max(top, max(u << 16, u & 0xffff0000u) & 0x7fffffffu);
    }
    return top;
  }
};

// A CTA takes a row, or (WARP) each of its eight warps one, a thread up to HOLD times eight of its values, which it keeps between the maximum and the rounding; what a
// long row has beyond that is read twice. A row with a value that is not finite gets NaN for its scale. Codes are written in eights, zeros behind the row.
template <typename T, bool VEC, bool WARP, int HOLD>
__global__ void __launch_bounds__(512) int8_rows_kernel(const T* __restrict__ x, long ldx, int rows, int K, int8_t* __restrict__ codes, long ldc, float* __restrict__ sx) {
  __shared__ uint32_t sh[16];
  release_next();
  const long r = WARP ? (long)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && r >= rows) return;
  const T* row = x + r * ldx;
  int8_t* to = codes + r * ldc;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x, eights = (K + 7) / 8;
  Int8Eight<T, VEC> v[HOLD], more;
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (tid + h * threads < eights) v[h].load(row + (tid + h * threads) * 8, K - (tid + h * threads) * 8);
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (tid + h * threads < eights) top = v[h].largest(top);
  for (int i = tid + HOLD * threads; i < eights; i += threads) {
    more.load(row + i * 8, K - i * 8);
    top = more.largest(top);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (!WARP) {
    if ((tid & 31) == 0) sh[tid >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, (tid & 31) < threads / 32 ? sh[tid & 31] : 0u);
  }
  float s, inv;
  const bool finite = int8_scale(top, s, inv);
  if (tid == 0) sx[r] = s;
  auto store = [&](int i, const Int8Eight<T, VEC>& e) {
    float2 f[4];
    e.values(f);
    *reinterpret_cast<uint2*>(to + i * 8) = finite ? int8_pack(f, s, inv) : make_uint2(0u, 0u);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (tid + h * threads < eights) store(tid + h * threads, v[h]);
  for (int i = tid + HOLD * threads; i < eights; i += threads) {
    more.load(row + i * 8, K - i * 8);
    store(i, more);
  }
}

static bool int8_rows_vec(const Int8Call& c) {
  return c.K % 8 == 0 && ((uintptr_t)c.x | (uintptr_t)(c.T > 1 ? c.ldx * (c.x_f32 ? 4 : 2) : 0)) % 16 == 0;
}

static int launch_int8_rows(const Int8Call& c, cudaStream_t st) {
  const bool vec = int8_rows_vec(c);
  // Instructions bound many rows, and a row costs each of its warps some 150 besides its values: then few warps a row, 64 values a lane. 8192 x 4096 in bf16: 21 us
  // (28 with eight warps a row and 16 values a lane); 2048 x 11008 17 (21). Fewer than two eights for each thread that the GPU holds: many warps, for the shortest
  // chain (301 x 1411: 2.6 us, 5.3 as above); a warp for each of many short rows.
  const long eights = (c.K + 7) / 8;
  const bool many = c.T * eights >= 2l * 148 * 2048, warps = many ? eights <= 256 : c.T > 296 && eights <= 128;
  const int hold = eights <= 64 ? 2 : eights <= 128 || !many ? 4 : 8;
  const long want = many ? (eights + 7) / 8 : c.K <= 512 ? 64 : c.K <= 1024 ? 128 : c.K <= 4096 ? 256 : 512;
  const int threads = (int)(warps ? 256 : want >= 512 ? 512 : (want + 31) / 32 * 32);
  const unsigned grid = (unsigned)(warps ? (c.T + 7) / 8 : c.T);
#define INV_ROW(E, V, W, H) int8_rows_kernel<E, V, W, H><<<grid, threads, 0, st>>>((const E*)c.x, c.ldx, (int)c.T, (int)c.K, c.codes, c.ldc, c.sx)
#define INV_ROWS(E, V)                                \
  do {                                                \
    if (!warps && hold <= 4) INV_ROW(E, V, false, 4); \
    else if (!warps) INV_ROW(E, V, false, 8);         \
    else if (hold == 2) INV_ROW(E, V, true, 2);       \
    else if (hold == 4) INV_ROW(E, V, true, 4);       \
    else INV_ROW(E, V, true, 8);                      \
  } while (0)
  if (c.x_f32) {
    if (vec) INV_ROWS(float, true);
    else INV_ROWS(float, false);
  } else {
    if (vec) INV_ROWS(__nv_bfloat16, true);
    else INV_ROWS(__nv_bfloat16, false);
  }
#undef INV_ROW
#undef INV_ROWS
  return -(int)cudaGetLastError();
}

// The scales are multiplied first: a sum of codes, up to 2^31, times the scale of a token of 1e32 and more would not fit. The conversion, the scales' product and the
// whole are rounded, half a step each.
__device__ __forceinline__ float int8_value(int sum, float sx, float sw, float bias) { return fmaf((float)sum, sx * sw, bias); }
// The quick exponential and quotient, as in the other products' epilogues (silu_f), for fp32 results too: off by 2 + 1.16 |x| and 2 units of 2^-23. Below -87 the quotient is 0
// in place of -5e-37. Neither has a branch, so that a warp stays together between its loads from tensor memory.
__device__ __forceinline__ float int8_silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }

// ---------------------------------------------------------------------------------------------- up to four rows
struct Int8Few {
  const void* x;                   // bf16 or fp32, or null: codes and scales are given
  const int8_t *codes, *q;
  const float *sx, *sw;
  const void* bias;
  void* out;
  long ldx, ldc, ldw, ldo;
  int T, N, K, cols, per, tiles;   // cols: output columns; per: of a tile
  int x_f32, x_vec, bias_f32, out_f32;
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
__device__ __forceinline__ float int8_bias(const void* b, int f32, int i) {
  return b == nullptr ? 0.f : f32 ? static_cast<const float*>(b)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(b)[i]);
}
// One launch: a CTA makes the codes of all rows for itself, in shared memory, while its first weights are on their way (every CTA reads x from L2, and with a kernel of
// their own in front the codes cost 1.5 us on the device and 4 on the host). Weights go from memory straight into registers and are multiplied there, with none of a
// tile's set-up.
//
// int8_few_kernel, one and two rows: products of four codes a lane and instruction. A warp reads 512 bytes of four weight rows at a time. A tile's rows by the slices
// of K are dealt out to the warps in equal runs, whose sums meet in shared memory, and tiles are as wide as spreads the weights over two CTAs an SM.
// int8_few_mma_kernel, three and four rows: a CTA takes 32 weight rows at a time (gated: 16 of the gate and their 16 of the up product) as the 16-row operand of
// warp-level matrix products, the activations as the other. Its eight warps take every eighth slice of K, 128 bytes of a row, and meet in shared memory. Both
// operands read a lane's bytes in the same order, which a sum over k does not notice.
//
// Neither kind of product is fast on this GPU: some 8 cycles a scheduler for 32 lanes' four codes, some 80 for 16 x 8 x 32. 6144 x 4096, us, in products of
// codes and of matrices: one row 7.4, 8.7; two 8.7, 9.4; four 11.6, 10.1. Against codes in front and tcgen05 tiles: one row 12288 x 4096 11.4, 13.6, 22016 x 4096 17.4,
// 18.8, 22016 x 11008 42.3, 42.8: any size. Two, three and four rows 7168 x 4096 9.7, 10.4, 10.8 against 10.7, 8192 x 4096 10.1, 11.1, 11.4 against 11.2, 12288 x 4096
// 12.5, 14.6, 15.0 against 14.1, 32768 x 1024 9.4, 10.3, 10.4 against 10.5: weights of up to 32 MB, where three and four rows are even. Long rows of few weights lose on the
// device, 2048 x 11008 11.3, 16.5, 17.4 against 9.9, and have the 4 us of a second launch on the host in return.

// Codes of all rows into shared memory, `pitch` apart, with zeros up to `width`, and their scales.
template <int TT>
__device__ __forceinline__ void int8_few_codes(const Int8Few& p, int8_t* few_codes, int pitch, int width, uint32_t (&tops)[FEW_WARPS][TT], float (&scales)[TT]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int eights = (p.K + 7) / 8, places = width / 8;
  if (p.x != nullptr) {
    // all rows' loads of a place at once
    auto codes = [&](auto* x, auto vec) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
      using Eight = Int8Eight<T, decltype(vec)::value>;
      uint32_t top[TT] = {};
      for (int i = tid; i < eights; i += FEW_WARPS * 32) {
        Eight e[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (t < p.T) e[t].load(x + t * p.ldx + i * 8, p.K - i * 8);
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (t < p.T) top[t] = e[t].largest(top[t]);
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        top[t] = __reduce_max_sync(0xffffffffu, top[t]);
        if (lane == 0) tops[warp][t] = top[t];
      }
      __syncthreads();
      float sx[TT], inv[TT];
      bool finite[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        finite[t] = int8_scale(__reduce_max_sync(0xffffffffu, lane < FEW_WARPS ? tops[lane][t] : 0u), sx[t], inv[t]);
        if (tid == t) scales[t] = sx[t];
      }
      for (int i = tid; i < places; i += FEW_WARPS * 32) {
        Eight e[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (t < p.T && i < eights) e[t].load(x + t * p.ldx + i * 8, p.K - i * 8);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          if (t >= p.T) break;
          float2 v[4];
          e[t].values(v);
          *reinterpret_cast<uint2*>(few_codes + t * pitch + i * 8) = i < eights && finite[t] ? int8_pack(v, sx[t], inv[t]) : make_uint2(0u, 0u);
        }
      }
    };
    if (p.x_f32) {
      if (p.x_vec) codes(static_cast<const float*>(p.x), std::true_type{});
      else codes(static_cast<const float*>(p.x), std::false_type{});
    } else {
      if (p.x_vec) codes(static_cast<const __nv_bfloat16*>(p.x), std::true_type{});
      else codes(static_cast<const __nv_bfloat16*>(p.x), std::false_type{});
    }
  } else {
    if (tid < p.T) scales[tid] = p.sx[tid];
    for (int t = 0; t < p.T; ++t)
      for (int i = tid; i < places; i += FEW_WARPS * 32) {
        const int8_t* from = p.codes + t * p.ldc + i * 8;
        uint2 v = make_uint2(0u, 0u);
        if (i * 8 + 8 <= p.K) v = *reinterpret_cast<const uint2*>(from);
        else
          for (int j = 0; i * 8 + j < p.K; ++j) (j < 4 ? v.x : v.y) |= ((uint32_t)from[j] & 255u) << (8 * (j % 4));
        *reinterpret_cast<uint2*>(few_codes + t * pitch + i * 8) = v;
      }
  }
  __syncthreads();
}

template <int TT, bool GATED>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) int8_few_kernel(const Int8Few p) {
  constexpr int UNIT = 4;                                    // rows that a warp takes a slice of at a time
  extern __shared__ __align__(16) int8_t few_codes[];        // [T] rows of whole slices
  __shared__ int part[TT * FEW_WIDEST];
  __shared__ uint32_t tops[FEW_WARPS][TT];
  __shared__ float scales[TT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slices = (p.K + FEW_SLICE - 1) / FEW_SLICE, pitch = slices * FEW_SLICE;
  release_next();
  for (int i = tid; i < TT * FEW_WIDEST; i += FEW_WARPS * 32) part[i] = 0;
  uint4 ring[FEW_RING][UNIT];
  int rows = 0, first = 0;                                   // of the tile; its first column
  auto fetch = [&](int group, int s, uint4 (&r)[UNIT]) {
#pragma unroll
    for (int t = 0; t < UNIT; ++t) {
      const int at = s * FEW_SLICE + lane * 16, i = group * UNIT + t, half = rows / 2;
      const long row = GATED && i >= half ? first + i - half + p.cols : first + i;
      r[t] = i < rows && at < p.K ? int8_stream(p.q + row * p.ldw + at) : make_uint4(0, 0, 0, 0);
    }
  };
  int tile = blockIdx.x, units = 0, unit = 0, end = 0, ahead = 0, group = 0, s = 0, next_group = 0, next_s = 0;
  auto advance = [&](int& group, int& s) {
    if (++s == slices) { s = 0; ++group; }
  };
  auto start = [&] {                                         // of a tile: this warp's run, and its first loads
    first = tile * p.per;
    rows = min(p.per, p.cols - first) * (GATED ? 2 : 1);
    units = (rows + UNIT - 1) / UNIT * slices;
    unit = ahead = units * warp / FEW_WARPS;
    end = units * (warp + 1) / FEW_WARPS;
    group = next_group = unit / slices;
    s = next_s = unit - group * slices;
#pragma unroll
    for (int u = 0; u < FEW_RING; ++u) {
      if (ahead == end) break;
      fetch(next_group, next_s, ring[u]);
      ++ahead;
      advance(next_group, next_s);
    }
  };
  start();
  int8_few_codes<TT>(p, few_codes, pitch, pitch, tops, scales);
  const int8_t* x = few_codes + lane * 16;
  while (true) {
    int acc[TT][UNIT] = {};
    auto flush = [&] {                                       // whole numbers, in whatever order
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        int mine = 0;
#pragma unroll
        for (int r = 0; r < UNIT; ++r) {
          const int all = __reduce_add_sync(0xffffffffu, acc[t][r]);
          if (lane == r) mine = all;
          acc[t][r] = 0;
        }
        if (lane < UNIT && group * UNIT + lane < rows) atomicAdd(&part[t * FEW_WIDEST + group * UNIT + lane], mine);
      }
    };
    while (unit < end) {
#pragma unroll
      for (int u = 0; u < FEW_RING; ++u) {
        if (unit == end) break;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          const uint4 b = *reinterpret_cast<const uint4*>(x + t * pitch + s * FEW_SLICE);
#pragma unroll
          for (int r = 0; r < UNIT; ++r) {
            acc[t][r] = __dp4a((int)ring[u][r].x, (int)b.x, acc[t][r]);
            acc[t][r] = __dp4a((int)ring[u][r].y, (int)b.y, acc[t][r]);
            acc[t][r] = __dp4a((int)ring[u][r].z, (int)b.z, acc[t][r]);
            acc[t][r] = __dp4a((int)ring[u][r].w, (int)b.w, acc[t][r]);
          }
        }
        if (ahead < end) {
          fetch(next_group, next_s, ring[u]);
          ++ahead;
          advance(next_group, next_s);
        }
        ++unit;
        if (s + 1 == slices || unit == end) flush();
        advance(group, s);
      }
    }
    __syncthreads();
    const int width = min(p.per, p.cols - first), now = first;
    const bool more = tile + (int)gridDim.x < p.tiles;
    if (more) {
      tile += gridDim.x;
      start();
    }
    for (int i = tid; i < width * TT; i += FEW_WARPS * 32) {
      const int t = i / width, c = i - t * width, col = now + c;
      const float sx = scales[t];
      float y = int8_value(part[t * FEW_WIDEST + c], sx, p.sw[col], int8_bias(p.bias, p.bias_f32, col));
      if (GATED) y = int8_silu(y) * int8_value(part[t * FEW_WIDEST + width + c], sx, p.sw[p.cols + col], int8_bias(p.bias, p.bias_f32, p.cols + col));
      if (p.out_f32) static_cast<float*>(p.out)[t * p.ldo + col] = y;
      else static_cast<__nv_bfloat16*>(p.out)[t * p.ldo + col] = __float2bfloat16_rn(y);
    }
    if (!more) break;
    __syncthreads();
    for (int i = tid; i < TT * FEW_WIDEST; i += FEW_WARPS * 32) part[i] = 0;
    __syncthreads();
  }
}

template <bool GATED>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) int8_few_mma_kernel(const Int8Few p) {
  extern __shared__ __align__(16) int8_t few_codes[];        // [T] rows of whole slices, pitch apart: 16 bytes off 128, so that eight lanes meet all banks
  __shared__ int part[FEW_WARPS * 8 * MMA_PL];                // the product has eight rows of activations
  __shared__ uint32_t tops[FEW_WARPS][FEW_ROWS];
  __shared__ float scales[FEW_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
  const int slices = (p.K + MMA_SLICE - 1) / MMA_SLICE, pitch = slices * MMA_SLICE + 16;
  release_next();
  uint4 ring[MMA_RING][4][2];
  auto fetch = [&](int tile, int s, uint4 (&r)[4][2]) {
    const int at = s * MMA_SLICE + tig * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = GATED ? min(tile * 16 + (t & 1) * 8 + g, p.cols - 1) + (t >> 1) * p.cols : min(tile * 32 + t * 8 + g, p.N - 1);
      const int8_t* from = p.q + (long)row * p.ldw + at;
#pragma unroll
      for (int i = 0; i < 2; ++i) r[t][i] = at + 64 * i < p.K ? int8_stream(from + 64 * i) : make_uint4(0, 0, 0, 0);
    }
  };
  int tile = blockIdx.x;
#pragma unroll
  for (int u = 0; u < MMA_RING; ++u)
    if (warp + u * FEW_WARPS < slices) fetch(tile, warp + u * FEW_WARPS, ring[u]);
  int8_few_codes<FEW_ROWS>(p, few_codes, pitch, slices * MMA_SLICE, tops, scales);
  const int8_t* x = few_codes + min(g, p.T - 1) * pitch + tig * 16;
  for (; tile < p.tiles; tile += gridDim.x) {
    int acc[2][4] = {};
    for (int s0 = warp; s0 < slices; s0 += MMA_RING * FEW_WARPS) {
#pragma unroll
      for (int u = 0; u < MMA_RING; ++u) {
        const int s = s0 + u * FEW_WARPS;
        if (s >= slices) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 b = *reinterpret_cast<const uint4*>(x + s * MMA_SLICE + 64 * i);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const uint4 lo = ring[u][2 * m][i], hi = ring[u][2 * m + 1][i];
            int8_mma(acc[m], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
            int8_mma(acc[m], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
          }
        }
        const int next = s + MMA_RING * FEW_WARPS;
        if (next < slices) fetch(tile, next, ring[u]);
        else if (tile + (int)gridDim.x < p.tiles && warp + u * FEW_WARPS < slices) fetch(tile + gridDim.x, warp + u * FEW_WARPS, ring[u]);
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      int* to = part + (warp * 8 + 2 * tig) * MMA_PL + m * 16 + g;
      to[0] = acc[m][0];
      to[MMA_PL] = acc[m][1];
      to[8] = acc[m][2];
      to[MMA_PL + 8] = acc[m][3];
    }
    __syncthreads();
    constexpr int COLS = GATED ? 16 : 32;
    const int t = tid / COLS, c = tid % COLS, col = tile * COLS + c;
    if (t < p.T && col < p.cols) {
      int a = 0, b = 0;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) {
        a += part[(w * 8 + t) * MMA_PL + c];
        if (GATED) b += part[(w * 8 + t) * MMA_PL + 16 + c];
      }
      const float s = scales[t];
      float y = int8_value(a, s, p.sw[col], int8_bias(p.bias, p.bias_f32, col));
      if (GATED) y = int8_silu(y) * int8_value(b, s, p.sw[p.cols + col], int8_bias(p.bias, p.bias_f32, p.cols + col));
      if (p.out_f32) static_cast<float*>(p.out)[t * p.ldo + col] = y;
      else static_cast<__nv_bfloat16*>(p.out)[t * p.ldo + col] = __float2bfloat16_rn(y);
    }
    __syncthreads();
  }
}

template <int TT, bool GATED>
static int launch_int8_few(const Int8Call& c, const Int8Plan& n, int device, cudaStream_t st) {
  constexpr bool MMA = TT > 2;
  static OncePerDevice once;
  const auto kernel = [] {
    if constexpr (MMA) return int8_few_mma_kernel<GATED>;
    else return int8_few_kernel<TT, GATED>;
  }();
  if (const int e = once.ask(device, [&] { return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_CODES); })) return -e;
  const Int8Few p = {c.x, c.codes, c.q, c.sx, c.sw, c.bias, c.out, c.ldx, c.ldc, c.ldw, c.ldo, (int)c.T, (int)c.N, (int)c.K, n.cols, n.per, n.tiles,
                     (int)c.x_f32, int8_rows_vec(c), (int)c.bias_f32, (int)c.out_f32};
  kernel<<<n.grid, n.threads, n.smem, st>>>(p);
  return -(int)cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------- few tiles
// Weight rows are the 128-row operand and TB activations the other one (tcgen05 kind::i8 on one SM), so that few activations fill an instruction. A cluster of up
// to four CTAs shares a tile: each has a part of K, leaves its sums in its shared memory and adds up its share of the tile's results from all of them (sums that met in
// global memory through atomics took 53 to 250 us of 64 x 4096 x 11008). Weight bytes bound it, but for its start and end: with the codes in front 16 rows of a gated
// 22016 x 4096 take 19.9 us, 4.6 TB/s, 64 rows of 4096 x 11008 14.7, 3.1 TB/s (the codes 2.6 us of them, the cluster's join 1.5).
struct Int8Split {
  const float *sx, *sw;
  const void* bias;
  void* out;
  int* status;
  long ldo;
  int T, cols, kb, t_tiles, parts, stages;     // kb: steps of 128 bytes of K; t_tiles: tiles of activations; parts: CTAs of a tile; stages: of the ring
  uint32_t inv_t, inv_parts;           // div_reciprocal
  int bias_f32, out_f32, fours;        // fours: four results of a row are stored at once
};

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// GATED: a tile's rows are 16 of the gate and the same 16 of the up product in turn (boxes of a map of three dimensions).
template <int TB, bool GATED>
__global__ void __launch_bounds__(i8s::THREADS, 2)
    int8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ Int8Split p) {
  using namespace i8s;
  constexpr int B_STAGE = TB * BK, COLS = GATED ? 64 : 128;
  constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TB >> 3) << 17) | ((128u >> 4) << 24);
  constexpr int TMEM_COLS = TB < 32 ? 32 : TB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  const int STAGES = p.stages;
  uint8_t* sB = smem + STAGES * A_STAGE;
  int* sums = reinterpret_cast<int*>(smem);                // [TB][128], once the stages have been used
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sB + STAGES * B_STAGE);
  uint64_t* empty_bar = full_bar + MAX_STAGES;
  uint64_t* tmem_full = empty_bar + MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* scales = reinterpret_cast<float*>(tmem_slot + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = div_by(blockIdx.x, p.parts, p.inv_parts), rank = (int)blockIdx.x - tile * p.parts;
  const int ct = div_by(tile, p.t_tiles, p.inv_t), t0 = (tile - ct * p.t_tiles) * TB, left = min(TB, p.T - t0), n0 = ct * COLS;
  const int k0 = rank * p.kb / p.parts, steps = (rank + 1) * p.kb / p.parts - k0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tmem_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  release_next();                                          // with tensor memory in hand: a kernel that starts early and takes some waits for this one's end

  if (warp == 0) {
    if (elect_one_sync()) {
      auto load_w = [&](int i, int s) {
        mbar_expect_tx(&full_bar[s], A_STAGE + B_STAGE);
        if constexpr (GATED) {
#pragma unroll
          for (int j = 0; j < 4; ++j) tma_load_3d(sA + s * A_STAGE + j * 4096, &tmap_w, &full_bar[s], (k0 + i) * BK, n0 + 16 * j, 0);
        } else {
          tma_load_2d(sA + s * A_STAGE, &tmap_w, &full_bar[s], (k0 + i) * BK, n0);
        }
      };
      auto load_x = [&](int i, int s) { tma_load_2d(sB + s * B_STAGE, &tmap_x, &full_bar[s], (k0 + i) * BK, t0); };
      const int head = min(steps, STAGES);                 // weights flow while the activations are still being made
      for (int i = 0; i < head; ++i) load_w(i, i);
      wait_previous();
      for (int i = 0; i < head; ++i) load_x(i, i);
      int s = 0;
      uint32_t ph = 0;
      for (int i = head; i < steps; ++i) {
        if (!mbar_wait(&empty_bar[s], ph, abort_flag, p.status, ERR_WAIT_EMPTY)) break;
        load_w(i, s);
        load_x(i, s);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (elect_one_sync()) {
      const uint64_t da0 = make_smem_desc(smem_u32(sA), 16, 1024, 2), db0 = make_smem_desc(smem_u32(sB), 16, 1024, 2);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0; i < steps; ++i) {
        if (!mbar_wait(&full_bar[s], ph, abort_flag, p.status, ERR_WAIT_FULL)) { ok = false; break; }
        tc_fence_after();
        const uint64_t da = da0 + (uint64_t)(s * (A_STAGE >> 4)), db = db0 + (uint64_t)(s * (B_STAGE >> 4));
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_i8(tmem_base, da + 2 * k, db + 2 * k, IDESC, i > 0 || k > 0 ? 1u : 0u);
        umma_commit(&empty_bar[s]);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (ok) umma_commit(tmem_full);
    }
  } else {
    const int q = warp & 3, row = q * 32 + lane;           // the lanes of tensor memory that this warp may read
    if (mbar_wait_warp(tmem_full, 0, abort_flag, p.status, ERR_WAIT_TMEM_FULL)) {
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < TB; c += 16) {
        if (c >= left) break;
        uint32_t r[16];
        tmem_ld_32x16(tmem_base + c + (uint32_t(q * 32) << 16), r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + row] = (int)r[j];
      }
      tc_fence_before();
    }
  }
  wait_previous();
  for (int t = threadIdx.x; t < left; t += THREADS) scales[t] = p.sx[t0 + t];
  __syncwarp();
  if (p.parts > 1) cluster_sync_all();
  else __syncthreads();
  if (*abort_flag) {                          // let the loads and products that are under way end before the memory they use is given up
    const uint64_t since = globaltimer_ns();
    while (globaltimer_ns() - since < 2000000ull) __nanosleep(1000);
  } else {
    // four columns a lane; a warp takes a token at a time, or two halves of the gated form one each
    constexpr int SUB = GATED ? 2 : 1;
    const int c = GATED ? (lane & 15) * 4 : lane * 4, col = n0 + c, in_row = GATED ? (c >> 4) * 32 + (c & 15) : c;
    float sw[SUB][4], bias[SUB][4];
#pragma unroll
    for (int h = 0; h < SUB; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool fine = col + i < p.cols;
        sw[h][i] = fine ? p.sw[h * p.cols + col + i] : 0.f;
        bias[h][i] = fine ? int8_bias(p.bias, p.bias_f32, h * p.cols + col + i) : 0.f;
      }
    const uint32_t base = smem_u32(sums) + in_row * 4;
#pragma unroll 2
    for (int t = rank + p.parts * (warp * SUB + (GATED ? lane >> 4 : 0)); t < left; t += p.parts * (THREADS / 32) * SUB) {
      int v[SUB][4] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= p.parts) break;
        const uint32_t there = mapa_shared(base + t * 512, j);
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
          const int4 w = ld_cluster_v4(there + h * 64);
          v[h][0] += w.x; v[h][1] += w.y; v[h][2] += w.z; v[h][3] += w.w;
        }
      }
      const float sx = scales[t];
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = int8_value(v[0][i], sx, sw[0][i], bias[0][i]);
        if (GATED) y[i] = int8_silu(y[i]) * int8_value(v[SUB - 1][i], sx, sw[SUB - 1][i], bias[SUB - 1][i]);
      }
      const long o = (long)(t0 + t) * p.ldo + col;
      if (p.fours && col + 3 < p.cols) {
        if (p.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) = make_float4(y[0], y[1], y[2], y[3]);
        else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + o) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (col + i >= p.cols) break;
          if (p.out_f32) static_cast<float*>(p.out)[o + i] = y[i];
          else static_cast<__nv_bfloat16*>(p.out)[o + i] = __float2bfloat16_rn(y[i]);
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (p.parts > 1) cluster_sync_all();                     // the others have read this CTA's sums
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int TB, bool GATED>
static int launch_int8_split(const Int8Call& c, const Int8Plan& n, bool early, int device, cudaStream_t st) {
  using namespace i8s;
  static OncePerDevice once;
  if (const int e = once.ask(device, [] { return (int)cudaFuncSetAttribute(int8_split_kernel<TB, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(TB, stages(TB, 1))); }))
    return -e;
  Int8Split p;
  p.sx = c.sx; p.sw = c.sw; p.bias = c.bias; p.out = c.out; p.ldo = c.ldo; p.T = (int)c.T; p.cols = n.cols; p.status = c.status;
  p.kb = n.kb; p.t_tiles = n.t_tiles; p.parts = n.parts; p.stages = n.stages;
  p.inv_t = div_reciprocal(p.t_tiles); p.inv_parts = div_reciprocal(p.parts);
  p.bias_f32 = (int)c.bias_f32; p.out_f32 = (int)c.out_f32;
  p.fours = c.ldo % 4 == 0 && (uintptr_t)c.out % 16 == 0;
  CUtensorMap tw, tx;
  const uint64_t K = c.K, N = c.N, T = c.T, ld = c.ldw;
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int rc = GATED ? make_tmap(&tw, u8, 3, c.q, {K, N / 2, 2}, {ld, ld * (N / 2)}, {BK, 16, 2}) : make_tmap(&tw, u8, 2, c.q, {K, N}, {ld}, {BK, 128});
  if (rc == 0) rc = make_tmap(&tx, u8, 2, c.codes, {K, T}, {(uint64_t)c.ldc}, {BK, TB});
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n.grid);
  cfg.blockDim = dim3(n.threads);
  cfg.dynamicSmemBytes = n.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  return -(int)cudaLaunchKernelEx(&cfg, int8_split_kernel<TB, GATED>, tw, tx, p);
}

// ---------------------------------------------------------------------------------------------- tiles
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
  uint32_t inv_n;              // div_reciprocal
  int bias_f32, boxes;         // boxes: results leave through TMA stores
  int* status;
};

// The pair protocol of the bf16 product (csrc/gemm_tcgen05_2cta.cu). GATED: the leader's half of the weights' rows are of the gate, the other CTA's of the up
// product, so a CTA finds both in its tensor memory. Many tiles are bound by the tensor cores, 88 % of whose cycles are busy: 8192 x 4096 x 22016 gated 478 us alone
// (3.1 POP/s), 600 with its codes call after call (2.5, the power limit). Few tiles by the last round of tiles: 2048 x 11008 x 4096 has 128 of them on 74 pairs, 34 us.
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
  release_next();                             // as above
  wait_previous();

  if (warp == 0) {
    if (elect_one_sync()) {
      int it = 0;
      bool ok = true;
      for (int w = pair; ok && w < total; w += npairs) {
        const int mt = div_by(w, p.n_tiles, p.inv_n), m0 = mt * BM + (int)cta * 128, n = (w - mt * p.n_tiles) * TN;
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
    // scales and biases of a tile come from memory under the tile before it (3003 x 512 x 4096 gated: 16.2 us without, 15.1 with)
    float next_scale[4], next_bias[4], next_sx = 0.f;
    auto fetch = [&](int w) {
      const int mt = div_by(w, p.n_tiles, p.inv_n), m0 = mt * BM + (int)cta * 128 + q * 32, n0 = (w - mt * p.n_tiles) * TN;
#pragma unroll
      for (int x = 0; x < 4; ++x) {           // gated: CW columns of the gate, then those of the up product
        const int c = n0 + half * CW + (GATED ? (x & 1) : x) * 32 + lane, at = GATED && x >= 2 ? p.cols + c : c;
        next_scale[x] = c < p.cols ? p.sw[at] : 0.f;
        next_bias[x] = c < p.cols ? int8_bias(p.bias, p.bias_f32, at) : 0.f;
      }
      next_sx = m0 + lane < p.T ? p.sx[m0 + lane] : 0.f;
    };
    int i = 0;
    if (pair < total) fetch(pair);
    for (int w = pair; w < total; w += npairs, ++i) {
      const int mt = div_by(w, p.n_tiles, p.inv_n), m0 = mt * BM + (int)cta * 128 + q * 32, n0 = (w - mt * p.n_tiles) * TN, acc = i & 1;
      const float sx = next_sx;
      __syncwarp();
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        scale[x * 32 + lane] = next_scale[x];
        bias[x * 32 + lane] = next_bias[x];
      }
      __syncwarp();
      if (w + npairs < total) fetch(w + npairs);
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
            y[j] = int8_value((int)r[j], sx, s4.x, b4.x);
            y[j + 1] = int8_value((int)r[j + 1], sx, s4.y, b4.y);
            y[j + 2] = int8_value((int)r[j + 2], sx, s4.z, b4.z);
            y[j + 3] = int8_value((int)r[j + 3], sx, s4.w, b4.w);
            if constexpr (GATED) {
              const float4 s5 = *reinterpret_cast<const float4*>(scale + 64 + c + x + j), b5 = *reinterpret_cast<const float4*>(bias + 64 + c + x + j);
              y[j] = int8_silu(y[j]) * int8_value((int)r2[j], sx, s5.x, b5.x);
              y[j + 1] = int8_silu(y[j + 1]) * int8_value((int)r2[j + 1], sx, s5.y, b5.y);
              y[j + 2] = int8_silu(y[j + 2]) * int8_value((int)r2[j + 2], sx, s5.z, b5.z);
              y[j + 3] = int8_silu(y[j + 3]) * int8_value((int)r2[j + 3], sx, s5.w, b5.w);
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
      if (lane == 0) mbar_arrive_remote_relaxed(mapa_shared(smem_u32(&tmem_empty[acc]), 0));
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
static int launch_int8_tiles(const Int8Call& c, const Int8Plan& n, bool early, int device, cudaStream_t st) {
  using namespace i8t;
  static OncePerDevice once;
  if (const int e = once.ask(device, [] { return (int)cudaFuncSetAttribute(int8_tile_kernel<GATED, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES); }))
    return -e;
  const int size = F32 ? 4 : 2;
  Int8Tiles p;
  p.sx = c.sx; p.sw = c.sw; p.bias = c.bias; p.out = c.out; p.ldo = c.ldo; p.T = (int)c.T; p.K = (int)c.K; p.cols = n.cols;
  p.m_tiles = n.t_tiles; p.n_tiles = n.tiles / n.t_tiles;
  p.inv_n = div_reciprocal(p.n_tiles); p.bias_f32 = (int)c.bias_f32; p.status = c.status;
  p.boxes = ((uintptr_t)c.out | (uintptr_t)(c.ldo * size)) % 16 == 0;
  CUtensorMap ta, tb, tc;
  int rc = make_tmap(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.codes, {(uint64_t)c.K, (uint64_t)c.T}, {(uint64_t)c.ldc}, {BK, 128});
  if (rc == 0) rc = make_tmap(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.q, {(uint64_t)c.K, (uint64_t)c.N}, {(uint64_t)c.ldw}, {BK, 128});
  tc = ta;
  if (rc == 0 && p.boxes) rc = F32 ? make_tmap_2d_f32(&tc, c.out, (uint64_t)n.cols, (uint64_t)c.T, (uint64_t)c.ldo, 32, 32)
                                   : make_tmap_2d_bf16(&tc, c.out, (uint64_t)n.cols, (uint64_t)c.T, (uint64_t)c.ldo, 64, 32);
  if (rc) return rc;
  launch_step(early, int8_tile_kernel<GATED, F32>, dim3(n.grid), n.threads, n.smem, st, ta, tb, tc, p);
  return -(int)cudaGetLastError();
}

}  // namespace inv

using namespace inv;

extern "C" int inv_int8_rows(const void* call) {
  const Int8Call& c = *static_cast<const Int8Call*>(call);
  if (c.T <= 0 || c.K <= 0) return 0;
  if (c.T > INT8_MOST || c.K > INT8_MOST) return -ERR_BAD_ARG;
  return launch_int8_rows(c, (cudaStream_t)c.stream);
}

// Whether a product makes the codes for itself and wants no place for them.
extern "C" int inv_int8_alone(long T, long N, long K) { return int8_route(T, N, K, false) == INT8_FEW; }

// The plan's numbers in their order, for who wants to look at them.
extern "C" int inv_int8_plan(long T, long N, long K, int gated, int* out) {
  if (T < 1 || T > INT8_MOST || N < 1 || N > INT8_MOST || K < 1 || K > INT8_MOST_K || (gated && N < 2)) return -ERR_BAD_ARG;
  const Int8Plan n = int8_plan(T, N, K, gated != 0);
  for (const int v : {n.route, n.cols, n.grid, n.cluster, n.threads, n.smem, n.tiles, n.t_tiles, n.tb, n.per, n.kb, n.parts, n.stages}) *out++ = v;
  return 0;
}

// Codes first where x is given and the product does not make them, then the product, which starts while they are made: the kernel of the codes is launched plainly, so everything in front of it is
// complete when the product's first weights are read.
extern "C" int inv_int8_linear(const void* call) {
  const Int8Call& c = *static_cast<const Int8Call*>(call);
  if (c.T <= 0 || c.N <= 0 || c.K <= 0) return 0;
  if (c.T > INT8_MOST || c.N > INT8_MOST || c.K > INT8_MOST_K || c.ldw % 16 || c.ldc % 16 || (((uintptr_t)c.q | (uintptr_t)c.codes) & 15) || (c.gated && c.N % 2) ||
      (c.gated && c.N < 2))
    return -ERR_BAD_ARG;
  cudaStream_t st = (cudaStream_t)c.stream;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device)) return -(int)e;
  const bool early = c.x != nullptr;
  const Int8Plan plan = int8_plan(c.T, c.N, c.K, c.gated != 0);
  const int route = plan.route, tb = plan.tb;
  if (route != INT8_FEW && (c.codes == nullptr || c.sx == nullptr)) return -ERR_BAD_ARG;
  if (route == INT8_FEW) {
#define INV_FEW(TT) (c.gated ? launch_int8_few<TT, true>(c, plan, device, st) : launch_int8_few<TT, false>(c, plan, device, st))
    return c.T == 1 ? INV_FEW(1) : c.T == 2 ? INV_FEW(2) : INV_FEW(4);
#undef INV_FEW
  }
  if (early)
    if (const int e = launch_int8_rows(c, st)) return e;
  if (route == INT8_SPLIT) {
#define INV_SPLIT(TB) (c.gated ? launch_int8_split<TB, true>(c, plan, early, device, st) : launch_int8_split<TB, false>(c, plan, early, device, st))
    return tb <= 16 ? INV_SPLIT(16) : tb <= 32 ? INV_SPLIT(32) : tb <= 64 ? INV_SPLIT(64) : INV_SPLIT(128);
#undef INV_SPLIT
  }
  if (c.gated) return c.out_f32 ? launch_int8_tiles<true, true>(c, plan, early, device, st) : launch_int8_tiles<true, false>(c, plan, early, device, st);
  return c.out_f32 ? launch_int8_tiles<false, true>(c, plan, early, device, st) : launch_int8_tiles<false, false>(c, plan, early, device, st);
}
