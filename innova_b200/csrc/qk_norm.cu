// Norms of query and key heads with the position rotation in the same pass, and their backward pass.
//
// qkv is token-major [T, (H + 2 Hkv) D]. A query or key head x becomes R_p(w * x * r) with r = (mean x^2 + eps)^-1/2, w the weight of the queries' or
// the keys' norm ([D], shared by the heads) and R_p the half-split rotation of its first `rot` values at the token's position; value heads are copied.
// Backward, with g = R_p^T dy and xh = x r:  dw = sum over tokens and heads of g xh,  dx = r (g w - xh mean(g w xh)).
//
// Both are bound by memory: forward reads and writes the buffer once, backward reads dy, reads x of the normed heads and writes dx. Heads live in the
// lanes of a warp as units that hold both halves of their rotation pairs (head_norm.cuh), with two 16-byte loads a lane and no shuffles but the sum
// over a head. A warp takes one token and walks over its heads, so that the token's cosines and sines are loaded once, and has the loads of several
// heads on their way at once.
#include "head_norm.cuh"
#include "inv_api.h"

namespace inv {

struct QkNorm {
  const void *x, *wq, *wk, *dy;
  void* y;                     // forward: the result; backward: dx
  const float *cos_t, *sin_t;
  const int* pos;              // position of every token; null: t % S
  float* part;                 // backward: sums of dw, [ctas_q, D] of the queries' norm and [the others, D] of the keys'
  int* status;
  int T, S, H, Hkv, D, rot, table_rows, chunk, ctas_q, chunk_q;      // backward: chunk of the key and value heads, chunk_q of the query heads
  long ld_x, ld_y, ld_dy;
  float eps, inv_d;
};

// Units that a lane has on its way at once.
template <typename T>
constexpr int UNITS = sizeof(T) == 2 ? 4 : 2;

template <typename T, int L>
__device__ __forceinline__ void load_turn(const QkNorm& p, int t, int u, const HeadUnit& h, Turn& turn) {
  if (p.rot) turn.load(p.cos_t, p.sin_t, p.rot, table_row(p.pos ? p.pos[t] : t % p.S, p.table_rows, p.status), u, h);
}

// A warp's share: token `t`, head slots [s0, s0 + chunk) of H + 2 Hkv. chunk: all of them where tokens alone fill the GPU.
template <typename T, int L>
__global__ void __launch_bounds__(256, 2) qk_norm_fwd_kernel(const __grid_constant__ QkNorm p) {
  constexpr int HPW = 32 / L, N = UNITS<T>;
  const int lane = threadIdx.x & 31, u = lane % L, sub = lane / L;
  const int slots = p.H + 2 * p.Hkv, per = (slots + p.chunk - 1) / p.chunk;
  const long item = blockIdx.x * 8l + (threadIdx.x >> 5);
  wait_previous();
  release_next();
  if (item >= (long)p.T * per) return;
  const int t = (int)(item / per), s0 = (int)(item % per) * p.chunk, s1 = min(slots, s0 + p.chunk);
  const HeadUnit h(u, p.D, p.rot);
  const T* x = (const T*)p.x + t * p.ld_x;
  T* y = (T*)p.y + t * p.ld_y;
  Turn turn;
  load_turn<T, L>(p, t, u, h, turn);
  for (int s = s0; s < s1; s += N * HPW) {
    RawUnit<T> raw[N];
#pragma unroll
    for (int j = 0; j < N; ++j) raw[j].fetch(x + (long)min(s + j * HPW + sub, s1 - 1) * p.D, h);      // lanes past the last head repeat it
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int slot = s + j * HPW + sub;
      if (s + j * HPW >= s1) break;
      const bool normed = slot < p.H + p.Hkv;
      uint64_t v[8];
      raw[j].get(v);
      head_norm<L>(v, (const T*)(slot < p.H ? p.wq : p.wk), h, p.inv_d, p.eps);
      if (normed) {
        turn.apply<false>(h, v);
        raw[j].set(v);
      }
      if (slot < s1 && h.has) raw[j].store(y + (long)slot * p.D, h);
    }
  }
}

// The first ctas_q CTAs take the query heads, the others the key and value heads: a lane then keeps the sums of one dw in registers. Warps walk over the
// tokens; a CTA adds its warps' sums in order and leaves one row.
template <typename T, int L>
__global__ void __launch_bounds__(256, 2) qk_norm_bwd_kernel(const __grid_constant__ QkNorm p) {
  constexpr int HPW = 32 / L, N = UNITS<T> / 2;
  __shared__ float sums[8][L * 16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane % L, sub = lane / L;
  const bool keys = (int)blockIdx.x >= p.ctas_q;
  const int first = keys ? p.H : 0, normed = keys ? p.H + p.Hkv : p.H, slots = keys ? 2 * p.Hkv : p.H, chunk = keys ? p.chunk : p.chunk_q;
  const int per = (slots + chunk - 1) / chunk, cta = keys ? blockIdx.x - p.ctas_q : blockIdx.x, ctas = keys ? gridDim.x - p.ctas_q : p.ctas_q;
  const HeadUnit h(u, p.D, p.rot);
  wait_previous();
  release_next();
  uint64_t dw[8], w[8];
  load_unit((const T*)(keys ? p.wk : p.wq), h, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0;
  for (long item = cta * 8l + warp; item < (long)p.T * per; item += ctas * 8l) {
    const int t = (int)(item / per), s0 = first + (int)(item - (long)t * per) * chunk, s1 = min(first + slots, s0 + chunk);
    const T *x = (const T*)p.x + t * p.ld_x, *dy = (const T*)p.dy + t * p.ld_dy;
    T* dx = (T*)p.y + t * p.ld_y;
    Turn turn;
    load_turn<T, L>(p, t, u, h, turn);
    for (int s = s0; s < s1; s += N * HPW) {
      RawUnit<T> rx[N], rg[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int slot = min(s + j * HPW + sub, s1 - 1);                        // lanes past the last head repeat it
        rg[j].fetch(dy + (long)slot * p.D, h);
        rx[j].fetch((slot < normed ? x : dy) + (long)slot * p.D, h);            // of values only the gradient
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (s + j * HPW >= s1) break;
        const int slot = s + j * HPW + sub;
        uint64_t v[8], g[8];
        rx[j].get(v);
        rg[j].get(g);
        const float r = head_rstd<L>(v, h, p.inv_d, p.eps);
        turn.apply<true>(h, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mul_pair(v[i], pair_of(r, r));       // xh
        if (slot < min(normed, s1)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) dw[i] = fma_pair(g[i], v[i], dw[i]);
        }
        uint64_t d0 = 0, d1 = 0;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          g[i] = mul_pair(g[i], w[i]);
          g[i + 1] = mul_pair(g[i + 1], w[i + 1]);
          d0 = fma_pair(g[i], v[i], d0);
          d1 = fma_pair(g[i + 1], v[i + 1], d1);
        }
        const float mean = head_sum<L>(add_pair(d0, d1), h) * -p.inv_d;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = mul_pair(pair_of(r, r), fma_pair(v[i], pair_of(mean, mean), g[i]));
        if (slot < normed) rg[j].set(g);
        if (slot < s1 && h.has) rg[j].store(dx + (long)slot * p.D, h);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 two = of_pair(dw[i / 2]);
    float v = i % 2 ? two.y : two.x;
#pragma unroll
    for (int o = 16; o >= L; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (sub == 0 && h.has) sums[warp][(i < 8 ? h.e0 : h.e1 - 8) + i] = v;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += 256) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sums[k][d];
    p.part[(long)blockIdx.x * p.D + d] = v;
  }
}

// dw[d] = (what is there, with `add`) + the sum of its rows, in an order that only their number decides. A CTA: 32 columns of the queries' or the keys'.
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* __restrict__ part, int rows_q, int rows, int D, void* dwq, void* dwk, int mode_q,
                                                          int mode_k) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  wait_previous();
  release_next();
  const int r0 = blockIdx.y ? rows_q : 0, r1 = blockIdx.y ? rows : rows_q;
  float v = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int r = r0 + warp; r < r1; r += 32) v += part[(long)r * D + d];
  }
  sums[warp][lane] = v;
  __syncthreads();
  v = sums[lane][warp];                              // warp <-> column, lane <-> the sum of a warp
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int col = blockIdx.x * 32 + warp;
  if (lane || col >= D) return;
  const int mode = blockIdx.y ? mode_k : mode_q;
  void* out = blockIdx.y ? dwk : dwq;
  if (mode == 2) ((float*)out)[col] += v;
  else if (mode == 1) ((float*)out)[col] = v;
  else ((__nv_bfloat16*)out)[col] = __float2bfloat16_rn(v);
}

// Slots a warp takes of a token: all, or as few as fill the GPU with warps (four to eight an SM hide the loads of a short call).
static int slot_chunk(int T, int slots, int hpw) {
  const int most = (slots + hpw - 1) / hpw * hpw;
  const long want = 148l * 32 / (T < 1 ? 1 : T);            // warps a token may have
  if (want <= 1) return most;
  int chunk = (int)((slots + want - 1) / want);
  chunk = (chunk + hpw - 1) / hpw * hpw;
  return chunk < most ? chunk : most;
}
// CTAs of the backward kernel, in proportion to the bytes of either side: dy, x and dx of a normed head, dy and dx of a value head. At most two an SM.
struct QkBwdCut {
  int chunk_q, chunk, ctas_q, ctas;
  QkBwdCut(int T, int H, int Hkv, int D) {
    const int hpw = 32 / head_lanes(D);
    const long want_q = H ? 148l * 2 * 3 * H / (3 * H + 5 * Hkv) : 0;
    chunk_q = slot_chunk(T, H, hpw);
    chunk = slot_chunk(T, 2 * Hkv, hpw);
    const long most_q = H ? ((long)T * ((H + chunk_q - 1) / chunk_q) + 7) / 8 : 0, most = Hkv ? ((long)T * ((2 * Hkv + chunk - 1) / chunk) + 7) / 8 : 0;
    const long lo_q = want_q > 0 || !H ? want_q : 1, lo = 148l * 2 - lo_q;
    ctas_q = (int)(most_q < lo_q ? most_q : lo_q);
    ctas = ctas_q + (int)(most < lo ? most : lo);
  }
};

}  // namespace inv

using namespace inv;

static int qk_norm_args(const QkNorm& p, int f32) {
  const int vec = f32 ? 4 : 8;
  if (p.D < 16 || p.D > 256 || p.D % 16 || p.rot < 0 || p.rot > p.D || p.rot % 16 || p.H < 0 || p.Hkv < 0 || p.H + p.Hkv < 1 || p.S < 1) return -ERR_BAD_ARG;
  if (p.rot && (!p.cos_t || !p.sin_t || p.table_rows < 1)) return -ERR_BAD_ARG;
  if (p.ld_x % vec || p.ld_y % vec || p.ld_dy % vec) return -ERR_BAD_ARG;
  if (((uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.dy | (uintptr_t)p.wq | (uintptr_t)p.wk | (uintptr_t)p.cos_t | (uintptr_t)p.sin_t) % 16) return -ERR_BAD_ARG;
  return 0;
}
#define INV_QK_L(T, KERNEL)                                                                                                   \
  switch (head_lanes(p.D)) {                                                                                                  \
    case 1: launch_early(KERNEL<T, 1>, grid, 256, 0, st, p); break;                                                                     \
    case 2: launch_early(KERNEL<T, 2>, grid, 256, 0, st, p); break;                                                                     \
    case 4: launch_early(KERNEL<T, 4>, grid, 256, 0, st, p); break;                                                                     \
    case 8: launch_early(KERNEL<T, 8>, grid, 256, 0, st, p); break;                                                                     \
    default: launch_early(KERNEL<T, 16>, grid, 256, 0, st, p);                                                                          \
  }

// x, y: [T, (H + 2 Hkv) D], bf16 or fp32 (then the weights are too), rows ld_x and ld_y apart. cos_t, sin_t: [table_rows, rot / 2] fp32.
extern "C" int inv_qk_norm_fwd(const void* x, long ld_x, void* y, long ld_y, const void* wq, const void* wk, const float* cos_t, const float* sin_t,
                               int table_rows, const int* pos, int T, int S, int H, int Hkv, int D, int rot, float eps, int f32, int* status,
                               void* stream) {
  QkNorm p{x, wq, wk, nullptr, y, cos_t, sin_t, pos, nullptr, status, T, S, H, Hkv, D, rot, table_rows, 0, 0, 0, ld_x, ld_y, 0, eps, 1.f / (float)D};
  if (int rc = qk_norm_args(p, f32)) return rc;
  if (T <= 0) return 0;
  const int slots = H + 2 * Hkv;
  p.chunk = slot_chunk(T, slots, 32 / head_lanes(D));
  const long items = (long)T * ((slots + p.chunk - 1) / p.chunk);
  const unsigned grid = (unsigned)((items + 7) / 8);
  cudaStream_t st = (cudaStream_t)stream;
  if (f32) { INV_QK_L(float, qk_norm_fwd_kernel) } else { INV_QK_L(__nv_bfloat16, qk_norm_fwd_kernel) }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}

// CTAs of the backward kernel, and so rows of [D] floats that its caller provides.
extern "C" int inv_qk_norm_bwd_grid(int T, int H, int Hkv, int D) {
  if (T <= 0 || D < 16 || D > 256 || H < 0 || Hkv < 0) return 0;
  return QkBwdCut(T, H, Hkv, D).ctas;
}

// dx, dy as y and x above. dwq, dwk: [D]; mode 0: bf16, written; 1: fp32, written; 2: fp32, added to.
extern "C" int inv_qk_norm_bwd(const void* x, long ld_x, const void* dy, long ld_dy, void* dx, long ld_dx, const void* wq, const void* wk,
                               const float* cos_t, const float* sin_t, int table_rows, const int* pos, void* dwq, int mode_q, void* dwk, int mode_k,
                               float* part, int T, int S, int H, int Hkv, int D, int rot, float eps, int f32, int* status, void* stream) {
  QkNorm p{x, wq, wk, dy, dx, cos_t, sin_t, pos, part, status, T, S, H, Hkv, D, rot, table_rows, 0, 0, 0, ld_x, ld_dx, ld_dy, eps, 1.f / (float)D};
  if (int rc = qk_norm_args(p, f32)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  unsigned grid = 0;
  if (T > 0) {
    const QkBwdCut cut(T, H, Hkv, D);
    p.chunk = cut.chunk;
    p.chunk_q = cut.chunk_q;
    p.ctas_q = cut.ctas_q;
    grid = (unsigned)cut.ctas;
    if (f32) { INV_QK_L(float, qk_norm_bwd_kernel) } else { INV_QK_L(__nv_bfloat16, qk_norm_bwd_kernel) }
  }
  launch_early(qk_norm_dw_kernel, dim3((D + 31) / 32, 2), 1024, 0, st, (const float*)part, p.ctas_q, (int)grid, D, dwq, dwk, mode_q, mode_k);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}
