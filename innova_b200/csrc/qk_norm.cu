// Norms of query and key heads with the position rotation in the same pass, and their backward pass.
//
// qkv is token-major [T, (H + 2 Hkv) D]. A query or key head x becomes R_p(w * x * r) with r = (mean x^2 + eps)^-1/2, w the weight of the queries' or
// the keys' norm ([D], shared by the heads) and R_p the half-split rotation of its first `rot` values at the token's position; value heads are copied.
// Backward, with g = R_p^T dy and xh = x r:  dw = sum over tokens and heads of g xh,  dx = r (g w - xh mean(g w xh)).
//
// Both are bound by memory: forward reads and writes the buffer once, backward reads dy, reads x of the normed heads and writes dx. Heads live in the
// lanes of a warp as units that hold both halves of their rotation pairs (head_norm.cuh), with two 16-byte loads a lane and no shuffles but the sum
// over a head. A warp takes one token and walks over its heads, so that the token's cosines and sines are loaded once.
#include "head_norm.cuh"
#include "inv_api.h"

namespace inv {

struct QkNorm {
  const void *x, *wq, *wk, *dy;
  void* y;                     // forward: the result; backward: dx
  const float *cos_t, *sin_t;
  const int* pos;              // position of every token; null: t % S
  float* part;                 // backward: [grid, 2, D] sums of dw
  int* status;
  int T, S, H, Hkv, D, rot, table_rows, chunk;
  long ld_x, ld_y, ld_dy;
  float eps, inv_d;
};

// A warp's share: token `t`, head slots [s0, s0 + chunk) of H + 2 Hkv. chunk: all of them where tokens alone fill the GPU.
template <typename T, int L>
__global__ void __launch_bounds__(256) qk_norm_fwd_kernel(const __grid_constant__ QkNorm p) {
  constexpr int HPW = 32 / L;
  const int lane = threadIdx.x & 31, u = lane % L, sub = lane / L;
  const int slots = p.H + 2 * p.Hkv, per = (slots + p.chunk - 1) / p.chunk;
  const long item = blockIdx.x * 8l + (threadIdx.x >> 5);
  if (item >= (long)p.T * per) return;
  const int t = (int)(item / per), s0 = (int)(item % per) * p.chunk, s1 = min(slots, s0 + p.chunk);
  const HeadUnit h(u, p.D, p.rot);
  Turn turn;
  if (p.rot && s0 < p.H + p.Hkv) turn.load(p.cos_t, p.sin_t, p.rot, table_row(p.pos ? p.pos[t] : t % p.S, p.table_rows, p.status), u, h);
  const T* x = (const T*)p.x + t * p.ld_x;
  T* y = (T*)p.y + t * p.ld_y;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int lo = max(s0, part ? p.H : 0), hi = min(s1, part ? p.H + p.Hkv : p.H);
    if (lo >= hi) continue;
    float w[16];
    load_unit((const T*)(part ? p.wk : p.wq), h, w);
#pragma unroll 2
    for (int s = lo; s < hi; s += HPW) {
      const bool ok = s + sub < hi;                 // lanes past the last head repeat it and store nothing
      const long at = (long)min(s + sub, hi - 1) * p.D;
      float v[16];
      load_unit(x + at, h, v);
      const float r = head_rstd<L>(v, p.inv_d, p.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = v[i] * r * w[i];
      turn.apply<false>(h, v);
      if (ok) store_unit(y + at, h, v);
    }
  }
  for (int s = max(s0, p.H + p.Hkv); s < s1; s += HPW)
    if (s + sub < s1) {
      const long at = (long)(s + sub) * p.D;
      float v[16];
      load_unit(x + at, h, v);
      store_unit(y + at, h, v);
    }
}

// Warps walk over the tokens and keep their sums of dw in registers; a CTA adds its warps' in order and leaves one row.
template <typename T, int L>
__global__ void __launch_bounds__(256) qk_norm_bwd_kernel(const __grid_constant__ QkNorm p) {
  constexpr int HPW = 32 / L;
  __shared__ float sums[8][2][L * 16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane % L, sub = lane / L;
  const int slots = p.H + 2 * p.Hkv, per = (slots + p.chunk - 1) / p.chunk;
  const HeadUnit h(u, p.D, p.rot);
  float dw[2][16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[0][i] = dw[1][i] = 0.f;
  for (long item = blockIdx.x * 8l + warp; item < (long)p.T * per; item += gridDim.x * 8l) {
    const int t = (int)(item / per), s0 = (int)(item % per) * p.chunk, s1 = min(slots, s0 + p.chunk);
    Turn turn;
    if (p.rot && s0 < p.H + p.Hkv) turn.load(p.cos_t, p.sin_t, p.rot, table_row(p.pos ? p.pos[t] : t % p.S, p.table_rows, p.status), u, h);
    const T *x = (const T*)p.x + t * p.ld_x, *dy = (const T*)p.dy + t * p.ld_dy;
    T* dx = (T*)p.y + t * p.ld_y;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int lo = max(s0, part ? p.H : 0), hi = min(s1, part ? p.H + p.Hkv : p.H);
      if (lo >= hi) continue;
      float w[16];
      load_unit((const T*)(part ? p.wk : p.wq), h, w);
      for (int s = lo; s < hi; s += HPW) {
        const bool ok = s + sub < hi;
        const long at = (long)min(s + sub, hi - 1) * p.D;
        float v[16], g[16];
        load_unit(x + at, h, v);
        load_unit(dy + at, h, g);
        const float r = head_rstd<L>(v, p.inv_d, p.eps);
        turn.apply<true>(h, g);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[i] *= r;                                // xh
          if (ok) dw[part][i] = fmaf(g[i], v[i], dw[part][i]);
          g[i] *= w[i];
          dot = fmaf(g[i], v[i], dot);
        }
        const float mean = head_sum<L>(dot) * p.inv_d;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = r * (g[i] - v[i] * mean);
        if (ok) store_unit(dx + at, h, g);
      }
    }
    for (int s = max(s0, p.H + p.Hkv); s < s1; s += HPW)
      if (s + sub < s1) {
        const long at = (long)(s + sub) * p.D;
        float v[16];
        load_unit(dy + at, h, v);
        store_unit(dx + at, h, v);
      }
  }
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = dw[part][i];
#pragma unroll
      for (int o = 16; o >= L; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (sub == 0 && h.has) sums[warp][part][(i < 8 ? h.e0 : h.e1 - 8) + i] = v;
    }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * p.D; e += 256) {
    const int part = e / p.D, d = e % p.D;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sums[w][part][d];
    p.part[(long)blockIdx.x * 2 * p.D + e] = v;
  }
}

// dw[part][d] = (what is there, with `add`) + the sum of `rows` rows, in an order that only their number decides. A CTA: 32 columns.
__global__ void __launch_bounds__(256) qk_norm_dw_kernel(const float* __restrict__ part, int rows, int D, void* dwq, void* dwk, int mode_q, int mode_k) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (e < 2 * D)
    for (int r = warp; r < rows; r += 8) v += part[(long)r * 2 * D + e];
  sums[warp][lane] = v;
  __syncthreads();
  if (warp || e >= 2 * D) return;
  v = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) v += sums[w][lane];
  const int mode = e < D ? mode_q : mode_k, d = e % D;
  void* out = e < D ? dwq : dwk;
  if (mode == 2) ((float*)out)[d] += v;
  else if (mode == 1) ((float*)out)[d] = v;
  else ((__nv_bfloat16*)out)[d] = __float2bfloat16_rn(v);
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
    case 1: KERNEL<T, 1><<<grid, 256, 0, st>>>(p); break;                                                                     \
    case 2: KERNEL<T, 2><<<grid, 256, 0, st>>>(p); break;                                                                     \
    case 4: KERNEL<T, 4><<<grid, 256, 0, st>>>(p); break;                                                                     \
    case 8: KERNEL<T, 8><<<grid, 256, 0, st>>>(p); break;                                                                     \
    default: KERNEL<T, 16><<<grid, 256, 0, st>>>(p);                                                                          \
  }

// x, y: [T, (H + 2 Hkv) D], bf16 or fp32 (then the weights are too), rows ld_x and ld_y apart. cos_t, sin_t: [table_rows, rot / 2] fp32.
extern "C" int inv_qk_norm_fwd(const void* x, long ld_x, void* y, long ld_y, const void* wq, const void* wk, const float* cos_t, const float* sin_t,
                               int table_rows, const int* pos, int T, int S, int H, int Hkv, int D, int rot, float eps, int f32, int* status,
                               void* stream) {
  QkNorm p{x, wq, wk, nullptr, y, cos_t, sin_t, pos, nullptr, status, T, S, H, Hkv, D, rot, table_rows, 0, ld_x, ld_y, 0, eps, 1.f / (float)D};
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

// CTAs of the backward kernel, and so rows of [2, D] floats that its caller provides.
extern "C" int inv_qk_norm_bwd_grid(int T, int H, int Hkv, int D) {
  if (T <= 0 || D < 16 || D > 256) return 0;
  const int slots = H + 2 * Hkv, chunk = slot_chunk(T, slots, 32 / head_lanes(D));
  const long ctas = ((long)T * ((slots + chunk - 1) / chunk) + 7) / 8;
  return (int)(ctas < 148 * 4 ? ctas : 148 * 4);
}

// dx, dy as y and x above. dwq, dwk: [D]; mode 0: bf16, written; 1: fp32, written; 2: fp32, added to.
extern "C" int inv_qk_norm_bwd(const void* x, long ld_x, const void* dy, long ld_dy, void* dx, long ld_dx, const void* wq, const void* wk,
                               const float* cos_t, const float* sin_t, int table_rows, const int* pos, void* dwq, int mode_q, void* dwk, int mode_k,
                               float* part, int T, int S, int H, int Hkv, int D, int rot, float eps, int f32, int* status, void* stream) {
  QkNorm p{x, wq, wk, dy, dx, cos_t, sin_t, pos, part, status, T, S, H, Hkv, D, rot, table_rows, 0, ld_x, ld_dx, ld_dy, eps, 1.f / (float)D};
  if (int rc = qk_norm_args(p, f32)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)inv_qk_norm_bwd_grid(T, H, Hkv, D);
  if (grid) {
    p.chunk = slot_chunk(T, H + 2 * Hkv, 32 / head_lanes(D));
    if (f32) { INV_QK_L(float, qk_norm_bwd_kernel) } else { INV_QK_L(__nv_bfloat16, qk_norm_bwd_kernel) }
  }
  qk_norm_dw_kernel<<<(2 * D + 31) / 32, 256, 0, st>>>(part, (int)grid, D, dwq, dwk, mode_q, mode_k);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}
