// Norms of query and key heads with the position rotation in the same pass, and their backward pass.
//
// qkv is token-major [T, (H + 2 Hkv) D]. A query or key head x becomes R_p(w * x * r) with r = (mean x^2 + eps)^-1/2, w the weight of the queries' or
// the keys' norm ([D], shared by the heads) and R_p the half-split rotation of its first `rot` values at the token's position; value heads are copied.
// Backward, with g = R_p^T dy and xh = x r:  dw = sum over tokens and heads of g xh,  dx = r (g w - xh mean(g w xh)).
//
// Both are bound by memory: forward reads and writes the buffer once, backward reads dy, reads x of the normed heads and writes dx. Heads live in the
// lanes of a warp as units that hold both halves of their rotation pairs (head_norm.cuh), with two 16-byte loads a lane and no shuffles but the sum
// over a head. The warps stay and take heads that lie one behind the other; what they read next is on its way meanwhile. 16384 tokens, 32 heads of 128 on
// 8, bf16: forward 72 us (5.6 TB/s), backward 114 (5.0), sums of dw 8 at most, all three in a graph 178; instructions, at two thirds of what the SMs can
// issue, come next to memory, so the arithmetic is in pairs.
#include "head_norm.cuh"
#include "inv_api.h"

namespace inv {

struct QkNorm {
  const void *x, *wq, *wk, *dy;
  void* y;                     // forward: the result; backward: dx
  const float *cos_t, *sin_t;
  const int* pos;              // position of every token; null: t % S
  float* part;                 // backward: sums of dw, [ctas_q, D] of the queries' norm and [the others, D] of the keys'; null: not asked for
  int* status;
  int T, S, H, Hkv, D, rot, table_rows, ctas_q;
  int rounds, rounds_q;        // steps of a run (Walk); backward: of the key and value heads, of the query heads
  uint32_t inv_s, inv_slots, inv_slots_q;      // div_reciprocal of S and of the head slots of a token (backward: key and value heads, query heads)
  long ld_x, ld_y, ld_dy;
  float eps, inv_d;
};

// The head slots of a call, a token's behind the other's, dealt to warps: 32 / L at a time, in runs of `stride` from `from` on. A run is one step, or the
// head slots of a token where those are whole steps: its angles are then loaded once.
struct Walk {
  long from, stride, jump;
  int base, step, all;
  __device__ __forceinline__ Walk(int step, int rounds, int warp, int warps, int all)
      : from((long)warp * step * rounds), stride((long)step * rounds), jump((long)warps * step * rounds), base((int)from), step(step), all(all) {}
  __device__ __forceinline__ bool more() const { return from < all; }
  __device__ __forceinline__ bool first() const { return base == from; }
  __device__ __forceinline__ void next() {
    base += step;
    if (base >= min(from + stride, (long)all)) {
      from += jump;
      base = (int)from;
    }
  }
};
// Token and head of a slot; one past the end repeats the last.
struct Slot {
  int tok, hd;
  bool in;
  __device__ __forceinline__ Slot(int s, int all, int slots, uint32_t inv) {
    const int at = min(s, all - 1);
    in = s < all;
    tok = div_by(at, slots, inv);
    hd = at - tok * slots;
  }
};
__device__ __forceinline__ void load_turn(const QkNorm& p, int t, int u, const HeadUnit& h, Turn& turn) {
  turn.load(p.cos_t, p.sin_t, p.rot, table_row(p.pos ? p.pos[t] : t - div_by(t, p.S, p.inv_s) * p.S, p.table_rows, p.status), u, h);
}

// With loads to registers, four units a lane, forward 75 us, and backward, two units, 140. Two CTAs an SM: forward with three 5 us more, with four 35.
template <typename T>
using QkFwdRing = UnitRing<T, 1, 6, 8>;
template <typename T>
using QkBwdRing = UnitRing<T, 2, sizeof(T) == 2 ? 3 : 2, 8>;

constexpr int QK_FWD_CTAS = 2;
template <typename T, int L>
__global__ void __launch_bounds__(256, QK_FWD_CTAS) qk_norm_fwd_kernel(const __grid_constant__ QkNorm p) {
  using Ring = QkFwdRing<T>;
  constexpr int HPW = 32 / L, ST = Ring::STAGES;
  extern __shared__ uint4 ring[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane % L, sub = lane / L;
  const int slots = p.H + 2 * p.Hkv, all = p.T * slots;
  const HeadUnit h(u, p.D, p.rot);
  wait_previous();
  release_next();
  uint4* mine = Ring::of_lane(ring);
  Walk now(HPW, p.rounds, blockIdx.x * 8 + warp, gridDim.x * 8, all), ahead = now;
  auto copy = [&](int stage) {
    if (ahead.more()) {
      const Slot s(ahead.base + sub, all, slots, p.inv_slots);
      Ring::copy(mine, stage, 0, (const T*)p.x + s.tok * p.ld_x + s.hd * p.D, h);
      ahead.next();
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) copy(i);
  Turn turn;
  for (int stage = 0; now.more(); now.next()) {
    const Slot s(now.base + sub, all, slots, p.inv_slots);
    if (p.rot && now.first()) load_turn(p, s.tok, u, h, turn);
    copies_wait<ST - 2>();
    RawUnit<T> raw;
    Ring::get(mine, stage, 0, raw);
    uint64_t v[8];
    raw.get(v);
    head_norm<L>(v, (const T*)(s.hd < p.H ? p.wq : p.wk), h, p.inv_d, p.eps);
    copy(stage ? stage - 1 : ST - 1);                // where the step before this one was
    if (++stage == ST) stage = 0;
    if (s.hd < p.H + p.Hkv) {
      turn.apply<false>(h, v);
      raw.set(v);
    }
    if (s.in && h.has) raw.store((T*)p.y + s.tok * p.ld_y + s.hd * p.D, h);
  }
}

// The first ctas_q CTAs take the query heads, the others the key and value heads: a lane then keeps the sums of one dw in registers. A CTA adds its warps'
// sums in order and leaves one row.
template <typename T, int L>
__global__ void __launch_bounds__(256, 2) qk_norm_bwd_kernel(const __grid_constant__ QkNorm p) {
  using Ring = QkBwdRing<T>;
  constexpr int HPW = 32 / L, ST = Ring::STAGES;
  extern __shared__ uint4 ring[];
  __shared__ float sums[8][L * 16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane % L, sub = lane / L;
  const bool keys = (int)blockIdx.x >= p.ctas_q;
  const int first = keys ? p.H : 0, normed = keys ? p.Hkv : p.H, slots = keys ? 2 * p.Hkv : p.H, all = p.T * slots;
  const uint32_t inv = keys ? p.inv_slots : p.inv_slots_q;
  const int cta = keys ? blockIdx.x - p.ctas_q : blockIdx.x, ctas = keys ? gridDim.x - p.ctas_q : p.ctas_q;
  const HeadUnit h(u, p.D, p.rot);
  wait_previous();
  release_next();
  uint4* mine = Ring::of_lane(ring);
  Walk now(HPW, keys ? p.rounds : p.rounds_q, cta * 8 + warp, ctas * 8, all), ahead = now;
  auto copy = [&](int stage) {
    if (ahead.more()) {
      const Slot s(ahead.base + sub, all, slots, inv);
      const int at = (first + s.hd) * p.D;
      const T* dy = (const T*)p.dy + s.tok * p.ld_dy + at;
      Ring::copy(mine, stage, 0, s.hd < normed ? (const T*)p.x + s.tok * p.ld_x + at : dy, h);      // of values only dy
      Ring::copy(mine, stage, 1, dy, h);
      ahead.next();
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) copy(i);
  uint64_t dw[8], w[8];
  load_unit((const T*)(keys ? p.wk : p.wq), h, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0;
  Turn turn;
  for (int stage = 0; now.more(); now.next()) {
    const Slot s(now.base + sub, all, slots, inv);
    if (p.rot && now.first()) load_turn(p, s.tok, u, h, turn);
    copies_wait<ST - 2>();
    RawUnit<T> rx, rg;
    Ring::get(mine, stage, 0, rx);
    Ring::get(mine, stage, 1, rg);
    uint64_t v[8], g[8];
    rx.get(v);
    rg.get(g);
    const float r = head_rstd<L>(v, h, p.inv_d, p.eps);
    copy(stage ? stage - 1 : ST - 1);                // where the step before this one was
    if (++stage == ST) stage = 0;
    turn.apply<true>(h, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mul_pair(v[i], pair_of(r, r));           // xh
    if (s.in && s.hd < normed) {
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
    if (s.hd < normed) rg.set(g);
    if (s.in && h.has) rg.store((T*)p.y + s.tok * p.ld_y + (first + s.hd) * p.D, h);
  }
  if (!p.part) return;
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
  const int r0 = blockIdx.y ? rows_q : 0, r1 = blockIdx.y ? rows : rows_q, mode = blockIdx.y ? mode_k : mode_q;
  if (mode == 3) return;
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
  void* out = blockIdx.y ? dwk : dwq;
  if (mode == 2) ((float*)out)[col] += v;
  else if (mode == 1) ((float*)out)[col] = v;
  else ((__nv_bfloat16*)out)[col] = __float2bfloat16_rn(v);
}

// A token's head slots where they are whole steps and that leaves each of the warps, which stay, two tokens or more; else a step, which deals them evenly.
static int qk_rounds(long T, int slots, int hpw, long ctas) { return slots > hpw && slots % hpw == 0 && T >= 16 * ctas ? slots / hpw : 1; }
static int qk_ctas(long T, int slots, int hpw, long share) {
  const long ctas = (T * slots + 8 * hpw - 1) / (8 * hpw);
  return (int)(ctas < share ? ctas : share);
}
// CTAs of the backward kernel, in proportion to the bytes of either side: dy, x and dx of a normed head, dy and dx of a value head.
struct QkBwdCut {
  int ctas_q, ctas;
  QkBwdCut(int T, int H, int Hkv, int D) {
    const int hpw = 32 / head_lanes(D);
    long share = H ? 296l * 3 * H / (3 * H + 5 * Hkv) : 0;
    if (H && share < 1) share = 1;
    ctas_q = qk_ctas(T, H, hpw, share);
    ctas = ctas_q + qk_ctas(T, 2 * Hkv, hpw, 296 - share);
  }
};

}  // namespace inv

using namespace inv;

// What a call's entry is given (the Python side packs the same fields in the same order).
struct QkNormDesc {
  const void* x;                   // [T, (H + 2 Hkv) D], bf16 or fp32 (then the weights are too), rows ld_x apart
  void* y;                         // forward: as x; backward: dx
  const void *wq, *wk;             // [D]
  const float *cos_t, *sin_t;      // [table_rows, rot / 2], or null with rot 0
  const int* pos;                  // [T], or null
  int* status;
  void* stream;
  // backward
  const void* dy;
  void *dwq, *dwk;                 // [D]; mode 0: bf16, written; 1: fp32, written; 2: fp32, added to; 3: not asked for
  float* part;                     // 296 rows of [D], or null with both modes 3
  long ld_x, ld_y, ld_dy, table_rows, T, S, H, Hkv, D, rot, f32, mode_q, mode_k;
  double eps;
};
static int qk_norm_args(const QkNormDesc& d, QkNorm& p) {
  const long vec = d.f32 ? 4 : 8, top = 0x7fff0000l;
  if (d.D < 16 || d.D > 256 || d.D % 16 || d.rot < 0 || d.rot > d.D || d.rot % 16 || d.H < 0 || d.Hkv < 0 || d.H + d.Hkv < 1 || d.S < 1 || d.S > top ||
      d.T < 0 || d.T > top || d.H + 2 * d.Hkv > top || d.T * (d.H + 2 * d.Hkv) > top)
    return -ERR_BAD_ARG;
  if (d.rot && (!d.cos_t || !d.sin_t || d.table_rows < 1 || d.table_rows > top)) return -ERR_BAD_ARG;
  if (d.ld_x % vec || d.ld_y % vec || d.ld_dy % vec) return -ERR_BAD_ARG;
  if (((uintptr_t)d.x | (uintptr_t)d.y | (uintptr_t)d.dy | (uintptr_t)d.wq | (uintptr_t)d.wk | (uintptr_t)d.cos_t | (uintptr_t)d.sin_t) % 16) return -ERR_BAD_ARG;
  p = QkNorm{d.x, d.wq, d.wk, d.dy, d.y, d.cos_t, d.sin_t, d.pos, d.part, d.status, (int)d.T, (int)d.S, (int)d.H, (int)d.Hkv, (int)d.D, (int)d.rot,
             (int)d.table_rows, 0, 0, 0, div_reciprocal((int)d.S), 0, 0, d.ld_x, d.ld_y, d.ld_dy, (float)d.eps, 1.f / (float)d.D};
  return 0;
}
template <typename T, int L>
static int qk_fwd(const QkNorm& p, unsigned grid, cudaStream_t st) {
  static OncePerDevice ready;
  if (int rc = raise_smem(qk_norm_fwd_kernel<T, L>, QkFwdRing<T>::BYTES, ready)) return rc;
  launch_early(qk_norm_fwd_kernel<T, L>, grid, 256, QkFwdRing<T>::BYTES, st, p);
  return 0;
}
template <typename T, int L>
static int qk_bwd(const QkNorm& p, unsigned grid, cudaStream_t st) {
  static OncePerDevice ready;
  if (int rc = raise_smem(qk_norm_bwd_kernel<T, L>, QkBwdRing<T>::BYTES, ready)) return rc;
  launch_early(qk_norm_bwd_kernel<T, L>, grid, 256, QkBwdRing<T>::BYTES, st, p);
  return 0;
}
#define INV_QK_L(T, LAUNCH)                    \
  switch (head_lanes(p.D)) {                   \
    case 1: return LAUNCH<T, 1>(p, grid, st);  \
    case 2: return LAUNCH<T, 2>(p, grid, st);  \
    case 4: return LAUNCH<T, 4>(p, grid, st);  \
    case 8: return LAUNCH<T, 8>(p, grid, st);  \
    default: return LAUNCH<T, 16>(p, grid, st); \
  }
static int qk_fwd(const QkNorm& p, bool f32, unsigned grid, cudaStream_t st) {
  if (f32) INV_QK_L(float, qk_fwd)
  INV_QK_L(__nv_bfloat16, qk_fwd)
}
static int qk_bwd(const QkNorm& p, bool f32, unsigned grid, cudaStream_t st) {
  if (f32) INV_QK_L(float, qk_bwd)
  INV_QK_L(__nv_bfloat16, qk_bwd)
}
#undef INV_QK_L

extern "C" int inv_qk_norm_fwd(const QkNormDesc* d) {
  QkNorm p;
  if (int rc = qk_norm_args(*d, p)) return rc;
  if (p.T == 0) return 0;
  const int slots = p.H + 2 * p.Hkv, hpw = 32 / head_lanes(p.D);
  p.inv_slots = div_reciprocal(slots);
  const unsigned grid = (unsigned)qk_ctas(p.T, slots, hpw, 148 * QK_FWD_CTAS);
  p.rounds = qk_rounds(p.T, slots, hpw, grid);
  cudaStream_t st = (cudaStream_t)d->stream;
  if (int rc = qk_fwd(p, d->f32 != 0, grid, st)) return rc;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}

extern "C" int inv_qk_norm_bwd(const QkNormDesc* d) {
  QkNorm p;
  if (int rc = qk_norm_args(*d, p)) return rc;
  const bool sums = d->mode_q != 3 || d->mode_k != 3;
  if (sums != (p.part != nullptr)) return -ERR_BAD_ARG;
  cudaStream_t st = (cudaStream_t)d->stream;
  unsigned grid = 0;
  if (p.T > 0) {
    const QkBwdCut cut(p.T, p.H, p.Hkv, p.D);
    p.inv_slots = div_reciprocal(p.Hkv ? 2 * p.Hkv : 1);
    p.inv_slots_q = div_reciprocal(p.H ? p.H : 1);
    const int hpw = 32 / head_lanes(p.D);
    p.rounds_q = qk_rounds(p.T, p.H, hpw, cut.ctas_q);
    p.rounds = qk_rounds(p.T, 2 * p.Hkv, hpw, cut.ctas - cut.ctas_q);
    p.ctas_q = cut.ctas_q;
    grid = (unsigned)cut.ctas;
    if (int rc = qk_bwd(p, d->f32 != 0, grid, st)) return rc;
  }
  if (sums)
    launch_early(qk_norm_dw_kernel, dim3((p.D + 31) / 32, 2), 1024, 0, st, (const float*)p.part, p.ctas_q, (int)grid, p.D, d->dwq, d->dwk, (int)d->mode_q,
                 (int)d->mode_k);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}
