// A whole mixture-of-experts layer for up to 64 tokens, in two launches.
//
//   p = softmax(R x);  y_t = r_t + [shared expert] + sum over the top_k largest p_te of p_te W2_e (silu(W1g_e x_t) * (W1u_e x_t))
//
// Such a layer reads every expert that some token goes to once and does little arithmetic, so weight bytes bound it. The training form (csrc/moe.cu) pads
// every expert to 128 rows and takes seven launches. Device times with 8 experts of 2048 x 5632, two for a token (in brackets the weights' bytes at 6.54 TB/s): 1 token 38 us
// (21), 4 tokens 69 (58), 16 tokens 92 (84), 64 tokens 102 (85), in 8 bits 31 (11), 50, 65 (42), 80 (43); 7 tokens, 6 of 64 experts of 1024 x 704 and a shared one 38 us
// (22). While it streams the second kernel reads 6.4 to 7 TB/s; the rest is the router with the launch behind it, 5 us, the fall from gate to down products, 3 to 5, and
// the sums with the end, 4. In 8 bits the conversions take two thirds of all issue slots.
//
// moe_few_router_kernel   a CTA a token: logits, softmax, the largest entries; clears the counters of the next kernel
// moe_few_kernel          gate and up products, down products and their sum, one CTA an SM, without a launch between them
//
// The second kernel's work is a list of items: 128 weight rows of one expert's gate and up product (eight and eight in turn) by all of K; then 128 rows of its down
// product by a part of K; then sums of 128 output columns for four tokens. CTAs draw items in order from a counter. Down items and sums wait for what they
// read; that comes from items drawn earlier, by CTAs that have all they need: a CTA draws its first item once it holds its tensor memory, for which it may have to wait
// for another stream's kernel on its SM. So every wait ends, whatever else runs on the GPU. An item is drawn when the one before it starts to load: one further ahead, the
// last items were spread less evenly (4 tokens of 8 experts 72.3 us, 69.5 so). How K is cut depends on the layer's sizes alone, and
// the parts are added in one order: a token's result depends on no order of arrival and on no other token. (Gate and up products in parts, added by
// the warp that finished the last one, made the SMs more even and were slower, 145 us against 114 for 64 tokens of the 24-layer mixture when it was tried: fences and
// counters take microseconds in a loaded memory system.)
//
// Weight rows are the 128-row operand of tcgen05 products, all tokens the other one, whichever experts they chose: columns that are not an expert's are computed
// and not looked at, which costs nothing that counts (128 x 64 x 64 takes 200 cycles, its 16 KB of weights 700 from memory). Down products take an
// expert's own activations, which lie one behind the other. Weights in 8 bits become bf16 on their way from shared to tensor memory, exactly; their scales are
// applied to the sums.
#include "gemm_common.cuh"
#include "once_per_device.h"

namespace inv {

constexpr int MF_TOKENS = 64, MF_EXPERTS = 256, MF_TOP = 16;
constexpr int MF_STEPS = 12;                       // of 128 bytes of K, of a down item at most
constexpr int MF_F = 64, MF_D = 128, MF_GROUP = 4; // columns of a gate and up item, of a down item; tokens of a sum

// What the entry is given; sizes in elements.
struct MoeFewCall {
  const __nv_bfloat16 *x, *router, *residual;      // [T, D] ldx apart; [E, D]; [T, D] ldr apart or null
  const void *gate_up, *down;                      // [E, 2F, D], [E, D, F], bf16 or int8
  const float *gate_up_scale, *down_scale;         // [E, 2F], [E, D], int8 only
  const void *shared_gate_up, *shared_down;        // [2F, D], [D, F], or null
  const float *shared_gate_up_scale, *shared_down_scale;
  __nv_bfloat16* out;                              // [T, D]
  int* counts;                                     // [E]
  void* work;
  int* status;
  void* stream;
  int64_t T, D, F, E, top_k, ldx, ldr, i8, work_bytes;
};

// How the work is cut, and where things stand in the workspace, in bytes.
struct MoeFewPlan {
  int slots, ld_act, f_tiles, d_tiles, experts, n_counters;
  int gate_steps, down_steps, down_per, down_parts;    // of K: in all, of a part, parts
  int tb, slices;                                      // tokens of a product's operand; slices of D in the router
  long choice, weight, counters, act, sums, bytes, items;
  MoeFewPlan(long T, long D, long F, long E, long top_k, bool shared, bool i8) {
    auto up = [](long v) { return (v + 255) / 256 * 256; };
    const int step = i8 ? 128 : 64;
    gate_steps = (int)((D + step - 1) / step);
    down_steps = (int)((F + step - 1) / step);
    down_parts = (down_steps + MF_STEPS - 1) / MF_STEPS;
    down_per = (down_steps + down_parts - 1) / down_parts;      // equal parts, but for the last
    down_parts = (down_steps + down_per - 1) / down_per;
    slots = (int)(T * top_k + (shared ? T : 0));
    experts = (int)((T * top_k < E ? T * top_k : E) + (shared ? 1 : 0));       // that are met, at most
    ld_act = (int)((F + 63) / 64 * 64);
    f_tiles = (int)((F + MF_F - 1) / MF_F);
    d_tiles = (int)((D + MF_D - 1) / MF_D);
    n_counters = 1 + experts + d_tiles;
    choice = 0;
    weight = up(choice + T * top_k * 4);
    counters = up(weight + T * top_k * 4);
    act = up(counters + n_counters * 4L);
    sums = up(act + (long)slots * ld_act * 2);
    bytes = up(sums + (long)down_parts * slots * D * 4);
    items = (long)experts * (f_tiles + d_tiles * down_parts) + d_tiles * ((T + MF_GROUP - 1) / MF_GROUP);
    tb = T <= 16 ? 16 : T <= 32 ? 32 : 64;
    slices = D >= 2048 ? 8 : D >= 1024 ? 4 : D >= 512 ? 2 : 1;
  }
};

// ---------------------------------------------------------------------------------------------- router
// 32 warps: slices of D times groups of experts, so that every load of a usual router is on its way at once.
__global__ void __launch_bounds__(1024) moe_few_router_kernel(const __nv_bfloat16* __restrict__ x, long ldx, const __nv_bfloat16* __restrict__ router, int D, int E,
                                                              int top_k, int slices, int* __restrict__ choice, float* __restrict__ weight,
                                                              int* __restrict__ counters, int n_counters) {
  constexpr int SLICES = 8, AT_ONCE = 8;
  __shared__ float part[SLICES][MF_EXPERTS], logit[MF_EXPERTS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t = blockIdx.x, slice = warp & (slices - 1), groups = 32 / slices;
  release_next();
  for (int i = t * 1024 + tid; i < n_counters; i += gridDim.x * 1024) counters[i] = 0;
  const uint4* row = reinterpret_cast<const uint4*>(x + (long)t * ldx);
  const int vecs = D / 8;
  // experts warp / slices, and every groups-th behind it
  for (int e0 = warp / slices; e0 < E; e0 += groups * AT_ONCE) {
    float s[AT_ONCE] = {};
    for (int i = slice * 32 + lane; i < vecs; i += slices * 32) {
      const uint4 a = row[i];
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
      uint4 b[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
        if (e0 + j * groups < E) b[j] = reinterpret_cast<const uint4*>(router + (long)(e0 + j * groups) * D)[i];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        if (e0 + j * groups >= E) break;
        const uint32_t bw[4] = {b[j].x, b[j].y, b[j].z, b[j].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          s[j] = fmaf(__uint_as_float(aw[q] << 16), __uint_as_float(bw[q] << 16), s[j]);
          s[j] = fmaf(__uint_as_float(aw[q] & 0xffff0000u), __uint_as_float(bw[q] & 0xffff0000u), s[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (e0 + j * groups >= E) break;
#pragma unroll
      for (int o = 16; o; o >>= 1) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
      if (lane == 0) part[slice][e0 + j * groups] = s[j];
    }
  }
  __syncthreads();
  if (tid < E) {
    float s = 0.f;
    for (int i = 0; i < slices; ++i) s += part[i][tid];
    logit[tid] = s;
  }
  __syncthreads();
  if (warp) return;
  constexpr int PER = MF_EXPERTS / 32;
  const int per = (E + 31) / 32;
  float p[PER], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j >= per) break;
    p[j] = j * 32 + lane < E ? logit[j * 32 + lane] : -INFINITY;
    top = fmaxf(top, p[j]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j >= per) break;
    p[j] = j * 32 + lane < E ? expf(p[j] - top) : 0.f;
    sum += p[j];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  // The largest first, ties to the lowest expert: the bits of numbers that are not negative are ordered as they are, with NaN above all, and one more than them is
  // above the 0 of what was taken. Every choice is another expert, whatever the probabilities hold.
  uint32_t key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j >= per) break;
    key[j] = j * 32 + lane < E ? (__float_as_uint(p[j] / sum) & 0x7fffffffu) + 1u : 0u;
  }
  for (int k = 0; k < top_k; ++k) {
    uint32_t best = 0;
    int e = MF_EXPERTS;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j >= per) break;
      if (key[j] > best) { best = key[j]; e = j * 32 + lane; }
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, best);
    e = __reduce_min_sync(0xffffffffu, best == most ? e : MF_EXPERTS);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j >= per) break;
      if (e == j * 32 + lane) key[j] = 0u;
    }
    if (lane == 0) {
      choice[t * top_k + k] = e;
      weight[t * top_k + k] = __uint_as_float(most - 1u);
    }
  }
}

// ---------------------------------------------------------------------------------------------- products
struct MoeFew {
  const __nv_bfloat16* residual;
  const float *gate_up_scale, *down_scale, *shared_gate_up_scale, *shared_down_scale;
  __nv_bfloat16* out;
  int *counts, *counters, *status;
  const int* choice;
  const float* weight;
  __nv_bfloat16* act;              // [slots, ld_act]
  float* sums;                     // [down_parts, slots, D]
  long ldr;
  int T, D, F, E, top_k, shared, ld_act, slots, f_tiles, d_tiles, experts;
  int gate_steps, down_steps, down_per, down_parts;
  uint32_t inv_k, inv_f, inv_down, inv_down_parts, inv_d;   // div_reciprocal
};

namespace mf {
constexpr int A_STAGE = 128 * 128, QUEUE = 2;
// Bytes of a weight row's step are 128: 64 or 128 values of K.
template <int TB, bool I8>
struct Shape {
  static constexpr int STEP = I8 ? 128 : 64, B_STAGE = (I8 ? 2 : 1) * TB * 128;
  static constexpr int PER_SM = I8 ? 1 : 2, ROOM = ((I8 ? 216 : 102) * 1024 - 1024) / (A_STAGE + B_STAGE), STAGES = ROOM < 12 ? ROOM : 12;
  static constexpr int ACC = 4, CONV = 4, SETS = I8 ? 2 : 1, SUM_AHEAD = I8 ? 2 : 4;   // buffers of sums and of converted weights; sets of four warps of sums
  // warps of weights, of products, of items, of tokens, of sums, of conversions
  static constexpr int SUMS = 4, CONVERT = SUMS + 4 * SETS, THREADS = 32 * (CONVERT + (I8 ? 4 * CONV : 0));
  static constexpr int SMEM = STAGES * (A_STAGE + B_STAGE) + 1024;
  static constexpr int COLS = ACC * TB + (I8 ? CONV * 64 : 0), TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static int grid(long items) { return (int)(items < 148 * PER_SM ? items : 148 * PER_SM); }
};
enum Kind { GATE, DOWN, SUM, END };
struct __align__(16) Item {
  int kind, a, tile, part;         // a: which of the experts that are met; SUM: part: the group of tokens
  int e, first, k0, steps;         // e: the expert, E for the shared one; its first slot; steps of K
};
}  // namespace mf

// Four codes into bf16, in two ways; neither rounds anything. Selections and logic have half the rate of products: the first way is mostly those, the second mostly products,
// and half the codes go each way (16 tokens of 8 experts of 2048 x 5632: 63.4 us; all the first way 66.5, all the second 64.5).
// 128 + (the lower seven bits), less 128, or 256 where the sign bit is set.
__device__ __forceinline__ void mf_widen_logic(uint32_t v, uint32_t& lo, uint32_t& hi) {
  const uint32_t m = v & 0x7f7f7f7fu, s = v & 0x80808080u, c = 0x43434343u;
  const uint32_t m0 = __byte_perm(m, c, 0x4140), m1 = __byte_perm(m, c, 0x4342), s0 = __byte_perm(s, c, 0x4140), s1 = __byte_perm(s, c, 0x4342);
  const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m0), *reinterpret_cast<const __nv_bfloat162*>(&s0));
  const __nv_bfloat162 b = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m1), *reinterpret_cast<const __nv_bfloat162*>(&s1));
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}
// With the sign bit flipped, u = code + 128, the pattern 0x4300 | u is p = 256 + code (code < 0) or 256 + 2 code: code = t - max(t / 2, 0), t = p - 256.
__device__ __forceinline__ uint32_t mf_widen_2(uint32_t p) {
  const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&p);
  const __nv_bfloat162 r = __hfma2_relu(v, __float2bfloat162_rn(0.5f), __float2bfloat162_rn(-128.f));
  const __nv_bfloat162 w = __hsub2(__hadd2(v, __float2bfloat162_rn(-256.f)), r);
  return *reinterpret_cast<const uint32_t*>(&w);
}
__device__ __forceinline__ void mf_widen_products(uint32_t v, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = v ^ 0x80808080u, c = 0x43434343u;
  lo = mf_widen_2(__byte_perm(u, c, 0x4140));
  hi = mf_widen_2(__byte_perm(u, c, 0x4342));
}
__device__ __forceinline__ void tmem_ld_32x1(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
}
__device__ __forceinline__ int mf_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void mf_release(int* p) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(p) : "memory");
}
__device__ __forceinline__ void mf_fence_proxy() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
// Until *p reaches n. False where the limit runs out.
__device__ __forceinline__ bool mf_wait(const int* p, int n, volatile int* abort_flag, int* status) {
  uint64_t t0 = 0;
  for (uint32_t spins = 1; mf_acquire(p) < n; ++spins) {
    if (spins & 0xff) continue;
    if (*abort_flag) return false;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    else if (now - t0 > INV_WAIT_LIMIT_NS) {
      *abort_flag = 1;
      atomicCAS(status, 0, (int)ERR_WAIT_MISC);
      return false;
    }
  }
  return true;
}

template <int TB, bool I8>
__global__ void __launch_bounds__(mf::Shape<TB, I8>::THREADS, mf::Shape<TB, I8>::PER_SM)
    moe_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_act, const __grid_constant__ CUtensorMap map_gate,
                   const __grid_constant__ CUtensorMap map_down, const __grid_constant__ CUtensorMap map_shared_gate,
                   const __grid_constant__ CUtensorMap map_shared_down, const __grid_constant__ MoeFew p) {
  using namespace mf;
  using S = Shape<TB, I8>;
  constexpr int STAGES = S::STAGES, B_STAGE = S::B_STAGE, STEP = S::STEP, ACC = S::ACC, CONV = S::CONV;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[STAGES], weights_bar[STAGES], empty_bar[STAGES], item_full[QUEUE], item_empty[QUEUE], acc_full[ACC], acc_empty[ACC], conv_full[CONV], conv_empty[CONV], taken;
  __shared__ uint32_t s_mask[MF_EXPERTS + 1][2];                 // tokens of an expert; E: of the shared one
  __shared__ uint16_t s_index[MF_EXPERTS], s_expert[MF_EXPERTS + 1], s_first[MF_EXPERTS + 2], s_slot[MF_TOKENS * MF_TOP];
  __shared__ Item s_item[QUEUE];
  __shared__ float s_weight[MF_TOKENS * MF_TOP];
  __shared__ uint8_t s_token[MF_TOKENS * (MF_TOP + 1)];          // of a slot
  __shared__ int s_n;
  __shared__ uint32_t tmem_slot;
  __shared__ int s_abort;
  volatile int* abort_flag = &s_abort;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_STAGE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, chosen = p.T * p.top_k;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full_bar[i], I8 ? 1 : 2);       // tokens, and weights where nothing converts them
      mbar_init(&weights_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < QUEUE; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 3 + 4 * S::SETS + (I8 ? 4 * CONV : 0));
    }
    for (int i = 0; i < ACC; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    for (int i = 0; i < CONV; ++i) {
      mbar_init(&conv_full[i], 4);
      mbar_init(&conv_empty[i], 1);
    }
    mbar_init(&taken, 1);
    s_abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_gate);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, S::TMEM);
    tmem_relinquish();
  }
  for (int i = tid; i < 2 * (MF_EXPERTS + 1); i += S::THREADS) (&s_mask[0][0])[i] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  release_next();                                  // with tensor memory in hand: a kernel that starts early and takes some waits for this one's end
  wait_previous();
  int ticket = 0;
  if (warp == 2 && lane == 0) ticket = atomicAdd(p.counters, 1);

  // Who goes where: the tokens of each expert, the experts that are met, and a slot for each choice, in the order of experts and of tokens within one.
  for (int i = tid; i < chosen; i += S::THREADS) {
    const int t = div_by(i, p.top_k, p.inv_k), e = p.choice[i];
    s_slot[i] = (uint16_t)e;
    s_weight[i] = p.weight[i];
    atomicOr(&s_mask[e][t >> 5], 1u << (t & 31));
  }
  if (p.shared && tid == 0) {
    s_mask[p.E][0] = p.T >= 32 ? 0xffffffffu : (1u << p.T) - 1;
    s_mask[p.E][1] = p.T >= 64 ? 0xffffffffu : p.T > 32 ? (1u << (p.T - 32)) - 1 : 0u;
  }
  __syncthreads();
  if (warp * 32 < p.E) {                           // a warp for 32 experts, which counts those before them as well
    int first = 0, active = 0;
    for (int e = lane; e < warp * 32; e += 32) {
      const int n = __popc(s_mask[e][0]) + __popc(s_mask[e][1]);
      first += __reduce_add_sync(0xffffffffu, n);
      active += __popc(__ballot_sync(0xffffffffu, n > 0));
    }
    const int e = warp * 32 + lane, n = e < p.E ? __popc(s_mask[e][0]) + __popc(s_mask[e][1]) : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t has = __ballot_sync(0xffffffffu, n > 0);
    const int a = active + __popc(has & ((1u << lane) - 1));
    if (n > 0) {
      s_expert[a] = (uint16_t)e;
      s_first[a] = (uint16_t)(first + sum - n);
    }
    if (e < p.E) {
      s_index[e] = (uint16_t)a;
      if (blockIdx.x == 0) p.counts[e] = n;
    }
    if (e == p.E - 1) {                            // behind them, the shared expert
      const int all = active + __popc(has);
      s_first[all] = (uint16_t)chosen;
      if (p.shared) {
        s_expert[all] = (uint16_t)p.E;
        s_first[all + 1] = (uint16_t)(chosen + p.T);
      }
      s_n = all + p.shared;
    }
  }
  __syncthreads();

  const int n_active = s_n, per_down = p.d_tiles * p.down_parts, n_gate = n_active * p.f_tiles, n_down = n_gate + n_active * per_down, n_items = n_down + p.d_tiles * ((p.T + MF_GROUP - 1) / MF_GROUP);
  int* done = p.counters + 1;                      // [experts] warps that have written activations
  int* down_done = done + p.experts;               // [d_tiles] warps that have written sums

  if (warp == 2) {
    // ---------------- items: drawn and described for the others ----------------
    if (lane == 0) {
      int qi = 0;
      uint32_t qph = 1, tph = 0;
      while (true) {
        Item it;
        int i = ticket;
        it.a = it.e = it.first = it.k0 = it.steps = 0;
        if (i < n_gate) {
          it.kind = GATE;
          it.a = div_by(i, p.f_tiles, p.inv_f);
          it.tile = i - it.a * p.f_tiles;
          it.part = 0;
          it.steps = p.gate_steps;
        } else if (i < n_down) {
          it.kind = DOWN;
          i -= n_gate;
          it.a = div_by(i, per_down, p.inv_down);
          i -= it.a * per_down;
          it.tile = div_by(i, p.down_parts, p.inv_down_parts);
          it.part = i - it.tile * p.down_parts;
          it.k0 = it.part * p.down_per;
          it.steps = min(p.down_per, p.down_steps - it.k0);
        } else {
          it.kind = i < n_items ? SUM : END;
          i -= n_down;
          it.part = div_by(i, p.d_tiles, p.inv_d);
          it.tile = i - it.part * p.d_tiles;
        }
        if (it.kind <= DOWN) {
          it.e = s_expert[it.a];
          it.first = s_first[it.a];
        }
        if (!mbar_wait(&item_empty[qi], qph, abort_flag, p.status, ERR_WAIT_MISC)) break;
        s_item[qi] = it;
        mbar_arrive(&item_full[qi]);
        if (++qi == QUEUE) { qi = 0; qph ^= 1; }
        if (it.kind == END || !mbar_wait(&taken, tph, abort_flag, p.status, ERR_WAIT_MISC)) break;
        tph ^= 1;
        ticket = atomicAdd(p.counters, 1);
      }
    }
  } else if (warp == 0) {
    // ---------------- weights: as far ahead as there is room ----------------
    if (elect_one_sync()) {
      int s = 0, qi = 0;
      uint32_t ph = 1, qph = 0;
      bool ok = true;
      while (ok) {
        if (!mbar_wait(&item_full[qi], qph, abort_flag, p.status, ERR_WAIT_MISC)) break;
        const Item it = s_item[qi];
        mbar_arrive(&item_empty[qi]);
        mbar_arrive(&taken);
        if (++qi == QUEUE) { qi = 0; qph ^= 1; }
        if (it.kind == END) break;
        if (it.kind == SUM) continue;
        const bool shared = it.e == p.E;
        const int plane = shared ? 0 : it.e, end = (it.k0 + it.steps) * STEP;
        const CUtensorMap* map = it.kind == GATE ? (shared ? &map_shared_gate : &map_gate) : (shared ? &map_shared_down : &map_down);
        for (int k = it.k0 * STEP; k < end; k += STEP) {
          if (!mbar_wait(&empty_bar[s], ph, abort_flag, p.status, ERR_WAIT_EMPTY)) { ok = false; break; }
          uint64_t* bar = I8 ? &weights_bar[s] : &full_bar[s];
          mbar_expect_tx(bar, A_STAGE);
          if (it.kind == GATE) tma_load_5d(sA + s * A_STAGE, map, bar, k, 0, 0, it.tile * (MF_F / 8), plane);
          else tma_load_3d(sA + s * A_STAGE, map, bar, k, it.tile * MF_D, plane);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 3) {
    // ---------------- tokens ----------------
    if (elect_one_sync()) {
      int s = 0, qi = 0, ready = -1;               // experts up to `ready` have their activations
      uint32_t ph = 1, qph = 0;
      bool ok = true;
      while (ok) {
        if (!mbar_wait(&item_full[qi], qph, abort_flag, p.status, ERR_WAIT_MISC)) break;
        const Item it = s_item[qi];
        mbar_arrive(&item_empty[qi]);
        if (++qi == QUEUE) { qi = 0; qph ^= 1; }
        if (it.kind == END) break;
        if (it.kind == SUM) continue;
        if (it.kind == DOWN && it.a > ready) {
          if (!mf_wait(&done[it.a], p.f_tiles * 4, abort_flag, p.status)) break;
          mf_fence_proxy();                          // activations were written by plain stores and are read by bulk copies
          ready = it.a;
        }
        const int row = it.kind == GATE ? 0 : it.first, end = (it.k0 + it.steps) * STEP;
        const CUtensorMap* map = it.kind == GATE ? &map_x : &map_act;
        for (int k = it.k0 * STEP; k < end; k += STEP) {
          if (!mbar_wait(&empty_bar[s], ph, abort_flag, p.status, ERR_WAIT_EMPTY)) { ok = false; break; }
          mbar_expect_tx(&full_bar[s], B_STAGE);
#pragma unroll
          for (int h = 0; h < (I8 ? 2 : 1); ++h) tma_load_2d(sB + s * B_STAGE + h * TB * 128, map, &full_bar[s], k + 64 * h, row);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- products ----------------
    if (elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_bf16(128, TB, 0, 0);
      const uint64_t da0 = make_smem_desc(smem_u32(sA), 16, 1024, 2), db0 = make_smem_desc(smem_u32(sB), 16, 1024, 2);
      int s = 0, qi = 0, acc = 0, cv = 0;
      uint32_t ph = 0, qph = 0, accph = 1, cvph = 0;
      bool ok = true;
      while (ok) {
        if (!mbar_wait(&item_full[qi], qph, abort_flag, p.status, ERR_WAIT_MISC)) break;
        const int kind = s_item[qi].kind, steps = s_item[qi].steps;
        mbar_arrive(&item_empty[qi]);
        if (++qi == QUEUE) { qi = 0; qph ^= 1; }
        if (kind == END) break;
        if (kind == SUM) continue;
        if (!mbar_wait(&acc_empty[acc], accph, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * TB;
        for (int j = 0; j < steps; ++j) {
          if (!mbar_wait(&full_bar[s], ph, abort_flag, p.status, ERR_WAIT_FULL)) { ok = false; break; }
          if (I8 && !mbar_wait(&conv_full[cv], cvph, abort_flag, p.status, ERR_WAIT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint64_t db = db0 + (uint64_t)(s * (B_STAGE >> 4));
          if constexpr (I8) {
            const uint32_t a = tmem_base + ACC * TB + cv * 64;
#pragma unroll
            for (int k = 0; k < 8; ++k) umma_bf16_tmem_a(d, a + k * 8, db + (k & 3) * 2 + (k >> 2) * (TB * 128 >> 4), idesc, j > 0 || k > 0 ? 1u : 0u);
            umma_commit(&conv_empty[cv]);
            if (++cv == CONV) { cv = 0; cvph ^= 1; }
          } else {
            const uint64_t da = da0 + (uint64_t)(s * (A_STAGE >> 4));
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16(d, da + k * 2, db + k * 2, idesc, j > 0 || k > 0 ? 1u : 0u);
          }
          umma_commit(&empty_bar[s]);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        umma_commit(&acc_full[acc]);
        if (++acc == ACC) { acc = 0; accph ^= 1; }
      }
    }
  } else if (warp < S::CONVERT) {
    // ---------------- sums: sets of four warps take items in turn ----------------
    const int q = warp & 3, row = q * 32 + lane;           // the lanes of tensor memory that this warp may read
    const int set = (warp - S::SUMS) >> 2;
    for (int i = tid - S::SUMS * 32; i < chosen; i += 128 * S::SETS) {
      const int t = div_by(i, p.top_k, p.inv_k), e = s_slot[i];
      const int below = t < 32 ? __popc(s_mask[e][0] & ((1u << t) - 1)) : __popc(s_mask[e][0]) + __popc(s_mask[e][1] & ((1u << (t - 32)) - 1));
      const int slot = s_first[s_index[e]] + below;
      s_slot[i] = (uint16_t)slot;
      s_token[slot] = (uint8_t)t;
    }
    if (p.shared && tid - S::SUMS * 32 < p.T) s_token[chosen + tid - S::SUMS * 32] = (uint8_t)(tid - S::SUMS * 32);
    asm volatile("bar.sync 1, %0;" ::"r"(128 * S::SETS) : "memory");
    int qi = 0, turn = 0, next_acc = 0;
    uint32_t qph = 0, next_accph = 0;
    while (true) {
      if (!mbar_wait_warp(&item_full[qi], qph, abort_flag, p.status, ERR_WAIT_MISC)) break;
      const Item it = s_item[qi];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[qi]);
      if (++qi == QUEUE) { qi = 0; qph ^= 1; }
      if (it.kind == END) break;
      const bool mine = turn == set;
      if (++turn == S::SETS) turn = 0;
      const int acc = next_acc;
      const uint32_t accph = next_accph;
      if (it.kind != SUM && ++next_acc == ACC) { next_acc = 0; next_accph ^= 1; }
      if (!mine) continue;
      if (it.kind == SUM) {
        // eight lanes of a warp have 32 columns between them and add every fourth of a token's parts; the four groups of lanes add up theirs
        const int col = it.tile * MF_D + q * 32 + (lane & 7) * 4, t0 = it.part * MF_GROUP, mine_t = t0 + (lane >> 3);
        uint2 residual = make_uint2(0, 0);
        if (p.residual != nullptr && mine_t < p.T && col < p.D) residual = *reinterpret_cast<const uint2*>(p.residual + mine_t * p.ldr + col);
        bool there = true;
        if (lane == 0) there = mf_wait(&down_done[it.tile], n_active * p.down_parts * 4, abort_flag, p.status);
        if (!__shfl_sync(0xffffffffu, there, 0)) break;
        __syncwarp();                              // what lane 0 acquired is the other lanes' too; a shuffle orders no memory
        float y[MF_GROUP][4] = {};
        if (col < p.D) {
          const int terms = (p.top_k + p.shared) * p.down_parts;
#pragma unroll S::SUM_AHEAD
          for (int i = lane >> 3; i < terms; i += 4) {
            const int k = div_by(i, p.down_parts, p.inv_down_parts), part = i - k * p.down_parts;
#pragma unroll
            for (int j = 0; j < MF_GROUP; ++j) {
              const int t = min(t0 + j, p.T - 1), c = t * p.top_k + k;
              const float w = k == p.top_k ? 1.f : s_weight[c];
              const float4 u = __ldcg(reinterpret_cast<const float4*>(p.sums + ((long)part * p.slots + (k == p.top_k ? chosen + t : s_slot[c])) * p.D + col));
              y[j][0] = fmaf(w, u.x, y[j][0]); y[j][1] = fmaf(w, u.y, y[j][1]); y[j][2] = fmaf(w, u.z, y[j][2]); y[j][3] = fmaf(w, u.w, y[j][3]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < MF_GROUP; ++j) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            y[j][x] += __shfl_xor_sync(0xffffffffu, y[j][x], 8);
            y[j][x] += __shfl_xor_sync(0xffffffffu, y[j][x], 16);
          }
          if (lane >> 3 == j && mine_t < p.T && col < p.D) {
            y[j][0] += __uint_as_float(residual.x << 16); y[j][1] += __uint_as_float(residual.x & 0xffff0000u);
            y[j][2] += __uint_as_float(residual.y << 16); y[j][3] += __uint_as_float(residual.y & 0xffff0000u);
            *reinterpret_cast<uint2*>(p.out + (long)mine_t * p.D + col) = make_uint2(pack_bf16x2(y[j][0], y[j][1]), pack_bf16x2(y[j][2], y[j][3]));
          }
        }
        continue;
      }
      const int e = it.e, first = it.first, n = s_first[it.a + 1] - first;
      const bool shared = e == p.E;
      // gate and up items: lanes of a warp hold eight columns of the gate, the same of the up product, and the next eight likewise
      const int f = it.tile * MF_F + q * 16 + (lane >> 4) * 8 + (lane & 7), col = it.tile * MF_D + row;
      float scale = 1.f;
      if (I8) {
        if (it.kind == GATE) scale = f < p.F ? (shared ? p.shared_gate_up_scale : p.gate_up_scale + (long)e * 2 * p.F)[f + (lane >> 3 & 1) * p.F] : 0.f;
        else scale = col < p.D ? (shared ? p.shared_down_scale : p.down_scale + (long)e * p.D)[col] : 0.f;
      }
      if (!mbar_wait_warp(&acc_full[acc], accph, abort_flag, p.status, ERR_WAIT_TMEM_FULL)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + acc * TB + (uint32_t(q * 32) << 16);
      if (it.kind == GATE) {
        // Two tokens at a time: lanes with the gate take the first of them, those with the up product the second.
        const bool second = lane & 8;
#pragma unroll 1
        for (int c = 0; c < n; c += 4) {
          uint32_t r[4];
          __syncwarp();                            // the stores below part the lanes, the loads want the whole warp
#pragma unroll
          for (int j = 0; j < 4; ++j) tmem_ld_32x1(taddr + s_token[first + min(c + j, n - 1)], r[j]);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const float u = __uint_as_float(r[j]) * scale, v = __uint_as_float(r[j + 1]) * scale, other = __shfl_xor_sync(0xffffffffu, second ? u : v, 8);
            const float g = second ? other : u, up = second ? v : other;
            const int slot = c + j + second;
            // rounded to bf16, the type of the next product's operands
            if (slot < n && f < p.F) p.act[(long)(first + slot) * p.ld_act + f] = __float2bfloat16_rn(g / (1.f + expf(-g)) * up);
          }
        }
      } else {
        float* to = p.sums + ((long)it.part * p.slots + first) * p.D + col;
#pragma unroll 1
        for (int c = 0; c < n; c += 16) {
          uint32_t r[16];
          tmem_ld_32x16(taddr + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < n && col < p.D) to[(long)(c + j) * p.D] = __uint_as_float(r[j]) * scale;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      __syncwarp();
      if (lane == 0) mf_release(it.kind == GATE ? &done[it.a] : &down_done[it.tile]);
    }
  } else if constexpr (I8) {
    // ---------------- conversions: groups of four warps take steps in turn, one buffer each ----------------
    const int q = warp & 3, row = q * 32 + lane, group = (warp - S::CONVERT) >> 2;
    int s = 0, qi = 0, cv = 0;
    uint32_t ph = 0, qph = 0, cvph = 1;
    bool ok = true;
    while (ok) {
      if (!mbar_wait_warp(&item_full[qi], qph, abort_flag, p.status, ERR_WAIT_MISC)) break;
      const int kind = s_item[qi].kind, steps = s_item[qi].steps;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[qi]);
      if (++qi == QUEUE) { qi = 0; qph ^= 1; }
      if (kind == END) break;
      if (kind == SUM) continue;
      for (int j = 0; j < steps; ++j) {
        if (cv == group) {
          if (!mbar_wait_warp(&weights_bar[s], ph, abort_flag, p.status, ERR_WAIT_FULL) ||
              !mbar_wait_warp(&conv_empty[cv], cvph, abort_flag, p.status, ERR_WAIT_EMPTY)) { ok = false; break; }
          tc_fence_after();
          const uint8_t* from = sA + s * A_STAGE + row * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint4 v = *reinterpret_cast<const uint4*>(from + (((4 * h + c) ^ (row & 7)) << 4));
              mf_widen_logic(v.x, w[8 * c], w[8 * c + 1]);
              mf_widen_products(v.y, w[8 * c + 2], w[8 * c + 3]);
              mf_widen_logic(v.z, w[8 * c + 4], w[8 * c + 5]);
              mf_widen_products(v.w, w[8 * c + 6], w[8 * c + 7]);
            }
            tmem_st_32x32(tmem_base + ACC * TB + cv * 64 + h * 32 + (uint32_t(q * 32) << 16), w);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&conv_full[cv]);
        }
        if (++s == STAGES) { s = 0; ph ^= 1; }
        if (++cv == CONV) { cv = 0; cvph ^= 1; }
      }
    }
  }

  __syncwarp();
  __syncthreads();
  if (s_abort) {                                           // let what is under way end before the memory it uses is given up
    const uint64_t since = globaltimer_ns();
    while (globaltimer_ns() - since < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::TMEM);
  }
}

struct MoeFewMaps {
  CUtensorMap x, act, gate, down, shared_gate, shared_down;
};

template <int TB, bool I8>
static int launch_moe_few(const MoeFewMaps& m, const MoeFew& p, long items, int device, cudaStream_t st) {
  using S = mf::Shape<TB, I8>;
  static OncePerDevice once;
  if (const int e = once.ask(device, [] { return (int)cudaFuncSetAttribute(moe_few_kernel<TB, I8>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); })) return -e;
  launch_early(moe_few_kernel<TB, I8>, dim3(S::grid(items)), S::THREADS, S::SMEM, st, m.x, m.act, m.gate, m.down, m.shared_gate, m.shared_down, p);
  return -(int)cudaGetLastError();
}

}  // namespace inv

using namespace inv;

extern "C" long inv_moe_few_bytes(long T, long D, long F, long E, long top_k, int shared, int i8) {
  return MoeFewPlan(T, D, F, E, top_k, shared != 0, i8 != 0).bytes;
}

template <int TB, bool I8>
static int* moe_few_shape(const MoeFewPlan& n, int* out) {
  using S = mf::Shape<TB, I8>;
  for (const int v : {S::grid(n.items), S::THREADS, S::SMEM, S::PER_SM, S::STAGES, S::STEP, S::COLS, S::TMEM}) *out++ = v;
  return out;
}
// The plan's numbers in their order, and those of the launch, for who wants to look at them.
extern "C" int inv_moe_few_plan(long T, long D, long F, long E, long top_k, int shared, int i8, int* out, long* places) {
  if (T < 1 || T > MF_TOKENS || D < 1 || F < 1 || E < 1 || E > MF_EXPERTS || top_k < 1 || top_k > MF_TOP || top_k > E) return -ERR_BAD_ARG;
  const MoeFewPlan n(T, D, F, E, top_k, shared != 0, i8 != 0);
  for (const int v : {n.slots, n.ld_act, n.f_tiles, n.d_tiles, n.experts, n.n_counters, n.gate_steps, n.down_steps, n.down_per, n.down_parts, n.tb, n.slices}) *out++ = v;
  for (const long v : {n.choice, n.weight, n.counters, n.act, n.sums, n.bytes, n.items}) *places++ = v;
#define INV_MF(TB) (i8 ? moe_few_shape<TB, true>(n, out) : moe_few_shape<TB, false>(n, out))
  n.tb == 16 ? INV_MF(16) : n.tb == 32 ? INV_MF(32) : INV_MF(64);
#undef INV_MF
  return 0;
}

extern "C" int inv_moe_few(const void* call) {
  const MoeFewCall& c = *static_cast<const MoeFewCall*>(call);
  if (c.T <= 0) return 0;
  const int grain = c.i8 ? 16 : 8;
  const bool shared = c.shared_gate_up != nullptr;
  if (c.T > MF_TOKENS || c.E < 1 || c.E > MF_EXPERTS || c.top_k < 1 || c.top_k > MF_TOP || c.top_k > c.E || c.D < grain || c.F < grain || c.D % grain ||
      c.F % grain || c.D > (1 << 24) || c.F > (1 << 24) || c.ldx % 8 || c.ldr % 4 ||
      (((uintptr_t)c.x | (uintptr_t)c.router | (uintptr_t)c.gate_up | (uintptr_t)c.down | (uintptr_t)c.shared_gate_up | (uintptr_t)c.shared_down |
        (uintptr_t)c.work | (uintptr_t)c.residual | (uintptr_t)c.out) & 15))
    return -ERR_BAD_ARG;
  const MoeFewPlan plan(c.T, c.D, c.F, c.E, c.top_k, shared, c.i8 != 0);
  if (c.work_bytes < plan.bytes || plan.items > (1 << 30)) return -ERR_BAD_ARG;
  cudaStream_t st = (cudaStream_t)c.stream;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device)) return -(int)e;
  char* work = static_cast<char*>(c.work);
  MoeFew p;
  p.residual = c.residual;
  p.gate_up_scale = c.gate_up_scale; p.down_scale = c.down_scale;
  p.shared_gate_up_scale = c.shared_gate_up_scale; p.shared_down_scale = c.shared_down_scale;
  p.out = c.out; p.counts = c.counts; p.counters = (int*)(work + plan.counters); p.status = c.status;
  p.choice = (const int*)(work + plan.choice); p.weight = (const float*)(work + plan.weight);
  p.act = (__nv_bfloat16*)(work + plan.act); p.sums = (float*)(work + plan.sums);
  p.ldr = c.ldr;
  p.T = (int)c.T; p.D = (int)c.D; p.F = (int)c.F; p.E = (int)c.E; p.top_k = (int)c.top_k; p.shared = shared; p.ld_act = plan.ld_act; p.slots = plan.slots;
  p.f_tiles = plan.f_tiles; p.d_tiles = plan.d_tiles; p.gate_steps = plan.gate_steps; p.down_steps = plan.down_steps; p.down_per = plan.down_per; p.down_parts = plan.down_parts; p.experts = plan.experts;
  p.inv_k = div_reciprocal(p.top_k); p.inv_f = div_reciprocal(p.f_tiles);
  p.inv_down = div_reciprocal(p.d_tiles * p.down_parts); p.inv_down_parts = div_reciprocal(p.down_parts); p.inv_d = div_reciprocal(p.d_tiles);
  const int tb = plan.tb;
  const CUtensorMapDataType bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, type = c.i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : bf16;
  const uint64_t D = c.D, F = c.F, E = c.E, size = c.i8 ? 1 : 2, row = D * size;
  const uint32_t wide = c.i8 ? 128 : 64;
  MoeFewMaps m;
  int rc = make_tmap(&m.x, bf16, 2, c.x, {D, (uint64_t)c.T}, {(uint64_t)c.ldx * 2}, {64, (uint32_t)tb});
  if (rc == 0) rc = make_tmap(&m.act, bf16, 2, p.act, {F, (uint64_t)plan.slots}, {(uint64_t)plan.ld_act * 2}, {64, (uint32_t)tb});
  if (rc == 0) rc = make_tmap(&m.gate, type, 5, c.gate_up, {D, 8, 2, F / 8, E}, {row, F * row, 8 * row, 2 * F * row}, {wide, 8, 2, MF_F / 8, 1});
  if (rc == 0) rc = make_tmap(&m.down, type, 3, c.down, {F, D, E}, {F * size, D * F * size}, {wide, 128, 1});
  m.shared_gate = m.gate;
  m.shared_down = m.down;
  if (rc == 0 && shared) rc = make_tmap(&m.shared_gate, type, 5, c.shared_gate_up, {D, 8, 2, F / 8, 1}, {row, F * row, 8 * row, 2 * F * row}, {wide, 8, 2, MF_F / 8, 1});
  if (rc == 0 && shared) rc = make_tmap(&m.shared_down, type, 3, c.shared_down, {F, D, 1}, {F * size, D * F * size}, {wide, 128, 1});
  if (rc) return rc;
  moe_few_router_kernel<<<(unsigned)p.T, 1024, 0, st>>>(c.x, c.ldx, c.router, p.D, p.E, p.top_k, plan.slices, (int*)p.choice, (float*)p.weight, p.counters, plan.n_counters);
  if (const cudaError_t e = cudaGetLastError()) return -(int)e;
#define INV_MF(TB) (c.i8 ? launch_moe_few<TB, true>(m, p, plan.items, device, st) : launch_moe_few<TB, false>(m, p, plan.items, device, st))
  return tb == 16 ? INV_MF(16) : tb == 32 ? INV_MF(32) : INV_MF(64);
#undef INV_MF
}
