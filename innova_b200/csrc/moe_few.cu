// A whole mixture-of-experts layer for up to 64 tokens, in two launches.
//
//   p = softmax(R x);  y_t = r_t + [shared expert] + sum over the top_k largest p_te of p_te W2_e (silu(W1g_e x_t) * (W1u_e x_t))
//
// Such a layer reads every expert that some token goes to once and does little arithmetic, so weight bytes bound it. The training form (csrc/moe.cu) pads
// every expert to 128 rows and takes seven launches.
//
// moe_few_router_kernel   a CTA a token: logits, softmax, the largest entries; clears the counters of the next kernel
// moe_few_kernel          gate and up products, then down products and their sum, without a launch between them
//
// The second kernel's work is a list of items: 16 columns of one expert's gate and up product, then 32 columns of one expert's down product. CTAs draw items in order
// from a counter. A down item waits until its expert's gate and up items are done; these were all drawn earlier, by CTAs that run and wait for nothing, so every
// wait ends, whatever else runs on the GPU. Down products of an expert go to memory in fp32; the CTA that finishes the last expert's part of 32 output
// columns adds them up in the order of the router's choices: no result depends on an order of arrival.
//
// Weights go from memory straight into the fragments of warp-level products, as the 16-row operand; tokens are the other one, eight at a time. (A tcgen05 tile
// has 128 rows of tokens or weights to fill, of which an item has 32.) Weights in 8 bits become bf16 in registers, exactly; their channel scales are applied to the sums.
#include "once_per_device.h"
#include "sm100_common.cuh"

namespace inv {

constexpr int MF_TOKENS = 64, MF_EXPERTS = 256, MF_TOP = 16;
constexpr int MF_WARPS = 8, MF_SLICE = 128, MF_PL = 36, MF_F = 16, MF_D = 32;

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

// Where things stand in the workspace, in bytes.
struct MoeFewPlan {
  long choice, weight, counters, act, part, bytes;
  int ld_act, n_counters, slots;
  __host__ __device__ MoeFewPlan(long T, long D, long F, long E, long top_k, bool shared) {
    auto up = [](long v) { return (v + 255) / 256 * 256; };
    slots = (int)(T * top_k + (shared ? T : 0));
    ld_act = (int)((F + 63) / 64 * 64);
    n_counters = (int)(1 + E + 1 + (D + MF_D - 1) / MF_D);
    choice = 0;
    weight = up(choice + T * top_k * 4);
    counters = up(weight + T * top_k * 4);
    act = up(counters + n_counters * 4);
    part = up(act + (long)slots * ld_act * 2);
    bytes = up(part + (long)slots * D * 4);
  }
};

// ---------------------------------------------------------------------------------------------- router
__global__ void __launch_bounds__(256) moe_few_router_kernel(const __nv_bfloat16* __restrict__ x, long ldx, const __nv_bfloat16* __restrict__ router, int D, int E,
                                                             int top_k, int* __restrict__ choice, float* __restrict__ weight, int* __restrict__ counters,
                                                             int n_counters) {
  __shared__ float logit[MF_EXPERTS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t = blockIdx.x;
  release_next();
  if (t == 0)
    for (int i = tid; i < n_counters; i += 256) counters[i] = 0;
  const uint4* row = reinterpret_cast<const uint4*>(x + t * ldx);
  const int vecs = D / 8;
  for (int e0 = warp * 4; e0 < E; e0 += 32) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const uint4* r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = reinterpret_cast<const uint4*>(router + (long)min(e0 + j, E - 1) * D);
    for (int i = lane; i < vecs; i += 32) {
      const uint4 a = row[i];
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 b = r[j][i];
        const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          s[j] = fmaf(__uint_as_float(aw[q] << 16), __uint_as_float(bw[q] << 16), s[j]);
          s[j] = fmaf(__uint_as_float(aw[q] & 0xffff0000u), __uint_as_float(bw[q] & 0xffff0000u), s[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int o = 16; o; o >>= 1) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
      if (lane == 0 && e0 + j < E) logit[e0 + j] = s[j];
    }
  }
  __syncthreads();
  if (warp) return;
  constexpr int PER = MF_EXPERTS / 32;
  float p[PER], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    p[j] = j * 32 + lane < E ? logit[j * 32 + lane] : -INFINITY;
    top = fmaxf(top, p[j]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    p[j] = j * 32 + lane < E ? expf(p[j] - top) : 0.f;
    sum += p[j];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  // The largest first, ties to the lowest expert: the bits of numbers that are not negative are ordered as they are, with NaN above all. Every choice is another expert,
  // whatever the probabilities hold.
  uint32_t taken = 0;
  for (int k = 0; k < top_k; ++k) {
    unsigned long long best = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = j * 32 + lane;
      const unsigned long long key = (unsigned long long)((__float_as_uint(p[j] / sum) & 0x7fffffffu) + 1u) << 32 | (uint32_t)(MF_EXPERTS - e);
      if (e < E && !(taken >> j & 1) && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    const int e = MF_EXPERTS - (int)(uint32_t)best;
    if ((e & 31) == lane) taken |= 1u << (e >> 5);
    if (lane == 0) {
      choice[t * top_k + k] = e;
      weight[t * top_k + k] = __uint_as_float((uint32_t)(best >> 32) - 1u);
    }
  }
}

// ---------------------------------------------------------------------------------------------- products
struct MoeFew {
  const __nv_bfloat16 *x, *residual;
  const uint8_t *gate_up, *down, *shared_gate_up, *shared_down;
  const float *gate_up_scale, *down_scale, *shared_gate_up_scale, *shared_down_scale;
  __nv_bfloat16* out;
  int *counts, *counters, *status;
  const int* choice;
  const float* weight;
  __nv_bfloat16* act;              // [slots, ld_act]
  float* part;                     // [slots, D]
  long ldx, ldr;
  int T, D, F, E, top_k, ld_act, f_tiles, d_tiles;
  uint32_t inv_f, inv_d;           // div_reciprocal
};

__device__ __forceinline__ void mf_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 mf_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// Four codes into bf16: 128 + (the lower seven bits), less 128, or 256 where the sign bit is set. Each is a number of eight bits, so nothing is rounded.
__device__ __forceinline__ void mf_widen(uint32_t v, uint32_t& lo, uint32_t& hi) {
  const uint32_t m = v & 0x7f7f7f7fu, s = v & 0x80808080u, c = 0x43434343u;
  const uint32_t m0 = __byte_perm(m, c, 0x4140), m1 = __byte_perm(m, c, 0x4342), s0 = __byte_perm(s, c, 0x4140), s1 = __byte_perm(s, c, 0x4342);
  const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m0), *reinterpret_cast<const __nv_bfloat162*>(&s0));
  const __nv_bfloat162 b = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m1), *reinterpret_cast<const __nv_bfloat162*>(&s1));
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ int mf_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// NT: tokens of an expert, in eights. I8: weights in 8 bits.
template <int NT, bool I8>
__global__ void __launch_bounds__(MF_WARPS * 32, 2) moe_few_kernel(const MoeFew p) {
  constexpr int THREADS = MF_WARPS * 32, UN = NT <= 4 ? 2 : 1, SLOTS = MF_TOKENS * (MF_TOP + 1);
  constexpr int ES = I8 ? 1 : 2;                           // bytes of a weight
  extern __shared__ float mf_part[];                       // [MF_WARPS][8 NT][MF_PL]
  __shared__ int s_first[MF_EXPERTS + 2];                  // first slot of an expert; E: the shared one's
  __shared__ uint16_t s_active[MF_EXPERTS + 1], s_token[SLOTS], s_slot[MF_TOKENS * MF_TOP];
  __shared__ int s_next, s_last, s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
  const int chosen = p.T * p.top_k;
  release_next();
  wait_previous();
  if (tid == 0) s_next = atomicAdd(p.counters, 2);
  // Slots: the choices in the order of their experts, tokens in order within an expert.
  int* s_count = reinterpret_cast<int*>(mf_part);          // before it holds sums
  for (int e = warp; e < p.E; e += MF_WARPS) {
    int n = 0;
    for (int i = 0; i < chosen; i += 32) n += __popc(__ballot_sync(0xffffffffu, i + lane < chosen && p.choice[i + lane] == e));
    if (lane == 0) s_count[e] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int first = 0, active = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int n = e0 + lane < p.E ? s_count[e0 + lane] : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const uint32_t has = __ballot_sync(0xffffffffu, n > 0);
      if (e0 + lane < p.E) {
        s_first[e0 + lane] = first + sum - n;
        if (n > 0) s_active[active + __popc(has & ((1u << lane) - 1))] = (uint16_t)(e0 + lane);
        if (blockIdx.x == 0) p.counts[e0 + lane] = n;
      }
      first += __shfl_sync(0xffffffffu, sum, 31);
      active += __popc(has);
    }
    if (lane == 0) {
      s_first[p.E] = first;
      if (p.shared_gate_up != nullptr) {
        s_active[active++] = (uint16_t)p.E;
        s_first[p.E + 1] = first + p.T;
      }
      s_n = active;
    }
  }
  __syncthreads();
  for (int e = warp; e < p.E; e += MF_WARPS) {
    int at = s_first[e];
    if (s_first[e + 1] == at) continue;
    for (int i = 0; i < chosen; i += 32) {
      const bool mine = i + lane < chosen && p.choice[i + lane] == e;
      const uint32_t has = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        const int slot = at + __popc(has & ((1u << lane) - 1));
        s_slot[i + lane] = (uint16_t)slot;
        s_token[slot] = (uint16_t)((i + lane) / p.top_k);
      }
      at += __popc(has);
    }
  }
  if (p.shared_gate_up != nullptr)
    for (int t = tid; t < p.T; t += THREADS) s_token[chosen + t] = (uint16_t)t;
  __syncthreads();

  const int n_active = s_n, n_gate = n_active * p.f_tiles, n_items = n_gate + n_active * p.d_tiles;
  struct Item {
    int a, tile;
    bool down;
  };
  auto decode = [&](int i) {
    Item it;
    it.down = i >= n_gate;
    const int j = it.down ? i - n_gate : i;
    it.a = it.down ? div_by(j, p.d_tiles, p.inv_d) : div_by(j, p.f_tiles, p.inv_f);
    it.tile = j - it.a * (it.down ? p.d_tiles : p.f_tiles);
    return it;
  };
  auto slices_of = [&](bool down) { return ((down ? p.F : p.D) * ES + MF_SLICE - 1) / MF_SLICE; };
  uint4 ring[UN][4][2];
  auto fetch = [&](const Item& it, int s, uint4 (&r)[4][2]) {
    const int e = s_active[it.a], width = (it.down ? p.F : p.D) * ES, rows = it.down ? p.D : 2 * p.F, at = s * MF_SLICE + tig * 32;
    const uint8_t* from = it.down ? (e == p.E ? p.shared_down : p.down) : (e == p.E ? p.shared_gate_up : p.gate_up);
    from += (long)(e == p.E ? 0 : e) * rows * width + at;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = it.down ? min(it.tile * MF_D + t * 8 + g, p.D - 1) : min(it.tile * MF_F + (t & 1) * 8 + g, p.F - 1) + (t >> 1) * p.F;
#pragma unroll
      for (int i = 0; i < 2; ++i) r[t][i] = at + 16 * i < width ? mf_stream(from + (long)row * width + 16 * i) : make_uint4(0, 0, 0, 0);
    }
  };
  int now = s_next, next = now + 1;
  Item it = decode(now);
  if (now < n_items) {
    const int slices = slices_of(it.down);
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (warp + u * MF_WARPS < slices) fetch(it, warp + u * MF_WARPS, ring[u]);
  }
  while (now < n_items) {
    const Item nx = decode(next);
    const int slices = slices_of(it.down), ahead = next < n_items ? slices_of(nx.down) : 0, width = it.down ? p.F : p.D;
    const int e = s_active[it.a], first = s_first[e], n = s_first[e + 1] - first;
    __syncthreads();                                       // s_next and the sums of the last item have been read
    if (tid == 0) {
      s_next = atomicAdd(p.counters, 1);
      if (it.down) {                                       // the expert's activations: written by CTAs that drew their items before this one
        const int* done = p.counters + 1 + it.a;
        uint64_t t0 = 0;
        for (uint32_t spins = 1; mf_acquire(done) < p.f_tiles; ++spins) {
          if (spins & 0xff) continue;
          const uint64_t clock = globaltimer_ns();
          if (t0 == 0) t0 = clock;
          else if (clock - t0 > INV_WAIT_LIMIT_NS) {
            atomicCAS(p.status, 0, (int)ERR_WAIT_MISC);
            break;
          }
        }
      }
    }
    if (it.down) __syncthreads();
    const __nv_bfloat16* xp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int slot = first + min(j * 8 + g, n - 1);
      xp[j] = (it.down ? p.act + (long)slot * p.ld_act : p.x + (long)s_token[slot] * p.ldx) + tig * 32 / ES;
    }
#pragma unroll
    for (int u = 0; u < UN; ++u)                           // a place that this item has no slice for
      if (warp + u * MF_WARPS >= slices && warp + u * MF_WARPS < ahead) fetch(nx, warp + u * MF_WARPS, ring[u]);
    float acc[NT][2][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[j][i / 4][i % 4] = 0.f;
    for (int s0 = warp; s0 < slices; s0 += UN * MF_WARPS) {
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int s = s0 + u * MF_WARPS;
        if (s >= slices) break;
        const int k0 = s * (MF_SLICE / ES), left = width - k0 - tig * 32 / ES;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (I8) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              uint32_t lo[8], hi[8];
              const uint4 a = ring[u][2 * m][i], b = ring[u][2 * m + 1][i];
              mf_widen(a.x, lo[0], lo[1]); mf_widen(a.y, lo[2], lo[3]); mf_widen(a.z, lo[4], lo[5]); mf_widen(a.w, lo[6], lo[7]);
              mf_widen(b.x, hi[0], hi[1]); mf_widen(b.y, hi[2], hi[3]); mf_widen(b.z, hi[4], hi[5]); mf_widen(b.w, hi[6], hi[7]);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (j && j * 8 >= n) break;
                uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
                if (left > 16 * i) {
                  v0 = *reinterpret_cast<const uint4*>(xp[j] + k0 + 16 * i);
                  v1 = *reinterpret_cast<const uint4*>(xp[j] + k0 + 16 * i + 8);
                }
                mf_mma(acc[j][m], lo[0], hi[0], lo[1], hi[1], v0.x, v0.y);
                mf_mma(acc[j][m], lo[2], hi[2], lo[3], hi[3], v0.z, v0.w);
                mf_mma(acc[j][m], lo[4], hi[4], lo[5], hi[5], v1.x, v1.y);
                mf_mma(acc[j][m], lo[6], hi[6], lo[7], hi[7], v1.z, v1.w);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              if (j && j * 8 >= n) break;
              uint4 v = make_uint4(0, 0, 0, 0);
              if (left > 8 * i) v = *reinterpret_cast<const uint4*>(xp[j] + k0 + 8 * i);
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                const uint4 lo = ring[u][2 * m][i], hi = ring[u][2 * m + 1][i];
                mf_mma(acc[j][m], lo.x, hi.x, lo.y, hi.y, v.x, v.y);
                mf_mma(acc[j][m], lo.z, hi.z, lo.w, hi.w, v.z, v.w);
              }
            }
          }
        }
        const int then = s + UN * MF_WARPS;
        if (then < slices) fetch(it, then, ring[u]);
        else if (warp + u * MF_WARPS < ahead) fetch(nx, warp + u * MF_WARPS, ring[u]);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (j && j * 8 >= n) break;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float* to = mf_part + ((warp * NT + j) * 8 + 2 * tig) * MF_PL + m * 16 + g;
        to[0] = acc[j][m][0];
        to[MF_PL] = acc[j][m][1];
        to[8] = acc[j][m][2];
        to[MF_PL + 8] = acc[j][m][3];
      }
    }
    __syncthreads();
    if (!it.down) {
      for (int i = tid; i < n * MF_F; i += THREADS) {
        const int j = i / MF_F, c = i % MF_F, f = it.tile * MF_F + c;
        if (f >= p.F) continue;
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < MF_WARPS; ++w) {
          a += mf_part[(w * NT * 8 + j) * MF_PL + c];
          b += mf_part[(w * NT * 8 + j) * MF_PL + MF_F + c];
        }
        if (I8) {
          const float* s = e == p.E ? p.shared_gate_up_scale : p.gate_up_scale + (long)e * 2 * p.F;
          a *= s[f];
          b *= s[p.F + f];
        }
        // rounded to bf16, the type of the next product's operands
        p.act[(long)(first + j) * p.ld_act + f] = __float2bfloat16_rn(a / (1.f + expf(-a)) * b);
      }
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        atomicAdd(p.counters + 1 + it.a, 1);
      }
    } else {
      for (int i = tid; i < n * MF_D; i += THREADS) {
        const int j = i / MF_D, c = i % MF_D, col = it.tile * MF_D + c;
        if (col >= p.D) continue;
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < MF_WARPS; ++w) a += mf_part[(w * NT * 8 + j) * MF_PL + c];
        if (I8) a *= (e == p.E ? p.shared_down_scale : p.down_scale + (long)e * p.D)[col];
        p.part[(long)(first + j) * p.D + col] = a;
      }
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(p.counters + 1 + p.E + 1 + it.tile, 1) == n_active - 1;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        for (int i = tid; i < p.T * MF_D; i += THREADS) {
          const int t = i / MF_D, col = it.tile * MF_D + i % MF_D;
          if (col >= p.D) continue;
          float y = p.residual == nullptr ? 0.f : __bfloat162float(p.residual[t * p.ldr + col]);
          if (p.shared_gate_up != nullptr) y += __ldcg(p.part + (long)(chosen + t) * p.D + col);
          for (int k = 0; k < p.top_k; ++k) y = fmaf(p.weight[t * p.top_k + k], __ldcg(p.part + (long)s_slot[t * p.top_k + k] * p.D + col), y);
          p.out[(long)t * p.D + col] = __float2bfloat16_rn(y);
        }
      }
    }
    now = next;
    next = s_next;
    it = nx;
  }
}

template <int NT, bool I8>
static int launch_moe_few(const MoeFew& p, int items, int device, cudaStream_t st) {
  constexpr int bytes = MF_WARPS * NT * 8 * MF_PL * 4;
  static OncePerDevice once;
  if (const int e = once.ask(device, [] { return (int)cudaFuncSetAttribute(moe_few_kernel<NT, I8>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); })) return -e;
  launch_early(moe_few_kernel<NT, I8>, dim3(items < 296 ? items : 296), MF_WARPS * 32, bytes, st, p);
  return -(int)cudaGetLastError();
}

}  // namespace inv

using namespace inv;

extern "C" long inv_moe_few_bytes(long T, long D, long F, long E, long top_k, int shared) { return MoeFewPlan(T, D, F, E, top_k, shared != 0).bytes; }

extern "C" int inv_moe_few(const void* call) {
  const MoeFewCall& c = *static_cast<const MoeFewCall*>(call);
  if (c.T <= 0) return 0;
  const int grain = c.i8 ? 16 : 8;
  const MoeFewPlan plan(c.T, c.D, c.F, c.E, c.top_k, c.shared_gate_up != nullptr);
  if (c.T > MF_TOKENS || c.E < 1 || c.E > MF_EXPERTS || c.top_k < 1 || c.top_k > MF_TOP || c.top_k > c.E || c.D < grain || c.F < grain || c.D % grain || c.F % grain ||
      c.ldx % 8 || c.work_bytes < plan.bytes || c.E * (2 * c.F / MF_F + c.D / MF_D + 4) > (1 << 30) ||
      (((uintptr_t)c.x | (uintptr_t)c.router | (uintptr_t)c.gate_up | (uintptr_t)c.down | (uintptr_t)c.shared_gate_up | (uintptr_t)c.shared_down |
        (uintptr_t)c.work) & 15))
    return -ERR_BAD_ARG;
  cudaStream_t st = (cudaStream_t)c.stream;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device)) return -(int)e;
  char* work = static_cast<char*>(c.work);
  MoeFew p;
  p.x = c.x; p.residual = c.residual;
  p.gate_up = (const uint8_t*)c.gate_up; p.down = (const uint8_t*)c.down;
  p.shared_gate_up = (const uint8_t*)c.shared_gate_up; p.shared_down = (const uint8_t*)c.shared_down;
  p.gate_up_scale = c.gate_up_scale; p.down_scale = c.down_scale;
  p.shared_gate_up_scale = c.shared_gate_up_scale; p.shared_down_scale = c.shared_down_scale;
  p.out = c.out; p.counts = c.counts; p.counters = (int*)(work + plan.counters); p.status = c.status;
  p.choice = (const int*)(work + plan.choice); p.weight = (const float*)(work + plan.weight);
  p.act = (__nv_bfloat16*)(work + plan.act); p.part = (float*)(work + plan.part);
  p.ldx = c.ldx; p.ldr = c.ldr;
  p.T = (int)c.T; p.D = (int)c.D; p.F = (int)c.F; p.E = (int)c.E; p.top_k = (int)c.top_k; p.ld_act = plan.ld_act;
  p.f_tiles = (p.F + MF_F - 1) / MF_F; p.d_tiles = (p.D + MF_D - 1) / MF_D;
  p.inv_f = div_reciprocal(p.f_tiles); p.inv_d = div_reciprocal(p.d_tiles);
  moe_few_router_kernel<<<(unsigned)p.T, 256, 0, st>>>(c.x, c.ldx, c.router, p.D, p.E, p.top_k, (int*)p.choice, (float*)p.weight, p.counters, plan.n_counters);
  if (const cudaError_t e = cudaGetLastError()) return -(int)e;
  const long met = (c.T * c.top_k < c.E ? c.T * c.top_k : c.E) + (c.shared_gate_up != nullptr);     // experts at most
  const long items = met * (p.f_tiles + p.d_tiles);
  const int n = (int)(items < 296 ? items : 296);
#define INV_MF(NT) (c.i8 ? launch_moe_few<NT, true>(p, n, device, st) : launch_moe_few<NT, false>(p, n, device, st))
  return p.T <= 8 ? INV_MF(1) : p.T <= 16 ? INV_MF(2) : p.T <= 32 ? INV_MF(4) : INV_MF(8);
#undef INV_MF
}
