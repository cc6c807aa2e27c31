// One head of a token in the lanes of a warp: RMS norm with a weight, half-split rotation, and their transposes. Shared by the stand-alone norm and
// rotation (qk_norm.cu) and the append to the paged 8-bit cache (paged_fp8.cu).
//
// A head of D values (a multiple of 16) is cut into D / 16 units of two runs of eight. A unit of the rotated part, the first `rot` values, holds the run
// u * 8 and its partner rot / 2 + u * 8, so that every pair of the rotation sits in one thread; behind it units are simply sixteen values in a row. A
// head takes the next power of two of lanes, of which D / 16 have a unit.
#pragma once
#include "once_per_device.h"
#include "sm100_common.cuh"

namespace inv {

__host__ __device__ constexpr int head_lanes(int D) {
  int l = 1;
  while (l * 16 < D) l *= 2;
  return l;
}

struct HeadUnit {
  int e0, e1;     // first element of the two runs
  bool has, turns;
  __device__ __forceinline__ HeadUnit(int u, int D, int rot) {
    has = u * 16 < D;
    turns = u * 16 < rot;
    e0 = turns ? u * 8 : has ? u * 16 : 0;              // a lane without a unit reads the head's first values
    e1 = turns ? rot / 2 + u * 8 : e0 + 8;
  }
};

// Two 32-bit values as one operand of the packed instructions.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float2 of_pair(uint64_t x) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 shared8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A unit as it lies in memory: fetched without a branch, so that several are on their way at once, and widened when they are there.
template <typename T>
struct RawUnit {
  static constexpr int N = sizeof(T) / 2;               // 16-byte pieces of a run
  uint4 r[2 * N];
  __device__ __forceinline__ void fetch(const T* head, const HeadUnit& u) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      r[i] = reinterpret_cast<const uint4*>(head + u.e0)[i];
      r[N + i] = reinterpret_cast<const uint4*>(head + u.e1)[i];
    }
  }
  __device__ __forceinline__ void store(T* head, const HeadUnit& u) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      reinterpret_cast<uint4*>(head + u.e0)[i] = r[i];
      reinterpret_cast<uint4*>(head + u.e1)[i] = r[N + i];
    }
  }
  __device__ __forceinline__ void get(uint64_t (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
      if constexpr (N == 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i * 4 + k] = pair_of(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
      } else {
        x[i * 2] = pair_of(__uint_as_float(w[0]), __uint_as_float(w[1]));
        x[i * 2 + 1] = pair_of(__uint_as_float(w[2]), __uint_as_float(w[3]));
      }
    }
  }
  __device__ __forceinline__ void set(const uint64_t (&x)[8]) {
    uint32_t w[8 * N];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = of_pair(x[i]);
      if constexpr (N == 1) {
        w[i] = cvt_bf16x2(v.x, v.y);
      } else {
        w[2 * i] = __float_as_uint(v.x);
        w[2 * i + 1] = __float_as_uint(v.y);
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) r[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
};
template <typename T>
__device__ __forceinline__ void load_unit(const T* head, const HeadUnit& u, uint64_t (&x)[8]) {
  RawUnit<T> raw;
  raw.fetch(head, u);
  raw.get(x);
}

// Units that a lane will read come by asynchronous copies into its own places of shared memory, which takes no registers and no barrier: a ring of STAGES
// steps of UNITS units for each of WARPS warps.
template <typename T, int UNITS, int STAGES_, int WARPS>
struct UnitRing {
  static constexpr int NP = RawUnit<T>::N, PIECES = UNITS * 2 * NP, STAGES = STAGES_, BYTES = WARPS * STAGES * PIECES * 32 * 16;
  __device__ __forceinline__ static uint4* of_lane(uint4* ring) { return ring + (threadIdx.x >> 5) * (STAGES * PIECES * 32) + (threadIdx.x & 31); }
  __device__ __forceinline__ static void copy(uint4* mine, int stage, int unit, const T* head, const HeadUnit& h) {
    const uint32_t to = smem_u32(mine + (stage * PIECES + unit * 2 * NP) * 32);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      copy16_async(to + i * 512, head + h.e0 + i * (16 / sizeof(T)));
      copy16_async(to + (NP + i) * 512, head + h.e1 + i * (16 / sizeof(T)));
    }
  }
  __device__ __forceinline__ static void get(const uint4* mine, int stage, int unit, RawUnit<T>& raw) {
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) raw.r[i] = mine[(stage * PIECES + unit * 2 * NP + i) * 32];
  }
};

// Sum over the L lanes of a head; what a lane without a unit brings counts for nothing.
template <int L>
__device__ __forceinline__ float head_sum(uint64_t two, const HeadUnit& u) {
  const float2 e = of_pair(two);
  float v = u.has ? e.x + e.y : 0.f;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// 1 / sqrt(mean of squares + eps)
template <int L>
__device__ __forceinline__ float head_rstd(const uint64_t (&x)[8], const HeadUnit& u, float inv_d, float eps) {
  uint64_t s0 = mul_pair(x[0], x[0]), s1 = mul_pair(x[1], x[1]);
#pragma unroll
  for (int i = 2; i < 8; i += 2) {
    s0 = fma_pair(x[i], x[i], s0);
    s1 = fma_pair(x[i + 1], x[i + 1], s1);
  }
  return rsqrtf(head_sum<L>(add_pair(s0, s1), u) * inv_d + eps);
}
template <int L, typename T>
__device__ __forceinline__ void head_norm(uint64_t (&x)[8], const T* weight, const HeadUnit& u, float inv_d, float eps) {
  uint64_t w[8];
  load_unit(weight, u, w);
  const float r = head_rstd<L>(x, u, inv_d, eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = mul_pair(mul_pair(x[i], pair_of(r, r)), w[i]);
}

// Cosines and sines of a unit's eight pairs at one position.
struct Turn {
  uint64_t c[4], s[4];
  __device__ __forceinline__ void load(const float* cos_t, const float* sin_t, int rot, int pos, int u, const HeadUnit& h) {
    const size_t at = (size_t)pos * (rot / 2) + (h.turns ? u * 8 : 0);
    take(reinterpret_cast<const float4*>(cos_t + at), reinterpret_cast<const float4*>(sin_t + at));
  }
  __device__ __forceinline__ void take(const float4* cosines, const float4* sines) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 a = cosines[i], b = sines[i];
      c[2 * i] = pair_of(a.x, a.y);
      c[2 * i + 1] = pair_of(a.z, a.w);
      s[2 * i] = pair_of(b.x, b.y);
      s[2 * i + 1] = pair_of(b.z, b.w);
    }
  }
  // (x1, x2) -> (x1 c - x2 s, x1 s + x2 c); INV: by the transpose. The products with x2 are rounded, those with x1 enter the sum as they are. Said here,
  // since a packed product and a sum behind it are made one instruction by the assembler in any case, whatever rounding they name.
  template <bool INV>
  __device__ __forceinline__ void apply(const HeadUnit& h, uint64_t (&x)[8]) const {
    if (!h.turns) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t a = x[i], b = x[i + 4], minus = 0x8000000080000000ull;
      x[i] = fma_pair(a, c[i], mul_pair(INV ? b : b ^ minus, s[i]));
      x[i + 4] = fma_pair(INV ? a ^ minus : a, s[i], mul_pair(b, c[i]));
    }
  }
  // The same with every product rounded by itself: what elementary operations give, to the bit, for values that are to be rounded to a few bits.
  __device__ __forceinline__ void apply_apart(const HeadUnit& h, uint64_t (&x)[8]) const {
    if (!h.turns) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = of_pair(x[i]), b = of_pair(x[i + 4]), k = of_pair(c[i]), n = of_pair(s[i]);
      x[i] = pair_of(__fsub_rn(__fmul_rn(a.x, k.x), __fmul_rn(b.x, n.x)), __fsub_rn(__fmul_rn(a.y, k.y), __fmul_rn(b.y, n.y)));
      x[i + 4] = pair_of(__fadd_rn(__fmul_rn(a.x, n.x), __fmul_rn(b.x, k.x)), __fadd_rn(__fmul_rn(a.y, n.y), __fmul_rn(b.y, k.y)));
    }
  }
};

// The table's row of a position; one outside the table is reported and takes the nearest row.
__device__ __forceinline__ int table_row(int pos, int rows, int* status) {
  if ((unsigned)pos < (unsigned)rows) return pos;
  atomicCAS(status, 0, ERR_BAD_ARG);
  return pos < 0 ? 0 : rows - 1;
}

// The kernel's shared memory on the current device. 0, or the entry's error code.
template <typename K>
static int raise_smem(K* kernel, int bytes, OncePerDevice& ready) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess)
    e = (cudaError_t)ready.ask(device, [&] { return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
  if (e != cudaSuccess) cudaGetLastError();          // returned here, not by the next entry that asks
  return -(int)e;
}

}  // namespace inv
