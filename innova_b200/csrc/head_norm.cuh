// One head of a token in the lanes of a warp: RMS norm with a weight, half-split rotation, and their transposes. Shared by the stand-alone norm and
// rotation (qk_norm.cu) and the append to the paged 8-bit cache (paged_fp8.cu).
//
// A head of D values (a multiple of 16) is cut into D / 16 units of two runs of eight. A unit of the rotated part, the first `rot` values, holds the run
// u * 8 and its partner rot / 2 + u * 8, so that every pair of the rotation sits in one thread; behind it units are simply sixteen values in a row. A
// head takes the next power of two of lanes, of which D / 16 have a unit.
#pragma once
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

__device__ __forceinline__ void load8(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

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
  __device__ __forceinline__ void get(const HeadUnit& u, float (&x)[16]) const {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (N == 1) {
          x[i * 8 + 2 * k] = u.has ? __uint_as_float(w[k] << 16) : 0.f;
          x[i * 8 + 2 * k + 1] = u.has ? __uint_as_float(w[k] & 0xffff0000u) : 0.f;
        } else {
          x[i * 4 + k] = u.has ? __uint_as_float(w[k]) : 0.f;
        }
      }
    }
  }
  __device__ __forceinline__ void set(const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      if constexpr (N == 1)
        r[i] = make_uint4(cvt_bf16x2(x[i * 8], x[i * 8 + 1]), cvt_bf16x2(x[i * 8 + 2], x[i * 8 + 3]), cvt_bf16x2(x[i * 8 + 4], x[i * 8 + 5]),
                          cvt_bf16x2(x[i * 8 + 6], x[i * 8 + 7]));
      else
        r[i] = make_uint4(__float_as_uint(x[i * 4]), __float_as_uint(x[i * 4 + 1]), __float_as_uint(x[i * 4 + 2]), __float_as_uint(x[i * 4 + 3]));
    }
  }
};
template <typename T>
__device__ __forceinline__ void load_unit(const T* head, const HeadUnit& u, float (&x)[16]) {
  RawUnit<T> raw;
  raw.fetch(head, u);
  raw.get(u, x);
}

// Sum over the L lanes of a head.
template <int L>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// 1 / sqrt(mean of squares + eps)
template <int L>
__device__ __forceinline__ float head_rstd(const float (&x)[16], float inv_d, float eps) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = fmaf(x[i], x[i], s);
  return 1.f / sqrtf(head_sum<L>(s) * inv_d + eps);
}

// Cosines and sines of a unit's eight pairs at one position.
struct Turn {
  float c[8], s[8];
  __device__ __forceinline__ void load(const float* cos_t, const float* sin_t, int rot, int pos, int u, const HeadUnit& h) {
    const size_t at = (size_t)pos * (rot / 2) + (h.turns ? u * 8 : 0);
    load8(cos_t + at, c);
    load8(sin_t + at, s);
  }
  // (x1, x2) -> (x1 c - x2 s, x1 s + x2 c); INV: by the transpose. Products are rounded by themselves, as written.
  template <bool INV>
  __device__ __forceinline__ void apply(const HeadUnit& h, float (&x)[16]) const {
    if (!h.turns) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[i], b = x[i + 8], sn = INV ? -s[i] : s[i];
      x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, sn));
      x[i + 8] = __fadd_rn(__fmul_rn(a, sn), __fmul_rn(b, c[i]));
    }
  }
};

// The table's row of a position; one outside the table is reported and takes the nearest row.
__device__ __forceinline__ int table_row(int pos, int rows, int* status) {
  if ((unsigned)pos < (unsigned)rows) return pos;
  atomicCAS(status, 0, ERR_BAD_ARG);
  return pos < 0 ? 0 : rows - 1;
}

}  // namespace inv
