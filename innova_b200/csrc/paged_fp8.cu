// Paged cache of keys and values in 8 bits with a scale for each page and head: append with norms and rotation on the way, and attention over it.
//
// Pools: codes [pages, Hkv, 16, D] float8 e4m3, scales [pages, Hkv] fp32; a token's value is code * scale. The scale of a page and head is the smallest
// power of two 2^e >= 2^-64 with |x| <= 448 * 2^e for all tokens stored there. A power of two: where a later token raises the scale, the codes of the
// earlier ones move by an exponent and keep their three bits (but for what falls under 2^-6 after the move), so that what a page reads as hardly
// depends on the portions it was written in. A value that is not finite makes the scale NaN and the page's tokens read as NaN, as it would without a cache.
//
// New tokens come packed: sequence i has tokens [cu[i], cu[i + 1]) of T, at positions start[i], start[i] + 1, ... of page table row rows[i]. Rows are
// distinct. What the tables say is checked against the pools' sizes; a bad entry is reported through *status and its page skipped.
#include "head_norm.cuh"
#include "inv_api.h"

#include <cuda_fp16.h>

namespace inv {

constexpr int FP8_PAGE = 16;

struct Fp8Pool {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int pages, Hkv;
};
struct Fp8Tokens {
  const int *rows, *cu, *start, *page_table;
  int n, T, table_rows, max_pages;
  int* status;
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t half2_of_e4m3x2(uint32_t two) {        // of the lower 16 bits
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((uint16_t)two));
  return d;
}
// Four codes times `f`, rounded to codes again.
__device__ __forceinline__ uint32_t requantise(uint32_t codes, float f) {
  const uint32_t a = half2_of_e4m3x2(codes), b = half2_of_e4m3x2(codes >> 16);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return e4m3x2(x.x * f, x.y * f) | (e4m3x2(y.x * f, y.y * f) << 16);
}
// The scale of a page whose largest value has these bits (sign off): 448 is 1.75 * 2^8.
__device__ __forceinline__ float scale_of_bits(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);      // biased by 127
  return __uint_as_float((uint32_t)max(e, 127 - 64) << 23);
}

// The page of the pool behind page `pg` of table row `row`, or -1.
__device__ __forceinline__ int pool_page(const Fp8Tokens& t, int pages, int row, int pg) {
  if ((unsigned)row < (unsigned)t.table_rows && (unsigned)pg < (unsigned)t.max_pages) {
    const int id = t.page_table[(long)row * t.max_pages + pg];
    if ((unsigned)id < (unsigned)pages) return id;
  }
  atomicCAS(t.status, 0, ERR_BAD_ARG);
  return -1;
}

// ---------------------------------------------------------------------------------------------- append
struct Fp8Append {
  const __nv_bfloat16 *q_in, *k_in, *v_in, *wq, *wk;   // rows ld_in apart, H, Hkv and Hkv heads side by side; weights null: no norm
  const float *cos_t, *sin_t;           // null: no rotation
  const int* pos;                       // positions of the rotation, per token; null: the token's place in its sequence
  __nv_bfloat16* q;
  long ld_in, ld_v, ld_q;
  int H, rot, table_rows;
  float eps;
};

// A CTA takes the new tokens of one page, and of the heads its share blockIdx.y. Sequence i owns the CTAs from cu[i] / 16 + 2 i on, which is enough for
// the pages that its tokens touch wherever it starts. A warp stores the keys or values of one head: all of the page's new tokens in its registers, so
// that their largest value is known before any is rounded; queries it takes by groups of tokens, whose angles are loaded once.
template <int D>
__global__ void __launch_bounds__(256) fp8_append_kernel(const __grid_constant__ Fp8Append a, const __grid_constant__ Fp8Pool pool,
                                                         const __grid_constant__ Fp8Tokens tk) {
  constexpr int L = D / 16, HPW = 32 / L, NIT = FP8_PAGE / HPW;
  __shared__ int found[2];
  if (threadIdx.x == 0) found[0] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < tk.n; i += 256) {
    const int base = tk.cu[i] / FP8_PAGE + 2 * i, next = tk.cu[i + 1] / FP8_PAGE + 2 * (i + 1);
    if (base <= (int)blockIdx.x && (int)blockIdx.x < next) {
      found[0] = i;
      found[1] = base;
    }
  }
  __syncthreads();
  const int seq = found[0];
  if (seq < 0) return;
  const int t0 = tk.cu[seq], count = tk.cu[seq + 1] - t0, start = tk.start[seq];
  if (t0 < 0 || count < 0 || count > tk.T - t0 || start < 0) {
    if (threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
    return;
  }
  const int pg = start / FP8_PAGE + ((int)blockIdx.x - found[1]);
  const int lo = max(start, pg * FP8_PAGE), m = min(start + count, (pg + 1) * FP8_PAGE) - lo;      // positions [lo, lo + m)
  if (m <= 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane % L, sub = lane / L;
  const int groups = (m + HPW - 1) / HPW;
  const int zs = gridDim.y, z = blockIdx.y;
  const int h0 = (int)((long)a.H * z / zs), h1 = (int)((long)a.H * (z + 1) / zs);
  const int g0 = (int)((long)pool.Hkv * 2 * z / zs), g1 = (int)((long)pool.Hkv * 2 * (z + 1) / zs);
  const int page = pool_page(tk, pool.pages, tk.rows[seq], pg);
  const HeadUnit h(u, D, a.rot);
  // queries: (group of tokens, a run of heads)
  const int run = max(1, (h1 - h0) * groups / 16), runs = (h1 - h0 + run - 1) / run;      // none without query heads
  const int n_kv = page < 0 ? 0 : g1 - g0;
  for (int item = warp; item < n_kv + groups * runs; item += 8) {
    if (item >= n_kv) {
      const int grp = (item - n_kv) % groups, hq = h0 + (item - n_kv) / groups * run;
      const int i = grp * HPW + sub;
      const bool ok = i < m;
      const int at = lo + min(i, m - 1), t = t0 + at - start;
      Turn turn;
      if (a.rot) turn.load(a.cos_t, a.sin_t, a.rot, table_row(a.pos ? a.pos[t] : at, a.table_rows, tk.status), u, h);
      float w[16];
      if (a.wq) load_unit(a.wq, h, w);
      const __nv_bfloat16* src = a.q_in + t * a.ld_in;
      __nv_bfloat16* dst = a.q + t * a.ld_q;
#pragma unroll 2
      for (int hd = hq; hd < min(h1, hq + run); ++hd) {
        float v[16];
        load_unit(src + hd * D, h, v);
        if (a.wq) {
          const float r = head_rstd<L>(v, 1.f / D, a.eps);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
        }
        turn.apply<false>(h, v);
        if (ok) store_unit(dst + hd * D, h, v);
      }
      continue;
    }
    const int g = g0 + item, hk = g >> 1, which = g & 1;         // 0 keys, 1 values
    const __nv_bfloat16* src = (which ? a.v_in : a.k_in) + hk * D;
    const long ld = which ? a.ld_v : a.ld_in;
    float x[NIT][16];
    uint32_t amax = 0;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      if (it >= groups) break;
      const int at = lo + min(it * HPW + sub, m - 1), t = t0 + at - start;      // lanes past the last token repeat it
      load_unit(src + t * ld, h, x[it]);
      if (!which) {
        if (a.wk) {
          float w[16];
          load_unit(a.wk, h, w);
          const float r = head_rstd<L>(x[it], 1.f / D, a.eps);
#pragma unroll
          for (int e = 0; e < 16; ++e) x[it][e] = x[it][e] * r * w[e];
        }
        if (a.rot) {
          Turn turn;
          turn.load(a.cos_t, a.sin_t, a.rot, table_row(a.pos ? a.pos[t] : at, a.table_rows, tk.status), u, h);
          turn.apply<false>(h, x[it]);
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = max(amax, __float_as_uint(x[it][e]) & 0x7fffffffu);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    float scale = scale_of_bits(amax);
    const long block = (long)page * pool.Hkv + hk;
    uint8_t* codes = (which ? pool.v : pool.k) + block * FP8_PAGE * D;
    float* scales = (which ? pool.v_scale : pool.k_scale) + block;
    const int slot0 = lo % FP8_PAGE;
    if (slot0 > 0) {                                             // earlier tokens of the sequence are in the page
      const float old = *scales;
      __syncwarp();
      if (scale > old) {
        const float f = old / scale;
        uint4* p = reinterpret_cast<uint4*>(codes);
        for (int i = lane; i < slot0 * (D / 16); i += 32) {
          uint4 c = p[i];
          c.x = requantise(c.x, f); c.y = requantise(c.y, f); c.z = requantise(c.z, f); c.w = requantise(c.w, f);
          p[i] = c;
        }
      } else if (scale <= old || old != old) {
        scale = old;
      }
    }
    const float inv = 1.f / scale;
    const bool number = scale == scale;
    if (lane == 0) *scales = scale;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      if (it * HPW + sub >= m) break;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = number ? e4m3x2(x[it][4 * e] * inv, x[it][4 * e + 1] * inv) | (e4m3x2(x[it][4 * e + 2] * inv, x[it][4 * e + 3] * inv) << 16) : 0u;
      uint8_t* dst = codes + (slot0 + it * HPW + sub) * D;
      *reinterpret_cast<uint2*>(dst + h.e0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + h.e1) = make_uint2(w[2], w[3]);
    }
  }
}

// ---------------------------------------------------------------------------------------------- attention
struct Fp8Attend {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  long ld_q, ld_o;
  int H, G;             // query heads; of one key head
  int window;           // > 0: a token sees the `window` latest positions, its own included
  float scale;
  int per_split;        // pages of a CTA
  int splits, tiles;
  float* part;          // splits > 1: [T, H, splits, D + 2] (maximum, sum, values)
  int* used;            // splits > 1: [T, H] splits that a row has
  // Rows of a token tree (or null): row t is of table row row_seq[t], which holds seq_lens[.] tokens, and sees those below tail_start[t] and of the 64
  // from there on the ones whose bit is set.
  const int *row_seq, *seq_lens, *tail_start;
  const unsigned long long* tail_mask;
};

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 load_stream2(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A lane's codes of one page: of the keys, tokens 4 (n / 2) + n % 2 and that + 2 (n = lane / 4), dimensions 64 j + 16 c on (c = lane % 4);
// of the values, tokens 4 c to 4 c + 3, dimensions n D / 8 on.
template <int D>
struct PageCodes {
  static constexpr int KP = D / 64, VW = D / 32;
  uint4 k[2][KP];
  uint32_t v[4][VW];
  __device__ __forceinline__ void load(const Fp8Pool& pool, int id, int hk, int lane) {
    const int n = lane >> 2, c = lane & 3;
    const long base = ((long)id * pool.Hkv + hk) * FP8_PAGE * D;
    const uint8_t* kp = pool.k + base + (4 * (n >> 1) + (n & 1)) * D + c * 16;
    const uint8_t* vp = pool.v + base + 4 * c * D + n * (D / 8);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < KP; ++i) k[j][i] = load_stream(kp + 2 * j * D + i * 64);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (D == 128) {
        const uint4 w = load_stream(vp + r * D);
        v[r][0] = w.x; v[r][1] = w.y; v[r][VW - 2] = w.z; v[r][VW - 1] = w.w;
      } else {
        const uint2 w = load_stream2(vp + r * D);
        v[r][0] = w.x; v[r][1] = w.y;
      }
    }
  }
};

// Sixteen rows (query tokens times the heads that share a key head) against a run of pages: grid = sequences x key heads x splits x row tiles, four warps
// that take a page in turn, each with a softmax of its own; they join at the end.
//
// Scores and values are products on m16n8k16 tensor instructions in fp16: a code is exact there, and so is a query up to 2^-24 of its row's largest value
// once the row is scaled by a power of two. Which dimension or token an index of a product means is free as long as both operands agree, so a lane's
// 16-byte pieces of a key row are its operands as they lie, and the tokens of a page are numbered such that a lane's four scores a row are the four tokens
// whose values it loads. Page scales multiply the scores, and the weights relative to the largest value scale so far, which the sums are kept in.
// Weights are 2^(s - m + 6) with a maximum that is raised only by scores above m + 8, so at most 2^14, and what fp16 rounds away of a weight is under
// 2^-30 of the largest one.
template <int D, bool TREE>
__global__ void __launch_bounds__(128) fp8_attend_kernel(const __grid_constant__ Fp8Attend a, const __grid_constant__ Fp8Pool pool,
                                                         const __grid_constant__ Fp8Tokens tk) {
  constexpr int NW = 4, KS = D / 16, NB = D / 8, KP = D / 64, VW = D / 32;
  constexpr float LIFT = 6.f, SLACK = 8.f;
  __shared__ float sm_m[NW][16], sm_l[NW][16];
  __shared__ float sm_o[NW][16][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  int x = blockIdx.x;
  const int tile = x % a.tiles;
  x /= a.tiles;
  const int split = x % a.splits;
  x /= a.splits;
  const int hk = x % pool.Hkv, seq = x / pool.Hkv;
  // rows r of the tile: token r / G, head r % G of the key head's
  int t0, row, rows, start = 0, len = 0, tail = 0;
  unsigned long long bits = 0;
  if (TREE) {
    t0 = seq;
    row = a.row_seq[seq];
    rows = a.G;
    if ((unsigned)row >= (unsigned)tk.table_rows) {
      if (threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
    } else {
      len = a.seq_lens[row];
      tail = a.tail_start ? a.tail_start[seq] : len;
      bits = a.tail_mask ? a.tail_mask[seq] : 0;
    }
  } else {
    t0 = tk.cu[seq];
    const int count = tk.cu[seq + 1] - t0;
    start = tk.start[seq];
    row = tk.rows[seq];
    if (t0 < 0 || count < 0 || count > tk.T - t0 || start < 0) {
      if (threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
      return;
    }
    rows = count * a.G;
    if (rows > 16 * a.tiles && threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);         // more new tokens than the caller said
  }
  const int r0 = tile * 16, nr = min(16, rows - r0);
  if (nr <= 0) return;
  const int first = start + r0 / a.G, last = start + (r0 + nr - 1) / a.G;       // positions of the tile's tokens
  const int hi = TREE ? len : last + 1, lo = !TREE && a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int pg_lo = lo / FP8_PAGE, pg_hi = (hi + FP8_PAGE - 1) / FP8_PAGE;
  const int p0 = pg_lo + split * a.per_split, p1 = split + 1 < a.splits ? min(pg_hi, p0 + a.per_split) : pg_hi;    // the last one takes the rest
  if (split > 0 && p0 >= p1) return;
  // visible positions of this lane's two rows: [vlo, vhi)
  int vlo[2], vhi[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int p = start + min(r0 + n + 8 * e, rows - 1) / a.G;
    vhi[e] = TREE ? len : p + 1;
    vlo[e] = !TREE && a.window > 0 ? p - a.window + 1 : 0;
  }
  const int all_lo = !TREE && a.window > 0 ? last - a.window + 1 : 0, all_hi = TREE ? min(tail, len) : first + 1;    // positions that every row sees

  // ---- queries ----
  uint32_t qa[KS][4];
  float qm[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = r0 + n + 8 * e;
    uint4 raw[KP][2];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        raw[j][i] = make_uint4(0, 0, 0, 0);
        if (n + 8 * e < nr) raw[j][i] = *reinterpret_cast<const uint4*>(a.q + (t0 + r / a.G) * a.ld_q + (hk * a.G + r % a.G) * D + j * 64 + c * 16 + i * 8);
        const uint32_t w[4] = {raw[j][i].x, raw[j][i].y, raw[j][i].z, raw[j][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = min(max((int)(top >> 7), 1), 253);                           // 2^(ex - 127): the row's largest value, but for its fraction
    const float down = __uint_as_float((uint32_t)(254 - ex) << 23);
    qm[e] = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)ex << 23);
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 v = raw[j][i >> 1];
        const uint32_t w0 = i & 1 ? v.z : v.x, w1 = i & 1 ? v.w : v.y;
        qa[j * 4 + i][e] = half2_of(__uint_as_float(w0 << 16) * down, __uint_as_float(w0 & 0xffff0000u) * down);
        qa[j * 4 + i][2 + e] = half2_of(__uint_as_float(w1 << 16) * down, __uint_as_float(w1 & 0xffff0000u) * down);
      }
  }

  float o[NB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, vref = 0.f, vinv = 0.f;
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  // A lane keeps number and scales of one of the warp's next 32 pages.
  int ids = -1;
  float kss = 0.f, vss = 0.f;
  auto look_up = [&](int pg) {
    ids = -1;
    if (pg < p1) {
      ids = pool_page(tk, pool.pages, row, pg);
      if (ids >= 0) {
        kss = pool.k_scale[(long)ids * pool.Hkv + hk];
        vss = pool.v_scale[(long)ids * pool.Hkv + hk];
      }
    }
  };
  const int mine = p1 > p0 + warp ? (p1 - p0 - warp + NW - 1) / NW : 0;          // pages of this warp
  PageCodes<D> next;
  int id_n = -1;
  float ks_n = 0.f, vs_n = 0.f;
  auto fetch = [&](int i) {
    if ((i & 31) == 0) look_up(p0 + warp + NW * (i + lane));
    id_n = __shfl_sync(0xffffffffu, ids, i & 31);
    ks_n = __shfl_sync(0xffffffffu, kss, i & 31);
    vs_n = __shfl_sync(0xffffffffu, vss, i & 31);
    if (id_n >= 0) next.load(pool, id_n, hk, lane);
  };
  if (mine > 0) fetch(0);
  for (int i = 0; i < mine; ++i) {
    const PageCodes<D> now = next;
    const int id = id_n, pos = (p0 + warp + NW * i) * FP8_PAGE;
    const float ks = ks_n, vs = vs_n;
    if (i + 1 < mine) fetch(i + 1);
    if (id < 0) continue;
    // ---- scores ----
    float s[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int q = 0; q < KP; ++q) {
        const uint32_t w[4] = {now.k[j][q].x, now.k[j][q].y, now.k[j][q].z, now.k[j][q].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t(&f)[4] = qa[q * 4 + k];
          mma_f16(s[j], f[0], f[1], f[2], f[3], half2_of_e4m3x2(w[k]), half2_of_e4m3x2(w[k] >> 16));
        }
      }
    }
    const float f0 = qm[0] * ks, f1 = qm[1] * ks;
    const bool whole = pos >= all_lo && pos + FP8_PAGE <= all_hi;
    bool over = vs > vref;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] *= e < 2 ? f0 : f1;
        if (!whole) {
          const int at = pos + 4 * c + 2 * j + (e & 1);
          bool seen = at >= vlo[e >> 1] && at < vhi[e >> 1];
          if (TREE) seen = seen && (at < tail || (at - tail < 64 && ((bits >> ((at - tail) & 63)) & 1ull)));
          if (!seen) s[j][e] = -INFINITY;
        }
        over |= s[j][e] > m[e >> 1] + SLACK;
      }
    if (__any_sync(0xffffffffu, over)) {
      const float beta = vs > vref ? vref / vs : 1.f;
      if (vs > vref) {
        vref = vs;
        vinv = 1.f / vs;
      }
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float up = fmaxf(m[e], mx);
        alpha[e] = up == m[e] ? 1.f : exp2_fast(m[e] - up);
        m[e] = up;
        l[e] *= alpha[e];
        alpha[e] *= beta;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        o[b][0] *= alpha[0];
        o[b][1] *= alpha[0];
        o[b][2] *= alpha[1];
        o[b][3] *= alpha[1];
      }
    }
    const float rel = vs * vinv;
    uint32_t pa[4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float w0 = exp2_fast(s[j][2 * e] - m[e] + LIFT), w1 = exp2_fast(s[j][2 * e + 1] - m[e] + LIFT), x0 = w0 * rel, x1 = w1 * rel;
        if (!whole) {                                 // nothing of a hidden place, whatever its scale and however little the row has seen
          if (s[j][2 * e] == -INFINITY) w0 = x0 = 0.f;
          if (s[j][2 * e + 1] == -INFINITY) w1 = x1 = 0.f;
        }
        l[e] += w0 + w1;
        pa[2 * j + e] = half2_of(x0, x1);
      }
    // ---- values ----
    const int keep = hi - pos - 4 * c;                // slots past the end hold whatever was there
#pragma unroll
    for (int q = 0; q < VW; ++q) {
      uint32_t v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = whole || r < keep ? now.v[r][q] : 0u;
      const uint32_t a01 = __byte_perm(v[0], v[1], 0x5140), b01 = __byte_perm(v[0], v[1], 0x7362);
      const uint32_t a23 = __byte_perm(v[2], v[3], 0x5140), b23 = __byte_perm(v[2], v[3], 0x7362);
      mma_f16(o[4 * q], pa[0], pa[1], pa[2], pa[3], half2_of_e4m3x2(a01), half2_of_e4m3x2(a23));
      mma_f16(o[4 * q + 1], pa[0], pa[1], pa[2], pa[3], half2_of_e4m3x2(a01 >> 16), half2_of_e4m3x2(a23 >> 16));
      mma_f16(o[4 * q + 2], pa[0], pa[1], pa[2], pa[3], half2_of_e4m3x2(b01), half2_of_e4m3x2(b23));
      mma_f16(o[4 * q + 3], pa[0], pa[1], pa[2], pa[3], half2_of_e4m3x2(b01 >> 16), half2_of_e4m3x2(b23 >> 16));
    }
  }

  // ---- the warps' shares ----
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (c == 0) {
      sm_m[warp][n + 8 * e] = m[e];
      sm_l[warp][n + 8 * e] = l[e];
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      sm_o[warp][n + 8 * e][2 * c * (D / 8) + b] = o[b][2 * e] * vref;
      sm_o[warp][n + 8 * e][(2 * c + 1) * (D / 8) + b] = o[b][2 * e + 1] * vref;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nr * D; i += 128) {
    const int r = i / D, d = i % D;
    float mm = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm_m[w][r]);
    float acc = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = mm == -INFINITY ? 1.f : exp2_fast(sm_m[w][r] - mm);
      acc += sm_o[w][r][d] * f;
      ll += sm_l[w][r] * f;
    }
    const int t = t0 + (r0 + r) / a.G, hd = hk * a.G + (r0 + r) % a.G;
    if (a.splits == 1) {
      a.out[t * a.ld_o + hd * D + d] = __float2bfloat16_rn(ll == 0.f ? 0.f : acc / ll);
      continue;
    }
    float* part = a.part + (((long)t * a.H + hd) * a.splits + split) * (D + 2);
    part[2 + d] = acc;
    if (d == 0) {
      part[0] = mm;
      part[1] = ll;
      if (split == 0) a.used[(long)t * a.H + hd] = max(1, min(a.splits, (pg_hi - pg_lo + a.per_split - 1) / a.per_split));
    }
  }
}

// Joins the splits of a row: a warp a row and head.
template <int D>
__global__ void __launch_bounds__(256) fp8_join_kernel(const float* __restrict__ part, const int* __restrict__ used, __nv_bfloat16* __restrict__ out,
                                                       long ld_o, int T, int H, int splits) {
  wait_previous();
  const long item = blockIdx.x * 8l + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long)T * H) return;
  const float* base = part + item * splits * (D + 2);
  const int ns = used[item];
  float mm = -INFINITY;
  for (int s = lane; s < ns; s += 32) mm = fmaxf(mm, base[(long)s * (D + 2)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  float acc[D / 32], ll = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int s = 0; s < ns; ++s) {
    const float* p = base + (long)s * (D + 2);
    const float f = mm == -INFINITY ? 1.f : exp2_fast(p[0] - mm);
    ll += p[1] * f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] += p[2 + lane + 32 * i] * f;
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    out[item / H * ld_o + item % H * D + lane + 32 * i] = __float2bfloat16_rn(ll == 0.f ? 0.f : acc[i] / ll);
}

}  // namespace inv

using namespace inv;

static bool fp8_bad_shape(int H, int Hkv, int D, int pages, int n, int T, int table_rows, int max_pages) {
  return (D != 64 && D != 128) || Hkv < 1 || H < Hkv || H % Hkv || pages < 1 || n < 0 || T < 0 || table_rows < 1 || max_pages < 1;
}
static bool off16(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) % 16 != 0;
}

// q_in [T, H D], k_in, v_in [T, Hkv D] bf16 -> q [T, H D] normed and rotated, and the pools. Queries and keys have rows ld_in apart, values ld_v, q
// ld_q; H may be 0. wq, wk [D] bf16 or null; cos_t, sin_t [rope_rows, rot / 2] fp32 or null with rot 0; pos [T] or null.
extern "C" int inv_fp8_append(const void* q_in, const void* k_in, long ld_in, const void* v_in, long ld_v, void* q, long ld_q, int H, int Hkv, int D,
                              const void* wq, const void* wk, float eps, const float* cos_t, const float* sin_t, int rope_rows, int rot, const int* pos,
                              void* k_pool, void* v_pool, float* k_scale, float* v_scale, int pages, const int* page_table, int table_rows,
                              int max_pages, const int* rows, const int* cu, const int* start, int n, int T, int* status, void* stream) {
  if (fp8_bad_shape(H ? H : Hkv, Hkv, D, pages, n, T, table_rows, max_pages) || rot < 0 || rot > D || rot % 16) return -ERR_BAD_ARG;
  if (rot && (!cos_t || !sin_t || rope_rows < 1)) return -ERR_BAD_ARG;
  if (ld_in % 8 || ld_v % 8 || ld_q % 8 || off16(q_in, k_in, v_in, q) || off16(wq, wk) || off16(cos_t, sin_t, k_pool, v_pool)) return -ERR_BAD_ARG;
  if (n == 0 || T == 0) return 0;
  const Fp8Append a{(const __nv_bfloat16*)q_in, (const __nv_bfloat16*)k_in, (const __nv_bfloat16*)v_in, (const __nv_bfloat16*)wq,
                    (const __nv_bfloat16*)wk, cos_t, sin_t, pos, (__nv_bfloat16*)q, ld_in, ld_v, ld_q, H, rot, rope_rows, eps};
  const Fp8Pool pool{(uint8_t*)k_pool, (uint8_t*)v_pool, k_scale, v_scale, pages, Hkv};
  const Fp8Tokens tk{rows, cu, start, page_table, n, T, table_rows, max_pages, status};
  const unsigned ctas = (unsigned)(T / FP8_PAGE + 2 * n);
  const dim3 grid(ctas, 1);
  if (D == 64) fp8_append_kernel<64><<<grid, 256, 0, (cudaStream_t)stream>>>(a, pool, tk);
  else fp8_append_kernel<128><<<grid, 256, 0, (cudaStream_t)stream>>>(a, pool, tk);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}

// Pages of a CTA, and from it CTAs along a sequence of `pages` pages.
static int pages_per_split(long units, int pages) {
  const long target = 148 * 12;
  long per = (units * pages + target - 1) / target;
  if (per < 32) per = 32;
  return (int)(per < pages ? per : pages);
}
// Splits that inv_fp8_attend will use, for its caller's workspace: [T, H, splits, D + 2] floats and [T, H] ints where there are several.
extern "C" int inv_fp8_attend_splits(int n, int Hkv, int G, int max_new, int max_len, int window) {
  if (n < 1 || Hkv < 1 || G < 1 || max_new < 1 || max_len < 1) return 1;
  const int tiles = (int)(((long)max_new * G + 15) / 16);
  const long span = window > 0 && (long)window + max_new < max_len ? (long)window + max_new : max_len;
  const int pages = (int)((span + 2 * FP8_PAGE - 2) / FP8_PAGE);
  return (pages + pages_per_split((long)n * Hkv * tiles, pages) - 1) / pages_per_split((long)n * Hkv * tiles, pages);
}

static int fp8_attend(Fp8Attend a, const Fp8Pool& pool, const Fp8Tokens& tk, int D, int max_new, int max_len, bool tree, cudaStream_t st) {
  const int G = a.H / pool.Hkv;
  a.G = G;
  a.tiles = (int)(((long)max_new * G + 15) / 16);
  a.splits = inv_fp8_attend_splits(tk.n, pool.Hkv, G, max_new, max_len, a.window);
  const long span = a.window > 0 && (long)a.window + max_new < max_len ? (long)a.window + max_new : max_len;
  const int pages = (int)((span + 2 * FP8_PAGE - 2) / FP8_PAGE);
  a.per_split = pages_per_split((long)tk.n * pool.Hkv * a.tiles, pages);
  if (a.splits > 1 && (!a.part || !a.used)) return -ERR_BAD_ARG;
  const long ctas = (long)tk.n * pool.Hkv * a.splits * a.tiles;
  if (ctas > 0x7fffffffl) return -ERR_BAD_ARG;
#define INV_FP8(DD, TR) fp8_attend_kernel<DD, TR><<<(unsigned)ctas, 128, 0, st>>>(a, pool, tk)
  if (D == 64) { if (tree) INV_FP8(64, true); else INV_FP8(64, false); }
  else { if (tree) INV_FP8(128, true); else INV_FP8(128, false); }
#undef INV_FP8
  if (a.splits > 1) {
    const dim3 grid((unsigned)(((long)tk.T * a.H + 7) / 8));
    if (D == 64) launch_early(fp8_join_kernel<64>, grid, 256, 0, st, a.part, a.used, a.out, a.ld_o, tk.T, a.H, a.splits);
    else launch_early(fp8_join_kernel<128>, grid, 256, 0, st, a.part, a.used, a.out, a.ld_o, tk.T, a.H, a.splits);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}

// q [T, H D] bf16, rows ld_q apart -> out [T, H D], rows ld_o apart: the token at position p of its sequence sees the cached positions up to p, with a
// window the latest `window` of them. No sequence has more than max_new new tokens or, with them, max_len tokens.
extern "C" int inv_fp8_attend(const void* q, long ld_q, void* out, long ld_o, int H, int Hkv, int D, float scale, int window, const void* k_pool,
                              const void* v_pool, const float* k_scale, const float* v_scale, int pages, const int* page_table, int table_rows,
                              int max_pages, const int* rows, const int* cu, const int* start, int n, int T, int max_new, int max_len, float* part,
                              int* used, int* status, void* stream) {
  if (fp8_bad_shape(H, Hkv, D, pages, n, T, table_rows, max_pages) || window < 0 || max_new < 1 || max_len < 1) return -ERR_BAD_ARG;
  if (ld_q % 8 || off16(q, k_pool, v_pool)) return -ERR_BAD_ARG;
  if (n == 0 || T == 0) return 0;
  Fp8Attend a{};
  a.q = (const __nv_bfloat16*)q; a.out = (__nv_bfloat16*)out; a.ld_q = ld_q; a.ld_o = ld_o; a.H = H; a.window = window; a.scale = scale;
  a.part = part; a.used = used;
  const Fp8Pool pool{(uint8_t*)k_pool, (uint8_t*)v_pool, (float*)k_scale, (float*)v_scale, pages, Hkv};
  const Fp8Tokens tk{rows, cu, start, page_table, n, T, table_rows, max_pages, status};
  return fp8_attend(a, pool, tk, D, max_new, max_len, false, (cudaStream_t)stream);
}

// One query token a row over shared sequences: row t belongs to table row row_seq[t], which holds seq_lens[row_seq[t]] tokens, and sees those below
// tail_start[t] and token tail_start[t] + i iff bit i of tail_mask[t] is set (both null: all).
extern "C" int inv_fp8_attend_tree(const void* q, long ld_q, void* out, long ld_o, int H, int Hkv, int D, float scale, const void* k_pool,
                                   const void* v_pool, const float* k_scale, const float* v_scale, int pages, const int* page_table, int table_rows,
                                   int max_pages, const int* row_seq, const int* seq_lens, const int* tail_start, const unsigned long long* tail_mask,
                                   int T, int max_len, float* part, int* used, int* status, void* stream) {
  if (fp8_bad_shape(H, Hkv, D, pages, T, T, table_rows, max_pages) || max_len < 1 || !row_seq || !seq_lens || !tail_start != !tail_mask) return -ERR_BAD_ARG;
  if (ld_q % 8 || off16(q, k_pool, v_pool)) return -ERR_BAD_ARG;
  if (T == 0) return 0;
  Fp8Attend a{};
  a.q = (const __nv_bfloat16*)q; a.out = (__nv_bfloat16*)out; a.ld_q = ld_q; a.ld_o = ld_o; a.H = H; a.scale = scale; a.part = part; a.used = used;
  a.row_seq = row_seq; a.seq_lens = seq_lens; a.tail_start = tail_start; a.tail_mask = tail_mask;
  const Fp8Pool pool{(uint8_t*)k_pool, (uint8_t*)v_pool, (float*)k_scale, (float*)v_scale, pages, Hkv};
  const Fp8Tokens tk{nullptr, nullptr, nullptr, page_table, T, T, table_rows, max_pages, status};
  return fp8_attend(a, pool, tk, D, 1, max_len, true, (cudaStream_t)stream);
}
