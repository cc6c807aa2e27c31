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

// The new tokens of a sequence, rows [t0, t0 + count) at positions [start, start + count). None where what the caller wrote cannot be: rows outside the
// tensor, positions behind the page table.
struct Fp8Span {
  int t0, count, start;
  bool fine;
  __device__ __forceinline__ Fp8Span(const Fp8Tokens& t, int cu0, int cu1, int start) : t0(cu0), count(cu1 - cu0), start(start) {
    fine = t0 >= 0 && count >= 0 && count <= t.T - t0 && start >= 0 && (long)start + count <= (long)t.max_pages * FP8_PAGE;
  }
  __device__ __forceinline__ Fp8Span(const Fp8Tokens& t, int seq) : Fp8Span(t, t.cu[seq], t.cu[seq + 1], t.start[seq]) {}
};

// ---------------------------------------------------------------------------------------------- append
struct Fp8Append {
  const __nv_bfloat16 *q_in, *k_in, *v_in, *wq, *wk;   // rows ld_in apart, H, Hkv and Hkv heads side by side; weights null: no norm
  const float *cos_t, *sin_t;           // null: no rotation
  const int* pos;                       // positions of the rotation, per token; null: the token's place in its sequence
  __nv_bfloat16* q;
  long ld_in, ld_v, ld_q;
  int H, rot, table_rows;
  uint32_t inv_h;                       // div_reciprocal
  float eps;
};

// Memory bounds it where there are many tokens: 2 x 8000 of 32 heads of 128 on 8, 369 MB in 65.5 us (5.6 TB/s). With rows in registers and angles read from
// the tables by each head, whose latency nothing hid, 82 us; with 32-bit rows in registers at one CTA an SM 193. A call of 64 x 1 takes 4.0 us, its chain of
// sequence, page, scale and store. Five CTAs an SM; four 5 us more, six 1.
constexpr int FP8_APPEND_CTAS = 5;
using Fp8AppendRing = UnitRing<__nv_bfloat16, 4, 2, 4>;
// A CTA takes the new tokens of one page, or with blockIdx.y a share of what they bring: items for its warps. Sequence i owns the CTAs from cu[i] / 16 + 2 i
// on, which is enough for the pages that its tokens touch wherever it starts. An item is the keys or the values of one head, all of the page's new tokens
// before a warp, so that their largest value is known before any is rounded; or a run of query heads. A warp's next item is on its way while it works on
// one, whose rows it reads again where it needs them (keys are normed and turned twice, for their largest value and for the codes).
template <int D>
__global__ void __launch_bounds__(128, FP8_APPEND_CTAS) fp8_append_kernel(const __grid_constant__ Fp8Append a, const __grid_constant__ Fp8Pool pool,
                                                            const __grid_constant__ Fp8Tokens tk) {
  constexpr int L = D / 16, HPW = 32 / L, NIT = FP8_PAGE / HPW, NQ = 4;
  using Raw = RawUnit<__nv_bfloat16>;
  using Ring = Fp8AppendRing;
  constexpr int ST = Ring::STAGES;
  extern __shared__ uint4 units[];
  __shared__ int found[5];
  __shared__ float4 cosines[FP8_PAGE][D / 8], sines[FP8_PAGE][D / 8];        // of the page's new tokens
  if (threadIdx.x == 0) found[0] = -1;
  __syncthreads();
  wait_previous();
  release_next();
  for (int i = threadIdx.x; i < tk.n; i += 128) {
    const int c0 = tk.cu[i], c1 = tk.cu[i + 1], start = tk.start[i], row = tk.rows[i];
    const int base = c0 / FP8_PAGE + 2 * i, next = c1 / FP8_PAGE + 2 * (i + 1);
    if (base <= (int)blockIdx.x && (int)blockIdx.x < next) {
      found[0] = base;
      found[1] = c0;
      found[2] = c1;
      found[3] = start;
      found[4] = row;
    }
  }
  __syncthreads();
  if (found[0] < 0) return;
  const Fp8Span span(tk, found[1], found[2], found[3]);
  const int t0 = span.t0, count = span.count, start = span.start, row = found[4];
  if (!span.fine) {
    if (threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
    return;
  }
  const int pg = start / FP8_PAGE + ((int)blockIdx.x - found[0]);
  const int lo = max(start, pg * FP8_PAGE), m = min(start + count, (pg + 1) * FP8_PAGE) - lo;      // positions [lo, lo + m)
  if (m <= 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane % L, sub = lane / L;
  const bool listed = (unsigned)row < (unsigned)tk.table_rows && (unsigned)pg < (unsigned)tk.max_pages;
  const int id = tk.page_table[listed ? (long)row * tk.max_pages + pg : 0];
  const HeadUnit h(u, D, a.rot);
  const int first = t0 + lo - start;                             // row of the page's first new token
  auto angles = [&](Turn& turn, int i) {
    const int at = h.turns ? u * 2 : 0;
    turn.take(cosines[i] + at, sines[i] + at);
  };
  const int n_kv = 2 * pool.Hkv, n_q = (m * a.H + NQ * HPW - 1) / (NQ * HPW);
  uint4* mine = Ring::of_lane(units);
  auto slot = [&](int item, int j, int& tok, int& hd) {          // the j-th head of a run in this lane
    const int s = (item - n_kv) * (NQ * HPW) + j * HPW + sub, at = min(s, m * a.H - 1);
    tok = div_by(at, a.H, a.inv_h);
    hd = at - tok * a.H;
    return s < m * a.H;
  };
  auto fetch = [&](int item, int stage) {
    if (item < n_kv) {
      const __nv_bfloat16* src = (item & 1 ? a.v_in : a.k_in) + (item >> 1) * D;
      const long ld = item & 1 ? a.ld_v : a.ld_in;
#pragma unroll
      for (int it = 0; it < NIT; ++it) Ring::copy(mine, stage, it, src + (first + min(it * HPW + sub, m - 1)) * ld, h);      // past the last token: the last
    } else if (item < n_kv + n_q) {
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        int tok, hd;
        slot(item, j, tok, hd);
        Ring::copy(mine, stage, j, a.q_in + (first + tok) * a.ld_in + hd * D, h);
      }
    }
    copies_commit();
  };
  const int item0 = blockIdx.y * 4 + warp, step = gridDim.y * 4;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) fetch(item0 + i * step, i);
  if (a.rot) {                                                   // every head of the page's tokens turns by them
    const int pieces = a.rot / 8;                                // of 16 bytes, of a token's cosines
    for (int i = threadIdx.x; i < m * pieces; i += 128) {
      const int tok = i / pieces, e = i - tok * pieces;
      const size_t at = (size_t)table_row(a.pos ? a.pos[first + tok] : lo + tok, a.table_rows, tk.status) * pieces + e;
      cosines[tok][e] = reinterpret_cast<const float4*>(a.cos_t)[at];
      sines[tok][e] = reinterpret_cast<const float4*>(a.sin_t)[at];
    }
    __syncthreads();
  }
  int stage = ST - 1;                                            // of the item that is fetched next
  for (int item = item0; item < n_kv + n_q; item += step) {
    fetch(item + (ST - 1) * step, stage);                        // where the item before this one was
    stage = stage + 1 == ST ? 0 : stage + 1;
    copies_wait<ST - 1>();
    if (item >= n_kv) {
      // ---- heads of tokens, one behind the other ----
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        int tok, hd;
        const bool in = slot(item, j, tok, hd);
        Raw raw;
        Ring::get(mine, stage, j, raw);
        uint64_t v[8];
        raw.get(v);
        if (a.wq) head_norm<L>(v, a.wq, h, 1.f / D, a.eps);
        if (a.rot) {
          Turn turn;
          angles(turn, tok);
          turn.apply<false>(h, v);
        }
        raw.set(v);
        if (in) raw.store(a.q + (first + tok) * a.ld_q + hd * D, h);
      }
      continue;
    }
    // ---- keys or values of a head ----
    const int hk = item >> 1, which = item & 1;                  // 0 keys, 1 values
    if (!listed || (unsigned)id >= (unsigned)pool.pages) {
      if (lane == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
      continue;
    }
    const long block = (long)id * pool.Hkv + hk;
    uint8_t* codes = (which ? pool.v : pool.k) + block * FP8_PAGE * D;
    float* scales = (which ? pool.v_scale : pool.k_scale) + block;
    const float old = *scales;
    auto values = [&](int it, uint64_t (&x)[8]) {
      Raw raw;
      Ring::get(mine, stage, it, raw);
      raw.get(x);
      if (which) return;
      if (a.wk) head_norm<L>(x, a.wk, h, 1.f / D, a.eps);
      if (a.rot) {
        Turn turn;
        angles(turn, min(it * HPW + sub, m - 1));
        turn.apply_apart(h, x);                                  // 2 x 8000 tokens 65.5 us either way; the queries too 16 x 500 with norms 53.3 -> 54.4
      }
    };
    uint32_t amax = 0;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      if (it * HPW >= m) break;
      uint64_t x[8];
      values(it, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = max(amax, max((uint32_t)x[e] & 0x7fffffffu, (uint32_t)(x[e] >> 32) & 0x7fffffffu));
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    float scale = scale_of_bits(amax);
    const int slot0 = lo % FP8_PAGE;
    __syncwarp();
    if (slot0 > 0) {                                             // earlier tokens of the sequence are in the page
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
      if (it * HPW >= m) break;
      uint64_t x[8];
      values(it, x);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 lo2 = of_pair(mul_pair(x[2 * e], pair_of(inv, inv))), hi2 = of_pair(mul_pair(x[2 * e + 1], pair_of(inv, inv)));
        w[e] = number ? e4m3x2(lo2.x, lo2.y) | (e4m3x2(hi2.x, hi2.y) << 16) : 0u;
      }
      if (it * HPW + sub < m) {
        uint8_t* dst = codes + (slot0 + it * HPW + sub) * D;
        *reinterpret_cast<uint2*>(dst + h.e0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(dst + h.e1) = make_uint2(w[2], w[3]);
      }
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
  uint32_t inv_tiles, inv_splits, inv_hkv, inv_g;     // div_reciprocal
  float *part, *part_ref;  // splits > 1: [T, H, splits, D] values; [T, H, splits, 3] ref, lift and the row sum
  int* used;            // splits > 1: [T, H] splits that a row has
  // Rows of a token tree (or null): row t is of table row row_seq[t], which holds seq_lens[.] tokens, and sees those below tail_start[t] and of the 64
  // from there on the ones whose bit is set.
  const int *row_seq, *seq_lens, *tail_start;
  const unsigned long long* tail_mask;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2 of a page's scale, a power of two from 2^-64 on (0, of a page never written, counts as that: its codes are 0); NaN stays.
__device__ __forceinline__ float log2_scale(float s) { return s == s ? (float)max((int)((__float_as_uint(s) >> 23) & 255) - 127, -64) : s; }
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// What a row sums, s being its scores in powers of two: 2^(s - ref), and values weighed with 2^(s - ref + log2 of their page's scale + lift), which is the
// product's fp16 operand. ref is such that the largest of these that the row has seen lies between 2^TOP and, SLACK lower, 2^6 (and is raised only when they
// leave that): what is rounded away of a weight is under 2^-30 of the row's largest weight times scale, whatever pages of large values weigh little or are
// not seen at all. With LIFT a term of the row sum is then between 2^-106 and 2^102 where it is the largest, so that fp32 holds it for scales of 2^-64 to 2^120.
// Differences of scores come first and are added to afterwards, so that both exponents are off by the same where scores are large.
constexpr float TOP = 14.f, SLACK = 8.f, LIFT = -24.f;
// A score of FAR and more leaves a float no room for the scale beside it. Such rows (far) have the largest score for ref, raised at every step, and a lift of
// their own for the scale. The tiles have no such rows: they report scores of twice that, where a weight may leave fp16.
constexpr float FAR = 4194304.f;
__device__ __forceinline__ bool is_far(float score) { return fabsf(score) > FAR && score > -INFINITY; }
// Partial sums meet at the largest ref and at the lift that the one with the largest weights has there. Their factors; 1 where none has seen a key.
__device__ __forceinline__ float lift_there(float ref, float lift, float to_ref) { return lift - (ref - to_ref); }
__device__ __forceinline__ float sum_factor(float ref, float to_ref) { return to_ref == -INFINITY ? 1.f : exp2_fast(ref - to_ref); }
__device__ __forceinline__ float values_factor(float ref, float lift, float to_ref, float to_lift) {
  return to_ref == -INFINITY ? 1.f : exp2_fast((ref - to_ref) + (to_lift - lift));
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

// In front of code that is to stay behind its branch: selects in its place would be paid for by every page.
__device__ __forceinline__ void rarely() { asm volatile(""); }

// The transpose of an 8 x 8 matrix of 16-bit values over the warp: a lane's pair of row lane / 4 becomes one of column lane / 4.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// Where the codes of a page lie in a warp's ring, and which of them a lane takes. A page's keys (and values) are lines of 128 bytes whose 16-byte pieces
// are exchanged by the line's number, so that the eight lanes of a read meet all banks. n = lane / 4, c = lane % 4. Row n
// and n + 8 of a score product are the tokens slot(0, n) and slot(1, n); a lane's values are those of the tokens of rows 2 c, 2 c + 1 and those + 8, from
// dimension col(n) on.
template <int D>
struct PageMap {
  static constexpr int KP = D / 64, VW = D / 32, BYTES = 2 * FP8_PAGE * D;
  static __device__ __forceinline__ int at(int byte) {                            // of 16 * D, a multiple of 8
    const int line = byte >> 7;
    return (line << 7) + ((((byte >> 4) ^ line) & 7) << 4) + (byte & 15);
  }
  static __device__ __forceinline__ int slot(int j, int n) { return D == 128 ? (n >> 1) + 4 * (n & 1) + 8 * j : n + 8 * j; }
  static __device__ __forceinline__ int col(int n) { return D == 128 ? ((n >> 1) + 4 * (n & 1)) * 16 : n * 8; }
};

// ST slots of two pages a warp.
template <int D, int NW, int ST>
constexpr int fp8_attend_smem() { return NW * ST * 2 * PageMap<D>::BYTES; }

// 8 NR rows (query tokens times the heads that share a key head) against a run of pages: grid = sequences x key heads x splits x row tiles. Four warps take
// two pages at a time in turn, each with a softmax of its own, and join at the end.
//
// Scores (keys times queries) and outputs (values times weights) are products on m16n8k16 tensor instructions in fp16, with the codes as the operand of 16
// rows, so that eight query rows fill the other one. A code is exact in fp16, and so is a query up to 2^-24 of its row's largest value once the row is
// scaled by a power of two. Which dimension or token an index of a product means is free as long as both operands agree, so a lane's 16-byte pieces of a
// key are its operands as they lie; the weights turn into the other product's operand by an 8 x 8 transpose. Scales of keys multiply the scores, scales of
// values are added to the exponent of the weights. Every score has two exponentials, one for the sum.
//
// Bound by memory where there are enough pages, by a warp's own chain of instructions where there are few. A warp keeps its next pages on their way through
// a ring of its own in shared memory, without registers and without a barrier of the CTA. Bulk copies in their place cost their issuing thread over a
// hundred cycles each: 8 contexts of up to 65000 tokens, 8 key heads of 128, took 99.7 us with each warp's first lane issuing them, 111 with a fifth warp.
// All shared memory is in the ring: three CTAs then fit the setting of 196 KB, and with 128 bytes more each take the next one from the first-level cache
// (the same 8 contexts 74 and 76.5 us).
template <int D, int NR, int NW, bool TREE, int ST>
__global__ void __launch_bounds__(NW * 32, (NR == 1 ? 12 : 8) / NW) fp8_attend_kernel(const __grid_constant__ Fp8Attend a,
                                                                                      const __grid_constant__ Fp8Pool pool,
                                                                                      const __grid_constant__ Fp8Tokens tk) {
  using M = PageMap<D>;
  constexpr int KS = D / 16, NI = D / 16, KP = M::KP, VW = M::VW, ROWS = 8 * NR, SLOT = 2 * M::BYTES;
  extern __shared__ __align__(128) uint8_t ring[];    // NW x ST slots; then the sums
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  int x = div_by(blockIdx.x, a.tiles, a.inv_tiles);
  const int tile = blockIdx.x - x * a.tiles, y = div_by(x, a.splits, a.inv_splits), split = x - y * a.splits;
  const int seq = div_by(y, pool.Hkv, a.inv_hkv), hk = y - seq * pool.Hkv;
  wait_previous();
  release_next();
  // rows r of the tile: token r / G, head r % G of the key head's
  int t0, row, rows, start = 0, len = 0, tail = 0;
  unsigned long long bits = 0;
  bool fine = true;
  if (TREE) {
    t0 = seq;
    row = a.row_seq[seq];
    rows = a.G;
    fine = (unsigned)row < (unsigned)tk.table_rows;
    if (fine) {
      len = a.seq_lens[row];
      fine = len <= tk.max_pages * (long)FP8_PAGE;
      if (!fine) len = 0;
      tail = a.tail_start ? a.tail_start[seq] : len;
      bits = a.tail_mask ? a.tail_mask[seq] : 0;
    }
  } else {
    const Fp8Span span(tk, seq);
    t0 = span.t0;
    start = span.start;
    row = tk.rows[seq];
    fine = span.fine;
    rows = fine ? span.count * a.G : 0;
    if (rows > ROWS * a.tiles) fine = false;         // more new tokens than the caller said
  }
  if (!fine && threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
  const int r0 = tile * ROWS, nr = min(ROWS, rows - r0);
  if (nr <= 0) return;
  const int first = start + div_by(r0, a.G, a.inv_g), last = start + div_by(r0 + nr - 1, a.G, a.inv_g);       // positions of the tile's tokens
  const int hi = TREE ? len : last + 1, lo = !TREE && a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int pg_lo = lo / FP8_PAGE, pg_hi = (hi + FP8_PAGE - 1) / FP8_PAGE;
  const int p0 = pg_lo + split * a.per_split, p1 = split + 1 < a.splits ? min(pg_hi, p0 + a.per_split) : pg_hi;    // the last one takes the rest
  if (split > 0 && p0 >= p1) return;

  // ---- the warp's pages: its step s takes p0 + 2 (warp + NW s) and the next ----
  // A lane keeps the number of a page of sixteen steps: `nf` of those that are fetched, ST - 1 steps ahead of `nc` with the scales of those that are worked
  // on; the next sixteen steps' are looked up in between, so that neither look-up is waited for.
  const int steps = max(0, ((p1 - p0 + 1) / 2 - warp + NW - 1) / NW);
  auto number_of = [&](int s) {                       // of step s + lane / 2
    const int pg = p0 + 2 * (warp + NW * (s + (lane >> 1))) + (lane & 1);
    return pg < p1 ? pool_page(tk, pool.pages, row, pg) : -1;
  };
  auto scale_at = [&](const float* scales, int id) { return id >= 0 ? scales[(long)id * pool.Hkv + hk] : 0.f; };
  const uint32_t slots = smem_u32(ring) + warp * ST * SLOT;
  const uint32_t even = M::at(lane * 16), odd = M::at((32 + lane) * 16) - 512;        // where a lane's piece of 512 bytes goes
  int nf = number_of(0), nn = -1;
  uint4 qraw[NR][KP][2];                              // the queries arrive with the pages' numbers
#pragma unroll
  for (int b = 0; b < NR; ++b) {
    const int r = r0 + min(b * 8 + n, nr - 1), tok = div_by(r, a.G, a.inv_g);             // rows past the tile's repeat its last
    const __nv_bfloat16* src = a.q + (t0 + tok) * a.ld_q + (hk * a.G + r - tok * a.G) * D + c * 16;
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) qraw[b][j][i] = *reinterpret_cast<const uint4*>(src + j * 64 + i * 8);
  }
  auto fetch = [&](int s) {                           // the pages of step s into their slot
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int id = __shfl_sync(0xffffffffu, nf, (2 * s + g) & 31);
      if (s < steps && id >= 0) {
        const long base = ((long)id * pool.Hkv + hk) * (FP8_PAGE * D) + lane * 16;
        const uint8_t *ksrc = pool.k + base, *vsrc = pool.v + base;
        const uint32_t dst = slots + (s % ST) * SLOT + g * M::BYTES;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          copy16_async(dst + q * 512 + (q & 1 ? odd : even), ksrc + q * 512);
          copy16_async(dst + FP8_PAGE * D + q * 512 + (q & 1 ? odd : even), vsrc + q * 512);
        }
      }
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) fetch(s);
  int nc = nf;
  float ksc = scale_at(pool.k_scale, nc), vsc = log2_scale(scale_at(pool.v_scale, nc)), ksn = 0.f, vsn = 0.f;

  // ---- queries: row n of a block of eight, as the second operand ----
  uint32_t qb[NR][KS][2];
  float qm[NR][2];                                                            // of this lane's columns: rows 2 c and 2 c + 1
  int vlo[NR][2], vhi[NR][2];                                                 // positions that they see: [vlo, vhi)
#pragma unroll
  for (int b = 0; b < NR; ++b) {
    uint4(&raw)[KP][2] = qraw[b];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {raw[j][i].x, raw[j][i].y, raw[j][i].z, raw[j][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = min(max((int)(top >> 7), 1), 253);                         // 2^(ex - 127): the row's largest value, but for its fraction
    const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)ex << 23);
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 v = raw[j][i >> 1];
        const uint32_t w0 = i & 1 ? v.z : v.x, w1 = i & 1 ? v.w : v.y;
        qb[b][j * 4 + i][0] = half2_of(__uint_as_float(w0 << 16) * down, __uint_as_float(w0 & 0xffff0000u) * down);
        qb[b][j * 4 + i][1] = half2_of(__uint_as_float(w1 << 16) * down, __uint_as_float(w1 & 0xffff0000u) * down);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      qm[b][e] = __shfl_sync(0xffffffffu, up, (2 * c + e) * 4);
      const int p = start + div_by(min(r0 + b * 8 + 2 * c + e, rows - 1), a.G, a.inv_g);
      vhi[b][e] = TREE ? len : p + 1;
      vlo[b][e] = !TREE && a.window > 0 ? p - a.window + 1 : 0;
    }
  }
  const int all_lo = !TREE && a.window > 0 ? last - a.window + 1 : 0, all_hi = TREE ? min(tail, len) : first + 1;  // positions that every row sees

  float o[NR][NI][4], l[NR][2], ref[NR][2], lift[NR][2];
  bool far = false;                                   // any of the warp's rows
#pragma unroll
  for (int b = 0; b < NR; ++b) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[b][i][e] = 0.f;
    ref[b][0] = ref[b][1] = -INFINITY;
    l[b][0] = l[b][1] = 0.f;
    lift[b][0] = lift[b][1] = LIFT;
  }

  for (int st = 0; st < steps; ++st) {
    if ((st & 15) == 0) {
      if (st > 0) {
        nc = nf;
        ksc = ksn;
        vsc = log2_scale(vsn);
      }
      nn = number_of(st + 16);
    }
    if ((st & 15) == 8) {
      ksn = scale_at(pool.k_scale, nn);
      vsn = scale_at(pool.v_scale, nn);
    }
    if (((st + ST - 1) & 15) == 0) nf = nn;
    const int at0 = (2 * st) & 31, there = (__ballot_sync(0xffffffffu, nc >= 0) >> at0) & 3, pos = (p0 + 2 * (warp + NW * st)) * FP8_PAGE;
    const float ks[2] = {__shfl_sync(0xffffffffu, ksc, at0), __shfl_sync(0xffffffffu, ksc, at0 + 1)};
    const float vs[2] = {__shfl_sync(0xffffffffu, vsc, at0), __shfl_sync(0xffffffffu, vsc, at0 + 1)};      // log2
    fetch(st + ST - 1);                              // into the slot of step st - 1, which every lane has read
    copies_wait<ST - 1>();
    __syncwarp();
    const uint32_t pages = slots + (st % ST) * SLOT;
    // ---- scores: 2 x 16 tokens x 8 rows ----
    float s[NR][2][4];
#pragma unroll
    for (int b = 0; b < NR; ++b)
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[b][g][e] = 0.f;
#pragma unroll
    for (int q = 0; q < KP; ++q) {
      uint32_t xs[2][4], ys[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint4 x4 = shared16(pages + g * M::BYTES + M::at(M::slot(0, n) * D + q * 64 + c * 16));
        const uint4 y4 = shared16(pages + g * M::BYTES + M::at(M::slot(1, n) * D + q * 64 + c * 16));
        xs[g][0] = x4.x; xs[g][1] = x4.y; xs[g][2] = x4.z; xs[g][3] = x4.w;
        ys[g][0] = y4.x; ys[g][1] = y4.y; ys[g][2] = y4.z; ys[g][3] = y4.w;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t k0 = half2_of_e4m3x2(xs[g][k]), k1 = half2_of_e4m3x2(ys[g][k]), k2 = half2_of_e4m3x2(xs[g][k] >> 16),
                         k3 = half2_of_e4m3x2(ys[g][k] >> 16);
#pragma unroll
          for (int b = 0; b < NR; ++b) mma_f16(s[b][g], k0, k1, k2, k3, qb[b][q * 4 + k][0], qb[b][q * 4 + k][1]);
        }
    }
    const bool whole = pos >= all_lo && pos + 2 * FP8_PAGE <= all_hi && there == 3;
    bool over = far;
#pragma unroll
    for (int b = 0; b < NR; ++b)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float f0 = qm[b][0] * ks[g], f1 = qm[b][1] * ks[g];
        s[b][g][0] *= f0;
        s[b][g][1] *= f1;
        s[b][g][2] *= f0;
        s[b][g][3] *= f1;
      }
    uint32_t hidden = 0;
    if (!whole) {
      rarely();
#pragma unroll
      for (int b = 0; b < NR; ++b)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = pos + g * FP8_PAGE + M::slot(e >> 1, n);
            bool seen = at >= vlo[b][e & 1] && at < vhi[b][e & 1] && ((there >> g) & 1);
            if (TREE) seen = seen && (at < tail || ((unsigned)(at - tail) < 64u && ((bits >> ((at - tail) & 63)) & 1ull)));
            if (!seen) {
              s[b][g][e] = -INFINITY;
              hidden |= 1u << (b * 8 + g * 4 + e);
            }
          }
    }
    float w[NR][2][4], up[NR][2][2];                 // scores over ref, then what the values are weighed with; a page's share in its exponent
    auto relate = [&](int b) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[b][g][e] = s[b][g][e] - ref[b][e & 1];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) up[b][g][e] = vs[g] + lift[b][e];
    };
#pragma unroll
    for (int b = 0; b < NR; ++b) {
      relate(b);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        over |= fmaxf(fmaxf(w[b][0][e], w[b][0][2 + e]) + up[b][0][e], fmaxf(w[b][1][e], w[b][1][2 + e]) + up[b][1][e]) > TOP;
    }
    if (__any_sync(0xffffffffu, over)) {
      auto highest = [&](int b, int e, float from) {             // of the row's scores over `from` with their page's scale
        float x = fmaxf(fmaxf(s[b][0][e], s[b][0][2 + e]) - from + vs[0], fmaxf(s[b][1][e], s[b][1][2 + e]) - from + vs[1]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
        return x;
      };
      float now[NR][2], alpha[NR][2];
#pragma unroll
      for (int b = 0; b < NR; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          now[b][e] = fmaxf(ref[b][e], highest(b, e, 0.f) + (SLACK - TOP + LIFT));
          alpha[b][e] = now[b][e] == ref[b][e] ? 1.f : exp2_fast(ref[b][e] - now[b][e]);
          far |= is_far(now[b][e]);
        }
      if (__any_sync(0xffffffffu, far)) {
        rarely();
        far = false;
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(fmaxf(s[b][0][e], s[b][0][2 + e]), fmaxf(s[b][1][e], s[b][1][2 + e]));
#pragma unroll
            for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top = fmaxf(ref[b][e], top);
            const float most = highest(b, e, is_far(top) ? top : 0.f), was = ref[b][e], raised = is_far(top) ? top : now[b][e];
            const float lifted = is_far(top) ? fminf(TOP - SLACK - most, lift_there(was, lift[b][e], raised)) : LIFT;
            const float step = was == raised ? 0.f : was - raised;
            l[b][e] *= exp2_fast(step);
            alpha[b][e] = exp2_fast(step + (lifted - lift[b][e]));
            ref[b][e] = raised;
            lift[b][e] = lifted;
            far |= is_far(top);
          }
        far = __any_sync(0xffffffffu, far);
      } else {
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[b][e] *= alpha[b][e];
            ref[b][e] = now[b][e];
          }
      }
#pragma unroll
      for (int b = 0; b < NR; ++b) {
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[b][k][e] *= alpha[b][e & 1];
        relate(b);
      }
    }
#pragma unroll
    for (int b = 0; b < NR; ++b)
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[b][g][e] = exp2_fast(w[b][g][e]);
          w[b][g][e] = exp2_fast(w[b][g][e] + up[b][g][e & 1]);
        }
    if (!whole) {                                    // nothing of a hidden place, whatever its scale and however little the row has seen
      rarely();
#pragma unroll
      for (int b = 0; b < NR; ++b)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((hidden >> (b * 8 + g * 4 + e)) & 1) s[b][g][e] = w[b][g][e] = 0.f;
    }
    uint32_t pb[NR][2][2];                           // weights of row n: tokens of rows 2 c, 2 c + 1 (and + 8) of the score product
#pragma unroll
    for (int b = 0; b < NR; ++b) {
      l[b][0] += (s[b][0][0] + s[b][0][2]) + (s[b][1][0] + s[b][1][2]);
      l[b][1] += (s[b][0][1] + s[b][0][3]) + (s[b][1][1] + s[b][1][3]);
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int h = 0; h < 2; ++h) pb[b][g][h] = transpose8(half2_of(w[b][g][2 * h], w[b][g][2 * h + 1]));
    }
    // ---- values: dimensions x 8 rows ----
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t v[4][VW];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = M::slot(r >> 1, 2 * c + (r & 1));
        const uint32_t src = pages + g * M::BYTES + FP8_PAGE * D + M::at(tok * D + M::col(n));
        if (D == 128) {
          const uint4 w = shared16(src);
          v[r][0] = w.x; v[r][1] = w.y; v[r][VW - 2] = w.z; v[r][VW - 1] = w.w;
        } else {
          const uint2 w = shared8(src);
          v[r][0] = w.x; v[r][1] = w.y;
        }
      }
      if (!whole) {                                   // slots past the end hold whatever was there
        rarely();
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (pos + g * FP8_PAGE + M::slot(r >> 1, 2 * c + (r & 1)) >= hi || !((there >> g) & 1)) {
#pragma unroll
            for (int q = 0; q < VW; ++q) v[r][q] = 0;
          }
      }
#pragma unroll
      for (int q = 0; q < VW; ++q) {                  // four dimensions of the lane: two products, rows n and n + 8 one dimension each
        const uint32_t a01 = __byte_perm(v[0][q], v[1][q], 0x5140), b01 = __byte_perm(v[0][q], v[1][q], 0x7362);
        const uint32_t a23 = __byte_perm(v[2][q], v[3][q], 0x5140), b23 = __byte_perm(v[2][q], v[3][q], 0x7362);
        const uint32_t va[4] = {half2_of_e4m3x2(a01), half2_of_e4m3x2(a01 >> 16), half2_of_e4m3x2(a23), half2_of_e4m3x2(a23 >> 16)};
        const uint32_t vb[4] = {half2_of_e4m3x2(b01), half2_of_e4m3x2(b01 >> 16), half2_of_e4m3x2(b23), half2_of_e4m3x2(b23 >> 16)};
#pragma unroll
        for (int b = 0; b < NR; ++b) {
          mma_f16(o[b][2 * q], va[0], va[1], va[2], va[3], pb[b][g][0], pb[b][g][1]);
          mma_f16(o[b][2 * q + 1], vb[0], vb[1], vb[2], vb[3], pb[b][g][0], pb[b][g][1]);
        }
      }
    }
    __syncwarp();
  }

  // ---- the warps' shares, each in its own part of the ring ----
  constexpr int SHARE = ST * SLOT / 4;               // floats of a warp's part: ROWS x D sums, behind them a row's ref, sum and lift
  static_assert(ROWS * (D + 3) <= SHARE, "sums fit the ring");
  float* sums = reinterpret_cast<float*>(ring);
  auto of_row = [&](int w, int what, int r) -> float& { return sums[w * SHARE + ROWS * (D + what) + r]; };
#pragma unroll
  for (int b = 0; b < NR; ++b)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], d);
      const int r = b * 8 + 2 * c + e;
      if (n == 0) {
        of_row(warp, 0, r) = ref[b][e];
        of_row(warp, 2, r) = lift[b][e];
        of_row(warp, 1, r) = l[b][e];
      }
      if (r < nr) {
        float* to = sums + warp * SHARE + r * D + M::col(n);
#pragma unroll
        for (int k = 0; k < NI; k += 2)
          *reinterpret_cast<float4*>(to + 2 * k) = make_float4(o[b][k][e], o[b][k][2 + e], o[b][k + 1][e], o[b][k + 1][2 + e]);
      }
    }
  const bool cta_far = __syncthreads_or(far);
  for (int i = threadIdx.x; i < nr * (D / 4); i += NW * 32) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float rr = of_row(0, 0, r);
#pragma unroll
    for (int w = 1; w < NW; ++w) rr = fmaxf(rr, of_row(w, 0, r));
    float to_lift = LIFT, acc[4] = {0.f, 0.f, 0.f, 0.f}, ll = 0.f;
    auto add = [&](int w, float f, float fv) {
      const float4 v = *reinterpret_cast<const float4*>(sums + w * SHARE + r * D + d);
      acc[0] += v.x * fv; acc[1] += v.y * fv; acc[2] += v.z * fv; acc[3] += v.w * fv;
      ll += of_row(w, 1, r) * f;
    };
    if (cta_far) {
      rarely();
      to_lift = INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) to_lift = fminf(to_lift, lift_there(of_row(w, 0, r), of_row(w, 2, r), rr));
#pragma unroll
      for (int w = 0; w < NW; ++w) add(w, sum_factor(of_row(w, 0, r), rr), values_factor(of_row(w, 0, r), of_row(w, 2, r), rr, to_lift));
    } else {
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = sum_factor(of_row(w, 0, r), rr);
        add(w, f, f);
      }
    }
    const int tok = div_by(r0 + r, a.G, a.inv_g), t = t0 + tok, hd = hk * a.G + r0 + r - tok * a.G;
    if (a.splits == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll, drop = cta_far ? exp2_fast(-to_lift) : exp2_fast(-LIFT);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = acc[i] * inv * drop;                      // inv first: the values' own scale is in the other one
      *reinterpret_cast<uint2*>(a.out + t * a.ld_o + hd * D + d) = make_uint2(cvt_bf16x2(acc[0], acc[1]), cvt_bf16x2(acc[2], acc[3]));
      continue;
    }
    const long at = ((long)t * a.H + hd) * a.splits + split;
    *reinterpret_cast<float4*>(a.part + at * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (d == 0) {
      a.part_ref[3 * at] = rr;
      a.part_ref[3 * at + 1] = to_lift;
      a.part_ref[3 * at + 2] = ll;
      if (split == 0) a.used[(long)t * a.H + hd] = max(1, min(a.splits, (pg_hi - pg_lo + a.per_split - 1) / a.per_split));
    }
  }
}

// ---------------------------------------------------------------------------------------------- attention of many rows
__host__ __device__ constexpr uint32_t make_idesc_f16(uint32_t M, uint32_t N, uint32_t b_mn_major) {
  return (1u << 4) | (b_mn_major << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);        // fp32 sums of fp16 operands
}

// One product step or commit of a converged warp: the thread is chosen inside, under a predicate, so that operands stay in uniform registers (a branch to
// one lane around them made each step cost about ninety cycles of its warp).
__device__ __forceinline__ void mma_of_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred one, add;\n"
      "elect.sync _|one, 0xffffffff;\n"
      "setp.ne.u32 add, %4, 0;\n"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, add;\n"
      "}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_of_warp_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred one, add;\n"
      "elect.sync _|one, 0xffffffff;\n"
      "setp.ne.u32 add, %4, 0;\n"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, add;\n"
      "}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_of_warp(uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred one;\n"
      "elect.sync _|one, 0xffffffff;\n"
      "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n"
      ::"r"(smem_u32(bar))
      : "memory");
}

constexpr int FT_M = 128, FT_N = 64, FT_PAGES = FT_N / FP8_PAGE, FT_ROWS = 2 * FT_M;
constexpr int FT_THREADS = 512;        // two groups of four warps for the softmax of a tile each, one that converts, one whose first warp issues the products
constexpr int FT_SLOTS = 4;            // of keys and of values
template <int D>
struct FtSmem {
  static constexpr int QUERIES = FT_M * D * 2, KEYS = FT_N * D * 2;        // fp16 rows in pieces of 64 columns with the 128-byte swizzle
  static constexpr int TOTAL = 2 * QUERIES + 2 * FT_SLOTS * KEYS + 1024;
};

// 256 rows (query tokens times the heads that share a key head) as two tiles against blocks of 64 keys on the tcgen05 tensor cores: prompts behind a cache,
// and drafts of more than a few tokens. grid = row tiles (the longest first) x splits x key heads x sequences, one CTA an SM.
//   warps 0-7    softmax, a row a thread: scores from tensor memory, weights in fp16 back in their place
//   warps 8-11   codes of the next blocks from the pages to registers, as fp16 to shared memory, for both tiles
//   warps 12-13  issue a tile's S = Q K^T and O += P V (P from tensor memory)
// A tile has two places for scores: the next block's are computed under this one's softmax, so that a row's chain does not wait for products (with one, and
// blocks of 128 keys, a tile's softmax and products took turns: 548 us in two parts against 514).
// 2 x 1500 tokens on 5500, 32 heads of 128 on 8: 363 us, 847 TFLOP/s. A block takes both tiles some 2100 cycles, of which the tensor cores are busy with
// 1260 (the queries are read from shared memory again for 64 keys each) and the exponentials' unit 1024: what bounds it is a row's chain of reading scores,
// maximum, exponentials and writing weights. Two threads a row, half of a block's keys each, shorten the chain but leave the conversion half the registers:
// 412 against 363 then. With barriers for keys and values apart the conversion was what every block waited for: 418.
// Scales of keys multiply the scores of their 16 columns in the exponential's argument, scales of values are added to it and taken out of the row sum again
// a page at a time, so neither costs anything a score. The sums and their references are those of the small kernel. Tensor memory, a tile 256 columns:
// scores (then weights) at 0 and 64, O at 128.
template <int D>
__global__ void __launch_bounds__(FT_THREADS, 1) fp8_attend_tile_kernel(const __grid_constant__ Fp8Attend a, const __grid_constant__ Fp8Pool pool,
                                                                        const __grid_constant__ Fp8Tokens tk) {
  using L = FtSmem<D>;
  constexpr int CH = D / 16, NS = FT_SLOTS;          // 16-byte pieces of a token's codes
  constexpr uint32_t T_COLS = 256, O_COL = 128, COLS = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = smem + 2 * L::QUERIES, *sV = sK + NS * L::KEYS;
  // s_full and p_full: [tile][even or odd block]
  __shared__ __align__(8) uint64_t q_full[2], full[NS], empty[NS], s_full[2][2], p_full[2][2], o_full[2];
  // Of a block's pages: the keys' scale, log2 of the values'; bit p of `present`: page p is there. Block j + 8 takes block j's place once the products of
  // block j + 4 are complete.
  __shared__ float2 scales[8][FT_PAGES];
  __shared__ uint32_t present[8];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = div_by(blockIdx.x, a.tiles, a.inv_tiles);
  const int tile = a.tiles - 1 - (blockIdx.x - x * a.tiles), y = div_by(x, a.splits, a.inv_splits), split = x - y * a.splits;
  const int seq = div_by(y, pool.Hkv, a.inv_hkv), hk = y - seq * pool.Hkv;
  wait_previous();
  release_next();
  const Fp8Span span(tk, seq);
  const int t0 = span.t0, start = span.start, row = tk.rows[seq], rows = span.fine ? span.count * a.G : 0;
  if ((!span.fine || rows > FT_ROWS * a.tiles) && threadIdx.x == 0) atomicCAS(tk.status, 0, ERR_BAD_ARG);
  const int r0 = tile * FT_ROWS, nr = min(FT_ROWS, rows - r0);
  if (nr <= 0) return;
  const int first = start + div_by(r0, a.G, a.inv_g), last = start + div_by(r0 + nr - 1, a.G, a.inv_g);
  const int hi = last + 1, lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  // key blocks start at whole blocks of the sequence; per_split is a multiple of a block's pages
  const int b_lo = lo / FT_N, b_hi = (hi + FT_N - 1) / FT_N, per = a.per_split / FT_PAGES;
  const int b0 = b_lo + split * per, b1 = split + 1 < a.splits ? min(b_hi, b0 + per) : b_hi;
  if (split > 0 && b0 >= b1) return;
  const int nb = b1 - b0, tiles = nr > FT_M ? 2 : 1;

  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&o_full[i], 1);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[i][b], 2);
        mbar_init(&p_full[i][b], 4);
      }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 4);
      mbar_init(&empty[i], tiles);
    }
    abort_word = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(&tmem_slot, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp >= 12) {
    // ---------------- products of tile t. A wait that is over costs its warp some 150 cycles all the same, so each tile has a warp to itself ----------------
    const int t = warp - 12;
    if (t < tiles) {
      constexpr uint32_t idesc_qk = make_idesc_f16(FT_M, FT_N, 0), idesc_pv = make_idesc_f16(FT_M, D, 1);
      const uint64_t desc_q = make_smem_desc(smem_u32(sQ) + t * L::QUERIES, 16, 1024, 2), desc_k = make_smem_desc(smem_u32(sK), 16, 1024, 2),
                     desc_v = make_smem_desc(smem_u32(sV), FT_N * 128, 1024, 2);               // steps of a product add to the address field
      const uint32_t t_s = tmem + t * T_COLS, t_o = t_s + O_COL;
      // scores of block j in the place of the weights of block j - 2, whose product is complete
      auto scores = [&](int j) -> bool {
        const int slot = j % NS;
        if (j > 1 && !mbar_wait_warp(&o_full[t], j & 1, abort_flag, tk.status, ERR_WAIT_TMEM_FULL)) return false;
        tc_fence_after();
        const uint64_t dk = desc_k + (uint64_t)(slot * L::KEYS >> 4);
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          mma_of_warp(t_s + (j & 1) * FT_N, desc_q + (((s / 4) * (FT_M * 128) + (s % 4) * 32) >> 4), dk + (((s / 4) * (FT_N * 128) + (s % 4) * 32) >> 4),
                      idesc_qk, s > 0);
        commit_of_warp(&s_full[t][j & 1]);
        if (lane == 0) mbar_arrive(&s_full[t][j & 1]);         // with it goes on what came with the keys: the block's scales
        __syncwarp();
        return true;
      };
      auto loaded = [&](int j) { return mbar_wait_warp(&full[j % NS], (j / NS) & 1, abort_flag, tk.status, ERR_WAIT_FULL); };
      auto values = [&](int j) -> bool {
        const int slot = j % NS;
        if (j + 2 < nb && !loaded(j + 2)) return false;                          // while the weights are not there yet
        if (!mbar_wait_warp(&p_full[t][j & 1], (j >> 1) & 1, abort_flag, tk.status, ERR_WAIT_MISC)) return false;
        tc_fence_after();
        const uint64_t dv = desc_v + (uint64_t)(slot * L::KEYS >> 4);
#pragma unroll
        for (int s = 0; s < FT_N / 16; ++s)          // 16 keys: eight packed columns of weights
          mma_of_warp_tmem(t_o, t_s + (j & 1) * FT_N + s * 8, dv + (s * 2048 >> 4), idesc_pv, (j > 0 || s > 0) ? 1u : 0u);
        commit_of_warp(&o_full[t]);
        commit_of_warp(&empty[slot]);
        return true;
      };
      bool ok = mbar_wait_warp(&q_full[t], 0, abort_flag, tk.status, ERR_WAIT_FULL) && loaded(0) && scores(0) && (nb == 1 || (loaded(1) && scores(1)));
      for (int j = 0; ok && j < nb; ++j) ok = values(j) && (j + 2 >= nb || scores(j + 2));
    }
  } else if (warp >= 8) {
    // ---------------- conversion: a thread takes the same piece of every sixteenth (D = 64: thirty-second) token ----------------
    const int tid = threadIdx.x - 256;
    constexpr int PER = FT_N * CH / 128, STEP = 128 / CH;      // pieces of a thread in a block; tokens from one to the next
    const int piece = tid % CH, tok0 = tid / CH, pages_lo = lo / FP8_PAGE, pages_hi = (hi + FP8_PAGE - 1) / FP8_PAGE;
    uint4 rk[2][PER], rv[2][PER];                    // of even and odd blocks, two ahead
    // Lanes 0 to 3 look a block's pages up: read three blocks ahead, checked two ahead and codes and scales read then, so that nothing is waited for. Loads
    // stand outside of branches, from a place that exists where there is none to read: behind a branch the compiler copies what was loaded, and so waits.
    const bool known = (unsigned)row < (unsigned)tk.table_rows;
    const int* list = tk.page_table + (known ? (long)row * tk.max_pages : 0);
    auto read_id = [&](int j) { return list[min((b0 + j) * FT_PAGES + lane, tk.max_pages - 1)]; };
    auto check_id = [&](int id, int j) {
      const int pg = (b0 + j) * FT_PAGES + lane;
      if (lane >= FT_PAGES || j >= nb || pg < pages_lo || pg >= pages_hi) return -1;       // a block may begin in front of the window: such pages are absent
      if (known && pg < tk.max_pages && (unsigned)id < (unsigned)pool.pages) return id;
      atomicCAS(tk.status, 0, ERR_BAD_ARG);
      return -1;
    };
    auto scale_at = [&](const float* of, int id) { return of[(long)max(id, 0) * pool.Hkv + hk]; };
    // A thread's place in a page is always the same; `at`: what it reads of page 0, key head 0.
    const uint8_t *k_at = pool.k + (tok0 % FP8_PAGE) * D + piece * 16, *v_at = pool.v + (tok0 % FP8_PAGE) * D + piece * 16;
    auto load = [&](uint4 (&k)[PER], uint4 (&v)[PER], int id) {
      const int head = max(id, 0) * pool.Hkv + hk;                               // under 2^31: there are as many scales
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const size_t off = (size_t)(unsigned)__shfl_sync(0xffffffffu, head, (tok0 + i * STEP) / FP8_PAGE) * (FP8_PAGE * D);
        k[i] = *reinterpret_cast<const uint4*>(k_at + off);
        v[i] = *reinterpret_cast<const uint4*>(v_at + off);
      }
    };
    const int at = 2 * piece;                                                    // 16-byte pieces `at` and `at` + 1 of a token's fp16 row
    const bool odd = piece >= CH / 2;                                            // lanes of the second half store in the other order: no bank twice
    const int to = (at >> 3) * (FT_N * 128) + tok0 * 128;
    const int x0 = (((at & 7) + (odd ? 1 : 0)) ^ (tok0 & 7)) << 4, x1 = (((at & 7) + (odd ? 0 : 1)) ^ (tok0 & 7)) << 4;
    auto store = [&](const uint4 (&raw)[PER], uint8_t* dst) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint4 r = raw[i];
        const uint32_t a0 = odd ? r.z : r.x, a1 = odd ? r.w : r.y, b0 = odd ? r.x : r.z, b1 = odd ? r.y : r.w;
        uint8_t* row = dst + to + i * STEP * 128;                                // STEP is a multiple of eight: the swizzle stays
        *reinterpret_cast<uint4*>(row + x0) = make_uint4(half2_of_e4m3x2(a0), half2_of_e4m3x2(a0 >> 16), half2_of_e4m3x2(a1), half2_of_e4m3x2(a1 >> 16));
        *reinterpret_cast<uint4*>(row + x1) = make_uint4(half2_of_e4m3x2(b0), half2_of_e4m3x2(b0 >> 16), half2_of_e4m3x2(b1), half2_of_e4m3x2(b1 >> 16));
      }
    };
    static_assert(STEP % FP8_PAGE == 0, "a thread's tokens share their place in a page, and a swizzle");
    int id[2] = {check_id(read_id(0), 0), check_id(read_id(1), 1)}, read = read_id(2);
    float ks[2] = {scale_at(pool.k_scale, id[0]), scale_at(pool.k_scale, id[1])}, vs[2] = {scale_at(pool.v_scale, id[0]), scale_at(pool.v_scale, id[1])};
#pragma unroll
    for (int e = 0; e < 2; ++e) load(rk[e], rv[e], id[e]);
    auto block = [&](int j, int e) -> bool {
      const int slot = j % NS;
      const uint32_t there = __ballot_sync(0xffffffffu, id[e] >= 0);
      if (!mbar_wait_warp(&empty[slot], ((j / NS) & 1) ^ 1, abort_flag, tk.status, ERR_WAIT_EMPTY)) return false;
      if (warp == 8) {
        if (lane < FT_PAGES) scales[j & 7][lane] = id[e] >= 0 ? make_float2(ks[e], log2_scale(vs[e])) : make_float2(0.f, -127.f);
        if (lane == 0) present[j & 7] = there;
      }
      if ((b0 + j + 1) * FT_N > hi || there != (1u << FT_PAGES) - 1) {           // values that are not there are nothing, whatever was read
        rarely();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int tok = tok0 + i * STEP;
          if ((b0 + j) * FT_N + tok >= hi || !((there >> (tok / FP8_PAGE)) & 1)) rv[e][i] = make_uint4(0, 0, 0, 0);
        }
      }
      store(rk[e], sK + slot * L::KEYS);
      store(rv[e], sV + slot * L::KEYS);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[slot]);
      id[e] = check_id(read, j + 2);
      read = read_id(j + 3);
      load(rk[e], rv[e], id[e]);
      ks[e] = scale_at(pool.k_scale, id[e]);
      vs[e] = scale_at(pool.v_scale, id[e]);
      return true;
    };
    for (int j = 0; j < nb; j += 2)
      if (!block(j, 0) || (j + 1 < nb && !block(j + 1, 1))) break;
  } else {
    // ---------------- softmax: thread <-> row r of tile t ----------------
    const int t = warp >> 2, r = threadIdx.x & 127, rt = t * FT_M + r, rr = r0 + min(rt, nr - 1), tok = div_by(rr, a.G, a.inv_g);
    const int hd = hk * a.G + rr - tok * a.G;
    const int kmax = start + tok, kmin = a.window > 0 ? kmax - a.window + 1 : 0;
    const uint32_t t_lane = tmem + (uint32_t((warp & 3) * 32) << 16), t_o = t_lane + t * T_COLS + O_COL;
    if (t < tiles) {
      float qm;
      {                                              // the row's queries, scaled by a power of two, as fp16 rows for the products
        const __nv_bfloat16* src = a.q + (t0 + tok) * a.ld_q + hd * D;
        uint4 w[D / 8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = *reinterpret_cast<const uint4*>(src + i * 8);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max(v[k] & 0x7fffu, (v[k] >> 16) & 0x7fffu));
        }
        const int ex = min(max((int)(top >> 7), 1), 253);
        const float sign = a.scale < 0.f ? -1.f : 1.f, down = sign * __uint_as_float((uint32_t)(254 - ex) << 23);
        qm = sign * a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)ex << 23);      // not negative: largest scores stay largest
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) h[k] = half2_of(__uint_as_float(v[k] << 16) * down, __uint_as_float(v[k] & 0xffff0000u) * down);
          *reinterpret_cast<uint4*>(sQ + t * L::QUERIES + (i >> 3) * (FT_M * 128) + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
      }
      const int all_lo = a.window > 0 ? last - a.window + 1 : 0, all_hi = first + 1;      // positions that every row sees
      float m = -INFINITY, l = 0.f, ref = -INFINITY;   // l: sum of 2^(s - m + TOP - SLACK); ref: the largest s + log2 of the value scale
      bool ok = true;
      for (int j = 0; j < nb; ++j) {
        if (!mbar_wait_warp(&s_full[t][j & 1], (j >> 1) & 1, abort_flag, tk.status, ERR_WAIT_TMEM_FULL)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[FT_N];
        const uint32_t t_s = t_lane + t * T_COLS + (j & 1) * FT_N;
#pragma unroll
        for (int cc = 0; cc < FT_N / 16; ++cc) tmem_ld_32x16(t_s + cc * 16, s + cc * 16);
        const float2* sc = scales[j & 7];
        const int k0 = (b0 + j) * FT_N;
        const uint32_t there = present[j & 7];
        const bool whole = k0 >= all_lo && k0 + FT_N <= all_hi && there == (1u << FT_PAGES) - 1;
        auto seen = [&](int i) { const int k = k0 + i; return k <= kmax && k >= kmin && ((there >> (i / FP8_PAGE)) & 1); };
        tmem_ld_wait();
        if (!whole) {
          rarely();
#pragma unroll
          for (int i = 0; i < FT_N; ++i)
            if (!seen(i)) s[i] = 0xff800000u;
        }
        // ---- the largest score, and the largest score and log2 of the value scale ----
        float mx = -INFINITY, rx = -INFINITY;
#pragma unroll
        for (int h = 0; h < FT_PAGES; ++h) {
          const uint32_t* u = s + h * 16;
          float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            x0 = fmax3(x0, __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
            x1 = fmax3(x1, __uint_as_float(u[i + 2]), __uint_as_float(u[i + 3]));
          }
          const float2 k = sc[h];
          const float top = fmaxf(x0, x1) * (qm * k.x);
          mx = fmaxf(mx, top);
          rx = fmaxf(rx, top + k.y);
        }
        // The last block passes here too, for the wait: the product after this one is waited for behind the loop, a barrier's parity tells a phase from its
        // neighbours only, and here it is sure that the phase before has ended and the one after has not.
        if (__any_sync(0xffffffffu, mx > m + SLACK || rx > ref + SLACK) || j == nb - 1) {
          rarely();
          const float up = j == 0 || mx > m + SLACK ? fmaxf(m, mx) : m;
          const float r_up = j == 0 || rx > ref + SLACK ? fmaxf(ref, rx) : ref;
          const float alpha = r_up == ref ? 1.f : exp2_fast(ref - r_up);
          l *= up == m ? 1.f : exp2_fast(m - up);
          m = up;
          ref = r_up;
          if (j > 0) {                                 // O is that of the blocks before, once the last one's product is complete
            if (!mbar_wait_warp(&o_full[t], (j - 1) & 1, abort_flag, tk.status, ERR_WAIT_TMEM_FULL)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const int steps = __any_sync(0xffffffffu, alpha != 1.f) ? D / 16 : 0;
#pragma unroll 1
            for (int cc = 0; cc < steps; ++cc) {
              uint32_t o[16];
              tmem_ld_32x16(t_o + cc * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x16(t_o + cc * 16, o);
            }
          }
        }
        // ---- weights: a page at a time, without a branch between pages where nothing is hidden, so that their chains overlap ----
        const float base = (TOP - SLACK) - (m == -INFINITY ? 0.f : m), shift = ref == -INFINITY ? 0.f : m - ref;
        auto weigh = [&](int h, bool masked) {
          uint32_t* u = s + h * 16;
          const float2 k = sc[h];
          // The page's value scale against the reference: 2^-60 and less leave nothing of a weight in fp16, so no less is said. Out of the sum again it is
          // taken, but for no number, which is in the weights.
          const float d = max_or_nan(k.y + shift, -60.f), f = qm * k.x, off = base + d, back = exp2_fast(fminf(60.f, -d));
          const uint64_t ff = pair_of(f, f), oo = pair_of(off, off);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 e = of_pair(fma_pair(pair_of(__uint_as_float(u[i]), __uint_as_float(u[i + 1])), ff, oo));
            u[i] = __float_as_uint(exp2_fast(e.x));
            u[i + 1] = __float_as_uint(exp2_fast(e.y));
          }
          if (masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!seen(h * 16 + i)) u[i] = 0u;
          }
          uint64_t sum0 = pair_of(__uint_as_float(u[0]), __uint_as_float(u[1])), sum1 = pair_of(__uint_as_float(u[2]), __uint_as_float(u[3]));
#pragma unroll
          for (int i = 4; i < 16; i += 4) {
            sum0 = add_pair(sum0, pair_of(__uint_as_float(u[i]), __uint_as_float(u[i + 1])));
            sum1 = add_pair(sum1, pair_of(__uint_as_float(u[i + 2]), __uint_as_float(u[i + 3])));
          }
          const float2 both = of_pair(add_pair(sum0, sum1));
          l = fmaf(both.x + both.y, back, l);
#pragma unroll
          for (int i = 0; i < 16; i += 2) s[h * 8 + i / 2] = half2_of(__uint_as_float(u[i]), __uint_as_float(u[i + 1]));
        };
        if (whole) {
#pragma unroll
          for (int h = 0; h < FT_PAGES; ++h) weigh(h, false);
        } else {
          rarely();
#pragma unroll
          for (int h = 0; h < FT_PAGES; ++h) weigh(h, true);
        }
        tmem_st_32x32(t_s, s);                         // over the scores, which are all in registers
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t][j & 1]);
      }
      if (ok) ok = mbar_wait_warp(&o_full[t], (nb - 1) & 1, abort_flag, tk.status, ERR_WAIT_TMEM_FULL);
      if (ok) {
        tc_fence_after();
        if (rt < nr && is_far(0.5f * m) && m < INFINITY) atomicCAS(tk.status, 0, ERR_BAD_ARG);
        l = l == 0.f ? 0.f : l * exp2_fast(m - ref - LIFT);                       // to the values' reference and lift
        const float inv = l == 0.f ? 0.f : 1.f / l, drop = exp2_fast(-LIFT);
        const long at = ((long)(t0 + tok) * a.H + hd) * a.splits + split;
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + cc * 32, o);
          tmem_ld_wait();
          if (rt < nr && a.splits == 1) {
            uint4* to = reinterpret_cast<uint4*>(a.out + (t0 + tok) * a.ld_o + hd * D + cc * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t h[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                h[k] = cvt_bf16x2(__uint_as_float(o[i * 8 + 2 * k]) * inv * drop, __uint_as_float(o[i * 8 + 2 * k + 1]) * inv * drop);
              to[i] = make_uint4(h[0], h[1], h[2], h[3]);
            }
          } else if (rt < nr) {
            float4* to = reinterpret_cast<float4*>(a.part + at * D + cc * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              to[i] = make_float4(__uint_as_float(o[i * 4]), __uint_as_float(o[i * 4 + 1]), __uint_as_float(o[i * 4 + 2]), __uint_as_float(o[i * 4 + 3]));
          }
          __syncwarp();
        }
        if (a.splits > 1 && rt < nr) {
          a.part_ref[3 * at] = ref;
          a.part_ref[3 * at + 1] = LIFT;
          a.part_ref[3 * at + 2] = l;
          if (split == 0) a.used[(long)(t0 + tok) * a.H + hd] = max(1, min(a.splits, (b_hi - b_lo + per - 1) / per));
        }
        tc_fence_before();
      }
    }
  }

  __syncthreads();
  if (*abort_flag) {                                 // a wait ran out: products on their way end before their memory goes
    const uint64_t since = globaltimer_ns();
    while (globaltimer_ns() - since < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

// The sequence of a row, by a warp: the last one that starts at or before it.
__device__ __forceinline__ int sequence_of(const Fp8Tokens& tk, int t, int lane) {
  int lo = 0;
  for (int len = tk.n; len > 1;) {
    const int step = (len + 31) / 32;
    const uint32_t below = __ballot_sync(0xffffffffu, lane * step < len && tk.cu[lo + lane * step] <= t);
    const int k = below ? 31 - __clz(below) : 0;
    lo += k * step;
    len = min(step, len - k * step);
  }
  return lo;
}

// Joins the splits of a row (a query token's head), D / 32 values a lane; rows that belong to no sequence stay as they are. WIDE: a CTA a row, whose warps
// share the splits; else a warp a row. With 63 splits of 32 rows a warp a row took most of 24 us.
template <int D, bool WIDE>
__global__ void __launch_bounds__(256) fp8_join_kernel(const __grid_constant__ Fp8Attend a, const __grid_constant__ Fp8Tokens tk, int tile_rows) {
  constexpr int E = D / 32, NW = WIDE ? 8 : 1;
  __shared__ float sm_l[8], sm_o[8][D];
  wait_previous();
  release_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, splits = a.splits;
  const long item = WIDE ? blockIdx.x : blockIdx.x * 8l + warp;
  if (item >= (long)tk.T * a.H) return;
  const int t = (int)(item / a.H), head = (int)(item - (long)t * a.H);
  if (!a.row_seq) {                                  // what the other kernel left out, of this row too
    const Fp8Span span(tk, sequence_of(tk, t, lane));
    if (!span.fine || t < span.t0 || t - span.t0 >= span.count || (long)(t - span.t0) * a.G + head % a.G >= (long)tile_rows * a.tiles) return;
  }
  const float* base = a.part + item * splits * D + lane * E;
  const float* ref = a.part_ref + item * splits * 3;
  const int ns = min(max(a.used[item], 0), splits);  // where a wait ran out there may be anything
  float rr = -INFINITY;
  bool far = false;
  for (int s = lane; s < ns; s += 32) {
    rr = fmaxf(rr, ref[3 * s]);
    far |= ref[3 * s + 1] != LIFT;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) rr = fmaxf(rr, __shfl_xor_sync(0xffffffffu, rr, o));
  float to_lift = LIFT;
  if (__any_sync(0xffffffffu, far)) {
    to_lift = INFINITY;
    for (int s = 0; s < ns; ++s) to_lift = fminf(to_lift, lift_there(ref[3 * s], ref[3 * s + 1], rr));
  }
  float acc[E], ll = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = WIDE ? warp : 0; s < ns; s += NW) {
    const float f = values_factor(ref[3 * s], ref[3 * s + 1], rr, to_lift);
    ll += ref[3 * s + 2] * sum_factor(ref[3 * s], rr);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] += base[(long)s * D + i] * f;
  }
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < E; ++i) sm_o[warp][lane * E + i] = acc[i];
    if (lane == 0) sm_l[warp] = ll;
    __syncthreads();
    if (warp) return;
    ll = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      ll += sm_l[w];
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] += sm_o[w][lane * E + i];
    }
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll, drop = ll == 0.f ? 0.f : exp2_fast(-to_lift);
  uint32_t* to = reinterpret_cast<uint32_t*>(a.out + t * a.ld_o + head * D + lane * E);
#pragma unroll
  for (int i = 0; i < E; i += 2) to[i / 2] = cvt_bf16x2(acc[i] * inv * drop, acc[i + 1] * inv * drop);
}

}  // namespace inv

using namespace inv;

static bool off16(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) % 16 != 0;
}

// What a call's entry is given (the Python side packs the same fields in the same order): pointers, sizes in 64 bits, numbers.
struct Fp8Where {                       // the pools, where a step's tokens belong, and where the work goes
  void *k, *v;
  float *k_scale, *v_scale;
  const int *page_table, *rows, *cu, *start;
  int* status;
  void* stream;
};
struct Fp8Sizes {
  long H, Hkv, D, pages, table_rows, max_pages, n, T;
  bool bad() const {
    constexpr long TOP = 0x7fffffff;
    return (D != 64 && D != 128) || Hkv < 1 || H < Hkv || H % Hkv || pages < 1 || n < 0 || T < 0 || table_rows < 1 || max_pages < 1 || H * D > TOP ||
           pages > TOP || table_rows > TOP || max_pages > TOP || n > TOP / 4 || T > TOP / 2;
  }
};

static Fp8Pool pool_of(const Fp8Where& w, const Fp8Sizes& s) { return {(uint8_t*)w.k, (uint8_t*)w.v, w.k_scale, w.v_scale, (int)s.pages, (int)s.Hkv}; }
static Fp8Tokens tokens_of(const Fp8Where& w, const Fp8Sizes& s) {
  return {w.rows, w.cu, w.start, w.page_table, (int)s.n, (int)s.T, (int)s.table_rows, (int)s.max_pages, w.status};
}

// q_in [T, H D], k_in, v_in [T, Hkv D] bf16 -> q [T, H D] normed and rotated, and the pools. Queries and keys have rows ld_in apart, values ld_v, q
// ld_q; H may be 0. wq, wk [D] bf16 or null; cos_t, sin_t [rope_rows, rot / 2] fp32 or null with rot 0; pos [T] or null.
struct Fp8AppendDesc {
  const void *q_in, *k_in, *v_in;
  void* q;
  const void *wq, *wk;
  const float *cos_t, *sin_t;
  const int* pos;
  Fp8Where at;
  Fp8Sizes size;
  long ld_in, ld_v, ld_q, rope_rows, rot;
  double eps;
};
extern "C" int inv_fp8_append(const Fp8AppendDesc* d) {
  const int H = (int)d->size.H, Hkv = (int)d->size.Hkv, D = (int)d->size.D, n = (int)d->size.n, T = (int)d->size.T, rot = (int)d->rot;
  Fp8Sizes s = d->size;
  if (s.H == 0) s.H = s.Hkv;
  if (s.bad() || d->rot < 0 || d->rot > D || rot % 16) return -ERR_BAD_ARG;
  if (rot && (!d->cos_t || !d->sin_t || d->rope_rows < 1 || d->rope_rows > 0x7fffffffl)) return -ERR_BAD_ARG;
  if (d->ld_in % 8 || d->ld_v % 8 || d->ld_q % 8 || off16(d->q_in, d->k_in, d->v_in, d->q) || off16(d->wq, d->wk) ||
      off16(d->cos_t, d->sin_t, d->at.k, d->at.v))
    return -ERR_BAD_ARG;
  if (n == 0 || T == 0) return 0;
  const Fp8Append a{(const __nv_bfloat16*)d->q_in, (const __nv_bfloat16*)d->k_in, (const __nv_bfloat16*)d->v_in, (const __nv_bfloat16*)d->wq,
                    (const __nv_bfloat16*)d->wk, d->cos_t, d->sin_t, d->pos, (__nv_bfloat16*)d->q, d->ld_in, d->ld_v, d->ld_q, H, rot, (int)d->rope_rows,
                    div_reciprocal(H ? H : 1), (float)d->eps};
  const Fp8Pool pool = pool_of(d->at, d->size);
  const Fp8Tokens tk = tokens_of(d->at, d->size);
  cudaStream_t st = (cudaStream_t)d->at.stream;
  const unsigned ctas = (unsigned)(T / FP8_PAGE + 2 * n);
  const int hpw = 512 / D, tokens = T / n < FP8_PAGE ? (T + n - 1) / n : FP8_PAGE;      // of an average page
  const int items = 2 * Hkv + (tokens * H + 4 * hpw - 1) / (4 * hpw);
  // An item a warp where there are few pages (128 sequences with a token each 6.1 us, six items 9.8), else six, behind one another (2 x 8000 tokens 65.5 us; two
  // items 74.6, twelve 73.1. 16 x 500 with norms 52.8, 49.8, 56.2).
  const int most = (items + 3) / 4, shares = ctas <= 296 ? most : (items + 23) / 24;
  const dim3 grid(ctas, shares < 65535 ? shares : 65535);
  if (D == 64) launch_early(fp8_append_kernel<64>, grid, 128, Fp8AppendRing::BYTES, st, a, pool, tk);
  else launch_early(fp8_append_kernel<128>, grid, 128, Fp8AppendRing::BYTES, st, a, pool, tk);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}

// Whether the kernel of 16-row tiles takes the rows of a sequence and key head, each tile reading the pages again, and not the one of 256: up to 32 rows of
// heads of 128 and 64 of 64, whose pages are half as large, and twice that while no SM has more than 64 pages to read. Small kernel and large one: 32 heads of
// 128 on 8, 16 sequences of 4000 with 8 / 12 / 16 new tokens each 59.7, 84.3, 109.7 and 69.8, 70.3, 70.5 us, 64 of 1000 66.5, 95.6, 116.2 and 86.7, 87.7, 88.2,
// four of 1000 13.3, 13.2, 13.5 and 16.4, 17.9, 18.3; 8 heads of 64 on 8, 16 of 4000 with 48 61.0 and 82.4.
static bool fp8_few_rows(long rows, int D, long units, int pages) {
  const int few = 4096 / D;
  return rows <= few || (rows <= 2 * few && (rows + 15) / 16 * units * pages <= 148 * 64);
}
// How an attention is cut: rows of a tile (8 `blocks`), warps and pages of a CTA, CTAs along a sequence.
struct Fp8Cut {
  int blocks, tiles, warps, per, splits;
  bool deep;             // one slot more a warp
  long floats(int T, int H, int D) const { return splits == 1 ? 0 : (long)T * H * (splits * (D + 3l) + 1); }      // of partial results
  Fp8Cut(int n, int Hkv, int G, int D, int max_new, int max_len, int window, bool tree) {
    const long rows = (long)max_new * G;
    const long reach = window > 0 && (long)window + max_new < max_len ? (long)window + max_new : max_len;
    blocks = rows <= 8 ? 1 : tree || fp8_few_rows(rows, D, (long)n * Hkv, (int)(reach / FP8_PAGE) + 1) ? 2 : FT_ROWS / 8;
    tiles = (int)((rows + 8 * blocks - 1) / (8 * blocks));
    const int tokens = max_new < 8 * blocks / G + 2 ? max_new : 8 * blocks / G + 2;       // of a tile
    const long span = window > 0 && (long)window + tokens < max_len ? (long)window + tokens : max_len;
    const int pages = (int)((span + (window > 0 ? 2 * FP8_PAGE - 2 : FP8_PAGE - 1)) / FP8_PAGE);       // a window may begin inside a page
    const long units = (long)n * Hkv * tiles;
    // Joining the splits costs about three microseconds, and a CTA as much before its first and behind its last page, so up to 64 pages stay together (64 x
    // 640 tokens, 512 units: 22.3 us, in two parts 25.9; 16 x 4 on 1000: 14.4 and 17.1). Longer ones are cut for two CTAs an SM, in parts of 16 pages or more
    // (2000 tokens, 16 units: 16 / 32 / 64 / 126 pages 7.5, 9.6, 12.1, 15.3 us; 32000, 8 units: 24 / 64 / 128 pages 23.5, 17.8, 19.9) and of 128 at most,
    // which evens unequal lengths out (8 of up to 65000: 128 / 192 / 512 pages 71.5, 84.6, 91.2 us; of 64999 each 165, 171, 209; 64 of 8000 164, 167). A
    // sequence alone has none to even out: its parts fill the GPU once (128000 tokens 53.3 us, in parts of 128 pages 63.3; 250000 95.1 and 101.9; with four
    // new tokens 100000 46.2 and 61.0, 200000 74.0 and 94.9; not so 300000 113.6 and 109.2). Where units alone fill the GPU several times, CTAs of two warps,
    // which are dealt out more evenly (1536 units of 63 pages: 38.3 us, four warps 43.0; 512 of 251 90.1 and 106.6).
    const bool many = blocks == 1 && units > 444 && pages <= 256;
    warps = many ? 2 : 4;
    // Four of them an SM have room for a third slot a warp (64 x 640 tokens, 512 units: 19.3 us, with three 18.2; 64 x 4000 90.3 and 86.2); more need six an
    // SM (96 x 640, 768 units: 26.6 and 33.5; 128 x 1000, 12 heads of 64, 1536 units: 38.5 and 44.6).
    deep = many && units <= 592;
    const long total = units * pages;
    long want = (total + 295) / 296;
    if (want > 128) {
      const long alone = n == 1 ? (total + (blocks == 1 ? 443 : 295)) / (blocks == 1 ? 444 : 296) : 0;
      want = alone > 128 ? alone : 128;
    }
    if (blocks == FT_ROWS / 8) {                                      // whole blocks of keys
      // One CTA an SM. A page takes a CTA about 0.25 us, all else as much as 24 pages; a join costs 10 of them and the partial results their bytes. Cut where
      // that comes out ahead (4 x 128 on 20000, 64 units: in 2 226 us, in 5 314, whole 424; 16 x 32 on 4000, 128 units: in 2 103, whole 87; 64 on 8000, 8
      // units: in 16 31, in 4 55).
      const int most = pages / (2 * FT_PAGES) < 64 ? pages / (2 * FT_PAGES) : 64;
      const double bytes = (double)n * max_new * Hkv * G * 8 * 130 / 1.2e6;
      double best = 0;
      for (int s = 1; s == 1 || s <= most; ++s) {
        const int p = ((pages + s - 1) / s + FT_PAGES - 1) / FT_PAGES * FT_PAGES, parts = (pages + p - 1) / p;
        const double cost = (double)((units * parts + 147) / 148) * (p + 24) + (s > 1 ? 10 + parts * bytes : 0);
        if (s == 1 || cost < best) {
          best = cost;
          per = p;
          splits = parts;
        }
      }
      return;
    }
    if (want < 16) want = 16;
    if (many || pages <= 64 || want > pages) want = pages;
    per = want < pages ? (int)((want + 1) & ~1l) : pages;          // warps take two
    splits = (pages + per - 1) / per;
  }
};
// Floats of workspace that an attention wants (0: none). A call's own: it holds partial results from one launch to the next.
extern "C" long inv_fp8_attend_floats(int n, int T, int H, int Hkv, int D, int max_new, int max_len, int window, int tree) {
  if (n < 1 || T < 1 || Hkv < 1 || H < Hkv || D < 1 || max_new < 1 || max_len < 1) return 0;
  const Fp8Cut cut(n, Hkv, H / Hkv, D, max_new, max_len, window, tree);
  return cut.floats(T, H, D);
}
template <int D>
static int fp8_attend_join(const Fp8Attend& a, const Fp8Tokens& tk, int tile_rows, cudaStream_t st) {
  const long items = (long)tk.T * a.H;
  if (a.splits > 4) launch_early(fp8_join_kernel<D, true>, dim3((unsigned)items), 256, 0, st, a, tk, tile_rows);
  else if (a.splits > 1) launch_early(fp8_join_kernel<D, false>, dim3((unsigned)((items + 7) / 8)), 256, 0, st, a, tk, tile_rows);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e;
}
template <int D, int NR, int NW, bool TREE, int ST = 2>
static int fp8_attend_launch(const Fp8Attend& a, const Fp8Pool& pool, const Fp8Tokens& tk, unsigned ctas, cudaStream_t st) {
  constexpr int SMEM = fp8_attend_smem<D, NW, ST>();
  static OncePerDevice ready;
  if (int rc = raise_smem(fp8_attend_kernel<D, NR, NW, TREE, ST>, SMEM, ready)) return rc;
  launch_early(fp8_attend_kernel<D, NR, NW, TREE, ST>, dim3(ctas), NW * 32, SMEM, st, a, pool, tk);
  return fp8_attend_join<D>(a, tk, 8 * NR, st);
}
template <int D>
static int fp8_attend_tile_launch(const Fp8Attend& a, const Fp8Pool& pool, const Fp8Tokens& tk, unsigned ctas, cudaStream_t st) {
  static OncePerDevice ready;
  if (int rc = raise_smem(fp8_attend_tile_kernel<D>, FtSmem<D>::TOTAL, ready)) return rc;
  launch_early(fp8_attend_tile_kernel<D>, dim3(ctas), FT_THREADS, FtSmem<D>::TOTAL, st, a, pool, tk);
  return fp8_attend_join<D>(a, tk, FT_ROWS, st);
}

static int fp8_attend(Fp8Attend a, const Fp8Pool& pool, const Fp8Tokens& tk, int D, int max_new, int max_len, float* work, long floats, cudaStream_t st) {
  a.G = a.H / pool.Hkv;
  const Fp8Cut cut(tk.n, pool.Hkv, a.G, D, max_new, max_len, a.window, a.row_seq != nullptr);
  a.tiles = cut.tiles;
  a.per_split = cut.per;
  a.splits = cut.splits;
  a.inv_tiles = div_reciprocal(a.tiles); a.inv_splits = div_reciprocal(a.splits); a.inv_hkv = div_reciprocal(pool.Hkv); a.inv_g = div_reciprocal(a.G);
  if (cut.splits > 1) {
    if (!work || off16(work) || floats < cut.floats(tk.T, a.H, D) || (long)tk.T * a.H > 0x7fffffffl) return -ERR_BAD_ARG;
    const long rows = (long)tk.T * a.H * cut.splits;
    a.part = work;
    a.part_ref = work + rows * D;
    a.used = (int*)(work + rows * (D + 3));
  }
  const long ctas = (long)tk.n * pool.Hkv * a.splits * a.tiles;
  if (ctas > 0x7fffffffl) return -ERR_BAD_ARG;
  const unsigned grid = (unsigned)ctas;
  if (cut.blocks == FT_ROWS / 8) return D == 64 ? fp8_attend_tile_launch<64>(a, pool, tk, grid, st) : fp8_attend_tile_launch<128>(a, pool, tk, grid, st);
#define INV_FP8(DD, TREE)                                                        \
  return cut.blocks == 2  ? fp8_attend_launch<DD, 2, 4, TREE>(a, pool, tk, grid, st) \
         : cut.warps == 4 ? fp8_attend_launch<DD, 1, 4, TREE>(a, pool, tk, grid, st) \
         : cut.deep       ? fp8_attend_launch<DD, 1, 2, TREE, 3>(a, pool, tk, grid, st) \
                          : fp8_attend_launch<DD, 1, 2, TREE>(a, pool, tk, grid, st)
  if (D == 64 && a.row_seq) INV_FP8(64, true);
  if (D == 64) INV_FP8(64, false);
  if (a.row_seq) INV_FP8(128, true);
  INV_FP8(128, false);
#undef INV_FP8
}

// q [T, H D] bf16, rows ld_q apart -> out [T, H D], rows ld_o apart: the token at position p of its sequence sees the cached positions up to p, with a
// window the latest `window` of them. No sequence has more than max_new new tokens or, with them, max_len tokens. work: inv_fp8_attend_floats of them.
// Rows of a token tree, where row_seq is given: row t belongs to table row row_seq[t], which holds seq_lens[row_seq[t]] tokens, and sees those below
// tail_start[t] and token tail_start[t] + i iff bit i of tail_mask[t] is set (both null: all). work: as for T sequences of one new token.
struct Fp8AttendDesc {
  const void* q;
  void* out;
  float* work;
  const int *row_seq, *seq_lens, *tail_start;
  const unsigned long long* tail_mask;
  Fp8Where at;
  Fp8Sizes size;
  long ld_q, ld_o, window, max_new, max_len, work_floats;
  double scale;
};
extern "C" int inv_fp8_attend(const Fp8AttendDesc* d) {
  constexpr long TOP = 0x7fffffff;
  if (d->size.bad() || d->window < 0 || d->max_new < 1 || d->max_len < 1 || d->max_new > TOP / 4 || d->max_len > TOP / 4) return -ERR_BAD_ARG;
  if (d->row_seq && (!d->seq_lens || !d->tail_start != !d->tail_mask || d->window || d->max_new != 1 || d->size.n != d->size.T)) return -ERR_BAD_ARG;
  if (d->ld_q % 8 || d->ld_o % 8 || off16(d->q, d->at.k, d->at.v, d->out)) return -ERR_BAD_ARG;
  if (d->size.n == 0 || d->size.T == 0) return 0;
  Fp8Attend a{};
  a.q = (const __nv_bfloat16*)d->q;
  a.out = (__nv_bfloat16*)d->out;
  a.ld_q = d->ld_q;
  a.ld_o = d->ld_o;
  a.H = (int)d->size.H;
  a.window = (int)(d->window < TOP ? d->window : TOP);
  a.scale = (float)d->scale;
  a.row_seq = d->row_seq;
  a.seq_lens = d->seq_lens;
  a.tail_start = d->tail_start;
  a.tail_mask = d->tail_mask;
  return fp8_attend(a, pool_of(d->at, d->size), tokens_of(d->at, d->size), (int)d->size.D, (int)d->max_new, (int)d->max_len, d->work,
                    d->work_floats, (cudaStream_t)d->at.stream);
}
