// Attention over the 4-bit KV cache (page layout: kv4.cuh) and the weight that it gives to every cached token.
//   out[row] = softmax(scale * q[row] K^T) V over keys first .. pos[row] of the row's sequence; rows without a key give zeros
//   mass[token] (=, +=) sum over the rows of a block and the query heads of a kv head of the softmax weight
#include <type_traits>

#include "attn_mma.cuh"
#include "kv4.cuh"

namespace {

using namespace kv4;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxUnits = 1024;      // groups of rows whose page counts a CTA keeps (streamed schedule)

struct AttnParams {
  const uint8_t* data; float* mass;
  Table t;
  const bf16* q; long ld_q;
  const int* row_seq; const int* row_pos;
  const bf16* gate; long ld_gate;
  bf16* out; long ld_o;
  float* part_o;            // [slots][pairs of a CTA][D]: sums over a part of a unit's pages, not divided
  float* part_ml;           // [slots][pairs of a CTA][2]: their softmax maximum (log2 domain) and sum
  long long* sched;         // streamed schedule: pages per CTA, then the pages before each group of rows
  float* fin;               // [M][Hq][2]: softmax maximum (log2 domain) and reciprocal sum of every row, or null
  unsigned int* status;     // device status block (bounded waits report here)
  int M, Hkv, G, window, block, add;
  int rows, groups;         // rows of a block that share a CTA, groups of them in a block
  int heads, subs;          // query heads of a kv head that share a CTA, CTAs a kv head
  int vec, vec_out;         // q rows are 8-byte aligned, output rows 4-byte
  int units, uheads;        // groups of rows in all; CTA head groups (kv heads * subs).  A unit is one of each
  int splits;               // CTAs a unit; 0: streamed
  int ctas, pairs;          // CTAs of the streamed schedule, pairs of a CTA
  int sms;
  float scale_log2;         // softmax scale * log2(e)
};

__device__ __forceinline__ int row_len(const AttnParams& p, int row) { return max(0, min(p.row_pos[row], p.t.width * kPage - 1) + 1); }
__device__ __forceinline__ int row_first(const AttnParams& p, int len) { return (p.window > 0 && len > p.window) ? len - p.window : 0; }

template <int D>
struct Ring {
  static constexpr int kStages = D == 256 ? 2 : 3;       // of two page records each
  static constexpr int kCtas = D == 256 ? 2 : 3;         // an SM: as many as the accumulators leave registers for without spills
  static constexpr int kWarpBytes = kStages * 2 * Geo<D>::kRecord + 2 * 32 * 4 * Geo<D>::kGroups;
  static constexpr int kBytes = kWarps * kWarpBytes;
};

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* src, uint32_t (&w)[N]) {
  static_assert(N == 1 || N == 2 || N % 4 == 0, "");
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(src);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + 16 * j);
      w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void load_floats(const float* src, float (&f)[N]) {
  uint32_t w[N];
  load_words<N>(reinterpret_cast<const uint8_t*>(src), w);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = __uint_as_float(w[i]);
}
template <int N>
__device__ __forceinline__ void store_floats(float* dst, const float (&f)[N]) {
  if constexpr (N == 2) {
    *reinterpret_cast<float2*>(dst) = make_float2(f[0], f[1]);
  } else {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) *reinterpret_cast<float4*>(dst + 4 * j) = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
  }
}

__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {         // 2 ulp; results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two elements of an output row: divided by the sum, gated, rounded; the row's statistics for the observed weight.
__device__ __forceinline__ void finish(const AttnParams& p, int row, int head, int d, int D, float o0, float o1, float mx, float l) {
  const float inv = l != 0.f ? 1.f / l : 0.f;
  o0 = l != 0.f ? o0 * inv : 0.f;
  o1 = l != 0.f ? o1 * inv : 0.f;
  const size_t col = (size_t)head * D + d;
  if (p.gate) {
    o0 *= sigmoid_f(__bfloat162float(p.gate[(size_t)row * p.ld_gate + col]));
    o1 *= sigmoid_f(__bfloat162float(p.gate[(size_t)row * p.ld_gate + col + 1]));
  }
  bf16* dst = p.out + (size_t)row * p.ld_o + col;
  if (p.vec_out) {
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o0, o1);
  } else {
    dst[0] = __float2bfloat16(o0);
    dst[1] = __float2bfloat16(o1);
  }
  if (p.fin && d == 0) {
    p.fin[2 * ((size_t)row * p.Hkv * p.G + head)] = mx;
    p.fin[2 * ((size_t)row * p.Hkv * p.G + head) + 1] = inv;
  }
}

// f16 x f16 -> f32, D += A B
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  attn_mma::mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
}

// Place of token n (of 8-token tile b) of an operand in its page: n = 2t and 2t + 1, the pair of a lane in the V operand, are the
// tokens t and 4 + (t ^ 1), so that neighbouring lanes read rows of different parity and the 64-byte rows of a 128-element head
// meet no bank conflict as the K operand and two-way ones as the V operand.
__device__ __forceinline__ int tok_of(int b, int n) { return 8 * b + ((n & 1) ? 4 + ((n >> 1) ^ 1) : (n >> 1)); }

// The codes of a 16-bit half word, two words at once (two tokens, or two places of a row): element i of the result holds
// nibble i of x's low half in its low half and of y's in its high half, as the fp16 number (code - 8) / 2: the nibble becomes
// the last mantissa bits of 1024 (or, four bits higher, of 1024 + 16 code), and one exact fp16 operation takes the offset away
// (halved, because a fused multiply-add with a factor of one is compiled to an addition, which takes the integer pipe's time).
// (Leaving the offset to the end, with the bare nibbles as fp16 subnormals, saves that operation and was measured to lose five
// bits of the fp32 sums: the MMA aligns a subnormal's product by its unnormalised exponent.)
// The constants come in registers whose value the compiler does not see: it would otherwise spend a second instruction on
// (p & mask) | magic for want of room for two constants in one.
struct Magic {
  uint32_t one, even, odd;
  __device__ __forceinline__ Magic() {
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(one));       // 1024
    asm volatile("mov.b32 %0, 0x38003800;" : "=r"(even));      // 1 / 2
    asm volatile("mov.b32 %0, 0x28002800;" : "=r"(odd));       // 1 / 32
  }
};
__device__ __forceinline__ uint32_t low_nibble(uint32_t p, uint32_t one) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(d) : "r"(p), "r"(one));      // (p & mask) | one
  return d;
}
__device__ __forceinline__ uint32_t high_nibble(uint32_t p, uint32_t one) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(d) : "r"(p), "r"(one));
  return d;
}
__device__ __forceinline__ void nibbles(const Magic& mg, uint32_t x, uint32_t y, bool high, uint32_t (&o)[4]) {
  const uint32_t p = attn_mma::prmt(x, y, high ? 0x7632u : 0x5410u);
  const uint32_t q = p >> 8;
  o[0] = h2_fma(low_nibble(p, mg.one), mg.even, 0xe008e008u);          // / 2 - 516
  o[1] = h2_fma(high_nibble(p, mg.one), mg.odd, 0xd080d080u);          // / 32 - 36
  o[2] = h2_fma(low_nibble(q, mg.one), mg.even, 0xe008e008u);
  o[3] = h2_fma(high_nibble(q, mg.one), mg.odd, 0xd080d080u);
}

__device__ __forceinline__ float exp2_pos(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // 2^e, -127 < e < 128

// The power of two that brings a query row whose largest magnitude has the bits ``mx`` to the top of fp16's range (exact: bf16 has
// fewer bits).  ``f``: what a product with the codes' halves has to be multiplied by (and by the group's maximum) to give the score in
// the log2 domain; positive, so that maxima stay maxima: a negative softmax scale goes into the operand.
__device__ __forceinline__ float q_scale(const AttnParams& p, uint32_t mx, float& f) {
  const int e = max((int)(mx >> 7), 14);                 // biased exponent
  const float up = e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(268 - e) << 23);   // 2^14 / 2^(e - 127)
  f = fmaxf(fabsf(p.scale_log2) * (2.f / 7.f / 16384.f) * exp2_pos(min(e - 127, 127)), 1e-37f);
  return p.scale_log2 < 0.f ? -up : up;
}

// Lane (g, t)'s part of one query row as the column operand of K Q^T (the row is pair g's): q times a power of two that fills
// fp16's range, k-step (group gi = 2 w + half, odd) made of the words w and w + NG / 2 of the lane's NG words of codes, nibbles
// odd and odd + 2.  Returns q_scale()'s factor.
template <int D>
__device__ __forceinline__ float load_q(const AttnParams& p, int row, int head, bool live, int t, uint32_t (&qb)[D / 32][2][2]) {
  constexpr int NG = D / 32;
  const unsigned short* src = reinterpret_cast<const unsigned short*>(p.q) + (size_t)row * p.ld_q + (size_t)head * D;
  uint2 raw[NG][2];
  uint32_t mx = 0;
#pragma unroll
  for (int gi = 0; gi < NG; ++gi)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const unsigned short* at = src + (t * NG + gi / 2 + y * (NG / 2)) * 8 + (gi & 1) * 4;
      if (!live) raw[gi][y] = make_uint2(0u, 0u);
      else if (p.vec) raw[gi][y] = *reinterpret_cast<const uint2*>(at);
      else raw[gi][y] = make_uint2(at[0] | ((uint32_t)at[1] << 16), at[2] | ((uint32_t)at[3] << 16));
      const uint32_t mm = __vmaxu2(raw[gi][y].x & 0x7fff7fffu, raw[gi][y].y & 0x7fff7fffu);
      mx = max(mx, max(mm & 0xffffu, mm >> 16));
    }
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  float f;
  const float up = q_scale(p, mx, f);
#pragma unroll
  for (int gi = 0; gi < NG; ++gi) {
    float a[4], b[4];
    a[0] = bf16lo_to_f(raw[gi][0].x) * up; a[1] = bf16hi_to_f(raw[gi][0].x) * up;
    a[2] = bf16lo_to_f(raw[gi][0].y) * up; a[3] = bf16hi_to_f(raw[gi][0].y) * up;
    b[0] = bf16lo_to_f(raw[gi][1].x) * up; b[1] = bf16hi_to_f(raw[gi][1].x) * up;
    b[2] = bf16lo_to_f(raw[gi][1].y) * up; b[3] = bf16hi_to_f(raw[gi][1].y) * up;
#pragma unroll
    for (int odd = 0; odd < 2; ++odd)
#pragma unroll
      for (int j = 0; j < 2; ++j) qb[gi][odd][j] = attn_mma::pack_f16x2(a[odd + 2 * j], b[odd + 2 * j]);
  }
  return f;
}

// Rows of unit group u and the tokens they see.
struct Rows {
  int row0, nr, slot;
  int len_hi, len_lo, first_lo, first_hi;                // longest and shortest row, earliest and latest first token
  int page_lo, pages;
};
__device__ __forceinline__ Rows rows_of(const AttnParams& p, int u) {
  Rows r;
  const int blk = u / p.groups, grp = u % p.groups;
  r.row0 = blk * p.block + grp * p.rows;
  r.nr = min(p.rows, p.block - grp * p.rows);
  r.slot = p.row_seq[blk * p.block];
  r.len_hi = 0; r.len_lo = 0x7fffffff; r.first_lo = 0x7fffffff; r.first_hi = 0;
  for (int i = 0; i < r.nr; ++i) {
    const int len = row_len(p, r.row0 + i), first = row_first(p, len);
    r.len_lo = min(r.len_lo, len);
    if (len > 0) {                                       // a row without keys widens nothing
      r.len_hi = max(r.len_hi, len);
      r.first_lo = min(r.first_lo, first); r.first_hi = max(r.first_hi, first);
    }
  }
  r.page_lo = r.len_hi > 0 ? r.first_lo / kPage : 0;
  r.pages = r.len_hi > 0 ? (r.len_hi + kPage - 1) / kPage - r.page_lo : 0;
  return r;
}

// Pages before each group of rows, in shared memory; returns the pages per CTA of the streamed schedule.  Up to 32 groups: every
// warp scans them in its lanes and writes the same values, so that no barrier is needed before its own reads.
__device__ __forceinline__ int pages_per_cta(const AttnParams& p, int run) {
  const long long total = (long long)run * p.uheads;
  const int per = total < 0x7fffffffLL - p.ctas ? ((int)total + p.ctas - 1) / p.ctas : (int)((total + p.ctas - 1) / p.ctas);
  return max(8, (per + 7) / 8 * 8);                      // whole steps of the four warps
}
__device__ __forceinline__ int stream_schedule(const AttnParams& p, int (&before)[kMaxUnits + 1]) {
  __shared__ int warp_sum_[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int run = 0;
  if (p.units <= 32) {
    const int n = lane < p.units ? rows_of(p, lane).pages : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    run = __shfl_sync(0xffffffffu, x, 31);
    if (lane < p.units) before[lane] = x - n;
    if (lane == 0) before[p.units] = run;
    __syncwarp();
    return pages_per_cta(p, run);
  }
  for (int base = 0; base < p.units; base += kThreads) {
    int n = base + tid < p.units ? rows_of(p, base + tid).pages : 0, x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum_[warp] = x;
    __syncthreads();
    int ahead = run;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) ahead += warp_sum_[w];
      run += warp_sum_[w];
    }
    if (base + tid < p.units) before[base + tid] = ahead + x - n;
    __syncthreads();
  }
  if (tid == 0) before[p.units] = run;
  __syncthreads();
  return pages_per_cta(p, run);
}

// Attention of up to 8 * HH (row, head) pairs of one kv head over one split of the sequence's pages.
//
// It has to keep up with the cache's bytes (18 D per 16 tokens and kv head): a record may cost a
// warp no more issue slots than four times the ~100 cycles in which an SM receives it, and unpacking takes most of them.  Hence
//   * a warp owns steps of two pages (32 tokens); a page is ONE bulk copy (the record is contiguous) into a per-warp ring;
//   * S^T[token][pair] = K Q^T with the codes, as the fp16 integers that they are, as the MMA's row operand: 16 tokens fill its
//     rows and 8 pairs its columns.  q is scaled by a power of two to fill fp16's range (bf16 has fewer bits: exact); a
//     quantisation group is two k-steps whose sum is scaled by the group's maximum in fp32;
//   * O^T[dim][pair] += V^T[dim][token] P^T[token][pair].  P is multiplied by the token's V maximum in fp32, rounded to fp16
//     (11 bits, against the output's 8) and transposed from the accumulator's layout to the column operand's by one movmatrix
//     per 8 tokens; a running power of two keeps the largest product at the top of fp16's range, whatever the values'
//     magnitude.  (Rounding P first and multiplying in fp16 saves 14 instructions a page and loses tokens whose values are
//     2^-24 of the largest ones.)
//   * the maxima are unpacked once a step, a token per lane, and handed round through shared memory.
// Softmax statistics, scores and outputs are fp32.
//
// Measured (5 heads a kv head of 128, 8 kv heads; merge included): 32 rows of 16384 to 32768 tokens 222 us, 4.1 TB/s, 0.63 of a copy;
// one row of 131072 tokens 47 us, 3.2 TB/s; 8 rows of 2500 to 4999 21 us.  The copies alone take 147 of the 222 us.  What is left is
// latency: twelve warps an SM, each with one chain of unpacking (160 of 350 instructions a page), MMA, softmax and MMA.  No pipe is full
// (issue slots 57 % busy, integer 47 %, tensor 20 %) and the largest stall is the fixed-latency wait.
template <int D, int HH>
__global__ void __launch_bounds__(kThreads, Ring<D>::kCtas) attn_kernel(const AttnParams p) {
  using Gm = Geo<D>;
  constexpr int NG = Gm::kGroups, WT = D / 64, PP = 8 * HH;
  constexpr int kStages = Ring<D>::kStages;
  constexpr int kOld = D + 4;                            // floats between the pairs of the merge buffer
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ float sm_ml[kWarps][PP][2];
  __shared__ int before[kMaxUnits + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const Magic mg;
  uint8_t* ring = smem + (size_t)warp * Ring<D>::kWarpBytes;
  float* am_k = reinterpret_cast<float*>(ring + kStages * 2 * Gm::kRecord);                  // [32 tokens][NG]
  float* am_v = am_k + 32 * NG;                                                              // [32 tokens][NG]
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[warp][s], 1);
    mbar_fence_init();
  }
  __syncwarp();
  grm_pdl_wait();
  uint32_t step = 0;                                     // steps of this warp so far: ring stage and barrier phase
  uint32_t limit = 4000000u;

  // the pages [at, end) of the flat list (group of rows, head group, page) that this CTA works on
  long long at = 0, end = 1;
  if (p.splits == 0) {
    const int q = stream_schedule(p, before);
    at = (long long)blockIdx.x * q;
    end = min(at + q, (long long)before[p.units] * p.uheads);
    if (blockIdx.x == 0) {
      if (tid == 0) p.sched[0] = q;
      for (int i = tid; i <= p.units; i += kThreads) p.sched[1 + i] = before[i];
    }
  }
  while (at < end) {
  int u, uh, n0, n1, part;
  Rows rw;
  if (p.splits == 0) {
    int lo = 0, hi = p.units;                            // the last group with at most `at` pages before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if ((long long)before[mid] * p.uheads <= at) lo = mid;
      else hi = mid;
    }
    u = lo;
    rw = rows_of(p, u);
    const long long rest = at - (long long)before[u] * p.uheads;
    uh = (int)(rest / rw.pages);
    n0 = (int)(rest % rw.pages);
    n1 = (int)min((long long)rw.pages, n0 + (end - at));
    at += n1 - n0;
    part = (int)blockIdx.x + u * p.uheads + uh;          // parts of a unit are consecutive, units too
  } else {
    u = blockIdx.z; uh = blockIdx.y;
    rw = rows_of(p, u);
    const int per = (rw.pages + p.splits - 1) / p.splits;
    n0 = min((int)blockIdx.x * per, rw.pages);
    n1 = min(n0 + per, rw.pages);
    at = end;
    part = (u * p.uheads + uh) * p.splits + blockIdx.x;
  }
  const int kvh = uh / p.subs, sub = uh % p.subs;
  // pairs of this CTA: the group's rows x heads head0 .. head0 + nh - 1 of the kv head
  const int row0 = rw.row0, nr = rw.nr, slot = rw.slot;
  const int head0 = sub * p.heads, nh = min(p.heads, p.G - head0), np = nr * nh;
  const int len_hi = rw.len_hi, len_lo = rw.len_lo, first_lo = rw.first_lo, first_hi = rw.first_hi;
  const int pbeg = rw.page_lo + n0, pend = rw.page_lo + n1;
  const int n_it = pbeg + 2 * warp < pend ? (pend - pbeg - 2 * warp + 2 * kWarps - 1) / (2 * kWarps) : 0;      // steps of two pages of this warp

  // ---- ring ----
  // page ids of 16 steps, a lane each; -1: not there.  The lane that holds an id issues its copy.
  auto load_ids = [&](int base) {
    const int pg = pbeg + 2 * (warp + kWarps * (base + (lane >> 1))) + (lane & 1);
    return pg < pend ? page_of(p.t, slot, pg) : -1;
  };
  int ids = load_ids(0), ids_next = load_ids(16);
  uint32_t mapped = __ballot_sync(0xffffffffu, ids >= 0), mapped_next = __ballot_sync(0xffffffffu, ids_next >= 0);
  auto issue = [&](int it, uint32_t st, int id, uint32_t map) {
    if ((lane >> 1) == (it & 15)) {
      uint64_t* bar = &bars[warp][st % kStages];
      if (!(lane & 1)) mbar_expect_tx(bar, Gm::kRecord * __popc(map >> lane & 3u));
      if (id >= 0)
        bulk_load(ring + (2 * (st % kStages) + (lane & 1)) * Gm::kRecord, p.data + ((size_t)id * p.Hkv + kvh) * Gm::kRecord, Gm::kRecord, bar);
    }
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (s < n_it) issue(s, step + s, ids, mapped);

  // ---- q: column operands of S^T for the pairs g and g + 8 ----
  uint32_t qb[HH][NG][2][2];
  constexpr float kLag = 1.f;
  float fh[HH][2], m[HH][2], l[HH][2], bar[HH][2], off[HH][2];          // of the pairs 2 t, 2 t + 1 (+ 8 x)
  int lim[HH][2], low[HH][2];
#pragma unroll
  for (int x = 0; x < HH; ++x) {
    const int pr = g + 8 * x;
    const bool live = pr < np;
    const int row = row0 + (live ? pr / nh : 0), head = kvh * p.G + head0 + (live ? pr % nh : 0);
    const int seen = live ? row_len(p, row) : 0;
    const float f = load_q<D>(p, row, head, live, t, qb[x]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      fh[x][j] = __shfl_sync(0xffffffffu, f, 8 * t + 4 * j);
      lim[x][j] = __shfl_sync(0xffffffffu, seen, 8 * t + 4 * j);
      low[x][j] = row_first(p, lim[x][j]);
      m[x][j] = bar[x][j] = -INFINITY; l[x][j] = 0.f;
      off[x][j] = 14.f - kLag;
    }
  }

  float acc[HH][NG][2][4];                               // O^T tiles [group][nibble pair]
#pragma unroll
  for (int x = 0; x < HH; ++x)
#pragma unroll
    for (int gi = 0; gi < NG; ++gi)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[x][gi][0][i] = acc[x][gi][1][i] = 0.f;
  int e_run = 14;                                        // biased exponent of the largest V maximum so far
  auto step_work = [&](auto edge_tag, const uint8_t* rec, int tok0, int have) {
    constexpr bool kEdge = decltype(edge_tag)::value;    // some token of the step is hidden from some row
    // ---- maxima as fp32, a token per lane; those of V normalised ----
    {
      const int pg = lane >> 4, tok = tok_of((lane >> 3) & 1, lane & 7);
      uint32_t w[NG];                                    // K: words 0 .. NG / 2 - 1, V: the others
      const uint8_t* src = rec + pg * Gm::kRecord + Gm::kAmax + tok * Gm::kAmaxTok;
      load_words<NG>(src, w);
      if constexpr (kEdge) {                             // a token that no row sees must not set the scale of the values
        const int at = tok0 + pg * kPage + tok;
        if (at >= len_hi || at < first_lo || !(have >> pg & 1))
#pragma unroll
          for (int j = 0; j < NG / 2; ++j) w[NG / 2 + j] = 0u;
      }
      float kf[NG];
#pragma unroll
      for (int j = 0; j < NG / 2; ++j) { kf[2 * j] = bf16lo_to_f(w[j]); kf[2 * j + 1] = bf16hi_to_f(w[j]); }
      store_floats<NG>(am_k + lane * NG, kf);
      uint32_t vm = w[NG / 2];
#pragma unroll
      for (int j = 1; j < NG / 2; ++j) vm = __vmaxu2(vm, w[NG / 2 + j]);
      if (__any_sync(0xffffffffu, max(vm & 0xffffu, vm >> 16) >= (uint32_t)(e_run + 1) << 7)) {
        int e = e_run;                                   // of the finite ones: a group that is not a number must not hide the others
#pragma unroll
        for (int j = 0; j < NG / 2; ++j) {
          const int lo = (int)(w[NG / 2 + j] >> 7) & 255, hi = (int)(w[NG / 2 + j] >> 23) & 255;
          e = max(e, max(lo < 255 ? lo : 0, hi < 255 ? hi : 0));
        }
        e = (int)__reduce_max_sync(0xffffffffu, (uint32_t)e);
        const float c = e - e_run < 127 ? exp2_pos(e_run - e) : 0.f;
        e_run = e;
#pragma unroll
        for (int x = 0; x < HH; ++x)
#pragma unroll
          for (int gi = 0; gi < NG; ++gi)
#pragma unroll
            for (int ii = 0; ii < 2; ++ii)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[x][gi][ii][i] *= c;
      }
      const float vs = exp2_pos(127 - e_run);            // the largest maximum becomes 1 .. 2
      float vf[NG];
#pragma unroll
      for (int j = 0; j < NG / 2; ++j) { vf[2 * j] = bf16lo_to_f(w[NG / 2 + j]) * vs; vf[2 * j + 1] = bf16hi_to_f(w[NG / 2 + j]) * vs; }
      store_floats<NG>(am_v + lane * NG, vf);
    }
    __syncwarp();
    // ---- S^T: rows are tokens, columns pairs; value i of a lane: page i >> 2, tile i >> 1 & 1 (token column g), pair 2 t + (i & 1) ----
    float s[HH][8];
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      uint32_t kw[2][NG];
      float km[2][NG];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        load_words<NG>(rec + pg * Gm::kRecord + tok_of(b, g) * Gm::kRow + t * (D / 8), kw[b]);
        load_floats<NG>(am_k + (16 * pg + 8 * b + g) * NG, km[b]);
      }
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        uint32_t n0[4], n1[4];
        nibbles(mg, kw[0][gi / 2], kw[0][gi / 2 + NG / 2], gi & 1, n0);
        nibbles(mg, kw[1][gi / 2], kw[1][gi / 2 + NG / 2], gi & 1, n1);
#pragma unroll
        for (int x = 0; x < HH; ++x) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          mma(c, n0[0], n1[0], n0[2], n1[2], qb[x][gi][0][0], qb[x][gi][0][1]);
          mma(c, n0[1], n1[1], n0[3], n1[3], qb[x][gi][1][0], qb[x][gi][1][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[x][4 * pg + i] = gi == 0 ? c[i] * km[i >> 1][gi] : fmaf(c[i], km[i >> 1][gi], s[x][4 * pg + i]);
        }
      }
    }
    // ---- online softmax.  The reference, kept in units of s, follows the maximum when that is 2^kLag times ahead of it (the first
    // tokens, then hardly ever: no shuffles, no rescaling); P comes with a factor of 2^(14 - kLag) and stays below 2^14 ----
    uint32_t hidden[HH];
    bool ahead = false;
#pragma unroll
    for (int x = 0; x < HH; ++x) {
      hidden[x] = 0u;
      if constexpr (kEdge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = tok0 + (i >> 2) * kPage + tok_of((i >> 1) & 1, g);
          if (at >= lim[x][i & 1] || at < low[x][i & 1] || !(have >> (i >> 2) & 1)) {
            hidden[x] |= 1u << i;
            s[x][i] = -INFINITY;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
        ahead = ahead || fmaxf(fmaxf(s[x][j], s[x][2 + j]), fmaxf(s[x][4 + j], s[x][6 + j])) > bar[x][j];
    }
    if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
      for (int x = 0; x < HH; ++x) {
        float corr[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(fmaxf(s[x][j], s[x][2 + j]), fmaxf(s[x][4 + j], s[x][6 + j]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[x][j], mx), ref = mn == -INFINITY ? 0.f : mn;
          corr[j] = exp2_fast((m[x][j] - ref) * fh[x][j]);
          m[x][j] = mn;
          bar[x][j] = mn + kLag / fh[x][j];
          off[x][j] = fmaf(-ref, fh[x][j], 14.f - kLag);
          l[x][j] *= corr[j];
        }
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int ii = 0; ii < 2; ++ii)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[x][gi][ii][i] *= corr[i & 1];
      }
    }
#pragma unroll
    for (int x = 0; x < HH; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[x][2 * i + j] = exp2_fast(fmaf(s[x][2 * i + j], fh[x][j], off[x][j]));
          sum += s[x][2 * i + j];
        }
        l[x][j] += sum;
      }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      uint32_t vw[4][WT];
      float vm[2][NG];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_words<WT>(rec + pg * Gm::kRecord + Gm::kV + tok_of(i >> 1, 2 * t + (i & 1)) * Gm::kRow + g * (4 * WT), vw[i]);
#pragma unroll
      for (int b = 0; b < 2; ++b) load_floats<NG>(am_v + (16 * pg + 8 * b + g) * NG, vm[b]);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        uint32_t pb[HH][2];
#pragma unroll
        for (int x = 0; x < HH; ++x)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            pb[x][b] = attn_mma::pack_f16x2(s[x][4 * pg + 2 * b] * vm[b][gi], s[x][4 * pg + 2 * b + 1] * vm[b][gi]);
            if constexpr (kEdge) {                       // 0 * NaN
              const uint32_t hd = hidden[x] >> (4 * pg + 2 * b);
              pb[x][b] &= ((hd & 1u) ? 0u : 0xffffu) | ((hd & 2u) ? 0u : 0xffff0000u);
            }
            pb[x][b] = transpose8x8(pb[x][b]);           // [token][pair] accumulator rows -> column operand
          }
        uint32_t v01[4], v23[4];
        nibbles(mg, vw[0][gi / 2], vw[1][gi / 2], gi & 1, v01);
        nibbles(mg, vw[2][gi / 2], vw[3][gi / 2], gi & 1, v23);
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
          for (int x = 0; x < HH; ++x) mma(acc[x][gi][ii], v01[2 * ii], v01[2 * ii + 1], v23[2 * ii], v23[2 * ii + 1], pb[x][0], pb[x][1]);
      }
    }
  };

  for (int it = 0; it < n_it; ++it, ++step) {
    const int tok0 = (pbeg + 2 * (warp + kWarps * it)) * kPage;
    const int have = (int)(mapped >> (2 * (it & 15))) & 3;
    // a wait that runs out is on record in the status block; the call's result is void then, so do not wait at length again
    if (!mbar_wait(&bars[warp][step % kStages], (step / kStages) & 1u, p.status, 0x4b563400u | warp, limit)) limit = 16;
    __syncwarp();
    if (have) {
      const uint8_t* rec = ring + (step % kStages) * 2 * Gm::kRecord;
      if (have != 3 || tok0 + 2 * kPage > len_lo || tok0 < first_hi) step_work(std::true_type{}, rec, tok0, have);
      else step_work(std::false_type{}, rec, tok0, 3);
    }
    __syncwarp();
    const int nx = it + kStages;
    if (nx < n_it) {
      const bool later = (nx ^ it) & 16;
      issue(nx, step + kStages, later ? ids_next : ids, later ? mapped_next : mapped);
    }
    if ((it & 15) == 15) {
      ids = ids_next;
      mapped = mapped_next;
      ids_next = load_ids(it + 17);
      mapped_next = __ballot_sync(0xffffffffu, ids_next >= 0);
    }
  }
#pragma unroll
  for (int x = 0; x < HH; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[x][j] += __shfl_xor_sync(0xffffffffu, l[x][j], o);
      if (g == 0) { sm_ml[warp][2 * t + j + 8 * x][0] = m[x][j] * fh[x][j]; sm_ml[warp][2 * t + j + 8 * x][1] = l[x][j] * (1.f / 8192.f); }
    }
  __syncthreads();                                       // the rings become the merge buffer [warp][pair][nibble of a lane][lane row g]
  float* so = reinterpret_cast<float*>(smem);
  {
    const float fo = exp2_pos(e_run - 127) * (2.f / 7.f / 8192.f);             // codes' half, maxima's and P's powers of two
#pragma unroll
    for (int x = 0; x < HH; ++x)
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pr = 2 * t + (i & 1) + 8 * x, j = gi * 4 + 2 * ii + (i >> 1);
            so[(warp * PP + pr) * kOld + j * 8 + g] = acc[x][gi][ii][i] * fo;
          }
  }
  __syncthreads();
  // ---- join the warps: thread = (pair, two dims) ----
  for (int i = tid; i < np * (D / 2); i += kThreads) {
    const int pr = i / (D / 2), d = 2 * (i % (D / 2));
    float mx = -INFINITY, f[kWarps], ls = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm_ml[w][pr][0]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = sm_ml[w][pr][0] == -INFINITY ? 1.f : exp2f(sm_ml[w][pr][0] - mx);
      ls += sm_ml[w][pr][1] != 0.f ? f[w] * sm_ml[w][pr][1] : 0.f;                  // zero: no key; a NaN sum counts
    }
    const int word = d / 8, at = ((word % WT) * 8 + d % 8) * 8 + word / WT;
    float o[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (sm_ml[w][pr][1] != 0.f) {
        o[0] += f[w] * so[(w * PP + pr) * kOld + at];
        o[1] += f[w] * so[(w * PP + pr) * kOld + at + 8];
      }
    if (p.splits == 1) {
      const int row = row0 + pr / nh, head = kvh * p.G + head0 + pr % nh;
      finish(p, row, head, d, D, o[0], o[1], mx, ls);
    } else {
      const size_t pi = (size_t)part * PP + pr;
      *reinterpret_cast<float2*>(p.part_o + pi * D + d) = make_float2(o[0], o[1]);
      if (d == 0) { p.part_ml[2 * pi] = mx; p.part_ml[2 * pi + 1] = ls; }
    }
  }
  if (p.splits == 0) {                                   // the merge buffer becomes the rings again
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
  }
}

// Attention of up to 128 (row, head) pairs of one kv head over one split of the pages, for blocks of many rows: a page is
// unpacked once for 128 pairs (the kernel above: once for 16), and the products run on tcgen05.
//
//   * Four warps unpack 64 tokens (a page each) into fp16 operand tiles of 128-byte swizzled rows: (code - 8) / 2 times the
//     group's maximum, which fp16 holds exactly (3 + 8 bits) once the maxima are scaled by a power of two, K by one of its own
//     page, V by a running one of the CTA.  A word of codes becomes the 16 bytes of dims (0, 4, 1, 5, 2, 6, 3, 7): q is laid out
//     and the output read in that order.
//   * One thread issues S = Q K^T (64 columns of TMEM, two buffers) and O += P V (V as it lies, tokens by dims: the MN-major
//     operand), so that S of the next tokens runs under the softmax of these.
//   * Four warps do the softmax, a pair a thread: no shuffles, the reference follows the maximum when that is 2^kLag ahead.  P, rounded
//     to fp16 (11 bits, against the output's 8), takes the place of S in TMEM.  S(j + 1) is on its way before P(j) is complete, so a
//     warp may be a block ahead of a slower one: P has a barrier for even and one for odd blocks, and an arrival for P(j + 1) never
//     counts for P(j).  Two blocks ahead it cannot be: S(j + 2) is issued after P V(j), which waits for every warp's P(j).
// A V group that is not finite would reach rows that do not see it as 0 * NaN: it is unpacked as zero, and the rows that see its
// token remember the group.  Scores, statistics and outputs are fp32.
//
// Four blocks of 32 rows x 40 heads over 8192 to 16384 tokens of 8 kv heads of 128: 138 us with the merge (the kernel above: 250), 0.2
// PFLOP/s.  Bound by the chain of 64 tokens (unpack, S, softmax, P V; 3500 instructions) with two CTAs an SM to overlap, and by the
// CTAs' start: issue slots are 42 % busy, the tensor pipe 21 %; the stalls are loads, barriers and fixed latencies.
template <int D>
struct Tile {
  static constexpr int kTok = 64, kRows = 128, kThreads = 288;
  static constexpr int kQ = kRows * D * 2, kK = kTok * D * 2;
  static constexpr int kBytes = kQ + 4 * kK + 1024;      // K and V twice
  static constexpr int kCols = D == 256 ? 512 : 256;     // TMEM: S [0, 64) and [64, 128), P in the place of S, O behind them
  static constexpr int kCtas = D == 256 ? 1 : 2;         // an SM
};

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]; A: a row a lane, two fp16 a column
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void smem_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// What the unpacking warps tell the softmax about 64 tokens.
struct alignas(16) TileNote {
  float kf[4];               // K: what a product of the page has to be multiplied by
  int e;                     // V: biased exponent of the largest maximum so far
  uint8_t have[4], bad[4];   // a page is there; it holds a V group that is not finite
  uint8_t groups[64];        // which ones, a bit each, by token
};

// rows_of(), by a warp.
__device__ __forceinline__ Rows rows_of_warp(const AttnParams& p, int u) {
  Rows r;
  const int blk = u / p.groups, grp = u % p.groups, lane = threadIdx.x & 31;
  r.row0 = blk * p.block + grp * p.rows;
  r.nr = min(p.rows, p.block - grp * p.rows);
  r.slot = p.row_seq[blk * p.block];
  int len_hi = 0, len_lo = 0x7fffffff, first_lo = 0x7fffffff, first_hi = 0;
  for (int i = lane; i < r.nr; i += 32) {
    const int len = row_len(p, r.row0 + i), first = row_first(p, len);
    len_lo = min(len_lo, len);
    if (len > 0) {                                       // a row without keys widens nothing
      len_hi = max(len_hi, len);
      first_lo = min(first_lo, first); first_hi = max(first_hi, first);
    }
  }
  r.len_hi = __reduce_max_sync(0xffffffffu, len_hi); r.len_lo = __reduce_min_sync(0xffffffffu, len_lo);
  r.first_lo = __reduce_min_sync(0xffffffffu, first_lo); r.first_hi = __reduce_max_sync(0xffffffffu, first_hi);
  r.page_lo = r.len_hi > 0 ? r.first_lo / kPage : 0;
  r.pages = r.len_hi > 0 ? (r.len_hi + kPage - 1) / kPage - r.page_lo : 0;
  return r;
}

// The 16 bytes that a word of codes becomes: dims 0, 4, 1, 5, 2, 6, 3, 7 times the maxima (of dims 0 - 3, of dims 4 - 7).
__device__ __forceinline__ uint4 unpack_word(const Magic& mg, uint32_t x, uint32_t a) {
  const uint32_t y = x >> 8;
  return make_uint4(h2_mul(h2_fma(low_nibble(x, mg.one), mg.even, 0xe008e008u), a), h2_mul(h2_fma(high_nibble(x, mg.one), mg.odd, 0xd080d080u), a),
                    h2_mul(h2_fma(low_nibble(y, mg.one), mg.even, 0xe008e008u), a), h2_mul(h2_fma(high_nibble(y, mg.one), mg.odd, 0xd080d080u), a));
}
// Largest exponent of the finite ones of two bf16 maxima.
__device__ __forceinline__ int top_exponent(uint32_t w) {
  const int lo = (int)(w >> 7) & 255, hi = (int)(w >> 23) & 255;
  return max(lo < 255 ? lo : 0, hi < 255 ? hi : 0);
}
// B operand with the dims contiguous: 64 of them a 128-byte swizzled row, a token a row, eight rows 1024 bytes.  One instruction takes
// 64 dims and 16 tokens, so that the only stride is the one between groups of eight tokens.
__device__ __forceinline__ uint64_t tokens_by_dims_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)(1024 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <int D>
__global__ void __launch_bounds__(Tile<D>::kThreads, Tile<D>::kCtas) tile_kernel(const AttnParams p) {
  using Gm = Geo<D>;
  using T = Tile<D>;
  constexpr int NG = Gm::kGroups, NW = NG / 2;           // words of a token's K (or V) maxima
  constexpr int kUnits = D / 64;                         // 16-byte units of K (or V) codes a lane and page
  constexpr int kBox = T::kTok * 128;                    // bytes of 64 dims of the tokens
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t b_q, b_p[2], b_k[2], b_v[2], b_s[2], b_o[2];
  __shared__ TileNote notes[4];                          // of blocks j mod 4
  __shared__ int v_top[2][4];
  __shared__ uint32_t tmem_holder;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = sQ + T::kQ, *sV = sK + 2 * T::kK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grm_pdl_wait();
  const int u = blockIdx.z, kvh = blockIdx.y;
  const Rows rw = rows_of_warp(p, u);
  const int np = rw.nr * p.G;
  int per = (rw.pages + p.splits - 1) / p.splits;
  per = (per + 3) / 4 * 4;
  const int n0 = min((int)blockIdx.x * per, rw.pages), n1 = min(n0 + per, rw.pages);
  const int pbeg = rw.page_lo + n0, pend = rw.page_lo + n1, nblk = (n1 - n0 + 3) / 4;
  if (tid == 0) {
    mbar_init(&b_q, 128);
    for (int i = 0; i < 2; ++i) { mbar_init(&b_p[i], 32 * ((np + 31) / 32)); mbar_init(&b_k[i], 128); mbar_init(&b_v[i], 128); mbar_init(&b_s[i], 1); mbar_init(&b_o[i], 1); }
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_holder, T::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  uint32_t limit = 4000000u;                             // a wait that runs out is on record in the status block: the next ones are short, the loops end as always

  if (warp == 8) {
    if (lane == 0 && nblk > 0) {
      constexpr uint32_t idesc = make_idesc(128, 64, 0, 0), idesc_mn = idesc | (1u << 16);
      auto issue_s = [&](int j) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma_f16(tmem + 64 * (j & 1), make_sw128_kmajor_desc(smem_u32(sQ) + (k >> 2) * (T::kRows * 128)) + (uint64_t)((k & 3) * 2),
                     make_sw128_kmajor_desc(smem_u32(sK) + (j & 1) * T::kK + (k >> 2) * kBox) + (uint64_t)((k & 3) * 2), idesc, k != 0 ? 1u : 0u);
        tc_commit(&b_s[j & 1]);
      };
      bool good = mbar_wait(&b_q, 0u, p.status, 0x4b563410u) && mbar_wait(&b_k[0], 0u, p.status, 0x4b563411u);
      if (good) issue_s(0);
      for (int j = 0; j < nblk && good; ++j) {
        if (j + 1 < nblk) {
          good = mbar_wait(&b_k[(j + 1) & 1], (uint32_t)((j + 1) >> 1) & 1u, p.status, 0x4b563412u);
          // its TMEM buffer holds P(j - 1): products with different accumulators are not ordered by their issue, so P V(j - 1) has to be
          // through with it (it runs beside the softmax of block j, which takes longer)
          if (j > 0) good = good && mbar_wait(&b_o[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, p.status, 0x4b56341au);
          if (!good) break;
          issue_s(j + 1);
        }
        good = mbar_wait(&b_p[j & 1], (uint32_t)(j >> 1) & 1u, p.status, 0x4b563413u) && mbar_wait(&b_v[j & 1], (uint32_t)(j >> 1) & 1u, p.status, 0x4b563414u);
        if (!good) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < D / 64; ++x)
#pragma unroll
          for (int k = 0; k < T::kTok / 16; ++k)
            tc_mma_f16_ts(tmem + 128 + 64 * x, tmem + 64 * (j & 1) + 8 * k,
                          tokens_by_dims_desc(smem_u32(sV) + (j & 1) * T::kK + x * kBox + k * 2048), idesc_mn, (k != 0 || j != 0) ? 1u : 0u);
        tc_commit(&b_o[j & 1]);
      }
    }
  } else if (warp >= 4) {
    // ---- unpack: a page a warp ----
    const Magic mg;
    const int w4 = warp - 4;
    // the page of the next 64 tokens is on its way while these are unpacked, the id of the one after that too
    uint4 ck[kUnits], cv[kUnits], ck_next[kUnits], cv_next[kUnits];
    uint32_t am[kUnits][2 * NW], am_next[kUnits][2 * NW];          // maxima: K, then V
    auto id_of = [&](int j) {
      const int pg = pbeg + 4 * j + w4;
      return pg < pend ? page_of(p.t, rw.slot, pg) : -1;
    };
    int id_next = id_of(0), id_after = id_of(1);
    auto fetch = [&](int id) {                           // (a page that is not there: any other, for nothing)
      const uint8_t* rec = p.data + ((size_t)max(id, 0) * p.Hkv + kvh) * Gm::kRecord;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        ck_next[i] = __ldg(reinterpret_cast<const uint4*>(rec) + lane + 32 * i);
        cv_next[i] = __ldg(reinterpret_cast<const uint4*>(rec + Gm::kV) + lane + 32 * i);
        load_words<2 * NW>(rec + Gm::kAmax + (lane + 32 * i) / (D / 32) * Gm::kAmaxTok, am_next[i]);
      }
    };
    fetch(id_next);
    int e_run = 14;
    for (int j = 0; j < nblk; ++j) {
      TileNote& note = notes[j & 3];
      const bool have = id_next >= 0;
      const int tok0 = (pbeg + 4 * j + w4) * kPage;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        ck[i] = ck_next[i]; cv[i] = cv_next[i];
#pragma unroll
        for (int n = 0; n < 2 * NW; ++n) am[i][n] = am_next[i][n];
      }
      if (!have || tok0 < rw.first_lo || tok0 + kPage > rw.len_hi) {       // a token that no row sees must not set a scale, nor be a NaN
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int at = tok0 + (lane + 32 * i) / (D / 32);
          if (!have || at < rw.first_lo || at >= rw.len_hi)
#pragma unroll
            for (int n = 0; n < 2 * NW; ++n) am[i][n] = 0u;
        }
      }
      id_next = id_after;
      fetch(id_next);
      id_after = id_of(j + 2);
      uint32_t k2 = 0, v2 = 0;
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
#pragma unroll
        for (int n = 0; n < NW; ++n) { k2 = __vmaxu2(k2, am[i][n]); v2 = __vmaxu2(v2, am[i][NW + n]); }
      int ek = (int)max(k2 & 0xffffu, k2 >> 16) >> 7, ev = (int)max(v2 & 0xffffu, v2 >> 16) >> 7;
      const bool odd = __any_sync(0xffffffffu, max(ek, ev) >= 255);
      bool bad = false;
      if (odd) {                                         // the largest finite ones, and the V groups that are not
        ek = ev = 0;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          uint32_t groups = 0;
#pragma unroll
          for (int n = 0; n < NW; ++n) {
            ek = max(ek, top_exponent(am[i][n]));
            uint32_t& v = am[i][NW + n];
            ev = max(ev, top_exponent(v));
            if ((v & 0x7f80u) == 0x7f80u) { groups |= 1u << (2 * n); v &= 0xffff0000u; }
            if ((v & 0x7f800000u) == 0x7f800000u) { groups |= 2u << (2 * n); v &= 0xffffu; }
          }
          const int x = lane + 32 * i;
          bad = bad || groups;
          if (x % (D / 32) == 0) note.groups[16 * w4 + x / (D / 32)] = (uint8_t)groups;
        }
        bad = __any_sync(0xffffffffu, bad);
      }
      ek = max(14, (int)__reduce_max_sync(0xffffffffu, (uint32_t)ek));
      ev = max(14, (int)__reduce_max_sync(0xffffffffu, (uint32_t)ev));
      if (lane == 0) {
        note.kf[w4] = exp2_pos(ek - 140);
        note.have[w4] = have; note.bad[w4] = bad;
        v_top[j & 1][w4] = ev;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
      for (int w = 0; w < 4; ++w) e_run = max(e_run, v_top[j & 1][w]);
      if (lane == 0 && w4 == 0) note.e = e_run;
      auto store = [&](uint8_t* tile, const uint4 (&c)[kUnits], int first, int e) {
        const float down = exp2_pos(140 - e);            // 2^13 / 2^(e - 127): a product with half a code stays below 2^16
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int x = lane + 32 * i, tok = 16 * w4 + x / (D / 32);
          uint32_t a[NW];
#pragma unroll
          for (int n = 0; n < NW; ++n) a[n] = attn_mma::pack_f16x2(bf16lo_to_f(am[i][first + n]) * down, bf16hi_to_f(am[i][first + n]) * down);
          const uint32_t c4[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int w = 4 * (x % (D / 32)) + k;
            *reinterpret_cast<uint4*>(tile + (w >> 3) * kBox + tok * 128 + (((w & 7) ^ (tok & 7)) << 4)) = unpack_word(mg, c4[k], a[k % NW]);
          }
        }
        smem_to_async();
      };
      if (j > 1 && !mbar_wait(&b_s[j & 1], (uint32_t)((j >> 1) - 1) & 1u, p.status, 0x4b563415u, limit)) limit = 16;
      store(sK + (j & 1) * T::kK, ck, 0, ek);
      mbar_arrive(&b_k[j & 1]);
      if (j > 1 && !mbar_wait(&b_o[j & 1], (uint32_t)((j >> 1) - 1) & 1u, p.status, 0x4b563416u, limit)) limit = 16;
      store(sV + (j & 1) * T::kK, cv, NW, e_run);
      mbar_arrive(&b_v[j & 1]);
    }
  } else {
    // ---- softmax: a pair a thread ----
    constexpr float kLag = 1.f;
    const bool live = tid < np;
    const int row = rw.row0 + (live ? tid / p.G : 0), head = kvh * p.G + (live ? tid % p.G : 0);
    const int hi = live ? row_len(p, row) : 0, lo = row_first(p, hi);
    float f;
    {
      const unsigned short* src = reinterpret_cast<const unsigned short*>(p.q) + (size_t)row * p.ld_q + (size_t)head * D;
      auto quad = [&](int i) -> uint2 {
        if (!live) return make_uint2(0u, 0u);
        if (p.vec) return __ldg(reinterpret_cast<const uint2*>(src) + i);
        const unsigned short* at = src + 4 * i;
        return make_uint2(at[0] | ((uint32_t)at[1] << 16), at[2] | ((uint32_t)at[3] << 16));
      };
      uint32_t mx = 0;
#pragma unroll 8
      for (int i = 0; i < D / 4; ++i) {
        const uint2 v = quad(i);
        const uint32_t mm = __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
        mx = max(mx, max(mm & 0xffffu, mm >> 16));
      }
      const float up = q_scale(p, mx, f);
#pragma unroll 4
      for (int w = 0; w < D / 8; ++w) {
        const uint2 a = quad(2 * w), b = quad(2 * w + 1);
        const uint4 v = make_uint4(attn_mma::pack_f16x2(bf16lo_to_f(a.x) * up, bf16lo_to_f(b.x) * up), attn_mma::pack_f16x2(bf16hi_to_f(a.x) * up, bf16hi_to_f(b.x) * up),
                                   attn_mma::pack_f16x2(bf16lo_to_f(a.y) * up, bf16lo_to_f(b.y) * up), attn_mma::pack_f16x2(bf16hi_to_f(a.y) * up, bf16hi_to_f(b.y) * up));
        *reinterpret_cast<uint4*>(sQ + (w >> 3) * (T::kRows * 128) + tid * 128 + (((w & 7) ^ (tid & 7)) << 4)) = v;
      }
      smem_to_async();
      mbar_arrive(&b_q);
    }
    const uint32_t t_row = tmem + ((uint32_t)(warp * 32) << 16);
    float m = -INFINITY, bar = -INFINITY, off = 14.f - kLag, l = 0.f;
    int e_run = 14;
    uint32_t poison = 0;                                 // V groups of a token that the row sees and that are not finite
    const bool on = nblk > 0 && 32 * warp < np;
    for (int j = 0; j < nblk && on; ++j) {
      if (!mbar_wait(&b_s[j & 1], (uint32_t)(j >> 1) & 1u, p.status, 0x4b563417u, limit)) limit = 16;
      __syncwarp();
      tc_fence_after();
      const TileNote& note = notes[j & 3];
      const int tok0 = (pbeg + 4 * j) * kPage;
      const uint32_t haves = *reinterpret_cast<const uint32_t*>(note.have), bads = *reinterpret_cast<const uint32_t*>(note.bad);
      const float4 k4 = *reinterpret_cast<const float4*>(note.kf);
      const float kf[4] = {fmaxf(f * k4.x, 1e-37f), fmaxf(f * k4.y, 1e-37f), fmaxf(f * k4.z, 1e-37f), fmaxf(f * k4.w, 1e-37f)};      // (0 * -inf)
      const bool edge = haves != 0x01010101u || tok0 + T::kTok > rw.len_lo || tok0 < rw.first_hi;
      const uint32_t ts = t_row + 64 * (j & 1);
      const int e_new = note.e;
      auto hide = [&](uint32_t (&r)[32], int half) {
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          const int at = tok0 + 32 * half + 16 * pg, a = lo - at, b = (haves >> (8 * (2 * half + pg)) & 255u) ? hi - at : 0;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < a || i >= b) r[16 * pg + i] = 0xff800000u;
        }
      };
      float mx = -INFINITY;
      uint32_t r[32];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        tmem_ld_32x32b_x32(ts + 32 * half, r);
        tmem_ld_wait();
        if (edge) hide(r, half);
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          float a = __uint_as_float(r[16 * pg]), b = __uint_as_float(r[16 * pg + 1]);
#pragma unroll
          for (int i = 2; i < 16; i += 2) { a = fmaxf(a, __uint_as_float(r[16 * pg + i])); b = fmaxf(b, __uint_as_float(r[16 * pg + i + 1])); }
          mx = fmaxf(mx, fmaxf(a, b) * kf[2 * half + pg]);
        }
      }
      float alpha = 1.f;
      if (mx > bar) {
        alpha = m == -INFINITY ? 0.f : exp2_fast(m - mx);
        m = mx;
        bar = mx + kLag;
        off = 14.f - kLag - mx;
        l *= alpha;
      }
      if (e_new != e_run) {                              // the values' power of two has moved: the sums follow, P does not
        alpha *= e_new - e_run < 127 ? exp2_pos(e_run - e_new) : 0.f;
        e_run = e_new;
      }
      if (bads)
        for (int i = 0; i < T::kTok; ++i) poison |= (note.bad[i >> 4] && tok0 + i >= lo && tok0 + i < hi) ? note.groups[i] : 0u;
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {       // O(j - 1) has to be there
        if (!mbar_wait(&b_o[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, p.status, 0x4b563418u, limit)) limit = 16;
        __syncwarp();
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          tmem_ld_32x32b_x32(t_row + 128 + 32 * c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
          tmem_st_x32(t_row + 128 + 32 * c, r);
        }
      }
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        tmem_ld_32x32b_x32(ts + 32 * half, r);
        tmem_ld_wait();
        if (edge) hide(r, half);
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float k = kf[2 * half + (i >> 3)];
          const float x = exp2_fast(fmaf(__uint_as_float(r[2 * i]), k, off)), y = exp2_fast(fmaf(__uint_as_float(r[2 * i + 1]), k, off));
          sum[0] += x; sum[1] += y;
          o[i] = attn_mma::pack_f16x2(x, y);
        }
        tmem_st_x16(ts + 16 * half, o);
      }
      l += sum[0] + sum[1];
      tmem_st_done();
      tc_fence_before();
      mbar_arrive(&b_p[j & 1]);
    }
    if (on) {
      mbar_wait(&b_o[(nblk - 1) & 1], (uint32_t)((nblk - 1) >> 1) & 1u, p.status, 0x4b563419u, limit);
      tc_fence_after();
    }
    // (a CTA without pages has nothing in TMEM: its sums are zero)
    const float ls = l * (1.f / 8192.f), fo = exp2_pos(e_run - 140);
    const size_t pi = ((size_t)(u * p.uheads + kvh) * p.splits + blockIdx.x) * T::kRows + tid;
    if (32 * warp < np) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        __syncwarp();
        if (on) {
          tmem_ld_32x32b_x32(t_row + 128 + 32 * c, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        if (live && (on || p.splits == 1)) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int g = (8 * c + 2 * w + (i & 1)) % NG;           // the group of dims i >> 1 (+ 4)
              o[(i >> 1) + 4 * (i & 1)] = (poison >> g & 1u) ? __uint_as_float(0x7fc00000u) : __uint_as_float(r[8 * w + i]) * (2.f / 7.f / 8192.f) * fo;
            }
            const int d = 32 * c + 8 * w;
            if (p.splits == 1) {
#pragma unroll
              for (int i = 0; i < 8; i += 2) finish(p, row, head, d + i, D, o[i], o[i + 1], m, ls);
            } else {
              float4* dst = reinterpret_cast<float4*>(p.part_o + pi * D + d);
              dst[0] = make_float4(o[0], o[1], o[2], o[3]);
              dst[1] = make_float4(o[4], o[5], o[6], o[7]);
            }
          }
        }
      }
      if (live && p.splits != 1) { p.part_ml[2 * pi] = m; p.part_ml[2 * pi + 1] = ls; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, T::kCols);
}

// Joins the parts of a unit: one CTA per (query head, row).  Groups of D / 2 threads (two dims each) take every n-th part and are
// joined in order: the result does not depend on timing.  Bound by the latency of its dependent loads: the parts' statistics are
// read once, and a group keeps eight parts in flight.
// kMergeThreads: 512 where a unit has many parts (74 of one row over 131072 tokens: 4 us less than with 256), 128 where it has few.
constexpr int kMergeParts = 512;
template <int D, int kMergeThreads>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const AttnParams p) {
  constexpr int kGroups = kMergeThreads / (D / 2), kMergeWarps = kMergeThreads / 32;
  __shared__ float2 wt[kMergeParts];                     // (weight, sum) of a part; a part without keys has a sum of zero
  __shared__ float red[kMergeWarps];
  __shared__ float2 so[kGroups][D / 2];
  __shared__ float sl[kGroups];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = tid / (D / 2), d = 2 * (tid % (D / 2));
  const int row = blockIdx.y, head = blockIdx.x;
  const int kvh = head / p.G, hg = head % p.G, blk = row / p.block, in = row % p.block;
  const int u = blk * p.groups + in / p.rows, uh = kvh * p.subs + hg / p.heads;
  const int nh = min(p.heads, p.G - hg / p.heads * p.heads), pr = (in % p.rows) * nh + hg % p.heads;
  grm_pdl_wait();
  long first = ((long)u * p.uheads + uh) * p.splits;
  int n = p.splits;
  if (p.splits == 0) {
    const long long q = p.sched[0], lo = p.sched[1 + u], pages = p.sched[2 + u] - lo;
    const long long beg = lo * p.uheads + uh * pages, last = beg + pages - 1;
    long long c0, c1;
    if (last < 0xffffffffLL) {                           // 32-bit division where it will do
      c0 = (uint32_t)beg / (uint32_t)q; c1 = (uint32_t)last / (uint32_t)q;
    } else {
      c0 = beg / q; c1 = last / q;
    }
    first = c0 + (long)u * p.uheads + uh;
    n = pages > 0 ? (int)(c1 - c0) + 1 : 0;
  }
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + first * p.pairs + pr;
  const float* po = p.part_o + (first * p.pairs + pr) * D + d;
  float mx = -INFINITY;
  for (int s = tid; s < n; s += kMergeThreads) {
    const float2 v = ml[(size_t)s * p.pairs];
    if (n <= kMergeParts) wt[s] = v;
    mx = fmaxf(mx, v.x);
  }
  mx = warp_max(mx);
  if (lane == 0) red[warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) mx = fmaxf(mx, red[w]);
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int base = 0; base < n; base += kMergeParts) {
    const int here = min(kMergeParts, n - base);
    for (int s = tid; s < here; s += kMergeThreads) {
      const float2 v = n <= kMergeParts ? wt[s] : ml[(size_t)(base + s) * p.pairs];
      wt[s] = make_float2(v.x == -INFINITY ? 1.f : exp2f(v.x - mx), v.y);
    }
    __syncthreads();
#pragma unroll 8
    for (int s = grp; s < here; s += kGroups) {
      const float2 v = *reinterpret_cast<const float2*>(po + (size_t)(base + s) * p.pairs * D);
      const float2 f = wt[s];
      if (f.y != 0.f) { l = fmaf(f.x, f.y, l); o0 = fmaf(f.x, v.x, o0); o1 = fmaf(f.x, v.y, o1); }      // a NaN sum counts
    }
    __syncthreads();
  }
  so[grp][d / 2] = make_float2(o0, o1);
  if (d == 0) sl[grp] = l;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 1; i < kGroups; ++i) {
      const float2 v = so[i][d / 2];
      o0 += v.x; o1 += v.y; l = l + sl[i];
    }
    finish(p, row, head, d, D, o0, o1, mx, l);
  }
}

// The observed weight: mass[token] (=, +=) sum over the rows and heads of a block of exp2(score - maximum) / sum.
//
// Scores are computed once more rather than stored: K is half of the cache, a stored score would be 4 bytes per query head.  A
// warp takes whole pages; the page's K becomes the MMA's row operand once, (code - 8) / 2 times its group's maximum, which fp16
// holds exactly (3 + 8 bits), and every tile of 8 (row, head) pairs is one column operand from shared memory: D / 16 MMAs and
// four exponentials a lane.  160 pairs over four sequences of 8192 to 16384 tokens x 8 kv heads of 128 take 82 us: MMAs (16 cycles of an
// SM a tile and page at D = 128; the tensor pipe is 44 % busy) in a chain behind operands from shared memory.  One row's 5 pairs take
// 20 us, 1.4 TB/s of K: latency, of the loads of one page at a time a warp and of the CTAs' start (queries, the search for blocks of
// the same sequence).  All rows of one sequence are summed by the CTAs of its first block, in the order of the rows:
// two blocks of one sequence neither race nor depend on timing.
template <int D>
struct MassTile {
  static constexpr int kSide = D == 256 ? 2 : 4;         // tiles worked on side by side: independent chains of MMAs
  static constexpr int kTiles = 2560 / D / kSide * kSide;       // tiles in shared memory at a time
  static constexpr int kBytes = kTiles * (32 * D / 2 + 8 * 24);       // operands, (factor, maximum, 1 / sum), (seen, first)
};
// The weights that a page's tokens g and g + 8 draw from the lane's pairs of tiles i0 .. i0 + kSide - 1, worked on side by side:
// independent chains of MMAs.
template <int D, bool kEdge, int kSide>
__device__ __forceinline__ void tile_sums(const uint32_t (&ka)[D / 32][2][4], const uint4* sq, const float4* sf, const int2* sl, int i0, float pf,
                                          int tok0, int lane, float (&sum)[2]) {
  constexpr int NG = D / 32;
  const int g = lane >> 2, t = lane & 3;
  float c[kSide][4];
#pragma unroll
  for (int i = 0; i < kSide; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
#pragma unroll
  for (int gi = 0; gi < NG; ++gi)
#pragma unroll
    for (int i = 0; i < kSide; ++i) {
      const uint4 q = sq[((i0 + i) * NG + gi) * 32 + lane];
      mma(c[i], ka[gi][0][0], ka[gi][0][1], ka[gi][0][2], ka[gi][0][3], q.x, q.y);
      mma(c[i], ka[gi][1][0], ka[gi][1][1], ka[gi][1][2], ka[gi][1][3], q.z, q.w);
    }
#pragma unroll
  for (int i = 0; i < kSide; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 f = sf[8 * (i0 + i) + 2 * t + j];
      const int2 lim = kEdge ? sl[8 * (i0 + i) + 2 * t + j] : make_int2(0, 0);
      const float k = f.x * pf;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float e = exp2_fast(fmaf(c[i][2 * r + j], k, -f.y));
        const int at = tok0 + g + 8 * r;
        if (!kEdge || (at < lim.x && at >= lim.y)) sum[r] = fmaf(e, f.z, sum[r]);
      }
    }
}
template <int D, bool kEdge>
__device__ __forceinline__ void page_sums(const uint32_t (&ka)[D / 32][2][4], const uint4* sq, const float4* sf, const int2* sl, int tiles, float pf,
                                          int tok0, int lane, float (&sum)[2]) {
  constexpr int kSide = MassTile<D>::kSide;
  int i = 0;
#pragma unroll 1
  for (; i + kSide <= tiles; i += kSide) tile_sums<D, kEdge, kSide>(ka, sq, sf, sl, i, pf, tok0, lane, sum);
#pragma unroll 1
  for (; i < tiles; ++i) tile_sums<D, kEdge, 1>(ka, sq, sf, sl, i, pf, tok0, lane, sum);
}

template <int D>
__global__ void __launch_bounds__(kThreads) mass_kernel(const AttnParams p, int nblocks, int pages, int per_cta) {
  using Gm = Geo<D>;
  constexpr int NG = Gm::kGroups, kTiles = MassTile<D>::kTiles;
  extern __shared__ __align__(128) uint8_t smem[];
  uint4* sq = reinterpret_cast<uint4*>(smem);                                        // [tile][NG][lane]
  float4* sf = reinterpret_cast<float4*>(smem + kTiles * 32 * D / 2);                // [tile][pair]
  int2* sl = reinterpret_cast<int2*>(smem + kTiles * (32 * D / 2 + 8 * 16));         // [tile][pair]
  __shared__ int s_len, s_dup;
  const int kvh = blockIdx.y, blk = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const Magic mg;
  if (tid == 0) { s_len = 0; s_dup = 0; }
  grm_pdl_wait();
  const int slot = p.row_seq[blk * p.block];
  __syncthreads();
  for (int b = tid; b < blk; b += kThreads)
    if (p.row_seq[b * p.block] == slot) s_dup = 1;
  int len = 0;
  for (int r = blk * p.block + tid; r < nblocks * p.block; r += kThreads)
    if (p.row_seq[r / p.block * p.block] == slot) len = max(len, row_len(p, r));
  atomicMax(&s_len, len);
  __syncthreads();
  if (s_dup) return;
  len = s_len;
  const int beg = blockIdx.x * per_cta, end = min(min(beg + per_cta, pages), (len + kPage - 1) / kPage);
  if (beg >= end) return;

  bool first = true;                                     // nothing of this call is in the mass yet
  for (int b = blk; b < nblocks; ++b) {
    if (p.row_seq[b * p.block] != slot) continue;
    const int np = p.block * p.G;
    for (int pair0 = 0; pair0 < np; pair0 += 8 * kTiles) {
      const int tiles = min(kTiles, (np - pair0 + 7) / 8);
      __syncthreads();
      for (int i = warp; i < tiles; i += kWarps) {
        const int pr = pair0 + 8 * i + g;
        const bool live = pr < np;
        const int row = b * p.block + (live ? pr / p.G : 0), head = kvh * p.G + (live ? pr % p.G : 0);
        uint32_t qb[NG][2][2];
        const float f = load_q<D>(p, row, head, live, t, qb);
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) sq[(i * NG + gi) * 32 + lane] = make_uint4(qb[gi][0][0], qb[gi][0][1], qb[gi][1][0], qb[gi][1][1]);
        if (t == 0) {
          const float* fin = p.fin + 2 * ((size_t)row * p.Hkv * p.G + head);
          const bool any = live && fin[1] != 0.f;        // a row without keys has no reciprocal sum
          const int seen = any ? row_len(p, row) : 0;
          sf[8 * i + g] = any ? make_float4(f, fin[0], fin[1], 0.f) : make_float4(0.f, 0.f, 0.f, 0.f);
          sl[8 * i + g] = make_int2(seen, row_first(p, seen));
        }
      }
      __syncthreads();
      int len_lo = 0x7fffffff, first_hi = 0;
      for (int i = lane; i < min(8 * tiles, np - pair0); i += 32) { len_lo = min(len_lo, sl[i].x); first_hi = max(first_hi, sl[i].y); }
      len_lo = __reduce_min_sync(0xffffffffu, len_lo);
      first_hi = __reduce_max_sync(0xffffffffu, first_hi);

      // the next page is on its way while a page is worked on, the id of the one after that too
      uint32_t kw[2][NG], am[2][NG / 2], kw_next[2][NG], am_next[2][NG / 2];
      int page = -1, page_next = beg + warp < end ? page_of(p.t, slot, beg + warp) : -1;
      int page_after = beg + warp + kWarps < end ? page_of(p.t, slot, beg + warp + kWarps) : -1;
      auto fetch = [&](int id) {
        const uint8_t* rec = p.data + ((size_t)max(id, 0) * p.Hkv + kvh) * Gm::kRecord;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          load_words<NG>(rec + (g + 8 * r) * Gm::kRow + t * (D / 8), kw_next[r]);
          load_words<NG / 2>(rec + Gm::kAmax + (g + 8 * r) * Gm::kAmaxTok, am_next[r]);
        }
      };
      fetch(page_next);
      for (int pg = beg + warp; pg < end; pg += kWarps) {
        const int tok0 = pg * kPage;
        page = page_next;
        page_next = page_after;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int j = 0; j < NG; ++j) kw[r][j] = kw_next[r][j];
#pragma unroll
          for (int j = 0; j < NG / 2; ++j) am[r][j] = tok0 + g + 8 * r < len ? am_next[r][j] : 0u;      // what lies behind must not set the scale
        }
        if (pg + kWarps < end) fetch(page_next);
        page_after = pg + 2 * kWarps < end ? page_of(p.t, slot, pg + 2 * kWarps) : -1;
        if (page < 0) continue;
        int e = 14;                                      // biased exponent of the page's largest finite maximum
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < NG / 2; ++j) {
            const int lo = (int)(am[r][j] >> 7) & 255, hi = (int)(am[r][j] >> 23) & 255;
            e = max(e, max(lo < 255 ? lo : 0, hi < 255 ? hi : 0));
          }
        e = __reduce_max_sync(0xffffffffu, e);
        const float down = exp2_pos(138 - e), pf = exp2_pos(e - 138);    // 2^11 / 2^(e - 127): a product with a code stays below 2^14
        uint32_t ka[NG][2][4];
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float a = ((gi & 1) ? bf16hi_to_f(am[r][gi / 2]) : bf16lo_to_f(am[r][gi / 2])) * down;
            const uint32_t aa = attn_mma::pack_f16x2(a, a);
            uint32_t n[4];
            nibbles(mg, kw[r][gi / 2], kw[r][gi / 2 + NG / 2], gi & 1, n);
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
              ka[gi][odd][r] = h2_mul(n[odd], aa);
              ka[gi][odd][2 + r] = h2_mul(n[odd + 2], aa);
            }
          }
        float sum[2] = {0.f, 0.f};
        if (tok0 + kPage > len_lo || tok0 < first_hi) page_sums<D, true>(ka, sq, sf, sl, tiles, pf, tok0, lane, sum);
        else page_sums<D, false>(ka, sq, sf, sl, tiles, pf, tok0, lane, sum);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
          sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        }
        if (t < 2) {
          const int at = g + 8 * t;
          const float w = t == 0 ? sum[0] : sum[1];
          float* dst = p.mass + ((size_t)page * p.Hkv + kvh) * kPage + at;
          if (tok0 + at < len) *dst = (first && !p.add) ? w : *dst + w;
        }
      }
      first = false;
    }
  }
}

// How a call is cut into CTAs, and what it needs as scratch.
struct Plan {
  int heads, subs, rows, groups, units, uheads, pairs, splits, ctas, sms;
  bool tile;                // 128 pairs a CTA
  long slots;               // parts that are stored
  long floats(long M, long Hq, long D, long observe) const {
    return (splits == 1 ? 0 : slots * pairs * (D + 2)) + (splits == 0 ? 2L * (units + 2) : 0) + (observe ? 2 * M * Hq : 0);
  }
};

int plan(Plan& pl, long M, long Hq, long Hkv, long D, long block, long max_len, long alone) {
  if (!fits(M, 1, 65535) || !fits(Hkv, 1, 65535) || !fits(Hq, 1, 16 * Hkv) || Hq % Hkv || !fits(block, 1, M) || M % block || !fits(max_len, 1, 0x7fffffff)) return -2;
  if (D != 64 && D != 128 && D != 256) return -2;
  const int G = (int)(Hq / Hkv), sms = sm_count();
  if (!sms) return -2;
  // (row, head) pairs of a CTA: one MMA column tile holds 8.  Two tiles where more pairs than that share the keys, except at
  // head_dim 256, whose accumulators fill the registers with one.
  // Tiles of 128 pairs pay where a block has many and the keys are long enough to carry the wider kernel's start (10 us).  Measured,
  // us without / with tiles, observed weight included: 160 pairs, 4 x 16384 tokens x 8 kv heads 375 / 268; 512 pairs at head_dim 64,
  // 2 x 8192 x 4 138 / 104; 96 pairs at head_dim 256, 2 x 8192 x 4 152 / 121; 40 pairs, 4 x 8192 x 8 109 / 104; but 20 pairs of
  // those 94 / 102, 40 pairs, 8192 x 8 56 / 61, 80 pairs, 2001 x 8 44 / 50.
  const long key_pages = (max_len + kPage - 1) / kPage;
  // alone: as in a call of one block, in this as in the cut of the keys below
  pl.tile = block * G >= 40 && (alone ? block : M) * Hq * key_pages >= 256L * 1024;
  const int most = pl.tile ? 128 : (D == 256 ? 8 : 16);
  pl.heads = G < most ? G : most;
  pl.subs = (G + pl.heads - 1) / pl.heads;
  pl.rows = pl.subs > 1 ? 1 : most / G;
  if (pl.rows > block) pl.rows = (int)block;
  pl.groups = (int)((block + pl.rows - 1) / pl.rows);
  if (pl.tile) pl.rows = (int)((block + pl.groups - 1) / pl.groups);       // tiles of like size
  pl.pairs = pl.tile ? 128 : (pl.rows * pl.heads <= 8 ? 8 : 16);
  const long units = M / block * pl.groups;
  if (units > 65535 || Hkv * pl.subs > 65535) return -2;
  pl.units = (int)units;
  pl.uheads = (int)Hkv * pl.subs;
  pl.sms = sms;
  pl.ctas = sms * (pl.tile ? (D == 256 ? Tile<256>::kCtas : Tile<128>::kCtas) : (D == 256 ? Ring<256>::kCtas : Ring<128>::kCtas));
  // alone: the keys of a block are cut as in a call of that block only, so that its rows get the same bits in both
  const long cells = (alone ? pl.groups : units) * pl.uheads, pages = (max_len + kPage - 1) / kPage;
  // Streamed: every CTA gets the same number of pages of the flat list, whatever the rows' lengths, at the price of a scan over
  // the rows and of parts that begin anywhere.  Split: a fixed number of CTAs a unit, at least eight pages (a step of the four
  // warps) each.  Measured, us split / streamed: 8 rows of up to 4999 tokens x 8 heads (45 pages a CTA) 20.7 / 24.5, 16 rows of
  // up to 8191 at head_dim 256 (110 pages) 51.0 / 54.1, 32 rows of up to 32768 (900 pages) 320 / 231.  A single block has nothing to
  // even out and is always split, at whatever length, so that its rows and those of `alone` calls are cut alike: one row of 200000
  // tokens x 8 heads 69.7 / 77.8, of 524288 152 / 156, of 262144 x 4 heads of 256 90 / 90.
  pl.splits = 0;
  if (pl.tile || alone || M == block || units > kMaxUnits || cells * pages < 256L * pl.ctas) {
    long s = pages / 8 < pl.ctas / cells ? pages / 8 : pl.ctas / cells;
    pl.splits = (int)(s < 1 ? 1 : s);
  }
  pl.slots = pl.splits == 0 ? pl.ctas + cells : units * pl.uheads * pl.splits;
  return 0;
}

template <int D, int HH>
int launch_attn(const AttnParams& p, cudaStream_t st) {
  constexpr int kMerge = kWarps * 8 * HH * (D + 4) * 4;
  constexpr int kSmem = Ring<D>::kBytes > kMerge ? Ring<D>::kBytes : kMerge;
  static unsigned long long ready = 0;
  const cudaError_t e = allow_smem(ready, (const void*)attn_kernel<D, HH>, kSmem);
  if (e != cudaSuccess) return (int)e;
  return (int)grm_launch_pdl(GRM_PDL_ATTN, attn_kernel<D, HH>, p.splits ? dim3(p.splits, p.uheads, p.units) : dim3(p.ctas), dim3(kThreads), kSmem, st, p);
}

template <int D>
int launch_tile(const AttnParams& p, cudaStream_t st) {
  static unsigned long long ready = 0;
  const cudaError_t e = allow_smem(ready, (const void*)tile_kernel<D>, Tile<D>::kBytes);
  if (e != cudaSuccess) return (int)e;
  return (int)grm_launch_pdl(GRM_PDL_ATTN, tile_kernel<D>, dim3(p.splits, p.uheads, p.units), dim3(Tile<D>::kThreads), Tile<D>::kBytes, st, p);
}

template <int D>
int launch(const AttnParams& p, int nblocks, int mass_pages, cudaStream_t st) {
  int rc;
  if (p.pairs == 128) rc = launch_tile<D>(p, st);
  else if constexpr (D == 256) rc = launch_attn<D, 1>(p, st);
  else rc = p.pairs == 8 ? launch_attn<D, 1>(p, st) : launch_attn<D, 2>(p, st);
  if (rc) return rc;
  if (p.splits != 1) {
    const dim3 grid(p.Hkv * p.G, p.M);
    const bool many = (p.splits ? p.splits : p.ctas / ((long)p.units * p.uheads)) >= 16;
    const cudaError_t e = many ? grm_launch_pdl(GRM_PDL_ATTN, merge_kernel<D, 512>, grid, dim3(512), 0, st, p)
                               : grm_launch_pdl(GRM_PDL_ATTN, merge_kernel<D, 128>, grid, dim3(128), 0, st, p);
    if (e != cudaSuccess) return (int)e;
  }
  if (p.mass) {
    // pages of a CTA: at least a page a warp, and about a wave of CTAs, four an SM; a quarter more where the pairs are quickly laid out,
    // since CTAs behind the end of a shorter sequence leave at once (one observed row, four sequences of 8192 to 16384 tokens: 92 us
    // of a call that sets and one that adds, against 104 with three waves and 108 with three quarters of one)
    const long cells = (long)mass_pages * p.Hkv * nblocks, ctas = (p.block * p.G <= 32 ? 5L : 4L) * p.sms;
    long per = cells / ctas;
    per = per < 1 ? 1 : per;
    per = (per + kWarps - 1) / kWarps * kWarps;
    static unsigned long long ready = 0;
    const cudaError_t e = allow_smem(ready, (const void*)mass_kernel<D>, MassTile<D>::kBytes);
    if (e != cudaSuccess) return (int)e;
    return (int)grm_launch_pdl(GRM_PDL_ATTN, mass_kernel<D>, dim3((unsigned)((mass_pages + per - 1) / per), p.Hkv, nblocks), dim3(kThreads), MassTile<D>::kBytes,
                               st, p, nblocks, mass_pages, (int)per);
  }
  return 0;
}

}  // namespace

constexpr int kNeedsScratch = -3;      // nothing was launched: the call wants grm_kv4_attn_scratch() words

// Scratch of a call in fp32 words, or -2 for arguments that are not served.
GRM_API long grm_kv4_attn_scratch(int M, int Hq, int Hkv, int D, int block, int max_len, int observe, int alone) {
  Plan pl;
  const int rc = plan(pl, M, Hq, Hkv, D, block, max_len, alone);
  return rc ? rc : pl.floats(M, Hq, D, observe);
}

// One record of 64-bit words (kv4::Args):
//   data, mass (or 0), table, slots, width, stride, pages, q, ld_q, row_seq, row_pos, gate (or 0), ld_gate, out, ld_o, scratch
//   (16-byte aligned, or 0: the call returns -3 where it needs some), M, Hq, Hkv, D, window, scale, block, observe (0 nothing, 1 set, 2 add), max_len,
//   alone
// max_len bounds the positions of the call's rows for the observed weight and sets how the keys are cut.
GRM_API int grm_kv4_attn(const void* words, void* stream) {
  Args a(words);
  AttnParams p;
  p.data = a.ptr<const uint8_t>(); p.mass = a.ptr<float>();
  if (!read_table(a, p.t)) return -2;
  p.q = a.ptr<const bf16>(); p.ld_q = a.num();
  p.row_seq = a.ptr<const int>(); p.row_pos = a.ptr<const int>();
  p.gate = a.ptr<const bf16>(); p.ld_gate = a.num();
  p.out = a.ptr<bf16>(); p.ld_o = a.num();
  float* s = a.ptr<float>();
  const long M = a.num(), Hq = a.num(), Hkv = a.num(), D = a.num(), window = a.num();
  p.scale_log2 = (float)(a.real() * 1.4426950408889634);
  const long block = a.num(), observe = a.num(), max_len = a.num(), alone = a.num();
  Plan pl;
  const int rc = plan(pl, M, Hq, Hkv, D, block, max_len, alone);
  if (rc) return rc;
  if (!fits(observe, 0, 2) || (observe && !p.mass)) return -2;
  if (!s && pl.floats(M, Hq, D, observe)) return kNeedsScratch;
  if (!observe) p.mass = nullptr;
  p.M = (int)M; p.Hkv = (int)Hkv; p.G = (int)(Hq / Hkv); p.window = (int)(fits(window, 1, 0x7fffffff) ? window : 0); p.block = (int)block;
  p.add = observe == 2;
  p.heads = pl.heads; p.subs = pl.subs; p.rows = pl.rows; p.groups = pl.groups;
  p.units = pl.units; p.uheads = pl.uheads; p.splits = pl.splits; p.ctas = pl.ctas; p.pairs = pl.pairs; p.sms = pl.sms;
  p.status = grm_status_ptr();
  p.vec = ((uintptr_t)p.q | (uintptr_t)(2 * p.ld_q)) % 8 == 0;
  p.vec_out = ((uintptr_t)p.out | (uintptr_t)(2 * p.ld_o)) % 4 == 0;
  p.sched = (long long*)s;
  if (pl.splits == 0) s += 2L * (pl.units + 2);
  p.part_o = s;
  if (pl.splits != 1) s += pl.slots * pl.pairs * D;
  p.part_ml = s;
  if (pl.splits != 1) s += pl.slots * pl.pairs * 2;
  p.fin = observe ? s : nullptr;
  const int mass_pages = (int)((max_len + kPage - 1) / kPage < p.t.width ? (max_len + kPage - 1) / kPage : p.t.width);
  switch (D) {
    case 64: return launch<64>(p, p.M / p.block, mass_pages, (cudaStream_t)stream);
    case 128: return launch<128>(p, p.M / p.block, mass_pages, (cudaStream_t)stream);
    default: return launch<256>(p, p.M / p.block, mass_pages, (cudaStream_t)stream);
  }
}
