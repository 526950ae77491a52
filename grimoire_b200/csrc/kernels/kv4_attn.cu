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
constexpr int kMaxSplits = 64;

struct AttnParams {
  const uint8_t* data; float* mass;
  Table t;
  const bf16* q; long ld_q;
  const int* row_seq; const int* row_pos;
  const bf16* gate; long ld_gate;
  bf16* out; long ld_o;
  float* part_o;            // [M][Hkv][splits][G][D]
  float* part_ml;           // [M][Hkv][splits][G][2]
  float* fin;               // [M][Hq][2]: softmax maximum (log2 domain) and reciprocal sum of every row, or null
  unsigned int* status;     // device status block (bounded waits report here)
  int M, Hkv, G, window, block, add;
  int rows, groups;         // rows of a block that share a CTA, groups of them in a block
  int heads, subs;          // query heads of a kv head that share a CTA, CTAs a kv head
  int vec;                  // q rows are 8-byte aligned
  float scale_log2;         // softmax scale * log2(e)
};

__device__ __forceinline__ int row_len(const AttnParams& p, int row) { return max(0, min(p.row_pos[row] + 1, p.t.width * kPage)); }
__device__ __forceinline__ int row_first(const AttnParams& p, int len) { return (p.window > 0 && len > p.window) ? len - p.window : 0; }

template <int D>
struct Ring {
  static constexpr int kStages = D == 256 ? 3 : 4;
  static constexpr int kBytes = kWarps * kStages * Geo<D>::kRecord;
};

__device__ __forceinline__ float deq(const uint8_t* row, const unsigned short* am, int d, int groups) {
  const int c = (row[d >> 1] >> (4 * (d & 1))) & 15;
  return (float)(c - 8) * __uint_as_float((uint32_t)am[(d >> 2) % groups] << 16) * (1.f / 7.f);
}

__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {         // 2 ulp; results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// f16 x f16 -> f32, D += A B
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  attn_mma::mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
}

// Place of token column n (of 8-token tile b) in its page: the columns that lane t of a quad owns in the accumulator fragment
// (2t, 2t + 1) are the tokens t and 4 + (t ^ 1) of the tile, so that neighbouring lanes read rows of different parity and the
// 64-byte rows of a 128-element head meet no bank conflict as the K operand.
__device__ __forceinline__ int tok_of(int b, int n) { return 8 * b + ((n & 1) ? 4 + ((n >> 1) ^ 1) : (n >> 1)); }

// The codes of a 16-bit half word, two words at once (two tokens, or two places of a row): element i of the result holds
// nibble i of x's low half in its low half and of y's in its high half, as the fp16 number code - 8: the nibble becomes the
// last mantissa bits of 1024 (or, four bits higher, of 1024 + 16 code), and one exact fp16 operation takes the offset away.
// (Leaving the offset to the end, with the bare nibbles as fp16 subnormals, saves that operation and was measured to lose five
// bits of the fp32 sums: the MMA aligns a subnormal's product by its unnormalised exponent.)
__device__ __forceinline__ void nibbles(uint32_t x, uint32_t y, bool high, uint32_t (&o)[4]) {
  const uint32_t p = attn_mma::prmt(x, y, high ? 0x7632u : 0x5410u);
  const uint32_t q = p >> 8;
  o[0] = h2_add((p & 0x000f000fu) | 0x64006400u, 0xe408e408u);                       // - 1032
  o[1] = h2_fma((p & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);          // / 16 - 72
  o[2] = h2_add((q & 0x000f000fu) | 0x64006400u, 0xe408e408u);
  o[3] = h2_fma((q & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);
}

__device__ __forceinline__ float exp2_pos(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // 2^e, -127 < e < 128

// Attention of up to 8 * HH (row, head) pairs of one kv head over one split of the sequence's pages.
//
// Bound by the cache's bytes (18 D per 16 tokens and kv head) and, close behind, by issue slots: one warp and page has to take
// less than four times the ~100 cycles in which an SM receives the record.  Hence
//   * a warp owns whole pages; each is ONE bulk copy (the record is contiguous) into a per-warp ring of kStages;
//   * S[pair][token] = Q K^T with the pairs as MMA rows and the codes, as the fp16 integers that they are, as the column
//     operand.  q is scaled by a power of two to fill fp16's range (bf16 has fewer bits: exact); a quantisation group is two
//     k-steps whose sum is scaled by the group's maximum in fp32;
//   * the accumulator fragment of S IS the column operand of O^T[dim][pair] += V^T[dim][token] P^T[token][pair]: no shuffle, and
//     8 pairs fill the MMA's 8 columns.  P is scaled by the token's V maximum before it is rounded to fp16 (11 bits, on top of
//     the output's 8); a running power of two keeps the largest maximum seen at the top of fp16's range, whatever the values'
//     magnitude.
// Softmax statistics, scores and outputs are fp32.
template <int D, int HH>
__global__ void __launch_bounds__(kThreads, D == 256 ? 2 : 3) attn_kernel(const AttnParams p) {
  using Gm = Geo<D>;
  constexpr int NG = Gm::kGroups, WT = D / 64, PP = 8 * HH;
  constexpr int kStages = Ring<D>::kStages;
  constexpr int kOld = D + 4;                           // floats between the pairs of the merge buffer
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ float sm_ml[kWarps][PP][2];
  const int split = blockIdx.x, nsplit = gridDim.x;
  const int kvh = blockIdx.y / p.subs, sub = blockIdx.y % p.subs;
  const int blk = blockIdx.z / p.groups, grp = blockIdx.z % p.groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  // pairs of this CTA: rows row0 .. row0 + nr - 1 of the block x heads head0 .. head0 + nh - 1 of the kv head
  const int row0 = blk * p.block + grp * p.rows, nr = min(p.rows, p.block - grp * p.rows);
  const int head0 = sub * p.heads, nh = min(p.heads, p.G - head0), np = nr * nh;
  const int slot = p.row_seq[blk * p.block];

  int len_hi = 0, len_lo = 0x7fffffff, first_lo = 0x7fffffff, first_hi = 0;      // over the rows that see a key at all
  for (int r = 0; r < nr; ++r) {
    const int len = row_len(p, row0 + r);
    if (len > 0) {
      const int first = row_first(p, len);
      len_hi = max(len_hi, len); len_lo = min(len_lo, len);
      first_lo = min(first_lo, first); first_hi = max(first_hi, first);
    } else {
      len_lo = 0;
    }
  }
  const int page_lo = len_hi > 0 ? first_lo / kPage : 0, page_hi = (len_hi + kPage - 1) / kPage;
  const int pps = (page_hi - page_lo + nsplit - 1) / nsplit;
  const int pbeg = page_lo + split * pps, pend = min(pbeg + pps, page_hi);
  const int n_it = pbeg + warp < pend ? (pend - pbeg - warp + kWarps - 1) / kWarps : 0;      // pages of this warp

  // ---- ring ----
  uint8_t* ring = smem + (size_t)warp * kStages * Gm::kRecord;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[warp][s], 1);
    mbar_fence_init();
  }
  __syncwarp();
  auto load_ids = [&](int base) { return base + lane < n_it ? page_of(p.t, slot, pbeg + warp + kWarps * (base + lane)) : -1; };
  int ids = load_ids(0), ids_next = load_ids(32);        // pages of iterations 32 i + lane and 32 (i + 1) + lane
  auto issue = [&](int it, int id) {
    if (lane == 0) {
      uint64_t* bar = &bars[warp][it % kStages];
      if (id >= 0) {
        mbar_expect_tx(bar, Gm::kRecord);
        bulk_load(ring + (it % kStages) * Gm::kRecord, p.data + ((size_t)id * p.Hkv + kvh) * Gm::kRecord, Gm::kRecord, bar);
      } else {
        mbar_arrive(bar);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (s < n_it) issue(s, __shfl_sync(0xffffffffu, ids, s));

  // ---- q: row operands of S for the pairs g and g + 8 ----
  // k-step (group gi = 2 w + half, odd): the words w and w + NG / 2 of lane t's NG words, nibbles odd and odd + 2
  uint32_t qa[HH][NG][2][2];
  float fh[HH], m[HH], l[HH];
  int lim[HH], low[HH];
#pragma unroll
  for (int x = 0; x < HH; ++x) {
    const int pr = g + 8 * x;
    const bool live = pr < np;
    const int row = row0 + (live ? pr / nh : 0), head = kvh * p.G + head0 + (live ? pr % nh : 0);
    lim[x] = live ? row_len(p, row) : 0;
    low[x] = row_first(p, lim[x]);
    m[x] = -INFINITY; l[x] = 0.f;
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
    const int e = max((int)(mx >> 7), 14);               // biased exponent of the largest magnitude
    const float up = e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(268 - e) << 23);   // 2^14 / 2^(e - 127)
    fh[x] = p.scale_log2 * (1.f / 7.f / 16384.f) * exp2_pos(min(e - 127, 127));                              // 1 / up
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
        for (int j = 0; j < 2; ++j) qa[x][gi][odd][j] = attn_mma::pack_f16x2(a[odd + 2 * j], b[odd + 2 * j]);
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
  uint32_t limit = 4000000u;

  auto page_work = [&](auto edge_tag, const uint8_t* rec, int tok0) {
    constexpr bool kEdge = decltype(edge_tag)::value;    // some token of the page is hidden from some row
    int tk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) tk[i] = tok_of(i >> 1, 2 * t + (i & 1));
    uint32_t am[4][NG];                                  // the lane's tokens: words 0 .. NG / 2 - 1 of K, then of V
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* src = rec + Gm::kAmax + tk[i] * Gm::kAmaxTok;
      if constexpr (NG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        am[i][0] = v.x; am[i][1] = v.y;
      } else {
#pragma unroll
        for (int j = 0; j < NG / 4; ++j) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + 16 * j);
          am[i][4 * j] = v.x; am[i][4 * j + 1] = v.y; am[i][4 * j + 2] = v.z; am[i][4 * j + 3] = v.w;
        }
      }
    }
    auto k_max = [&](int i, int gi) { return (gi & 1) ? bf16hi_to_f(am[i][gi / 2]) : bf16lo_to_f(am[i][gi / 2]); };
    auto v_max = [&](int i, int gi) { return (gi & 1) ? bf16hi_to_f(am[i][NG / 2 + gi / 2]) : bf16lo_to_f(am[i][NG / 2 + gi / 2]); };
    // ---- S ----
    float s[HH][4];
#pragma unroll
    for (int x = 0; x < HH; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint8_t* src = rec + tok_of(b, g) * Gm::kRow + t * (D / 8);
      uint32_t kw[NG];
      if constexpr (NG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        kw[0] = v.x; kw[1] = v.y;
      } else {
#pragma unroll
        for (int j = 0; j < NG / 4; ++j) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + 16 * j);
          kw[4 * j] = v.x; kw[4 * j + 1] = v.y; kw[4 * j + 2] = v.z; kw[4 * j + 3] = v.w;
        }
      }
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        uint32_t nb[4];
        nibbles(kw[gi / 2], kw[gi / 2 + NG / 2], gi & 1, nb);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        mma(c, qa[0][gi][0][0], HH == 2 ? qa[HH - 1][gi][0][0] : 0u, qa[0][gi][0][1], HH == 2 ? qa[HH - 1][gi][0][1] : 0u, nb[0], nb[2]);
        mma(c, qa[0][gi][1][0], HH == 2 ? qa[HH - 1][gi][1][0] : 0u, qa[0][gi][1][1], HH == 2 ? qa[HH - 1][gi][1][1] : 0u, nb[1], nb[3]);
#pragma unroll
        for (int x = 0; x < HH; ++x)
#pragma unroll
          for (int j = 0; j < 2; ++j) s[x][2 * b + j] = fmaf(c[2 * x + j], k_max(2 * b + j, gi), s[x][2 * b + j]);
      }
    }
    if constexpr (kEdge) {                               // a token that no row sees must not set the scale of the values
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tok0 + tk[i] >= len_hi || tok0 + tk[i] < first_lo)
#pragma unroll
          for (int j = 0; j < NG / 2; ++j) am[i][NG / 2 + j] = 0u;
    }
    // ---- running scale of the values: the exponent of the largest finite maximum ----
    uint32_t vm = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NG / 2; ++j) vm = __vmaxu2(vm, am[i][NG / 2 + j]);
    int e = (int)(max(vm & 0xffffu, vm >> 16) >> 7);
    e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
    e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
    if (e >= 255) {                                      // a group that is not a number: it must not hide the others
      e = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          const int one = (int)(__float_as_uint(v_max(i, gi)) >> 23);
          e = one < 255 ? max(e, one) : e;
        }
      e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
      e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
    }
    float corr_e = 1.f;
    if (e > e_run) {
      corr_e = e - e_run < 127 ? exp2_pos(e_run - e) : 0.f;
      e_run = e;
    }
    const float vs = __uint_as_float((uint32_t)(268 - e_run) << 23);           // 2^14 / 2^(e_run - 127): the largest P is below 2^15
    // ---- online softmax ----
    float corr[HH];
    bool change = corr_e != 1.f;
#pragma unroll
    for (int x = 0; x < HH; ++x) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[x][i] *= fh[x];
        if (kEdge && (tok0 + tk[i] >= lim[x] || tok0 + tk[i] < low[x])) s[x][i] = -INFINITY;
        mx = fmaxf(mx, s[x][i]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[x], mx), ref = mn == -INFINITY ? 0.f : mn;
      corr[x] = exp2_fast(m[x] - ref);
      change = change || corr[x] != 1.f;
      m[x] = mn;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[x][i] = exp2_fast(s[x][i] - ref);
        sum += s[x][i];
      }
      l[x] = fmaf(l[x], corr[x], sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] *= vs;
      corr[x] *= corr_e;
    }
    if (__any_sync(0xffffffffu, change)) {
#pragma unroll
      for (int x = 0; x < HH; ++x) {
        const float ca = __shfl_sync(0xffffffffu, corr[x], 8 * t), cb = __shfl_sync(0xffffffffu, corr[x], 8 * t + 4);
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int ii = 0; ii < 2; ++ii) {
            acc[x][gi][ii][0] *= ca; acc[x][gi][ii][1] *= cb; acc[x][gi][ii][2] *= ca; acc[x][gi][ii][3] *= cb;
          }
      }
    }
    // ---- O^T += V^T P^T ----
    uint32_t vw[4][WT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* src = rec + Gm::kV + tk[i] * Gm::kRow + g * (4 * WT);
      if constexpr (WT == 1) {
        vw[i][0] = *reinterpret_cast<const uint32_t*>(src);
      } else if constexpr (WT == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        vw[i][0] = v.x; vw[i][1] = v.y;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        vw[i][0] = v.x; vw[i][1] = v.y; vw[i][2] = v.z; vw[i][3] = v.w;
      }
    }
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      uint32_t pb[HH][2];
#pragma unroll
      for (int x = 0; x < HH; ++x) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = s[x][i] * v_max(i, gi);
          if (kEdge && (tok0 + tk[i] >= lim[x] || tok0 + tk[i] < low[x])) v[i] = 0.f;      // 0 * NaN
        }
        pb[x][0] = attn_mma::pack_f16x2(v[0], v[1]);
        pb[x][1] = attn_mma::pack_f16x2(v[2], v[3]);
      }
      uint32_t v01[4], v23[4];
      nibbles(vw[0][gi / 2], vw[1][gi / 2], gi & 1, v01);
      nibbles(vw[2][gi / 2], vw[3][gi / 2], gi & 1, v23);
#pragma unroll
      for (int ii = 0; ii < 2; ++ii)
#pragma unroll
        for (int x = 0; x < HH; ++x) mma(acc[x][gi][ii], v01[2 * ii], v01[2 * ii + 1], v23[2 * ii], v23[2 * ii + 1], pb[x][0], pb[x][1]);
    }
  };

  for (int it = 0; it < n_it; ++it) {
    const int id = __shfl_sync(0xffffffffu, ids, it & 31);
    const int stage = it % kStages, pg = pbeg + warp + kWarps * it;
    const bool here = __all_sync(0xffffffffu, mbar_wait(&bars[warp][stage], (uint32_t)(it / kStages) & 1u, p.status, 0x4b563400u | warp, limit));
    if (!here) limit = 16;                               // the call has failed: do not wait at length again
    const int tok0 = pg * kPage;
    if (id >= 0 && here) {
      const uint8_t* rec = ring + stage * Gm::kRecord;
      if (tok0 + kPage > len_lo || tok0 < first_hi) page_work(std::true_type{}, rec, tok0);
      else page_work(std::false_type{}, rec, tok0);
    }
    __syncwarp();
    const int nx = it + kStages;
    if (nx < n_it) issue(nx, __shfl_sync(0xffffffffu, (nx >> 5) == (it >> 5) ? ids : ids_next, nx & 31));
    if ((it & 31) == 31) {
      ids = ids_next;
      ids_next = load_ids(((it >> 5) + 2) * 32);
    }
  }
#pragma unroll
  for (int x = 0; x < HH; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    if (t == 0) { sm_ml[warp][g + 8 * x][0] = m[x]; sm_ml[warp][g + 8 * x][1] = l[x]; }
  }
  __syncthreads();                                       // the rings become the merge buffer [warp][pair][nibble of a lane][lane row g]
  float* so = reinterpret_cast<float*>(smem);
  {
    const float fo = exp2_pos(e_run - 127) * (1.f / 7.f / 16384.f);
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
    const int row = row0 + pr / nh, hd = head0 + pr % nh;
    const size_t pi = (((size_t)row * p.Hkv + kvh) * nsplit + split) * p.G + hd;
    *reinterpret_cast<float2*>(p.part_o + pi * D + d) = make_float2(o[0], o[1]);
    if (d == 0) { p.part_ml[2 * pi] = mx; p.part_ml[2 * pi + 1] = ls; }
  }
}

// Joins the splits of a row in split order, applies the gate, leaves (maximum, 1 / sum) for the weights.
__global__ void __launch_bounds__(128) merge_kernel(const AttnParams p, int nsplit, int D) {
  const int kvh = blockIdx.y, row = blockIdx.z, g = blockIdx.x;
  const size_t pi = ((size_t)row * p.Hkv + kvh) * nsplit * p.G + g;
  float mx = -INFINITY;
  for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, p.part_ml[2 * (pi + (size_t)s * p.G)]);
  float l = 0.f;
  for (int s = 0; s < nsplit; ++s) {
    const float* ml = p.part_ml + 2 * (pi + (size_t)s * p.G);
    if (ml[1] != 0.f) l += (ml[0] == -INFINITY ? 1.f : exp2f(ml[0] - mx)) * ml[1];
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int head = kvh * p.G + g;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float o = 0.f;
    for (int s = 0; s < nsplit; ++s) {
      const size_t at = pi + (size_t)s * p.G;
      const float* ml = p.part_ml + 2 * at;
      if (ml[1] != 0.f) o += (ml[0] == -INFINITY ? 1.f : exp2f(ml[0] - mx)) * p.part_o[at * D + d];
    }
    o = l != 0.f ? o * inv : 0.f;
    if (p.gate) o *= 1.f / (1.f + __expf(-__bfloat162float(p.gate[(size_t)row * p.ld_gate + (size_t)head * D + d])));
    p.out[(size_t)row * p.ld_o + (size_t)head * D + d] = __float2bfloat16(o);
  }
  if (p.fin && threadIdx.x == 0) {
    p.fin[2 * ((size_t)row * p.Hkv * p.G + head)] = mx;
    p.fin[2 * ((size_t)row * p.Hkv * p.G + head) + 1] = inv;
  }
}

// One CTA per (page, kv head, block of rows).  All rows of one sequence are summed by the CTA of its first block, in the
// order of the rows, so that two blocks of one sequence neither race nor depend on the order of CTAs.
template <int D>
__global__ void __launch_bounds__(128) mass_kernel(const AttnParams p, int nblocks) {
  using Gm = Geo<D>;
  __shared__ float sk[kPage][D + 1];
  __shared__ float part[8][kPage];
  __shared__ int s_len;
  const int pg = blockIdx.x, kvh = blockIdx.y, blk = blockIdx.z;
  const int tid = threadIdx.x;
  const int slot = p.row_seq[blk * p.block];
  for (int b = 0; b < blk; ++b)
    if (p.row_seq[b * p.block] == slot) return;
  const int page = page_of(p.t, slot, pg);
  if (page < 0) return;
  if (tid == 0) {
    int len = 0;
    for (int b = blk; b < nblocks; ++b)
      if (p.row_seq[b * p.block] == slot)
        for (int r = 0; r < p.block; ++r) len = max(len, p.row_pos[b * p.block + r] + 1);
    s_len = len;
  }
  const uint8_t* rec = p.data + ((size_t)page * p.Hkv + kvh) * Gm::kRecord;
  for (int i = tid; i < kPage * D; i += 128) {
    const int tok = i / D, d = i % D;
    sk[tok][d] = deq(rec + tok * Gm::kRow, reinterpret_cast<const unsigned short*>(rec + Gm::kAmax + tok * Gm::kAmaxTok), d, Gm::kGroups);
  }
  __syncthreads();
  const int tok = tid & 15, part_id = tid >> 4, t = pg * kPage + tok;
  float sum = 0.f;
  for (int b = blk; b < nblocks; ++b) {
    if (p.row_seq[b * p.block] != slot) continue;
    for (int i = part_id; i < p.block * p.G; i += 8) {
      const int row = b * p.block + i / p.G, head = kvh * p.G + i % p.G;
      const int len = p.row_pos[row] + 1, first = (p.window > 0 && len > p.window) ? len - p.window : 0;
      if (t >= len || t < first) continue;
      const bf16* q = p.q + (size_t)row * p.ld_q + (size_t)head * D;
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(__bfloat162float(q[d]), sk[tok][d], s);
      const float* f = p.fin + 2 * ((size_t)row * p.Hkv * p.G + head);
      sum += exp2f(s * p.scale_log2 - f[0]) * f[1];
    }
  }
  part[part_id][tok] = sum;
  __syncthreads();
  if (part_id == 0 && t < min(s_len, p.t.width * kPage)) {
    float w = 0.f;
    for (int i = 0; i < 8; ++i) w += part[i][tok];
    float* dst = p.mass + ((size_t)page * p.Hkv + kvh) * kPage + tok;
    *dst = p.add ? *dst + w : w;
  }
}

template <int D, int HH>
int launch_attn(const AttnParams& p, int splits, int nblocks, cudaStream_t st) {
  constexpr int kMerge = kWarps * 8 * HH * (D + 4) * 4;
  constexpr int kSmem = Ring<D>::kBytes > kMerge ? Ring<D>::kBytes : kMerge;
  cudaError_t e = cudaFuncSetAttribute(attn_kernel<D, HH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return (int)e;
  attn_kernel<D, HH><<<dim3(splits, p.Hkv * p.subs, nblocks * p.groups), kThreads, kSmem, st>>>(p);
  GRM_LAUNCH_RET();
}

template <int D>
int launch(AttnParams p, int splits, int nblocks, int mass_pages, cudaStream_t st) {
  // (row, head) pairs of a CTA: one MMA column tile holds 8.  Two tiles where more pairs than that share the keys, except at
  // head_dim 256, whose accumulators fill the registers with one.
  constexpr int kMost = D == 256 ? 8 : 16;
  p.heads = p.G < kMost ? p.G : kMost;
  p.subs = (p.G + p.heads - 1) / p.heads;
  p.rows = p.subs > 1 ? 1 : kMost / p.G;
  if (p.rows > p.block) p.rows = p.block;
  p.groups = (p.block + p.rows - 1) / p.rows;
  if ((long)p.Hkv * p.subs > 65535 || (long)nblocks * p.groups > 65535) return -2;
  int rc;
  if constexpr (D == 256) rc = launch_attn<D, 1>(p, splits, nblocks, st);
  else rc = p.rows * p.heads <= 8 ? launch_attn<D, 1>(p, splits, nblocks, st) : launch_attn<D, 2>(p, splits, nblocks, st);
  if (rc) return rc;
  merge_kernel<<<dim3(p.G, p.Hkv, p.M), 128, 0, st>>>(p, splits, D);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  if (p.mass) mass_kernel<D><<<dim3(mass_pages, p.Hkv, nblocks), 128, 0, st>>>(p, nblocks);
  GRM_LAUNCH_RET();
}

}  // namespace

// Scratch of a call in fp32 words: the split partials and, with ``observe``, the softmax statistics of every row.
GRM_API long grm_kv4_attn_scratch(int M, int Hq, int D, int splits, int observe) {
  return (long)M * Hq * splits * (D + 2) + (observe ? 2L * M * Hq : 0);
}

// observe: 0 nothing, 1 set, 2 add.  max_len bounds the positions of the call's rows for the observed weight.
GRM_API int grm_kv4_attn(const void* data, void* mass, const void* table, int slots_n, int width, long stride, int pages, const void* q, long ld_q,
                         const void* row_seq, const void* row_pos, const void* gate, long ld_gate, void* out, long ld_o, void* scratch, int M, int Hq,
                         int Hkv, int D, int splits, int window, float scale, int block, int observe, int max_len, void* stream) {
  if (M < 1 || M > 65535 || Hkv < 1 || Hkv > 65535 || Hq % Hkv || Hq / Hkv > 16 || splits < 1 || splits > kMaxSplits || block < 1 || M % block) return -2;
  if (!table || slots_n < 1 || width < 1 || width > (1 << 27) || pages < 1 || !scratch || (observe && !mass) || max_len < 1) return -2;
  AttnParams p;
  p.data = (const uint8_t*)data; p.mass = observe ? (float*)mass : nullptr;
  p.t = Table{(const int*)table, slots_n, width, stride, pages};
  p.q = (const bf16*)q; p.ld_q = ld_q; p.row_seq = (const int*)row_seq; p.row_pos = (const int*)row_pos;
  p.gate = (const bf16*)gate; p.ld_gate = ld_gate; p.out = (bf16*)out; p.ld_o = ld_o;
  p.M = M; p.Hkv = Hkv; p.G = Hq / Hkv; p.window = window; p.block = block; p.add = observe == 2;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = grm_status_ptr();
  p.vec = ((uintptr_t)q | (uintptr_t)(2 * ld_q)) % 8 == 0;
  p.part_o = (float*)scratch;
  p.part_ml = p.part_o + (size_t)M * Hq * splits * D;
  p.fin = observe ? p.part_ml + (size_t)M * Hq * splits * 2 : nullptr;
  const int mass_pages = (max_len + kPage - 1) / kPage < width ? (max_len + kPage - 1) / kPage : width;
  switch (D) {
    case 64: return launch<64>(p, splits, M / block, mass_pages, (cudaStream_t)stream);
    case 128: return launch<128>(p, splits, M / block, mass_pages, (cudaStream_t)stream);
    case 256: return launch<256>(p, splits, M / block, mass_pages, (cudaStream_t)stream);
    default: return -2;
  }
}
