// Writing, reading back, selecting and moving tokens of the 4-bit KV cache (page layout: kv4.cuh).
//   kv4_append    bf16 K / V rows -> codes and maxima of their page slots (mass of the token starts at zero)
//   kv4_gather    pages -> dense bf16 rows of whole sequences (what prompt attention over a cached history works on)
//   kv4_select    per (sequence, kv head) the tokens that stay when the cache is cut to `keep` tokens
//   kv4_compact   moves those tokens to fresh pages
#include "kv4.cuh"

namespace {

using namespace kv4;

// ---------------------------------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------------------------------
struct AppendParams {
  uint8_t* data; float* mass;
  const bf16* k; const bf16* v; long ld_k, ld_v;
  const int* row_pos; const int* row_seq;
  Table t;
  int M, Hkv, vec;
};

// A warp per row and head: the 2 * D / 4 quads of K and V go round the lanes, so a lane's quads all lie in one group and
// the group's maximum is a butterfly over the lanes with the same (K / V, quad mod groups).
//
// The codes equal those of 64-bit arithmetic.  7 x / maximum is a quotient of an 11-bit and an 8-bit integer (times a power of
// two): it either is a multiple of one half, or at least 2^-13 away from one.  Both are first scaled by a power of two that brings
// the maximum near one (exact, nothing overflows); x7 times the approximate reciprocal, corrected by its exact residual once, is
// within an ulp of the quotient and equals it where it is a multiple of one half; adding 1.5 * 2^23 rounds to even.
//
// kHeads heads of a row a warp: one where there are few rows, four (their loads in flight together, one look into the table) where
// there are many.
//
// 4096 rows x 8 heads x 128 (21.5 MB in and out, part of it from L2) take 8.9 us, 2.4 TB/s, where the bytes alone take 3.3: a warp
// loads once, computes and leaves, so the wait for its loads is the largest stall (5.3 an issue; issue slots 60 % busy, integer pipe
// 49 %).  One row takes 1.8 us, which is a launch in a graph.
template <int D, int kHeads>
__global__ void __launch_bounds__(128) append_kernel(const AppendParams p) {
  using G = Geo<D>;
  constexpr int kQuads = D / 4, kRegs = (2 * kQuads + 31) / 32;
  grm_pdl_wait();
  const long wid = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int sets = (p.Hkv + kHeads - 1) / kHeads;
  if (wid >= (long)p.M * sets) return;
  const int row = (int)(wid / sets), h0 = (int)(wid % sets) * kHeads;
  const int pos = p.row_pos[row];
  const int page = pos < 0 ? -1 : page_of(p.t, p.row_seq[row], pos / kPage);
  if (page < 0) return;
  const int slot = pos % kPage;
  uint2 x[kHeads][kRegs];          // 4 bf16 each
#pragma unroll
  for (int n = 0; n < kHeads; ++n)
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int idx = lane + 32 * i, which = idx / kQuads, quad = idx % kQuads;
      const bf16* src = (which ? p.v + (size_t)row * p.ld_v : p.k + (size_t)row * p.ld_k) + (size_t)min(h0 + n, p.Hkv - 1) * D + 4 * quad;
      if (p.vec) {
        x[n][i] = *reinterpret_cast<const uint2*>(src);
      } else {
        const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
        x[n][i].x = s[0] | ((uint32_t)s[1] << 16);
        x[n][i].y = s[2] | ((uint32_t)s[3] << 16);
      }
    }
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    if (h0 + n >= p.Hkv) break;
    // magnitude bits order like the values, with infinity and then NaN on top
    uint32_t mx[kRegs];
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const uint32_t m = __vmaxu2(x[n][i].x & 0x7fff7fffu, x[n][i].y & 0x7fff7fffu);
      mx[i] = max(m & 0xffffu, m >> 16);
    }
    if constexpr (D == 256) {                     // registers 0, 1 are K, 2, 3 are V; both quads of a lane are in group lane % 8
      mx[0] = mx[1] = max(mx[0], mx[1]);
      mx[2] = mx[3] = max(mx[2], mx[3]);
    }
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      if (D == 256 && (i & 1)) { mx[i] = mx[i - 1]; continue; }
#pragma unroll
      for (int o = G::kGroups; o < (kQuads < 32 ? kQuads : 32); o <<= 1) mx[i] = max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
    }
    uint8_t* rec = p.data + ((size_t)page * p.Hkv + h0 + n) * G::kRecord;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int idx = lane + 32 * i, which = idx / kQuads, quad = idx % kQuads;
      const int e = (int)(mx[i] >> 7);                    // biased exponent of the maximum
      const float scale = __uint_as_float((uint32_t)max(254 - e, 1) << 23), top = __uint_as_float(mx[i] << 16) * scale;
      float r;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(top));
      const bool ok = mx[i] > 0u && mx[i] < 0x7f80u;      // an empty group has codes of zero; one that is not finite reads back as NaN
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = j < 2 ? x[n][i].x : x[n][i].y;
        const float f = (j & 1) ? bf16hi_to_f(b) : bf16lo_to_f(b);
        const float x7 = f * scale * 7.f, t = x7 * r;
        const float q = fmaf(fmaf(-t, top, x7), r, t) + 12582920.f;      // 1.5 * 2^23 + 8: the code in the last bits
        word |= (ok ? __float_as_uint(q) & 15u : 8u) << (4 * j);
      }
      const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
      if (!(lane & 1)) *reinterpret_cast<uint32_t*>(rec + which * G::kV + slot * G::kRow + 2 * quad) = word | (other << 16);
      if (quad < G::kGroups)
        *reinterpret_cast<unsigned short*>(rec + G::kAmax + slot * G::kAmaxTok + 2 * (which * G::kGroups + quad)) = (unsigned short)mx[i];
    }
    if (p.mass && lane == 0) p.mass[((size_t)page * p.Hkv + h0 + n) * kPage + slot] = 0.f;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// gather
// ---------------------------------------------------------------------------------------------------------------------
struct GatherParams {
  const uint8_t* data;
  Table t;
  const int* slots; const int* lengths;
  bf16* out_k; bf16* out_v;
  long ld_k, ld_v, batch_k, batch_v;
  int T, Hkv, vec;
};

// One CTA per (page, kv head, sequence): the record is read once, 8 elements (a word of codes) a thread and turn.  code * maximum / 7
// is a ratio of integers of 11 and 3 bits: it is a bf16 or lies at least 2^-12 from a rounding boundary, so the product with the
// rounded seventh of the maximum rounds to the same bf16 as the exact value.  Bound by bytes, most of them written: 36001 tokens x 8 heads
// x 128 (190 MB) take 35 us, 5.4 TB/s, 0.82 of a copy; one thousand 2.4 us.
template <int D>
__global__ void __launch_bounds__(128) gather_kernel(const GatherParams p) {
  using G = Geo<D>;
  constexpr int kWords = D / 8, kTurns = 2 * kPage * kWords / 128;
  const int s = blockIdx.z, h = blockIdx.y, pg = blockIdx.x;
  grm_pdl_wait();
  const int slot = p.slots ? p.slots[s] : s;
  const int len = p.lengths ? min(p.lengths[s], p.T) : p.T;
  if (pg * kPage >= len) return;
  const int page = page_of(p.t, slot, pg);
  if (page < 0) return;
  const uint8_t* rec = p.data + ((size_t)page * p.Hkv + h) * G::kRecord;
  uint32_t c[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) c[k] = __ldg(reinterpret_cast<const uint32_t*>(rec) + threadIdx.x + 128 * k);
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int i = threadIdx.x + 128 * k, which = i / (kPage * kWords), in = i / kWords % kPage, w = i % kWords;
    const int tok = pg * kPage + in;
    if (tok >= len) continue;
    const uint32_t am = __ldg(reinterpret_cast<const uint32_t*>(rec + G::kAmax + in * G::kAmaxTok + 2 * which * G::kGroups) + w % (G::kGroups / 2));
    const float a[2] = {bf16lo_to_f(am) * (1.f / 7.f), bf16hi_to_f(am) * (1.f / 7.f)};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[2];
#pragma unroll
      for (int y = 0; y < 2; ++y)                        // 2^23 + code, less 2^23 + 8
        v[y] = (__uint_as_float(((c[k] >> (8 * j + 4 * y)) & 15u) | 0x4b000000u) - 8388616.f) * a[j >> 1];
      o[j] = pack_bf16x2(v[0], v[1]);
    }
    bf16* dst = which ? p.out_v + s * p.batch_v + tok * p.ld_v : p.out_k + s * p.batch_k + tok * p.ld_k;
    dst += (size_t)h * D + 8 * w;
    if (p.vec) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
      unsigned short* d = reinterpret_cast<unsigned short*>(dst);
#pragma unroll
      for (int j = 0; j < 4; ++j) { d[2 * j] = (unsigned short)o[j]; d[2 * j + 1] = (unsigned short)(o[j] >> 16); }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// select
// ---------------------------------------------------------------------------------------------------------------------
struct SelectParams {
  const float* mass;
  Table t;
  const int* slots; const int* lengths;
  int* idx;                // [S][Hkv][keep]
  int Hkv, keep, recent, sink;
};

// Order of fp32 values as unsigned integers; NaN, like a token without a page, comes last.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;
  if ((b << 1) == 0u) return 0x80000000u;                   // -0 and +0 are equal
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int kSelThreads = 1024, kSelBins = 2048;
constexpr int kSelKeys = 32768;          // keys that a CTA keeps in shared memory

__device__ __forceinline__ void cluster_sync_() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_load(const int* local, int rank) {      // the same variable of another CTA of the cluster
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
// Inclusive sums over the CTA's threads.
__device__ __forceinline__ int block_scan(int v, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = lane < warp ? warp_sums[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  __syncthreads();
  return v + before;
}

// One cluster of CTAs per (kv head, sequence), each with a stretch of the tokens whose keys it reads once into shared memory (a
// stretch too long for that is read again in every pass).  Radix selection: three passes of 11, 11 and 10 bits over the tokens
// that are neither among the first `sink` nor the last `recent` find the key of the last token that stays and how many tokens
// of exactly that key do, the earliest ones; the histograms of the cluster are added through distributed shared memory.  Then
// every warp writes the kept positions of its own stretch behind those of the stretches before it.  2000 tokens x 8 heads take 10 us,
// the barriers and launch of a few short passes; eight sequences of up to 32768 27 us, one of 100000 37 us, where the 4 bytes a token
// take 1.3: five walks over the keys in shared memory (issue slots 57 % busy; per issue 2.7 cycles of fixed-latency waits, 2.1 for
// loads, 1.5 at barriers).
__global__ void __launch_bounds__(kSelThreads) select_kernel(const SelectParams p, int nctas) {
  extern __shared__ __align__(16) uint32_t keys[];       // [kSelKeys]
  __shared__ int hist[kSelBins];
  __shared__ int warp_sums[32], w_eq[33], w_gt[33], s_bin, s_left, tot[2];
  const int rank = (int)(blockIdx.x % nctas), h = blockIdx.x / nctas, s = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grm_pdl_wait();
  const int slot = p.slots ? p.slots[s] : s;
  const int n = max(0, min(p.lengths[s], p.t.width * kPage));
  int* out = p.idx + ((size_t)s * p.Hkv + h) * p.keep;
  if (n <= p.keep) {
    for (int i = rank * kSelThreads + tid; i < p.keep; i += nctas * kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int lo = min(p.sink, n), hi = max(n - p.recent, lo);
  const int per = (n + nctas * kPage - 1) / (nctas * kPage) * kPage;
  const int beg = min(rank * per, n), end = min(beg + per, n), len = end - beg;
  const bool cached = per <= kSelKeys;
  auto key_of = [&](int t) -> uint32_t {
    const int page = page_of(p.t, slot, t / kPage);
    return page < 0 ? 0u : order_key(__ldg(p.mass + ((size_t)page * p.Hkv + h) * kPage + t % kPage));
  };
  if (cached) {                                          // four tokens of a page a thread
    for (int i = 4 * tid; i < len; i += 4 * kSelThreads) {
      const int page = page_of(p.t, slot, (beg + i) / kPage);
      uint4 k = make_uint4(0u, 0u, 0u, 0u);
      if (page >= 0) {
        const float4 m = __ldg(reinterpret_cast<const float4*>(p.mass + ((size_t)page * p.Hkv + h) * kPage + (beg + i) % kPage));
        k = make_uint4(order_key(m.x), order_key(m.y), order_key(m.z), order_key(m.w));
      }
      *reinterpret_cast<uint4*>(keys + i) = k;
    }
  }
  auto key = [&](int t) -> uint32_t { return cached ? keys[t - beg] : key_of(t); };
  const int want = p.keep - lo - (n - hi);               // tokens to take from [lo, hi); fewer than there are
  uint32_t prefix = 0;
  int need = want;
  const int from = max(beg, lo), to = min(end, hi);
#pragma unroll 1
  for (int pass = 0; pass < 3 && want > 0; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
    const int above = pass == 1 ? 21 : 10;               // bits below those that are settled
    for (int b = tid; b < kSelBins; b += kSelThreads) hist[b] = 0;
    __syncthreads();
    for (int base = from; base < to; base += kSelThreads) {
      const int t = base + tid;
      const uint32_t k = t < to ? key(t) : 0u;
      const bool in = t < to && (pass == 0 || (k >> above) == prefix);
      // tokens that were never looked at share one key: a warp counts them together
      const bool zero = in && k == 0x80000000u;
      const uint32_t zeros = __ballot_sync(0xffffffffu, zero);
      if (in && !zero) atomicAdd(&hist[(k >> shift) & digits], 1);
      if (zeros && lane == 0) atomicAdd(&hist[(0x80000000u >> shift) & digits], __popc(zeros));
    }
    cluster_sync_();
    // bins in falling order, two a thread
    const int b1 = kSelBins - 1 - 2 * tid, b0 = b1 - 1;
    int c1 = 0, c0 = 0;
    for (int r = 0; r < nctas; ++r) { c1 += cluster_load(&hist[b1], r); c0 += cluster_load(&hist[b0], r); }
    const int sum = block_scan(c1 + c0, warp_sums), before = sum - c1 - c0;
    if (before < need && need <= sum) {
      const bool first = need <= before + c1;
      s_bin = first ? b1 : b0;
      s_left = need - before - (first ? 0 : c1);
    }
    cluster_sync_();                                     // s_bin is there; nobody reads this pass's histogram any more
    prefix = pass == 2 ? (prefix << 10) | (uint32_t)s_bin : (prefix << 11) | (uint32_t)s_bin;
    need = s_left;
  }
  if (cached) __syncthreads();                           // (no pass has run where nothing is wanted)
  // prefix: the key of the last kept token; need: how many tokens with that key stay
  auto rank_of = [&](int t, bool& gt, bool& eq) {
    const bool cand = t >= lo && t < hi;
    const uint32_t k = (cand && want > 0) ? key(t) : 0u;
    gt = !cand || (want > 0 && k > prefix);
    eq = cand && want > 0 && k == prefix;
  };
  const int wper = (len + 32 * 32 - 1) / (32 * 32) * 32, wbeg = beg + min(warp * wper, len), wend = min(wbeg + wper, end);
  int n_gt = 0, n_eq = 0;
  for (int t = wbeg + lane; t < wend; t += 32) {
    bool gt, eq;
    rank_of(t, gt, eq);
    n_gt += gt; n_eq += eq;
  }
  n_gt = __reduce_add_sync(0xffffffffu, n_gt);
  n_eq = __reduce_add_sync(0xffffffffu, n_eq);
  if (lane == 0) { w_gt[warp] = n_gt; w_eq[warp] = n_eq; }
  __syncthreads();
  if (tid == 0) {
    int a = 0, b = 0;
    for (int w = 0; w < 32; ++w) { a += w_gt[w]; b += w_eq[w]; }
    tot[0] = a; tot[1] = b;
  }
  cluster_sync_();
  int gt_before = 0, eq_before = 0;
  for (int r = 0; r < rank; ++r) { gt_before += cluster_load(&tot[0], r); eq_before += cluster_load(&tot[1], r); }
  for (int w = 0; w < warp; ++w) { gt_before += w_gt[w]; eq_before += w_eq[w]; }
  for (int t0 = wbeg; t0 < wend; t0 += 32) {
    const int t = t0 + lane;
    bool gt = false, eq = false;
    if (t < wend) rank_of(t, gt, eq);
    const uint32_t gts = __ballot_sync(0xffffffffu, gt), eqs = __ballot_sync(0xffffffffu, eq), under = (1u << lane) - 1u;
    const int eq_here = eq_before + __popc(eqs & under);
    const int to = gt_before + __popc(gts & under) + min(eq_here, need);
    if ((gt || (eq && eq_here < need)) && to < p.keep) out[to] = t;          // (more only where the weights change meanwhile)
    gt_before += __popc(gts);
    eq_before += __popc(eqs);
  }
  cluster_sync_();                                       // the totals stay readable until everybody has read them
}

// ---------------------------------------------------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------------------------------------------------
struct CompactParams {
  uint8_t* data; float* mass;
  Table src;
  const int* slots;
  const int* idx;          // [S][Hkv][keep]
  const int* dst; long dst_stride;      // fresh pages [S][>= ceil(keep / 16)]
  int Hkv, keep;
};

// One CTA per (eight pages of kept tokens, kv head, sequence): the sources of its 128 tokens are looked up side by side, then codes and
// maxima are copied as they are, 16 bytes (the maxima at head_dim 64: 8) a thread and turn, loads ahead of stores.  Eight times 4096 of
// 32768 tokens x 8 heads x 128 (80 MB) take 23 us, 3.4 TB/s: rows of 64 bytes from all over the cache (64 tokens a CTA: the same).
constexpr int kMoveTokens = 128;
template <int D>
__global__ void __launch_bounds__(256) compact_kernel(const CompactParams p) {
  using G = Geo<D>;
  constexpr int kRowUnits = G::kRow / 16;                // units of a token's K (or V) codes
  constexpr int kTurns = kMoveTokens * 2 * kRowUnits / 256;
  __shared__ long long from[kMoveTokens], to[kMoveTokens];       // (page * kv heads + head) * 16 + place; -1: nothing to move
  const int s = blockIdx.z, h = blockIdx.y, j0 = blockIdx.x * kMoveTokens;
  grm_pdl_wait();
  if (threadIdx.x < kMoveTokens) {
    const int j = j0 + threadIdx.x;
    long long a = -1, b = -1;
    if (j < p.keep) {
      const int t = p.idx[((size_t)s * p.Hkv + h) * p.keep + j], dst = p.dst[(size_t)s * p.dst_stride + j / kPage];
      const int page = t < 0 ? -1 : page_of(p.src, p.slots ? p.slots[s] : s, t / kPage);
      if (page >= 0 && (unsigned)dst < (unsigned)p.src.pages) {
        a = ((long long)page * p.Hkv + h) * kPage + t % kPage;
        b = ((long long)dst * p.Hkv + h) * kPage + j % kPage;
        if (p.mass) p.mass[b] = p.mass[a];
      }
    }
    from[threadIdx.x] = a; to[threadIdx.x] = b;
  }
  __syncthreads();
  auto record = [&](long long at) { return p.data + (size_t)(at / kPage) * G::kRecord; };
  uint4 v[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int i = threadIdx.x + 256 * k, tok = i / (2 * kRowUnits), u = i % (2 * kRowUnits);
    const long long a = from[tok];
    if (a >= 0) v[k] = *reinterpret_cast<const uint4*>(record(a) + (u / kRowUnits) * G::kV + (int)(a % kPage) * G::kRow + 16 * (u % kRowUnits));
  }
  constexpr int kAmaxUnits = G::kAmaxTok / 8, kMaxTurns = (kMoveTokens * kAmaxUnits + 255) / 256;
  uint2 m[kMaxTurns];
#pragma unroll
  for (int k = 0; k < kMaxTurns; ++k) {
    const int i = threadIdx.x + 256 * k, tok = i / kAmaxUnits;
    if (tok < kMoveTokens && from[tok] >= 0)
      m[k] = *reinterpret_cast<const uint2*>(record(from[tok]) + G::kAmax + (int)(from[tok] % kPage) * G::kAmaxTok + 8 * (i % kAmaxUnits));
  }
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int i = threadIdx.x + 256 * k, tok = i / (2 * kRowUnits), u = i % (2 * kRowUnits);
    const long long b = to[tok];
    if (b >= 0) *reinterpret_cast<uint4*>(record(b) + (u / kRowUnits) * G::kV + (int)(b % kPage) * G::kRow + 16 * (u % kRowUnits)) = v[k];
  }
#pragma unroll
  for (int k = 0; k < kMaxTurns; ++k) {
    const int i = threadIdx.x + 256 * k, tok = i / kAmaxUnits;
    if (tok < kMoveTokens && to[tok] >= 0)
      *reinterpret_cast<uint2*>(record(to[tok]) + G::kAmax + (int)(to[tok] % kPage) * G::kAmaxTok + 8 * (i % kAmaxUnits)) = m[k];
  }
}

}  // namespace

// CALL, which returns, with DD for the head dimension
#define KV4_DISPATCH(D, ...)                                    \
  switch (D) {                                                  \
    case 64: { constexpr int DD = 64; __VA_ARGS__; }            \
    case 128: { constexpr int DD = 128; __VA_ARGS__; }          \
    case 256: { constexpr int DD = 256; __VA_ARGS__; }          \
    default: return -2;                                         \
  }

// Every entry point takes its arguments as one record of 64-bit words (kv4::Args), in the order of the list above it.

// data, mass (or 0), table, slots, width, stride, pages, k, v, ld_k, ld_v, row_pos, row_seq, M, Hkv, D, vec (rows 8-byte aligned)
// data: uint8 [pages][Hkv][18 * D]; mass: fp32 [pages][Hkv][16]; k / v: bf16 rows of Hkv * D.
GRM_API int grm_kv4_append(const void* words, void* stream) {
  Args a(words);
  AppendParams p;
  p.data = a.ptr<uint8_t>(); p.mass = a.ptr<float>();
  if (!read_table(a, p.t)) return -2;
  p.k = a.ptr<const bf16>(); p.v = a.ptr<const bf16>(); p.ld_k = a.num(); p.ld_v = a.num();
  p.row_pos = a.ptr<const int>(); p.row_seq = a.ptr<const int>();
  const long M = a.num(), Hkv = a.num(), D = a.num();
  p.vec = a.num() != 0;
  if (!fits(M, 1, 0x7fffffff) || !fits(Hkv, 1, 0x7fffffff) || (M * Hkv + 3) / 4 > 0x7fffffffL) return -2;
  p.M = (int)M; p.Hkv = (int)Hkv;
  if (M * Hkv < 8192) {
    KV4_DISPATCH(D, return (int)grm_launch_pdl(GRM_PDL_ATTN, append_kernel<DD, 1>, dim3((unsigned)((M * Hkv + 3) / 4)), dim3(128), 0, (cudaStream_t)stream, p));
  } else {
    KV4_DISPATCH(D, return (int)grm_launch_pdl(GRM_PDL_ATTN, append_kernel<DD, 4>, dim3((unsigned)((M * ((Hkv + 3) / 4) + 3) / 4)), dim3(128), 0, (cudaStream_t)stream, p));
  }
}

// data, table, slots, width, stride, pages, seq (or 0), lengths (or 0), out_k, out_v, ld_k, ld_v, batch_k, batch_v, S, T, Hkv, D,
// vec (rows 16-byte aligned).  out_k / out_v: bf16 [S][T][Hkv * D], strides in elements.
GRM_API int grm_kv4_gather(const void* words, void* stream) {
  Args a(words);
  GatherParams p;
  p.data = a.ptr<const uint8_t>();
  if (!read_table(a, p.t)) return -2;
  p.slots = a.ptr<const int>(); p.lengths = a.ptr<const int>(); p.out_k = a.ptr<bf16>(); p.out_v = a.ptr<bf16>();
  p.ld_k = a.num(); p.ld_v = a.num(); p.batch_k = a.num(); p.batch_v = a.num();
  const long S = a.num(), T = a.num(), Hkv = a.num(), D = a.num();
  p.vec = a.num() != 0;
  if (!fits(S, 1, 65535) || !fits(T, 1, 0x7fffffff - kPage) || !fits(Hkv, 1, 65535)) return -2;
  p.T = (int)T; p.Hkv = (int)Hkv;
  KV4_DISPATCH(D, return (int)grm_launch_pdl(GRM_PDL_ATTN, gather_kernel<DD>, dim3((unsigned)((T + kPage - 1) / kPage), (unsigned)Hkv, (unsigned)S), dim3(128), 0, (cudaStream_t)stream, p));
}

// mass, table, slots, width, stride, pages, seq (or 0), lengths, idx (int32 [S][Hkv][keep]), S, Hkv, keep, recent, sink
GRM_API int grm_kv4_select(const void* words, void* stream) {
  Args a(words);
  SelectParams p;
  p.mass = a.ptr<const float>();
  if (!read_table(a, p.t)) return -2;
  p.slots = a.ptr<const int>(); p.lengths = a.ptr<const int>(); p.idx = a.ptr<int>();
  const long S = a.num(), Hkv = a.num(), keep = a.num(), recent = a.num(), sink = a.num();
  if (!fits(S, 1, 65535) || !fits(Hkv, 1, 0x7fffffff) || !fits(keep, 1, 0x7fffffff) || !fits(recent, 0, keep) || !fits(sink, 0, keep - recent)) return -2;
  p.Hkv = (int)Hkv; p.keep = (int)keep; p.recent = (int)recent; p.sink = (int)sink;
  // CTAs a (kv head, sequence): a stretch of up to 4096 tokens is quickest in one (no sums across CTAs); longer ones are shared by up
  // to eight, as many as run at once with a CTA an SM (its registers allow no more), or as it takes to keep the keys.  Measured, us
  // with one CTA to two an SM / as it is: 4 sequences of 16384 tokens x 8 kv heads 81 / 18, 8 of 8192 33 / 14; with 16384 keys a
  // CTA / 32768: 8 of 32768 43 / 27
  const int sms = sm_count();
  if (!sms) return -2;
  int n = 1;
  while (n < 8 && (long)p.t.width * kPage > 4096L * n && (S * Hkv * 2 * n <= sms || (long)p.t.width * kPage > (long)kSelKeys * n)) n *= 2;
  if (Hkv * n > 0x7fffffffL) return -2;
  static unsigned long long ready = 0;
  const cudaError_t e = allow_smem(ready, (const void*)select_kernel, kSelKeys * 4);
  if (e != cudaSuccess) return (int)e;
  const long most = (p.t.width + n - 1L) / n * kPage;           // tokens of a CTA
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(Hkv * n), (unsigned)S); cfg.blockDim = dim3(kSelThreads); cfg.dynamicSmemBytes = 4 * (size_t)(most < kSelKeys ? most : kSelKeys); cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)n; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = (grm_pdl_enabled() & GRM_PDL_ATTN) ? 1 : 0;
  cfg.attrs = at; cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, select_kernel, p, n);
}

// data, mass (or 0), table, slots, width, stride, pages, seq (or 0), idx, dst (int32 [S][>= ceil(keep / 16)]), dst_stride, S, Hkv, D, keep
GRM_API int grm_kv4_compact(const void* words, void* stream) {
  Args a(words);
  CompactParams p;
  p.data = a.ptr<uint8_t>(); p.mass = a.ptr<float>();
  if (!read_table(a, p.src)) return -2;
  p.slots = a.ptr<const int>(); p.idx = a.ptr<const int>(); p.dst = a.ptr<const int>(); p.dst_stride = a.num();
  const long S = a.num(), Hkv = a.num(), D = a.num(), keep = a.num();
  if (!fits(S, 1, 65535) || !fits(Hkv, 1, 65535) || !fits(keep, 1, 0x7fffffff - kMoveTokens)) return -2;
  p.Hkv = (int)Hkv; p.keep = (int)keep;
  KV4_DISPATCH(D, return (int)grm_launch_pdl(GRM_PDL_ATTN, compact_kernel<DD>, dim3((unsigned)((keep + kMoveTokens - 1) / kMoveTokens), (unsigned)Hkv, (unsigned)S), dim3(256), 0, (cudaStream_t)stream, p));
}
