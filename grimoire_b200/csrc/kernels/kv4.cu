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

// One warp per (row, kv head): the 2 * D / 4 quads of K and V go round the lanes, so a lane's quads all lie in one group and
// the group's maximum is a butterfly over the lanes with the same (K / V, quad mod groups).  7 x / maximum is a quotient of an
// 11-bit and an 8-bit integer (times powers of two; 7 / 8 and 1 / 8 so that nothing overflows): a correctly rounded fp32
// division never lands on another side of a rounding boundary than the exact quotient, so the codes equal those of 64-bit
// arithmetic.
template <int D>
__global__ void __launch_bounds__(128) append_kernel(const AppendParams p) {
  using G = Geo<D>;
  constexpr int kQuads = D / 4, kRegs = (2 * kQuads + 31) / 32;
  const long wid = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (wid >= (long)p.M * p.Hkv) return;
  const int row = (int)(wid / p.Hkv), h = (int)(wid % p.Hkv);
  const int pos = p.row_pos[row];
  const int page = pos < 0 ? -1 : page_of(p.t, p.row_seq[row], pos / kPage);
  if (page < 0) return;
  const int slot = pos % kPage;
  uint2 x[kRegs];          // 4 bf16 each
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int idx = lane + 32 * i, which = idx / kQuads, quad = idx % kQuads;
    const bf16* src = (which ? p.v + (size_t)row * p.ld_v : p.k + (size_t)row * p.ld_k) + (size_t)h * D + 4 * quad;
    if (p.vec) {
      x[i] = *reinterpret_cast<const uint2*>(src);
    } else {
      const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
      x[i].x = s[0] | ((uint32_t)s[1] << 16);
      x[i].y = s[2] | ((uint32_t)s[3] << 16);
    }
  }
  // magnitude bits order like the values, with infinity and then NaN on top
  uint32_t mx[kRegs];
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const uint32_t a = x[i].x & 0x7fff7fffu, b = x[i].y & 0x7fff7fffu;
    const uint32_t m = __vmaxu2(a, b);
    mx[i] = max(m & 0xffffu, m >> 16);
  }
  if constexpr (D == 256) {                       // registers 0, 1 are K, 2, 3 are V; both quads of a lane are in group lane % 8
    mx[0] = mx[1] = max(mx[0], mx[1]);
    mx[2] = mx[3] = max(mx[2], mx[3]);
  }
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    if (D == 256 && (i & 1)) { mx[i] = mx[i - 1]; continue; }
#pragma unroll
    for (int o = G::kGroups; o < (kQuads < 32 ? kQuads : 32); o <<= 1) mx[i] = max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
  }
  uint8_t* rec = p.data + ((size_t)page * p.Hkv + h) * G::kRecord;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int idx = lane + 32 * i, which = idx / kQuads, quad = idx % kQuads;
    const float amax = __uint_as_float(mx[i] << 16);
    const bool ok = mx[i] > 0u && mx[i] < 0x7f80u;        // an empty group has codes of zero; one that is not finite reads back as NaN
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = j < 2 ? x[i].x : x[i].y;
      const float f = (j & 1) ? bf16hi_to_f(b) : bf16lo_to_f(b);
      const int q = ok ? __float2int_rn(__fdiv_rn(0.875f * f, 0.125f * amax)) : 0;
      word |= (uint32_t)(q + 8) << (4 * j);
    }
    const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
    if (!(lane & 1)) *reinterpret_cast<uint32_t*>(rec + which * G::kV + slot * G::kRow + 2 * quad) = word | (other << 16);
    if (quad < G::kGroups)
      *reinterpret_cast<unsigned short*>(rec + G::kAmax + slot * G::kAmaxTok + 2 * (which * G::kGroups + quad)) = (unsigned short)mx[i];
  }
  if (p.mass && lane == 0) p.mass[((size_t)page * p.Hkv + h) * kPage + slot] = 0.f;
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

// x / 7 rounded correctly: one Newton correction of the product with the rounded reciprocal (Markstein).
__device__ __forceinline__ float div7(float x) {
  constexpr float r = 1.f / 7.f;
  const float y = x * r;
  const float z = fmaf(fmaf(-7.f, y, x), r, y);
  return isfinite(z) ? z : y;
}

// One thread per 8 elements (a word of codes) of K or V: T * Hkv * 2 * D / 8 words a sequence.
template <int D>
__global__ void __launch_bounds__(256) gather_kernel(const GatherParams p) {
  using G = Geo<D>;
  constexpr int kWords = D / 8;
  const int s = blockIdx.y;
  const int slot = p.slots ? p.slots[s] : s;
  const int len = p.lengths ? min(p.lengths[s], p.T) : p.T;
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int w = (int)(i % kWords);
  const int which = (int)(i / kWords % 2);
  const long th = i / (2 * kWords);
  const int h = (int)(th % p.Hkv);
  const long tok = th / p.Hkv;
  if (tok >= len) return;
  const int page = page_of(p.t, slot, (int)(tok / kPage));
  if (page < 0) return;
  const int in = (int)(tok % kPage);
  const uint8_t* rec = p.data + ((size_t)page * p.Hkv + h) * G::kRecord;
  const uint32_t c = *reinterpret_cast<const uint32_t*>(rec + which * G::kV + in * G::kRow + 4 * w);
  const unsigned short* am = reinterpret_cast<const unsigned short*>(rec + G::kAmax + in * G::kAmaxTok) + which * G::kGroups;
  const float a0 = __uint_as_float((uint32_t)am[(2 * w) % G::kGroups] << 16);
  const float a1 = __uint_as_float((uint32_t)am[(2 * w + 1) % G::kGroups] << 16);
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = j < 2 ? a0 : a1;
    const float lo = 0.125f * (float)((int)((c >> (8 * j)) & 15u) - 8), hi = 0.125f * (float)((int)((c >> (8 * j + 4)) & 15u) - 8);
    o[j] = pack_bf16x2(8.f * div7(lo * a), 8.f * div7(hi * a));      // an eighth on the way: code * maximum may exceed fp32
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

constexpr int kSelThreads = 1024;

// One CTA per (kv head, sequence).  Radix selection: four passes of 8 bits over the tokens that are neither among the first
// `sink` nor the last `recent` find the key of the last token that stays and how many tokens of exactly that key do; one
// more pass writes the kept positions in order.
__global__ void __launch_bounds__(kSelThreads) select_kernel(const SelectParams p) {
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  __shared__ int w_eq[kSelThreads / 32], w_keep[kSelThreads / 32];
  const int h = blockIdx.x, s = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = p.slots ? p.slots[s] : s;
  const int n = max(0, min(p.lengths[s], p.t.width * kPage));
  int* out = p.idx + ((size_t)s * p.Hkv + h) * p.keep;
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int lo = min(p.sink, n), hi = max(n - p.recent, lo);
  auto key = [&](int t) -> uint32_t {
    const int page = page_of(p.t, slot, t / kPage);
    return page < 0 ? 0u : order_key(__ldg(p.mass + ((size_t)page * p.Hkv + h) * kPage + t % kPage));
  };
  uint32_t prefix = 0;
  int need = p.keep - lo - (n - hi);                        // tokens to take from [lo, hi); fewer than there are
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = lo + tid; t < hi; t += kSelThreads) {
      const uint32_t k = key(t);
      if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int left = need, b = 255;
      while (b > 0 && hist[b] < left) left -= hist[b--];
      s_prefix = (prefix << 8) | (uint32_t)b;
      s_need = left;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // prefix: the key of the last kept token; need: how many tokens with that key stay, the earliest ones
  const bool none = p.keep - lo - (n - hi) == 0;
  int eq0 = 0, out0 = 0;
  for (int t0 = 0; t0 < n; t0 += kSelThreads) {
    const int t = t0 + tid;
    const bool cand = t >= lo && t < hi;
    const uint32_t k = (cand && !none) ? key(t) : 0u;
    const bool eq = cand && !none && k == prefix;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) w_eq[warp] = __popc(eqs);
    __syncthreads();
    int before = eq0, all_eq = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) { before += w < warp ? w_eq[w] : 0; all_eq += w_eq[w]; }
    before += __popc(eqs & ((1u << lane) - 1u));
    const bool keep = t < n && (!cand || (!none && (k > prefix || (eq && before < need))));
    const uint32_t ks = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) w_keep[warp] = __popc(ks);
    __syncthreads();
    int at = out0, all_keep = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) { at += w < warp ? w_keep[w] : 0; all_keep += w_keep[w]; }
    at += __popc(ks & ((1u << lane) - 1u));
    if (keep && at < p.keep) out[at] = t;
    eq0 += all_eq;
    out0 += all_keep;
  }
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

// One CTA of 8-byte movers per (page of 16 kept tokens, kv head, sequence): codes and maxima are copied as they are.
template <int D>
__global__ void __launch_bounds__(128) compact_kernel(const CompactParams p) {
  using G = Geo<D>;
  constexpr int kUnits = (2 * G::kRow + G::kAmaxTok) / 8;   // 8-byte units of a token
  const int s = blockIdx.z, h = blockIdx.y, pg = blockIdx.x;
  const int dst = p.dst[(size_t)s * p.dst_stride + pg];
  if ((unsigned)dst >= (unsigned)p.src.pages) return;
  const int slot = p.slots ? p.slots[s] : s;
  const int* idx = p.idx + ((size_t)s * p.Hkv + h) * p.keep + (size_t)pg * kPage;
  const size_t dbase = (size_t)dst * p.Hkv + h;
  for (int i = threadIdx.x; i < kPage * kUnits; i += blockDim.x) {
    const int tok = i / kUnits, u = i % kUnits;
    if (pg * kPage + tok >= p.keep) continue;
    const int from = idx[tok];
    if (from < 0) continue;
    const int page = page_of(p.src, slot, from / kPage);
    if (page < 0) continue;
    const size_t sbase = (size_t)page * p.Hkv + h;
    const int in = from % kPage;
    constexpr int kRowUnits = G::kRow / 8;
    auto off = [&](int r) {
      return u < kRowUnits ? r * G::kRow + 8 * u
                           : (u < 2 * kRowUnits ? G::kV + r * G::kRow + 8 * (u - kRowUnits) : G::kAmax + r * G::kAmaxTok + 8 * (u - 2 * kRowUnits));
    };
    *reinterpret_cast<uint2*>(p.data + dbase * G::kRecord + off(tok)) = *reinterpret_cast<const uint2*>(p.data + sbase * G::kRecord + off(in));
    if (u == 0 && p.mass) p.mass[dbase * kPage + tok] = p.mass[sbase * kPage + in];
  }
}

}  // namespace

#define KV4_DISPATCH(D, CALL)                                   \
  switch (D) {                                                  \
    case 64: { constexpr int DD = 64; CALL; break; }            \
    case 128: { constexpr int DD = 128; CALL; break; }          \
    case 256: { constexpr int DD = 256; CALL; break; }          \
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
  KV4_DISPATCH(D, (append_kernel<DD><<<(unsigned)((M * Hkv + 3) / 4), 128, 0, (cudaStream_t)stream>>>(p)));
  GRM_LAUNCH_RET();
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
  if (!fits(S, 1, 65535) || !fits(T, 1, 0x7fffffff) || !fits(Hkv, 1, 0x7fffffff)) return -2;
  p.T = (int)T; p.Hkv = (int)Hkv;
  const long blocks = (T * Hkv * (D / 4) + 255) / 256;
  if (blocks > 0x7fffffffL) return -2;
  KV4_DISPATCH(D, (gather_kernel<DD><<<dim3((unsigned)blocks, (unsigned)S), 256, 0, (cudaStream_t)stream>>>(p)));
  GRM_LAUNCH_RET();
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
  select_kernel<<<dim3((unsigned)Hkv, (unsigned)S), kSelThreads, 0, (cudaStream_t)stream>>>(p);
  GRM_LAUNCH_RET();
}

// data, mass (or 0), table, slots, width, stride, pages, seq (or 0), idx, dst (int32 [S][>= ceil(keep / 16)]), dst_stride, S, Hkv, D, keep
GRM_API int grm_kv4_compact(const void* words, void* stream) {
  Args a(words);
  CompactParams p;
  p.data = a.ptr<uint8_t>(); p.mass = a.ptr<float>();
  if (!read_table(a, p.src)) return -2;
  p.slots = a.ptr<const int>(); p.idx = a.ptr<const int>(); p.dst = a.ptr<const int>(); p.dst_stride = a.num();
  const long S = a.num(), Hkv = a.num(), D = a.num(), keep = a.num();
  if (!fits(S, 1, 65535) || !fits(Hkv, 1, 65535) || !fits(keep, 1, 0x7fffffff - kPage)) return -2;
  p.Hkv = (int)Hkv; p.keep = (int)keep;
  KV4_DISPATCH(D, (compact_kernel<DD><<<dim3((unsigned)((keep + kPage - 1) / kPage), (unsigned)Hkv, (unsigned)S), 128, 0, (cudaStream_t)stream>>>(p)));
  GRM_LAUNCH_RET();
}
