// Attention over the 4-bit KV cache (page layout: kv4.cuh) and the weight that it gives to every cached token.
//   out[row] = softmax(scale * q[row] K^T) V over keys first .. pos[row] of the row's sequence; rows without a key give zeros
//   mass[token] (=, +=) sum over the rows of a block and the query heads of a kv head of the softmax weight
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
  int M, Hkv, G, window, block, add;
  float scale_log2;         // softmax scale * log2(e)
};

__device__ __forceinline__ float deq(const uint8_t* row, const unsigned short* am, int d, int groups) {
  const int c = (row[d >> 1] >> (4 * (d & 1))) & 15;
  return (float)(c - 8) * __uint_as_float((uint32_t)am[(d >> 2) % groups] << 16) * (1.f / 7.f);
}

template <int D, int GP>
__global__ void __launch_bounds__(kThreads) attn_kernel(const AttnParams p) {
  using Gm = Geo<D>;
  constexpr int R = D / 32;
  __shared__ float sq[GP][D];
  __shared__ float sm[kWarps][GP], sl[kWarps][GP];
  __shared__ float so[kWarps][D];
  const int split = blockIdx.x, nsplit = gridDim.x, kvh = blockIdx.y, row = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = p.row_seq[row];
  const int len = max(0, min(p.row_pos[row] + 1, p.t.width * kPage));
  const int first = (p.window > 0 && len > p.window) ? len - p.window : 0;
  const int page_lo = first / kPage, page_hi = (len + kPage - 1) / kPage;
  const int pps = (page_hi - page_lo + nsplit - 1) / nsplit;
  const int pbeg = page_lo + split * pps, pend = min(pbeg + pps, page_hi);
  for (int i = tid; i < p.G * D; i += kThreads)
    sq[i / D][i % D] = __bfloat162float(p.q[(size_t)row * p.ld_q + (size_t)(kvh * p.G) * D + i]);
  __syncthreads();
  float m[GP], l[GP], acc[GP][R];
#pragma unroll
  for (int g = 0; g < GP; ++g) {
    m[g] = -INFINITY; l[g] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) acc[g][r] = 0.f;
  }
  for (int pg = pbeg + warp; pg < pend; pg += kWarps) {
    const int page = page_of(p.t, slot, pg);
    if (page < 0) continue;
    const uint8_t* rec = p.data + ((size_t)page * p.Hkv + kvh) * Gm::kRecord;
    for (int tok = 0; tok < kPage; ++tok) {
      const int t = pg * kPage + tok;
      if (t < first || t >= len) continue;
      const unsigned short* am = reinterpret_cast<const unsigned short*>(rec + Gm::kAmax + tok * Gm::kAmaxTok);
      float k[R], v[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        k[r] = deq(rec + tok * Gm::kRow, am, lane + 32 * r, Gm::kGroups);
        v[r] = deq(rec + Gm::kV + tok * Gm::kRow, am + Gm::kGroups, lane + 32 * r, Gm::kGroups);
      }
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        if (g < p.G) {
          float s = 0.f;
#pragma unroll
          for (int r = 0; r < R; ++r) s = fmaf(sq[g][lane + 32 * r], k[r], s);
          s = warp_sum(s) * p.scale_log2;
          const float mn = fmaxf(m[g], s);
          const float c = m[g] == -INFINITY ? 0.f : exp2f(m[g] - mn);
          const float e = exp2f(s - mn);
          m[g] = mn;
          l[g] = fmaf(l[g], c, e);
#pragma unroll
          for (int r = 0; r < R; ++r) acc[g][r] = fmaf(acc[g][r], c, e * v[r]);
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GP; ++g)
    if (lane == 0) { sm[warp][g] = m[g]; sl[warp][g] = l[g]; }
  for (int g = 0; g < p.G; ++g) {
    __syncthreads();
#pragma unroll
    for (int gg = 0; gg < GP; ++gg)
      if (gg == g)
#pragma unroll
        for (int r = 0; r < R; ++r) so[warp][lane + 32 * r] = acc[gg][r];
    __syncthreads();
    float mx = -INFINITY;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[w][g]);
    float ls = 0.f, f[kWarps];
    for (int w = 0; w < kWarps; ++w) {
      f[w] = sm[w][g] == -INFINITY ? 0.f : exp2f(sm[w][g] - mx);
      ls += f[w] * sl[w][g];
    }
    const size_t pi = (((size_t)row * p.Hkv + kvh) * nsplit + split) * p.G + g;
    for (int d = tid; d < D; d += kThreads) {
      float o = 0.f;
      for (int w = 0; w < kWarps; ++w) o += sl[w][g] != 0.f ? f[w] * so[w][d] : 0.f;
      p.part_o[pi * D + d] = o;
    }
    if (tid == 0) { p.part_ml[2 * pi] = mx; p.part_ml[2 * pi + 1] = ls; }
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

template <int D>
int launch(const AttnParams& p, int splits, int nblocks, int mass_pages, cudaStream_t st) {
  const dim3 grid(splits, p.Hkv, p.M);
  if (p.G <= 4) attn_kernel<D, 4><<<grid, kThreads, 0, st>>>(p);
  else if (p.G <= 8) attn_kernel<D, 8><<<grid, kThreads, 0, st>>>(p);
  else attn_kernel<D, 16><<<grid, kThreads, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  merge_kernel<<<dim3(p.G, p.Hkv, p.M), 128, 0, st>>>(p, splits, D);
  e = cudaGetLastError();
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
