// The 4-bit KV page, shared by the kernels that write, read, weigh and move it (kv4.cu, kv4_attn.cu).
//
// A (page, kv head) record of 18 * D bytes holds 16 tokens:
//   K codes [16][D / 2] | V codes [16][D / 2] | maxima [16][K, V][D / 32] bf16
// Element d of a token's row is (code - 8) * maximum[(d / 4) % (D / 32)] / 7 with code = round(7 x / maximum) + 8 in 1..15,
// element d in byte d / 2 (low half for even d).  A quantisation group is 32 elements: the quads (4 consecutive elements)
// whose index has the same remainder mod D / 32.  Quads are dealt out because a 32-bit word of codes then holds exactly two
// groups, one per 16-bit half, which is what the tensor-core operands of the attention kernel want: an operand register pairs
// the same nibble of two words (or two tokens), so both of its elements share one maximum.
#pragma once
#include "common.cuh"

namespace kv4 {

constexpr int kPage = 16;
constexpr int kMaxWidth = 1 << 20;                   // pages of a sequence: sums over 1024 sequences fit 32 bits

template <int D>
struct Geo {
  static constexpr int kGroups = D / 32;             // maxima of a row
  static constexpr int kRow = D / 2;                 // bytes of a token's codes (K or V)
  static constexpr int kAmaxTok = 4 * kGroups;       // bytes of a token's maxima (K then V)
  static constexpr int kV = kPage * kRow;            // offset of the V codes
  static constexpr int kAmax = 2 * kPage * kRow;     // offset of the maxima
  static constexpr int kRecord = kAmax + kPage * kAmaxTok;
  static_assert(kRecord == 18 * D, "page record");
};

// Pages of one sequence.  A table entry outside [0, pages) maps nothing: its tokens do not exist for any reader or writer.
struct Table {
  const int* table;       // [slots][width]
  int slots, width;       // rows, entries a row
  long stride;            // entries between rows
  int pages;              // pages in the pool
};
__device__ __forceinline__ int page_of(const Table& t, int slot, int index) {
  if ((unsigned)slot >= (unsigned)t.slots || (unsigned)index >= (unsigned)t.width) return -1;
  const int p = __ldg(t.table + (size_t)slot * t.stride + index);
  return (unsigned)p < (unsigned)t.pages ? p : -1;
}

// Arguments of a call as 64-bit words (pointers, integers; the one fraction as the bits of a double) in the order of the entry
// point's list: a record that the caller packs at once costs it a third of what thirty separate arguments do.
struct Args {
  const long long* w;
  int at = 0;
  explicit Args(const void* words) : w((const long long*)words) {}
  template <typename T>
  T* ptr() { return (T*)(uintptr_t)w[at++]; }
  long num() { return (long)w[at++]; }
  double real() {
    union { long long i; double d; } u;
    u.i = w[at++];
    return u.d;
  }
};
inline bool fits(long v, long lo, long hi) { return v >= lo && v <= hi; }
// table, slots, width, stride, pages
inline bool read_table(Args& a, Table& t) {
  t.table = a.ptr<const int>();
  const long slots = a.num(), width = a.num();
  t.stride = a.num();
  const long pages = a.num();
  if (!t.table || !fits(slots, 1, 0x7fffffff) || !fits(width, 1, kMaxWidth) || !fits(pages, 1, 0x7fffffff)) return false;
  t.slots = (int)slots; t.width = (int)width; t.pages = (int)pages;
  return true;
}

// The multiprocessors of the current device (0 where that fails).
inline int sm_count() {
  static int known[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!known[dev] && cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return known[dev];
}

// Opts a kernel in to its dynamic shared memory, once per device (bit of ``ready``; setting it twice does no harm).
inline cudaError_t allow_smem(unsigned long long& ready, const void* kernel, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (ready >> (dev & 63) & 1)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) ready |= 1ull << (dev & 63);
  return e;
}

}  // namespace kv4
