// Device helpers shared by the 8-bit cache's kernels.
#pragma once
#include "fp8_cache_kernels.h"
#include "pagecopy_kernels.h"

namespace bikv {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Addresses are put together from integers: the explicit address space keeps the accesses global_*.
#define BIKV_G __attribute__((address_space(1)))
template <class T>
__device__ __forceinline__ T gload(uint64_t addr) {
  return *(const BIKV_G T*)addr;
}
template <class T>
__device__ __forceinline__ void gstore(uint64_t addr, T v) {
  *(BIKV_G T*)addr = v;
}

__device__ __forceinline__ void raise_flag(uint32_t* status, int slot) {
  *(volatile BIKV_G uint32_t*)(status + slot) = 1u;
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uni64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// A sequence as the kernels use it. One whose numbers make no sense (a negative length, more tokens than
// its table row has pages for, rows outside the caller's tensors) is dropped as a whole: no rows, no keys.
struct Seq {
  int64_t first;   // first row of the caller's tensors
  int n;           // rows
  int len;         // tokens in the cache
  bool ok;
};
__device__ __forceinline__ Seq read_seq(const SeqArgs& s, int64_t b) {
  const int64_t len = s.kv_lens[b];
  int64_t lo = b, hi = b + 1;
  if (s.q_starts) {
    lo = s.q_starts[b];
    hi = s.q_starts[b + 1];
  }
  Seq r;
  r.ok = len >= 0 && len <= s.max_len && lo >= 0 && hi >= lo && hi <= s.n_rows;
  r.first = r.ok ? lo : 0;
  r.n = r.ok ? (int)(hi - lo) : 0;
  r.len = r.ok ? (int)len : 0;
  return r;
}

// The largest b < n_seqs whose first_slot(b) is not beyond `slot`. first_slot grows with b, so a 64-way search by a
// whole wave finds it in one step for 64 sequences, two for 4096. With row numbers that do not grow
// the result is some b in range: callers check that the slot is one of that sequence's.
template <class F>
__device__ __forceinline__ int64_t find_seq(int64_t n_seqs, int64_t slot, int lane, F first_slot) {
  int64_t lo = 0, n = n_seqs;       // the answer is in [lo, lo + n)
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const int64_t b = lo + step * lane;
    const bool le = step * lane < n && first_slot(b) <= slot;
    const uint64_t m = __ballot(le);
    const int last = m ? 63 - __builtin_clzll(m) : 0;
    lo = lo + step * last;
    n = n - step * last < step ? n - step * last : step;
  }
  return uni64(lo);
}

}  // namespace bikv
