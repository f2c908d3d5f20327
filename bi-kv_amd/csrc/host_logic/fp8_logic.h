// Arithmetic of the 8-bit cache's kernels that has nothing to do with the GPU. HIP-free: tests compile it with the
// host compiler.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define BIKV_HD __host__ __device__ __forceinline__
#else
#define BIKV_HD inline
#endif

namespace bikv {

// n / d for 0 <= n < 2^31 without a division: (n * mul) >> shift with mul = floor(2^shift / d) + 1,
// shift = 31 + ceil(log2 d). mul * d = 2^shift + e with 0 < e <= d, so the product is too large by
// n e / d < 2^31 2^ceil(log2 d) / d, less than one step of the quotient.
struct FastDiv {
  uint32_t d;
  uint32_t shift;
  uint64_t mul;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return {d, 31 + s, (uint64_t(1) << (31 + s)) / d + 1};
}
BIKV_HD uint32_t divide(uint32_t n, const FastDiv& f) { return (uint32_t)((n * f.mul) >> f.shift); }

// Threads of a launch are numbered with 32 bits.
inline bool launch_fits(int64_t groups, int64_t threads_each) { return groups < (int64_t(1) << 32) / threads_each; }

// append: a wave for each page slot, K or V, and head, four to a workgroup. With row numbers there are as many slots as n_rows tokens of n_seqs
// sequences can touch pages.
constexpr int kAppendThreads = 256;
inline int64_t append_units(bool one_each, int64_t n_seqs, int64_t n_rows, int page_tokens) { return one_each ? n_seqs : n_rows / page_tokens + 2 * n_seqs; }
inline int64_t append_groups(int64_t units, int heads) { return (units * 2 * heads + 3) / 4; }

// `total` steps of work in at most `slots` equal shares of at least `min_steps`: slot s has [begin, end), step x
// lies in share x / per.
struct Share {
  uint32_t per, begin, end;
};
BIKV_HD Share share_of(uint32_t total, uint32_t slots, uint32_t min_steps, uint32_t slot) {
  Share s;
  s.per = (total + slots - 1) / slots;
  if (s.per < min_steps) s.per = min_steps;
  const uint64_t begin = (uint64_t)slot * s.per, end = begin + s.per;
  s.begin = begin < total ? (uint32_t)begin : total;
  s.end = end < total ? (uint32_t)end : total;
  return s;
}

}  // namespace bikv
