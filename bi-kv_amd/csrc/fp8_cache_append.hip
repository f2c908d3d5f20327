// New keys and values into the 8-bit cache (gfx950).
//
// A page of one layer holds, for K and for V, page_tokens x heads x head_dim bytes of e4m3 and one fp32 scale
// s per head; byte c stands for e4m3(c) * s. New tokens fill rows [r0, r1) of a page. With
//   amax = max |x| over those rows of one head (finite values only),
//   need = the smallest power of two, not under 2^-126, with amax <= 448 need,
// the page's scale becomes
//   r0 == 0 (nothing older in the page): need
//   r0 >  0: its old scale s while 448 s >= amax, else need; rows [0, r0) are then rounded once more,
//            c' = e4m3(e4m3(c) * s / need).
// Powers of two because they cost an e4m3 value nothing: dividing by one moves its exponent and keeps its
// three bits, so a row that is rescaled when its page's scale grows stays as it was first rounded (but for
// values that reach e4m3's subnormals), however many tokens arrive one at a time. New values are x / scale, rounded
// to the nearest e4m3 value, ties to even; the quotient is exact in fp32 for a power of two. A NaN or an infinity becomes
// NaN and takes no part in amax. Rows behind the new ones are left as they are.
//
// Bound by memory: 2 bytes read and 1 written per value. One wave per (page, head, K or V): a row of a head
// is 16 bytes a lane, the rows of a page of up to 32 tokens (head_dim 128) stay in registers between the
// maximum and the rounding, so that they are read once; longer pages are read twice, the second time
// out of the caches. The maximum is taken over the bits of two values at a time, and values are divided and rounded two
// at a time by the conversion that takes a power of two along; only a page with a NaN or an infinity, or an old scale that is no
// power of two, goes value by value (with that for all, 29 us where it is 21 now). No LDS, no barrier, no atomics.
// Measured: 16k tokens of 16 prompts, 8 heads of 128: 98 MB in 21 us, 4.7 TB/s; 9 chunks of up to 299 tokens
// in pages of 50: 7.6 us; one token to each of 8 sequences: 4.2 us, a launch and the lookups. Where every touched page outgrows its scale,
// and its older rows are rounded again, these take 21, 7.9 and 5.8 us.
#include "fp8_cache_device.h"

namespace bikv {

template <int TYPE>
__device__ __forceinline__ float widen(uint32_t half_bits) {
  if constexpr (TYPE == 0) return __uint_as_float(half_bits << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)half_bits);
}

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The smallest power of two >= 2^-126 with amax <= 448 s; 448 = 1.75 * 2^8.
__device__ __forceinline__ float needed_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -126 ? -126 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Division by the page's scale. A normal power of two (every scale this kernel makes) divides by a
// product with its inverse, which is exact; another scale, of a cache that was filled elsewhere, divides.
struct Divider {
  float s, inv;
  bool pow2;
  __device__ __forceinline__ explicit Divider(float scale) : s(scale) {
    const uint32_t b = __float_as_uint(scale);
    pow2 = (b & 0x807fffffu) == 0 && b >= 0x00800000u && b < 0x7e800000u;   // 2^-126 .. 2^125: the inverse is normal
    inv = pow2 ? __uint_as_float(0x7f000000u - b) : 0.f;
  }
  __device__ __forceinline__ float operator()(float x) const {
    if (pow2) return x * inv;
    return s == 0.f ? x * 0.f : x / s;       // a zero scale is kept only where every value is zero
  }
};

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Four values, two to a word as they were read, divided by a power of two and rounded to the nearest e4m3.
template <int TYPE>
__device__ __forceinline__ uint32_t pack4_scaled(uint32_t ab, uint32_t cd, float s) {
  s16x2 w{0, 0};
  if constexpr (TYPE == 0) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, ab), s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, cd), s, true);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, ab), s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, cd), s, true);
  }
  return __builtin_bit_cast(uint32_t, w);
}

template <int D, int TYPE>
__global__ __launch_bounds__(kAppendThreads) void fp8_append_kernel(const AppendArgs a) {
  constexpr int kLanesPerRow = D / 8;
  constexpr int kRows = 64 / kLanesPerRow;    // rows a wave reads with one instruction
  constexpr int kVecs = 8, kOld = 4;
  constexpr int kChunk = kRows * kVecs;       // rows held in registers
  const int lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * 4 + uni(threadIdx.x >> 6);    // below 2^31: the host sees to it
  const uint32_t H = (uint32_t)a.layer.heads;
  const int h = (int)(w % H);
  const int kv = (int)((w / H) & 1);
  const int64_t u = w / H / 2;
  if (u >= a.units) return;
  const int P = (int)a.layer.page_tokens.d;

  // Page slots: without row numbers sequence b has the one slot b. With them it has the slots from
  // floor(q_starts[b] / P) + 2 b on, at least floor(n / P) + 2 of them, which is as many pages as n tokens can touch.
  int64_t b = u, j = 0;
  if (a.seq.q_starts) {
    auto first_slot = [&](int64_t i) {
      int64_t q = a.seq.q_starts[i];
      q = q < 0 ? 0 : q > a.seq.n_rows ? a.seq.n_rows : q;
      return (int64_t)divide((uint32_t)q, a.layer.page_tokens) + 2 * i;
    };
    b = find_seq(a.seq.n_seqs, u, lane, first_slot);
    j = u - first_slot(b);
    if (h == 0 && kv == 0 && u < a.seq.n_seqs) {
      const Seq s = read_seq(a.seq, u);
      if ((!s.ok || s.n > s.len) && lane == 0) raise_flag(a.status, ST_SLOT_SRC);
    }
  }
  const Seq s = read_seq(a.seq, b);
  if (!s.ok || s.n > s.len) {
    if (lane == 0) raise_flag(a.status, ST_SLOT_SRC);
    return;
  }
  const int start = s.len - s.n;
  const int64_t page_no = (int64_t)divide((uint32_t)start, a.layer.page_tokens) + j;
  if (j < 0 || s.n == 0 || page_no * P >= s.len) return;
  const int64_t pid = a.seq.table[b * a.seq.table_stride + page_no];      // not looked at before the new values are on their way
  const int base = (int)(page_no * P);
  const int r0 = start > base ? start - base : 0;
  const int r1 = s.len - base < P ? s.len - base : P;
  const int n = r1 - r0;

  const int sub = lane / kLanesPerRow;
  const int d = (lane % kLanesPerRow) * 8;
  const int64_t row = kv ? a.v_row : a.k_row, head = kv ? a.v_head : a.k_head;
  const uint64_t src = (uint64_t)(kv ? a.v : a.k) + 2 * ((s.first + (base + r0 - start)) * row + h * head + d);
  u32x4 x[kVecs];
  constexpr uint32_t kInf = TYPE == 0 ? 0x7f80u : 0x7c00u;
  u16x2 top{0, 0};                            // the largest |x| by its bits, which order like the values; two lanes of 16 bits
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int r = c0 + i * kRows + sub;
      x[i] = u32x4{0, 0, 0, 0};
      if (r < n) x[i] = gload<u32x4>(src + 2 * (uint64_t)(r * row));
    }
  };
  load(0);
  __builtin_amdgcn_sched_barrier(0);
  if ((uint64_t)pid >= (uint64_t)a.layer.n_pages) {
    if (lane == 0) raise_flag(a.status, ST_SLOT_PAGE);
    return;
  }
  const uint64_t page = (uint64_t)(kv ? a.layer.v : a.layer.k) + (uint64_t)(pid * a.layer.page_stride) + h * D + d;
  const uint64_t scale_at = (uint64_t)(kv ? a.layer.vs : a.layer.ks) + (uint64_t)(pid * a.layer.scale_stride) + 4 * h;

  const float s_old = r0 > 0 ? gload<float>(scale_at) : 0.f;
  const int chunks = (n + kChunk - 1) / kChunk;
  for (int c = 0; c < chunks; ++c) {
    if (c > 0) load(c * kChunk);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[i][e] & 0x7fff7fffu));
  }
  uint32_t bits = top[0] > top[1] ? top[0] : top[1];
  for (int m = 32; m > 0; m >>= 1) {
    const uint32_t other = __shfl_xor(bits, m);
    bits = bits > other ? bits : other;
  }
  bits = uni(bits);
  const bool finite = bits < kInf;            // of every value: the usual case
  float amax = widen<TYPE>(bits);
  if (!finite) {                              // the largest of those that are
    amax = 0.f;
    for (int c = 0; c < chunks; ++c) {
      if (chunks > 1) load(c * kChunk);
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lo = fabsf(widen<TYPE>(x[i][e] & 0xffffu)), hi = fabsf(widen<TYPE>(x[i][e] >> 16));
          if (finite_bits(lo)) amax = fmaxf(amax, lo);
          if (finite_bits(hi)) amax = fmaxf(amax, hi);
        }
    }
    for (int m = 32; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
  }

  const bool kept = r0 > 0 && 448.f * s_old >= amax;
  const float scale = kept ? s_old : needed_scale(amax);
  const Divider by(scale);
  const bool plain = uni(finite && by.pow2);
  if (r0 > 0 && !kept) {
    for (int q0 = 0; q0 < r0; q0 += kRows * kOld) {        // kOld loads in flight; more would cost registers, and waves, in every call
      u32x2 old[kOld];
#pragma unroll
      for (int i = 0; i < kOld; ++i) {
        const int r = q0 + i * kRows + sub;
        old[i] = u32x2{0, 0};
        if (r < r0) old[i] = gload<u32x2>(page + (uint64_t)(r * a.layer.token_stride));
      }
#pragma unroll
      for (int i = 0; i < kOld; ++i) {
        const int r = q0 + i * kRows + sub;
        if (r < r0) {
          u32x2 c = old[i];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[e], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[e], true);
            c[e] = pack4(by(lo[0] * s_old), by(lo[1] * s_old), by(hi[0] * s_old), by(hi[1] * s_old));
          }
          gstore<u32x2>(page + (uint64_t)(r * a.layer.token_stride), c);
        }
      }
    }
  }
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c * kChunk);
    if (plain) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int r = c * kChunk + i * kRows + sub;
        if (r < n)
          gstore<u32x2>(page + (uint64_t)((r0 + r) * a.layer.token_stride),
                        u32x2{pack4_scaled<TYPE>(x[i][0], x[i][1], scale), pack4_scaled<TYPE>(x[i][2], x[i][3], scale)});
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int r = c * kChunk + i * kRows + sub;
      if (r < n) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[e] = widen<TYPE>((x[i][e / 2] >> (16 * (e & 1))) & 0xffffu);
          f[e] = finite_bits(f[e]) ? by(f[e]) : __uint_as_float(0x7fc00000u);
        }
        gstore<u32x2>(page + (uint64_t)((r0 + r) * a.layer.token_stride), u32x2{pack4(f[0], f[1], f[2], f[3]), pack4(f[4], f[5], f[6], f[7])});
      }
    }
  }
  if (lane == 0 && !kept) gstore<float>(scale_at, scale);
}

hipError_t launch_fp8_append(int head_dim, int type, const AppendArgs& a, hipStream_t stream) {
  const dim3 grid((uint32_t)append_groups(a.units, a.layer.heads)), block(kAppendThreads);
  if (head_dim == 128) {
    if (type == 0) hipLaunchKernelGGL((fp8_append_kernel<128, 0>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((fp8_append_kernel<128, 1>), grid, block, 0, stream, a);
  } else {
    if (type == 0) hipLaunchKernelGGL((fp8_append_kernel<64, 0>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((fp8_append_kernel<64, 1>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace bikv
