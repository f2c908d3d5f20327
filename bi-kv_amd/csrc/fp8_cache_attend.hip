// Attention over the 8-bit cache (gfx950).
//
// Row (t, i) of sequence b is query head i of its t-th new token; with g query heads to a KV head, KV head
// h = i / g. Over the keys j the row sees (all len of them, or the first len - n + t + 1 when causal)
//   z_j = scale * q . k_j * ks_j        k_j, v_j: e4m3 bytes of the cache, ks_j, vs_j: their page's fp32 scales
//   out = sum_j exp(z_j - lse) vs_j v_j       lse = log sum_j exp(z_j)
// and a row that sees no key gets out = 0, lse = -inf.
//
// Both forms make one pass over the keys with a running maximum m and sum l per row (in log2 units, fp32),
// and rescale what they have summed when m grows. Products run on the matrix cores, transposed:
// S^T = K Q^T and O^T = V^T P^T. A lane of S^T then holds a few keys of ONE row, which is the layout the second product
// takes its P^T operand in, as long as V^T's keys are put in the same order: P never crosses lanes or
// memory. K is widened to q's type and Q K^T is exact up to fp32 sums. P is rounded to fp16 (11 bits; bf16's 8 would
// cost as much as the output's own rounding): p vs 2^(8 - r), so that neither a page's scale nor a small p leaves fp16's range; the
// exponent r comes off again at the end. Where q is fp16, 11 bits would cost as much as the output's own rounding, and P goes as
// the sum of two fp16 numbers. l sums the unrounded p.
//
// r: while the V scales of the keys read so far lie within 2^kSpread of each other, the largest one's exponent, the same for all rows of
// a tile. A row's largest p vs 2^(8 - r) is then 1 at least, whichever of these keys the row sees: a weight p vs keeps 11 bits
// down to 2^-14 of the row's largest one, and no weight, of either type, is off by more than 2^-25 of that for want of range. Once they lie farther
// apart each row has an r of its own, that of the largest p vs among the keys it does see ("wide" steps, to the end of the tile): a page that a row
// does not see, or hardly attends to, takes no bits from the pages it does. They cost few rows 3 to 8 %, many rows a third.
#include "fp8_cache_device.h"

#include <cstddef>

namespace bikv {

constexpr float kMinusInf = -__builtin_huge_valf();
constexpr int kNoKey = 0x7fffffff;      // position of a key that no row sees
constexpr int kPShift = 8;              // p is scaled by 2^8 in fp16: p down to 2^-22 stays normal
// z is taken against a row's last reference m, which moves only when some z exceeds it by more than this: p may be up to 2^4, p
// 2^kPShift vs 2^-r < 2^(4 + 8 + 1) is in fp16's range, and most steps rescale nothing and reduce nothing across lanes. With 0
// 6 chunks of up to 900 tokens behind up to 8192 take 789 us where they take 777 with 4.
constexpr float kSlack = 4.f;
constexpr int kSpread = 8;
constexpr int kLeastR = -400;           // below any exponent that is left over in a sum

// Four e4m3 bytes as two pairs of q's type.
template <int TYPE>
__device__ __forceinline__ u32x2 widen4(uint32_t c) {
  if constexpr (TYPE == 0)
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, 1.f, true))};
  else
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, 1.f, true))};
}

template <int TYPE>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (TYPE == 0)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {      // nearest, ties to even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
// x less the fp16 value in the pair's low (0) or high (1) half: one instruction, where widening and subtracting are two.
template <int HIGH>
__device__ __forceinline__ float less_half(float x, uint32_t pair) {
  float y;
  if constexpr (HIGH) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(pair), "v"(x));
  else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(pair), "v"(x));
  return y;
}
template <int TYPE>
__device__ __forceinline__ uint32_t narrow(float a, float b) {
  if constexpr (TYPE == 0)
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
  else
    return pack_f16(a, b);
}

// 0xff in each byte that is a NaN in e4m3.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ((((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }
// Reads one key's row of V again and keeps, by place, the first key that holds a NaN there. Rows see keys up to some
// position, so a row's output is NaN at a place exactly if that first key is one it sees. Rare: small, not fast.
template <int D>
__device__ __forceinline__ void note_nans(int* nan_at, uint64_t row, int pos) {
#pragma nounroll
  for (int d = 0; d < D; d += 4) {
    uint32_t bad = nan_bytes(gload<uint32_t>(row + d));
#pragma nounroll
    for (int k = 0; bad != 0; ++k, bad >>= 8)
      if (bad & 1u) atomicMin(nan_at + d + k, pos);
  }
}

// Exponent of a page's V scale, -126 where it is zero, subnormal or not finite.
__device__ __forceinline__ int scale_exponent(float s) {
  const int e = (int)((__float_as_uint(s) >> 23) & 0xffu);
  return e == 0 || e == 255 ? -126 : e - 127;
}
__device__ __forceinline__ bool scale_is_finite(float s) { return (__float_as_uint(s) & 0x7f800000u) != 0x7f800000u; }
// The largest and the smallest exponent among the lanes' scales, -126 and 127 from lanes without one or with one that is not
// finite (it spoils the rows that see it, and has no say in the others').
struct Exponents { int top, low; };
__device__ __forceinline__ Exponents exponents_of(bool there, float s) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const short e = (short)scale_exponent(s);
  s16x2 most{there ? e : (short)-126, (short)(there && scale_is_finite(s) ? -e : -127)};       // both in one word: half the exchanges
  for (int k = 32; k > 0; k >>= 1) most = __builtin_elementwise_max(most, __builtin_bit_cast(s16x2, __shfl_xor(__builtin_bit_cast(int, most), k)));
  return {uni(most[0]), uni(-most[1])};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Wide steps: vs = mantissa * 2^exponent, the mantissa less than 1. A scale that is zero or not finite has the exponent -inf.
__device__ __forceinline__ float wide_exponent(float vs) { return vs != 0.f && scale_is_finite(vs) ? (float)__builtin_amdgcn_frexp_expf(vs) : kMinusInf; }
__device__ __forceinline__ float wide_mantissa(float vs) { return __builtin_amdgcn_frexp_mantf(vs); }
// A row's r after a step whose largest weight is below 2^top and in which the row's reference moved up by `moved`.
__device__ __forceinline__ int row_exponent(int r, float moved, float top) {
  const int older = r - (int)fminf(moved, 1000.f), now = (int)ceilf(fmaxf(top, (float)kLeastR)), y = older > now ? older : now;
  return y > kLeastR ? y : kLeastR;
}

// ---------------------------------------------------------------------------------------------
// Few rows per sequence: a workgroup takes a tile of 16 or 32 rows over a run of key steps, its waves the KV
// heads; where there are more waves than heads, several waves share a head and take its steps in turn.
//
// Measured, with fp8_join_few_kernel: 64 sequences of 1024 to 8192 tokens, 64 query and 8 KV heads of 128, bf16, one new token
// each: 612 MB in 118 + 7 us, 5.2 TB/s while the first kernel runs; 3 of 32k, 32 heads: 186 MB in 37 + 8 us. 24 of up to 5000
// with up to 5 new tokens, 28 and 4 heads: 69 MB in 30 + 6 us; by time stamps its workgroups take 23.5 us on average and 30 at most: 2 to find
// their share, 2 until a tile's first rows are there, 11 for 5 steps (2.2 us each; twice the buffers changed nothing), 6 until the waves
// of a head have joined their sums, the waiting for the slowest of them included. One of 777, 12 and 2 heads: 13 us; 1.8 to find the tile, 2 until the
// first rows are there, 4 for two steps, 4 to join eight waves; the rest is the launch.
//
// Bound by memory: every byte of K and V is read once per row tile. Each wave copies its own steps' rows into its own part
// of LDS (global_load_lds, 16 bytes a lane, whole rows) and never waits for another wave while it goes: scales and the next
// page ids first, then K, then V, each refilled for the next step as soon as it has been read, with the waits
// counted by hand. Eight waves of 256 registers fill a CU; for D = 128 that is not quite enough: 32-row tiles spill 19 (bf16) or 26 (fp16) of
// them, 16-row tiles of fp16 3, where a tile begins and ends. The heads of a page stand side by side in memory, so the waves of a workgroup together read whole
// pages: copies alone run at 6.2 TB/s this way and at 5.2 TB/s with every head in a workgroup of its own. From LDS a lane takes its
// operands' bytes: for K 16 bytes of a key's row (a matrix product does not mind in which order it sums, so the four lanes
// of a row take the 16-byte pieces as they lie), for V the D/16 bytes at one place of its own eight keys' rows, which it
// transposes in registers. At the end the waves of a head join their sums in LDS.
//
// Two ways of cutting the work, chosen by the host: every tile a workgroup of its own (no second launch), or, where sequences
// may be long, even shares: the tiles of all sequences times their key steps form one line, share s of which is slot s's.
// A tile's steps have a few steps' room before them, which stands for what beginning a tile costs a workgroup.
// A tile that lies in one share is finished there; of the others each share leaves (O, m, l), and
// fp8_join_few_kernel joins them.
// ---------------------------------------------------------------------------------------------
template <int D, int TYPE, int NT, int NK>
struct Few {
  static constexpr int kM = 16 * NT;       // rows of a tile
  static constexpr int kWaves = kFewWaves;
  static constexpr int kKeys = 16 * NK;    // keys of a step
  static constexpr int kDT = D / 16;       // bytes of a V row per lane, and row tiles of O^T
  static constexpr int kChunks = D / 16;   // 16-byte pieces of a key's row
  static constexpr int kCopies = kKeys * D / 1024;   // copies of 1 KiB that bring a step's K (or V)
};

// Global memory straight into LDS: lane i's 16 (4) bytes land at `lds` + 16 i (4 i). Written out so that the kernel
// itself says which copies it waits for: the compiler would wait for all of them before any read of LDS.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"      // m0 is a reserved register: named all the same, for the compiler keeps values in it
__device__ __forceinline__ void copy16_to_lds(uint64_t src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void copy4_to_lds(uint64_t src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most N of the wave's newest vector memory accesses are under way.
template <int N>
__device__ __forceinline__ void wait_vmem() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// A barrier for what the workgroup has in LDS: __syncthreads would also wait until stores to global memory have arrived.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
template <class T>
__device__ __forceinline__ uint32_t lds_address(T* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) T*)p;
}

__device__ __forceinline__ uint32_t tiles_of(const Seq& s, const FastDiv& group, int m) { return ((uint32_t)s.n * group.d + m - 1) / m; }
__device__ __forceinline__ uint32_t steps_of(const Seq& s, int keys) { return s.len <= keys ? 1 : ((uint32_t)s.len + keys - 1) / keys; }
template <int M, int KEYS>
__device__ __forceinline__ uint32_t weight_of(const AttendArgs& a, int64_t b) {
  if (b >= a.seq.n_seqs) return 0;
  const Seq s = read_seq(a.seq, b);
  if (!s.ok) raise_flag(a.status, ST_SLOT_SRC);
  return tiles_of(s, a.group, M) * (steps_of(s, KEYS) + (uint32_t)a.begin_cost);
}

// The number of the row tile that sequence b's first row begins: with one token each the sequences have as many tiles
// each; else, if every sequence may leave one tile unfilled, a rising function of b with room for all of its tiles.
template <int M>
__device__ __forceinline__ int64_t first_tile(const AttendArgs& a, int64_t b) {
  if (!a.seq.q_starts) return b * ((a.group.d + M - 1) / M);
  int64_t q = a.seq.q_starts[b];
  q = q < 0 ? 0 : q > a.seq.n_rows ? a.seq.n_rows : q;
  return q * a.group.d / M + b;
}

// The line's length (the host sees to it that it stays below 2^31).
template <int M, int KEYS>
__device__ __forceinline__ uint32_t line_length(const AttendArgs& a, int lane) {
  uint32_t sum = 0;
  for (int64_t b = lane; b < a.seq.n_seqs; b += 64) sum += weight_of<M, KEYS>(a, b);
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  return (uint32_t)uni((int)sum);
}
// The sequence that step x (below the line's length) belongs to, and where in it.
template <int M, int KEYS>
__device__ __forceinline__ int64_t seq_at(const AttendArgs& a, uint32_t x, int lane, uint32_t* local) {
  uint32_t run = 0;
  for (int64_t base = 0; base < a.seq.n_seqs; base += 64) {
    const uint32_t w = weight_of<M, KEYS>(a, base + lane);
    uint32_t upto = w;
    for (int m = 1; m < 64; m <<= 1) {
      const uint32_t y = __shfl_up(upto, m);
      if (lane >= m) upto += y;
    }
    upto += run;
    const uint64_t m = __ballot(upto > x);
    if (m) {
      const int src = __builtin_ctzll(m);
      *local = (uint32_t)uni((int)(x - __shfl(upto - w, src)));
      return base + src;
    }
    run = (uint32_t)uni((int)__shfl(upto, 63));
  }
  *local = 0;
  return a.seq.n_seqs;
}

template <int D, int TYPE, int NT, int NK>
__global__ __launch_bounds__((64 * Few<D, TYPE, NT, NK>::kWaves), 2) void fp8_attend_few_kernel(const AttendArgs a) {
  using C = Few<D, TYPE, NT, NK>;
  constexpr int kM = C::kM, kKeys = C::kKeys, kDT = C::kDT, kChunks = C::kChunks, kCopies = C::kCopies, kWaves = C::kWaves;
  constexpr int kQK = D / 32;              // matrix steps of q . k
  struct Meta {
    u32x4 kv[2][kKeys * kChunks];          // K, V
    uint64_t off[2][kKeys];                // byte offset of the key's row in its plane; of this step and the next
    float ks_in[64], vs_in[64];            // the copies' targets: a step's scales, the next step's page ids
    uint32_t pid_in[2][64];
    float ks[kKeys], vs[kKeys];
    float ex[kKeys];                       // wide steps: the exponents of the V scales, whose mantissas are in vs
    int pos[kKeys];
    int nan_at[D];                         // by place: the first key with a NaN in V that not every row sees
    int r[kM];                             // wide steps: the rows' r
  };
  static_assert(offsetof(Meta, ks) % 16 == 0 && offsetof(Meta, vs) % 16 == 0 && offsetof(Meta, ex) % 16 == 0 && sizeof(Meta) % 16 == 0, "");
  __shared__ Meta metas[kWaves];
  __shared__ float sums[kWaves][2][kM];    // the waves' m and l
  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63;
  const int quad = lane >> 4, col = lane & 15;
  Meta& meta = metas[wave];
  const uint32_t H = (uint32_t)a.layer.heads;
  // the workgroup's heads: `hw` of them from h0 on; wave i does head h0 + i % hw and is its turn i / hw of `ways`
  const uint32_t hw = (uint32_t)a.heads_per_group, groups = (H + hw - 1) / hw;
  const int slot = (int)(blockIdx.x / groups), h0 = (int)((blockIdx.x - slot * groups) * hw);
  const int ways = kWaves / (int)hw, way = wave / (int)hw;
  const int h_raw = h0 + wave - way * (int)hw;
  const bool works = way < ways && h_raw < (int)H;
  const int h = h_raw < (int)H ? h_raw : h0;
  const int G = (int)a.group.d;
  const int P = (int)a.layer.page_tokens.d;

  const uint64_t kbase = (uint64_t)a.layer.k + h * D, vbase = (uint64_t)a.layer.v + h * D;
  const uint64_t ksbase = (uint64_t)a.layer.ks + 4 * h, vsbase = (uint64_t)a.layer.vs + 4 * h;
  const uint32_t lds_k = (uint32_t)uni((int)lds_address(meta.kv[0])), lds_v = (uint32_t)uni((int)lds_address(meta.kv[1]));
  const uint32_t lds_ks = (uint32_t)uni((int)lds_address(meta.ks_in)), lds_vs = (uint32_t)uni((int)lds_address(meta.vs_in));
  const uint32_t lds_pid = (uint32_t)uni((int)lds_address(meta.pid_in));
  // rows whose pieces would meet in a bank: those a whole sweep of the 64 banks (256 bytes) apart
  auto swizzle = [](int row) { return (row / (16 / kChunks)) & (kChunks - 1); };

  Seq seq = {0, 0, 0, false};
  int64_t seq_of = -1;                     // the sequence that `seq` is
  Share line = {1, 0, 0};
  JoinHead join = {0, 0, 0, 0, 0};
  uint32_t local = 0;                      // step of the line within sequence b
  int64_t b = 0;
  if (a.slots > 0) {
    const uint32_t total = line_length<kM, kKeys>(a, lane);
    line = share_of(total, (uint32_t)a.slots, (uint32_t)a.min_steps, (uint32_t)slot);
    if (line.begin < line.end) b = seq_at<kM, kKeys>(a, line.begin, lane, &local);
  } else {
    b = find_seq(a.seq.n_seqs, slot, lane, [&](int64_t i) { return first_tile<kM>(a, i); });
    if (h0 == 0 && tid == 0 && slot < a.seq.n_seqs && !read_seq(a.seq, slot).ok) raise_flag(a.status, ST_SLOT_SRC);
    seq = read_seq(a.seq, b);
    seq_of = b;
    const int64_t tile = slot - first_tile<kM>(a, b);
    if (!seq.ok || tile < 0 || tile >= (int64_t)tiles_of(seq, a.group, kM)) return;
    const uint32_t steps = (uint32_t)uni((int)steps_of(seq, kKeys));
    local = (uint32_t)uni((int)tile) * steps;                    // the host sets begin_cost to 0
    line = {steps, 0, steps};
  }

  uint32_t at = line.begin;
  while (at < line.end && b < a.seq.n_seqs) {
    if (seq_of != b) {
      seq = read_seq(a.seq, b);
      seq_of = b;
    }
    const int steps = uni((int)steps_of(seq, kKeys));
    // a tile's place on the line: its begin_cost, then its steps
    const int room = steps + a.begin_cost;
    const uint32_t weight = (uint32_t)uni((int)(tiles_of(seq, a.group, kM) * (uint32_t)room));
    if (local >= weight) {
      ++b;
      local = 0;
      continue;
    }
    const int tile = (int)(local / (uint32_t)room);
    const int x0 = (int)local - tile * room;
    int taken = room - x0;
    if ((uint32_t)taken > line.end - at) taken = (int)(line.end - at);
    const int step0 = x0 > a.begin_cost ? x0 - a.begin_cost : 0;
    const int count = x0 + taken - a.begin_cost - step0;
    if (count <= 0) break;                                       // the share ends before the tile's steps begin: the next one has them all
    const bool first_of_share = at == line.begin;
    const bool whole = count == steps;
    const int rows = uni((int)((int64_t)seq.n * G - (int64_t)tile * kM < kM ? (int64_t)seq.n * G - (int64_t)tile * kM : kM));
    const int len = uni(seq.len);
    const int before = a.causal ? uni(seq.len - seq.n) : 0;     // keys older than the call's own (negative: some rows see none)
    if (step0 == 0 && !whole) {
      int parts = (int)((at + (room - x0) - 1) / line.per) - slot + 1;
      if (parts > a.slots - slot) parts = a.slots - slot;          // row numbers that make no sense may have wrapped the line's length
      join = {seq.first, tile, rows, parts, 2 * slot + (first_of_share ? 0 : 1)};
    }

    const int last_tok = uni((int)divide((uint32_t)(tile * kM + rows - 1), a.group));
    const int first_tok = uni((int)divide((uint32_t)(tile * kM), a.group));
    int seen = a.causal ? before + last_tok + 1 : len;           // keys that the tile's last row sees
    seen = seen < 0 ? 0 : seen;
    int all = a.causal ? before + first_tok + 1 : len;           // keys that every row sees
    all = all < 0 ? 0 : all;
    int end = step0 + count;
    if (end > (seen + kKeys - 1) / kKeys) end = (seen + kKeys - 1) / kKeys;
    const int begin = works ? step0 + way : end;                 // the wave's steps: begin, begin + ways, ...

    // A step's copies into LDS, in the order in which they are waited for: scales and the next step's page ids, K, V.
    // Keys that are not there (behind the sequence, or on a page the pool does not have) read the
    // plane's first row and are masked by position.
    const uint64_t trow = (uint64_t)(a.seq.table + b * a.seq.table_stride);
    auto key_of = [&](int step) { return step * kKeys + (lane & (kKeys - 1)); };
    auto copy_pages = [&](int step) {
      int key = key_of(step);
      key = key < seen ? key : seen - 1;
      const uint64_t src = trow + 8 * (uint64_t)divide((uint32_t)key, a.layer.page_tokens);
      copy4_to_lds(src, lds_pid);
      copy4_to_lds(src + 4, lds_pid + 256);
    };
    bool bad_page = false;
    auto copy_scales = [&](int step, int which) {                // returns the position of the lane's key
      const int key = key_of(step);
      const uint64_t pid = meta.pid_in[0][lane] | ((uint64_t)meta.pid_in[1][lane] << 32);
      const bool in = key < seen, ok = in && pid < (uint64_t)a.layer.n_pages;
      bad_page |= in && !ok;
      const int64_t page = ok ? (int64_t)pid : 0;
      uint32_t in_page = (uint32_t)key - divide((uint32_t)key, a.layer.page_tokens) * (uint32_t)P;
      in_page = ok ? in_page : 0;
      meta.off[which][lane & (kKeys - 1)] = (uint64_t)(page * a.layer.page_stride) + (uint64_t)in_page * (uint64_t)a.layer.token_stride;
      copy4_to_lds(ksbase + (uint64_t)(page * a.layer.scale_stride), lds_ks);
      copy4_to_lds(vsbase + (uint64_t)(page * a.layer.scale_stride), lds_vs);
      return ok ? key : kNoKey;
    };
    // A row's 16-byte pieces are XOR-ed with its number on the way, so that reads of a column spread over the banks; a
    // copy still takes whole rows.
    auto copy_rows = [&](int which, uint64_t base, uint32_t lds) {       // a loop: its code, not its time, is what the first step waits for
#pragma nounroll
      for (int i = 0; i < kCopies; ++i) {
        const int row = i * (64 / kChunks) + lane / kChunks;
        copy16_to_lds(base + meta.off[which][row] + 16 * ((lane & (kChunks - 1)) ^ swizzle(row)), lds + 1024 * i);
      }
    };

    if (begin < end) copy_pages(begin);
    // The lane's rows: row tile*kM + 16 t + col.
    uint32_t tok[NT];
    int head[NT], limit[NT];
    bool live[NT];
    u32x4 q[NT][kQK];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = 16 * t + col;
      live[t] = r < rows;
      const uint32_t row = (uint32_t)(tile * kM + (live[t] ? r : 0));
      tok[t] = divide(row, a.group);
      head[t] = h * G + (int)(row - tok[t] * G);
      limit[t] = a.causal ? before + (int)tok[t] + 1 : len;
      if (limit[t] < 0) limit[t] = 0;
      const uint64_t src = (uint64_t)a.q + 2 * ((seq.first + tok[t]) * a.q_row + head[t] * a.q_head);
#pragma unroll
      for (int j = 0; j < kQK; j += 2) {
        const uint64_t p = src + 2 * (32 * j + 16 * quad);
        q[t][j] = gload<u32x4>(p);
        q[t][j + 1] = gload<u32x4>(p + 16);
      }
    }

#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < kQK; ++j) asm volatile("" : "+v"(q[t][j]));     // here before the copies are counted

    f32x4 o[NT][kDT];
    float m[NT], l[NT];
    int r_exp = -126, r_low = 127;         // exponents of the V scales read so far
    bool wide = false, spoilt = false;
    for (int d = lane; d < D; d += 64) meta.nan_at[d] = kNoKey;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kMinusInf;
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < kDT; ++i) o[t][i] = f32x4{0, 0, 0, 0};
    }

    auto compute = [&](int step, int which, int pos, bool more) {
      wait_vmem<kCopies>();                                      // all but V
      const float ks_in = meta.ks_in[lane], vs_in = meta.vs_in[lane];
      // a larger V scale than any before: what is summed moves to its exponent, or the steps are wide from here on
      const int e = pos != kNoKey ? scale_exponent(vs_in) : -126;
      if (!wide && __ballot(e > r_exp || (e < r_low && pos != kNoKey && scale_is_finite(vs_in)))) {
        const Exponents now = exponents_of(pos != kNoKey, vs_in);
        const int top = now.top > r_exp ? now.top : r_exp;
        r_low = now.low < r_low ? now.low : r_low;
        wide = top - r_low > kSpread;
        if (wide && lane < kM) meta.r[lane] = r_exp;
        const int by = wide ? 0 : r_exp - top;                   // no branch: in two ways the sums would be held twice
        r_exp = wide ? r_exp : top;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < kDT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[t][i][c] = ldexpf(o[t][i][c], by);
      }
      meta.ks[lane & (kKeys - 1)] = ks_in * a.scale_log2;
      meta.vs[lane & (kKeys - 1)] = wide ? wide_mantissa(vs_in) : ldexpf(vs_in, kPShift - r_exp);
      if (wide) meta.ex[lane & (kKeys - 1)] = wide_exponent(vs_in);
      meta.pos[lane & (kKeys - 1)] = pos;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const bool edge = (step + 1) * kKeys > all || __ballot(pos == kNoKey) != 0;

      __builtin_amdgcn_sched_barrier(0);
      // S^T = K Q^T; what it needs from LDS is asked for at once, not piece by piece with a wait for each
      u32x4 kx[NK][D / 64];
      f32x4 ks[NK], vs[NK];
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int j = 0; j < D / 64; ++j) kx[i][j] = meta.kv[0][(16 * i + col) * kChunks + ((4 * j + quad) ^ swizzle(16 * i + col))];
#pragma unroll
      for (int i = 0; i < NK; ++i) ks[i] = *reinterpret_cast<const f32x4*>(&meta.ks[16 * i + 4 * quad]);
      __builtin_amdgcn_sched_barrier(0);
      f32x4 s[NT][NK];
#pragma unroll
      for (int i = 0; i < NK; ++i) {
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          u32x4 f[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const u32x2 lo = widen4<TYPE>(kx[i][j][2 * half]), hi = widen4<TYPE>(kx[i][j][2 * half + 1]);
            f[half] = u32x4{lo[0], lo[1], hi[0], hi[1]};
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            s[t][i] = mfma16<TYPE>(f[0], q[t][2 * j], s[t][i]);
            s[t][i] = mfma16<TYPE>(f[1], q[t][2 * j + 1], s[t][i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NK; ++i) vs[i] = *reinterpret_cast<const f32x4*>(&meta.vs[16 * i + 4 * quad]);
      __builtin_amdgcn_sched_barrier(0);
      int next = kNoKey;
      if (more) {
        next = copy_scales(step + ways, which ^ 1);
        copy_pages(step + 2 * ways);
        copy_rows(which ^ 1, kbase, lds_k);
      }
      __builtin_amdgcn_sched_barrier(0);
      // softmax: the lane's keys are 16 i + 4 quad + c
      const float counted = wide ? 0.f : 1.f;
      u32x4 p[NT][NK / 2], p_low[NT][TYPE == 1 ? NK / 2 : 1];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t hidden = 0;                     // bit per key of the lane: the row does not see it
        float top = kMinusInf;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[t][i][c] *= ks[i][c];
        if (edge) {
#pragma unroll
          for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (meta.pos[16 * i + 4 * quad + c] >= limit[t]) {
                s[t][i][c] = kMinusInf;
                hidden |= 1u << (4 * i + c);
              }
        }
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) top = fmaxf(top, s[t][i][c]);
        if (wide || __ballot(top > m[t] + kSlack)) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float now = fmaxf(m[t], top);
          const float grow = now == kMinusInf ? 1.f : exp2_fast(m[t] - now);       // 0 at the first key
          const float moved = now == m[t] ? 0.f : now - m[t];
          m[t] = now;
          l[t] *= grow;
#pragma unroll
          for (int i = 0; i < kDT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[t][i][c] *= grow;
          if (wide) {                              // l by itself; z then takes the scale's exponent along, relative to the row's r
            float most = kMinusInf;
#pragma unroll
            for (int i = 0; i < NK; ++i) {
              const f32x4 ex = *reinterpret_cast<const f32x4*>(&meta.ex[16 * i + 4 * quad]);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                s[t][i][c] -= m[t] == kMinusInf ? 0.f : m[t];
                l[t] += exp2_fast(s[t][i][c]);
                most = fmaxf(most, s[t][i][c] + ex[c]);
              }
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const int was = meta.r[16 * t + col], r = row_exponent(was, moved, most);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            meta.r[16 * t + col] = r;
#pragma unroll
            for (int i = 0; i < kDT; ++i)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[t][i][c] = ldexpf(o[t][i][c], was - r);
#pragma unroll
            for (int i = 0; i < NK; ++i) {
              const f32x4 ex = *reinterpret_cast<const f32x4*>(&meta.ex[16 * i + 4 * quad]);
#pragma unroll
              for (int c = 0; c < 4; ++c) s[t][i][c] += ex[c] + (float)(kPShift - r);
            }
          }
        }
        const float from = wide || m[t] == kMinusInf ? 0.f : m[t];
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float e = exp2_fast(s[t][i][c] - from);
            l[t] = fmaf(e, counted, l[t]);
            s[t][i][c] = e * vs[i][c];
          }
        if (edge) {                              // 0 times a scale that is not finite
#pragma unroll
          for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if ((hidden >> (4 * i + c)) & 1u) s[t][i][c] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float f0 = s[t][i][2 * c], f1 = s[t][i][2 * c + 1];
            const uint32_t y = pack_f16(f0, f1);
            p[t][i / 2][2 * (i & 1) + c] = y;
            if constexpr (TYPE == 1) p_low[t][i / 2][2 * (i & 1) + c] = pack_f16(less_half<0>(f0, y), less_half<1>(f1, y));
          }
      }
      if (more) wait_vmem<4 + kCopies>();                        // all but what has just been asked for
      else wait_vmem<0>();
      uint32_t xv[NK][4][kDT / 4];
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = 16 * i + 4 * quad + c;
          const uint32_t* piece = reinterpret_cast<const uint32_t*>(&meta.kv[1][row * kChunks + ((col * kDT / 16) ^ swizzle(row))]) + (col * kDT / 4) % 4;
          if constexpr (kDT == 8) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(piece);
            xv[i][c][0] = x[0];
            xv[i][c][1] = x[1];
          } else {
            xv[i][c][0] = piece[0];
          }
        }
      // V^T operands: eight keys' bytes at four places, transposed
      auto operands = [&](int i, int dw, u32x4 (&f)[4]) {
        u32x2 x8[8];                             // [key] -> places (0, 1) and (2, 3) of the dword
#pragma unroll
        for (int c = 0; c < 8; ++c) x8[c] = widen4<1>(xv[i + c / 4][c & 3][dw]);
#pragma unroll
        for (int pl = 0; pl < 4; ++pl)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            f[pl][c] = __builtin_amdgcn_perm(x8[2 * c + 1][pl / 2], x8[2 * c][pl / 2], pl & 1 ? 0x07060302u : 0x05040100u);
      };
      if (edge) {
        // Bytes of keys that nobody sees become zero, and so does a NaN: the rows that see its key get it at the end.
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool gone = meta.pos[16 * i + 4 * quad + c] == kNoKey;
#pragma unroll
            for (int dw = 0; dw < kDT / 4; ++dw) {
              const uint32_t bytes = gone ? 0 : xv[i][c][dw], bad = nan_bytes(bytes);
              any |= bad;
              xv[i][c][dw] = bytes & ~bad;
            }
          }
        if (__ballot(any != 0)) {
          spoilt = true;
          if (lane < kKeys && pos != kNoKey) note_nans<D>(meta.nan_at, vbase + meta.off[which][lane], pos);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // O^T += V^T P^T, 32 keys at a time
#pragma unroll
      for (int i = 0; i < NK; i += 2)
#pragma unroll
        for (int dw = 0; dw < kDT / 4; ++dw) {
          u32x4 f[4];
          operands(i, dw, f);
#pragma unroll
          for (int pl = 0; pl < 4; ++pl)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              o[t][4 * dw + pl] = mfma16<1>(f[pl], p[t][i / 2], o[t][4 * dw + pl]);
              if constexpr (TYPE == 1) o[t][4 * dw + pl] = mfma16<1>(f[pl], p_low[t][i / 2], o[t][4 * dw + pl]);
            }
        }
      __builtin_amdgcn_sched_barrier(0);
      if (more) copy_rows(which ^ 1, vbase, lds_v);
      __builtin_amdgcn_sched_barrier(0);
      return next;
    };

    if (begin < end) {
      wait_vmem<0>();
      int pos = copy_scales(begin, 0);
      copy_pages(begin + ways);
      copy_rows(0, kbase, lds_k);
      copy_rows(0, vbase, lds_v);
      int which = 0;
      for (int step = begin; step < end; step += ways, which ^= 1) pos = compute(step, which, pos, step + ways < end);
      if (bad_page) raise_flag(a.status, ST_SLOT_PAGE);
    }

    // The lane holds, of row 16 t + col, places kDT * (4 quad + c) + dt.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (spoilt) {
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int from = meta.nan_at[kDT * (4 * quad + c) + dt];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (from < limit[t]) o[t][dt][c] = __uint_as_float(0x7fc00000u);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] += __shfl_xor(l[t], 16);
      l[t] += __shfl_xor(l[t], 32);
    }
    auto r_of = [&](int t) { return (wide ? meta.r[16 * t + col] : r_exp) - kPShift; };    // what comes off the row's sums
    const int64_t part0 = ((int64_t)(2 * slot + (first_of_share ? 0 : 1)) * H) * kM;       // the segment's place among the parts
    // What is known of a row once all of its keys in the segment are: its lse, or its (m, l)
    auto leave_sum = [&](int r, uint32_t token, int hd, float top, float sum) {
      if (whole) {
        if (a.lse) a.lse[(seq.first + token) * (int64_t)(H * G) + hd] = sum == 0.f ? kMinusInf : (top + __log2f(sum)) * 0.69314718055994530942f;
      } else {
        const int64_t part = part0 + (int64_t)h * kM + r;
        a.part_ml[2 * part] = top;
        a.part_ml[2 * part + 1] = sum;
      }
    };
    if (ways == 1) {
      if (works)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (!live[t]) continue;
          const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];
          const int off = r_of(t);
          if (quad == 0) leave_sum(16 * t + col, tok[t], head[t], m[t], l[t]);
          const uint64_t dst = whole ? (uint64_t)a.out + 2 * ((seq.first + tok[t]) * a.o_row + head[t] * a.o_head)
                                     : (uint64_t)(a.part_o + (part0 + (int64_t)h * kM + 16 * t + col) * D);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float y[kDT];
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt) y[dt] = ldexpf(o[t][dt][c] * inv, off);
            const int d = kDT * (4 * quad + c);
            if (whole) {
              if constexpr (kDT == 8)
                gstore<u32x4>(dst + 2 * d, u32x4{narrow<TYPE>(y[0], y[1]), narrow<TYPE>(y[2], y[3]), narrow<TYPE>(y[4], y[5]), narrow<TYPE>(y[6], y[7])});
              else
                gstore<u32x2>(dst + 2 * d, u32x2{narrow<TYPE>(y[0], y[1]), narrow<TYPE>(y[2], y[3])});
            } else {
#pragma unroll
              for (int dt = 0; dt < kDT; dt += 4) gstore<f32x4>(dst + 4 * (d + dt), f32x4{y[dt], y[dt + 1], y[dt + 2], y[dt + 3]});
            }
          }
        }
    } else {
      // The waves of a head: each brings its sums to the common maximum and divides them by the common l; 16 rows at a time
      // go through the waves' K and V space, which is free by now.
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (quad == 0) {
          sums[wave][0][16 * t + col] = m[t];
          sums[wave][1][16 * t + col] = l[t];
        }
      lds_barrier();
      const int first = wave - way * (int)hw;                        // the head's first wave; the others follow hw apart
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int r = 16 * t + col;
        float top = kMinusInf, sum = 0.f;
        float mi[kWaves], li[kWaves];                                // all at once: a loop would wait for LDS at every turn
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          const int from_wave = i < ways ? first + i * (int)hw : first;
          mi[i] = sums[from_wave][0][r];
          li[i] = i < ways ? sums[from_wave][1][r] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = fmaxf(top, mi[i]);
        const float from = top == kMinusInf ? 0.f : top;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) sum += li[i] == 0.f ? 0.f : li[i] * exp2_fast(mi[i] - from);
        const float mine = l[t] == 0.f ? 0.f : exp2_fast(m[t] - from) / sum;
        const int off = r_of(t);
        float* space = reinterpret_cast<float*>(meta.kv);            // 16 rows of D floats
        // a row's 16-byte pieces are XOR-ed with its number: sixteen lanes write sixteen rows at one place
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int dt = 0; dt < kDT; dt += 4) {
            f32x4 y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = ldexpf(o[t][dt + k][c] * mine, off);
            *reinterpret_cast<f32x4*>(space + col * D + 4 * (((kDT * (4 * quad + c) + dt) / 4) ^ (col & (D / 4 - 1)))) = y;
          }
        if (works && way == 0 && quad == 0 && live[t]) leave_sum(r, tok[t], head[t], top, sum);
        lds_barrier();
        // way i of the head adds up rows i, i + ways, ...; four places a lane
        constexpr int kRowLanes = D / 4, kRowsAtOnce = 64 / kRowLanes;
        const int j = lane % kRowLanes;
        for (int rr = way * kRowsAtOnce + lane / kRowLanes; works && rr < 16 && 16 * t + rr < rows; rr += ways * kRowsAtOnce) {
          f32x4 y = {0, 0, 0, 0};
          f32x4 x[kWaves];
#pragma unroll
          for (int i = 0; i < kWaves; ++i)
            x[i] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(metas[i < ways ? first + i * (int)hw : first].kv) + rr * D + 4 * (j ^ (rr & (D / 4 - 1))));
#pragma unroll
          for (int i = 0; i < kWaves; ++i)
            if (i < ways) y += x[i];
          const uint32_t row = (uint32_t)(tile * kM + 16 * t + rr), tk = divide(row, a.group);
          if (whole)
            gstore<u32x2>((uint64_t)a.out + 2 * ((seq.first + tk) * a.o_row + (h * G + (int)(row - tk * G)) * a.o_head + 4 * j),
                          u32x2{narrow<TYPE>(y[0], y[1]), narrow<TYPE>(y[2], y[3])});
          else
            gstore<f32x4>((uint64_t)(a.part_o + (part0 + (int64_t)h * kM + 16 * t + rr) * D + 4 * j), y);
        }
        lds_barrier();                                             // before the space is written again
      }
    }
    at += taken;
    local += taken;
  }
  if (a.slots > 1 && h0 == 0 && tid == 0) a.part_join[slot] = join;
}

// Joins `n` partial results of one row: weights l_i 2^(m_i - max m). A wave does a row; `at(i)` is the index of the
// i-th part. Parts that saw no key have weight 0 and are not read.
template <int D, int TYPE, class F>
__device__ __forceinline__ void join_row(const AttendArgs& a, int lane, int n, F at, int64_t row, int head, int q_heads) {
  float top = kMinusInf;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, a.part_ml[2 * at(i)]);
  for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
  const float from = top == kMinusInf ? 0.f : top;
  constexpr int kLanes = D / 4;             // lanes that hold one part's row, four floats each
  constexpr int kParts = 64 / kLanes;       // parts read at once
  const int sub = lane / kLanes, d = (lane % kLanes) * 4;
  f32x4 o = {0, 0, 0, 0};
  float sum = 0.f;
  for (int base = 0; base < n; base += 64) {
    float w = 0.f;
    int64_t idx = 0;
    if (base + lane < n) {
      idx = at(base + lane);
      w = a.part_ml[2 * idx + 1];
      if (w != 0.f) w *= exp2_fast(a.part_ml[2 * idx] - from);
    }
    sum += w;
    const int here = n - base < 64 ? n - base : 64;
    constexpr int kAtOnce = 8;              // loads under way
    for (int i0 = 0; i0 < here; i0 += kParts * kAtOnce) {
      f32x4 y[kAtOnce];
      float wi[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = i0 + u * kParts + sub, in = i < here ? i : here - 1;
        wi[u] = __shfl(w, in);
        wi[u] = i < here ? wi[u] : 0.f;
        y[u] = gload<f32x4>((uint64_t)(a.part_o + at(base + in) * D + d));
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (wi[u] != 0.f)                   // what a part without weight holds was never written
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] += wi[u] * y[u][c];
    }
  }
  for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
#pragma unroll
  for (int k = 32; k >= kLanes; k >>= 1)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] += __shfl_xor(o[c], k);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (sub == 0)
    gstore<u32x2>((uint64_t)a.out + 2 * (row * a.o_row + head * a.o_head + d),
                  u32x2{narrow<TYPE>(o[0] * inv, o[1] * inv), narrow<TYPE>(o[2] * inv, o[3] * inv)});
  if (a.lse && lane == 0) a.lse[row * q_heads + head] = sum == 0.f ? kMinusInf : (top + __log2f(sum)) * 0.69314718055994530942f;
}

// A wave per row, a workgroup per (slot, KV head) and four rows: joins the tile that begins in the slot's share and ends behind it, if
// there is one (the slot has left word). The parts are summed in the order of the shares, so the result does not depend on timing.
template <int D, int TYPE, int M>
__global__ __launch_bounds__(256) void fp8_join_few_kernel(const AttendArgs a) {
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int H = a.layer.heads, G = (int)a.group.d;
  const int slot = blockIdx.x / H, h = blockIdx.x - slot * H;
  const JoinHead j = a.part_join[slot];
  const int r = blockIdx.y * 4 + wave;
  if (r < j.rows) {
    const uint32_t row = (uint32_t)(j.tile * M + r), tok = divide(row, a.group);
    auto at = [&](int i) { return ((int64_t)(i == 0 ? j.first_index : 2 * (slot + i)) * H + h) * M + r; };
    join_row<D, TYPE>(a, lane, j.parts, at, j.first_row + tok, h * G + (int)(row - tok * G), H * G);
  }
}

// ---------------------------------------------------------------------------------------------
// Many rows per sequence: a workgroup of four waves does 128 rows of one KV head, 32 a wave, over the
// keys 64 at a time.
//
// Measured: a prompt of 4096 tokens, 32 query and 8 KV heads of 128, fp16, causal: 137 GFLOP in 250 us (550 TFLOP/s); 6 chunks of
// up to 900 tokens behind up to 8192, 64 and 8 heads, bf16: 556 GFLOP in 777 us (715 TFLOP/s); 5 of up to 700 tokens and
// 1500 keys, 16 and 2 heads of 64, fp16, not causal: 9.3 GFLOP in 40 us.
//
// Bound by what the matrix products (4 D flops per visible row and key), the softmax beside them (an exp2 and some six other
// instructions per row and key) and the reads from LDS (a wave's 32 rows need the whole step's K and V) take together: of the
// second case's time the matrix cores are busy 28 %, the vector units 45 %, LDS 37 %, and two waves to a SIMD, all that
// registers allow, overlap little of it. So products and softmax are interleaved by halves of a step, and what a step needs from
// LDS is read half a step ahead. For 64-wide heads it is the length of that chain, 2.3 us a step, also for a wave that has
// its SIMD to itself. fp16 rows carry P in two halves (see the file's head: P has 11 bits, as much as the output), which makes
// twice the products of O.
//
// K and V are widened once per workgroup. Threads bring them as bytes into registers while the step before is computed, K as
// 16-byte pieces of rows, V as four bytes of each of eight keys, and put them into LDS afterwards: K as [key][D] in
// q's type, V transposed as [D][key] in fp16 with the keys in the order in which P lies in the lanes. 16-byte
// pieces of a row are XOR-ed with the row number, so that neither the writes nor the reads of a column meet in
// a bank. Two LDS buffers, one barrier a step.
//
// A tile's keys are cut into `slots` parts where the tiles alone would not fill the chip; the parts' results are
// joined by fp8_join_many_kernel.
// ---------------------------------------------------------------------------------------------
constexpr int kWide = 1 << 20;          // in r's place: the step is a wide one

template <int TYPE>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (TYPE == 0)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int D, int TYPE>
__global__ __launch_bounds__(kManyThreads, 2) void fp8_attend_many_kernel(const AttendArgs a) {
  constexpr int kKeys = kManyKeys;
  constexpr int kChunks = D / 8;                  // 16-byte pieces of a K row in LDS
  constexpr int kLoads = D / 64;                  // 16-byte pieces of K a thread brings per step
  constexpr int kRowThreads = D / 4;              // threads that bring one row of V, four bytes each
  struct alignas(16) Meta {                       // four floats are read at a time
    uint64_t off[kKeys];
    float ks[kKeys], vs[kKeys];                   // as they are in the cache; then times the softmax's scale and log2(e), and times 2^(kPShift - r)
    float ex[kKeys];                              // wide steps: the exponents of the V scales, whose mantissas are in vs then
    int pos[kKeys];
    int gone, r;                                  // some key is nobody's; the largest exponent of V's scales up to here, or kWide
    Exponents e;                                  // of V's scales here
  };
  static_assert(offsetof(Meta, ks) % 16 == 0 && offsetof(Meta, vs) % 16 == 0 && offsetof(Meta, ex) % 16 == 0 && sizeof(Meta) % 16 == 0, "");
  __shared__ uint32_t pids_in[4][2][kKeys];       // page ids of the keys to be looked up next, low and high words
  __shared__ int nan_at[D];                       // by place: the first key with a NaN in V that not every row sees
  __shared__ int spoilt;
  __shared__ int row_r[kManyRows];                // wide steps: the rows' r
  __shared__ u32x4 k_lds[2][kKeys * kChunks];
  __shared__ u32x4 v_lds[2][D * 8];
  __shared__ Meta metas[8];
  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63;
  const int half = lane >> 5, col = lane & 31;
  const uint32_t H = (uint32_t)a.layer.heads;
  const uint32_t id = blockIdx.x;
  const int h = (int)(id % H);
  const uint32_t rest = id / H;
  const int part = (int)(rest % (uint32_t)a.slots);
  const int64_t slot = a.tiles - 1 - (int64_t)(rest / (uint32_t)a.slots);   // the last rows of a prompt see most keys: first
  const int G = (int)a.group.d;
  const int P = (int)a.layer.page_tokens.d;

  const int64_t b = find_seq(a.seq.n_seqs, slot, lane, [&](int64_t i) { return first_tile<kManyRows>(a, i); });
  if (h == 0 && part == 0 && slot < a.seq.n_seqs && tid == 0 && !read_seq(a.seq, slot).ok) raise_flag(a.status, ST_SLOT_SRC);
  const Seq seq = read_seq(a.seq, b);
  const int64_t tile64 = slot - first_tile<kManyRows>(a, b);
  const int64_t n_rows = (int64_t)seq.n * G;
  if (!seq.ok || tile64 < 0 || tile64 * kManyRows >= n_rows) return;
  const int tile = uni((int)tile64);
  const int rows = uni((int)(n_rows - (int64_t)tile * kManyRows < kManyRows ? n_rows - (int64_t)tile * kManyRows : kManyRows));
  const int len = uni(seq.len);
  const int before = uni(seq.len - seq.n);
  const int row0 = tile * kManyRows;
  auto sees = [&](int row) {                       // keys that row `row` of the sequence sees
    const int n = a.causal ? before + (int)divide((uint32_t)row, a.group) + 1 : len;
    return n < 0 ? 0 : n;
  };
  const int seen = uni(sees(row0 + rows - 1));
  const int steps = (seen + kKeys - 1) / kKeys;
  const int per = (steps + a.slots - 1) / a.slots;
  const int t0 = part * per, t1 = t0 + per < steps ? t0 + per : steps;

  auto opaque = [](uint32_t x) {                   // keeps the compiler from holding in registers what it could work out again
    asm volatile("" : "+v"(x));
    return x;
  };
  // the wave's rows: row0 + 32 wave + col
  struct Row { int r; bool live; uint32_t tok; int head; };
  auto my_row = [&](int c) {
    Row y;
    y.r = 32 * wave + c;
    y.live = y.r < rows;
    const uint32_t row = (uint32_t)(row0 + (y.live ? y.r : 0));
    y.tok = divide(row, a.group);
    y.head = h * G + (int)(row - y.tok * G);
    return y;
  };
  const int limit = sees(row0 + (32 * wave + col < rows ? 32 * wave + col : 0));
  const int wave_last = 32 * wave + 31 < rows ? 32 * wave + 31 : rows - 1;
  const int wave_seen = uni(32 * wave < rows ? sees(row0 + wave_last) : 0);
  const int wave_all = uni(32 * wave < rows ? sees(row0 + 32 * wave) : 0);
  const int all = uni(sees(row0));                 // keys that every row of the tile sees
  u32x4 q[D / 16];
  {
    const Row me = my_row(col);
    const uint64_t src = (uint64_t)a.q + 2 * ((seq.first + me.tok) * a.q_row + me.head * a.q_head);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) q[j] = gload<u32x4>(src + 2 * (16 * j + 8 * half));
  }

  const uint64_t kbase = (uint64_t)a.layer.k + h * D, vbase = (uint64_t)a.layer.v + h * D;
  const uint64_t trow = (uint64_t)(a.seq.table + b * a.seq.table_stride);
  // The keys of four steps are looked up at a time, a step's by each wave, in stages a step or more apart and through
  // copies into LDS that hold no registers meanwhile: page ids; with them places and scales; with the scales
  // their largest exponent; with those of all four what is left of the steps' metas. Step t's is metas[(t - t0) & 7].
  uint32_t (*pid_in)[kKeys] = pids_in[wave];
  const uint32_t lds_pid = (uint32_t)uni((int)lds_address(pid_in));
  auto table_at = [&](int t) {
    int key = t * kKeys + lane;
    key = key < seen ? key : seen - 1;
    return trow + 8 * (uint64_t)divide((uint32_t)key, a.layer.page_tokens);
  };
  auto copy_pages = [&](int t) {
    copy4_to_lds(table_at(t), lds_pid);
    copy4_to_lds(table_at(t) + 4, lds_pid + 4 * kKeys);
  };
  bool bad_page = false;
  auto look_up = [&](int t, uint64_t pid, Meta& m) {
    const int key = t * kKeys + lane;
    const bool in = key < seen, ok = in && pid < (uint64_t)a.layer.n_pages;
    bad_page |= in && !ok;
    const int64_t page = ok ? (int64_t)pid : 0;                    // keys that are not there read the plane's first row
    uint32_t in_page = (uint32_t)key - divide((uint32_t)key, a.layer.page_tokens) * (uint32_t)P;
    in_page = ok ? in_page : 0;
    m.off[lane] = (uint64_t)(page * a.layer.page_stride) + (uint64_t)in_page * (uint64_t)a.layer.token_stride;
    m.pos[lane] = ok ? key : kNoKey;
    const bool gone = __ballot(!ok) != 0;
    if (lane == 0) m.gone = gone;
    copy4_to_lds((uint64_t)a.layer.ks + 4 * h + (uint64_t)(page * a.layer.scale_stride), (uint32_t)uni((int)lds_address(m.ks)));
    copy4_to_lds((uint64_t)a.layer.vs + 4 * h + (uint64_t)(page * a.layer.scale_stride), (uint32_t)uni((int)lds_address(m.vs)));
  };
  auto find_exponents = [&](Meta& m) {
    const Exponents e = exponents_of(m.pos[lane] != kNoKey, m.vs[lane]);
    if (lane == 0) m.e = e;
  };
  int r_seen = -126, r_low = 127;
  auto finish = [&](int first, Meta& m) {                          // first: the ring's index of the four steps' first
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int top = uni(metas[first + i].e.top), low = uni(metas[first + i].e.low);
      r_seen = top > r_seen ? top : r_seen;
      r_low = low < r_low ? low : r_low;
    }
    const bool wide = r_seen - r_low > kSpread;
    m.ks[lane] *= a.scale_log2;
    const float vs = m.vs[lane];
    m.vs[lane] = wide ? wide_mantissa(vs) : ldexpf(vs, kPShift - r_seen);
    if (wide) m.ex[lane] = wide_exponent(vs);
    if (lane == 0) m.r = wide ? kWide : r_seen;
  };

  // Bringing a step's bytes: of K a thread takes whole 16-byte pieces, of V four bytes of each of eight keys.
  const int vg = tid / kRowThreads & 7, v_at = 4 * (tid % kRowThreads);
  u32x4 raw_k[kLoads];
  uint32_t raw_v[8];
  auto v_key = [&](int c) { return 16 * (vg >> 1) + 8 * (c >> 2) + 4 * (vg & 1) + (c & 3); };
  // Byte offsets in a buffer. A row's 16-byte pieces are XOR-ed with a number that all rows the same lane touches share, so
  // every access is one base, XOR a constant, plus a constant. The bases go through an empty asm in every step:
  // otherwise the compiler keeps each of the two dozen sums in a register of its own and spills them.
  constexpr int kKRow = 2 * D, kVRow = 2 * kKeys;
  auto swizzle_k = [](int key) { return kChunks == 16 ? key & 15 : (key >> 1) & 7; };
  auto swizzle_v = [](int d) { return ((d >> 1) & 7) ^ ((d >> 4) & 1); };
  auto at_k = [&](int buf, uint32_t off) -> u32x4& { return *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(k_lds) + buf * (int)sizeof(k_lds[0]) + off); };
  auto at_v = [&](int buf, uint32_t off) -> u32x4& { return *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(v_lds) + buf * (int)sizeof(v_lds[0]) + off); };
  constexpr int kPieces = D / 16;
  const uint32_t k_write = (tid / kPieces) * kKRow + 16 * ((2 * (tid % kPieces)) ^ swizzle_k(tid / kPieces));
  const uint32_t v_write = v_at * kVRow + 16 * (vg ^ swizzle_v(v_at));
  const uint32_t k_read = col * kKRow + 16 * (half ^ swizzle_k(col)), v_read = col * kVRow + 16 * (half ^ swizzle_v(col));
  auto bring = [&](const Meta& m) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) raw_k[i] = gload<u32x4>(kbase + m.off[i * (256 / kPieces) + tid / kPieces] + 16 * (tid % kPieces));
#pragma unroll
    for (int c = 0; c < 8; ++c) raw_v[c] = gload<uint32_t>(vbase + m.off[v_key(c)] + v_at);
  };
  auto put = [&](int t, int buf, const Meta& m, bool gone) {
    static_assert(256 / kPieces % 16 == 0, "the rows of a thread's pieces share their swizzle");
    const uint32_t k_at = opaque(k_write);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x2 lo = widen4<TYPE>(raw_k[i][2 * e]), hi = widen4<TYPE>(raw_k[i][2 * e + 1]);
        at_k(buf, (k_at ^ (16 * e)) + i * (256 / kPieces) * kKRow) = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    if ((t + 1) * kKeys > all || gone) {
      // bytes of keys that nobody sees become zero, and so does a NaN: the rows that see its key get it at the end
      uint32_t any = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint32_t bytes = m.pos[v_key(c)] == kNoKey ? 0 : raw_v[c], bad = nan_bytes(bytes);
        any |= bad;
        raw_v[c] = bytes & ~bad;
      }
      if (__ballot(any != 0)) {
        spoilt = 1;
        if (m.pos[lane] != kNoKey) note_nans<D>(nan_at, vbase + m.off[lane], m.pos[lane]);
      }
    }
    if (tid < 8 * kRowThreads) {
      const uint32_t at = opaque(v_write);
      u32x2 x8[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) x8[c] = widen4<1>(raw_v[c]);
#pragma unroll
      for (int pl = 0; pl < 4; ++pl) {
        u32x4 f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          f[c] = __builtin_amdgcn_perm(x8[2 * c + 1][pl / 2], x8[2 * c][pl / 2], pl & 1 ? 0x07060302u : 0x05040100u);
        at_v(buf, (at ^ (16 * (pl >> 1))) + pl * kVRow) = f;
      }
    }
  };

  f32x16 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m_run = kMinusInf, l_run = 0.f;
  int r_exp = -126;
  auto scale_sums = [&](float by) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int c = 0; c < 16; ++c) o[i][c] *= by;
  };

  auto shift_sums = [&](int by) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int c = 0; c < 16; ++c) o[i][c] = ldexpf(o[i][c], by);
  };

  auto compute = [&](int t, int buf, const Meta& meta, int r, bool gone) {
    const bool wide = r == kWide;
    if (r != r_exp) {
      if (wide) row_r[32 * wave + col] = r_exp;
      shift_sums(wide ? 0 : r_exp - r);
      r_exp = r;
    }
    const bool edge = (t + 1) * kKeys > wave_all || gone;
    // Operands are read from LDS half a step ahead of the products that use them, each into the registers of the
    // operand just used; left alone, the compiler reads each one right before its product and waits for it.
    f32x16 s[2];
    u32x4 kf[D / 16];
    f32x4 ks[2][4];
    auto read_ks = [&](int kb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) ks[kb][i] = *reinterpret_cast<const f32x4*>(&meta.ks[32 * kb + 8 * i + 4 * half]);
    };
    const uint32_t k_at = opaque(k_read), v_at = opaque(v_read);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) kf[j] = at_k(buf, k_at ^ (32 * j));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      s[0] = mfma32<TYPE>(kf[j], q[j], s[0]);
      kf[j] = at_k(buf, (k_at ^ (32 * j)) + 32 * kKRow);
      __builtin_amdgcn_sched_barrier(0);
    }
    // The lane's keys: 32 kb + 8 (i / 4) + 4 half + i % 4.
    const float from = m_run == kMinusInf ? 0.f : m_run;
    float top = kMinusInf;
    auto take_z = [&](int kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = fmaf(s[kb][i], ks[kb][i / 4][i & 3], -from);
    };
    read_ks(0);
    if constexpr (D == 64) read_ks(1);             // the larger head has no registers for both
    __builtin_amdgcn_sched_barrier(0);
    // the first half's z stand between the second half's products
#pragma unroll
    for (int j = 0; j < D / 16; ++j) s[1] = mfma32<TYPE>(kf[j], q[j], s[1]);
    take_z(0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (D != 64) read_ks(1);
    __builtin_amdgcn_sched_barrier(0);
    take_z(1);
    uint32_t hidden = 0;
    if (edge) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (meta.pos[32 * kb + 8 * (i / 4) + 4 * half + (i & 3)] >= limit) {
            s[kb][i] = kMinusInf;
            hidden |= 1u << (16 * kb + i);
          }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    const float counted = wide ? 0.f : 1.f;
    if (wide || __ballot(top > kSlack || (m_run == kMinusInf && top > kMinusInf))) {
      top = fmaxf(top, __shfl_xor(top, 32));
      // a row moves if it has to or has no reference yet; its two lanes agree
      const bool move = top > kSlack || (m_run == kMinusInf && top > kMinusInf);
      const float by = move ? top : 0.f;
      const float grow = m_run == kMinusInf ? 0.f : exp2_fast(-by);
      const float moved = m_run == kMinusInf ? __builtin_huge_valf() : by;
      if (move) m_run = from + by;
      l_run *= grow;
      scale_sums(grow);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] -= by;
      if (wide) {                                    // l by itself; z then takes the scale's exponent along, relative to the row's r
        float most = kMinusInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 ex = *reinterpret_cast<const f32x4*>(&meta.ex[32 * kb + 8 * i + 4 * half]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              l_run += exp2_fast(s[kb][4 * i + c]);
              most = fmaxf(most, s[kb][4 * i + c] + ex[c]);
            }
          }
        most = fmaxf(most, __shfl_xor(most, 32));
        const int was = row_r[32 * wave + col], r_now = row_exponent(was, moved, most);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        row_r[32 * wave + col] = r_now;
        shift_sums(was - r_now);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 ex = *reinterpret_cast<const f32x4*>(&meta.ex[32 * kb + 8 * i + 4 * half]);
#pragma unroll
            for (int c = 0; c < 4; ++c) s[kb][4 * i + c] += ex[c] + (float)(kPShift - r_now);
          }
      }
    }
    f32x4 vs[2][4];
    auto read_vs = [&](int kb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) vs[kb][i] = *reinterpret_cast<const f32x4*>(&meta.vs[32 * kb + 8 * i + 4 * half]);
    };
    u32x4 vf[2][D / 32];
    auto read_v = [&](int kb, int s2, int dt) { vf[s2][dt] = at_v(buf, (v_at ^ (32 * (2 * kb + s2))) + 32 * dt * kVRow); };
    read_vs(0);
    read_vs(1);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) read_v(0, s2, dt);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 pf[2][2], pf_low[2][2];
    auto weights = [&](int kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = exp2_fast(s[kb][i]);
        l_run = fmaf(e, counted, l_run);
        s[kb][i] = e * vs[kb][i / 4][i & 3];
      }
    };
    auto blank = [&](int kb) {                     // 0 times a scale that is not finite
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((hidden >> (16 * kb + i)) & 1u) s[kb][i] = 0.f;
    };
    auto pack = [&](int kb) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const uint32_t y = pack_f16(s[kb][i], s[kb][i + 1]);
        pf[kb][i / 8][(i & 7) / 2] = y;
        if constexpr (TYPE == 1) pf_low[kb][i / 8][(i & 7) / 2] = pack_f16(less_half<0>(s[kb][i], y), less_half<1>(s[kb][i + 1], y));
      }
    };
    auto gather = [&](int kb, int s2, int dt) {
      o[dt] = mfma32<1>(vf[s2][dt], pf[kb][s2], o[dt]);
      if constexpr (TYPE == 1) o[dt] = mfma32<1>(vf[s2][dt], pf_low[kb][s2], o[dt]);
    };
    weights(0);
    if (edge) blank(0);
    pack(0);
    __builtin_amdgcn_sched_barrier(0);
    // the second half's exponentials stand between the first half's products
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        gather(0, s2, dt);
        read_v(1, s2, dt);
      }
    weights(1);
    if (edge) blank(1);
    pack(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) gather(1, s2, dt);
    __builtin_amdgcn_sched_barrier(0);
  };

  if (t0 < t1) {
    // Step t's bytes are brought while step t - 1 is computed.
    look_up(t0 + wave, gload<uint64_t>(table_at(t0 + wave)), metas[wave]);
    copy_pages(t0 + 4 + wave);
    for (int d = tid; d < D; d += 256) nan_at[d] = kNoKey;
    if (tid == 0) spoilt = 0;
    lds_barrier();
    bring(metas[0]);
    wait_vmem<0>();
    find_exponents(metas[wave]);
    lds_barrier();
    finish(0, metas[wave]);
    int gone = uni(metas[0].gone);
    put(t0, 0, metas[0], gone);
    lds_barrier();
    for (int t = t0; t < t1; ++t) {
      const int i = t - t0, ahead = (i & 4) ^ 4;   // ahead: where the ring has the next four steps
      if ((i & 3) == 0) {
        wait_vmem<0>();                            // the page ids, asked for four steps ago
        look_up(t + 4 + wave, pid_in[0][lane] | ((uint64_t)pid_in[1][lane] << 32), metas[ahead + wave]);
        copy_pages(t + 8 + wave);
      } else if ((i & 3) == 1) {
        wait_vmem<0>();                            // the scales, asked for a step ago
        find_exponents(metas[ahead + wave]);
      } else if ((i & 3) == 3) {
        finish(ahead, metas[ahead + wave]);
      }
      const int r_read = metas[i & 7].r, gone_read = metas[(i + 1) & 7].gone;      // read here: their wait is the one that bring has anyway
      bring(metas[(i + 1) & 7]);
      const int r = uni(r_read), gone_next = uni(gone_read);
      if (t * kKeys < wave_seen) compute(t, i & 1, metas[i & 7], r, gone);
      if (t + 1 < t1) put(t + 1, (i & 1) ^ 1, metas[(i + 1) & 7], gone_next);
      gone = gone_next;
      lds_barrier();
    }
    wait_vmem<0>();                                // no copy into LDS outlives the workgroup
    if (bad_page) raise_flag(a.status, ST_SLOT_PAGE);
    if (spoilt)
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (nan_at[32 * i + 8 * (e / 4) + 4 * half + (e & 3)] < limit) o[i][e] = __uint_as_float(0x7fc00000u);
  }

  l_run += __shfl_xor(l_run, 32);
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
  const int off = (r_exp == kWide ? row_r[32 * wave + col] : r_exp) - kPShift;       // what comes off the row's sums
  const Row me = my_row((int)opaque((uint32_t)col));
  const uint32_t tok = me.tok;
  const int head = me.head, r = me.r, by_half = (int)opaque((uint32_t)half);
  if (!me.live) return;
  if (a.slots == 1) {
    const uint64_t dst = (uint64_t)a.out + 2 * ((seq.first + tok) * a.o_row + head * a.o_head);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = ldexpf(o[i][4 * j + c] * inv, off);
        gstore<u32x2>(dst + 2 * (32 * i + 8 * j + 4 * by_half), u32x2{narrow<TYPE>(y[0], y[1]), narrow<TYPE>(y[2], y[3])});
      }
    if (a.lse && by_half == 0)
      a.lse[(seq.first + tok) * (int64_t)(H * G) + head] = l_run == 0.f ? kMinusInf : (m_run + __log2f(l_run)) * 0.69314718055994530942f;
  } else {
    const int64_t at = ((slot * H + h) * a.slots + part) * kManyRows + r;
    if (l_run != 0.f) {
      const uint64_t dst = (uint64_t)(a.part_o + at * D);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4 y;
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] = ldexpf(o[i][4 * j + c] * inv, off);
          gstore<f32x4>(dst + 4 * (32 * i + 8 * j + 4 * by_half), y);
        }
    }
    if (by_half == 0) {
      a.part_ml[2 * at] = m_run;
      a.part_ml[2 * at + 1] = l_run;
    }
  }
}

// Joins the parts of a tile's keys: D/4 threads a row, each with a share of the parts' (m, l) and four places over all parts, four
// parts' places under way at a time.
template <int D, int TYPE>
__global__ __launch_bounds__(256) void fp8_join_many_kernel(const AttendArgs a) {
  constexpr int kRows = 256 / (D / 4);            // rows of a workgroup
  const int lane = threadIdx.x & 63;
  const int H = a.layer.heads, G = (int)a.group.d;
  const uint32_t id = blockIdx.x;
  const int r = (int)(id % (kManyRows / kRows)) * kRows + threadIdx.x / (D / 4), d = 4 * (threadIdx.x % (D / 4));
  const uint32_t rest = id / (kManyRows / kRows);
  const int h = (int)(rest % (uint32_t)H);
  const int64_t slot = rest / (uint32_t)H;
  const int64_t b = find_seq(a.seq.n_seqs, slot, lane, [&](int64_t i) { return first_tile<kManyRows>(a, i); });
  const Seq seq = read_seq(a.seq, b);
  const int64_t tile = slot - first_tile<kManyRows>(a, b);
  if (!seq.ok || tile < 0 || tile * kManyRows + r >= (int64_t)seq.n * G) return;
  const uint32_t row = (uint32_t)(tile * kManyRows + r), tok = divide(row, a.group);
  auto at = [&](int i) { return ((slot * H + h) * a.slots + i) * kManyRows + r; };
  constexpr int kLanes = D / 4, kMine = kMostParts / kLanes;
  const int mine = threadIdx.x % kLanes, first_lane = lane - mine;
  float w[kMine], l[kMine], top = kMinusInf;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int i = k * kLanes + mine;
    w[k] = kMinusInf;
    l[k] = 0.f;
    if (i < a.slots) {
      w[k] = a.part_ml[2 * at(i)];
      l[k] = a.part_ml[2 * at(i) + 1];
    }
    top = fmaxf(top, w[k]);
  }
#pragma unroll
  for (int k = 1; k < kLanes; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
  const float from = top == kMinusInf ? 0.f : top;
  f32x4 o = {0, 0, 0, 0};
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    w[k] = l[k] == 0.f ? 0.f : l[k] * exp2_fast(w[k] - from);
    sum += w[k];
  }
#pragma unroll
  for (int k = 1; k < kLanes; k <<= 1) sum += __shfl_xor(sum, k);
#pragma unroll
  for (int k = 0; k < kMine; ++k)
    for (int i0 = k * kLanes; i0 < (k + 1) * kLanes && i0 < a.slots; i0 += 4) {
      f32x4 y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = gload<f32x4>((uint64_t)(a.part_o + at(i0 + u < a.slots ? i0 + u : a.slots - 1) * D + d));
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float wi = __shfl(w[k], first_lane + i0 + u - k * kLanes);
        if (i0 + u < a.slots && wi != 0.f)        // what a part that saw no key holds was never written
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] += wi * y[u][c];
      }
    }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int head = h * G + (int)(row - tok * G);
  gstore<u32x2>((uint64_t)a.out + 2 * ((seq.first + tok) * a.o_row + head * a.o_head + d),
                u32x2{narrow<TYPE>(o[0] * inv, o[1] * inv), narrow<TYPE>(o[2] * inv, o[3] * inv)});
  if (a.lse && d == 0) a.lse[(seq.first + tok) * (int64_t)(H * G) + head] = sum == 0.f ? kMinusInf : (top + __log2f(sum)) * 0.69314718055994530942f;
}

// ---------------------------------------------------------------------------------------------
template <int D, int TYPE, int NT, int NK>
static hipError_t launch_few(const AttendPlan& p, const AttendArgs& a, hipStream_t s) {
  static_assert(Few<D, TYPE, NT, NK>::kWaves == kFewWaves, "the plan's workgroup");
  hipLaunchKernelGGL((fp8_attend_few_kernel<D, TYPE, NT, NK>), dim3((uint32_t)p.groups), dim3(p.threads), 0, s, a);
  if (p.slots > 1) hipLaunchKernelGGL((fp8_join_few_kernel<D, TYPE, 16 * NT>), dim3((uint32_t)(p.slots * a.layer.heads), 4 * NT), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int D, int TYPE>
static hipError_t launch_form(const AttendPlan& p, const AttendArgs& a, hipStream_t s) {
  switch (p.form) {
    case ATTEND_FEW_16: return launch_few<D, TYPE, 1, 4>(p, a, s);
    case ATTEND_FEW_32: return launch_few<D, TYPE, 2, 2>(p, a, s);
    default: break;
  }
  hipLaunchKernelGGL((fp8_attend_many_kernel<D, TYPE>), dim3((uint32_t)p.groups), dim3(p.threads), 0, s, a);
  if (p.slots > 1)
    hipLaunchKernelGGL((fp8_join_many_kernel<D, TYPE>), dim3((uint32_t)(p.tiles * a.layer.heads * (kManyRows * D / 1024))), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_fp8_attend(const AttendPlan& p, int head_dim, int type, const AttendArgs& args, hipStream_t stream) {
  AttendArgs a = args;
  a.slots = p.slots;
  a.min_steps = p.min_steps;
  a.begin_cost = p.begin_cost;
  a.tiles = p.tiles;
  a.heads_per_group = p.heads_per_group;
  if (head_dim == 128) return type == 0 ? launch_form<128, 0>(p, a, stream) : launch_form<128, 1>(p, a, stream);
  return type == 0 ? launch_form<64, 0>(p, a, stream) : launch_form<64, 1>(p, a, stream);
}

}  // namespace bikv
