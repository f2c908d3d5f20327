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
// cost as much as the output's own rounding): p vs 2^(8 - r) with r the largest exponent of vs so far, so that
// neither a page's scale nor a small p leaves fp16's range; the exponent comes off again at the end.
// l sums the unrounded p.
#include "fp8_cache_device.h"

namespace bikv {

constexpr float kMinusInf = -__builtin_huge_valf();
constexpr int kNoKey = 0x7fffffff;      // position of a key that no row sees
constexpr int kPShift = 8;              // p is scaled by 2^8 in fp16: p down to 2^-22 stays normal

template <int TYPE> struct QType;
template <> struct QType<0> { typedef bf16x8 V8; };
template <> struct QType<1> { typedef f16x8 V8; };

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

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
}
template <int TYPE>
__device__ __forceinline__ uint32_t narrow(float a, float b) {
  if constexpr (TYPE == 0)
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
  else
    return pack_f16(a, b);
}

// 0xffff in each half that is a NaN in fp16.
__device__ __forceinline__ uint32_t nan_halves(uint32_t x) {
  const uint32_t t = ((x & 0x7fff7fffu) + 0x03ff03ffu) & 0x80008000u;    // sign bit set where the magnitude is over 0x7c00
  return (t >> 15) * 0xffffu;
}

// Exponent of a page's V scale, -126 where it is zero, subnormal or not finite.
__device__ __forceinline__ int scale_exponent(float s) {
  const int e = (int)((__float_as_uint(s) >> 23) & 0xffu);
  return e == 0 || e == 255 ? -126 : e - 127;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---------------------------------------------------------------------------------------------
// Few rows per sequence: one wave per (tile of up to 64 rows, KV head, run of key steps).
//
// Bound by memory: every byte of K and V is read once per row tile. Waves share nothing and never meet at a
// barrier. A lane reads its operands' bytes straight from the cache: for K 16 bytes of a
// key's row (a matrix product does not mind in which order it sums, so the four lanes of a row take the
// 16-byte pieces as they lie), for V the D/16 bytes at one place of its own eight keys' rows, which the
// lane transposes in registers. The loads of the next step are issued before the present one is computed.
//
// The work is cut evenly: row tiles of all sequences times their key steps form one line, share s of
// it belongs to slot s (every KV head has its own wave per slot). A tile that lies in one share is
// finished there; the others leave (O, m, l) per share and fp8_join_few_kernel joins them.
// ---------------------------------------------------------------------------------------------
template <int D, int TYPE, int NT, int NK>
struct Few {
  static constexpr int kM = 16 * NT;       // rows of a tile
  static constexpr int kKeys = 16 * NK;    // keys of a step
  static constexpr int kDT = D / 16;       // bytes of a V row per lane, and row tiles of O^T
};

__device__ __forceinline__ int64_t tiles_of(const Seq& s, const FastDiv& group, int m) {
  return ((int64_t)s.n * group.d + m - 1) / m;
}
__device__ __forceinline__ int steps_of(const Seq& s, int keys) { return s.len <= keys ? 1 : (s.len + keys - 1) / keys; }

// The line of work, as one wave sees it.
struct Line {
  int64_t total;    // steps
  int64_t begin;    // of this share
  int64_t end;
};
__device__ __forceinline__ Line share_of(int64_t total, int slots, int min_steps, int slot) {
  const int64_t want = (total + min_steps - 1) / min_steps;
  const int64_t n = want < slots ? (want > 0 ? want : 1) : slots;
  const int64_t per = total / n, more = total - per * n;
  Line l;
  l.total = total;
  l.begin = slot < n ? slot * per + (slot < more ? slot : more) : total;
  l.end = slot < n ? l.begin + per + (slot < more ? 1 : 0) : total;
  return l;
}
// The share that step x of the line lies in.
__device__ __forceinline__ int slot_of(int64_t total, int slots, int min_steps, int64_t x) {
  const int64_t want = (total + min_steps - 1) / min_steps;
  const int64_t n = want < slots ? (want > 0 ? want : 1) : slots;
  const int64_t per = total / n, more = total - per * n;
  const int64_t cut = more * (per + 1);
  return (int)(x < cut ? x / (per + 1) : more + (x - cut) / per);
}

template <int M, int KEYS>
__device__ __forceinline__ int64_t line_length(const AttendArgs& a, int lane) {
  int64_t sum = 0;
  for (int64_t b = lane; b < a.seq.n_seqs; b += 64) {
    const Seq s = read_seq(a.seq, b);
    sum += tiles_of(s, a.group, M) * steps_of(s, KEYS);
  }
  return uni64(wave_sum64(sum));
}
// The sequence that step x (below the line's length) belongs to, and where in it.
template <int M, int KEYS>
__device__ __forceinline__ int64_t seq_at(const AttendArgs& a, int64_t x, int lane, int64_t* local) {
  int64_t run = 0;
  for (int64_t base = 0; base < a.seq.n_seqs; base += 64) {
    int64_t w = 0;
    if (base + lane < a.seq.n_seqs) {
      const Seq s = read_seq(a.seq, base + lane);
      w = tiles_of(s, a.group, M) * steps_of(s, KEYS);
    }
    const int64_t upto = run + wave_scan64(w, lane);
    const uint64_t m = __ballot(upto > x);
    if (m) {
      const int src = __builtin_ctzll(m);
      *local = uni64(x - shfl64(upto - w, src));
      return uni64(base + src);
    }
    run = uni64(shfl64(upto, 63));
  }
  *local = 0;
  return a.seq.n_seqs;
}

template <int D, int TYPE, int NT, int NK>
__global__ __launch_bounds__(256, NT == 1 ? 2 : 1) void fp8_attend_few_kernel(const AttendArgs a) {
  using C = Few<D, TYPE, NT, NK>;
  constexpr int kM = C::kM, kKeys = C::kKeys, kDT = C::kDT;
  constexpr int kQK = D / 32;              // matrix steps of q . k
  struct Meta {
    uint64_t off[kKeys];                   // byte offset of the key's row in its plane
    float ks[kKeys], vs[kKeys];
    int pos[kKeys];
  };
  __shared__ Meta metas[4];
  const int wave = uni(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int quad = lane >> 4, col = lane & 15;
  Meta& meta = metas[wave];
  const uint32_t w = blockIdx.x * 4 + wave;
  const uint32_t H = (uint32_t)a.layer.heads;
  const int h = (int)(w % H), slot = (int)(w / H);
  if (slot >= a.slots) return;
  const int G = (int)a.group.d;
  const int P = (int)a.layer.page_tokens.d;

  const int64_t total = line_length<kM, kKeys>(a, lane);
  if (w == 0)
    for (int64_t b = lane; b < a.seq.n_seqs; b += 64)
      if (!read_seq(a.seq, b).ok) raise_flag(a.status, ST_SLOT_SRC);
  const Line line = share_of(total, a.slots, a.min_steps, slot);
  if (line.begin >= line.end) return;
  int64_t local = 0;
  int64_t b = seq_at<kM, kKeys>(a, line.begin, lane, &local);

  const uint64_t kbase = (uint64_t)a.layer.k + h * D, vbase = (uint64_t)a.layer.v + h * D;
  const uint64_t ksbase = (uint64_t)a.layer.ks + 4 * h, vsbase = (uint64_t)a.layer.vs + 4 * h;

  int64_t at = line.begin;
  while (at < line.end && b < a.seq.n_seqs) {
    const Seq seq = read_seq(a.seq, b);
    const int steps = uni(steps_of(seq, kKeys));
    const int64_t weight = uni64(tiles_of(seq, a.group, kM) * steps);
    if (local >= weight) {
      ++b;
      local = 0;
      continue;
    }
    const int tile = (int)(local / steps);
    const int step0 = (int)(local - (int64_t)tile * steps);
    int count = steps - step0;
    if (count > line.end - at) count = (int)(line.end - at);
    const bool first_of_share = at == line.begin;
    const bool whole = count == steps;
    const int rows = uni((int)((int64_t)seq.n * G - (int64_t)tile * kM < kM ? (int64_t)seq.n * G - (int64_t)tile * kM : kM));
    const int len = uni(seq.len);
    const int before = a.causal ? uni(seq.len - seq.n) : 0;     // keys older than the call's own (negative: some rows see none)

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
    const int last_tok = uni((int)divide((uint32_t)(tile * kM + rows - 1), a.group));
    const int first_tok = uni((int)divide((uint32_t)(tile * kM), a.group));
    int seen = a.causal ? before + last_tok + 1 : len;           // keys that the tile's last row sees
    seen = seen < 0 ? 0 : seen;
    int all = a.causal ? before + first_tok + 1 : len;           // keys that every row sees
    all = all < 0 ? 0 : all;
    int end = step0 + count;
    if (end > (seen + kKeys - 1) / kKeys) end = (seen + kKeys - 1) / kKeys;

    f32x4 o[NT][kDT];
    float m[NT], l[NT];
    int r_exp = -126;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kMinusInf;
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < kDT; ++i) o[t][i] = f32x4{0, 0, 0, 0};
    }

    const uint64_t trow = (uint64_t)(a.seq.table + b * a.seq.table_stride);
    auto page_of = [&](int step) -> int64_t {                   // the page id of the lane's key
      const int key = step * kKeys + lane;
      if (lane >= kKeys || key >= seen) return -1;
      return gload<int64_t>(trow + 8 * (uint64_t)divide((uint32_t)key, a.layer.page_tokens));
    };
    struct Data {
      u32x4 k[NK][D / 64];
      uint32_t v[NK][4][kDT / 4];
      float ks, vs;
      int pos;
    };
    // Issues a step's loads: the page ids are there. Keys that are not there (behind the sequence, or
    // on a page the pool does not have) read the plane's first row instead, and are masked by position.
    auto fetch = [&](int step, int64_t pid, Data& x) {
      const int key = step * kKeys + lane;
      bool ok = lane < kKeys && key < seen;
      if (ok && (uint64_t)pid >= (uint64_t)a.layer.n_pages) {
        raise_flag(a.status, ST_SLOT_PAGE);
        ok = false;
      }
      x.pos = ok ? key : kNoKey;
      x.ks = 0.f;
      x.vs = 0.f;
      uint64_t off = 0;
      if (ok) {
        const uint32_t in_page = (uint32_t)key - divide((uint32_t)key, a.layer.page_tokens) * (uint32_t)P;
        off = (uint64_t)(pid * a.layer.page_stride) + (uint64_t)in_page * (uint64_t)a.layer.token_stride;
        x.ks = gload<float>(ksbase + (uint64_t)(pid * a.layer.scale_stride));
        x.vs = gload<float>(vsbase + (uint64_t)(pid * a.layer.scale_stride));
      }
      if (lane < kKeys) meta.off[lane] = off;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const uint64_t p = kbase + meta.off[16 * i + col] + 16 * quad;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) x.k[i][j] = gload<u32x4>(p + 64 * j);
      }
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t p = vbase + meta.off[16 * i + 4 * quad + e] + kDT * col;
          if constexpr (kDT == 8) {
            const u32x2 c = gload<u32x2>(p);
            x.v[i][e][0] = c[0];
            x.v[i][e][1] = c[1];
          } else {
            x.v[i][e][0] = gload<uint32_t>(p);
          }
        }
    };
    auto compute = [&](int step, Data& x) {
      // a larger V scale than any before: what is summed moves to its exponent
      const int e = scale_exponent(x.vs);
      if (__ballot(x.pos != kNoKey && e > r_exp)) {
        int top = x.pos != kNoKey ? e : -126;
        for (int k = 32; k > 0; k >>= 1) {
          const int y = __shfl_xor(top, k);
          top = y > top ? y : top;
        }
        top = uni(top);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < kDT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[t][i][c] = ldexpf(o[t][i][c], r_exp - top);
        r_exp = top;
      }
      if (lane < kKeys) {
        meta.ks[lane] = x.ks * a.scale_log2;
        meta.vs[lane] = ldexpf(x.vs, kPShift - r_exp);
        meta.pos[lane] = x.pos;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const bool edge = (step + 1) * kKeys > all || __ballot(lane < kKeys && x.pos == kNoKey) != 0;

      // S^T = K Q^T
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
            const u32x2 lo = widen4<TYPE>(x.k[i][j][2 * half]), hi = widen4<TYPE>(x.k[i][j][2 * half + 1]);
            f[half] = u32x4{lo[0], lo[1], hi[0], hi[1]};
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            s[t][i] = mfma16<TYPE>(f[0], q[t][2 * j], s[t][i]);
            s[t][i] = mfma16<TYPE>(f[1], q[t][2 * j + 1], s[t][i]);
          }
        }
      }
      // softmax: the lane's keys are 16 i + 4 quad + c
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float top = kMinusInf;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const f32x4 ks = *reinterpret_cast<const f32x4*>(&meta.ks[16 * i + 4 * quad]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[t][i][c] *= ks[c];
            if (edge && meta.pos[16 * i + 4 * quad + c] >= limit[t]) s[t][i][c] = kMinusInf;
            top = fmaxf(top, s[t][i][c]);
          }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = fmaxf(m[t], top);
        const float from = now == kMinusInf ? 0.f : now;
        const float grow = exp2_fast(m[t] - from);              // 0 at the first key
        m[t] = now;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[t][i][c] = exp2_fast(s[t][i][c] - from);
            sum += s[t][i][c];
          }
        l[t] = l[t] * grow + sum;
#pragma unroll
        for (int i = 0; i < kDT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[t][i][c] *= grow;
      }
      // O^T += V^T P^T, 32 keys at a time
#pragma unroll
      for (int i = 0; i < NK; i += 2) {
        u32x4 p[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const f32x4 vs = *reinterpret_cast<const f32x4*>(&meta.vs[16 * (i + half) + 4 * quad]);
            float f[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              f[c] = s[t][i + half][c] * vs[c];
              if (edge && meta.pos[16 * (i + half) + 4 * quad + c] >= limit[t]) f[c] = 0.f;   // whatever the scale is
            }
            p[t][2 * half] = pack_f16(f[0], f[1]);
            p[t][2 * half + 1] = pack_f16(f[2], f[3]);
          }
        uint32_t gone = 0;                                       // eight keys' bits: nobody sees them
        if (edge)
#pragma unroll
          for (int c = 0; c < 8; ++c) gone |= (meta.pos[16 * (i + c / 4) + 4 * quad + (c & 3)] == kNoKey ? 1u : 0u) << c;
#pragma unroll
        for (int dw = 0; dw < kDT / 4; ++dw) {
          u32x2 x8[8];                                           // [key] -> places (0, 1) and (2, 3) of the dword
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t bytes = x.v[i + c / 4][c & 3][dw];
            if (edge) bytes = (gone >> c) & 1u ? 0u : bytes;
            x8[c] = widen4<1>(bytes);
          }
#pragma unroll
          for (int pl = 0; pl < 4; ++pl) {
            u32x4 f;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              f[c] = __builtin_amdgcn_perm(x8[2 * c + 1][pl / 2], x8[2 * c][pl / 2], pl & 1 ? 0x07060302u : 0x05040100u);
            const int dt = 4 * dw + pl;
            if (edge) {
              // A NaN in V reaches the rows that see its key and no others: it is taken out of the
              // product, and a second product counts, per output, the visible keys that hold one.
              u32x4 bad;
#pragma unroll
              for (int c = 0; c < 4; ++c) bad[c] = nan_halves(f[c]);
              if (__ballot((bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  u32x4 vis, one;
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    const int k0 = 16 * (i + c / 2) + 4 * quad + 2 * (c & 1);
                    vis[c] = (meta.pos[k0] < limit[t] ? 0x3c00u : 0u) | (meta.pos[k0 + 1] < limit[t] ? 0x3c000000u : 0u);
                    one[c] = bad[c] & 0x3c003c00u;
                  }
                  const f32x4 n = mfma16<1>(one, vis, f32x4{0, 0, 0, 0});
#pragma unroll
                  for (int c = 0; c < 4; ++c)
                    if (n[c] > 0.f) o[t][dt][c] = __uint_as_float(0x7fc00000u);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) f[c] &= ~bad[c];
              }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t][dt] = mfma16<1>(f, p[t], o[t][dt]);
          }
        }
      }
    };

    if (step0 < end) {
      Data x0, x1;
      int64_t pid = page_of(step0);
      fetch(step0, pid, x0);
      pid = step0 + 1 < end ? page_of(step0 + 1) : -1;
      for (int step = step0; step < end; step += 2) {
        if (step + 1 < end) {
          fetch(step + 1, pid, x1);
          pid = step + 2 < end ? page_of(step + 2) : -1;
        }
        compute(step, x0);
        if (step + 1 >= end) break;
        if (step + 2 < end) {
          fetch(step + 2, pid, x0);
          pid = step + 3 < end ? page_of(step + 3) : -1;
        }
        compute(step + 1, x1);
      }
    }

    // The lane holds, of row 16 t + col, places kDT * (4 quad + c) + dt.
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] += __shfl_xor(l[t], 16);
      l[t] += __shfl_xor(l[t], 32);
      const float inv = l[t] > 0.f ? 1.f / l[t] : (l[t] == 0.f ? 0.f : l[t]);     // a NaN sum stays one
      if (!live[t]) continue;
      if (whole) {
        const uint64_t dst = (uint64_t)a.out + 2 * ((seq.first + tok[t]) * a.o_row + head[t] * a.o_head);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t y[kDT / 2];
#pragma unroll
          for (int dt = 0; dt < kDT; dt += 2)
            y[dt / 2] = narrow<TYPE>(ldexpf(o[t][dt][c] * inv, r_exp - kPShift), ldexpf(o[t][dt + 1][c] * inv, r_exp - kPShift));
          if constexpr (kDT == 8) gstore<u32x4>(dst + 2 * kDT * (4 * quad + c), u32x4{y[0], y[1], y[2], y[3]});
          else gstore<u32x2>(dst + 2 * kDT * (4 * quad + c), u32x2{y[0], y[1]});
        }
        if (a.lse && quad == 0)
          a.lse[(seq.first + tok[t]) * (int64_t)(H * G) + head[t]] = l[t] == 0.f ? kMinusInf : (m[t] + __log2f(l[t])) * 0.69314718055994530942f;
      } else {
        const int64_t part = ((int64_t)(2 * slot + (first_of_share ? 0 : 1)) * H + h) * kM + 16 * t + col;
        const uint64_t dst = (uint64_t)(a.part_o + part * D);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int dt = 0; dt < kDT; dt += 4) {
            f32x4 y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = ldexpf(o[t][dt + k][c] * inv, r_exp - kPShift);
            gstore<f32x4>(dst + 4 * (kDT * (4 * quad + c) + dt), y);
          }
        if (quad == 0) {
          a.part_ml[2 * part] = m[t];
          a.part_ml[2 * part + 1] = l[t];
        }
      }
    }
    at += count;
    local += count;
  }
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
#pragma unroll 4
    for (int i = 0; i < here; i += kParts) {
      const float wi = __shfl(w, i + sub);
      if (i + sub < here && wi != 0.f) {
        const f32x4 y = gload<f32x4>((uint64_t)(a.part_o + at(base + i + sub) * D + d));
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += wi * y[c];
      }
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

// One workgroup per (slot, KV head): joins the tile that begins in the slot's share and ends behind it, if
// there is one. The parts are summed in the order of the shares, so the result does not depend on timing.
template <int D, int TYPE, int NT, int NK>
__global__ __launch_bounds__(256) void fp8_join_few_kernel(const AttendArgs a) {
  using C = Few<D, TYPE, NT, NK>;
  constexpr int kM = C::kM, kKeys = C::kKeys;
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int H = a.layer.heads, G = (int)a.group.d;
  const int h = blockIdx.x % H, slot = blockIdx.x / H;
  const int64_t total = line_length<kM, kKeys>(a, lane);
  const Line line = share_of(total, a.slots, a.min_steps, slot);
  if (line.begin >= line.end || line.end >= total) return;
  int64_t local = 0;
  const int64_t b = seq_at<kM, kKeys>(a, line.end - 1, lane, &local);
  if (b >= a.seq.n_seqs) return;
  const Seq seq = read_seq(a.seq, b);
  const int steps = steps_of(seq, kKeys);
  const int tile = (int)(local / steps);
  const int64_t tile_begin = line.end - 1 - (local - (int64_t)tile * steps), tile_end = tile_begin + steps;
  if (tile_end <= line.end || tile_begin < line.begin) return;
  const int last = slot_of(total, a.slots, a.min_steps, tile_end - 1);
  const int first_index = 2 * slot + (tile_begin == line.begin ? 0 : 1);
  const int64_t left = (int64_t)seq.n * G - (int64_t)tile * kM;
  const int rows = (int)(left < kM ? left : kM);
  for (int r = wave; r < rows; r += 4) {
    const uint32_t row = (uint32_t)(tile * kM + r), tok = divide(row, a.group);
    auto at = [&](int i) { return ((int64_t)(i == 0 ? first_index : 2 * (slot + i)) * H + h) * kM + r; };
    join_row<D, TYPE>(a, lane, last - slot + 1, at, seq.first + tok, h * G + (int)(row - tok * G), H * G);
  }
}

// ---------------------------------------------------------------------------------------------
// Many rows per sequence: a workgroup of four waves does 128 rows of one KV head, 32 a wave, over the
// keys 64 at a time.
//
// Bound by the matrix cores (4 D flops per visible row and key) and by what stands beside them: one exp2 per row
// and key, and the widening of K and V, which is done once per workgroup: two waves bring K, two V, as
// bytes into registers while the step before is computed, then widened into LDS: K as [key][D] in
// q's type, V transposed as [D][key] in fp16 with the keys in the order in which P lies in the lanes. 16-byte
// pieces of a row are XOR-ed with the row number, so that neither the writes nor the reads of a column meet in
// a bank. Two LDS buffers, one barrier a step.
//
// A tile's keys are cut into `slots` parts where the tiles alone would not fill the chip; the parts' results are
// joined by fp8_join_many_kernel.
// ---------------------------------------------------------------------------------------------
constexpr int kManyRows = 128;
constexpr int kManyKeys = 64;

template <int TYPE>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (TYPE == 0)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ int64_t first_tile(const AttendArgs& a, int64_t b) {
  int64_t q = b;
  if (a.seq.q_starts) {
    q = a.seq.q_starts[b];
    q = q < 0 ? 0 : q > a.seq.n_rows ? a.seq.n_rows : q;
  }
  return q * a.group.d / kManyRows + b;
}

template <int D, int TYPE>
__global__ __launch_bounds__(256, 2) void fp8_attend_many_kernel(const AttendArgs a) {
  constexpr int kKeys = kManyKeys;
  constexpr int kChunks = D / 8;                  // 16-byte pieces of a K row in LDS
  constexpr int kVB = D / 16;                     // bytes of a V row per thread
  constexpr int kLoads = D / 32;                  // 16-byte registers a thread brings per step
  struct Meta {
    uint64_t off[kKeys];
    float ks[kKeys], vs[kKeys];
    int pos[kKeys];
    int gone;
  };
  __shared__ u32x4 k_lds[2][kKeys * kChunks];
  __shared__ u32x4 v_lds[2][D * 8];
  __shared__ Meta metas[3];
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

  const int64_t b = find_seq(a.seq.n_seqs, slot, lane, [&](int64_t i) { return first_tile(a, i); });
  if (h == 0 && part == 0 && slot < a.seq.n_seqs && tid == 0 && !read_seq(a.seq, slot).ok) raise_flag(a.status, ST_SLOT_SRC);
  const Seq seq = read_seq(a.seq, b);
  const int64_t tile64 = slot - first_tile(a, b);
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

  // the wave's rows: row0 + 32 wave + col
  const int r = 32 * wave + col;
  const bool live = r < rows;
  const uint32_t row = (uint32_t)(row0 + (live ? r : 0));
  const uint32_t tok = divide(row, a.group);
  const int head = h * G + (int)(row - tok * G);
  const int limit = sees((int)row);
  const int wave_last = 32 * wave + 31 < rows ? 32 * wave + 31 : rows - 1;
  const int wave_seen = uni(32 * wave < rows ? sees(row0 + wave_last) : 0);
  const int wave_all = uni(32 * wave < rows ? sees(row0 + 32 * wave) : 0);
  u32x4 q[D / 16];
  {
    const uint64_t src = (uint64_t)a.q + 2 * ((seq.first + tok) * a.q_row + head * a.q_head);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) q[j] = gload<u32x4>(src + 2 * (16 * j + 8 * half));
  }

  const uint64_t kbase = (uint64_t)a.layer.k + h * D, vbase = (uint64_t)a.layer.v + h * D;
  const uint64_t trow = (uint64_t)(a.seq.table + b * a.seq.table_stride);
  auto page_of = [&](int t) -> int64_t {
    const int key = t * kKeys + lane;
    if (key >= seen) return -1;
    return gload<int64_t>(trow + 8 * (uint64_t)divide((uint32_t)key, a.layer.page_tokens));
  };
  struct Key { uint64_t off; float ks, vs; int pos; };
  auto look_up = [&](int t, int64_t pid) {
    Key k = {0, 0.f, 0.f, kNoKey};
    const int key = t * kKeys + lane;
    if (key < seen) {
      if ((uint64_t)pid >= (uint64_t)a.layer.n_pages) {
        raise_flag(a.status, ST_SLOT_PAGE);
      } else {
        const uint32_t in_page = (uint32_t)key - divide((uint32_t)key, a.layer.page_tokens) * (uint32_t)P;
        k.off = (uint64_t)(pid * a.layer.page_stride) + (uint64_t)in_page * (uint64_t)a.layer.token_stride;
        k.ks = gload<float>((uint64_t)a.layer.ks + 4 * h + (uint64_t)(pid * a.layer.scale_stride));
        k.vs = gload<float>((uint64_t)a.layer.vs + 4 * h + (uint64_t)(pid * a.layer.scale_stride));
        k.pos = key;
      }
    }
    return k;
  };
  auto put_meta = [&](Meta& m, const Key& k) {
    m.off[lane] = k.off;
    m.ks[lane] = k.ks * a.scale_log2;
    m.vs[lane] = k.vs;
    m.pos[lane] = k.pos;
    const bool gone = __ballot(k.pos == kNoKey) != 0;
    if (lane == 0) m.gone = gone;
  };

  // Bringing a step's bytes: waves 0 and 1 K, waves 2 and 3 V.
  const int p = tid & 127;
  const bool brings_v = wave >= 2;
  u32x4 raw[kLoads];
  auto bring = [&](const Meta& m) {
    if (!brings_v) {
      constexpr int kRowLanes = D / 16;             // threads that read one row
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int key = i * (128 / kRowLanes) + p / kRowLanes;
        raw[i] = gload<u32x4>(kbase + m.off[key] + 16 * (p % kRowLanes));
      }
    } else {
      const int g = p >> 4, at = (p & 15) * kVB;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int key = 16 * (g >> 1) + 8 * (c >> 2) + 4 * (g & 1) + (c & 3);
        const uint64_t src = vbase + m.off[key] + at;
        if constexpr (kVB == 8) {
          const u32x2 y = gload<u32x2>(src);
          raw[c / 2][2 * (c & 1)] = y[0];
          raw[c / 2][2 * (c & 1) + 1] = y[1];
        } else {
          raw[c / 4][c & 3] = gload<uint32_t>(src);
        }
      }
    }
  };
  auto put = [&](int buf, const Meta& m) {
    if (!brings_v) {
      constexpr int kRowLanes = D / 16;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int key = i * (128 / kRowLanes) + p / kRowLanes, c = 2 * (p % kRowLanes);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x2 lo = widen4<TYPE>(raw[i][2 * e]), hi = widen4<TYPE>(raw[i][2 * e + 1]);
          k_lds[buf][key * kChunks + ((c + e) ^ (key & (kChunks - 1)))] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      }
    } else {
      const int g = p >> 4, c16 = p & 15;
      uint32_t gone = 0;
      if (m.gone)
#pragma unroll
        for (int c = 0; c < 8; ++c) gone |= (m.pos[16 * (g >> 1) + 8 * (c >> 2) + 4 * (g & 1) + (c & 3)] == kNoKey ? 1u : 0u) << c;
#pragma unroll
      for (int dw = 0; dw < kVB / 4; ++dw) {
        u32x2 x8[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t bytes;
          if constexpr (kVB == 8) bytes = raw[c / 2][2 * (c & 1) + dw];
          else bytes = raw[c / 4][c & 3];
          x8[c] = widen4<1>((gone >> c) & 1u ? 0u : bytes);
        }
#pragma unroll
        for (int pl = 0; pl < 4; ++pl) {
          u32x4 f;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            f[c] = __builtin_amdgcn_perm(x8[2 * c + 1][pl / 2], x8[2 * c][pl / 2], pl & 1 ? 0x07060302u : 0x05040100u);
          const int d = c16 * kVB + 4 * dw + pl;
          v_lds[buf][d * 8 + (g ^ ((d >> 1) & 7))] = f;
        }
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

  auto compute = [&](int t, int buf, const Meta& meta) {
    {
      const float vs = meta.vs[lane];
      const int e = meta.pos[lane] == kNoKey ? -126 : scale_exponent(vs);
      if (__ballot(e > r_exp)) {
        int top = e;
        for (int k = 32; k > 0; k >>= 1) {
          const int y = __shfl_xor(top, k);
          top = y > top ? y : top;
        }
        top = uni(top);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int c = 0; c < 16; ++c) o[i][c] = ldexpf(o[i][c], r_exp - top);
        r_exp = top;
      }
    }
    const bool edge = (t + 1) * kKeys > wave_all || meta.gone;
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
      const int key = 32 * kb + col;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
        s[kb] = mfma32<TYPE>(k_lds[buf][key * kChunks + ((2 * j + half) ^ (key & (kChunks - 1)))], q[j], s[kb]);
    }
    // the lane's keys: 32 kb + 8 (i / 4) + 4 half + i % 4
    float top = kMinusInf;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 ks = *reinterpret_cast<const f32x4*>(&meta.ks[32 * kb + 8 * j + 4 * half]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float z = s[kb][4 * j + c] * ks[c];
          if (edge && meta.pos[32 * kb + 8 * j + 4 * half + c] >= limit) z = kMinusInf;
          s[kb][4 * j + c] = z;
          top = fmaxf(top, z);
        }
      }
    top = fmaxf(top, __shfl_xor(top, 32));
    if (__ballot(top > m_run)) {
      const float now = fmaxf(m_run, top);
      const float grow = now == kMinusInf ? 1.f : exp2_fast(m_run - now);
      m_run = now;
      l_run *= grow;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int c = 0; c < 16; ++c) o[i][c] *= grow;
    }
    const float from = m_run == kMinusInf ? 0.f : m_run;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        u32x4 pf;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key0 = 32 * kb + 16 * s2 + 8 * j + 4 * half;
          const f32x4 vs = *reinterpret_cast<const f32x4*>(&meta.vs[key0]);
          float f[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float e = exp2_fast(s[kb][8 * s2 + 4 * j + c] - from);
            l_run += e;
            f[c] = e * ldexpf(vs[c], kPShift - r_exp);
            if (edge && meta.pos[key0 + c] >= limit) f[c] = 0.f;
          }
          pf[2 * j] = pack_f16(f[0], f[1]);
          pf[2 * j + 1] = pack_f16(f[2], f[3]);
        }
        const int g = 2 * (2 * kb + s2) + half;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const int d = 32 * dt + col;
          u32x4 f = v_lds[buf][d * 8 + (g ^ ((d >> 1) & 7))];
          if (edge) {
            u32x4 bad;
#pragma unroll
            for (int c = 0; c < 4; ++c) bad[c] = nan_halves(f[c]);
            if (__ballot((bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
              u32x4 vis, one;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int k0 = 32 * kb + 16 * s2 + 8 * (c >> 1) + 4 * half + 2 * (c & 1);
                vis[c] = (meta.pos[k0] < limit ? 0x3c00u : 0u) | (meta.pos[k0 + 1] < limit ? 0x3c000000u : 0u);
                one[c] = bad[c] & 0x3c003c00u;
                f[c] &= ~bad[c];
              }
              f32x16 n;
#pragma unroll
              for (int c = 0; c < 16; ++c) n[c] = 0.f;
              n = mfma32<1>(one, vis, n);
#pragma unroll
              for (int c = 0; c < 16; ++c)
                if (n[c] > 0.f) o[dt][c] = __uint_as_float(0x7fc00000u);
            }
          }
          o[dt] = mfma32<1>(f, pf, o[dt]);
        }
      }
  };

  if (t0 < t1) {
    // Step t's bytes are brought while step t - 1 is computed, its keys' places one step earlier.
    Key next = {0, 0.f, 0.f, kNoKey};
    int64_t pid = -1;
    if (wave == 0) {
      put_meta(metas[0], look_up(t0, page_of(t0)));
      if (t0 + 1 < t1) put_meta(metas[1], look_up(t0 + 1, page_of(t0 + 1)));
      if (t0 + 2 < t1) pid = page_of(t0 + 2);
    }
    __syncthreads();
    bring(metas[0]);
    put(0, metas[0]);
    __syncthreads();
    int mi = 0;
    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
      const int m1 = mi == 2 ? 0 : mi + 1, m2 = m1 == 2 ? 0 : m1 + 1;
      if (t + 1 < t1) bring(metas[m1]);
      if (wave == 0 && t + 2 < t1) {
        next = look_up(t + 2, pid);
        if (t + 3 < t1) pid = page_of(t + 3);
      }
      if (t * kKeys < wave_seen) compute(t, buf, metas[mi]);
      if (t + 1 < t1) put(buf ^ 1, metas[m1]);
      if (wave == 0 && t + 2 < t1) put_meta(metas[m2], next);
      __syncthreads();
      mi = m1;
    }
  }

  l_run += __shfl_xor(l_run, 32);
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
  if (!live) return;
  if (a.slots == 1) {
    const uint64_t dst = (uint64_t)a.out + 2 * ((seq.first + tok) * a.o_row + head * a.o_head);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = ldexpf(o[i][4 * j + c] * inv, r_exp - kPShift);
        gstore<u32x2>(dst + 2 * (32 * i + 8 * j + 4 * half), u32x2{narrow<TYPE>(y[0], y[1]), narrow<TYPE>(y[2], y[3])});
      }
    if (a.lse && half == 0)
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
          for (int c = 0; c < 4; ++c) y[c] = ldexpf(o[i][4 * j + c] * inv, r_exp - kPShift);
          gstore<f32x4>(dst + 4 * (32 * i + 8 * j + 4 * half), y);
        }
    }
    if (half == 0) {
      a.part_ml[2 * at] = m_run;
      a.part_ml[2 * at + 1] = l_run;
    }
  }
}

// A wave per row: joins the parts of a tile's keys.
template <int D, int TYPE>
__global__ __launch_bounds__(256) void fp8_join_many_kernel(const AttendArgs a) {
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int H = a.layer.heads, G = (int)a.group.d;
  const uint32_t id = blockIdx.x;
  const int r = (int)(id % (kManyRows / 4)) * 4 + wave;
  const uint32_t rest = id / (kManyRows / 4);
  const int h = (int)(rest % (uint32_t)H);
  const int64_t slot = rest / (uint32_t)H;
  const int64_t b = find_seq(a.seq.n_seqs, slot, lane, [&](int64_t i) { return first_tile(a, i); });
  const Seq seq = read_seq(a.seq, b);
  const int64_t tile = slot - first_tile(a, b);
  if (!seq.ok || tile < 0 || tile * kManyRows + r >= (int64_t)seq.n * G) return;
  const uint32_t row = (uint32_t)(tile * kManyRows + r), tok = divide(row, a.group);
  auto at = [&](int i) { return ((slot * H + h) * a.slots + i) * kManyRows + r; };
  join_row<D, TYPE>(a, lane, a.slots, at, seq.first + tok, h * G + (int)(row - tok * G), H * G);
}

// ---------------------------------------------------------------------------------------------
AttendPlan plan_fp8_attend(int head_dim, int heads, int group, int64_t n_seqs, int64_t n_rows, int64_t max_len) {
  AttendPlan p = {};
  const int64_t all = n_rows * group;                      // rows of one KV head
  const int64_t mean = (all + n_seqs - 1) / n_seqs;
  if (mean <= 64) {
    p.form = mean <= 16 ? ATTEND_FEW_16 : mean <= 32 ? ATTEND_FEW_32 : ATTEND_FEW_64;
    p.rows = mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
    // as many waves as the chip holds at once: 256 CUs x 4 SIMDs x 2 (one where a wave has all registers)
    const int64_t waves = p.form == ATTEND_FEW_16 ? 2048 : 1024;
    int64_t slots = waves / heads;
    p.slots = (int32_t)(slots < 1 ? 1 : slots);
    p.min_steps = 1;
    p.part_rows = 2 * (int64_t)p.slots * heads * p.rows;
  } else {
    p.form = ATTEND_MANY;
    p.rows = kManyRows;
    p.tiles = all / kManyRows + n_seqs;
    int64_t parts = 512 / (p.tiles * heads);
    const int64_t steps = (max_len + kManyKeys - 1) / kManyKeys;
    if (parts > steps / 4) parts = steps / 4;
    p.slots = (int32_t)(parts < 1 ? 1 : parts);
    p.part_rows = p.slots > 1 ? p.tiles * heads * p.slots * kManyRows : 0;
  }
  return p;
}

template <int D, int TYPE, int NT, int NK>
static hipError_t launch_few(const AttendPlan& p, const AttendArgs& a, hipStream_t s) {
  const int64_t waves = (int64_t)p.slots * a.layer.heads;
  hipLaunchKernelGGL((fp8_attend_few_kernel<D, TYPE, NT, NK>), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, s, a);
  if (p.slots > 1) hipLaunchKernelGGL((fp8_join_few_kernel<D, TYPE, NT, NK>), dim3((uint32_t)waves), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int D, int TYPE>
static hipError_t launch_form(const AttendPlan& p, const AttendArgs& a, hipStream_t s) {
  switch (p.form) {
    case ATTEND_FEW_16: return launch_few<D, TYPE, 1, 4>(p, a, s);
    case ATTEND_FEW_32: return launch_few<D, TYPE, 2, 2>(p, a, s);
    case ATTEND_FEW_64: return launch_few<D, TYPE, 4, 2>(p, a, s);
    default: break;
  }
  hipLaunchKernelGGL((fp8_attend_many_kernel<D, TYPE>), dim3((uint32_t)(p.tiles * a.layer.heads * p.slots)), dim3(256), 0, s, a);
  if (p.slots > 1)
    hipLaunchKernelGGL((fp8_join_many_kernel<D, TYPE>), dim3((uint32_t)(p.tiles * a.layer.heads * (kManyRows / 4))), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_fp8_attend(const AttendPlan& p, int head_dim, int type, const AttendArgs& args, hipStream_t stream) {
  AttendArgs a = args;
  a.slots = p.slots;
  a.min_steps = p.min_steps;
  a.tiles = p.tiles;
  if (head_dim == 128) return type == 0 ? launch_form<128, 0>(p, a, stream) : launch_form<128, 1>(p, a, stream);
  return type == 0 ? launch_form<64, 0>(p, a, stream) : launch_form<64, 1>(p, a, stream);
}

}  // namespace bikv
