// How a call of the 8-bit cache's attention is cut into work, from what the host knows of it alone. HIP-free: tests compile
// it with the host compiler.
#pragma once
#include <stdint.h>

namespace bikv {

enum : int { ATTEND_FEW_16 = 0, ATTEND_FEW_32 = 1, ATTEND_MANY = 2 };
constexpr int kFewWaves = 8;             // waves of a few rows' workgroup, of 256 registers: they fill a CU
constexpr int kManyRows = 128;           // rows of a many rows' tile
constexpr int kManyKeys = 64;            // and its keys a step
constexpr int kManyThreads = 256;
constexpr int kMostParts = 64;           // a tile's keys are cut into no more

struct AttendPlan {
  int form;
  int rows;                  // rows of a tile
  int32_t slots;             // few rows: shares the work is cut into, 0 = a workgroup per tile; many rows: parts a tile's keys are cut into
  int32_t min_steps;
  int32_t begin_cost;
  int32_t heads_per_group;
  int64_t tiles;
  int64_t part_rows;         // rows of partial results the call may need (x head_dim floats + 2 floats)
  int64_t groups;            // workgroups of the launch that reads the cache, and their threads
  int threads;
};

// Row tiles of `m` rows: with one token each the sequences have as many tiles each; else every sequence may leave one unfilled.
inline int64_t tiles_in_all(bool one_each, int group, int64_t n_seqs, int64_t n_rows, int m) {
  return one_each ? n_seqs * (((int64_t)group + m - 1) / m) : n_rows * group / m + n_seqs;
}
inline int64_t steps_of_keys(int64_t len, int keys) { return len <= keys ? 1 : (len + keys - 1) / keys; }

// one_each: no row numbers, a sequence has one row.
inline AttendPlan plan_fp8_attend(int heads, int group, bool one_each, int64_t n_seqs, int64_t n_rows, int64_t max_len) {
  AttendPlan p = {};
  const int64_t all = n_rows * group;                      // rows of one KV head
  const int64_t mean = (all + n_seqs - 1) / n_seqs;
  // Up to 16 rows of a sequence on average: few rows (3 sequences of 32k, 8 KV heads, 16 rows: 58 us against 69 as many rows; 64 of
  // 3000: 113 and 137). Up to 32: where the sequences are many enough for the shares (64 of 3000, 21 rows, 4 heads, 63 us against
  // 119; 12 of 4500, 33 and 35; but 6 of 3000, 27 and 23; one of 20000, 43 and 30). More: many rows; a 64-row tile of the first
  // kind took two to three times as long.
  const int m = mean <= 16 ? 16 : 32, keys = m == 16 ? 64 : 32;
  const int64_t tiles = tiles_in_all(one_each, group, n_seqs, n_rows, m);
  const int waves = kFewWaves, side_by_side = heads < waves ? heads : waves;
  // 3 steps of each wave of a head: 64 sequences of 100 to 4000 tokens, 3 new each, 28 and 4 heads, take 51 us, 64 without and 59
  // with one; 64 of 1k to 8k, 64 and 8 heads, 140, 148 and 144.
  const int min_steps = waves / side_by_side, begin_cost = 3 * min_steps;
  if ((mean <= 16 || (mean <= 32 && n_seqs >= 8)) && tiles * (steps_of_keys(max_len, keys) + begin_cost) < (int64_t(1) << 31)) {   // the line's length
    p.form = m == 16 ? ATTEND_FEW_16 : ATTEND_FEW_32;
    p.rows = m;
    p.tiles = tiles;
    p.heads_per_group = side_by_side;
    if (max_len <= 1024) {
      // A workgroup per tile, no second launch: 11.5 us against 16 for a sequence of 500 tokens, 15 against 16 at 1000; at 1500
      // shares are ahead (18.7 against 17.1), and at 4000 by half (35 against 22). Where there are few tiles a head
      // gets more waves, of more workgroups: 8 sequences of up to 1000 tokens, 8 KV heads, take 14 us, 52 without; 42 of them 21 and 53. But
      // no more workgroups than CUs, each of which holds one (42 short sequences 12.6 us, 19.4 in twice as many).
      auto groups = [&](int32_t per) { return tiles * ((heads + per - 1) / per); };
      while (p.heads_per_group > 1 && groups((p.heads_per_group + 1) / 2) <= 256) p.heads_per_group = (p.heads_per_group + 1) / 2;
      p.slots = 0;
    } else {
      // one workgroup for each of the 256 CUs, which is what one holds of this size
      const int64_t slots = 256 / ((heads + p.heads_per_group - 1) / p.heads_per_group);
      p.slots = (int32_t)(slots < 1 ? 1 : slots);
    }
    p.min_steps = waves / p.heads_per_group;
    p.begin_cost = p.slots > 0 ? begin_cost : 0;             // the heads of a workgroup are as they were, then
    p.part_rows = p.slots > 1 ? 2 * (int64_t)p.slots * heads * p.rows : 0;
    p.groups = (p.slots > 0 ? p.slots : p.tiles) * ((heads + p.heads_per_group - 1) / p.heads_per_group);
    p.threads = 64 * kFewWaves;
  } else {
    p.form = ATTEND_MANY;
    p.rows = kManyRows;
    p.tiles = tiles_in_all(one_each, group, n_seqs, n_rows, kManyRows);
    // Parts of a tile's keys. The chip holds 512 of these workgroups, two to a CU, so `n` of them take ceil(n / 512) rounds of their
    // steps, and some two steps more to begin and to end (two again where empty workgroups, of tiles that sequences may have
    // and these do not, take a place first); the parts' sums are written and read again, 115 of them in a step's time. 33 sequences of
    // 40 to 64 rows over 4000 keys, 8 KV heads: 243 us in one part, 184 in three; 300 new tokens of each of 2 sequences of 3500, 4
    // KV heads: 52 us in 6 parts, 119 in one and 66 in 12. From 1024 tiles on the rounds even out by themselves. Parts have
    // four steps at least, and their sums take 140 MB at most.
    const int64_t tiles_likely = one_each ? p.tiles : all / kManyRows + n_seqs / 2, n = heads * (tiles_likely > n_seqs ? tiles_likely : n_seqs);
    const int64_t steps = steps_of_keys(max_len, kManyKeys);
    p.slots = 1;
    if (n < 1024) {
      int64_t least = -1;
      for (int64_t parts = 1; parts <= kMostParts && (parts == 1 || (parts <= steps / 4 && p.tiles * heads * parts <= 2048)); ++parts) {
        const int64_t cost = (n * parts + 511) / 512 * ((steps + parts - 1) / parts + 2) + (parts > 1 ? n * parts / 115 + 2 : 0) + (p.tiles * heads * parts > 512 ? 2 : 0);
        if (least < 0 || cost < least) {
          least = cost;
          p.slots = (int32_t)parts;
        }
      }
    }
    p.part_rows = p.slots > 1 ? p.tiles * heads * p.slots * kManyRows : 0;
    p.groups = p.tiles * heads * p.slots;
    p.threads = kManyThreads;
  }
  return p;
}

}  // namespace bikv
