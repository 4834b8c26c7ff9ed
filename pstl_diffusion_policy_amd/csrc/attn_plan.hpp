// attn_plan.hpp -- the choice of a forward attention kernel and of its grid: integer arithmetic on sizes, no device code, so that
// the CPU tests compile it by itself.
#pragma once
#include <stdint.h>

namespace pstl {
namespace attn {

// ---- forward ---------------------------------------------------------------------------------------------------------
constexpr int kMaxSplits = 1024;
enum Kind { kManyRows, kShort, kShortPairs, kFewRows };
struct FwdPlan {
  Kind kind;
  int n_tiles, splits, tiles_per_split, cus_per_xcd;
};
inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// B sequences, Hk key heads, R packed rows (queries x heads that share a key head) and Lk keys each
inline bool plan_in_pairs(int B, int Hk, int R, int Lk) {
  return Lk <= 16 && R <= 16 && (int64_t)B * Hk * Hk < (1ll << 31);
}
inline FwdPlan plan_forward(int B, int Hk, int R, int Lk, bool f32, int cus) {
  const int64_t units = (int64_t)B * Hk;
  FwdPlan p = {kManyRows, ceil_div(R, 128), 1, 0, cus >= 8 ? cus / 8 : 1};
  if (units == 0 || R == 0) return p;      // nothing to launch, nothing to divide
  // (up to 32 keys one tile holds them; 4096 x 12 tokens, 8 heads of 32, bf16: 22 us, one unit to a wavefront 29, many-rows 130)
  if (Lk <= 32) {
    p.kind = plan_in_pairs(B, Hk, R, Lk) ? kShortPairs : kShort;
    p.n_tiles = ceil_div(R, 32);
    return p;
  }
  // the few-rows kernel spreads 32-row tiles, and the keys of each, over the chip, and reads the keys again for every tile.  It is
  // taken while the 128-row workgroups would fill no more than a quarter of the compute units (float32, whose products take
  // sixteen times as long: half of them).  Time of it and of the many-rows kernel, 8 heads of 64, bf16: 256 queries on 4096 keys
  // 22 and 63 us, 1024 causal 16 and 19, 256 on 512 10 and 12, 512 on 64 6.5 and 5.1, and at 114 workgroups (777 x 1301, heads of
  // 80) 58 and 31; float32: 1024 causal 36 and 87, 128 on 128 9 and 16, 4 x 256 on 64 18 and 11, 114 workgroups 150 and 167, 200 (4 x
  // 777) 119 and 71.
  // Up to 32 rows a 128-row workgroup would leave three wavefronts idle: 4 x 32 queries on 4096 keys 15 and 68 us; 64 sequences of
  // 128 keys, 8.8 and 7.3, are what that costs.
  const int64_t wgs = units * p.n_tiles;
  const bool few = R <= 32 || (f32 ? wgs * 2 <= cus && Lk >= 128 : wgs * 4 <= cus && Lk >= 256);
  if (!few) return p;
  p.kind = kFewRows;
  p.n_tiles = ceil_div(R, 32);
  const int64_t jobs = units * p.n_tiles;
  // a part has at least 8 tiles (two per wavefront), and up to 16 tiles are not divided at all: joining costs a launch of 4 us
  const int key_tiles = ceil_div(Lk, 32), most = key_tiles <= 16 ? 1 : ceil_div(key_tiles, 8);
  // one workgroup per compute unit: its four wavefronts keep 64 KB of keys and values in flight; more workgroups only add
  // starts and joins (4 x 32768 keys, 16 / 2 heads of 128, fp16: 1, 2, 3, 4 per unit took 30, 35, 42, 45 us)
  const int64_t want = jobs >= cus ? 1 : cus / jobs;
  p.splits = (int)(want < most ? want : most);
  if (p.splits > kMaxSplits) p.splits = kMaxSplits;
  p.tiles_per_split = ceil_div(ceil_div(key_tiles, p.splits), 4) * 4;
  p.splits = ceil_div(key_tiles, p.tiles_per_split);
  return p;
}

}  // namespace attn
}  // namespace pstl
