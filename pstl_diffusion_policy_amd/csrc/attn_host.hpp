// attn_host.hpp -- host side of the attention entry points: argument checks and the choice of a kernel.
#pragma once
#include <math.h>

#include "attn_core.hpp"

namespace pstl {
namespace attn {

enum Check { kCheckShape, kCheckForward, kCheckBackward };

inline int mat_ok(const pstl_attn_mat& m, int el, bool needed) {
  if (!m.p) return needed ? PSTL_ERR_ARG : PSTL_OK;
  const int64_t per = 16 / el;      // rows are read 16 bytes at a time
  if (!aligned16(m.p) || m.stride_b % per || m.stride_l % per || m.stride_h % per) return PSTL_ERR_ARG;
  return PSTL_OK;
}

inline int attn_args(const pstl_attn* c, Args* a, Check what) {
  if (!c) return PSTL_ERR_ARG;
  if (c->dtype != PSTL_F32 && c->dtype != PSTL_BF16 && c->dtype != PSTL_F16) return PSTL_ERR_SHAPE;
  if (c->B < 0 || c->Lq < 0 || c->Lk < 0 || c->Hq < 1 || c->Hk < 1) return PSTL_ERR_ARG;
  if (c->D < 8 || c->D > PSTL_ATTN_MAX_D || c->D % 8 || c->Hq % c->Hk) return PSTL_ERR_SHAPE;
  const int64_t G = c->Hq / c->Hk, R = (int64_t)c->Lq * G;
  // 32-bit row and key indexes with room for the tiles past the end, and the exact division of a row index by G
  if (R * G >= (1ll << 31) || R >= (1ll << 30) || c->Lk >= (1 << 30) || (int64_t)c->B * c->Hk >= (1ll << 30)) return PSTL_ERR_SHAPE;
  if (!(c->scale > 0.0f) || !(c->scale * kLog2e < INFINITY)) return PSTL_ERR_ARG;
  const int thr = c->dropout_256;
  if (thr < 0 || thr > 255) return PSTL_ERR_ARG;
  *a = Args();
  auto mat = [](const pstl_attn_mat& m) { return Mat{(char*)m.p, m.stride_b, m.stride_l, m.stride_h}; };
  a->q = mat(c->q), a->k = mat(c->k), a->v = mat(c->v), a->o = mat(c->o);
  a->dout = mat(c->dout), a->dq = mat(c->dq), a->dk = mat(c->dk), a->dv = mat(c->dv);
  a->lse = c->lse, a->key_mask = c->key_mask, a->mask_sb = c->mask_stride_b, a->q_lens = c->q_lens, a->k_lens = c->k_lens;
  a->part = c->work, a->delta = c->work, a->seed = c->seed, a->seed_dev = c->seed_dev;
  a->B = c->B, a->Lq = c->Lq, a->Lk = c->Lk, a->Hk = c->Hk, a->G = (int)G, a->D = c->D, a->R = (int)R, a->causal = c->causal != 0;
  a->g_magic = G > 1 ? (uint32_t)((1ull << 32) / (uint64_t)G + 1) : 0;
  a->hk_magic = c->Hk > 1 ? (uint32_t)((1ull << 32) / (uint64_t)c->Hk + 1) : 0;
  a->scale = c->scale, a->c = c->scale * kLog2e;
  a->thr = (uint32_t)thr, a->keep_inv = 256.0f / (float)(256 - thr);
  if (what == kCheckShape) return PSTL_OK;
  const int el = c->dtype == PSTL_F32 ? 4 : 2;
  const bool rows = (int64_t)c->B * R > 0, keys = (int64_t)c->B * c->Lk > 0;
  for (int e : {mat_ok(c->q, el, rows), mat_ok(c->o, el, rows), mat_ok(c->k, el, keys), mat_ok(c->v, el, keys)})
    if (e) return e;
  if (what == kCheckBackward) {
    for (int e : {mat_ok(c->dout, el, rows), mat_ok(c->dq, el, rows), mat_ok(c->dk, el, keys), mat_ok(c->dv, el, keys)})
      if (e) return e;
    if (rows && (!c->lse || !c->work)) return PSTL_ERR_ARG;
  }
  return PSTL_OK;
}

// lets a kernel use `bytes` of dynamic LDS (more than 64 KB must be asked for), once per device
template <auto Kernel>
inline int allow_lds(int bytes) {
  static DeviceOnce once;
  const int dev = current_device();
  if (once.done(dev)) return PSTL_OK;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return PSTL_ERR_LAUNCH;
  once.set(dev);
  return PSTL_OK;
}

// ---- forward ---------------------------------------------------------------------------------------------------------
constexpr int kMaxSplits = 1024;
enum Kind { kManyRows, kShort, kShortPairs, kFewRows };
struct FwdPlan {
  Kind kind;
  int n_tiles, splits, tiles_per_split, cus_per_xcd;
};
inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// two units share a wavefront (attn_core.hpp, Slot)
inline bool in_pairs(const Args& a) {
  return a.Lk <= 16 && a.R <= 16 && (int64_t)a.B * a.Hk * a.Hk < (1ll << 31);
}
inline FwdPlan plan_forward(const Args& a, bool f32, int cus) {
  const int64_t units = (int64_t)a.B * a.Hk;
  FwdPlan p = {kManyRows, ceil_div(a.R, 128), 1, 0, cus >= 8 ? cus / 8 : 1};
  // (up to 32 keys one tile holds them; 4096 x 12 tokens, 8 heads of 32, bf16: 22 us, one unit to a wavefront 29, many-rows 130)
  if (a.Lk <= 32) {
    p.kind = in_pairs(a) ? kShortPairs : kShort;
    p.n_tiles = ceil_div(a.R, 32);
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
  const bool few = a.R <= 32 || (f32 ? wgs * 2 <= cus && a.Lk >= 128 : wgs * 4 <= cus && a.Lk >= 256);
  if (!few) return p;
  p.kind = kFewRows;
  p.n_tiles = ceil_div(a.R, 32);
  const int64_t jobs = units * p.n_tiles;
  // a part has at least 8 tiles (two per wavefront), and up to 16 tiles are not divided at all: joining costs a launch of 4 us
  const int key_tiles = ceil_div(a.Lk, 32), most = key_tiles <= 16 ? 1 : ceil_div(key_tiles, 8);
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
