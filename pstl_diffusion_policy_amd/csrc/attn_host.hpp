// attn_host.hpp -- host side of the attention entry points: argument checks (the choice of a kernel: attn_plan.hpp).
#pragma once
#include <math.h>

#include "attn_core.hpp"
#include "attn_plan.hpp"

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

// does a launch of that many workgroups have fewer than 2^32 threads, the most that a grid can hold?
inline bool grid_fits(int64_t workgroups, int threads) { return workgroups * threads < (1ll << 32); }

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

// two units share a wavefront (attn_core.hpp, Slot)
inline bool in_pairs(const Args& a) { return plan_in_pairs(a.B, a.Hk, a.R, a.Lk); }
inline FwdPlan plan_forward(const Args& a, bool f32, int cus) { return plan_forward(a.B, a.Hk, a.R, a.Lk, f32, cus); }

}  // namespace attn
}  // namespace pstl
