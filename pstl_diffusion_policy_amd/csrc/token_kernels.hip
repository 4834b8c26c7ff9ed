// token_kernels.hip -- the elementwise neighbours of attention: RMS norm of queries and keys per head with the position rotation
// in the same pass (and its backward pass), and dropout + residual with a mask that is never stored.
#include "attn_host.hpp"

namespace pstl {
namespace attn {
namespace {

// ---- per-head norm + rotation ----------------------------------------------------------------------------------------
//   xhat = x / sqrt(mean_d x^2 + eps);  z = w o xhat;  y = rotate(z, pos f):  (a, b) -> (a cos - b sin, b cos + a sin) per pair
//   dz = rotate(dy, -pos f);  dw = sum dz o xhat;  dx = (w o dz - xhat mean_d(w o dz o xhat)) / sqrt(...)
// Bound by memory (forward: read x, write y; backward: read x and dy, write dx).  A thread owns two 8-element chunks of one head,
// half the rotated width apart, so that both pair orders are rotated inside the thread; `lanes` (a power of two) consecutive
// lanes make a head.  The angles of a token are shared by all its heads: they are formed once per workgroup, in 64 bits and in
// revolutions (pos f / 2 pi less its whole part), because a float32 angle of position 10^6 is off by 0.06 rad.
struct RopeArgs {
  Mat x[2], y[2], dy[2], dx[2];      // [0] queries, [1] keys
  const float* w[2];
  const int64_t* pos;
  int64_t pos_sb;
  const double* freq;
  float* part;                       // (workgroups, 2, D) sums of dz o xhat
  int heads[2];
  int L, D, rot, pairs, lanes, lane_shift, interleaved, per_block;
  int64_t tokens;
  float eps;
};
constexpr int kRopeTable = 2048;     // (cos, sin) entries of a workgroup

template <typename T>
__device__ inline f32x8 up8(const T* p) {
  return __builtin_convertvector(load8<T>(p), f32x8);
}
template <typename T>
__device__ inline void down8(T* p, f32x8 v) {
  const Frag<T> f = __builtin_convertvector(v, Frag<T>);
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<u32x4v*>(p) = __builtin_bit_cast(u32x4v, f);
  } else {
    reinterpret_cast<f32x4*>(p)[0] = __builtin_shufflevector(f, f, 0, 1, 2, 3);
    reinterpret_cast<f32x4*>(p)[1] = __builtin_shufflevector(f, f, 4, 5, 6, 7);
  }
}
__device__ inline void rotate(f32x8& a, f32x8& b, const float2* cs, const RopeArgs& p, int chunk, float sign) {
  if (p.interleaved) {
    const float2 *c0 = cs + 4 * chunk, *c1 = c0 + (p.rot >> 2);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const float2 u = c0[m], v = c1[m];
      const float a0 = a[2 * m], a1 = a[2 * m + 1], b0 = b[2 * m], b1 = b[2 * m + 1], us = sign * u.y, vs = sign * v.y;
      a[2 * m] = a0 * u.x - a1 * us, a[2 * m + 1] = a1 * u.x + a0 * us;
      b[2 * m] = b0 * v.x - b1 * vs, b[2 * m + 1] = b1 * v.x + b0 * vs;
    }
  } else {
    const float2* c0 = cs + 8 * chunk;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const float2 u = c0[m];
      const float a0 = a[m], b0 = b[m], us = sign * u.y;
      a[m] = a0 * u.x - b0 * us, b[m] = b0 * u.x + a0 * us;
    }
  }
}
__device__ inline float lanes_sum(float v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ inline float dot8(f32x8 a, f32x8 b) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = __builtin_fmaf(a[j], b[j], s);
  return s;
}

template <typename T, bool BWD>
__global__ __launch_bounds__(256) void k_qk_norm_rope(RopeArgs p) {
  __shared__ float2 table[kRopeTable];
  __shared__ float sums[4][64][17];
  const int tid = threadIdx.x, half = p.rot >> 1;
  // a thread's place inside a head is the same in every iteration (256 is a multiple of `lanes`)
  const int c = tid & (p.lanes - 1);
  const bool pair = c < p.pairs;
  const int d0 = pair ? 8 * c : p.rot + 8 * (c - p.pairs), d1 = d0 + half;
  const bool ok = d0 < p.D;
  const f32x8 zero = {};
  f32x8 wa[2], wb[2], ga[2], gb[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    wa[s] = ok ? up8<float>(p.w[s] + d0) : zero;
    wb[s] = ok && pair ? up8<float>(p.w[s] + d1) : zero;
    ga[s] = zero, gb[s] = zero;
  }
  for (int64_t t0 = (int64_t)blockIdx.x * p.per_block; t0 < p.tokens; t0 += (int64_t)gridDim.x * p.per_block) {
    const int nt = (int)min((int64_t)p.per_block, p.tokens - t0);
    __syncthreads();
    for (int e = tid; e < nt * half; e += 256) {
      const int tt = e / half, i = e - tt * half;
      const int64_t tok = t0 + tt, b = tok / p.L, l = tok - b * p.L;
      const double rev = (double)p.pos[b * p.pos_sb + l] * (p.freq[i] * 0.15915494309189533577);
      const float x = 2.0f * (float)(rev - __builtin_rint(rev));
      table[e] = float2{cospif(x), sinpif(x)};
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int H = p.heads[s], n = (nt * H) << p.lane_shift;
      for (int u = tid; u < n; u += 256) {
        const int th = u >> p.lane_shift, tt = th / H, h = th - tt * H;
        const int64_t tok = t0 + tt, b = tok / p.L, l = tok - b * p.L;
        const T* x = reinterpret_cast<const T*>(p.x[s].p) + b * p.x[s].sb + l * p.x[s].sl + h * p.x[s].sh;
        f32x8 a = ok ? up8<T>(x + d0) : zero, bb = ok && pair ? up8<T>(x + d1) : zero;
        const float ss = lanes_sum(dot8(a, a) + dot8(bb, bb), p.lanes);
        const float rstd = 1.0f / __builtin_sqrtf(ss / (float)p.D + p.eps);
        a *= rstd, bb *= rstd;
        if (!BWD) {
          a *= wa[s], bb *= wb[s];
          if (pair) rotate(a, bb, table + tt * half, p, c, 1.0f);
          T* y = reinterpret_cast<T*>(p.y[s].p) + b * p.y[s].sb + l * p.y[s].sl + h * p.y[s].sh;
          if (ok) down8<T>(y + d0, a);
          if (ok && pair) down8<T>(y + d1, bb);
        } else {
          const T* dy = reinterpret_cast<const T*>(p.dy[s].p) + b * p.dy[s].sb + l * p.dy[s].sl + h * p.dy[s].sh;
          f32x8 za = ok ? up8<T>(dy + d0) : zero, zb = ok && pair ? up8<T>(dy + d1) : zero;
          if (pair) rotate(za, zb, table + tt * half, p, c, -1.0f);
          ga[s] += za * a, gb[s] += zb * bb;
          za *= wa[s], zb *= wb[s];
          const float mean = lanes_sum(dot8(za, a) + dot8(zb, bb), p.lanes) / (float)p.D;
          T* dx = reinterpret_cast<T*>(p.dx[s].p) + b * p.dx[s].sb + l * p.dx[s].sl + h * p.dx[s].sh;
          if (ok) down8<T>(dx + d0, (za - a * mean) * rstd);
          if (ok && pair) down8<T>(dx + d1, (zb - bb * mean) * rstd);
        }
      }
    }
  }
  if (BWD) {      // sums of the workgroup, in a fixed order: over the lanes of a wavefront that share a place, then the wavefronts
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        for (int o = p.lanes; o < 64; o <<= 1) {
          ga[s][j] += __shfl_xor(ga[s][j], o);
          gb[s][j] += __shfl_xor(gb[s][j], o);
        }
      __syncthreads();
      if (lane < p.lanes)
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[wave][lane][j] = ga[s][j], sums[wave][lane][8 + j] = gb[s][j];
      __syncthreads();
      for (int e = tid; e < p.lanes * 16; e += 256) {
        const int lc = e >> 4, j = e & 15, second = j >> 3;
        const bool lp = lc < p.pairs;
        const int d = (lp ? 8 * lc + second * half : p.rot + 8 * (lc - p.pairs)) + (j & 7);
        if (d >= p.D || (second && !lp)) continue;
        p.part[((int64_t)blockIdx.x * 2 + s) * p.D + d] = sums[0][lc][j] + sums[1][lc][j] + sums[2][lc][j] + sums[3][lc][j];
      }
    }
  }
}

// dw[s][d] = sum over the workgroups' parts: one workgroup per (s, 32 elements), 32 strided sums each, joined in order.  Bound by
// the latency of its loads: eight are in flight per thread (8 strided sums with one load in flight took 60 us for 2048 parts).
__global__ __launch_bounds__(1024) void k_qk_norm_rope_dw(const float* part, int blocks, int D, float* dwq, float* dwk) {
  __shared__ float s[32][32];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, d = (int)blockIdx.x * 32 + lane, which = blockIdx.y;
  float sum = 0.0f;
  if (d < D) {
    for (int i0 = g; i0 < blocks; i0 += 256) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i0 + 32 * u < blocks ? part[((int64_t)(i0 + 32 * u) * 2 + which) * D + d] : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += v[u];
    }
  }
  s[g][lane] = sum;
  __syncthreads();
  if (g == 0 && d < D) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += s[i][lane];
    (which ? dwk : dwq)[d] = v;
  }
}

int rope_args(const pstl_qk_rope* c, RopeArgs* p, bool backward) {
  if (!c) return PSTL_ERR_ARG;
  if (c->dtype != PSTL_F32 && c->dtype != PSTL_BF16 && c->dtype != PSTL_F16) return PSTL_ERR_SHAPE;
  if (c->B < 0 || c->L < 0 || c->Hq < 1 || c->Hk < 1 || !(c->eps >= 0.0f)) return PSTL_ERR_ARG;
  if (c->D < 8 || c->D > PSTL_ROPE_MAX_D || c->D % 8 || c->rot < 16 || c->rot > c->D || c->rot % 16) return PSTL_ERR_SHAPE;
  if (c->Hq > 65536 || c->Hk > 65536) return PSTL_ERR_SHAPE;
  *p = RopeArgs();
  const int el = c->dtype == PSTL_F32 ? 4 : 2;
  const bool any = (int64_t)c->B * c->L > 0;
  const pstl_attn_mat* in[2] = {&c->q, &c->k};
  const pstl_attn_mat* out[2] = {backward ? &c->dq : &c->yq, backward ? &c->dk : &c->yk};
  const pstl_attn_mat* up[2] = {&c->dyq, &c->dyk};
  auto mat = [](const pstl_attn_mat& m) { return Mat{(char*)m.p, m.stride_b, m.stride_l, m.stride_h}; };
  for (int s = 0; s < 2; ++s) {
    if (int e = mat_ok(*in[s], el, any)) return e;
    if (int e = mat_ok(*out[s], el, any)) return e;
    if (backward)
      if (int e = mat_ok(*up[s], el, any)) return e;
    p->x[s] = mat(*in[s]), p->y[s] = p->dx[s] = mat(*out[s]), p->dy[s] = mat(*up[s]);
  }
  if (!c->wq || !c->wk || !c->inv_freq || (any && !c->positions) || !aligned16(c->wq) || !aligned16(c->wk)) return PSTL_ERR_ARG;
  if (backward && (!c->dwq || !c->dwk || !c->work)) return PSTL_ERR_ARG;
  p->w[0] = c->wq, p->w[1] = c->wk, p->pos = c->positions, p->pos_sb = c->pos_stride_b, p->freq = c->inv_freq;
  p->part = c->work, p->heads[0] = c->Hq, p->heads[1] = c->Hk;
  p->L = c->L, p->D = c->D, p->rot = c->rot, p->interleaved = c->interleaved != 0, p->eps = c->eps;
  p->pairs = c->rot / 16;
  const int need = p->pairs + (c->D - c->rot) / 8;
  while (p->lanes = 1 << p->lane_shift, p->lanes < need) ++p->lane_shift;
  p->tokens = (int64_t)c->B * c->L;
  return PSTL_OK;
}
constexpr int kRopeMaxBlocks = 2048;
// workgroups and tokens per workgroup and iteration: one token each while that does not fill the chip, else a few, so that the
// angles' table is shared by at least two iterations of the heads' loop
void rope_grid(RopeArgs* p, int* blocks) {
  const int units = (p->heads[0] + p->heads[1]) << p->lane_shift;
  int per = 1;
  while (per < 32 && per * units < 1024 && p->tokens > (int64_t)per * 2 * kRopeMaxBlocks && 2 * per * (p->rot / 2) <= kRopeTable) per *= 2;
  p->per_block = per;
  const int64_t n = (p->tokens + per - 1) / per;
  *blocks = (int)(n < kRopeMaxBlocks ? n : kRopeMaxBlocks);
}

// ---- dropout + residual ------------------------------------------------------------------------------------------------
//   y = residual + m x / keep,   m_n = [16 bits of philox((n + offset) / 8, 'DROP')  >=  65536 p]
// Bound by memory; one draw of 128 bits serves eight elements.  A multiplication by the mask would turn a dropped infinity into
// NaN: dropped elements are selected away.
struct DropArgs {
  const void *x, *res;
  void* y;
  int64_t n;
  uint64_t offset, seed;
  const uint64_t* seed_dev;
  uint32_t thr;
  float gain;
};
constexpr uint32_t kDropElTag = 0x44524F50u;

__device__ inline void drop_bits8(uint64_t seed, uint64_t first, uint32_t (&bits)[8]) {      // decisions of elements first .. + 7
  const uint64_t g = first >> 3;
  const u32x4 a = philox4x32(u32x4{(uint32_t)g, (uint32_t)(g >> 32), 0u, kDropElTag}, (uint32_t)seed, (uint32_t)(seed >> 32));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) bits[j] = (w[j >> 1] >> (16 * (j & 1))) & 0xffffu;
}

template <typename T>
__global__ __launch_bounds__(256) void k_dropout_add(DropArgs p, int vec) {
  const int64_t v = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (v >= p.n) return;
  const uint64_t seed = p.seed_dev ? uniform_u64(p.seed_dev) : p.seed;
  const uint64_t first = (uint64_t)v + p.offset;
  const uint32_t sh = (uint32_t)first & 7u;
  uint32_t bits[8];
  drop_bits8(seed, first, bits);
  if (sh) {       // (the same for every thread: v is a multiple of 8) the eight elements straddle two draws
    uint32_t next[8], all[8];
    drop_bits8(seed, first + 8, next);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      all[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if ((uint32_t)i == ((j + sh) & 7u)) all[j] = (j + sh) < 8u ? bits[i] : next[i];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) bits[j] = all[j];
  }
  const T *x = static_cast<const T*>(p.x) + v, *res = p.res ? static_cast<const T*>(p.res) + v : nullptr;
  T* y = static_cast<T*>(p.y) + v;
  if (vec && v + 8 <= p.n) {
    f32x8 a = up8<T>(x);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = bits[j] >= p.thr ? a[j] * p.gain : 0.0f;
    if (res) a += up8<T>(res);
    down8<T>(y, a);
  } else {
    const int m = (int)min((int64_t)8, p.n - v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < m) {
        const float a = bits[j] >= p.thr ? (float)x[j] * p.gain : 0.0f;
        y[j] = (T)(res ? a + (float)res[j] : a);
      }
  }
}

template <typename T>
int rope_launch(RopeArgs& p, bool backward, float* dwq, float* dwk, hipStream_t st) {
  int blocks;
  rope_grid(&p, &blocks);
  if (blocks > 0) {
    if (backward)
      hipLaunchKernelGGL((k_qk_norm_rope<T, true>), dim3(blocks), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((k_qk_norm_rope<T, false>), dim3(blocks), dim3(256), 0, st, p);
    if (int e = launch_status()) return e;
  }
  if (backward)
    hipLaunchKernelGGL(k_qk_norm_rope_dw, dim3((p.D + 31) / 32, 2), dim3(1024), 0, st, p.part, blocks, p.D, dwq, dwk);
  return launch_status();
}
int rope_run(const pstl_qk_rope* c, bool backward, void* stream) {
  RopeArgs p;
  if (int e = rope_args(c, &p, backward)) return e;
  switch (c->dtype) {
    case PSTL_F32: return rope_launch<float>(p, backward, c->dwq, c->dwk, as_stream(stream));
    case PSTL_BF16: return rope_launch<__bf16>(p, backward, c->dwq, c->dwk, as_stream(stream));
    default: return rope_launch<_Float16>(p, backward, c->dwq, c->dwk, as_stream(stream));
  }
}

}  // namespace
}  // namespace attn
}  // namespace pstl

using namespace pstl;
using namespace pstl::attn;

extern "C" int pstl_qk_norm_rope(const pstl_qk_rope* c, void* stream) { return rope_run(c, false, stream); }
extern "C" int pstl_qk_norm_rope_backward(const pstl_qk_rope* c, void* stream) { return rope_run(c, true, stream); }
extern "C" size_t pstl_qk_norm_rope_work_floats(const pstl_qk_rope* c) {
  return c && c->D > 0 && c->D <= PSTL_ROPE_MAX_D ? (size_t)kRopeMaxBlocks * 2 * c->D : 0;
}

extern "C" int pstl_dropout_add(int dtype, int64_t n, const void* x, const void* residual, void* y, int threshold, int64_t seed,
                                const uint64_t* seed_dev, int64_t offset, void* stream) {
  if (dtype != PSTL_F32 && dtype != PSTL_BF16 && dtype != PSTL_F16) return PSTL_ERR_SHAPE;
  if (n < 0 || threshold < 0 || threshold > 65536 || offset < 0) return PSTL_ERR_ARG;
  if (n == 0) return PSTL_OK;
  if (!x || !y) return PSTL_ERR_ARG;
  const uintptr_t el = dtype == PSTL_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) % el) return PSTL_ERR_ARG;
  const int64_t blocks = (n + 2047) / 2048;
  if (blocks >= (1ll << 31)) return PSTL_ERR_SHAPE;
  DropArgs p = {x, residual, y, n, (uint64_t)offset, (uint64_t)seed, seed_dev, (uint32_t)threshold,
                threshold < 65536 ? 65536.0f / (float)(65536 - threshold) : 0.0f};
  const int vec = aligned16(x) && aligned16(y) && aligned16(residual);
  const dim3 grid((unsigned)blocks), block(256);
  switch (dtype) {
    case PSTL_F32: hipLaunchKernelGGL(k_dropout_add<float>, grid, block, 0, as_stream(stream), p, vec); break;
    case PSTL_BF16: hipLaunchKernelGGL(k_dropout_add<__bf16>, grid, block, 0, as_stream(stream), p, vec); break;
    default: hipLaunchKernelGGL(k_dropout_add<_Float16>, grid, block, 0, as_stream(stream), p, vec); break;
  }
  return launch_status();
}
