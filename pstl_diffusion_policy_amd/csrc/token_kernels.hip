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
// 4 x 4096 tokens, 20 heads of 128, bf16: forward 40 us (168 MB = 4.2 TB/s), backward 71 us (252 MB = 3.6 TB/s: its wavefronts wait
// 75 % of their cycles, because a thread's first loads stand behind the barriers and the angles of its table; the vector pipe is
// busy half of the time); 2048 x 20 tokens, 16 heads of 32, float32: 41 and 57 us.
// (Heads summed by shuffles through the LDS and queries' and keys' gradients in one workgroup: 43 and 93 us.)
struct RopeArgs {
  Mat x[2], y[2], dy[2], dx[2];      // [0] queries, [1] keys
  const float* w[2];
  const int64_t* pos;
  int64_t pos_sb;
  const double* freq;
  float* part;                       // (workgroups, 2, D) sums of dz o xhat
  int heads[2];
  uint32_t head_magic[2];            // x / heads = umulhi(x, magic) for heads > 1 (x heads < 2^32: kRopeTokens and the heads are bounded)
  int L, D, rot, pairs, lanes, lane_shift, interleaved, per_block, tokens;
  float eps, inv_d;
};
constexpr int kRopeTable = 2048;     // (cos, sin) entries of a workgroup
constexpr int kRopeTokens = 32;      // tokens of a workgroup and iteration, at most

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
    const f32x4 *c0 = reinterpret_cast<const f32x4*>(cs + 4 * chunk), *c1 = reinterpret_cast<const f32x4*>(cs + 4 * chunk + (p.rot >> 2));
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const f32x4 uu = c0[m >> 1], vv = c1[m >> 1];
      const float ux = uu[2 * (m & 1)], us = sign * uu[2 * (m & 1) + 1], vx = vv[2 * (m & 1)], vs = sign * vv[2 * (m & 1) + 1];
      const float a0 = a[2 * m], a1 = a[2 * m + 1], b0 = b[2 * m], b1 = b[2 * m + 1];
      a[2 * m] = a0 * ux - a1 * us, a[2 * m + 1] = a1 * ux + a0 * us;
      b[2 * m] = b0 * vx - b1 * vs, b[2 * m + 1] = b1 * vx + b0 * vs;
    }
  } else {
    const f32x4* c0 = reinterpret_cast<const f32x4*>(cs + 8 * chunk);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const f32x4 uu = c0[m >> 1];
      const float ux = uu[2 * (m & 1)], us = sign * uu[2 * (m & 1) + 1];
      const float a0 = a[m], b0 = b[m];
      a[m] = a0 * ux - b0 * us, b[m] = b0 * ux + a0 * us;
    }
  }
}
// sum over the `lanes` (1, 2, ... 32) neighbouring lanes of a head.  Inside a row of 16 by DPP: once the sums of 2, 4, 8 lanes are
// equal in their groups, mirroring a group of 4, 8, 16 brings the other half's.
template <int CTRL>
__device__ inline float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ inline float lanes_sum(float v, int lanes) {
  if (lanes > 1) v = dpp_add<0xB1>(v);       // quad_perm [1,0,3,2]
  if (lanes > 2) v = dpp_add<0x4E>(v);       // quad_perm [2,3,0,1]
  if (lanes > 4) v = dpp_add<0x141>(v);      // row_half_mirror
  if (lanes > 8) v = dpp_add<0x140>(v);      // row_mirror
  if (lanes > 16) v += __shfl_xor(v, 16);
  return v;
}
// 1 / sqrt(v): v_rsq_f32 (good to a step) and one Newton step; an overflowed sum of squares keeps its 0
__device__ inline float inv_sqrt(float v) {
  const float r = __builtin_amdgcn_rsqf(v), e = __builtin_fmaf(-v * r, r, 1.0f);
  return v < INFINITY ? __builtin_fmaf(0.5f * r, e, r) : r;
}
__device__ inline float dot8(f32x8 a, f32x8 b) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = __builtin_fmaf(a[j], b[j], s);
  return s;
}

template <typename T, bool BWD>
__global__ __launch_bounds__(256, 4) void k_qk_norm_rope(RopeArgs p) {
  __shared__ __attribute__((aligned(16))) char lds[BWD ? 4 * 32 * 17 * 4 : kRopeTable * 8];
  __shared__ __attribute__((aligned(16))) float weight[2][PSTL_ROPE_MAX_D];
  __shared__ int2 place[kRopeTokens];      // (sequence, position in it) of the iteration's tokens
  float2* table = reinterpret_cast<float2*>(lds);
  static_assert(4 * 32 * 17 * 4 >= 1024 * 8, "the backward table fits");
  const int tid = threadIdx.x, half = p.rot >> 1;
  // a thread's place inside a head is the same in every iteration (256 is a multiple of `lanes`)
  const int c = tid & (p.lanes - 1);
  const bool pair = c < p.pairs;
  const int d0 = pair ? 8 * c : p.rot + 8 * (c - p.pairs), d1 = d0 + half;
  const bool ok = d0 < p.D;
  const f32x8 zero = {};
  f32x8 ga = zero, gb = zero;
  const int s_first = BWD ? (int)blockIdx.y : 0, s_end = BWD ? s_first + 1 : 2;      // (backward: queries or keys, one set of sums)
  for (int s = s_first; s < s_end; ++s)
    for (int d = tid; d < p.D; d += 256) weight[s][d] = p.w[s][d];
  const int w0 = ok ? d0 : 0, w1 = ok && pair ? d1 : 0;      // (a lane without elements multiplies zeros)
  for (int t0 = (int)blockIdx.x * p.per_block; t0 < p.tokens; t0 += (int)gridDim.x * p.per_block) {
    const int nt = min(p.per_block, p.tokens - t0);
    __syncthreads();
    if (tid < nt) {
      const int b = (t0 + tid) / p.L;
      place[tid] = int2{b, t0 + tid - b * p.L};
    }
    __syncthreads();
    for (int e = tid; e < nt * half; e += 256) {
      const int tt = e / half, i = e - tt * half;
      const int2 at = place[tt];
      const double rev = (double)p.pos[at.x * p.pos_sb + at.y] * (p.freq[i] * 0.15915494309189533577);
      const float x = 2.0f * (float)(rev - __builtin_rint(rev));
      table[e] = float2{cospif(x), sinpif(x)};
    }
    __syncthreads();
#pragma unroll
    for (int s = s_first; s < s_end; ++s) {
      const int H = p.heads[s], n = (nt * H) << p.lane_shift;
      for (int u = tid; u < n; u += 256) {
        const int th = u >> p.lane_shift, tt = H == 1 ? th : (int)__umulhi((uint32_t)th, p.head_magic[s]), h = th - tt * H;
        const int2 at = place[tt];
        const T* x = reinterpret_cast<const T*>(p.x[s].p) + at.x * p.x[s].sb + at.y * p.x[s].sl + h * p.x[s].sh;
        f32x8 a = ok ? up8<T>(x + d0) : zero, bb = ok && pair ? up8<T>(x + d1) : zero;
        f32x8 za, zb;
        if (BWD) {
          const T* dy = reinterpret_cast<const T*>(p.dy[s].p) + at.x * p.dy[s].sb + at.y * p.dy[s].sl + h * p.dy[s].sh;
          za = ok ? up8<T>(dy + d0) : zero, zb = ok && pair ? up8<T>(dy + d1) : zero;
        }
        const float ss = lanes_sum(dot8(a, a) + dot8(bb, bb), p.lanes);
        const float rstd = inv_sqrt(__builtin_fmaf(ss, p.inv_d, p.eps));
        a *= rstd, bb *= rstd;
        if (!BWD) {
          a *= up8<float>(&weight[s][w0]), bb *= up8<float>(&weight[s][w1]);
          if (pair) rotate(a, bb, table + tt * half, p, c, 1.0f);
          T* y = reinterpret_cast<T*>(p.y[s].p) + at.x * p.y[s].sb + at.y * p.y[s].sl + h * p.y[s].sh;
          if (ok) down8<T>(y + d0, a);
          if (ok && pair) down8<T>(y + d1, bb);
        } else {
          if (pair) rotate(za, zb, table + tt * half, p, c, -1.0f);
          ga += za * a, gb += zb * bb;
          za *= up8<float>(&weight[s][w0]), zb *= up8<float>(&weight[s][w1]);
          const float mean = lanes_sum(dot8(za, a) + dot8(zb, bb), p.lanes) * p.inv_d;
          T* dx = reinterpret_cast<T*>(p.dx[s].p) + at.x * p.dx[s].sb + at.y * p.dx[s].sl + h * p.dx[s].sh;
          if (ok) down8<T>(dx + d0, (za - a * mean) * rstd);
          if (ok && pair) down8<T>(dx + d1, (zb - bb * mean) * rstd);
        }
      }
    }
  }
  if (BWD) {      // sums of the workgroup, in a fixed order: over the lanes of a wavefront that share a place, then the wavefronts
    const int lane = tid & 63, wave = tid >> 6;
    float(*sums)[32][17] = reinterpret_cast<float(*)[32][17]>(lds);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      for (int o = p.lanes; o < 64; o <<= 1) {
        ga[j] += __shfl_xor(ga[j], o);
        gb[j] += __shfl_xor(gb[j], o);
      }
    __syncthreads();
    if (lane < p.lanes)
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[wave][lane][j] = ga[j], sums[wave][lane][8 + j] = gb[j];
    __syncthreads();
    for (int e = tid; e < p.lanes * 16; e += 256) {
      const int lc = e >> 4, j = e & 15, second = j >> 3;
      const bool lp = lc < p.pairs;
      const int d = (lp ? 8 * lc + second * half : p.rot + 8 * (lc - p.pairs)) + (j & 7);
      if (d >= p.D || (second && !lp)) continue;
      p.part[((int64_t)blockIdx.x * 2 + s_first) * p.D + d] = sums[0][lc][j] + sums[1][lc][j] + sums[2][lc][j] + sums[3][lc][j];
    }
  }
}

// dw[s][d] = sum over the workgroups' parts: one workgroup per (s, 16 elements), 64 strided sums each, joined in a fixed order.  In 64
// bits: up to 2048 parts of either sign are added one after another, which in 32 bits was most of a weight gradient's error (2.3e-7
// of its size against 1.1e-7 at 2048 x 20 tokens, 8 heads of 32, float32).  Bound by the latency of its loads: sixteen are in flight
// per thread (past the end the last part again, not counted: a branch around each load would wait for it before the next, 19 us).
// 2048 parts of 32 and 128 elements take 4.6 and 5.3 us.
__global__ __launch_bounds__(1024) void k_qk_norm_rope_dw(const float* part, int blocks, int D, float* dwq, float* dwk) {
  __shared__ double s[64][16];
  const int lane = threadIdx.x & 15, g = threadIdx.x >> 4, d = (int)blockIdx.x * 16 + lane, which = blockIdx.y;
  double sum = 0.0;
  if (d < D) {
    for (int i0 = g; i0 < blocks; i0 += 1024) {
      float v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = part[((int64_t)min(i0 + 64 * u, blocks - 1) * 2 + which) * D + d];
#pragma unroll
      for (int u = 0; u < 16; ++u) sum += i0 + 64 * u < blocks ? (double)v[u] : 0.0;
    }
  }
  s[g][lane] = sum;
  __syncthreads();
  if (g < 8) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += s[g + 8 * i][lane];
    s[g][lane] = sum;      // (of this column's rows g + 8 i only this thread reads and writes)
  }
  __syncthreads();
  if (g == 0 && d < D) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += s[i][lane];
    (which ? dwk : dwq)[d] = (float)sum;
  }
}

constexpr int kRopeMaxBlocks = 2048;
int rope_args(const pstl_qk_rope* c, RopeArgs* p, bool backward) {
  if (!c) return PSTL_ERR_ARG;
  if (c->dtype != PSTL_F32 && c->dtype != PSTL_BF16 && c->dtype != PSTL_F16) return PSTL_ERR_SHAPE;
  if (c->B < 0 || c->L < 0 || c->Hq < 1 || c->Hk < 1 || !(c->eps >= 0.0f)) return PSTL_ERR_ARG;
  if (c->D < 8 || c->D > PSTL_ROPE_MAX_D || c->D % 8 || c->rot < 16 || c->rot > c->D || c->rot % 16) return PSTL_ERR_SHAPE;
  if (c->Hq > 8192 || c->Hk > 8192) return PSTL_ERR_SHAPE;
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
  if ((int64_t)c->B * c->L >= (1ll << 30)) return PSTL_ERR_SHAPE;      // (32-bit tokens)
  p->tokens = c->B * c->L;
  auto magic = [](int d) { return d > 1 ? (uint32_t)((1ull << 32) / (uint64_t)d + 1) : 0u; };
  p->head_magic[0] = magic(c->Hq), p->head_magic[1] = magic(c->Hk);
  p->inv_d = 1.0f / (float)c->D;
  return PSTL_OK;
}
// workgroups and tokens per workgroup and iteration: one token each while that does not fill the chip, else as many as give every
// thread a few heads, so that the angles' table and the barriers around it are shared
void rope_grid(RopeArgs* p, int* blocks) {
  const int units = (p->heads[0] + p->heads[1]) << p->lane_shift, table = 1024;
  int per = 1;
  while (per < kRopeTokens && per * units < 2048 && p->tokens > per * 2 * kRopeMaxBlocks && 2 * per * (p->rot / 2) <= table) per *= 2;
  p->per_block = per;
  const int64_t n = ((int64_t)p->tokens + per - 1) / per;
  *blocks = (int)(n < kRopeMaxBlocks ? n : kRopeMaxBlocks);
}

// ---- dropout + residual ------------------------------------------------------------------------------------------------
//   y = residual + m x / keep,   m_n = [16 bits of philox((n + offset) / 8, 'DROP')  >=  65536 p]
// Bound by memory: 16384 x 1024, bf16, with residual: 101 MB in 20 us = 5.0 TB/s, the rate of a copy; backward 67 MB in 13 us.  One
// draw of 128 bits serves eight elements.  A multiplication by the mask would turn a dropped infinity into
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
      hipLaunchKernelGGL((k_qk_norm_rope<T, true>), dim3(blocks, 2), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((k_qk_norm_rope<T, false>), dim3(blocks), dim3(256), 0, st, p);
    if (int e = launch_status()) return e;
  }
  if (backward)
    hipLaunchKernelGGL(k_qk_norm_rope_dw, dim3((p.D + 15) / 16, 2), dim3(1024), 0, st, p.part, blocks, p.D, dwq, dwk);
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
  if (!grid_fits(blocks, 256)) return PSTL_ERR_SHAPE;
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
