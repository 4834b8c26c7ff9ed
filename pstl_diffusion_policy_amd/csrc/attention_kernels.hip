// attention_kernels.hip -- softmax attention, forward: O = softmax(scale Q K^T) V over padded, ragged, grouped-head batches.
//
//   S_rj = scale q_r . k_j,  j < limit(r) and not hidden;   P = exp(S - lse_r),  lse_r = log sum_j exp(S_rj);   O = (m P / keep) V
// One pass over the keys with the running maximum and sum (32 bits); a row that sees no key gives zeros and lse = -inf.
// Scores are formed TRANSPOSED (S^T = K Q^T): a lane holds one row's scores, so that maximum, sum and rescaling need one exchange
// between the lane halves, and the probabilities are the second operand of O^T = V^T P^T where they stand (attn_core.hpp).
// Arithmetic: products of 16-bit inputs on v_mfma_f32_32x32x16 with 32-bit sums; the probabilities are rounded to the inputs' type
// for the second product (half a step of a value <= 1; the sum that divides them is taken before that rounding).  float32
// inputs: v_mfma_f32_32x32x2, nothing is rounded below 32 bits.
#include "attn_host.hpp"

namespace pstl {
namespace attn {
namespace {

template <typename T>
constexpr int block_keys() {
  return sizeof(T) == 2 ? 64 : 32;
}

// ---- many rows: 128 packed rows per workgroup, 32 per wavefront; tiles of keys and values shared through the LDS -----------
template <typename T, int DK, bool DROP>
__global__ __launch_bounds__(256, 2) void k_attn_fwd(Args a) {
  constexpr int W = lds_width(DK), BN = block_keys<T>(), NS = BN / 32;
  typedef Tile<T, W> TL;
  constexpr int kTileBytes = BN * TL::kRowBytes, kPer = BN * TL::kChunks / 256;
  __shared__ __attribute__((aligned(16))) char lds[2][2][kTileBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, col = lane & 31;
  const int work = xcd_order((int)blockIdx.x, (int)gridDim.x);
  const int unit = work / a.n_tiles, tile = a.n_tiles - 1 - (work - unit * a.n_tiles);   // (causal: the longest first)
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int r0 = tile * 128 + wave * 32, r = r0 + col;
  const int qi = row_query(a, r);
  const bool live = r < a.R && qi < n.q;
  const int lim = live ? row_limit(a, n, qi) : 0;
  // keys that some row of the workgroup sees; keys that every live row of the wavefront sees
  const int q_first = row_query(a, tile * 128), q_last = min(row_query(a, min(tile * 128 + 127, a.R - 1)), n.q - 1);
  const int kend = q_first < n.q ? row_limit(a, n, q_last) : 0;
  const int q_wave = row_query(a, r0), all_see = a.causal ? max(min(q_wave + n.k - n.q + 1, n.k), 0) : n.k;

  Frag<T> qf[DK / 16];
  load_row_frags<T, DK>(live ? row_ptr<T>(a, a.q, b, hk, r) : nullptr, live, a.D, hi, qf);
  f32x16 acc[DK / 32] = {};
  float m = -INFINITY, l = 0.0f;
  const uint64_t seed = DROP ? drop_seed(a) : 0;

  u32x4v stage[2][kPer];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = tid + 256 * i, row = id / TL::kChunks, c = (id % TL::kChunks) ^ TL::swz(row), key = k0 + row;
      const int d = c * TL::kChunkEl;
      bool ok = key < n.k && d < a.D;
      if (ok && a.key_mask) ok = a.key_mask[b * a.mask_sb + key] != 0;   // hidden keys may hold anything: 0 * NaN is NaN
      stage[0][i] = ok ? *reinterpret_cast<const u32x4v*>(key_ptr<T>(a.k, b, hk, key) + d) : u32x4v{0, 0, 0, 0};
      stage[1][i] = ok ? *reinterpret_cast<const u32x4v*>(key_ptr<T>(a.v, b, hk, key) + d) : u32x4v{0, 0, 0, 0};
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      *reinterpret_cast<u32x4v*>(&lds[buf][0][(tid + 256 * i) * 16]) = stage[0][i];
      *reinterpret_cast<u32x4v*>(&lds[buf][1][(tid + 256 * i) * 16]) = stage[1][i];
    }
  };
  if (kend > 0) {
    fetch(0);
    store(0);
  }
  __syncthreads();
  int buf = 0;
  for (int k0 = 0; k0 < kend; k0 += BN, buf ^= 1) {
    const bool more = k0 + BN < kend;
    if (more) fetch(k0 + BN);
    const char *kt = lds[buf][0], *vt = lds[buf][1];
    f32x16 s[NS] = {};
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) s[j] = mma(TL::row(kt, 32 * j + col, t, hi), qf[t], s[j]);
    if (k0 + BN > all_see || a.key_mask) {
      uint64_t vis = ~0ull;
      if (a.key_mask) {
        const int key = k0 + lane;
        vis = __ballot(key < n.k && lane < BN && a.key_mask[b * a.mask_sb + key] != 0) >> (4 * hi);
      }
#pragma unroll
      for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int g = 0; g < 16; ++g) {
          const int o = 32 * j + 8 * (g >> 2) + (g & 3);
          const bool see = k0 + o + 4 * hi < lim && ((vis >> o) & 1);
          s[j][g] = see ? s[j][g] : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int g = 0; g < 16; ++g) mx = fmaxf(mx, s[j][g]);
    const float m_new = fmaxf(m, half_max(mx) * a.c), mu = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - mu);
    m = m_new;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int g = 0; g < 16; ++g) {
        s[j][g] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][g], a.c, -mu));
        sum += s[j][g];
      }
    l = __builtin_fmaf(l, alpha, sum);
    if (DROP) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        uint32_t w[4];
        drop_words_rows(seed, (uint32_t)unit, r, k0 + 32 * j, lane, w);
#pragma unroll
        for (int g = 0; g < 16; ++g) s[j][g] = kept(w, g, a.thr) ? s[j][g] : 0.0f;
      }
    }
    if (__any(alpha != 1.0f)) {
#pragma unroll
      for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 16; ++g) acc[dt][g] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag<T> p = acc_frag<T>(s[j], t);
#pragma unroll
        for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = mma(TL::col(vt, 32 * j + 16 * t, dt, lane), p, acc[dt]);
      }
    if (more) store(buf ^ 1);
    __syncthreads();
  }
  l = half_sum(l);
  if (r >= a.R) return;
  const float inv = l > 0.0f ? (DROP ? a.keep_inv : 1.0f) / l : (l == 0.0f ? 0.0f : l);   // (a NaN sum stays one)
  if (hi == 0 && a.lse) a.lse[(int64_t)unit * a.R + r] = live && l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  store_col<T, DK>(row_ptr<T>(a, a.o, b, hk, r), a.D, hi, acc, live ? inv : 0.0f);
}

// ---- few rows: 32 packed rows; every wavefront walks keys of its own ----------------------------------------------------
// SPLIT: the four wavefronts of a workgroup (and `splits` workgroups) share one set of rows and divide its keys; their results
// are joined in the LDS (and by k_attn_join).  Otherwise every wavefront has rows of its own (many short sequences).
// Keys go straight to the matrix operands; values pass through the wavefront's own LDS tile to be read by columns.
template <typename T, int DK, bool DROP, bool SPLIT>
__global__ __launch_bounds__(256) void k_attn_fwd_few(Args a) {
  constexpr int W = lds_width(DK);
  typedef Tile<T, W> TL;
  constexpr int kTileBytes = 32 * TL::kRowBytes, kPer = 32 * TL::kChunks / 64;
  constexpr int kJoinBytes = SPLIT ? 32 * DK * 4 : 0, kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
  __shared__ __attribute__((aligned(16))) char lds[4][kWaveBytes];
  __shared__ float stat[4][2][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, col = lane & 31;
  const int jobs = a.B * a.Hk * a.n_tiles;
  int job, split = 0;
  if (SPLIT) {
    const int work = xcd_order((int)blockIdx.x, (int)gridDim.x);
    job = work / a.splits, split = work - job * a.splits;
  } else {
    job = (int)blockIdx.x * 4 + wave;
    if (job >= jobs) return;       // (no workgroup barrier below in this form)
  }
  const int unit = job / a.n_tiles, tile = job - unit * a.n_tiles;
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int r = tile * 32 + col, qi = row_query(a, r);
  const bool live = r < a.R && qi < n.q;
  const int lim = live ? row_limit(a, n, qi) : 0;
  const int q_first = row_query(a, tile * 32), q_last = min(row_query(a, min(tile * 32 + 31, a.R - 1)), n.q - 1);
  const int kall = q_first < n.q ? row_limit(a, n, q_last) : 0;
  const int t_lo = SPLIT ? split * a.tiles_per_split + wave : 0, t_step = SPLIT ? 4 : 1;
  const int kend = SPLIT ? min(kall, (split + 1) * a.tiles_per_split * 32) : kall;

  Frag<T> qf[DK / 16];
  load_row_frags<T, DK>(live ? row_ptr<T>(a, a.q, b, hk, r) : nullptr, live, a.D, hi, qf);
  f32x16 acc[DK / 32] = {};
  float m = -INFINITY, l = 0.0f;
  const uint64_t seed = DROP ? drop_seed(a) : 0;
  char* vt = lds[wave];
  for (int k0 = t_lo * 32; k0 < kend; k0 += 32 * t_step) {
    const int key = k0 + col;
    const bool key_ok = key < n.k && (!a.key_mask || a.key_mask[b * a.mask_sb + key] != 0);
    const uint32_t vis = (uint32_t)__ballot(key_ok);
    Frag<T> kf[DK / 16];
    load_row_frags<T, DK>(key_ok ? key_ptr<T>(a.k, b, hk, key) : nullptr, key_ok, a.D, hi, kf);
    u32x4v stage[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = lane + 64 * i, row = id / TL::kChunks, d = ((id % TL::kChunks) ^ TL::swz(row)) * TL::kChunkEl;
      const bool ok = ((vis >> row) & 1) && d < a.D;
      stage[i] = ok ? *reinterpret_cast<const u32x4v*>(key_ptr<T>(a.v, b, hk, k0 + row) + d) : u32x4v{0, 0, 0, 0};
    }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < kPer; ++i) *reinterpret_cast<u32x4v*>(vt + (lane + 64 * i) * 16) = stage[i];
    wave_lds_fence();
    f32x16 s = {};
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) s = mma(kf[t], qf[t], s);
    float mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      const int o = 8 * (g >> 2) + 4 * hi + (g & 3);
      const bool see = k0 + o < lim && ((vis >> o) & 1);
      s[g] = see ? s[g] : -INFINITY;
      mx = fmaxf(mx, s[g]);
    }
    const float m_new = fmaxf(m, half_max(mx) * a.c), mu = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - mu);
    m = m_new;
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      s[g] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g], a.c, -mu));
      sum += s[g];
    }
    l = __builtin_fmaf(l, alpha, sum);
    if (DROP) {
      uint32_t w[4];
      drop_words_rows(seed, (uint32_t)unit, r, k0, lane, w);
#pragma unroll
      for (int g = 0; g < 16; ++g) s[g] = kept(w, g, a.thr) ? s[g] : 0.0f;
    }
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 16; ++g) acc[dt][g] *= alpha;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> p = acc_frag<T>(s, t);
#pragma unroll
      for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = mma(TL::col(vt, 16 * t, dt, lane), p, acc[dt]);
    }
  }
  l = half_sum(l);
  if constexpr (!SPLIT) {
    if (r >= a.R) return;
    const float inv = l > 0.0f ? (DROP ? a.keep_inv : 1.0f) / l : (l == 0.0f ? 0.0f : l);
    if (hi == 0 && a.lse) a.lse[(int64_t)unit * a.R + r] = live && l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
    store_col<T, DK>(row_ptr<T>(a, a.o, b, hk, r), a.D, hi, acc, live ? inv : 0.0f);
  } else {
    // join the wavefronts: common maximum, then the sum of the rescaled parts in the fixed order 0..3
    if (hi == 0) stat[wave][0][col] = m;
    __syncthreads();
    const float mj = fmaxf(fmaxf(stat[0][0][col], stat[1][0][col]), fmaxf(stat[2][0][col], stat[3][0][col]));
    const float f = __builtin_amdgcn_exp2f(m - (mj == -INFINITY ? 0.0f : mj));
    if (hi == 0) stat[wave][1][col] = l * f;
    float* part = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = acc[dt][4 * g + c] * f;
        *reinterpret_cast<f32x4*>(part + col * DK + 32 * dt + 8 * g + 4 * hi) = v;
      }
    __syncthreads();
    for (int e = tid; e < 32 * (DK / 4); e += 256) {
      const int row = e / (DK / 4), d = (e - row * (DK / 4)) * 4, rr = tile * 32 + row;
      if (rr >= a.R || d >= a.D) continue;
      f32x4 v = {};
      float ls = 0.0f, mr = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w]) + row * DK + d);
        ls += stat[w][1][row];
        mr = fmaxf(mr, stat[w][0][row]);
      }
      if (a.splits > 1) {
        const int64_t units = (int64_t)a.B * a.Hk, at = ((int64_t)split * units + unit) * a.R + rr;
        *reinterpret_cast<f32x4*>(a.part + at * a.D + d) = v;
        if (d == 0) {
          float* st = a.part + (int64_t)a.splits * units * a.R * a.D + 2 * at;
          st[0] = mr, st[1] = ls;
        }
      } else {
        const bool lv = row_query(a, rr) < n.q;
        const float inv = lv ? (ls > 0.0f ? (DROP ? a.keep_inv : 1.0f) / ls : (ls == 0.0f ? 0.0f : ls)) : 0.0f;
        typedef typename Vec<T>::x4 V4;
        *reinterpret_cast<V4*>(row_ptr<T>(a, a.o, b, hk, rr) + d) = __builtin_convertvector(v * inv, V4);
        if (d == 0 && a.lse)
          a.lse[(int64_t)unit * a.R + rr] = lv && ls != 0.0f ? (mr + __builtin_amdgcn_logf(ls)) * kLn2 : -INFINITY;
      }
    }
  }
}

// joins the parts of a split call: thread = (row, four elements)
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(Args a, float gain) {
  const int per = a.D / 4;
  const int64_t units = (int64_t)a.B * a.Hk, rows = units * a.R, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= rows * per) return;
  const int64_t row = e / per;
  const int d = (int)(e - row * per) * 4, unit = (int)(row / a.R), r = (int)(row - (int64_t)unit * a.R);
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const float* st = a.part + (int64_t)a.splits * rows * a.D;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, st[2 * (s * rows + row)]);
  const float mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  f32x4 v = {};
  for (int s = 0; s < a.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(st[2 * (s * rows + row)] - mu);
    l += f * st[2 * (s * rows + row) + 1];
    v += f * *reinterpret_cast<const f32x4*>(a.part + (s * rows + row) * a.D + d);
  }
  const float inv = l > 0.0f ? gain / l : (l == 0.0f ? 0.0f : l);
  typedef typename Vec<T>::x4 V4;
  *reinterpret_cast<V4*>(row_ptr<T>(a, a.o, b, hk, r) + d) = __builtin_convertvector(v * inv, V4);
  if (d == 0 && a.lse) a.lse[row] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

template <typename T, int DK, bool DROP>
int launch(const Args& a0, const FwdPlan& p, hipStream_t st) {
  Args a = a0;
  a.n_tiles = p.n_tiles, a.splits = p.splits, a.tiles_per_split = p.tiles_per_split;
  const int64_t units = (int64_t)a.B * a.Hk;
  if (p.kind == kManyRows) {
    hipLaunchKernelGGL((k_attn_fwd<T, DK, DROP>), dim3((unsigned)(units * p.n_tiles)), dim3(256), 0, st, a);
  } else if (p.kind == kFewRowsOwn) {
    hipLaunchKernelGGL((k_attn_fwd_few<T, DK, DROP, false>), dim3((unsigned)((units * p.n_tiles + 3) / 4)), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((k_attn_fwd_few<T, DK, DROP, true>), dim3((unsigned)(units * p.n_tiles * p.splits)), dim3(256), 0, st, a);
    if (p.splits > 1) {
      if (int e = launch_status()) return e;
      const int64_t n = units * a.R * (a.D / 4);
      hipLaunchKernelGGL((k_attn_join<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, DROP ? a.keep_inv : 1.0f);
    }
  }
  return launch_status();
}

template <typename T, int DK>
int launch_drop(const Args& a, const FwdPlan& p, hipStream_t st) {
  return a.thr ? launch<T, DK, true>(a, p, st) : launch<T, DK, false>(a, p, st);
}
template <typename T>
int launch_dim(const Args& a, const FwdPlan& p, hipStream_t st) {
  if (a.D <= 32) return launch_drop<T, 32>(a, p, st);
  if (a.D <= 64) return launch_drop<T, 64>(a, p, st);
  if (a.D <= 96) return launch_drop<T, 96>(a, p, st);
  return launch_drop<T, 128>(a, p, st);
}

}  // namespace
}  // namespace attn
}  // namespace pstl

using namespace pstl;
using namespace pstl::attn;

extern "C" size_t pstl_attention_work_floats(const pstl_attn* c) {
  Args a;
  if (attn_args(c, &a, kCheckShape) != PSTL_OK) return 0;
  const FwdPlan p = plan_forward(a, device_cus());
  return p.splits > 1 ? (size_t)p.splits * a.B * a.Hk * a.R * (a.D + 2) : 0;
}

extern "C" int pstl_attention(const pstl_attn* c, void* stream) {
  Args a;
  if (int e = attn_args(c, &a, kCheckForward)) return e;
  if ((int64_t)a.B * a.R == 0) return PSTL_OK;
  const FwdPlan p = plan_forward(a, device_cus());
  if (p.splits > 1 && !a.part) return PSTL_ERR_ARG;
  if ((int64_t)a.B * a.Hk * p.n_tiles * p.splits >= (1ll << 31)) return PSTL_ERR_SHAPE;
  switch (c->dtype) {
    case PSTL_F32: return launch_dim<float>(a, p, as_stream(stream));
    case PSTL_BF16: return launch_dim<__bf16>(a, p, as_stream(stream));
    default: return launch_dim<_Float16>(a, p, as_stream(stream));
  }
}
