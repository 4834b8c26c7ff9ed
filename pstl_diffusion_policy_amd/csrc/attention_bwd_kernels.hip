// attention_bwd_kernels.hip -- softmax attention, backward: the probabilities are formed again from q, k and the saved lse.
//
//   P = exp(S - lse);  delta_r = sum_d dO_rd O_rd;  dV = (m P / keep)^T dO;  dP = dO V^T;  dS = P o (m dP / keep - delta)
//   dQ = scale dS K;   dK = scale dS^T Q
// Two launches without atomics, so that a result does not depend on the order in which workgroups finish: k_attn_bwd_q (a lane
// holds one row: S^T, dP^T, dQ^T; it also leaves delta) and k_attn_bwd_kv or _kv_duo (a lane holds one key: S, dP, dK^T, dV^T;
// packed rows make the sum over the heads that share a key head part of the same accumulator).  S and dP are formed in both: seven products
// instead of five, against a second pass over dQ in memory.  Sequences of at most 32 keys have one launch (k_attn_bwd_short).
// Arithmetic: P and dS are rounded to the inputs' type as operands of dV, dQ and dK; all sums are 32-bit.  Above 32 keys delta is
// formed from the rounded O: the sum over d averages its roundings, and the unrounded O would be another tensor to keep for the
// backward pass.  Error of dQ and dK in bf16, of their size: 0.0025 at 4 x 2048 causal tokens, heads of 128 (their own rounding 0.0017,
// dS 0.0017, delta 0.0007), 0.0026 at 182 (delta 0.0010: the first rows of a causal call average few values).
#include "attn_host.hpp"

namespace pstl {
namespace attn {
namespace {

template <typename T>
constexpr int block_len() {
  return sizeof(T) == 2 ? 64 : 32;
}
template <typename T, int DK>
constexpr int waves_per_simd_q() {
  return sizeof(T) == 2 ? 2 : DK <= 32 ? 2 : 1;
}
template <typename T, int DK>
constexpr int waves_per_simd_kv() {
  return sizeof(T) == 2 || DK <= 32 ? 2 : 1;
}

// sum over d of the product of two rows (row fragments; both lane halves)
template <typename T, int DK>
__device__ inline float row_dot(const Frag<T> (&x)[DK / 16], const Frag<T> (&y)[DK / 16]) {
  float s = 0.0f;
#pragma unroll
  for (int t = 0; t < DK / 16; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf((float)x[t][j], (float)y[t][j], s);
  return half_sum(s);
}

// ---- dQ: 128 packed rows per workgroup, 32 per wavefront ---------------------------------------------------------------
// Q, dO and dQ stay in registers, keys and values pass through the LDS as in the forward kernel; 16-bit types run two wavefronts
// per SIMD, so that one's matrix products stand beside the other's exponentials (one per SIMD with the scores formed a step ahead:
// 212 us).  4 x 2048 causal, 16/4 heads of 128, bf16: 138 us, 103 GF = 750 TF; the matrix pipe is busy 44 % of the time and the
// vector pipe 35 %, the rest is LDS latency and the barrier of a tile.  (Copies asked for behind the products instead of right
// behind the barrier: no difference.)
template <typename T, int DK, bool DROP>
__global__ __launch_bounds__(256, (waves_per_simd_q<T, DK>())) void k_attn_bwd_q(Args a) {
  constexpr int W = lds_width(DK), BN = block_len<T>(), NS = BN / 32;
  typedef Tile<T, W> TL;
  typedef RowPipe<T, W, BN> Pipe;
  __shared__ __attribute__((aligned(16))) char lds[2][2][Pipe::kTileBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
  const Work wk = causal_order((int)blockIdx.x, a.n_tiles, a.B * a.Hk, a.cus_per_xcd);
  const int unit = wk.unit, base = wk.tile * 128;
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int r0 = base + wave * 32, r = r0 + col;
  const int qi = row_query(a, r);
  const bool live = r < a.R && qi < n.q;
  const int lim = live ? row_limit(a, n, qi) : 0;
  const int q_first = row_query(a, base), q_last = min(row_query(a, min(base + 127, a.R - 1)), n.q - 1);
  const int kend = q_first < n.q ? row_limit(a, n, q_last) : 0;
  const int q_wave = row_query(a, r0);
  const int all_see = r0 + 32 > a.R || row_query(a, r0 + 31) >= n.q ? 0 : a.causal ? max(min(q_wave + n.k - n.q + 1, n.k), 0) : n.k;

  const Pipe kp(key_ptr<T>(a.k, b, hk, 0), a.k.sl, a.Lk, a.D, tid), vp(key_ptr<T>(a.v, b, hk, 0), a.v.sl, a.Lk, a.D, tid);
  KeyMask<BN> km(a, b, n.k, lane);
  if (a.D < W) kp.clear(lds[0][0]), kp.clear(lds[1][0]), vp.clear(lds[0][1]), vp.clear(lds[1][1]);
  if (kend > 0) km.fetch(0), kp.issue(0, lds[0][0]), vp.issue(0, lds[0][1]);
  Frag<T> qf[DK / 16], dof[DK / 16];
  load_row_frags<T, DK>(live ? row_ptr<T>(a, a.q, b, hk, r) : nullptr, live, a.D, hi, qf);
  load_row_frags<T, DK>(live ? row_ptr<T>(a, a.dout, b, hk, r) : nullptr, live, a.D, hi, dof);
  float delta, lse2;
  {
    Frag<T> of[DK / 16];
    load_row_frags<T, DK>(live ? row_ptr<T>(a, a.o, b, hk, r) : nullptr, live, a.D, hi, of);
    delta = row_dot<T, DK>(dof, of);
    lse2 = live ? a.lse[(int64_t)unit * a.R + r] * kLog2e : 0.0f;
    if (hi == 0 && r < a.R) a.delta[(int64_t)unit * a.R + r] = delta;
  }
  f32x16 acc[DK / 32] = {};
  const uint64_t seed = DROP ? drop_seed(a) : 0;
  int buf = 0;
  for (int k0 = 0; k0 < kend; k0 += BN, buf ^= 1) {
    copies_done();
    const uint64_t visible = km.bits(k0);
    if (k0 + BN > n.k || a.key_mask) kp.hide(lds[buf][0], visible);      // (dP of a hidden key is selected away)
    __syncthreads();
    if (k0 + BN < kend) km.fetch(k0 + BN), kp.issue(k0 + BN, lds[buf ^ 1][0]), vp.issue(k0 + BN, lds[buf ^ 1][1]);
    const char *kt = lds[buf][0], *vt = lds[buf][1];
    const bool masked = k0 + BN > all_see || a.key_mask;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) s = mma(TL::row(kt, 32 * j + col, t, hi), qf[t], s);
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) dp = mma(TL::row(vt, 32 * j + col, t, hi), dof[t], dp);
      uint32_t w[4];
      if (DROP) drop_words_rows(seed, (uint32_t)unit, r, k0 + 32 * j, lane, w);
#pragma unroll
      for (int g = 0; g < 16; ++g) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g], a.c, -lse2));
        float dpv = dp[g];
        if (DROP) dpv = kept(w, g, a.thr) ? dpv * a.keep_inv : 0.0f;
        s[g] = p * (dpv - delta);
      }
      if (masked) {
        asm volatile("");      // (a branch, not a select per score)
        const uint32_t see = seen_bits<false>((uint32_t)(visible >> (32 * j)), min(max(lim - k0 - 32 * j, 0), 32), lane) >> (4 * hi);
#pragma unroll
        for (int g = 0; g < 16; ++g) s[g] = (see >> (8 * (g >> 2) + (g & 3))) & 1 ? s[g] : 0.0f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag<T> ds = acc_frag<T>(s, t);
#pragma unroll
        for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = mma(TL::col(kt, 32 * j + 16 * t, dt, lane), ds, acc[dt]);
      }
    }
  }
  if (r >= a.R) return;
  if (!live || lse2 == -INFINITY) {      // (a row that sees nothing: selected away, as in the forward kernel)
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = f32x16{};
  }
  store_col<T, DK>(row_ptr<T>(a, a.dq, b, hk, r), a.D, hi, acc, a.scale);
}

// ---- dK, dV: 64 keys per workgroup --------------------------------------------------------------------------------------
// float32, and 16-bit types up to D = 64.
// Wavefronts 0, 1 take 32 keys each and the even 32-row steps, wavefronts 2, 3 the same keys and the odd steps; their sums are
// joined in the LDS at the end.  (128 keys per workgroup, all steps in every wavefront: half the workgroups, which a causal mask
// makes uneven.)
// 16-bit types: S and dP of a wavefront's NEXT step are formed (matrix pipe) beside the exponentials of the present one, so rows
// are copied two steps ahead into three buffers.  4 x 2048 causal, 16/4 heads of 64, bf16: 219 us with dQ (k_attn_bwd_kv_duo
// 226); heads of 128, float32: 2.18 ms with dQ, 241 GF = 110 of the 153 TF that a large float32 product reaches here.
template <typename T, int DK>
constexpr bool kv_ahead() {
  return sizeof(T) == 2;
}
template <typename T, int DK>
constexpr int kv_lds() {
  constexpr int tiles = (kv_ahead<T, DK>() ? 6 : 4) * 64 * lds_width(DK) * (int)sizeof(T), join = 2 * 32 * DK * 4;
  return tiles > join ? tiles : join;
}
template <typename T, int DK, bool DROP>
__global__ __launch_bounds__(256, (waves_per_simd_kv<T, DK>())) void k_attn_bwd_kv(Args a) {
  constexpr int W = lds_width(DK), BM = 64;
  constexpr bool kAhead = kv_ahead<T, DK>();
  constexpr int NB = kAhead ? 3 : 2;
  typedef Tile<T, W> TL;
  typedef PackedPipe<T, W, BM> Pipe;
  extern __shared__ __attribute__((aligned(16))) char lds[];      // [NB][2][kTileBytes]: Q and dO of NB steps
  __shared__ __attribute__((aligned(16))) float row_lse[NB][BM], row_delta[NB][BM];
  __shared__ __attribute__((aligned(16))) int row_lim[NB][BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
  const int kg = wave & 1, part = wave >> 1;
  const Work wk = causal_order((int)blockIdx.x, a.n_tiles, a.B * a.Hk, a.cus_per_xcd);
  const int unit = wk.unit, key0 = (a.n_tiles - 1 - wk.tile) * 64;      // (causal: the first keys are seen by the most rows)
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int key = key0 + kg * 32 + col;
  const bool live = key < n.k && (!a.key_mask || a.key_mask[b * a.mask_sb + key] != 0);
  const int r_end = key0 < n.k ? n.q * a.G : 0;
  const int r_begin = a.causal && r_end > 0 ? max(key0 - (n.k - n.q), 0) * a.G / BM * BM : 0;

  Frag<T> kf[DK / 16], vf[DK / 16];
  load_row_frags<T, DK>(live ? key_ptr<T>(a.k, b, hk, key) : nullptr, live, a.D, hi, kf);
  load_row_frags<T, DK>(live ? key_ptr<T>(a.v, b, hk, key) : nullptr, live, a.D, hi, vf);
  f32x16 dk[DK / 32] = {}, dv[DK / 32] = {};
  const uint64_t seed = DROP ? drop_seed(a) : 0;

  const Pipe qp(a, a.q, b, hk, r_end, tid), dop(a, a.dout, b, hk, r_end, tid);
  auto tile_at = [&](int buf, int which) { return lds + (2 * buf + which) * Pipe::kTileBytes; };
  if (a.D < W)
    for (int i = 0; i < 2 * NB; ++i) qp.clear(lds + i * Pipe::kTileBytes);
  float st_lse = 0.0f, st_delta = 0.0f;      // (asked for before the copies and looked at when those have arrived)
  auto issue = [&](int m0, int buf) {
    if (tid < BM) {
      const int64_t r = (int64_t)unit * a.R + min(m0 + tid, r_end - 1);
      st_lse = a.lse[r], st_delta = a.delta[r];
    }
    qp.issue(m0, tile_at(buf, 0));
    dop.issue(m0, tile_at(buf, 1));
  };
  auto arrive = [&](int m0, int buf) {      // (a barrier must follow)
    copies_done();
    if (m0 + BM > r_end) qp.hide(tile_at(buf, 0), m0), dop.hide(tile_at(buf, 1), m0);
    if (tid < BM) {
      const bool ok = m0 + tid < r_end;
      row_lse[buf][tid] = ok ? st_lse * kLog2e : 0.0f, row_delta[buf][tid] = ok ? st_delta : 0.0f;
      row_lim[buf][tid] = ok ? row_limit(a, n, row_query(a, m0 + tid)) : 0;
    }
  };
  const int o0 = 32 * part;
  f32x16 s = {}, dp = {};
  auto products = [&](int buf, f32x16& x, f32x16& y) {
    x = f32x16{}, y = f32x16{};
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) x = mma(TL::row(tile_at(buf, 0), o0 + col, t, hi), kf[t], x);
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) y = mma(TL::row(tile_at(buf, 1), o0 + col, t, hi), vf[t], y);
  };
  if (r_begin < r_end) {
    issue(r_begin, 0);
    if (kAhead) {
      arrive(r_begin, 0);
      __syncthreads();
      if (r_begin + BM < r_end) issue(r_begin + BM, 1);
      products(0, s, dp);
    }
  }
  int buf = 0;
  for (int m0 = r_begin; m0 < r_end; m0 += BM) {
    const int buf1 = buf + 1 == NB ? 0 : buf + 1, buf2 = buf1 + 1 == NB ? 0 : buf1 + 1;
    if (kAhead) {      // rows of the next step
      if (m0 + BM < r_end) arrive(m0 + BM, buf1);
      __syncthreads();
      if (m0 + 2 * BM < r_end) issue(m0 + 2 * BM, buf2);
    } else {
      arrive(m0, buf);
      __syncthreads();
      if (m0 + BM < r_end) issue(m0 + BM, buf1);
      products(buf, s, dp);
    }
    const char *qt = tile_at(buf, 0), *dot = tile_at(buf, 1);
    // rows see more keys the later they are: no masks when the step's first row sees the wavefront's last key
    const bool masked = m0 + BM > r_end || (a.causal && row_lim[buf][o0] < key0 + kg * 32 + 32);
    // (behind the last step: products of whatever the buffer holds, never looked at)
    f32x16 s1, dp1;
    if (kAhead) products(buf1, s1, dp1);
    uint32_t w[4];
    if (DROP) drop_words_keys(seed, (uint32_t)unit, m0 + o0, key, lane, w);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = o0 + 8 * q + 4 * hi;
      const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_lse[buf][o]), delta = *reinterpret_cast<const f32x4*>(&row_delta[buf][o]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int g = 4 * q + c;
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g], a.c, -lse[c]));
        const bool keep = !DROP || kept(w, g, a.thr);
        const float dpv = DROP ? (keep ? dp[g] * a.keep_inv : 0.0f) : dp[g];
        s[g] = keep ? p : 0.0f;
        dp[g] = p * (dpv - delta[c]);
      }
    }
    if (masked) {
      asm volatile("");      // (a branch, not a select per score)
#pragma unroll
      for (int g = 0; g < 16; ++g) {
        const bool see = key < row_lim[buf][o0 + 8 * (g >> 2) + 4 * hi + (g & 3)];
        s[g] = see ? s[g] : 0.0f, dp[g] = see ? dp[g] : 0.0f;
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> p = acc_frag<T>(s, t), ds = acc_frag<T>(dp, t);
#pragma unroll
      for (int dt = 0; dt < DK / 32; ++dt) {
        dv[dt] = mma(TL::col(dot, o0 + 16 * t, dt, lane), p, dv[dt]);
        dk[dt] = mma(TL::col(qt, o0 + 16 * t, dt, lane), ds, dk[dt]);
      }
    }
    if (kAhead) s = s1, dp = dp1;
    buf = buf1;
  }
  // the odd steps' sums into the even steps' wavefronts: (register, lane) by (register, lane)
  __syncthreads();
  float* x = reinterpret_cast<float*>(lds) + kg * (DK / 32) * 2048 + lane * 4;
  auto give = [&](const f32x16 (&v)[DK / 32]) {
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(x + dt * 1024 + q * 256) = f32x4{v[dt][4 * q], v[dt][4 * q + 1], v[dt][4 * q + 2], v[dt][4 * q + 3]};
  };
  auto take = [&](f32x16 (&v)[DK / 32]) {
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(x + dt * 1024 + q * 256);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[dt][4 * q + c] += y[c];
      }
  };
  if (part) give(dk);
  __syncthreads();
  if (!part) take(dk);
  __syncthreads();
  if (part) give(dv);
  __syncthreads();
  if (part) return;
  take(dv);
  if (key >= a.Lk) return;
  if (!live) {      // (a hidden key's column holds sums of no meaning, infinities among them: it is written as zeros)
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt) dk[dt] = f32x16{}, dv[dt] = f32x16{};
  }
  store_col<T, DK>(key_ptr<T>(a.dk, b, hk, key), a.D, hi, dk, a.scale);
  store_col<T, DK>(key_ptr<T>(a.dv, b, hk, key), a.D, hi, dv, DROP ? a.keep_inv : 1.0f);
}

// 16-bit types, D > 64: K, V, dK and dV of 32 keys take 192 registers per lane, which leaves one wavefront per SIMD.  Here eight
// wavefronts share them: 4 + w forms S, P and dV of 32 keys and every second 32-row step, and hands P (32 bits; the sign bit
// marks a dropped probability) through the LDS to w on the same SIMD, which forms dP, dS and dK.  The second kind passes its
// barrier between dP and dS, the first before S: one is in the matrix pipe while the other forms exponentials.  Copies are asked
// for behind the first product: 32 KB take 500 cycles to issue, which right behind the barrier nobody had anything to do in.
// 4 x 2048 causal, 16/4 heads of 128, bf16: 218 us, 137 GF = 630 TF (on the day of these trials 204 us: one wavefront per SIMD with all four: 241 us; both kinds
// forming S for themselves: 245 us; copies right behind the barrier: 219 us; columns of Q and dO read ahead of the exponentials:
// no gain).  At D <= 64 everything fits two wavefronts per SIMD in k_attn_bwd_kv, and the handing over only costs (219 -> 226 us).
template <typename T, int DK>
constexpr int kv_duo_lds() {
  return 6 * 64 * lds_width(DK) * (int)sizeof(T) + 2 * 4 * 4096;
}
template <typename T, int DK, bool DROP>
__global__ __launch_bounds__(512, 2) void k_attn_bwd_kv_duo(Args a) {
  constexpr int W = lds_width(DK), BM = 64;
  typedef Tile<T, W> TL;
  typedef PackedPipe<T, W, BM> Pipe;
  static_assert(4 * (DK / 32) * 4096 <= 6 * Pipe::kTileBytes, "the sums are joined in the tiles' place");
  extern __shared__ __attribute__((aligned(16))) char lds[];      // [3][2][kTileBytes]: Q and dO of three steps; [2][4][4096]: P
  __shared__ __attribute__((aligned(16))) float row_lse[3][BM], row_delta[3][BM];
  __shared__ __attribute__((aligned(16))) int row_lim[3][BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
  const int kg = wave & 1, part = (wave >> 1) & 1, first = wave >> 2;      // first: S, P, dV; else dP, dS, dK
  const Work wk = causal_order((int)blockIdx.x, a.n_tiles, a.B * a.Hk, a.cus_per_xcd);
  const int unit = wk.unit, key0 = (a.n_tiles - 1 - wk.tile) * 64;      // (causal: the first keys are seen by the most rows)
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int key = key0 + kg * 32 + col;
  const bool live = key < n.k && (!a.key_mask || a.key_mask[b * a.mask_sb + key] != 0);
  const int r_end = key0 < n.k ? n.q * a.G : 0;
  const int r_begin = a.causal && r_end > 0 ? max(key0 - (n.k - n.q), 0) * a.G / BM * BM : 0;

  Frag<T> kv[DK / 16];      // this key's K or V
  load_row_frags<T, DK>(live ? key_ptr<T>(first ? a.k : a.v, b, hk, key) : nullptr, live, a.D, hi, kv);
  f32x16 acc[DK / 32] = {};
  const uint64_t seed = DROP ? drop_seed(a) : 0;

  const Pipe pipe(a, first ? a.dout : a.q, b, hk, r_end, tid & 255);      // each half of the workgroup copies one of the two
  auto tile_at = [&](int buf, int which) { return lds + (2 * buf + which) * Pipe::kTileBytes; };
  char* const p_at = lds + 6 * Pipe::kTileBytes + (wave & 3) * 4096 + lane * 16;
  if (a.D < W)
    for (int i = 0; i < 3; ++i) pipe.clear(tile_at(i, first));
  float st_lse = 0.0f, st_delta = 0.0f;      // (asked for before the copies and looked at when those have arrived)
  auto issue = [&](int m0, int buf) {
    if (tid < BM) {
      const int64_t r = (int64_t)unit * a.R + min(m0 + tid, r_end - 1);
      st_lse = a.lse[r], st_delta = a.delta[r];
    }
    pipe.issue(m0, tile_at(buf, first));
  };
  const int o0 = 32 * part;
  // makes step m0 visible
  auto turn = [&](int m0, int buf) {
    if (m0 < r_end) {
      copies_done();
      if (m0 + BM > r_end) pipe.hide(tile_at(buf, first), m0);
      if (tid < BM) {
        const bool ok = m0 + tid < r_end;
        row_lse[buf][tid] = ok ? st_lse * kLog2e : 0.0f, row_delta[buf][tid] = ok ? st_delta : 0.0f;
        row_lim[buf][tid] = ok ? row_limit(a, n, row_query(a, m0 + tid)) : 0;
      }
    }
    __syncthreads();
  };
  if (r_begin < r_end) issue(r_begin, 0);
  if (!first) {
    turn(r_begin, 0);
    if (r_begin + BM < r_end) issue(r_begin + BM, 1);
  }
  int buf = 0, slot = 0;
  for (int m0 = r_begin; m0 < r_end; m0 += BM, slot ^= 4 * 4096) {
    const int next = buf == 2 ? 0 : buf + 1;
    if (first) turn(m0, buf);
    f32x4 stat[4];      // lse or delta
#pragma unroll
    for (int q = 0; q < 4; ++q) stat[q] = *reinterpret_cast<const f32x4*>((first ? row_lse[buf] : row_delta[buf]) + o0 + 8 * q + 4 * hi);
    f32x16 s = {};
    const char* rows = tile_at(buf, 1 - first);
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) s = mma(TL::row(rows, o0 + col, t, hi), kv[t], s);      // S or dP
    if (!first)
      turn(m0 + BM, next);
    else if (m0 + BM < r_end)
      issue(m0 + BM, next);
    // rows see more keys the later they are: no masks when the step's first row sees the wavefront's last key
    const bool masked = m0 + BM > r_end || (a.causal && row_lim[buf][o0] < key0 + kg * 32 + 32);
    uint32_t w[4];
    if (first) {
      if (DROP) drop_words_keys(seed, (uint32_t)unit, m0 + o0, key, lane, w);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int c = 0; c < 4; ++c) s[4 * q + c] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + c], a.c, -stat[q][c]));
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 p = *reinterpret_cast<const f32x4*>(p_at + slot + q * 1024);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x = p[c];
          const float dpv = DROP ? (__builtin_signbitf(x) ? 0.0f : s[4 * q + c] * a.keep_inv) : s[4 * q + c];
          s[4 * q + c] = (DROP ? __builtin_fabsf(x) : x) * (dpv - stat[q][c]);
        }
      }
      if (m0 + 2 * BM < r_end) issue(m0 + 2 * BM, next == 2 ? 0 : next + 1);
    }
    if (masked) {
      asm volatile("");      // (a branch, not a select per score; dS too: a row that does not see the key may hold anything)
#pragma unroll
      for (int g = 0; g < 16; ++g) s[g] = key < row_lim[buf][o0 + 8 * (g >> 2) + 4 * hi + (g & 3)] ? s[g] : 0.0f;
    }
    if (first) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 p;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int g = 4 * q + c;
          const bool keep = !DROP || kept(w, g, a.thr);
          p[c] = keep ? s[g] : -s[g];
          s[g] = keep ? s[g] : 0.0f;
        }
        *reinterpret_cast<f32x4*>(p_at + slot + q * 1024) = p;
      }
    }
    const char* other = tile_at(buf, first);      // dV += dO^T P, dK += Q^T dS
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> f = acc_frag<T>(s, t);
#pragma unroll
      for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = mma(TL::col(other, o0 + 16 * t, dt, lane), f, acc[dt]);
    }
    buf = next;
  }
  if (first) turn(r_end, 0);
  // the odd steps' sums into the even steps' wavefronts: (register, lane) by (register, lane)
  __syncthreads();
  float* x = reinterpret_cast<float*>(lds) + (2 * first + kg) * (DK / 32) * 1024 + lane * 4;
  if (part) {
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(x + dt * 1024 + q * 256) =
            f32x4{acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]};
  }
  __syncthreads();
  if (part || key >= a.Lk) return;
#pragma unroll
  for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(x + dt * 1024 + q * 256);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[dt][4 * q + c] += y[c];
    }
  if (!live) {      // (a hidden key's column holds sums of no meaning, infinities among them: it is written as zeros)
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = f32x16{};
  }
  store_col<T, DK>(key_ptr<T>(first ? a.dv : a.dk, b, hk, key), a.D, hi, acc, !first ? a.scale : DROP ? a.keep_inv : 1.0f);
}

// ---- at most 32 keys: one wavefront per (sequence, key head), or per pair of them, everything in one pass ------------------
// K and V stay in the LDS, rows come 32 at a time; delta is the row sum of P o m dP / keep, so that O is not read.  dK and dV need P
// and dS with a key per lane: 16-bit types form S and dP a second time in that layout; float32, whose products take sixteen times
// as long, turns P and dS through the LDS when there is one row tile (their tiles take the places of V and K): 2048 x 20 tokens,
// 8 heads of 32, float32, dropout: 112 us (formed twice: 128 us); 294 MB = 2.6 TB/s of 5.0, beside five products of 32 x 32 x 32
// per unit, 5.4 GF = 35 us at the float32 matrix rate, and the exponentials and draws of 16384 tiles.
// One wavefront walks ALL rows of its unit: few units with many rows (4096 queries of one sequence on 32 keys, 8 heads: 8
// wavefronts, 128 tiles one after another) leave most of the chip idle.
template <typename T, int DK>
constexpr int bwd_short_waves() {
  return DK <= 32 ? 2 : short_waves<T, DK>(4);
}
// ONE: at most 32 rows
template <typename T, int DK, bool DROP, bool PAIR, bool ONE>
__global__ __launch_bounds__(64 * (bwd_short_waves<T, DK>()), DK <= 64 ? 2 : 1) void k_attn_bwd_short(Args a) {
  constexpr int NW = bwd_short_waves<T, DK>();
  constexpr bool kTurn = sizeof(T) == 4 && ONE;
  typedef Rows32<T, DK> RW;
  constexpr int kTileBytes = 32 * RW::TL::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[NW][4][kTileBytes];
  __shared__ __attribute__((aligned(16))) float row_stat[NW][2][32];
  __shared__ __attribute__((aligned(16))) uint32_t row_see[NW][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = lane >> 5, col = lane & 31;
  const int units = a.B * a.Hk, u0 = ((int)blockIdx.x * NW + wave) * (PAIR ? 2 : 1);
  if (u0 >= units) return;       // (no workgroup barrier below)
  char *kt = lds[wave][0], *vt = lds[wave][1], *qt = lds[wave][2], *dot = lds[wave][3];
  auto key_at = [&](const Mat& m) {
    return [&, m](int row) -> T* {
      const Slot s = slot_of<PAIR>(a, u0, units, row);
      return s.ok && s.at < a.Lk ? key_ptr<T>(m, s.b, s.hk, s.at) : nullptr;
    };
  };
  RW kr, vr;
  kr.load(key_at(a.k), a.D, lane);
  vr.load(key_at(a.v), a.D, lane);
  const Slot me = slot_of<PAIR>(a, u0, units, col);
  const Lens n = lens_lane(a, me.b);
  const bool key_on = me.ok && me.at < n.k && (!a.key_mask || a.key_mask[me.b * a.mask_sb + me.at] != 0);
  const uint32_t keys_on = (uint32_t)__ballot(key_on);
  const uint64_t seed = DROP ? drop_seed(a) : 0;
  f32x16 dk[DK / 32] = {}, dv[DK / 32] = {};
  for (int m0 = 0; m0 < (ONE ? min(a.R, 1) : a.R); m0 += 32) {
    auto row_at = [&](const Mat& m) {
      return [&, m](int row) -> T* {
        const Slot s = slot_of<PAIR>(a, u0, units, row);
        return s.ok && m0 + s.at < a.R ? row_ptr<T>(a, m, s.b, s.hk, m0 + s.at) : nullptr;
      };
    };
    RW qr, dor;
    qr.load(row_at(a.q), a.D, lane);
    dor.load(row_at(a.dout), a.D, lane);
    const int r = m0 + me.at, qi = row_query(a, r);
    const uint32_t see = seen_bits<PAIR>(keys_on, me.ok && r < a.R ? row_limit(a, n, qi) : 0, lane);
    const bool live = see != 0;      // (a row that sees nothing is left out, as one behind the length is)
    const uint32_t rows_on = (uint32_t)__ballot(live);
    const float lse2 = live ? a.lse[(int64_t)me.unit * a.R + r] * kLog2e : 0.0f;
    wave_lds_fence();
    if (m0 == 0) {
      kr.put(kt, keys_on, lane);
      vr.put(vt, keys_on, lane);
    }
    qr.put(qt, rows_on, lane);
    dor.put(dot, rows_on, lane);
    wave_lds_fence();
    // rows in the lanes: delta, dQ
    f32x16 s = row_product<T, DK>(kt, qt, lane), dp = row_product<T, DK>(vt, dot, lane);
    uint32_t w[4];
    if (DROP) drop_words_rows<PAIR>(seed, (uint32_t)me.unit, r, 0, lane, w);
    float delta = 0.0f;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      const bool on = ((see >> (4 * hi)) >> (8 * (g >> 2) + (g & 3))) & 1;
      const float p = on ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[g], a.c, -lse2)) : 0.0f;
      float dpv = on ? dp[g] : 0.0f;
      if (DROP) dpv = kept(w, g, a.thr) ? dpv * a.keep_inv : 0.0f;
      delta = __builtin_fmaf(p, dpv, delta);
      s[g] = p, dp[g] = dpv;
    }
    delta = half_sum(delta);
    f32x16 dq[DK / 32] = {};
    if constexpr (kTurn) {
      f32x16 pk;      // m P
#pragma unroll
      for (int g = 0; g < 16; ++g) {
        pk[g] = !DROP || kept(w, g, a.thr) ? s[g] : 0.0f;
        s[g] = s[g] * (dp[g] - delta);
      }
      Turned::put(vt, pk, lane);
      contract<T, DK, PAIR>(dq, kt, s, lane);
      wave_lds_fence();
      Turned::put(kt, s, lane);
      contract<T, DK, PAIR>(dv, dot, Turned::frag(vt, 0, lane), Turned::frag(vt, 1, lane), lane);
      wave_lds_fence();
      contract<T, DK, PAIR>(dk, qt, Turned::frag(kt, 0, lane), Turned::frag(kt, 1, lane), lane);
    } else {
#pragma unroll
      for (int g = 0; g < 16; ++g) s[g] = s[g] * (dp[g] - delta);
      if (hi == 0) row_stat[wave][0][col] = lse2, row_stat[wave][1][col] = delta, row_see[wave][col] = see;
      contract<T, DK, PAIR>(dq, kt, s, lane);
      wave_lds_fence();
      // keys in the lanes: dK, dV
      s = row_product<T, DK>(qt, kt, lane), dp = row_product<T, DK>(dot, vt, lane);
      if (DROP) drop_words_keys<PAIR>(seed, (uint32_t)me.unit, m0, me.at, lane, w);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int o = 8 * q + 4 * hi;
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_stat[wave][0][o]), dl = *reinterpret_cast<const f32x4*>(&row_stat[wave][1][o]);
        const u32x4v sees = *reinterpret_cast<const u32x4v*>(&row_see[wave][o]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int g = 4 * q + c;
          const bool on = (sees[c] >> col) & 1;
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g], a.c, -lse[c]));
          const bool keep = !DROP || kept(w, g, a.thr);
          const float dpv = DROP ? (keep ? dp[g] * a.keep_inv : 0.0f) : dp[g];
          s[g] = on && keep ? p : 0.0f;
          dp[g] = on ? p * (dpv - dl[c]) : 0.0f;
        }
      }
      contract<T, DK, PAIR>(dv, dot, s, lane);
      contract<T, DK, PAIR>(dk, qt, dp, lane);
    }
    wave_lds_fence();
    RW::from_acc(qt, col, hi, dq, a.scale, live);
    wave_lds_fence();
    RW::store(qt, row_at(a.dq), a.D, lane);
  }
  wave_lds_fence();
  RW::from_acc(kt, col, hi, dk, a.scale, key_on);
  RW::from_acc(vt, col, hi, dv, DROP ? a.keep_inv : 1.0f, key_on);
  wave_lds_fence();
  RW::store(kt, key_at(a.dk), a.D, lane);
  RW::store(vt, key_at(a.dv), a.D, lane);
}

template <typename T, int DK, bool DROP>
int launch(const Args& a0, hipStream_t st) {
  Args a = a0;
  a.cus_per_xcd = device_cus() >= 8 ? device_cus() / 8 : 1;
  const int64_t units = (int64_t)a.B * a.Hk;
  if (a.Lk <= 32) {
    constexpr int NW = bwd_short_waves<T, DK>();
    const bool pair = in_pairs(a);
    const int64_t jobs = pair ? (units + 1) / 2 : units;
    if (!grid_fits((jobs + NW - 1) / NW, 64 * NW)) return PSTL_ERR_SHAPE;
    const dim3 grid((unsigned)((jobs + NW - 1) / NW)), block(64 * NW);
    if (pair)
      hipLaunchKernelGGL((k_attn_bwd_short<T, DK, DROP, true, true>), grid, block, 0, st, a);
    else if (a.R <= 32)
      hipLaunchKernelGGL((k_attn_bwd_short<T, DK, DROP, false, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((k_attn_bwd_short<T, DK, DROP, false, false>), grid, block, 0, st, a);
    return launch_status();
  }
  constexpr bool kDuo = sizeof(T) == 2 && DK > 64;
  if (!grid_fits(units * ceil_div(a.R, 128), 256) || !grid_fits(units * ceil_div(a.Lk, 64), kDuo ? 512 : 256)) return PSTL_ERR_SHAPE;
  if (a.R > 0) {
    a.n_tiles = ceil_div(a.R, 128);
    hipLaunchKernelGGL((k_attn_bwd_q<T, DK, DROP>), dim3((unsigned)(units * a.n_tiles)), dim3(256), 0, st, a);
    if (int e = launch_status()) return e;
  }
  a.n_tiles = ceil_div(a.Lk, 64);
  const dim3 grid((unsigned)(units * a.n_tiles));
  if constexpr (kDuo) {
    a.cus_per_xcd = 1 << 24;      // one workgroup per compute unit
    constexpr int kBytes = kv_duo_lds<T, DK>();
    if (int e = allow_lds<k_attn_bwd_kv_duo<T, DK, DROP>>(kBytes)) return e;
    hipLaunchKernelGGL((k_attn_bwd_kv_duo<T, DK, DROP>), grid, dim3(512), kBytes, st, a);
  } else {
    if (waves_per_simd_kv<T, DK>() == 1) a.cus_per_xcd = 1 << 24;
    constexpr int kBytes = kv_lds<T, DK>();
    if (int e = allow_lds<k_attn_bwd_kv<T, DK, DROP>>(kBytes)) return e;
    hipLaunchKernelGGL((k_attn_bwd_kv<T, DK, DROP>), grid, dim3(256), kBytes, st, a);
  }
  return launch_status();
}
template <typename T, int DK>
int launch_drop(const Args& a, hipStream_t st) {
  return a.thr ? launch<T, DK, true>(a, st) : launch<T, DK, false>(a, st);
}
template <typename T>
int launch_dim(const Args& a, hipStream_t st) {
  if (a.D <= 32) return launch_drop<T, 32>(a, st);
  if (a.D <= 64) return launch_drop<T, 64>(a, st);
  if (a.D <= 96) return launch_drop<T, 96>(a, st);
  return launch_drop<T, 128>(a, st);
}

}  // namespace
}  // namespace attn
}  // namespace pstl

using namespace pstl;
using namespace pstl::attn;

extern "C" size_t pstl_attention_backward_work_floats(const pstl_attn* c) {
  Args a;
  if (attn_args(c, &a, kCheckShape) != PSTL_OK) return 0;
  return (size_t)a.B * a.Hk * a.R + 1;
}

extern "C" int pstl_attention_backward(const pstl_attn* c, void* stream) {
  Args a;
  if (int e = attn_args(c, &a, kCheckBackward)) return e;
  if (a.B == 0 || (a.R == 0 && a.Lk == 0)) return PSTL_OK;
  switch (c->dtype) {
    case PSTL_F32: return launch_dim<float>(a, as_stream(stream));
    case PSTL_BF16: return launch_dim<__bf16>(a, as_stream(stream));
    default: return launch_dim<_Float16>(a, as_stream(stream));
  }
}
