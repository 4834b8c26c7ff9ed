// attention_kernels.hip -- softmax attention, forward: O = softmax(scale Q K^T) V over padded, ragged, grouped-head batches.
//
//   S_rj = scale q_r . k_j,  j < limit(r) and not hidden;   P = exp(S - lse_r),  lse_r = log sum_j exp(S_rj);   O = (m P / keep) V
// One pass over the keys with the running maximum and sum (32 bits); a row that sees no key gives zeros and lse = -inf: its sum is 0
// and its result is selected, not multiplied, away (an infinity that other rows of its tile see has come into it as 0 x inf).
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
// The scores of the NEXT 32 keys are formed (matrix pipe) beside the exponentials of the present ones (vector pipe).  16-bit types:
// fragments of keys are read from the LDS a step before their product, so that a tile of keys is used up one tile ahead of its
// values.
// The maximum that the exponents are taken against moves only when a score exceeds it by more than 2^8: P is then at most 256
// in 32 bits, the sums stay exact to their rounding, and the accumulators are hardly ever rescaled.
// Bound by the matrix pipe beside the exponentials of two wavefronts per SIMD (busy 53 and 52 % at 8192 tokens).  bf16, causal, 16/4
// heads of 128: 8192 tokens 306 us = 900 TF under the profiler and 278 us a pass without it, 990 TF of the 1239 that a large product
// reaches here; 4 x 2048 tokens 102 us = 670 TF (its 1024 workgroups are two rounds, in which the matrix pipe is busy 42 % and the
// vector pipe 46 %).  16-bit heads over 96 wide without dropout spill 7 registers, 32 bytes of scratch a lane: 40 MB written where
// output and lse are 34.  When these were tried the kernel took 280 and 94 us: 64 rows per wavefront at one wavefront per SIMD: 461 and 150 us;
// tiles through registers instead of copies: 458 and 107 us; copies asked for behind the products: 330 and 102 us.  float32,
// 4 x 2048: 727 us, 69 GF = 95 of 153 TF.
template <typename T, int DK, bool DROP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DK > 64 ? 1 : 2) void k_attn_fwd(Args a) {
  constexpr int W = lds_width(DK), BN = block_keys<T>(), NS = BN / 32;
  typedef RowPipe<T, W, BN> Pipe;
  typedef Tile<T, W> TL;
  __shared__ __attribute__((aligned(16))) char lds_k[2][Pipe::kTileBytes], lds_v[2][Pipe::kTileBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
  const Work wk = causal_order((int)blockIdx.x, a.n_tiles, a.B * a.Hk, a.cus_per_xcd);
  const int unit = wk.unit, base = wk.tile * 128;
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int r0 = base + wave * 32, r = r0 + col, qi = row_query(a, r);
  const bool live = r < a.R && qi < n.q;
  const int lim = live ? row_limit(a, n, qi) : 0;
  Frag<T> qf[DK / 16];
  load_row_frags<T, DK>(live ? row_ptr<T>(a, a.q, b, hk, r) : nullptr, live, a.D, hi, qf);
  // keys that some row of the workgroup sees; keys that every live row of the wavefront sees
  const int q_first = row_query(a, base), q_last = min(row_query(a, min(base + 127, a.R - 1)), n.q - 1);
  const int kend = q_first < n.q ? row_limit(a, n, q_last) : 0;
  const int q_wave = row_query(a, r0), all_see = a.causal ? max(min(q_wave + n.k - n.q + 1, n.k), 0) : n.k;

  f32x16 acc[DK / 32] = {};
  float m = -INFINITY, l = 0.0f;
  const uint64_t seed = DROP ? drop_seed(a) : 0;

  const Pipe kp(key_ptr<T>(a.k, b, hk, 0), a.k.sl, a.Lk, a.D, tid), vp(key_ptr<T>(a.v, b, hk, 0), a.v.sl, a.Lk, a.D, tid);
  KeyMask<BN> km(a, b, n.k, lane);
  if (a.D < W) kp.clear(lds_k[0]), kp.clear(lds_k[1]), vp.clear(lds_v[0]), vp.clear(lds_v[1]);
  constexpr bool kAhead = NS == 2 && !(DROP && DK == 128);      // (the draws need the registers there)
  Frag<T> kf[kAhead ? DK / 16 : 1];      // the fragments of the next scores
  auto read_keys = [&](const char* kt, int j) {
#pragma unroll
    for (int t = 0; t < (kAhead ? DK / 16 : 0); ++t) kf[t] = TL::row(kt, 32 * j + col, t, hi);
  };
  f32x16 s = {};
  if (kend > 0) {
    kp.issue(0, lds_k[0]);
    copies_done();
    __syncthreads();
    vp.issue(0, lds_v[0]);
    km.fetch(0);
    if (BN < kend) kp.issue(BN, lds_k[1]);
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) s = mma(TL::row(lds_k[0], col, t, hi), qf[t], s);
    read_keys(lds_k[0], 1);
  }
  int buf = 0;
  for (int k0 = 0; k0 < kend; k0 += BN, buf ^= 1) {
    copies_done();         // V of this tile, K of the next
    const uint64_t visible = km.bits(k0);
    if (k0 + BN > n.k || a.key_mask) vp.hide(lds_v[buf], visible);
    __syncthreads();
    if (k0 + BN < kend) vp.issue(k0 + BN, lds_v[buf ^ 1]), km.fetch(k0 + BN);
    // (without kAhead the second half of this tile's keys is still to be read: their buffer is filled again behind that)
    if (kAhead || NS == 1) {
      if (k0 + 2 * BN < kend) kp.issue(k0 + 2 * BN, lds_k[buf]);
    }
    const char *vt = lds_v[buf], *kt = lds_k[buf ^ 1];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      Frag<T> vf[DK / 32];      // the first half of the values' fragments (both do not fit the registers at DK = 128)
      if (kAhead) {
#pragma unroll
        for (int dt = 0; dt < DK / 32; ++dt) vf[dt] = TL::col(vt, 32 * j, dt, lane);
      }
      if (k0 + BN > all_see || a.key_mask) {
        asm volatile("");      // (a branch, not a select per score)
        const uint32_t see = seen_bits<false>((uint32_t)(visible >> (32 * j)), min(max(lim - k0 - 32 * j, 0), 32), lane) >> (4 * hi);
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = (see >> (8 * (x >> 2) + (x & 3))) & 1 ? s[x] : -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int x = 1; x < 16; ++x) mx = fmaxf(mx, s[x]);
      mx *= a.c;
      if (__any(mx > m + 8.0f)) {
        const float to = fmaxf(m, half_max(mx)), alpha = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.0f : to));
        m = to;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[dt][x] *= alpha;
      }
      // (behind the last tile: scores of whatever the buffer holds, never looked at)
      f32x16 next = {};
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) {
        if constexpr (kAhead)
          next = mma(kf[t], qf[t], next);
        else
          next = mma(j + 1 < NS ? TL::row(lds_k[buf], 32 * (j + 1) + col, t, hi) : TL::row(kt, col, t, hi), qf[t], next);
      }
      read_keys(kt, j);
      const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], a.c, -mu));
        l += s[x];
      }
      if (DROP) {
        uint32_t w[4];
        drop_words_rows(seed, (uint32_t)unit, r, k0 + 32 * j, lane, w);
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = kept(w, x, a.thr) ? s[x] : 0.0f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag<T> p = acc_frag<T>(s, t);
#pragma unroll
        for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = mma(kAhead && t == 0 ? vf[dt] : TL::col(vt, 32 * j + 16 * t, dt, lane), p, acc[dt]);
      }
      s = next;
      if (!kAhead && NS == 2 && j == 0) {
        __syncthreads();
        if (k0 + 2 * BN < kend) kp.issue(k0 + 2 * BN, lds_k[buf]);
      }
    }
  }
  l = half_sum(l);
  if (r >= a.R) return;
  const bool on = live && l != 0.0f;
  const float inv = !on ? 0.0f : l > 0.0f ? (DROP ? a.keep_inv : 1.0f) / l : l;      // (a NaN sum stays one)
  if (hi == 0 && a.lse) a.lse[(int64_t)unit * a.R + r] = on ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  if (!on) {
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt) acc[dt] = f32x16{};
  }
  store_col<T, DK>(row_ptr<T>(a, a.o, b, hk, r), a.D, hi, acc, inv);
}

// ---- at most 32 keys: one wavefront per 32 packed rows, or per pair of units of at most 16 rows and keys -----------------
// Bound by memory: q, k and v pass through the wavefront's LDS tiles and o leaves the same way, so that neighbouring lanes touch
// neighbouring 16 bytes (fragments read straight from global memory touch 32 rows per instruction: 82 us at 4096 x 12 tokens, 8
// heads of 32, float32; like this, one unit per wavefront, 59 us; with two units of at most 16 to a wavefront and the values in
// the keys' place 57 us, 201 MB = 3.5 TB/s).
template <typename T, int DK, bool DROP, bool PAIR>
__global__ __launch_bounds__(64 * (short_waves<T, DK>(2))) void k_attn_fwd_short(Args a) {
  constexpr int NW = short_waves<T, DK>(2);
  typedef Rows32<T, DK> RW;
  constexpr int kTileBytes = 32 * RW::TL::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[NW][2][kTileBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = lane >> 5, col = lane & 31;
  const int units = a.B * a.Hk, groups = PAIR ? (units + 1) / 2 : units;
  const int job = (int)blockIdx.x * NW + wave;
  if (job >= groups * a.n_tiles) return;       // (no workgroup barrier below)
  const int group = job / a.n_tiles, tile = job - group * a.n_tiles, u0 = PAIR ? 2 * group : group;
  char *kt = lds[wave][0], *qt = lds[wave][1];      // keys, then values; queries, then results
  // (loads are bounded by the tensors, not by the lengths and masks, so that they do not wait for those)
  RW kr, vr, qr;
  auto key_at = [&](const Mat& m) {
    return [&, m](int row) -> const T* {
      const Slot s = slot_of<PAIR>(a, u0, units, row);
      return s.ok && s.at < a.Lk ? key_ptr<T>(m, s.b, s.hk, s.at) : nullptr;
    };
  };
  auto row_at = [&](const Mat& m) {
    return [&, m](int row) -> T* {
      const Slot s = slot_of<PAIR>(a, u0, units, row);
      const int r = tile * 32 + s.at;
      return s.ok && r < a.R ? row_ptr<T>(a, m, s.b, s.hk, r) : nullptr;
    };
  };
  kr.load(key_at(a.k), a.D, lane);
  qr.load(row_at(a.q), a.D, lane);
  vr.load(key_at(a.v), a.D, lane);
  const Slot me = slot_of<PAIR>(a, u0, units, col);
  const Lens n = lens_lane(a, me.b);
  const int r = tile * 32 + me.at, qi = row_query(a, r);
  const bool key_on = me.ok && me.at < n.k && (!a.key_mask || a.key_mask[me.b * a.mask_sb + me.at] != 0);
  const bool live = me.ok && r < a.R && qi < n.q;
  const uint32_t keys_on = (uint32_t)__ballot(key_on), rows_on = (uint32_t)__ballot(live);
  const uint32_t see = seen_bits<PAIR>(keys_on, live ? row_limit(a, n, qi) : 0, lane) >> (4 * hi);
  kr.put(kt, keys_on, lane);
  qr.put(qt, rows_on, lane);
  wave_lds_fence();
  f32x16 s = row_product<T, DK>(kt, qt, lane);
  wave_lds_fence();
  vr.put(kt, keys_on, lane);
  float mx = -INFINITY;
#pragma unroll
  for (int g = 0; g < 16; ++g) {
    s[g] = (see >> (8 * (g >> 2) + (g & 3))) & 1 ? s[g] : -INFINITY;
    mx = fmaxf(mx, s[g]);
  }
  const float m = half_max(mx) * a.c, mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
#pragma unroll
  for (int g = 0; g < 16; ++g) {
    s[g] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g], a.c, -mu));
    l += s[g];
  }
  l = half_sum(l);
  if (DROP) {
    uint32_t w[4];
    drop_words_rows<PAIR>(drop_seed(a), (uint32_t)me.unit, r, 0, lane, w);
#pragma unroll
    for (int g = 0; g < 16; ++g) s[g] = kept(w, g, a.thr) ? s[g] : 0.0f;
  }
  f32x16 acc[DK / 32] = {};
  wave_lds_fence();
  contract<T, DK, PAIR>(acc, kt, s, lane);
  const bool on = live && l != 0.0f;
  const float inv = l > 0.0f ? (DROP ? a.keep_inv : 1.0f) / l : l;      // (a NaN sum stays one)
  if (hi == 0 && a.lse && me.ok && r < a.R)
    a.lse[(int64_t)me.unit * a.R + r] = on ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  wave_lds_fence();
  RW::from_acc(qt, col, hi, acc, inv, on);
  wave_lds_fence();
  RW::store(qt, row_at(a.o), a.D, lane);
}

// ---- few rows, many keys: 32 packed rows; every wavefront walks keys of its own ------------------------------------------
// The four wavefronts of a workgroup (and `splits` workgroups) share one set of rows and divide its keys; their results are
// joined in the LDS (and by k_attn_join).  Bound by reading the keys and values once: tiles of 32 keys are fetched a tile ahead
// into registers, 16 bytes per lane along the rows, and pass through the wavefront's own LDS tiles.  4 x up to 32768 keys, 16 / 2
// heads of 128, fp16, 117 MB: 30 us = 3.9 TB/s, and 4 us for the join (two tiles ahead: no gain; one query on 300 keys: 8.6 us,
// latency).
template <typename T, int DK, bool DROP>
__global__ __launch_bounds__(256) void k_attn_fwd_few(Args a) {
  typedef Rows32<T, DK> RW;
  typedef typename RW::TL TL;
  constexpr int kTileBytes = 32 * TL::kRowBytes;
  constexpr int kJoinBytes = 32 * DK * 4, kWaveBytes = 2 * kTileBytes > kJoinBytes ? 2 * kTileBytes : kJoinBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];       // 4 x kWaveBytes
  __shared__ float stat[4][2][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, col = lane & 31;
  // (in the grid's order: a sequence's parts go to all XCDs, so that short sequences leave none of them idle)
  const int job = (int)blockIdx.x / a.splits, split = (int)blockIdx.x - job * a.splits;
  const int unit = job / a.n_tiles, tile = job - unit * a.n_tiles;
  const int b = unit / a.Hk, hk = unit - b * a.Hk;
  const Lens n = lens_of(a, b);
  const int r = tile * 32 + col, qi = row_query(a, r);
  const bool live = r < a.R && qi < n.q;
  const int lim = live ? row_limit(a, n, qi) : 0;
  const int q_first = row_query(a, tile * 32), q_last = min(row_query(a, min(tile * 32 + 31, a.R - 1)), n.q - 1);
  const int kall = q_first < n.q ? row_limit(a, n, q_last) : 0;
  const int k_lo = (split * a.tiles_per_split + wave) * 32, kend = min(kall, (split + 1) * a.tiles_per_split * 32);

  Frag<T> qf[DK / 16];
  load_row_frags<T, DK>(live ? row_ptr<T>(a, a.q, b, hk, r) : nullptr, live, a.D, hi, qf);
  f32x16 acc[DK / 32] = {};
  float m = -INFINITY, l = 0.0f;
  const uint64_t seed = DROP ? drop_seed(a) : 0;
  char *kt = lds + wave * kWaveBytes, *vt = kt + kTileBytes;
  RW kr, vr;
  uint32_t vis = 0;
  auto fetch = [&](int k0) {
    auto at = [&](const Mat& mt) {
      return [&, mt](int row) -> const T* { return k0 + row < n.k ? key_ptr<T>(mt, b, hk, k0 + row) : nullptr; };
    };
    kr.load(at(a.k), a.D, lane);
    vr.load(at(a.v), a.D, lane);
    vis = (uint32_t)__ballot(k0 + col < n.k && (!a.key_mask || a.key_mask[b * a.mask_sb + k0 + col] != 0));
  };
  if (k_lo < kend) fetch(k_lo);
  for (int k0 = k_lo; k0 < kend; k0 += 128) {
    wave_lds_fence();
    kr.put(kt, vis, lane);
    vr.put(vt, vis, lane);
    const uint32_t see = seen_bits<false>(vis, min(max(lim - k0, 0), 32), lane) >> (4 * hi);
    if (k0 + 128 < kend) fetch(k0 + 128);
    wave_lds_fence();
    f32x16 s = {};
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) s = mma(TL::row(kt, col, t, hi), qf[t], s);
    float mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      s[g] = (see >> (8 * (g >> 2) + (g & 3))) & 1 ? s[g] : -INFINITY;
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
    contract<T, DK, false>(acc, vt, s, lane);
  }
  l = half_sum(l);
  // join the wavefronts: common maximum, then the sum of the rescaled parts in the fixed order 0..3
  if (hi == 0) stat[wave][0][col] = m;
  __syncthreads();
  const float mj = fmaxf(fmaxf(stat[0][0][col], stat[1][0][col]), fmaxf(stat[2][0][col], stat[3][0][col]));
  const float f = __builtin_amdgcn_exp2f(m - (mj == -INFINITY ? 0.0f : mj));
  if (hi == 0) stat[wave][1][col] = l * f;
  float* part = reinterpret_cast<float*>(lds + wave * kWaveBytes);
  const int rows = min(a.R - tile * 32, 32);
  if (col < rows) {
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = acc[dt][4 * g + c] * f;
        *reinterpret_cast<f32x4*>(part + col * DK + 32 * dt + 8 * g + 4 * hi) = v;
      }
  }
  __syncthreads();
  for (int e = tid; e < rows * (DK / 4); e += 256) {
    const int row = e / (DK / 4), d = (e - row * (DK / 4)) * 4, rr = tile * 32 + row;
    if (d >= a.D) continue;
    f32x4 v = {};
    float ls = 0.0f, mr = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * kWaveBytes) + row * DK + d);
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
      const bool lv = row_query(a, rr) < n.q && ls != 0.0f;
      const float inv = ls > 0.0f ? (DROP ? a.keep_inv : 1.0f) / ls : ls;
      typedef typename Vec<T>::x4 V4;
      v = lv ? v * inv : f32x4{};
      *reinterpret_cast<V4*>(row_ptr<T>(a, a.o, b, hk, rr) + d) = __builtin_convertvector(v, V4);
      if (d == 0 && a.lse) a.lse[(int64_t)unit * a.R + rr] = lv ? (mr + __builtin_amdgcn_logf(ls)) * kLn2 : -INFINITY;
    }
  }
}

// joins the parts of a split call: one workgroup per row; eight groups of 32 lanes (four elements each) sum every eighth part,
// and the groups' sums are joined in order.  Latency: 64 rows of 32 parts take 4 us (one lane a row and element: 36 us).
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(Args a, float gain) {
  __shared__ float weight[kMaxSplits], red[8];
  __shared__ f32x4 sums[8][32];
  const int tid = threadIdx.x, lane = tid & 31, g = tid >> 5;
  const int64_t rows = (int64_t)a.B * a.Hk * a.R, row = blockIdx.x;
  const int unit = (int)(row / a.R), r = (int)(row - (int64_t)unit * a.R), b = unit / a.Hk, hk = unit - b * a.Hk;
  const float* st = a.part + (int64_t)a.splits * rows * a.D;
  float m = -INFINITY;
  for (int s = tid; s < a.splits; s += 256) {
    const float x = st[2 * (s * rows + row)];
    weight[s] = x;
    m = fmaxf(m, x);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) red[g] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
  const float mu = m == -INFINITY ? 0.0f : m;
  __syncthreads();
  float l = 0.0f;
  for (int s = tid; s < a.splits; s += 256) {
    const float f = __builtin_amdgcn_exp2f(weight[s] - mu);
    weight[s] = f;
    l += f * st[2 * (s * rows + row) + 1];
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) l += __shfl_xor(l, o);
  if (lane == 0) red[g] = l;
  __syncthreads();
  f32x4 v = {};
  const int d = 4 * lane;
  if (d < a.D) {
#pragma unroll 4
    for (int s = g; s < a.splits; s += 8) v += weight[s] * *reinterpret_cast<const f32x4*>(a.part + (s * rows + row) * a.D + d);
  }
  sums[g][lane] = v;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) l += red[i];
  if (g == 0 && d < a.D) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += sums[i][lane];
    const float inv = l > 0.0f ? gain / l : l;
    typedef typename Vec<T>::x4 V4;
    v = l != 0.0f ? v * inv : f32x4{};      // (a row that sees nothing)
    *reinterpret_cast<V4*>(row_ptr<T>(a, a.o, b, hk, r) + d) = __builtin_convertvector(v, V4);
  }
  if (tid == 0 && a.lse) a.lse[row] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

template <typename T, int DK, bool DROP>
int launch(const Args& a0, const FwdPlan& p, hipStream_t st) {
  Args a = a0;
  a.n_tiles = p.n_tiles, a.splits = p.splits, a.tiles_per_split = p.tiles_per_split, a.cus_per_xcd = p.cus_per_xcd;
  const int64_t units = (int64_t)a.B * a.Hk;
  if (p.kind == kManyRows) {
    if (!grid_fits(units * p.n_tiles, 256)) return PSTL_ERR_SHAPE;
    hipLaunchKernelGGL((k_attn_fwd<T, DK, DROP>), dim3((unsigned)(units * p.n_tiles)), dim3(256), 0, st, a);
  } else if (p.kind == kShort || p.kind == kShortPairs) {
    constexpr int NW = short_waves<T, DK>(2);
    const bool pair = p.kind == kShortPairs;
    const int64_t jobs = (pair ? (units + 1) / 2 : units) * p.n_tiles;
    if (!grid_fits((jobs + NW - 1) / NW, 64 * NW)) return PSTL_ERR_SHAPE;
    const dim3 grid((unsigned)((jobs + NW - 1) / NW)), block(64 * NW);
    if (pair)
      hipLaunchKernelGGL((k_attn_fwd_short<T, DK, DROP, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((k_attn_fwd_short<T, DK, DROP, false>), grid, block, 0, st, a);
  } else {
    constexpr int kTile2 = 2 * 32 * lds_width(DK) * (int)sizeof(T), kJoin = 32 * DK * 4, kBytes = 4 * (kTile2 > kJoin ? kTile2 : kJoin);
    if (!grid_fits(units * p.n_tiles * p.splits, 256) || (p.splits > 1 && !grid_fits(units * a.R, 256))) return PSTL_ERR_SHAPE;
    if (int e = allow_lds<k_attn_fwd_few<T, DK, DROP>>(kBytes)) return e;
    hipLaunchKernelGGL((k_attn_fwd_few<T, DK, DROP>), dim3((unsigned)(units * p.n_tiles * p.splits)), dim3(256), kBytes, st, a);
    if (p.splits > 1) {
      if (int e = launch_status()) return e;
      hipLaunchKernelGGL((k_attn_join<T>), dim3((unsigned)(units * a.R)), dim3(256), 0, st, a, DROP ? a.keep_inv : 1.0f);
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
  const FwdPlan p = plan_forward(a, c->dtype == PSTL_F32, device_cus());
  return p.splits > 1 ? (size_t)p.splits * a.B * a.Hk * a.R * (a.D + 2) : 0;
}

extern "C" int pstl_attention(const pstl_attn* c, void* stream) {
  Args a;
  if (int e = attn_args(c, &a, kCheckForward)) return e;
  if ((int64_t)a.B * a.R == 0) return PSTL_OK;
  const FwdPlan p = plan_forward(a, c->dtype == PSTL_F32, device_cus());
  if (p.splits > 1 && !a.part) return PSTL_ERR_ARG;
  switch (c->dtype) {
    case PSTL_F32: return launch_dim<float>(a, p, as_stream(stream));
    case PSTL_BF16: return launch_dim<__bf16>(a, p, as_stream(stream));
    default: return launch_dim<_Float16>(a, p, as_stream(stream));
  }
}
