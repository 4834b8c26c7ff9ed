// attn_core.hpp -- building blocks of the attention kernels: element types, 32 x 32 matrix tiles, the swizzled LDS tile, packed
// rows and the dropout decisions.
//
// Matrix tiles.  Every product is built from 32 x 32 accumulator tiles: lane l holds column l % 32, and register 4a + c (a, c in
// 0..3) row 8a + 4 (l / 32) + c.  An operand fragment ("Frag") is eight values of the contraction index per lane: row (first
// operand) or column (second operand) l % 32, slots 8 (l / 32) + j.  For 16-bit types one fragment pair is one
// v_mfma_f32_32x32x16; for float32 the same fragments are eight v_mfma_f32_32x32x2 (slot j of both lane halves at a time), so
// that both arithmetics share every layout.  A contraction over keys (or rows) pairs slots 0..3 with tile rows 4 (l / 32) + j and
// slots 4..7 with 8 + 4 (l / 32) + j - 4: exactly the registers 8t .. 8t + 7 of an accumulator tile, which therefore become the
// second operand of the next product without leaving the lane.
//
// Packed rows.  The G = Hq / Hk query heads that share a key head are rows of one matrix: row r = i G + g is query i of head
// hk G + g.  Keys and values are then read once for all G heads, and the gradients of shared heads are sums inside one
// accumulator, in a fixed order.
#pragma once
#include "pstl_common.hpp"
#include "rng.hpp"

namespace pstl {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  typedef f32x8 x8;
  typedef f32x4 x4;
};
template <>
struct Vec<__bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
};
template <>
struct Vec<_Float16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
};
template <typename T>
using Frag = typename Vec<T>::x8;

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

__device__ inline f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// registers 8t .. 8t + 7 of an accumulator tile as an operand fragment (rounded to T: to nearest even)
template <typename T>
__device__ inline Frag<T> acc_frag(const f32x16& s, int t) {
  f32x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = s[8 * t + j];
  return __builtin_convertvector(v, Frag<T>);
}

template <typename T>
__device__ inline Frag<T> zero_frag() {
  Frag<T> z;
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = (T)0.0f;
  return z;
}

// eight consecutive elements of global memory (16-byte aligned)
template <typename T>
__device__ inline Frag<T> load8(const T* p) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_bit_cast(Frag<T>, *reinterpret_cast<const u32x4v*>(p));
  } else {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// this lane's value and the other lane half's: v_permlane32_swap_b32 exchanges the upper half of one register with the lower half
// of another.  (The two operands are kept apart by an empty asm: with one value in both, the compiler names one register twice
// and nothing is exchanged.)
__device__ inline f32x2 both_halves(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x), v = u;
  asm("" : "+v"(v));
  const auto p = __builtin_amdgcn_permlane32_swap(u, v, false, false);
  return f32x2{__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1])};
}
__device__ inline float half_max(float x) {
  const f32x2 p = both_halves(x);
  return fmaxf(p[0], p[1]);
}
__device__ inline float half_sum(float x) {
  const f32x2 p = both_halves(x);
  return p[0] + p[1];
}

// ---- LDS tiles ----------------------------------------------------------------------------------------------------
// A tile of rows of W elements (a power of two) is stored row after row in 16-byte chunks; chunk c of row r sits at position
// c ^ swz(r).  Rows 0..15 then put the same chunk on different banks (row fragments), and the four rows x 64 bytes that half a
// wavefront takes in one transposing 16-bit read lie on 64 different ones (column fragments).
template <typename T, int W>
struct Tile {
  static constexpr int kChunkEl = 16 / (int)sizeof(T);
  static constexpr int kChunks = W / kChunkEl;
  static constexpr int kRowBytes = W * (int)sizeof(T);
  __device__ static inline int swz(int r) {
    if constexpr (kChunks == 4) return (r >> 2) & 3;
    if constexpr (kChunks == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  __device__ static inline int chunk_off(int r, int c) { return r * kRowBytes + ((c ^ swz(r)) << 4); }
  // row fragment: row `r`, elements 16 t + 8 hi + 0..7
  __device__ static inline Frag<T> row(const char* lds, int r, int t, int hi) {
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(Frag<T>, *reinterpret_cast<const u32x4v*>(lds + chunk_off(r, 2 * t + hi)));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(lds + chunk_off(r, 4 * t + 2 * hi));
      const f32x4 b = *reinterpret_cast<const f32x4*>(lds + chunk_off(r, 4 * t + 2 * hi + 1));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // column fragment: element 32 dt + l % 32, slots = rows r0 + 4 hi + 0..3 and r0 + 8 + 4 hi + 0..3   (r0 a multiple of 16).
  // 16-bit: ds_read_b64_tr_b16 hands lane i of a group of 16 the four rows' element i; lane i addresses row i / 4, elements
  // 4 (i % 4) .. + 3.
  __device__ static inline Frag<T> col(const char* lds, int r0, int dt, int lane) {
    const int hi = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      typedef s16x4 __attribute__((address_space(3))) * lds_p;
      const int i = lane & 15, d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
      const int r = r0 + 4 * hi + (i >> 2);
      const char* p0 = lds + chunk_off(r, d >> 3) + (d & 7) * 2;
      const char* p1 = lds + chunk_off(r + 8, d >> 3) + (d & 7) * 2;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p0);
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p1);
      return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int d = 32 * dt + (lane & 31);
      Frag<T> v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = r0 + 4 * hi + (j & 3) + 8 * (j >> 2);
        v[j] = *reinterpret_cast<const float*>(lds + chunk_off(r, d >> 2) + (d & 3) * 4);
      }
      return v;
    }
  }
};

// orders the LDS traffic of ONE wavefront (its instructions reach the LDS in order; this keeps the compiler to that order)
__device__ inline void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- dropout of probabilities ----------------------------------------------------------------------------------------
// The decision for (row r, key j) of unit u = b Hk + hk is byte j % 4 of word r % 4 of philox(j / 4, r / 4, u, 'ATTD') under the
// seed: a function of the element alone, whatever the kernel, tile or layout.  One draw serves a 4 x 4 patch, i.e. 16 elements
// of 8 bits (16 bits per element would double the draws, and at D = 64 those of 8 bits already cost a third: 4 x 2048 causal, 16/4
// heads, bf16, takes 85 us forward instead of 59 and 268 backward instead of 219); the probability is therefore a multiple of
// 1/256, and the scale is the inverse of the REALISED keep probability.  A quad of lanes shares the four patches its 16 registers touch: lane i of the quad draws patch i, then the
// words move across the quad by DPP -- one draw per lane and 32 x 32 tile in either layout.
constexpr uint32_t kDropTag = 0x41545444u;

template <int A>
__device__ inline uint32_t quad_bcast(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, A * 0x55, 0xf, 0xf, true);
}

// lane = row r (any), registers = keys key0 + 8a + 4 hi + c (key0 a multiple of 32): W[a] = the four decision bytes of register
// group a, key c in byte c.  PAIR: the tile holds two units of 16 keys (groups 0, 1 and 2, 3), `unit` and r are the lane's own.
template <bool PAIR = false>
__device__ inline void drop_words_rows(uint64_t seed, uint32_t unit, int r, int key0, int lane, uint32_t (&W)[4]) {
  const uint32_t i = lane & 3, hi = lane >> 5;
  const u32x4 w = philox4x32(u32x4{(uint32_t)(key0 >> 2) + 2 * (PAIR ? i & 1 : i) + hi, (uint32_t)(r >> 2), unit, kDropTag}, (uint32_t)seed,
                             (uint32_t)(seed >> 32));
  // W[a] = word i of lane a: a 4 x 4 transposition inside the quad
#define PSTL_TR(A)                                                                                                \
  {                                                                                                               \
    const uint32_t x0 = quad_bcast<A>(w.x), x1 = quad_bcast<A>(w.y), x2 = quad_bcast<A>(w.z), x3 = quad_bcast<A>(w.w); \
    const uint32_t lo = (i & 1) ? x1 : x0, up = (i & 1) ? x3 : x2;                                                \
    W[A] = (i & 2) ? up : lo;                                                                                     \
  }
  PSTL_TR(0) PSTL_TR(1) PSTL_TR(2) PSTL_TR(3)
#undef PSTL_TR
}

// lane = key, registers = rows row0 + 8a + 4 hi + c (row0 a multiple of 32): byte c of W[a] = the decision of row c of group a
template <bool PAIR = false>
__device__ inline void drop_words_keys(uint64_t seed, uint32_t unit, int row0, int key, int lane, uint32_t (&W)[4]) {
  const uint32_t i = lane & 3, hi = lane >> 5, sh = 8 * i;
  const u32x4 w = philox4x32(u32x4{(uint32_t)(key >> 2), (uint32_t)(row0 >> 2) + 2 * (PAIR ? i & 1 : i) + hi, unit, kDropTag}, (uint32_t)seed,
                             (uint32_t)(seed >> 32));
#define PSTL_TR(A)                                                                                          \
  W[A] = ((quad_bcast<A>(w.x) >> sh) & 255u) | (((quad_bcast<A>(w.y) >> sh) & 255u) << 8) |                 \
         (((quad_bcast<A>(w.z) >> sh) & 255u) << 16) | (((quad_bcast<A>(w.w) >> sh) & 255u) << 24);
  PSTL_TR(0) PSTL_TR(1) PSTL_TR(2) PSTL_TR(3)
#undef PSTL_TR
}
__device__ inline bool kept(const uint32_t (&W)[4], int reg, uint32_t thr) {
  return ((W[reg >> 2] >> (8 * (reg & 3))) & 255u) >= thr;
}

// ---- arguments -------------------------------------------------------------------------------------------------------
struct Mat {      // (B, L, H, D), elements of a row consecutive; strides in elements
  char* p;
  int64_t sb, sl, sh;
};
struct Args {
  Mat q, k, v, o, dout, dq, dk, dv;
  float* lse;                 // (B, Hk, R): natural logarithm, -inf for a row that sees no key
  float* delta;               // (B, Hk, R): sum_d dO O                      (backward's work)
  const uint8_t* key_mask;    // (B, Lk), 0 = hidden, or null
  int64_t mask_sb;
  const int *q_lens, *k_lens; // (B) or null
  float* part;                // (splits, units, rows, D) then (splits, units, rows, 2): partial results of a split call
  const uint64_t* seed_dev;
  uint64_t seed;
  int B, Lq, Lk, Hk, G, D, R, causal;
  uint32_t g_magic;           // r / G = umulhi(r, g_magic) for G > 1  (R G < 2^32, checked by the host)
  uint32_t hk_magic;          // unit / Hk likewise, where a kernel divides lane by lane (short sequences in pairs)
  float scale, c;             // c = scale log2(e)
  uint32_t thr;               // a probability is dropped when its byte is below thr
  float keep_inv;             // 256 / (256 - thr)
  int n_tiles, splits, tiles_per_split, cus_per_xcd;
};

__device__ inline int row_query(const Args& a, int r) { return a.G == 1 ? r : (int)__umulhi((uint32_t)r, a.g_magic); }
__device__ inline uint64_t drop_seed(const Args& a) { return a.seed_dev ? uniform_u64(a.seed_dev) : a.seed; }

// lengths of sequence b, clamped to the tensors
struct Lens {
  int q, k;
};
__device__ inline Lens lens_of(const Args& a, int b) {
  Lens n;
  n.q = a.q_lens ? min(max(__builtin_amdgcn_readfirstlane(a.q_lens[b]), 0), a.Lq) : a.Lq;
  n.k = a.k_lens ? min(max(__builtin_amdgcn_readfirstlane(a.k_lens[b]), 0), a.Lk) : a.Lk;
  return n;
}
// keys [0, limit) are what query i sees (before the key mask); causal masks are aligned to the sequences' ends
__device__ inline int row_limit(const Args& a, Lens n, int i) {
  if (i >= n.q) return 0;
  if (!a.causal) return n.k;
  return min(max(i + n.k - n.q + 1, 0), n.k);
}
template <typename T>
__device__ inline T* row_ptr(const Args& a, const Mat& m, int b, int hk, int r) {
  const int i = row_query(a, r), g = r - i * a.G;
  return reinterpret_cast<T*>(m.p) + b * m.sb + i * m.sl + (int64_t)(hk * a.G + g) * m.sh;
}
template <typename T>
__device__ inline T* key_ptr(const Mat& m, int b, int hk, int j) {
  return reinterpret_cast<T*>(m.p) + b * m.sb + j * m.sl + hk * m.sh;
}

// workgroups are dealt to the 8 XCDs in turn: gives every XCD a consecutive share of [0, n), so that the workgroups that read the
// same keys share one L2
__device__ inline int xcd_order(int x, int n) {
  const int q = n >> 3, rem = n & 7, xcd = x & 7;
  return xcd * q + min(xcd, rem) + (x >> 3);
}

// Order of the workgroups of a causal launch.  All tiles of a unit stay on one XCD (or on 8 / units of them); inside an XCD the
// longest come first, and every second round of `round` tiles runs backwards: with two workgroups on a compute unit at once
// (round = compute units of an XCD) they are a long and a short one; with one (round past the grid) the next free unit takes the
// longest that is left.  Where the units do not divide the XCDs evenly: xcd_order, longest first.
struct Work {
  int unit, tile;
};
__device__ inline Work causal_order(int x, int n_tiles, int units, int round_len) {
  const int total = n_tiles * units, xcd = x & 7, q = x >> 3;
  int share = 0;                      // XCDs that share a unit's tiles
  if (units % 8 == 0) share = 1;
  else if (8 % units == 0 && n_tiles % (8 / units) == 0) share = 8 / units;
  if (share == 0) {
    const int w = xcd_order(x, total), unit = w / n_tiles;
    return Work{unit, n_tiles - 1 - (w - unit * n_tiles)};
  }
  const int per = total >> 3, round = q / round_len, i = q - round * round_len, width = min(round_len, per - round * round_len);
  const int pos = round * round_len + ((round & 1) ? width - 1 - i : i);
  const int here = share > 1 ? 1 : units >> 3, u = pos % here;      // units of this XCD
  return share > 1 ? Work{xcd / share, n_tiles - 1 - (pos * share + xcd % share)} : Work{xcd * here + u, n_tiles - 1 - pos / here};
}

// ---- tiles of keys and values, copied to the LDS without passing through registers ----------------------------------------
// 256 threads copy BN rows with global_load_lds_dwordx4: lane l of a wavefront writes 16 bytes at the wavefront's LDS address +
// 16 l, so the swizzle is a permutation of the chunks that the lanes fetch.  The copies are inline asm because the compiler would
// wait for them before any LDS read; copies_done() is the wait.  Rows past the tensor repeat its last row; rows that the mask or
// the lengths hide are overwritten by zeros after their arrival where a product contracts over them (a hidden NaN times a zero
// probability is NaN).
__device__ inline void copy16(const void* g, uint32_t lds_wave) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds_wave) : "memory", "m0");
}
__device__ inline void copy16(const void* base, uint32_t offset, uint32_t lds_wave) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds_wave) : "memory", "m0");
}
__device__ inline void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ inline uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
template <typename T>
__device__ inline T* uniform_ptr(T* p) {      // (readfirstlane gives a SIGNED word: each half through an unsigned one)
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<T*>(((uint64_t)hi << 32) | lo);
}

template <typename T, int W, int BN>
struct RowPipe {      // one tensor's rows (keys) of one unit
  typedef Tile<T, W> TL;
  static constexpr int kTileBytes = BN * TL::kRowBytes, kPer = BN * TL::kChunks / 256, kRowStep = 256 / TL::kChunks;
  const char* base;
  int64_t stride;      // bytes
  int rows, D, tid;    // rows of the tensor
  bool near;           // a tile's rows lie within 2^31 bytes
  __device__ RowPipe(const T* first, int64_t stride_el, int rows_, int D_, int tid_)
      : base(uniform_ptr(reinterpret_cast<const char*>(first))), stride(stride_el * (int)sizeof(T)), rows(rows_), D(D_), tid(tid_) {
    near = stride >= 0 && stride < (1ll << 31) / BN;
  }
  __device__ inline int row(int i) const { return tid / TL::kChunks + i * kRowStep; }
  __device__ inline int chunk(int i) const { return (tid % TL::kChunks) ^ TL::swz(row(i)); }
  // chunks past D never arrive: they are zeroed once
  __device__ inline void clear(char* tile) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (chunk(i) * TL::kChunkEl >= D) *reinterpret_cast<u32x4v*>(tile + (tid + 256 * i) * 16) = u32x4v{0, 0, 0, 0};
  }
  __device__ inline void issue(int k0, const char* tile) const {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(tile) + (tid >> 6) * 1024);
    if (near && k0 + BN <= rows) {
      const char* at = base + k0 * stride;
      const uint32_t off = (uint32_t)(tid / TL::kChunks) * (uint32_t)stride;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (chunk(i) * TL::kChunkEl < D) copy16(at + i * kRowStep * stride, off + chunk(i) * 16, to + i * 4096);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (chunk(i) * TL::kChunkEl < D) copy16(base + min(k0 + row(i), rows - 1) * stride + chunk(i) * 16, to + i * 4096);
    }
  }
  __device__ inline void hide(char* tile, uint64_t visible) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (!((visible >> row(i)) & 1)) *reinterpret_cast<u32x4v*>(tile + (tid + 256 * i) * 16) = u32x4v{0, 0, 0, 0};
  }
};
template <typename T, int W, int BM>
struct PackedPipe {      // one tensor's packed rows [0, end) of one unit
  typedef Tile<T, W> TL;
  static constexpr int kTileBytes = BM * TL::kRowBytes, kPer = BM * TL::kChunks / 256, kRowStep = 256 / TL::kChunks;
  const Args& a;
  const char* base;
  int64_t sl, sh;      // bytes
  int end, tid;
  uint32_t off;        // of this thread's first row in a tile
  bool near;           // a tile is a fixed pattern within 2^31 bytes
  __device__ PackedPipe(const Args& a_, const Mat& m, int b, int hk, int end_, int tid_) : a(a_), end(end_), tid(tid_) {
    base = uniform_ptr(m.p + (b * m.sb + (int64_t)(hk * a.G) * m.sh) * (int)sizeof(T));
    sl = m.sl * (int)sizeof(T), sh = m.sh * (int)sizeof(T);
    near = kRowStep % a.G == 0 && sl >= 0 && sh >= 0 && sl < (1ll << 30) / BM && sh < (1ll << 30) / BM;
    const int i = row_query(a, tid / TL::kChunks), g = tid / TL::kChunks - i * a.G;
    off = near ? (uint32_t)i * (uint32_t)sl + (uint32_t)g * (uint32_t)sh : 0;
  }
  __device__ inline int row(int i) const { return tid / TL::kChunks + i * kRowStep; }
  __device__ inline int chunk(int i) const { return (tid % TL::kChunks) ^ TL::swz(row(i)); }
  __device__ inline void clear(char* tile) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (chunk(i) * TL::kChunkEl >= a.D) *reinterpret_cast<u32x4v*>(tile + (tid + 256 * i) * 16) = u32x4v{0, 0, 0, 0};
  }
  __device__ inline void issue(int m0, const char* tile) const {      // m0: a multiple of BM
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(tile) + (tid >> 6) * 1024);
    if (near && m0 + BM <= end) {
      const char* at = base + row_query(a, m0) * sl;
      const int64_t step = (uint32_t)row_query(a, kRowStep) * sl;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (chunk(i) * TL::kChunkEl < a.D) copy16(at + i * step, off + chunk(i) * 16, to + i * 4096);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (chunk(i) * TL::kChunkEl < a.D) {
          const int r = min(m0 + row(i), end - 1), q = row_query(a, r);
          copy16(base + q * sl + (r - q * a.G) * sh + chunk(i) * 16, to + i * 4096);
        }
    }
  }
  __device__ inline void hide(char* tile, int m0) const {      // rows past the end: zeros
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (m0 + row(i) >= end) *reinterpret_cast<u32x4v*>(tile + (tid + 256 * i) * 16) = u32x4v{0, 0, 0, 0};
  }
};
// which keys of a tile are visible to anyone, as bits; the mask's bytes are fetched a tile ahead
template <int BN>
struct KeyMask {
  const uint8_t* mask;
  int n_k, last, lane;
  uint8_t next;
  __device__ KeyMask(const Args& a, int b, int n_k_, int lane_)
      : mask(a.key_mask ? a.key_mask + b * a.mask_sb : nullptr), n_k(n_k_), last(a.Lk - 1), lane(lane_), next(1) {}
  __device__ inline void fetch(int k0) {
    if (mask) next = mask[min(k0 + lane, last)];
  }
  __device__ inline uint64_t bits(int k0) const {
    const uint64_t all = BN == 64 ? ~0ull : (1ull << BN) - 1;
    if (mask) return __ballot(lane < BN && k0 + lane < n_k && next != 0);
    return k0 + BN > n_k ? (n_k > k0 ? (1ull << (n_k - k0)) - 1 : 0) : all;
  }
};

// row fragments of one packed row straight from global memory; zeros past D and for rows that are not there
template <typename T, int DK>
__device__ inline void load_row_frags(const T* p, bool ok, int D, int hi, Frag<T> (&f)[DK / 16]) {
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) {
    const int d = 16 * t + 8 * hi;
    f[t] = (ok && d < D) ? load8<T>(p + d) : zero_frag<T>();
  }
}

// stores an accumulator column (lane = row / key; registers = elements 32 dt + 8a + 4 hi + c) times `scale`
template <typename T, int DK>
__device__ inline void store_col(T* p, int D, int hi, const f32x16 (&acc)[DK / 32], float scale) {
  typedef typename Vec<T>::x4 V4;
#pragma unroll
  for (int dt = 0; dt < DK / 32; ++dt) {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * dt + 8 * a + 4 * hi;
      f32x4 v;
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = acc[dt][4 * a + c] * scale;
      if (d < D) *reinterpret_cast<V4*>(p + d) = __builtin_convertvector(v, V4);
    }
  }
}

constexpr int lds_width(int dk) { return dk <= 32 ? 32 : dk <= 64 ? 64 : 128; }

// ---- short sequences: 32 packed rows and 32 keys, one wavefront ---------------------------------------------------------
// PAIR: two units (sequence, key head) of at most 16 rows and 16 keys share a wavefront: rows and keys 0..15 are the first's,
// 16..31 the second's.  A score between the two is masked away, and their sums never meet: the contraction over the first
// sixteen slots belongs to the first unit, the other sixteen to the second, each with an accumulator of its own (0 * NaN is NaN,
// and one unit's NaN must not reach its neighbour).
struct Slot {        // what a row of the tile stands for
  int unit, b, hk, at;
  bool ok;
};
template <bool PAIR>
__device__ inline Slot slot_of(const Args& a, int first_unit, int units, int row) {
  Slot s;
  s.unit = PAIR ? first_unit + (row >> 4) : first_unit;
  s.at = PAIR ? row & 15 : row;
  s.ok = s.unit < units;
  const int u = s.ok ? s.unit : first_unit;
  s.b = PAIR ? (a.Hk == 1 ? u : (int)__umulhi((uint32_t)u, a.hk_magic)) : u / a.Hk;
  s.hk = u - s.b * a.Hk;
  return s;
}
__device__ inline Lens lens_lane(const Args& a, int b) {
  Lens n;
  n.q = a.q_lens ? min(max(a.q_lens[b], 0), a.Lq) : a.Lq;
  n.k = a.k_lens ? min(max(a.k_lens[b], 0), a.Lk) : a.Lk;
  return n;
}
// 32 rows of global memory to / from an LDS tile, 16 bytes per lane, neighbouring lanes on neighbouring chunks
template <typename T, int DK>
struct Rows32 {
  typedef Tile<T, lds_width(DK)> TL;
  static constexpr int kPer = 32 * TL::kChunks / 64;
  u32x4v v[kPer];
  template <typename F>
  __device__ inline void load(F ptr, int D, int lane) {      // ptr(row) -> the row's first element, or null
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = lane + 64 * i, row = id / TL::kChunks, d = ((id % TL::kChunks) ^ TL::swz(row)) * TL::kChunkEl;
      const T* p = ptr(row);
      v[i] = p && d < D ? *reinterpret_cast<const u32x4v*>(p + d) : u32x4v{0, 0, 0, 0};
    }
  }
  __device__ inline void put(char* tile, uint32_t rows_on, int lane) const {      // rows that are off: zeros
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = lane + 64 * i, row = id / TL::kChunks;
      *reinterpret_cast<u32x4v*>(tile + id * 16) = (rows_on >> row) & 1 ? v[i] : u32x4v{0, 0, 0, 0};
    }
  }
  template <typename F>
  __device__ static inline void store(const char* tile, F ptr, int D, int lane) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = lane + 64 * i, row = id / TL::kChunks, d = ((id % TL::kChunks) ^ TL::swz(row)) * TL::kChunkEl;
      T* p = ptr(row);
      if (p && d < D) *reinterpret_cast<u32x4v*>(p + d) = *reinterpret_cast<const u32x4v*>(tile + id * 16);
    }
  }
  // an accumulator column (lane = row) into the tile's row
  __device__ static inline void from_acc(char* tile, int row, int hi, const f32x16 (&acc)[DK / 32], float scale, bool on) {
    typedef typename Vec<T>::x4 V4;
#pragma unroll
    for (int dt = 0; dt < DK / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 x;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = on ? acc[dt][4 * g + c] * scale : 0.0f;
        const int d = 32 * dt + 8 * g + 4 * hi;
        *reinterpret_cast<V4*>(tile + TL::chunk_off(row, d / TL::kChunkEl) + (d % TL::kChunkEl) * (int)sizeof(T)) =
            __builtin_convertvector(x, V4);
      }
  }
};
// sum over the tile's 32 slots of  A(slot) x f(slot):  acc[dt] += columns of `tile` times the fragments f0 (slots 0..15), f1; PAIR:
// the lane's half
template <typename T, int DK, bool PAIR>
__device__ inline void contract(f32x16 (&acc)[DK / 32], const char* tile, const Frag<T>& f0, const Frag<T>& f1, int lane) {
  typedef Tile<T, lds_width(DK)> TL;
  const bool second = (lane & 16) != 0;
#pragma unroll
  for (int dt = 0; dt < DK / 32; ++dt) {
    if constexpr (PAIR) {
      const f32x16 x0 = mma(TL::col(tile, 0, dt, lane), f0, acc[dt]), x1 = mma(TL::col(tile, 16, dt, lane), f1, acc[dt]);
#pragma unroll
      for (int g = 0; g < 16; ++g) acc[dt][g] = second ? x1[g] : x0[g];
    } else {
      acc[dt] = mma(TL::col(tile, 0, dt, lane), f0, acc[dt]);
      acc[dt] = mma(TL::col(tile, 16, dt, lane), f1, acc[dt]);
    }
  }
}
template <typename T, int DK, bool PAIR>
__device__ inline void contract(f32x16 (&acc)[DK / 32], const char* tile, const f32x16& s, int lane) {
  contract<T, DK, PAIR>(acc, tile, acc_frag<T>(s, 0), acc_frag<T>(s, 1), lane);
}
// Float tile T[key][row] of 32 x 32 from an accumulator whose lanes are rows and registers keys; its row fragments then are the
// contraction's operand for lanes that are keys (slots: rows)
struct Turned {
  typedef Tile<float, 32> TL;
  __device__ static inline void put(char* tile, const f32x16& s, int lane) {
    const int hi = lane >> 5, row = lane & 31;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      const int key = 8 * (g >> 2) + 4 * hi + (g & 3);
      *reinterpret_cast<float*>(tile + TL::chunk_off(key, row >> 2) + (row & 3) * 4) = s[g];
    }
  }
  // slots 0..3: rows 16 t + 4 hi + 0..3, slots 4..7: rows 16 t + 8 + 4 hi + 0..3 -- the order of Tile::col
  __device__ static inline f32x8 frag(const char* tile, int t, int lane) {
    const int hi = lane >> 5, key = lane & 31;
    const f32x4 a = *reinterpret_cast<const f32x4*>(tile + TL::chunk_off(key, 4 * t + hi));
    const f32x4 b = *reinterpret_cast<const f32x4*>(tile + TL::chunk_off(key, 4 * t + 2 + hi));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};
// the tile's product over the element index: result(row i of x, lane = row of y)
template <typename T, int DK>
__device__ inline f32x16 row_product(const char* x, const char* y, int lane) {
  typedef Tile<T, lds_width(DK)> TL;
  f32x16 s = {};
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) s = mma(TL::row(x, lane & 31, t, lane >> 5), TL::row(y, lane & 31, t, lane >> 5), s);
  return s;
}
// the keys of the tile that this lane's row sees, as bits (lim: its first `lim` keys)
template <bool PAIR>
__device__ inline uint32_t seen_bits(uint32_t keys_on, int lim, int lane) {
  if constexpr (PAIR) {
    const uint32_t own = (1u << min(lim, 16)) - 1u;
    return keys_on & (own << (lane & 16));
  } else {
    return keys_on & (lim >= 32 ? ~0u : (1u << lim) - 1u);
  }
}
template <typename T, int DK>
constexpr int short_waves(int tiles) {      // wavefronts (each with its own tiles) per workgroup
  return tiles * 32 * lds_width(DK) * (int)sizeof(T) <= 16384 ? 4 : tiles * 32 * lds_width(DK) * (int)sizeof(T) <= 32768 ? 2 : 1;
}

}  // namespace attn
}  // namespace pstl
