// What the kernels of differential attention share: the staged tiles, their
// fragments, the per-key masks and the weight of the second map.
//
//   S_t = scale q_t k_t^T + bias  (t = 1, 2),  P_t = softmax over the keys
//   out = (P_1 - lambda P_2) v,  lambda_h = exp(a_1 . b_1) - exp(a_2 . b_2) + init
//
// The heads of one key/value head are worked on together: its query rows are
// the nq queries of each of the heads / kv_heads query heads, one after the
// other, so that a single token's heads fill one 16-row tile and read the
// cache once. In bf16 a score starts as bias / scale, in the accumulator of its
// matrix instruction, and is left unscaled: the exponent of a weight is one fma,
// 2^(s scale log2(e) - M), with the row's maximum M in log2 units. Each of a
// score's sums is then rounded at bias / scale's size, which float32 results show
// (1e-6 of the output): there the bias comes to the scaled score, in log2 units.
// A bias that is -inf in its unit (-inf and the types' lowest values) is no key.
// Where a bias is so large that M's own rounding counts as an exponent, the
// products s scale log2(e) are rounded like it (far_scores).
#pragma once

#include "fjx_common.hpp"
#include "fjx_kernels.hpp"

namespace fjx {

// strides in elements: item, head, token
template <typename T>
struct HeadsView {
  T* p;
  int64_t item, head, token;
};

template <typename T>
struct DiffAttnParams {
  HeadsView<const T> q, k, v;  // [items][2 H][nq][D], [items][2 Hk][nk][D], [items][Hk][nk][2 D]
  HeadsView<T> out;            // [items][H][nq][2 D]
  HeadsView<const T> bias;     // [items / share][H][nq][nk] (item: plane, token: query), or null
  const uint8_t* mask;         // [items][nk] or null
  const float* lam;            // [4][H][D]: a_1, b_1, a_2, b_2
  float* stats;                // [items][2 H][nq] row statistics, or null
  int64_t items, nq, nk, share;
  int heads, group;            // query heads, and those of one key/value head
  float scale, scale_log2, inv_scale, init;  // scale_log2: times log2(e)
  // keys split over workgroups: key blocks of one split, and the partial
  // results [split][items][H nq rows][2 maps]: values [2 D], then (max, sum)
  int splits;
  int64_t split_blocks;
  float* part_o;
  float* part_ml;
  // backward
  HeadsView<const T> dout;     // [items][H][nq][2 D]
  HeadsView<T> dq, dk, dv;
  HeadsView<T> dbias;          // as bias, or null
  const float* saved;          // the forward pass's stats
  float* delta;                // [items][2 H][nq]: rowsum(P_t dP) / rowsum(P_t)
  float* norm;                 // the same: 1 / rowsum(P_t), 0 for a row without keys
  float* dlam;                 // [4][H][D]
  float* part_bias;            // [chunks][planes][H][nq][nk] partial sums of dbias
  int64_t chunk_items;         // items of one chunk
  int chunks;
};

// waves a SIMD that the registers are held to
template <typename T, int D> constexpr int kDaWaves = sizeof(T) == 2 && D == 32 ? 2 : 1;

// a bias starts its score's sum, as bias / scale, or is added to the scaled score
template <typename T> constexpr bool kBiasFirst = sizeof(T) == 2;
template <typename T>
__device__ __forceinline__ float bias_unit(float inv_scale) { return kBiasFirst<T> ? inv_scale : kLog2e; }
template <typename T>
__device__ __forceinline__ f32x4 score_start(const f32x4& b) { return kBiasFirst<T> ? b : f32x4{0.f, 0.f, 0.f, 0.f}; }
// the exponent of a weight, less `base`, in log2 units, from its score's sum s
template <typename T>
__device__ __forceinline__ float exponent(float s, float b, float scale_log2, float base) {
  return kBiasFirst<T> ? fmaf(s, scale_log2, -base) : fmaf(s, scale_log2, b) - base;
}

// In bf16 an exponent is the rounding of s scale log2(e) - M with M rounded: off by up
// to half a step of M for all of a row's keys alike, which cancels in the softmax as
// long as 2 to that is a number. Rows with |M| > kFar (a step of 2; the bias of a
// whole row at -1e10 gave 2^512) take products rounded by themselves, whose largest is M
// exactly. Returns the factor that is left for the exponents' fma. The branch costs the
// forward pass up to 2 % (18.2 -> 18.6 us at 4 x 499 tokens).
constexpr float kFar = 16777216.f;
template <int NT>
__device__ __forceinline__ float far_scores(bool far, float scale_log2, f32x4 (&s)[NT]) {
  if (!far) return scale_log2;
#pragma unroll
  for (int kt = 0; kt < NT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = s[kt][r] * scale_log2;
      asm("" : "+v"(x));  // not one fma with what is subtracted from it
      s[kt][r] = x;
    }
  return 1.f;
}

// How the waves of a workgroup share its rows (for the keys' gradients: its keys)
// and a staged block: KS of them have a tile of 16 rows and a KS-th of a block each.
// KS 1: four waves, four tiles, blocks of 64; 4: four waves, one tile, blocks of
// 128; 2: eight waves, four tiles, blocks of 128.
template <int KS>
struct DaForm {
  static constexpr int kWaves = KS == 2 ? 8 : 4, kThreads = 64 * kWaves;
  static constexpr int kTiles = kWaves / KS;
  static constexpr int kBlock = KS == 1 ? 64 : 128;
};

constexpr int kDaKeys = 64;  // keys (or, for the keys' gradients, queries) of a staged block

// one staged block: the two maps' D columns side by side, and 2 D columns; rows
// padded by 16 bytes so that 16 rows' 16-byte pieces fall on distinct banks
template <typename T, int D, int ROWS>
struct DaTile {
  static constexpr int kPitch = 2 * D + 16 / (int)sizeof(T);
  T a[ROWS][kPitch];
  T b[ROWS][kPitch];
};

// 8 k-slots of a column operand: rows row0 + 4 g + 0..3 and row0 + 16 + 4 g +
// 0..3 (g = lane / 16) of column col0 + lane % 16, the rows that a lane's
// accumulators of two adjacent 16-row score tiles hold
__device__ __forceinline__ bf16x8 col_frag(const bf16* tile, int pitch, int row0, int col0, int lane) {
  // ds_read_b64_tr_b16: the 16 lanes of a group name 4 rows x 16 columns in
  // row order, and lane i gets the 4 rows of column i
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s16x4 lds4;
  const bf16* p = tile + (row0 + 4 * (lane >> 4) + ((lane >> 2) & 3)) * pitch + col0 + 4 * (lane & 3);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * pitch));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ f32x8 col_frag(const float* tile, int pitch, int row0, int col0, int lane) {
  const float* p = tile + (row0 + 4 * (lane >> 4)) * pitch + col0 + (lane & 15);
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = p[e * pitch];
    v[4 + e] = p[(16 + e) * pitch];
  }
  return v;
}

// 4 contiguous elements with element alignment only (rows of an odd length)
template <typename T> struct Quad;
template <> struct Quad<bf16> { typedef bf16x4 type; typedef bf16x4 any __attribute__((aligned(2))); };
template <> struct Quad<float> { typedef f32x4 type; typedef f32x4 any __attribute__((aligned(4))); };

// the bias of a lane's 4 keys of each of NT tiles, from k0 on (its own 4 g
// within); zeros past the last key, which its flag takes out
template <typename T, int NT>
__device__ __forceinline__ void bias_tile(const T* bias, int64_t k0, int64_t nk, bool whole, typename Quad<T>::type (&bv)[NT]) {
  if (whole) {
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) bv[kt] = *reinterpret_cast<const typename Quad<T>::any*>(bias + k0 + 16 * kt);
  } else {
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) bv[kt][r] = k0 + 16 * kt + r < nk ? bias[k0 + 16 * kt + r] : from_f32<T>(0.f);
  }
}

// One instruction where fminf and fmaxf quiet both operands first: for values
// that no signalling NaN can be among, results of arithmetic.
__device__ __forceinline__ float plain_min(float a, float b) {
  float r;
  asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float plain_max(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// Which keys of a block take part: +inf, or -inf for one that does not, so
// that the minimum with its bias (or 0) is -inf whatever the bias holds, a NaN
// among it; and whether all of 64 do, the usual case.
template <int ROWS>
struct alignas(16) KeyFlags {
  float on[ROWS];
  int all[ROWS / 64];
  // by threads 0 .. ROWS - 1
  __device__ __forceinline__ void set(int t, bool part) {
    on[t] = part ? INFINITY : -INFINITY;
    const bool every = __builtin_amdgcn_ballot_w64(part) == ~0ull;
    if ((t & 63) == 0) all[t >> 6] = every;
  }
  __device__ __forceinline__ bool whole() const {
    int v = all[0];
#pragma unroll
    for (int i = 1; i < ROWS / 64; ++i) v &= all[i];
    return __builtin_amdgcn_readfirstlane(v);
  }
  // b = min(b, flag) for a lane's keys
  template <int NT>
  __device__ __forceinline__ void apply(int key_w, int lg, f32x4 (&b)[NT]) const {
    if (__builtin_amdgcn_readfirstlane(all[key_w >> 6])) return;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      const f32x4 f = *reinterpret_cast<const f32x4*>(&on[key_w + 16 * kt + 4 * lg]);
#pragma unroll
      for (int r = 0; r < 4; ++r) b[kt][r] = plain_min(b[kt][r], f[r]);
    }
  }
};

// what a row's maximum (in log2 units) subtracts in the exponent: itself, or 0
// where the row has no key (every weight is then 2^-inf)
__device__ __forceinline__ float exponent_base(float m) { return m == -INFINITY ? 0.f : m; }

// max over the 4 lanes {l % 16 + 16 g}
__device__ __forceinline__ float group_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const uint32_t v = __builtin_bit_cast(uint32_t, plain_max(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return plain_max(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// lambda of `head`, the lane's own; the 4 lanes of a row take a quarter of
// the two dot products each. e[0], e[1]: the two exponentials
template <int D>
__device__ __forceinline__ float da_lambda(const float* lam, int heads, int head, float init, int lane, float* e = nullptr) {
  float dot[2] = {0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float* a = lam + ((int64_t)(2 * t) * heads + head) * D + (lane >> 4) * (D / 4);
    const float* b = a + (int64_t)heads * D;
#pragma unroll
    for (int d = 0; d < D / 4; d += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(a + d), y = *reinterpret_cast<const f32x4*>(b + d);
#pragma unroll
      for (int r = 0; r < 4; ++r) dot[t] = fmaf(x[r], y[r], dot[t]);
    }
    dot[t] = group_sum(dot[t]);
  }
  const float e1 = expf(dot[0]), e2 = expf(dot[1]);
  if (e) e[0] = e1, e[1] = e2;
  return e1 - e2 + init;
}

// The pieces of one block that a thread moves from memory to LDS: 16 bytes
// of a row at a time, the same columns of every `step`-th row. Rows past n,
// and those that the mask takes out, are zeros: a weight of zero times what
// padding holds there must stay zero.
template <typename T, int D, int ROWS, int THREADS>
struct DaStage {
  static constexpr int kE = 16 / (int)sizeof(T);           // elements of a piece
  static constexpr int kPa = D / kE;                       // pieces of a row of the first two
  static constexpr int kPk = 4 * kPa;                      // pieces of a row in all
  static constexpr int kStep = THREADS / kPk;              // rows between a thread's pieces
  static constexpr int kN = ROWS / kStep;                  // pieces of a thread
  static_assert(THREADS % kPk == 0 && ROWS % kStep == 0, "whole pieces");
  u32x4 r[kN];
  const T* src;
  int64_t pitch;
  int row, which;
  int lds;  // the first piece's place in the tile

  // a, b: the rows' bases; a_head: elements between the two a tiles
  __device__ __forceinline__ void init(const T* a, int64_t a_head, int64_t a_token, const T* b, int64_t b_token,
                                       int t) {
    const int in = t % kPk;
    row = t / kPk;
    which = in / kPa;  // 0, 1: the a tiles; 2, 3: the halves of b
    const int col = (in % kPa) * kE + (which == 3 ? D : 0);
    lds = ((which >> 1) * ROWS + row) * DaTile<T, D, ROWS>::kPitch + in % (2 * kPa) * kE;
    pitch = which < 2 ? a_token : b_token;
    src = (which < 2 ? a + which * a_head : b) + col + row * pitch;
  }
  // rows row0 .. row0 + ROWS - 1; `all`: every one is there and takes part,
  // else on[x] says so of row x
  __device__ __forceinline__ void load(int64_t row0, bool all, const float* on) {
    const T* p = src + row0 * pitch;
    if (all) {
#pragma unroll
      for (int i = 0; i < kN; ++i) r[i] = *reinterpret_cast<const u32x4*>(p + i * kStep * pitch);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        r[i] = u32x4{0, 0, 0, 0};
        if (on[row + i * kStep] > 0.f) r[i] = *reinterpret_cast<const u32x4*>(p + i * kStep * pitch);
      }
    }
  }
  __device__ __forceinline__ void store(DaTile<T, D, ROWS>& tile) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) *reinterpret_cast<u32x4*>(&tile.a[0][0] + lds + i * kStep * tile.kPitch) = r[i];
  }
};

// workgroups in an order that keeps neighbours (the tiles of one item, which
// read the same keys) on one of the 8 XCDs, to which the hardware deals block
// after block in turn; grids are multiples of 8 blocks
__device__ __forceinline__ uint32_t xcd_order(uint32_t blk, uint32_t blocks) { return (blk & 7) * (blocks >> 3) + (blk >> 3); }

}  // namespace fjx
