// What the kernels of packed attention share: finding a tile's sequence, staged
// blocks and their fragments, the limits of a row.
//
//   sequence s: queries [q_starts[s], q_starts[s + 1]), keys from k_starts[s] on
//   S = scale q k^T over the keys that the row sees,  P = softmax(S),  out = P v
//
// The query heads that share a key/value head are worked on together: the rows of
// a sequence are its queries, and of each the heads / kv_heads heads one after the
// other, so that a single token's heads fill a tile and read the cache once, and
// consecutive rows see (nearly) the same keys.
//
// The host knows the number of sequences and of tokens, not the lengths. Sequence s
// has the tiles from t(s) = floor(first row / R) + s on: t(s + 1) - t(s) is at least
// its rows / R rounded up, so that no two share a tile, and there are at most
// (rows / R) + sequences in all; a tile finds its sequence by a search in t, and one
// that has no rows returns.
#pragma once

#include <type_traits>

#include "fjx_common.hpp"
#include "fjx_kernels.hpp"

namespace fjx {

// strides in elements
template <typename T>
struct PackedView {
  T* p;
  int64_t head, token;
};

// token offsets, [n] int32 or int64 in device memory
struct PackedInts {
  const void* p;
  int wide;
};

// how a call is cut (PkForm), 16-row tiles of a wave
struct PackedForm {
  int groups, ks, tiles;
  int count;    // workgroups for one key/value head
  int2* order;  // [count], to be filled with the tiles in the order of their work, or null
  __host__ __device__ int rows() const { return 16 * groups * tiles; }  // of a workgroup
};
constexpr int kPackedOrder = 12288;  // tiles that are sorted at most

template <typename T>
struct PackedParams {
  PackedView<const T> q, k, v;  // [H][tq][d], [Hk][tk][d], [Hk][tk][d]
  PackedView<T> out;            // [H][tq][d]
  PackedView<T> rest;           // what out's rounding left, or null
  float* lse;                   // [H][tq][2]: the row's maximum and log2 of its sum (log2 units), or null
  PackedInts q_starts, k_starts, k_lengths;  // [seqs + 1], [seqs + 1], [seqs] or null
  int64_t tq, tk;
  int seqs, heads, group, d;
  float scale, scale_log2;      // scale_log2: times log2(e)
  int causal;
  int zero_tail;                // rows of no sequence are written as zeros
  int tiles;                    // of a launch, for one key/value head
  const int2* order;            // [tiles] {sequence, its tile}, those with the most work first; or null
  // keys (dk, dv: the group's heads) over several workgroups, whose sums a second kernel joins
  int splits;
  float* part_o;                // [splits][H][tq][DP]
  float* part_ml;               // [splits][H][tq][2]
  // backward
  PackedView<const T> dout, o, o_rest;
  PackedView<T> dq, dk, dv;
  float* delta;                 // [H][tq]: rowsum(dO out)
  float* part_dk;               // [splits][Hk][tk][DP]
  float* part_dv;
};

__device__ __forceinline__ int64_t packed_int(const PackedInts& a, int i, int64_t most) {
  const int64_t v = a.wide ? static_cast<const int64_t*>(a.p)[i] : static_cast<const int32_t*>(a.p)[i];
  return v < 0 ? 0 : v > most ? most : v;
}
// the first token of sequence s; offsets that lead out of the buffer end at its ends
__device__ __forceinline__ int64_t packed_start(const PackedInts& a, int s, int64_t tokens) {
  return s == 0 ? 0 : packed_int(a, s, tokens);
}

struct PackedSpan {
  int seq;         // seqs: the rows behind the last sequence
  int tile;        // of the sequence
  int q0, nq, k0, nk, cap;  // first query, queries, first key, keys, and keys with the unused ones behind them
};

// The sequence of `tile` among tiles of 2^shift rows of which a token has `per`,
// counted over a's offsets: 64 probes at a time. False for a tile past the last.
__device__ __forceinline__ bool packed_find(const PackedInts& a, int seqs, int64_t tokens, int per, int shift, int tile,
                                            int lane, int& seq, int& at) {
  auto first = [&](int s) { return (int)((packed_start(a, s, tokens) * per) >> shift) + s; };
  int lo = 0, n = seqs + 1;  // the last s of [lo, lo + n) whose first tile is not behind `tile`; s = 0 starts at 0
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int s = lo + lane * step;
    const bool in = lane * step < n && first(s) <= tile;
    const uint64_t votes = __builtin_amdgcn_ballot_w64(in);
    // offsets that descend leave votes behind a gap: the first run counts
    const int run = votes == ~0ull ? 64 : (int)__builtin_ctzll(~votes);
    const int hop = run > 0 ? run - 1 : 0;
    lo += hop * step;
    n = n - hop * step < step ? n - hop * step : step;
  }
  seq = __builtin_amdgcn_readfirstlane(lo);
  at = tile - __builtin_amdgcn_readfirstlane(first(seq));
  return at >= 0;
}

// what there is of sequence s.seq
template <typename T>
__device__ __forceinline__ void packed_sequence(const PackedParams<T>& P, bool by_keys, PackedSpan& s) {
  const int64_t q0 = packed_start(P.q_starts, s.seq, P.tq), k0 = packed_start(P.k_starts, s.seq, P.tk);
  int64_t q1 = P.tq, k1 = P.tk, nk = 0;
  if (s.seq < P.seqs) {
    q1 = packed_int(P.q_starts, s.seq + 1, P.tq);
    k1 = packed_int(P.k_starts, s.seq + 1, P.tk);
    if (k1 < k0) k1 = k0;
    nk = P.k_lengths.p ? packed_int(P.k_lengths, s.seq, k1 - k0) : k1 - k0;
  }
  s.q0 = (int)q0;
  s.nq = s.seq < P.seqs || !by_keys ? (int)(q1 > q0 ? q1 - q0 : 0) : 0;
  s.k0 = (int)k0;
  s.nk = (int)nk;
  s.cap = (int)(k1 > k0 ? k1 - k0 : 0);
}

// the sequence and the tile of a workgroup, the `at`-th of a key/value head
template <typename T>
__device__ __forceinline__ bool packed_span(const PackedParams<T>& P, bool by_keys, int per, int shift, int at, int lane,
                                            PackedSpan& s) {
  if (P.order) {
    const int2 o = P.order[at];
    s.seq = __builtin_amdgcn_readfirstlane(o.x);
    s.tile = __builtin_amdgcn_readfirstlane(o.y);
    if (s.seq < 0) return false;
  } else if (!packed_find(by_keys ? P.k_starts : P.q_starts, P.seqs, by_keys ? P.tk : P.tq, per, shift, at, lane, s.seq, s.tile)) {
    return false;
  }
  packed_sequence(P, by_keys, s);
  s.q0 = __builtin_amdgcn_readfirstlane(s.q0);
  s.nq = __builtin_amdgcn_readfirstlane(s.nq);
  s.k0 = __builtin_amdgcn_readfirstlane(s.k0);
  s.nk = __builtin_amdgcn_readfirstlane(s.nk);
  s.cap = __builtin_amdgcn_readfirstlane(s.cap);
  return true;
}

// How the waves of a workgroup share its rows (for the keys' gradients: its keys) and the
// blocks that it walks: G groups of waves with tiles of their own, KS waves in each with
// the same tiles and a KS-th of a block. Every group reads a whole block from LDS, so that
// few groups of many rows read least. One group: its waves have staged rows of their own,
// and need no barrier.
template <int G, int KS>
struct PkForm {
  static constexpr int kWaves = G * KS, kThreads = 64 * kWaves;
  static constexpr bool kPrivate = G == 1;
  static constexpr int kBlock = KS == 1 ? 64 : 128;             // of all waves
  static constexpr int kOwn = kBlock / KS;                      // of one
  static constexpr int kStage = kPrivate ? kOwn : kBlock;       // rows staged together
  static constexpr int kSets = kPrivate ? KS : 1;               // of such rows
  static constexpr int kOwners = kPrivate ? 1 : kWaves;         // waves that stage them
  static constexpr int kRest = (kStage + 63) / 64;              // waves that fetch a value for each
  // waves a SIMD that the registers are held to, where a workgroup's LDS (two stages of
  // two operands) leaves room for as many
  template <typename T, int DP>
  static constexpr int kSimd =
      kWaves / 4 * (sizeof(T) == 2 && 2 * 2 * kStage * kSets * DP * (int)sizeof(T) <= 75 * 1024 ? 2 : 1) >= 2 ? 2 : 1;
  // the wave's place: its group, its part of a block, where that begins among its
  // staged rows, and as which of the owners it stages
  int group, part, at, stager;
  __device__ __forceinline__ explicit PkForm(int wave)
      : group(wave % G), part(wave / G), at(kPrivate ? 0 : kOwn * (wave / G)), stager(kPrivate ? 0 : wave) {}
  // the first of the wave's staged rows in a block
  __device__ __forceinline__ int staged() const { return kPrivate ? kOwn * part : 0; }
  // which of the waves with the same rows writes column tile u, after their sums were joined
  __device__ __forceinline__ bool writes(int u) const { return u % KS == part; }
};

// Rows of DP elements in LDS, 16-byte piece c of row r in slot c ^ f(r) of its row.
// A fragment read takes 16 rows, four pieces side by side; the hardware serves lanes
// {0-3, 12-15, 20-23, 24-27} and such sets together, 16 pieces over 64 banks: they are
// distinct where f maps rows {0-3, 12-15} to a set closed under exchanging neighbours.
// A transposing read takes 8 rows of two pieces: distinct where f / 2 is distinct in
// rows 0-7 and in 8-15. float32 reads columns element by element, 4 rows apart.
template <typename T, int DP>
struct PkRows {
  static constexpr int kE = 16 / (int)sizeof(T);       // elements of a piece
  static constexpr int kCh = DP / kE;                  // pieces of a row
  static constexpr int kRowBytes = DP * (int)sizeof(T);
  static constexpr int kC = DP / 32;                   // k-steps of a product over a row
  static constexpr int kU = DP / 16;                   // 16-column tiles of a row
  static constexpr int kPer = kCh < 16 ? kCh : 16;     // f repeats every 16 rows
  __device__ static __forceinline__ int f(int r) {
    const int j = (r & 15) * kPer / 16;
    if (sizeof(T) == 4) return j;
    constexpr int half = kPer / 2;
    return j < half ? 2 * j : 2 * ((j + half / 2) % half) + 1;
  }
};

// The addresses of a lane's fragments within a staged tile, in bytes: those of other
// k-steps and columns by exclusive or, of other rows (multiples of 16) by addition.
template <typename T, int DP>
struct PkLane {
  typedef PkRows<T, DP> Rows;
  typedef typename Frag<T>::type F;
  static constexpr int kCols = sizeof(T) == 2 ? 1 : 4;
  uint32_t row, col[kCols];
  __device__ __forceinline__ void init(int lane) {
    const int li = lane & 15, lg = lane >> 4;
    row = li * Rows::kRowBytes + (((sizeof(T) == 2 ? lg : 2 * lg) ^ Rows::f(li)) << 4);
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * lg + ((lane >> 2) & 3);
      col[0] = r * Rows::kRowBytes + ((((lane >> 1) & 1) ^ Rows::f(r)) << 4) + 8 * (lane & 1);
    } else {
#pragma unroll
      for (int e = 0; e < kCols; ++e) {
        const int r = 4 * lg + e;
        col[e] = r * Rows::kRowBytes + (((li >> 2) ^ Rows::f(r)) << 4) + 4 * (li & 3);
      }
    }
  }
  // elements 32 c + 8 lg .. + 7 of row row0 + li (row0 a multiple of 16)
  __device__ __forceinline__ F at_row(const unsigned char* tile, int row0, int c) const {
    const unsigned char* p = tile + row0 * Rows::kRowBytes;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const F*>(p + (row ^ (64 * c)));
    } else {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(p + (row ^ (128 * c)));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(p + (row ^ (128 * c + 16)));
      return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }
  // rows row0 + 4 lg + 0..3 and row0 + 16 + 4 lg + 0..3 of column 16 u + li: the rows
  // that a lane's accumulators of two adjacent 16-row tiles hold
  __device__ __forceinline__ F at_col(const unsigned char* tile, int row0, int u) const {
    const unsigned char* p = tile + row0 * Rows::kRowBytes;
    if constexpr (sizeof(T) == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const unsigned char* a = p + (col[0] ^ (32 * u));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(a));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(a + 16 * Rows::kRowBytes));
      return __builtin_bit_cast(F, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      F v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned char* a = p + (col[e] ^ (64 * u));
        v[e] = *reinterpret_cast<const float*>(a);
        v[4 + e] = *reinterpret_cast<const float*>(a + 16 * Rows::kRowBytes);
      }
      return v;
    }
  }
};

// Copies ROWS rows of d <= DP elements from memory to LDS without registers
// (buffer_load ... lds: a wave's 64 pieces side by side). Rows past the last and
// columns past d come as zeros, from past the resource's end: a weight of zero times
// what lies there must stay zero. WAVES waves share the work.
template <typename T, int DP, int ROWS, int WAVES>
struct PkCopy {
  typedef PkRows<T, DP> Rows;
  static constexpr int kRpi = 64 / Rows::kCh > 0 ? 64 / Rows::kCh : 1;  // rows of one instruction
  static constexpr int kG = 16 / kRpi;                                 // instructions of 16 rows
  static constexpr int kN = ROWS * Rows::kCh / 64 / WAVES;             // instructions of a wave
  static constexpr int kSub = kG > WAVES ? kG / WAVES : 1;             // distinct offsets of a lane
  static_assert(Rows::kCh <= 64 && ROWS % 16 == 0 && kN >= 1, "whole instructions");
  uint32_t off[kSub];
  uint32_t pitch;  // bytes between rows
  __device__ __forceinline__ void init(int64_t token, int d, int wave, int lane) {
    pitch = (uint32_t)(token * (int64_t)sizeof(T));
#pragma unroll
    for (int i = 0; i < kSub; ++i) {
      const int sub = WAVES >= kG ? wave % kG : wave + WAVES * i;
      const int r = sub * kRpi + lane / Rows::kCh;
      const int c = (lane % Rows::kCh) ^ Rows::f(r);
      off[i] = c * Rows::kE < d ? r * pitch + 16 * c : 0x80000000u;
    }
  }
  // rows row0 .. of `src` (row 0 at src, n rows in all) to `tile`
  __device__ __forceinline__ void issue(const T* src, int64_t row0, int64_t n, int d, unsigned char* tile, int wave) const {
    const int64_t left = n - row0;
    const int64_t rows = left < ROWS ? left : ROWS;
    const int bytes = rows > 0 ? (int)((rows - 1) * pitch + d * (int)sizeof(T)) : 0;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(reinterpret_cast<const char*>(src) + row0 * (int64_t)pitch), (short)0, bytes, 0x00020000);
    // their sums, kept through a loop, took more scalars than there are
    typedef __attribute__((address_space(3))) unsigned char lds_byte;
    uint32_t step = pitch, to = (uint32_t)(uintptr_t)(lds_byte*)tile;
    asm volatile("" : "+s"(step), "+s"(to));
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      // 16-row group and place of instruction `wave + WAVES i`
      const int group = WAVES >= kG ? wave / kG + i * (WAVES / kG) : i / kSub;
      const uint32_t o = off[WAVES >= kG ? 0 : i % kSub];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_byte*)(uintptr_t)(to + (wave + WAVES * i) * 1024), 16, o + (uint32_t)(16 * group) * step, 0, 0, 0);
    }
  }
};

// N products use(i, load(i)) whose fragments come from LDS: those of the next four are on
// their way while four are worked on. Left to itself the compiler reads one or two ahead,
// and a wave waits for LDS between any two products.
template <int N, typename L, typename U>
__device__ __forceinline__ void pk_ahead(L load, U use) {
  typedef decltype(load(0)) F;
  constexpr int kGroup = sizeof(F) > 16 ? 2 : 4, kGroups = (N + kGroup - 1) / kGroup;
  F f[2][kGroup];
#pragma unroll
  for (int j = 0; j < kGroup; ++j)
    if (j < N) f[0][j] = load(j);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (kGroup * (g + 1) + j < N) f[(g + 1) & 1][j] = load(kGroup * (g + 1) + j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (kGroup * g + j < N) use(kGroup * g + j, f[g & 1][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Behind the use of a stage and the issue of the next: what this wave has in flight is
// complete, its fragment reads too, and where waves share stages, theirs.
template <typename Form>
__device__ __forceinline__ void pk_sync() {
  lds_wait<0>();
  if constexpr (!Form::kPrivate) lds_barrier();
  asm volatile("" ::: "memory");
}

// what a row's maximum (in log2 units) subtracts in the exponent: itself, or 0
// where the row has no key yet (every weight is then 2^-inf)
__device__ __forceinline__ float pk_base(float m) { return m == -INFINITY ? 0.f : m; }

// a row's statistics: its maximum and log2 of its sum; +inf for a row without keys,
// whose weights are then zeros in the backward pass as well
__device__ __forceinline__ f32x2 pk_stats(float m, float sum) {
  return f32x2{pk_base(m), sum == 0.f ? INFINITY : log2f(sum)};
}

// scores times their factor, each product rounded by itself: not one fma with what is
// subtracted from it
template <int NT>
__device__ __forceinline__ void pk_round(float by, f32x4 (&s)[NT]) {
#pragma unroll
  for (int kt = 0; kt < NT; ++kt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = s[kt][e] * by;
      asm("" : "+v"(x));
      s[kt][e] = x;
    }
}

// The accumulators of a group's waves added, through LDS (PITCH floats a row), 16 rows of
// each at a time; wave j of a group gets the column tiles u with u % KS == j.
template <int G, int KS, int R, int U, int PITCH>
__device__ __forceinline__ void pk_sum_waves(float* lds, const PkForm<G, KS>& f, int li, int lg, f32x4 (&x)[R][U]) {
  auto slot = [&](int j) { return ((j * G + f.group) * 16 + li) * PITCH + 4 * lg; };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) lds[slot(f.part) + 16 * u + e] = x[r][u][e];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!f.writes(u)) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) a += lds[slot(j) + 16 * u + e];
        x[r][u][e] = a;
      }
    }
  }
}
template <int G, int KS, int PITCH>
constexpr int kPkSumBytes = G * KS * 16 * PITCH * 4;

// max over the 4 lanes {l % 16 + 16 g}
__device__ __forceinline__ float lanes4_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const uint32_t v = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// f(G, KS, R) for the forms that packed_form chooses; float32 has one tile a wave
template <typename T, typename F>
void pk_form(const PackedForm& form, F f) {
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 4> Four;
  if (form.groups == 1) return f(One{}, Four{}, One{});
  if constexpr (sizeof(T) == 2) {
    if (form.groups == 2) return f(Two{}, Four{}, Two{});
    if (form.tiles == 2) return form.ks == 2 ? f(Four{}, Two{}, Two{}) : f(Four{}, One{}, Two{});
  }
  if (form.ks == 2) return f(Four{}, Two{}, One{});
  f(Four{}, One{}, One{});
}

// the orders that `rows` and `keys` ask for
template <typename T>
void launch_packed_order(const PackedParams<T>& P, const PackedForm& rows, const PackedForm& keys, hipStream_t st);
template <typename T>
void launch_packed_fwd(const PackedParams<T>& P, const PackedForm& form, hipStream_t st);
template <typename T>
void launch_packed_bwd(const PackedParams<T>& P, const PackedForm& rows, const PackedForm& keys, hipStream_t st);

}  // namespace fjx
