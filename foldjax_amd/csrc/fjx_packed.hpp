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
// floor(rows / R) + sequences + 1 in all, the one more for the rows behind the last
// sequence; a tile finds its sequence by a search in t, and one that has no rows returns.
#pragma once

#include <type_traits>

#include "fjx_common.hpp"
#include "fjx_kernels.hpp"
#include "fjx_packed_plan.hpp"

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

template <typename T>
struct PackedParams {
  PackedView<const T> q, k, v;  // [H][tq][d], [Hk][tk][d], [Hk][tk][d]
  PackedView<T> out;            // [H][tq][d]
  PackedView<T> rest;           // what out's rounding left, or null
  float* lse;                   // [H][tq][2]: the row's maximum and log2 of its sum, unrounded (log2 units), or null
  PackedInts q_starts, k_starts, k_lengths;  // [seqs + 1], [seqs + 1], [seqs] or null
  int64_t tq, tk;
  int seqs, heads, group, d;
  uint32_t group_inv;           // x / group = (x group_inv) >> 21 for x < group + 128
  float scale, scale_log2;      // scale_log2: times log2(e)
  int causal;
  int zero_tail;                // rows of no sequence are written as zeros
  int tiles;                    // of a launch, for one key/value head
  const PackedTile* order;      // [tiles], those with the most work first; or null
  int tile0;                    // the first tile of this launch
  // keys (dk, dv: the group's heads) over several workgroups, whose sums a second kernel joins
  int splits;
  float* part_o;                // [splits][H][tq][DP]
  float* part_ml;               // [splits][H][tq][2]
  float* part_l;                // [splits][H][tq]: sums of unrounded bf16 weights, where lse is asked for
  // backward
  PackedView<const T> dout, o, o_rest;
  PackedView<T> dq, dk, dv;
  float* delta;                 // [H][tq]: rowsum(dO out)
  float* part_dk;               // [splits][Hk][tk][DP]
  float* part_dv;
  int part_rows;                // rows of all heads that a part of a key tile walks, about
};

__device__ __forceinline__ int64_t packed_int(const PackedInts& a, int i, int64_t most) {
  const int64_t v = a.wide ? static_cast<const int64_t*>(a.p)[i] : static_cast<const int32_t*>(a.p)[i];
  return v < 0 ? 0 : v > most ? most : v;
}
// the first token of sequence s; offsets that lead out of the buffer end at its ends
__device__ __forceinline__ int64_t packed_start(const PackedInts& a, int s, int64_t tokens) {
  return s == 0 ? 0 : packed_int(a, s, tokens);
}

// the sequence's tokens, from its offsets as they are
template <typename T>
__device__ __forceinline__ void packed_tokens(const PackedParams<T>& P, bool by_keys, int q0, int q1, int k0, int k1, int length,
                                              PackedTile& s) {
  const bool real = s.seq < P.seqs;
  if (!real) q1 = (int)P.tq, k1 = (int)P.tk;
  s.q0 = q0;
  s.nq = (real || !by_keys) && q1 > q0 ? q1 - q0 : 0;
  s.k0 = k0;
  s.cap = k1 > k0 ? k1 - k0 : 0;
  s.nk = !real ? 0 : length < s.cap ? length : s.cap;
}

// The sequence of tile `at` among tiles of 2^shift rows of which a token has `per`
// (by_keys: of keys). False for a tile past the last. For up to 63 sequences a lane has
// the offsets of one, and one trip to memory tells all there is to know.
template <typename T>
__device__ __forceinline__ bool packed_find(const PackedParams<T>& P, bool by_keys, int per, int shift, int at, int lane,
                                            PackedTile& s) {
  const PackedInts& own = by_keys ? P.k_starts : P.q_starts;
  const int64_t tokens = by_keys ? P.tk : P.tq;
  auto first = [&](int64_t start, int seq) { return (int)((start * per) >> shift) + seq; };
  if (P.seqs < 64) {
    const int i = lane < P.seqs ? lane : P.seqs;
    const int qv = (int)packed_start(P.q_starts, i, P.tq), kv = (int)packed_start(P.k_starts, i, P.tk);
    const int lv = P.k_lengths.p ? (int)packed_int(P.k_lengths, lane < P.seqs ? lane : 0, P.tk) : 0x7fffffff;
    const int f = first(by_keys ? kv : qv, i);
    const uint64_t votes = __builtin_amdgcn_ballot_w64(lane <= P.seqs && f <= at);
    // offsets that descend leave votes behind a gap: the first run counts
    const int run = votes == ~0ull ? 64 : (int)__builtin_ctzll(~votes);
    const int seq = run > 0 ? run - 1 : 0, next = seq < P.seqs ? seq + 1 : seq;
    s.seq = seq;
    s.tile = at - __builtin_amdgcn_readlane(f, seq);
    packed_tokens(P, by_keys, __builtin_amdgcn_readlane(qv, seq), __builtin_amdgcn_readlane(qv, next),
                  __builtin_amdgcn_readlane(kv, seq), __builtin_amdgcn_readlane(kv, next), __builtin_amdgcn_readlane(lv, seq), s);
    return s.tile >= 0;
  }
  int lo = 0, n = P.seqs + 1;  // the last s of [lo, lo + n) whose first tile is not behind `at`; s = 0 starts at 0
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int seq = lo + lane * step;
    const bool in = lane * step < n && first(packed_start(own, seq, tokens), seq) <= at;
    const uint64_t votes = __builtin_amdgcn_ballot_w64(in);
    const int run = votes == ~0ull ? 64 : (int)__builtin_ctzll(~votes);
    const int hop = run > 0 ? run - 1 : 0;
    lo += hop * step;
    n = n - hop * step < step ? n - hop * step : step;
  }
  s.seq = __builtin_amdgcn_readfirstlane(lo);
  const int next = s.seq < P.seqs ? s.seq + 1 : s.seq;
  const int q0 = (int)packed_start(P.q_starts, s.seq, P.tq), k0 = (int)packed_start(P.k_starts, s.seq, P.tk);
  s.tile = at - __builtin_amdgcn_readfirstlane(first(by_keys ? k0 : q0, s.seq));
  packed_tokens(P, by_keys, __builtin_amdgcn_readfirstlane(q0),
                __builtin_amdgcn_readfirstlane((int)packed_start(P.q_starts, next, P.tq)), __builtin_amdgcn_readfirstlane(k0),
                __builtin_amdgcn_readfirstlane((int)packed_start(P.k_starts, next, P.tk)),
                P.k_lengths.p && s.seq < P.seqs ? __builtin_amdgcn_readfirstlane((int)packed_int(P.k_lengths, s.seq, P.tk)) : 0x7fffffff,
                s);
  return s.tile >= 0;
}

// the sequence and the tile of a workgroup, the `at`-th of a key/value head
template <typename T>
__device__ __forceinline__ bool packed_tile(const PackedParams<T>& P, bool by_keys, int per, int shift, int at, int lane,
                                            PackedTile& s) {
  if (!P.order) return packed_find(P, by_keys, per, shift, at, lane, s);
  const PackedTile o = P.order[at];
  s.seq = __builtin_amdgcn_readfirstlane(o.seq);
  s.tile = __builtin_amdgcn_readfirstlane(o.tile);
  s.q0 = __builtin_amdgcn_readfirstlane(o.q0);
  s.nq = __builtin_amdgcn_readfirstlane(o.nq);
  s.k0 = __builtin_amdgcn_readfirstlane(o.k0);
  s.nk = __builtin_amdgcn_readfirstlane(o.nk);
  s.cap = __builtin_amdgcn_readfirstlane(o.cap);
  return s.seq >= 0;
}

// A workgroup's rows from row0 on: query and head (of the group) of its x-th. One
// division for them all; those of a lane by a product (group_inv).
struct PackedRows {
  int query, rest, group;
  uint32_t inv;
  template <typename T>
  __device__ __forceinline__ PackedRows(const PackedParams<T>& P, int row0) : group(P.group), inv(P.group_inv) {
    query = row0 / group;
    rest = row0 - query * group;
  }
  __device__ __forceinline__ void at(int x, int& q, int& head) const {
    const uint32_t y = rest + x, n = (y * inv) >> 21;
    q = query + n;
    head = y - n * group;
  }
};

// How the waves of a workgroup share its rows (for the keys' gradients: its keys) and the
// blocks that it walks: G groups of waves with tiles of their own, KS waves in each with
// the same tiles and a KS-th of a block. One group: its waves have staged rows of their own, and
// need no barrier.
template <int G, int KS, int BLOCK = KS == 1 ? 64 : 128>
struct PkForm {
  static constexpr int kG = G, kKS = KS, kWaves = G * KS, kThreads = 64 * kWaves;
  static constexpr bool kPrivate = G == 1;
  static constexpr int kBlock = BLOCK;                          // of all waves
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
};

// The kernel's arguments, read from memory where they are used (each packed kernel has them as its only ones).
template <typename T>
__device__ __forceinline__ const __attribute__((address_space(4))) PackedParams<T>* pk_late() {
  auto* p = (const __attribute__((address_space(4))) PackedParams<T>*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

template <typename T, int DP, int G, int KS>
struct PkFormOf {
  typedef PkForm<G, KS, KS == 1 || (KS == 2 && DP * sizeof(T) >= 512) ? 64 : 128> type;
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
// (buffer_load ... lds: a wave's 64 pieces side by side), one block after the other. Rows
// past the last and columns past d come as zeros, from past the resource's end: a weight of
// zero times what lies there must stay zero. WAVES waves share the work.
template <typename T, int DP, int ROWS, int WAVES>
struct PkCopy {
  typedef PkRows<T, DP> Rows;
  static constexpr int kRpi = 64 / Rows::kCh > 0 ? 64 / Rows::kCh : 1;  // rows of one instruction
  static constexpr int kG = 16 / kRpi;                                 // instructions of 16 rows
  static constexpr int kN = ROWS * Rows::kCh / 64 / WAVES;             // instructions of a wave
  static constexpr int kSub = kG > WAVES ? kG / WAVES : 1;             // distinct offsets of a lane
  static_assert(Rows::kCh <= 64 && ROWS % 16 == 0 && kN >= 1, "whole instructions");
  uint32_t off[kSub];
  uint32_t pitch;    // bytes between rows
  uint64_t from;     // address of the next block's first row
  int left, row;     // rows from there on; bytes of a row
  __device__ __forceinline__ void init(int64_t token, int d, int wave, int lane) {
    pitch = (uint32_t)(token * (int64_t)sizeof(T));
    row = d * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < kSub; ++i) {
      const int sub = WAVES >= kG ? wave % kG : wave + WAVES * i;
      const int r = sub * kRpi + lane / Rows::kCh;
      const int c = (lane % Rows::kCh) ^ Rows::f(r);
      off[i] = c * Rows::kE < d ? r * pitch + 16 * c : 0x80000000u;
    }
  }
  // begins at row row0 of the n at src
  __device__ __forceinline__ void begin(const T* src, int row0, int n) {
    from = (uint64_t)(uintptr_t)src + (uint64_t)row0 * pitch;
    left = n - row0;
  }
  // a block to `tile`; the next one is `step` rows on
  __device__ __forceinline__ void issue(unsigned char* tile, int wave, int step) {
    const uint32_t bytes = left <= 0 ? 0u : (uint32_t)((left < ROWS ? left : ROWS) - 1) * pitch + (uint32_t)row;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>((uintptr_t)from), (short)0, (int)bytes, 0x00020000);
    // their sums, kept through a loop, took more scalars than there are
    typedef __attribute__((address_space(3))) unsigned char lds_byte;
    uint32_t by = pitch, to = (uint32_t)(uintptr_t)(lds_byte*)tile;
    asm volatile("" : "+s"(by), "+s"(to));
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      // 16-row group and place of instruction `wave + WAVES i`
      const int group = WAVES >= kG ? wave / kG + i * (WAVES / kG) : i / kSub;
      const uint32_t o = off[WAVES >= kG ? 0 : i % kSub];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_byte*)(uintptr_t)(to + (wave + WAVES * i) * 1024), 16,
                                               o + (uint32_t)(16 * group) * by, 0, 0, 0);
    }
    from += (uint64_t)step * pitch;
    left -= step;
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

// A workgroup's accumulators to memory by way of LDS: 16 rows of each wave, then put(row,
// c, x) for each row of the groups and its 8 columns from c on, x being where they lie, the
// j-th wave's of a group j * kPart floats on. Few instructions, where each lane's stores
// to its own rows were most of a small call's time, and whole rows of memory.
template <typename Form, int DP>
struct PkOut {
  static constexpr int kPitch = DP + 4, kRows = 16 * Form::kG, kPart = kRows * kPitch;
  static constexpr int kBytes = Form::kKS * kPart * 4;
  template <int U, typename Put>
  __device__ static __forceinline__ void write(unsigned char* raw, const Form& f, int t, const f32x4 (&x)[U], Put put) {
    float* lds = reinterpret_cast<float*>(raw);
    const int li = t & 15, lg = (t >> 4) & 3;
    __syncthreads();
    float* mine = lds + f.part * kPart + (16 * f.group + li) * kPitch + 4 * lg;
#pragma unroll
    for (int u = 0; u < U; ++u) *reinterpret_cast<f32x4*>(mine + 16 * u) = x[u];
    __syncthreads();
#pragma unroll 1
    for (int i = t; i < kRows * (DP / 8); i += Form::kThreads) {
      const int row = i / (DP / 8), c = i % (DP / 8) * 8;
      put(row, c, lds + row * kPitch + c);
    }
  }
  // the sum of a group's waves
  __device__ static __forceinline__ f32x8 sum(const float* x) {
    f32x8 v = load8(x);
#pragma unroll
    for (int j = 1; j < Form::kKS; ++j) {
      const f32x8 o = load8(x + j * kPart);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += o[e];
    }
    return v;
  }
};

// The larger of two, NaN if either is: unlike fmaxf it takes values as they come, three at a
// time (17 -> 13 instructions for 16 scores and the lanes; 1 % of the forward pass).
__device__ __forceinline__ float pk_most(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// max over the 4 lanes {l % 16 + 16 g}
__device__ __forceinline__ float lanes4_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const uint32_t v = __builtin_bit_cast(uint32_t, pk_most(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return pk_most(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// launch(P, grid) for a call's workgroups: key/value heads, tiles and parts, in as many
// launches as a grid's second axis takes
template <typename T, typename F>
void pk_grid(PackedParams<T> P, F launch) {
  constexpr int kMost = 65535;
  for (P.tile0 = 0; P.tile0 < P.tiles; P.tile0 += kMost)
    launch(P, dim3(P.heads / P.group, P.tiles - P.tile0 < kMost ? P.tiles - P.tile0 : kMost, P.splits));
}

// f(G, KS, R) for the forms that packed_form chooses; float32 has one tile a wave
template <typename T, typename F>
void pk_form(const PackedForm& form, F f) {
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 4> Four;
  if (form.groups == 1) return f(One{}, Four{}, One{});
  if constexpr (sizeof(T) == 2) {
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
