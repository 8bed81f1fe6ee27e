// How a call of packed attention is cut into workgroups: rules on its counts of sequences,
// tokens and heads, its width and type. Host only but for the types that the kernels share,
// standard headers only.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace fjx {

constexpr int kPackedOrder = 12288, kPackedOrderSeqs = 1023;  // tiles that are sorted at most, and their sequences

// a tile of a sequence: first query, queries, first key, keys, and keys with the unused
// ones behind them. Sequence `seqs`: the rows behind the last one
struct alignas(16) PackedTile {
  int seq, tile, q0, nq, k0, nk, cap, pad;
};

// how a call is cut (PkForm), 16-row tiles of a wave
struct PackedForm {
  int groups, ks, tiles;
  int count;          // tiles for one key/value head
  PackedTile* order;  // [count], to be filled with the tiles in the order of their work, or null
  constexpr int rows() const { return 16 * groups * tiles; }  // of a workgroup
};

// How a call is cut. The host knows how many sequences and tokens there are, not how
// long each is: the rules take all lengths as alike.
struct PackedPlan {
  PackedForm rows, keys;
  int splits;                // of the keys (forward, keywise), of the heads that share keys (dk, dv)
  size_t part_o, part_ml;    // workspace bytes: forward; backward: one of dk, dv and D
  int part_rows;
  size_t rows_order, keys_order;
};

inline size_t packed_bytes(size_t n) { return (n + 255) / 256 * 256; }  // a workspace's parts begin at multiples of 256
inline int packed_width(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
// `wgs`: workgroups of 64 rows (keys) there are, `walk`: keys (rows) that one walks;
// `few`: so few wgs are one wave's rows with its own keys each; `pairs`: from so many on a
// wave has two tiles; `alone`: from so many on also all keys of a block. us by form, KS 4 /
// KS 2 / KS 1 with one tile / KS 2 / KS 1 with two:
//   forward  126 workgroups 1003 keys d 64         8.7 / 10.9 / 14.6 / 15.6 / 20.5
//            216            851       128         21.0 / 15.4 / 19.4 / 22.2 / 27.6
//            258            686        64         17.5 / 13.4 / 16.4 / 16.0 / 20.8
//            496            245        24         14.1 /  9.4 /  8.9 / 10.3 / 10.2
//            520            4099      128          107 / 56.6 / 64.9 / 64.1 / 87.9
//           1024            1638      128          160 / 83.4 / 75.9 / 70.8 / 96.1
//           2048            2730      128          586 /  296 /  264 /  230 /  219
//           4096            8192       64          641 /  370 /  349 /  301 /  295
//   dk, dv (the backward pass with them, dq's form the same)
//           1016            4049       64          251 /  202 /  238 /  216 /  231
//           1024            4096       64         1101 /  849 / 1035 /  889 / 1182
//           4096            8192       64         1580 / 1177 / 1135 / 1122 / 1090
//   float32  132            701        64           36 /   39 /   42
//            256            2048      128          107 /  144 /  148
//            456            1774      128          163 /  147 /  149
// (rows of several long sequences sorted). Where `pairs` and `alone` lie, KS 2 with one / KS 2 /
// KS 1 with two tiles, four sequences, causal and all keys (d 128: 8 heads, d 64: 16 on 4):
//   forward  640  d 128    43 /  45 /  59   68 /  60 /  66
//            768           57 /  55 /  74   90 /  81 /  77
//           1024           86 /  70 /  95  145 / 135 / 126
//           1536          167 / 130 / 144  287 / 226 / 211
//           2048          269 / 209 / 198  503 / 386 / 402
//            768  d 64     21 /  21 /  28   31 /  29 /  34
//           1024           30 /  33 /  41   48 /  46 /  52
//           1280           40 /  40 /  50   64 /  60 /  65
//           2048           79 /  67 /  78  138 / 127 / 132
//           3200          167 / 138 / 138  321 / 260 / 256
//           4096          262 / 218 / 210  494 / 404 / 413
//   dq (the backward pass with it)
//            768  d 128   167 / 169 / 194  272 / 265 / 259
//           2048          841 / 785 / 766  1590 / 1492 / 1501
//           1280  d 64    128 / 131 / 137  202 / 202 / 206
//           2048          247 / 253 / 249  448 / 459 / 454
//           3200          530 / 537 / 510  979 / 974 / 943
// Up to d 64 two tiles begin to pay at 1280 to 2048 where it is causal and at 640 to 768 with all
// keys, which a workspace's size does not know: 1024 lies between (all keys, d 24, 1264: 54 / 48).
inline PackedForm packed_form(int64_t rows, int64_t seqs, int64_t wgs, int64_t walk, int64_t few, int64_t pairs, int64_t alone) {
  PackedForm f = {};
  f.groups = 4;
  f.tiles = 1;
  if (walk > 64 && (rows <= 16 * seqs || wgs < few))
    f.groups = 1, f.ks = 4;
  else if (walk < 320 || wgs < 128)
    f.ks = 1;
  else if (wgs < pairs)
    f.ks = 2;
  else
    f.ks = wgs < alone ? 2 : 1, f.tiles = 2;
  f.count = (int)std::min<int64_t>(rows / f.rows() + seqs + 1, 1 << 30);
  return f;
}
// Sorting the tiles by their work takes a launch, 4 us: for calls of several sequences
// that walk 16384 blocks of 64 and more in all (the forward pass of 5 causal sequences,
// 8192 tokens, 85 -> 77 us with it, of 6 with 16384 254 -> 234)
inline bool packed_sorted(const PackedForm& f, int64_t seqs, int64_t wgs, int64_t walk) {
  return f.groups > 1 && f.count && f.count <= kPackedOrder && seqs > 1 && seqs <= kPackedOrderSeqs && wgs * walk >= (int64_t)16384 * 64;
}
inline int64_t packed_few(bool bf, int64_t d) { return bf ? 128 : d <= 64 ? 256 : 384; }
inline int64_t packed_pairs(bool bf, int64_t d) { return !bf ? INT64_MAX : d <= 64 ? 1024 : 768; }
inline PackedPlan packed_fwd_plan(int64_t tq, int64_t tk, int64_t seqs, int64_t heads, int64_t kvh, int64_t d, bool bf) {
  const int64_t group = heads / kvh, rows = tq * group, wgs = kvh * ((rows + 63) / 64), walk = tk / seqs;
  PackedPlan p = {};
  p.rows = packed_form(rows, seqs, wgs, walk, packed_few(bf, d), packed_pairs(bf, d), d <= 64 ? 3200 : 2048);
  p.splits = 1;
  if (p.rows.groups == 1) {
    const int64_t tiles = kvh * std::max(seqs, rows / 16);
    // two blocks of 128 keys a split at least, were the lengths alike
    const int64_t want = tiles <= 128 ? std::min<int64_t>(512 / tiles, walk / 256) : 1;
    if (want > 1) {
      p.splits = (int)want;
      const size_t r = (size_t)heads * tq * p.splits;
      p.part_o = packed_bytes(r * packed_width(d) * sizeof(float));
      p.part_ml = packed_bytes(r * 3 * sizeof(float));  // maxima and sums, and the statistics' sums
    }
  }
  if (packed_sorted(p.rows, seqs, wgs, walk)) p.rows_order = packed_bytes((size_t)p.rows.count * sizeof(PackedTile));
  return p;
}
inline PackedPlan packed_bwd_plan(int64_t tq, int64_t tk, int64_t seqs, int64_t heads, int64_t kvh, int64_t d, bool bf) {
  const int64_t group = heads / kvh, rows = tq * group, wgs = kvh * ((rows + 63) / 64), walk = tk / seqs;
  const int64_t key_wgs = kvh * ((tk + 63) / 64);
  PackedPlan p = {};
  p.splits = 1;
  // Workgroups that walk long and, causal, uneven ways: the heads that share keys in parts, of
  // an eighth of a workgroup's share of the card (of 128 channels one a CU, else two) were the
  // lengths alike. us of the backward pass with every tile in 4 parts / with parts of a half /
  // an eighth / a 16th, causal: 8192 tokens in 5 sequences, d 128 (2 parts: 283)  291 / 316 /
  // 270 / 270; one sequence of 8192, d 64  353 / 384 / 330 / 332; 4099 and 4000, d 64
  // 199 / 210 / 188 / 187; one of 1003, d 64  30.4 / 32 / 31.0 / 31
  if (group > 1 && tk && key_wgs < 1024) {
    p.splits = (int)std::min(group, std::max<int64_t>(2, (1024 + key_wgs - 1) / key_wgs));
    p.part_rows = (int)std::max<int64_t>(256, tq * group / seqs * key_wgs / (d > 64 ? 256 : 512) / 8);
  }
  if (tq) p.rows = packed_form(rows, seqs, wgs, walk, packed_few(bf, d), packed_pairs(bf, d), 2048);
  // two tiles of keys a wave would take more registers than two waves a SIMD have at 128 channels
  if (tk) p.keys = packed_form(tk, seqs, key_wgs * p.splits, tq / seqs, packed_few(bf, d),
                                bf && d <= 64 ? 2048 : INT64_MAX, 0);
  if (p.splits > 1) p.part_o = packed_bytes((size_t)p.splits * kvh * tk * packed_width(d) * sizeof(float));
  p.part_ml = packed_bytes((size_t)heads * tq * sizeof(float));
  if (packed_sorted(p.rows, seqs, wgs, walk)) p.rows_order = packed_bytes((size_t)p.rows.count * sizeof(PackedTile));
  if (packed_sorted(p.keys, seqs, key_wgs * group, tq / seqs)) p.keys_order = packed_bytes((size_t)p.keys.count * sizeof(PackedTile));
  return p;
}

}  // namespace fjx
