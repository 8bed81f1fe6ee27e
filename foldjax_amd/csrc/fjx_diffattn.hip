// Differential attention, forward: one pass over the keys with the running
// maximum and sum of both softmaxes.
#include "fjx_diffattn.hpp"

namespace fjx {

namespace {

// A wave holds 16 query rows, lane l row l % 16 of them, and walks the keys in
// tiles of 16: S_t^T = K_t Q_t^T leaves the lane 4 keys of its own row a tile
// (keys 4 g + r, g = l / 16), so a row's maximum and sum are the lane's own
// values and two lane swaps, and the weights of two tiles are the operand of
// O_t^T = V^T P_t^T as they lie.
//
// The two outputs are subtracted at the end, where they may nearly cancel (two
// maps that are almost the same, lambda near one), so a bf16 weight would be
// rounded relative to a sum several times the result: weights go into the
// product as two bf16 parts.
// A weight may exceed 1 by up to 2^kSlack before the maximum is moved, which
// saves the outputs' rescaling in all but the first blocks of a row.
constexpr float kSlack = 8.f;

// What bounds it: vector instructions (an exponential, its fma and two bf16 parts
// a weight and map: 6 to a matrix instruction) and the matrix instructions, which
// on one SIMD run beside other waves' vector work only in part. 499 rows of 499
// tokens, 2 heads with their bias: 280 us (at the clock that the card has after a
// hundred passes, as all figures here), the SIMDs 60 % in vector and 29 % in matrix
// instructions; 245 rows of 245: 47 us, 45 and 18 %, a quarter of it the workgroups'
// starts and ends (4 blocks of keys each). One token of 8 sequences against 16384
// keys (134 MB, keywise and split): 25.7 us, the copy rate, and 4.8 for the join.
//
// KS 4 (keywise): the four waves share one 16-row tile and take 32 keys each of a
// 128-key block, for calls with few rows; KS 1: each has 16 rows of its own and
// walks every 64-key block.
template <typename T, int D, int KS>
__global__ __launch_bounds__((DaForm<KS>::kThreads), (kDaWaves<T, D> + (kDaWaves<T, D> > 1))) void diffattn_fwd_kernel(DiffAttnParams<T> P) {
  typedef DaForm<KS> Form;
  constexpr int kRows = Form::kBlock;          // keys of a block
  constexpr int kNt = kRows / KS / 16;         // key tiles of a wave in one
  // one block in LDS where the waves share it, for the sake of a second and third
  // workgroup on a CU (two blocks: 18.6 -> 23.5 us at 4 x 499 tokens)
  constexpr int kBufs = KS == 4 ? 1 : 2;
  constexpr int kC = D / 32, kU = 2 * D / 16;  // k-steps of a score, tiles of 16 values
  typedef typename Frag<T>::type F;
  typedef DaTile<T, D, kRows> Tile;
  constexpr size_t kMerge = Form::kWaves * 16 * 2 * (2 * D + 4) * sizeof(float);
  constexpr size_t kBytes = kBufs * sizeof(Tile);
  static_assert(KS == 1 || kBytes >= kMerge, "the waves' sums");
  __shared__ __attribute__((aligned(16))) unsigned char raw[kBytes];
  __shared__ __attribute__((aligned(16))) KeyFlags<kRows> flags[3];  // of the block at hand and the next two
  __shared__ float lams[Form::kWaves][16];  // of the waves' rows
  Tile* tiles = reinterpret_cast<Tile*>(raw);

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = P.heads / P.group;
  // 32 bits from here to the item: a launch has fewer than 2^23 workgroups
  const uint32_t nq = (uint32_t)P.nq, rows = P.group * nq;  // of one key/value head
  const uint32_t row_blocks = (rows + Form::kTiles * 16 - 1) / (Form::kTiles * 16);
  uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= (uint32_t)P.items * kvh * row_blocks * P.splits) return;
  const uint32_t rb = id % row_blocks;
  id /= row_blocks;
  const uint32_t split = id % (uint32_t)P.splits;
  id /= (uint32_t)P.splits;
  const int kv = id % (uint32_t)kvh;
  const int64_t item = id / (uint32_t)kvh;

  const int tile_of = wave % Form::kTiles, ks = wave / Form::kTiles;  // its tile of 16 rows, and its part of a block's keys
  const uint32_t row = (rb * Form::kTiles + tile_of) * 16 + li;
  const bool row_on = row < rows;
  const uint32_t row_c = row_on ? row : rows - 1;
  const int hg = row_c / nq;
  const uint32_t qi = row_c - hg * nq;
  const int head = kv * P.group + hg;

  DaStage<T, D, kRows, Form::kThreads> st;
  st.init(P.k.p + item * P.k.item + 2 * kv * P.k.head, P.k.head, P.k.token, P.v.p + item * P.v.item + kv * P.v.head,
          P.v.token, t);
  const uint8_t* mask = P.mask ? P.mask + item * P.nk : nullptr;
  const bool biased = P.bias.p != nullptr;
  const T* bias = P.bias.p + (biased ? (item / P.share) * P.bias.item + head * P.bias.head + qi * P.bias.token : 0);

  const int64_t blocks = (P.nk + kRows - 1) / kRows;
  const int64_t blk0 = split * P.split_blocks;
  const int64_t blk1 = blk0 + P.split_blocks < blocks ? blk0 + P.split_blocks : blocks;

  // The loads on which others wait go first: the mask, whose flags say which rows of
  // the block to load, then what the loop starts with; lambda's vectors come in
  // while the block does.
  // a block's flags in two steps: the mask on its way while a block is worked on
  uint8_t part = 0;
  auto look = [&](int64_t blk) {
    const int64_t k = blk * kRows + t;
    part = t < kRows && k < P.nk;
    if (part && mask) part = mask[k];
  };
  auto put_flags = [&](int at) {
    if (t < kRows) flags[at].set(t, part != 0);
  };
  const int key_w = kRows / KS * ks;  // this wave's keys of a block
  typename Quad<T>::type bv[kNt] = {};  // zeros without a bias
  auto load_bias = [&](int64_t blk) {
    bias_tile<T, kNt>(bias, blk * kRows + key_w + 4 * lg, P.nk, (blk + 1) * kRows <= P.nk, bv);
  };
  look(blk0);
  const uint8_t part0 = part;
  look(blk0 + 1);
  F qf[2][kC];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < kC; ++c)
      qf[m][c] = load8(P.q.p + item * P.q.item + (2 * head + m) * P.q.head + qi * P.q.token + 32 * c + 8 * lg);
  if (biased) load_bias(blk0);
  if (t < kRows) flags[0].set(t, part0 != 0);
  put_flags(1);
  __syncthreads();
  st.load(blk0 * kRows, flags[0].whole(), flags[0].on);
  // kept in LDS: in a register through the loop it was the one that spilled
  const float lam_own = da_lambda<D>(P.lam, P.heads, head, P.init, lane);
  if (lg == 0) lams[wave][li] = lam_own;

  // the sums of the weights: in bf16 a row of ones times their parts, on the
  // matrix cores, which have the time; lane l gets its own row's
  constexpr bool kOnes = sizeof(T) == 2;
  F ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = from_f32<T>(1.f);
  float m[2] = {-INFINITY, -INFINITY};
  f32x4 l[2], o[2][kU];
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) {
    l[mp] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kU; ++u) o[mp][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  st.store(tiles[0]);
  __syncthreads();

  int cur = 0;  // the block's flags
  for (int64_t blk = blk0; blk < blk1; ++blk) {
    const int buf = kBufs == 2 ? (int)(blk - blk0) & 1 : 0;
    const Tile& tile = tiles[buf];
    const bool more = blk + 1 < blk1;
    const int next = cur == 2 ? 0 : cur + 1;
    f32x4 b[kNt];
#pragma unroll
    for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) b[kt][r] = to_f32(bv[kt][r]) * bias_unit<T>(P.inv_scale);
    flags[cur].apply(key_w, lg, b);
    if (more) {
      st.load((blk + 1) * kRows, flags[next].whole(), flags[next].on);
      if (biased) load_bias(blk + 1);
      look(blk + 2);
    }
    const int after = next == 2 ? 0 : next + 1;
    cur = next;
    f32x4 s[2][kNt];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
      for (int mp = 0; mp < 2; ++mp) {
        s[mp][kt] = score_start<T>(b[kt]);
#pragma unroll
        for (int c = 0; c < kC; ++c) mma(s[mp][kt], load8(&tile.a[key_w + 16 * kt + li][D * mp + 32 * c + 8 * lg]), qf[mp][c]);
      }
#pragma unroll
    for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
      for (int mp = 0; mp < 2; ++mp)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (!kBiasFirst<T>) s[mp][kt][r] = fmaf(s[mp][kt][r], P.scale_log2, b[kt][r]);
          top[mp] = fmaxf(top[mp], s[mp][kt][r]);
        }
    top[0] = group_max(top[0]) * (kBiasFirst<T> ? P.scale_log2 : 1.f);
    top[1] = group_max(top[1]) * (kBiasFirst<T> ? P.scale_log2 : 1.f);
    if (__builtin_amdgcn_ballot_w64(top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
#pragma unroll
      for (int mp = 0; mp < 2; ++mp) {
        const float mn = fmaxf(m[mp], top[mp]);
        const float alpha = __builtin_amdgcn_exp2f(m[mp] - exponent_base(mn));  // 0 where no key was before
        m[mp] = mn;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          l[mp][r] *= alpha;
#pragma unroll
          for (int u = 0; u < kU; ++u) o[mp][u][r] *= alpha;
        }
      }
    }
    const float bases[2] = {exponent_base(m[0]), exponent_base(m[1])};
    float by = P.scale_log2;
    if (kBiasFirst<T>) {
      const bool far = __builtin_amdgcn_ballot_w64(fmaxf(fabsf(bases[0]), fabsf(bases[1])) > kFar);
      by = far_scores(far, by, s[0]);
      far_scores(far, P.scale_log2, s[1]);
    }
    F pf[2][kNt / 2][kParts<T>];
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      const float base = bases[mp];
      float p[kNt / 2][8];
#pragma unroll
      for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(kBiasFirst<T> ? fmaf(s[mp][kt][r], by, -base) : s[mp][kt][r] - base);
          if (!kOnes) l[mp][r] += e;
          p[kt >> 1][4 * (kt & 1) + r] = e;
        }
#pragma unroll
      for (int c = 0; c < kNt / 2; ++c) {
        parts(p[c], pf[mp][c]);
        if (kOnes) mma_parts(l[mp], ones, pf[mp][c]);
      }
    }
#pragma unroll
    for (int c = 0; c < kNt / 2; ++c)
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const F v = col_frag(&tile.b[0][0], Tile::kPitch, key_w + 32 * c, 16 * u, lane);
        mma_parts(o[0][u], v, pf[0][c]);
        mma_parts(o[1][u], v, pf[1][c]);
      }
    if (kBufs == 1) __syncthreads();
    if (more) {
      st.store(tiles[kBufs == 2 ? buf ^ 1 : 0]);
      put_flags(after);
    }
    __syncthreads();
  }
  float ls[2];
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) ls[mp] = kOnes ? l[mp][0] : group_sum((l[mp][0] + l[mp][1]) + (l[mp][2] + l[mp][3]));

  constexpr int kOwn = kU / KS;
  const int u0 = ks * kOwn;
  if constexpr (KS > 1) {
    // the partial rows of the waves that share them, on the largest of their maxima
    constexpr int kPo = 2 * D + 2;
    float* ml = reinterpret_cast<float*>(raw);       // [wave][map][row][2]
    float* po = ml + Form::kWaves * 2 * 16 * 2;      // [wave][map][row][2 D + 2]
    auto slot = [&](int j, int mp) { return ((Form::kTiles * j + tile_of) * 2 + mp) * 16 + li; };  // of the tile's j-th wave
    if (lg == 0)
      for (int mp = 0; mp < 2; ++mp) {
        ml[slot(ks, mp) * 2] = m[mp];
        ml[slot(ks, mp) * 2 + 1] = ls[mp];
      }
    __syncthreads();
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      float mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) mx = fmaxf(mx, ml[slot(j, mp) * 2]);
      const float base = exponent_base(mx);
#pragma unroll
      for (int j = 0; j < KS; ++j) sum = fmaf(ml[slot(j, mp) * 2 + 1], __builtin_amdgcn_exp2f(ml[slot(j, mp) * 2] - base), sum);
      const float alpha = __builtin_amdgcn_exp2f(m[mp] - base);
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) po[slot(ks, mp) * kPo + 16 * u + 4 * lg + r] = o[mp][u][r] * alpha;
      m[mp] = mx;
      ls[mp] = sum;
    }
    __syncthreads();
    // each wave takes its share of the tiles of 16 values
#pragma unroll
    for (int mp = 0; mp < 2; ++mp)
#pragma unroll
      for (int u = 0; u < kOwn; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float a = 0.f;
#pragma unroll
          for (int j = 0; j < KS; ++j) a += po[slot(j, mp) * kPo + 16 * (u0 + u) + 4 * lg + r];
          o[mp][u][r] = a;
        }
  }
  if (!row_on) return;
  const bool first = lg == 0 && ks == 0;
  const int64_t at = item * P.heads * P.nq + (int64_t)head * P.nq + qi;
  if (P.splits > 1) {
    const int64_t base = (split * (P.items * P.heads * P.nq) + at) * 2;
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      if (first) *reinterpret_cast<f32x2*>(P.part_ml + (base + mp) * 2) = f32x2{m[mp], ls[mp]};
#pragma unroll
      for (int u = 0; u < kOwn; ++u)
        *reinterpret_cast<f32x4*>(P.part_o + (base + mp) * (2 * D) + 16 * (u0 + u) + 4 * lg) = o[mp][u];
    }
    return;
  }
  float inv[2];
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) {
    inv[mp] = ls[mp] == 0.f ? 0.f : 1.f / ls[mp];  // a row without keys is zeros
    if (first && P.stats)  // +inf for such a row: its weights are zeros in the backward pass as well
      P.stats[(item * 2 * P.heads + 2 * head + mp) * P.nq + qi] = ls[mp] == 0.f ? INFINITY : m[mp] + log2f(ls[mp]);
  }
  inv[1] *= lams[wave][li];
  T* out = P.out.p + item * P.out.item + head * P.out.head + qi * P.out.token;
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = o[0][u][r] * inv[0] - o[1][u][r] * inv[1];
    store4f(out + 16 * (u0 + u) + 4 * lg, v);
  }
}

// The splits of a row joined: a workgroup a row, wave w taking every fourth
// split from w on for both maps, lane l holding 2 D / 64 values.
template <typename T, int D>
__global__ __launch_bounds__(256) void diffattn_join_kernel(DiffAttnParams<T> P) {
  constexpr int kV = 2 * D / 64;
  __shared__ float lds_o[4][2][2 * D];
  __shared__ float lds_l[4][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = P.items * P.heads * P.nq, at = blockIdx.x;
  const int64_t qi = at % P.nq, ih = at / P.nq;
  const int head = (int)(ih % P.heads);
  const int64_t item = ih / P.heads;
  float base[2], mx[2] = {-INFINITY, -INFINITY};
  for (int s = lane; s < P.splits; s += 64) {
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) mx[mp] = fmaxf(mx[mp], P.part_ml[((s * rows + at) * 2 + mp) * 2]);
  }
  const float lam = da_lambda<D>(P.lam, P.heads, head, P.init, lane);
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) {
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) mx[mp] = fmaxf(mx[mp], shfl_xor(mx[mp], x));
    base[mp] = exponent_base(mx[mp]);
  }
  float l[2] = {0.f, 0.f}, o[2][kV] = {};
#pragma unroll 8
  for (int s = wave; s < P.splits; s += 4) {
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      const int64_t i = (s * rows + at) * 2 + mp;
      const f32x2 v = *reinterpret_cast<const f32x2*>(P.part_ml + i * 2);
      const float w = __builtin_amdgcn_exp2f(v[0] - base[mp]);
      l[mp] = fmaf(v[1], w, l[mp]);
#pragma unroll
      for (int j = 0; j < kV; ++j) o[mp][j] = fmaf(P.part_o[i * (2 * D) + 64 * j + lane], w, o[mp][j]);
    }
  }
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) {
    if (lane == 0) lds_l[wave][mp] = l[mp];
#pragma unroll
    for (int j = 0; j < kV; ++j) lds_o[wave][mp][64 * j + lane] = o[mp][j];
  }
  __syncthreads();
  if (wave) return;
  float res[kV] = {};
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) {
    const float sum = (lds_l[0][mp] + lds_l[1][mp]) + (lds_l[2][mp] + lds_l[3][mp]);
    const float inv = (sum == 0.f ? 0.f : 1.f / sum) * (mp ? -lam : 1.f);
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const int x = 64 * j + lane;
      res[j] = fmaf((lds_o[0][mp][x] + lds_o[1][mp][x]) + (lds_o[2][mp][x] + lds_o[3][mp][x]), inv, res[j]);
    }
    if (lane == 0 && P.stats)
      P.stats[(item * 2 * P.heads + 2 * head + mp) * P.nq + qi] = sum == 0.f ? INFINITY : base[mp] + log2f(sum);
  }
  T* out = P.out.p + item * P.out.item + head * P.out.head + qi * P.out.token;
#pragma unroll
  for (int j = 0; j < kV; ++j) out[64 * j + lane] = from_f32<T>(res[j]);
}

template <typename T, int D, int KS>
void fwd_form(const DiffAttnParams<T>& P, hipStream_t st) {
  constexpr int kTile = DaForm<KS>::kTiles * 16;
  const int64_t blocks = P.items * (P.heads / P.group) * P.splits * ((P.group * P.nq + kTile - 1) / kTile);
  diffattn_fwd_kernel<T, D, KS><<<(unsigned)((blocks + 7) / 8 * 8), DaForm<KS>::kThreads, 0, st>>>(P);
}

template <typename T, int D>
void fwd(const DiffAttnParams<T>& P, bool keywise, hipStream_t st) {
  if (keywise) {
    fwd_form<T, D, 4>(P, st);
    if (P.splits > 1) diffattn_join_kernel<T, D><<<(unsigned)(P.items * P.heads * P.nq), 256, 0, st>>>(P);
    return;
  }
  fwd_form<T, D, 1>(P, st);
}

}  // namespace

template <typename T>
void launch_diffattn_fwd(const DiffAttnParams<T>& P, int d, bool keywise, hipStream_t st) {
  if (d == 32)
    fwd<T, 32>(P, keywise, st);
  else
    fwd<T, 64>(P, keywise, st);
}
template void launch_diffattn_fwd<bf16>(const DiffAttnParams<bf16>&, int, bool, hipStream_t);
template void launch_diffattn_fwd<float>(const DiffAttnParams<float>&, int, bool, hipStream_t);

}  // namespace fjx
