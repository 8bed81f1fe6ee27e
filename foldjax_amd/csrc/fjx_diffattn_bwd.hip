// Differential attention, backward. With dP = dO v^T and
//   D_t = rowsum(P_t dP),  dS_1 = P_1 (dP - D_1),  dS_2 = -lambda P_2 (dP - D_2):
//   dq_t = scale dS_t k_t,  dk_t = scale dS_t^T q_t,  dv = (P_1 - lambda P_2)^T dO,
//   dbias = dS_1 + dS_2,  dlambda = -sum D_2
// The weights come again from the scores and the forward pass's row statistics
// L_t = log2 sum 2^x: P_t = 2^(x - L_t). L's own rounding is a factor of all of a row's
// weights: 1e-6 of them at |L| = 32, but of the order of 1 under the biases of -1e5 and
// beyond that masks add to whole rows (where L is the maximum alone, and the weights
// add up to the number of keys). So the kernel for dq divides by the sum of P_t, and
// leaves it for the others, which divide too wherever a row has |L| > kFarSum. Every
// sum has one owner and one order: no atomics, and the same bits each time.
//
// dS's rows sum to zero, so its products may cancel: like the weights it goes
// into them as two bf16 parts, and a gradient is off by its own rounding. With
// one part dq and dk were off by 1.4 times as much (1.5 at a few keys).
#include "fjx_diffattn.hpp"

namespace fjx {

namespace {

constexpr float kFarSum = 256.f;  // there the factor is 1 + 5e-6
// |L| beyond `most`, and not for want of keys
__device__ __forceinline__ bool row_far(float L, float most) { return fabsf(L) > most && L < INFINITY; }

// sums of the scores of the wave's 16 rows and NT key tiles from row `key_w` of a
// block on, one map; b: bias in its unit
template <typename T, int D, int ROWS, int NT>
__device__ __forceinline__ void tile_scores(const DaTile<T, D, ROWS>& tile, int mp, int key_w,
                                            const typename Frag<T>::type (&qf)[D / 32], const f32x4 (&b)[NT], int li, int lg,
                                            f32x4 (&s)[NT]) {
#pragma unroll
  for (int kt = 0; kt < NT; ++kt) {
    s[kt] = score_start<T>(b[kt]);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) mma(s[kt], load8(&tile.a[key_w + 16 * kt + li][D * mp + 32 * c + 8 * lg]), qf[c]);
  }
}

// the weights in their place
template <typename T, int NT>
__device__ __forceinline__ void to_weights(const f32x4 (&b)[NT], float scale_log2, float L, f32x4 (&s)[NT]) {
#pragma unroll
  for (int kt = 0; kt < NT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) s[kt][r] = __builtin_amdgcn_exp2f(exponent<T>(s[kt][r], b[kt][r], scale_log2, L));
}

// dP of the same
template <typename T, int D, int ROWS, int NT>
__device__ __forceinline__ void tile_dp(const DaTile<T, D, ROWS>& tile, int key_w, const typename Frag<T>::type (&dof)[2 * D / 32],
                                        int li, int lg, f32x4 (&dp)[NT]) {
#pragma unroll
  for (int kt = 0; kt < NT; ++kt) {
    dp[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 2 * D / 32; ++c) mma(dp[kt], load8(&tile.b[key_w + 16 * kt + li][32 * c + 8 * lg]), dof[c]);
  }
}

__device__ __forceinline__ float sum8(const float (&x)[8]) {
  return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

// dq and D_t in one walk over the keys. A wave holds 16 query rows (lane l row
// l % 16) as in the forward pass. D_t is known only at the end, so two sums
// are kept, U = sum P_t (dP - c_t) k and W = sum P_t k, and
//   dq_t = scale (U - (D_t - c_t) W) / sum P_t
// whatever c_t is; D_t - c_t comes from the sum of P_t (dP - c_t). (The weights'
// own sum is one but for the rounding of L; lambda's gradient is the sum of all D_2,
// of either sign, and shows what they have in common.) But the two terms cancel,
// down to their operands' bits, unless c_t is near D_t: where one key has nearly
// all the weight dq is what the others have left of it. So c_t is the mean of dP
// under map t over the keys so far, moved before a block's own terms are formed,
//   c -> c + e:  U -> U - e W,  sum P (dP - c) -> less e sum P,
// until the keys it is taken from have kEnough of the weight: with A of it, it is
// within sum P |dP - D| / A of D, and what is lost is 1 / A of the rounding of dS
// itself. Rows are mostly there after a block or two; the waves that share a row each
// have a centre of their own keys, joined at the end. (c is subtracted from dP here:
// as the start of dP's accumulators it left D_2 off by 1e-6 in common.) Against a
// first walk for D_t alone this trades a second set of scores, dP and exponentials
// for the products W, half the time. W takes two bf16 parts as well.
// Bound like the forward kernel, with two waves a SIMD (256 registers; at 64 channels
// one): 69 us at 245 rows of 245 tokens and 2 heads, 50 % vector and 13 % matrix
// instructions, a quarter of it starts and ends; 23 us at 4 x 499 tokens and 6 heads (62
// and 19 with one centre of the first block for both maps, which lost dq's digits in
// rows of one heavy key, and without far rows). 64 of a block's vector instructions are
// copies still: the sums of P and P (dP - c) come after parts() has overwritten them.
//
// KS 4: the four waves share 16 rows and take 32 keys each of a 128-key block, for
// calls with few rows; KS 1: each has rows of its own.
constexpr float kEnough = 1.f / 16;

template <typename T, int D, int KS>
__global__ __launch_bounds__((DaForm<KS>::kThreads), (D == 32 ? 2 : 1)) void diffattn_dq_kernel(DiffAttnParams<T> P) {
  typedef DaForm<KS> Form;
  constexpr int kRows = Form::kBlock, kNt = kRows / KS / 16, kBufs = KS == 4 ? 1 : 2;
  constexpr int kC = D / 32, kU = D / 16;
  typedef typename Frag<T>::type F;
  typedef DaTile<T, D, kRows> Tile;
  constexpr int kPo = D + 2;
  static_assert(KS == 1 || kBufs * sizeof(Tile) >= Form::kWaves * 2 * 16 * kPo * sizeof(float), "the waves' sums");
  __shared__ __attribute__((aligned(16))) Tile tiles[kBufs];
  __shared__ __attribute__((aligned(16))) KeyFlags<kRows> flags[3];  // of the block at hand and the next two
  __shared__ float lams[Form::kWaves][16];  // of the waves' rows
  __shared__ float joined[Form::kWaves][2][3][16];  // of the waves' rows and maps: center, weight, off

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = P.heads / P.group;
  const uint32_t nq = (uint32_t)P.nq, rows = P.group * nq, row_blocks = (rows + Form::kTiles * 16 - 1) / (Form::kTiles * 16);
  uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= (uint32_t)P.items * kvh * row_blocks) return;
  const uint32_t rb = id % row_blocks;
  id /= row_blocks;
  const int kv = id % (uint32_t)kvh;
  const int64_t item = id / (uint32_t)kvh;
  const int tile_of = wave % Form::kTiles, ks = wave / Form::kTiles;  // its tile of 16 rows, and its part of a block's keys
  const uint32_t row = (rb * Form::kTiles + tile_of) * 16 + li;
  const bool row_on = row < rows;
  const uint32_t row_c = row_on ? row : rows - 1;
  const int hg = row_c / nq;
  const uint32_t qi = row_c - hg * nq;
  const int head = kv * P.group + hg;
  const int key_w = kRows / KS * ks;  // this wave's keys of a block

  DaStage<T, D, kRows, Form::kThreads> st;
  st.init(P.k.p + item * P.k.item + 2 * kv * P.k.head, P.k.head, P.k.token, P.v.p + item * P.v.item + kv * P.v.head,
          P.v.token, t);
  const uint8_t* mask = P.mask ? P.mask + item * P.nk : nullptr;
  const bool biased = P.bias.p != nullptr;
  const T* bias = P.bias.p + (biased ? (item / P.share) * P.bias.item + head * P.bias.head + qi * P.bias.token : 0);

  // as in the forward kernel: the mask's loads, on which the block's wait, go first
  uint8_t part = 0;
  auto look = [&](int64_t blk) {
    const int64_t k = blk * kRows + t;
    part = t < kRows && k < P.nk;
    if (part && mask) part = mask[k];
  };
  auto put_flags = [&](int at) {
    if (t < kRows) flags[at].set(t, part != 0);
  };
  typename Quad<T>::type bv[kNt] = {};  // zeros without a bias
  const int64_t blocks = (P.nk + kRows - 1) / kRows;
  auto load_bias = [&](int64_t blk) {
    bias_tile<T, kNt>(bias, blk * kRows + key_w + 4 * lg, P.nk, (blk + 1) * kRows <= P.nk, bv);
  };
  look(0);
  const uint8_t part0 = part;
  look(1);
  F qf[2][kC], dof[2 * kC];
  float L[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    L[m] = P.saved[(item * 2 * P.heads + 2 * head + m) * P.nq + qi];
#pragma unroll
    for (int c = 0; c < kC; ++c)
      qf[m][c] = load8(P.q.p + item * P.q.item + (2 * head + m) * P.q.head + qi * P.q.token + 32 * c + 8 * lg);
  }
#pragma unroll
  for (int c = 0; c < 2 * kC; ++c)
    dof[c] = load8(P.dout.p + item * P.dout.item + head * P.dout.head + qi * P.dout.token + 32 * c + 8 * lg);
  if (biased) load_bias(0);
  if (t < kRows) flags[0].set(t, part0 != 0);
  put_flags(1);
  __syncthreads();
  st.load(0, flags[0].whole(), flags[0].on);
  const float lam_own = da_lambda<D>(P.lam, P.heads, head, P.init, lane);  // kept in LDS, as there
  if (lg == 0) lams[wave][li] = lam_own;

  // of each map: c_t, the lane's sums of P and of P (dP - c), and whether c_t is to
  // move yet (not in a row without keys, to the end in a far one, whose weights are not
  // yet divided by their sum)
  float center[2] = {0.f, 0.f}, weight[2] = {0.f, 0.f}, off[2] = {0.f, 0.f};
  bool moves[2] = {L[0] < INFINITY, L[1] < INFINITY};
  const bool far = __builtin_amdgcn_ballot_w64(row_far(L[0], kFar) || row_far(L[1], kFar));
  f32x4 us[2][kU], ws[2][kU];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int u = 0; u < kU; ++u) us[m][u] = ws[m][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  st.store(tiles[0]);
  __syncthreads();
  uint32_t row_e = row_c;
  asm("" : "+v"(row_e));
  int at = 0;
  for (int64_t blk = 0; blk < blocks; ++blk) {
    const int buf = kBufs == 2 ? (int)blk & 1 : 0;
    const Tile& tile = tiles[buf];
    const bool more = blk + 1 < blocks;
    const int next = at == 2 ? 0 : at + 1;
    f32x4 b[kNt];
#pragma unroll
    for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) b[kt][r] = to_f32(bv[kt][r]) * bias_unit<T>(P.inv_scale);
    flags[at].apply(key_w, lg, b);
    if (more) {
      st.load((blk + 1) * kRows, flags[next].whole(), flags[next].on);
      if (biased) load_bias(blk + 1);
      look(blk + 2);
    }
    const int after = next == 2 ? 0 : next + 1;
    at = next;
    f32x4 dp[kNt], p[2][kNt];
    tile_dp<T, D, kRows, kNt>(tile, key_w, dof, li, lg, dp);
#pragma unroll
    for (int m = 0; m < 2; ++m) tile_scores<T, D, kRows, kNt>(tile, m, key_w, qf[m], b, li, lg, p[m]);
    float by = P.scale_log2;
    if (kBiasFirst<T>) {
      far_scores(far, P.scale_log2, p[0]);
      by = far_scores(far, P.scale_log2, p[1]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) to_weights<T>(b, by, L[m], p[m]);
    if (__builtin_amdgcn_ballot_w64(moves[0] || moves[1])) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float sp = 0.f, sd = 0.f;
#pragma unroll
        for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sp += p[m][kt][r];
            sd = fmaf(p[m][kt][r], dp[kt][r] - center[m], sd);
          }
        sp = group_sum(sp + weight[m]);
        sd = group_sum(sd);
        // the keys before it add nothing to sd: c_t is their mean
        const float move = moves[m] && sp > 0.f ? sd / sp : 0.f;
        moves[m] = moves[m] && !(sp >= kEnough && fabsf(L[m]) <= kFarSum);
        center[m] += move;
        off[m] = fmaf(-move, weight[m], off[m]);
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) us[m][u][r] = fmaf(-move, ws[m][u][r], us[m][u][r]);
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < kNt / 2; ++c) {
        float u8[8], w8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w8[e] = p[m][2 * c + (e >> 2)][e & 3];
          u8[e] = w8[e] * (dp[2 * c + (e >> 2)][e & 3] - center[m]);
        }
        off[m] += sum8(u8);
        weight[m] += sum8(w8);
        F uf[kParts<T>], wf[kParts<T>];
        parts(u8, uf);
        parts(w8, wf);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const F kf = col_frag(&tile.a[0][D * m], Tile::kPitch, key_w + 32 * c, 16 * u, lane);
          mma_parts(us[m][u], kf, uf);
          mma_parts(ws[m][u], kf, wf);
        }
      }
    if (kBufs == 1) __syncthreads();
    if (more) {
      st.store(tiles[kBufs == 2 ? buf ^ 1 : 0]);
      put_flags(after);
    }
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    off[m] = group_sum(off[m]);
    weight[m] = group_sum(weight[m]);
  }
  if constexpr (KS > 1) {  // the waves' sums, through the tiles' memory
    if (lg == 0)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        joined[wave][m][0][li] = center[m];
        joined[wave][m][1][li] = weight[m];
        joined[wave][m][2][li] = off[m];
      }
    __syncthreads();
    // all the keys' weight, and their sum of P (dP - c) around this wave's centre
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      weight[m] = off[m] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const float (&of)[3][16] = joined[Form::kTiles * j + tile_of][m];
        weight[m] += of[1][li];
        off[m] += fmaf(of[1][li], of[0][li] - center[m], of[2][li]);
      }
    }
  }
  // the row's head and query again: through the loop they took the registers that a
  // second wave a SIMD needs
  const uint32_t hg_e = row_e / nq, qi_e = row_e - hg_e * nq;
  const int head_e = kv * P.group + hg_e;
  float by[2];  // dq's factors; and D_t - c_t in `off`
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    weight[m] = weight[m] > 0.f ? 1.f / weight[m] : 0.f;  // a row without keys is zeros
    off[m] *= weight[m];
    by[m] = P.scale * weight[m] * (m ? -lams[wave][li] : 1.f);
  }
  if constexpr (KS > 1) {
    float* po = reinterpret_cast<float*>(&tiles[0]);  // [wave][map][row][D + 2]
    auto slot = [&](int j, int m) { return (((Form::kTiles * j + tile_of) * 2 + m) * 16 + li) * kPo; };  // of the tile's j-th wave
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) po[slot(ks, m) + 16 * u + 4 * lg + r] = us[m][u][r] - off[m] * ws[m][u][r];
    __syncthreads();
    // each wave writes its share of the two maps' tiles of 16 columns
    constexpr int kOwn = 2 * kU / KS;
    const int m = ks * 2 / KS, first = ks * kOwn % kU;
    if (!row_on) return;
    if (lg == 0 && first == 0) {
      const int64_t at = (item * 2 * P.heads + 2 * head_e + m) * P.nq + qi_e;
      P.delta[at] = off[m] + center[m];
      P.norm[at] = weight[m];
    }
    T* out = P.dq.p + item * P.dq.item + (2 * head_e + m) * P.dq.head + qi_e * P.dq.token;
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      const int col = 16 * (first + u) + 4 * lg;
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) x += po[slot(j, m) + col + r];
        v[r] = x * by[m];
      }
      store4f(out + col, v);
    }
    return;
  }
  if (!row_on) return;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (lg == 0) {
      const int64_t at = (item * 2 * P.heads + 2 * head_e + m) * P.nq + qi_e;
      P.delta[at] = off[m] + center[m];
      P.norm[at] = weight[m];
    }
    T* out = P.dq.p + item * P.dq.item + (2 * head_e + m) * P.dq.head + qi_e * P.dq.token;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = (us[m][u][r] - off[m] * ws[m][u][r]) * by[m];
      store4f(out + 16 * u + 4 * lg, v);
    }
  }
}

// dlambda_h = -sum over items and queries of D_2, and the four vectors'
// gradients from it, by one workgroup a head: the first of the launch for dk
// and dv, in whose shadow they run.
template <typename T, int D, int WAVES>
__device__ __forceinline__ void dlambda_of(const DiffAttnParams<T>& P, int head, double (&lds)[WAVES]) {
  const int t = threadIdx.x;
  const int64_t n = P.items * P.nq;
  double s = 0.;  // many numbers of either sign
#pragma unroll 8
  for (int64_t i = t; i < n; i += 64 * WAVES) {
    const int64_t item = n >> 32 ? i / P.nq : (uint32_t)i / (uint32_t)P.nq;
    s += P.delta[(item * 2 * P.heads + 2 * head + 1) * P.nq + i - item * P.nq];
  }
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) s += __shfl_xor(s, x, 64);
  if ((t & 63) == 0) lds[t >> 6] = s;
  __syncthreads();
  if (t >= 64) return;
  double sum = 0.;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) sum += lds[w];
  const float dl = (float)-sum;
  float e[2];
  da_lambda<D>(P.lam, P.heads, head, P.init, t, e);
  if (t < D) {
    const int64_t st = (int64_t)P.heads * D, at = (int64_t)head * D + t;
    const float g[2] = {dl * e[0], -dl * e[1]};
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      P.dlam[2 * m * st + at] = g[m] * P.lam[(2 * m + 1) * st + at];
      P.dlam[(2 * m + 1) * st + at] = g[m] * P.lam[2 * m * st + at];
    }
  }
}

// dk and dv: a wave owns 16 keys (lane l key l % 16, its k and v in registers)
// and walks the query blocks of every head that shares them. S_t = Q_t K_t^T
// leaves the lane 4 queries of its key a tile, the operand of dS_t^T Q_t and of
// (P_1 - lambda P_2)^T dO as they lie. It also writes dbias, where every item has
// a plane of its own. KS 4: the four waves share 16 keys and take 32 queries each
// of a 128-query block, for calls with few keys; 2: two of eight share 16 and take
// 64 each, so that a CU with one workgroup has two waves a SIMD. Bound like the
// kernel for dq (41 % vector, 14 % matrix instructions): 62 us at 245 rows of 245
// tokens and 2 heads, 22 us with dbias at 4 x 499 and 6.
template <typename T, int D, int KS, bool DBIAS>
__global__ __launch_bounds__((DaForm<KS>::kThreads), (kDaWaves<T, D>)) void diffattn_dkv_kernel(DiffAttnParams<T> P) {
  typedef DaForm<KS> Form;
  constexpr int kC = D / 32, kU = D / 16, kQ = Form::kBlock, kQt = kQ / KS / 16, kBufs = KS == 4 ? 1 : 2;
  typedef typename Frag<T>::type F;
  typedef DaTile<T, D, kQ> Tile;
  constexpr int kPo = 4 * D + 2;
  static_assert(KS == 1 || kBufs * sizeof(Tile) >= Form::kWaves * 16 * kPo * sizeof(float), "the waves' sums");
  __shared__ __attribute__((aligned(16))) Tile tiles[kBufs];
  __shared__ __attribute__((aligned(16))) float row_stat[kBufs][4][kQ];  // L_1, L_2, D_1, D_2
  __shared__ __attribute__((aligned(16))) float far_norm[kBufs][2][kQ];  // log2 of rows' norms, 0 for |L| <= kFarSum
  __shared__ int far_rows[kBufs][Form::kWaves];  // whether a wave staged such an L
  __shared__ __attribute__((aligned(16))) float zeros[kQ];
  __shared__ float query_on[kQ];
  __shared__ double lam_lds[Form::kWaves];

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = P.heads / P.group;
  const uint32_t key_blocks = (P.nk + Form::kTiles * 16 - 1) / (Form::kTiles * 16);
  const uint32_t lams = (P.heads + 7) / 8 * 8;
  if (blockIdx.x < lams) {
    if (blockIdx.x < (uint32_t)P.heads) dlambda_of<T, D, Form::kWaves>(P, blockIdx.x, lam_lds);
    return;
  }
  uint32_t id = xcd_order(blockIdx.x - lams, gridDim.x - lams);
  if (id >= (uint32_t)P.items * kvh * key_blocks) return;
  const uint32_t kb = id % key_blocks;
  id /= key_blocks;
  const int kv = id % (uint32_t)kvh;
  const int64_t item = id / (uint32_t)kvh;
  const int tile_of = wave % Form::kTiles, ks = wave / Form::kTiles;  // its tile of 16 keys, and its part of a block's queries
  const int64_t key = ((int64_t)kb * Form::kTiles + tile_of) * 16 + li;
  const int q_w = kQ / KS * ks;  // this wave's queries of a block
  const bool in = key < P.nk;
  uint8_t there = in;
  if (in && P.mask) there = P.mask[item * P.nk + key];

  F kf[2][kC], vf[2 * kC];  // loaded beside the mask, and zeros where that takes the key out
  const int64_t key_there = in ? key : 0;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < kC; ++c)
      kf[m][c] = load8(P.k.p + item * P.k.item + (2 * kv + m) * P.k.head + key_there * P.k.token + 32 * c + 8 * lg);
#pragma unroll
  for (int c = 0; c < 2 * kC; ++c)
    vf[c] = load8(P.v.p + item * P.v.item + kv * P.v.head + key_there * P.v.token + 32 * c + 8 * lg);
  const bool biased = P.bias.p != nullptr;
  const bool part = there != 0;
  const float key_on = part ? INFINITY : -INFINITY;
  const bool all_on = __builtin_amdgcn_ballot_w64(part) == ~0ull;
  const int64_t plane = biased ? item / P.share : 0;
  const int h0 = kv * P.group;
  const T* bias = biased ? P.bias.p + plane * P.bias.item + h0 * P.bias.head : nullptr;
  const uint32_t key_c = in ? (uint32_t)key : 0;

  T* dbias = DBIAS ? P.dbias.p + plane * P.dbias.item + h0 * P.dbias.head : nullptr;

  const uint32_t nq = (uint32_t)P.nq;  // the queries in 32 bits: below 2^31
  const int q_blocks = (nq + kQ - 1) / kQ;
  DaStage<T, D, kQ, Form::kThreads> st;
  st.init(P.q.p + item * P.q.item + 2 * h0 * P.q.head, P.q.head, P.q.token, P.dout.p + item * P.dout.item + h0 * P.dout.head,
          P.dout.token, t);
  const int64_t head_step = st.which < 2 ? 2 * P.q.head : P.dout.head;
  const T* src0 = st.src;
  // the last block's queries, as KeyFlags::on
  if (t < kQ) {
    query_on[t] = (uint32_t)(q_blocks - 1) * kQ + t < nq ? 1.f : -1.f;
    zeros[t] = 0.f;
  }
  __syncthreads();
  constexpr int kStats = 4 * kQ / Form::kThreads;  // statistics that a thread stages
  float stat[kStats];
  // of the first one's row; the statistics of this item's first head and map
  uint32_t stat_at = 0;
  const int64_t stats0 = (item * 2 * P.heads + 2 * h0) * (int64_t)nq;
  const float *saved = P.saved + stats0, *delta = P.delta + stats0, *norm = P.norm + stats0;
  auto fetch = [&](int hg, int qb) {
    const uint32_t q0 = (uint32_t)qb * kQ;
    st.src = src0 + hg * head_step;
    st.load(q0, q0 + kQ <= nq, query_on);
#pragma unroll
    for (int i = 0; i < kStats; ++i) {
      const int which = (t + Form::kThreads * i) / kQ;
      const uint32_t q = q0 + (t + Form::kThreads * i) % kQ;
      const uint32_t at = (2 * hg + (which & 1)) * nq + q;  // heads nq is below 2^27 a key/value head
      stat[i] = which < 2 ? INFINITY : 0.f;  // past the last query: weights of zero
      if (q < nq) stat[i] = (which < 2 ? saved : delta)[at];
      if (i == 0) stat_at = at;
    }
  };
  auto put = [&](int buf) {
    st.store(tiles[buf]);
#pragma unroll
    for (int i = 0; i < kStats; ++i) row_stat[buf][(t + Form::kThreads * i) / kQ][(t + Form::kThreads * i) % kQ] = stat[i];
    // kStats 1: L in the first half of the threads, 2: in the first of each one's
    const bool is_L = kStats == 2 || t < 2 * kQ;
    const bool far = is_L && row_far(stat[0], kFarSum);
    const bool any = __builtin_amdgcn_ballot_w64(far);
    if (lane == 0) far_rows[buf][wave] = any;
    if (is_L) far_norm[buf][t / kQ][t % kQ] = far ? __builtin_amdgcn_logf(norm[stat_at]) : 0.f;
  };
  // a lane's element of the bias in a tile's 16 rows (less than 2^23 elements
  // apart): its row and its key. The scalar address goes from tile to tile (of dbias
  // from row to row) by a step that is not to be known before the loop: its multiples,
  // kept there, took more scalars than there are
  const uint32_t bias_row = (uint32_t)P.bias.token, dbias_row = (uint32_t)P.dbias.token;
  const uint32_t lane_bias = 4 * lg * bias_row + key_c, lane_dbias = 4 * lg * dbias_row + key_c;
  T bq[kQt][4] = {};  // zeros without a bias
  auto fetch_bias = [&](int hg, int qb) {
    const T* p = bias + hg * P.bias.head;
    const uint32_t q0 = (uint32_t)qb * kQ + q_w;
    uint32_t step = bias_row;
    asm volatile("" : "+s"(step));
    p += (uint64_t)q0 * step;
    if ((uint32_t)(qb + 1) * kQ <= nq) {
#pragma unroll
      for (int qt = 0; qt < kQt; ++qt, p += 16 * step)
#pragma unroll
        for (int r = 0; r < 4; ++r) bq[qt][r] = p[lane_bias + r * bias_row];
    } else {
      const int left = (int)nq - (int)q0 - 4 * lg;
#pragma unroll
      for (int qt = 0; qt < kQt; ++qt, p += 16 * step)
#pragma unroll
        for (int r = 0; r < 4; ++r) bq[qt][r] = 16 * qt + r < left ? p[lane_bias + r * bias_row] : from_f32<T>(0.f);
    }
  };

  f32x4 dk[2][kU], dv[2 * kU];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int u = 0; u < kU; ++u) dk[m][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2 * kU; ++u) dv[u] = f32x4{0.f, 0.f, 0.f, 0.f};

  // for the end, a lane's: the loop has no scalar to spare
  int to_item = (int)item, to_kv = kv;
  asm("" : "+v"(to_item), "+v"(to_kv));
  fetch(0, 0);
  if (biased) fetch_bias(0, 0);
  float lam = da_lambda<D>(P.lam, P.heads, h0, P.init, lane);
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    if (!part) kf[0][c] = kf[1][c] = F{};
    if (!part) vf[c] = vf[kC + c] = F{};
  }
  put(0);
  __syncthreads();
  int turn = 0;
  for (int hg = 0; hg < P.group; ++hg) {
    if (hg) lam = da_lambda<D>(P.lam, P.heads, h0 + hg, P.init, lane);
    for (int qb = 0; qb < q_blocks; ++qb, turn ^= 1) {
      const int buf = kBufs == 2 ? turn : 0;
      const Tile& tile = tiles[buf];
      const bool same = qb + 1 < q_blocks;
      const bool more = same || hg + 1 < P.group;
      f32x4 b[kQt];
#pragma unroll
      for (int qt = 0; qt < kQt; ++qt)
#pragma unroll
        for (int r = 0; r < 4; ++r) b[qt][r] = to_f32(bq[qt][r]) * bias_unit<T>(P.inv_scale);
      if (!all_on) {
#pragma unroll
        for (int qt = 0; qt < kQt; ++qt)
#pragma unroll
          for (int r = 0; r < 4; ++r) b[qt][r] = plain_min(b[qt][r], key_on);
      }
      if (more) {
        fetch(same ? hg : hg + 1, same ? qb + 1 : 0);
        if (biased) fetch_bias(same ? hg : hg + 1, same ? qb + 1 : 0);
      }
      f32x4 s[2][kQt], dp[kQt];
#pragma unroll
      for (int qt = 0; qt < kQt; ++qt) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          s[m][qt] = score_start<T>(b[qt]);
#pragma unroll
          for (int x = 0; x < kC; ++x) mma(s[m][qt], load8(&tile.a[q_w + 16 * qt + li][D * m + 32 * x + 8 * lg]), kf[m][x]);
        }
        dp[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2 * kC; ++x) mma(dp[qt], load8(&tile.b[q_w + 16 * qt + li][32 * x + 8 * lg]), vf[x]);
      }
      int far = 0;
#pragma unroll
      for (int w = 0; w < Form::kWaves; ++w) far |= far_rows[buf][w];
      float by = P.scale_log2;
      const float* ls = &row_stat[buf][0][0];  // L_1 and, `ls2` further on, L_2
      int ls2 = kQ;
      if (__builtin_amdgcn_readfirstlane(far)) {
        // the exponents of divided weights in the scores' place, with no more to subtract
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int qt = 0; qt < kQt; ++qt) {
            const f32x4 L = *reinterpret_cast<const f32x4*>(&row_stat[buf][m][q_w + 16 * qt + 4 * lg]);
            const f32x4 n = *reinterpret_cast<const f32x4*>(&far_norm[buf][m][q_w + 16 * qt + 4 * lg]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float e = exponent<T>(s[m][qt][r], b[qt][r], by, L[r]);
              if (kBiasFirst<T> && row_far(L[r], kFar)) {
                e = s[m][qt][r] * by;
                asm("" : "+v"(e));  // rounded, as in far_scores
                e -= L[r];
              }
              s[m][qt][r] = e + n[r];
            }
          }
#pragma unroll
        for (int qt = 0; qt < kQt; ++qt) b[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
        by = 1.f;
        ls = zeros;
        ls2 = 0;
      }
      T db[kQt][4];
#pragma unroll
      for (int c = 0; c < kQt / 2; ++c) {
        float comb[8], ds[2][8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int qt = 2 * c + j;
          f32x4 rs[4];
#pragma unroll
          for (int w = 0; w < 4; ++w)
            rs[w] = *reinterpret_cast<const f32x4*>(w < 2 ? ls + w * ls2 + q_w + 16 * qt + 4 * lg
                                                          : &row_stat[buf][w][q_w + 16 * qt + 4 * lg]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p1 = __builtin_amdgcn_exp2f(exponent<T>(s[0][qt][r], b[qt][r], by, rs[0][r]));
            const float p2 = lam * __builtin_amdgcn_exp2f(exponent<T>(s[1][qt][r], b[qt][r], by, rs[1][r]));
            comb[4 * j + r] = p1 - p2;
            ds[0][4 * j + r] = p1 * (dp[qt][r] - rs[2][r]);
            ds[1][4 * j + r] = p2 * (rs[3][r] - dp[qt][r]);
            if (DBIAS) db[qt][r] = from_f32<T>(ds[0][4 * j + r] + ds[1][4 * j + r]);
          }
        }
        F cf[kParts<T>], df0[kParts<T>], df1[kParts<T>];
        parts(comb, cf);
        parts(ds[0], df0);
        parts(ds[1], df1);
#pragma unroll
        for (int u = 0; u < 2 * kU; ++u) mma_parts(dv[u], col_frag(&tile.b[0][0], Tile::kPitch, q_w + 32 * c, 16 * u, lane), cf);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          mma_parts(dk[0][u], col_frag(&tile.a[0][0], Tile::kPitch, q_w + 32 * c, 16 * u, lane), df0);
          mma_parts(dk[1][u], col_frag(&tile.a[0][D], Tile::kPitch, q_w + 32 * c, 16 * u, lane), df1);
        }
      }
      if (DBIAS && in) {
        const uint32_t q0 = (uint32_t)qb * kQ + q_w;
        uint32_t step = dbias_row;
        asm volatile("" : "+s"(step));
        T* p = dbias + hg * P.dbias.head + (uint64_t)q0 * step;
        if ((uint32_t)(qb + 1) * kQ <= nq) {
#pragma unroll
          for (int qt = 0; qt < kQt; ++qt, p += 12 * step)
#pragma unroll
            for (int r = 0; r < 4; ++r, p += step) p[lane_dbias] = db[qt][r];
        } else {
          const int left = (int)nq - (int)q0 - 4 * lg;
#pragma unroll
          for (int qt = 0; qt < kQt; ++qt, p += 12 * step)
#pragma unroll
            for (int r = 0; r < 4; ++r, p += step)
              if (16 * qt + r < left) p[lane_dbias] = db[qt][r];
        }
      }
      if (kBufs == 1) __syncthreads();
      if (more) put(kBufs == 2 ? buf ^ 1 : 0);
      __syncthreads();
    }
  }
  if constexpr (KS > 1) {  // the waves' sums, through the tiles' memory: [wave][key][dk_1, dk_2, dv]
    float* po = reinterpret_cast<float*>(&tiles[0]);
    float* own = po + (wave * 16 + li) * kPo + 4 * lg;
#pragma unroll
    for (int u = 0; u < 4 * kU; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) own[16 * u + r] = u < 2 * kU ? dk[u / kU][u % kU][r] : dv[u < 2 * kU ? 0 : u - 2 * kU][r];
    __syncthreads();
    if (!in) return;
    // each wave writes 4 / KS of dk_1, dk_2 and the two halves of dv
#pragma unroll
    for (int x = 0; x < 4 / KS; ++x) {
      const int part_of = ks * (4 / KS) + x;
      T* out = part_of < 2 ? P.dk.p + to_item * P.dk.item + (2 * to_kv + part_of) * P.dk.head + key * P.dk.token
                           : P.dv.p + to_item * P.dv.item + to_kv * P.dv.head + key * P.dv.token + (part_of - 2) * D;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < KS; ++j) sum += po[((Form::kTiles * j + tile_of) * 16 + li) * kPo + part_of * D + 16 * u + 4 * lg + r];
          v[r] = part_of < 2 ? sum * P.scale : sum;
        }
        store4f(out + 16 * u + 4 * lg, v);
      }
    }
    return;
  }
  if (!in) return;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    T* out = P.dk.p + to_item * P.dk.item + (2 * to_kv + m) * P.dk.head + key * P.dk.token;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = dk[m][u][r] * P.scale;
      store4f(out + 16 * u + 4 * lg, v);
    }
  }
  T* out = P.dv.p + to_item * P.dv.item + to_kv * P.dv.head + key * P.dv.token;
#pragma unroll
  for (int u = 0; u < 2 * kU; ++u) {
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = dv[u][r];
    store4f(out + 16 * u + 4 * lg, v);
  }
}

// dbias of a plane that several items share (the rows of a triangle attention):
// a workgroup owns 64 queries x 64 keys of one head and adds dS over the items
// of its chunk in registers; the chunks' sums are added by diffattn_bias_sum.
// What bounds it is the 32 KB of k, v, q and dO that each item of a tile brings from
// L2: 40 us at 245 rows of 245 tokens and 2 heads, 6.4 TB/s (three waves a SIMD in
// place of two change it by a few percent).
template <typename T, int D>
__global__ __launch_bounds__(256, (kDaWaves<T, D> + (kDaWaves<T, D> > 1))) void diffattn_dbias_kernel(DiffAttnParams<T> P) {
  constexpr int kC = D / 32;
  typedef typename Frag<T>::type F;
  typedef DaTile<T, D, kDaKeys> Tile;
  __shared__ __attribute__((aligned(16))) Tile tiles[2];
  __shared__ __attribute__((aligned(16))) KeyFlags<kDaKeys> flags[3];  // of the item at hand and the next two

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t planes = (uint32_t)P.items / (uint32_t)P.share;
  const uint32_t kbs = (P.nk + 63) / 64, qbs = (P.nq + 63) / 64;
  uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= planes * P.heads * kbs * qbs * P.chunks) return;
  const int64_t kb = id % kbs;
  id /= kbs;
  const int64_t qb = id % qbs;
  id /= qbs;
  const int head = id % (uint32_t)P.heads;
  id /= (uint32_t)P.heads;
  const int chunk = id % (uint32_t)P.chunks;
  const int64_t plane = id / (uint32_t)P.chunks;
  const int kv = head / P.group;
  const uint32_t qi = (uint32_t)qb * 64 + 16 * wave + li, nq = (uint32_t)P.nq;
  const uint32_t qc = qi < nq ? qi : nq - 1;
  const int64_t i0 = plane * P.share + chunk * P.chunk_items;
  const int64_t i1 = i0 + P.chunk_items < (plane + 1) * P.share ? i0 + P.chunk_items : (plane + 1) * P.share;

  const float lam = da_lambda<D>(P.lam, P.heads, head, P.init, lane);
  typename Quad<T>::type bv[4];
  bias_tile<T, 4>(P.bias.p + plane * P.bias.item + head * P.bias.head + qc * P.bias.token, kb * 64 + 4 * lg, P.nk,
                  (kb + 1) * 64 <= P.nk, bv);

  DaStage<T, D, kDaKeys, 256> st;
  st.init(P.k.p + i0 * P.k.item + 2 * kv * P.k.head, P.k.head, P.k.token, P.v.p + i0 * P.v.item + kv * P.v.head,
          P.v.token, t);
  const int64_t item_step = st.which < 2 ? P.k.item : P.v.item;
  F qf[2][kC], dof[2 * kC], qn[2][kC], don[2 * kC];
  float rs[4], rn[4];
  auto fetch = [&](int64_t item, int at) {
    st.load(kb * 64, flags[at].whole(), flags[at].on);
    st.src += item_step;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int64_t at = (item * 2 * P.heads + 2 * head + m) * P.nq + qc;
      rn[m] = P.saved[at];
      rn[2 + m] = P.delta[at];
#pragma unroll
      for (int c = 0; c < kC; ++c)
        qn[m][c] = load8(P.q.p + item * P.q.item + (2 * head + m) * P.q.head + qc * P.q.token + 32 * c + 8 * lg);
    }
#pragma unroll
    for (int c = 0; c < 2 * kC; ++c)
      don[c] = load8(P.dout.p + item * P.dout.item + head * P.dout.head + qc * P.dout.token + 32 * c + 8 * lg);
  };
  uint8_t part = 0;  // as in the kernel for dq
  auto look = [&](int64_t item) {
    const int64_t k = kb * 64 + t;
    part = t < kDaKeys && item < i1 && k < P.nk;
    if (part && P.mask) part = P.mask[item * P.nk + k];
  };
  auto put_flags = [&](int at) {
    if (t < kDaKeys) flags[at].set(t, part != 0);
  };
  f32x4 acc[4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) acc[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
  look(i0);
  put_flags(0);
  look(i0 + 1);
  put_flags(1);
  __syncthreads();
  fetch(i0, 0);
  st.store(tiles[0]);
  __syncthreads();
  int buf = 0, at = 0;
  for (int64_t item = i0; item < i1; ++item, buf ^= 1) {
    const Tile& tile = tiles[buf];
    const bool more = item + 1 < i1;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < kC; ++c) qf[m][c] = qn[m][c];
#pragma unroll
    for (int c = 0; c < 2 * kC; ++c) dof[c] = don[c];
#pragma unroll
    for (int w = 0; w < 4; ++w) rs[w] = rn[w];
    f32x4 b[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) b[kt][r] = to_f32(bv[kt][r]) * bias_unit<T>(P.inv_scale);
    flags[at].apply(0, lg, b);
    at = at == 2 ? 0 : at + 1;
    if (more) {
      fetch(item + 1, at);
      look(item + 2);
    }
    const bool far_sum = __builtin_amdgcn_ballot_w64(row_far(rs[0], kFarSum) || row_far(rs[1], kFarSum));
    const bool far = far_sum && __builtin_amdgcn_ballot_w64(row_far(rs[0], kFar) || row_far(rs[1], kFar));
    f32x4 dp[4];
    tile_dp<T, D, kDaKeys, 4>(tile, 0, dof, li, lg, dp);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f32x4 p[4];
      tile_scores<T, D, kDaKeys, 4>(tile, m, 0, qf[m], b, li, lg, p);
      to_weights<T>(b, kBiasFirst<T> ? far_scores(far, P.scale_log2, p) : P.scale_log2, rs[m], p);
      if (far_sum) {
        const float n = P.norm[(item * 2 * P.heads + 2 * head + m) * P.nq + qc];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[kt][r] *= n;
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[kt][r] = fmaf(m ? p[kt][r] * -lam : p[kt][r], dp[kt][r] - rs[2 + m], acc[kt][r]);
    }
    if (more) {
      st.store(tiles[buf ^ 1]);
      put_flags(at == 2 ? 0 : at + 1);
    }
    __syncthreads();
  }
  if (qi >= nq) return;
  float* out = P.part_bias + (((int64_t)chunk * planes + plane) * P.heads + head) * P.nq * P.nk + qi * P.nk;
  const int64_t k0 = kb * 64 + 4 * lg;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (k0 + 16 * kt + r < P.nk) out[k0 + 16 * kt + r] = acc[kt][r];
}

template <typename T>
__global__ __launch_bounds__(256) void diffattn_bias_sum_kernel(DiffAttnParams<T> P) {
  const int64_t per = P.items / P.share * P.heads * P.nq * P.nk;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < per; i += gridDim.x * 256ll) {
    float s = 0.f;
#pragma unroll 8
    for (int c = 0; c < P.chunks; ++c) s += P.part_bias[c * per + i];
    const int64_t k = i % P.nk, q = i / P.nk % P.nq, ph = i / (P.nk * P.nq);
    P.dbias.p[ph / P.heads * P.dbias.item + ph % P.heads * P.dbias.head + q * P.dbias.token + k] = from_f32<T>(s);
  }
}

unsigned eights(int64_t blocks) { return (unsigned)((blocks + 7) / 8 * 8); }

template <typename T, int D, int KS>
void dq_form(const DiffAttnParams<T>& P, hipStream_t st) {
  constexpr int kTile = DaForm<KS>::kTiles * 16;
  const int64_t blocks = P.items * (P.heads / P.group) * ((P.group * P.nq + kTile - 1) / kTile);
  diffattn_dq_kernel<T, D, KS><<<eights(blocks), DaForm<KS>::kThreads, 0, st>>>(P);
}
template <typename T, int D, int KS>
void dkv_form(const DiffAttnParams<T>& P, hipStream_t st) {
  constexpr int kTile = DaForm<KS>::kTiles * 16;
  const unsigned blocks = eights(P.heads) + eights(P.items * (P.heads / P.group) * ((P.nk + kTile - 1) / kTile));
  if (P.dbias.p && P.share == 1)
    diffattn_dkv_kernel<T, D, KS, true><<<blocks, DaForm<KS>::kThreads, 0, st>>>(P);
  else
    diffattn_dkv_kernel<T, D, KS, false><<<blocks, DaForm<KS>::kThreads, 0, st>>>(P);
}

template <typename T, int D>
void bwd(const DiffAttnParams<T>& P, hipStream_t st) {
  const int64_t kvh = P.heads / P.group;
  // Waves with rows (keys) of their own cost the least work; they share 16 where
  // that leaves too few workgroups for the card's 256 CUs. us own / shared by four,
  // 499 tokens: dq in bf16 at D = 32 at 120 workgroups 22.9 / 16.9, 144 22.4 / 25.6; at
  // D = 64 120 29.8 / 34.0 (the one form that would rather change over earlier), 144
  // 29.7 / 48.4; float32 D = 32 120 49.0 / 34.4, 144 49.0 / 48.4; D = 64 120 86.9 / 70.7,
  // 144 88 / 102. dk and dv in bf16 at D = 64 120 39.2 / 35.3, 144 39.6 / 51.6; float32 D =
  // 32 120 54.2 / 45.9, 144 55.1 / 66.5; D = 64 120 94 / 73, 144 95 / 106; bf16 at D = 32,
  // own / by two / by four: 120 24.9 / 20.9 / 16.5, 144 25.5 / 21.3 / 25.3, 192 26.4 /
  // 22.0 / 26.2, 240 27.1 / 23.6 / 29.9 (one such workgroup fits a CU; the other types'
  // registers leave one wave a SIMD). By two gained nothing in the forward kernel and dq
  // (18.3 and 19.5 either way at 192).
  constexpr bool kPaired = sizeof(T) == 2 && D == 32;
  const int64_t heads = P.items * kvh, rows = P.group * P.nq;
  const int64_t row_wgs = heads * ((rows + 63) / 64), key_wgs = heads * ((P.nk + 63) / 64);
  if (row_wgs < 128)
    dq_form<T, D, 4>(P, st);
  else
    dq_form<T, D, 1>(P, st);
  if (key_wgs < 128)
    dkv_form<T, D, 4>(P, st);
  else if (kPaired && P.nq > 64 && key_wgs <= 256)
    dkv_form<T, D, kPaired ? 2 : 1>(P, st);
  else
    dkv_form<T, D, 1>(P, st);
  if (P.dbias.p && P.share > 1) {
    const int64_t planes = P.items / P.share;
    diffattn_dbias_kernel<T, D><<<eights(planes * P.heads * P.chunks * ((P.nk + 63) / 64) * ((P.nq + 63) / 64)), 256, 0, st>>>(P);
    const int64_t blocks = (planes * P.heads * P.nq * P.nk + 255) / 256;
    diffattn_bias_sum_kernel<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, st>>>(P);
  }
}

}  // namespace

template <typename T>
void launch_diffattn_bwd(const DiffAttnParams<T>& P, int d, hipStream_t st) {
  if (d == 32)
    bwd<T, 32>(P, st);
  else
    bwd<T, 64>(P, st);
}
template void launch_diffattn_bwd<bf16>(const DiffAttnParams<bf16>&, int, hipStream_t);
template void launch_diffattn_bwd<float>(const DiffAttnParams<float>&, int, hipStream_t);

}  // namespace fjx
