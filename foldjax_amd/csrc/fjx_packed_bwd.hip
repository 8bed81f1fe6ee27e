// Packed attention, backward. With dP = dO v^T and D = rowsum(dO out):
//   dS = P (dP - D),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T dO
// The weights come again from the scores and the forward pass's row statistics, the
// maximum M and log2 of the sum l: P = 2^(s scale log2(e) - M - log2 l).
// Every sum has one owner and one order: no atomics, and the same bits each time. So
// dq and the keys' gradients are two walks with the scores and dP taken twice, seven
// products in place of five.
//
// dS's rows sum to zero. Where one key has nearly all of a row's weight dP - D is what
// the others have left of it, and D must be known to more bits than a bf16 output has:
// it is taken from the output and what its rounding left (17 bits; the forward pass
// applies rounded weights, but in D they are off in proportion to dS itself). For the
// same reason dq takes bf16's dS in two parts (17 bits): rounded once, what a row's dS
// lose is as large as dq's own rounding (0.0026 of dq against 0.0017). What the applied
// weights' rounding leaves in D stays, times the keys' weighted mean: where all keys share a
// part of 4 times their spread dq is off by 0.0056 (0.0083 with one part). dk and dv sum over rows, where nothing
// cancels so: weights and dS enter their products rounded once, relative to themselves.
//
// us of dq / dk and dv: a step of 8192 causal tokens in 5 sequences of 43 to 4099, 8 heads
// of 128 on 2: 106 / 142 and the join's 11; of 6 crops of 1 to 1003 residues, 16 heads of
// 24: 19.0 / 17.7. No one thing bounds them. In variants of the first that left out work,
// half the column fragments' reads were 3 % of both, the exponentials and dS 4 %, the
// staging of further blocks 8 %, and all blocks but the first left a quarter to a third:
// finding the tile, the first loads, the outputs. Vector instructions a score, one of them
// an exponential: 5 for dq, 4 for dk and dv (7 and 6 with D and the logarithm subtracted
// by themselves: 5 % and 2 % slower). Two tiles of keys a wave at 128 channels, on one
// wave a SIMD, halve the reads and took 360 us where two waves take 299.
#include "fjx_packed.hpp"

namespace fjx {

namespace {

constexpr float kFar = 16777216.f;  // as in the forward pass

// The exponent of a weight is s scale log2(e) - M - log2 l. bf16 rows whose |M| is up to
// kNear take M + log2 l as one number, half a step of which, 2^-13, is a 16th of a weight's
// own rounding: one fma. Others have M subtracted from their scores (rounded products where
// they are far, as in the forward pass) and the logarithm apart.
constexpr float kNear = 2048.f;
template <typename T> constexpr bool kJoined = sizeof(T) == 2;
template <int N, typename M>
__device__ __forceinline__ void pk_less(float scale, bool far, M m, f32x4 (&s)[N]) {
  if (far) pk_round(scale, s);
  const float by = far ? 1.f : scale;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[j][e] = fmaf(s[j][e], by, -m(j, e));
}

// dq, and D for the other kernel: rows and blocks as in the forward pass.
template <typename T, int DP, int G, int KS, int R>
__global__ __launch_bounds__((PkForm<G, KS>::kThreads), (PkFormOf<T, DP, G, KS>::type::template kSimd<T, DP>)) void packed_dq_kernel(PackedParams<T> P) {
  typedef typename PkFormOf<T, DP, G, KS>::type Form;
  typedef PkRows<T, DP> Rows;
  typedef typename Frag<T>::type F;
  constexpr int kC = Rows::kC, kU = Rows::kU;
  constexpr int kNt = Form::kOwn / 16;
  constexpr int kTileRows = 16 * R * G, kShift = __builtin_ctz(kTileRows);
  constexpr int kOperand = Form::kStage * Rows::kRowBytes;
  constexpr int kSets = Form::kSets;
  constexpr int kStages = 4 * kOperand * kSets <= 160 * 1024 ? 2 : 1;
  typedef PkOut<Form, DP> Out;
  constexpr int kRaw = kStages * 2 * kOperand * kSets;  // and at the end the outputs' way
  __shared__ __attribute__((aligned(16))) unsigned char raw[kRaw > Out::kBytes ? kRaw : Out::kBytes];
  __shared__ int2 places[R][16 * G];  // the rows' heads and tokens; head -1: no such row

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Form form(wave);
  const int kv = blockIdx.x;
  const int nth = P.tile0 + blockIdx.y;  // in the forward pass's order
  PackedTile sp;
  if (!packed_tile(P, false, P.group, kShift, P.order ? nth : P.tiles - 1 - nth, lane, sp)) return;
  const int row0 = sp.tile * kTileRows, rows = sp.nq * P.group - row0;  // those from row0 on
  if (rows <= 0) return;
  const int row_w = 16 * R * form.group;
  const PackedRows place(P, row0);

  int lim[R];
  F qf[R][kC], dof[R][kC];
  float m[R], log_sum[R], delta[R];
  bool any_far = false, any_off = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int x = row_w + 16 * r + li;
    int qi, head;
    place.at(x < rows ? x : rows - 1, qi, head);
    head += kv * P.group;
    const int64_t token = sp.q0 + qi;
    lim[r] = P.causal ? qi + (sp.nk - sp.nq) + 1 : sp.nk;
    if (lg == 0 && form.part == 0) places[r][16 * form.group + li] = make_int2(x < rows ? head : -1, (int)token);
    const T* q = P.q.p + head * P.q.head + token * P.q.token + 8 * lg;
    const T* dout = P.dout.p + head * P.dout.head + token * P.dout.token + 8 * lg;
    const T* o = P.o.p + head * P.o.head + token * P.o.token + 8 * lg;
    const T* rest = P.o_rest.p + head * P.o_rest.head + token * P.o_rest.token + 8 * lg;
    float d = 0.f;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      qf[r][c] = dof[r][c] = F{};
      if (32 * c + 8 * lg >= P.d) continue;
      qf[r][c] = load8(q + 32 * c);
      dof[r][c] = load8(dout + 32 * c);
      float x[8], y[8];
      to_f32x8(dof[r][c], x);
      to_f32x8(load8(o + 32 * c), y);
      if (P.o_rest.p) {
        float z[8];
        to_f32x8(load8(rest + 32 * c), z);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] += z[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) d = fmaf(x[e], y[e], d);
    }
    delta[r] = group_sum(d);
    const int64_t at_row = (int64_t)head * P.tq + token;
    const f32x2 stats = *reinterpret_cast<const f32x2*>(P.lse + at_row * 2);
    m[r] = stats[0];
    log_sum[r] = stats[1];
    any_far = any_far || fabsf(m[r]) > kFar;
    any_off = any_off || !kJoined<T> || fabsf(m[r]) > kNear;
    if (lg == 0 && form.part == 0 && x < rows) P.delta[at_row] = delta[r];
  }
  const bool far = __builtin_amdgcn_ballot_w64(any_far), off = __builtin_amdgcn_ballot_w64(any_off);
  const float by = off ? 1.f : P.scale_log2;
  float base[R];  // what is still to be subtracted from a score times by
#pragma unroll
  for (int r = 0; r < R; ++r) base[r] = off ? log_sum[r] : m[r] + log_sum[r];
  int q_last, h_last;
  place.at((kTileRows < rows ? kTileRows : rows) - 1, q_last, h_last);
  const int most = P.causal ? q_last + (sp.nk - sp.nq) + 1 : sp.nk;
  const int lim_lo = __builtin_amdgcn_readfirstlane(lim[0]);
  const int lim_hi = row_w < rows ? __builtin_amdgcn_readlane(lim[R - 1], 15) : 0;
  const int blocks = most > 0 ? (int)((uint32_t)(most + Form::kBlock - 1) / Form::kBlock) : 0;

  unsigned char* const mine = raw + (Form::kPrivate ? wave * kStages * 2 * kOperand : 0);
  PkCopy<T, DP, Form::kStage, Form::kOwners> kcopy, vcopy;
  kcopy.init(P.k.token, P.d, form.stager, lane);
  vcopy.init(P.v.token, P.d, form.stager, lane);
  kcopy.begin(P.k.p + kv * P.k.head + (int64_t)sp.k0 * P.k.token, form.staged(), sp.nk);
  vcopy.begin(P.v.p + kv * P.v.head + (int64_t)sp.k0 * P.v.token, form.staged(), sp.nk);
  auto stage = [&](int at) {  // the next block
    unsigned char* s = mine + at * 2 * kOperand;
    kcopy.issue(s, form.stager, Form::kBlock);
    vcopy.issue(s + kOperand, form.stager, Form::kBlock);
  };
  PkLane<T, DP> at;
  at.init(lane);
  f32x4 dq[R][kU];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int u = 0; u < kU; ++u) dq[r][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (kStages == 2) {
    if (blocks) stage(0);
    pk_sync<Form>();
  }
  for (int blk = 0; blk < blocks; ++blk) {
    const int cur = kStages == 2 ? blk & 1 : 0;
    if (kStages == 1) {
      stage(0);
      pk_sync<Form>();
    } else if (blk + 1 < blocks) {
      stage(cur ^ 1);
    }
    const unsigned char* kt_ = mine + cur * 2 * kOperand + form.at * Rows::kRowBytes;
    const unsigned char* vt_ = kt_ + kOperand;
    const int key0 = blk * Form::kBlock + Form::kOwn * form.part;
    if (key0 < lim_hi) {
      const bool masked = key0 + 16 * kNt > lim_lo;
#pragma unroll
      for (int pair = 0; pair < kNt / 2; ++pair) {
        f32x4 s[R][2], dp[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[r][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            dp[r][j] = f32x4{-delta[r], -delta[r], -delta[r], -delta[r]};  // dP - D from the start
          }
        pk_ahead<2 * kC>([&](int i) { return at.at_row(kt_, 32 * pair + 16 * (i / kC), i % kC); },
                         [&](int i, const F& kf) {
#pragma unroll
                           for (int r = 0; r < R; ++r) mma(s[r][i / kC], kf, qf[r][i % kC]);
                         });
        pk_ahead<2 * kC>([&](int i) { return at.at_row(vt_, 32 * pair + 16 * (i / kC), i % kC); },
                         [&](int i, const F& vf) {
#pragma unroll
                           for (int r = 0; r < R; ++r) mma(dp[r][i / kC], vf, dof[r][i % kC]);
                         });
        if (off) {
#pragma unroll
          for (int r = 0; r < R; ++r) pk_less(P.scale_log2, far, [&](int, int) { return m[r]; }, s[r]);
        }
        if (masked) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int left = lim[r] - key0 - 32 * pair - 4 * lg;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[r][j][e] = 16 * j + e < left ? s[r][j][e] : -INFINITY;
          }
        }
        F dsf[R][kParts<T>];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float ds[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            ds[e] = __builtin_amdgcn_exp2f(fmaf(s[r][e >> 2][e & 3], by, -base[r])) * dp[r][e >> 2][e & 3];
          parts(ds, dsf[r]);
        }
        pk_ahead<kU>([&](int u) { return at.at_col(kt_, 32 * pair, u); },
                     [&](int u, const F& kf) {
#pragma unroll
                       for (int r = 0; r < R; ++r) mma_parts(dq[r][u], kf, dsf[r]);
                     });
      }
    }
    pk_sync<Form>();
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    Out::write(raw, form, t, dq[r], [&](int row, int c, const float* x) {
      const int2 to = places[r][row];
      if (to.x < 0 || c >= P.d) return;
      const f32x8 v = Out::sum(x);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v[e] * P.scale;
      store8(P.dq.p + to.x * P.dq.head + to.y * P.dq.token + c, pack8<T>(y));
    });
}

// A key tile's walk: the blocks of queries in which any row sees its first key, and in how
// many parts the heads that share it are dealt to workgroups: a tile's walk depends on its
// sequence and, causal, its place in that, so that long ones have parts and short ones none.
struct PkWalk {
  int first, last, parts;
  template <typename T>
  __device__ __forceinline__ PkWalk(const PackedParams<T>& P, const PackedTile& sp, int key0, int block) {
    const int shift = sp.nq - sp.nk;
    first = (uint32_t)(P.causal && key0 + shift > 0 ? key0 + shift : 0) / block;
    last = key0 < sp.nk ? (int)((uint32_t)(sp.nq + block - 1) / block) : 0;
    if (last < first) last = first;
    parts = 1;
    if (P.splits > 1) {
      const int n = (int)(((uint32_t)(last - first) * block * P.group + P.part_rows - 1) / P.part_rows);
      parts = n < 1 ? 1 : n < P.splits ? n : P.splits;
    }
  }
};

// dk and dv: a wave holds R tiles of 16 keys, lane l key l % 16 of each, and walks the
// queries of every head that shares them in tiles of 16: S = Q K^T and dP = dO V^T leave
// the lane 4 queries of its own keys, as the operands of dV^T = dO^T P and dK^T = Q^T dS.
// KS 1: four waves with keys of their own; 4: the waves share keys and split the queries.
template <typename T, int DP, int G, int KS, int R>
__global__ __launch_bounds__((PkForm<G, KS>::kThreads), (PkFormOf<T, DP, G, KS>::type::template kSimd<T, DP>)) void packed_dkv_kernel(PackedParams<T> P) {
  typedef typename PkFormOf<T, DP, G, KS>::type Form;
  typedef PkRows<T, DP> Rows;
  typedef typename Frag<T>::type F;
  constexpr int kC = Rows::kC, kU = Rows::kU;
  constexpr int kNt = Form::kOwn / 16;  // query tiles of a wave in a block
  constexpr int kTileKeys = 16 * R * G, kShift = __builtin_ctz(kTileKeys);
  constexpr int kOperand = Form::kStage * Rows::kRowBytes;
  constexpr int kSets = Form::kSets;
  constexpr int kStages = 4 * kOperand * kSets <= 156 * 1024 ? 2 : 1;
  typedef PkOut<Form, DP> Out;
  constexpr int kRaw = kStages * 2 * kOperand * kSets;  // and at the end the outputs' way
  __shared__ __attribute__((aligned(16))) unsigned char raw[kRaw > Out::kBytes ? kRaw : Out::kBytes];
  __shared__ __attribute__((aligned(16))) float rowstat[kSets][kStages][3 + kJoined<T>][Form::kStage];  // M, log2 of the sum, -D, M + the second
  __shared__ int rowfar[kSets][kStages][Form::kRest];  // 1: a row past kNear, 2: one past kFar

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Form form(wave);
  const int kv = blockIdx.x / P.splits, part = blockIdx.x - kv * P.splits;
  PackedTile sp;
  if (!packed_tile(P, true, 1, kShift, P.tile0 + blockIdx.y, lane, sp)) return;
  const int key0 = sp.tile * kTileKeys;
  if (key0 >= sp.cap) return;
  const PkWalk walk(P, sp, key0, Form::kBlock);
  const int parts = __builtin_amdgcn_readfirstlane(walk.parts);
  if (part >= parts) return;
  const int key_w = key0 + 16 * R * form.group;
  const int shift = sp.nq - sp.nk;  // a causal row i sees the keys up to i - shift

  F kf[R][kC], vf[R][kC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int key = key_w + 16 * r + li;
    const int64_t token = (int64_t)sp.k0 + key;
    const T* k = P.k.p + kv * P.k.head + token * P.k.token + 8 * lg;
    const T* v = P.v.p + kv * P.v.head + token * P.v.token + 8 * lg;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const bool in = key < sp.nk && 32 * c + 8 * lg < P.d;
      kf[r][c] = in ? load8(k + 32 * c) : F{};
      vf[r][c] = in ? load8(v + 32 * c) : F{};
    }
  }
  const int h0 = P.group * part / parts, h1 = P.group * (part + 1) / parts;  // the heads of this part
  const int qb0 = walk.first, qb1 = walk.last;
  const int turns = qb1 > qb0 ? (h1 - h0) * (qb1 - qb0) : 0;

  const int set = Form::kPrivate ? wave : 0;
  unsigned char* const mine = raw + set * kStages * 2 * kOperand;
  const int stat_row = Form::kPrivate ? lane : t;  // of a staged block, of which the thread fetches the statistics
  PkCopy<T, DP, Form::kStage, Form::kOwners> qcopy, ocopy;
  qcopy.init(P.q.token, P.d, form.stager, lane);
  ocopy.init(P.dout.token, P.d, form.stager, lane);
  int next_h = h0, next_b = qb0;  // of the next block to stage
  f32x2 st_m = {0.f, INFINITY};
  float st_d = 0.f;
  auto stage = [&](int at) {
    const int head = kv * P.group + next_h, row0 = next_b * Form::kBlock + form.staged();
    if (next_b == qb0) {
      qcopy.begin(P.q.p + head * P.q.head + (int64_t)sp.q0 * P.q.token, row0, sp.nq);
      ocopy.begin(P.dout.p + head * P.dout.head + (int64_t)sp.q0 * P.dout.token, row0, sp.nq);
    }
    unsigned char* s = mine + at * 2 * kOperand;
    qcopy.issue(s, form.stager, Form::kBlock);
    ocopy.issue(s + kOperand, form.stager, Form::kBlock);
    st_m = f32x2{0.f, INFINITY};  // rows past the last: weights of zero
    st_d = 0.f;
    if (stat_row < Form::kStage && row0 + stat_row < sp.nq) {
      const int64_t at_row = (int64_t)head * P.tq + sp.q0 + row0 + stat_row;
      st_m = *reinterpret_cast<const f32x2*>(P.lse + at_row * 2);
      st_d = P.delta[at_row];
    }
    if (++next_b == qb1) {
      next_b = qb0;
      ++next_h;
    }
  };
  auto put_stats = [&](int at) {
    if (stat_row < Form::kStage) {
      rowstat[set][at][0][stat_row] = st_m[0];
      rowstat[set][at][1][stat_row] = st_m[1];
      rowstat[set][at][2][stat_row] = -st_d;
      if constexpr (kJoined<T>) rowstat[set][at][3][stat_row] = st_m[0] + st_m[1];
      const int far = (__builtin_amdgcn_ballot_w64(!kJoined<T> || fabsf(st_m[0]) > kNear) ? 1 : 0) |
                      (__builtin_amdgcn_ballot_w64(fabsf(st_m[0]) > kFar) ? 2 : 0);
      if (stat_row % 64 == 0) rowfar[set][at][stat_row / 64] = far;
    }
  };
  PkLane<T, DP> at;
  at.init(lane);
  f32x4 dk[R][kU], dv[R][kU];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int u = 0; u < kU; ++u) dk[r][u] = dv[r][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (kStages == 2) {
    if (turns) {
      stage(0);
      put_stats(0);
    }
    pk_sync<Form>();
  }
  int qb = qb0;
  for (int turn = 0; turn < turns; ++turn) {
    const int cur = kStages == 2 ? turn & 1 : 0;
    if (kStages == 1) {
      stage(0);
      put_stats(0);
      pk_sync<Form>();
    } else if (turn + 1 < turns) {
      stage(cur ^ 1);
    }
    const unsigned char* qt_ = mine + cur * 2 * kOperand + form.at * Rows::kRowBytes;
    const unsigned char* ot_ = qt_ + kOperand;
    const int row0 = qb * Form::kBlock + Form::kOwn * form.part;
    // rows from key + shift on see a key
    if (!P.causal || row0 + 16 * kNt > key_w + shift) {
      const bool masked = P.causal && row0 < key_w + 16 * R - 1 + shift;
      int any_far = 0;
#pragma unroll
      for (int i = 0; i < Form::kRest; ++i) any_far |= rowfar[set][cur][i];
      const int flags = __builtin_amdgcn_readfirstlane(any_far);
      const bool off = flags & 1, far = flags & 2;
      const float by = off ? 1.f : P.scale_log2;
      const float* const stats = rowstat[set][cur][0];
      const float* const bases = rowstat[set][cur][kJoined<T> && !off ? 3 : 1];
#pragma unroll
      for (int pair = 0; pair < kNt / 2; ++pair) {
        f32x4 s[R][2], dp[R][2];
        const int row = form.at + 32 * pair + 4 * lg;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(stats + 2 * Form::kStage + row + 16 * j);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            s[r][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            dp[r][j] = d4;  // dP - D from the start
          }
        }
        pk_ahead<2 * kC>([&](int i) { return at.at_row(qt_, 32 * pair + 16 * (i / kC), i % kC); },
                         [&](int i, const F& qf) {
#pragma unroll
                           for (int r = 0; r < R; ++r) mma(s[r][i / kC], qf, kf[r][i % kC]);
                         });
        pk_ahead<2 * kC>([&](int i) { return at.at_row(ot_, 32 * pair + 16 * (i / kC), i % kC); },
                         [&](int i, const F& of) {
#pragma unroll
                           for (int r = 0; r < R; ++r) mma(dp[r][i / kC], of, vf[r][i % kC]);
                         });
        if (off) {
          f32x4 m4[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) m4[j] = *reinterpret_cast<const f32x4*>(stats + row + 16 * j);
#pragma unroll
          for (int r = 0; r < R; ++r) pk_less(P.scale_log2, far, [&](int j, int e) { return m4[j][e]; }, s[r]);
        }
        if (masked) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int from = key_w + 16 * r + li + shift - row0 - 32 * pair - 4 * lg;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[r][j][e] = 16 * j + e >= from ? s[r][j][e] : -INFINITY;
          }
        }
        F pf[R], dsf[R];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x4 b4 = *reinterpret_cast<const f32x4*>(bases + row + 16 * j);
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float p = __builtin_amdgcn_exp2f(fmaf(s[r][j][e], by, -b4[e]));
              pf[r][4 * j + e] = from_f32<T>(p);
              dsf[r][4 * j + e] = from_f32<T>(p * dp[r][j][e]);
            }
        }
        pk_ahead<2 * kU>([&](int i) { return at.at_col(i & 1 ? qt_ : ot_, 32 * pair, i / 2); },
                         [&](int i, const F& f) {
#pragma unroll
                           for (int r = 0; r < R; ++r) {
                             if (i & 1)
                               mma(dk[r][i / 2], f, dsf[r]);
                             else
                               mma(dv[r][i / 2], f, pf[r]);
                           }
                         });
      }
    }
    if (++qb == qb1) qb = qb0;
    if (kStages == 2 && turn + 1 < turns) put_stats(cur ^ 1);
    pk_sync<Form>();
  }
  // The arguments are read again here: kept through the walk, they would spill scalar registers.
  const auto* L = pk_late<T>();
  // dk, then dv; keys that are not there have zeros
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r)
      Out::write(raw, form, t, i ? dv[r] : dk[r], [&](int row, int c, const float* x) {
        const int key = key0 + 16 * (R * (row / 16) + r) + row % 16;
        if (key >= sp.cap) return;
        const f32x8 v = Out::sum(x);
        const int64_t token = (int64_t)sp.k0 + key;
        const float by = key < sp.nk ? i || parts > 1 ? 1.f : L->scale : 0.f;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = by == 0.f ? 0.f : v[e] * by;
        if (parts > 1) {
          const int kvh = L->heads / L->group;
          store8((i ? L->part_dv : L->part_dk) + (((int64_t)part * kvh + kv) * L->tk + token) * DP + c, pack8<float>(y));
          return;
        }
        if (c >= L->d) return;
        T* to = i ? L->dv.p : L->dk.p;
        const int64_t head = i ? L->dv.head : L->dk.head, step = i ? L->dv.token : L->dk.token;
        store8(to + kv * head + token * step + c, pack8<T>(y));
      });
}

// The parts of dk and dv added, where a tile (of 2^shift keys) has several: a workgroup 16
// keys, 8 elements a thread.
template <typename T, int DP>
__global__ __launch_bounds__(2 * DP) void packed_dkv_join_kernel(PackedParams<T> P, int shift, int block) {
  PackedTile sp;
  if (!packed_tile(P, true, 1, shift, P.tile0 + blockIdx.y, threadIdx.x & 63, sp)) return;
  const int key0 = sp.tile << shift, kv = blockIdx.x, key = key0 + 16 * blockIdx.z + threadIdx.x / (DP / 8);
  const int c = threadIdx.x % (DP / 8) * 8;
  if (key >= sp.cap || c >= P.d) return;
  const int parts = PkWalk(P, sp, key0, block).parts;
  if (parts == 1) return;
  const int64_t all = (int64_t)(P.heads / P.group) * P.tk * DP, token = (int64_t)sp.k0 + key;
  const int64_t at = (kv * P.tk + token) * DP + c;
  f32x8 a = load8(P.part_dk + at), b = load8(P.part_dv + at);
  for (int s = 1; s < parts; ++s) {
    a += load8(P.part_dk + s * all + at);
    b += load8(P.part_dv + s * all + at);
  }
  float x[8], y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = a[e] * P.scale, y[e] = b[e];
  store8(P.dk.p + kv * P.dk.head + token * P.dk.token + c, pack8<T>(x));
  store8(P.dv.p + kv * P.dv.head + token * P.dv.token + c, pack8<T>(y));
}

template <typename T, int DP>
void bwd(PackedParams<T> P, const PackedForm& rows, const PackedForm& keys, hipStream_t st) {
  const int splits = P.splits;
  launch_packed_order(P, rows, keys, st);
  P.splits = 1;
  P.tiles = rows.count;
  P.order = rows.order;
  pk_form<T>(rows, [&](auto g, auto ks, auto r) {
    constexpr int G = decltype(g)::value, KS = decltype(ks)::value, R = decltype(r)::value;
    pk_grid(P, [&](const PackedParams<T>& Q, dim3 grid) {
      packed_dq_kernel<T, DP, G, KS, R><<<grid, PkForm<G, KS>::kThreads, 0, st>>>(Q);
    });
  });
  if (!keys.count) return;
  P.splits = splits;
  P.tiles = keys.count;
  P.order = keys.order;
  pk_form<T>(keys, [&](auto g, auto ks, auto r) {
    constexpr int G = decltype(g)::value, KS = decltype(ks)::value, R = decltype(r)::value;
    // two tiles of keys a wave: at 128 channels they would take more registers than two waves
    // a SIMD have, and are taken only where workgroups are many
    if constexpr (DP * R <= 128 && (KS * R <= 2 || G == 1))
      pk_grid(P, [&](const PackedParams<T>& Q, dim3 grid) {
        // a tile's parts side by side, so that the longest tiles begin with all of theirs
        packed_dkv_kernel<T, DP, G, KS, R><<<dim3(grid.x * splits, grid.y), PkForm<G, KS>::kThreads, 0, st>>>(Q);
        if (splits > 1)
          packed_dkv_join_kernel<T, DP><<<dim3(grid.x, grid.y, G * R), 2 * DP, 0, st>>>(Q, __builtin_ctz(keys.rows()),
                                                                                        PkFormOf<T, DP, G, KS>::type::kBlock);
      });
  });
}

}  // namespace

template <typename T>
void launch_packed_bwd(const PackedParams<T>& P, const PackedForm& rows, const PackedForm& keys, hipStream_t st) {
  if (P.d <= 32)
    bwd<T, 32>(P, rows, keys, st);
  else if (P.d <= 64)
    bwd<T, 64>(P, rows, keys, st);
  else
    bwd<T, 128>(P, rows, keys, st);
}
template void launch_packed_bwd<bf16>(const PackedParams<bf16>&, const PackedForm&, const PackedForm&, hipStream_t);
template void launch_packed_bwd<float>(const PackedParams<float>&, const PackedForm&, const PackedForm&, hipStream_t);

}  // namespace fjx
