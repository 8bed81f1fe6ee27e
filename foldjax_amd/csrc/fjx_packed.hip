// Packed attention, forward: one pass over a row's keys with the running maximum
// and sum of the softmax.
#include "fjx_packed.hpp"

namespace fjx {

namespace {

// A wave holds R tiles of 16 rows, lane l row l % 16 of each, and walks the keys in
// tiles of 16: S^T = K Q^T leaves the lane 4 keys of its own row a tile (keys 4 g + r,
// g = l / 16), so a row's maximum and sum are the lane's own values and two lane swaps,
// and the weights of two key tiles are the operand of O^T = V^T P^T as they lie.
//
// A bf16 weight is rounded once (half a step, 2^-8 of itself at most), and the outputs'
// sum is that of the rounded weights, taken by the matrix cores as a row of ones times them:
// the weights that are applied add up to one, and an output is off by less than its own
// rounding. A weight may exceed 1 by up to 2^kSlack before the maximum is moved, which
// saves the outputs' rescaling in all but the first blocks of a row.
//
// Blocks of keys and values come by LDS DMA, the next while one is worked on, fragments
// from LDS a product ahead. What bounds it: long prompts the issue of vector beside matrix
// instructions (16384 causal tokens in 6 sequences of up to 9001, 8 heads of 128 on 2: 220 us,
// 990 TFLOP/s, where a large product reaches 1400; the matrix cores busy in 47 % of the cycles,
// 3.4 vector instructions to one of theirs, waves issuing in 41 % of theirs and waiting to
// issue in as many); narrow heads the vector instructions,
// 5 a score and one of them an exponential, against two matrix products of 24 channels,
// and the ways in and out (6 crops of 1 to 1003 residues, 16 heads of 24: 13.8 us, of them
// 3.4 until a workgroup's first block is there and 5.8 walking; 14.8 with the statistics);
// single tokens memory (8 caches of 9 to 16384 tokens: 19.5 us, 4.5 TB/s, and the join 3.8).
constexpr float kSlack = 8.f;

// An exponent is the rounding of s scale log2(e) - M with M rounded: off by up to half
// a step of M for all of a row's keys alike, which cancels in the softmax while 2 to that
// is a number. Rows with |M| beyond take products rounded by themselves, whose largest is
// M exactly.
constexpr float kFar = 16777216.f;

// SUMS: also the sum of the weights before their rounding, for the statistics. The rounded
// ones' is off by up to half a step of bf16 where a few keys have the weight (0.3 % measured),
// and the gradients' weights, which come anew, would all be off by that: a vector
// instruction a score more, where statistics are asked for.
template <typename T, int DP, int G, int KS, int R, bool SUMS>
__global__ __launch_bounds__((PkForm<G, KS>::kThreads), (PkFormOf<T, DP, G, KS>::type::template kSimd<T, DP>)) void packed_fwd_kernel(PackedParams<T> P) {
  typedef typename PkFormOf<T, DP, G, KS>::type Form;
  typedef PkRows<T, DP> Rows;
  typedef typename Frag<T>::type F;
  constexpr int kC = Rows::kC, kU = Rows::kU;
  constexpr int kNt = Form::kOwn / 16;  // key tiles of a wave in a block
  constexpr int kTileRows = 16 * R * G, kShift = __builtin_ctz(kTileRows);
  constexpr int kOperand = Form::kStage * Rows::kRowBytes;
  constexpr int kSets = Form::kSets;
  constexpr int kStages = 4 * kOperand * kSets <= 160 * 1024 ? 2 : 1;
  typedef PkOut<Form, DP> Out;
  constexpr int kRaw = kStages * 2 * kOperand * kSets;  // and at the end the outputs' way
  __shared__ __attribute__((aligned(16))) unsigned char raw[kRaw > Out::kBytes ? kRaw : Out::kBytes];
  __shared__ f32x2 wave_ml[R][KS][16 * G];  // maxima and sums
  __shared__ float wave_l[SUMS ? R : 1][KS][16 * G];  // sums of unrounded weights
  __shared__ int2 places[R][16 * G];        // the rows' heads and tokens; head -1: no such row

  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Form form(wave);
  const int kv = blockIdx.x, split = blockIdx.z;
  // without an order of their work, from the last tile on: causal rows with the most keys first
  const int nth = P.tile0 + blockIdx.y;
  PackedTile sp;
  if (!packed_tile(P, false, P.group, kShift, P.order ? nth : P.tiles - 1 - nth, lane, sp)) return;
  if (sp.seq == P.seqs && !P.zero_tail) return;
  const int row0 = sp.tile * kTileRows, rows = sp.nq * P.group - row0;  // those from row0 on
  if (rows <= 0) return;
  const int row_w = 16 * R * form.group;
  const PackedRows place(P, row0);

  // of the lane's rows: head, token, and the keys that it sees: those before lim
  int lim[R];
  F qf[R][kC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int x = row_w + 16 * r + li;
    int qi, head;
    place.at(x < rows ? x : rows - 1, qi, head);
    head += kv * P.group;
    lim[r] = P.causal ? qi + (sp.nk - sp.nq) + 1 : sp.nk;
    if (lg == 0 && form.part == 0) places[r][16 * form.group + li] = make_int2(x < rows ? head : -1, sp.q0 + qi);
    const T* q = P.q.p + head * P.q.head + (int64_t)(sp.q0 + qi) * P.q.token + 8 * lg;
#pragma unroll
    for (int c = 0; c < kC; ++c) qf[r][c] = 32 * c + 8 * lg < P.d ? load8(q + 32 * c) : F{};
  }
  int q_last, h_last;
  place.at((kTileRows < rows ? kTileRows : rows) - 1, q_last, h_last);
  const int most = P.causal ? q_last + (sp.nk - sp.nq) + 1 : sp.nk;  // keys that the workgroup's rows see
  const int lim_lo = __builtin_amdgcn_readfirstlane(lim[0]);      // that all of the wave's rows see,
  const int lim_hi = row_w < rows ? __builtin_amdgcn_readlane(lim[R - 1], 15) : 0;  // and that any does
  const int blocks = most > 0 ? (int)((uint32_t)(most + Form::kBlock - 1) / Form::kBlock) : 0;
  int blk0 = 0, blk1 = blocks;
  if (P.splits > 1) {
    const int each = (blocks + P.splits - 1) / P.splits;
    blk0 = split * each < blocks ? split * each : blocks;
    blk1 = blk0 + each < blocks ? blk0 + each : blocks;
  }

  unsigned char* const mine = raw + (Form::kPrivate ? wave * kStages * 2 * kOperand : 0);
  PkCopy<T, DP, Form::kStage, Form::kOwners> kcopy, vcopy;
  kcopy.init(P.k.token, P.d, form.stager, lane);
  vcopy.init(P.v.token, P.d, form.stager, lane);
  kcopy.begin(P.k.p + kv * P.k.head + (int64_t)sp.k0 * P.k.token, blk0 * Form::kBlock + form.staged(), sp.nk);
  vcopy.begin(P.v.p + kv * P.v.head + (int64_t)sp.k0 * P.v.token, blk0 * Form::kBlock + form.staged(), sp.nk);
  auto stage = [&](int at) {  // the next block
    unsigned char* s = mine + at * 2 * kOperand;
    kcopy.issue(s, form.stager, Form::kBlock);
    vcopy.issue(s + kOperand, form.stager, Form::kBlock);
  };
  PkLane<T, DP> at;
  at.init(lane);

  constexpr bool kOnes = sizeof(T) == 2;
  F ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = from_f32<T>(1.f);
  float m[R], unrounded[R];
  f32x4 l[R], o[R][kU];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    unrounded[r] = 0.f;
    l[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kU; ++u) o[r][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool far = false;

  if (kStages == 2) {
    if (blk0 < blk1) stage(0);
    pk_sync<Form>();
  }
  for (int blk = blk0; blk < blk1; ++blk) {
    const int cur = kStages == 2 ? (blk - blk0) & 1 : 0;
    if (kStages == 1) {
      stage(0);
      pk_sync<Form>();
    } else if (blk + 1 < blk1) {
      stage(cur ^ 1);
    }
    const unsigned char* kt_ = mine + cur * 2 * kOperand + form.at * Rows::kRowBytes;
    const unsigned char* vt_ = kt_ + kOperand;
    const int key0 = blk * Form::kBlock + Form::kOwn * form.part;
    if (key0 < lim_hi) {
      f32x4 s[R][kNt];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int kt = 0; kt < kNt; ++kt) s[r][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
      pk_ahead<kNt * kC>([&](int i) { return at.at_row(kt_, 16 * (i / kC), i % kC); },
                         [&](int i, const F& kf) {
#pragma unroll
                           for (int r = 0; r < R; ++r) mma(s[r][i / kC], kf, qf[r][i % kC]);
                         });
      if (key0 + 16 * kNt > lim_lo) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int left = lim[r] - key0 - 4 * lg;
#pragma unroll
          for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[r][kt][e] = 16 * kt + e < left ? s[r][kt][e] : -INFINITY;
        }
      }
      float top[R];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        top[r] = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < kNt; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[r] = pk_most(top[r], s[r][kt][e]);
        top[r] = lanes4_max(top[r]) * P.scale_log2;
        moved = moved || top[r] > m[r] + kSlack;
      }
      if (__builtin_amdgcn_ballot_w64(moved)) {
        bool any = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float mn = fmaxf(m[r], top[r]);
          const float alpha = __builtin_amdgcn_exp2f(m[r] - pk_base(mn));  // 0 where no key was before
          m[r] = mn;
          any = any || fabsf(pk_base(mn)) > kFar;
          if (SUMS) unrounded[r] *= alpha;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            l[r][e] *= alpha;
#pragma unroll
            for (int u = 0; u < kU; ++u) o[r][u][e] *= alpha;
          }
        }
        far = __builtin_amdgcn_ballot_w64(any);
      }
      float by = P.scale_log2;
      if (far) {
        by = 1.f;
#pragma unroll
        for (int r = 0; r < R; ++r) pk_round(P.scale_log2, s[r]);
      }
      F pf[R][kNt / 2];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float base = pk_base(m[r]);
#pragma unroll
        for (int c = 0; c < kNt / 2; ++c) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(s[r][2 * c + (e >> 2)][e & 3], by, -base));
            if (!kOnes) l[r][e & 3] += p[e];
          }
          if (SUMS) unrounded[r] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
          pf[r][c] = pack8<T>(p);
          if (kOnes) mma(l[r], ones, pf[r][c]);
        }
      }
      pk_ahead<kNt / 2 * kU>([&](int i) { return at.at_col(vt_, 32 * (i / kU), i % kU); },
                             [&](int i, const F& vf) {
#pragma unroll
                               for (int r = 0; r < R; ++r) mma(o[r][i % kU], vf, pf[r][i / kU]);
                             });
    }
    pk_sync<Form>();
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (SUMS) {
      const float sum = group_sum(unrounded[r]);
      if (lg == 0) wave_l[r][form.part][16 * form.group + li] = sum;
    }
    if (lg == 0 || !kOnes) {
      const float sum = kOnes ? l[r][0] : group_sum((l[r][0] + l[r][1]) + (l[r][2] + l[r][3]));
      if (lg == 0) wave_ml[r][form.part][16 * form.group + li] = f32x2{m[r], sum};
    }
  }
  // rows come together on the largest of their waves' maxima
#pragma unroll
  for (int r = 0; r < R; ++r)
    Out::write(raw, form, t, o[r], [&](int row, int c, const float* x) {
      const int2 to = places[r][row];
      if (to.x < 0) return;
      float mx = -INFINITY, sum = 0.f, all = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) mx = fmaxf(mx, wave_ml[r][j][row][0]);
      f32x8 v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const f32x2 ml = wave_ml[r][j][row];
        const float w = __builtin_amdgcn_exp2f(ml[0] - pk_base(mx));
        const f32x8 y = load8(x + j * Out::kPart);
        sum = fmaf(ml[1], w, sum);
        if (SUMS) all = fmaf(wave_l[r][j][row], w, all);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(y[e], w, v[e]);
      }
      const int64_t at_row = (int64_t)to.x * P.tq + to.y;
      if (P.splits > 1) {
        const int64_t part = (int64_t)split * P.heads * P.tq + at_row;
        if (c == 0) *reinterpret_cast<f32x2*>(P.part_ml + part * 2) = f32x2{mx, sum};
        if (SUMS && c == 0) P.part_l[part] = all;
        store8(P.part_o + part * DP + c, v);
        return;
      }
      if (c == 0 && P.lse) *reinterpret_cast<f32x2*>(P.lse + at_row * 2) = pk_stats(mx, SUMS ? all : sum);
      if (c >= P.d) return;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row without keys is zeros
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v[e] * inv;
      store8(P.out.p + to.x * P.out.head + to.y * P.out.token + c, pack8<T>(y));
      if (!P.rest.p) return;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] -= round_to<T>(y[e]);
      store8(P.rest.p + to.x * P.rest.head + to.y * P.rest.token + c, pack8<T>(y));
    });
}

// The splits of a row joined: a workgroup a row, wave w taking every fourth split
// from w on, lane l holding DP / 64 values (of DP = 32 half the lanes one).
template <typename T, int DP, bool SUMS>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedParams<T> P) {
  constexpr int kV = DP > 64 ? DP / 64 : 1;
  __shared__ float lds_o[4][DP];
  __shared__ float lds_l[4];
  __shared__ float lds_all[SUMS ? 4 : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = P.heads * P.tq, at = blockIdx.x;
  const int64_t token = at % P.tq;
  const int head = (int)(at / P.tq);
  // rows of no sequence have no parts
  if (token >= packed_int(P.q_starts, P.seqs, P.tq) && !P.zero_tail) return;
  float mx = -INFINITY;
  for (int s = lane; s < P.splits; s += 64) mx = fmaxf(mx, P.part_ml[(s * rows + at) * 2]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) mx = fmaxf(mx, shfl_xor(mx, x));
  const float base = pk_base(mx);
  float l = 0.f, all = 0.f, o[kV] = {};
#pragma unroll 8
  for (int s = wave; s < P.splits; s += 4) {
    const int64_t i = s * rows + at;
    const f32x2 v = *reinterpret_cast<const f32x2*>(P.part_ml + i * 2);
    const float w = __builtin_amdgcn_exp2f(v[0] - base);
    l = fmaf(v[1], w, l);
    if (SUMS) all = fmaf(P.part_l[i], w, all);
#pragma unroll
    for (int j = 0; j < kV; ++j)
      if (64 * j + lane < DP) o[j] = fmaf(P.part_o[i * DP + 64 * j + lane], w, o[j]);
  }
  if (lane == 0) lds_l[wave] = l;
  if (SUMS && lane == 0) lds_all[wave] = all;
#pragma unroll
  for (int j = 0; j < kV; ++j)
    if (64 * j + lane < DP) lds_o[wave][64 * j + lane] = o[j];
  __syncthreads();
  if (wave) return;
  const float sum = (lds_l[0] + lds_l[1]) + (lds_l[2] + lds_l[3]);
  if (lane == 0 && P.lse)
    *reinterpret_cast<f32x2*>(P.lse + at * 2) = pk_stats(mx, SUMS ? (lds_all[0] + lds_all[1]) + (lds_all[2] + lds_all[3]) : sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* out = P.out.p + head * P.out.head + token * P.out.token;
  T* rest = P.rest.p + head * P.rest.head + token * P.rest.token;
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const int x = 64 * j + lane;
    if (x >= P.d) continue;
    const float v = ((lds_o[0][x] + lds_o[1][x]) + (lds_o[2][x] + lds_o[3][x])) * inv;
    out[x] = from_f32<T>(v);
    if (P.rest.p) rest[x] = from_f32<T>(v - round_to<T>(v));
  }
}

// The tiles of one key/value head by their work, longest first: they are dealt to the
// card in this order, and the last to end are short ones (8 causal sequences of one
// length leave half the card idle at the end else, a long one that comes last more).
// One workgroup: a tile's work, the number of key blocks (dk, dv: query blocks) that
// it walks, kept in LDS, then a counting sort by 256 classes of it. The order within a
// class changes nothing but who starts first.
template <typename T>
__global__ __launch_bounds__(1024) void packed_order_kernel(PackedParams<T> P, PackedForm by_rows, PackedForm of_keys) {
  // a workgroup for each order that is asked for
  const bool by_keys = !by_rows.order || blockIdx.x;
  const PackedForm form = by_keys ? of_keys : by_rows;
  PackedTile* const order = form.order;
  const int count = form.count, shift = __builtin_ctz(form.rows());
  constexpr int kClasses = 256;
  __shared__ int work[kPackedOrder], seqs[kPackedOrder];
  __shared__ int classes[kClasses], most;
  __shared__ int q_at[kPackedOrderSeqs + 1], k_at[kPackedOrderSeqs + 1], length[kPackedOrderSeqs + 1];
  const int t = threadIdx.x;
  if (t < kClasses) classes[t] = 0;
  if (t == 0) most = 0;
  __syncthreads();
  const int per = by_keys ? 1 : P.group;
  // the offsets, fetched once: the search and both passes over the tiles wait for no memory
  for (int s = t; s <= P.seqs; s += 1024) {
    q_at[s] = (int)packed_start(P.q_starts, s, P.tq);
    k_at[s] = (int)packed_start(P.k_starts, s, P.tk);
    length[s] = P.k_lengths.p && s < P.seqs ? (int)packed_int(P.k_lengths, s, P.tk) : 0x7fffffff;
  }
  __syncthreads();
  auto first = [&](int s) { return (int)(((int64_t)(by_keys ? k_at : q_at)[s] * per) >> shift) + s; };
  auto tile_of = [&](int i, int seq) {
    PackedTile s;
    const int next = seq < P.seqs ? seq + 1 : seq;
    s.seq = seq;
    s.tile = i - first(seq);
    s.pad = 0;
    packed_tokens(P, by_keys, q_at[seq], q_at[next], k_at[seq], k_at[next], length[seq], s);
    return s;
  };
  for (int i = t; i < count; i += 1024) {
    int lo = 0, hi = P.seqs + 1;  // the last s whose first tile is not behind i
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first(mid) <= i)
        lo = mid;
      else
        hi = mid;
    }
    const PackedTile s = tile_of(i, lo);
    const int64_t row0 = (int64_t)s.tile << shift, rows = by_keys ? s.cap : (int64_t)s.nq * P.group;
    int blocks = -1;
    if (s.tile >= 0 && row0 < rows && (s.seq < P.seqs || P.zero_tail)) {
      int64_t walk;
      if (by_keys) {
        const int64_t from = P.causal && row0 + s.nq - s.nk > 0 ? row0 + s.nq - s.nk : 0;  // the first query
        walk = row0 < s.nk && from < s.nq ? s.nq - from : 0;
      } else {
        const int64_t last = (row0 + (1 << shift) < rows ? row0 + (1 << shift) : rows) - 1;
        walk = P.causal ? last / P.group + s.nk - s.nq + 1 : s.nk;
      }
      blocks = walk > 0 ? (int)((walk + 63) / 64) : 0;
      atomicMax(&most, blocks);
    }
    work[i] = blocks;
    seqs[i] = s.seq;
  }
  __syncthreads();
  const int top = most + 1;
  auto class_of = [&](int w) { return kClasses - 1 - (int)((int64_t)w * kClasses / top); };
  for (int i = t; i < count; i += 1024)
    if (work[i] >= 0) atomicAdd(&classes[class_of(work[i])], 1);
  __syncthreads();
  if (t < 64) {  // where each class begins
    int c[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = sum;
      sum += classes[4 * t + j];
    }
    int before = sum;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const int o = __shfl_up(before, x, 64);
      if (t >= x) before += o;
    }
    before -= sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) classes[4 * t + j] = before + c[j];
    if (t == 63) most = before + sum;
  }
  __syncthreads();
  for (int i = t; i < count; i += 1024)
    if (work[i] >= 0) order[atomicAdd(&classes[class_of(work[i])], 1)] = tile_of(i, seqs[i]);
  for (int i = most + t; i < count; i += 1024) order[i].seq = -1;
}

template <typename T, int DP, bool SUMS>
void fwd(const PackedParams<T>& P, const PackedForm& form, hipStream_t st) {
  pk_form<T>(form, [&](auto g, auto ks, auto r) {
    constexpr int G = decltype(g)::value, KS = decltype(ks)::value, R = decltype(r)::value;
    pk_grid(P, [&](const PackedParams<T>& Q, dim3 grid) {
      packed_fwd_kernel<T, DP, G, KS, R, SUMS><<<grid, PkForm<G, KS>::kThreads, 0, st>>>(Q);
    });
  });
  if (P.splits > 1) packed_join_kernel<T, DP, SUMS><<<(unsigned)(P.heads * P.tq), 256, 0, st>>>(P);
}
template <typename T, int DP>
void fwd(const PackedParams<T>& P, const PackedForm& form, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (P.lse) return fwd<T, DP, true>(P, form, st);
  fwd<T, DP, false>(P, form, st);
}

}  // namespace

template <typename T>
void launch_packed_order(const PackedParams<T>& P, const PackedForm& rows, const PackedForm& keys, hipStream_t st) {
  const int orders = (rows.order != nullptr) + (keys.order != nullptr);
  if (orders) packed_order_kernel<T><<<orders, 1024, 0, st>>>(P, rows, keys);
}
template void launch_packed_order<bf16>(const PackedParams<bf16>&, const PackedForm&, const PackedForm&, hipStream_t);
template void launch_packed_order<float>(const PackedParams<float>&, const PackedForm&, const PackedForm&, hipStream_t);

template <typename T>
void launch_packed_fwd(const PackedParams<T>& P, const PackedForm& form, hipStream_t st) {
  launch_packed_order(P, form, PackedForm{}, st);
  if (P.d <= 32)
    fwd<T, 32>(P, form, st);
  else if (P.d <= 64)
    fwd<T, 64>(P, form, st);
  else
    fwd<T, 128>(P, form, st);
}
template void launch_packed_fwd<bf16>(const PackedParams<bf16>&, const PackedForm&, hipStream_t);
template void launch_packed_fwd<float>(const PackedParams<float>&, const PackedForm&, hipStream_t);

}  // namespace fjx
