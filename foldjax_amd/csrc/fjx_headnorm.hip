// The norm of each head's queries and keys and their rotation by position, one pass
// over memory for both, and its gradients.
//
//   n = x / sqrt(mean(x^2) + eps) * w          (x itself without a weight)
//   y = (n_a cos t - n_b sin t, n_a sin t + n_b cos t) for each pair (a, b) of
//   channels, t = position * frequency; channels behind the pairs as they are
//   dn = dy rotated back;  dx = rstd (u - h mean(u h)), u = dn w, h = x rstd;
//   dw = sum over tokens and heads of dn h
//
// A team of lanes takes a token and walks its heads, so that a token's cosines are
// computed once: 8 channels a lane, 4 pairs with both members (two pieces of 4
// channels, which half a row lies between when pairs are (i, i + half)). Angles are
// taken in 64 bits and reduced in turns: float32 would lose 1e-2 of an angle at position
// 1e5. A row stays in registers.
//
// Memory bounds it: queries and keys of 16384 tokens, 8 + 2 heads of 128, 17.1 us (84 MB,
// 4.9 TB/s; a copy of as many bytes 16.1); with gradients at 8192 tokens 11.5 and 16.2, and
// 3.8 for the workgroups' sums of the weights' gradients; smaller calls the latency of a
// token's chain (positions, cosines in 64 bits, a row), 4.2.
#include <type_traits>

#include "fjx_common.hpp"
#include "fjx_kernels.hpp"

namespace fjx {

namespace {

constexpr int kBatch = 4, kBwdBatch = 2;  // heads whose loads are on their way together

template <typename T> struct Quad4;
template <> struct Quad4<bf16> { typedef bf16x4 type; };
template <> struct Quad4<float> { typedef f32x4 type; };
__device__ __forceinline__ void widen(const bf16x4& v, float (&o)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(v[e]);
}
__device__ __forceinline__ void widen(const f32x4& v, float (&o)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = v[e];
}

// what a lane needs of its token: cosines and sines of its 4 pairs
struct Turn {
  float c[4], s[4];
};

template <typename T>
__device__ __forceinline__ Turn turn_of(const HeadNormParams<T>& P, int64_t item, int64_t token, int unit) {
  Turn r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    r.c[e] = 1.f;
    r.s[e] = 0.f;
  }
  if (4 * unit >= P.pairs) return r;
  double turns[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int pair = 4 * unit + e;
    const int axis = (pair >= P.axis_end[0]) + (pair >= P.axis_end[1]) + (pair >= P.axis_end[2]);
    const int64_t at = axis * P.pos_axis + item * P.pos_item + token;
    const double pos = P.pos_wide ? (double)static_cast<const int64_t*>(P.positions)[at]
                                  : (double)static_cast<const int32_t*>(P.positions)[at];
    turns[e] = pos * P.frequencies[pair] * 0.15915494309189535;  // 1 / (2 pi)
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sincospif((float)(2.0 * (turns[e] - rint(turns[e]))), &r.s[e], &r.c[e]);
  return r;
}

// both pieces of a lane turned; BACK: by the negative angle
template <bool NEXT, bool BACK>
__device__ __forceinline__ void rotate(const Turn& t, float (&a)[4], float (&b)[4]) {
  auto two = [](float c, float s, float& x, float& y) {
    const float x0 = x, y0 = y;
    x = BACK ? fmaf(x0, c, y0 * s) : fmaf(x0, c, -y0 * s);
    y = BACK ? fmaf(y0, c, -x0 * s) : fmaf(y0, c, x0 * s);
  };
  if constexpr (NEXT) {  // pairs of neighbours
    two(t.c[0], t.s[0], a[0], a[1]);
    two(t.c[1], t.s[1], a[2], a[3]);
    two(t.c[2], t.s[2], b[0], b[1]);
    two(t.c[3], t.s[3], b[2], b[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) two(t.c[e], t.s[e], a[e], b[e]);
  }
}

// the sum over the TEAM lanes of a row, by lane permutes of vector instructions: within
// quads, by mirrors of 8 and 16 lanes (whose halves hold one value each by then), and
// of two rows of 16
template <int CTRL>
__device__ __forceinline__ float add_lanes(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
template <int TEAM>
__device__ __forceinline__ float team_sum(float v) {
  v = quad_sum(v);
  if constexpr (TEAM >= 8) v = add_lanes<0x141>(v);
  if constexpr (TEAM >= 16) v = add_lanes<0x140>(v);
  if constexpr (TEAM >= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t x0 = x[0], x1 = x[1];
    v = __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1);
  }
  return v;
}

__device__ __forceinline__ float dot4(const float (&x)[4], const float (&y)[4], float s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) s = fmaf(x[e], y[e], s);
  return s;
}

// the first channels of a lane's two pieces
template <bool NEXT, typename T>
__device__ __forceinline__ void pieces_of(const HeadNormParams<T>& P, int unit, int& a, int& b) {
  const bool halves = !NEXT && 4 * unit < P.pairs;
  a = halves ? 4 * unit : 8 * unit;
  b = halves ? P.pairs + 4 * unit : 8 * unit + 4;
}

// A workgroup's heads, of [queries, keys] one after the other, are the same for all its
// teams: addresses are a head's, scalar, and the token's, a lane's own.
struct Heads {
  int q0, q1, k0, k1;
};
template <typename T>
__device__ __forceinline__ Heads heads_of(const HeadNormParams<T>& P, int chunk) {
  const int q = P.heads[0], h0 = chunk * P.per_chunk, h1 = h0 + P.per_chunk;
  Heads r;
  r.q0 = h0 < q ? h0 : q;
  r.q1 = h1 < q ? h1 : q;
  r.k0 = h0 > q ? h0 - q : 0;
  r.k1 = h1 - q < P.heads[1] ? h1 - q : P.heads[1];
  return r;
}
template <typename V>
__device__ __forceinline__ int64_t place_in(const V& v, int64_t item, int64_t token, int ca) {
  return item * v.item + token * v.token + ca;
}

// both pieces of a batch of heads, as they lie in memory; off: the lane's first piece
// in a head, step: from there to the second
template <typename T, int N>
struct Batch {
  typename Quad4<T>::type a[N], b[N];
  template <typename V>
  __device__ __forceinline__ void load(const V& v, int h, int h1, int64_t off, int step) {
    const T* p = v.p + h * v.head;
    int64_t head = v.head;
    asm volatile("" : "+s"(head));  // its multiples, kept through a loop, took more scalars than there are
#pragma unroll
    for (int x = 0; x < N; ++x, p += head) {
      a[x] = b[x] = typename Quad4<T>::type{};
      if (h + x >= h1) continue;
      a[x] = *reinterpret_cast<const typename Quad4<T>::type*>(p + off);
      b[x] = *reinterpret_cast<const typename Quad4<T>::type*>(p + off + step);
    }
  }
};

template <typename T>
__device__ __forceinline__ void weights_of(const T* w, int ca, int cb, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  if (!w) return;
  load4f(w + ca, o);
  load4f(w + cb, o + 4);
}

// Lanes behind a row's last channel (a row is 3/4 of a team at 24 channels) take its
// last piece again, with a share of nothing in its sums, and write nothing.
template <typename T, int TEAM, bool NEXT, int I>
__device__ __forceinline__ void norm_heads(const HeadNormParams<T>& P, int h0, int h1, int64_t from, int64_t to, int step,
                                           const float (&w)[8], const Turn& turn, Batch<T, kBatch>& x, bool on) {
  const bool normed = P.w[I] != nullptr;
  for (int h = h0; h < h1; h += kBatch) {
    if (h > h0) x.load(P.x[I], h, h1, from, step);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (h + j >= h1) break;
      float a[4], b[4];
      widen(x.a[j], a);
      widen(x.b[j], b);
      if (normed) {
        const float ss = dot4(a, a, dot4(b, b, 0.f));
        const float rstd = __builtin_amdgcn_rsqf(team_sum<TEAM>(on ? ss : 0.f) * P.inv_d + P.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] *= rstd * w[e];
          b[e] *= rstd * w[4 + e];
        }
      }
      rotate<NEXT, false>(turn, a, b);
      if (!on) continue;
      T* p = P.y[I].p + (h + j) * P.y[I].head;
      store4f(p + to, a);
      store4f(p + to + step, b);
    }
  }
}

// The first batch's loads go out before the cosines are computed.
template <typename T, int TEAM, bool NEXT>
__global__ __launch_bounds__(256) void headnorm_kernel(HeadNormParams<T> P) {
  const int64_t block = P.first + blockIdx.x, group = block / P.chunks;
  const Heads hs = heads_of(P, (int)(block - group * P.chunks));
  const int64_t id = group * (256 / TEAM) + threadIdx.x / TEAM;
  if (id >= P.items * P.tokens) return;  // a whole team
  const int64_t item = id / P.tokens, token = id - item * P.tokens;
  int unit = threadIdx.x % TEAM;
  const bool on = 8 * unit < P.d;
  if (!on) unit = P.d / 8 - 1;
  int ca, cb;
  pieces_of<NEXT>(P, unit, ca, cb);
  Batch<T, kBatch> x;
  const int64_t from_q = place_in(P.x[0], item, token, ca), from_k = place_in(P.x[1], item, token, ca);
  if (hs.q0 < hs.q1)
    x.load(P.x[0], hs.q0, hs.q1, from_q, cb - ca);
  else
    x.load(P.x[1], hs.k0, hs.k1, from_k, cb - ca);
  float w[8];
  weights_of(P.w[hs.q0 < hs.q1 ? 0 : 1], ca, cb, w);
  const Turn turn = turn_of(P, item, token, unit);
  if (hs.q0 < hs.q1) {
    norm_heads<T, TEAM, NEXT, 0>(P, hs.q0, hs.q1, from_q, place_in(P.y[0], item, token, ca), cb - ca, w, turn, x, on);
    if (hs.k0 >= hs.k1) return;
    x.load(P.x[1], hs.k0, hs.k1, from_k, cb - ca);
    weights_of(P.w[1], ca, cb, w);
  }
  norm_heads<T, TEAM, NEXT, 1>(P, hs.k0, hs.k1, from_k, place_in(P.y[1], item, token, ca), cb - ca, w, turn, x, on);
}

// The gradients of the same, y being those of the outputs and g those of the inputs.
// The weights' gradients are summed over a team's heads and tokens in registers, then
// over the workgroup's teams; headnorm_dw_kernel adds the workgroups' sums
// [gridDim.x][2][d] in one order.
template <typename T, int TEAM, bool NEXT>
__global__ __launch_bounds__(256, 3) void headnorm_bwd_kernel(HeadNormParams<T> P) {
  constexpr int kTeams = 256 / TEAM;
  __shared__ float sums[2][8 * TEAM][kTeams + 1];
  const int group = blockIdx.x / P.chunks, groups = gridDim.x / P.chunks;
  const Heads hs = heads_of(P, blockIdx.x - group * P.chunks);
  const int team = threadIdx.x / TEAM;
  int unit = threadIdx.x % TEAM;
  const bool on = 8 * unit < P.d;
  if (!on) unit = P.d / 8 - 1;
  int ca, cb;
  pieces_of<NEXT>(P, unit, ca, cb);
  const int step = cb - ca;
  float dw[2][8] = {};
  for (int64_t id = (int64_t)group * kTeams + team; id < P.items * P.tokens; id += (int64_t)groups * kTeams) {
    const int64_t item = id / P.tokens, token = id - item * P.tokens;
    Turn turn;
    bool turned = false;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {  // queries, keys: one code for both
      const int h0 = i ? hs.k0 : hs.q0, h1 = i ? hs.k1 : hs.q1;
      if (h0 >= h1) continue;
      const HeadNormView<const T> vx = P.x[i];
      const HeadNormView<T> vy = P.y[i], vg = P.g[i];
      const bool normed = P.w[i] != nullptr;
      const int64_t from = place_in(vy, item, token, ca), from_x = place_in(vx, item, token, ca), to = place_in(vg, item, token, ca);
      Batch<T, kBwdBatch> dy, x;
      dy.load(vy, h0, h1, from, step);
      if (normed) x.load(vx, h0, h1, from_x, step);
      float w[8], d[8] = {};
      weights_of(P.w[i], ca, cb, w);
      if (!turned) turn = turn_of(P, item, token, unit);
      turned = true;
      for (int h = h0; h < h1; h += kBwdBatch) {
        if (h > h0) {
          dy.load(vy, h, h1, from, step);
          if (normed) x.load(vx, h, h1, from_x, step);
        }
        T* out = vg.p + h * vg.head;
        int64_t head = vg.head;
        asm volatile("" : "+s"(head));
#pragma unroll
        for (int j = 0; j < kBwdBatch; ++j, out += head) {
          if (h + j >= h1) break;
          float a[4], b[4];
          widen(dy.a[j], a);
          widen(dy.b[j], b);
          rotate<NEXT, true>(turn, a, b);
          if (normed) {
            float xa[4], xb[4], ss = 0.f, ux = 0.f;
            widen(x.a[j], xa);
            widen(x.b[j], xb);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              ss = fmaf(xa[e], xa[e], fmaf(xb[e], xb[e], ss));
              ux = fmaf(a[e] * w[e], xa[e], fmaf(b[e] * w[4 + e], xb[e], ux));
            }
            const float rstd = __builtin_amdgcn_rsqf(team_sum<TEAM>(on ? ss : 0.f) * P.inv_d + P.eps);
            const float mean = team_sum<TEAM>(on ? ux : 0.f) * P.inv_d * rstd;  // of u h
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float ha = xa[e] * rstd, hb = xb[e] * rstd;
              d[e] = fmaf(a[e], ha, d[e]);
              d[4 + e] = fmaf(b[e], hb, d[4 + e]);
              a[e] = rstd * (a[e] * w[e] - ha * mean);
              b[e] = rstd * (b[e] * w[4 + e] - hb * mean);
            }
          }
          if (!on) continue;
          store4f(out + to, a);
          store4f(out + to + step, b);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (i)
          dw[1][e] += d[e];
        else
          dw[0][e] += d[e];
      }
    }
  }
  if (!P.part) return;
  if (on)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[i][e < 4 ? ca + e : cb + e - 4][team] = dw[i][e];
  __syncthreads();
  for (int x = threadIdx.x; x < 2 * P.d; x += 256) {
    const float* p = x < P.d ? sums[0][x] : sums[1][x - P.d];
    float s = 0.f;
#pragma unroll 8
    for (int g = 0; g < kTeams; ++g) s += p[g];
    P.part[(int64_t)blockIdx.x * 2 * P.d + x] = s;
  }
}

// the workgroups' sums of the two weights, [blocks][2][d], added: 16 channels a
// workgroup, 64 threads each, so that a thread's few loads are on their way together
__global__ __launch_bounds__(1024) void headnorm_dw_kernel(const float* __restrict__ part, float* __restrict__ dwq,
                                                           float* __restrict__ dwk, int blocks, int d) {
  __shared__ float lds[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int ch = blockIdx.x * 16 + c;
  float s = 0.f;
#pragma unroll 8
  for (int b = g; b < blocks; b += 64) s += part[(int64_t)b * 2 * d + ch];
  lds[g][c] = s;
  __syncthreads();
  if (g >= 16) return;
  // a column's 64 sums by 16 lanes
  const int x = threadIdx.x >> 4, q = threadIdx.x & 15;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += lds[16 * i + q][x];
#pragma unroll
  for (int i = 8; i >= 1; i >>= 1) s += shfl_xor(s, i);
  const int out = blockIdx.x * 16 + x;
  float* dst = out < d ? dwq : dwk;
  if (q == 0 && dst) dst[out < d ? out : out - d] = s;
}

template <typename F>
void by_width(int d, bool next, F f) {
  auto both = [&](auto team) {
    if (next)
      f(team, std::true_type{});
    else
      f(team, std::false_type{});
  };
  if (d <= 32) return both(std::integral_constant<int, 4>{});
  if (d <= 64) return both(std::integral_constant<int, 8>{});
  if (d <= 128) return both(std::integral_constant<int, 16>{});
  both(std::integral_constant<int, 32>{});
}

int team_of(int d) { return d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32; }

// The heads of a token over `chunks` workgroups where the tokens alone do not fill the card
template <typename T>
void cut(HeadNormParams<T>& p) {
  const int64_t threads = p.items * p.tokens * team_of(p.d);
  const int heads = p.heads[0] + p.heads[1];
  const int64_t want = ((int64_t)1 << 17) / threads;
  const int most = (heads + kBatch - 1) / kBatch;
  p.chunks = (int)(want < 1 ? 1 : want < most ? want : most);
  p.per_chunk = (((heads + p.chunks - 1) / p.chunks) + kBatch - 1) / kBatch * kBatch;
  p.chunks = (heads + p.per_chunk - 1) / p.per_chunk;
  p.inv_d = 1.f / p.d;
}
// workgroups of tokens, and of all
template <typename T>
int64_t blocks_of(const HeadNormParams<T>& p) {
  return (p.items * p.tokens * team_of(p.d) + 255) / 256;
}
template <typename T>
int bwd_blocks_of(const HeadNormParams<T>& p) {
  const int64_t most = 1024 / p.chunks, blocks = blocks_of(p);
  return (int)(blocks < most ? blocks : most) * p.chunks;
}

}  // namespace

int headnorm_bwd_blocks(int64_t items, int64_t tokens, int heads, int d) {
  HeadNormParams<float> p = {};
  p.items = items;
  p.tokens = tokens;
  p.heads[0] = heads;
  p.d = d;
  cut(p);
  return bwd_blocks_of(p);
}

template <typename T>
void launch_headnorm(HeadNormParams<T> p, hipStream_t st) {
  cut(p);
  by_width(p.d, p.neighbours, [&](auto team, auto next) {
    constexpr int kTeam = decltype(team)::value;
    constexpr bool kNext = decltype(next)::value;
    for_pieces(blocks_of(p) * p.chunks, [&](int64_t first, unsigned blocks) {
      HeadNormParams<T> q = p;
      q.first = first;
      headnorm_kernel<T, kTeam, kNext><<<blocks, 256, 0, st>>>(q);
    });
  });
}

template <typename T>
void launch_headnorm_bwd(HeadNormParams<T> p, float* dwq, float* dwk, hipStream_t st) {
  cut(p);
  const int blocks = bwd_blocks_of(p);
  by_width(p.d, p.neighbours, [&](auto team, auto next) {
    headnorm_bwd_kernel<T, decltype(team)::value, decltype(next)::value><<<blocks, 256, 0, st>>>(p);
  });
  if (p.part) headnorm_dw_kernel<<<2 * p.d / 16, 1024, 0, st>>>(p.part, dwq, dwk, blocks, p.d);
}

template void launch_headnorm<bf16>(HeadNormParams<bf16>, hipStream_t);
template void launch_headnorm<float>(HeadNormParams<float>, hipStream_t);
template void launch_headnorm_bwd<bf16>(HeadNormParams<bf16>, float*, float*, hipStream_t);
template void launch_headnorm_bwd<float>(HeadNormParams<float>, float*, float*, hipStream_t);

}  // namespace fjx
