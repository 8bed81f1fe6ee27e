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
#include <type_traits>

#include "fjx_common.hpp"
#include "fjx_kernels.hpp"

namespace fjx {

namespace {

constexpr int kBatch = 4;  // heads whose loads are on their way together

__device__ __forceinline__ void load4(const bf16* p, float* o) { load4f(p, o); }
__device__ __forceinline__ void load4(const float* p, float* o) { load4f(p, o); }

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
    const int pair = 4 * unit + e;
    if (pair >= P.pairs) continue;
    const int axis = (pair >= P.axis_end[0]) + (pair >= P.axis_end[1]) + (pair >= P.axis_end[2]);
    const int64_t at = axis * P.pos_axis + item * P.pos_item + token;
    const double pos = P.pos_wide ? (double)static_cast<const int64_t*>(P.positions)[at]
                                  : (double)static_cast<const int32_t*>(P.positions)[at];
    const double turns = pos * P.frequencies[pair] * 0.15915494309189535;  // 1 / (2 pi)
    sincospif((float)(2.0 * (turns - rint(turns))), &r.s[e], &r.c[e]);
  }
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

template <int TEAM>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int x = TEAM / 2; x >= 1; x >>= 1) v += shfl_xor(v, x);
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

template <typename T, int TEAM, bool NEXT>
__global__ __launch_bounds__(256) void headnorm_kernel(HeadNormParams<T> P) {
  const int unit = threadIdx.x % TEAM;
  const int64_t id = (P.first + blockIdx.x) * (256 / TEAM) + threadIdx.x / TEAM;
  if (id >= P.items * P.tokens * P.chunks) return;  // a whole team
  const int chunk = (int)(id % P.chunks);
  const int64_t at = id / P.chunks, item = at / P.tokens, token = at - item * P.tokens;
  const bool on = 8 * unit < P.d;
  int ca, cb;
  pieces_of<NEXT>(P, unit, ca, cb);
  const Turn turn = turn_of(P, item, token, unit);
  const int h0 = chunk * P.per_chunk, h1 = h0 + P.per_chunk < P.heads[0] + P.heads[1] ? h0 + P.per_chunk : P.heads[0] + P.heads[1];
  float w[2][8] = {};
  if (on)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (P.w[i]) {
        load4(P.w[i] + ca, w[i]);
        load4(P.w[i] + cb, w[i] + 4);
      }
  for (int h = h0; h < h1; h += kBatch) {
    float a[kBatch][4], b[kBatch][4];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[x][e] = b[x][e] = 0.f;
      if (!on || h + x >= h1) continue;
      const int i = h + x >= P.heads[0];
      const HeadNormView<const T>& v = P.x[i];
      const T* p = v.p + item * v.item + (h + x - (i ? P.heads[0] : 0)) * v.head + token * v.token;
      load4(p + ca, a[x]);
      load4(p + cb, b[x]);
    }
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      if (h + x >= h1) break;
      const int i = h + x >= P.heads[0];
      if (P.w[i]) {
        const float rstd = __builtin_amdgcn_rsqf(team_sum<TEAM>(dot4(a[x], a[x], dot4(b[x], b[x], 0.f))) / P.d + P.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[x][e] *= rstd * (i ? w[1][e] : w[0][e]);
          b[x][e] *= rstd * (i ? w[1][4 + e] : w[0][4 + e]);
        }
      }
      rotate<NEXT, false>(turn, a[x], b[x]);
      if (!on) continue;
      const HeadNormView<T>& v = P.y[i];
      T* p = v.p + item * v.item + (h + x - (i ? P.heads[0] : 0)) * v.head + token * v.token;
      store4f(p + ca, a[x]);
      store4f(p + cb, b[x]);
    }
  }
}

// y: the gradients of the outputs, g: those of the inputs. The weights' gradients are
// summed over a team's heads and tokens in registers, then over the workgroup's teams;
// headnorm_dw_kernel adds the workgroups' sums [gridDim.x][2][d] in one order.
template <typename T, int TEAM, bool NEXT>
__global__ __launch_bounds__(256) void headnorm_bwd_kernel(HeadNormParams<T> P) {
  constexpr int kTeams = 256 / TEAM;
  __shared__ float sums[2][8 * TEAM];
  const int unit = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const bool on = 8 * unit < P.d;
  int ca, cb;
  pieces_of<NEXT>(P, unit, ca, cb);
  float w[2][8] = {}, dw[2][8] = {};
  if (on)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (P.w[i]) {
        load4(P.w[i] + ca, w[i]);
        load4(P.w[i] + cb, w[i] + 4);
      }
  const int64_t all = P.items * P.tokens * P.chunks;
  for (int64_t id = (int64_t)blockIdx.x * kTeams + team; id < all; id += (int64_t)gridDim.x * kTeams) {
    const int chunk = (int)(id % P.chunks);
    const int64_t at = id / P.chunks, item = at / P.tokens, token = at - item * P.tokens;
    const Turn turn = turn_of(P, item, token, unit);
    const int h0 = chunk * P.per_chunk, h1 = h0 + P.per_chunk < P.heads[0] + P.heads[1] ? h0 + P.per_chunk : P.heads[0] + P.heads[1];
    for (int h = h0; h < h1; h += kBatch) {
      float a[kBatch][4], b[kBatch][4], xa[kBatch][4], xb[kBatch][4];
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[x][e] = b[x][e] = xa[x][e] = xb[x][e] = 0.f;
        if (!on || h + x >= h1) continue;
        const int i = h + x >= P.heads[0];
        const int head = h + x - (i ? P.heads[0] : 0);
        const T* p = P.y[i].p + item * P.y[i].item + head * P.y[i].head + token * P.y[i].token;
        load4(p + ca, a[x]);
        load4(p + cb, b[x]);
        if (!P.w[i]) continue;
        p = P.x[i].p + item * P.x[i].item + head * P.x[i].head + token * P.x[i].token;
        load4(p + ca, xa[x]);
        load4(p + cb, xb[x]);
      }
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        if (h + x >= h1) break;
        const int i = h + x >= P.heads[0];
        rotate<NEXT, true>(turn, a[x], b[x]);
        if (P.w[i]) {
          float ua[4], ub[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ua[e] = a[x][e] * (i ? w[1][e] : w[0][e]);
            ub[e] = b[x][e] * (i ? w[1][4 + e] : w[0][4 + e]);
          }
          const float ss = team_sum<TEAM>(dot4(xa[x], xa[x], dot4(xb[x], xb[x], 0.f)));
          const float ux = team_sum<TEAM>(dot4(ua, xa[x], dot4(ub, xb[x], 0.f)));
          const float rstd = __builtin_amdgcn_rsqf(ss / P.d + P.eps);
          const float mean = ux / P.d * rstd;  // of u h
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ha = xa[x][e] * rstd, hb = xb[x][e] * rstd;
            const float da = a[x][e] * ha, db = b[x][e] * hb;
            dw[0][e] += i ? 0.f : da;
            dw[1][e] += i ? da : 0.f;
            dw[0][4 + e] += i ? 0.f : db;
            dw[1][4 + e] += i ? db : 0.f;
            a[x][e] = rstd * (ua[e] - ha * mean);
            b[x][e] = rstd * (ub[e] - hb * mean);
          }
        }
        if (!on) continue;
        T* p = P.g[i].p + item * P.g[i].item + (h + x - (i ? P.heads[0] : 0)) * P.g[i].head + token * P.g[i].token;
        store4f(p + ca, a[x]);
        store4f(p + cb, b[x]);
      }
    }
  }
  if (!P.part) return;
  for (int g = 0; g < kTeams; ++g) {  // the workgroup's teams, one after the other
    __syncthreads();
    if (team == g && on)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float& s = sums[i][e < 4 ? ca + e : cb + e - 4];
          s = g ? s + dw[i][e] : dw[i][e];
        }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 2 * P.d; x += 256)
    P.part[(int64_t)blockIdx.x * 2 * P.d + x] = sums[x >= P.d][x >= P.d ? x - P.d : x];
}

// the workgroups' sums of the two weights, [blocks][2][d], added: 16 waves of a
// workgroup take every sixteenth
__global__ __launch_bounds__(1024) void headnorm_dw_kernel(const float* __restrict__ part, float* __restrict__ dwq,
                                                           float* __restrict__ dwk, int blocks, int d) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ch = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (ch < 2 * d) {
#pragma unroll 8
    for (int b = wave; b < blocks; b += 16) s += part[(int64_t)b * 2 * d + ch];
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave || ch >= 2 * d) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += lds[w][lane];
  float* out = ch < d ? dwq : dwk;
  if (out) out[ch < d ? ch : ch - d] = s;
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

// The heads of a token over `chunks` teams where the tokens alone do not fill the card
template <typename T>
void cut(HeadNormParams<T>& p) {
  const int64_t threads = p.items * p.tokens * team_of(p.d);
  const int heads = p.heads[0] + p.heads[1];
  const int64_t want = ((int64_t)1 << 18) / threads;
  const int most = (heads + kBatch - 1) / kBatch;
  p.chunks = (int)(want < 1 ? 1 : want < most ? want : most);
  p.per_chunk = (heads + p.chunks - 1) / p.chunks;
  p.chunks = (heads + p.per_chunk - 1) / p.per_chunk;
}

}  // namespace

int headnorm_bwd_blocks(int64_t items, int64_t tokens, int heads, int d) {
  HeadNormParams<float> p = {};
  p.items = items;
  p.tokens = tokens;
  p.heads[0] = heads;
  p.d = d;
  cut(p);
  const int64_t blocks = (items * tokens * p.chunks * team_of(d) + 255) / 256;
  return (int)(blocks < 1024 ? blocks : 1024);
}

template <typename T>
void launch_headnorm(HeadNormParams<T> p, hipStream_t st) {
  cut(p);
  by_width(p.d, p.neighbours, [&](auto team, auto next) {
    constexpr int kTeam = decltype(team)::value;
    constexpr bool kNext = decltype(next)::value;
    for_pieces((p.items * p.tokens * p.chunks * kTeam + 255) / 256, [&](int64_t first, unsigned blocks) {
      HeadNormParams<T> q = p;
      q.first = first;
      headnorm_kernel<T, kTeam, kNext><<<blocks, 256, 0, st>>>(q);
    });
  });
}

template <typename T>
void launch_headnorm_bwd(HeadNormParams<T> p, float* dwq, float* dwk, hipStream_t st) {
  cut(p);
  const int blocks = headnorm_bwd_blocks(p.items, p.tokens, p.heads[0] + p.heads[1], p.d);
  by_width(p.d, p.neighbours, [&](auto team, auto next) {
    headnorm_bwd_kernel<T, decltype(team)::value, decltype(next)::value><<<blocks, 256, 0, st>>>(p);
  });
  if (p.part) headnorm_dw_kernel<<<(2 * p.d + 63) / 64, 1024, 0, st>>>(p.part, dwq, dwk, blocks, p.d);
}

template void launch_headnorm<bf16>(HeadNormParams<bf16>, hipStream_t);
template void launch_headnorm<float>(HeadNormParams<float>, hipStream_t);
template void launch_headnorm_bwd<bf16>(HeadNormParams<bf16>, float*, float*, hipStream_t);
template void launch_headnorm_bwd<float>(HeadNormParams<float>, float*, float*, hipStream_t);

}  // namespace fjx
