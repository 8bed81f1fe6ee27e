// Root-mean-square norm with the residual's addition, its 8-bit output and its
// gradients. One pass over memory: a row stays in the registers of the lanes
// that share it, 8 channels (16 bytes of bf16) a lane and piece.
//
//   h = x + r;  y = h rstd w,  rstd = (mean h^2 + eps)^-1/2
//   codes: scale = max |y| / most over a row or a group of channels, y / scale
//          in e4m3 (most = 448) or int8 (127)
//   dx = rstd (t - n mean(t n)) + dh,  t = dy w, n = h rstd;  dw = sum over rows of dy n
//
// Bound by memory: 1003 x 1003 rows of 128 bf16 channels with the residual into e4m3
// codes and the sum (901 MB) 148 us, 6.1 TB/s; 120050 rows of 64 float32 channels
// forward 13.1 us (61 MB) and backward 18.7 (92 MB), 4.7 and 4.9 TB/s, then 4.7 for dw.
#include <type_traits>

#include "fjx_common.hpp"
#include "fjx_kernels.hpp"

namespace fjx {

namespace {

// The sum over the TEAM lanes of a row: within a wave, or (TEAM 256) over the
// four waves of the workgroup through LDS.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* lds) {
#pragma unroll
  for (int x = (TEAM < 64 ? TEAM : 64) / 2; x >= 1; x >>= 1) v += shfl_xor(v, x);
  if constexpr (TEAM > 64) {
    __syncthreads();  // the last sum's values are read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
  return v;
}
// the maximum of |values| as bits, where a NaN is the largest of all
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
template <int TEAM>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t* lds) {
#pragma unroll
  for (int x = (TEAM < 64 ? TEAM : 64) / 2; x >= 1; x >>= 1) {
    const uint32_t o = __shfl_xor(v, x, 64);
    v = o > v ? o : v;
  }
  if constexpr (TEAM > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) v = lds[w] > v ? lds[w] : v;
  }
  return v;
}

template <typename T, int TEAM, int PIECES, int CODES>
__global__ __launch_bounds__(256) void rmsnorm_kernel(RmsNormParams<T> P) {
  __shared__ float lds[4];
  __shared__ uint32_t lds_u[4];
  constexpr int kTeams = 256 / TEAM;
  const int lane = threadIdx.x % TEAM;
  int64_t row = (P.first + blockIdx.x) * kTeams + threadIdx.x / TEAM;
  const bool row_on = row < P.rows;
  if (!row_on) row = P.rows - 1;  // stays for the sums
  const int64_t at = row * P.c;
  float h[PIECES][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int ch = (i * TEAM + lane) * 8;
    if (ch < P.c) {
      to_f32x8(load8(P.x + at + ch), h[i]);
      if (P.residual) {
        float r[8];
        to_f32x8(load8(P.residual + at + ch), r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] += r[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
  }
  const float rstd = __builtin_amdgcn_rsqf(team_sum<TEAM>(ss, lds) / P.c + P.eps);
  uint32_t top[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int ch = (i * TEAM + lane) * 8;
    top[i] = 0;
    if (ch >= P.c) continue;
    // the sum goes out rounded, the norm is taken of the unrounded one
    if (P.h && row_on) store8(P.h + at + ch, pack8<T>(h[i]));
    float w[8];
    to_f32x8(load8(P.w + ch), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[i][e] *= rstd * w[e];
      if (CODES) top[i] = abs_bits(h[i][e]) > top[i] ? abs_bits(h[i][e]) : top[i];
    }
    if (!CODES && row_on) store8(P.y + at + ch, pack8<T>(h[i]));
  }
  if constexpr (CODES != 0) {
    const float most = CODES == 1 ? 448.f : 127.f;
    const bool by_row = P.group == P.c;
    if (by_row) {
      uint32_t v = top[0];
#pragma unroll
      for (int i = 1; i < PIECES; ++i) v = top[i] > v ? top[i] : v;
      v = team_max<TEAM>(v, lds_u);
#pragma unroll
      for (int i = 0; i < PIECES; ++i) top[i] = v;
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        for (int x = P.group / 16; x >= 1; x >>= 1) {  // group / 8 adjacent lanes
          const uint32_t o = __shfl_xor(top[i], x, 64);
          top[i] = o > top[i] ? o : top[i];
        }
    }
    if (!row_on) return;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int ch = (i * TEAM + lane) * 8;
      if (ch >= P.c) continue;
      const float amax = __builtin_bit_cast(float, top[i]);
      const bool none = amax < 1e-30f;  // no scale for what float32's reciprocals cannot reach: zeros
      const float inv = none ? 0.f : most / amax;
      if (ch % P.group == 0) P.scales[row * (P.c / P.group) + ch / P.group] = none ? 0.f : amax / most;
      uint32_t q[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float a = h[i][e] * inv, b = h[i][e + 1] * inv;
        if constexpr (CODES == 1) {
          q[e / 4] = (e & 2) ? __builtin_amdgcn_cvt_pk_fp8_f32(a, b, q[e / 4], true)
                             : __builtin_amdgcn_cvt_pk_fp8_f32(a, b, q[e / 4], false);
        } else {
          const int ia = (int)fminf(fmaxf(rintf(a), -127.f), 127.f), ib = (int)fminf(fmaxf(rintf(b), -127.f), 127.f);
          q[e / 4] |= ((uint32_t)(ia & 255) | (uint32_t)(ib & 255) << 8) << (8 * (e & 2));
        }
      }
      *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(P.codes) + at + ch) = u32x2{q[0], q[1]};
    }
  }
}

// dx a row at a time, dw summed over the rows of a workgroup in registers, the
// workgroups' sums [gridDim.x][c] added by rmsnorm_dw_kernel in one order.
template <typename T, int TEAM, int PIECES>
__global__ __launch_bounds__(256) void rmsnorm_bwd_kernel(RmsNormBwdParams<T> P) {
  constexpr int kTeams = 256 / TEAM;
  __shared__ float lds[4];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  float w[PIECES][8], dw[PIECES][8];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int ch = (i * TEAM + lane) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = dw[i][e] = 0.f;
    if (ch < P.c) to_f32x8(load8(P.w + ch), w[i]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < P.rows; r0 += (int64_t)gridDim.x * kTeams) {
    const bool row_on = r0 + team < P.rows;
    const int64_t at = (row_on ? r0 + team : P.rows - 1) * P.c;
    float h[PIECES][8], t[PIECES][8];
    float ss = 0.f, tn = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int ch = (i * TEAM + lane) * 8;
      if (ch < P.c) {
        to_f32x8(load8(P.h + at + ch), h[i]);
        to_f32x8(load8(P.dy + at + ch), t[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = t[i][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(h[i][e], h[i][e], ss);
        tn = fmaf(t[i][e] * w[i][e], h[i][e], tn);
      }
    }
    const float rstd = __builtin_amdgcn_rsqf(team_sum<TEAM>(ss, lds) / P.c + P.eps);
    const float mean = team_sum<TEAM>(tn, lds) / P.c * rstd;  // of t n
    if (!row_on) continue;  // a whole team at once, and the last round
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int ch = (i * TEAM + lane) * 8;
      if (ch >= P.c) continue;
      float o[8], add[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (P.dh) to_f32x8(load8(P.dh + at + ch), add);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n = h[i][e] * rstd;
        dw[i][e] = fmaf(t[i][e], n, dw[i][e]);
        o[e] = fmaf(rstd, t[i][e] * w[i][e] - n * mean, add[e]);
      }
      store8(P.dx + at + ch, pack8<T>(o));
    }
  }
  // the workgroup's teams, one after the other
  __shared__ float sums[PIECES * TEAM * 8];
  for (int g = 0; g < kTeams; ++g) {
    __syncthreads();
    if (team == g) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float& s = sums[(i * 8 + e) * TEAM + lane];
          s = g ? s + dw[i][e] : dw[i][e];
        }
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < P.c; x += 256) {
    const int piece = x / 8;
    P.part[(int64_t)blockIdx.x * P.c + x] = sums[(piece / TEAM * 8 + x % 8) * TEAM + piece % TEAM];
  }
}

__global__ __launch_bounds__(1024) void rmsnorm_dw_kernel(const float* __restrict__ part, float* __restrict__ dw, int blocks, int c) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ch = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (ch < c) {
#pragma unroll 8
    for (int b = wave; b < blocks; b += 16) s += part[(int64_t)b * c + ch];
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave || ch >= c) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += lds[w][lane];
  dw[ch] = s;
}

// lanes that share a row and 8-channel pieces of each: one piece up to 512
// channels, so that narrow rows leave few lanes idle, then up to 4 of a wave,
// then of a workgroup
template <typename F>
void by_width(int c, F f) {
  const int p = c / 8;
  if (p <= 8) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
  if (p <= 16) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  if (p <= 32) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  if (p <= 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  if (p <= 128) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  if (p <= 256) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  if (p <= 512) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
}

}  // namespace

int rmsnorm_bwd_blocks(int64_t rows, int c) {
  int64_t blocks = 0;
  by_width(c, [&](auto team, auto) { blocks = (rows * team.value + 255) / 256; });
  // a row a team while that leaves a workgroup a CU, then two and more
  if (blocks > 256) blocks = blocks / 2 > 256 ? blocks / 2 : 256;
  return (int)(blocks < 1024 ? blocks : 1024);
}

template <typename T>
void launch_rmsnorm(const RmsNormParams<T>& p, int codes, hipStream_t st) {
  by_width(p.c, [&](auto team, auto pieces) {
    constexpr int kTeam = team.value, kPieces = pieces.value;
    for_pieces((p.rows * kTeam + 255) / 256, [&](int64_t first, unsigned blocks) {
      RmsNormParams<T> q = p;
      q.first = first;
      if (codes == 0)
        rmsnorm_kernel<T, kTeam, kPieces, 0><<<blocks, 256, 0, st>>>(q);
      else if (codes == 1)
        rmsnorm_kernel<T, kTeam, kPieces, 1><<<blocks, 256, 0, st>>>(q);
      else
        rmsnorm_kernel<T, kTeam, kPieces, 2><<<blocks, 256, 0, st>>>(q);
    });
  });
}

template <typename T>
void launch_rmsnorm_bwd(const RmsNormBwdParams<T>& p, float* dw, hipStream_t st) {
  const int blocks = rmsnorm_bwd_blocks(p.rows, p.c);
  by_width(p.c, [&](auto team, auto pieces) {
    rmsnorm_bwd_kernel<T, decltype(team)::value, decltype(pieces)::value><<<blocks, 256, 0, st>>>(p);
  });
  rmsnorm_dw_kernel<<<(p.c + 63) / 64, 1024, 0, st>>>(p.part, dw, blocks, p.c);
}

template void launch_rmsnorm<bf16>(const RmsNormParams<bf16>&, int, hipStream_t);
template void launch_rmsnorm<float>(const RmsNormParams<float>&, int, hipStream_t);
template void launch_rmsnorm_bwd<bf16>(const RmsNormBwdParams<bf16>&, float*, hipStream_t);
template void launch_rmsnorm_bwd<float>(const RmsNormBwdParams<float>&, float*, hipStream_t);

}  // namespace fjx
