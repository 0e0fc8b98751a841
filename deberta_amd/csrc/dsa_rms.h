// dsa_rms.h — RMS norm with the residual's addition (gfx950):
//   z = dropout(x + bias) + res,  r = 1 / sqrt(mean(z^2) + eps),  y = z r w
// and its backward, for g = dy w and the gradient u that arrives at z itself:
//   dz = r (g - z r^2 mean(g z)) + u;  dres = dz;  dx = keep ? dz / (1 - p) : 0
//   dbias = column sums of dx,  dw = column sums of dy z r
// and the forward with y in 8 bits (e4m3) and a scale a row or a group of
// columns.
//
// A row is held in registers by a team of W waves, NC chunks of eight columns
// a lane: x and res are read once, y and z written once.  The squares are
// summed in fp32 from the unrounded z, and y comes from the unrounded z.  The
// backward forms z again from x, bias, res and the keep bits rather than
// reading the z that was returned: where the stream is bf16 that z is
// rounded, and dw, held in fp32, would carry its 2^-9.
#pragma once

#include <type_traits>

#include "dsa_hidden.h"

namespace dsa {
namespace hid {

struct fp8 {};  // y as e4m3 bytes with scales

struct RmsRows {
  const void *x, *bias, *res, *w, *dy, *dzu;
  void *y, *z, *dx, *dres;
  float *rstd, *yscale, *part;
  int64_t xs, xe, rs0, rs1, re, ys, zs, dys, dye, dzus, dzue, dxs, drs;
  uint32_t N, rpg;
  int C, bias_dt, w_dt, group;
  int rows;  // backward: rows a team takes
  float eps;
  Drop d;
};

// rows a block takes at a time: one team of four waves or more, four teams of one
template <int W>
constexpr int rms_teams() { return W == 1 ? 4 : 1; }
template <int W>
constexpr int rms_threads() { return 64 * W * rms_teams<W>(); }

// The team's sum of x, in every lane, in a fixed order.  buf: two sets of W
// floats, used in turn, so that one barrier a sum is enough.
template <int W>
DSA_DEV float team_sum(float x, float* buf, int wr, int& turn) {
  x = wave_sum(x);
  if constexpr (W > 1) {
    float* b = buf + (turn & 1) * W;
    ++turn;
    b[wr] = x;  // every lane the same value
    __syncthreads();
    x = b[0];
#pragma unroll
    for (int i = 1; i < W; ++i) x += b[i];
  }
  return x;
}

// z of the lane's chunks of row r, and their keep bits
template <int NC, int W, typename TX, typename TR>
DSA_DEV void rms_load_z(const RmsRows& p, uint32_t r, int first, float (&z)[NC][8], uint32_t (&keep)[NC]) {
  raw8<TX> x[NC];
  raw8<TR> res[NC];
  const int64_t xo = (int64_t)r * p.xs;
  const int64_t ro = p.res ? res_row(r, p.rpg, p.N, p.rs0, p.rs1) : 0;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = 8 * (first + 64 * W * k);
    x[k] = ld8<TX>(p.x, xo + c, p.xe, p.C - c);
    if (p.res) res[k] = ld8<TR>(p.res, ro + c, p.re, p.C - c);
  }
  if (p.d.t) {
#pragma unroll
    for (int k = 0; k < NC; ++k) keep[k] = hidden_keep8(p.d, r, first + 64 * W * k);
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = 8 * (first + 64 * W * k), n = p.C - c;
    cvt8<TX>(x[k], n, z[k]);
    if (p.bias) {
      float b[8];
      ld_param8(p.bias, p.bias_dt, c, n, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[k][e] += b[e];
    }
    if (p.d.t) apply_keep(keep[k], p.d.scale, z[k]);
    if (p.res) {
      float v[8];
      cvt8<TR>(res[k], n, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[k][e] += v[e];
    }
  }
}

// The largest of the bit patterns of |v|: the largest magnitude, where an
// infinity is above every finite value and a NaN above both.
DSA_DEV uint32_t mag(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

template <int NC, int W, typename TX, typename TR, typename TZ, typename TY>
__global__ __launch_bounds__(rms_threads<W>()) void rms_fwd_kernel(RmsRows p) {
  __shared__ float buf[2 * W];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv % W, first = wr * 64 + lane;
  const uint32_t r = blockIdx.x * rms_teams<W>() + wv / W;
  if (r >= p.N) return;  // the whole team; a block has barriers only where it is one team
  float z[NC][8];
  uint32_t keep[NC];
  rms_load_z<NC, W, TX, TR>(p, r, first, z, keep);
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += z[k][e] * z[k][e];
  int turn = 0;
  const float rstd = 1.f / sqrtf(team_sum<W>(s, buf, wr, turn) / (float)p.C + p.eps);
  if (p.rstd && wr == 0 && lane == 0) p.rstd[r] = rstd;
  if (p.z) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k);
      st8<TZ>(p.z, (int64_t)r * p.zs + c, p.C - c, z[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = 8 * (first + 64 * W * k), n = p.C - c;
    float w[8];
    ld_param8(p.w, p.w_dt, c, n, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[k][e] = z[k][e] * rstd * w[e];
    if constexpr (!std::is_same<TY, fp8>::value) st8<TY>(p.y, (int64_t)r * p.ys + c, n, z[k]);
  }
  if constexpr (std::is_same<TY, fp8>::value) {
    __shared__ uint32_t mbuf[W];
    uint32_t m[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      m[k] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m[k] = max(m[k], mag(z[k][e]));
    }
    int ng = 1;
    if (p.group) {  // a power of two of columns: group / 8 neighbouring lanes
      ng = p.C / p.group;
      for (int o = 1; o < p.group / 8; o <<= 1) {
#pragma unroll
        for (int k = 0; k < NC; ++k) m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], o));
      }
    } else {
      uint32_t a = 0;
#pragma unroll
      for (int k = 0; k < NC; ++k) a = max(a, m[k]);
      for (int o = 1; o < 64; o <<= 1) a = max(a, (uint32_t)__shfl_xor((int)a, o));
      if constexpr (W > 1) {
        mbuf[wr] = a;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) a = max(a, mbuf[i]);
      }
#pragma unroll
      for (int k = 0; k < NC; ++k) m[k] = a;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k), n = p.C - c;
      if (n <= 0) continue;
      const float a = __builtin_bit_cast(float, m[k]);
      // every value below the smallest normal scale's range: zeros
      const bool tiny = a < 448.f * 0x1p-126f;
      const float scale = a < __builtin_inff() ? (tiny ? 1.f : a / 448.f) : __builtin_nanf("");
      const float inv = tiny ? 1.f : 448.f / a;
      uint32_t q[2];
      if (a < __builtin_inff()) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[k][e] = fminf(fmaxf(z[k][e] * inv, -448.f), 448.f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int v = 0;
          v = __builtin_amdgcn_cvt_pk_fp8_f32(z[k][4 * h], z[k][4 * h + 1], v, false);
          v = __builtin_amdgcn_cvt_pk_fp8_f32(z[k][4 * h + 2], z[k][4 * h + 3], v, true);
          q[h] = (uint32_t)v;
        }
      } else {
        q[0] = q[1] = 0x7f7f7f7fu;  // NaN
      }
      uint8_t* out = static_cast<uint8_t*>(p.y) + (int64_t)r * p.ys + c;
      if (n >= 8) {
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        typedef u2 u2u __attribute__((aligned(1)));
        *reinterpret_cast<u2u*>(out) = u2{q[0], q[1]};
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < n) out[e] = (uint8_t)(q[e / 4] >> (8 * (e % 4)));
      }
      if (p.group ? c % p.group == 0 : c == 0) p.yscale[(int64_t)r * ng + (p.group ? c / p.group : 0)] = scale;
    }
  }
}

// Rows [rows * team, + rows), team counted over the grid.  dw's and dbias's
// partial sums of the block go to part[block][1 or 2][C].
template <int NC, int W, typename TX, typename TR, typename TZ, typename TDY>
__global__ __launch_bounds__(rms_threads<W>()) void rms_bwd_kernel(RmsRows p) {
  __shared__ float buf[2 * W];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv % W, first = wr * 64 + lane;
  const int64_t r0 = ((int64_t)blockIdx.x * rms_teams<W>() + wv / W) * p.rows;
  float sw[NC][8], sb[NC][8];
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[k][e] = sb[k][e] = 0.f;
  int turn = 0;
#pragma unroll 1
  for (int i = 0; i < p.rows; ++i) {
    const int64_t r64 = r0 + i;
    if (r64 >= p.N) break;  // the whole team
    const uint32_t r = (uint32_t)r64;
    raw8<TDY> dyr[NC];
    raw8<TZ> ur[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k);
      dyr[k] = ld8<TDY>(p.dy, r64 * p.dys + c, p.dye, p.C - c);
      if (p.dzu) ur[k] = ld8<TZ>(p.dzu, r64 * p.dzus + c, p.dzue, p.C - c);
    }
    float z[NC][8], g[NC][8];
    uint32_t keep[NC];
    rms_load_z<NC, W, TX, TR>(p, r, first, z, keep);
    const float rstd = p.rstd[r];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k), n = p.C - c;
      float w[8];
      cvt8<TDY>(dyr[k], n, g[k]);
      ld_param8(p.w, p.w_dt, c, n, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[k][e] *= rstd;  // the normed value
        sw[k][e] += g[k][e] * z[k][e];
        g[k][e] *= w[e];
        s += g[k][e] * z[k][e];
      }
    }
    const float m = team_sum<W>(s, buf, wr, turn) / (float)p.C;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k), n = p.C - c;
      float u[8];
      if (p.dzu) {
        cvt8<TZ>(ur[k], n, u);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) g[k][e] = rstd * (g[k][e] - z[k][e] * m) + u[e];
      if (p.dres) st8<TR>(p.dres, r64 * p.drs + c, n, g[k]);
      if (p.d.t) apply_keep(keep[k], p.d.scale, g[k]);
      if (p.dx) st8<TX>(p.dx, r64 * p.dxs + c, n, g[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sb[k][e] += g[k][e];
    }
  }
  if (!p.part) return;
  const int sums = p.bias ? 2 : 1;
  float* out = p.part + (int64_t)blockIdx.x * sums * p.C;
  if constexpr (W > 1) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < p.C) {
          out[c + e] = sw[k][e];
          if (sums == 2) out[p.C + c + e] = sb[k][e];
        }
    }
  } else {
    // the four waves' sums, added in wave order
    __shared__ float red[2 * 512 * NC];
    for (int v = 0; v < 4; ++v) {
      if (wv == v) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const int c = 8 * (first + 64 * k);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < p.C) {
              red[c + e] = v == 0 ? sw[k][e] : red[c + e] + sw[k][e];
              if (sums == 2) red[p.C + c + e] = v == 0 ? sb[k][e] : red[p.C + c + e] + sb[k][e];
            }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < sums * p.C; i += 256) out[i] = red[i];
  }
}

}  // namespace hid
}  // namespace dsa
