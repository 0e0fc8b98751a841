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

// The columns of a lane's chunk k from column c on: only the last chunk may
// lie past the row, or hold less than eight columns (TAIL).
template <int NC, bool TAIL>
DSA_DEV int rms_cols(int C, int c, int k) {
  return k < NC - 1 ? 8 : TAIL ? C - c : c < C ? 8 : 0;
}

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

// The lane's chunks of a row of x and the residual as they lie in memory.
template <int NC, int W, typename TX, typename TR, bool TAIL>
struct RawZ {
  raw8<TX> x[NC];
  raw8<TR> res[NC];
  DSA_DEV void load(const RmsRows& p, uint32_t r, int first) {
    const int64_t xo = (int64_t)r * p.xs;
    const int64_t ro = p.res ? res_row(r, p.rpg, p.N, p.rs0, p.rs1) : 0;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k);
      x[k] = ld8<TX, TAIL>(p.x, xo + c, p.xe, rms_cols<NC, TAIL>(p.C, c, k));
      if (p.res) res[k] = ld8<TR, TAIL>(p.res, ro + c, p.re, rms_cols<NC, TAIL>(p.C, c, k));
    }
  }
};

// The random words of the lane's chunks of row r.
template <int NC, int W>
DSA_DEV void rms_words(const RmsRows& p, uint32_t r, int first, uint4 (&words)[NC]) {
  if (!p.d.on) return;
#pragma unroll
  for (int k = 0; k < NC; ++k) words[k] = hidden_words(p.d, r, first + 64 * W * k);
}

// chunk k of z = dropout(x + bias) + res
template <int NC, int W, typename TX, typename TR, bool TAIL>
DSA_DEV void rms_z(const RmsRows& p, const RawZ<NC, W, TX, TR, TAIL>& raw, int k, int n, const float (&bias)[8], uint4 words,
                   float (&z)[8]) {
  cvt8<TX, TAIL>(raw.x[k], n, z);
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += bias[e];
  }
  if (p.d.on) drop8(p.d, words, z);
  if (p.res) {
    float v[8];
    cvt8<TR, TAIL>(raw.res[k], n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += v[e];
  }
}

// The largest of the bit patterns of |v|: the largest magnitude, where an
// infinity is above every finite value and a NaN above both.
DSA_DEV uint32_t mag(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

template <int NC, int W, typename TX, typename TR, typename TZ, typename TY, bool TAIL>
__global__ __launch_bounds__(rms_threads<W>()) void rms_fwd_kernel(RmsRows p) {
  __shared__ float buf[2 * W];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv % W, first = wr * 64 + lane;
  const uint32_t r = blockIdx.x * rms_teams<W>() + wv / W;
  if (r >= p.N) return;  // the whole team; a block has barriers only where it is one team
  RawZ<NC, W, TX, TR, TAIL> raw;
  raw.load(p, r, first);
  uint4 words[NC];
  rms_words<NC, W>(p, r, first, words);  // while the loads are in flight
  float z[NC][8];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = 8 * (first + 64 * W * k), n = rms_cols<NC, TAIL>(p.C, c, k);
    float bias[8];
    ld_param8<TAIL>(p.bias, p.bias_dt, c, n, bias);
    rms_z<NC, W, TX, TR, TAIL>(p, raw, k, n, bias, words[k], z[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += z[k][e] * z[k][e];
  }
  int turn = 0;
  const float rstd = 1.f / sqrtf(team_sum<W>(s, buf, wr, turn) / (float)p.C + p.eps);
  if (p.rstd && wr == 0 && lane == 0) p.rstd[r] = rstd;
  if (p.z) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k);
      st8<TZ, TAIL>(p.z, (int64_t)r * p.zs + c, rms_cols<NC, TAIL>(p.C, c, k), z[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = 8 * (first + 64 * W * k), n = rms_cols<NC, TAIL>(p.C, c, k);
    float w[8];
    ld_param8<TAIL>(p.w, p.w_dt, c, n, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[k][e] = z[k][e] * rstd * w[e];
    if constexpr (!std::is_same<TY, fp8>::value) st8<TY, TAIL>(p.y, (int64_t)r * p.ys + c, n, z[k]);
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
      const int c = 8 * (first + 64 * W * k), n = rms_cols<NC, TAIL>(p.C, c, k);
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

// What the backward reads of a row.
template <int NC, int W, typename TX, typename TR, typename TZ, typename TDY, bool TAIL>
struct RawBwd {
  RawZ<NC, W, TX, TR, TAIL> z;
  raw8<TDY> dy[NC];
  raw8<TZ> u[NC];
  float rstd;
  DSA_DEV void load(const RmsRows& p, uint32_t r, int first) {
    z.load(p, r, first);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k);
      dy[k] = ld8<TDY, TAIL>(p.dy, (int64_t)r * p.dys + c, p.dye, rms_cols<NC, TAIL>(p.C, c, k));
      if (p.dzu) u[k] = ld8<TZ, TAIL>(p.dzu, (int64_t)r * p.dzus + c, p.dzue, rms_cols<NC, TAIL>(p.C, c, k));
    }
    rstd = p.rstd[r];
  }
};

// Rows [rows * team, + rows), team counted over the grid.  dw's and dbias's
// partial sums of the block go to part[block][1 or 2][C].
//
// A block stays for many rows (the launch holds as many blocks as run at
// once), so that the partial sums are few.  A row's own latency is then
// what bounds it: the next row is loaded while the row is worked on, where
// its registers allow (PRE), and w and the bias stay in registers (KEEP).
template <int NC, int W, typename TX, typename TR, typename TZ, typename TDY, bool TAIL>
__global__ __launch_bounds__(rms_threads<W>()) void rms_bwd_kernel(RmsRows p) {
  typedef RawBwd<NC, W, TX, TR, TZ, TDY, TAIL> Raw;
  constexpr bool KEEP = W < 16;  // sixteen waves have 128 registers each
  constexpr bool PRE = KEEP && sizeof(Raw) <= 4 * 44;
  __shared__ float buf[2 * W];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv % W, first = wr * 64 + lane;
  const int64_t r0 = ((int64_t)blockIdx.x * rms_teams<W>() + wv / W) * p.rows;
  const int64_t left = (int64_t)p.N - r0;
  const int rows = (int)(left < p.rows ? left : p.rows);  // of this team; none: at most 0
  float sw[NC][8], sb[NC][8], w[NC][8], bias[NC][8];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = 8 * (first + 64 * W * k);
    if (KEEP) ld_param8<TAIL>(p.w, p.w_dt, c, rms_cols<NC, TAIL>(p.C, c, k), w[k]);
    if (KEEP) ld_param8<TAIL>(p.bias, p.bias_dt, c, rms_cols<NC, TAIL>(p.C, c, k), bias[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[k][e] = sb[k][e] = 0.f;
  }
  int turn = 0;
  Raw next;
  if (PRE && rows > 0) next.load(p, (uint32_t)r0, first);
#pragma unroll 1
  for (int i = 0; i < rows; ++i) {
    const uint32_t r = (uint32_t)(r0 + i);
    Raw raw;
    if (PRE) {
      raw = next;
      if (i + 1 < rows) next.load(p, r + 1, first);
    } else {
      raw.load(p, r, first);
    }
    uint4 words[NC];
    rms_words<NC, W>(p, r, first, words);
    float z[NC][8], g[NC][8];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k), n = rms_cols<NC, TAIL>(p.C, c, k);
      if (!KEEP) ld_param8<TAIL>(p.w, p.w_dt, c, n, w[k]);
      if (!KEEP) ld_param8<TAIL>(p.bias, p.bias_dt, c, n, bias[k]);
      rms_z<NC, W, TX, TR, TAIL>(p, raw.z, k, n, bias[k], words[k], z[k]);
      cvt8<TDY, TAIL>(raw.dy[k], n, g[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[k][e] *= raw.rstd;  // the normed value
        sw[k][e] += g[k][e] * z[k][e];
        g[k][e] *= w[k][e];
        s += g[k][e] * z[k][e];
      }
    }
    const float m = team_sum<W>(s, buf, wr, turn) / (float)p.C;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = 8 * (first + 64 * W * k), n = rms_cols<NC, TAIL>(p.C, c, k);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[k][e] = raw.rstd * (g[k][e] - z[k][e] * m);
      if (p.dzu) {
        float u[8];
        cvt8<TZ, TAIL>(raw.u[k], n, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[k][e] += u[e];
      }
      if (p.dres) st8<TR, TAIL>(p.dres, (int64_t)r * p.drs + c, n, g[k]);
      if (p.d.on) drop8(p.d, words[k], g[k]);
      if (p.dx) st8<TX, TAIL>(p.dx, (int64_t)r * p.dxs + c, n, g[k]);
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
      const int c = 8 * (first + 64 * W * k), n = rms_cols<NC, TAIL>(p.C, c, k);
      st8<float, TAIL>(out, c, n, sw[k]);
      if (sums == 2) st8<float, TAIL>(out, p.C + c, n, sb[k]);
    }
  } else {
    // the four waves' sums, added in wave order
    __shared__ float red[2 * 512 * NC];
    for (int v = 0; v < 4; ++v) {
      if (wv == v) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const int c = 8 * (first + 64 * k);
          if (c < p.C) {  // columns past the row lie inside red, and are not read
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              red[c + e] = v == 0 ? sw[k][e] : red[c + e] + sw[k][e];
              red[512 * NC + c + e] = v == 0 ? sb[k][e] : red[512 * NC + c + e] + sb[k][e];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.C; i += 256) {
      out[i] = red[i];
      if (sums == 2) out[p.C + i] = red[512 * NC + i];
    }
  }
}

}  // namespace hid
}  // namespace dsa
