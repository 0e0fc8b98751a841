// dsa_rms.h — RMS norm with the residual's addition (gfx950):
//   z = dropout(x + bias) + res,  r = 1 / sqrt(mean(z^2) + eps),  y = z r w
// and its backward, for g = dy w and the gradient u that arrives at z itself:
//   dz = r (g - z r^2 mean(g z)) + u;  dres = dz;  dx = keep ? dz / (1 - p) : 0
//   dbias = column sums of dx,  dw = column sums of dy z r
// and the forward with y in 8 bits (e4m3) and a scale a row or a group of
// columns.
//
// A row is held in registers by a team: W waves of NC chunks of eight columns
// a lane, or L lanes of a wave where rows are narrow (64 / L rows a wave).  x
// and res are read once, y and z written once.  The squares are summed in
// fp32 from the unrounded z, and y comes from the unrounded z.  The backward
// forms z again from x, bias, res and the keep bits rather than reading the z
// that was returned: where the stream is bf16 that z is rounded, and dw, held
// in fp32, would carry its 2^-9.
//
// Every load of a row is made by every lane, so that the compiler can keep
// the next row's in flight while it waits for this one's (behind a condition
// it waits for both): lanes past the row load its last chunk, a residual or
// gradient that is not there is read from a tensor that is, always the same
// row, and not used.  Not so where a row ends in a cut chunk (TAIL): its loads
// are behind the condition that the tensor goes on behind the row (row8).
//
// HBM bounds all but the smallest: 16384 x 768 bf16 with bias, dropout and
// residual 21.8 us forward (101 MB, 4.6 TB/s) and 30.0 backward (151 MB, 5.0),
// 16384 x 4096 bf16 on a float32 stream 164 (940 MB, 5.7) and 270 (1342 MB,
// 5.0); 9971 x 1024 in 8 bits 14.0 (71 MB, 5.1).  Of the rate at the next
// multiple of eight, odd bf16 widths (33.5 million values, 513 to 8191 columns)
// reach 77 to 96% forward and 57 to 84% backward; dropout, whose accesses are as
// unaligned and unconditional but for the last chunk, 82 to 92%.
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
  uint32_t r0;         // forward: the launch's first row
  int C, bias_dt, w_dt, group;
  int has_res, has_u;  // whether res and dzu are there
  int rows;            // backward: rows a team takes
  float eps;
  Drop d;
};

// teams a block: one of four waves or more, or four waves of 64 / L
template <int L, int W>
constexpr int rms_teams() { return W == 1 ? 4 * (64 / L) : 1; }
template <int W>
constexpr int rms_threads() { return W == 1 ? 256 : 64 * W; }

// A lane's place: its chunks are first, first + 64 W, ...; all but the last
// lie in the row whole.
template <int L, int NC, int W, bool TAIL>
struct Place {
  int lane, wv, wr, first;
  // of the last chunk: its columns, and which of them exist as bits to AND
  // (without TAIL all or none)
  int n;
  uint32_t mask[TAIL ? 8 : 1];
  DSA_DEV explicit Place(int C) {
    lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wr = wv % W;
    first = L < 64 ? lane % L : wr * 64 + lane;
    n = C - col(NC - 1);
#pragma unroll
    for (int e = 0; e < (TAIL ? 8 : 1); ++e) mask[e] = e < n ? 0xffffffffu : 0u;
  }
  DSA_DEV int col(int k) const { return 8 * (first + 64 * W * k); }
  // the column to load chunk k from
  DSA_DEV int load_col(int C, int k) const { return k < NC - 1 ? col(k) : min(col(k), (C - 1) / 8 * 8); }
  DSA_DEV int cols(int k) const { return k < NC - 1 ? 8 : TAIL ? n : n > 0 ? 8 : 0; }
  // zeroes what is past the row
  DSA_DEV void clip(int k, float (&v)[8]) const {
    if (k < NC - 1) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v[e]) & mask[TAIL ? e : 0]);
  }
};

// Eight columns from column c of the row at element `row` of a tensor that
// ends at element `extent`.  A TAIL row's last chunk reads on past the row,
// but for the tensor's last: what it gets there is clipped.
template <typename T, bool TAIL>
DSA_DEV raw8<T> row8(const void* base, int64_t row, int64_t extent, int c, int C) {
  if (!TAIL || row + (C + 7) / 8 * 8 <= extent) {
    const char* p = static_cast<const char*>(base) + row * (int64_t)sizeof(T);
    return *reinterpret_cast<const typename Raw8<T>::v8u*>(p + (uint32_t)c * (uint32_t)sizeof(T));
  }
  raw8<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = static_cast<const T*>(base)[row + min(c + e, C - 1)];
  return r;
}

// The team's sum of x, in every lane, in a fixed order.  buf: two sets of W
// floats, used in turn, so that one barrier a sum is enough.
template <int L, int W>
DSA_DEV float team_sum(float x, float* buf, int wr, int& turn) {
  x = lanes_sum<L>(x);
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
template <int NC, typename TX, typename TR, bool TAIL>
struct RawZ {
  raw8<TX> x[NC];
  raw8<TR> res[NC];
  template <typename P>
  DSA_DEV void load(const RmsRows& p, uint32_t r, const P& at) {
    const int64_t xo = (int64_t)r * p.xs, ro = res_row(r, p.rpg, p.N, p.rs0, p.rs1);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = at.load_col(p.C, k);
      x[k] = row8<TX, TAIL>(p.x, xo, p.xe, c, p.C);
      res[k] = row8<TR, TAIL>(p.res, ro, p.re, c, p.C);
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
template <int NC, typename TX, typename TR, bool TAIL, typename P>
DSA_DEV void rms_z(const RmsRows& p, const RawZ<NC, TX, TR, TAIL>& raw, const P& at, int k, const float (&bias)[8], uint4 words,
                   float (&z)[8]) {
  cvt8<TX, false>(raw.x[k], 8, z);
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += bias[e];
  }
  if (p.d.on) drop8(p.d, words, z);
  if (p.has_res) {
    float v[8];
    cvt8<TR, false>(raw.res[k], 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += v[e];
  }
  at.clip(k, z);
}

// The largest of the bit patterns of |v|: the largest magnitude, where an
// infinity is above every finite value and a NaN above both.
DSA_DEV uint32_t mag(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

template <int L, int NC, int W, typename TX, typename TR, typename TZ, typename TY, bool TAIL>
__global__ __launch_bounds__(rms_threads<W>()) void rms_fwd_kernel(RmsRows p) {
  __shared__ float buf[2 * W];
  const Place<L, NC, W, TAIL> at(p.C);
  const int lane = at.lane, wr = at.wr;
  const uint32_t r = p.r0 + blockIdx.x * (uint32_t)rms_teams<L, W>() + at.wv / W * (64 / L) + (L < 64 ? lane / L : 0);
  if (r >= p.N) return;  // the whole team; a block has barriers only where it is one team
  RawZ<NC, TX, TR, TAIL> raw;
  raw.load(p, r, at);
  uint4 words[NC];
  rms_words<NC, W>(p, r, at.first, words);  // while the loads are in flight
  float z[NC][8];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    float bias[8];
    ld_param8<TAIL>(p.bias, p.bias_dt, at.col(k), at.cols(k), bias);
    rms_z<NC, TX, TR, TAIL>(p, raw, at, k, bias, words[k], z[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += z[k][e] * z[k][e];
  }
  int turn = 0;
  const float rstd = 1.f / sqrtf(team_sum<L, W>(s, buf, wr, turn) / (float)p.C + p.eps);
  if (p.rstd && at.first == 0) p.rstd[r] = rstd;
  if (p.z) {
#pragma unroll
    for (int k = 0; k < NC; ++k) st8<TZ, TAIL>(p.z, (int64_t)r * p.zs + at.col(k), at.cols(k), z[k]);
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    float w[8];
    ld_param8<TAIL>(p.w, p.w_dt, at.col(k), at.cols(k), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[k][e] = z[k][e] * rstd * w[e];
    if constexpr (!std::is_same<TY, fp8>::value) st8<TY, TAIL>(p.y, (int64_t)r * p.ys + at.col(k), at.cols(k), z[k]);
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
    if (p.group) {  // a power of two of columns: group / 8 neighbouring lanes, of the team's
      ng = p.C / p.group;
      for (int o = 1; o < p.group / 8; o <<= 1) {
#pragma unroll
        for (int k = 0; k < NC; ++k) m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], o));
      }
    } else {
      uint32_t a = 0;
#pragma unroll
      for (int k = 0; k < NC; ++k) a = max(a, m[k]);
      for (int o = 1; o < L; o <<= 1) a = max(a, (uint32_t)__shfl_xor((int)a, o));
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
      const int c = at.col(k), n = at.cols(k);
      if (n <= 0) continue;
      const float a = __builtin_bit_cast(float, m[k]);
      // one division a group rather than one a value: of 10.2 million bytes 5
      // are then one step from the float64 definition's (4 by a division each),
      // all within two half steps of fp32 of the border between the bytes.
      // Every value below the smallest normal scale's range: zeros
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
template <int NC, typename TX, typename TR, typename TZ, typename TDY, bool TAIL>
struct RawBwd {
  RawZ<NC, TX, TR, TAIL> z;
  raw8<TDY> dy[NC];
  raw8<TZ> u[NC];
  float rstd;
  template <typename P>
  DSA_DEV void load(const RmsRows& p, uint32_t r, const P& at) {
    z.load(p, r, at);
    rstd = p.rstd[r];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = at.load_col(p.C, k);
      dy[k] = row8<TDY, TAIL>(p.dy, (int64_t)r * p.dys, p.dye, c, p.C);
      u[k] = row8<TZ, TAIL>(p.dzu, (int64_t)r * p.dzus, p.dzue, c, p.C);
    }
  }
};

// Rows [rows * team, + rows), but of a wave with several teams: these take
// neighbouring rows.  dw's and dbias's partial sums of the block go to
// part[block][1 or 2][C].
//
// A block stays for many rows (the launch holds as many blocks as run at
// once), so that the partial sums are few.  A row's own latency is then
// what bounds it: the next row is loaded while the row is worked on, where
// its registers allow (PRE), and w and the bias stay in registers (KEEP).
// Sixteen waves have 128 registers each.  With two chunks a lane (past 8192
// columns) their column sums lie in LDS, w and the bias are read again for every
// row and no row is loaded ahead; with one chunk all of it is in registers.
// Neither form fits whole: the compiler spills up to 14 registers a lane where
// rows are whole and 5 to 57 where they are cut.
template <int L, int NC, int W, typename TX, typename TR, typename TZ, typename TDY, bool TAIL>
__global__ __launch_bounds__(rms_threads<W>()) void rms_bwd_kernel(RmsRows p) {
  typedef RawBwd<NC, TX, TR, TZ, TDY, TAIL> Raw;
  typedef float f4 __attribute__((ext_vector_type(4)));
  constexpr int G = 64 / L;  // rows a wave takes at a time
  constexpr bool LDS = NC * W >= 32, KEEP = !LDS, PRE = KEEP && sizeof(Raw) <= 4 * 44;
  __shared__ float buf[2 * W];
  __shared__ f4 cs[LDS ? 4 * NC * 64 * W : 1];  // [dw or dbias][chunk][half][thread]
  const Place<L, NC, W, TAIL> at(p.C);
  const int lane = at.lane, wv = at.wv, wr = at.wr;
  const int64_t r0 = ((int64_t)blockIdx.x * (W == 1 ? 4 : 1) + wv / W) * p.rows * G;  // the wave's first row
  const int64_t left = ((int64_t)p.N - r0 + G - 1) / G;
  const int rows = (int)(left < p.rows ? left : p.rows);  // of this team; none: at most 0
  float sw[NC][8], sb[NC][8], w[NC][8], bias[NC][8];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    if (KEEP) ld_param8<TAIL>(p.w, p.w_dt, at.col(k), at.cols(k), w[k]);
    if (KEEP) ld_param8<TAIL>(p.bias, p.bias_dt, at.col(k), at.cols(k), bias[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[k][e] = sb[k][e] = 0.f;
    if constexpr (LDS) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        cs[(2 * k + h) * 64 * W + threadIdx.x] = cs[(2 * (NC + k) + h) * 64 * W + threadIdx.x] = f4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // adds v to the lane's sums j (0: dw, 1: dbias) of chunk k
  auto add = [&](int j, int k, const float(&v)[8], float(&sum)[8]) {
    if constexpr (LDS) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f4& c = cs[(2 * (j * NC + k) + h) * 64 * W + threadIdx.x];
        c += f4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
  };
  auto row = [&](int i) {
    const int64_t r = r0 + (int64_t)i * G + (L < 64 ? lane / L : 0);
    return (uint32_t)(r < p.N ? r : p.N - 1);  // teams past the last row repeat it
  };
  int turn = 0;
  Raw next;
  if (PRE && rows > 0) next.load(p, row(0), at);
#pragma unroll 1
  for (int i = 0; i < rows; ++i) {
    const uint32_t r = row(i);
    const bool there = L == 64 || r0 + (int64_t)i * G + lane / L < p.N;
    Raw raw;
    if (PRE) {
      raw = next;
      next.load(p, row(min(i + 1, rows - 1)), at);
    } else {
      raw.load(p, r, at);
    }
    uint4 words[NC];
    rms_words<NC, W>(p, r, at.first, words);
    float z[NC][8], g[NC][8];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (!KEEP) ld_param8<TAIL>(p.w, p.w_dt, at.col(k), at.cols(k), w[k]);
      if (!KEEP) ld_param8<TAIL>(p.bias, p.bias_dt, at.col(k), at.cols(k), bias[k]);
      rms_z<NC, TX, TR, TAIL>(p, raw.z, at, k, bias[k], words[k], z[k]);
      cvt8<TDY, false>(raw.dy[k], 8, g[k]);
      at.clip(k, g[k]);
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[k][e] *= raw.rstd;  // the normed value
        t[e] = g[k][e] * z[k][e];
        if (L < 64 && !there) t[e] = 0.f;
        g[k][e] *= w[k][e];
        s += g[k][e] * z[k][e];
      }
      add(0, k, t, sw[k]);
    }
    const float m = team_sum<L, W>(s, buf, wr, turn) / (float)p.C;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = at.col(k), n = there ? at.cols(k) : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[k][e] = raw.rstd * (g[k][e] - z[k][e] * m);
      if (p.has_u) {
        float u[8];
        cvt8<TZ, false>(raw.u[k], 8, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[k][e] += u[e];
      }
      if (p.dres) st8<TR, TAIL>(p.dres, (int64_t)r * p.drs + c, n, g[k]);
      if (p.d.on) drop8(p.d, words[k], g[k]);
      if (p.dx) st8<TX, TAIL>(p.dx, (int64_t)r * p.dxs + c, n, g[k]);
      if (L < 64 && !there) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[k][e] = 0.f;
      }
      add(1, k, g[k], sb[k]);
    }
  }
  if (!p.part) return;
  const int sums = p.bias ? 2 : 1;
  float* out = p.part + (int64_t)blockIdx.x * sums * p.C;
  if constexpr (W > 1) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if constexpr (LDS) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sw[k][e] = cs[(2 * k + e / 4) * 64 * W + threadIdx.x][e % 4];
          sb[k][e] = cs[(2 * (NC + k) + e / 4) * 64 * W + threadIdx.x][e % 4];
        }
      }
      st8<float, TAIL>(out, at.col(k), at.cols(k), sw[k]);
      if (sums == 2) st8<float, TAIL>(out, p.C + at.col(k), at.cols(k), sb[k]);
    }
  } else {
    // a wave's teams, then the four waves' sums in wave order
    __shared__ float red[2 * 8 * L * NC];
#pragma unroll
    for (int o = L; o < 64; o <<= 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sw[0][e] += __shfl_xor(sw[0][e], o);
        sb[0][e] += __shfl_xor(sb[0][e], o);
      }
    }
    for (int v = 0; v < 4; ++v) {
      if (wv == v && lane < L) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const int c = at.col(k);
          if (c < p.C) {  // columns past the row lie inside red, and are not read
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              red[c + e] = v == 0 ? sw[k][e] : red[c + e] + sw[k][e];
              red[8 * L * NC + c + e] = v == 0 ? sb[k][e] : red[8 * L * NC + c + e] + sb[k][e];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.C; i += 256) {
      out[i] = red[i];
      if (sums == 2) out[p.C + i] = red[8 * L * NC + i];
    }
  }
}

}  // namespace hid
}  // namespace dsa
