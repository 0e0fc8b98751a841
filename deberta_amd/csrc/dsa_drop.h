// dsa_drop.h — hidden dropout with the bias before it and the residual after
// it (gfx950):
//   y = keep ? (x + bias) / (1 - p) : 0, + res
//   dx = keep ? dy / (1 - p) : 0,  dbias = column sums of dx
// The keep bits come from the position and the seed (dsa_hidden.h).
//
// A thread owns one chunk of eight columns (its bias stays in registers) and
// takes rows 'subs' apart; the chunks of a row lie in consecutive threads, so
// that a wave reads whole lines.  Four rows' loads are issued before the
// first is used: the Philox rounds run while they are in flight.
//
// HBM bounds both: of 16384 x 768 bf16 values with bias and residual the
// forward takes 14.3 us (75 MB, 5.3 TB/s) and the backward 13.4 (50 MB) and 3.9
// for the partial sums of dbias; 33.5 million values of any even width run at
// 6.1 to 6.3 TB/s without dbias, where a large copy reaches 4.9.
#pragma once

#include "dsa_hidden.h"

namespace dsa {
namespace hid {

constexpr int DROP_T = 256;  // chunks (threads) a block takes at most
constexpr int DROP_SUM_T = 512;  // the same of a backward with dbias: larger blocks leave fewer partial sums
constexpr int DROP_U = 4;    // rows whose loads are issued together

struct DropRows {
  const void *x, *bias, *res, *dy;
  void *y, *dx;
  float* part;  // backward: [blocks][C] column sums, or null
  void* dbias;  // backward of one block: the column sums themselves, or null
  int64_t xs, xe, rs0, rs1, re, ys, dys, dye, dxs;  // row strides and extents, elements
  uint32_t N, rpg;  // rows; rows of a residual group
  int C, bias_dt;
  int cw, subs;     // chunks of a row in a block; rows a block takes at a time
  int rows;         // rows a thread takes
  Drop d;
};

template <typename TX, typename TR, typename TY, bool TAIL>
__global__ __launch_bounds__(DROP_T) void drop_fwd_kernel(DropRows p) {
  const int sub = threadIdx.x / p.cw, chunk = blockIdx.y * p.cw + (int)threadIdx.x - sub * p.cw;
  const int c = 8 * chunk, n = p.C - c;
  if (sub >= p.subs || n <= 0) return;  // all others: eight columns, or the row's last
  float bias[8];
  ld_param8<TAIL>(p.bias, p.bias_dt, c, n, bias);
  const int64_t r0 = (int64_t)blockIdx.x * p.rows * p.subs + sub;
  for (int i = 0; i < p.rows; i += DROP_U) {
    raw8<TX> x[DROP_U];
    raw8<TR> res[DROP_U];
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
      const uint32_t r = (uint32_t)min(r0 + (int64_t)(i + u) * p.subs, (int64_t)p.N - 1);
      x[u] = ld8<TX, TAIL>(p.x, (int64_t)r * p.xs + c, p.xe, n);
      if (p.res) res[u] = ld8<TR, TAIL>(p.res, res_row(r, p.rpg, p.N, p.rs0, p.rs1) + c, p.re, n);
    }
    uint4 words[DROP_U];
    if (p.d.on) {
#pragma unroll
      for (int u = 0; u < DROP_U; ++u) words[u] = hidden_words(p.d, r0 + (int64_t)(i + u) * p.subs, chunk);
    }
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
      const int64_t r = r0 + (int64_t)(i + u) * p.subs;
      if (r >= p.N) return;
      float v[8];
      cvt8<TX, TAIL>(x[u], 8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += bias[e];
      if (p.d.on) drop8(p.d, words[u], v);
      if (p.res) {
        float w[8];
        cvt8<TR, TAIL>(res[u], 8, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += w[e];
      }
      st8<TY, TAIL>(p.y, r * p.ys + c, n, v);
    }
  }
}

// dx and, where part or dbias is given, the block's column sums of it: the sums
// of a thread's rows, then of the block's row groups in their order.
template <typename TDY, typename TX, bool TAIL>
__global__ __launch_bounds__(DROP_SUM_T) void drop_bwd_kernel(DropRows p) {
  __shared__ float red[DROP_SUM_T * 8];
  const int sub = threadIdx.x / p.cw, in_row = (int)threadIdx.x - sub * p.cw, chunk = blockIdx.y * p.cw + in_row;
  const int c = 8 * chunk, n = sub < p.subs ? p.C - c : 0;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows * p.subs + sub;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (n > 0) {
    for (int i = 0; i < p.rows; i += DROP_U) {
      raw8<TDY> dy[DROP_U];
#pragma unroll
      for (int u = 0; u < DROP_U; ++u) {
        const int64_t r = min(r0 + (int64_t)(i + u) * p.subs, (int64_t)p.N - 1);
        dy[u] = ld8<TDY, TAIL>(p.dy, r * p.dys + c, p.dye, n);
      }
      uint4 words[DROP_U];
      if (p.d.on) {
#pragma unroll
        for (int u = 0; u < DROP_U; ++u) words[u] = hidden_words(p.d, r0 + (int64_t)(i + u) * p.subs, chunk);
      }
#pragma unroll
      for (int u = 0; u < DROP_U; ++u) {
        const int64_t r = r0 + (int64_t)(i + u) * p.subs;
        if (r < p.N) {
          float v[8];
          cvt8<TDY, TAIL>(dy[u], n, v);
          if (p.d.on) drop8(p.d, words[u], v);
          if (p.dx) st8<TX, TAIL>(p.dx, r * p.dxs + c, n, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += v[e];
        }
      }
    }
  }
  if (!p.part && !p.dbias) return;  // uniform over the block
#pragma unroll
  for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = sum[e];
  __syncthreads();
  if (sub != 0 || n <= 0) return;
  for (int s = 1; s < p.subs; ++s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += red[(s * p.cw + in_row) * 8 + e];
  }
  if (!p.dbias) st8<float, TAIL>(p.part, (int64_t)blockIdx.x * p.C + c, n, sum);
  else if (p.bias_dt == kBF16) st8<bf16, TAIL>(p.dbias, c, n, sum);
  else st8<float, TAIL>(p.dbias, c, n, sum);
}

}  // namespace hid
}  // namespace dsa
