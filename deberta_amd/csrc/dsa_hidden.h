// dsa_hidden.h — what the operators on hidden states share (gfx950): rows of
// any width, stride and element alignment in chunks of eight columns, the
// keep bits of hidden dropout and sums over a wave.  The operators
// (dsa_drop.h, dsa_rms.h, dsa_embed.h) are bound by HBM traffic.
//
// A lane holds chunks of eight consecutive columns: one 16-byte access for
// bf16, two for fp32, and one Philox call for dropout.  The accesses are
// declared with the alignment of one element: gfx950's global memory
// instructions take any address, so an odd row stride or first column needs
// no kernel of its own.  An odd width does (TAIL: C is no multiple of
// eight): its rows end in a chunk of fewer columns, which is read in one
// access where the eight elements lie inside the tensor (they are then the
// next row's), element by element where they do not (the last row), zeroed
// in registers past the row, and written element by element.  In one kernel
// for both the lanes' conditions would take more scalar registers than
// there are: their spills were a third of the RMS backward's instructions.
#pragma once

#include "dsa_common.h"
#include "dsa_dropout.h"

namespace dsa {
namespace hid {

constexpr int kBF16 = 1;  // DSA_BF16 (DSA_F32 = 0)

template <typename T>
struct Raw8 {
  typedef T v8 __attribute__((ext_vector_type(8)));
  typedef v8 v8u __attribute__((aligned(sizeof(T))));
};
template <typename T>
using raw8 = typename Raw8<T>::v8;

// The lane's n columns from element off of a tensor that ends at element
// `extent` (n <= 0: nothing, zeros; without TAIL n >= 8 otherwise).
template <typename T, bool TAIL>
DSA_DEV raw8<T> ld8(const void* base, int64_t off, int64_t extent, int n) {
  raw8<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)0.f;
  const T* p = static_cast<const T*>(base) + off;
  if (TAIL ? n >= 8 || (n > 0 && off + 8 <= extent) : n > 0) {
    r = *reinterpret_cast<const typename Raw8<T>::v8u*>(p);
  } else if (TAIL && n > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) r[e] = p[e];
  }
  return r;
}

// the n first values as fp32, zero behind them (what ld8 gave for n <= 0 is zero)
template <typename T, bool TAIL>
DSA_DEV void cvt8(const raw8<T>& r, int n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)r[e];
  if (TAIL && n > 0 && n < 8) {
#pragma unroll
    for (int e = 1; e < 8; ++e) v[e] = e < n ? v[e] : 0.f;
  }
}

// Stores the first n of eight values (n <= 0: none).  Where n is below eight
// it is the same in every lane that has such a chunk: C % 8.
template <typename T, bool TAIL>
DSA_DEV void st8(void* base, int64_t off, int n, const float (&v)[8]) {
  if (n <= 0) return;
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef T v2 __attribute__((ext_vector_type(2)));
  typedef v4 v4u __attribute__((aligned(sizeof(T))));
  typedef v2 v2u __attribute__((aligned(sizeof(T))));
  T* p = static_cast<T*>(base) + off;
  raw8<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)v[e];
  if (!TAIL || n >= 8) {
    *reinterpret_cast<typename Raw8<T>::v8u*>(p) = r;
    return;
  }
  const int u = __builtin_amdgcn_readfirstlane(n);
  if (u & 4) *reinterpret_cast<v4u*>(p) = v4{r[0], r[1], r[2], r[3]};
  if (u & 2) *reinterpret_cast<v2u*>(p + (u & 4)) = u & 4 ? v2{r[4], r[5]} : v2{r[0], r[1]};
  if (u & 1) p[u - 1] = u & 4 ? (u & 2 ? r[6] : r[4]) : (u & 2 ? r[2] : r[0]);
}

// A parameter vector's chunk, its type known at run time (read once a block
// or from the caches).
template <bool TAIL>
DSA_DEV void ld_param8(const void* p, int dt, int c, int n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (!p || n <= 0) return;
  if (dt == kBF16) cvt8<bf16, TAIL>(ld8<bf16, TAIL>(p, c, (int64_t)c + n, n), n, v);
  else cvt8<float, TAIL>(ld8<float, TAIL>(p, c, (int64_t)c + n, n), n, v);
}

// element offset of the residual's row r
DSA_DEV int64_t res_row(uint32_t r, uint32_t rpg, uint32_t N, int64_t rs0, int64_t rs1) {
  if (rpg >= N) return (int64_t)r * rs1;
  const uint32_t g = r / rpg;
  return (int64_t)g * rs0 + (int64_t)(r - g * rpg) * rs1;
}

// Hidden dropout's keep bits.  The value at row r (all leading dimensions
// flattened) and column c of a call with threshold t is kept where
//   x = Philox4x32-10(counter = (c / 8, r & 0xffffffff, r >> 32, kHiddenDomain),
//                     key = (seed & 0xffffffff, seed >> 32))
//   u = c % 8;  (x[u / 2] >> (16 * (u % 2))) & 0xffff >= t
// so it depends on the position and the seed alone, not on strides, types or
// the launch, and the backward draws the same bits again: nothing is stored.
// A value is dropped with probability t / 65536 exactly.  Sixteen bits a
// value make one call serve a lane's chunk: about 20 32-bit products and 60
// other operations for eight values, which a bf16 stream hides behind its
// 32 bytes of traffic; with 32 bits a value they would not hide.
constexpr uint32_t kHiddenDomain = 0x68696464u;  // the attention's counters end in the batch row

struct Drop {
  uint32_t on;      // 0: no dropout
  uint32_t lim;     // (t << 16) - 1: a value is kept where its 16 bits, shifted up, are above
                    // (t = 65536: none is)
  uint32_t k0, k1;  // the seed's low and high words
  float scale;      // 65536 / (65536 - t); 0 where everything is dropped
};

// the random words of a chunk
DSA_DEV uint4 hidden_words(const Drop& d, int64_t row, int chunk) {
  return philox4x32_10((uint32_t)chunk, (uint32_t)row, (uint32_t)((uint64_t)row >> 32), kHiddenDomain, d.k0, d.k1);
}

// A dropped value is 0 whatever it was (NaN and infinities included).  The
// words are kept rather than a mask of bits: a compare a value either way,
// and no bit to set and test.
DSA_DEV void drop8(const Drop& d, uint4 x, float (&v)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    v[2 * u] = (w[u] << 16) > d.lim ? v[2 * u] * d.scale : 0.f;
    v[2 * u + 1] = w[u] > d.lim ? v[2 * u + 1] * d.scale : 0.f;
  }
}

// One data-parallel step of a sum over the lanes of a row of 16 (the
// instruction's own lane patterns: no trip through LDS).
template <int CTRL>
DSA_DEV float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
DSA_DEV float lane_value(float x, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
// The sum of x over each L neighbouring lanes, in a fixed order, in every lane.
template <int L>
DSA_DEV float lanes_sum(float x) {
  static_assert(L == 16 || L == 32 || L == 64, "");
  x += dpp<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x += dpp<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x += dpp<0x141>(x);  // row_half_mirror: the other quad of eight lanes
  x += dpp<0x140>(x);  // row_mirror: the other eight of sixteen
  if constexpr (L == 32) x += __shfl_xor(x, 16);
  if constexpr (L == 64) x = (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
  return x;
}

// ---------------------------------------------------------------------------
// out[j][c] = sum over i < nparts of part[i * stride + j * C + c].  A block
// takes SUM_C columns (one line of each part) in SUM_G groups: group g sums
// parts g, g + SUM_G, ... into eight independent sums (eight loads in
// flight), then the groups' sums are added in their order, so the result
// does not depend on scheduling.
constexpr int SUM_C = 32, SUM_G = 32;

struct SumParts {
  const float* part;
  int64_t nparts, stride;
  int C;
  void* out[2];
  int dt[2];
};

static __global__ __launch_bounds__(SUM_C * SUM_G) void sum_parts_kernel(SumParts p) {
  __shared__ float red[SUM_G][SUM_C + 1];
  const int col = threadIdx.x % SUM_C, g = threadIdx.x / SUM_C, j = blockIdx.y;
  if (!p.out[j]) return;  // uniform over the block
  const int c = blockIdx.x * SUM_C + col;
  const float* base = p.part + (int64_t)j * p.C + min(c, p.C - 1);
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t i = g; i < p.nparts; i += 8 * SUM_G) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t k = i + u * SUM_G;
      const float v = base[min(k, p.nparts - 1) * p.stride];
      a[u] += k < p.nparts ? v : 0.f;
    }
  }
  red[g][col] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  __syncthreads();
  if (g != 0 || c >= p.C) return;
  float s = red[0][col];
#pragma unroll
  for (int i = 1; i < SUM_G; ++i) s += red[i][col];
  if (p.dt[j] == kBF16) static_cast<bf16*>(p.out[j])[c] = (bf16)s;
  else static_cast<float*>(p.out[j])[c] = s;
}

}  // namespace hid
}  // namespace dsa
