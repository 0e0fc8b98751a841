// dsa_vocab.h — log probabilities over a vocabulary (gfx950).  For a row of V
// logits x, z = x / T:
//   m = max x,  s = sum exp(z - m / T),  u = sum exp(z - m / T) (z - m / T)
//   lse = m / T + ln s,  log p_j = (x_j - m) / T - ln s
//   entropy = -sum p ln p = ln s - u / s        (both terms are positive)
// and the k largest, in one pass over the row with a running maximum: where a
// batch of values has a larger one, s and u are scaled to it.  The gradient is
//   dx_j = 1 / T (p_j (a + b ln p_j) + sum_t c_t [j = id_t])
// with a and b the row's and c_t given for a few tokens:
//   log probabilities  a = -g - sum g_top - g_H H + g_lse, b = -g_H, c = g, g_top
//   distillation       a = g T^2 Q, b = 0, c_t = -g T^2 q_t, Q = sum q
//
// x - m is formed before its scaling: m / T rounded by itself would move every
// probability of a row whose logits are large, and a row of the type's lowest
// value (a mask that leaves nothing) would overflow; so it has p = 1 / V.  (One
// fused product from a rounded origin, with this form beside it for such rows, and
// the entropy's guard against 0 times -inf taken out of the loop: a fifth fewer
// instructions and no faster, 58 to 94 registers a lane cost what they saved.)
//
// The k largest come out of the same pass.  It keeps the maximum of each
// segment of 64 columns.  A number that the maxima of k segments reach is reached
// by k values at least, so the k largest lie in the segments that reach it and
// are among their values that do: about as many lines of the row as there are
// values to find are read again, and the ranks of what reaches the bound are counted
// (write_top).  Where more than 512 segments or values reach the number, the k segments
// whose maxima are largest (equal ones: the first) are selected exactly, and of their
// values the k largest (top_of_segments): a value outside of them, at most its own
// segment's maximum, has k larger ones before it.  The number is one of 16 bits, so that
// is a row with thousands of values near its largest that are equal in their upper 16
// bits: equal ones in bf16, ones of the same 2^-7 of their value in fp32.  (512 x 128100
// fp32 normals of deviation 2, and the same plus 1000, us: 20 largest 45 and 54, 64 48
// and 69, 128 52 and 90; in bf16, of which 1000 leaves every fourth whole number, 29 and
// 33, 31 and 34, 33 and 69.)
//
// HBM bounds it where there are many rows; of 128100 bf16 columns, us and TB/s of
// what has to move (kernels that only read reach 6.4 to 7.0 so, that copy 6.1):
//   forward   1229 rows in parts 55 + 5 to join (315 MB, 5.3), 4096 rows of a
//             distillation 152 + 17 (1.05 GB, 6.9 the parts by themselves); 64 largest of
//             2048 rows, whole, 95 to 98 a pass of a settled card (525 MB, 5.5), 102 to
//             133 in the first hundred behind an idle one
//   backward  1229 rows 95 (630 MB, 6.6, in part from the last-level cache), 4096 rows
//             of a distillation 379 (2.10 GB, 5.5), of a loss with 85% of the rows left
//             out 198 (1.21 GB, 6.1)
// With few rows it is the chain of a launch, a part's batch, a join and its reads: one
// row 3.8 + 5.1 us with its 5 largest, 16 by one block (and its host side 8.7).
#pragma once

#include <type_traits>

#include "dsa_lanes.h"

namespace dsa {
namespace voc {

constexpr int kSeg = 64;      // columns of a segment
constexpr int kBins = 1024;   // of a selection's histogram
constexpr int kMost = 128;    // entries of a row
constexpr int kRow = 1 << 30;  // vectors: as many as a row has
constexpr int kPartWaves = 4;  // of a block that has a part of a row
constexpr int kUnroll = 4;    // 16-byte loads in flight a lane
constexpr float kLowest = -3.402823466e+38f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1000.f;  // 2^kFar is 0

struct VocabRows {
  const void *x, *ids, *teacher;
  const float *teacher_lse, *dlp, *dent, *dlse, *dtop;
  float *lp, *ent, *lse, *top_lp, *loss;
  float4* stats;  // m, ln s, entropy, 1 / s
  int64_t* top_ids;
  void* dx;
  int64_t xs, dxs, dlp_s, dent_s, dlse_s, ignore;
  int64_t row0;    // the launch's first row
  int V, top, K, ids64, teacher_bf16;
  int keys;        // LDS words for a selection's keys
  int parts, per;  // blocks a row, 16-byte vectors a block
  float4* part;    // [N, parts, kPartWaves]: m, s, u of a wave's share
  uint32_t* seg;   // [N, segs]: the segments' maxima
  int segs;
  float inv_t, t;
  float c;         // log2(e) / T
};

// ---------------------------------------------------------------------------
// values

template <typename T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);  // values of a 16-byte access
};
typedef uint32_t raw __attribute__((ext_vector_type(4)));
typedef raw raw2 __attribute__((aligned(2)));  // aligned as a bf16 is
typedef raw raw4 __attribute__((aligned(4)));

template <typename T>
DSA_DEV void unpack(const raw& r, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = r[i];  // (a bit cast of the element itself takes the vector's first)
    if constexpr (sizeof(T) == 2) {
      v[2 * i] = __builtin_bit_cast(float, w << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
    } else {
      v[i] = __builtin_bit_cast(float, w);
    }
  }
}
// -inf in every place
template <typename T>
DSA_DEV raw raw_none() {
  const uint32_t w = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  return raw{w, w, w, w};
}

// The larger of two or three, a NaN giving way (a signalling one where
// nan_gives_way has run).  The instruction by itself: fmaxf of values that come
// from memory quiets each one first, an instruction a value.
DSA_DEV float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
DSA_DEV float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Takes the wave out of IEEE mode (bit 9 of the mode register), in which the maximum
// of a number and a signalling NaN is a NaN: it would hide the values beside it from
// a row's largest.  Before the wave's first load, which stays behind it.
DSA_DEV void nan_gives_way() {
  __builtin_amdgcn_s_setreg(1 | 9 << 6, 0);
  asm volatile("" ::: "memory");
}
template <int N>
DSA_DEV float max_of(const float* v) {
  static_assert(N % 2 == 0, "");
  float m = max2(v[0], v[1]);
#pragma unroll
  for (int i = 2; i < N; i += 2) m = max3(m, v[i], v[i + 1]);
  return m;
}

// The maxima of four numbers over each L = 8 or 16 neighbouring lanes, one
// instruction a step and number.  A step reads what the last but three wrote: the
// two wait states between a vector instruction and another that reads its register
// across lanes; two more for what was written before.
template <int L>
DSA_DEV void max_of_lanes(float (&v)[4]) {
  static_assert(L == 8 || L == 16, "");
#define DSA_STEP(how)                                                \
  "v_max_f32_dpp %0, %0, %0 " how " row_mask:0xf bank_mask:0xf\n\t" \
  "v_max_f32_dpp %1, %1, %1 " how " row_mask:0xf bank_mask:0xf\n\t" \
  "v_max_f32_dpp %2, %2, %2 " how " row_mask:0xf bank_mask:0xf\n\t" \
  "v_max_f32_dpp %3, %3, %3 " how " row_mask:0xf bank_mask:0xf\n\t"
  asm("s_nop 1\n\t" DSA_STEP("quad_perm:[1,0,3,2]") DSA_STEP("quad_perm:[2,3,0,1]") DSA_STEP("row_half_mirror")
      : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
  if (L == 16)
    asm("s_nop 1\n\t" DSA_STEP("row_mirror") : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#undef DSA_STEP
}

DSA_DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Whole numbers that order as the values do (NaN as -inf, -0 as +0), above 0.
// bf16's are 16 bits.
template <typename T>
DSA_DEV uint32_t key_of(float x) {
  const int b = __builtin_bit_cast(int, (x == x ? x : -__builtin_inff()) + 0.f);
  const uint32_t k = (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
  return sizeof(T) == 2 ? k >> 16 : k;
}
template <typename T>
DSA_DEV float of_key(uint32_t k) {
  if (sizeof(T) == 2) {
    const uint32_t b = k & 0x8000u ? k ^ 0x8000u : ~k & 0xffffu;
    return __builtin_bit_cast(float, b << 16);
  }
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

DSA_DEV int64_t load_id(const void* ids, int ids64, int64_t i) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int*>(ids)[i];
}

// ---------------------------------------------------------------------------
// the running sums

// x's exponent in a row with maximum m: c = log2(e) / T
DSA_DEV float exponent(float x, float m, float c) { return (x - m) * c; }

struct Run {
  float m, s, u;  // u in units of ln 2
};
DSA_DEV Run run_none() { return Run{kLowest, 0.f, 0.f}; }

// the sums as of a maximum that is no smaller
template <bool ENT>
DSA_DEV void raise(Run& r, float m, float c) {
  const float d = fmaxf(exponent(r.m, m, c), kFar), f = exp2_(d);
  if (ENT) r.u = f * fmaf(d, r.s, r.u);
  r.s *= f;
  r.m = m;
}
template <int E, bool ENT>
DSA_DEV void add(Run& r, const float* x, float most, float c) {
  if (most > r.m) raise<ENT>(r, most, c);
  float s[2] = {0.f, 0.f}, u[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = exponent(x[e], r.m, c), p = exp2_(t);
    s[e & 1] += p;
    if (ENT) u[e & 1] = fmaf(p, fmaxf(t, kFar), u[e & 1]);  // 0 where t is -inf
  }
  r.s += s[0] + s[1];
  if (ENT) r.u += u[0] + u[1];
}

DSA_DEV float wave_max_f(float x) {
  x = max2(x, hid::dpp<0xB1>(x));
  x = max2(x, hid::dpp<0x4E>(x));
  x = max2(x, hid::dpp<0x141>(x));
  x = max2(x, hid::dpp<0x140>(x));  // of 16 lanes
  return max2(max3(hid::lane_value(x, 0), hid::lane_value(x, 16), hid::lane_value(x, 32)), hid::lane_value(x, 48));
}
// The wave's sums out of its lanes', in every lane.
template <bool ENT>
DSA_DEV Run wave_run(Run r, float c) {
  raise<ENT>(r, wave_max_f(r.m), c);
  r.s = hid::lanes_sum<64>(r.s);
  if (ENT) r.u = hid::lanes_sum<64>(r.u);
  return r;
}
// The block's sums out of its threads', red: 3 words a wave.  leave_run by all of
// them, then, behind a barrier, run_of by whoever needs them.
template <bool ENT>
DSA_DEV void leave_run(Run r, float c, float* red) {
  r = wave_run<ENT>(r, c);
  if ((threadIdx.x & 63) == 0) {
    float* w = red + 3 * (threadIdx.x >> 6);
    w[0] = r.m, w[1] = r.s, w[2] = r.u;
  }
}
template <int NT, bool ENT>
DSA_DEV Run run_of(const float* red, float c) {
  float most = kLowest;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) most = max2(most, red[3 * i]);
  Run all{most, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    Run w{red[3 * i], red[3 * i + 1], red[3 * i + 2]};
    raise<ENT>(w, most, c);
    all.s += w.s, all.u += w.u;
  }
  return all;
}
template <int NT, bool ENT>
DSA_DEV Run block_run(Run r, float c, float* red) {
  if constexpr (NT == 64) return wave_run<ENT>(r, c);
  leave_run<ENT>(r, c, red);
  __syncthreads();
  return run_of<NT, ENT>(red, c);
}

// ---------------------------------------------------------------------------
// a row in 16-byte accesses: it starts `pad` values behind a 128-byte border, and
// positions count from there, so that a wave's access is of whole lines.  Vectors
// v0 .. v1 - 1 lie in the row whole; the values before and behind them are taken
// one by one, a lane each.
template <typename T>
struct Line {
  static constexpr int N = Vec<T>::N;
  const T* row;
  const T* base;  // of position 0
  int V, pad, v0, v1, head, edges, tail0;
  DSA_DEV Line(const void* x, int64_t stride, int64_t r, int cols) : V(cols) {
    row = static_cast<const T*>(x) + r * stride;
    pad = (int)(reinterpret_cast<uintptr_t>(row) & 127u) / (int)sizeof(T);
    base = row - pad;
    v0 = (pad + N - 1) / N;
    v1 = max((int)(((int64_t)pad + V) / N), v0);
    head = min(V, v0 * N - pad);
    tail0 = min(V, v1 * N - pad);  // the row's first value behind the vectors
    edges = head + (V - tail0);
  }
  DSA_DEV int edge(int i) const { return i < head ? i : tail0 + (i - head); }
  template <bool FAR = false>
  DSA_DEV raw load(int v) const {
    const raw* at = reinterpret_cast<const raw*>(base) + v;
    return FAR ? __builtin_nontemporal_load(at) : *at;
  }
};

// The sums of a thread over its share of positions from `from` to `to` vectors (a
// multiple of 64 each, or the row's end); with SEG the keys of the maxima of the
// `segs` segments from there on, for which the caller waits.  FAR: past the caches.
template <typename T, int NT, bool ENT, bool SEG, bool FAR>
DSA_DEV Run stream(const Line<T>& l, int from, int to, float c, uint32_t* keys, int segs) {
  constexpr int N = Vec<T>::N, E = kUnroll * N, L = kSeg / N;
  const int tid = threadIdx.x;
  const int first = max(from, l.v0), end = min(to, l.v1);
  Run r = run_none();
  if (SEG) {
    for (int i = tid; i < segs; i += NT) keys[i] = 0xff800000u;  // -inf
    __syncthreads();
  }
  // the next batch is loaded before this one is worked on (behind the end the
  // last vector again)
  raw next[kUnroll];
  if (first < end) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) next[i] = l.template load<FAR>(min(max(from + i * NT + tid, first), end - 1));
    for (int vb = from; vb < end; vb += NT * kUnroll) {
      raw q[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) q[i] = next[i];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) next[i] = l.template load<FAR>(min(vb + (i + kUnroll) * NT + tid, end - 1));
      if (vb < first || vb + NT * kUnroll > end) {
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
          const int v = vb + i * NT + tid;
          if (v < first || v >= end) q[i] = raw_none<T>();
        }
      }
      float x[E], most[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        unpack<T>(q[i], x + i * N);
        most[i] = max_of<N>(x + i * N);
      }
      add<E, ENT>(r, x, max_of<kUnroll>(most), c);
      if (SEG) {
        max_of_lanes<L>(most);
        if (tid % L == 0) {
          uint32_t* to = keys + (vb - from + tid) / L;
#pragma unroll
          for (int i = 0; i < kUnroll; ++i)
            if (vb + i * NT + tid < end) to[i * (NT / L)] = __builtin_bit_cast(uint32_t, most[i]);
        }
      }
    }
  }
  if (SEG) {
    __syncthreads();
    for (int i = tid; i < segs; i += NT) keys[i] = key_of<T>(__builtin_bit_cast(float, keys[i]));
    __syncthreads();
  }
  const int head = from == 0 ? l.head : 0, tail = l.v1 >= from && l.v1 < to ? l.V - l.tail0 : 0;
  if (tid < head + tail) {
    const int j = tid < head ? tid : l.tail0 + (tid - head);
    const float x = (float)l.row[j];
    add<1, ENT>(r, &x, max2(x, kLowest), c);
    if (SEG) atomicMax(&keys[(l.pad + j) / kSeg - from / L], key_of<T>(x));
  }
  return r;
}

// ---------------------------------------------------------------------------
// the largest

constexpr uint32_t kCands = 512;  // segments, and values, that compete in write_top

struct Shared {
  uint32_t* keys;
  uint32_t* hist;    // kBins
  uint64_t* cand;    // kCands
  int* seg;          // kCands
  int* list;         // kMost
  uint32_t* picked;  // kMost
  uint32_t* word;    // 24
  float* sums;       // m, ln s
};
constexpr int kSharedWords = kBins + 3 * kCands + 2 * kMost + 24 + 2;
DSA_DEV Shared shared_at(uint32_t* lds, int keys) {  // keys: a multiple of 4
  Shared s;
  s.keys = lds;
  s.hist = lds + keys;
  uint32_t* at = s.hist + kBins;
  s.cand = reinterpret_cast<uint64_t*>(at);
  s.seg = reinterpret_cast<int*>(at + 2 * kCands);
  s.list = s.seg + kCands;
  s.picked = reinterpret_cast<uint32_t*>(s.list + kMost);
  s.word = s.picked + kMost;
  s.sums = reinterpret_cast<float*>(s.word + 24);
  return s;
}

// The sum over the threads before this one; w: a word a wave and one.  The
// caller waits before the next use of w.
template <int NT>
DSA_DEV uint32_t block_before(uint32_t x, uint32_t* w) {
  const int lane = threadIdx.x & 63;
  uint32_t all = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(all, o);
    if (lane >= o) all += y;
  }
  if constexpr (NT > 64) {
    if (lane == 63) w[threadIdx.x >> 6] = all;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int i = 0; i < NT / 64 - 1; ++i) before += i < (int)(threadIdx.x >> 6) ? w[i] : 0u;
    all += before;
  }
  return all - x;
}

// The places of the `need` largest of key(0) .. key(n - 1), equal ones by their
// place, into sh.list in the order of their places (0 < need <= n, need <= kMost,
// n < 2^16).
//
// Keys are counted into bins of equal width between the least and the largest,
// the bin that holds the last one wanted is cut into bins again, and so on until
// all of a bin are wanted or its keys are equal: one round where the keys span
// at most 1024, at most four (10 bits a round).
template <int NT, typename F>
DSA_DEV void choose(const Shared& sh, int n, int need, F key) {
  constexpr int W = NT / 64, PER = kBins / NT;
  const int tid = threadIdx.x;
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = tid; i < n; i += NT) {
    const uint32_t k = key(i);
    lo = min(lo, k), hi = max(hi, k);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) lo = min(lo, (uint32_t)__shfl_xor(lo, o)), hi = max(hi, (uint32_t)__shfl_xor(hi, o));
  if constexpr (W > 1) {
    if ((tid & 63) == 0) sh.word[2 * (tid >> 6)] = lo, sh.word[2 * (tid >> 6) + 1] = hi;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) lo = min(lo, sh.word[2 * i]), hi = max(hi, sh.word[2 * i + 1]);
  }
  int want = need;
  uint32_t equal;  // of the keys at lo, how many are taken; all above it are
  for (;;) {
    const uint32_t span = hi - lo;
    const int shift = span < (uint32_t)kBins ? 0 : 22 - __builtin_clz(span);
    for (int i = tid; i < kBins; i += NT) sh.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = key(i);
      if (k >= lo && k <= hi) atomicAdd(&sh.hist[(k - lo) >> shift], 1u);
    }
    __syncthreads();
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += sh.hist[kBins - 1 - (tid * PER + i)];
    uint32_t above = block_before<NT>(mine, sh.word);
    __syncthreads();
    if (above < (uint32_t)want && above + mine >= (uint32_t)want) {  // one thread
      int b = kBins - 1 - tid * PER;
      while (above + sh.hist[b] < (uint32_t)want) above += sh.hist[b--];
      sh.word[0] = (uint32_t)b, sh.word[1] = (uint32_t)want - above, sh.word[2] = sh.hist[b];
    }
    __syncthreads();
    const uint32_t bin = sh.word[0], here = sh.word[2];
    want = (int)sh.word[1];
    lo += bin << shift;
    hi = min(hi, lo + ((1u << shift) - 1u));
    equal = here == (uint32_t)want ? (uint32_t)n : (uint32_t)want;
    __syncthreads();
    if (here == (uint32_t)want || shift == 0) break;
  }
  const int per = (n + NT - 1) / NT, first = min(n, tid * per), last = min(n, first + per);
  uint32_t counts = 0;  // above lo, and at lo in the upper half
  for (int i = first; i < last; ++i) {
    const uint32_t k = key(i);
    counts += k > lo ? 1u : k == lo ? 0x10000u : 0u;
  }
  const uint32_t before = block_before<NT>(counts, sh.word);
  uint32_t over = before & 0xffffu, at = before >> 16;
  for (int i = first; i < last; ++i) {
    const uint32_t k = key(i);
    if (k > lo || (k == lo && at < equal)) sh.list[over + min(at, equal)] = i;
    over += k > lo, at += k == lo;
  }
  __syncthreads();
}

// The k-th largest of 64 G numbers, G a lane, cut to its upper 16 bits, by one
// wave: a bit at a time, by counting the numbers that reach it.
template <int G>
DSA_DEV uint32_t kth_largest(const uint32_t (&g)[G], int k) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t trial = t | 1u << bit;
    int n = 0;
#pragma unroll
    for (int u = 0; u < G; ++u) n += __popcll(__ballot(g[u] >= trial));
    t = n >= k ? trial : t;
  }
  return t;
}
// A number that at least k of the threads' values reach: the k-th largest of the
// maxima of 64 groups of threads up to k = 32, of 256 from there on, where the k-th
// of 64 is too low a bound (512 x 128128 bf16, of 256 and of 64 groups: 16 largest
// 29.4 and 28.8 us, 32 29.8 and 29.3, 48 30.1 and 30.8, 64 30.9 and 46.6).  Meanwhile
// the second wave does `other`.
template <int NT, typename F>
DSA_DEV uint32_t reached(uint32_t most, int k, const Shared& sh, F other) {
  static_assert(NT >= 256 && NT <= kBins && kMost <= 256, "");
  const int tid = threadIdx.x;
  uint32_t* all = sh.hist;
  all[tid] = most;
  __syncthreads();
  if (tid < 64) {
    uint32_t g[4], one[1] = {0};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      g[u] = 0;
      for (int i = tid + 64 * u; i < NT; i += 256) g[u] = max(g[u], all[i]);
      one[0] = max(one[0], g[u]);
    }
    const uint32_t t = k <= 32 ? kth_largest(one, k) : kth_largest(g, k);
    if (tid == 0) sh.word[0] = t;
  } else if (tid < 128) {
    other();
  }
  __syncthreads();
  return sh.word[0];
}

// Appends to a list of *count entries: f(e, place) for every bit e < 8 of the lanes'
// m, with one addition a wave.
template <typename F>
DSA_DEV void append(uint32_t m, uint32_t* count, F f) {
  const uint64_t some = __ballot(m != 0);
  if (some == 0) return;
  // how many the lanes before have, and all: the bits of the lanes' counts
  const uint32_t mine = (uint32_t)__popc(m);
  uint32_t total = 0, at = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint64_t with = __ballot(mine >> b & 1);
    total += (uint32_t)__popcll(with) << b;
    at += __builtin_amdgcn_mbcnt_hi((uint32_t)(with >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)with, 0)) << b;
  }
  if (m == 0) return;
  uint32_t first = 0;
  if ((int)(threadIdx.x & 63) == __builtin_ctzll(some)) first = atomicAdd(count, total);
  at += __builtin_amdgcn_readfirstlane(first);
  for (; m; m &= m - 1) f(__builtin_ctz(m), at++);
}

DSA_DEV int round_8(int n) { return (n + 7) & ~7; }

template <typename T>
DSA_DEV uint32_t wide_key(uint32_t k) { return sizeof(T) == 2 ? k << 16 : k; }

// One of the row's largest.
template <typename T>
DSA_DEV void put_top(const VocabRows& p, int64_t r, int rank, int j, uint32_t key, const Shared& sh) {
  p.top_ids[r * p.top + rank] = j;
  p.top_lp[r * p.top + rank] = fmaf(exponent(of_key<T>(key), sh.sums[0], p.c), kLn2, -sh.sums[1]);
}

// The row's largest, from its segments' maxima in sh.keys: those of the k
// segments whose maxima are largest (read again at every step: this is for rows
// with thousands of values that are equal in their upper 16 bits).
template <typename T, int NT>
DSA_DEV void top_of_segments(const Line<T>& l, const VocabRows& p, int64_t r, const Shared& sh) {
  const int tid = threadIdx.x, k = p.top;
  const int segs = (l.pad + p.V - 1) / kSeg + 1, found = min(k, segs);
  choose<NT>(sh, segs, found, [&](int i) { return sh.keys[i]; });
  if (tid < found) sh.picked[tid] = (uint32_t)sh.list[tid];
  __syncthreads();
  const auto column = [&](int i) { return (int)sh.picked[i / kSeg] * kSeg + i % kSeg - l.pad; };
  const auto key = [&](int i) {
    const int j = column(i);
    return j >= 0 && j < p.V ? key_of<T>((float)l.row[j]) : 0u;
  };
  choose<NT>(sh, found * kSeg, k, key);
  if (tid < k) sh.hist[tid] = key(sh.list[tid]);
  __syncthreads();
  if (tid < k) {
    const uint32_t mine = sh.hist[tid];
    int rank = 0;
    for (int o = 0; o < k; ++o) rank += sh.hist[o] > mine || (sh.hist[o] == mine && o < tid);
    put_top<T>(p, r, rank, column(sh.list[tid]), mine, sh);
  }
}

// f(vector's values, column of the first, of the n that are the row's) for the
// 16-byte pieces of the first `found` segments of sh.seg, four loads of a thread
// in flight.
template <typename T, int NT, typename F>
DSA_DEV void values_of(const Line<T>& l, const Shared& sh, int found, F f) {
  constexpr int N = Vec<T>::N, L = kSeg / N, U = 4;
  const int n = found * L;
  for (int i0 = threadIdx.x; i0 < n; i0 += U * NT) {
    int v[U];
    raw q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT;
      v[u] = i < n ? sh.seg[i / L] * L + i % L : -1;
      q[u] = raw_none<T>();
      if (v[u] >= l.v0 && v[u] < l.v1) q[u] = l.load(v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v[u] < 0) continue;
      float x[N];
      const int j = v[u] * N - l.pad;
      if (v[u] >= l.v0 && v[u] < l.v1) {
        unpack<T>(q[u], x);
        f(x, j, 0, N);
      } else {
        const int lo = max(0, -j), hi = min(N, l.V - j);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = e >= lo && e < hi ? (float)l.row[j + e] : -__builtin_inff();
        f(x, j, lo, hi);
      }
    }
  }
}

// The given token's logit, NaN outside the vocabulary.
template <typename T>
DSA_DEV float given(const Line<T>& l, const VocabRows& p, int64_t id) {
  return p.lp && id >= 0 && id < p.V ? (float)l.row[id] : __builtin_nanf("");
}

// One thread: the row's results; x: the given token's logit.
DSA_DEV void write_row(const VocabRows& p, int64_t r, const Run& all, float ln_s, float x) {
  const float ent = ln_s - kLn2 * all.u / all.s;
  if (p.lp) p.lp[r] = fmaf(exponent(x, all.m, p.c), kLn2, -ln_s);
  if (p.ent) p.ent[r] = ent;
  if (p.lse) p.lse[r] = fmaf(all.m, p.inv_t, ln_s);
  if (p.stats) p.stats[r] = float4{all.m, ln_s, ent, 1.f / all.s};
}

// The same where few values compete, as nearly always: a bound that k values
// reach leaves a few segments, and of those a few values, whose ranks are counted
// (value and place in one number, so that equal values go by their place).  Where
// there are more than kCands of either, top_of_segments takes over.  The row's other
// results too, from its waves' sums in red and the given token's logit x: a wave has
// them ready while another looks for the bound (64 largest of 2048 x 128100 bf16 96.7
// to 95.8 us, 10 of 512 x 128128 32.0 to 31.5, against one after the other).  Keys and
// red may be fresh: a barrier comes first.
template <typename T, int NT>
DSA_DEV void write_top(const Line<T>& l, const VocabRows& p, int64_t r, const Shared& sh, const float* red, float x) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, k = p.top;
  const int segs = (l.pad + p.V - 1) / kSeg + 1;
  const uint32_t least = wide_key<T>(key_of<T>(-__builtin_inff()));
  constexpr int U = 2048 / NT;  // keys of a thread in a step
  uint32_t most = 0;
  __syncthreads();
  for (int i = 0; i < segs; i += U * NT) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i + u * NT + tid;
      const uint32_t key = sh.keys[min(at, segs - 1)];
      most = max(most, at < segs ? key : 0u);
    }
  }
  if (tid == 0) sh.word[1] = 0, sh.word[2] = 0;
  uint32_t bound = reached<NT>(wide_key<T>(most), k, sh, [&] {
    const Run sums = run_of<NT, true>(red, p.c);
    const float ln_s = logf(sums.s);
    if (tid == 64) {
      write_row(p, r, sums, ln_s, x);
      sh.sums[0] = sums.m, sh.sums[1] = ln_s;
    }
  });
  for (int i = 0; i < segs; i += U * NT) {
    uint32_t in = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i + u * NT + tid;
      in |= (uint32_t)(at < segs && wide_key<T>(sh.keys[min(at, segs - 1)]) >= bound) << u;
    }
    append(in, &sh.word[1], [&](int u, uint32_t at) {
      if (at < kCands) sh.seg[at] = i + u * NT + tid;
    });
  }
  __syncthreads();
  const uint32_t found = sh.word[1];
  __syncthreads();  // what follows writes the word again
  for (int round = 0; round < 2 && found <= kCands; ++round) {
    // the segments' bound may be far below their values', where there are few segments
    if (round == 1 || (segs < 4 * k && found * kSeg > kCands)) {
      round = 1;
      float top = -__builtin_inff();
      values_of<T, NT>(l, sh, (int)found, [&](const float* x, int, int, int) { top = max2(top, max_of<N>(x)); });
      bound = max(bound, reached<NT>(wide_key<T>(key_of<T>(top)), k, sh, [] {}));
    }
    const bool all = bound <= least;  // NaN are -inf here
    const float limit = all ? -__builtin_inff() : of_key<T>(sizeof(T) == 2 ? bound >> 16 : bound);
    values_of<T, NT>(l, sh, (int)found, [&](const float* x, int j, int lo, int hi) {
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) in |= (uint32_t)(e >= lo && e < hi && (all || x[e] >= limit)) << e;
      append(in, &sh.word[2], [&](int e, uint32_t at) {
        if (at < kCands) sh.cand[at] = (uint64_t)key_of<T>((float)l.row[j + e]) << 32 | (uint32_t)~(j + e);
      });
    });
    __syncthreads();
    const int n = (int)sh.word[2];
    if (n <= (int)kCands) {
      // up to a multiple of 8, which is what a step compares
      if (tid >= n && tid < round_8(n)) sh.cand[tid] = 0;
      if (NT < (int)kCands && tid + NT >= n && tid + NT < round_8(n)) sh.cand[tid + NT] = 0;
      __syncthreads();
      for (int t = tid; t < n; t += NT) {
        const uint64_t mine = sh.cand[t];
        int rank = 0;
        for (int o = 0; o < n; o += 8) {
          uint64_t other[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) other[u] = sh.cand[o + u];
#pragma unroll
          for (int u = 0; u < 8; ++u) rank += other[u] > mine;
        }
        if (rank < k) put_top<T>(p, r, rank, (int)~(uint32_t)mine, (uint32_t)(mine >> 32), sh);
      }
      return;
    }
    __syncthreads();
    if (tid == 0) sh.word[2] = 0;
    __syncthreads();
  }
  top_of_segments<T, NT>(l, p, r, sh);
}

// ---------------------------------------------------------------------------
// forward: a block a row

// what a row that is left out gives
template <int NT>
DSA_DEV void write_none(const VocabRows& p, int64_t r) {
  const int tid = threadIdx.x;
  if (tid == 0) {
    if (p.lp) p.lp[r] = 0.f;
    if (p.ent) p.ent[r] = 0.f;
    if (p.lse) p.lse[r] = 0.f;
    if (p.stats) p.stats[r] = float4{0.f, 0.f, 0.f, 0.f};
  }
  for (int t = tid; t < p.top; t += NT) p.top_lp[r * p.top + t] = 0.f, p.top_ids[r * p.top + t] = -1;
}

template <typename T, int NT, bool TOP, bool FAR>
__global__ __launch_bounds__(NT) void logprobs_fwd_kernel(VocabRows p) {
  extern __shared__ __align__(16) uint32_t lds[];
  if (TOP) nan_gives_way();
  __shared__ float red[3 * (NT / 64)];
  const int64_t r = p.row0 + blockIdx.x;
  const int64_t id = p.ids ? load_id(p.ids, p.ids64, r) : 0;
  if (p.ids && id == p.ignore) {
    write_none<NT>(p, r);
    return;
  }
  const Line<T> l(p.x, p.xs, r, p.V);
  const float x = given(l, p, id);  // early: its way from memory is long
  const Run mine = stream<T, NT, true, TOP, FAR>(l, 0, kRow, p.c, lds, p.segs);
  if constexpr (TOP) {
    leave_run<true>(mine, p.c, red);
    write_top<T, NT>(l, p, r, shared_at(lds, p.keys), red, x);
  } else {
    const Run all = block_run<NT, true>(mine, p.c, red);
    if (threadIdx.x == 0) write_row(p, r, all, logf(all.s), x);
  }
}

// A part of a row by a block, where rows are few or long: its waves' sums, and its
// segments' maxima, for the row's join.
template <typename T, int NT, bool ENT, bool SEG, bool FAR>
DSA_DEV void write_part(const VocabRows& p, int64_t r, int part, uint32_t* keys) {
  constexpr int L = kSeg / Vec<T>::N;
  const Line<T> l(p.x, p.xs, r, p.V);
  const int from = part * p.per;
  const int first = from / L, n = min(p.per / L, p.segs - first);  // segments
  const Run w = wave_run<ENT>(stream<T, NT, ENT, SEG, FAR>(l, from, from + p.per, p.c, keys, n), p.c);
  if ((threadIdx.x & 63) == 0)
    p.part[(r * p.parts + part) * (NT / 64) + threadIdx.x / 64] = float4{w.m, w.s, w.u, 0.f};
  if (SEG) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) p.seg[r * p.segs + first + i] = keys[i];
  }
}

template <typename T, int NT, bool TOP, bool FAR>
__global__ __launch_bounds__(NT) void logprobs_part_kernel(VocabRows p) {
  extern __shared__ __align__(16) uint32_t lds[];
  if (TOP) nan_gives_way();
  const int64_t r = p.row0 + blockIdx.x / (uint32_t)p.parts;
  if (p.ids && load_id(p.ids, p.ids64, r) == p.ignore) return;
  write_part<T, NT, true, TOP, FAR>(p, r, blockIdx.x % (uint32_t)p.parts, lds);
}

// A thread's share of a row's parts; q: its first (part_of).
DSA_DEV float4 part_of(const VocabRows& p, int64_t r) {
  const int n = p.parts * kPartWaves;
  return (int)threadIdx.x < n ? p.part[r * n + threadIdx.x] : float4{kLowest, 0.f, 0.f, 0.f};
}
template <int NT, bool ENT>
DSA_DEV Run join_parts(const VocabRows& p, int64_t r, float4 q) {
  Run all{q.x, q.y, q.z};
  const int n = p.parts * kPartWaves;
  for (int i = NT + threadIdx.x; i < n; i += NT) {
    q = p.part[r * n + i];
    Run w{q.x, q.y, q.z};
    const float m = max2(all.m, w.m);
    raise<ENT>(all, m, p.c);
    raise<ENT>(w, m, p.c);
    all.s += w.s, all.u += w.u;
  }
  return all;
}

template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_join_kernel(VocabRows p) {
  extern __shared__ __align__(16) uint32_t lds[];
  if (TOP) nan_gives_way();
  __shared__ float red[3 * (NT / 64)];
  const int64_t r = p.row0 + blockIdx.x;
  const int64_t id = p.ids ? load_id(p.ids, p.ids64, r) : 0;
  if (p.ids && id == p.ignore) {
    write_none<NT>(p, r);
    return;
  }
  const Line<T> l(p.x, p.xs, r, p.V);
  const float x = given(l, p, id);
  const float4 q = part_of(p, r);
  if constexpr (TOP) {
    // the loads of 2048 keys in flight; keys past the segments are not read
    constexpr int U = 2048 / NT;
    const uint32_t* seg = p.seg + r * p.segs;
    for (int i = threadIdx.x; i < p.segs; i += U * NT) {
      uint32_t k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) k[u] = seg[min(i + u * NT, p.segs - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * NT < p.segs) lds[i + u * NT] = k[u];
    }
  }
  const Run mine = join_parts<NT, true>(p, r, q);
  if constexpr (TOP) {
    leave_run<true>(mine, p.c, red);
    write_top<T, NT>(l, p, r, shared_at(lds, p.keys), red, x);
  } else {
    const Run all = block_run<NT, true>(mine, p.c, red);
    if (threadIdx.x == 0) write_row(p, r, all, logf(all.s), x);
  }
}

// ---------------------------------------------------------------------------
// a teacher's entries: two a lane of a wave

struct Entries {
  int64_t id[2];
  float q[2], log_q[2];
  float total;  // sum of q
  bool any;     // an id that is an entry's
  bool bad;     // one outside the vocabulary
};
DSA_DEV Entries entries_of(const VocabRows& p, int64_t r) {
  Entries e;
  const int lane = threadIdx.x & 63;
  float t[2], most = kLowest;
  bool bad = false, any = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int k = lane + 64 * i;
    const bool in = k < p.K;
    const int64_t at = r * p.K + min(k, p.K - 1);
    e.id[i] = in ? load_id(p.ids, p.ids64, at) : -1;
    const float v = p.teacher_bf16 ? (float)static_cast<const bf16*>(p.teacher)[at] : static_cast<const float*>(p.teacher)[at];
    t[i] = e.id[i] >= 0 ? v : -__builtin_inff();
    any |= e.id[i] >= 0;
    bad |= e.id[i] >= p.V;
    most = max2(most, t[i]);
  }
  e.any = __ballot(any) != 0;
  e.bad = __ballot(bad) != 0;
  if (p.teacher_lse) {
    const float lse = p.teacher_lse[r];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e.log_q[i] = t[i] * p.inv_t - lse;
      e.q[i] = expf(e.log_q[i]);
    }
    e.total = hid::lanes_sum<64>(e.q[0] + e.q[1]);
    return e;
  }
  most = wave_max_f(most);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e.log_q[i] = (t[i] - most) * p.inv_t;
    e.q[i] = expf(e.log_q[i]);
  }
  const float sum = hid::lanes_sum<64>(e.q[0] + e.q[1]);
  // every entry's logit -inf: there is none
  const float ln = logf(sum), inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 2; ++i) e.q[i] *= inv, e.log_q[i] -= ln;
  e.total = sum == 0.f ? 0.f : sum * inv == sum * inv ? 1.f : __builtin_nanf("");
  return e;
}

// What a row without entries gives.
DSA_DEV void write_no_loss(const VocabRows& p, int64_t r) {
  if (threadIdx.x != 0) return;
  p.loss[r] = 0.f;
  if (p.stats) p.stats[r] = float4{0.f, 0.f, 0.f, 0.f};
}

// By one wave: the row's loss.
template <typename T>
DSA_DEV void write_loss(const VocabRows& p, int64_t r, const Entries& e, const Run& all) {
  const T* row = static_cast<const T*>(p.x) + r * p.xs;
  const float ln_s = logf(all.s);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (e.id[i] < 0 || e.id[i] >= p.V || e.q[i] == 0.f) continue;
    const float log_p = fmaf(exponent((float)row[e.id[i]], all.m, p.c), kLn2, -ln_s);
    sum += e.q[i] * (e.log_q[i] - log_p);
  }
  sum = hid::lanes_sum<64>(sum);
  if (threadIdx.x == 0) {
    p.loss[r] = e.bad ? __builtin_nanf("") : p.t * (p.t * sum);  // T^2 may be no float32's
    if (p.stats) p.stats[r] = float4{all.m, ln_s, 0.f, 1.f / all.s};
  }
}

template <typename T, int NT, bool FAR>
__global__ __launch_bounds__(NT) void distill_fwd_kernel(VocabRows p) {
  __shared__ float red[3 * (NT / 64)];
  const int64_t r = p.row0 + blockIdx.x;
  const Entries e = entries_of(p, r);  // by every wave
  if (!e.any) {
    write_no_loss(p, r);
    return;
  }
  const Line<T> l(p.x, p.xs, r, p.V);
  const Run all = block_run<NT, false>(stream<T, NT, false, false, FAR>(l, 0, kRow, p.c, nullptr, 0), p.c, red);
  if (threadIdx.x < 64) write_loss<T>(p, r, e, all);
}

template <typename T, int NT, bool FAR>
__global__ __launch_bounds__(NT) void distill_part_kernel(VocabRows p) {
  const int64_t r = p.row0 + blockIdx.x / (uint32_t)p.parts;
  bool any = false;  // by every wave
  for (int k = threadIdx.x & 63; k < p.K; k += 64) any |= load_id(p.ids, p.ids64, r * p.K + k) >= 0;
  if (__ballot(any) == 0) return;
  write_part<T, NT, false, false, FAR>(p, r, blockIdx.x % (uint32_t)p.parts, nullptr);
}

// (4096 rows of 128 entries 14 us by a wave each, each entry's logit a line of its
// own from memory; handed on by the parts, which had them in the caches, 6 and 5
// more in the parts.)
template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_join_kernel(VocabRows p) {
  __shared__ float red[3 * (NT / 64)];
  const int64_t r = p.row0 + blockIdx.x;
  const Entries e = entries_of(p, r);  // by every wave
  if (!e.any) {
    write_no_loss(p, r);
    return;
  }
  const Run all = block_run<NT, false>(join_parts<NT, false>(p, r, part_of(p, r)), p.c, red);
  if (threadIdx.x < 64) write_loss<T>(p, r, e, all);
}

// ---------------------------------------------------------------------------
// backward: e = exp2((x - m) c), dx = e (a + b (x - m) c) and, at a few
// columns, a term more

// the row's constants, and how many columns have a term of their own in LDS (behind
// them up to a multiple of 4 column -1)
struct Grad {
  float m, a, b;
  int n;
};
template <bool B>
DSA_DEV float grad_of(const Grad& g, float t) {
  const float e = exp2_(t);
  return B ? e * fmaf(g.b, fmaxf(t, kFar), g.a) : e * g.a;
}

template <typename T>
DSA_DEV void pack(const float* v, raw& r) {
  if constexpr (sizeof(T) == 2) {
    typedef bf16 v8 __attribute__((ext_vector_type(8)));
    v8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (bf16)v[i];
    r = __builtin_bit_cast(raw, o);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, v[i]);
  }
}

template <bool FAR>
DSA_DEV void store(raw* to, raw v) {
  if (FAR) __builtin_nontemporal_store(v, to);
  else *to = v;
}

// A block's part of a row: vectors lo .. hi - 1, and the row's single values with
// the first part.
template <typename T>
struct Part {
  Line<T> l;
  int from, lo, hi, edges;
  DSA_DEV Part(const VocabRows& p, int64_t r, int part) : l(p.dx, p.dxs, r, p.V) {
    from = part * p.per, lo = max(from, l.v0), hi = min(l.v1, from + p.per);
    edges = part == 0 ? l.edges : 0;
  }
  DSA_DEV bool has(int j) const {
    const int at = l.pad + j, v = at / Line<T>::N;
    return v >= l.v0 && v < l.v1 ? v >= lo && v < hi : edges > 0;
  }
};

// A part of a row of the gradient in 16-byte stores; the logits' row may lie
// otherwise to 16-byte borders.  FAR: past the caches, for gradients that do not
// stay in them (their lines would be written back while the next kernel reads).
template <typename T, int NT, bool B, bool FAR>
DSA_DEV void write_grad(const VocabRows& p, int64_t r, const Part<T>& part, const Grad& g, const int* col, const float* term) {
  constexpr int N = Vec<T>::N;
  typedef typename std::conditional<sizeof(T) == 2, raw2, raw4>::type rawu;
  const int tid = threadIdx.x;
  const Line<T>& l = part.l;
  T* out = const_cast<T*>(l.row);
  const T* row = static_cast<const T*>(p.x) + r * p.xs;
  const T* base = row - l.pad;
  for (int vb = part.from; vb < part.hi && part.lo < part.hi; vb += NT * kUnroll) {
    raw q[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const rawu* at = reinterpret_cast<const rawu*>(base + (int64_t)min(max(vb + i * NT + tid, part.lo), part.hi - 1) * N);
      q[i] = FAR ? __builtin_nontemporal_load(at) : *at;
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int v = vb + i * NT + tid;
      float x[N];
      unpack<T>(q[i], x);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = grad_of<B>(g, exponent(x[e], g.m, p.c));
      pack<T>(x, q[i]);
      if (v >= part.lo && v < part.hi) store<FAR>(reinterpret_cast<raw*>(out - l.pad) + v, q[i]);
    }
  }
  if (tid < part.edges) {
    const int j = l.edge(tid);
    out[j] = (T)grad_of<B>(g, exponent((float)row[j], g.m, p.c));
  }
  // the columns with terms are written again, behind the barrier
  __syncthreads();
  for (int t = tid; t < g.n; t += NT) {
    const int j = col[t];
    if (j < 0 || !part.has(j)) continue;
    // those of the same column in their order, four a step (4096 x 4000 bf16 with 128
    // entries 40 us one by one, 31 so; a pass of 1229 x 128100 with 64 169.7 and 167.2)
    float sum = 0.f;
    bool first = true;
    for (int o = 0; o < g.n; o += 4) {
      const int4 c = *reinterpret_cast<const int4*>(col + o);
      const float4 w = *reinterpret_cast<const float4*>(term + o);
      const int cs[4] = {c.x, c.y, c.z, c.w};
      const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool same = cs[i] == j;
        sum += same ? ws[i] : 0.f;
        first = first && !(same && o + i < t);
      }
    }
    if (first) out[j] = (T)(grad_of<B>(g, exponent((float)row[j], g.m, p.c)) + sum);
  }
}

// A row that is left out, past the caches too: the loss of 4096 x 128100 of which 85%
// are left out 285 us through them, 240 past them.
template <typename T, int NT, bool FAR>
DSA_DEV void write_zeros(const Part<T>& part) {
  T* out = const_cast<T*>(part.l.row);
  for (int v = part.from + threadIdx.x; v < part.hi; v += NT)
    if (v >= part.lo) store<FAR>(reinterpret_cast<raw*>(out - part.l.pad) + v, raw{0u, 0u, 0u, 0u});
  if ((int)threadIdx.x < part.edges) out[part.l.edge(threadIdx.x)] = (T)0.f;
}

template <typename T, int NT, bool B, bool FAR>
__global__ __launch_bounds__(NT) void logprobs_bwd_kernel(VocabRows p) {
  __shared__ __align__(16) int col[kMost + 4];
  __shared__ __align__(16) float term[kMost + 4];
  const int tid = threadIdx.x;
  const int64_t r = p.row0 + blockIdx.x / (uint32_t)p.parts;
  const Part<T> part(p, r, blockIdx.x % (uint32_t)p.parts);
  const int64_t id = p.ids ? load_id(p.ids, p.ids64, r) : 0;
  if (p.ids && id == p.ignore) {
    write_zeros<T, NT, FAR>(part);
    return;
  }
  const float4 st = p.stats[r];
  const float g = p.dlp ? p.dlp[r * p.dlp_s] : 0.f;
  const float gh = B ? p.dent[r * p.dent_s] : 0.f;
  float a = -g - gh * st.z;
  if (p.dlse) a += p.dlse[r * p.dlse_s];
  const int k = p.dtop ? p.top : 0;
  if (p.dtop) {
    const int lane = tid & 63;
    float sum = 0.f;
    for (int t = lane; t < k; t += 64) sum += p.dtop[r * k + t];
    a -= hid::lanes_sum<64>(sum);
    for (int t = tid; t < k; t += NT) {
      const int64_t j = p.top_ids[r * k + t];
      col[1 + t] = j >= 0 && j < p.V ? (int)j : -1;
      term[1 + t] = p.dtop[r * k + t] * p.inv_t;
    }
  }
  const bool in = p.dlp && id >= 0 && id < p.V;
  if (tid == 0) col[0] = in ? (int)id : -1, term[0] = g * p.inv_t;
  if (tid < 3) col[1 + k + tid] = -1;  // up to a multiple of 4
  Grad d;
  d.m = st.x, d.n = 1 + k;
  // p_j (a + b ln p_j) / T with ln p_j = ln 2 t - ln s, p_j = e / s
  a = (a + gh * st.y) * p.inv_t * st.w;
  if (p.dlp && !in && g != 0.f) a = __builtin_nanf("");
  // a row without probabilities (1 / s infinite or NaN): e = 0 would hide it
  if (B && !(st.w <= -kLowest)) a = __builtin_nanf("");
  d.a = a;
  d.b = -gh * p.inv_t * kLn2 * st.w;
  write_grad<T, NT, B, FAR>(p, r, part, d, col, term);
}

template <typename T, int NT, bool FAR>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(VocabRows p) {
  __shared__ __align__(16) int col[kMost];
  __shared__ __align__(16) float term[kMost];
  const int64_t r = p.row0 + blockIdx.x / (uint32_t)p.parts;
  const Part<T> part(p, r, blockIdx.x % (uint32_t)p.parts);
  const Entries e = entries_of(p, r);
  if (!e.any) {
    write_zeros<T, NT, FAR>(part);
    return;
  }
  const float4 st = p.stats[r];
  const float g = p.dlp[r * p.dlp_s] * p.t;
  Grad d;
  d.m = st.x, d.b = 0.f, d.n = p.K;
  d.a = e.bad && g != 0.f ? __builtin_nanf("") : g * e.total * st.w;
  if (threadIdx.x < 64) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = threadIdx.x + 64 * i;
      col[k] = k < p.K && e.id[i] < p.V ? (int)e.id[i] : -1, term[k] = -g * e.q[i];
    }
  }
  write_grad<T, NT, false, FAR>(p, r, part, d, col, term);
}

}  // namespace voc
}  // namespace dsa
