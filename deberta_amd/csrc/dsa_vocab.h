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
// value (a mask that leaves nothing) would overflow; so it has p = 1 / V.
//
// The k largest come out of the same pass.  It keeps the maximum of each
// segment of 64 columns.  The k segments whose maxima are largest (equal ones:
// the first) hold the k largest values: each of these k maxima is one of them
// or below them, so a value outside these segments, at most its own segment's
// maximum, has k larger ones before it.  Only those are read again (k 128-byte
// lines of bf16), and the k largest of them are chosen.  Nothing depends on
// the data but which lines these are.
#pragma once

#include <type_traits>

#include "dsa_lanes.h"

namespace dsa {
namespace voc {

constexpr int kSeg = 64;      // columns of a segment
constexpr int kBins = 1024;   // of a selection's histogram
constexpr int kMost = 128;    // entries of a row
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

// The larger of two or three, a NaN giving way.  The instruction by itself:
// fmaxf of values that come from memory quiets each one first, an instruction
// a value.
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
template <int N>
DSA_DEV float max_of(const float* v) {
  static_assert(N % 2 == 0, "");
  float m = max2(v[0], v[1]);
#pragma unroll
  for (int i = 2; i < N; i += 2) m = max3(m, v[i], v[i + 1]);
  return m;
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

struct Run {
  float m, s, u;
};
DSA_DEV Run run_none() { return Run{kLowest, 0.f, 0.f}; }

// the sums as of a larger maximum
template <bool ENT>
DSA_DEV void raise(Run& r, float m, float c) {
  const float d = fmaxf((r.m - m) * c, kFar), f = exp2_(d);
  if (ENT) r.u = f * fmaf(d, r.s, r.u);  // in units of ln 2
  r.s *= f;
  r.m = m;
}
template <int E, bool ENT>
DSA_DEV void add(Run& r, const float* x, float most, float c) {
  if (most > r.m) raise<ENT>(r, most, c);
  float s[2] = {0.f, 0.f}, u[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = (x[e] - r.m) * c, p = exp2_(t);
    s[e & 1] += p;
    if (ENT) u[e & 1] = fmaf(p, fmaxf(t, kFar), u[e & 1]);  // 0 where t is -inf
  }
  r.s += s[0] + s[1];
  if (ENT) r.u += u[0] + u[1];
}

DSA_DEV float wave_max_f(float x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x = max2(x, __shfl_xor(x, o));
  return x;
}
// The block's sums out of its threads', in every thread; red: 3 words a wave.
template <int NT, bool ENT>
DSA_DEV Run block_run(Run r, float c, float* red) {
  constexpr int W = NT / 64;
  const float m = wave_max_f(r.m);
  raise<ENT>(r, m, c);
  r.s = hid::lanes_sum<64>(r.s);
  if (ENT) r.u = hid::lanes_sum<64>(r.u);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) {
      float* w = red + 3 * (threadIdx.x >> 6);
      w[0] = r.m, w[1] = r.s, w[2] = r.u;
    }
    __syncthreads();
    float most = kLowest;
#pragma unroll
    for (int i = 0; i < W; ++i) most = max2(most, red[3 * i]);
    Run all{most, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Run w{red[3 * i], red[3 * i + 1], red[3 * i + 2]};
      raise<ENT>(w, most, c);
      all.s += w.s, all.u += w.u;
    }
    r = all;
  }
  return r;
}

// ---------------------------------------------------------------------------
// a row in 16-byte accesses: it starts `pad` values behind a 16-byte border,
// and positions count from there.  Vectors v0 .. v1 - 1 lie in the row whole;
// the values before and behind them are taken one by one, a lane each.
template <typename T>
struct Line {
  static constexpr int N = Vec<T>::N;
  const T* row;
  const T* base;  // of position 0
  int pad, v0, v1, head, edges, tail0;
  DSA_DEV Line(const void* x, int64_t stride, int64_t r, int V) {
    row = static_cast<const T*>(x) + r * stride;
    pad = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(T);
    base = row - pad;
    v0 = pad ? 1 : 0;
    v1 = max((int)(((int64_t)pad + V) / N), v0);
    head = min(V, v0 * N - pad);
    tail0 = min(V, v1 * N - pad);  // the row's first value behind the vectors
    edges = head + (V - tail0);
  }
  DSA_DEV int edge(int i) const { return i < head ? i : tail0 + (i - head); }
  DSA_DEV raw load(int v) const { return reinterpret_cast<const raw*>(base)[v]; }
};

// The sums of a thread over its share of the row; with SEG the segments'
// maxima into keys (all of them: the caller has cleared them, and waits).
template <typename T, int NT, bool ENT, bool SEG>
DSA_DEV Run stream(const Line<T>& l, float c, uint32_t* keys) {
  constexpr int N = Vec<T>::N, E = kUnroll * N;
  const int tid = threadIdx.x;
  Run r = run_none();
  const int end = l.v1 > l.v0 ? l.v1 : 0;
  for (int vb = 0; vb < end; vb += NT * kUnroll) {
    raw q[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) q[i] = l.load(min(max(vb + i * NT + tid, l.v0), l.v1 - 1));
    if (vb < l.v0 || vb + NT * kUnroll > l.v1) {
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int v = vb + i * NT + tid;
        if (v < l.v0 || v >= l.v1) q[i] = raw_none<T>();
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
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        float g = most[i];  // over the 64 / N lanes of the segment
        g = max2(g, hid::dpp<0xB1>(g));
        g = max2(g, hid::dpp<0x4E>(g));
        g = max2(g, hid::dpp<0x141>(g));
        if (N == 4) g = max2(g, hid::dpp<0x140>(g));
        const int v = vb + i * NT + tid;
        if (tid % (kSeg / N) == 0 && v < l.v1) keys[v / (kSeg / N)] = key_of<T>(g);
      }
    }
  }
  if (SEG) __syncthreads();
  if (tid < l.edges) {
    const int j = l.edge(tid);
    const float x = (float)l.row[j];
    add<1, ENT>(r, &x, max2(x, kLowest), c);
    if (SEG) atomicMax(&keys[(l.pad + j) / kSeg], key_of<T>(x));
  }
  return r;
}

// ---------------------------------------------------------------------------
// the largest

struct Shared {
  uint32_t* keys;
  uint32_t* hist;  // kBins
  int* list;       // kMost
  uint32_t* picked;  // kMost
  uint32_t* word;  // 24
};
constexpr int kSharedWords = kBins + 2 * kMost + 24;
DSA_DEV Shared shared_at(uint32_t* lds, int keys) {
  Shared s;
  s.keys = lds;
  s.hist = lds + keys;
  s.list = reinterpret_cast<int*>(s.hist + kBins);
  s.picked = s.hist + kBins + kMost;
  s.word = s.hist + kBins + 2 * kMost;
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

// The places of the `need` largest of keys[0 .. n), equal ones by their place,
// into sh.list in the order of their places (0 < need <= n, need <= kMost).
//
// Keys are counted into bins of equal width between the least and the largest,
// the bin that holds the last one wanted is cut into bins again, and so on until
// all of a bin are wanted or its keys are equal: one round where the keys span
// at most 1024, at most four (10 bits a round).
template <int NT>
DSA_DEV void choose(const Shared& sh, int n, int need) {
  constexpr int W = NT / 64, PER = kBins / NT;
  const int tid = threadIdx.x;
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = tid; i < n; i += NT) lo = min(lo, sh.keys[i]), hi = max(hi, sh.keys[i]);
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
      const uint32_t k = sh.keys[i];
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
    const uint32_t k = sh.keys[i];
    counts += k > lo ? 1u : k == lo ? 0x10000u : 0u;
  }
  const uint32_t before = block_before<NT>(counts, sh.word);
  uint32_t over = before & 0xffffu, at = before >> 16;
  for (int i = first; i < last; ++i) {
    const uint32_t k = sh.keys[i];
    if (k > lo || (k == lo && at < equal)) sh.list[over + min(at, equal)] = i;
    over += k > lo, at += k == lo;
  }
  __syncthreads();
}

// The row's largest, from its segments' maxima in sh.keys.
template <typename T, int NT>
DSA_DEV void write_top(const Line<T>& l, const VocabRows& p, int64_t r, const Shared& sh, float m, float ln_s) {
  const int tid = threadIdx.x, k = p.top;
  const int segs = (l.pad + p.V - 1) / kSeg + 1, found = min(k, segs);
  choose<NT>(sh, segs, found);
  if (tid < found) sh.picked[tid] = (uint32_t)sh.list[tid];
  __syncthreads();
  for (int i = tid; i < found * kSeg; i += NT) {
    const int j = (int)sh.picked[i / kSeg] * kSeg + i % kSeg - l.pad;
    sh.keys[i] = j >= 0 && j < p.V ? key_of<T>((float)l.row[j]) : 0u;
  }
  __syncthreads();
  choose<NT>(sh, found * kSeg, k);
  for (int t = tid; t < k; t += NT) {
    const int i = sh.list[t];
    const uint32_t mine = sh.keys[i];
    int rank = 0;
    for (int o = 0; o < k; ++o) {
      const uint32_t other = sh.keys[sh.list[o]];
      rank += other > mine || (other == mine && o < t);
    }
    const int j = (int)sh.picked[i / kSeg] * kSeg + i % kSeg - l.pad;
    p.top_ids[r * k + rank] = j;
    p.top_lp[r * k + rank] = (of_key<T>(mine) - m) * p.inv_t - ln_s;
  }
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

// One thread: the row's results.
template <typename T>
DSA_DEV void write_row(const Line<T>& l, const VocabRows& p, int64_t r, const Run& all, float ln_s, int64_t id) {
  const float ent = ln_s - kLn2 * all.u / all.s;
  if (p.lp)
    p.lp[r] = id >= 0 && id < p.V ? ((float)l.row[id] - all.m) * p.inv_t - ln_s : __builtin_nanf("");
  if (p.ent) p.ent[r] = ent;
  if (p.lse) p.lse[r] = fmaf(all.m, p.inv_t, ln_s);
  if (p.stats) p.stats[r] = float4{all.m, ln_s, ent, 1.f / all.s};
}

template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_fwd_kernel(VocabRows p) {
  extern __shared__ uint32_t lds[];
  __shared__ float red[3 * (NT / 64)];
  const int64_t r = p.row0 + blockIdx.x;
  const int64_t id = p.ids ? load_id(p.ids, p.ids64, r) : 0;
  if (p.ids && id == p.ignore) {
    write_none<NT>(p, r);
    return;
  }
  const Line<T> l(p.x, p.xs, r, p.V);
  if (TOP) {
    for (int i = threadIdx.x; i < p.keys; i += NT) lds[i] = 0;
    __syncthreads();
  }
  const Run all = block_run<NT, true>(stream<T, NT, true, TOP>(l, p.c, lds), p.c, red);
  const float ln_s = logf(all.s);
  if (threadIdx.x == 0) write_row(l, p, r, all, ln_s, id);
  if (TOP) {
    __syncthreads();
    write_top<T, NT>(l, p, r, shared_at(lds, p.keys), all.m, ln_s);
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

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_fwd_kernel(VocabRows p) {
  __shared__ float red[3 * (NT / 64)];
  const int64_t r = p.row0 + blockIdx.x;
  const Entries e = entries_of(p, r);  // by every wave
  if (!e.any) {
    if (threadIdx.x == 0) {
      p.loss[r] = 0.f;
      if (p.stats) p.stats[r] = float4{0.f, 0.f, 0.f, 0.f};
    }
    return;
  }
  const Line<T> l(p.x, p.xs, r, p.V);
  const Run all = block_run<NT, false>(stream<T, NT, false, false>(l, p.c, nullptr), p.c, red);
  const float ln_s = logf(all.s);
  if (threadIdx.x >= 64) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (e.id[i] < 0 || e.id[i] >= p.V || e.q[i] == 0.f) continue;
    const float log_p = ((float)l.row[e.id[i]] - all.m) * p.inv_t - ln_s;
    sum += e.q[i] * (e.log_q[i] - log_p);
  }
  sum = hid::lanes_sum<64>(sum);
  if (threadIdx.x == 0) {
    p.loss[r] = e.bad ? __builtin_nanf("") : p.t * p.t * sum;
    if (p.stats) p.stats[r] = float4{all.m, ln_s, 0.f, 1.f / all.s};
  }
}

// ---------------------------------------------------------------------------
// backward: e = exp2((x - m) c), dx = e (a + b (x - m) c) and, at a few
// columns, a term more

// the row's constants, and the columns with a term of their own in LDS
struct Grad {
  float m, a, b;
  int n;
};
template <bool B>
DSA_DEV float grad_of(const Grad& g, float c, float x) {
  const float t = (x - g.m) * c, e = exp2_(t);
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

// A row of the gradient in 16-byte stores; the logits' row may lie otherwise
// to 16-byte borders.
template <typename T, int NT, bool B>
DSA_DEV void write_grad(const VocabRows& p, int64_t r, const Grad& g, const int* col, const float* term) {
  constexpr int N = Vec<T>::N;
  typedef typename std::conditional<sizeof(T) == 2, raw2, raw4>::type rawu;
  const int tid = threadIdx.x;
  const Line<T> l(p.dx, p.dxs, r, p.V);
  T* out = const_cast<T*>(l.row);
  const T* row = static_cast<const T*>(p.x) + r * p.xs;
  const T* base = row - l.pad;
  for (int vb = l.v0; vb < l.v1; vb += NT * kUnroll) {
    raw q[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      q[i] = *reinterpret_cast<const rawu*>(base + (int64_t)min(vb + i * NT + tid, l.v1 - 1) * N);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int v = vb + i * NT + tid;
      float x[N];
      unpack<T>(q[i], x);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = grad_of<B>(g, p.c, x[e]);
      pack<T>(x, q[i]);
      if (v < l.v1) reinterpret_cast<raw*>(out - l.pad)[v] = q[i];
    }
  }
  if (tid < l.edges) {
    const int j = l.edge(tid);
    out[j] = (T)grad_of<B>(g, p.c, (float)row[j]);
  }
  // the columns with terms are written again, behind the barrier
  __syncthreads();
  for (int t = tid; t < g.n; t += NT) {
    const int j = col[t];
    if (j < 0) continue;
    float sum = 0.f;
    bool first = true;
    for (int o = 0; o < g.n; ++o) {
      const bool same = col[o] == j;
      if (same) sum += term[o];
      if (same && o < t) first = false;
    }
    if (first) out[j] = (T)(grad_of<B>(g, p.c, (float)row[j]) + sum);
  }
}

template <typename T, int NT>
DSA_DEV void write_zeros(const VocabRows& p, int64_t r) {
  const Line<T> l(p.dx, p.dxs, r, p.V);
  T* out = const_cast<T*>(l.row);
  for (int v = l.v0 + threadIdx.x; v < l.v1; v += NT) reinterpret_cast<raw*>(out - l.pad)[v] = raw{0u, 0u, 0u, 0u};
  if ((int)threadIdx.x < l.edges) out[l.edge(threadIdx.x)] = (T)0.f;
}

template <typename T, int NT, bool B>
__global__ __launch_bounds__(NT) void logprobs_bwd_kernel(VocabRows p) {
  __shared__ int col[kMost + 1];
  __shared__ float term[kMost + 1];
  const int tid = threadIdx.x;
  const int64_t r = p.row0 + blockIdx.x;
  const int64_t id = p.ids ? load_id(p.ids, p.ids64, r) : 0;
  if (p.ids && id == p.ignore) {
    write_zeros<T, NT>(p, r);
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
  Grad d;
  d.m = st.x, d.n = 1 + k;
  // p_j (a + b ln p_j) / T with ln p_j = ln 2 t - ln s, p_j = e / s
  a = (a + gh * st.y) * p.inv_t * st.w;
  if (p.dlp && !in && g != 0.f) a = __builtin_nanf("");
  // a row without probabilities (1 / s infinite or NaN): e = 0 would hide it
  if (B && !(st.w <= -kLowest)) a = __builtin_nanf("");
  d.a = a;
  d.b = -gh * p.inv_t * kLn2 * st.w;
  write_grad<T, NT, B>(p, r, d, col, term);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(VocabRows p) {
  __shared__ int col[kMost];
  __shared__ float term[kMost];
  const int64_t r = p.row0 + blockIdx.x;
  const Entries e = entries_of(p, r);
  if (!e.any) {
    write_zeros<T, NT>(p, r);
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
      if (k < p.K) col[k] = e.id[i] < p.V ? (int)e.id[i] : -1, term[k] = -g * e.q[i];
    }
  }
  write_grad<T, NT, false>(p, r, d, col, term);
}

}  // namespace voc
}  // namespace dsa
