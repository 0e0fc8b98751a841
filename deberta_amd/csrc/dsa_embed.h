// dsa_embed.h — the token embedding (gfx950): out[n] = scale W[ids[n]], and
// its gradient dW[v] = scale * sum of dout[n] over the positions n that hold
// token v, by sorted tokens.
//
// The gradient:
//   1. the positions are sorted by token, stably, with a radix sort whose
//      digits cover the vocabulary's bits (two digits of nine bits up to
//      262143 tokens).  The padding token and ids outside the table take the
//      key V, behind every token;
//   2. while it runs, other workgroups of the same launches clear dW (the
//      largest part of the traffic where the batch is smaller than the
//      vocabulary);
//   3. the sorted positions are cut in chunks of equal length, one wave a
//      chunk and 512 columns, whatever the tokens' frequencies are: a wave
//      sums its rows of dout token by token, in fp32, in the order of the
//      positions.  A token that lies in one chunk is written at once, one
//      that crosses a border leaves a partial sum for each chunk;
//   4. the partial sums of a token are joined in the order of the chunks.
// No float is added atomically: equal inputs give equal bits.
#pragma once

#include "dsa_hidden.h"

namespace dsa {
namespace hid {

constexpr int EMB_T = 256;      // chunks (threads) a lookup block takes at most
constexpr int EMB_U = 4;        // rows whose loads are issued together
constexpr int SORT_T = 512;     // threads of a sort workgroup
constexpr int SORT_R = 8;       // keys a thread holds
constexpr int SORT_TILE = SORT_T * SORT_R;
constexpr int SORT_BITS = 9;    // a digit's bits at most: SORT_T >= 2^SORT_BITS
constexpr int SORT_D = 1 << SORT_BITS;
constexpr int SORT_W = SORT_T / 64;
constexpr int FILL_IT = 8;      // 16-byte stores a thread of a fill workgroup makes

struct EmbedRows {
  const void *ids, *w;
  void* y;
  int64_t V, ws, ys;
  uint32_t N;
  int C, ids64;
  int cw, subs, rows;
  float scale;
};

DSA_DEV int64_t ld_id(const void* ids, int64_t i, int ids64) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// Threads as in drop_fwd_kernel.  An id outside [0, V) reads nothing and
// gives a row of NaN.
template <typename TW, typename TY, bool TAIL>
__global__ __launch_bounds__(EMB_T) void embed_fwd_kernel(EmbedRows p) {
  const int sub = threadIdx.x / p.cw, chunk = blockIdx.y * EMB_T + (int)threadIdx.x - sub * p.cw;
  const int c = 8 * chunk, n = p.C - c;
  if (sub >= p.subs || n <= 0) return;
  const int64_t extent = (p.V - 1) * p.ws + p.C;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows * p.subs + sub;
  for (int i = 0; i < p.rows; i += EMB_U) {
    int64_t id[EMB_U];
    raw8<TW> w[EMB_U];
#pragma unroll
    for (int u = 0; u < EMB_U; ++u)
      id[u] = ld_id(p.ids, min(r0 + (int64_t)(i + u) * p.subs, (int64_t)p.N - 1), p.ids64);
#pragma unroll
    for (int u = 0; u < EMB_U; ++u) {
      const bool ok = (uint64_t)id[u] < (uint64_t)p.V;
      w[u] = ld8<TW, TAIL>(p.w, ok ? id[u] * p.ws + c : c, extent, ok ? n : 0);
    }
#pragma unroll
    for (int u = 0; u < EMB_U; ++u) {
      const int64_t r = r0 + (int64_t)(i + u) * p.subs;
      if (r >= p.N) return;
      float v[8];
      cvt8<TW, TAIL>(w[u], 8, v);
      const float s = (uint64_t)id[u] < (uint64_t)p.V ? p.scale : __builtin_nanf("");
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= s;
      st8<TY, TAIL>(p.y, r * p.ys + c, n, v);
    }
  }
}

// ---------------------------------------------------------------------------
// the sort

struct SortParams {
  const void* ids;
  int64_t V, padding;     // padding < 0: none
  const uint32_t *kin, *pin;  // sorted so far (null: from ids)
  uint32_t *kout, *pout;
  uint32_t* counts;       // [tiles][SORT_D]
  char* fill;             // the part of dW that this launch clears
  int64_t fill_bytes;
  uint32_t N;
  int ids64, tiles, per_tile;  // per_tile: runs of SORT_TILE keys a workgroup takes
  int shift, bits;        // the digit: (key >> shift) & ((1 << bits) - 1)
  int passes;             // embed_sort_one_kernel: digits, from the lowest
};

DSA_DEV uint32_t token_key(const SortParams& s, uint32_t i) {
  const int64_t id = ld_id(s.ids, i, s.ids64);
  return (uint64_t)id < (uint64_t)s.V && id != s.padding ? (uint32_t)id : (uint32_t)s.V;
}

// workgroup `b` of the launch's fill workgroups
DSA_DEV void fill_zero(const SortParams& s, int64_t b) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const int64_t n16 = s.fill_bytes / 16, at = b * SORT_T * FILL_IT + threadIdx.x;
#pragma unroll
  for (int i = 0; i < FILL_IT; ++i) {
    const int64_t k = at + (int64_t)i * SORT_T;
    if (k < n16) reinterpret_cast<u4*>(s.fill)[k] = u4{0u, 0u, 0u, 0u};
  }
  if (b == 0 && threadIdx.x == 0)
    for (int64_t k = 16 * n16; k < s.fill_bytes; k += 2) *reinterpret_cast<uint16_t*>(s.fill + k) = 0;
}

struct SortLds {
  uint32_t cnt[SORT_W][SORT_D];
  uint32_t wave[SORT_W];
};

// For the thread's keys (wave w's are the tile's w-th run of 64 * SORT_R, key
// j of lane l at 64 j + l of it; valid where `ok`): how many keys of the same
// digit lie before it in its wave, and the wave's counts in l.cnt[w].
template <int R>
DSA_DEV void wave_ranks(SortLds& l, const uint32_t (&digit)[R], const bool (&ok)[R], int bits, uint32_t (&rank)[R]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // volatile: every access is made, in this order
  typedef __attribute__((address_space(3))) volatile uint32_t lds_u32;
  lds_u32* cnt = (lds_u32*)l.cnt[w];
  for (int d = lane; d < SORT_D; d += 64) cnt[d] = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    uint64_t peers = __ballot(ok[j]);
    for (int b = 0; b < bits; ++b) {
      const bool one = (digit[j] >> b) & 1;
      const uint64_t m = __ballot(one);
      peers &= one ? m : ~m;
    }
    const uint32_t before = __builtin_amdgcn_mbcnt_hi((uint32_t)(peers >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)peers, 0));
    // the wave's LDS accesses complete in their order: every lane reads
    // before the first of a digit's lanes writes
    const uint32_t base = ok[j] ? cnt[digit[j]] : 0;
    rank[j] = base + before;
    if (ok[j] && before == 0) cnt[digit[j]] = base + (uint32_t)__popcll(peers);
  }
}

// Thread d's digit count `mine` -> the sum of the counts of lower digits.
DSA_DEV uint32_t digit_scan(SortLds& l, uint32_t mine) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t s = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_up((int)s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 63) l.wave[w] = s;
  __syncthreads();
  for (int i = 0; i < w; ++i) s += l.wave[i];
  return s - mine;
}

// counts[tile][digit]: the tile's keys of each digit
static __global__ __launch_bounds__(SORT_T) void embed_count_kernel(SortParams s) {
  if ((int)blockIdx.x >= s.tiles) {
    fill_zero(s, (int)blockIdx.x - s.tiles);
    return;
  }
  __shared__ uint32_t cnt[SORT_D];
  for (int d = threadIdx.x; d < SORT_D; d += SORT_T) cnt[d] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * s.per_tile * SORT_TILE;
  const int64_t n1 = min(n0 + (int64_t)s.per_tile * SORT_TILE, (int64_t)s.N);
  const uint32_t mask = (1u << s.bits) - 1;
  for (int64_t i = n0 + threadIdx.x; i < n1; i += SORT_T) {
    const uint32_t key = s.kin ? s.kin[i] : token_key(s, (uint32_t)i);
    atomicAdd(&cnt[(key >> s.shift) & mask], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_D; d += SORT_T) s.counts[(int64_t)blockIdx.x * SORT_D + d] = cnt[d];
}

// Moves the tile's keys and positions to their places by one digit.
static __global__ __launch_bounds__(SORT_T) void embed_scatter_kernel(SortParams s) {
  if ((int)blockIdx.x >= s.tiles) {
    fill_zero(s, (int)blockIdx.x - s.tiles);
    return;
  }
  __shared__ SortLds l;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = threadIdx.x;
  const uint32_t mask = (1u << s.bits) - 1;
  // thread d: where digit d of this tile begins in the sorted order
  uint32_t before = 0, total = 0;
  for (int i = 0; i < s.tiles; ++i) {
    const uint32_t c = s.counts[(int64_t)i * SORT_D + t];
    total += c;
    before += i < (int)blockIdx.x ? c : 0;
  }
  uint32_t begin = digit_scan(l, total) + before;
  for (int run = 0; run < s.per_tile; ++run) {
    const int64_t n0 = ((int64_t)blockIdx.x * s.per_tile + run) * SORT_TILE + w * 64 * SORT_R + lane;
    uint32_t key[SORT_R], pos[SORT_R], digit[SORT_R], rank[SORT_R];
    bool ok[SORT_R];
#pragma unroll
    for (int j = 0; j < SORT_R; ++j) {
      const int64_t i = n0 + 64 * j;
      ok[j] = i < s.N;
      key[j] = !ok[j] ? 0 : s.kin ? s.kin[i] : token_key(s, (uint32_t)i);
      pos[j] = !ok[j] ? 0 : s.pin ? s.pin[i] : (uint32_t)i;
      digit[j] = (key[j] >> s.shift) & mask;
    }
    wave_ranks(l, digit, ok, s.bits, rank);
    __syncthreads();
    // thread d: the waves' counts of digit d become their first places
    uint32_t at = begin;
#pragma unroll
    for (int i = 0; i < SORT_W; ++i) {
      const uint32_t c = l.cnt[i][t];
      l.cnt[i][t] = at;
      at += c;
    }
    begin = at;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_R; ++j) {
      if (ok[j]) {
        const uint32_t to = l.cnt[w][digit[j]] + rank[j];
        s.kout[to] = key[j];
        s.pout[to] = pos[j];
      }
    }
    __syncthreads();
  }
}

// At most SORT_TILE positions: one workgroup sorts them by every digit in LDS.
static __global__ __launch_bounds__(SORT_T) void embed_sort_one_kernel(SortParams s) {
  if (blockIdx.x > 0) {
    fill_zero(s, (int64_t)blockIdx.x - 1);
    return;
  }
  __shared__ SortLds l;
  __shared__ uint32_t ks[SORT_TILE], ps[SORT_TILE];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = threadIdx.x;
  const int n0 = w * 64 * SORT_R + lane;
  const uint32_t mask = (1u << s.bits) - 1;
  uint32_t key[SORT_R], pos[SORT_R], digit[SORT_R], rank[SORT_R];
  bool ok[SORT_R];
#pragma unroll
  for (int j = 0; j < SORT_R; ++j) {
    const uint32_t i = (uint32_t)(n0 + 64 * j);
    ok[j] = i < s.N;
    key[j] = ok[j] ? token_key(s, i) : 0;
    pos[j] = i;
  }
  for (int pass = 0; pass < s.passes; ++pass) {
#pragma unroll
    for (int j = 0; j < SORT_R; ++j) digit[j] = (key[j] >> (pass * s.bits)) & mask;
    wave_ranks(l, digit, ok, s.bits, rank);
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int i = 0; i < SORT_W; ++i) total += l.cnt[i][t];
    uint32_t at = digit_scan(l, total);
#pragma unroll
    for (int i = 0; i < SORT_W; ++i) {
      const uint32_t c = l.cnt[i][t];
      l.cnt[i][t] = at;
      at += c;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_R; ++j) {
      if (ok[j]) {
        const uint32_t to = l.cnt[w][digit[j]] + rank[j];
        ks[to] = key[j];
        ps[to] = pos[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_R; ++j) {
      if (ok[j]) {
        key[j] = ks[n0 + 64 * j];
        pos[j] = ps[n0 + 64 * j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < SORT_R; ++j) {
    if (ok[j]) {
      s.kout[n0 + 64 * j] = key[j];
      s.pout[n0 + 64 * j] = pos[j];
    }
  }
}

// ---------------------------------------------------------------------------
// the sums

struct EmbedSums {
  const uint32_t *keys, *pos;  // sorted
  const void* dy;
  void* dw;
  float* part;  // [chunks][2][C]: the chunk's first and last token where they cross its borders
  int64_t dys, dye, dws;
  uint32_t V, N, chunks;
  int C, slabs, K;  // slabs of 512 columns; positions a chunk (at most 64)
  float scale;
};

template <typename TDY, typename TW, bool TAIL>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedSums p) {
  const int lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ch = item / (uint32_t)p.slabs;
  if (ch >= p.chunks) return;
  const int c = (int)(item - ch * p.slabs) * 512 + lane * 8, n = p.C - c;
  const uint32_t i0 = ch * (uint32_t)p.K, i1 = min(i0 + (uint32_t)p.K, p.N);
  const uint32_t i = i0 + lane;
  const uint32_t key = i < i1 ? p.keys[i] : p.V, pos = i < i1 ? p.pos[i] : 0;
  const uint32_t next = i < i1 && i + 1 < p.N ? p.keys[i + 1] : p.V;
  const int m = __popcll(__ballot(key < p.V));  // the chunk's tokens: the keys V come last
  if (m == 0) return;
  const uint64_t ends = __ballot(lane < m && key != next);
  // the chunk's first token began before it
  bool carried = i0 > 0 && p.keys[i0 - 1] == (uint32_t)__builtin_amdgcn_readlane(key, 0);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  constexpr int U = 8;
  for (int j0 = 0; j0 < m; j0 += U) {
    raw8<TDY> dy[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = (uint32_t)__builtin_amdgcn_readlane(pos, min(j0 + u, m - 1));
      dy[u] = ld8<TDY, TAIL>(p.dy, (int64_t)r * p.dys + c, p.dye, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u;
      if (j < m) {
        float v[8];
        cvt8<TDY, TAIL>(dy[u], n, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += v[e];
        const bool end = (ends >> j) & 1;
        if (end || j == m - 1) {
          if (carried || !end) {
            float* out = p.part + ((int64_t)ch * 2 + (carried ? 0 : 1)) * p.C;
            st8<float, TAIL>(out, c, n, acc);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = acc[e] * p.scale;
            st8<TW, TAIL>(p.dw, (int64_t)(uint32_t)__builtin_amdgcn_readlane(key, j) * p.dws + c, n, v);
          }
          carried = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// Block (chunk, slab): the token that begins in the chunk and goes on past
// its end, from the chunk's own partial sum and those of the chunks behind.
template <typename TW, bool TAIL>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedSums p) {
  __shared__ float red[3][64][8];
  const int lane = threadIdx.x & 63, q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ch = blockIdx.x / (uint32_t)p.slabs;
  const int c = (int)(blockIdx.x - ch * p.slabs) * 512 + lane * 8, n = p.C - c;
  const uint64_t i0 = (uint64_t)ch * p.K, i1 = i0 + p.K;
  if (i1 >= p.N) return;
  const uint32_t key = p.keys[i1];
  if (key >= p.V || p.keys[i1 - 1] != key) return;
  if (i0 > 0 && p.keys[i0 - 1] == key) return;  // it began before
  // the chunks behind that begin with the token: the keys are sorted
  uint32_t last = ch;
  for (;;) {
    const uint64_t at = ((uint64_t)last + 1 + lane) * p.K;
    const int more = __popcll(__ballot(at < p.N && p.keys[at < p.N ? at : 0] == key));
    last += more;
    if (more < 64) break;
  }
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t extent = (int64_t)p.chunks * 2 * p.C;
  constexpr int U = 4;
  if (q == 0) cvt8<float, TAIL>(ld8<float, TAIL>(p.part, ((int64_t)ch * 2 + 1) * p.C + c, extent, n), n, acc);
  for (int64_t k0 = (int64_t)ch + 1 + q; k0 <= last; k0 += 4 * U) {
    raw8<float> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = ld8<float, TAIL>(p.part, min(k0 + 4 * u, (int64_t)last) * 2 * p.C + c, extent, n);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + 4 * u <= last) {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += e < n ? v[u][e] : 0.f;
      }
  }
  if (q > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red[q - 1][lane][e] = acc[e];
  }
  __syncthreads();
  if (q > 0) return;
#pragma unroll
  for (int v = 0; v < 3; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += red[v][lane][e];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= p.scale;
  st8<TW, TAIL>(p.dw, (int64_t)key * p.dws + c, n, acc);
}

}  // namespace hid
}  // namespace dsa
