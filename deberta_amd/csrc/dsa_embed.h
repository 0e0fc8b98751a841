// dsa_embed.h — the token embedding (gfx950): out[n] = scale W[ids[n]], and
// its gradient dW[v] = scale * sum of dout[n] over the positions n that hold
// token v, by sorted tokens.
//
// The gradient:
//   1. the positions are sorted by token, stably: up to RANK_N positions by
//      counting, for each, the positions before it (every pair is compared,
//      on all compute units, in one launch); more with a radix sort whose
//      digits cover the vocabulary's bits (two digits of nine bits up to
//      262143 tokens; two launches a digit).  The padding token and ids
//      outside the table take the key V, behind every token;
//   2. while it runs, other workgroups of the same launches clear dW (the
//      largest part of the traffic where the batch is smaller than the
//      vocabulary).  Of the radix sort's launches the first marks the tokens
//      that occur and the others clear the rows of those that do not, so that
//      no row is written twice; beside the counting sort every row is cleared;
//   3. the sorted positions are cut in chunks of equal length, one wave a
//      chunk and 512 columns, whatever the tokens' frequencies are: a wave
//      sums its rows of dout token by token, in fp32, in the order of the
//      positions.  A token that lies in one chunk is written at once, one
//      that crosses a border leaves a partial sum for each chunk;
//   4. the partial sums of a token are joined in the order of the chunks.
// No float is added atomically: equal inputs give equal bits.
//
// HBM bounds the large ones: 8192 positions x 768 fp32 in 128100 tokens take
// 12.7 us forward, then 62.6 for the places and the 394 MB of dW (6.3 TB/s),
// 12.2 for the sums and 4.9 to join them; 131072 x 1024 bf16 take 89, 61 (five
// launches), 65 and 8.  The chain of launches bounds small ones (2723 x 513:
// 26 us, of which the bytes need 12).
#pragma once

#include "dsa_hidden.h"

namespace dsa {
namespace hid {

// A lane's eight columns of what it would take from column c on: where they
// would pass the row's end, the row's last eight.  Two lanes then take the
// same columns and write the same values, and no width of eight or more needs
// a condition.  NARROW: rows of fewer than eight columns.
template <bool NARROW>
DSA_DEV int embed_col(int C, int c) { return NARROW ? c : min(c, C - 8); }

constexpr int EMB_T = 256;      // chunks (threads) a lookup block takes at most
constexpr int EMB_U = 4;        // rows whose loads are issued together
constexpr int SORT_T = 512;     // threads of a sort workgroup
constexpr int SORT_R = 8;       // keys a thread holds
constexpr int SORT_TILE = SORT_T * SORT_R;
constexpr int SORT_BITS = 9;    // a digit's bits at most: SORT_T >= 2^SORT_BITS
constexpr int SORT_D = 1 << SORT_BITS;
constexpr int SORT_W = SORT_T / 64;
constexpr int FILL_BYTES = 65536;  // of dW, about, a fill workgroup clears
// Positions the counting sort takes at most: as many as leave 19 bits of a word
// to the token.  It compares every pair and is still the faster one there; the
// two meet at about twice as many.  The gradient's kernels, counting / radix, us:
// 513 bf16 columns of 50021 tokens 21.7 / 43.2 for 2723 positions, 35 / 52 for
// 8192, 52 / 55 for 16384 (a build with 14 bits); 768 fp32 of 128100 81 / 95,
// 84 / 106, 108 / 114; 1024 bf16 of 128100 43 / 58, 51 / 72, 65 / 74.
constexpr int RANK_BITS = 13;
constexpr int RANK_N = 1 << RANK_BITS;

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
template <typename TW, typename TY, bool NARROW>
__global__ __launch_bounds__(EMB_T) void embed_fwd_kernel(EmbedRows p) {
  const int sub = threadIdx.x / p.cw, chunk = blockIdx.y * p.cw + (int)threadIdx.x - sub * p.cw;
  const int c = embed_col<NARROW>(p.C, 8 * chunk), n = p.C - c;
  if (sub >= p.subs || 8 * chunk >= p.C) return;
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
      w[u] = ld8<TW, NARROW>(p.w, ok ? id[u] * p.ws + c : c, extent, ok ? n : 0);
    }
#pragma unroll
    for (int u = 0; u < EMB_U; ++u) {
      const int64_t r = r0 + (int64_t)(i + u) * p.subs;
      if (r >= p.N) return;
      float v[8];
      cvt8<TW, NARROW>(w[u], 8, v);
      const float s = (uint64_t)id[u] < (uint64_t)p.V ? p.scale : __builtin_nanf("");
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= s;
      st8<TY, NARROW>(p.y, r * p.ys + c, n, v);
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
  uint8_t* occurs;        // [V] tokens that occur, or null
  void* dw;               // [V, C]; this launch clears rows [fill0, fill1), fill_rows a workgroup
  int64_t fill0, fill1;
  int C, fill_rows;
  uint32_t N;
  int ids64, tiles, per_tile;  // per_tile: runs of SORT_TILE keys a workgroup takes
  int shift, bits;        // the digit: (key >> shift) & ((1 << bits) - 1)
};

DSA_DEV uint32_t token_key(const SortParams& s, uint32_t i) {
  const int64_t id = ld_id(s.ids, i, s.ids64);
  return (uint64_t)id < (uint64_t)s.V && id != s.padding ? (uint32_t)id : (uint32_t)s.V;
}

// Workgroup `b` of the launch's fill workgroups: its rows of dW, but those of
// tokens that occur, 16 bytes a thread at a time; consecutive threads write
// consecutive bytes.
template <typename TW, bool NARROW>
DSA_DEV void fill_zero(const SortParams& s, int b) {
  constexpr int E = NARROW ? 1 : 16 / (int)sizeof(TW);  // elements a store
  typedef TW vec __attribute__((ext_vector_type(E)));
  typedef vec vecu __attribute__((aligned(sizeof(TW))));
  const int64_t v0 = s.fill0 + (int64_t)b * s.fill_rows;
  const int64_t left = s.fill1 - v0;
  const uint32_t rows = (uint32_t)(left < s.fill_rows ? left : s.fill_rows), units = (uint32_t)(s.C + E - 1) / E;
  vec zero;
#pragma unroll
  for (int e = 0; e < E; ++e) zero[e] = (TW)0.f;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < rows * units; i += SORT_T) {
    const uint32_t r = i / units;
    const int c = min(E * (int)(i - r * units), s.C - E);
    if (s.occurs && s.occurs[v0 + r]) continue;
    *reinterpret_cast<vecu*>(static_cast<TW*>(s.dw) + (v0 + r) * s.C + c) = zero;
  }
}

// Clears the marks of the tokens that occur.
static __global__ __launch_bounds__(SORT_T) void embed_unmark_kernel(SortParams s) {
  const int64_t v0 = ((int64_t)blockIdx.x * SORT_T + threadIdx.x) * 16;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  if (v0 < s.V) *reinterpret_cast<u4*>(s.occurs + v0) = u4{0u, 0u, 0u, 0u};  // [V] rounded up to 16
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
template <typename TW, bool NARROW>
__global__ __launch_bounds__(SORT_T) void embed_count_kernel(SortParams s) {
  if ((int)blockIdx.x >= s.tiles) {
    fill_zero<TW, NARROW>(s, (int)blockIdx.x - s.tiles);
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
    if (!s.kin && key < (uint32_t)s.V) s.occurs[key] = 1;
    atomicAdd(&cnt[(key >> s.shift) & mask], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_D; d += SORT_T) s.counts[(int64_t)blockIdx.x * SORT_D + d] = cnt[d];
}

// Moves the tile's keys and positions to their places by one digit.
template <typename TW, bool NARROW>
__global__ __launch_bounds__(SORT_T) void embed_scatter_kernel(SortParams s) {
  if ((int)blockIdx.x >= s.tiles) {
    fill_zero<TW, NARROW>(s, (int)blockIdx.x - s.tiles);
    return;
  }
  __shared__ SortLds l;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = threadIdx.x;
  const uint32_t mask = (1u << s.bits) - 1;
  // thread d: where digit d of this tile begins in the sorted order
  uint32_t before = 0, total = 0;
#pragma unroll 16
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

// At most RANK_N positions of a vocabulary below 2^(32 - RANK_BITS): the key
// and the position in one 32-bit word, and a position's place is the number
// of smaller words.  A workgroup places 64 positions, one a lane; its waves
// share the comparisons.  All words lie in its LDS and are read four at a
// time, the same four by all lanes.
template <typename TW, bool NARROW>
__global__ __launch_bounds__(SORT_T) void embed_rank_kernel(SortParams s) {
  if ((int)blockIdx.x >= s.tiles) {
    fill_zero<TW, NARROW>(s, (int)blockIdx.x - s.tiles);
    return;
  }
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  __shared__ __align__(16) uint32_t words[RANK_N];
  __shared__ uint32_t part[SORT_W][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n4 = ((int)s.N + 3) / 4;
  for (int i = threadIdx.x; i < 4 * n4; i += SORT_T)
    words[i] = i < (int)s.N ? token_key(s, (uint32_t)i) << RANK_BITS | (uint32_t)i : 0xffffffffu;
  __syncthreads();
  const int i = (int)blockIdx.x * 64 + lane;
  const uint32_t mine = i < (int)s.N ? words[i] : 0u;
  uint32_t place = 0;
#pragma unroll 4
  for (int q = w; q < n4; q += SORT_W) {
    const u4 v = reinterpret_cast<const u4*>(words)[q];
#pragma unroll
    for (int e = 0; e < 4; ++e) place += v[e] < mine ? 1u : 0u;
  }
  part[w][lane] = place;
  __syncthreads();
  if (w > 0 || i >= (int)s.N) return;
#pragma unroll
  for (int v = 1; v < SORT_W; ++v) place += part[v][lane];
  s.kout[place] = mine >> RANK_BITS;
  s.pout[place] = (uint32_t)i;
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

// A wave: one chunk of positions, 512 columns.  A wave keeps two batches of
// rows in flight: the next is loaded while one is summed.  Every batch is
// loaded whole (past the chunk's end its last row again): a load behind a
// condition would make the compiler wait for the newer batch with the older.
// dout is read past the caches in bf16, where one instruction takes whole
// lines: it is read once, and the lines of dW that the fill has just written
// stay in the last-level cache instead.  Of 131072 x 1024 bf16 positions and
// 128100 tokens that took the sums from 107 to 66 us.
template <typename TDY, typename TW, bool NARROW>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedSums p) {
  constexpr int U = sizeof(TDY) == 2 ? 8 : 4;  // rows a batch
  const int lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ch = item / (uint32_t)p.slabs;
  if (ch >= p.chunks) return;
  const int c0 = (int)(item - ch * p.slabs) * 512 + lane * 8, c = embed_col<NARROW>(p.C, c0);
  const int n = c0 < p.C ? p.C - c : 0;  // lanes past the row load with the others, and write nothing
  const uint32_t i0 = ch * (uint32_t)p.K, i1 = min(i0 + (uint32_t)p.K, p.N);
  const uint32_t i = i0 + lane;
  const uint32_t key = i < i1 ? p.keys[i] : p.V, pos = i < i1 ? p.pos[i] : 0;
  const uint32_t next = i < i1 && i + 1 < p.N ? p.keys[i + 1] : p.V;
  const uint32_t prev = i0 > 0 ? p.keys[i0 - 1] : p.V;
  const int m = __popcll(__ballot(key < p.V));  // the chunk's tokens: the keys V come last
  if (m == 0) return;
  const uint64_t ends = __ballot(lane < m && key != next);
  // the chunk's first token began before it
  bool carried = __builtin_amdgcn_readfirstlane(prev) == __builtin_amdgcn_readfirstlane(key);
  const uint32_t cb = (uint32_t)c * (uint32_t)sizeof(TDY);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto load = [&](int j0, raw8<TDY>(&dy)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = (uint32_t)__builtin_amdgcn_readlane(pos, min(j0 + u, m - 1));
      const char* row = static_cast<const char*>(p.dy) + (int64_t)r * p.dys * (int64_t)sizeof(TDY);  // uniform
      typedef const typename Raw8<TDY>::v8u* ptr;
      if constexpr (NARROW) dy[u] = ld8<TDY, true>(p.dy, (int64_t)r * p.dys + c, p.dye, n);
      else if constexpr (sizeof(TDY) == 2) dy[u] = __builtin_nontemporal_load(reinterpret_cast<ptr>(row + cb));
      else dy[u] = *reinterpret_cast<ptr>(row + cb);
    }
  };
  auto sum = [&](int j0, const raw8<TDY>(&dy)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u;
      if (j < m) {
        float v[8];
        cvt8<TDY, NARROW>(dy[u], n, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += v[e];
        const bool end = (ends >> j) & 1;
        if (end || j == m - 1) {
          if (carried || !end) {
            st8<float, NARROW>(p.part + ((int64_t)ch * 2 + (carried ? 0 : 1)) * p.C, c, n, acc);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = acc[e] * p.scale;
            st8<TW, NARROW>(p.dw, (int64_t)(uint32_t)__builtin_amdgcn_readlane(key, j) * p.dws + c, n, v);
          }
          carried = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        }
      }
    }
  };
  raw8<TDY> a[U], b[U];
  load(0, a);
  for (int j0 = 0; j0 < m; j0 += 2 * U) {
    load(j0 + U, b);
    sum(j0, a);
    load(j0 + 2 * U, a);
    sum(j0 + U, b);
  }
}

// The sum of the token that begins in chunk ch and goes on to chunk `last`:
// the lane's columns of ch's partial sum, and by every `waves`-th chunk from
// q on of those behind.
template <bool NARROW>
DSA_DEV void join_parts(const EmbedSums& p, uint32_t ch, uint32_t last, int q, int waves, int c, int n, float (&acc)[8]) {
  constexpr int U = 8;
  const int64_t extent = (int64_t)p.chunks * 2 * p.C;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  if (q == 0) cvt8<float, NARROW>(ld8<float, NARROW>(p.part, ((int64_t)ch * 2 + 1) * p.C + c, extent, n), n, acc);
  for (int64_t k0 = (int64_t)ch + 1 + q; k0 <= last; k0 += waves * U) {
    raw8<float> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = ld8<float, NARROW>(p.part, min(k0 + waves * u, (int64_t)last) * 2 * p.C + c, extent, n);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + waves * u <= last) {
        float w[8];
        cvt8<float, NARROW>(v[u], n, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += w[e];
      }
  }
}

// A block: JOIN_W chunks and 512 columns; wave q looks whether a token begins in
// its chunk and goes on past the chunk's end.  One that ends within JOIN_ONE
// chunks is joined by the wave, which loads eight chunks' sums at once, a longer
// one by the whole block, tokens in turn.  The gradient's kernels with every token
// by the block, and with 2, 8 and 32 chunks by the wave: 2723 x 513 30.3, 24.2,
// 22.6, 22.6 us, 30000 x 768 of 2000 tokens 56.8, 51.2, 49.9, 50.4.
constexpr uint32_t JOIN_ONE = 8;
constexpr int JOIN_W = 8;

template <typename TW, bool NARROW>
__global__ __launch_bounds__(64 * JOIN_W) void embed_join_kernel(EmbedSums p) {
  __shared__ float red[JOIN_W - 1][64][8];
  __shared__ uint32_t far[JOIN_W][2];  // per wave: its chunk's last chunk (0: none to share), the token
  const int lane = threadIdx.x & 63, q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ch0 = blockIdx.x / (uint32_t)p.slabs * JOIN_W, ch = ch0 + q;
  const int c0 = (int)(blockIdx.x % (uint32_t)p.slabs) * 512 + lane * 8, c = embed_col<NARROW>(p.C, c0);
  const int n = c0 < p.C ? p.C - c : 0;
  const uint64_t i0 = (uint64_t)ch * p.K, i1 = i0 + p.K;
  float acc[8];
  if (lane == 0) far[q][0] = 0;
  if (i1 < p.N) {
    const uint32_t key = p.keys[i1], own = p.keys[i1 - 1], prev = i0 > 0 ? p.keys[i0 - 1] : p.V;
    if (key < p.V && own == key && prev != key) {  // with prev == key it began before
      // the chunks behind that begin with the token: the keys are sorted
      uint32_t last = ch;
      for (;;) {
        const uint64_t at = ((uint64_t)last + 1 + lane) * p.K;
        const int more = __popcll(__ballot(at < p.N && p.keys[at < p.N ? at : 0] == key));
        last += more;
        if (more < 64) break;
      }
      if (last - ch <= JOIN_ONE) {
        join_parts<NARROW>(p, ch, last, 0, 1, c, n, acc);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= p.scale;
        st8<TW, NARROW>(p.dw, (int64_t)key * p.dws + c, n, acc);
      } else if (lane == 0) {
        far[q][0] = last;
        far[q][1] = key;
      }
    }
  }
  __syncthreads();
  for (int v = 0; v < JOIN_W; ++v) {
    const uint32_t last = far[v][0], key = far[v][1];
    if (last == 0) continue;  // uniform over the block
    join_parts<NARROW>(p, ch0 + v, last, q, JOIN_W, c, n, acc);
    if (q > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red[q - 1][lane][e] = acc[e];
    }
    __syncthreads();
    if (q == 0) {
#pragma unroll
      for (int w = 0; w < JOIN_W - 1; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += red[w][lane][e];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= p.scale;
      st8<TW, NARROW>(p.dw, (int64_t)key * p.dws + c, n, acc);
    }
    __syncthreads();
  }
}

}  // namespace hid
}  // namespace dsa
