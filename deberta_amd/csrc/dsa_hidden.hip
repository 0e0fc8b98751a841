// dsa_hidden.hip — C ABI of the operators on hidden states (declared in
// include/dsa_block.h): argument checks, launch shapes and launches of hidden
// dropout, the RMS norm and the embedding.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/dsa_block.h"
#include "dsa_drop.h"
#include "dsa_embed.h"
#include "dsa_host.h"
#include "dsa_rms_launch.h"

using namespace dsa::host;
namespace hid = dsa::hid;

// Compiled in translation units of their own (dsa_rms_inst.hip).
namespace dsa {
namespace host {
#define DSA_EXTERN(TX, TR)                                                                  \
  extern template int launch_rms_fwd<TX, TR>(hid::RmsRows, int, hipStream_t);               \
  extern template int launch_rms_bwd<TX, TR>(const hid::RmsRows&, int, int64_t, hipStream_t);
DSA_EXTERN(bf16, bf16)
DSA_EXTERN(bf16, float)
DSA_EXTERN(float, bf16)
DSA_EXTERN(float, float)
#undef DSA_EXTERN
}  // namespace host
}  // namespace dsa

namespace {

constexpr int64_t kMaxRows = 0x7fffffffLL;
constexpr int kMaxEmbedC = 1 << 30;

template <typename T>
struct Tag {
  typedef T type;
};
template <typename F>
void by_type(int dt, F f) {
  if (dt == DSA_BF16) f(Tag<dsa::bf16>{});
  else f(Tag<float>{});
}

// f(NARROW): whether rows hold fewer than the eight columns of a lane
template <typename F>
void by_narrow(int C, F f) {
  if (C < 8) f(std::true_type{});
  else f(std::false_type{});
}

bool elem_aligned(const void* p, int dt) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elem_bytes(dt) - 1)) == 0; }
// a tensor of rows: given, its type known, aligned to its elements
bool rows_given(const void* p, int64_t stride, int dt) { return p && dtype_ok(dt) && elem_aligned(p, dt) && stride >= 0; }
bool vec_given(const void* p, int dt) { return p && dtype_ok(dt) && elem_aligned(p, dt); }

// The type of a sum of x and a residual (x's own without one).
int stream_dtype(int x_dt, const void* res, int res_dt) {
  return x_dt == DSA_BF16 && (!res || res_dt == DSA_BF16) ? DSA_BF16 : DSA_F32;
}

bool res_ok(const void* res, const int64_t* strides, int64_t per_group, int dt) {
  return !res || (dtype_ok(dt) && elem_aligned(res, dt) && strides[0] >= 0 && strides[1] >= 0 && per_group >= 1);
}
// elements from the residual's first to behind the last that a row reads
int64_t res_extent(const int64_t* strides, int64_t per_group, int64_t N, int C) {
  const int64_t g = (N - 1) / per_group;
  // the last row of the last group, or of the last full one
  const int64_t in_last = (N - 1) - g * per_group;
  int64_t last = g * strides[0] + in_last * strides[1];
  if (g > 0) last = std::max(last, (g - 1) * strides[0] + (per_group - 1) * strides[1]);
  return last + C;
}

// Keep bits of a call: threshold in [0, 65536].
hid::Drop drop_params(uint32_t t, uint64_t seed) {
  hid::Drop d;
  d.on = t != 0;
  d.lim = (uint32_t)((uint64_t)t << 16) - 1u;
  d.k0 = (uint32_t)seed;
  d.k1 = (uint32_t)(seed >> 32);
  d.scale = t < 65536u ? (float)(65536.0 / (65536.0 - (double)t)) : 0.f;
  return d;
}

// Threads of a block whose threads own a chunk of eight columns each: cw
// chunks of a row, subs rows at a time, slabs blocks beside each other that
// share the row evenly.
struct ChunkGrid {
  int cw, subs, slabs, threads;
};
ChunkGrid chunk_grid(int C, int most) {
  ChunkGrid g;
  const int chunks = (int)cdiv(C, 8);
  g.slabs = (int)cdiv(chunks, most);
  g.cw = (int)cdiv(chunks, g.slabs);
  g.subs = most / g.cw;
  g.threads = round_up(g.cw * g.subs, 64);
  return g;
}
bool grid_ok(int64_t blocks, int slabs, int threads) {
  return blocks * threads <= 0xffffffffLL && blocks <= kMaxRows && slabs <= 65535;
}

// Sums the blocks' partial sums part[nparts][sums][C] into out0 (the first of
// the sums) and out1 (the second); a null one is left out.
int sum_parts(const float* part, int64_t nparts, int sums, int C, void* out0, int dt0, void* out1, int dt1, hipStream_t st) {
  hid::SumParts p{};
  p.part = part, p.nparts = nparts, p.stride = (int64_t)sums * C, p.C = C;
  p.out[0] = out0, p.out[1] = out1;
  p.dt[0] = dt0, p.dt[1] = dt1;
  hipLaunchKernelGGL(hid::sum_parts_kernel, dim3((unsigned)cdiv(C, hid::SUM_C), out1 ? 2 : 1),
                     dim3(hid::SUM_C * hid::SUM_G), 0, st, p);
  return launch_check("sum_parts_kernel");
}

// ---- dropout ----------------------------------------------------------------

// rows a thread takes in the backward with dbias: at most about 512 blocks
// leave partial sums, and where a thread's rows are 16 at most one block takes
// all and writes dbias itself, without a second launch.  From the first kernel's
// start to the last one's end, one block / several, whatever the width (128 to
// 2048): 8 rows 5.6 to 6.6 us / 12.5 to 14 (7 of them in the kernels), 16 rows 9.2
// to 10.1 / 12 to 15, 32 rows 16 to 17 / 12 to 15.
int drop_sum_rows(int64_t N, int subs) {
  if (N <= 16 * subs) return (int)cdiv(cdiv(N, subs), hid::DROP_U) * hid::DROP_U;
  return (int)std::max<int64_t>(hid::DROP_U, cdiv(cdiv(N, (int64_t)subs * 512), hid::DROP_U) * hid::DROP_U);
}
int64_t drop_sum_blocks(int64_t N, int C) {
  const ChunkGrid g = chunk_grid(C, hid::DROP_SUM_T);
  return cdiv(N, (int64_t)drop_sum_rows(N, g.subs) * g.subs);
}

int check_dropout(const dsa_dropout_args* a, bool bwd) {
  if (!a) return fail("dsa: null arguments");
  if (a->N < 1 || a->N > kMaxRows || a->C < 1)
    return fail("dsa_dropout: N in [1, 2^31) and C >= 1 required, got N=%lld C=%d", (long long)a->N, a->C);
  if (a->threshold > 65536u) return fail("dsa_dropout: threshold must be in [0, 65536], got %u", a->threshold);
  if (!bwd) {
    if (!rows_given(a->x, a->x_stride, a->x_dtype)) return fail("dsa_dropout: bad x");
    if (!res_ok(a->res, a->res_strides, a->rows_per_group, a->res_dtype)) return fail("dsa_dropout: bad res");
    if (a->bias && !vec_given(a->bias, a->bias_dtype)) return fail("dsa_dropout: bad bias");
    if (!rows_given(a->y, a->y_stride, a->y_dtype) || a->y_dtype != stream_dtype(a->x_dtype, a->res, a->res_dtype))
      return fail("dsa_dropout: bad y (float32 unless x and res are both bf16)");
    return 0;
  }
  if (!rows_given(a->dy, a->dy_stride, a->dy_dtype)) return fail("dsa_dropout: bad dy");
  if (!a->dx && !a->dbias) return fail("dsa_dropout: dx or dbias is required");
  if (a->dx && !rows_given(a->dx, a->dx_stride, a->dx_dtype)) return fail("dsa_dropout: bad dx");
  if (a->dbias) {
    if (!vec_given(a->dbias, a->bias_dtype)) return fail("dsa_dropout: bad dbias");
    const size_t need = dsa_block_workspace_bytes(DSA_BLOCK_DROPOUT, a->N, a->C);  // none for one block
    if (need && (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)))
      return fail("dsa_dropout: workspace of %zu bytes (16-byte aligned) required", need);
  }
  return 0;
}

// ---- RMS norm ---------------------------------------------------------------

// rows a team takes in the backward
int rms_sum_rows(int64_t N, int C) { return (int)cdiv(N, (int64_t)rms_blocks_of(C) * rms_teams_of(C)); }
int64_t rms_sum_blocks(int64_t N, int C) { return cdiv(N, (int64_t)rms_sum_rows(N, C) * rms_teams_of(C)); }

int check_rms(const dsa_rms_args* a, bool quant, bool bwd) {
  if (!a) return fail("dsa: null arguments");
  if (a->N < 1 || a->N > kMaxRows || a->C < 1 || a->C > kMaxRmsC)
    return fail("dsa_add_rms: N in [1, 2^31) and C in [1, %d] required, got N=%lld C=%d", kMaxRmsC, (long long)a->N, a->C);
  if (a->threshold > 65536u) return fail("dsa_add_rms: threshold must be in [0, 65536], got %u", a->threshold);
  if (!rows_given(a->x, a->x_stride, a->x_dtype)) return fail("dsa_add_rms: bad x");
  if (!res_ok(a->res, a->res_strides, a->rows_per_group, a->res_dtype)) return fail("dsa_add_rms: bad res");
  if (a->bias && !vec_given(a->bias, a->bias_dtype)) return fail("dsa_add_rms: bad bias");
  if (!vec_given(a->weight, a->weight_dtype)) return fail("dsa_add_rms: bad weight");
  if (bwd && !a->rstd) return fail("dsa_add_rms: rstd is required");
  if (!bwd) {
    if (!a->y || a->y_stride < a->C) return fail("dsa_add_rms: bad y");
    if (!quant && !rows_given(a->y, a->y_stride, a->y_dtype)) return fail("dsa_add_rms: bad y");
    if (a->z && (!elem_aligned(a->z, stream_dtype(a->x_dtype, a->res, a->res_dtype)) || a->z_stride < a->C))
      return fail("dsa_add_rms: bad z");
    if (quant) {
      if (!a->scales) return fail("dsa_add_rms_quant: scales is required");
      const int g = a->group_size;
      if (g && (g < 32 || g > 512 || (g & (g - 1)) || a->C % g))
        return fail("dsa_add_rms_quant: group_size must be 0 or a power of two in [32, 512] that divides C, got %d for C=%d", g, a->C);
    }
    return 0;
  }
  if (!rows_given(a->dy, a->dy_stride, a->dy_dtype)) return fail("dsa_add_rms: bad dy");
  const int z_dt = stream_dtype(a->x_dtype, a->res, a->res_dtype);
  if (a->dzu && !rows_given(a->dzu, a->dzu_stride, z_dt)) return fail("dsa_add_rms: bad dzu");
  if (a->dx && !rows_given(a->dx, a->dx_stride, a->x_dtype)) return fail("dsa_add_rms: bad dx");
  if (a->dres && (!a->res || !rows_given(a->dres, a->dres_stride, a->res_dtype))) return fail("dsa_add_rms: bad dres");
  if (a->dweight && !vec_given(a->dweight, a->weight_dtype)) return fail("dsa_add_rms: bad dweight");
  if (a->dbias && (!a->bias || !vec_given(a->dbias, a->bias_dtype))) return fail("dsa_add_rms: bad dbias");
  if (a->dweight || a->dbias) {
    const size_t need = dsa_block_workspace_bytes(DSA_BLOCK_RMS, a->N, a->C);
    if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace))
      return fail("dsa_add_rms: workspace of %zu bytes (16-byte aligned) required", need);
  }
  return 0;
}

hid::RmsRows rms_params(const dsa_rms_args* a) {
  hid::RmsRows p{};
  p.x = a->x, p.bias = a->bias, p.res = a->res, p.w = a->weight, p.dy = a->dy, p.dzu = a->dzu;
  p.y = a->y, p.z = a->z, p.dx = a->dx, p.dres = a->dres;
  p.rstd = a->rstd, p.yscale = a->scales;
  p.xs = a->x_stride, p.xe = (a->N - 1) * a->x_stride + a->C;
  if (a->res) {
    p.rs0 = a->res_strides[0], p.rs1 = a->res_strides[1];
    p.re = res_extent(a->res_strides, a->rows_per_group, a->N, a->C);
    p.has_res = 1;
  } else {  // the first row of x, over and over
    p.res = a->x, p.re = p.xe;
  }
  p.ys = a->y_stride, p.zs = a->z_stride;
  p.dys = a->dy_stride, p.dye = (a->N - 1) * a->dy_stride + a->C;
  p.dzus = a->dzu_stride, p.dzue = (a->N - 1) * a->dzu_stride + a->C;
  p.has_u = a->dzu != nullptr;
  if (!p.has_u) {  // the first row of whichever of x and res has z's type
    const bool as_x = a->x_dtype == stream_dtype(a->x_dtype, a->res, a->res_dtype);
    p.dzu = as_x ? a->x : a->res;
    p.dzus = 0, p.dzue = as_x ? p.xe : p.re;
  }
  p.dxs = a->dx_stride, p.drs = a->dres_stride;
  p.N = (uint32_t)a->N;
  p.rpg = (uint32_t)std::min<int64_t>(a->res ? a->rows_per_group : a->N, a->N);
  p.C = a->C, p.bias_dt = a->bias_dtype, p.w_dt = a->weight_dtype, p.group = a->group_size;
  p.eps = a->eps;
  p.d = drop_params(a->threshold, a->seed);
  return p;
}

int rms_fwd(const dsa_rms_args* a, bool quant, const char* what, void* stream) {
  g_err.clear();
  if (check_rms(a, quant, false)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, what)) return 1;
  const hid::RmsRows p = rms_params(a);
  const int y_dt = quant ? kFp8 : a->y_dtype;
  int rc = 0;
  by_type(a->x_dtype, [&](auto tx) {
    by_type(a->res ? a->res_dtype : a->x_dtype, [&](auto tr) {
      rc = launch_rms_fwd<typename decltype(tx)::type, typename decltype(tr)::type>(p, y_dt, st);
    });
  });
  return rc;
}

// ---- embedding --------------------------------------------------------------

int bit_length(int64_t v) {
  int b = 0;
  while (v >> b) ++b;
  return b;
}
// positions a chunk of the sums: enough chunks for 2048 waves, at most 64
int embed_chunk(int64_t N, int slabs) {
  int k = 8;
  while (k < 64 && N * slabs > (int64_t)2048 * k) k *= 2;
  return k;
}
struct EmbedPlan {
  bool rank;  // sorted by counting
  int bits, passes, tiles, per_tile, slabs, K;
  int64_t chunks;
  size_t keys, counts, marks, part, total;  // bytes: a key or position buffer, the counts, the marks, the partial sums
};
EmbedPlan embed_plan(int64_t N, int C, int64_t V) {
  EmbedPlan e;
  const int all = bit_length(V);
  e.passes = (int)cdiv(all, hid::SORT_BITS);
  e.bits = (int)cdiv(all, e.passes);
  e.rank = N <= hid::RANK_N && all <= 32 - hid::RANK_BITS;
  e.per_tile = (int)cdiv(N, (int64_t)hid::SORT_TILE * 256);
  e.tiles = e.rank ? (int)cdiv(N, 64) : (int)cdiv(N, (int64_t)hid::SORT_TILE * e.per_tile);
  e.slabs = (int)cdiv(C, 512);
  e.K = embed_chunk(N, e.slabs);
  e.chunks = cdiv(N, e.K);
  e.keys = align_up((size_t)N * 4, 256);
  e.counts = e.rank ? 0 : align_up((size_t)e.tiles * hid::SORT_D * 4, 256);
  e.marks = e.rank ? 0 : align_up((size_t)V, 256);
  e.part = align_up((size_t)e.chunks * 2 * C * sizeof(float), 256);
  e.total = e.keys * (!e.rank && e.passes > 1 ? 4 : 2) + e.counts + e.marks + e.part;
  return e;
}

int check_embed(const dsa_embed_args* a, bool bwd) {
  if (!a) return fail("dsa: null arguments");
  if (a->N < 1 || a->N > kMaxRows || a->C < 1 || a->V < 1 || a->V > kMaxRows - 1)
    return fail("dsa_embed: N in [1, 2^31), C >= 1 and V in [1, 2^31 - 2] required, got N=%lld C=%d V=%lld",
                (long long)a->N, a->C, (long long)a->V);
  if (a->ids_bytes != 4 && a->ids_bytes != 8) return fail("dsa_embed: ids must be int64 or int32");
  if (!a->ids || (reinterpret_cast<uintptr_t>(a->ids) & (uintptr_t)(a->ids_bytes - 1))) return fail("dsa_embed: bad ids");
  if (!bwd) {
    if (!rows_given(a->weight, a->weight_stride, a->weight_dtype)) return fail("dsa_embed: bad weight");
    if (!rows_given(a->y, a->y_stride, a->y_dtype)) return fail("dsa_embed: bad y");
    return 0;
  }
  // the sums take a column's byte offset in 32 bits
  if (a->C > kMaxEmbedC) return fail("dsa_embed: the backward takes at most 2^30 columns, got C=%d", a->C);
  if (!dtype_ok(a->weight_dtype)) return fail("dsa_embed: bad weight dtype");
  if (!rows_given(a->dy, a->dy_stride, a->dy_dtype)) return fail("dsa_embed: bad dy");
  if (!a->dweight || !aligned16(a->dweight)) return fail("dsa_embed: dweight must be given and 16-byte aligned");
  const size_t need = dsa_embed_workspace_bytes(a->N, a->C, a->V);
  if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace))
    return fail("dsa_embed: workspace of %zu bytes (16-byte aligned) required", need);
  return 0;
}

}  // namespace

namespace dsa {
namespace host {
// for dsa_block_workspace_bytes
size_t drop_workspace(int64_t N, int C) {
  const int64_t nb = drop_sum_blocks(N, C);
  return nb == 1 ? 0 : align_up((size_t)nb * C * sizeof(float), 256);
}
size_t rms_workspace(int64_t N, int C) { return align_up((size_t)rms_sum_blocks(N, C) * 2 * C * sizeof(float), 256); }
}  // namespace host
}  // namespace dsa

extern "C" {

int dsa_dropout_fwd(const dsa_dropout_args* a, void* stream) {
  g_err.clear();
  if (check_dropout(a, false)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_dropout_fwd")) return 1;
  const ChunkGrid g = chunk_grid(a->C, hid::DROP_T);
  hid::DropRows p{};
  p.x = a->x, p.bias = a->bias, p.res = a->res, p.y = a->y;
  p.xs = a->x_stride, p.xe = (a->N - 1) * a->x_stride + a->C, p.ys = a->y_stride;
  if (a->res) {
    p.rs0 = a->res_strides[0], p.rs1 = a->res_strides[1];
    p.re = res_extent(a->res_strides, a->rows_per_group, a->N, a->C);
  }
  p.N = (uint32_t)a->N;
  p.rpg = (uint32_t)std::min<int64_t>(a->res ? a->rows_per_group : a->N, a->N);
  p.C = a->C, p.bias_dt = a->bias_dtype;
  p.cw = g.cw, p.subs = g.subs, p.rows = hid::DROP_U;
  p.d = drop_params(a->threshold, a->seed);
  const int64_t nb = cdiv(a->N, (int64_t)p.rows * g.subs);
  if (!grid_ok(nb, g.slabs, g.threads)) return fail("dsa_dropout: too many rows or columns for one launch");
  by_type(a->x_dtype, [&](auto tx) {
    by_type(a->res ? a->res_dtype : a->x_dtype, [&](auto tr) {
      typedef typename decltype(tx)::type TX;
      typedef typename decltype(tr)::type TR;
      by_tail(a->C, [&](auto tail) {
        hipLaunchKernelGGL((hid::drop_fwd_kernel<TX, TR, stream_t<TX, TR>, decltype(tail)::value>),
                           dim3((unsigned)nb, (unsigned)g.slabs), dim3((unsigned)g.threads), 0, st, p);
      });
    });
  });
  return launch_check("drop_fwd_kernel");
}

int dsa_dropout_bwd(const dsa_dropout_args* a, void* stream) {
  g_err.clear();
  if (check_dropout(a, true)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_dropout_bwd")) return 1;
  const ChunkGrid g = chunk_grid(a->C, a->dbias ? hid::DROP_SUM_T : hid::DROP_T);
  hid::DropRows p{};
  p.dy = a->dy, p.dx = a->dx;
  p.dys = a->dy_stride, p.dye = (a->N - 1) * a->dy_stride + a->C, p.dxs = a->dx_stride;
  p.N = (uint32_t)a->N, p.C = a->C;
  p.cw = g.cw, p.subs = g.subs;
  p.rows = a->dbias ? drop_sum_rows(a->N, g.subs) : hid::DROP_U;
  p.d = drop_params(a->threshold, a->seed);
  const int64_t nb = cdiv(a->N, (int64_t)p.rows * g.subs);
  if (a->dbias) {
    p.bias_dt = a->bias_dtype;
    if (nb == 1) p.dbias = a->dbias;
    else p.part = static_cast<float*>(a->workspace);
  }
  if (!grid_ok(nb, g.slabs, g.threads)) return fail("dsa_dropout: too many rows or columns for one launch");
  by_type(a->dy_dtype, [&](auto tdy) {
    by_type(a->dx ? a->dx_dtype : a->dy_dtype, [&](auto tx) {
      by_tail(a->C, [&](auto tail) {
        hipLaunchKernelGGL((hid::drop_bwd_kernel<typename decltype(tdy)::type, typename decltype(tx)::type, decltype(tail)::value>),
                           dim3((unsigned)nb, (unsigned)g.slabs), dim3((unsigned)g.threads), 0, st, p);
      });
    });
  });
  if (launch_check("drop_bwd_kernel")) return 1;
  if (!p.part) return 0;
  return sum_parts(p.part, nb, 1, a->C, a->dbias, a->bias_dtype, nullptr, 0, st);
}

int dsa_add_rms_fwd(const dsa_rms_args* a, void* stream) { return rms_fwd(a, false, "dsa_add_rms_fwd", stream); }

int dsa_add_rms_quant(const dsa_rms_args* a, void* stream) { return rms_fwd(a, true, "dsa_add_rms_quant", stream); }

int dsa_add_rms_bwd(const dsa_rms_args* a, void* stream) {
  g_err.clear();
  if (check_rms(a, false, true)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_add_rms_bwd")) return 1;
  hid::RmsRows p = rms_params(a);
  p.part = a->dweight || a->dbias ? static_cast<float*>(a->workspace) : nullptr;
  p.rows = rms_sum_rows(a->N, a->C);
  const int64_t nb = rms_sum_blocks(a->N, a->C);
  int rc = 0;
  by_type(a->x_dtype, [&](auto tx) {
    by_type(a->res ? a->res_dtype : a->x_dtype, [&](auto tr) {
      rc = launch_rms_bwd<typename decltype(tx)::type, typename decltype(tr)::type>(p, a->dy_dtype, nb, st);
    });
  });
  if (rc || !p.part) return rc;
  return sum_parts(p.part, nb, a->bias ? 2 : 1, a->C, a->dweight, a->weight_dtype, a->dbias, a->bias_dtype, st);
}

size_t dsa_embed_workspace_bytes(int64_t N, int32_t C, int64_t V) {
  if (N < 1 || N > kMaxRows || C < 1 || V < 1 || V > kMaxRows - 1) return 0;
  return embed_plan(N, C, V).total;
}

int dsa_embed_fwd(const dsa_embed_args* a, void* stream) {
  g_err.clear();
  if (check_embed(a, false)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_embed_fwd")) return 1;
  const ChunkGrid g = chunk_grid(a->C, hid::EMB_T);
  hid::EmbedRows p{};
  p.ids = a->ids, p.w = a->weight, p.y = a->y;
  p.V = a->V, p.ws = a->weight_stride, p.ys = a->y_stride;
  p.N = (uint32_t)a->N, p.C = a->C, p.ids64 = a->ids_bytes == 8;
  p.cw = g.cw, p.subs = g.subs, p.rows = hid::EMB_U, p.scale = a->scale;
  const int64_t nb = cdiv(a->N, (int64_t)p.rows * g.subs);
  if (!grid_ok(nb, g.slabs, g.threads)) return fail("dsa_embed: too many rows or columns for one launch");
  by_type(a->weight_dtype, [&](auto tw) {
    by_type(a->y_dtype, [&](auto ty) {
      by_narrow(a->C, [&](auto narrow) {
        hipLaunchKernelGGL((hid::embed_fwd_kernel<typename decltype(tw)::type, typename decltype(ty)::type, decltype(narrow)::value>),
                           dim3((unsigned)nb, (unsigned)g.slabs), dim3((unsigned)g.threads), 0, st, p);
      });
    });
  });
  return launch_check("embed_fwd_kernel");
}

int dsa_embed_bwd(const dsa_embed_args* a, void* stream) {
  g_err.clear();
  if (check_embed(a, true)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_embed_bwd")) return 1;
  const EmbedPlan e = embed_plan(a->N, a->C, a->V);
  if (!grid_ok(cdiv(e.chunks, hid::JOIN_W) * cdiv(a->C, 512), 1, 64 * hid::JOIN_W))
    return fail("dsa_embed: too many rows or columns for one launch");
  char* ws = static_cast<char*>(a->workspace);
  uint32_t* buf[4];  // keys and positions, twice
  for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t*>(ws + i * e.keys);
  ws += e.keys * (!e.rank && e.passes > 1 ? 4 : 2);
  hid::SortParams s{};
  s.ids = a->ids, s.V = a->V, s.padding = a->padding;
  s.counts = reinterpret_cast<uint32_t*>(ws);
  s.occurs = e.rank ? nullptr : reinterpret_cast<uint8_t*>(ws + e.counts);
  float* part = reinterpret_cast<float*>(ws + e.counts + e.marks);
  s.N = (uint32_t)a->N, s.ids64 = a->ids_bytes == 8;
  s.tiles = e.tiles, s.per_tile = e.per_tile, s.bits = e.bits;
  s.dw = a->dweight, s.C = a->C;
  s.fill_rows = (int)std::max<int64_t>(1, hid::FILL_BYTES / ((int64_t)a->C * elem_bytes(a->weight_dtype)));
  // each launch of the sort but the first of several clears its share of dW
  const int64_t share = cdiv(a->V, e.rank ? 1 : 2 * e.passes - 1);
  if (!grid_ok(e.tiles + cdiv(share, s.fill_rows), 1, hid::SORT_T)) return fail("dsa_embed: the table is too large for one launch");
  const dim3 block(hid::SORT_T);
  auto grid = [&](bool fill) {
    s.fill0 = s.fill1;
    if (fill) s.fill1 = std::min(s.fill0 + share, a->V);
    return dim3((unsigned)(e.tiles + cdiv(s.fill1 - s.fill0, s.fill_rows)));
  };
  int rc = 0;
  if (!e.rank) {
    hipLaunchKernelGGL(hid::embed_unmark_kernel, dim3((unsigned)cdiv(a->V, 16 * hid::SORT_T)), block, 0, st, s);
    if (launch_check("embed_unmark_kernel")) return 1;
  }
  by_type(a->weight_dtype, [&](auto tw) {
    by_narrow(a->C, [&](auto narrow) {
      typedef typename decltype(tw)::type TW;
      constexpr bool T = decltype(narrow)::value;
      if (e.rank) {
        s.kout = buf[0], s.pout = buf[1];
        hipLaunchKernelGGL((hid::embed_rank_kernel<TW, T>), grid(true), block, 0, st, s);
        rc = launch_check("embed_rank_kernel");
        return;
      }
      for (int pass = 0; pass < e.passes && !rc; ++pass) {
        s.shift = pass * e.bits;
        s.kout = buf[2 * (pass & 1)], s.pout = buf[2 * (pass & 1) + 1];
        hipLaunchKernelGGL((hid::embed_count_kernel<TW, T>), grid(pass > 0), block, 0, st, s);
        if ((rc = launch_check("embed_count_kernel"))) return;
        hipLaunchKernelGGL((hid::embed_scatter_kernel<TW, T>), grid(true), block, 0, st, s);
        rc = launch_check("embed_scatter_kernel");
        s.kin = s.kout, s.pin = s.pout;
      }
    });
  });
  if (rc) return rc;
  const uint32_t *keys = s.kout, *pos = s.pout;
  hid::EmbedSums p{};
  p.keys = keys, p.pos = pos, p.dy = a->dy, p.dw = a->dweight, p.part = part;
  p.dys = a->dy_stride, p.dye = (a->N - 1) * a->dy_stride + a->C, p.dws = a->C;
  p.V = (uint32_t)a->V, p.N = (uint32_t)a->N, p.chunks = (uint32_t)e.chunks;
  p.C = a->C, p.slabs = e.slabs, p.K = e.K, p.scale = a->scale;
  by_type(a->dy_dtype, [&](auto tdy) {
    by_type(a->weight_dtype, [&](auto tw) {
      by_narrow(a->C, [&](auto narrow) {
        typedef typename decltype(tdy)::type TDY;
        typedef typename decltype(tw)::type TW;
        constexpr bool T = decltype(narrow)::value;
        const dim3 grid((unsigned)cdiv(e.chunks * e.slabs, 4)), block(256);
        hipLaunchKernelGGL((hid::embed_sum_kernel<TDY, TW, T>), grid, block, 0, st, p);
      });
    });
  });
  if (launch_check("embed_sum_kernel")) return 1;
  if (e.chunks == 1) return 0;
  by_type(a->weight_dtype, [&](auto tw) {
    by_narrow(a->C, [&](auto narrow) {
      hipLaunchKernelGGL((hid::embed_join_kernel<typename decltype(tw)::type, decltype(narrow)::value>),
                         dim3((unsigned)(cdiv(e.chunks, hid::JOIN_W) * p.slabs)), dim3(64 * hid::JOIN_W), 0, st, p);
    });
  });
  return launch_check("embed_join_kernel");
}

}  // extern "C"
