// dsa_vocab.hip — C ABI of the operators on a vocabulary's logits (declared in
// include/dsa_vocab.h): argument checks, launch shapes and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/dsa_vocab.h"
#include "dsa_host.h"
#include "dsa_vocab.h"

using namespace dsa::host;
namespace voc = dsa::voc;

namespace {

constexpr int64_t kMaxRows = 1LL << 36;  // a workspace of them in parts is below 2^61 bytes
constexpr int64_t kMaxV = (1LL << 31) - 128;  // positions of a row and its 16-byte borders are 32-bit
constexpr int64_t kLaunchBlocks = 1LL << 22;  // a launch's threads fit 32 bits

bool elem_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

bool one_or_none(int64_t stride) { return stride == 0 || stride == 1; }

// logits, or a gradient of their shape
int check_rows(const char* what, const char* name, const void* p, int64_t stride, int dt) {
  if (!p) return fail("%s: %s are required", what, name);
  if (!elem_aligned(p, elem_bytes(dt))) return fail("%s: %s are not aligned to their elements", what, name);
  if (stride < 0) return fail("%s: %s have rows of stride %lld", what, name, (long long)stride);
  return 0;
}

int check_sizes(const char* what, int64_t N, int64_t V, int dt) {
  if (!dtype_ok(dt)) return fail("%s: unknown dtype %d", what, dt);
  if (N < 0 || N > kMaxRows) return fail("%s: N must be in [0, 2^36], got %lld", what, (long long)N);
  if (V < 1 || V > kMaxV) return fail("%s: V must be in [1, 2^31 - 128], got %lld", what, (long long)V);
  return 0;
}

bool good_scale(float s) { return s >= 0x1p-100f && s <= 0x1p100f; }

// Launches `launch(row0, rows)` over all rows, `parts` blocks each.
template <typename F>
int by_rows(int64_t N, int parts, const char* what, F launch) {
  const int64_t most = std::max<int64_t>(1, kLaunchBlocks / parts);
  for (int64_t r = 0; r < N; r += most) {
    launch(r, (unsigned)std::min(most, N - r));
    if (launch_check(what)) return 1;
  }
  return 0;
}

voc::VocabRows rows_of(const dsa_logprobs_args* a) {
  voc::VocabRows p{};
  p.x = a->logits, p.xs = a->logits_stride, p.ids = a->ids, p.ids64 = a->ids_bytes == 8, p.ignore = a->ignore_index;
  p.lp = a->logprobs, p.ent = a->entropy, p.lse = a->lse, p.top_lp = a->top_logprobs, p.top_ids = a->top_ids;
  p.stats = reinterpret_cast<float4*>(a->stats);
  p.dlp = a->dlogprobs, p.dent = a->dentropy, p.dlse = a->dlse, p.dtop = a->dtop;
  p.dlp_s = a->dlogprobs_stride, p.dent_s = a->dentropy_stride, p.dlse_s = a->dlse_stride;
  p.dx = a->dlogits, p.dxs = a->dlogits_stride;
  p.V = (int)a->V, p.top = a->top_k;
  p.inv_t = a->inv_temperature;
  p.c = (float)((double)a->inv_temperature * 1.4426950408889634);
  return p;
}

int check_logprobs(const dsa_logprobs_args* a, bool bwd) {
  const char* what = bwd ? "dsa_logprobs_bwd" : "dsa_logprobs_fwd";
  if (!a) return fail("%s: no arguments", what);
  if (check_sizes(what, a->N, a->V, a->dtype)) return 1;
  if (!good_scale(a->inv_temperature)) return fail("%s: inv_temperature must be in [2^-100, 2^100]", what);
  if (a->top_k < 0 || a->top_k > std::min<int64_t>(a->V, DSA_VOCAB_MAX_ENTRIES))
    return fail("%s: top_k must be in [0, min(V, %d)], got %d", what, DSA_VOCAB_MAX_ENTRIES, a->top_k);
  if (a->top_k && a->V > DSA_VOCAB_MAX_TOP_V) return fail("%s: top_k needs V of at most %d", what, DSA_VOCAB_MAX_TOP_V);
  if (a->ids && a->ids_bytes != 4 && a->ids_bytes != 8) return fail("%s: ids_bytes must be 4 or 8, got %d", what, a->ids_bytes);
  if (a->N == 0) return 0;
  if (check_rows(what, "logits", a->logits, a->logits_stride, a->dtype)) return 1;
  if (a->ids && !elem_aligned(a->ids, a->ids_bytes)) return fail("%s: ids are not aligned to their elements", what);
  if (a->stats && !aligned16(a->stats)) return fail("%s: stats must be 16-byte aligned", what);
  if (!bwd) {
    if (a->logprobs && !a->ids) return fail("%s: logprobs need ids", what);
    if (a->top_k && !(a->top_logprobs && a->top_ids)) return fail("%s: top_k needs top_logprobs and top_ids", what);
    return 0;
  }
  if (!a->stats) return fail("%s: stats are required", what);
  if (!a->dlogprobs && !a->dentropy && !a->dlse && !a->dtop) return fail("%s: a gradient is required", what);
  if (a->dlogprobs && !a->ids) return fail("%s: dlogprobs need ids", what);
  if (a->dtop && !(a->top_k && a->top_ids)) return fail("%s: dtop needs top_k and top_ids", what);
  if (!one_or_none(a->dlogprobs_stride) || !one_or_none(a->dentropy_stride) || !one_or_none(a->dlse_stride))
    return fail("%s: the gradients' strides must be 0 or 1", what);
  if (check_rows(what, "dlogits", a->dlogits, a->dlogits_stride, a->dtype)) return 1;
  return a->dlogits_stride < a->V && a->N > 1 ? fail("%s: dlogits' rows overlap", what) : 0;
}

voc::VocabRows rows_of(const dsa_distill_args* a) {
  voc::VocabRows p{};
  p.x = a->logits, p.xs = a->logits_stride, p.ids = a->teacher_ids, p.ids64 = a->ids_bytes == 8;
  p.teacher = a->teacher, p.teacher_bf16 = a->teacher_dtype == DSA_BF16, p.teacher_lse = a->teacher_lse;
  p.loss = a->loss, p.stats = reinterpret_cast<float4*>(a->stats);
  p.dlp = a->dloss, p.dlp_s = a->dloss_stride, p.dx = a->dlogits, p.dxs = a->dlogits_stride;
  p.V = (int)a->V, p.K = a->K;
  p.t = a->temperature;
  p.inv_t = (float)(1.0 / (double)a->temperature);
  p.c = (float)(1.4426950408889634 / (double)a->temperature);
  return p;
}

int check_distill(const dsa_distill_args* a, bool bwd) {
  const char* what = bwd ? "dsa_distill_bwd" : "dsa_distill_fwd";
  if (!a) return fail("%s: no arguments", what);
  if (check_sizes(what, a->N, a->V, a->dtype)) return 1;
  if (!dtype_ok(a->teacher_dtype)) return fail("%s: unknown teacher_dtype %d", what, a->teacher_dtype);
  if (!good_scale(a->temperature)) return fail("%s: temperature must be in [2^-100, 2^100]", what);
  if (a->K < 1 || a->K > DSA_VOCAB_MAX_ENTRIES) return fail("%s: K must be in [1, %d], got %d", what, DSA_VOCAB_MAX_ENTRIES, a->K);
  if (a->ids_bytes != 4 && a->ids_bytes != 8) return fail("%s: ids_bytes must be 4 or 8, got %d", what, a->ids_bytes);
  if (a->N == 0) return 0;
  if (check_rows(what, "logits", a->logits, a->logits_stride, a->dtype)) return 1;
  if (!a->teacher_ids || !elem_aligned(a->teacher_ids, a->ids_bytes)) return fail("%s: teacher_ids are missing or not aligned", what);
  if (!a->teacher || !elem_aligned(a->teacher, elem_bytes(a->teacher_dtype)))
    return fail("%s: the teacher's logits are missing or not aligned", what);
  if (a->stats && !aligned16(a->stats)) return fail("%s: stats must be 16-byte aligned", what);
  if (!bwd) return a->loss ? 0 : fail("%s: loss is required", what);
  if (!a->stats || !a->dloss) return fail("%s: stats and dloss are required", what);
  if (!one_or_none(a->dloss_stride)) return fail("%s: dloss' stride must be 0 or 1", what);
  if (check_rows(what, "dlogits", a->dlogits, a->dlogits_stride, a->dtype)) return 1;
  return a->dlogits_stride < a->V && a->N > 1 ? fail("%s: dlogits' rows overlap", what) : 0;
}

constexpr int kThreads = 512, kThreadsNarrow = 256;  // of a block that has a row (by_width)
constexpr int kPart = 64 * voc::kPartWaves;  // of one that has a part of a row
constexpr int kPartMost = 2048, kPartLeast = 256;  // 16-byte vectors of a part
constexpr int kBack = 512;
constexpr int kBackPer = 2048;
// Gradients past the caches from here on.  With the two products that read it a
// step of 160 x 128100 bf16 (41 MB) takes 537 us through the caches and 541 past
// them, of 512 rows (131 MB) 663 and 655, of 1229 rows 1382 and 1356.
constexpr double kFarBytes = 64 << 20;
// Logits that a forward reads past the caches: of the last level's size and more,
// where no backward reads them again (the 64 largest of 2048 x 128100 bf16 102
// and 95 us), and those of a distillation from twice that on (4096 rows with the
// gradient 582 and 551; 1229 rows, 315 MB, 171 and 168).  Not those of a loss, whose
// rows may be left out, so that fewer bytes are read again than there are: 1229
// rows 152 and 164, 4096 of which 85% are left out 240 and 292.
constexpr double kFarLogits = 256 << 20;

template <typename F>
void by_bool(bool b, F f) {
  if (b) f(std::true_type{});
  else f(std::false_type{});
}
// f(threads of a block that has a row).  Many narrow rows are bound by each row's chain of
// steps, so more of them at once: 4096 x 1001 bf16 19.8 us by 512 threads and 11.4 by
// 256, with the 16 largest 51.9 and 28.4, 4096 x 16000 40.2 and 31.1, 2223 x 40155 43.8
// and 37.4; of 160 KB a row and few rows alike (2223 x 40155 fp32 58.8 and 59.5, 512 x
// 16000 bf16 9.5 and 9.0, 256 rows 7.9 and 7.9, with the 128 largest 12.9 and 15.3); wide
// rows the other way (2048 x 128100 bf16 92.5 and 95.2, fp32 159.8 and 171.1).
template <typename F>
void by_width(int64_t N, int64_t row_bytes, F f) {
  if (N >= 512 && row_bytes <= 128 << 10) f(std::integral_constant<int, kThreadsNarrow>{});
  else f(std::integral_constant<int, kThreads>{});
}
// f(threads of a block that joins a row's parts).  The join by 64 threads of a row in 63
// parts 3.4 us, in 513 10.5, in 2442 45, by 1024 2.5, 2.8 and 5.8; a pass of 24 rows in 257
// parts 36.9 and 33.3, of 100 rows in 17 parts 15.3 and 15.8.
constexpr int kPartsOfAWave = 32;
template <bool TOP, typename F>
void by_parts(int parts, F f) {
  if constexpr (TOP) f(std::integral_constant<int, 256>{});  // of 2^19 columns at most
  else if (parts <= kPartsOfAWave) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 1024>{});
}
double bytes_of(int64_t N, int64_t V, size_t elem) { return (double)N * (double)V * (double)elem; }

// How a forward cuts its rows.
struct Cut {
  int parts, per, segs;
  size_t part_bytes, bytes;
};

// Whether rows go in parts, joined by a second launch.  A block's time goes by its
// row's columns, bf16 and fp32 alike (a lane's chain of loads and sums), that of parts
// by all bytes, behind a launch more.  us of a pass whole and in parts, by rows:
//   82000  bf16    8:  9.6 11.7    96:  9.9 10.8
//   128100 bf16    8: 11.6 10.7    96: 12.1 10.7   160: 12.9 12.7   192: 13.3 13.9
//   128100 fp32    8: 12.1 10.7    64: 12.3 11.3    96: 13.1 14.3
//   262144 bf16    8: 19.9 11.2   128: 21.7 17.3   192: 21.8 21.7   250: 22.3 25.2
//   262144 fp32    8: 21.4 10.9    48: 21.4 13.7    96: 22.0 19.8   128: 22.2 24.0
//   524288 fp32    8: 38.4 10.6    96: 40.6 33.3   128: 48.3 43.9
//   2^20   fp32    8: 73.7 11.0    64: 87.0 44.3
// and with the largest, whose search is one block's either way (5, 20 or 64 of them):
//   48000  bf16    8: 10.2 12.1 (20)
//   64000  bf16    8: 13.2 13.2    64: 13.6 13.9   100: 13.6 14.6 (64)
//   82000  bf16    8: 14.1 12.3    96: 14.2 13.9   160: 14.1 15.2 (5)
//   50021  fp32    8: 12.4 11.9   100: 12.4 12.9 (20)
//   64000  fp32    8: 15.0 14.4    64: 15.2 15.2   100: 15.2 16.8 (64)
//   128100 bf16    8: 16.7 11.9   128: 17.5 16.2   160: 17.7 17.5   192: 18.0 19.0 (5)
//   128100 fp32    8: 19.1 12.0    64: 19.3 14.5    96: 19.8 17.0   128: 19.4 19.5 (5)
//   262144 bf16    8: 29.9 16.4   128: 30.7 27.1   192: 31.5 31.7 (64)
//   262144 fp32    8: 34.9 16.9    96: 35.7 30.1   128: 35.8 34.2   160: 35.9 38.9 (64)
// So rows go in parts while their bytes are below lines over the columns.  Without the
// largest none below 70000 columns, 41 MB of 128100, 102 of 262144, and all of 333000 and
// more (by the next rule).  With them none below 51000 in bf16, 46000 in fp32, whose search
// is the longer, 38 MB of 128100 and 53, and none of so many bytes that whole rows are read
// past the caches.  A lane of a whole row adds up 41 batches at most then, 64 with the largest.
//
// And many bytes are read faster where
// neighbouring blocks read neighbouring lines: the loss of 1229 x 128100 with its
// gradient 161.6 and 152.2, of 777 x 50021 fp32 80.1 and 76.9 (in between, 512 x
// 128100 23.9 and 26.5), but not with the largest to find, whose search then has
// nothing to hide behind: 64 of 2048 rows 93 and 115.
bool in_parts(int64_t N, int64_t V, int elem, int top) {
  const double bytes = bytes_of(N, V, elem), cols = (double)V;
  if (top) return bytes < std::min(elem == 2 ? std::min(650. * (cols - 51000.), 460. * (cols - 45000.)) : 640. * (cols - 46000.), kFarLogits);
  return bytes < std::min(700. * (cols - 70000.), 455. * (cols - 38000.)) || bytes >= 128 << 20;
}

Cut cut_of(int64_t N, int64_t V, int dt, int top) {
  Cut c{};
  const int64_t most = V / (dt == DSA_BF16 ? 8 : 4) + 9;  // vectors, wherever a row begins
  c.segs = (int)(V / voc::kSeg) + 2;
  c.parts = 1, c.per = kPartMost;
  if (!in_parts(N, V, elem_bytes(dt), top)) return c;
  // 128100 bf16 in 63 parts 4.2 us, in 8 parts 5.0
  while (c.per > kPartLeast && N * cdiv(most, c.per) < 512) c.per /= 2;
  c.parts = (int)cdiv(most, c.per);
  if (c.parts == 1) return c;
  c.part_bytes = (size_t)N * c.parts * voc::kPartWaves * sizeof(float4);
  c.bytes = c.part_bytes + (top ? (size_t)N * c.segs * 4 : 0);
  return c;
}
int take(voc::VocabRows& p, const Cut& c, void* ws, size_t bytes, const char* what) {
  p.parts = c.parts, p.per = c.per, p.segs = c.segs;
  if (c.bytes == 0) return 0;
  if (!ws || bytes < c.bytes || !aligned16(ws)) return fail("%s: the workspace needs %zu bytes, 16-byte aligned", what, c.bytes);
  p.part = static_cast<float4*>(ws);
  p.seg = reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + c.part_bytes);
  return 0;
}
// backward
template <typename T>
void cut_back(voc::VocabRows& p) {
  p.per = kBackPer;
  p.parts = (int)cdiv(p.V / voc::Vec<T>::N + 9, p.per);
}

template <typename T, bool TOP>
int logprobs_fwd(voc::VocabRows p, int64_t N, hipStream_t st) {
  size_t lds = 0;
  if (TOP) {
    p.keys = round_up(p.segs, 4);
    lds = (size_t)(p.keys + voc::kSharedWords) * 4;
  }
  const bool far = !p.stats && bytes_of(N, p.V, sizeof(T)) >= kFarLogits;
  if (p.parts == 1)
    return by_rows(N, 1, "logprobs_fwd_kernel", [&](int64_t r, unsigned rows) {
      p.row0 = r;
      by_bool(far, [&](auto f) {
        by_width(N, (int64_t)p.V * sizeof(T), [&](auto n) {
          constexpr int NT = decltype(n)::value;
          constexpr bool FAR = decltype(f)::value && (TOP || NT == kThreadsNarrow);  // so many bytes of wide rows are in parts
          hipLaunchKernelGGL((voc::logprobs_fwd_kernel<T, NT, TOP, FAR>), dim3(rows), dim3(NT), lds, st, p);
        });
      });
    });
  const size_t part_lds = TOP ? (size_t)p.per * 16 / sizeof(T) / voc::kSeg * 4 : 0;
  return by_rows(N, p.parts, "logprobs_part_kernel", [&](int64_t r, unsigned rows) {
           p.row0 = r;
           by_bool(far, [&](auto f) {
             constexpr bool FAR = !TOP && decltype(f)::value;  // with the largest, parts are for few bytes
             hipLaunchKernelGGL((voc::logprobs_part_kernel<T, kPart, TOP, FAR>), dim3(rows * p.parts), dim3(kPart), part_lds, st, p);
           });
         }) ||
         by_rows(N, 1, "logprobs_join_kernel", [&](int64_t r, unsigned rows) {
           p.row0 = r;
           by_parts<TOP>(p.parts, [&](auto n) {
             constexpr int NT = decltype(n)::value;
             hipLaunchKernelGGL((voc::logprobs_join_kernel<T, NT, TOP>), dim3(rows), dim3(NT), lds, st, p);
           });
         });
}

template <typename T>
int logprobs_bwd(voc::VocabRows p, int64_t N, hipStream_t st) {
  cut_back<T>(p);
  return by_rows(N, p.parts, "logprobs_bwd_kernel", [&](int64_t r, unsigned rows) {
    p.row0 = r;
    const dim3 grid(rows * p.parts), block(kBack);
    by_bool(bytes_of(N, p.V, sizeof(T)) >= kFarBytes, [&](auto f) {
      constexpr bool FAR = decltype(f)::value;
      if (p.dent) hipLaunchKernelGGL((voc::logprobs_bwd_kernel<T, kBack, true, FAR>), grid, block, 0, st, p);
      else hipLaunchKernelGGL((voc::logprobs_bwd_kernel<T, kBack, false, FAR>), grid, block, 0, st, p);
    });
  });
}

template <typename T>
int distill_fwd(voc::VocabRows p, int64_t N, hipStream_t st) {
  const bool far = bytes_of(N, p.V, sizeof(T)) >= (p.stats ? 2 * kFarLogits : kFarLogits);
  if (p.parts == 1)
    return by_rows(N, 1, "distill_fwd_kernel", [&](int64_t r, unsigned rows) {
      p.row0 = r;
      by_bool(far, [&](auto f) {
        by_width(N, (int64_t)p.V * sizeof(T), [&](auto n) {
          constexpr int NT = decltype(n)::value;
          constexpr bool FAR = decltype(f)::value && NT == kThreadsNarrow;
          hipLaunchKernelGGL((voc::distill_fwd_kernel<T, NT, FAR>), dim3(rows), dim3(NT), 0, st, p);
        });
      });
    });
  return by_rows(N, p.parts, "distill_part_kernel", [&](int64_t r, unsigned rows) {
           p.row0 = r;
           by_bool(far, [&](auto f) {
             hipLaunchKernelGGL((voc::distill_part_kernel<T, kPart, decltype(f)::value>), dim3(rows * p.parts), dim3(kPart), 0, st, p);
           });
         }) ||
         by_rows(N, 1, "distill_join_kernel", [&](int64_t r, unsigned rows) {
           p.row0 = r;
           by_parts<false>(p.parts, [&](auto n) {
             constexpr int NT = decltype(n)::value;
             hipLaunchKernelGGL((voc::distill_join_kernel<T, NT>), dim3(rows), dim3(NT), 0, st, p);
           });
         });
}

template <typename T>
int distill_bwd(voc::VocabRows p, int64_t N, hipStream_t st) {
  cut_back<T>(p);
  return by_rows(N, p.parts, "distill_bwd_kernel", [&](int64_t r, unsigned rows) {
    p.row0 = r;
    by_bool(bytes_of(N, p.V, sizeof(T)) >= kFarBytes, [&](auto f) {
      hipLaunchKernelGGL((voc::distill_bwd_kernel<T, kBack, decltype(f)::value>), dim3(rows * p.parts), dim3(kBack), 0, st, p);
    });
  });
}

}  // namespace

extern "C" {

size_t dsa_vocab_workspace_bytes(int64_t N, int64_t V, int32_t dtype, int32_t top_k) {
  return N > 0 && N <= kMaxRows && V > 0 && V <= kMaxV ? cut_of(N, V, dtype, top_k).bytes : 0;
}

int dsa_logprobs_fwd(const dsa_logprobs_args* a, void* stream) {
  g_err.clear();
  if (check_logprobs(a, false)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_logprobs_fwd")) return 1;
  voc::VocabRows p = rows_of(a);
  if (take(p, cut_of(a->N, a->V, a->dtype, a->top_k), a->workspace, a->workspace_bytes, "dsa_logprobs_fwd")) return 1;
  if (a->top_k) return a->dtype == DSA_BF16 ? logprobs_fwd<dsa::bf16, true>(p, a->N, st) : logprobs_fwd<float, true>(p, a->N, st);
  return a->dtype == DSA_BF16 ? logprobs_fwd<dsa::bf16, false>(p, a->N, st) : logprobs_fwd<float, false>(p, a->N, st);
}

int dsa_logprobs_bwd(const dsa_logprobs_args* a, void* stream) {
  g_err.clear();
  if (check_logprobs(a, true)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_logprobs_bwd")) return 1;
  const voc::VocabRows p = rows_of(a);
  return a->dtype == DSA_BF16 ? logprobs_bwd<dsa::bf16>(p, a->N, st) : logprobs_bwd<float>(p, a->N, st);
}

int dsa_distill_fwd(const dsa_distill_args* a, void* stream) {
  g_err.clear();
  if (check_distill(a, false)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_distill_fwd")) return 1;
  voc::VocabRows p = rows_of(a);
  if (take(p, cut_of(a->N, a->V, a->dtype, 0), a->workspace, a->workspace_bytes, "dsa_distill_fwd")) return 1;
  return a->dtype == DSA_BF16 ? distill_fwd<dsa::bf16>(p, a->N, st) : distill_fwd<float>(p, a->N, st);
}

int dsa_distill_bwd(const dsa_distill_args* a, void* stream) {
  g_err.clear();
  if (check_distill(a, true)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_distill_bwd")) return 1;
  const voc::VocabRows p = rows_of(a);
  return a->dtype == DSA_BF16 ? distill_bwd<dsa::bf16>(p, a->N, st) : distill_bwd<float>(p, a->N, st);
}

}  // extern "C"
