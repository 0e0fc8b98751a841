// dsa_vocab.hip — C ABI of the operators on a vocabulary's logits (declared in
// include/dsa_vocab.h): argument checks, launch shapes and launches.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/dsa_vocab.h"
#include "dsa_host.h"
#include "dsa_vocab.h"

using namespace dsa::host;
namespace voc = dsa::voc;

namespace {

constexpr int64_t kMaxRows = 1LL << 40;
constexpr int64_t kMaxV = (1LL << 31) - 128;  // positions of a row and its 16-byte borders are 32-bit
constexpr int64_t kLaunchRows = 1LL << 22;    // a launch's threads fit 32 bits

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
  if (N < 0 || N > kMaxRows) return fail("%s: N must be in [0, 2^40], got %lld", what, (long long)N);
  if (V < 1 || V > kMaxV) return fail("%s: V must be in [1, 2^31 - 128], got %lld", what, (long long)V);
  return 0;
}

bool good_scale(float s) { return s >= 0x1p-100f && s <= 0x1p100f; }

// Launches `launch(row0, rows)` over all rows.
template <typename F>
int by_rows(int64_t N, const char* what, F launch) {
  for (int64_t r = 0; r < N; r += kLaunchRows) {
    launch(r, (unsigned)std::min(kLaunchRows, N - r));
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

constexpr int kThreads = 256;

template <typename T>
int logprobs_fwd(voc::VocabRows p, int64_t N, hipStream_t st) {
  if (!p.top)
    return by_rows(N, "logprobs_fwd_kernel", [&](int64_t r, unsigned rows) {
      p.row0 = r;
      hipLaunchKernelGGL((voc::logprobs_fwd_kernel<T, kThreads, false>), dim3(rows), dim3(kThreads), 0, st, p);
    });
  const int segs = p.V / voc::kSeg + 2;  // at most, wherever a row begins
  p.keys = std::max(segs, std::min(p.top, segs) * voc::kSeg);
  const size_t lds = (size_t)(p.keys + voc::kSharedWords) * 4;
  return by_rows(N, "logprobs_fwd_kernel", [&](int64_t r, unsigned rows) {
    p.row0 = r;
    hipLaunchKernelGGL((voc::logprobs_fwd_kernel<T, kThreads, true>), dim3(rows), dim3(kThreads), lds, st, p);
  });
}

template <typename T>
int logprobs_bwd(voc::VocabRows p, int64_t N, hipStream_t st) {
  return by_rows(N, "logprobs_bwd_kernel", [&](int64_t r, unsigned rows) {
    p.row0 = r;
    if (p.dent) hipLaunchKernelGGL((voc::logprobs_bwd_kernel<T, kThreads, true>), dim3(rows), dim3(kThreads), 0, st, p);
    else hipLaunchKernelGGL((voc::logprobs_bwd_kernel<T, kThreads, false>), dim3(rows), dim3(kThreads), 0, st, p);
  });
}

template <typename T>
int distill(voc::VocabRows p, int64_t N, bool bwd, hipStream_t st) {
  return by_rows(N, bwd ? "distill_bwd_kernel" : "distill_fwd_kernel", [&](int64_t r, unsigned rows) {
    p.row0 = r;
    if (bwd) hipLaunchKernelGGL((voc::distill_bwd_kernel<T, kThreads>), dim3(rows), dim3(kThreads), 0, st, p);
    else hipLaunchKernelGGL((voc::distill_fwd_kernel<T, kThreads>), dim3(rows), dim3(kThreads), 0, st, p);
  });
}

}  // namespace

extern "C" {

size_t dsa_vocab_workspace_bytes(int64_t, int64_t, int32_t, int32_t) { return 0; }

int dsa_logprobs_fwd(const dsa_logprobs_args* a, void* stream) {
  g_err.clear();
  if (check_logprobs(a, false)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_logprobs_fwd")) return 1;
  const voc::VocabRows p = rows_of(a);
  return a->dtype == DSA_BF16 ? logprobs_fwd<dsa::bf16>(p, a->N, st) : logprobs_fwd<float>(p, a->N, st);
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
  const voc::VocabRows p = rows_of(a);
  return a->dtype == DSA_BF16 ? distill<dsa::bf16>(p, a->N, false, st) : distill<float>(p, a->N, false, st);
}

int dsa_distill_bwd(const dsa_distill_args* a, void* stream) {
  g_err.clear();
  if (check_distill(a, true)) return 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (refuse_capture(st, "dsa_distill_bwd")) return 1;
  const voc::VocabRows p = rows_of(a);
  return a->dtype == DSA_BF16 ? distill<dsa::bf16>(p, a->N, true, st) : distill<float>(p, a->N, true, st);
}

}  // extern "C"
