// dsa_rms_launch.h — the RMS norm's launches.  Each pair of x's and the
// residual's types is compiled in a translation unit of its own
// (dsa_rms_inst.hip with DSA_TX and DSA_TR); dsa_hidden.hip declares them.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "dsa_host.h"
#include "dsa_rms.h"

namespace dsa {
namespace host {

constexpr int kFp8 = 2;  // y's type beside DSA_F32 and DSA_BF16
constexpr int kMaxRmsC = 16384;

// Rows a block takes at a time: four waves with a row each up to 1024 columns
// (what a wave holds in registers), beyond that one row for the whole block.
inline int rms_teams_of(int C) { return C <= 1024 ? 4 : 1; }

// f(NC, W): chunks a lane and waves a row (its team).  Two chunks a lane at
// most: the backward keeps four fp32 values a column (w, the bias and both
// sums) beside the row itself.
template <typename F>
void by_width(int C, F f) {
  using std::integral_constant;
  if (C <= 512) f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (C <= 1024) f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  else if (C <= 2048) f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (C <= 4096) f(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  else if (C <= 8192) f(integral_constant<int, 2>{}, integral_constant<int, 8>{});
  else f(integral_constant<int, 2>{}, integral_constant<int, 16>{});
}

// f(TAIL): whether rows end in a chunk of fewer than eight columns
template <typename F>
void by_tail(int C, F f) {
  if (C % 8) f(std::true_type{});
  else f(std::false_type{});
}

template <typename TX, typename TR>
using stream_t = std::conditional_t<std::is_same<TX, TR>::value, TX, float>;

template <typename TX, typename TR>
int launch_rms_fwd(const hid::RmsRows& p, int y_dt, hipStream_t st) {
  typedef stream_t<TX, TR> TZ;
  by_width(p.C, [&](auto nc, auto w) {
    by_tail(p.C, [&](auto tail) {
      constexpr int NC = decltype(nc)::value, W = decltype(w)::value;
      constexpr bool T = decltype(tail)::value;
      const dim3 grid((unsigned)cdiv(p.N, hid::rms_teams<W>())), block(hid::rms_threads<W>());
      if (y_dt == kFp8) hipLaunchKernelGGL((hid::rms_fwd_kernel<NC, W, TX, TR, TZ, hid::fp8, T>), grid, block, 0, st, p);
      else if (y_dt == DSA_BF16) hipLaunchKernelGGL((hid::rms_fwd_kernel<NC, W, TX, TR, TZ, bf16, T>), grid, block, 0, st, p);
      else hipLaunchKernelGGL((hid::rms_fwd_kernel<NC, W, TX, TR, TZ, float, T>), grid, block, 0, st, p);
    });
  });
  return launch_check("rms_fwd_kernel");
}

template <typename TX, typename TR>
int launch_rms_bwd(const hid::RmsRows& p, int dy_dt, int64_t blocks, hipStream_t st) {
  typedef stream_t<TX, TR> TZ;
  by_width(p.C, [&](auto nc, auto w) {
    by_tail(p.C, [&](auto tail) {
      constexpr int NC = decltype(nc)::value, W = decltype(w)::value;
      constexpr bool T = decltype(tail)::value;
      const dim3 grid((unsigned)blocks), block(hid::rms_threads<W>());
      if (dy_dt == DSA_BF16) hipLaunchKernelGGL((hid::rms_bwd_kernel<NC, W, TX, TR, TZ, bf16, T>), grid, block, 0, st, p);
      else hipLaunchKernelGGL((hid::rms_bwd_kernel<NC, W, TX, TR, TZ, float, T>), grid, block, 0, st, p);
    });
  });
  return launch_check("rms_bwd_kernel");
}

}  // namespace host
}  // namespace dsa
