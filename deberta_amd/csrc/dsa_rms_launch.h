// dsa_rms_launch.h — the RMS norm's launches.  Each pair of x's and the
// residual's types is compiled in a translation unit of its own
// (dsa_rms_inst.hip with DSA_TX and DSA_TR); dsa_hidden.hip declares them.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "dsa_host.h"
#include "dsa_rms.h"

namespace dsa {
namespace host {

constexpr int kFp8 = 2;  // y's type beside DSA_F32 and DSA_BF16
constexpr int kMaxRmsC = 16384;

// f(L, NC, W): lanes a row where it takes less than a wave, chunks a lane,
// waves a row; at most two chunks a lane.
//
// Past 2048 columns the backward takes one chunk a lane and twice the waves of
// the forward.  It keeps four fp32 values a column (w, the bias and both sums)
// beside the row itself, and with fewer, larger blocks it leaves fewer partial
// sums: 8192 x 4096 bf16 4.56 TB/s against 4.18 with two chunks and 512 blocks
// of four waves, 4096 x 8192 4.42 against 3.97.  The forward has no such sums
// and loses on widths that fill the waves badly: 8176 x 4104 4.1 against 5.3.
template <bool BWD, typename F>
void by_width(int C, F f) {
  using std::integral_constant;
  integral_constant<int, 16> i16;
  integral_constant<int, 32> i32;
  integral_constant<int, 64> i64;
  integral_constant<int, 1> i1;
  integral_constant<int, 2> i2;
  integral_constant<int, 4> i4;
  integral_constant<int, 8> i8;
  if (C <= 128) f(i16, i1, i1);
  else if (C <= 256) f(i32, i1, i1);
  else if (C <= 512) f(i64, i1, i1);
  else if (C <= 1024) f(i64, i2, i1);
  else if (C <= 2048) f(i64, i1, i4);
  else if (C > 8192) f(i64, i2, i16);
  else if constexpr (BWD) {
    if (C <= 4096) f(i64, i1, i8);
    else f(i64, i1, i16);
  } else {
    if (C <= 4096) f(i64, i2, i4);
    else f(i64, i2, i8);
  }
}
// Teams a block of the backward, and the blocks that run at once: two a
// compute unit of four waves, one of eight or sixteen.
inline int rms_teams_of(int C) {
  int n = 0;
  by_width<true>(C, [&](auto l, auto, auto w) { n = hid::rms_teams<decltype(l)::value, decltype(w)::value>(); });
  return n;
}
inline int rms_blocks_of(int C) { return C <= 2048 ? 512 : 256; }

// f(TAIL): whether rows end in a chunk of fewer than eight columns
template <typename F>
void by_tail(int C, F f) {
  if (C % 8) f(std::true_type{});
  else f(std::false_type{});
}

template <typename TX, typename TR>
using stream_t = std::conditional_t<std::is_same<TX, TR>::value, TX, float>;

// One launch for all rows, or for as many as its 2^32 - 1 threads hold (2^28
// rows of at most 128 columns).
template <typename TX, typename TR>
int launch_rms_fwd(hid::RmsRows p, int y_dt, hipStream_t st) {
  typedef stream_t<TX, TR> TZ;
  by_width<false>(p.C, [&](auto l, auto nc, auto w) {
    by_tail(p.C, [&](auto tail) {
      constexpr int L = decltype(l)::value, NC = decltype(nc)::value, W = decltype(w)::value;
      constexpr bool T = decltype(tail)::value;
      const dim3 block(hid::rms_threads<W>());
      const int64_t most = 0xffffffffLL / block.x;  // blocks
      for (int64_t b = 0, all = cdiv(p.N, hid::rms_teams<L, W>()); b < all; b += most) {
        const dim3 grid((unsigned)std::min(most, all - b));
        p.r0 = (uint32_t)(b * hid::rms_teams<L, W>());
        if (y_dt == kFp8) hipLaunchKernelGGL((hid::rms_fwd_kernel<L, NC, W, TX, TR, TZ, hid::fp8, T>), grid, block, 0, st, p);
        else if (y_dt == DSA_BF16) hipLaunchKernelGGL((hid::rms_fwd_kernel<L, NC, W, TX, TR, TZ, bf16, T>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((hid::rms_fwd_kernel<L, NC, W, TX, TR, TZ, float, T>), grid, block, 0, st, p);
      }
    });
  });
  return launch_check("rms_fwd_kernel");
}

template <typename TX, typename TR>
int launch_rms_bwd(const hid::RmsRows& p, int dy_dt, int64_t blocks, hipStream_t st) {
  typedef stream_t<TX, TR> TZ;
  by_width<true>(p.C, [&](auto l, auto nc, auto w) {
    by_tail(p.C, [&](auto tail) {
      constexpr int L = decltype(l)::value, NC = decltype(nc)::value, W = decltype(w)::value;
      constexpr bool T = decltype(tail)::value;
      const dim3 grid((unsigned)blocks), block(hid::rms_threads<W>());
      if (dy_dt == DSA_BF16) hipLaunchKernelGGL((hid::rms_bwd_kernel<L, NC, W, TX, TR, TZ, bf16, T>), grid, block, 0, st, p);
      else hipLaunchKernelGGL((hid::rms_bwd_kernel<L, NC, W, TX, TR, TZ, float, T>), grid, block, 0, st, p);
    });
  });
  return launch_check("rms_bwd_kernel");
}

}  // namespace host
}  // namespace dsa
