// dsa_rms_inst.hip — the RMS norm's kernels for x of type DSA_TX and a
// residual of type DSA_TR (macros of the build): see dsa_rms_launch.h.
#include "dsa_rms_launch.h"

namespace dsa {
namespace host {
template int launch_rms_fwd<DSA_TX, DSA_TR>(hid::RmsRows, int, hipStream_t);
template int launch_rms_bwd<DSA_TX, DSA_TR>(const hid::RmsRows&, int, int64_t, hipStream_t);
}  // namespace host
}  // namespace dsa
