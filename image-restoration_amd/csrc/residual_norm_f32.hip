// The kernels of residual_norm.h for float activations.
#define JIRF_RN_KERNELS
#include <algorithm>

#include "residual_norm.h"

namespace jirf {
template <> void rn_launch_fwd<float>(const RnArgs& a, const RnForm& f, hipStream_t s) { launch_fwd<float>(a, f, s); }
template <> void rn_launch_bwd<float>(const RnArgs& a, const RnForm& f, int mode, bool params, hipStream_t s) {
  launch_bwd<float>(a, f, mode, params, s);
}
}  // namespace jirf
