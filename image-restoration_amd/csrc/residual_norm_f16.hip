// The kernels of residual_norm.h for _Float16 activations.
#define JIRF_RN_KERNELS
#include <algorithm>

#include "residual_norm.h"

namespace jirf {
template <> void rn_launch_fwd<_Float16>(const RnArgs& a, const RnForm& f, hipStream_t s) { launch_fwd<_Float16>(a, f, s); }
template <> void rn_launch_bwd<_Float16>(const RnArgs& a, const RnForm& f, int mode, bool params, hipStream_t s) {
  launch_bwd<_Float16>(a, f, mode, params, s);
}
}  // namespace jirf
