// The layer norm's kernels for tensors of F16.
#include "layer_norm_kernels.h"

namespace fmhc {

template int ln_fwd_run<FMHC_DTYPE_F16>(const LnFwdArgs&, hipStream_t);
template int ln_bwd_run<FMHC_DTYPE_F16>(const LnBwdArgs&, hipStream_t);

}  // namespace fmhc
