// The RMS norm's kernels for tensors of F32.
#include "rms_norm_kernels.h"

namespace fmhc {

template int rms_fwd_run<FMHC_DTYPE_F32>(const RmsFwdArgs&, hipStream_t);
template int rms_bwd_run<FMHC_DTYPE_F32>(const RmsBwdArgs&, hipStream_t);

}  // namespace fmhc
