#include "layernorm_launch_impl.cuh"

namespace lab200 {
template cudaError_t ln_fwd<SRMS_F32>(const LnArgs&, LnPlace);
template cudaError_t ln_bwd<SRMS_F32>(LnArgs, LnPlace);
template int ln_bwd_parts<SRMS_F32>(const LnArgs&, LnPlace);
}  // namespace lab200
