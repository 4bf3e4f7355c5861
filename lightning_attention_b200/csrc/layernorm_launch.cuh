// Which layer norm kernel a call takes, and its launch. Each tensor type is compiled in a file of its own (layernorm_*.cu).
#pragma once
#include <cuda_runtime.h>

#include "launch_count.h"
#include "layernorm_kernels.cuh"

namespace lab200 {

constexpr int LN_MAX_PARTS = 320;  // parts of dw and db: at most two CTAs for each SM, and a few to spare

struct LnPlace { int device, sms; cudaStream_t st; };  // the current device, its SMs

template <int DT> cudaError_t ln_fwd(const LnArgs& a, LnPlace at);
template <int DT> cudaError_t ln_bwd(LnArgs a, LnPlace at);  // sets a.nparts; does not join the parts
template <int DT> int ln_bwd_parts(const LnArgs& a, LnPlace at);

inline unsigned ln_capped(long long want, long long most) { return static_cast<unsigned>(want < 1 ? 1 : want > most ? most : want); }

}  // namespace lab200
