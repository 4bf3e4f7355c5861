// C-ABI entry points of the layer norms and the 8-bit activation checkpoints (declared in include/lightning_b200.h).
// Host side only: argument checks, kernel selection and launches.
#include <cuda_runtime.h>
#include <math.h>

#include "../../include/lightning_b200.h"
#include "launch_count.h"
#include "layernorm_kernels.cuh"

using namespace lab200;

namespace {

bool dtype_known(int dt) { return dt == LAB200_F32 || dt == LAB200_F16 || dt == LAB200_BF16; }
int launched() {
  count_launch();
  return cudaGetLastError() == cudaSuccess ? LAB200_OK : LAB200_ERR_CUDA;
}
bool rows_ok(long long M, int N, long long ld) { return M <= 1 || ld >= N; }
// What the kernels' index arithmetic takes: 32 bits within a row, 64 over all of them, with room for byte offsets.
bool size_ok(long long M, int N, long long ld) {
  const long long widest = ld > N ? ld : N;
  return M >= 0 && N >= 1 && N <= (1 << 30) && widest <= (1LL << 58) && (M == 0 || widest <= (1LL << 58) / M);
}
unsigned capped(long long want, long long most) { return static_cast<unsigned>(want < 1 ? 1 : want > most ? most : want); }

// Parts that the sums over rows are cut into: one for 32 rows, at most 64.
int ln_parts(long long M) { return static_cast<int>(M <= 0 ? 0 : M >= 64 * 32 ? 64 : (M + 31) / 32); }

template <int DT>
int ln_fwd(const LnArgs& a, cudaStream_t st) {
  ln_fwd_any_kernel<DT><<<capped(a.M, 1 << 20), 256, 0, st>>>(a);
  return launched();
}

template <int DT>
int ln_bwd(LnArgs a, cudaStream_t st) {
  if (a.M > 0 && (a.dx || a.dgate)) {
    ln_bwd_any_kernel<DT><<<capped(a.M, 1 << 20), 256, 0, st>>>(a);
    if (const int rc = launched()) return rc;
  }
  if (!a.dw && !a.db) return LAB200_OK;
  const unsigned cols = capped((a.N - 1) / 32 + 1, 1 << 20);
  a.nparts = ln_parts(a.M);
  if (a.nparts) {
    ln_bwd_columns_kernel<DT><<<dim3(cols, a.nparts), 256, 0, st>>>(a);
    if (const int rc = launched()) return rc;
  }
  ln_bwd_join_kernel<<<cols, 256, 0, st>>>(a.partial, a.nparts, a.N, a.dw, a.db, a.wdt);
  return launched();
}

}  // namespace

extern "C" {

int lab200_layernorm_fwd(const void* x, long long ldx, const void* gate, long long ldg, const void* weight, const void* bias, int wdtype, void* y,
                         float* stats, void* xcodes, void* xscales, void* gcodes, void* gscales, long long M, int N, float eps, int dtype, void* stream) {
  if (!size_ok(M, N, ldx) || (gate && !size_ok(M, N, ldg)) || !rows_ok(M, N, ldx) || (gate && !rows_ok(M, N, ldg))) return LAB200_ERR_SHAPE;
  if (!dtype_known(dtype) || ((weight || bias) && wdtype != dtype && wdtype != LAB200_F32)) return LAB200_ERR_DTYPE;
  if (!(eps >= 0.f) || isinf(eps)) return LAB200_ERR_SHAPE;
  if (M == 0) return LAB200_OK;
  if (!x || !y || !xcodes != !xscales || !gcodes != !gscales || (gcodes && !gate) || (gate && !xcodes != !gcodes)) return LAB200_ERR_SHAPE;
  LnArgs a = {};
  a.x = x; a.ldx = ldx; a.gate = gate; a.ldg = ldg; a.weight = weight; a.bias = bias; a.wdt = wdtype; a.y = y;
  a.stats = reinterpret_cast<float2*>(stats);
  a.xcodes = static_cast<int8_t*>(xcodes); a.xscales = static_cast<uint8_t*>(xscales);
  a.gcodes = static_cast<int8_t*>(gcodes); a.gscales = static_cast<uint8_t*>(gscales);
  a.M = M; a.N = N; a.eps = eps;
  if (reinterpret_cast<uintptr_t>(stats) & 7) return LAB200_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == LAB200_F32 ? ln_fwd<SRMS_F32>(a, st) : dtype == LAB200_F16 ? ln_fwd<SRMS_F16>(a, st) : ln_fwd<SRMS_BF16>(a, st);
}

size_t lab200_layernorm_bwd_workspace_bytes(long long M, int N) {
  return N < 1 ? 0 : static_cast<size_t>(ln_parts(M)) * 2 * N * sizeof(float);
}

int lab200_layernorm_bwd(const void* x, long long ldx, const void* gate, long long ldg, const void* xcodes, const void* xscales, const void* gcodes,
                         const void* gscales, const float* stats, const void* dy, long long lddy, const void* weight, const void* bias, int wdtype,
                         void* dx, void* dgate, void* dweight, void* dbias, void* workspace, size_t workspace_bytes, long long M, int N, int dtype,
                         void* stream) {
  if (!size_ok(M, N, lddy) || !rows_ok(M, N, lddy) || (x && (!size_ok(M, N, ldx) || !rows_ok(M, N, ldx))) ||
      (gate && (!size_ok(M, N, ldg) || !rows_ok(M, N, ldg))))
    return LAB200_ERR_SHAPE;
  if (!dtype_known(dtype) || ((weight || bias || dweight || dbias) && wdtype != dtype && wdtype != LAB200_F32)) return LAB200_ERR_DTYPE;
  if (M > 0 && (!stats || !dy || !x == !xcodes || !xcodes != !xscales || (gate && gcodes) || !gcodes != !gscales || (gate && xcodes) || (gcodes && x)))
    return LAB200_ERR_SHAPE;
  if (dgate && M > 0 && !gate && !gcodes) return LAB200_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(stats) & 7) return LAB200_ERR_ALIGN;
  if ((dweight || dbias) && M > 0 && (!workspace || workspace_bytes < lab200_layernorm_bwd_workspace_bytes(M, N))) return LAB200_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return LAB200_ERR_ALIGN;
  LnArgs a = {};
  a.x = x; a.ldx = ldx; a.gate = gate; a.ldg = ldg; a.weight = weight; a.bias = bias; a.wdt = wdtype;
  a.xcodes = static_cast<int8_t*>(const_cast<void*>(xcodes)); a.xscales = static_cast<uint8_t*>(const_cast<void*>(xscales));
  a.gcodes = static_cast<int8_t*>(const_cast<void*>(gcodes)); a.gscales = static_cast<uint8_t*>(const_cast<void*>(gscales));
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.dy = dy; a.lddy = lddy; a.dx = dx; a.dgate = dgate; a.dw = dweight; a.db = dbias;
  a.partial = static_cast<float*>(workspace);
  a.M = M; a.N = N;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == LAB200_F32 ? ln_bwd<SRMS_F32>(a, st) : dtype == LAB200_F16 ? ln_bwd<SRMS_F16>(a, st) : ln_bwd<SRMS_BF16>(a, st);
}

int lab200_pack8(const void* x, long long ldx, void* codes, void* scales, long long M, int N, int dtype, void* stream) {
  if (!size_ok(M, N, ldx) || !rows_ok(M, N, ldx)) return LAB200_ERR_SHAPE;
  if (!dtype_known(dtype)) return LAB200_ERR_DTYPE;
  if (M == 0) return LAB200_OK;
  if (!x || !codes || !scales) return LAB200_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* c = static_cast<int8_t*>(codes);
  auto* s = static_cast<uint8_t*>(scales);
  const unsigned grid = capped((M * ((N - 1) / PK_GROUP + 1) + 7) / 8, 1 << 20);
  if (dtype == LAB200_F32) pack8_any_kernel<SRMS_F32><<<grid, 256, 0, st>>>(x, ldx, c, s, M, N);
  else if (dtype == LAB200_F16) pack8_any_kernel<SRMS_F16><<<grid, 256, 0, st>>>(x, ldx, c, s, M, N);
  else pack8_any_kernel<SRMS_BF16><<<grid, 256, 0, st>>>(x, ldx, c, s, M, N);
  return launched();
}

int lab200_unpack8(const void* codes, const void* scales, void* y, long long M, int N, int dtype, void* stream) {
  if (!size_ok(M, N, N)) return LAB200_ERR_SHAPE;
  if (!dtype_known(dtype)) return LAB200_ERR_DTYPE;
  if (M == 0) return LAB200_OK;
  if (!y || !codes || !scales) return LAB200_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* c = static_cast<const int8_t*>(codes);
  auto* s = static_cast<const uint8_t*>(scales);
  const unsigned grid = capped((M * ((N - 1) / PK_GROUP + 1) + 7) / 8, 1 << 20);
  if (dtype == LAB200_F32) unpack8_any_kernel<SRMS_F32><<<grid, 256, 0, st>>>(c, s, y, M, N);
  else if (dtype == LAB200_F16) unpack8_any_kernel<SRMS_F16><<<grid, 256, 0, st>>>(c, s, y, M, N);
  else unpack8_any_kernel<SRMS_BF16><<<grid, 256, 0, st>>>(c, s, y, M, N);
  return launched();
}

}  // extern "C"
