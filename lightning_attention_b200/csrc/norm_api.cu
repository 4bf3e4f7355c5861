// C-ABI entry points of the layer norms and the 8-bit activation checkpoints (declared in include/lightning_b200.h).
// Host side only: argument checks, kernel selection and launches.
#include <cuda_runtime.h>
#include <math.h>

#include <atomic>

#include "../../include/lightning_b200.h"
#include "layernorm_launch.cuh"

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

// Whether each pointer (NULL ones too) is a multiple of the size of what it points to.
int size_of(int dtype) { return dtype == LAB200_F32 ? 4 : 2; }
template <class... Ptr>
bool whole(int size, Ptr... p) {
  return ((reinterpret_cast<uintptr_t>(p) % size == 0) && ...);
}

// The current device and its number of SMs, which is asked for once.
LnPlace place(cudaStream_t st) {
  static std::atomic<int> known[64];
  LnPlace at{0, 148, st};
  if (cudaGetDevice(&at.device) != cudaSuccess) {
    cudaGetLastError();
    return at;
  }
  int n = at.device < 64 ? known[at.device].load(std::memory_order_relaxed) : 0;
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, at.device) == cudaSuccess && at.device < 64)
    known[at.device].store(n, std::memory_order_relaxed);
  if (n > 0) at.sms = n;
  return at;
}

// How a call's rows are given out to warps: by packs of P values, or (P 0) by groups. Contiguous rows of whole groups are one row.
constexpr int PK_U = 4, PK_U_ANY = 8;
PkRows pk_rows(long long M, long long N, int P, bool contiguous) {
  if (P && contiguous && N % PK_GROUP == 0) N *= M, M = 1;
  PkRows r = {};
  r.M = M;
  r.ngroups = (N - 1) / PK_GROUP + 1;
  r.npack = P ? N / P : N;
  const long long units = P ? r.ngroups * (PK_GROUP / P) : r.ngroups, per = P ? 32 * PK_U : PK_U_ANY, per_row = (units + per - 1) / per;
  r.items = M * per_row;
  r.per_row = M == 1 ? 0 : static_cast<int>(per_row);
  // rows that fill their last item well are left to warps, whose place costs less (20000 x 1000 in 12 us
  // against 15; 27408 x 312 in 14 against 6, a warp having 40 packs for 128; value by value 27965 x 562
  // in 27 us against 35; 374506 x 51 in 117 against 51, a warp having 2 groups for 8)
  if (M > 1 && units * 10 < per_row * per * (P ? 9 : 6) && M * units <= (1ll << 31) - per) {
    // n / d = umulhi(n, ceil(2^(31 + l) / d)) >> (l - 1) for n < 2^31, d > 1 and 2^(l - 1) < d <= 2^l: the factor is too large by less
    // than d / 2^(31 + l), which n times stays below 1 / d
    int l = 1;
    while ((1ll << l) < units) ++l;
    r.units = static_cast<uint32_t>(units);
    r.magic = static_cast<uint32_t>(((1ull << (31 + l)) + units - 1) / units);
    r.shift = l - 1;
    r.items = (M * units + per - 1) / per;
  }
  return r;
}

bool aligned_params(const LnArgs& a) { return !((reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias)) & 15); }

// dw and db from their parts: a CTA per 32 columns, its 32 warps take every 32nd part. No part: zeros. 148 parts of 128 to 5120 columns
// in 3.0 to 4.3 us, most of it the launch and one chain of loads.
__global__ void __launch_bounds__(1024) ln_bwd_join_kernel(const float* __restrict__ partial, int nparts, int N, void* dw, void* db, int wdt) {
  __shared__ float red[2][32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long c0 = static_cast<long long>(blockIdx.x) * 32; c0 < N; c0 += static_cast<long long>(gridDim.x) * 32) {
    const int col = static_cast<int>(c0) + lane;
    const bool on = lane < N - c0;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll 5
    for (int p = warp; p < nparts; p += 32) {
      const float* from = partial + static_cast<size_t>(p) * 2 * N + col;
      s0 += on ? from[0] : 0.f;
      s1 += on ? from[N] : 0.f;
    }
    red[0][warp][lane] = s0;
    red[1][warp][lane] = s1;
    __syncthreads();
    if (warp < 2) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) v += red[warp][k][lane];
      if (on) ln_param_out(warp ? db : dw, wdt, col, v);
    }
    __syncthreads();
  }
}

template <int DT>
int run_bwd(LnArgs a, cudaStream_t st) {
  if (a.M > 0) {
    const LnPlace at = place(st);
    if (a.partial) a.nparts = ln_bwd_parts<DT>(a, at);
    if (ln_bwd<DT>(a, at) != cudaSuccess) return LAB200_ERR_CUDA;
  }
  if (!a.dw && !a.db) return LAB200_OK;
  ln_bwd_join_kernel<<<ln_capped((a.N - 1) / 32 + 1, 1 << 20), 1024, 0, st>>>(a.partial, a.nparts, a.N, a.dw, a.db, a.wdt);
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
  if (!whole(8, stats) || !whole(size_of(dtype), x, gate, y) || !whole(size_of(wdtype), weight, bias)) return LAB200_ERR_ALIGN;
  a.vec_params = aligned_params(a);
  const LnPlace at = place(static_cast<cudaStream_t>(stream));
  // groups of 32 values do not keep to the packs of odd rows: those are checkpointed on their own
  if (xcodes && N % (dtype == LAB200_F32 ? 4 : 8)) {
    int rc = lab200_pack8(x, ldx, xcodes, xscales, M, N, dtype, stream);
    if (rc == LAB200_OK && gate) rc = lab200_pack8(gate, ldg, gcodes, gscales, M, N, dtype, stream);
    if (rc != LAB200_OK) return rc;
    a.xcodes = a.gcodes = nullptr;
    a.xscales = a.gscales = nullptr;
  }
  const cudaError_t rc = dtype == LAB200_F32 ? ln_fwd<SRMS_F32>(a, at) : dtype == LAB200_F16 ? ln_fwd<SRMS_F16>(a, at) : ln_fwd<SRMS_BF16>(a, at);
  return rc == cudaSuccess ? LAB200_OK : LAB200_ERR_CUDA;
}

size_t lab200_layernorm_bwd_workspace_bytes(long long M, int N) {
  return N < 1 || M < 1 ? 0 : static_cast<size_t>(M + 8 < LN_MAX_PARTS ? M + 8 : LN_MAX_PARTS) * 2 * N * sizeof(float);
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
  if (!whole(8, stats) || !whole(size_of(dtype), x, gate, dy, dx, dgate) || !whole(size_of(wdtype), weight, bias, dweight, dbias)) return LAB200_ERR_ALIGN;
  if ((dweight || dbias) && M > 0 && (!workspace || workspace_bytes < lab200_layernorm_bwd_workspace_bytes(M, N))) return LAB200_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return LAB200_ERR_ALIGN;
  LnArgs a = {};
  a.x = x; a.ldx = ldx; a.gate = gate; a.ldg = ldg; a.weight = weight; a.bias = bias; a.wdt = wdtype;
  a.xcodes = static_cast<int8_t*>(const_cast<void*>(xcodes)); a.xscales = static_cast<uint8_t*>(const_cast<void*>(xscales));
  a.gcodes = static_cast<int8_t*>(const_cast<void*>(gcodes)); a.gscales = static_cast<uint8_t*>(const_cast<void*>(gscales));
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.dy = dy; a.lddy = lddy; a.dx = dx; a.dgate = dgate; a.dw = dweight; a.db = dbias;
  a.partial = dweight || dbias ? static_cast<float*>(workspace) : nullptr;
  a.M = M; a.N = N;
  a.vec_params = aligned_params(a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == LAB200_F32 ? run_bwd<SRMS_F32>(a, st) : dtype == LAB200_F16 ? run_bwd<SRMS_F16>(a, st) : run_bwd<SRMS_BF16>(a, st);
}

int lab200_pack8(const void* x, long long ldx, void* codes, void* scales, long long M, int N, int dtype, void* stream) {
  if (!size_ok(M, N, ldx) || !rows_ok(M, N, ldx)) return LAB200_ERR_SHAPE;
  if (!dtype_known(dtype)) return LAB200_ERR_DTYPE;
  if (M == 0) return LAB200_OK;
  if (!x || !codes || !scales) return LAB200_ERR_SHAPE;
  const int esz = size_of(dtype);
  if (!whole(esz, x)) return LAB200_ERR_ALIGN;
  if (M == 1) ldx = N;
  auto* c = static_cast<int8_t*>(codes);
  auto* s = static_cast<uint8_t*>(scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool packs = !((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ldx) * esz | static_cast<uintptr_t>(N) * esz) & 15) &&
                     !(reinterpret_cast<uintptr_t>(codes) % (16 / esz));
  const PkRows r = pk_rows(M, N, packs ? 16 / esz : 0, ldx == N);
  const unsigned grid = ln_capped((r.items + 7) / 8, 16LL * place(st).sms);
#define LAB200_PACK(DT) \
  !packs && r.units ? pack8_any_kernel<DT, PK_U_ANY, true><<<grid, 256, 0, st>>>(x, ldx, c, s, N, r) \
  : !packs ? pack8_any_kernel<DT, PK_U_ANY, false><<<grid, 256, 0, st>>>(x, ldx, c, s, N, r) \
  : r.units ? pack8_kernel<DT, PK_U, true><<<grid, 256, 0, st>>>(x, ldx, c, s, r) : pack8_kernel<DT, PK_U, false><<<grid, 256, 0, st>>>(x, ldx, c, s, r)
  if (dtype == LAB200_F32) LAB200_PACK(SRMS_F32);
  else if (dtype == LAB200_F16) LAB200_PACK(SRMS_F16);
  else LAB200_PACK(SRMS_BF16);
#undef LAB200_PACK
  return launched();
}

int lab200_unpack8(const void* codes, const void* scales, void* y, long long M, int N, int dtype, void* stream) {
  if (!size_ok(M, N, N)) return LAB200_ERR_SHAPE;
  if (!dtype_known(dtype)) return LAB200_ERR_DTYPE;
  if (M == 0) return LAB200_OK;
  if (!y || !codes || !scales) return LAB200_ERR_SHAPE;
  const int esz = size_of(dtype);
  if (!whole(esz, y)) return LAB200_ERR_ALIGN;
  auto* c = static_cast<const int8_t*>(codes);
  auto* s = static_cast<const uint8_t*>(scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool packs = !((reinterpret_cast<uintptr_t>(y) | static_cast<uintptr_t>(N) * esz) & 15) && !(reinterpret_cast<uintptr_t>(codes) % (16 / esz));
  const PkRows r = pk_rows(M, N, packs ? 16 / esz : 0, true);
  const unsigned grid = ln_capped((r.items + 7) / 8, 16LL * place(st).sms);
#define LAB200_UNPACK(DT) \
  !packs && r.units ? unpack8_any_kernel<DT, PK_U_ANY, true><<<grid, 256, 0, st>>>(c, s, y, N, r) \
  : !packs ? unpack8_any_kernel<DT, PK_U_ANY, false><<<grid, 256, 0, st>>>(c, s, y, N, r) \
  : r.units ? unpack8_kernel<DT, PK_U, true><<<grid, 256, 0, st>>>(c, s, y, r) : unpack8_kernel<DT, PK_U, false><<<grid, 256, 0, st>>>(c, s, y, r)
  if (dtype == LAB200_F32) LAB200_UNPACK(SRMS_F32);
  else if (dtype == LAB200_F16) LAB200_UNPACK(SRMS_F16);
  else LAB200_UNPACK(SRMS_BF16);
#undef LAB200_UNPACK
  return launched();
}

}  // extern "C"
