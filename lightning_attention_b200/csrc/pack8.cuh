// 8-bit activation checkpoints: 32 consecutive values of a row share one exponent byte E, each keeps a signed byte.
//
//   step = 2^(E - 133);   code = rint(x / step), in [-127, 127];   value = code * step
//   E    = exponent field of the group's largest magnitude, one more where that would round to 128 steps; 7 <= E <= 254
//
// so a group's largest value is 63.5 to 127.5 steps and every value is off by at most half a step, 2^-7 of that largest value
// (values of 127.5 * 2^121 and above, where E is at its end, come back as 127 * 2^121). The step is a power of two so that
// scaling is exact: a code is one rounding of the exact quotient whatever computes it, and the value it stands for is exact in
// fp32 and bf16. A group that holds an infinity or a NaN has E = 255 and comes back as NaN.
#pragma once
#include <stdint.h>

#include "srmsnorm_kernels.cuh"

namespace lab200 {

constexpr int PK_GROUP = 32;

// Exponent byte of a group from the largest bit pattern of |x| (NaN > infinity > finite in that order).
__device__ __forceinline__ uint32_t pk_exponent(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  return min(max((amax_bits + 0x10000u) >> 23, 7u), 254u);
}
__device__ __forceinline__ float pk_step(uint32_t e) { return __uint_as_float(e == 255u ? 0x7fffffffu : (e - 6u) << 23); }
__device__ __forceinline__ float pk_inv_step(uint32_t e) { return __uint_as_float(e == 255u ? 0u : (260u - e) << 23); }
// The code of one value; a group of E = 255 gets zeros (inv = 0 makes 0 or NaN of its values, and NaN converts to 0).
__device__ __forceinline__ int pk_code(float x, float inv) { return min(max(__float2int_rn(x * inv), -127), 127); }

// A checkpoint's value in a 16-bit type: exact, but that a group's largest fp16 value may round up past 65504.
template <int DT>
__device__ __forceinline__ float pk_value(int code, float step) {
  float v = static_cast<float>(code) * step;
  if constexpr (DT == SRMS_F16) v = v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v;  // comparisons keep a NaN
  return v;
}

// The largest magnitude of P values, as bits; a NaN among them wins.
template <int P>
__device__ __forceinline__ uint32_t pk_abs_max(const float* f) {
  float m = fabsf(f[0]);
#pragma unroll
  for (int e = 1; e < P; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(f[e])));
  return __float_as_uint(m);
}
// Its maximum over LANES adjacent lanes, which hold one group.
template <int LANES>
__device__ __forceinline__ uint32_t pk_group_max(uint32_t bits) {
  if constexpr (LANES == 32) return __reduce_max_sync(0xffffffffu, bits);
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  return bits;
}
// P codes, four to a word. Adding 1.5 * 2^23 rounds to a whole number, to nearest even, and leaves it in the low byte: exact, as
// x * inv is. Groups of E = 254 (whose codes may have to be held at 127) and 255 take the checked way.
template <int P>
__device__ __forceinline__ void pk_codes(const float* f, uint32_t e, uint32_t* w) {
  const float inv = pk_inv_step(e);
  uint32_t c[P];
  if (e < 254u) {
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = __float_as_uint(fmaf(f[i], inv, 12582912.f));
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = static_cast<uint32_t>(pk_code(f[i], inv));
  }
  if constexpr (P == 1) {
    w[0] = c[0];
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 4) w[i / 4] = __byte_perm(__byte_perm(c[i], c[i + 1], 0x0040), __byte_perm(c[i + 2], c[i + 3], 0x0040), 0x5410);
  }
}
// Two adjacent codes of a word as fp32 values: a byte b, moved by 128, in the low byte of 2^23 makes 2^23 + b + 128.
__device__ __forceinline__ unsigned long long pk_two(uint32_t w, int e) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t lo = __byte_perm(u, 0x4b000000u, 0x7440 + e), hi = __byte_perm(u, 0x4b000000u, 0x7441 + e);
  unsigned long long v, r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  asm("{ .reg .b64 c; mov.b64 c, {%2, %2}; add.rn.f32x2 %0, %1, c; }" : "=l"(r) : "l"(v), "r"(__float_as_uint(-8388736.f)));
  return r;
}

// A warp per group, a lane per value: any row length, stride and alignment.
template <int DT>
__global__ void __launch_bounds__(256)
pack8_any_kernel(const void* __restrict__ x_, long long ldx, int8_t* __restrict__ codes, uint8_t* __restrict__ scales, long long M, int N) {
  using E = SrmsElem<DT>;
  const auto* x = static_cast<const typename E::T*>(x_);
  const int ng = (N - 1) / PK_GROUP + 1, lane = threadIdx.x & 31;
  const long long total = M * ng, step = static_cast<long long>(gridDim.x) * 8;
  for (long long g = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); g < total; g += step) {
    const long long row = g / ng;
    const int col = static_cast<int>(g - row * ng) * PK_GROUP + lane;
    const bool on = lane < N - (col - lane);
    const float v = on ? E::ld(x + row * ldx + col) : 0.f;
    const uint32_t e = pk_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(v))));
    if (on) codes[row * N + col] = static_cast<int8_t>(pk_code(v, pk_inv_step(e)));
    if (lane == 0) scales[g] = static_cast<uint8_t>(e);
  }
}

template <int DT>
__global__ void __launch_bounds__(256)
unpack8_any_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y_, long long M, int N) {
  using E = SrmsElem<DT>;
  auto* y = static_cast<typename E::T*>(y_);
  const int ng = (N - 1) / PK_GROUP + 1, lane = threadIdx.x & 31;
  const long long total = M * ng, step = static_cast<long long>(gridDim.x) * 8;
  for (long long g = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); g < total; g += step) {
    const long long row = g / ng;
    const int col = static_cast<int>(g - row * ng) * PK_GROUP + lane;
    if (lane < N - (col - lane)) E::st(y + row * N + col, pk_value<DT>(codes[row * N + col], pk_step(scales[g])));
  }
}

}  // namespace lab200
