// Layer norm with weight and bias, alone or followed by a sigmoid gate, forward and backward for sm_100a.
//
//   forward : m = mean(x); r = 1 / sqrt(mean((x - m)^2) + eps); xh = (x - m) r; n = xh w + b; y = n, or n s with s = sigmoid(gate)
//   backward: t = dy, or dy s; u = t w
//             dx = r (u - mean(u) - xh mean(u xh));  dw = sum over rows of t xh;  db = sum over rows of t
//             dgate = dy n s (1 - s)
// In place of x and gate the backward pass may take their 8-bit checkpoints (pack8.cuh), which the forward pass then writes.
//
// Statistics and sums are fp32. The variance is taken around the computed mean and corrected by what that mean was off by, so a
// row whose values are far from zero loses nothing to its offset in y. Sums over rows go through partial sums of a fixed order
// (no atomics): a call's results are the same every time.
#pragma once
#include "pack8.cuh"

namespace lab200 {

struct LnArgs {
  const void *x, *gate;          // gate NULL: none
  long long ldx, ldg;            // elements from one row to the next
  int8_t *xcodes, *gcodes;       // forward: written where not NULL; backward: read in place of x, gate where not NULL
  uint8_t *xscales, *gscales;
  const void *weight, *bias;     // NULL: ones, zeros
  int wdt;                       // their type
  void* y;
  float2* stats;                 // (m, r) of each row; forward: NULL where nobody wants them
  const void* dy;
  long long lddy;
  void *dx, *dgate, *dw, *db;    // NULL: not wanted
  float* partial;                // [nparts][2][N]: a part of dw and db each
  int nparts;
  long long M;
  int N;
  float eps;
};

__device__ __forceinline__ float ln_param(const void* p, int wdt, int i, float without) {
  if (!p) return without;
  if (wdt == SRMS_F32) return static_cast<const float*>(p)[i];
  if (wdt == SRMS_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void ln_param_out(void* p, int wdt, int i, float v) {
  if (!p) return;
  if (wdt == SRMS_F32) static_cast<float*>(p)[i] = v;
  else if (wdt == SRMS_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// sigmoid(v) and sigmoid(-v). exp(80) is finite and sigmoid(-80) = 2e-35 nothing next to 1, so the bound changes no result and
// keeps inf * 0 out; a NaN passes the comparison.
__device__ __forceinline__ void ln_sigmoid(float v, float* s, float* rest) {
  const float e = __expf(v < -80.f ? 80.f : -v);
  *s = __fdividef(1.f, 1.f + e);
  *rest = e * *s;
}

// 1 / sqrt(variance + eps) from the means of d and d^2, d = x - (the mean as computed). A NaN stays one.
__device__ __forceinline__ float ln_rstd(float d1, float d2, float eps) {
  const float v = d2 - d1 * d1;
  return 1.f / sqrtf((v < 0.f ? 0.f : v) + eps);
}

// One value of x or gate in the backward pass, from the tensor or from its checkpoint.
template <int DT>
__device__ __forceinline__ float ln_saved(const void* p, long long ld, const int8_t* codes, const uint8_t* scales, long long row, int col, int N) {
  if (codes) return pk_value<SRMS_F32>(codes[row * N + col], pk_step(scales[row * ((N - 1) / PK_GROUP + 1) + col / PK_GROUP]));
  return SrmsElem<DT>::ld(static_cast<const typename SrmsElem<DT>::T*>(p) + row * ld + col);
}

// ---- rows of any length, stride and alignment: a CTA per row, element by element, each row read again for each sum ----------
template <int DT>
__global__ void __launch_bounds__(256) ln_fwd_any_kernel(const LnArgs a) {
  using E = SrmsElem<DT>;
  using T = typename E::T;
  __shared__ float red[16];
  const int N = a.N, lane = threadIdx.x & 31;
  const float inv_n = 1.f / static_cast<float>(N);
  for (long long row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* g = a.gate ? static_cast<const T*>(a.gate) + row * a.ldg : nullptr;
    T* y = static_cast<T*>(a.y) + row * N;
    float s = 0.f;
    for (int i = threadIdx.x; i < N; i += 256) s += E::ld(x + i);
    const float m = group_sum<256>(s, red, threadIdx.x) * inv_n;
    float d1 = 0.f, d2 = 0.f;
    for (int i = threadIdx.x; i < N; i += 256) { const float d = E::ld(x + i) - m; d1 += d; d2 = fmaf(d, d, d2); }
    d1 = group_sum<256>(d1, red, threadIdx.x) * inv_n;
    d2 = group_sum<256>(d2, red, threadIdx.x) * inv_n;
    const float r = ln_rstd(d1, d2, a.eps);
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(m + d1, r);
    for (int i = threadIdx.x; i < N; i += 256) {
      float v = fmaf((E::ld(x + i) - m - d1) * r, ln_param(a.weight, a.wdt, i, 1.f), ln_param(a.bias, a.wdt, i, 0.f));
      if (g) {
        float sg, rest;
        ln_sigmoid(E::ld(g + i), &sg, &rest);
        v *= sg;
      }
      E::st(y + i, v);
    }
    if (a.xcodes) {
      const int ng = (N - 1) / PK_GROUP + 1;
      for (int k = threadIdx.x >> 5; k < ng; k += 8) {
        const int i = k * PK_GROUP + lane;
        const bool on = lane < N - k * PK_GROUP;
        const float v = on ? E::ld(x + i) : 0.f;
        const uint32_t e = pk_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(v))));
        if (on) a.xcodes[row * N + i] = static_cast<int8_t>(pk_code(v, pk_inv_step(e)));
        if (lane == 0) a.xscales[row * ng + k] = static_cast<uint8_t>(e);
        if (g) {
          const float u = on ? E::ld(g + i) : 0.f;
          const uint32_t f = pk_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(u))));
          if (on) a.gcodes[row * N + i] = static_cast<int8_t>(pk_code(u, pk_inv_step(f)));
          if (lane == 0) a.gscales[row * ng + k] = static_cast<uint8_t>(f);
        }
      }
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(256) ln_bwd_any_kernel(const LnArgs a) {
  using E = SrmsElem<DT>;
  using T = typename E::T;
  __shared__ float red[16];
  const int N = a.N;
  const float inv_n = 1.f / static_cast<float>(N);
  const bool gated = a.gate || a.gcodes;
  for (long long row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float2 st = a.stats[row];
    float c1 = 0.f, c2 = 0.f;
    for (int i = threadIdx.x; i < N; i += 256) {
      const float xh = (ln_saved<DT>(a.x, a.ldx, a.xcodes, a.xscales, row, i, N) - st.x) * st.y;
      float t = E::ld(dy + i);
      if (gated) {
        float sg, rest;
        ln_sigmoid(ln_saved<DT>(a.gate, a.ldg, a.gcodes, a.gscales, row, i, N), &sg, &rest);
        const float n = fmaf(xh, ln_param(a.weight, a.wdt, i, 1.f), ln_param(a.bias, a.wdt, i, 0.f));
        if (a.dgate) E::st(static_cast<T*>(a.dgate) + row * N + i, t * n * sg * rest);
        t *= sg;
      }
      const float u = t * ln_param(a.weight, a.wdt, i, 1.f);
      c1 += u;
      c2 = fmaf(u, xh, c2);
    }
    c1 = group_sum<256>(c1, red, threadIdx.x) * inv_n;
    c2 = group_sum<256>(c2, red, threadIdx.x) * inv_n;
    if (!a.dx) continue;
    for (int i = threadIdx.x; i < N; i += 256) {
      const float xh = (ln_saved<DT>(a.x, a.ldx, a.xcodes, a.xscales, row, i, N) - st.x) * st.y;
      float t = E::ld(dy + i);
      if (gated) {
        float sg, rest;
        ln_sigmoid(ln_saved<DT>(a.gate, a.ldg, a.gcodes, a.gscales, row, i, N), &sg, &rest);
        t *= sg;
      }
      E::st(static_cast<T*>(a.dx) + row * N + i, (t * ln_param(a.weight, a.wdt, i, 1.f) - c1 - xh * c2) * st.y);
    }
  }
}

// Part blockIdx.y of dw and db of 32 columns: eight warps take every eighth row of the part's.
template <int DT>
__global__ void __launch_bounds__(256) ln_bwd_columns_kernel(const LnArgs a) {
  using E = SrmsElem<DT>;
  using T = typename E::T;
  __shared__ float red[2][8][32];
  const int N = a.N, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long per = (a.M + a.nparts - 1) / a.nparts, lo = per * blockIdx.y, hi = min(a.M, lo + per);
  const bool gated = a.gate || a.gcodes;
  for (long long c0 = static_cast<long long>(blockIdx.x) * 32; c0 < N; c0 += static_cast<long long>(gridDim.x) * 32) {
    const int col = static_cast<int>(c0) + lane;
    float dw = 0.f, db = 0.f;
    if (lane < N - c0) {
      for (long long row = lo + warp; row < hi; row += 8) {
        const float2 st = a.stats[row];
        const float xh = (ln_saved<DT>(a.x, a.ldx, a.xcodes, a.xscales, row, col, N) - st.x) * st.y;
        float t = E::ld(static_cast<const T*>(a.dy) + row * a.lddy + col);
        if (gated) {
          float sg, rest;
          ln_sigmoid(ln_saved<DT>(a.gate, a.ldg, a.gcodes, a.gscales, row, col, N), &sg, &rest);
          t *= sg;
        }
        dw = fmaf(t, xh, dw);
        db += t;
      }
    }
    red[0][warp][lane] = dw;
    red[1][warp][lane] = db;
    __syncthreads();
    if (warp < 2 && lane < N - c0) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += red[warp][k][lane];
      a.partial[(static_cast<size_t>(blockIdx.y) * 2 + warp) * N + col] = s;
    }
    __syncthreads();
  }
}

// dw and db from their parts: a CTA per 32 columns, its eight warps take every eighth part. No part: zeros.
__global__ void __launch_bounds__(256) ln_bwd_join_kernel(const float* __restrict__ partial, int nparts, int N, void* dw, void* db, int wdt) {
  __shared__ float red[2][8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long c0 = static_cast<long long>(blockIdx.x) * 32; c0 < N; c0 += static_cast<long long>(gridDim.x) * 32) {
    const int col = static_cast<int>(c0) + lane;
    const bool on = lane < N - c0;
    float s[2] = {0.f, 0.f};
    for (int p = warp; on && p < nparts; p += 8) {
      s[0] += partial[(static_cast<size_t>(p) * 2) * N + col];
      s[1] += partial[(static_cast<size_t>(p) * 2 + 1) * N + col];
    }
    red[0][warp][lane] = s[0];
    red[1][warp][lane] = s[1];
    __syncthreads();
    if (warp < 2 && on) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += red[warp][k][lane];
      ln_param_out(warp ? db : dw, wdt, col, v);
    }
    __syncthreads();
  }
}

}  // namespace lab200
