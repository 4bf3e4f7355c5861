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
  bool vec_params;               // and whether they may be read 16 bytes at a time
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

// sigmoid(v) and sigmoid(-v) from -v / ln 2: 1 / (1 + e) and e / (1 + e), e = 2^(-v / ln 2) by the approximate instructions
// (relative errors of 2^-22). The bound on e keeps inf * 0 out: with it sigmoid(v) stays at 2^-116 where it would go on to zero. A NaN
// passes it.
constexpr float LN_MINUS_LOG2E = -1.4426950408889634f;
__device__ __forceinline__ void ln_sigmoid2(float arg, float* s, float* rest) {
  float e;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(e) : "f"(arg), "f"(116.f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(*s) : "f"(1.f + e));
  *rest = e * *s;
}
__device__ __forceinline__ void ln_sigmoid(float v, float* s, float* rest) { ln_sigmoid2(v * LN_MINUS_LOG2E, s, rest); }

// 1 / sqrt(variance + eps) from the means of d and d^2, d = x - (the mean as computed). A NaN stays one.
__device__ __forceinline__ float ln_rstd(float d1, float d2, float eps) {
  const float v = d2 - d1 * d1;
  return 1.f / sqrtf((v < 0.f ? 0.f : v) + eps);
}

// One value of x or gate in the backward pass, from the tensor or from its checkpoint.
template <int DT>
__device__ __forceinline__ float ln_saved(const void* p, long long ld, const int8_t* codes, const uint8_t* scales, long long row, int col, int N) {
  if (codes) return static_cast<float>(codes[row * N + col]) * (pk_step(scales[row * ((N - 1) / PK_GROUP + 1) + col / PK_GROUP]));
  return SrmsElem<DT>::ld(static_cast<const typename SrmsElem<DT>::T*>(p) + row * ld + col);
}

// ---- rows of any length, stride and alignment: a CTA per row, element by element, each row read again for each sum ----------
// For C callers' rows that the Python operators would copy, and for rows past what teams hold:
//   rows that packs divide      forward 16384 values of 16 bits (gated 11872: shared memory), 8192 of 32; backward 8192
//   rows that packs do not      8185 of 16 bits, 8189 of 32; gated, backward, 4089 and 4093: weight and bias of columns that each team has for
//                               itself stay in registers beside the two sums, and with 16 values a thread they do not fit
// Bound by instructions: 32768 x 4096 bf16 in 1040 us, both passes.
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

// ---- rows in packs of 16 bytes ---------------------------------------------------------------------------------------------
// A pack is P = 8 (16-bit) or 4 (fp32) values. Copies into shared memory run ahead (cp.async), every value comes from memory once in
// each pass, and CTAs walk over the rows with what belongs to the columns at hand.
//
// ODD: rows of a contiguous tensor whose length P does not divide. The packs are those of the whole tensor: a row begins `shift` =
// row * N mod P values into its first one and shares that and its last one with its neighbours. Teams take every so-manieth row
// with a step that is a multiple of the shifts' period, so that a team's shift, and with it each thread's columns, stay the same.
struct LnPackEdge { int lo, hi; };  // the values of a pack that belong to the row
template <int P, bool ODD>
__device__ __forceinline__ LnPackEdge ln_edge(int k, int shift, int N) {
  return {ODD && k == 0 ? shift : 0, ODD ? min(P, N + shift - k * P) : P};
}

// Two fp32 values in one 64-bit register: the packed arithmetic of sm_100 does both at once.
using f2 = unsigned long long;
__device__ __forceinline__ f2 f2_of(float lo, float hi) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ f2 f2_all(float v) { return f2_of(v, v); }
__device__ __forceinline__ float2 f2_get(f2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ float f2_sum(f2 v) { const float2 t = f2_get(v); return t.x + t.y; }

// Copies of 4, 8 or 16 bytes into shared memory that the thread does not wait for; with a size, so many are read and the rest is zero.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int n) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `stages` - 2 of the thread's groups are under way.
__device__ __forceinline__ void copies_wait(int stages) {
  if (stages == 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
}
__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 shared_f4(uint32_t at) {
  const uint4 v = shared16(at);
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ void shared_put(uint32_t at, float4 v) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

template <int DT>
struct LnPack {
  static constexpr int ESZ = DT == SRMS_F32 ? 4 : 2, P = 16 / ESZ, H = P / 2;
  static constexpr int LANES = PK_GROUP / P;  // adjacent packs that hold one group of a checkpoint
  using T = typename SrmsElem<DT>::T;

  __device__ static void unpack(const uint4& raw, f2* out) {
    float f[P];
    SrmsVec<DT>::unpack(raw, f);
#pragma unroll
    for (int j = 0; j < H; ++j) out[j] = f2_of(f[2 * j], f[2 * j + 1]);
  }
  __device__ static void floats(const f2* v, float* f) {
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const float2 t = f2_get(v[j]);
      f[2 * j] = t.x; f[2 * j + 1] = t.y;
    }
  }
  __device__ static void store(void* to, const f2* in) {
    float f[P];
    floats(in, f);
    SrmsPack<1> o;
    o.q[0] = SrmsVec<DT>::pack(f);
    st_stream<1>(static_cast<SrmsPack<1>*>(to), o);
  }
  // P values of weight or bias (`p` NULL: `without`), whatever their type and alignment.
  __device__ static void params(const void* p, int wdt, bool vec, int k, float without, float* f) {
#pragma unroll
    for (int e = 0; e < P; ++e) f[e] = without;
    if (!p) return;
    if (!vec) {
#pragma unroll
      for (int e = 0; e < P; ++e) f[e] = ln_param(p, wdt, k * P + e, without);
    } else if (wdt == SRMS_F32) {
#pragma unroll
      for (int e = 0; e < P; e += 4) *reinterpret_cast<float4*>(f + e) = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + k * P + e));
    } else if constexpr (DT != SRMS_F32) {
      SrmsVec<DT>::unpack(__ldg(static_cast<const uint4*>(p) + k), f);
    }
  }
  // Odd rows: zeros in place of the values of a pack that belong to another row, those before `lo` and from `hi` on.
  __device__ static void cut(f2* v, int lo, int hi) {
    float f[P];
    floats(v, f);
#pragma unroll
    for (int j = 0; j < H; ++j)
      v[j] = f2_of(2 * j >= lo && 2 * j < hi ? f[2 * j] : 0.f, 2 * j + 1 >= lo && 2 * j + 1 < hi ? f[2 * j + 1] : 0.f);
  }
  // Stores the values from `lo` to `hi` - 1 of a pack.
  __device__ static void store_part(void* to, const f2* in, int lo, int hi) {
    float f[P];
    floats(in, f);
#pragma unroll
    for (int e = 0; e < P; ++e)
      if (e >= lo && e < hi) SrmsElem<DT>::st(static_cast<T*>(to) + e, f[e]);
  }
  // Weight or bias from column c on, of which some may be no columns.
  __device__ static void params_at(const void* p, int wdt, int c, int N, float without, f2* out) {
    float f[P];
#pragma unroll
    for (int e = 0; e < P; ++e) f[e] = c + e >= 0 && c + e < N ? ln_param(p, wdt, c + e, without) : without;
#pragma unroll
    for (int j = 0; j < H; ++j) out[j] = f2_of(f[2 * j], f[2 * j + 1]);
  }
  // The checkpoint of pack k of a row (its words, and its values), whose group LANES adjacent lanes hold; all lanes of a warp call
  // it, `on`: there is such a pack.
  __device__ static void quantise(const uint4& words, const f2* x, int8_t* codes, uint8_t* scales, int k, bool on) {
    const uint32_t ex = pk_pack_exponent<DT>(words);
    uint32_t w[P / 4];
    pk_pack_codes<P>(x, ex, w);
    if (on) {
      if constexpr (P == 8) reinterpret_cast<uint2*>(codes)[k] = make_uint2(w[0], w[1]);
      else reinterpret_cast<uint32_t*>(codes)[k] = w[0];
      if (k % LANES == 0) scales[k / LANES] = static_cast<uint8_t>(ex);
    }
  }
  // P fp32 values for each pack, in planes of four: what adjacent lanes read lies next to each other.
  __device__ static void plane_put(uint32_t plane, int npack, int k, const float* f) {
#pragma unroll
    for (int e = 0; e < P; e += 4) shared_put(plane + (e / 4 * npack + k) * 16, make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]));
  }
  __device__ static void plane_get(uint32_t plane, int npack, int k, f2* out) {
#pragma unroll
    for (int e = 0; e < P; e += 4) {
      const float4 v = shared_f4(plane + (e / 4 * npack + k) * 16);
      out[e / 2] = f2_of(v.x, v.y);
      out[e / 2 + 1] = f2_of(v.z, v.w);
    }
  }
};

extern __shared__ __align__(16) char ln_shared[];

// ---- forward -----------------------------------------------------------------------------------------------------------------
// A row is a team's of T threads, V packs a thread: T a power of two up to 32 (several rows in a warp) or a multiple of 32. A warp
// has the mean and the squares about it of its part of a row from shuffles; the parts are joined by the formula for the variance of
// a union, a lane to a part, behind the only barrier of a row. Each thread has places of its own in the ring of copies, so that it needs none.
// Most threads of a CTA: 20 warps of up to 96 registers hide more than 16 of 128 do (32768 x 4096 bf16: 91 us, 100; 16384 x 5120 gated,
// writing checkpoints: 122, 130). Gated rows of which the copies of 640 threads do not fit beside weight and bias (from 7784 values on) take 512,
// up to 11872 values: 8192 x 8192 gated, writing checkpoints, 103 us, 403 value by value.
// So do fp32 rows of several warps that packs do not divide, whose weight and bias are in registers: 8192 x 1001 gated 22 us, 25 with 640 threads.
// Bound by memory without a gate or checkpoints (5.9 TB/s at 32768 x 4096 bf16), else by instructions too (with both 187 us, 5.8 TB/s).
constexpr int LN_FWD_THREADS = 640, LN_FWD_FEWER = 512;

// Strides from one of a team's rows to its next, in bytes: all teams' rows at once. As arguments they cost the kernels no registers.
struct LnSteps {
  long long rows, x, gate, dy, out, codes, scales;
  LnSteps() = default;
  LnSteps(const LnArgs& a, int esz, long long all_teams)
      : rows(all_teams), x(all_teams * a.ldx * esz), gate(all_teams * a.ldg * esz), dy(all_teams * a.lddy * esz), out(all_teams * a.N * esz),
        codes(all_teams * a.N), scales(all_teams * ((a.N - 1) / PK_GROUP + 1)) {}
};

// parts: the warps of a team of several, rounded up to 4, 8 or 16, less one.
struct LnFwdPlan { int T, stages, parts; LnSteps step; };

template <int DT, int V, int G, bool ODD, bool GATE, bool SAVE, int THREADS = LN_FWD_THREADS>
__global__ void __launch_bounds__(THREADS) ln_fwd_kernel(const LnArgs a, const LnFwdPlan plan) {
  using K = LnPack<DT>;
  constexpr int P = K::P, H = K::H;
  static_assert(!(ODD && SAVE), "groups of 32 values do not keep to the packs of odd rows");
  // of each team's warps: mean, squares, count of their part; two halves in turn. What a team does not fill has a count of zero.
  constexpr int WARPS = THREADS / 32, TEAMS = G > 32 ? THREADS / 64 : 1;
  __shared__ float4 slots[TEAMS][2][WARPS];
  const int T = G <= 32 ? G : plan.T, team = threadIdx.x / T, t = threadIdx.x - team * T, lanes = blockDim.x, warp = t >> 5;
  const int N = a.N, ng = (N - 1) / PK_GROUP + 1, teams = lanes / T;
  const uint32_t wplane = static_cast<uint32_t>(__cvta_generic_to_shared(ln_shared)), bplane = wplane + N * 4, ring = (ODD ? wplane : bplane + N * 4) + threadIdx.x * 16;
  constexpr uint32_t PITCH = THREADS * 16, STAGE = PITCH * V * (GATE ? 2 : 1);
  const uint32_t ring_end = plan.stages * STAGE;
  if constexpr (G > 32)
    for (int i = threadIdx.x; i < TEAMS * 2 * WARPS; i += lanes) slots[0][0][i] = make_float4(0.f, 0.f, 0.f, 0.f);
  const long long row = static_cast<long long>(blockIdx.x) * teams + team;
  const long long first = G < 32 ? static_cast<long long>(blockIdx.x) * teams + (threadIdx.x & ~31) / T : row;
  // rows of this team, and of the team in its warp that has most
  const int mine = row < a.M ? static_cast<int>((a.M - 1 - row) / plan.step.rows) + 1 : 0;
  const int most = G >= 32 ? mine : first < a.M ? static_cast<int>((a.M - 1 - first) / plan.step.rows) + 1 : 0;
  const int shift = ODD ? static_cast<int>(row * N % P) : 0, npack = (N + shift + P - 1) / P;
  const char *x_from = static_cast<const char*>(a.x) + (row * a.ldx - shift) * K::ESZ + t * 16, *g_from = static_cast<const char*>(a.gate) + (row * a.ldg - shift) * K::ESZ + t * 16;
  uint32_t in = 0, out = 0;
  const auto start = [&](int n) {
    if (n < mine) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (t + i * T < npack) {
          if constexpr (ODD) {
            const int size = ln_edge<P, ODD>(t + i * T, shift, N).hi * K::ESZ;
            copy_async<16>(ring + in + i * PITCH, x_from + i * T * 16, size);
            if constexpr (GATE) copy_async<16>(ring + in + (V + i) * PITCH, g_from + i * T * 16, size);
          } else {
            copy_async<16>(ring + in + i * PITCH, x_from + i * T * 16);
            if constexpr (GATE) copy_async<16>(ring + in + (V + i) * PITCH, g_from + i * T * 16);
          }
        }
    }
    copies_commit();
    x_from += plan.step.x;
    if constexpr (GATE) g_from += plan.step.gate;
    in = in + STAGE == ring_end ? 0 : in + STAGE;
  };
  for (int k = 1; k < plan.stages; ++k) start(k - 1);
  // weight and bias: in shared memory, or, where each team has columns of its own in a pack, in registers
  f2 wr[ODD ? V : 1][H], br[ODD ? V : 1][H];
  if constexpr (ODD) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      K::params_at(a.weight, a.wdt, (t + i * T) * P - shift, N, 1.f, wr[i]);
      K::params_at(a.bias, a.wdt, (t + i * T) * P - shift, N, 0.f, br[i]);
    }
  } else {
    for (int k = threadIdx.x; k < npack; k += lanes) {
      float f[P];
      K::params(a.weight, a.wdt, a.vec_params, k, 1.f, f);
      K::plane_put(wplane, npack, k, f);
      K::params(a.bias, a.wdt, a.vec_params, k, 0.f, f);
      K::plane_put(bplane, npack, k, f);
    }
  }
  if constexpr (!ODD || G > 32) __syncthreads();
  int count = 0;  // values of a row that this warp (or sub-warp team) has
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const LnPackEdge e = ln_edge<P, ODD>(t + i * T, shift, N);
    count += t + i * T < npack ? e.hi - e.lo : 0;
  }
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
  const float fcount = static_cast<float>(count), inv_count = count ? 1.f / fcount : 0.f, inv_n = 1.f / static_cast<float>(N);
  int turn = 0;
  char* y = static_cast<char*>(a.y) + (row * N - shift) * K::ESZ + t * 16;
  int8_t* xc = SAVE ? a.xcodes + row * N : nullptr;
  uint8_t* xs = SAVE ? a.xscales + row * ng : nullptr;
  const long long gate_codes = a.gcodes - a.xcodes, gate_scales = a.gscales - a.xscales;  // from x's to the gate's
  float2* stats = a.stats ? a.stats + row : nullptr;
  for (int n = 0; n < most; ++n, y += plan.step.out) {
    const bool live = G >= 32 || n < mine;
    copies_wait(plan.stages);
    uint4 raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = live && t + i * T < npack ? shared16(ring + out + i * PITCH) : make_uint4(0, 0, 0, 0);
    const uint32_t gates = ring + out + V * PITCH;
    out = out + STAGE == ring_end ? 0 : out + STAGE;
    start(n + plan.stages - 1);
    f2 v[V][H];
    f2 s = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      K::unpack(raw[i], v[i]);
      const LnPackEdge e = ln_edge<P, ODD>(t + i * T, shift, N);
      if (ODD && (e.lo > 0 || e.hi < P)) K::cut(v[i], e.lo, e.hi);
      f2 part = v[i][0];
#pragma unroll
      for (int j = 1; j < H; ++j) part = f2_add(part, v[i][j]);
      s = f2_add(s, part);
      if constexpr (SAVE) K::quantise(raw[i], v[i], xc, xs, t + i * T, live && t + i * T < npack);
    }
    float m = f2_sum(s);
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    m *= inv_count;
    const f2 minus_m = f2_all(-m);
    f2 d1 = 0, d2 = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f2 p1 = 0, p2 = 0;
#pragma unroll
      for (int j = 0; j < H; ++j) v[i][j] = f2_add(v[i][j], minus_m);
      const LnPackEdge e = ln_edge<P, ODD>(t + i * T, shift, N);
      if (ODD && (e.lo > 0 || e.hi < P)) K::cut(v[i], e.lo, e.hi);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        p1 = f2_add(p1, v[i][j]);
        p2 = f2_fma(v[i][j], v[i][j], p2);
      }
      if (t + i * T < npack) {  // packs behind the row's end take no part
        d1 = f2_add(d1, p1);
        d2 = f2_add(d2, p2);
      }
    }
    float q1 = f2_sum(d1), q2 = f2_sum(d2);
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
      q1 += __shfl_xor_sync(0xffffffffu, q1, o);
      q2 += __shfl_xor_sync(0xffffffffu, q2, o);
    }
    // what the warp's mean was off by, and the squares about the corrected one
    float mean = q1 * inv_count;  // counted from m
    float squares = fmaf(-mean, q1, q2);
    if constexpr (G > 32) {
      float4* slot = slots[team][turn];
      if ((t & 31) == 0) slot[warp] = make_float4(m + mean, squares, fcount, 0.f);
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(T) : "memory");
      // A lane takes a part. The row's mean first, counted from the first part's, then the squares about it: a sum of positive terms, so that a
      // short part far from the rest (a last warp of four values, outliers) cancels nothing, and all warps get the same mean and spread.
      const float4 part = slot[t & plan.parts];
      const float ref = slot[0].x;
      const auto over_parts = [&](float s) {
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (plan.parts > 3) s += __shfl_xor_sync(0xffffffffu, s, 4);
        if (plan.parts > 7) s += __shfl_xor_sync(0xffffffffu, s, 8);
        return s;
      };
      const float from_ref = over_parts(part.z * (part.x - ref)) * inv_n, d = part.x - ref - from_ref;
      squares = over_parts(fmaf(part.z * d, d, part.y));
      mean = ref - m + from_ref;
      turn ^= 1;
    }
    squares *= inv_n;
    const float r = 1.f / sqrtf((squares < 0.f ? 0.f : squares) + a.eps);
    if (stats && t == 0 && live) *stats = make_float2(m + mean, r);
    if (a.stats) stats += plan.step.rows;
    const f2 off = f2_all(-mean * r), rr = f2_all(r);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int k = t + i * T;
      const bool on = live && k < npack;
      f2 u[H];
      if constexpr (GATE) {
        const uint4 words = on ? shared16(gates + i * PITCH) : make_uint4(0, 0, 0, 0);
        K::unpack(words, u);
        if constexpr (SAVE) K::quantise(words, u, xc + gate_codes, xs + gate_scales, k, on);
#pragma unroll
        for (int j = 0; j < H; ++j) u[j] = f2_mul(u[j], f2_all(LN_MINUS_LOG2E));
      }
      if (on) {
        f2 w[H], b[H];
        if constexpr (!ODD) {
          K::plane_get(wplane, npack, k, w);
          K::plane_get(bplane, npack, k, b);
        }
#pragma unroll
        for (int j = 0; j < H; ++j) {
          v[i][j] = f2_fma(f2_fma(v[i][j], rr, off), ODD ? wr[ODD ? i : 0][j] : w[j], ODD ? br[ODD ? i : 0][j] : b[j]);
          if constexpr (GATE) {
            const float2 gv = f2_get(u[j]);
            float s0, s1, rest;
            ln_sigmoid2(gv.x, &s0, &rest);
            ln_sigmoid2(gv.y, &s1, &rest);
            v[i][j] = f2_mul(v[i][j], f2_of(s0, s1));
          }
        }
        const LnPackEdge e = ln_edge<P, ODD>(k, shift, N);
        if (ODD && (e.lo > 0 || e.hi < P)) K::store_part(y + i * T * 16, v[i], e.lo, e.hi);
        else K::store(y + i * T * 16, v[i]);
      }
    }
    if constexpr (SAVE) {
      xc += plan.step.codes;
      xs += plan.step.scales;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- backward ----------------------------------------------------------------------------------------------------------------
// A row is a team's of T threads, V packs a thread (E = P V values), as in the forward pass, and a thread's columns are the same for
// all rows: it sums dw and db in registers. The copies of a row's dy, x and gate (or their checkpoints) run some rows ahead, into
// places that are each thread's own. Bound by memory where an SM holds two teams or more (32768 x 4096 bf16: 134 us, 6.0 TB/s), by
// instructions and the chain of a row with checkpoints and a gate (219 us, 5.0 TB/s).
//
// WIDE: rows for 257 to 320 threads, in 16 bits and without a gate, have two teams to an SM in 640 threads of 96 registers, where 512 threads
// of 128 have one. For this a row's values are not kept over its barrier but taken from the ring and worked out again behind it, and the
// weight is in shared memory. 16384 x 5120 bf16: 92 us, 109 with one team; from checkpoints 106 and 112. fp32 160 and 156, from checkpoints
// 177 and 166: not there.
constexpr int LN_BWD_THREADS = 512, LN_BWD_WIDE = 640;  // most of a CTA
constexpr int LN_BWD_SLOTS = LN_BWD_THREADS / 64 * 2 * 128;  // two halves of 16 warps' two sums for each team of several warps

struct LnBwdPlan { int T, stages; LnSteps step; };

// What a team reads row by row: a tensor, or (SAVED) its checkpoint.
// PLACE: bytes from a thread's place for one pack to that for the next.
template <int DT, int V, int LANES, bool ODD, bool SAVED>
struct LnRows {
  using K = LnPack<DT>;
  static constexpr int P = K::P, H = K::H, PACK = SAVED ? P : 16, UNIT = PACK / P, PLACE = LANES * PACK, BYTES = V * PLACE;
  const char *p, *base;   // the thread's first pack of the row to start; somewhere in the tensor
  const uint8_t* e_from;  // the exponents of the row after the one at hand, those of the thread's first pack (ODD: of the row)
  uint32_t at;
  uint32_t e[SAVED ? V : 1], e2[SAVED && ODD ? V : 1];  // of a pack's group, and of the next one where the pack reaches into that

  __device__ void init(const void* tensor, long long ld, const int8_t* codes, const uint8_t* scales, int N, long long row, int t, int shift, uint32_t ring) {
    base = SAVED ? reinterpret_cast<const char*>(codes) : static_cast<const char*>(tensor);
    const long long pitch = SAVED ? N : ld;
    p = base + (row * pitch - shift) * UNIT + t * PACK;
    at = ring + threadIdx.x * PACK;
    if constexpr (SAVED) {
      const int ng = (N - 1) / PK_GROUP + 1;
      e_from = scales + row * ng + (ODD ? 0 : t / K::LANES);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        e[i] = 7;
        if constexpr (ODD) e2[i] = 7;
      }
    }
  }
  // Zeros in the thread's places of a stage: packs behind the row's end are not copied.
  __device__ void clear(uint32_t stage) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int w = 0; w < PACK / 4; ++w) asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + at + i * PLACE + 4 * w), "r"(0) : "memory");
  }
  // FILL: teams that share a warp, of which one may have no row: its places become zero.
  template <bool FILL>
  __device__ void start(uint32_t stage, bool live, int t, int T, int npack, int shift, int N, long long step) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (t + i * T < npack) {
        const char* from = p + i * T * PACK;
        const uint32_t to = stage + at + i * PLACE;
        if (FILL && !live) {
          copy_async<PACK>(to, base, 0);
        } else if constexpr (!ODD) {
          copy_async<PACK>(to, from);
        } else {
          const int n = ln_edge<P, ODD>(t + i * T, shift, N).hi * UNIT;
          if (SAVED && n < PACK) {  // part of a pack of codes: whole words, and the last one's bytes
#pragma unroll
            for (int w = 0; w < PACK; w += 4) copy_async<4>(to + w, from + (w < n ? w : 0), w < n ? min(4, n - w) : 0);
          } else {
            copy_async<PACK>(to, from, n);
          }
        }
      }
    p += step;
  }
  __device__ void start_scales(bool live, int t, int T, int npack, int shift, int N, long long step) {
    if constexpr (SAVED) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int k = t + i * T;
        if (live && k < npack) {
          e[i] = __ldg(e_from + (ODD ? max(k * P - shift, 0) / PK_GROUP : i * T / K::LANES));
          if constexpr (ODD) e2[i] = __ldg(e_from + min(k * P - shift + P - 1, N - 1) / PK_GROUP);
        }
      }
      e_from += step;
    }
  }
  struct Words { uint32_t w[PACK / 4]; };
  __device__ Words fetch(uint32_t stage, int i) const {
    const uint32_t from = stage + at + i * PLACE;
    Words v;
    if constexpr (PACK == 16) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]) : "r"(from) : "memory");
    else if constexpr (PACK == 8) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.w[0]), "=r"(v.w[1]) : "r"(from) : "memory");
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v.w[0]) : "r"(from) : "memory");
    return v;
  }
  // The values of pack i, with AFFINE times `by` plus `plus` (a checkpoint's step takes the factor in for nothing).
  template <bool AFFINE>
  __device__ void values(const Words& v, int i, int t, int T, int shift, float by, float plus, f2* out) const {
    const f2 plus2 = f2_all(plus);
    if constexpr (!SAVED) {
      K::unpack(make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]), out);
      if constexpr (AFFINE) {
        const f2 by2 = f2_all(by);
#pragma unroll
        for (int j = 0; j < H; ++j) out[j] = f2_fma(out[j], by2, plus2);
      }
    } else {
      const float unit = AFFINE ? pk_step(e[i]) * by : pk_step(e[i]);
      f2 units = f2_all(unit);
#pragma unroll
      for (int c = 0; c < P; c += 2) {
        if constexpr (ODD) {
          // the next group begins with the value whose column is a multiple of 32
          const float unit2 = AFFINE ? pk_step(e2[i]) * by : pk_step(e2[i]);
          const int next = PK_GROUP - ((t + i * T) * P - shift + PK_GROUP) % PK_GROUP;
          units = f2_of(c < next ? unit : unit2, c + 1 < next ? unit : unit2);
        }
        out[c / 2] = AFFINE ? f2_fma(pk_two(v.w[c / 4], c % 4), units, plus2) : f2_mul(pk_two(v.w[c / 4], c % 4), units);
      }
    }
  }
};

// Sums of two values over a team. In a warp the halves exchange what they do not keep, so that both take one shuffle a step. Teams of
// several warps: `slot` has two halves, used in turn, so that one barrier is enough: who writes a half again has seen everybody
// arrive at the barrier after the one that guarded its reading. What a team does not fill of `slot` is zero.
template <int G>
__device__ __forceinline__ float2 team_sum(float2 v, uint32_t slot, int t, int T, int team) {
  if constexpr (G < 32) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
  } else {
    const bool upper = threadIdx.x & 16;
    float keep = upper ? v.y : v.x;
    keep += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, o);
    if constexpr (G == 32) {
      const float other = __shfl_xor_sync(0xffffffffu, keep, 16);
      return upper ? make_float2(other, keep) : make_float2(keep, other);
    } else {
      if ((t & 15) == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(slot + (t >> 4) * 4), "f"(keep) : "memory");
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(T) : "memory");
      f2 s = 0;
      const auto add = [&](int from, int to) {
#pragma unroll
        for (int w = from; w < to; ++w) {
          const float4 u = shared_f4(slot + w * 16);
          s = f2_add(s, f2_add(f2_of(u.x, u.y), f2_of(u.z, u.w)));
        }
      };
      add(0, 2);
      if (T > 128) add(2, 4);
      if (T > 256) add(4, 8);
      return f2_get(s);
    }
  }
}

template <int DT, int E, int G, bool ODD, bool GATE, bool SAVED, bool WIDE = false>
__global__ void __launch_bounds__(WIDE ? LN_BWD_WIDE : LN_BWD_THREADS) ln_bwd_kernel(const LnArgs a, const LnBwdPlan plan) {
  using K = LnPack<DT>;
  constexpr int P = K::P, H = K::H, V = E / P;
  constexpr bool FILL = G < 32;
  static_assert(!WIDE || (G > 32 && !ODD && !GATE), "what WIDE is for");
  // Weight and bias: in registers, or, with a gate or in WIDE, where these would not do: in shared memory (PLANES), or, in fp32 with a gate,
  // where that would not either, read again for each row.
  constexpr bool PLANES = WIDE || (GATE && !ODD && (DT != SRMS_F32 || SAVED)), AGAIN = GATE && !ODD && !PLANES, HELD = !PLANES && !AGAIN;
  constexpr int LANES = WIDE ? LN_BWD_WIDE : LN_BWD_THREADS;
  using In = LnRows<DT, V, LANES, ODD, SAVED>;
  using Dy = LnRows<DT, V, LANES, ODD, false>;
  constexpr uint32_t STAGE = Dy::BYTES + In::BYTES * (GATE ? 2 : 1), SLOTS = G > 32 ? LN_BWD_SLOTS : 0;
  const int T = G <= 32 ? G : plan.T, team = threadIdx.x / T, t = threadIdx.x - team * T, lanes = blockDim.x, teams = lanes / T;
  const int N = a.N;
  const float inv_n = 1.f / static_cast<float>(N);
  // shared memory: the teams' slots, weight and bias, the ring
  constexpr uint32_t PLANE = (WIDE ? LANES / 2 : LANES) * V * 16;  // four values of each pack
  const uint32_t slots = static_cast<uint32_t>(__cvta_generic_to_shared(ln_shared)), planes = slots + SLOTS;
  const uint32_t ring = PLANES ? planes + (GATE ? 2 : 1) * (P / 4) * PLANE : planes, ring_end = plan.stages * STAGE;
  uint32_t slot = slots + (G > 32 ? team * 256 : 0);
  if constexpr (G > 32)
    for (int i = threadIdx.x; i < SLOTS / 4; i += lanes) asm volatile("st.shared.u32 [%0], %1;" ::"r"(slots + 4 * i), "r"(0) : "memory");
  const long long row = static_cast<long long>(blockIdx.x) * teams + team;
  const long long first = FILL ? static_cast<long long>(blockIdx.x) * teams + (threadIdx.x & ~31) / T : row;
  // rows of this team, and of the team in its warp that has most
  const int mine = row < a.M ? static_cast<int>((a.M - 1 - row) / plan.step.rows) + 1 : 0;
  const int most = !FILL ? mine : first < a.M ? static_cast<int>((a.M - 1 - first) / plan.step.rows) + 1 : 0;
  const int shift = ODD ? static_cast<int>(row * N % P) : 0, npack = (N + shift + P - 1) / P;
  In x, g;
  Dy dy;
  dy.init(a.dy, a.lddy, nullptr, nullptr, N, row, t, shift, ring);
  x.init(a.x, a.ldx, a.xcodes, a.xscales, N, row, t, shift, ring + Dy::BYTES);
  if constexpr (GATE) g.init(a.gate, a.ldg, a.gcodes, a.gscales, N, row, t, shift, ring + Dy::BYTES + In::BYTES);
  uint32_t in = 0, out = 0;
  const auto start = [&](int n) {
    if (FILL || n < mine) {
      dy.template start<FILL>(in, n < mine, t, T, npack, shift, N, plan.step.dy);
      x.template start<FILL>(in, n < mine, t, T, npack, shift, N, SAVED ? plan.step.codes : plan.step.x);
      if constexpr (GATE) g.template start<FILL>(in, n < mine, t, T, npack, shift, N, SAVED ? plan.step.codes : plan.step.gate);
    }
    copies_commit();
    in = in + STAGE == ring_end ? 0 : in + STAGE;
  };
  const float2* st_from = a.stats + row;
  float2 st = make_float2(0.f, 0.f);
  const auto start_small = [&](int n) {
    const bool live = n < mine;
    if (FILL && !live) st = make_float2(0.f, 0.f);
    if (live) st = __ldg(st_from);
    st_from += plan.step.rows;
    x.start_scales(live, t, T, npack, shift, N, plan.step.scales);
    if constexpr (GATE) g.start_scales(live, t, T, npack, shift, N, plan.step.scales);
  };
  for (int k = 0; k < plan.stages; ++k) {
    dy.clear(k * STAGE);
    x.clear(k * STAGE);
    if constexpr (GATE) g.clear(k * STAGE);
  }
  for (int k = 1; k < plan.stages; ++k) start(k - 1);
  start_small(0);
  f2 w[HELD ? V : 1][H], b[HELD && GATE ? V : 1][H], dw[V][H], db[V][H];
  const auto columns = [&](int i, bool bias, f2* out) {  // weight or bias of pack i's columns
    const int k = t + i * T;
    const void* from = bias ? a.bias : a.weight;
    if constexpr (ODD) {
      K::params_at(from, a.wdt, k * P - shift, N, bias ? 0.f : 1.f, out);
    } else {
      float f[P];
      K::params(k < npack ? from : nullptr, a.wdt, a.vec_params, k, bias ? 0.f : 1.f, f);
#pragma unroll
      for (int j = 0; j < H; ++j) out[j] = f2_of(f[2 * j], f[2 * j + 1]);
    }
  };
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (HELD) columns(i, false, w[i]);
    if constexpr (HELD && GATE) columns(i, true, b[i]);
#pragma unroll
    for (int j = 0; j < H; ++j) dw[i][j] = db[i][j] = 0;
  }
  if constexpr (PLANES)
    for (int k = threadIdx.x; k < V * T; k += lanes)  // those behind the row's end too: they are multiplied by zero
#pragma unroll
      for (int which = 0; which < (GATE ? 2 : 1); ++which) {
        float f[P];
        K::params(k >= npack ? nullptr : which ? a.bias : a.weight, a.wdt, a.vec_params, k, which ? 0.f : 1.f, f);
#pragma unroll
        for (int e = 0; e < P; e += 4) shared_put(planes + (which * (P / 4) + e / 4) * PLANE + k * 16, make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]));
      }
  // Weight or bias of pack i from where they are.
  const auto weights = [&](int i, bool bias, f2* out) {
    if constexpr (PLANES) {
#pragma unroll
      for (int e = 0; e < P; e += 4) {
        const float4 v = shared_f4(planes + t * 16 + i * T * 16 + ((bias ? P / 4 : 0) + e / 4) * PLANE);
        out[e / 2] = f2_of(v.x, v.y);
        out[e / 2 + 1] = f2_of(v.z, v.w);
      }
    } else if constexpr (AGAIN) {
      columns(i, bias, out);
    } else {
#pragma unroll
      for (int j = 0; j < H; ++j) out[j] = bias ? b[GATE ? i : 0][j] : w[i][j];
    }
  };
  if constexpr (PLANES || G > 32) __syncthreads();
  char *dx = static_cast<char*>(a.dx) + (row * N - shift) * K::ESZ + t * 16, *dg = static_cast<char*>(a.dgate) + (row * N - shift) * K::ESZ + t * 16;
  for (int n = 0; n < most; ++n, dx += plan.step.out, dg += plan.step.out) {
    const bool live = !FILL || n < mine;
    copies_wait(plan.stages);
    if constexpr (WIDE) {
      const uint32_t at = out;
      const In row_x = x;  // its exponents
      const float r = st.y, minus_mr = -st.x * st.y;
      // dy with the weight's factor and xh of pack i; dy alone
      const auto take = [&](int i, f2* sv, f2* xh, f2* d) {
        f2 wk[H];
        const typename Dy::Words dy_words = dy.fetch(at, i);
        const typename In::Words x_words = x.fetch(at, i);
        weights(i, false, wk);
        dy.template values<false>(dy_words, i, t, T, shift, 1.f, 0.f, d);
        row_x.template values<true>(x_words, i, t, T, shift, r, minus_mr, xh);
#pragma unroll
        for (int j = 0; j < H; ++j) sv[j] = f2_mul(wk[j], d[j]);
      };
      f2 c1 = 0, c2 = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f2 sv[H], xh[H], d[H];
        take(i, sv, xh, d);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          db[i][j] = f2_add(db[i][j], d[j]);
          dw[i][j] = f2_fma(d[j], xh[j], dw[i][j]);
          c1 = f2_add(c1, sv[j]);
          c2 = f2_fma(sv[j], xh[j], c2);
        }
      }
      out = out + STAGE == ring_end ? 0 : out + STAGE;
      start(n + plan.stages - 1);
      start_small(n + 1);
      const float2 c = team_sum<G>(make_float2(f2_sum(c1), f2_sum(c2)), slot, t, T, team);
      slot = slots + team * 256 + ((n & 1) ? 0 : 128);
      const float by = -inv_n * r;
      const f2 rr = f2_all(r), k1 = f2_all(c.x * by), k2 = f2_all(c.y * by);
      if (a.dx) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          f2 sv[H], xh[H], d[H];
          take(i, sv, xh, d);
#pragma unroll
          for (int j = 0; j < H; ++j) sv[j] = f2_fma(sv[j], rr, f2_fma(xh[j], k2, k1));
          if (t + i * T < npack) K::store(dx + i * T * 16, sv);
        }
      }
      continue;
    }
    f2 xh[V][H], s[V][H];  // s: dy, then with the gate's factor, then with the weight's
    typename Dy::Words dy_words[V];
    typename In::Words x_words[V], g_words[GATE ? V : 1];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dy_words[i] = dy.fetch(out, i);
      x_words[i] = x.fetch(out, i);
      if constexpr (GATE) g_words[i] = g.fetch(out, i);
    }
    out = out + STAGE == ring_end ? 0 : out + STAGE;
    const float r = st.y, minus_mr = -st.x * st.y;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const LnPackEdge e = ln_edge<P, ODD>(t + i * T, shift, N);
      dy.template values<false>(dy_words[i], i, t, T, shift, 1.f, 0.f, s[i]);
      x.template values<true>(x_words[i], i, t, T, shift, r, minus_mr, xh[i]);
      if (ODD && (e.lo > 0 || e.hi < P)) {
        K::cut(s[i], e.lo, e.hi);
        K::cut(xh[i], e.lo, e.hi);
      }
    }
    if constexpr (GATE) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int k = t + i * T;
        const LnPackEdge e = ln_edge<P, ODD>(k, shift, N);
        const bool part = ODD && (e.lo > 0 || e.hi < P);
        if (k < npack) {
          f2 u[H], wk[H], bk[H];
          g.template values<true>(g_words[i], i, t, T, shift, LN_MINUS_LOG2E, 0.f, u);
          if (part) K::cut(u, e.lo, e.hi);
          weights(i, false, wk);
          weights(i, true, bk);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            const float2 gv = f2_get(u[j]);
            float s0, s1, r0, r1;
            ln_sigmoid2(gv.x, &s0, &r0);
            ln_sigmoid2(gv.y, &s1, &r1);
            s[i][j] = f2_mul(s[i][j], f2_of(s0, s1));
            u[j] = f2_mul(f2_mul(s[i][j], f2_fma(xh[i][j], wk[j], bk[j])), f2_of(r0, r1));
          }
          if (a.dgate && live) {
            if (part) K::store_part(dg + i * T * 16, u, e.lo, e.hi);
            else K::store(dg + i * T * 16, u);
          }
        }
      }
    }
    f2 c1 = 0, c2 = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f2 wk[H];
      weights(i, false, wk);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        db[i][j] = f2_add(db[i][j], s[i][j]);
        dw[i][j] = f2_fma(s[i][j], xh[i][j], dw[i][j]);
        s[i][j] = f2_mul(wk[j], s[i][j]);
        c1 = f2_add(c1, s[i][j]);
        c2 = f2_fma(s[i][j], xh[i][j], c2);
      }
    }
    // With a gate, where registers run out, the sums' halves meet before the copies start, else behind that, where they overlap:
    // 32768 x 4096 bf16 gated from checkpoints 219 us and 231, 16384 x 5120 without a gate 117 and 111.
    float2 c;
    if constexpr (GATE) c = make_float2(f2_sum(c1), f2_sum(c2));
    start(n + plan.stages - 1);
    start_small(n + 1);
    if constexpr (!GATE) c = make_float2(f2_sum(c1), f2_sum(c2));
    c = team_sum<G>(c, slot, t, T, team);
    const float by = -inv_n * r;
    const f2 rr = f2_all(r), k1 = f2_all(c.x * by), k2 = f2_all(c.y * by);
    if (a.dx && live) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < H; ++j) s[i][j] = f2_fma(s[i][j], rr, f2_fma(xh[i][j], k2, k1));
        const LnPackEdge e = ln_edge<P, ODD>(t + i * T, shift, N);
        if (t + i * T < npack) {
          if (ODD && (e.lo > 0 || e.hi < P)) K::store_part(dx + i * T * 16, s[i], e.lo, e.hi);
          else K::store(dx + i * T * 16, s[i]);
        }
      }
    }
    if constexpr (G > 32) slot = slots + team * 256 + ((n & 1) ? 0 : 128);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!a.partial) return;
  float* sums = reinterpret_cast<float*>(ln_shared);
  if constexpr (ODD) {
    // The CTA's part of dw and db: teams have columns of their own in a pack, so their sums meet by column in shared memory. A number of
    // threads add up a column's teams, each every so-manieth one, and one of them these in turn.
    const int parts = N < lanes ? min(lanes / N, teams) : 1;
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float f[P];
        f2 both[H];
#pragma unroll
        for (int j = 0; j < H; ++j) both[j] = which ? db[i][j] : dw[i][j];
        K::floats(both, f);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const int col = (t + i * T) * P - shift + e;
          if (col >= 0 && col < N) sums[team * N + col] = f[e];
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < parts * N; c += lanes) {
        const int part = c / N, col = c - part * N;
        float sum = 0.f;
        for (int k = part; k < teams; k += parts) sum += sums[k * N + col];
        sums[part * N + col] = sum;  // team `part` is this thread's alone
      }
      __syncthreads();
      for (int col = threadIdx.x; col < N; col += lanes) {
        float sum = 0.f;
        for (int k = 0; k < parts; ++k) sum += sums[k * N + col];
        a.partial[(static_cast<size_t>(blockIdx.x) * 2 + which) * N + col] = sum;
      }
    }
    return;
  }
  // The CTA's part of dw and db: its teams' (for rows within a warp, its warps') sums in their order, through shared memory.
  constexpr int LW = G < 32 ? G : 32;
  const int span = G <= 32 ? 32 : T, TT = G <= 32 ? LW : T, units = lanes / span, unit = threadIdx.x / span, tt = threadIdx.x - unit * span;
  const bool holds = tt < TT;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float acc[E];
#pragma unroll
    for (int i = 0; i < V; ++i) K::floats(which ? db[i] : dw[i], acc + i * P);
#pragma unroll
    for (int o = LW; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
    if (units > 1) {
      __syncthreads();
      if (holds && unit > 0)
#pragma unroll
        for (int e = 0; e < E; ++e) sums[((unit - 1) * E + e) * TT + tt] = acc[e];
      __syncthreads();
      if (holds && unit == 0)
        for (int u = 0; u < units - 1; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += sums[(u * E + e) * TT + tt];
    }
    if (holds && unit == 0) {
      float* to = a.partial + (static_cast<size_t>(blockIdx.x) * 2 + which) * N;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int k = tt + i * T;
        if (k < npack)
#pragma unroll
          for (int e = 0; e < P; e += 4)
            reinterpret_cast<float4*>(to + static_cast<size_t>(k) * P)[e / 4] = make_float4(acc[i * P + e], acc[i * P + e + 1], acc[i * P + e + 2], acc[i * P + e + 3]);
      }
    }
  }
}

}  // namespace lab200
