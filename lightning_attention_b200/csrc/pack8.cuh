// 8-bit activation checkpoints: 32 consecutive values of a row share one exponent byte E, each keeps a signed byte.
//
//   step = 2^(E - 133);   code = rint(x / step), in [-127, 127];   value = code * step
//   E    = exponent field of the group's largest magnitude, one more where that would round to 128 steps; 7 <= E <= 254
//
// so a group's largest value is 63.75 (where E is raised) to 127.5 steps and every value is off by at most half a step, 1 / 127.5 of that
// largest value. At E's ends that bound is another: groups below 2^-120 have the step 2^-126, and their values up to half of it come back
// as zero; values of 127.5 * 2^121 and above come back as 127 * 2^121, up to a step less. The step is a power of two so that
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

// A checkpoint's value before it becomes fp16: what rounded up past the type's largest value is held there. A NaN stays one.
template <int DT>
__device__ __forceinline__ float pk_bound(float v) {
  if constexpr (DT == SRMS_F16) v = v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v;
  return v;
}

// Exponent byte of the group of which this lane has a pack of 16 bytes and adjacent lanes the rest (4 lanes of 16-bit values, 8 of
// fp32); all lanes of a warp call it. Magnitudes of each type compare as whole numbers, infinities and NaN above the rest; 16-bit
// ones two at a time.
template <int DT>
__device__ __forceinline__ uint32_t pk_pack_exponent(const uint4& w) {
  constexpr uint32_t ALL = 0xffffffffu;
  if constexpr (DT == SRMS_F32) {
    uint32_t m = max(max(w.x & 0x7fffffffu, w.y & 0x7fffffffu), max(w.z & 0x7fffffffu, w.w & 0x7fffffffu));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(ALL, m, o));
    return pk_exponent(m);
  } else {
    uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(ALL, m, o));
    m = max(m & 0xffffu, m >> 16);
    if constexpr (DT == SRMS_BF16) return pk_exponent(m << 16);
    return pk_exponent(__float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m)))));
  }
}
// P codes, four to a word, from pairs of fp32 values. Adding 1.5 * 2^23 rounds to a whole number, to nearest even, and leaves it in the
// low byte: exact, as x * inv is. Groups of E = 254 (whose codes may have to be held at 127) and 255 take the checked way.
template <int P>
__device__ __forceinline__ void pk_pack_codes(const unsigned long long* x, uint32_t e, uint32_t* w) {
  const float inv = pk_inv_step(e);
  uint32_t c[P];
  if (e < 254u) {
#pragma unroll
    for (int i = 0; i < P; i += 2)
      asm("{ .reg .b64 s, m, r; mov.b64 s, {%3, %3}; mov.b64 m, {%4, %4}; fma.rn.f32x2 r, %2, s, m; mov.b64 {%0, %1}, r; }"
          : "=r"(c[i]), "=r"(c[i + 1]) : "l"(x[i / 2]), "r"(__float_as_uint(inv)), "r"(__float_as_uint(12582912.f)));
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      float lo, hi;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x[i / 2]));
      c[i] = static_cast<uint32_t>(pk_code(lo, inv));
      c[i + 1] = static_cast<uint32_t>(pk_code(hi, inv));
    }
  }
#pragma unroll
  for (int i = 0; i < P; i += 4) w[i / 4] = __byte_perm(__byte_perm(c[i], c[i + 1], 0x0040), __byte_perm(c[i + 2], c[i + 3], 0x0040), 0x5410);
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

// ---- pack and unpack on their own: streaming kernels, bound by memory (3 1/32 bytes for each 16-bit value; 1048576 x 128 bf16 in
// 68 + 62 us, 0.91 and 1.0 of the measured copy bandwidth) ---------------------------------------------------------------------------
// Where packs of 16 bytes divide the rows, a thread has U packs, 32 apart, so that adjacent lanes hold a group and U accesses are under
// way. Contiguous rows of whole groups count as one row; otherwise rows are counted in whole groups, the last one's missing packs
// included, and a pack's row comes from a multiplication (`magic`) in place of a division. Past 2^31 packs a warp stays in one row.
struct PkRows {
  long long M, npack, ngroups, items;  // packs (without: groups) of a row, its groups; what warps take at a time
  int per_row;                         // items of a row
  uint32_t units, magic, shift;        // packs of a row counted in whole groups; 0: a warp stays in one row
};

__device__ __forceinline__ void pk_item(const PkRows& r, long long item, long long* row, long long* k) {
  if (r.M == 1) {
    *row = 0;
    *k = item;
  } else if (item < (1ll << 31)) {  // a division in 32 bits
    *row = static_cast<uint32_t>(item) / static_cast<uint32_t>(r.per_row);
    *k = item - *row * r.per_row;
  } else {
    *row = item / r.per_row;
    *k = item - *row * r.per_row;
  }
}
// Where a thread's packs of an item are: row and number of pack i, npack or more where there is none. UNITS: r.units is given.
template <int U, bool UNITS>
struct PkPlaces {
  long long row, k0;
  uint32_t q0;
  __device__ PkPlaces(const PkRows& r, long long item, int lane) {
    if constexpr (UNITS) {
      q0 = static_cast<uint32_t>(item) * (32 * U) + lane;
    } else {
      pk_item(r, item, &row, &k0);
      k0 = k0 * (32 * U) + lane;
    }
  }
  __device__ long long row_of(const PkRows& r, int i) const { return UNITS ? __umulhi(q0 + 32 * i, r.magic) >> r.shift : row; }
  __device__ long long pack_of(const PkRows& r, int i) const {
    if constexpr (!UNITS) return k0 + 32 * i;
    const uint32_t y = __umulhi(q0 + 32 * i, r.magic) >> r.shift;
    return y < r.M ? q0 + 32 * i - y * r.units : static_cast<uint32_t>(r.npack);
  }
};

template <int DT, int U, bool UNITS>
__global__ void __launch_bounds__(256)
pack8_kernel(const void* __restrict__ x_, long long ldx, int8_t* __restrict__ codes, uint8_t* __restrict__ scales, const PkRows r) {
  constexpr int P = SrmsVec<DT>::EPV, LANES = PK_GROUP / P, ESZ = 16 / P;
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); item < r.items; item += step) {
    const PkPlaces<U, UNITS> at(r, item, lane);
    SrmsPack<1> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const long long k = at.pack_of(r, i);
      v[i].q[0] = make_uint4(0, 0, 0, 0);
      if (k < r.npack) v[i] = ld_stream<1>(reinterpret_cast<const SrmsPack<1>*>(static_cast<const char*>(x_) + at.row_of(r, i) * ldx * ESZ) + k);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float f[P];
      SrmsVec<DT>::unpack(v[i].q[0], f);
      unsigned long long two[P / 2];
#pragma unroll
      for (int c = 0; c < P; c += 2) asm("mov.b64 %0, {%1, %2};" : "=l"(two[c / 2]) : "f"(f[c]), "f"(f[c + 1]));
      const uint32_t e = pk_pack_exponent<DT>(v[i].q[0]);
      uint32_t w[P / 4];
      pk_pack_codes<P>(two, e, w);
      const long long row = at.row_of(r, i), k = at.pack_of(r, i);
      if (k < r.npack) {
        auto* to = reinterpret_cast<uint32_t*>(codes + row * r.npack * P);
        if constexpr (P == 8) reinterpret_cast<uint2*>(to)[k] = make_uint2(w[0], w[1]);
        else to[k] = w[0];
        if (k % LANES == 0) scales[row * r.ngroups + k / LANES] = static_cast<uint8_t>(e);
      }
    }
  }
}

template <int DT, int U, bool UNITS>
__global__ void __launch_bounds__(256)
unpack8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y_, const PkRows r) {
  constexpr int P = SrmsVec<DT>::EPV, LANES = PK_GROUP / P;
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); item < r.items; item += step) {
    const PkPlaces<U, UNITS> at(r, item, lane);
    uint32_t w[U][P / 4], e[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const long long row = at.row_of(r, i), k = at.pack_of(r, i);
      if (k < r.npack) {
        const auto* from = reinterpret_cast<const uint32_t*>(codes + row * r.npack * P);
        if constexpr (P == 8) {
          const uint2 v = __ldcs(reinterpret_cast<const uint2*>(from) + k);
          w[i][0] = v.x; w[i][P / 4 - 1] = v.y;
        } else {
          w[i][0] = __ldcs(from + k);
        }
        e[i] = __ldg(scales + row * r.ngroups + k / LANES);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const long long row = at.row_of(r, i), k = at.pack_of(r, i);
      if (k < r.npack) {
        const float unit = pk_step(e[i]);
        float f[P];
#pragma unroll
        for (int c = 0; c < P; c += 2) {
          const unsigned long long two = pk_two(w[i][c / 4], c % 4);
          float lo, hi;
          asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(two));
          f[c] = pk_bound<DT>(lo * unit);
          f[c + 1] = pk_bound<DT>(hi * unit);
        }
        SrmsPack<1> o;
        o.q[0] = SrmsVec<DT>::pack(f);
        st_stream<1>(reinterpret_cast<SrmsPack<1>*>(y_) + row * r.npack + k, o);
      }
    }
  }
}

// Any row length, stride and alignment: a warp takes U adjacent groups at a time, a lane a value of each. As with packs, the groups are
// those of a row, or (UNITS) of all rows in turn, where a row would leave a warp little to do: 374506 x 51 bf16 in 51 + 40 us, 117 + 81 with
// warps that stay in a row.
template <int U, bool UNITS>
struct PkGroups {
  long long row, scale;  // of the first group; where its exponent is
  int g0, left;          // its number in the row, groups that there are from it on
  __device__ PkGroups(const PkRows& r, long long item) {
    if constexpr (UNITS) {
      const uint32_t q = static_cast<uint32_t>(item) * U, y = r.units == 1 ? q : __umulhi(q, r.magic) >> r.shift;
      row = y;
      scale = q;
      g0 = q - y * r.units;
      left = static_cast<int>(static_cast<uint32_t>(r.M) * r.units - q);
    } else {
      long long k;
      pk_item(r, item, &row, &k);
      g0 = static_cast<int>(k) * U;
      scale = row * r.ngroups + g0;
      left = static_cast<int>(r.ngroups) - g0;
    }
  }
  // Calls f(i, p) for each of U groups, p where the lane's value of it is (`from`: that of the first one, rows `ld` apart) or NULL.
  template <class T, class F>
  __device__ void each(const PkRows& r, int N, int lane, T* from, long long ld, F&& f) const {
    int rest = N - g0 * PK_GROUP - lane;  // values of the row from the lane's on
#pragma unroll
    for (int i = 0; i < U; ++i) {
      f(i, i < left && rest > 0 ? from : nullptr);
      rest -= PK_GROUP;
      from += PK_GROUP;
      if (UNITS && rest + lane <= 0) {
        rest = N - lane;
        from += ld - static_cast<long long>(r.units) * PK_GROUP;
      }
    }
  }
};

template <int DT, int U, bool UNITS>
__global__ void __launch_bounds__(256)
pack8_any_kernel(const void* __restrict__ x_, long long ldx, int8_t* __restrict__ codes, uint8_t* __restrict__ scales, int N, const PkRows r) {
  using E = SrmsElem<DT>;
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); item < r.items; item += step) {
    const PkGroups<U, UNITS> at(r, item);
    const int c0 = at.g0 * PK_GROUP + lane;
    float v[U];
    at.each(r, N, lane, static_cast<const typename E::T*>(x_) + at.row * ldx + c0, ldx, [&](int i, const typename E::T* x) { v[i] = x ? E::ld(x) : 0.f; });
    uint32_t mine = 0;  // lane i keeps the exponent of group i
    at.each(r, N, lane, codes + at.row * N + c0, N, [&](int i, int8_t* to) {
      const uint32_t e = pk_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(v[i]))));
      // as in pk_pack_codes
      const int code = e < 254u ? __float_as_int(fmaf(v[i], pk_inv_step(e), 12582912.f)) : pk_code(v[i], pk_inv_step(e));
      if (to) *to = static_cast<int8_t>(code);
      if (lane == i) mine = e;
    });
    if (lane < U && lane < at.left) scales[at.scale + lane] = static_cast<uint8_t>(mine);
  }
}

template <int DT, int U, bool UNITS>
__global__ void __launch_bounds__(256)
unpack8_any_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y_, int N, const PkRows r) {
  using E = SrmsElem<DT>;
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); item < r.items; item += step) {
    const PkGroups<U, UNITS> at(r, item);
    const long long first = at.row * N + at.g0 * PK_GROUP + lane;
    int v[U];
    uint32_t e[U];
    at.each(r, N, lane, codes + first, N, [&](int i, const int8_t* from) {
      if (from) {
        v[i] = *from;
        e[i] = __ldg(scales + at.scale + i);
      }
    });
    at.each(r, N, lane, static_cast<typename E::T*>(y_) + first, N, [&](int i, typename E::T* y) {
      if (y) E::st(y, pk_bound<DT>(static_cast<float>(v[i]) * pk_step(e[i])));
    });
  }
}

}  // namespace lab200
