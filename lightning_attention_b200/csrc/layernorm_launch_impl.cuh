#pragma once
#include "layernorm_launch.cuh"

namespace lab200 {

constexpr int LN_SHARED = 232448;  // bytes of shared memory that a CTA may have

// Whether packs of 16 bytes divide every row of every tensor of the call, and whole words its checkpoints.
inline bool ln_packs(const LnArgs& a, int esz) {
  uintptr_t bits = static_cast<uintptr_t>(a.N) * esz;
  const auto tensor = [&](const void* p, long long ld) {
    if (!p) return;
    bits |= reinterpret_cast<uintptr_t>(p);
    if (a.M > 1) bits |= static_cast<uintptr_t>(ld) * esz;
  };
  tensor(a.x, a.ldx);
  tensor(a.gate, a.ldg);
  tensor(a.y, a.N);
  tensor(a.dy, a.lddy);
  tensor(a.dx, a.N);
  tensor(a.dgate, a.N);
  const uintptr_t codes = reinterpret_cast<uintptr_t>(a.xcodes) | reinterpret_cast<uintptr_t>(a.gcodes);
  const uintptr_t scales = reinterpret_cast<uintptr_t>(a.xscales) | reinterpret_cast<uintptr_t>(a.gscales);
  return bits % 16 == 0 && codes % (16 / esz) == 0 && scales % 4 == 0;
}

template <class Kern, class Plan>
cudaError_t ln_launch(Kern kern, unsigned grid, int cta, size_t shared, cudaStream_t st, const LnArgs& a, const Plan& plan) {
  cudaError_t rc = shared > 40 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared)) : cudaSuccess;
  if (rc == cudaSuccess) {
    kern<<<grid, cta, shared, st>>>(a, plan);
    count_launch();
  }
  const cudaError_t last = cudaGetLastError();
  return rc == cudaSuccess ? last : rc;
}

template <int DT>
cudaError_t ln_fwd_any(const LnArgs& a, LnPlace at) {
  ln_fwd_any_kernel<DT><<<ln_capped(a.M, 1 << 20), 256, 0, at.st>>>(a);
  count_launch();
  return cudaGetLastError();
}

template <int DT, int V, int G>
cudaError_t ln_fwd_team(const LnArgs& a, LnPlace at, int T) {
  const bool gate = a.gate, save = a.xcodes;
  const int cta = 512 / T * T, stage = cta * 16 * V * (gate ? 2 : 1);
  const long long teams = cta / T, ctas = (a.M + teams - 1) / teams;
  const size_t planes = static_cast<size_t>(a.N) * 8;
  int stages = static_cast<int>((LN_SHARED - 1024 - planes) / stage);
  if (stages < 2) return ln_fwd_any<DT>(a, at);
  stages = stages > 4 ? 4 : stages;
  const LnFwdPlan plan{T, stages};
  const size_t shared = planes + static_cast<size_t>(stages) * stage;
  const unsigned grid = ln_capped(ctas, at.sms);
  if (gate) return save ? ln_launch(ln_fwd_kernel<DT, V, G, true, true>, grid, cta, shared, at.st, a, plan)
                        : ln_launch(ln_fwd_kernel<DT, V, G, true, false>, grid, cta, shared, at.st, a, plan);
  return save ? ln_launch(ln_fwd_kernel<DT, V, G, false, true>, grid, cta, shared, at.st, a, plan)
              : ln_launch(ln_fwd_kernel<DT, V, G, false, false>, grid, cta, shared, at.st, a, plan);
}

template <int DT>
cudaError_t ln_fwd(const LnArgs& a, LnPlace at) {
  using K = LnPack<DT>;
  const int npack = a.N / K::P;
  if (!ln_packs(a, K::ESZ) || npack > 512 * 4) return ln_fwd_any<DT>(a, at);
  const auto team = [&](int v) { return (npack + v * 32 - 1) / (v * 32) * 32; };
  if (npack <= 512 && a.M * team(4) < 148 * 256) return npack <= 32 ? ln_fwd_team<DT, 1, 32>(a, at, 32) : ln_fwd_team<DT, 1, 64>(a, at, team(1));
  if (npack <= 16 && K::LANES <= 4) return ln_fwd_team<DT, 4, 4>(a, at, 4);
  if (npack <= 32) return ln_fwd_team<DT, 4, 8>(a, at, 8);
  if (npack <= 64) return ln_fwd_team<DT, 4, 16>(a, at, 16);
  if (npack <= 128) return ln_fwd_team<DT, 4, 32>(a, at, 32);
  return ln_fwd_team<DT, 4, 64>(a, at, team(4));
}

struct LnBwdLaunch { LnBwdPlan plan; int G, cta; size_t shared; int parts; };

// False: no kernel that keeps rows in registers takes the call.
template <int DT>
bool ln_bwd_plan(const LnArgs& a, LnPlace at, LnBwdLaunch* l) {
  using K = LnPack<DT>;
  constexpr int E = 16, V = E / K::P;
  const bool gate = a.gate || a.gcodes, saved = a.xcodes;
  const int npack = a.N / K::P;
  if (!ln_packs(a, K::ESZ) || npack > LN_BWD_THREADS * V) return false;
  const int G = npack <= 8 * V ? 8 : npack <= 16 * V ? 16 : npack <= 32 * V ? 32 : 64;
  const int T = G <= 32 ? G : (npack + V * 32 - 1) / (V * 32) * 32;
  l->G = G;
  // up to 512 threads; one team more where that is a good part of a CTA's
  int teams = 512 / T;
  if ((teams + 1) * T <= LN_BWD_THREADS && teams <= 1) ++teams;
  l->cta = teams * T;
  const size_t in = static_cast<size_t>(V) * LN_PITCH / 16 * (saved ? K::P : 16), stage = static_cast<size_t>(V) * LN_PITCH + in * (gate ? 2 : 1);
  const size_t fixed = (G > 32 ? 10 * 2 * 160 : 0) + (gate ? static_cast<size_t>(a.N) * 8 : 0);
  const int units = l->cta / (G <= 32 ? 32 : T);
  const size_t sums = static_cast<size_t>(units - 1) * E * T * 4;
  const int stages = static_cast<int>((LN_SHARED - fixed) / stage);
  if (fixed > LN_SHARED || stages < 2) return false;
  l->plan = {T, stages > 4 ? 4 : stages};
  l->shared = fixed + l->plan.stages * stage;
  if (sums > l->shared) l->shared = sums;
  const long long ctas = (a.M + teams - 1) / teams;
  l->parts = static_cast<int>(ln_capped(ctas, at.sms < LN_MAX_PARTS ? at.sms : LN_MAX_PARTS));
  return (a.M + teams - 1) / teams / l->parts < (1 << 30);
}

template <int DT, int G>
cudaError_t ln_bwd_team(const LnArgs& a, LnPlace at, const LnBwdLaunch& l) {
  const bool gate = a.gate || a.gcodes, saved = a.xcodes;
  if (gate) return saved ? ln_launch(ln_bwd_kernel<DT, G, true, true>, l.parts, l.cta, l.shared, at.st, a, l.plan)
                         : ln_launch(ln_bwd_kernel<DT, G, true, false>, l.parts, l.cta, l.shared, at.st, a, l.plan);
  return saved ? ln_launch(ln_bwd_kernel<DT, G, false, true>, l.parts, l.cta, l.shared, at.st, a, l.plan)
               : ln_launch(ln_bwd_kernel<DT, G, false, false>, l.parts, l.cta, l.shared, at.st, a, l.plan);
}

template <int DT>
int ln_bwd_parts(const LnArgs& a, LnPlace at) {
  LnBwdLaunch l;
  return ln_bwd_plan<DT>(a, at, &l) ? l.parts : static_cast<int>(a.M >= 64 * 32 ? 64 : (a.M + 31) / 32);
}

template <int DT>
cudaError_t ln_bwd(LnArgs a, LnPlace at) {
  LnBwdLaunch l;
  if (ln_bwd_plan<DT>(a, at, &l))
    return l.G == 8 ? ln_bwd_team<DT, 8>(a, at, l) : l.G == 16 ? ln_bwd_team<DT, 16>(a, at, l) : l.G == 32 ? ln_bwd_team<DT, 32>(a, at, l) : ln_bwd_team<DT, 64>(a, at, l);
  if (a.dx || a.dgate) {
    ln_bwd_any_kernel<DT><<<ln_capped(a.M, 1 << 20), 256, 0, at.st>>>(a);
    count_launch();
    if (const cudaError_t rc = cudaGetLastError()) return rc;
  }
  if (!a.partial) return cudaSuccess;
  a.nparts = ln_bwd_parts<DT>(a, at);
  ln_bwd_columns_kernel<DT><<<dim3(ln_capped((a.N - 1) / 32 + 1, 1 << 20), a.nparts), 256, 0, at.st>>>(a);
  count_launch();
  return cudaGetLastError();
}

}  // namespace lab200
