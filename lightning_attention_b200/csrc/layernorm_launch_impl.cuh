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

struct LnBwdLaunch { LnBwdPlan plan; int vp, cta; size_t shared; int parts; };

// False: a row has too many packs.
template <int DT>
bool ln_bwd_plan(const LnArgs& a, LnPlace at, LnBwdLaunch* l) {
  using K = LnPack<DT>;
  const bool gate = a.gate || a.gcodes, saved = a.xcodes;
  const int npack = a.N / K::P, ng = (a.N - 1) / PK_GROUP + 1;
  if (!ln_packs(a, K::ESZ) || npack > 512 * 4) return false;
  l->vp = npack <= 640 ? 1 : npack <= 1024 ? 2 : 4;
  LnBwdPlan& p = l->plan;
  p.ct = (npack + l->vp - 1) / l->vp;
  p.rg = p.ct >= 512 ? 1 : 512 / p.ct;
  const int kr = 4 / l->vp;
  int rows = p.rg * kr;
  if (rows > 512) rows = 512;
  // few rows: tiles that leave no SM without one
  const long long fair = (a.M + at.sms - 1) / at.sms;
  if (rows > fair) rows = static_cast<int>(fair);
  p.rows = rows;
  l->cta = (p.rg * p.ct + 31) / 32 * 32;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes * 4 < npack) p.lanes *= 2;
  p.warps = (npack + 127) / 128;
  if (p.warps > l->cta / 32) return false;
  const uint32_t xp = saved ? K::P : 16, tile = static_cast<uint32_t>(rows) * npack;
  const uint32_t scales = saved ? ((static_cast<uint32_t>(rows) * ng + 3 + 15) & ~15u) : 0;
  p.dy_at = 0;
  p.x_at = tile * 16;
  p.g_at = p.x_at + ((tile * xp + 15) & ~15u);
  p.st_at = p.g_at + (gate ? ((tile * xp + 15) & ~15u) : 0);
  p.xs_at = p.st_at + ((static_cast<uint32_t>(rows) * 8 + 15) & ~15u);
  p.gs_at = p.xs_at + scales;
  p.stage_bytes = p.gs_at + (gate ? scales : 0);
  const size_t fixed = static_cast<size_t>(a.N) * 4 + ((rows * p.warps * 8 + 15) & ~15);
  int stages = static_cast<int>((LN_SHARED - fixed) / p.stage_bytes);
  if (stages < 2) return false;
  p.stages = stages > 4 ? 4 : stages;
  l->shared = fixed + static_cast<size_t>(p.stages) * p.stage_bytes;
  const size_t tree = static_cast<size_t>(p.rg / 2) * l->vp * K::P * p.ct * 4;
  if (tree > l->shared) l->shared = tree;
  const long long tiles = (a.M + rows - 1) / rows;
  l->parts = static_cast<int>(ln_capped(tiles, at.sms < LN_MAX_PARTS ? at.sms : LN_MAX_PARTS));
  return true;
}

template <int DT, int VP>
cudaError_t ln_bwd_packs(const LnArgs& a, LnPlace at, const LnBwdLaunch& l) {
  const bool gate = a.gate || a.gcodes, saved = a.xcodes;
  if (gate) return saved ? ln_launch(ln_bwd_kernel<DT, VP, true, true>, l.parts, l.cta, l.shared, at.st, a, l.plan)
                         : ln_launch(ln_bwd_kernel<DT, VP, true, false>, l.parts, l.cta, l.shared, at.st, a, l.plan);
  return saved ? ln_launch(ln_bwd_kernel<DT, VP, false, true>, l.parts, l.cta, l.shared, at.st, a, l.plan)
               : ln_launch(ln_bwd_kernel<DT, VP, false, false>, l.parts, l.cta, l.shared, at.st, a, l.plan);
}

template <int DT>
int ln_bwd_parts(const LnArgs& a, LnPlace at) {
  LnBwdLaunch l;
  return ln_bwd_plan<DT>(a, at, &l) ? l.parts : static_cast<int>(a.M >= 64 * 32 ? 64 : (a.M + 31) / 32);
}

template <int DT>
cudaError_t ln_bwd(LnArgs a, LnPlace at) {
  LnBwdLaunch l;
  if (ln_bwd_plan<DT>(a, at, &l)) return l.vp == 1 ? ln_bwd_packs<DT, 1>(a, at, l) : l.vp == 2 ? ln_bwd_packs<DT, 2>(a, at, l) : ln_bwd_packs<DT, 4>(a, at, l);
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
