#pragma once
#include <atomic>

#include "layernorm_launch.cuh"

namespace lab200 {

constexpr int LN_SHARED = 232448;  // bytes of shared memory that a CTA may have

enum LnRowKind { LN_ANY, LN_PACKS, LN_ODD };

// How a call's rows may be read: in packs of 16 bytes that divide every row of every tensor (and words that divide its checkpoints);
// in the packs of whole contiguous tensors; element by element.
inline LnRowKind ln_kind(const LnArgs& a, int esz) {
  uintptr_t bits = 0;  // of pointers and row strides
  bool contiguous = true;
  const auto tensor = [&](const void* p, long long ld) {
    if (!p) return;
    bits |= reinterpret_cast<uintptr_t>(p);
    if (a.M > 1 && ld != a.N) bits |= static_cast<uintptr_t>(ld) * esz, contiguous = false;
  };
  tensor(a.x, a.ldx);
  tensor(a.gate, a.ldg);
  tensor(a.y, a.N);
  tensor(a.dy, a.lddy);
  tensor(a.dx, a.N);
  tensor(a.dgate, a.N);
  const uintptr_t codes = reinterpret_cast<uintptr_t>(a.xcodes) | reinterpret_cast<uintptr_t>(a.gcodes);
  if (bits % 16 || codes % (16 / esz)) return LN_ANY;
  return a.N % (16 / esz) == 0 ? LN_PACKS : contiguous ? LN_ODD : LN_ANY;
}

// Rows after which the shifts of odd rows repeat.
inline int ln_period(int N, int P) {
  int q = P;
  while (q > 1 && (static_cast<long long>(N) * (q / 2)) % P == 0) q /= 2;
  return q;
}
// `ctas` of `teams` each, a few more or (past `most`) fewer, so that all teams together are a multiple of the period.
inline long long ln_even(long long ctas, long long most, int teams, int period) {
  int unit = period;
  while (unit > 1 && (static_cast<long long>(unit / 2) * teams) % period == 0) unit /= 2;
  ctas = (ctas + unit - 1) / unit * unit;
  return ctas <= most ? ctas : most / unit * unit > 0 ? most / unit * unit : unit;
}

// Static shared memory that a kernel may have beside its dynamic part.
constexpr int LN_STATIC = LN_FWD_THREADS / 64 * 2 * (LN_FWD_THREADS / 32) * 16;

// KERN has had its limit of dynamic shared memory raised on the devices whose bits are set.
template <auto KERN>
std::atomic<unsigned long long> ln_raised{0};

template <auto KERN, class Plan>
cudaError_t ln_launch(unsigned grid, int cta, size_t shared, LnPlace at, const LnArgs& a, const Plan& plan) {
  const unsigned long long bit = at.device < 64 ? 1ull << at.device : 0;
  if (!(ln_raised<KERN>.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t rc = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SHARED - LN_STATIC);
    if (rc != cudaSuccess) {
      cudaGetLastError();
      return rc;
    }
    ln_raised<KERN>.fetch_or(bit, std::memory_order_relaxed);
  }
  KERN<<<grid, cta, shared, at.st>>>(a, plan);
  count_launch();
  return cudaGetLastError();
}

template <int DT>
cudaError_t ln_fwd_any(const LnArgs& a, LnPlace at) {
  ln_fwd_any_kernel<DT><<<ln_capped(a.M, 1 << 20), 256, 0, at.st>>>(a);
  count_launch();
  return cudaGetLastError();
}

template <int DT, int V, int G, bool ODD>
cudaError_t ln_fwd_team(const LnArgs& a, LnPlace at, int T) {
  const bool gate = a.gate, save = a.xcodes;
  constexpr bool WIDEST = G > 32 && V == 4 && !ODD;  // the kernels that may want more room than there is
  constexpr int MOST = ODD && G > 32 && DT == SRMS_F32 ? LN_FWD_FEWER : LN_FWD_THREADS;
  constexpr size_t room = LN_SHARED - LN_STATIC;
  const size_t planes = ODD ? 0 : static_cast<size_t>(a.N) * 8;
  const auto stage_of = [&](int threads) { return threads * 16 * V * (gate ? 2 : 1); };
  const bool fewer = WIDEST && gate && planes + 2 * stage_of(LN_FWD_THREADS) > room;
  const int threads = fewer ? LN_FWD_FEWER : MOST, teams = threads / T, cta = teams * T, stage = stage_of(threads);
  int stages = planes > room ? 0 : static_cast<int>((room - planes) / stage);
  if (stages < 2) return ln_fwd_any<DT>(a, at);
  stages = stages > 4 ? 4 : stages;
  const size_t shared = planes + static_cast<size_t>(stages) * stage;
  const unsigned grid = static_cast<unsigned>(ln_even((a.M + teams - 1) / teams, at.sms, teams, ODD ? ln_period(a.N, LnPack<DT>::P) : 1));
  const LnFwdPlan plan{T, stages, T > 256 ? 15 : T > 128 ? 7 : 3, LnSteps(a, LnPack<DT>::ESZ, static_cast<long long>(grid) * teams)};
  if constexpr (ODD) {
    return gate ? ln_launch<ln_fwd_kernel<DT, V, G, true, true, false, MOST>>(grid, cta, shared, at, a, plan)
                : ln_launch<ln_fwd_kernel<DT, V, G, true, false, false, MOST>>(grid, cta, shared, at, a, plan);
  } else {
    if constexpr (WIDEST)
      if (fewer) return save ? ln_launch<ln_fwd_kernel<DT, V, G, false, true, true, LN_FWD_FEWER>>(grid, cta, shared, at, a, plan)
                           : ln_launch<ln_fwd_kernel<DT, V, G, false, true, false, LN_FWD_FEWER>>(grid, cta, shared, at, a, plan);
    if (gate) return save ? ln_launch<ln_fwd_kernel<DT, V, G, false, true, true>>(grid, cta, shared, at, a, plan)
                          : ln_launch<ln_fwd_kernel<DT, V, G, false, true, false>>(grid, cta, shared, at, a, plan);
    return save ? ln_launch<ln_fwd_kernel<DT, V, G, false, false, true>>(grid, cta, shared, at, a, plan)
                : ln_launch<ln_fwd_kernel<DT, V, G, false, false, false>>(grid, cta, shared, at, a, plan);
  }
}

template <int DT>
cudaError_t ln_fwd(const LnArgs& a, LnPlace at) {
  using K = LnPack<DT>;
  const LnRowKind kind = ln_kind(a, K::ESZ);
  const auto team = [](int npack, int v) { return (npack + v * 32 - 1) / (v * 32) * 32; };
  if (kind == LN_ODD && !a.xcodes) {
    constexpr int V = 16 / K::P;
    const int npack = (a.N + 2 * K::P - 2) / K::P;  // of the row that begins last in its first pack
    if (npack <= 4 * V) return ln_fwd_team<DT, V, 4, true>(a, at, 4);
    if (npack <= 8 * V) return ln_fwd_team<DT, V, 8, true>(a, at, 8);
    if (npack <= 32 * V) return ln_fwd_team<DT, V, 32, true>(a, at, 32);
    if (npack <= 512 * V) return ln_fwd_team<DT, V, 64, true>(a, at, team(npack, V));
  }
  const int npack = a.N / K::P;
  if (kind != LN_PACKS || npack > 512 * 4) return ln_fwd_any<DT>(a, at);
  // Rows of which one for each team of one pack a thread fills the GPU once or less: more threads to a row then cost less than they gain.
  // Measured with one pack and with four, bf16, rows from memory: 1 x 2048 in 3.3 and 3.5 us, 296 x 2048 in 3.9 and 5.1, 888 x 2048 in 6.5
  // and 5.8; 888 x 768 in 4.2 and 4.5, 1184 x 768 in 5.4 and 4.6.
  if (npack <= 512 && a.M * (npack <= 32 ? 32 : team(npack, 1)) <= at.sms * 640LL)
    return npack <= 32 ? ln_fwd_team<DT, 1, 32, false>(a, at, 32) : ln_fwd_team<DT, 1, 64, false>(a, at, team(npack, 1));
  if (npack <= K::LANES) return ln_fwd_team<DT, 1, K::LANES, false>(a, at, K::LANES);
  if (npack <= 2 * K::LANES) return ln_fwd_team<DT, 2, K::LANES, false>(a, at, K::LANES);
  if (npack <= 16) return ln_fwd_team<DT, 16 / K::LANES, K::LANES, false>(a, at, K::LANES);
  if (npack <= 32) return ln_fwd_team<DT, 4, 8, false>(a, at, 8);
  if (npack <= 64) return ln_fwd_team<DT, 4, 16, false>(a, at, 16);
  if (npack <= 128) return ln_fwd_team<DT, 4, 32, false>(a, at, 32);
  return ln_fwd_team<DT, 4, 64, false>(a, at, team(npack, 4));
}

struct LnBwdLaunch { LnBwdPlan plan; LnRowKind kind; bool wide; int G, cta; size_t shared; int parts; };

// False: no kernel that keeps rows in registers takes the call.
template <int DT>
bool ln_bwd_plan(const LnArgs& a, LnPlace at, LnBwdLaunch* l) {
  using K = LnPack<DT>;
  const bool gate = a.gate || a.gcodes, saved = a.xcodes;
  l->kind = ln_kind(a, K::ESZ);
  if (l->kind == LN_ANY) return false;
  const bool odd = l->kind == LN_ODD;
  const int npack = odd ? (a.N + 2 * K::P - 2) / K::P : a.N / K::P;  // odd rows: of the one that begins last in its first pack
  const auto team = [&](int e) { return (npack + e / K::P * 32 - 1) / (e / K::P * 32) * 32; };
  const int E = odd && gate ? 8 : 16, V = E / K::P;
  if (npack > LN_BWD_THREADS * V) return false;
  l->G = npack <= 2 * V ? 2 : npack <= 4 * V ? 4 : npack <= 8 * V ? 8 : npack <= 16 * V ? 16 : npack <= 32 * V ? 32 : 64;
  const int T = l->G <= 32 ? l->G : team(E);
  l->wide = K::P == 8 && !odd && !gate && T > LN_BWD_THREADS / 2 && T <= LN_BWD_WIDE / 2;
  const int lanes = l->wide ? LN_BWD_WIDE : LN_BWD_THREADS, teams = lanes / T;
  l->cta = teams * T;
  const size_t in = static_cast<size_t>(V) * lanes * (saved ? K::P : 16), stage = static_cast<size_t>(V) * lanes * 16 + in * (gate ? 2 : 1);
  // the kernel's slots and planes
  const size_t planes = l->wide ? lanes / 2 : gate && !odd && (K::P == 8 || saved) ? 2 * lanes : 0;
  const size_t fixed = (l->G > 32 ? LN_BWD_SLOTS : 0) + planes * (K::P / 4) * V * 16;
  const int units = l->cta / (l->G <= 32 ? 32 : T);
  const size_t sums = odd ? static_cast<size_t>(teams) * a.N * 4 : static_cast<size_t>(units - 1) * E * T * 4;
  constexpr size_t room = LN_SHARED - LN_STATIC;
  const int stages = fixed > room ? 0 : static_cast<int>((room - fixed) / stage);
  if (stages < 2) return false;
  l->plan.T = T;
  l->plan.stages = stages > 4 ? 4 : stages;
  l->shared = fixed + l->plan.stages * stage;
  if (sums > l->shared) l->shared = sums;
  const long long most = at.sms < LN_MAX_PARTS ? at.sms : LN_MAX_PARTS;
  l->parts = static_cast<int>(ln_even((a.M + teams - 1) / teams, most, teams, odd ? ln_period(a.N, K::P) : 1));
  l->plan.step = LnSteps(a, K::ESZ, static_cast<long long>(l->parts) * teams);
  return a.M / teams / l->parts < (1 << 30);
}

template <int DT, int G, bool ODD>
cudaError_t ln_bwd_team(const LnArgs& a, LnPlace at, const LnBwdLaunch& l) {
  const bool gate = a.gate || a.gcodes, saved = a.xcodes;
  constexpr int E = 16, EG = ODD ? 8 : 16;
  if (gate) return saved ? ln_launch<ln_bwd_kernel<DT, EG, G, ODD, true, true>>(l.parts, l.cta, l.shared, at, a, l.plan)
                         : ln_launch<ln_bwd_kernel<DT, EG, G, ODD, true, false>>(l.parts, l.cta, l.shared, at, a, l.plan);
  if constexpr (G > 32 && !ODD && LnPack<DT>::P == 8)
    if (l.wide) return saved ? ln_launch<ln_bwd_kernel<DT, E, G, false, false, true, true>>(l.parts, l.cta, l.shared, at, a, l.plan)
                             : ln_launch<ln_bwd_kernel<DT, E, G, false, false, false, true>>(l.parts, l.cta, l.shared, at, a, l.plan);
  return saved ? ln_launch<ln_bwd_kernel<DT, E, G, ODD, false, true>>(l.parts, l.cta, l.shared, at, a, l.plan)
               : ln_launch<ln_bwd_kernel<DT, E, G, ODD, false, false>>(l.parts, l.cta, l.shared, at, a, l.plan);
}

template <int DT, bool ODD>
cudaError_t ln_bwd_teams(const LnArgs& a, LnPlace at, const LnBwdLaunch& l) {
  switch (l.G) {
    case 2: return ln_bwd_team<DT, 2, ODD>(a, at, l);
    case 4: return ln_bwd_team<DT, 4, ODD>(a, at, l);
    case 8: return ln_bwd_team<DT, 8, ODD>(a, at, l);
    case 16: return ln_bwd_team<DT, 16, ODD>(a, at, l);
    case 32: return ln_bwd_team<DT, 32, ODD>(a, at, l);
    default: return ln_bwd_team<DT, 64, ODD>(a, at, l);
  }
}

template <int DT>
int ln_bwd_parts(const LnArgs& a, LnPlace at) {
  LnBwdLaunch l;
  return ln_bwd_plan<DT>(a, at, &l) ? l.parts : static_cast<int>(a.M >= 64 * 32 ? 64 : (a.M + 31) / 32);
}

template <int DT>
cudaError_t ln_bwd(LnArgs a, LnPlace at) {
  LnBwdLaunch l;
  if (ln_bwd_plan<DT>(a, at, &l)) {
    return l.kind == LN_ODD ? ln_bwd_teams<DT, true>(a, at, l) : ln_bwd_teams<DT, false>(a, at, l);
  }
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
