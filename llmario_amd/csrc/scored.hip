// scored.hip — attention with shaped scores (lmh_attend_scored) on gfx950 matrix cores: a unit launch as
// units.hip's (unit_wave.h) whose scores s = scale q.K pass through
//     cap * tanh(s / cap)               when there is a cap
//     s - slopes[head] * |pos - key|    when there are slopes
// before the softmax, and whose rows may each see a range of keys of their own (prefix and document masks).
// A row that sees no key is zeros.
//
// A launch takes decode rows, drafted tokens and every width the kernel of long segments (scored_prompt.hip) has no
// instance of. Pages are read once per unit, so HBM bounds large calls: one token of 32 sequences on 512 .. 4,096 keys,
// 32/8 heads of 128, f16, cap 50: 40 us, 5.8 TB/s of the 6.9 a plain read reaches, VALU 15 % and matrix pipe 7 % of its
// time; 8 on 32,768 q8_0 keys with slopes 99 .. 112 us, 5.2 .. 5.8 TB/s, VALU 44 % (codes to f16, a unit's scales).
// Smaller ones are bound by the chain of a wave's steps and the widest unit's share of a workgroup: 48 sequences of
// packed documents, 40/8 heads, bf16, 127 MB: 31 us, one wave per SIMD; 8 rows beside 120 of a prompt, 32 heads of 80:
// 26 us, 3.4 TB/s; one f32 row of 256 keys 10 us, a launch and five dependent round trips. Cut units' merge: 4.1 us.
#include "unit_wave.h"

#include <atomic>

namespace lmh {
namespace {

template <int F, int HDP, int HDVP, int NB>
__global__ __launch_bounds__((64 * unit_w<F, HDP, HDVP, NB, true>()))
__attribute__((amdgpu_waves_per_eu(unit_wpe<F, HDP, HDVP, NB, true>())))
void scored_unit_kernel(PageGeom g, UnitGeom u, ScoreGeom sc, const UnitWave* waves, const float* q, float* out, MergeCopy mc) {
  extern __shared__ __attribute__((aligned(16))) float scored_lds[];
  copy_merges(mc, blockIdx.x, gridDim.x);
  unit_wave<F, HDP, HDVP, NB, NB == 1 && !Cfg<F, HDP, HDVP, NB>::ROWS, true>(g, u, waves, q, out, scored_lds, sc);
}

}  // namespace

uint32_t scored_waves(uint32_t kv_type, uint32_t hd, uint32_t hdv, uint32_t layout, uint32_t nb) {
  uint32_t w = 0;
  with_instance(kv_type, hd, hdv, layout, [&](auto f, auto a, auto b) {
    constexpr int F = decltype(f)::value, A = decltype(a)::value, B = decltype(b)::value;
    if (nb == 1) w = unit_w<F, A, B, 1, true>();
    else if (two_blocks<F, A, B>()) w = unit_w<F, A, B, 2, true>();
  });
  return w;
}

// As unit_waves_per_cu: asked of the runtime once per kernel and device.
uint32_t scored_waves_per_cu(int32_t device, uint32_t kv_type, uint32_t hd, uint32_t hdv, uint32_t layout, uint32_t nb) {
  constexpr int DEVICES = 16;   // devices beyond these are asked each time
  uint32_t n = 4;
  auto ask = [&](auto f, auto a, auto b, auto nbt) {
    constexpr int F = decltype(f)::value, A = decltype(a)::value, B = decltype(b)::value, NB = decltype(nbt)::value;
    if constexpr (NB == 1 || two_blocks<F, A, B>()) {
      static std::atomic<uint32_t> known[DEVICES];
      const bool keep = device >= 0 && device < DEVICES;
      if (keep && (n = known[device].load(std::memory_order_relaxed)) != 0) return;
      int blocks = 0;
      const bool ok = hipSetDevice(device) == hipSuccess &&
                      hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, scored_unit_kernel<F, A, B, NB>, 256, 0) == hipSuccess && blocks > 0;
      n = ok ? 4 * (uint32_t)blocks : 4;
      if (ok && keep) known[device].store(n, std::memory_order_relaxed);
    }
  };
  with_instance(kv_type, hd, hdv, layout, [&](auto f, auto a, auto b) {
    if (nb == 1) ask(f, a, b, std::integral_constant<int, 1>{});
    else ask(f, a, b, std::integral_constant<int, 2>{});
  });
  return n;
}

hipError_t launch_scored_units(const PageGeom& g, const UnitGeom& u, const ScoreGeom& sc, uint32_t nb, uint32_t w, const UnitWave* waves,
                               uint32_t n_wg, const float* q, float* out, const MergeCopy& mc, hipStream_t s, const LaunchEv& ev) {
  if (n_wg == 0) return hipSuccess;
  hipError_t e = hipErrorInvalidValue;
  auto go = [&](auto f, auto a, auto b, auto nbt) {
    constexpr int F = decltype(f)::value, A = decltype(a)::value, B = decltype(b)::value, NB = decltype(nbt)::value;
    if constexpr (NB == 1 || two_blocks<F, A, B>()) {
      using C = Cfg<F, A, B, NB, true>;
      if (w == 0 || w > (uint32_t)unit_w<F, A, B, NB, true>()) return;
      const uint32_t lds = w * 4 * std::max(C::QF, u.shared ? C::LF : 0);
      LMH_LAUNCH(ev, (scored_unit_kernel<F, A, B, NB>), dim3(n_wg), dim3(64 * w), lds, s, g, u, sc, waves, q, out, mc);
      e = hipGetLastError();
    }
  };
  with_instance(g.kv_type, g.hd, g.hdv, g.layout, [&](auto f, auto a, auto b) {
    if (nb == 1) go(f, a, b, std::integral_constant<int, 1>{});
    else if (nb == 2) go(f, a, b, std::integral_constant<int, 2>{});
  });
  return e;
}

}  // namespace lmh
