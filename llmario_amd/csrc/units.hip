// units.hip — attention of multi-row segments the prefill kernel has no instance for, and of every
// row of the row layout and f32 pages, on gfx950 matrix cores.
//
// Computes what `attend` computes (crates/engine/model/src/forward.rs:585-807). A unit is up to
// 16 * NB columns (token, query head) of one segment and KV head, flattened token-major as the
// prefill kernel's units are, over the key pages its columns see. A unit's keys are shared by 1 to W
// consecutive waves of one workgroup (the planner packs units into workgroups), whose partials merge
// in LDS; a unit longer than a workgroup's waves should walk runs as key pieces whose partials a
// merge launch combines. So the rows of a short segment (a run of drafted tokens) read each page
// once, not once per row, and wide heads, f32 pages and rows off the tile layout run on the matrix
// cores.
//
// Per step of KT page tiles (32 keys; 16 on f32 pages), operands straight from HBM to registers:
//   S^T[keys x cols] = K . Q^T       16-bit: v_mfma_f32_16x16x32, Q as hi + lo parts of the type
//                                    f32:    v_mfma_f32_16x16x4f32
//   O^T[dims x cols] += V^T . P^T    16-bit: v_mfma_f32_16x16x32_f16, P as f16 hi + lo parts
//                                    f32:    v_mfma_f32_16x16x4f32
// with the same lazy online softmax, precision and q8_0 scheme as the decode work item
// (decode_tile.h); in the row layout Q and P have three parts of the pages' 16-bit type (24 bits, as in
// f32; bf16 there takes P.V in bf16). One step's operands are held; a register is requested again for the
// next step as soon as its products are issued, so every load has a whole step to arrive in (the two-tile
// buffers of the decode item would not leave room for a second column block).
//
// Measured, one step of lmh_attend, against a decode item per row (before; the row layout's and f32
// pages' on the VALU): 24 sequences x 4 rows on 512 .. 4,096 keys (32/8 heads, hd 128, bf16, 190 MB of
// pages): 98.5 -> 42 us, 36.6 of them this kernel (202 MB read at 5.5 TB/s, 5.9 at four times the contexts:
// bound by HBM) and 4.4 the cut units' merge; hd 256 prompts of 600 and 800 tokens, window 1,024: 225 -> 62 us
// (57 before non-finite V of a masked key was kept out: the masked steps wait for V to test it), bound by the
// chain of one wave per SIMD's steps and a second, partly filled round of workgroups (waves resident 62 % of
// the time, issuing VALU 25 % and in the matrix pipe 12 %), two of 2,048: 410 TFLOP/s; hd 80, 32 heads of
// their own K/V, 8 decode rows and a 120-token chunk: 1,038 -> 29 us (23.5 + merge 4.1; 85 MB; decode rows
// alone at 8,000 keys: 5.0 TB/s); f32 prompts of 450 and 390 tokens, hd 64: 102 -> 23 us (four steps a wave:
// the chain from its record to its merge; matrix pipe 21 %). The row layout's loads are ordinary ones: a row's
// lines are touched by several lanes' loads, and as streaming loads they were fetched again for each (8,000
// keys at hd 80: 200 -> 140 us).
//
// An instance of the row layout or of f32 pages takes every width up to its own: lanes past a row's end
// hold zeros (K) or re-read the row's first dims into blocks that are never stored (V).
//
// Row layout and f32 pages hold key rows as they are, so the operands' element order is chosen to
// suit the loads: 16-bit V pairs two dims per lane (a dword per key and 32-dim block: block 2b + p
// holds dims 32b + 2m + p, m = 0..15), f32 K and V four (a float4; f32 K chunk c, product i: k index
// g is dim 16c + 4g + i; V block 4b + j: dims 64b + 4m + j).
#include "unit_wave.h"

#include <atomic>

namespace lmh {
namespace {

template <int F, int HDP, int HDVP, int NB>
__global__ __launch_bounds__((64 * unit_w<F, HDP, HDVP, NB>()))
__attribute__((amdgpu_waves_per_eu(unit_wpe<F, HDP, HDVP, NB>())))
void unit_kernel(PageGeom g, UnitGeom u, const UnitWave* waves, const float* q, float* out, MergeCopy mc) {
  extern __shared__ __attribute__((aligned(16))) float unit_lds[];
  copy_merges(mc, blockIdx.x, gridDim.x);
  unit_wave<F, HDP, HDVP, NB, NB == 1 && !Cfg<F, HDP, HDVP, NB>::ROWS>(g, u, waves, q, out, unit_lds);
}

}  // namespace

uint32_t unit_waves(uint32_t kv_type, uint32_t hd, uint32_t hdv, uint32_t layout, uint32_t nb) {
  uint32_t w = 0;
  with_instance(kv_type, hd, hdv, layout, [&](auto f, auto a, auto b) {
    constexpr int F = decltype(f)::value, A = decltype(a)::value, B = decltype(b)::value;
    if (nb == 1) w = unit_w<F, A, B, 1>();
    else if (two_blocks<F, A, B>()) w = unit_w<F, A, B, 2>();
  });
  return w;
}

// Asked of the runtime once per kernel and device (a query takes ~10 us, which each new cache's first call
// paid); a query that fails is asked again by the next call.
uint32_t unit_waves_per_cu(int32_t device, uint32_t kv_type, uint32_t hd, uint32_t hdv, uint32_t layout, uint32_t nb) {
  constexpr int DEVICES = 16;   // devices beyond these are asked each time
  uint32_t n = 4;
  auto ask = [&](auto f, auto a, auto b, auto nbt) {   // without LDS, 4-wave workgroups: what the registers allow
    constexpr int F = decltype(f)::value, A = decltype(a)::value, B = decltype(b)::value, NB = decltype(nbt)::value;
    if constexpr (NB == 1 || two_blocks<F, A, B>()) {
      static std::atomic<uint32_t> known[DEVICES];
      const bool keep = device >= 0 && device < DEVICES;
      if (keep && (n = known[device].load(std::memory_order_relaxed)) != 0) return;
      int blocks = 0;
      const bool ok = hipSetDevice(device) == hipSuccess &&
                      hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, unit_kernel<F, A, B, NB>, 256, 0) == hipSuccess && blocks > 0;
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

hipError_t launch_units(const PageGeom& g, const UnitGeom& u, uint32_t nb, uint32_t w, const UnitWave* waves, uint32_t n_wg,
                        const float* q, float* out, const MergeCopy& mc, hipStream_t s, const LaunchEv& ev) {
  if (n_wg == 0) return hipSuccess;
  hipError_t e = hipErrorInvalidValue;
  auto go = [&](auto f, auto a, auto b, auto nbt) {
    constexpr int F = decltype(f)::value, A = decltype(a)::value, B = decltype(b)::value, NB = decltype(nbt)::value;
    if constexpr (NB == 1 || two_blocks<F, A, B>()) {
      if (w == 0 || w > (uint32_t)unit_w<F, A, B, NB>()) return;
      const uint32_t lds = w * 4 * std::max(Cfg<F, A, B, NB>::QF, u.shared ? Cfg<F, A, B, NB>::LF : 0);
      LMH_LAUNCH(ev, (unit_kernel<F, A, B, NB>), dim3(n_wg), dim3(64 * w), lds, s, g, u, waves, q, out, mc);
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
