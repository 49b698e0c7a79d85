// scored_prompt.hip — attention with shaped scores (lmh_attend_scored) of long segments on gfx950 matrix cores.
//
// A unit is up to 8 * COLS columns (token, query head) of one segment and KV head, flattened token-major as
// units.hip's, over the key pages its columns see; one workgroup of 8 waves (two per SIMD, four on heads of 64) takes a unit, wave w its
// columns COLS * w .. (COLS: 32 as two 16-column blocks on heads of 128; 16 on 256, whose O and Q fill the registers of
// two waves per SIMD, and on 64, where two workgroups to a CU hide each other's latencies: 8,192 packed tokens of 16
// heads 46 us against 56 with 32 columns). The workgroup walks 64-key tiles:
// all its waves share each tile's K and V through LDS, so pages are read once per unit and expanded once:
//   f16: as they are. bf16: widened to f16. q8_0: code * scale as f16 hi + lo parts (exact: 7 + 11 bits).
//   S^T[keys x cols] = K . Q^T       v_mfma_f32_16x16x32_f16, Q as f16 hi + lo parts of the column scaled by a
//                                    power of two to below 1 (22 bits of its largest element)
//   O^T[dims x cols] += V^T . P^T    v_mfma_f32_16x16x32_f16, weights as f16 hi + lo parts
// (q8_0: K hi . Q hi + K hi . Q lo + K lo . Q hi, and V likewise.) f16 has less range than bf16 or a scaled code: K
// and V are scaled by powers of two taken from the largest magnitude of the unit's first tile when that lies outside
// 2^0 .. 2^8 (q8_0, whose small products are multiples of 2^-24 and so exact: 2^-6 .. 2^8), to 2^3 .. 2^4. Computed again
// on the vector units in f32, straight from the pages (redo): all columns of a unit whose K leaves f16's range later;
// columns whose outputs are not finite (a NaN or an infinity in V, seen or not); and columns whose outputs are so small
// that V's rounding below 2^-17 (bf16; half a step, 2^-25) could be seen in them: n keys, a largest output M with
// M sqrt(n) < 2^-5 (V of their keys 2^-5 and less of the first tile's). K's rounding there is not looked for: it moves a
// score by 2^-25 of what the first tile's keys score.
//
// Per tile: the next tile's pages are requested into registers, the tile in LDS is multiplied, then the registers are
// expanded into the other LDS buffer and one barrier publishes it. All 64 keys' scores are formed before their softmax, so
// that the second half's weights can issue beside the first half's products (32 keys at a time: q8_0 prompts 106.2 us, 104.8
// so; four prompts of 2,048 370.7 and 365).
//
// Q and the weights in two parts are two products per pair (q8_0: three), so half (a third) of a large product's
// 1,260 TFLOP/s is the ceiling. Measured, us, with the share of the matrix pipe and of VALU issue: four prompts of 2,048
// tokens whose first halves see each other, 32/8 heads of 128, bf16: 365, 531 TFLOP/s, 39 % and 35 % (the unit launch 627; a
// third LDS buffer with the next tile's scores issued ahead of this one's softmax 406 .. 421); three of 401 .. 2,047 on
// q8_0 pages with a cap 102, 25 % and 33 %, and units of uneven lengths; 8,192 packed tokens of 16/4 heads of 64, f16, 42,
// 19 % and 32 %: 1,024 units of few tiles, much of it their way from the record to the first tile; two of 600 .. 1,100 tokens,
// 16/4 heads of 256, bf16, window 1,024, cap 50, 49 and the pieces' merge 5.5, 13 % and 21 %, one workgroup to a CU. A unit's
// time outside its walk, 128-wide heads, by the clock: its record from host memory 2.0 us, Q requested and converted 2 .. 3,
// the first tile's arrival, maxima and expansion 2, the first pass through the walk's code 1.3, its stores 2.
// Traffic is small beside that (0.4 .. 1.1 TB/s). No LDS bank conflicts on 16-bit pages; q8_0's 8-byte V stores have a few.
#include "decode_tile.h"
#include "score.h"

namespace lmh {
namespace {

using namespace dtile;

constexpr int PW = 8, NTH = 64 * PW, BK = 64;

template <int KVT, int HD>
struct Shape {
  static constexpr bool Q8 = KVT == KV_Q8, BF = KVT == KV_BF16;
  static constexpr int NCB = HD == 128 ? 2 : 1, COLS = 16 * NCB;
  static constexpr int NC = HD / 32, NJ = HD / 16;
  static constexpr int SIDE = BK * HD * 2;                  // bytes of a tile's K or V part in LDS
  static constexpr int PARTS = Q8 ? 2 : 1;
  static constexpr int STAGE = 2 * SIDE * PARTS;            // [K hi][K lo][V hi][V lo]
  static constexpr int LDS = 2 * STAGE + 128;               // .. and the workgroup's words
  static constexpr int NI = HD == 64 ? 1 : Q8 ? HD / 64 : NC / 2;   // staged items per wave and tile
  static constexpr int ROWS_I = Q8 ? 1 : 2;                 // 1 KiB page rows of an item
};

// One f32 value of key m, dim d of a tile-layout page (K or V) of head base `head`, tile `sub` of the block.
template <int KVT>
__device__ inline float page_value(const uint8_t* head, uint32_t sub, uint32_t tile, uint32_t scale, uint32_t tile_s, bool is_v, uint32_t m,
                                   uint32_t d, uint32_t hd) {
  const uint8_t* t = head + (size_t)sub * tile;
  if constexpr (KVT == KV_Q8) {
    const float c = (float)*(const int8_t*)(t + (is_v ? vq8_off(m, d) : kq8_off(m, d)));
    return c * h_to_f(*(const uint16_t*)(head + scale + (size_t)sub * tile_s + (m * (hd / 32) + d / 32) * 2));
  } else {
    const uint16_t b = *(const uint16_t*)(t + (is_v ? v16_off(m, d) : k16_off(m, d)));
    return KVT == KV_F16 ? h_to_f(b) : __uint_as_float((uint32_t)b << 16);
  }
}

// Column (row, head) of a unit in f32 from the pages, one wave: lanes over keys for the scores, over dims for the sums.
// out: the row's HD values, or its partial (raw sums, then reference and sum).
template <int KVT, int HD>
__device__ __forceinline__ void redo(const PageGeom& g, const UnitGeom& u, const ScoreGeom& sc, uint32_t seq, uint32_t kvh, uint32_t head,
                                  uint32_t pos, uint32_t first, uint32_t end, const float* q, float* out, bool partial) {
  constexpr int ND = HD / 64;
  const uint32_t lane = threadIdx.x & 63u, bt_mask = (1u << g.bt_shift) - 1u;
  const int32_t* tab = g.table + (size_t)seq * g.bps;
  float m = -INFINITY, l = 0.f, o[ND];
  for (int i = 0; i < ND; i++) o[i] = 0.f;
  const float slope = sc.slopes ? sc.slopes[head] * LOG2E : 0.f;
#pragma clang loop unroll(disable)
  for (uint32_t k0 = first; k0 < end; k0 += 64) {
    const uint32_t key = min(k0 + lane, end - 1), n = min(64u, end - k0);
    const uint8_t* b = g.pool + (size_t)(uint32_t)tab[key >> g.bt_shift] * g.block_bytes;
    const uint8_t* kh = b + g.k_off + (size_t)kvh * g.k_head;
    float s = 0.f;
#pragma clang loop unroll_count(16)
    for (uint32_t d = 0; d < (uint32_t)HD; d++)
      s = fmaf(q[d], page_value<KVT>(kh, (key & bt_mask) >> 4, g.k_tile, g.k_scale, g.k_tile_s, false, key & 15u, d, HD), s);
    float p[1] = {s * u.scale_log2};
    if (sc.cap_log2 > 0.f) cap_scores<1>(p, sc.cap_log2);
    if (sc.slopes) bias_scores<1>(p, slope, (float)(int)(key - pos), [](int) { return 0.f; });
    if (lane >= n) p[0] = -INFINITY;
    float mn = fmaxf(m, p[0]);
    for (int x = 32; x >= 1; x >>= 1) mn = fmaxf(mn, __shfl_xor(mn, x));
    const float ref = mn == -INFINITY ? 0.f : mn, alpha = exp2_fast(m - ref), w = lane < n ? exp2_fast(p[0] - ref) : 0.f;
    float sum = w;
    for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x);
    l = l * alpha + sum;
    m = mn;
    for (int i = 0; i < ND; i++) o[i] *= alpha;
#pragma clang loop unroll(disable)
    for (uint32_t j0 = 0; j0 < n; j0 += 8)
#pragma unroll
      for (uint32_t e = 0; e < 8; e++) {
        const uint32_t kj = min(k0 + j0 + e, end - 1);   // (past the last: read again, not added)
        const float wj = __shfl(w, (int)(j0 + e));
        const uint8_t* vh = g.pool + (size_t)(uint32_t)tab[kj >> g.bt_shift] * g.block_bytes + g.v_off + (size_t)kvh * g.v_head;
        for (int i = 0; i < ND; i++) {
          const float v = page_value<KVT>(vh, (kj & bt_mask) >> 4, g.v_tile, g.v_scale, g.v_tile_s, true, kj & 15u, lane + 64 * i, HD);
          o[i] = j0 + e < n ? fmaf(wj, v, o[i]) : o[i];
        }
      }
  }
  const float mul = partial ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
  for (int i = 0; i < ND; i++) out[lane + 64 * i] = o[i] * mul;
  if (partial && lane == 0) {
    out[HD] = m;
    out[HD + 1] = l;
  }
}

// CAP, BIAS: the launch has a cap, slopes (a test in the walk would split its code, and the compiler computes a short
// branch's values ahead of the test).
template <int KVT, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(NTH) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 4 : 2, HD == 64 ? 4 : 2)))
void scored_prompt_kernel(PageGeom g, UnitGeom u, ScoreGeom sc, const PromptItem* items, const float* q, float* out, MergeCopy mc) {
  using C = Shape<KVT, HD>;
  constexpr bool Q8 = C::Q8, BF = C::BF;
  constexpr int NCB = C::NCB, COLS = C::COLS, NC = C::NC, NJ = C::NJ, NI = C::NI;
  extern __shared__ __attribute__((aligned(16))) uint8_t prompt_lds[];
  uint32_t* words = (uint32_t*)(prompt_lds + 2 * C::STAGE);   // [8] K maxima, [8] V maxima, [16] the redo flag, [17] some V is not 0
  copy_merges(mc, blockIdx.x, gridDim.x);
  const uint32_t lane = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t hq = lane & 15u, grp = lane >> 4, G = u.group;
  // the unit's record: one load, a word per lane, broadcast to scalar registers
  const uint32_t word = lane < sizeof(PromptItem) / 4 ? ((const uint32_t*)(items + blockIdx.x))[lane] : 0u;
  auto fld = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)word, i); };
  const uint32_t seq = fld(0), kvh = fld(1), row0 = fld(2), pos0 = fld(3), c_off = fld(4), n_col = fld(5), page0 = fld(6),
                 n_pages = fld(7), slot = fld(8), stride = fld(9);
  const uint32_t page_end = page0 + n_pages, n_tiles = (n_pages + 3) / 4;

  // ---- page tiles of a staged item: item i of wave w is a K item (two chunk rows of a page tile; q8_0: a row of codes)
  // or a V item (the same dim row of page tiles 2h and 2h + 1, the two of half h; q8_0: a row of codes of one)
  auto is_k = [&](int i) -> bool { return HD == 64 ? w < 4 : i < NI / 2; };
  auto index = [&](int i) -> uint32_t { return HD == 64 ? w & 3u : w + 8u * (i % (NI / 2 ? NI / 2 : 1)); };
  // the page tiles (0 .. 3 of the 64-key tile) an item reads, and its row there
  auto tile_of = [&](int i, int r) -> uint32_t {
    const uint32_t x = index(i);
    if constexpr (Q8) return x / (HD / 64);
    return is_k(i) ? x / (NC / 2) : 2 * (x / NC) + r;
  };
  auto row_of = [&](int i, int r) -> uint32_t {
    const uint32_t x = index(i);
    if constexpr (Q8) return x % (HD / 64);
    return is_k(i) ? x % (NC / 2) * 2 + r : x % NC;
  };
  typedef const __attribute__((address_space(4))) int32_t cint;
  cint* tab = (cint*)(uintptr_t)(g.table + (size_t)seq * g.bps);
  const uint32_t bt_mask = (1u << g.bt_shift) - 1u;
  int blk[NI][C::ROWS_I];
  auto page_of = [&](uint32_t t, int i, int r) -> uint32_t { return min(page0 + 4 * t + tile_of(i, r), page_end - 1); };
  auto ids = [&](uint32_t t) {
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int r = 0; r < C::ROWS_I; r++) blk[i][r] = r == 1 && NI > 1 && is_k(i) ? blk[i][0] : tab[(page_of(t, i, r) << 4) >> g.bt_shift];
  };
  uint4 raw[NI][C::ROWS_I];
  uint32_t rs[NI][Q8 ? 4 : 1];   // q8_0: the scales (K: the key's two chunks; V: of four keys)
  auto request = [&](uint32_t t) {   // with the block ids of tile t
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const bool k = is_k(i);
#pragma unroll
      for (int r = 0; r < C::ROWS_I; r++) {
        const uint32_t sub = ((page_of(t, i, r) << 4) & bt_mask) >> 4;
        const uint8_t* head = g.pool + (size_t)(uint32_t)blk[i][r] * g.block_bytes + (k ? g.k_off + (size_t)kvh * g.k_head : g.v_off + (size_t)kvh * g.v_head);
        raw[i][r] = *(const uint4*)(head + (size_t)sub * (k ? g.k_tile : g.v_tile) + row_of(i, r) * 1024 + lane * 16);
        if constexpr (Q8) {
          const uint8_t* s = head + (k ? g.k_scale : g.v_scale) + (size_t)sub * (k ? g.k_tile_s : g.v_tile_s) + row_of(i, r) * 4;
          if (k) rs[i][0] = *(const uint32_t*)(s + hq * (2 * NC));
          else {
#pragma unroll
            for (int e = 0; e < 4; e++) rs[i][e] = *(const uint32_t*)(s + (4 * grp + e) * (2 * NC));
          }
        }
      }
    }
  };
  // ---- the wave's columns, and their Q on its way; then the first tile; then the rows' ranges, which lie in host memory
  // (2 us), so that they are waited for last
  uint32_t ct[NCB], ch[NCB], cpos[NCB];
  bool cv[NCB];
  f4 qv[NCB][NC][2];
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    const uint32_t c = w * COLS + 16 * x + hq;
    cv[x] = c < n_col;
    ct[x] = cv[x] ? (c + c_off) / G : 0;
    ch[x] = cv[x] ? (c + c_off) - ct[x] * G : 0;
    cpos[x] = pos0 + ct[x];
    const float* qrow = q + ((size_t)(row0 + ct[x]) * u.n_head + (size_t)kvh * G + ch[x]) * HD;
#pragma unroll
    for (int k = 0; k < NC; k++)
#pragma unroll
      for (int e = 0; e < 2; e++) qv[x][k][e] = cv[x] ? *(const f4u*)(qrow + 32 * k + 8 * grp + 4 * e) : f4u{0.f, 0.f, 0.f, 0.f};
  }
  __builtin_amdgcn_sched_barrier(0);
  ids(0);
  request(0);
  ids(1);
  __builtin_amdgcn_sched_barrier(0);
  uint2 range[NCB];   // first and last key
  float slope[NCB];
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    range[x] = make_uint2((u.window > 0 && cpos[x] + 1 > u.window) ? cpos[x] + 1 - u.window : 0, cpos[x]);
    if (sc.ranges) range[x] = sc.ranges[row0 + ct[x]];
    slope[x] = BIAS && cv[x] ? sc.slopes[kvh * G + ch[x]] * LOG2E : 0.f;
  }
  __builtin_amdgcn_sched_barrier(0);

  // ---- Q as the B operand of S^T = K Q^T: each column times 2^-e to below 1, in two parts
  float qscale[NCB];
  h8 qp[2][NCB][NC];
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    float am = 0.f;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int i = 0; i < 8; i++) am = fmaxf(am, fabsf(qv[x][c][i >> 2][i & 3]));
    const int e = min(max(__builtin_amdgcn_frexp_expf(xmax_groups(am)), -126), 126);
    const float mul = ldexpf(1.0f, -e);
    qscale[x] = ldexpf(u.scale_log2, e);
#pragma unroll
    for (int c = 0; c < NC; c++) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; i++) split_pair(qv[x][c][i >> 1][2 * (i & 1)] * mul, qv[x][c][i >> 1][2 * (i & 1) + 1] * mul, hi[i], lo[i]);
      qp[0][x][c] = __builtin_bit_cast(h8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
      qp[1][x][c] = __builtin_bit_cast(h8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
    }
  }

  // ---- the powers of two of K and V (bf16, q8_0), from the first tile
  float k_mul = 1.f, v_mul = 1.f;
  int v_exp = 0;
  if (threadIdx.x == 0) words[16] = words[17] = 0;
  if constexpr (BF || Q8) {
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < NI; i++) {
      uint32_t t = 0;
      auto see = [&](uint32_t x) { t = max(t, max(x & 0x7fffu, (x >> 16) & 0x7fffu)); };
      if constexpr (Q8) {
        see(rs[i][0]);
        if (!is_k(i)) {
          see(rs[i][1]);
          see(rs[i][2]);
          see(rs[i][3]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 2; r++) {
          see(raw[i][r].x);
          see(raw[i][r].y);
          see(raw[i][r].z);
          see(raw[i][r].w);
        }
      }
      if (is_k(i)) top[0] = max(top[0], t);
      else top[1] = max(top[1], t);
    }
    top[0] = row_max(top[0]);
    top[1] = row_max(top[1]);
#pragma unroll
    for (int x = 16; x < 64; x <<= 1) {
      top[0] = max(top[0], (uint32_t)__shfl_xor((int)top[0], x));
      top[1] = max(top[1], (uint32_t)__shfl_xor((int)top[1], x));
    }
    if (lane == 0) {
      words[w] = top[0];
      words[8 + w] = top[1];
    }
    __syncthreads();
    uint32_t km = 0, vm = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      km = max(km, words[i]);
      vm = max(vm, words[8 + i]);
    }
    auto exponent = [&](uint32_t bits) -> int {   // of the largest value: in [2^(e-1), 2^e); 0 in the usual range
      const float f = Q8 ? h_to_f((uint16_t)bits) * 127.0f : __uint_as_float(bits << 16);
      if (!(f < INFINITY) || f == 0.f) return 0;
      const int e = __builtin_amdgcn_frexp_expf(f);
      return e >= (Q8 ? -6 : 1) && e <= 8 ? 0 : min(max(e - 4, -120), 120);
    };
    const int ke = __builtin_amdgcn_readfirstlane(exponent(km));
    v_exp = __builtin_amdgcn_readfirstlane(exponent(vm));
    k_mul = ldexpf(1.0f, -ke);
    v_mul = ldexpf(1.0f, -v_exp);
#pragma unroll
    for (int x = 0; x < NCB; x++) qscale[x] = ldexpf(qscale[x], ke);
  }

  // ---- registers into an LDS buffer
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  uint32_t v_bits = 0;   // of all V written by this lane (bf16)
  u16x2 k_top = 0;   // largest |K| bits written by this lane (bf16, q8_0): 0x7c00 and more left f16's range
  const bool plain = k_mul == 1.f && v_mul == 1.f;   // uniform
  auto widen = [&](uint32_t x, float mul) -> uint32_t {   // two bf16
    f2 y = f2{__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)};
    if (!plain) {
      y *= mul;
      asm volatile("" : "+v"(y));   // not ahead of the test
    }
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(y, h2));
  };
  auto widen4 = [&](uint4 x, float mul) -> uint4 { return make_uint4(widen(x.x, mul), widen(x.y, mul), widen(x.z, mul), widen(x.w, mul)); };
  auto note = [&](uint32_t x) { k_top = __builtin_elementwise_max(k_top, __builtin_bit_cast(u16x2, x & 0x7fff7fffu)); };
  // two codes times their scales as hi and lo parts
  auto expand = [&](float a, float b, uint32_t& hi, uint32_t& lo) { split_pair(a, b, hi, lo); };
  auto write = [&](uint32_t buf) {
    uint8_t* st = prompt_lds + buf * C::STAGE;
    uint8_t* const kst = st;
    uint8_t* const vst = st + C::PARTS * C::SIDE;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      if constexpr (Q8) {
        const uint32_t t = tile_of(i, 0), r = row_of(i, 0);
        const uint32_t* cw = (const uint32_t*)&raw[i][0];
        if (is_k(i)) {   // codes 0 .. 7: chunk 2r of key hq, 8 .. 15: chunk 2r + 1
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float s = h_to_f((uint16_t)(c ? rs[i][0] >> 16 : rs[i][0])) * k_mul;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t x = cw[2 * c + (e >> 1)] >> (16 * (e & 1));
              expand((float)(int8_t)x * s, (float)(int8_t)(x >> 8) * s, hi[e], lo[e]);
              note(hi[e]);
            }
            uint8_t* at = kst + (t * NC + 2 * r + c) * 1024 + lane * 16;
            *(uint4*)at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *(uint4*)(at + C::SIDE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        } else {         // word j: dims block 4r + j, keys 4 grp .. + 3
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float s[4];
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = h_to_f((uint16_t)(j >> 1 ? rs[i][e] >> 16 : rs[i][e])) * v_mul;
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint32_t x = cw[j] >> (16 * e);
              expand((float)(int8_t)x * s[2 * e], (float)(int8_t)(x >> 8) * s[2 * e + 1], hi[e], lo[e]);
            }
            uint8_t* at = vst + ((t >> 1) * NJ + 4 * r + j) * 1024 + lane * 16 + (t & 1) * 8;
            *(uint2*)at = make_uint2(hi[0], hi[1]);
            *(uint2*)(at + C::SIDE) = make_uint2(lo[0], lo[1]);
          }
        }
      } else if (is_k(i)) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
          uint4 x = raw[i][r];
          if constexpr (BF) {
            x = widen4(x, k_mul);
            note(x.x);
            note(x.y);
            note(x.z);
            note(x.w);
          }
          *(uint4*)(kst + (tile_of(i, r) * NC + row_of(i, r)) * 1024 + lane * 16) = x;
        }
      } else {           // [4 keys of dim d | of dim d + 16] of both tiles into blocks 2b and 2b + 1 of 8 keys
        uint4 a = raw[i][0], b = raw[i][1];
        if constexpr (BF) {
          v_bits |= (a.x | a.y | a.z) | (a.w | b.x | b.y) | (b.z | b.w);
          a = widen4(a, v_mul);
          b = widen4(b, v_mul);
        }
        uint8_t* at = vst + ((tile_of(i, 0) >> 1) * NJ + 2 * row_of(i, 0)) * 1024 + lane * 16;
        *(uint4*)at = make_uint4(a.x, a.y, b.x, b.y);
        *(uint4*)(at + 1024) = make_uint4(a.z, a.w, b.z, b.w);
      }
    }
  };
  write(0);
  // ---- the keys the columns see
  uint32_t clo[NCB], clen[NCB];   // a column sees keys clo .. clo + clen - 1 of the unit's
  uint32_t lo_max = 0, hi_min = 0, lo_min = 0, end_max = 0;   // (the least of x as the most of ~x)
  bool any = false;   // some column of the wave sees a key
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    clo[x] = range[x].x;
    const uint32_t last = min(range[x].y, (page_end << 4) - 1);
    clen[x] = clo[x] <= last ? last + 1 - clo[x] : 0;
    if (cv[x]) {
      lo_max = max(lo_max, clo[x]);
      hi_min = max(hi_min, ~last);
      if (clen[x]) {
        lo_min = max(lo_min, ~clo[x]);
        end_max = max(end_max, last);
        any = true;
      }
    }
  }
  lo_max = __builtin_amdgcn_readfirstlane(row_max(lo_max));
  const uint32_t end_min = ~(uint32_t)__builtin_amdgcn_readfirstlane(row_max(hi_min));
  lo_min = ~(uint32_t)__builtin_amdgcn_readfirstlane(row_max(lo_min));     // no column of the wave sees a key outside lo_min .. end_max
  end_max = __builtin_amdgcn_readfirstlane(row_max(end_max));
  any = __ballot(any) != 0;
  __syncthreads();

  // ---- the walk
  constexpr int VP = 4;   // V operands of a tile requested before its softmax (none: q8_0 prompts 104.8 -> 107.7 us)
  constexpr float UP = 7.0f;   // weights up to 2^15: more of them in f16's range
  // a column's weights are taken against mref = m - UP, m a score of it that none exceeds by more than 8 (room: how far
  // scores may exceed mref; -inf before its first, while every score is -inf)
  float mref[NCB], room[NCB], lsum[NCB];
  f4 O[NCB][NJ];
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    mref[x] = 0.f;
    room[x] = -INFINITY;
    lsum[x] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; j++) O[x][j] = f4{0.f, 0.f, 0.f, 0.f};
  }
#pragma clang loop unroll(disable)
  for (uint32_t t = 0; t < n_tiles; t++) {
    if (t + 1 < n_tiles) {
      request(t + 1);
      ids(t + 2);
    }
    const uint8_t* st = prompt_lds + (t & 1) * C::STAGE + lane * 16;
    const uint32_t key0 = (page0 + 4 * t) << 4;
    if (any && key0 <= end_max && key0 + 63 >= lo_min) {   // uniform over the wave
      f4 s[NCB][4];
#pragma unroll
      for (int x = 0; x < NCB; x++)
#pragma unroll
        for (int kk = 0; kk < 4; kk++) s[x][kk] = f4{0.f, 0.f, 0.f, 0.f};
      // (products into one accumulator wait for each other: two key blocks' between them)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int c = 0; c < NC; c++) {
          h8 kc[2];
#pragma unroll
          for (int kk = 0; kk < 2; kk++) kc[kk] = *(const h8*)(st + ((2 * h + kk) * NC + c) * 1024);
#pragma unroll
          for (int p = 0; p < 2; p++)
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
              for (int x = 0; x < NCB; x++) s[x][2 * h + kk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[kk], qp[p][x][c], s[x][2 * h + kk], 0, 0, 0);
          if constexpr (Q8) {
#pragma unroll
            for (int kk = 0; kk < 2; kk++) kc[kk] = *(const h8*)(st + ((2 * h + kk) * NC + c) * 1024 + C::SIDE);
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
              for (int x = 0; x < NCB; x++) s[x][2 * h + kk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[kk], qp[0][x][c], s[x][2 * h + kk], 0, 0, 0);
          }
        }
      // the first of V's operands on their way before the softmax
      const uint8_t* const vst = st + C::PARTS * C::SIDE;
      h8 vpre[VP];
#pragma unroll
      for (int j = 0; j < VP; j++) vpre[j] = *(const h8*)(vst + j * 1024);
      __builtin_amdgcn_sched_barrier(0);
      const bool need_mask = key0 + 63 > end_min || key0 < lo_max;
      float p[NCB][16];   // scores less the reference mref
#pragma unroll
      for (int x = 0; x < NCB; x++) {
        if constexpr (CAP) {
#pragma unroll
          for (int i = 0; i < 16; i++) p[x][i] = s[x][i >> 2][i & 3] * qscale[x];
          cap_scores<16>(p[x], sc.cap_log2);
#pragma unroll
          for (int i = 0; i < 16; i++) p[x][i] -= mref[x];
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) p[x][i] = fmaf(s[x][i >> 2][i & 3], qscale[x], -mref[x]);
        }
        if constexpr (BIAS) bias_scores<16>(p[x], slope[x], (float)(int)(key0 + 4 * grp - cpos[x]), [](int i) { return (float)(16 * (i >> 2) + (i & 3)); });
        if (need_mask) {
          const uint32_t at = key0 + 4 * grp - clo[x];   // (keys before clo wrap round)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            p[x][i] = at + 16 * (i >> 2) + (i & 3) < clen[x] ? p[x][i] : -INFINITY;
            asm volatile("" : "+v"(p[x][i]));   // not ahead of the test
          }
        }
        float lm = p[x][0];
#pragma unroll
        for (int i = 1; i < 16; i++) lm = fmaxf(lm, p[x][i]);
        if (__ballot(lm > room[x])) {   // some column's largest score is 8 past its m, or its first
          const float tm = xmax_groups(lm) + mref[x];
          if (tm - mref[x] > room[x]) {
            const float nref = tm - UP, alpha = room[x] == -INFINITY ? 0.f : exp2_fast(mref[x] - nref);
            lsum[x] *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; j++) O[x][j] *= alpha;
#pragma unroll
            for (int i = 0; i < 16; i++) p[x][i] -= nref - mref[x];
            mref[x] = nref;
            room[x] = UP + 8.0f;
          }
        }
      }
      // weights of half h; those of the second beside the products of the first
      h8 ph[2][NCB], pl[2][NCB];
      auto weights = [&](int h) {
#pragma unroll
        for (int x = 0; x < NCB; x++) {
          float* e = p[x] + 8 * h;
#pragma unroll
          for (int i = 0; i < 8; i++) e[i] = exp2_fast(e[i]);
          lsum[x] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
          uint32_t hw[4], lw[4];
#pragma unroll
          for (int i = 0; i < 4; i++) split_pair(e[2 * i], e[2 * i + 1], hw[i], lw[i]);
          ph[h][x] = __builtin_bit_cast(h8, make_uint4(hw[0], hw[1], hw[2], hw[3]));
          pl[h][x] = __builtin_bit_cast(h8, make_uint4(lw[0], lw[1], lw[2], lw[3]));
        }
      };
      auto products = [&](int h) {
        const uint8_t* const vh = vst + h * NJ * 1024;
#pragma unroll
        for (int j0 = 0; j0 < NJ; j0 += 2) {
          h8 va[2];
#pragma unroll
          for (int e = 0; e < 2; e++) va[e] = h == 0 && j0 + e < VP ? vpre[j0 + e < VP ? j0 + e : 0] : *(const h8*)(vh + (j0 + e) * 1024);
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int x = 0; x < NCB; x++) O[x][j0 + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], ph[h][x], O[x][j0 + e], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int x = 0; x < NCB; x++) O[x][j0 + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], pl[h][x], O[x][j0 + e], 0, 0, 0);
          if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 2; e++) va[e] = *(const h8*)(vh + (j0 + e) * 1024 + C::SIDE);
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
              for (int x = 0; x < NCB; x++) O[x][j0 + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], ph[h][x], O[x][j0 + e], 0, 0, 0);
          }
        }
      };
      weights(0);
      products(0);
      weights(1);
      products(1);
    }
    if (t + 1 < n_tiles) write((t + 1) & 1);
    __syncthreads();
  }

  // ---- results
  if constexpr (BF || Q8) {
    if (max(k_top[0], k_top[1]) >= 0x7c00) words[16] = 1;
    if (BF && (v_bits & 0x7fff7fffu)) words[17] = 1;
    __syncthreads();
  }
  const bool all = (BF || Q8) && words[16] != 0, lossy = BF ? words[17] != 0 : Q8 && v_mul < 1.f;
  bool bad[NCB], some = false;
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    lsum[x] = xsum_groups(lsum[x]);
    float z = lsum[x];
#pragma unroll
    for (int j = 0; j < NJ; j++) z += (O[x][j][0] + O[x][j][1]) + (O[x][j][2] + O[x][j][3]);
    bad[x] = all || !__builtin_isfinite(z);
    if (lossy) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; j++) top = fmaxf(top, fmaxf(fmaxf(fabsf(O[x][j][0]), fabsf(O[x][j][1])), fmaxf(fabsf(O[x][j][2]), fabsf(O[x][j][3]))));
      top = xmax_groups(top);
      bad[x] |= top * top * (float)min(clen[x], n_pages << 4) < lsum[x] * lsum[x] * 0x1p-10f;
    }
    bad[x] &= cv[x];
    some |= bad[x];
  }
  auto row_at = [&](uint32_t tok, uint32_t head) -> float* {
    if (slot == NO_SLOT) return out + ((size_t)(row0 + tok) * u.n_head + (size_t)kvh * G + head) * HD;
    return u.part + ((size_t)(slot + tok * stride) * u.ng + head) * (HD + 4);
  };
  if (__builtin_expect(__ballot(some) != 0, 0)) {
    uint32_t again = 0;   // a bit per column of the wave
#pragma unroll
    for (int x = 0; x < NCB; x++) {
      uint64_t b = __ballot(bad[x]);
      b |= b >> 32;
      b |= b >> 16;
      again |= ((uint32_t)b & 0xffffu) << (16 * x);
      cv[x] = cv[x] && !(again >> (16 * x + hq) & 1u);
    }
#pragma clang loop unroll(disable)
    for (; again; again &= again - 1) {
      const uint32_t a = w * COLS + (uint32_t)__builtin_ctz(again) + c_off, tok = a / G, head = a - tok * G, pos = pos0 + tok;
      uint32_t first = (u.window > 0 && pos + 1 > u.window) ? pos + 1 - u.window : 0, last = pos;
      if (sc.ranges) {
        const uint2 r = sc.ranges[row0 + tok];
        first = r.x;
        last = r.y;
      }
      first = max(first, page0 << 4);
      const uint32_t end = first > last ? first : min(last + 1, page_end << 4);   // (end <= first: it sees nothing here)
      redo<KVT, HD>(g, u, sc, seq, kvh, kvh * G + head, pos, first, end,
                    q + ((size_t)(row0 + tok) * u.n_head + (size_t)kvh * G + head) * HD, row_at(tok, head), slot != NO_SLOT);
    }
  }
#pragma unroll
  for (int x = 0; x < NCB; x++) {
    if (!cv[x]) continue;
    float* op = row_at(ct[x], ch[x]);
    const float mul = (slot != NO_SLOT ? 1.0f : lsum[x] == 0.f ? 0.f : 1.0f / lsum[x]) * ldexpf(1.0f, v_exp);
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const f4 o = O[x][j] * mul;
      *(f4u*)(op + 16 * j + 4 * grp) = f4u{o[0], o[1], o[2], o[3]};
    }
    if (slot != NO_SLOT && grp == 0) {
      op[HD] = room[x] == -INFINITY ? -INFINITY : mref[x];   // the reference the weights were taken against
      op[HD + 1] = lsum[x];
    }
  }
}

// f(type, width) of the instance that takes a geometry; false: none does.
template <typename Fn>
bool with_prompt(uint32_t kv_type, uint32_t hd, uint32_t hdv, uint32_t layout, Fn&& f) {
  if (layout != LAYOUT_TILES || hd != hdv) return false;
#define LMH_P(T, H)                                                                              \
  if (kv_type == T && hd == H) {                                                                 \
    f(std::integral_constant<uint32_t, T>{}, std::integral_constant<int, H>{});                  \
    return true;                                                                                 \
  }
  LMH_P(KV_F16, 64) LMH_P(KV_F16, 128) LMH_P(KV_F16, 256) LMH_P(KV_BF16, 64) LMH_P(KV_BF16, 128) LMH_P(KV_BF16, 256)
  LMH_P(KV_Q8, 64) LMH_P(KV_Q8, 128)
#undef LMH_P
  return false;
}

}  // namespace

uint32_t scored_prompt_cols(uint32_t kv_type, uint32_t hd, uint32_t hdv, uint32_t layout) {
  uint32_t n = 0;
  with_prompt(kv_type, hd, hdv, layout, [&](auto t, auto h) { n = PW * Shape<decltype(t)::value, decltype(h)::value>::COLS; });
  return n;
}

hipError_t launch_scored_prompts(const PageGeom& g, const UnitGeom& u, const ScoreGeom& sc, const PromptItem* items, uint32_t n_items,
                                 const float* q, float* out, const MergeCopy& mc, hipStream_t s, const LaunchEv& ev) {
  if (n_items == 0) return hipSuccess;
  hipError_t e = hipErrorInvalidValue;
  with_prompt(g.kv_type, g.hd, g.hdv, g.layout, [&](auto t, auto h) {
    constexpr int T = decltype(t)::value, H = decltype(h)::value;
#define LMH_PROMPT(CAP, BIAS) \
  LMH_LAUNCH(ev, (scored_prompt_kernel<T, H, CAP, BIAS>), dim3(n_items), dim3(NTH), (Shape<T, H>::LDS), s, g, u, sc, items, q, out, mc)
    if (sc.cap_log2 > 0.f) {
      if (sc.slopes) LMH_PROMPT(true, true);
      else LMH_PROMPT(true, false);
    } else {
      if (sc.slopes) LMH_PROMPT(false, true);
      else LMH_PROMPT(false, false);
    }
#undef LMH_PROMPT
    e = hipGetLastError();
  });
  return e;
}

}  // namespace lmh
