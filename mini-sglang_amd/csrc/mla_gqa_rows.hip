// Grouped-head attention for many rows (tokens times group): whole prompts, and chunks over a paged cache. See mla_gqa.h for
// the mathematics.
//
// One CTA per (request, 32 NW rows, KV head, piece of the keys), NW waves x 32 rows, two waves per SIMD: NW 4 (two CTAs
// on a compute unit) or 8 (one). With KS 2 a CTA has two of four waves, each for half of the keys, joined at the end.
//  * Keys stream in stages of 32 through a K ring and a V ring in LDS, filled by 16-byte DMA loads whose sources are
//    per token, so that a page may end anywhere (rows of a paged cache are looked up a window at a time into LDS).
//    Keys past the last repeat it. 16-byte chunks are permuted within a row (kchunk, vchunk), so that neither the K
//    reads (16 rows at a time) nor the transposing V reads meet in a bank.
//  * S^T[32 keys x 32 rows] = K . Q^T and O^T[D dims x 32 rows] += V^T . P^T on 32x32x16 bf16 MFMA; queries and O stay
//    in registers.
//  * Software pipeline: step j issues the score MFMAs of stage j + 1 and then the value MFMAs of stage j - 1 while the
//    vector ALU runs the softmax of stage j, spread over the MFMAs.
//  * Online softmax in the log2 domain against a lazy row reference: the maximum of the wave's first stage, moved (with O
//    and l rescaled, and the stage redone) only when a lane's numerators of a stage sum past 2^32. The reference is a
//    rounded product m = round(max s * scale), the numerators are 2^(fma(s, scale, -m) - d): d = fma(max s, scale, -m), what
//    the rounding left out, keeps the largest at 1. Below |m| = 2^24 it is at most half a bit and taken as 0, which keeps the
//    subtraction out of the loop; a wave with a row past that redoes its stages.
// Bound: the MFMAs, and under them power: prompts of 7.8k and 8.1k tokens with 64 and 8 heads of 128 take 1.76 ms, 1164
// TFLOP/s, with the MFMAs busy for 62 % of the cycles at 1.4 to 1.8 GHz from dispatch to dispatch (alone, on random operands,
// they run at 1829 TFLOP/s and 1.74 GHz); four chunks of 2048 on up to 8192, pages of 64, 1.17 ms, 1170 TFLOP/s. Short calls
// are bound by their CTA's chain: 1.2 us to find the request, 2 to the first stage, 0.45 a stage for a lone CTA, 1 to 1.8 for
// the results.
// Waves of 64 rows (one per SIMD; each K and V operand read once for two MFMAs) took 1098 TFLOP/s where these took 1170.
#include <type_traits>

#include "mla_gqa.h"

namespace mla {
namespace {

typedef float f32x16_t __attribute__((__vector_size__(64)));

constexpr int kStage = 32;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLazyMax = 4294967296.0f;
constexpr float kFar = 16777216.0f;  // references from here on have a rounding that counts

template <int N>
using ic = std::integral_constant<int, N>;
template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(ic<I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// Rings: group n is K stage n and V stage n - 2. Step j issues group j + kDist, scores stage j + 1, adds the values of
// stage j - 1 and reads ahead into K stage j + 2. Every kSync steps a barrier makes the groups up to j + kSync + 1
// visible, those of the steps up to the next barrier. A slot is refilled kRing - kDist + 1 steps after its stage's last
// read (K stage s in step s - 1, V stage s in step s + 1), which must pass a barrier: kRing >= kDist + kSync - 1.
template <int NW>
struct Rings;
template <>
struct Rings<4> {
  static constexpr int kSync = 1, kDist = 4, kRing = 4, kWindow = 2048;
};
template <>
struct Rings<8> {
  static constexpr int kSync = 2, kDist = 7, kRing = 8, kWindow = 4096;
};
template <int NW>
constexpr bool rings_ok() {
  using S = Rings<NW>;
  return S::kRing >= S::kDist + S::kSync - 1 && S::kDist >= S::kSync + 2 && S::kRing % 2 == 0 && S::kRing % S::kSync == 0 &&
         S::kWindow >= (2 * S::kRing + S::kDist) * kStage;
}
static_assert(rings_ok<4>() && rings_ok<8>(), "ring lengths");

// Position of 16-byte chunk c of token t in a K / V row of an LDS tile. A 16-byte read serves 16 lanes at a time, of each
// 32 lanes 0-3, 12-15 and 20-27, then the others: their tokens' chunks lie in different banks.
template <int D>
__device__ __forceinline__ int kchunk(int c, int t) {
  return D == 128 ? c ^ (t & 15) : c ^ ((t >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int vchunk(int c, int t) {
  return D == 128 ? c ^ (4 * (t & 3)) : c ^ (4 * ((t >> 1) & 1));
}

__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Pins a value to its slot of the instruction stream (volatile statements keep their order).
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void pin(uint32_t& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void pin(f32x16_t& x) { asm volatile("" : "+v"(x)); }

// The softmax of a stage as 24 micro-operations: for u = 3 k + r (pair k of a lane's 16 scores), r < 2 is the exponential
// of score 2 k + r, r == 2 adds the pair to the row sum and packs it. Spread over a step's MFMA slots in proportion to
// their cost.
constexpr int kUops = 24;
constexpr int uop_total(int n) {
  int t = 0;
  for (int u = 0; u < n; ++u) t += u % 3 < 2 ? 5 : 6;
  return t;
}
constexpr int uop_slot(int u, int slots) { return uop_total(u) * slots / uop_total(kUops); }

template <int D, int NW, int KS, bool kPaged>
__global__ __launch_bounds__(64 * NW * KS, 2) void gqa_rows_kernel(const GqaParams p) {
  using S = Rings<NW>;
  constexpr int kRows = 32 * NW, kRowB = D * 2, kTileB = kStage * kRowB;
  constexpr int kKs = D / 16, kDb = D / 32, kVs = 2 * kDb;  // K operands, 32-dim blocks, V operands of a stage
  constexpr int kSlots = kVs + kKs;                         // MFMAs of a step
  constexpr int kLd = kTileB / 1024 / NW;                   // a wave's K (V) loads of a stage, 1 KB each
  static_assert(kLd >= 1, "every wave loads K and V");
  constexpr int kPerLoad = 1024 / kRowB;  // tokens of a load
  constexpr int kRingB = S::kRing * kTileB;
  constexpr int kAK = D == 128 ? 4 : 3, kAV = 3;  // operands read ahead
  static_assert(kAK <= kVs && kAV <= kKs, "read ahead by less than a step");
  __shared__ __attribute__((aligned(1024))) char smem[KS * 2 * kRingB];
  static_assert(KS == 1 || !kPaged, "one window of rows");
  __shared__ int s_row[kPaged ? S::kWindow : 1];

  const int lane = threadIdx.x & 63;
  const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_all % NW, part = wave_all / NW;  // part: of the keys
  GqaItem it;
  if (!gqa_find<kRows, true>(p, blockIdx.x, it)) return;
  const int E = it.r.E, L = it.r.L, P = it.r.P, G = p.group;
  const int c32 = lane & 31, g32 = lane >> 5;
  const int row0 = it.block * kRows + 32 * wave;  // the wave's first row
  const int tok0 = row0 / G, rem0 = row0 - tok0 * G;
  const float inv_g = 1.f / (float)G;
  // token and head of the wave's row i (rem0 + i < G + 32: exact)
  auto tok_of = [&](int i) __attribute__((always_inline)) { return tok0 + (int)(((float)(rem0 + i) + 0.5f) * inv_g); };
  auto head_of = [&](int i, int tok) __attribute__((always_inline)) { return it.head * G + rem0 + i - (tok - tok0) * G; };
  const int last_tok = min(E - 1, (it.block * kRows + kRows - 1) / G);
  const int k0_all = it.piece * it.C, k1_all = min(it.pieces > 1 ? k0_all + it.C : L, P + last_tok + 1);
  // stages, of each part alike (the last part's may lie past its keys)
  const int nst = __builtin_amdgcn_readfirstlane(k1_all > k0_all ? ((k1_all - k0_all + kStage - 1) / kStage + KS - 1) / KS : 0);
  const int k0 = k0_all + part * nst * kStage, k1 = part + 1 < KS ? min(k0 + nst * kStage, k1_all) : k1_all;
  int W = 0;  // stages that the wave needs
  if (tok0 < E) W = (min(k1, P + min(E - 1, (row0 + 31) / G) + 1) - k0 + kStage - 1) / kStage;
  W = __builtin_amdgcn_readfirstlane(max(W, 0));
  // the first stage with a key that some row of the wave does not see
  const int j_diag = __builtin_amdgcn_readfirstlane(max(min(P + tok0 + 1, k1) - k0, 0) >> 5);

  const int tok = tok_of(c32), head = head_of(c32, tok);
  const bool live = tok < E;
  // last key of the lane's row, from k0; rows past the last query repeat the request's first (and are not written)
  const int limit = min(live ? P + tok : k1 - 1, k1 - 1) - k0;
  bf16x8 qf[kKs];
  {
    const __bf16* q = p.q + (int64_t)(it.r.q0 + (live ? tok : 0)) * p.q_stride_t + (int64_t)(live ? head : it.head * G) * p.q_stride_h + 8 * g32;
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(q + 16 * ks);
  }

  f32x16_t O[kDb];
#pragma unroll
  for (int db = 0; db < kDb; ++db) O[db] = f32x16_t{};
  float m_ref = kLowest, negm = -kLowest, d_ref = 0.f, l_run = 0.f;
  uint64_t far = 0;  // lanes whose reference is past kFar

  if (nst > 0) {
    // ---- sources: token t of the piece
    const int last = L - 1 - k0;
    int w0 = 0;  // first token of the window
    auto fill = [&]() __attribute__((always_inline)) {
      if constexpr (kPaged) {
        const int need = min(S::kWindow, (nst + S::kDist + S::kRing) * kStage - w0);
        for (int t0 = 0; t0 < need; t0 += 4 * 64 * NW) {
          int r[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t = t0 + threadIdx.x + 64 * NW * u;
            if (t < need) r[u] = gqa_row(p, it.b, it.r.q0, k0 + min(w0 + t, last));
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t = t0 + threadIdx.x + 64 * NW * u;
            if (t < need) s_row[t] = r[u];
          }
        }
      }
    };
    fill();
    // load i of a wave covers kPerLoad tokens of the stage, lane's token tk[i], 16-byte chunk position lane % (D / 8)
    const char* kb[kLd];
    const char* vb[kLd];
    int tk[kLd];
#pragma unroll
    for (int i = 0; i < kLd; ++i) {
      tk[i] = (wave * kLd + i) * kPerLoad + lane / (D / 8);
      const int c = lane % (D / 8);
      kb[i] = reinterpret_cast<const char*>(p.k + (int64_t)it.head * p.k_head_stride) + kchunk<D>(c, tk[i]) * 16;
      vb[i] = reinterpret_cast<const char*>(p.v + (int64_t)it.head * p.v_head_stride) + vchunk<D>(c, tk[i]) * 16;
    }
    const uint32_t ks_b = (uint32_t)(p.k_row_stride * 2), vs_b = (uint32_t)(p.v_row_stride * 2);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(MLA_LDS char*)smem + part * 2 * kRingB + wave * kLd * 1024;
    int row[kLd], row_1[kLd], row_v[kLd];  // of group n's K stage, the one before, and V stage n - 2
    auto rows_of = [&](int n) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kLd; ++i) {
        row_v[i] = row_1[i];
        row_1[i] = row[i];
        if constexpr (kPaged) row[i] = s_row[n * kStage - w0 + tk[i]];
        else row[i] = it.r.q0 + k0 + min(n * kStage + tk[i], last);
      }
    };
    auto dma = [&](int n, uint32_t kslot, uint32_t vslot) __attribute__((always_inline)) {
      const int i = n % kLd;
      if (n < kLd) dma16_vaddr(kb[i] + (uint64_t)(uint32_t)row[i] * ks_b, lds0 + kslot * kTileB + i * 1024);
      else dma16_vaddr(vb[i] + (uint64_t)(uint32_t)row_v[i] * vs_b, lds0 + kRingB + vslot * kTileB + i * 1024);
    };
    auto group_now = [&](int n) __attribute__((always_inline)) {
      rows_of(n);
#pragma unroll
      for (int l = 0; l < 2 * kLd; ++l) dma(l, n % S::kRing, (n + S::kRing - 2) % S::kRing);
    };
    auto sync_groups = [&](auto ng) __attribute__((always_inline)) {
      wait_vmcnt<2 * kLd * decltype(ng)::value>();
      __builtin_amdgcn_s_barrier();
    };

    barrier_lds();  // s_row is written
    rows_of(0);     // groups 0 and 1 fill V slots of no stage with V stage 0
#pragma unroll
    for (int i = 0; i < kLd; ++i) row_1[i] = row[i];
    for (int n = 0; n < S::kDist - 1; ++n) group_now(n);
    // the queries stay in registers and have landed here, with the first groups issued behind them; the wait is
    // explicit, since the compiler does not count the DMA loads
    wait_vmcnt<0>();
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) asm volatile("" : "+v"(qf[ks]));

    // ---- operand reads
    int k_off[kKs], v_off[kDb];
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) k_off[ks] = part * 2 * kRingB + c32 * kRowB + kchunk<D>(2 * ks + g32, c32) * 16;
    // V^T operand: keys 16 ksp + 8 e + 4 g32 + 0..3 (e = 0, 1) of dims 32 db + 16 (gq & 1) + ..., as the numerators lie
    const int gq = lane >> 4, a16 = lane & 15, vt = 4 * (gq >> 1) + (a16 >> 2);
#pragma unroll
    for (int db = 0; db < kDb; ++db) v_off[db] = part * 2 * kRingB + kRingB + vt * kRowB + vchunk<D>(4 * db + 2 * (gq & 1) + ((a16 & 3) >> 1), vt) * 16 + (a16 & 1) * 8;
    auto kread = [&](int slot, int ks) __attribute__((always_inline)) {
      return *reinterpret_cast<const MLA_LDS bf16x8*>((const MLA_LDS char*)smem + slot * kTileB + k_off[ks]);
    };
    auto vread = [&](int slot, int st) __attribute__((always_inline)) {
      const MLA_LDS char* base = (const MLA_LDS char*)smem + slot * kTileB + v_off[st >> 1] + 16 * (st & 1) * kRowB;
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((MLA_LDS bf16x4*)base);
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((MLA_LDS bf16x4*)(base + 8 * kRowB));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    f32x16_t sc[2];  // [parity]: scores of the stage being softmaxed / being computed
    u32x4 pb[2][2];  // [parity]: bf16 numerators P^T
    bf16x8 vop[kAV + 1], kop[kAK + 1];
    auto mask = [&](f32x16_t& s, int j, bool all) __attribute__((always_inline)) {
      const int lim = all ? -1 : limit - j * kStage - 4 * g32;  // score i: key 8 (i / 4) + 4 g32 + i % 4
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + (i & 3) > lim) s[i] = -INFINITY;
    };
    // the reference of a stage by itself: m, and what its rounding left out
    auto top_of = [&](const f32x16_t& s, float& m, float& d) __attribute__((always_inline)) {
      float t = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) t = fmaxf(t, s[i]);
      t = max_halves(t);
      m = fmaxf(t * p.scale_log2, kLowest);  // (a stage of -inf alone: its numerators are 0)
      d = fabsf(m) >= kFar && m > kLowest ? fmaf(t, p.scale_log2, -m) : 0.f;
    };
    auto refer = [&](float m, float d) __attribute__((always_inline)) {
      m_ref = m;
      negm = -m;
      d_ref = d;
      far = __ballot(fabsf(m) >= kFar && m > kLowest);
    };
    auto redo = [&](const f32x16_t& s, u32x4 (&dst)[2], float& l_step) __attribute__((always_inline)) {
      float m, d;
      top_of(s, m, d);
      if (!(m > m_ref || (m == m_ref && d > d_ref))) m = m_ref, d = d_ref;
      const float fr = __builtin_amdgcn_exp2f((m_ref - m) + (d_ref - d));
      refer(m, d);
      l_run *= fr;
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[2 * k], p.scale_log2, negm) - d_ref);
        const float e1 = __builtin_amdgcn_exp2f(fmaf(s[2 * k + 1], p.scale_log2, negm) - d_ref);
        l += e0 + e1;
        dst[k >> 2][k & 3] = pack_bf16x2(e0, e1);
      }
      l_step = l;
#pragma unroll
      for (int db = 0; db < kDb; ++db) {
        O[db] *= fr;
        pin(O[db]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    // ---- pipelined step; U: its number modulo the rings
    auto step_fast = [&](auto u_c) __attribute__((always_inline)) {
      constexpr int U = decltype(u_c)::value, par = U & 1;
      constexpr int v_prev = (U + S::kRing - 1) % S::kRing, k_next = (U + 1) % S::kRing, k_next2 = (U + 2) % S::kRing;
      constexpr int kslot = (U + S::kDist) % S::kRing, vslot = (U + S::kDist + S::kRing - 2) % S::kRing;
      constexpr int kDmaEvery = kSlots / (2 * kLd);
      float l_step, ev[2];
      static_for<kSlots>([&](auto s_c) __attribute__((always_inline)) {
        constexpr int s = decltype(s_c)::value;
        if constexpr (s < kKs) {
          if constexpr (s == 0) sc[par ^ 1] = f32x16_t{};
          sc[par ^ 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop[s % (kAK + 1)], qf[s], sc[par ^ 1], 0, 0, 0);
        } else {
          constexpr int st = s - kKs;
          O[st >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vop[st % (kAV + 1)], __builtin_bit_cast(bf16x8, pb[par ^ 1][st & 1]), O[st >> 1], 0, 0, 0);
          pin(O[st >> 1]);
        }
        if constexpr (s % kDmaEvery == kDmaEvery - 1) dma(s / kDmaEvery, kslot, vslot);
        {  // operand reads
          constexpr int ks = s + kAK, ksn = s + kAK - kSlots, st = s - kKs + kAV;
          if constexpr (ks < kKs) kop[ks % (kAK + 1)] = kread(k_next, ks);
          if constexpr (ksn >= 0 && ksn < kAK) kop[ksn % (kAK + 1)] = kread(k_next2, ksn);
          if constexpr (st >= 0 && st < kVs) vop[st % (kAV + 1)] = vread(v_prev, st);
        }
        static_for<kUops>([&](auto w_c) __attribute__((always_inline)) {
          constexpr int u = decltype(w_c)::value, k = u / 3, r = u % 3;
          if constexpr (uop_slot(u, kSlots) == s) {
            if constexpr (r < 2) {
              ev[r] = __builtin_amdgcn_exp2f(fmaf(sc[par][2 * k + r], p.scale_log2, negm));
              pin(ev[r]);
            } else {
              l_step = k == 0 ? ev[0] + ev[1] : l_step + ev[0] + ev[1];
              uint32_t x = pack_bf16x2(ev[0], ev[1]);
              pin(l_step);
              pin(x);
              pb[par][k >> 2][k & 3] = x;
            }
          }
        });
        __builtin_amdgcn_sched_barrier(0);
      });
      if ((__ballot(l_step >= kLazyMax) | far) != 0) redo(sc[par], pb[par], l_step);
      l_run += l_step;
    };
    auto step = [&](auto u_c, int j) __attribute__((always_inline)) {
      constexpr int U = decltype(u_c)::value, par = U & 1;
      if (j > nst) return;
      if constexpr (U % S::kSync == 0) sync_groups(ic<S::kDist - 2 - S::kSync>{});
      if (__builtin_expect(j <= W && W > 0, 1)) {
        rows_of(j + S::kDist);
        if (__builtin_expect(j >= j_diag || j == W, 0)) mask(sc[par], j, j == W);
        if constexpr (U == 0) if (__builtin_expect(j == 0, 0)) {
          float m, d;
          top_of(sc[par], m, d);
          refer(m, d);
        }
        step_fast(u_c);
        if constexpr (U == 0) if (__builtin_expect(j == 0, 0))
          // step 0 has no stage before it: its value pass multiplied zeros with what the V ring's last slot held
#pragma unroll
          for (int db = 0; db < kDb; ++db) O[db] = f32x16_t{};
      } else {
        group_now(j + S::kDist);
      }
    };

    pb[1][0] = pb[1][1] = u32x4{};
    // step -1: the scores of stage 0
    __builtin_amdgcn_s_barrier();
    group_now(S::kDist - 1);
    if (W > 0) {
      sc[0] = f32x16_t{};
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kread(0, ks), qf[ks], sc[0], 0, 0, 0);
#pragma unroll
      for (int ks = 0; ks < kAK; ++ks) kop[ks] = kread(1, ks);
    }
    for (int j0 = 0; j0 <= nst; j0 += S::kRing) {
      if constexpr (kPaged) {
        // the next kRing steps issue K stages j0 + kDist .. j0 + kDist + kRing - 1
        if (__builtin_expect((j0 + S::kDist + S::kRing) * kStage > w0 + S::kWindow, 0)) {
          barrier_lds();  // every wave is done with the window
          w0 = (j0 + S::kDist) * kStage;
          fill();
          barrier_lds();
        }
      }
      static_for<S::kRing>([&](auto u_c) __attribute__((always_inline)) { step(u_c, j0 + decltype(u_c)::value); });
    }
    wait_vmcnt<0>();  // the last groups have landed before the CTA ends
  }

  if constexpr (KS == 2) {
    // the second part's O to the first's waves, lane by lane, through its own rings, its sums through the first's V ring;
    // the first's K ring serves the output
    static_assert(NW * 64 * kDb * 16 * 4 <= 2 * kRingB && NW * 64 * 3 * 4 <= kRingB && NW * 32 * kRowB <= kRingB, "they fit");
    MLA_LDS float* s = (MLA_LDS float*)((MLA_LDS char*)smem + 2 * kRingB) + wave * 64 * kDb * 16 + lane;
    MLA_LDS float* s_ml = (MLA_LDS float*)((MLA_LDS char*)smem + kRingB) + wave * 192 + lane;
    __syncthreads();  // both are done with their rings
    if (part == 1) {
#pragma unroll
      for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[64 * (16 * db + i)] = O[db][i];
      s_ml[0] = m_ref;
      s_ml[64] = l_run;
      s_ml[128] = d_ref;
    }
    __syncthreads();
    if (part == 1) return;
    const float m1 = s_ml[0], l1 = s_ml[64], d1 = s_ml[128];
    const bool second = m1 > m_ref || (m1 == m_ref && d1 > d_ref);
    const float m = second ? m1 : m_ref, d = second ? d1 : d_ref;
    const float f0 = __builtin_amdgcn_exp2f((m_ref - m) + (d_ref - d)), f1 = __builtin_amdgcn_exp2f((m1 - m) + (d1 - d));
    m_ref = m;
    d_ref = d;
    l_run = l_run * f0 + l1 * f1;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) O[db][i] = O[db][i] * f0 + s[64 * (16 * db + i)] * f1;
  }
  // ---- results: a lane holds row c32, dims 32 db + 8 i4 + 4 g32 + 0..3
  const float l = sum_halves(l_run);
  const bool some = l > 0.f || l != l;
  const float inv = some ? 1.f / l : 0.f;
  const f32x2 lse2 = gqa_lse(some, m_ref, d_ref + log2f(l));
  const int64_t at = (int64_t)it.slot * kRows + 32 * wave + c32;
  if (it.slot >= 0) {
    if (live) {
#pragma unroll
      for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          f32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = O[db][4 * i4 + i] * inv;
          *reinterpret_cast<f32x4*>(p.ws_o + at * D + 32 * db + 8 * i4 + 4 * g32) = v;
        }
      if (g32 == 0) p.ws_lse[at] = lse2;
    }
  } else {
    if (p.lse != nullptr && g32 == 0 && live) p.lse[(int64_t)(it.r.q0 + tok) * p.lse_stride_t + head] = lse2[0] * 0.69314718055994531f;
    auto packed = [&](int db, int i4) __attribute__((always_inline)) {
      return u32x2{pack_bf16x2(O[db][4 * i4] * inv, O[db][4 * i4 + 1] * inv), pack_bf16x2(O[db][4 * i4 + 2] * inv, O[db][4 * i4 + 3] * inv)};
    };
    auto out_row = [&](int t, int h) __attribute__((always_inline)) { return p.out + (int64_t)(it.r.q0 + t) * p.out_stride_t + (int64_t)h * p.out_stride_h; };
    if (p.out_16b) {
      // whole rows at a time, through the wave's part of the rings
      if constexpr (KS == 1) barrier_lds();  // every wave is done with them
      MLA_LDS char* mine = (MLA_LDS char*)smem + wave * 32 * kRowB;
      constexpr int kCh = D / 8;
#pragma unroll
      for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          *reinterpret_cast<MLA_LDS u32x2*>(mine + c32 * kRowB + ((4 * db + i4) ^ (c32 % kCh)) * 16 + 8 * g32) = packed(db, i4);
#pragma unroll
      for (int i = 0; i < 32 * kCh / 64; ++i) {
        const int r = i * (64 / kCh) + lane / kCh, c = lane % kCh;
        const u32x4 v = *reinterpret_cast<const MLA_LDS u32x4*>(mine + r * kRowB + (c ^ (r % kCh)) * 16);
        const int t = tok_of(r);
        if (t < E) *reinterpret_cast<u32x4*>(out_row(t, head_of(r, t)) + 8 * c) = v;
      }
    } else if (live) {
#pragma unroll
      for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) *reinterpret_cast<u32x2*>(out_row(tok, head) + 32 * db + 8 * i4 + 4 * g32) = packed(db, i4);
    }
  }
  // finite sums times 0 are 0
  float zero = 0.f;
#pragma unroll
  for (int db = 0; db < kDb; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) zero = fmaf(O[db][i], 0.f, zero);
  uint64_t bad = __ballot(live && zero != 0.f && l < INFINITY);
  if (__builtin_expect(bad != 0, 0)) {
    gqa_rows_again<D>(p, it, row0, (bad | bad >> 32) & 0xffffffff, k0_all, k1_all, (int64_t)it.slot * kRows + 32 * wave);
  }
}

template <int D, int NW>
void launch_rows(const GqaParams& p, unsigned grid, hipStream_t stream) {
  if (p.page_table != nullptr) hipLaunchKernelGGL((gqa_rows_kernel<D, NW, 1, true>), dim3(grid), dim3(64 * NW), 0, stream, p);
  else hipLaunchKernelGGL((gqa_rows_kernel<D, NW, 1, false>), dim3(grid), dim3(64 * NW), 0, stream, p);
}

}  // namespace

hipError_t launch_gqa_merge(const GqaParams& p, int dim, int rows, hipStream_t stream);

hipError_t launch_gqa_rows(const GqaParams& p, int dim, int rows, hipStream_t stream) {
  // the workspace holds pieces of 128 rows
  if (rows == 256 && (p.target > 0 || dim != 128)) return hipErrorInvalidValue;
  if (p.wide && (rows == 256 || p.page_table != nullptr)) return hipErrorInvalidValue;
  const int64_t grid = gqa_ctas(p, rows);
  if (p.wide) {
    if (dim == 128) hipLaunchKernelGGL((gqa_rows_kernel<128, 4, 2, false>), dim3((unsigned)grid), dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((gqa_rows_kernel<64, 4, 2, false>), dim3((unsigned)grid), dim3(512), 0, stream, p);
  } else if (rows == 256) launch_rows<128, 8>(p, (unsigned)grid, stream);
  else if (dim == 128) launch_rows<128, 4>(p, (unsigned)grid, stream);
  else launch_rows<64, 4>(p, (unsigned)grid, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.target > 0) e = launch_gqa_merge(p, dim, rows, stream);
  return e;
}

}  // namespace mla
