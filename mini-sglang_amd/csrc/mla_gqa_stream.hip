// Grouped-head attention for few rows (tokens times group): single tokens, chunks of up to 32 rows over a paged cache, with
// the keys of a batch split over the chip and joined by an fp32 log-sum-exp merge, and chunks and prompts of which few
// CTAs come. See mla_gqa.h.
//
// One CTA per (request, rows, KV head, piece of the keys). Its NW waves take tiles of 32 keys in turn and share
// nothing until the end, so there is no barrier in the stream: a wave brings a tile's K and V into the MFMAs' operand
// layouts through private LDS tiles, and requests the next tile before it computes the present one.
// Bound: HBM (each K and V row is read once), and below some 20 MB the chain of dependent loads (lengths, page, tile) and
// the merge's launch. Measured with the merge: 64 requests of 1k to 8k tokens, 64 and 8 heads of 128, 223 us (5.8 TB/s);
// 8 of 32k to 128k, 8 heads and 1, 60 us (5.4 TB/s); 16 chunks of 1 to 8 on 1k to 16k, 32 and 8 heads, pages of one
// token, 112 us (5.1 TB/s); one request of 1500, 32 and 8 heads, 9.6 us; in one piece, eight waves: three chunks of 5 to
// 60 on up to 500, 28 and 4 heads, 8.2 us; seven prompts of 1 to 300, 8 and 2 heads of 64, four waves, 6.4 us.
#include <type_traits>

#include "mla_gqa.h"

namespace mla {
namespace {

constexpr int kTileKeys = 32;
constexpr float kLowest = -3.4028234663852886e38f;

// NB blocks of 16 rows, NW waves
template <int D, int NB, int NW>
__global__ __launch_bounds__(64 * NW, 2) void gqa_stream_kernel(const GqaParams p) {
  constexpr int kRows = 16 * NB, kRowB = D * 2, kChunks = D / 8, kKs = D / 32, kDb = D / 16;
  constexpr int kLoads = kTileKeys * kChunks / 64;  // 16-byte loads of a lane per K or V tile
  __shared__ __attribute__((aligned(16))) char s_k[NW][kTileKeys * kRowB], s_v[NW][kTileKeys * kRowB];
  __shared__ float s_m[NW][16], s_l[NW][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  GqaItem it;
  if (!gqa_find<kRows, false>(p, blockIdx.x, it)) return;
  const int C = it.C;
  const int E = it.r.E, L = it.r.L, P = it.r.P, G = p.group;
  const int a16 = lane & 15, g = lane >> 4;
  int limit[NB];
  bf16x8 qf[NB][kKs];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = it.block * kRows + 16 * nb + a16, tok = r / G;
    const bool live = tok < E;
    limit[nb] = live ? P + tok : -1;
    const __bf16* q = p.q + (int64_t)(it.r.q0 + (live ? tok : 0)) * p.q_stride_t + (int64_t)(it.head * G + (live ? r % G : 0)) * p.q_stride_h;
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) qf[nb][ks] = *reinterpret_cast<const bf16x8*>(q + 32 * ks + 8 * g);
  }
  const int last_tok = min(E - 1, (it.block * kRows + kRows - 1) / G);
  const int first_limit = P + it.block * kRows / G;  // of the item's first row: no key up to it is masked
  const int k0 = it.piece * C, k1 = min(it.pieces > 1 ? k0 + C : L, P + last_tok + 1);
  // of the lane's 16-byte chunk; row strides in bytes, below 2^32 by the host. As 32 bits an address is one multiply-add,
  // which eight waves on their own gain by (a prompt of 8000, one head 76 -> 70 us; chunks of 64 on 900 13.8 -> 13.2); streams
  // at HBM's rate lose (16 chunks of 1 to 8 on 1k to 16k 107 -> 109, decode of 32k to 128k 59.4 -> 60.3).
  using stride_t = std::conditional_t<NW == 8, uint32_t, int64_t>;
  const char* kh = reinterpret_cast<const char*>(p.k + (int64_t)it.head * p.k_head_stride + lane % kChunks * 8);
  const char* vh = reinterpret_cast<const char*>(p.v + (int64_t)it.head * p.v_head_stride + lane % kChunks * 8);
  const stride_t ks_b = (stride_t)(p.k_row_stride * 2), vs_b = (stride_t)(p.v_row_stride * 2);

  f32x4 O[NB][kDb];
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = kLowest;
    l[nb] = 0.f;
#pragma unroll
    for (int db = 0; db < kDb; ++db) O[nb][db] = f32x4{};
  }
  // A tile is loaded row by row, 16 lanes (D 64: 8) to a row, and goes through the wave's own LDS tiles into the operand
  // layouts: with loads straight into the K operand's (a 16-byte chunk of 16 rows each), 64 requests of 1k to 8k tokens, 8
  // KV heads, took 263 us where this takes 231. Non-temporal, since a row is read once (257 us without). Two tiles in
  // flight a wave gained nothing (229 us / 235; four chunks of 64 on 900 keys 15.5 / 16.6). row: of token t < 32 of the tile
  // in lane t.
  u32x4 kr[kLoads], vr[kLoads];
  auto rows = [&](int t0) __attribute__((always_inline)) { return gqa_row(p, it.b, it.r.q0, min(t0 + (lane & 31), L - 1)); };
  auto load = [&](int row) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const std::conditional_t<NW == 8, uint64_t, int64_t> rw = (stride_t)__shfl(row, (u * 64 + lane) / kChunks);
      kr[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kh + rw * ks_b));
      vr[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vh + rw * vs_b));
    }
  };
  // 16-byte chunk c of token t: pairs of chunks permuted, so that neither the K reads (16 rows' chunks c and c + 1) nor
  // the transposing V reads (8 rows' chunk pairs) meet in a bank
  auto pos = [&](int t, int c) __attribute__((always_inline)) { return t * kRowB + (D == 128 ? c ^ (2 * (t & 7)) : c ^ (2 * ((t >> 1) & 3))) * 16; };

  constexpr int kStep = NW * kTileKeys;
  int t0 = k0 + kTileKeys * wave, row_next = 0;
  if (t0 < k1) {
    const int row = rows(t0);
    row_next = rows(t0 + kStep);
    load(row);
  }
  for (; t0 < k1; t0 += kStep) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int at = pos((u * 64 + lane) / kChunks, lane % kChunks);
      *reinterpret_cast<u32x4*>(s_k[wave] + at) = kr[u];
      *reinterpret_cast<u32x4*>(s_v[wave] + at) = vr[u];
    }
    if (t0 + kStep < k1) load(row_next);
    if (t0 + 2 * kStep < k1) row_next = rows(t0 + 2 * kStep);
    f32x4 sc[NB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 kc[kKs];
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) kc[ks] = *reinterpret_cast<const bf16x8*>(s_k[wave] + pos(16 * h + a16, 4 * ks + g));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        sc[nb][h] = f32x4{};
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) sc[nb][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kc[ks], qf[nb][ks], sc[nb][h], 0, 0, 0);
      }
    }
    u32x4 pb[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      // the scaled scores are rounded before their maximum is taken from them: the largest numerator is 1 at any size
#pragma clang fp contract(off)
      f32x4(&s)[2] = sc[nb];
      // score (h, i) of a lane: row a16, key t0 + 16 h + 4 g + i
      float top = kLowest;
      const bool masked = t0 + kTileKeys - 1 > first_limit || t0 + kTileKeys > k1;
      const int lim = min(limit[nb], k1 - 1) - t0 - 4 * g;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[h][i] *= p.scale_log2;
          if (masked && 16 * h + i > lim) s[h][i] = -INFINITY;
          top = fmaxf(top, s[h][i]);
        }
      top = wave_max_g(top);
      if (__ballot(top > m[nb]) != 0) {
        const float m_new = fmaxf(m[nb], top), f = __builtin_amdgcn_exp2f(m[nb] - m_new);
        m[nb] = m_new;
        l[nb] *= f;
#pragma unroll
        for (int db = 0; db < kDb; ++db) O[nb][db] *= f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(s[h][i] - m[nb]);
          l[nb] += e[i];
        }
        pb[nb][2 * h] = pack_bf16x2(e[0], e[1]);
        pb[nb][2 * h + 1] = pack_bf16x2(e[2], e[3]);
      }
    }
#pragma unroll
    for (int db = 0; db < kDb; ++db) {
      // tokens 4 g + 0..3 and 16 + 4 g + 0..3 of dim 16 db + a16, as the numerators lie
      const int t = 4 * g + (a16 >> 2), c = 2 * db + ((a16 & 3) >> 1);
      auto at = [&](int tt) { return (MLA_LDS bf16x4*)(s_v[wave] + pos(tt, c) + (a16 & 1) * 8); };
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at(t));
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at(t + 16));
      const bf16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, pb[nb]), O[nb][db], 0, 0, 0);
    }
  }

  // ---- the waves' results joined, one block of 16 rows at a time: a wave's O in its own V tile, fp32 [16 rows][D]
  static_assert(16 * D * 4 <= kTileKeys * kRowB, "a block's O fits the wave's V tile");
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float lw = wave_sum_g(l[nb]);
    if (nb > 0) __syncthreads();
    // lane: row a16, dims 16 db + 4 g + 0..3, 16-byte chunks rotated by the row
#pragma unroll
    for (int db = 0; db < kDb; ++db)
      *reinterpret_cast<f32x4*>(s_v[wave] + a16 * (D * 4) + ((4 * db + g + a16) % (D / 4)) * 16) = O[nb][db];
    if (g == 0) {
      s_m[wave][a16] = m[nb];
      s_l[wave][a16] = lw;
    }
    __syncthreads();
    // kTpr threads a row, 4 dims each at a time
    constexpr int kTpr = 4 * NW;
    const int row = threadIdx.x / kTpr, x = threadIdx.x % kTpr;
    float mt = s_m[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) mt = fmaxf(mt, s_m[w][row]);
    float f[NW], lt = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = __builtin_amdgcn_exp2f(s_m[w][row] - mt);
      lt += f[w] * s_l[w][row];
    }
    const bool some = lt > 0.f || lt != lt;
    const float inv = some ? 1.f / lt : 0.f;
    const f32x2 lse2 = gqa_lse(some, mt, log2f(lt));
    const int r = it.block * kRows + 16 * nb + row, tok = r / G, head = it.head * G + r % G;
    float zero = 0.f;
#pragma unroll
    for (int c = tok < E ? x : D; c < D / 4; c += kTpr) {
      f32x4 o = f32x4{};
#pragma unroll
      for (int w = 0; w < NW; ++w) o += *reinterpret_cast<const f32x4*>(s_v[w] + row * (D * 4) + ((c + row) % (D / 4)) * 16) * f[w];
#pragma unroll
      for (int i = 0; i < 4; ++i) zero = fmaf(o[i], 0.f, zero);
      o *= inv;
      if (it.slot >= 0) {
        *reinterpret_cast<f32x4*>(p.ws_o + ((int64_t)it.slot * kRows + 16 * nb + row) * D + 4 * c) = o;
      } else {
        u32x2 v{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
        *reinterpret_cast<u32x2*>(p.out + (int64_t)(it.r.q0 + tok) * p.out_stride_t + (int64_t)head * p.out_stride_h + 4 * c) = v;
      }
    }
    if (x == 0 && tok < E) {
      if (it.slot >= 0) p.ws_lse[(int64_t)it.slot * kRows + 16 * nb + row] = lse2;
      else if (p.lse != nullptr) p.lse[(int64_t)(it.r.q0 + tok) * p.lse_stride_t + head] = lse2[0] * 0.69314718055994531f;
    }
    uint64_t bad = __ballot(zero != 0.f && lt < INFINITY);  // finite sums times 0 are 0
    if (__builtin_expect(bad != 0, 0)) {
      constexpr int kWr = 64 / kTpr;  // rows of a wave
      uint64_t rows = 0;
#pragma unroll
      for (int i = 0; i < kWr; ++i)
        if ((bad >> (i * kTpr) & ((1ull << kTpr) - 1)) != 0) rows |= 1ull << i;
      const int r0 = 16 * nb + kWr * wave;
      gqa_rows_again<D>(p, it, it.block * kRows + r0, rows, k0, k1, (int64_t)it.slot * kRows + r0);
    }
  }
}

// Partial results of requests in pieces, joined: lse = log2 sum_i 2^lse_i, out = sum_i 2^(lse_i - lse) o_i, with lse_i of two
// floats each (gqa_lse).
// One CTA per (query, query head): its waves take every fourth piece (kWaves 4), or a wave per row (kWaves 1). Weights are
// times 2^-12: up to 2^12 pieces of the largest values sum up within fp32's range. (Exact but for products below its normal
// range: results of 2^-126 are as far off as larger ones, measured over 131,072 keys.)
// Bound: dependent loads (lengths, the pieces' lse, their rows). 4.3 us for 32 rows, 7 for 4096 rows of 64 requests.
template <int D, int kRows, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void gqa_merge_kernel(const GqaParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = p.kv_heads * p.group, t = blockIdx.x / heads, h = blockIdx.x % heads;
  GqaRequest r{0, 0, 0, 0};
  if (lane < p.batch) r = gqa_request(p, lane);
  const int C = gqa_piece_keys<kRows>(p, r);
  int slots = 0, tok = -1, pieces = 1;
  for (int c0 = 0; c0 < p.batch && tok < 0; c0 += 64) {
    if (c0 > 0) {
      r = GqaRequest{0, 0, 0, 0};
      if (c0 + lane < p.batch) r = gqa_request(p, c0 + lane);
    }
    const int pi = gqa_pieces(r.L, C);
    const int ns = pi > 1 ? gqa_blocks<kRows>(p, r) * pi * p.kv_heads : 0, sincl = wave_iscan(ns);
    const uint64_t hit = __ballot(t >= r.q0 && t < r.q0 + r.E);
    if (hit != 0) {
      const int fl = __builtin_ctzll(hit);
      tok = t - __builtin_amdgcn_readlane(r.q0, fl);
      pieces = __builtin_amdgcn_readlane(pi, fl);
      slots += __builtin_amdgcn_readlane(sincl - ns, fl);
    } else {
      slots += __builtin_amdgcn_readlane(sincl, 63);
    }
  }
  if (tok < 0 || pieces == 1) return;
  const int rr = tok * p.group + h % p.group, row = rr % kRows;
  // piece i of the row's block and head: slot0 + i kv_heads
  const int64_t slot0 = slots + (int64_t)(rr / kRows) * pieces * p.kv_heads + h / p.group;
  const f32x2* lse = p.ws_lse + slot0 * kRows + row;
  const float* part = p.ws_o + (slot0 * kRows + row) * D + (D / 64) * lane;
  const int64_t ls = (int64_t)p.kv_heads * kRows, os = ls * D;
  typedef float part_t __attribute__((ext_vector_type(D / 64)));
  // parts wave, wave + kWaves, ... eight in flight; the first eight are requested before the LSEs are waited for
  part_t x[8];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const part_t*>(part + min(i + u * kWaves, pieces - 1) * os);
  };
  load(wave);
  f32x2 own{-INFINITY, 0.f};  // of piece `lane`
  if (lane < pieces) own = lse[lane * ls];
  float mt = fmaxf(own[0], kLowest);
  for (int i = 64 + lane; i < pieces; i += 64) mt = fmaxf(mt, lse[i * ls][0]);
  mt = wave_max64(mt);
  // of the largest LSEs that are alike in fp32 the largest rest; below 2^24 at most half a bit, and left in the weights
  float rest = 0.f;
  if (__ballot(fabsf(mt) >= 16777216.f) != 0) {
    rest = own[0] == mt ? own[1] : kLowest;
    for (int i = 64 + lane; i < pieces; i += 64) {
      const f32x2 x = lse[i * ls];
      if (x[0] == mt) rest = fmaxf(rest, x[1]);
    }
    rest = wave_max64(rest);
  }
  float lt = 0.f;
  part_t o = {};
  for (int i0 = 0; i0 < pieces; i0 += 64) {  // 64 pieces at a time: their weights in the lanes
    float f = 0.f;
    if (i0 + lane < pieces) {
      const f32x2 x = i0 == 0 ? own : lse[(i0 + lane) * ls];
      f = __builtin_amdgcn_exp2f((x[0] - mt) + (x[1] - rest)) * 0x1p-12f;
    }
    lt += wave_sum64(f);
    const int n = min(64, pieces - i0);
    for (int i = wave; i < n; i += 8 * kWaves) {
      if (i0 + i > wave) load(i0 + i);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = i + u * kWaves;
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(j, 63)));
        if (j < n) o += x[u] * w;
      }
    }
  }
  if constexpr (kWaves > 1) {
    __shared__ part_t s_o[kWaves][64];
    s_o[wave][lane] = o;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) o += s_o[w][lane];
  }
  const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
  __bf16* out = p.out + (int64_t)t * p.out_stride_t + (int64_t)h * p.out_stride_h + (D / 64) * lane;
  if constexpr (D == 128) *reinterpret_cast<uint32_t*>(out) = pack_bf16x2(o[0] * inv, o[1] * inv);
  else *out = (__bf16)(o[0] * inv);
  if (lane == 0 && p.lse != nullptr)
    p.lse[(int64_t)t * p.lse_stride_t + h] = lt > 0.f || lt != lt ? (mt + (rest + log2f(lt * 0x1p12f))) * 0.69314718055994531f : -INFINITY;
}

template <int D, int NB>
void launch_stream(const GqaParams& p, int64_t grid, hipStream_t stream) {
  if (p.wide) hipLaunchKernelGGL((gqa_stream_kernel<D, NB, 8>), dim3((unsigned)grid), dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((gqa_stream_kernel<D, NB, 4>), dim3((unsigned)grid), dim3(256), 0, stream, p);
}

}  // namespace

hipError_t launch_gqa_merge(const GqaParams& p, int dim, int rows, hipStream_t stream) {
  const int64_t grid = (int64_t)p.total_q * p.kv_heads * p.group;
  // few rows are cut into many pieces
#define MLA_MERGE(D, R)                                                                                            \
  if (dim == D && rows == R) {                                                                                     \
    if (grid <= 2048) hipLaunchKernelGGL((gqa_merge_kernel<D, R, 4>), dim3((unsigned)grid), dim3(256), 0, stream, p); \
    else hipLaunchKernelGGL((gqa_merge_kernel<D, R, 1>), dim3((unsigned)grid), dim3(64), 0, stream, p);             \
  }
  MLA_MERGE(64, 16)
  MLA_MERGE(64, 32)
  MLA_MERGE(64, 128)
  MLA_MERGE(128, 16)
  MLA_MERGE(128, 32)
  MLA_MERGE(128, 128)
#undef MLA_MERGE
  return hipGetLastError();
}

hipError_t launch_gqa_stream(const GqaParams& p, int dim, int rows, hipStream_t stream) {
  const int64_t grid = gqa_ctas(p, rows);
  if (dim == 128) rows == 16 ? launch_stream<128, 1>(p, grid, stream) : launch_stream<128, 2>(p, grid, stream);
  else rows == 16 ? launch_stream<64, 1>(p, grid, stream) : launch_stream<64, 2>(p, grid, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.target > 0) e = launch_gqa_merge(p, dim, rows, stream);
  return e;
}

}  // namespace mla
