// Grouped-head attention for few rows: single tokens and chunks of up to 64 rows (tokens times group) over a paged
// cache, with the keys of a batch split over the chip and joined by an fp32 log-sum-exp merge. See mla_gqa.h.
//
// One CTA per (request, rows, KV head, piece of the keys). Its four waves take tiles of 32 keys in turn and share
// nothing until the end, so there is no barrier in the stream: a wave loads a tile's K straight into the operand layout
// of the score MFMA and its V through a private LDS tile that transposes it, and requests the next tile before it
// computes the present one. Bound: HBM (each K and V row is read once).
#include "mla_gqa.h"

namespace mla {
namespace {

constexpr int kTileKeys = 32;
constexpr float kLowest = -3.4028234663852886e38f;

// NB blocks of 16 rows
template <int D, int NB>
__global__ __launch_bounds__(256, 2) void gqa_stream_kernel(const GqaParams p) {
  constexpr int kRows = 16 * NB, kRowB = D * 2, kChunks = D / 8, kKs = D / 32, kDb = D / 16;
  constexpr int kVLoads = kTileKeys * kChunks / 64;  // 16-byte loads of a lane per V tile
  __shared__ __attribute__((aligned(16))) char s_v[4][kTileKeys * kRowB];
  __shared__ float s_m[4][16], s_l[4][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int C = gqa_split_keys<kRows>(p);
  GqaItem it;
  if (!gqa_find<kRows>(p, C, blockIdx.x, it)) return;
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
  const __bf16* kh = p.k + (int64_t)it.head * p.k_head_stride;
  const __bf16* vh = p.v + (int64_t)it.head * p.v_head_stride;

  f32x4 O[NB][kDb];
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = kLowest;
    l[nb] = 0.f;
#pragma unroll
    for (int db = 0; db < kDb; ++db) O[nb][db] = f32x4{};
  }
  u32x4 kr[2][kKs], vr[kVLoads];
  auto load = [&](int t0) __attribute__((always_inline)) {
    // token t < 32 of the tile: its row is in lane t (keys past the last repeat it)
    const int64_t row = gqa_row(p, it.b, it.r.q0, min(t0 + (lane & 31), L - 1));
    const int lo = (int)row, hi = (int)(row >> 32);
    auto row_of = [&](int t) { return (int64_t)(uint32_t)__shfl(lo, t) | (int64_t)__shfl(hi, t) << 32; };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __bf16* src = kh + row_of(16 * h + a16) * p.k_row_stride + 8 * g;
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) kr[h][ks] = *reinterpret_cast<const u32x4*>(src + 32 * ks);
    }
#pragma unroll
    for (int u = 0; u < kVLoads; ++u) {
      const int i = u * 64 + lane;
      vr[u] = *reinterpret_cast<const u32x4*>(vh + row_of(i / kChunks) * p.v_row_stride + i % kChunks * 8);
    }
  };
  // V chunk c (16 bytes) of token t: pairs of chunks permuted, so that the 8 tokens of a transposing read differ
  auto vpos = [&](int t, int c) { return t * kRowB + (D == 128 ? c ^ (2 * (t & 7)) : c ^ (2 * ((t >> 1) & 3))) * 16; };

  int t0 = k0 + kTileKeys * wave;
  if (t0 < k1) load(t0);
  for (; t0 < k1; t0 += 4 * kTileKeys) {
    bf16x8 kc[2][kKs];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) kc[h][ks] = __builtin_bit_cast(bf16x8, kr[h][ks]);
#pragma unroll
    for (int u = 0; u < kVLoads; ++u) {
      const int i = u * 64 + lane;
      *reinterpret_cast<u32x4*>(s_v[wave] + vpos(i / kChunks, i % kChunks)) = vr[u];
    }
    if (t0 + 4 * kTileKeys < k1) load(t0 + 4 * kTileKeys);
    u32x4 pb[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{};
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kc[h][ks], qf[nb][ks], s[h], 0, 0, 0);
      }
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
      auto at = [&](int tt) { return (MLA_LDS bf16x4*)(s_v[wave] + vpos(tt, c) + (a16 & 1) * 8); };
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
    // thread: row threadIdx / 16, dims in steps of 64 from 4 (threadIdx % 16)
    const int row = threadIdx.x >> 4, x = threadIdx.x & 15;
    float mt = s_m[0][row];
#pragma unroll
    for (int w = 1; w < 4; ++w) mt = fmaxf(mt, s_m[w][row]);
    float f[4], lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = __builtin_amdgcn_exp2f(s_m[w][row] - mt);
      lt += f[w] * s_l[w][row];
    }
    const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
    const float lse2 = lt > 0.f || lt != lt ? mt + log2f(lt) : -INFINITY;
    const int r = it.block * kRows + 16 * nb + row, tok = r / G, head = it.head * G + r % G;
    if (tok >= E) continue;
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
      const int c = 16 * d + x;
      f32x4 o = f32x4{};
#pragma unroll
      for (int w = 0; w < 4; ++w) o += *reinterpret_cast<const f32x4*>(s_v[w] + row * (D * 4) + ((c + row) % (D / 4)) * 16) * f[w];
      o *= inv;
      if (it.slot >= 0) {
        *reinterpret_cast<f32x4*>(p.ws_o + ((int64_t)it.slot * kRows + 16 * nb + row) * D + 4 * c) = o;
      } else {
        u32x2 v{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
        *reinterpret_cast<u32x2*>(p.out + (int64_t)(it.r.q0 + tok) * p.out_stride_t + (int64_t)head * p.out_stride_h + 4 * c) = v;
      }
    }
    if (x == 0) {
      if (it.slot >= 0) p.ws_lse[(int64_t)it.slot * kRows + 16 * nb + row] = lse2;
      else if (p.lse != nullptr) p.lse[(int64_t)(it.r.q0 + tok) * p.lse_stride_t + head] = lse2 * 0.69314718055994531f;
    }
  }
}

// Partial results of split requests joined: one wave per 16 rows... of (request, block, head), a row at a time:
//   lse = log2 sum_i 2^lse_i, out = sum_i 2^(lse_i - lse) o_i.
// A CTA takes (block of kRows rows, head) number blockIdx.x of the batch, counted as the attention kernels count their
// items with every request in one piece.
template <int D, int kRows>
__global__ __launch_bounds__(256) void gqa_merge_kernel(const GqaParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int C = gqa_split_keys<kRows>(p);
  // the request of this (block, head), and the slots before it
  int acc = 0, slots = 0, b = -1, local = 0, pieces = 1;
  GqaRequest r{0, 0, 0, 0};
  for (int c0 = 0; c0 < p.batch && b < 0; c0 += 64) {
    const int i = c0 + lane;
    GqaRequest ri{0, 0, 0, 0};
    int n = 0, ns = 0, pi = 1;
    if (i < p.batch) {
      ri = gqa_request(p, i);
      pi = ri.L > C ? (ri.L + C - 1) / C : 1;
      n = (ri.E * p.group + kRows - 1) / kRows * p.kv_heads;
      ns = pi > 1 ? n * pi : 0;
    }
    int incl = n, sincl = ns;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o), w = __shfl_up(sincl, o);
      if (lane >= o) {
        incl += u;
        sincl += w;
      }
    }
    const int item = blockIdx.x;
    const uint64_t hit = __ballot(item >= acc + incl - n && item < acc + incl);
    if (hit != 0) {
      const int fl = __builtin_ctzll(hit);
      b = c0 + fl;
      local = item - acc - __builtin_amdgcn_readlane(incl - n, fl);
      slots += __builtin_amdgcn_readlane(sincl - ns, fl);
      pieces = __builtin_amdgcn_readlane(pi, fl);
      r.q0 = __builtin_amdgcn_readlane(ri.q0, fl);
      r.E = __builtin_amdgcn_readlane(ri.E, fl);
      r.L = __builtin_amdgcn_readlane(ri.L, fl);
    } else {
      acc += __shfl(incl, 63);
      slots += __shfl(sincl, 63);
    }
  }
  if (b < 0 || pieces == 1) return;
  const int head = local % p.kv_heads, block = local / p.kv_heads;
  const int64_t slot0 = slots + (int64_t)block * pieces * p.kv_heads + head;  // piece i: + i kv_heads
  for (int row = wave; row < kRows; row += 4) {
    const int rr = block * kRows + row, tok = rr / p.group, h = head * p.group + rr % p.group;
    if (tok >= r.E) break;
    float mt = kLowest;
    for (int i = lane; i < pieces; i += 64) mt = fmaxf(mt, p.ws_lse[(slot0 + (int64_t)i * p.kv_heads) * kRows + row]);
    mt = wave_max64(mt);
    float lt = 0.f, o[D / 64] = {};
    for (int i = 0; i < pieces; ++i) {
      const int64_t at = (slot0 + (int64_t)i * p.kv_heads) * kRows + row;
      const float f = __builtin_amdgcn_exp2f(p.ws_lse[at] - mt);
      lt += f;
#pragma unroll
      for (int d = 0; d < D / 64; ++d) o[d] += f * p.ws_o[at * D + (D / 64) * lane + d];
    }
    const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
    __bf16* out = p.out + (int64_t)(r.q0 + tok) * p.out_stride_t + (int64_t)h * p.out_stride_h + (D / 64) * lane;
    if constexpr (D == 128) *reinterpret_cast<uint32_t*>(out) = pack_bf16x2(o[0] * inv, o[1] * inv);
    else *out = (__bf16)(o[0] * inv);
    if (lane == 0 && p.lse != nullptr)
      p.lse[(int64_t)(r.q0 + tok) * p.lse_stride_t + h] = lt > 0.f || lt != lt ? (mt + log2f(lt)) * 0.69314718055994531f : -INFINITY;
  }
}

template <int D, int NB>
void launch_stream(const GqaParams& p, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((gqa_stream_kernel<D, NB>), dim3((unsigned)grid), dim3(256), 0, stream, p);
}

}  // namespace

hipError_t launch_gqa_merge(const GqaParams& p, int dim, int rows, hipStream_t stream) {
  const int64_t blocks = ((int64_t)p.total_q * p.group + rows - 1) / rows + p.batch;
  const dim3 grid((unsigned)(blocks * p.kv_heads)), cta(256);
#define MLA_MERGE(D, R) \
  if (dim == D && rows == R) hipLaunchKernelGGL((gqa_merge_kernel<D, R>), grid, cta, 0, stream, p)
  MLA_MERGE(64, 16);
  MLA_MERGE(64, 32);
  MLA_MERGE(64, 64);
  MLA_MERGE(64, 128);
  MLA_MERGE(128, 16);
  MLA_MERGE(128, 32);
  MLA_MERGE(128, 64);
  MLA_MERGE(128, 128);
#undef MLA_MERGE
  return hipGetLastError();
}

hipError_t launch_gqa_stream(const GqaParams& p, int dim, hipStream_t stream) {
  const int64_t most = (int64_t)p.max_q * p.group;
  const int rows = most <= 16 ? 16 : most <= 32 ? 32 : 64;
  const int64_t blocks = ((int64_t)p.total_q * p.group + rows - 1) / rows + p.batch;
  const int64_t grid = blocks * p.kv_heads + p.target;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  if (dim == 128) rows == 16 ? launch_stream<128, 1>(p, grid, stream) : rows == 32 ? launch_stream<128, 2>(p, grid, stream) : launch_stream<128, 4>(p, grid, stream);
  else rows == 16 ? launch_stream<64, 1>(p, grid, stream) : rows == 32 ? launch_stream<64, 2>(p, grid, stream) : launch_stream<64, 4>(p, grid, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.target > 0) e = launch_gqa_merge(p, dim, rows, stream);
  return e;
}

}  // namespace mla
