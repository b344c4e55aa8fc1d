// Grouped-head attention for many rows: whole prompts, and chunks of more than 64 rows (tokens times group) over a
// paged cache. See mla_gqa.h for the mathematics.
//
// One CTA per (request, 128 rows, KV head, piece of the keys), four waves x 32 rows. Stages of 32 keys go through LDS;
// S^T[32 keys x 32 rows] = K . Q^T and O^T[D dims x 32 rows] += V^T . P^T on 32x32x16 bf16 MFMA, queries and O in
// registers, online softmax in the log2 domain.
#include "mla_gqa.h"

namespace mla {
namespace {

typedef float f32x16_t __attribute__((__vector_size__(64)));

constexpr int kRows = 128;
constexpr int kStage = 32;
constexpr float kLowest = -3.4028234663852886e38f;

// 16-byte chunk c of token t in a K / V row of an LDS tile
template <int D>
__device__ __forceinline__ int kchunk(int c, int t) {
  const int hi = ((t >> 3) ^ (t >> 4)) & 1;
  return D == 128 ? c ^ ((t & 7) | (hi << 3)) : c ^ (((t >> 1) & 3) | (hi << 2));
}
template <int D>
__device__ __forceinline__ int vchunk(int c, int t) {
  return D == 128 ? c ^ (4 * (t & 3)) : c ^ (4 * ((t >> 1) & 1));
}

template <int D>
__global__ __launch_bounds__(256, 2) void gqa_rows_kernel(const GqaParams p) {
  constexpr int kRowB = D * 2, kChunks = D / 8, kKs = D / 16, kDb = D / 32;
  __shared__ __attribute__((aligned(16))) char s_k[kStage * kRowB];
  __shared__ __attribute__((aligned(16))) char s_v[kStage * kRowB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  GqaItem it;
  if (!gqa_find<kRows>(p, blockIdx.x, it)) return;
  const int C = it.C;
  const int E = it.r.E, L = it.r.L, P = it.r.P, G = p.group;
  const int c32 = lane & 31, g32 = lane >> 5;
  const int r = it.block * kRows + 32 * wave + c32;  // this lane's row
  const int tok = r / G, head = it.head * G + r % G;
  const bool live = tok < E;
  const int limit = live ? P + tok : -1;  // last key
  const int last_tok = min(E - 1, (it.block * kRows + kRows - 1) / G);
  const int k0 = it.piece * C, k1 = min(it.pieces > 1 ? k0 + C : L, P + last_tok + 1);

  bf16x8 qf[kKs];
  {
    const __bf16* q = p.q + (int64_t)(it.r.q0 + (live ? tok : 0)) * p.q_stride_t + (int64_t)(live ? head : it.head * G) * p.q_stride_h;
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(q + 16 * ks + 8 * g32);
  }
  f32x16_t O[kDb];
#pragma unroll
  for (int db = 0; db < kDb; ++db) O[db] = f32x16_t{};
  float m = kLowest, l = 0.f;
  const __bf16* kh = p.k + (int64_t)it.head * p.k_head_stride;
  const __bf16* vh = p.v + (int64_t)it.head * p.v_head_stride;
  const int gq = lane >> 4, a16 = lane & 15;

  for (int t0 = k0; t0 < k1; t0 += kStage) {
    __syncthreads();
    for (int i = threadIdx.x; i < kStage * kChunks; i += 256) {
      const int t = i / kChunks, c = i % kChunks;
      const int row = gqa_row(p, it.b, it.r.q0, min(t0 + t, L - 1));  // keys past the last repeat it
      *reinterpret_cast<u32x4*>(s_k + t * kRowB + kchunk<D>(c, t) * 16) = *reinterpret_cast<const u32x4*>(kh + (int64_t)row * p.k_row_stride + c * 8);
      *reinterpret_cast<u32x4*>(s_v + t * kRowB + vchunk<D>(c, t) * 16) = *reinterpret_cast<const u32x4*>(vh + (int64_t)row * p.v_row_stride + c * 8);
    }
    __syncthreads();
    f32x16_t s = f32x16_t{};
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) {
      const bf16x8 a = *reinterpret_cast<const bf16x8*>(s_k + c32 * kRowB + kchunk<D>(2 * ks + g32, c32) * 16);
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[ks], s, 0, 0, 0);
    }
    const int lim = min(limit, k1 - 1) - t0 - 4 * g32;  // score i is of key t0 + 8 (i / 4) + 4 g32 + i % 4
    float top = kLowest;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = 8 * (i >> 2) + (i & 3) > lim ? -INFINITY : s[i] * p.scale_log2;
      top = fmaxf(top, s[i]);
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m_new = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    l *= f;
#pragma unroll
    for (int db = 0; db < kDb; ++db) O[db] *= f;
    u32x4 pb[2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float e0 = __builtin_amdgcn_exp2f(s[2 * k] - m), e1 = __builtin_amdgcn_exp2f(s[2 * k + 1] - m);
      l += e0 + e1;
      pb[k >> 2][k & 3] = pack_bf16x2(e0, e1);
    }
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int ksp = 0; ksp < 2; ++ksp) {
        // keys 16 ksp + 8 e + 4 g32 + 0..3 (e = 0, 1) of dims 32 db + ..., as the numerators lie
        const int t = 16 * ksp + 4 * (gq >> 1) + (a16 >> 2), c = 4 * db + 2 * (gq & 1) + ((a16 & 3) >> 1);
        auto at = [&](int tt) { return (MLA_LDS bf16x4*)(s_v + tt * kRowB + vchunk<D>(c, tt) * 16 + (a16 & 1) * 8); };
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at(t));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at(t + 8));
        const bf16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        O[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, pb[ksp]), O[db], 0, 0, 0);
      }
  }
  l += __shfl_xor(l, 32);
  if (!live) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const float lse2 = l > 0.f || l != l ? m + log2f(l) : -INFINITY;
  if (it.slot >= 0) {
    const int64_t row = (int64_t)it.slot * kRows + 32 * wave + c32;
    float* o = p.ws_o + row * D;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = O[db][4 * i4 + i] * inv;
        *reinterpret_cast<f32x4*>(o + 32 * db + 8 * i4 + 4 * g32) = v;
      }
    if (g32 == 0) p.ws_lse[row] = lse2;
    return;
  }
  __bf16* o = p.out + (int64_t)(it.r.q0 + tok) * p.out_stride_t + (int64_t)head * p.out_stride_h;
#pragma unroll
  for (int db = 0; db < kDb; ++db)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      u32x2 v;
      v[0] = pack_bf16x2(O[db][4 * i4] * inv, O[db][4 * i4 + 1] * inv);
      v[1] = pack_bf16x2(O[db][4 * i4 + 2] * inv, O[db][4 * i4 + 3] * inv);
      *reinterpret_cast<u32x2*>(o + 32 * db + 8 * i4 + 4 * g32) = v;
    }
  if (p.lse != nullptr && g32 == 0)
    p.lse[(int64_t)(it.r.q0 + tok) * p.lse_stride_t + head] = lse2 * 0.69314718055994531f;
}

}  // namespace

hipError_t launch_gqa_merge(const GqaParams& p, int dim, int rows, hipStream_t stream);

hipError_t launch_gqa_rows(const GqaParams& p, int dim, hipStream_t stream) {
  // sum over requests of ceil(E group / rows), then of ceil(L / C) pieces each
  const int64_t blocks = ((int64_t)p.total_q * p.group + kRows - 1) / kRows + p.batch;
  const int64_t grid = blocks * p.kv_heads + p.target;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  if (dim == 128) hipLaunchKernelGGL(gqa_rows_kernel<128>, dim3((unsigned)grid), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(gqa_rows_kernel<64>, dim3((unsigned)grid), dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.target > 0) e = launch_gqa_merge(p, dim, kRows, stream);
  return e;
}

}  // namespace mla
