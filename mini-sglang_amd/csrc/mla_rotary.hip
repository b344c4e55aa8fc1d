// Queries and keys of models with grouped heads, from a fused projection's output to attention: RMSNorm of each head, the
// rotation by position, and the rows of K and V into a paged cache, in one launch.
//
// Row x of D dims, weight w, angle a_i of pair i:  y = x / sqrt(mean(x^2) + eps) * w, then for the first R dims
//   y_p, y_q -> y_p cos a_i - y_q sin a_i, y_q cos a_i + y_p sin a_i,   (p, q) = (i, i + R/2) or (2 i, 2 i + 1).
// fp32 throughout, rounded to bf16 once, at the store.
//
// A row is D / 8 lanes' (a wave holds 4 rows of 128 or 8 of 64), 8 dims a lane in two chunks of 4 that hold both halves of
// its pairs: no lane needs another's values but for the sum of squares, which is 3 or 4 DPP steps. Rows of one token are
// next to each other in a wave, so they share the angles.
// Bound: HBM for many tokens (8192 of 64 and 8 heads of 128, with V: 340 MB in 63 us, 5.4 TB/s), a launch and two dependent
// loads (position, angles) for few (64 tokens 3.7 us).
#include "mla_common.h"
#include "mla_device.h"

namespace mla {
namespace {

// Sum over the kLanes (8 or 16) lanes of a row; every lane gets it.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
  auto add = [&](auto ctrl) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  add(std::integral_constant<int, 0xb1>{});   // lane ^ 1
  add(std::integral_constant<int, 0x4e>{});   // lane ^ 2
  add(std::integral_constant<int, 0x141>{});  // 7 - lane, of 8
  if constexpr (kLanes == 16) add(std::integral_constant<int, 0x140>{});  // 15 - lane, of 16
  return v;
}

__device__ __forceinline__ void unpack4(const u32x2 w, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// U rows a lane
template <int D, int U>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkNormRopeParams p) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes, kStep = kRows * U;
  const int lane = threadIdx.x & 63, x = lane % kLanes;
  const int heads = p.q_heads + p.kv_heads, rows = heads + (p.v != nullptr ? p.kv_heads : 0);
  const uint32_t groups = (rows + kStep - 1) / kStep;  // waves of a token
  const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= p.tokens * groups) return;
  const int t = (int)(item / groups), r0 = (int)(item % groups) * kStep + lane / kLanes;
  int64_t slot = t;
  if (p.slots != nullptr) slot = p.index_bits == 32 ? ((const int32_t*)p.slots)[t] : ((const int64_t*)p.slots)[t];
  const bool stored = slot >= 0 && slot < p.out_rows;
  // the lane's dims: chunks a and b of 4
  const int R = p.rotary_dim;
  const bool turns = 8 * x < R;
  const int a = turns && !p.interleaved ? 4 * x : 8 * x, b = turns && !p.interleaved ? 4 * x + R / 2 : 8 * x + 4;
  f32x4 c{}, s{};
  if (turns) {
    const float* cs = p.cos_sin + (int64_t)min(max(p.positions[t], 0), p.max_position - 1) * R + 4 * x;
    c = *reinterpret_cast<const f32x4*>(cs);
    s = *reinterpret_cast<const f32x4*>(cs + R / 2);
  }
  u32x2 xa[U] = {}, xb[U] = {};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = r0 + u * kRows;
    if (r >= rows) continue;
    const __bf16* in = r < p.q_heads ? p.q + (int64_t)t * p.q_stride_t + (int64_t)r * p.q_stride_h
                       : r < heads   ? p.k + (int64_t)t * p.k_stride_t + (int64_t)(r - p.q_heads) * p.k_stride_h
                                     : p.v + (int64_t)t * p.v_stride_t + (int64_t)(r - heads) * p.v_stride_h;
    xa[u] = *reinterpret_cast<const u32x2*>(in + a);
    xb[u] = *reinterpret_cast<const u32x2*>(in + b);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = r0 + u * kRows;
    // (rows past the last take part in the sums of their own lanes only)
    float f[8];
    unpack4(xa[u], f);
    unpack4(xb[u], f + 4);
    const __bf16* w = r < p.q_heads ? p.q_weight : p.k_weight;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
    ss = row_sum<kLanes>(ss);
    if (r >= rows) continue;
    if (r < heads) {
      if (w != nullptr) {
        const float mean = ss * (1.f / D) + p.eps;
        float inv = rsqrtf(mean);
        // Squares of 2^64 and more pass fp32's range, those of 2^-63 and less are not exact: the row is taken again, times a power of two.
        // (All lanes of the row have the same sum. Large values stay themselves for the product, as 1 / norm is at least 2^-128.)
        if (__builtin_expect(!(mean >= 0x1p-100f && mean <= 3.4028234663852886e38f), 0)) {
          const bool small = mean < 0x1p-100f;
          const float by = small ? 0x1p86f : 0x1p-80f;
          ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = f[i] * by;
            ss = fmaf(x, x, ss);
            if (small) f[i] = x;
          }
          inv = rsqrtf(row_sum<kLanes>(ss) * (1.f / D) + p.eps * by * by);
          if (!small) inv *= by;
        }
        float g[8];
        unpack4(*reinterpret_cast<const u32x2*>(w + a), g);
        unpack4(*reinterpret_cast<const u32x2*>(w + b), g + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * g[i];  // (at most sqrt(D) times the weight)
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& lo = p.interleaved ? f[2 * i] : f[i];
          float& hi = p.interleaved ? f[2 * i + 1] : f[4 + i];
          const float was = lo;
          lo = was * c[i] - hi * s[i];
          hi = hi * c[i] + was * s[i];
        }
      }
      if (w != nullptr || turns) {
        xa[u] = u32x2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
        xb[u] = u32x2{pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
      }
    }
    if (r >= p.q_heads && !stored) continue;
    __bf16* out = r < p.q_heads ? p.q_out + (int64_t)t * p.qo_stride_t + (int64_t)r * p.qo_stride_h
                  : r < heads   ? p.k_out + slot * p.ko_stride_row + (int64_t)(r - p.q_heads) * p.ko_stride_h
                                : p.v_out + slot * p.vo_stride_row + (int64_t)(r - heads) * p.vo_stride_h;
    if constexpr (U == 1) {
      *reinterpret_cast<u32x2*>(out + a) = xa[u];
      *reinterpret_cast<u32x2*>(out + b) = xb[u];
    } else {
      __builtin_nontemporal_store(xa[u], reinterpret_cast<u32x2*>(out + a));
      __builtin_nontemporal_store(xb[u], reinterpret_cast<u32x2*>(out + b));
    }
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(const QkNormRopeParams& p, int dim, hipStream_t stream) {
  const int rows = p.q_heads + p.kv_heads + (p.v != nullptr ? p.kv_heads : 0);
  // Rows of a lane: one while all waves run at once, more where their loads should be in flight together. us for 1 / 2 / 4, 64
  // and 8 heads of 128 with V: 128 tokens (2560 waves of one row) 3.7 / 4.0 / 4.8; 256 4.5 / 4.4 / 5.1; 2048 20.4 / 16.0 / 16.0;
  // 8192 (163840) 88 / 66.9 / 63.4. Non-temporal stores with more than one: 68.8 and 66.6 without. (Loads stay temporal: a
  // projection's output lies in the caches; 2048 tokens 16.0, 19.9 with non-temporal ones.)
  const int step = 512 / dim;  // rows of a wave
  const int64_t waves = (int64_t)p.tokens * ((rows + step - 1) / step);
  const int u = waves <= 4096 ? 1 : waves <= 98304 ? 2 : 4;
  const dim3 grid((unsigned)(((int64_t)p.tokens * ((rows + step * u - 1) / (step * u)) + 3) / 4));
#define MLA_ROTARY(D, U) \
  if (dim == D && u == U) hipLaunchKernelGGL((qk_norm_rope_kernel<D, U>), grid, dim3(256), 0, stream, p);
  MLA_ROTARY(64, 1)
  MLA_ROTARY(64, 2)
  MLA_ROTARY(64, 4)
  MLA_ROTARY(128, 1)
  MLA_ROTARY(128, 2)
  MLA_ROTARY(128, 4)
#undef MLA_ROTARY
  return hipGetLastError();
}

}  // namespace mla
