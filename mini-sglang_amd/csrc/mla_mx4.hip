// Rows of K and V into a cache that holds them in 4 bits, and back (mla_mx4.h: the format).
//
// A lane takes 8 dims: 16 bytes of bf16, 4 of codes. Four lanes share a block of 32; its largest magnitude is found in two
// DPP steps on the bits (bf16 magnitudes order like whole numbers, infinities and NaN above all of them). The power of two
// is exact to divide by, so rounding to the nearest code is the only rounding, in one instruction for two values.
// Bound: HBM for many rows, a launch for few. 8192 rows of 8 heads of 128, 43 MB: in 11.0 us, out 9.6 (13.3 and 12.6 with a
// thread for K and one for V); 64 rows 3 us each.
#include "mla_mx4.h"

namespace mla {
namespace {

// 8 dims of a row of K and of V
struct Piece {
  int t, head, x;
  int64_t row;  // of the pool
};
template <int D>
__device__ __forceinline__ Piece mx4_piece(const Mx4Rows& p, uint32_t i) {
  constexpr int kLanes = D / 8;
  Piece r;
  r.x = (int)(i % kLanes);
  const uint32_t row = i / kLanes;
  r.t = (int)(row / (uint32_t)p.kv_heads);
  r.head = (int)(row - (uint32_t)r.t * p.kv_heads);
  r.row = p.index_bits == 32 ? ((const int32_t*)p.indices)[r.t] : ((const int64_t*)p.indices)[r.t];
  return r;
}
__device__ __forceinline__ uint8_t* mx4_codes(const Mx4Rows& p, const Mx4View& pool, const Piece& c) {
  return pool.codes + (c.row >> p.log2_ps) * pool.c_page + (c.row & ((1 << p.log2_ps) - 1)) * pool.c_tok + c.head * pool.c_head + 4 * c.x;
}
__device__ __forceinline__ uint8_t* mx4_scale(const Mx4Rows& p, const Mx4View& pool, const Piece& c) {
  return pool.scales + (c.row >> p.log2_ps) * pool.s_page + (c.row & ((1 << p.log2_ps) - 1)) * pool.s_tok + c.head * pool.s_head + c.x / 4;
}

// Codes of 8 values (two a word) and their block's scale, by all four lanes of a block.
__device__ __forceinline__ uint32_t mx4_round(const u32x4 w, uint32_t& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, w[k] >> 16 & 0x7fffu));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));  // lane ^ 2
  const uint32_t e = top >> 7;
  scale = e == 255 ? 255 : e > 2 ? e - 2 : 0;
  const float f = __uint_as_float(scale << 23);
  auto two = [](uint32_t x) { return __builtin_bit_cast(bf16x2, x); };
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[0]), f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[1]), f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[2]), f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[3]), f, 3);
  return e == 255 ? 0 : codes;
}

template <int D>
__global__ __launch_bounds__(256) void mx4_store_kernel(const Mx4Rows p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;  // 32 bits by the host
  if (i >= (uint32_t)p.rows * p.kv_heads * (D / 8)) return;  // whole rows: a block's four lanes leave together
  const Piece c = mx4_piece<D>(p, i);
  const u32x4 k = *reinterpret_cast<const u32x4*>(p.k + (int64_t)c.t * p.k_stride_t + (int64_t)c.head * p.k_stride_h + 8 * c.x);
  const u32x4 v = *reinterpret_cast<const u32x4*>(p.v + (int64_t)c.t * p.v_stride_t + (int64_t)c.head * p.v_stride_h + 8 * c.x);
  uint32_t ks, vs;
  const uint32_t kc = mx4_round(k, ks), vc = mx4_round(v, vs);
  if (c.row < 0 || c.row >= p.pool_rows) return;
  *reinterpret_cast<uint32_t*>(mx4_codes(p, p.k_pool, c)) = kc;
  *reinterpret_cast<uint32_t*>(mx4_codes(p, p.v_pool, c)) = vc;
  if (c.x % 4 == 0) {
    *mx4_scale(p, p.k_pool, c) = (uint8_t)ks;
    *mx4_scale(p, p.v_pool, c) = (uint8_t)vs;
  }
}

template <int D>
__global__ __launch_bounds__(256) void mx4_load_kernel(const Mx4Rows p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= (uint32_t)p.rows * p.kv_heads * (D / 8)) return;
  const Piece c = mx4_piece<D>(p, i);
  u32x4 k{}, v{};
  if (c.row >= 0 && c.row < p.pool_rows) {
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(mx4_codes(p, p.k_pool, c)), vc = *reinterpret_cast<const uint32_t*>(mx4_codes(p, p.v_pool, c));
    const uint32_t ks = *mx4_scale(p, p.k_pool, c), vs = *mx4_scale(p, p.v_pool, c);
    k = mx4_values(kc, ks << 23);
    v = mx4_values(vc, vs << 23);
  }
  *reinterpret_cast<u32x4*>(p.k_out + (int64_t)c.t * p.k_stride_t + (int64_t)c.head * p.k_stride_h + 8 * c.x) = k;
  *reinterpret_cast<u32x4*>(p.v_out + (int64_t)c.t * p.v_stride_t + (int64_t)c.head * p.v_stride_h + 8 * c.x) = v;
}

}  // namespace

hipError_t launch_mx4_rows(const Mx4Rows& p, int dim, bool load, hipStream_t stream) {
  const int64_t pieces = (int64_t)p.rows * p.kv_heads * (dim / 8);
  const dim3 grid((unsigned)((pieces + 255) / 256));
  if (load) {
    if (dim == 128) hipLaunchKernelGGL(mx4_load_kernel<128>, grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(mx4_load_kernel<64>, grid, dim3(256), 0, stream, p);
  } else {
    if (dim == 128) hipLaunchKernelGGL(mx4_store_kernel<128>, grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(mx4_store_kernel<64>, grid, dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace mla
