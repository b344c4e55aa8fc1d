// Rows of K and V into a cache that holds them in 4 bits, and back (mla_mx4.h: the format).
//
// A lane takes 8 dims: 16 bytes of bf16, 4 of codes. Four lanes share a block of 32; its largest magnitude is found in two
// DPP steps on the bits (bf16 magnitudes order like whole numbers, infinities and NaN above all of them). The power of two
// is exact to divide by, so rounding to the nearest code is the only rounding, in one instruction for two values.
#include "mla_mx4.h"

namespace mla {
namespace {

// (row, pool) of 16-byte piece `i` of the rows of K, then of V
struct Piece {
  int t, head, x;
  bool v;
};
template <int D>
__device__ __forceinline__ Piece mx4_piece(const Mx4Rows& p, uint32_t i) {
  constexpr int kLanes = D / 8;
  Piece r;
  r.x = (int)(i % kLanes);
  const uint32_t row = i / kLanes, heads = 2 * p.kv_heads;
  r.t = (int)(row / heads);
  const int h = (int)(row - r.t * heads);
  r.v = h >= p.kv_heads;
  r.head = r.v ? h - p.kv_heads : h;
  return r;
}

__device__ __forceinline__ int64_t mx4_index(const Mx4Rows& p, int t) {
  return p.index_bits == 32 ? ((const int32_t*)p.indices)[t] : ((const int64_t*)p.indices)[t];
}

template <int D>
__global__ __launch_bounds__(256) void mx4_store_kernel(const Mx4Rows p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;  // 32 bits by the host
  if (i >= (uint32_t)p.rows * 2 * p.kv_heads * (D / 8)) return;  // whole rows: a block's four lanes leave together
  const Piece c = mx4_piece<D>(p, i);
  const int64_t row = mx4_index(p, c.t);
  const __bf16* in = c.v ? p.v + (int64_t)c.t * p.v_stride_t + (int64_t)c.head * p.v_stride_h
                         : p.k + (int64_t)c.t * p.k_stride_t + (int64_t)c.head * p.k_stride_h;
  const u32x4 w = *reinterpret_cast<const u32x4*>(in + 8 * c.x);
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, w[k] >> 16 & 0x7fffu));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));  // lane ^ 2
  const uint32_t e = top >> 7, scale = e == 255 ? 255 : e > 2 ? e - 2 : 0;
  uint32_t codes = 0;
  if (e != 255) {
    const float f = __uint_as_float(scale << 23);
    auto two = [&](uint32_t x) { return __builtin_bit_cast(bf16x2, x); };
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[0]), f, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[1]), f, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[2]), f, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, two(w[3]), f, 3);
  }
  if (row < 0 || row >= p.pool_rows) return;
  const int64_t page = row >> p.log2_ps, tok = row & ((1 << p.log2_ps) - 1);
  const Mx4View& pool = c.v ? p.v_pool : p.k_pool;
  *reinterpret_cast<uint32_t*>(pool.codes + page * pool.c_page + tok * pool.c_tok + c.head * pool.c_head + 4 * c.x) = codes;
  if (c.x % 4 == 0) pool.scales[page * pool.s_page + tok * pool.s_tok + c.head * pool.s_head + c.x / 4] = (uint8_t)scale;
}

template <int D>
__global__ __launch_bounds__(256) void mx4_load_kernel(const Mx4Rows p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;  // 32 bits by the host
  if (i >= (uint32_t)p.rows * 2 * p.kv_heads * (D / 8)) return;
  const Piece c = mx4_piece<D>(p, i);
  const int64_t row = mx4_index(p, c.t);
  u32x4 w{};
  if (row >= 0 && row < p.pool_rows) {
    const int64_t page = row >> p.log2_ps, tok = row & ((1 << p.log2_ps) - 1);
    const Mx4View& pool = c.v ? p.v_pool : p.k_pool;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(pool.codes + page * pool.c_page + tok * pool.c_tok + c.head * pool.c_head + 4 * c.x);
    w = mx4_values(codes, (uint32_t)pool.scales[page * pool.s_page + tok * pool.s_tok + c.head * pool.s_head + c.x / 4] << 23);
  }
  __bf16* out = c.v ? p.v_out + (int64_t)c.t * p.v_stride_t + (int64_t)c.head * p.v_stride_h
                    : p.k_out + (int64_t)c.t * p.k_stride_t + (int64_t)c.head * p.k_stride_h;
  *reinterpret_cast<u32x4*>(out + 8 * c.x) = w;
}

}  // namespace

hipError_t launch_mx4_rows(const Mx4Rows& p, int dim, bool load, hipStream_t stream) {
  const int64_t pieces = (int64_t)p.rows * 2 * p.kv_heads * (dim / 8);
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
