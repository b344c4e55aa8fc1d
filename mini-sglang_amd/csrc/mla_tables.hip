// The tables of a scheduler step, from its requests' lengths: pages given to the new tokens, token table rows, page
// table, slots, positions and query offsets, in one launch (integer work, bit-exact).
//
// Request b has cached tokens [0, c) and new tokens [c, d); it takes pages first = ceil(c / ps) .. last - 1 = ceil(d / ps)
// - 1 of its row, the free slots base_b + 0, 1, ..., base_b = the pages that the requests before it take.
#include "mla_common.h"

namespace mla {
namespace {

constexpr int kPer = 4;             // tokens, and page table columns, of a thread, in flight together
constexpr int kChunk = 256 * kPer;  // of a CTA

template <bool kPow2>
__device__ __forceinline__ int page_of(int t, int ps, int log2_ps) {
  return kPow2 ? t >> log2_ps : t / ps;
}

// CTA (x, b) takes the x-th kChunk tokens and columns of request b; it sums the lengths before b itself, in the one round
// trip that its own lengths take. Bound: writes, and with few tokens the launch and three dependent loads (lengths, free
// slot, store). 256 prompts of up to 8192 tokens at page size 1, 23 MB: 10.5 us, 1.6 more with the tokens of a thread one after
// the other, 0.1 more with four neighbouring ones a thread and 16-byte stores; a decode step of 64 requests 4.2.
template <bool kPow2>
__global__ __launch_bounds__(256) void page_tables_kernel(const PageTablesParams p) {
  __shared__ int s_sum[4][3];
  const int b = blockIdx.y, ps = p.page_size;
  auto page = [&](int t) { return page_of<kPow2>(t, ps, p.log2_ps); };
  // lengths, cut to the table's width
  auto lens = [&](int i, int& c, int& d) {
    c = min(max(p.cached_lens[i], 0), p.tt_cols);
    d = min(max(p.device_lens[i], c), p.tt_cols);
  };
  int c, d;
  lens(b, c, d);
  int32_t* row = p.token_table + (int64_t)min(max(p.table_idx[b], 0), p.tt_rows - 1) * p.tt_stride;
  // pages of the requests before b, of all; new tokens before b. Sums stop at 2^31 - 1: a wrapped one would pass for few
  // pages, or for an offset in front of out_loc.
  int sum[3] = {0, 0, 0};
  auto add = [](int x, int y) { return __builtin_elementwise_add_sat(x, y); };
  for (int i = threadIdx.x; i < p.batch; i += 256) {
    int ci, di;
    lens(i, ci, di);
    const int n = i < p.alloc_reqs ? page(di + ps - 1) - page(ci + ps - 1) : 0;
    sum[1] = add(sum[1], n);
    if (i < b) {
      sum[0] = add(sum[0], n);
      sum[2] = add(sum[2], di - ci);
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum[k] = add(sum[k], __shfl_xor(sum[k], o));
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6][k] = sum[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) sum[k] = add(add(s_sum[0][k], s_sum[1][k]), add(s_sum[2][k], s_sum[3][k]));
  const int before = sum[0], all = sum[1], fresh_before = sum[2];
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.cu_seqlens_q[b] = fresh_before;
    if (b == p.batch - 1) p.cu_seqlens_q[p.batch] = add(fresh_before, d - c);
    if (b == 0) *p.pages_taken = all;
  }
  // slots and positions that no token has: -1, which no row is stored at, and 0
  auto none = [&](int64_t n, int64_t stride) {
    for (; n < p.total_new; n += stride) {
      p.out_loc[n] = -1;
      p.positions[n] = 0;
    }
  };
  const int64_t ctas = gridDim.x, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (all > min(p.num_free, 0x7ffffffe)) {  // out of pages: the token table stays, the others hold nothing
    none(b * ctas * 256 + id, ctas * p.batch * 256);
    for (int64_t i = id; i < p.pt_cols; i += ctas * 256) p.page_table[b * p.pt_stride + i] = 0;
    return;
  }
  if (b == p.batch - 1) none(add(fresh_before, d - c) + id, ctas * 256);
  const int first = page(c + ps - 1), last = page(d + ps - 1);
  const bool takes = b < p.alloc_reqs;
  const int32_t* free_slots = p.free_slots + before - first;  // page j of the row: free_slots[j]
  // tokens from c to the end of the last page taken
  const int span = (takes && last > first ? min(last * ps, p.tt_cols) : d) - c;
  // once, unless a request has more new tokens than the launch was made for
  const unsigned need = max(span, p.pt_cols);
  for (unsigned x = blockIdx.x * kChunk; x < need; x += gridDim.x * kChunk) {
    const int x0 = x + threadIdx.x;
    int loc[kPer], head[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = x0 + 256 * u, pos = c + i, j = page(pos);
      if (i < span) loc[u] = takes && j >= first ? free_slots[j] + pos - j * ps : row[pos];
      if (i < last) head[u] = takes && i >= first ? free_slots[i] : row[i * ps];
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = x0 + 256 * u, pos = c + i;
      const int64_t n = (int64_t)fresh_before + i;
      if (i < span && takes && page(pos) >= first) row[pos] = loc[u];
      if (i < span && pos < d && n < p.total_new) {
        p.out_loc[n] = loc[u];
        p.positions[n] = pos;
      }
      if (i < p.pt_cols) {
        const int v = i < last ? head[u] : 0;
        p.page_table[b * p.pt_stride + i] = kPow2 ? v >> p.log2_ps : v / ps - (v % ps != 0 && v < 0);
      }
    }
  }
}

}  // namespace

hipError_t launch_page_tables(const PageTablesParams& p, int32_t max_extend, hipStream_t stream) {
  // tokens of a request, to the end of its last page; within the table, so that a thread's index stays below 2^31
  const int64_t tokens = (int64_t)(max_extend < p.tt_cols ? max_extend : p.tt_cols) + p.page_size - 1;
  const int64_t most = tokens > p.pt_cols ? tokens : p.pt_cols;
  const dim3 grid((unsigned)((most + kChunk - 1) / kChunk > 0 ? (most + kChunk - 1) / kChunk : 1), (unsigned)p.batch);
  if (p.log2_ps >= 0) hipLaunchKernelGGL(page_tables_kernel<true>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(page_tables_kernel<false>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mla
