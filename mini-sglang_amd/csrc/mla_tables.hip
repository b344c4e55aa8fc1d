// The tables of a scheduler step, from its requests' lengths: pages given to the new tokens, token table rows, page
// table, slots, positions and query offsets, in one launch (integer work, bit-exact).
//
// Request b has cached tokens [0, c) and new tokens [c, d); it takes pages first = ceil(c / ps) .. last - 1 = ceil(d / ps)
// - 1 of its row, the free slots base_b + 0, 1, ..., base_b = the pages that the requests before it take.
#include "mla_common.h"

namespace mla {
namespace {

constexpr int kChunk = 2048;  // tokens, and page table columns, of a CTA

__device__ __forceinline__ int block_sum(int v, int* s) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0] + s[1] + s[2] + s[3];
  __syncthreads();
  return v;
}

template <bool kPow2>
__device__ __forceinline__ int page_of(int t, int ps, int log2_ps) {
  return kPow2 ? t >> log2_ps : t / ps;
}

template <bool kPow2>
__global__ __launch_bounds__(256) void page_tables_kernel(const PageTablesParams p) {
  __shared__ int s_sum[4];
  const int b = blockIdx.y, x0 = blockIdx.x * kChunk, ps = p.page_size;
  auto page = [&](int t) { return page_of<kPow2>(t, ps, p.log2_ps); };
  // lengths, cut to the table's width
  auto lens = [&](int i, int& c, int& d) {
    c = min(max(p.cached_lens[i], 0), p.tt_cols);
    d = min(max(p.device_lens[i], c), p.tt_cols);
  };
  int before = 0, all = 0, fresh_before = 0;  // pages of the requests before b, of all; new tokens before b
  for (int i = threadIdx.x; i < p.batch; i += 256) {
    int c, d;
    lens(i, c, d);
    const int n = i < p.alloc_reqs ? page(d + ps - 1) - page(c + ps - 1) : 0;
    all += n;
    if (i < b) {
      before += n;
      fresh_before += d - c;
    }
  }
  before = block_sum(before, s_sum);
  all = block_sum(all, s_sum);
  fresh_before = block_sum(fresh_before, s_sum);
  int c, d;
  lens(b, c, d);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.cu_seqlens_q[b] = fresh_before;
    if (b == p.batch - 1) p.cu_seqlens_q[p.batch] = fresh_before + d - c;
    if (b == 0) *p.pages_taken = all;
  }
  if (all > p.num_free) return;  // out of pages: no table is touched
  const int first = page(c + ps - 1), last = page(d + ps - 1);
  const bool takes = b < p.alloc_reqs;
  int32_t* row = p.token_table + (int64_t)min(max(p.table_idx[b], 0), p.tt_rows - 1) * p.tt_stride;
  const int32_t* free_slots = p.free_slots + before - first;  // page j of the row: free_slots[j]
  // tokens from c to the end of the last page taken
  const int end = takes && last > first ? min(last * ps, p.tt_cols) : d;
  for (int i = x0 + threadIdx.x; i < min(x0 + kChunk, end - c); i += 256) {
    const int pos = c + i, j = page(pos);
    int loc;
    if (takes && j >= first) row[pos] = loc = free_slots[j] + pos - j * ps;
    else loc = row[pos];
    const int64_t n = (int64_t)fresh_before + i;
    if (pos < d && n < p.total_new) {
      p.out_loc[n] = loc;
      p.positions[n] = pos;
    }
  }
  for (int j = x0 + threadIdx.x; j < min(x0 + kChunk, p.pt_cols); j += 256) {
    int v = 0;
    if (j < last) v = takes && j >= first ? free_slots[j] : row[j * ps];
    p.page_table[b * p.pt_stride + j] = kPow2 ? v >> p.log2_ps : v / ps - (v % ps != 0 && v < 0);
  }
}

}  // namespace

hipError_t launch_page_tables(const PageTablesParams& p, int32_t max_extend, hipStream_t stream) {
  const int64_t tokens = (int64_t)max_extend + p.page_size - 1;  // of a request, to the end of its last page
  const int64_t most = tokens > p.pt_cols ? tokens : p.pt_cols;
  const dim3 grid((unsigned)((most + kChunk - 1) / kChunk > 0 ? (most + kChunk - 1) / kChunk : 1), (unsigned)p.batch);
  if (p.log2_ps >= 0) hipLaunchKernelGGL(page_tables_kernel<true>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(page_tables_kernel<false>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mla
