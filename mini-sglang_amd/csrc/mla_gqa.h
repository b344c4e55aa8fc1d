// Attention with per-head K and V of equal width (64 or 128) shared by groups of query heads, over packed prompts and
// over a paged cache: types and device helpers of its kernels (gfx950).
//
// Per request b of E new tokens and L keys (P = L - E before the chunk): query i attends keys j <= P + i,
//   s_j = scale q . k_j,  lse = ln sum_j exp s_j,  out = sum_j exp(s_j - lse) v_j;
// a query without keys gives out = 0, lse = -inf.
//
// The query heads of a KV head are rows of one matrix product: row r of (request, KV head) is query r / group of head
// r % group, so a K or V row is read once for all of them, and one new token fills group rows of a tile.
#pragma once

#include "mla_common.h"
#include "mla_device.h"

namespace mla {

struct GqaParams {
  const __bf16* q;  // [T, Hq, D]
  int64_t q_stride_t, q_stride_h;
  // K of (token row r, KV head h) at k + r * k_row_stride + h * k_head_stride, V likewise. Row of key j: packed
  // (page_table null) cu_seqlens_q[b] + j, else page_table[b, j >> log2_ps] << log2_ps | j & (ps - 1)
  const __bf16* k;
  int64_t k_row_stride, k_head_stride;
  const __bf16* v;
  int64_t v_row_stride, v_head_stride;
  int32_t num_pages, log2_ps;
  const int32_t* page_table;
  int64_t pt_stride;
  int32_t max_keys;             // keys that a page table row can hold (longer lengths are cut)
  const int32_t* cu_seqlens_q;  // [B + 1], or null: request b is query b
  const int32_t* seq_lens_k;    // [B], or null: as many keys as queries
  int32_t batch, total_q, kv_heads, group;
  int32_t max_q;  // queries of a request that the launch covers
  float scale_log2;
  __bf16* out;  // [T, Hq, D]
  int64_t out_stride_t, out_stride_h;
  float* lse;  // [T, Hq] or null
  int64_t lse_stride_t;
  float* ws_o;    // [slots, rows, D] partial outputs of split requests, normalised
  float* ws_lse;  // [slots, rows] their log2-domain LSEs
  int32_t target;  // items that a batch's keys are split into, about (0: no splitting)
};

// A request as the kernels see it; every read is bounded by what the host knows, whatever the device arrays hold.
struct GqaRequest {
  int q0, E, L, P;  // first query, queries, keys, keys before the first query
};
__device__ __forceinline__ GqaRequest gqa_request(const GqaParams& p, int b) {
  GqaRequest r;
  if (p.cu_seqlens_q != nullptr) {
    r.q0 = min(max(p.cu_seqlens_q[b], 0), p.total_q);
    r.E = min(max(p.cu_seqlens_q[b + 1], r.q0), p.total_q) - r.q0;
  } else {
    r.q0 = b;
    r.E = 1;
  }
  r.L = p.seq_lens_k != nullptr ? min(max(p.seq_lens_k[b], 0), p.max_keys) : r.E;
  r.P = r.L - r.E;
  r.E = min(r.E, p.max_q);
  return r;
}

__device__ __forceinline__ int wave_isum(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ int64_t wave_isum64(int64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Keys of a split: the batch's keys, weighted with the row blocks that read them, over `target` items, in whole tiles
// of 64 and at least kMin. Requests of more keys are cut into ceil(L / C) pieces. Every kernel of a call computes the
// same C from the same lengths, so no plan is made on the host and a captured launch follows its lengths.
// Sum over split requests of their pieces: ceil(L / C) <= 2 L / C, so 2 target slots hold them all.
constexpr int kGqaMinSplit = 256;
template <int kRows>
__device__ __forceinline__ int gqa_split_keys(const GqaParams& p) {
  if (p.target <= 0) return 0x7fffffff;
  const int lane = threadIdx.x & 63;
  int64_t cost = 0;
  for (int c0 = 0; c0 < p.batch; c0 += 64) {
    const int b = c0 + lane;
    if (b < p.batch) {
      const GqaRequest r = gqa_request(p, b);
      cost += (int64_t)((r.E * p.group + kRows - 1) / kRows) * r.L;
    }
  }
  cost = wave_isum64(cost) * p.kv_heads;
  const int64_t c = (cost / p.target + 64) / 64 * 64;  // above cost / target
  return (int)min(max(c, (int64_t)kGqaMinSplit), (int64_t)0x7fffffc0);
}

// Item `item` of the batch: request, block of kRows rows, KV head, piece of the keys. Items of a request are
// ((block, piece), head), heads fastest. slot: of the item's partial result, < 0 for a request in one piece.
struct GqaItem {
  int b, block, head, piece, pieces, slot;
  GqaRequest r;
};
template <int kRows>
__device__ __forceinline__ bool gqa_find(const GqaParams& p, int C, int item, GqaItem& it) {
  const int lane = threadIdx.x & 63;
  int acc = 0, slots = 0;
  for (int c0 = 0; c0 < p.batch; c0 += 64) {
    const int b = c0 + lane;
    GqaRequest r{0, 0, 0, 0};
    int n = 0, ns = 0, pieces = 1;
    if (b < p.batch) {
      r = gqa_request(p, b);
      pieces = r.L > C ? (r.L + C - 1) / C : 1;
      n = (r.E * p.group + kRows - 1) / kRows * pieces * p.kv_heads;
      ns = pieces > 1 ? n : 0;
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
    const uint64_t hit = __ballot(item >= acc + incl - n && item < acc + incl);
    if (hit != 0) {
      const int fl = __builtin_ctzll(hit);
      const int local = item - acc - __builtin_amdgcn_readlane(incl - n, fl);
      it.b = c0 + fl;
      it.pieces = __builtin_amdgcn_readlane(pieces, fl);
      it.head = local % p.kv_heads;
      it.piece = local / p.kv_heads % it.pieces;
      it.block = local / p.kv_heads / it.pieces;
      it.slot = it.pieces > 1 ? slots + __builtin_amdgcn_readlane(sincl - ns, fl) + local : -1;
      it.r.q0 = __builtin_amdgcn_readlane(r.q0, fl);
      it.r.E = __builtin_amdgcn_readlane(r.E, fl);
      it.r.L = __builtin_amdgcn_readlane(r.L, fl);
      it.r.P = __builtin_amdgcn_readlane(r.P, fl);
      return true;
    }
    acc += __shfl(incl, 63);
    slots += __shfl(sincl, 63);
  }
  return false;
}

// Token row of key j of request b (packed prompts: q0 + j); page ids are clamped into the pool.
__device__ __forceinline__ int64_t gqa_row(const GqaParams& p, int b, int q0, int j) {
  if (p.page_table == nullptr) return q0 + j;
  const int pid = min(max(p.page_table[(int64_t)b * p.pt_stride + (j >> p.log2_ps)], 0), p.num_pages - 1);
  return ((int64_t)pid << p.log2_ps) + (j & ((1 << p.log2_ps) - 1));
}

hipError_t launch_gqa_rows(const GqaParams& p, int dim, hipStream_t stream);    // many rows a request
hipError_t launch_gqa_stream(const GqaParams& p, int dim, hipStream_t stream);  // up to 64 rows a request

}  // namespace mla
