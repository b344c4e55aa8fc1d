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

#include <limits.h>

#include "mla_common.h"
#include "mla_device.h"

namespace mla {

typedef float f32x2 __attribute__((ext_vector_type(2)));

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
  f32x2* ws_lse;  // [slots, rows] their log2-domain LSEs: the nearest fp32, and the rest
  int32_t target;  // items that a batch's keys are split into, about (0: no splitting), a power of two
  int32_t log2_target;
  int32_t fit;     // at most `target`, where that can be
  int32_t wide;    // eight waves a CTA instead of four, sharing an item's keys
  int32_t out_16b;  // rows of out start 16-byte aligned
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

// Inclusive scan over the wave (lane 63 holds the whole): DPP row shifts, then row broadcasts; a ds_bpermute step
// would wait out the LDS latency each time.
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T v, F&& f) {
  static_assert(sizeof(T) == 4, "one register");
  auto step = [&](auto ctrl, auto rows) {
    const int w = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    v = f(v, __builtin_bit_cast(T, w));  // lanes without a source add the bits of 0
  };
  step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr:1
  step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15 to rows 1 and 3
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_iscan(int v) {
  return wave_scan(v, [](int a, int b) { return a + b; });
}
// Keys of a piece, C: the batch's keys, weighted with the row blocks that read them, over `target` items, in whole tiles
// of 64 and at least gqa_min_split; with `fit`, enlarged until the pieces are at most `target` (the CTAs that run at once:
// one more piece would be a round of its own). Requests of more keys are cut into ceil(L / C) pieces. Every kernel of a
// call computes the same C from the same lengths, so no plan is made on the host and a captured launch follows its
// lengths; in whole numbers, since the kernels find each other's partial results by it: a sum that one of them rounds
// otherwise would join foreign ones. C is above cost / target, so a batch has fewer than `target` pieces more than
// blocks; a request in pieces has L > C, so ceil(L / C) <= 2 L / C, and 2 target slots hold every piece. The cost counts
// 16 keys as one; requests stay in one piece where it passes 2^26 for one of them (or of every 64th), 2^30 keys of one block.
// Least keys of a piece: a tile for each wave of the stream kernel; 16 stages of the blocks (their joining takes 6 us).
template <int kRows>
constexpr int gqa_min_split() {
  return kRows <= 32 ? 128 : 512;
}
template <int kRows>
__device__ __forceinline__ int gqa_blocks(const GqaParams& p, const GqaRequest& r) {
  return (r.E * p.group + kRows - 1) / kRows;
}
__device__ __forceinline__ int gqa_pieces(int L, int C) { return L > C ? (L - 1) / C + 1 : 1; }
// r: request `lane` (batches of more than 64 requests read the others here)
template <int kRows>
__device__ __forceinline__ int gqa_piece_keys(const GqaParams& p, const GqaRequest& r) {
  if (p.target <= 0) return 0x7fffffff;
  const int lane = threadIdx.x & 63;
  constexpr uint32_t kMost = (1u << 26) - 1;  // of a lane: the wave's sum fits 32 bits
  auto cost_of = [&](const GqaRequest& x) {
    const uint64_t c = (uint64_t)(uint32_t)gqa_blocks<kRows>(p, x) * (uint32_t)((x.L + 15) >> 4);
    return c < kMost ? (uint32_t)c : kMost;
  };
  uint32_t cost = lane < p.batch ? cost_of(r) : 0;
  for (int b = 64 + lane; b < p.batch; b += 64) cost = min(cost + cost_of(gqa_request(p, b)), kMost);
  if (__ballot(cost == kMost) != 0) return 0x7fffffc0;
  cost = (uint32_t)__builtin_amdgcn_readlane(wave_iscan((int)cost), 63);
  const uint64_t c = ((uint64_t)cost * (uint32_t)(16 * p.kv_heads) >> p.log2_target) + 64;
  int C = c < 0x7fffffc0 ? (int)c & ~63 : 0x7fffffc0;
  // blocks: `target` items are two CTAs a compute unit; short pieces, half as many. One against two, 64 query and 8 KV
  // heads unless said: 8 chunks of 100 tokens on 2000 (32 heads) 53 / 64 us, 4 of 256 on 4000 (32) 96 / 106; one of 512 on
  // 8000 190 / 182, one of 4096 on 28,000 (8 and 1) 585 / 535
  if (kRows >= 128 && C < 2560) C *= 2;
  C = max(C, gqa_min_split<kRows>());
  if (p.fit && p.batch <= 64) {
    for (int i = 0; i < 4 && C < (1 << 24); ++i) {
      const int n = lane < p.batch ? gqa_blocks<kRows>(p, r) * gqa_pieces(r.L, C) * p.kv_heads : 0;
      const int items = __builtin_amdgcn_readlane(wave_iscan(n), 63);
      if (items <= p.target) break;
      C = (int)(((uint64_t)C * (uint32_t)items >> p.log2_target) + 64) & ~63;
    }
  }
  return __builtin_amdgcn_readfirstlane(C);
}

// Item `item` of the batch: request, block of kRows rows, KV head, piece of the keys. Items of a request are
// ((block, piece), head), heads fastest. kLong: a request's last blocks, which see the most keys, come first, and of up
// to 64 requests the longest, so that no long item runs alone at the end. slot: of the item's partial result, < 0 for a request in one piece.
struct GqaItem {
  int b, block, head, piece, pieces, C, slot;
  GqaRequest r;
};
template <int kRows, bool kLong>
__device__ __forceinline__ bool gqa_find(const GqaParams& p, int item, GqaItem& it) {
  const int lane = threadIdx.x & 63;
  GqaRequest r{0, 0, 0, 0};
  if (lane < p.batch) r = gqa_request(p, lane);
  it.C = gqa_piece_keys<kRows>(p, r);
  int acc = 0, slots = 0;
  for (int c0 = 0; c0 < p.batch; c0 += 64) {
    if (c0 > 0) {
      r = GqaRequest{0, 0, 0, 0};
      if (c0 + lane < p.batch) r = gqa_request(p, c0 + lane);
    }
    const int pieces = gqa_pieces(r.L, it.C);
    const int n = gqa_blocks<kRows>(p, r) * pieces * p.kv_heads, ns = pieces > 1 ? n : 0;
    const int incl = wave_iscan(n), sincl = wave_iscan(ns);
    int first = acc + incl - n;  // the request's first item
    if constexpr (kLong) {
      if (p.batch <= 64) {  // after those of longer requests, and of as long ones before it
        // (keys of 2^25 and more count as alike: the order is any). Constant lanes, 16 at a time: a readlane of a
        // loop's counter took 60 ns.
        const int key = min(r.L, (1 << 25) - 1) * 64 + 63 - lane;
        first = 0;
        auto group = [&](auto g0) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int ni = __builtin_amdgcn_readlane(n, decltype(g0)::value + i);
            first += __builtin_amdgcn_readlane(key, decltype(g0)::value + i) > key ? ni : 0;
          }
        };
        group(std::integral_constant<int, 0>{});
        if (p.batch > 16) group(std::integral_constant<int, 16>{});
        if (p.batch > 32) group(std::integral_constant<int, 32>{});
        if (p.batch > 48) group(std::integral_constant<int, 48>{});
      }
    }
    const uint64_t hit = __ballot(item >= first && item < first + n);
    if (hit != 0) {
      const int fl = __builtin_ctzll(hit);
      const int local = item - __builtin_amdgcn_readlane(first, fl);
      it.b = c0 + fl;
      it.pieces = __builtin_amdgcn_readlane(pieces, fl);
      it.head = local % p.kv_heads;
      it.piece = local / p.kv_heads % it.pieces;
      it.block = local / p.kv_heads / it.pieces;
      if constexpr (kLong) it.block = __builtin_amdgcn_readlane(n, fl) / (it.pieces * p.kv_heads) - 1 - it.block;
      it.slot = it.pieces > 1 ? slots + __builtin_amdgcn_readlane(sincl - ns, fl) +
                                    (it.block * it.pieces + it.piece) * p.kv_heads + it.head : -1;
      it.r.q0 = __builtin_amdgcn_readlane(r.q0, fl);
      it.r.E = __builtin_amdgcn_readlane(r.E, fl);
      it.r.L = __builtin_amdgcn_readlane(r.L, fl);
      it.r.P = __builtin_amdgcn_readlane(r.P, fl);
      it.C = ((it.r.L + it.pieces - 1) / it.pieces + 63) & ~63;  // of the request: pieces alike
      return true;
    }
    acc += __builtin_amdgcn_readlane(incl, 63);
    slots += __builtin_amdgcn_readlane(sincl, 63);
  }
  return false;
}

// LSE m + t of a row, log2 domain, and what its rounding leaves out (from |m| = 2^24 on as large as the sum's logarithm, by
// which pieces of like scores differ).
__device__ __forceinline__ f32x2 gqa_lse(bool some, float m, float t) {
  const float sum = m + t;
  return some ? f32x2{sum, (m - sum) + t} : f32x2{-INFINITY, 0.f};
}

// Token row of key j of request b (packed prompts: q0 + j); page ids are clamped into the pool. The host keeps pools
// below 2^31 rows.
__device__ __forceinline__ int gqa_row(const GqaParams& p, int b, int q0, int j) {
  if (p.page_table == nullptr) return q0 + j;
  const int pid = min(max(p.page_table[(int64_t)b * p.pt_stride + (j >> p.log2_ps)], 0), p.num_pages - 1);
  return (pid << p.log2_ps) + (j & ((1 << p.log2_ps) - 1));
}

// For rows (bits of `rows`, row0 + bit) whose values are not finite although their sums of numerators are. Either V holds an
// infinity or a NaN at a key that such a row attends, and that is its result; or at a key that it does not attend, and the
// matrix product (weight zero times it) put it there; or finite values added up past fp32's range before a maximum that
// makes them small was seen (numerators are relative to a running or a lazy reference). The last two are computed again,
// row by row by the whole wave, until NaN throughout: slow (0.13 ms per 1000 keys) and rare. One pass over the item's V tells
// which: each lane notes for its dims the first key that is not finite, and compares with what the row came out as. (It skips
// to the first row's last key once that explains all that came out.)
// The reference is a running maximum of its own, not the products': the scores here are sums in another order. A second sum
// of values times 2^-32 stays in range whatever they are (below 2^31 keys), and is the result where the first did not.
// at: row0's row of the workspace.
template <int D>
__device__ __forceinline__ void gqa_rows_again(const GqaParams& p, const GqaItem& it, int row0, uint64_t rows, int k0, int k1, int64_t at) {
  constexpr int kN = D / 64;  // dims of a lane
  typedef __bf16 dims_t __attribute__((ext_vector_type(kN)));
  typedef float part_t __attribute__((ext_vector_type(kN)));
  constexpr int kU = 8, kScan = 16;  // keys in flight (32: no faster)
  const int d0 = (threadIdx.x & 63) * kN, hi = min(it.r.L, k0 + ((k1 - k0 + 31) & ~31));
  auto load = [&](const __bf16* x) { return __builtin_convertvector(*reinterpret_cast<const dims_t*>(x + d0), part_t); };
  auto value = [&](int64_t row) { return load(p.v + row * p.v_row_stride + (int64_t)it.head * p.v_head_stride); };
  auto finite = [](float x) { return x * 0.f == 0.f; };
  // the rows' stores, by other lanes of the wave, have landed
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  wait_vmcnt<0>();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  auto token = [&](int r) { return r / p.group; };
  auto end_of = [&](int r) { return min(k1, it.r.P + token(r) + 1); };
  auto partial = [&](int r) { return p.ws_o + (at + (r - row0)) * D + d0; };
  auto out_row = [&](int r) {
    return p.out + (int64_t)(it.r.q0 + token(r)) * p.out_stride_t + (int64_t)(it.head * p.group + r % p.group) * p.out_stride_h;
  };
  auto result = [&](int r) { return it.slot >= 0 ? *reinterpret_cast<const part_t*>(partial(r)) : load(out_row(r)); };
  bool bad[kN] = {};  // dims of the lane in which some row is not finite
  for (uint64_t left = rows; left != 0; left &= left - 1) {
    const part_t was = result(row0 + __builtin_ctzll(left));
#pragma unroll
    for (int e = 0; e < kN; ++e) bad[e] = bad[e] || !finite(was[e]);
  }
  int first[kN], last = -1;  // keys of the lane's dims that are not finite
#pragma unroll
  for (int e = 0; e < kN; ++e) first[e] = INT_MAX;
  const int end0 = end_of(row0 + __builtin_ctzll(rows));  // all of the rows attend the keys before it
  for (int j = k0; j < hi;) {
    part_t v[kScan];
#pragma unroll
    for (int u = 0; u < kScan; ++u) v[u] = value(gqa_row(p, it.b, it.r.q0, min(j + u, hi - 1)));
#pragma unroll
    for (int u = 0; u < kScan; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (!finite(v[u][e])) {
          last = min(j + u, hi - 1);
          first[e] = min(first[e], last);
        }
    j += kScan;
    bool open = false;
#pragma unroll
    for (int e = 0; e < kN; ++e) open = open || (bad[e] && first[e] >= end0);
    if (__ballot(open) == 0) j = max(j, end0);
  }
  for (; rows != 0; rows &= rows - 1) {
    const int r = row0 + __builtin_ctzll(rows), tok = token(r), head = it.head * p.group + r % p.group, end = end_of(r);
    const part_t was = result(r);
    bool again = last >= end;
#pragma unroll
    for (int e = 0; e < kN; ++e) again = again || (!finite(was[e]) && first[e] >= end);
    if (__ballot(again) == 0) continue;
    const part_t q = load(p.q + (int64_t)(it.r.q0 + tok) * p.q_stride_t + (int64_t)head * p.q_stride_h);
    part_t o = {}, small = {};
    float l = 0.f, m = -3.4028234663852886e38f;
    for (int j = k0; j < end; j += kU) {
      part_t x[kU], v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t row = gqa_row(p, it.b, it.r.q0, min(j + u, end - 1));
        x[u] = q * load(p.k + row * p.k_row_stride + (int64_t)it.head * p.k_head_stride);
        v[u] = value(row);
      }
      float s[kU], top = m;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float sum = x[u][0];
        if constexpr (kN == 2) sum += x[u][1];
        s[u] = wave_sum64(sum);
        if (j + u >= end) s[u] = -INFINITY;
        top = fmaxf(top, s[u]);
      }
      // unscaled differences: exact next to the maximum, at any size of the scores
      const float f = __builtin_amdgcn_exp2f((m - top) * p.scale_log2);
      m = top;
      l *= f;
      o *= f;
      small *= f;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float e = __builtin_amdgcn_exp2f((s[u] - m) * p.scale_log2);
        if (j + u < end) {
          l += e;
          o += e * v[u];
          small += e * (v[u] * 0x1p-32f);
        }
      }
      bool done = small[0] != small[0];
      if constexpr (kN == 2) done = done && small[1] != small[1];
      if (__ballot(!done) == 0) break;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < kN; ++e) o[e] = finite(o[e]) ? o[e] * inv : small[e] * inv * 0x1p32f;
    if (it.slot >= 0) *reinterpret_cast<part_t*>(partial(r)) = o;
    else *reinterpret_cast<dims_t*>(out_row(r) + d0) = __builtin_convertvector(o, dims_t);
  }
}

// CTAs of a launch of `rows` rows: sum over requests of ceil(E group / rows), then of ceil(L / C) pieces each.
inline int64_t gqa_ctas(const GqaParams& p, int rows) {
  return (((int64_t)p.total_q * p.group + rows - 1) / rows + p.batch) * p.kv_heads + p.target;
}
// Whether a call's launches hold fewer than 2^32 threads each, the merge's too: looked at before the first of them.
inline bool gqa_grids_ok(const GqaParams& p, int rows) {
  auto ok = [](int64_t ctas, int threads) { return ctas <= 0x7fffffff && ctas * threads <= (int64_t)UINT32_MAX; };
  return ok(gqa_ctas(p, rows), p.wide || rows == 256 ? 512 : 256) && (p.target == 0 || ok((int64_t)p.total_q * p.kv_heads * p.group, 64));
}

hipError_t launch_gqa_rows(const GqaParams& p, int dim, int rows, hipStream_t stream);    // blocks of 128 or 256 rows
hipError_t launch_gqa_stream(const GqaParams& p, int dim, int rows, hipStream_t stream);  // CTAs of 16 or 32 rows

}  // namespace mla
