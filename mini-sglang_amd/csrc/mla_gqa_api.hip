// extern "C" entry points of the grouped-head attention and of the step's tables (declared in include/mla_amd.h):
// argument checks, the choice of kernel, and launches.
#include <math.h>

#include <algorithm>

#include "mla_gqa.h"

namespace mla {
namespace {

int done(hipError_t e, const char* who) {
  if (e != hipSuccess) return api_error(MLA_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
  api_error(MLA_OK, "%s", "");
  return MLA_OK;
}
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool is_pow2(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

// A launch's kernel: CTAs of 16 or 32 rows that stream keys, or (rows 128) blocks; how many items a paged batch is cut
// into (target, fit: mla_gqa.h; 0: requests in one piece), and whether its CTAs are the wide ones.
struct Choice {
  int rows, target;
  bool fit, wide;
};

// CTAs that run at once, two a compute unit, and about how many pieces of different length even out.
constexpr int kFit = 512;
constexpr int kTarget = 2048;
constexpr int kBlocksTarget = 512;
static_assert(!(kFit & (kFit - 1)) && !(kTarget & (kTarget - 1)) && !(kBlocksTarget & (kBlocksTarget - 1)), "powers of two");
constexpr int kBlock = 128;
// A paged batch of at least this many blocks fills the chip without cutting keys; up to this many keys (by the page
// table's width) cutting them gains nothing over joining the pieces: in blocks, and streamed by more CTAs than run at once.
constexpr int kBlocksEnough = 1024;
constexpr int kOnePieceBlocks = 1024;
constexpr int kOnePieceMany = 1600;
// Prompts of at least this many tokens on average (head_dim 128), in blocks alone on their compute units: two halves of a
// block's keys side by side. With / without, us: 3000, 8 heads and 1 46 / 51; 4000, 4 and 1 57 / 65, at head_dim 64 42 / 52;
// 1000, 16 and 2 23 / 23, at head_dim 64 17 / 18; four of 300, 8 and 2 15 / 12.
constexpr int64_t kAloneTokens = 2048;
// CTAs of 16 rows, four waves each, that run at once (head_dim 64: as many as its registers allow; 128: two a compute unit, and
// some more of ragged requests): up to here their chains are shorter than a block's. Against blocks, us, head_dim 64: seven
// prompts of 1 to 300, 8 and 2 heads 6.4 / 9.1; four of 300 8.0 / 10.0; one of 1000, 16 and 2 (1000 CTAs) 16 / 18; eight of
// 300, 8 and 2 (1200) 11 / 10; 128: nine of 1 to 300, 8 and 2 (550) 10 / 12; 600, 16 and 4 (600) 15 / 16; sixteen of 100
// (800) 10.1 / 9.4. Paged, up to 512 keys: sixteen chunks of 20 on 400, 32 and 8 heads of 64, 11.1 / 12.6; twenty of 30 and
// 10 on 200 9.4 / 10.9, on 900 21 / 20.
constexpr int64_t kAtOnce64 = 1024;
constexpr int64_t kAtOnce128 = 600;
// Requests of more than 16 rows are streamed in pieces up to this many CTAs of 16 rows times keys.
constexpr int64_t kFewWork = 1 << 18;

// Blocks of 256 rows (head_dim 128): they read keys once for twice the rows, but start and end alone on their compute
// unit. 256 / 128 rows: prompts of 8k tokens, 64 and 8 heads 1797 / 1894 us; one of 4096, 32 heads 149 / 156; four of 2048
// 330 / 325; six of 250 to 1900, 32 heads 85 / 82; 64 of 100 55 / 46; four chunks of 2048 on up to 8k tokens 1190 / 1264;
// one prompt of 8192, 8 and 1 heads (256 wide blocks) 191 / 173. avg: tokens of an average request; keys: of the longest,
// by what the host knows.
bool wide_blocks(int dim, int64_t blocks, int64_t avg, int64_t keys) {
  return dim == 128 && blocks >= kBlocksEnough && avg >= 1024 && keys >= 2560;
}

// batch, total_q, most: requests, their queries, the most rows (queries times group) of one; keys: the most keys of one
// (paged), or 0: packed prompts.
//
// Where 16- or 32-row CTAs of eight waves are no more than the compute units, each takes a request's keys in one piece:
// their waves share the keys, so that a lone CTA's chain is short. 16 / 32 rows / blocks, us, head_dim 128 unless said:
// prompts of 2000, 2 and 2 heads 20 / 25 / 36; 4000, 2 and 1 51 / 43 / 63; four of 300, 8 and 2 (304 CTAs of 32 rows) 16 /
// 17 / 12; four chunks of 64 on 900, 8 heads and 1 15 / 19 / 23, on 2000 24 / 29 / 25, 32 and 8 heads 27 / 19 / 24. Against
// cut keys: 8 CTAs on 600 keys 10 / 11, on 1000 13 / 11; 128 on 1000 19 / 19; 256 on 1000 25 / 31, on 3000 67 / 73; at
// head_dim 64 8 on 1000 9.1 / 9.4, 128 on 2000 21 / 20. With more CTAs, one token a request, 8 KV heads: 40 requests of up
// to 1600 45 / 46, 64 56 / 63, 256 186 / 202; 40 of up to 3000 75 / 67, 256 327 / 333.
// Few rows on longer keys are cut in CTAs of 16 rows: a chunk of 100 on 2000, 8 heads and 1, 17 in blocks 21; on 4000 20,
// 22; on 8000 26, 24. Else up to 32 rows are streamed, bound by reading K and V: 64 chunks of 8 on 1k to 8k, 32 and 8
// heads, 256, in blocks 277; with 64 and 8 heads (64 rows) 432, 297.
Choice choose(int dim, int32_t batch, int64_t total_q, int32_t group, int32_t kv_heads, int64_t most, int64_t keys) {
  auto ctas = [&](int rows) { return std::max<int64_t>((total_q * group + rows - 1) / rows, batch) * kv_heads; };
  auto one_piece = [&](int64_t n) { return 2 * n <= kFit && (keys == 0 || keys * dim <= (512 + 4 * n) * 128); };
  for (int rows : {16, 32}) {
    if (one_piece(ctas(rows))) return {rows, 0, false, true};
    if (most <= rows) break;
  }
  const int64_t blocks = (total_q * group + kBlock - 1) / kBlock * kv_heads;
  const int64_t avg = total_q / batch;
  const bool at_once = ctas(16) <= (dim == 64 ? kAtOnce64 : kAtOnce128);
  if (keys == 0) {
    if (wide_blocks(dim, blocks, avg, avg)) return {2 * kBlock, 0, false, false};
    const bool halves = 2 * ctas(kBlock) <= kFit && avg * 128 >= kAloneTokens * dim;
    return at_once && !halves ? Choice{16, 0, false, false} : Choice{kBlock, 0, false, halves};
  }
  if (most > 32 && keys <= 512 && at_once) return {16, 0, false, false};
  if (most > 16 && 2 * ctas(16) <= kFit && ctas(16) * keys <= kFewWork) return {16, kFit, true, false};
  if (most <= 32) {
    const int rows = most <= 16 ? 16 : 32;
    if (2 * ctas(rows) <= kFit) return {rows, kFit, true, false};
    return {rows, keys <= kOnePieceMany ? 0 : kTarget, false, false};
  }
  if (blocks >= kBlocksEnough || keys <= kOnePieceBlocks) return {wide_blocks(dim, blocks, avg, keys) ? 2 * kBlock : kBlock, 0, false, false};
  return {kBlock, kBlocksTarget, false, false};
}

// Rows of partial results: 2 target pieces of any choice for requests of up to `most` rows.
int64_t workspace_rows(int64_t most) {
  static_assert(2 * kTarget * 32 >= 2 * kBlocksTarget * kBlock && 2 * kTarget * 32 >= 2 * kFit * 16, "32 rows streamed need the most");
  static_assert(2 * kTarget * 16 >= 2 * kFit * 16, "and 16 rows");
  return 2 * (int64_t)kTarget * (most <= 16 ? 16 : 32);
}

int check_heads(const char* who, int32_t q_heads, int32_t kv_heads, int32_t dim) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: %d query heads are no multiple of %d KV heads", who, q_heads, kv_heads);
  if (q_heads > 4096) return api_error(MLA_ERR_UNSUPPORTED, "%s: at most 4096 query heads, got %d", who, q_heads);
  if (dim != 64 && dim != 128) return api_error(MLA_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128, got %d", who, dim);
  return MLA_OK;
}

// What all three attention entry points check; fills p but for the keys' addressing.
int attention_params(const char* who, GqaParams& p, const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                     int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                     int64_t v_head_stride, int32_t batch, int32_t total_q, int32_t q_heads, int32_t kv_heads,
                     int32_t dim, float scale, void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
                     int64_t lse_stride_t) {
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr)
    return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 8))
    return api_error(MLA_ERR_INVALID_ARG, "%s: q, k and v must be 16-byte and out 8-byte aligned", who);
  if (k_row_stride > 0x7fffffff || v_row_stride > 0x7fffffff)
    return api_error(MLA_ERR_UNSUPPORTED, "%s: k and v rows lie more than 4 GiB apart", who);
  if (q_stride_t % 8 || q_stride_h % 8 || q_stride_t < 0 || q_stride_h < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: q strides (%lld, %lld) must be non-negative multiples of 8", who,
                     (long long)q_stride_t, (long long)q_stride_h);
  if (k_row_stride % 8 || k_head_stride % 8 || v_row_stride % 8 || v_head_stride % 8 || k_row_stride < 0 ||
      k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: k and v strides must be non-negative multiples of 8", who);
  // rows of out must not overlap, tokens outside heads or heads outside tokens
  const bool by_token = (q_heads == 1 || out_stride_h >= dim) && (total_q == 1 || out_stride_t >= (q_heads - 1) * out_stride_h + dim);
  const bool by_head = (total_q == 1 || out_stride_t >= dim) && (q_heads == 1 || out_stride_h >= (total_q - 1) * out_stride_t + dim);
  if (out_stride_t % 4 || out_stride_h % 4 || out_stride_t < 0 || out_stride_h < 0 || !(by_token || by_head))
    return api_error(MLA_ERR_INVALID_ARG, "%s: out strides (%lld, %lld) must be multiples of 4 and hold %d tokens of %d heads of %d",
                     who, (long long)out_stride_t, (long long)out_stride_h, total_q, q_heads, dim);
  if (lse != nullptr && total_q > 1 && lse_stride_t < q_heads)
    return api_error(MLA_ERR_INVALID_ARG, "%s: lse_stride_t %lld < %d heads", who, (long long)lse_stride_t, q_heads);
  if (!(scale > 0.f) || !isfinite(scale)) return api_error(MLA_ERR_INVALID_ARG, "%s: bad scale", who);
  if (batch > 65535) return api_error(MLA_ERR_UNSUPPORTED, "%s: at most 65535 requests, got %d", who, batch);
  if ((int64_t)total_q * q_heads > 0x7fffffff) return api_error(MLA_ERR_UNSUPPORTED, "%s: total_q * q_heads passes 2^31", who);
  p.q = static_cast<const __bf16*>(q);
  p.q_stride_t = q_stride_t;
  p.q_stride_h = q_stride_h;
  p.k = static_cast<const __bf16*>(k);
  p.k_row_stride = k_row_stride;
  p.k_head_stride = k_head_stride;
  p.v = static_cast<const __bf16*>(v);
  p.v_row_stride = v_row_stride;
  p.v_head_stride = v_head_stride;
  p.batch = batch;
  p.total_q = total_q;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<__bf16*>(out);
  p.out_stride_t = out_stride_t;
  p.out_stride_h = out_stride_h;
  p.out_16b = aligned(out, 16) && out_stride_t % 8 == 0 && out_stride_h % 8 == 0;
  p.lse = lse;
  p.lse_stride_t = lse_stride_t;
  return MLA_OK;
}

int launch(const char* who, GqaParams& p, const Choice& c, int dim, void* stream) {
  p.target = c.target;
  for (p.log2_target = 0; (1 << p.log2_target) < c.target;) ++p.log2_target;
  p.fit = c.fit;
  p.wide = c.wide;
  if (!gqa_grids_ok(p, c.rows))
    return api_error(MLA_ERR_UNSUPPORTED, "%s: %d rows of %d heads are more than a launch holds", who, p.total_q, p.kv_heads * p.group);
  return done(c.rows >= kBlock ? launch_gqa_rows(p, dim, c.rows, (hipStream_t)stream) : launch_gqa_stream(p, dim, c.rows, (hipStream_t)stream), who);
}

int paged(const char* who, const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_pool,
          int64_t k_row_stride, int64_t k_head_stride, const void* v_pool, int64_t v_row_stride, int64_t v_head_stride,
          int32_t num_pages, int32_t page_size, const int32_t* page_table, int32_t pt_cols, int64_t pt_stride,
          const int32_t* cu_seqlens_q, const int32_t* seq_lens_k, int32_t batch, int32_t total_q, int32_t max_q,
          int32_t q_heads, int32_t kv_heads, int32_t dim, float scale, void* workspace, int64_t workspace_bytes,
          void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse, int64_t lse_stride_t, void* stream) {
  if (batch < 0 || total_q < 0 || max_q < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: batch %d, total_q %d, max_q %d", who, batch, total_q, max_q);
  if (int rc = check_heads(who, q_heads, kv_heads, dim)) return rc;
  if (batch == 0 || total_q == 0 || max_q == 0) return done(hipSuccess, who);
  if (page_table == nullptr || seq_lens_k == nullptr || (workspace == nullptr && workspace_bytes != 0))
    return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!is_pow2(page_size)) return api_error(MLA_ERR_UNSUPPORTED, "%s: page_size %d must be a power of two", who, page_size);
  if (num_pages < 1 || pt_cols < 1 || (batch > 1 && pt_stride < pt_cols))
    return api_error(MLA_ERR_INVALID_ARG, "%s: num_pages %d, pt_cols %d, pt_stride %lld", who, num_pages, pt_cols, (long long)pt_stride);
  if ((int64_t)num_pages * page_size > 0x7fffffff)
    return api_error(MLA_ERR_UNSUPPORTED, "%s: a pool of %d pages of %d passes 2^31 rows", who, num_pages, page_size);
  GqaParams p = {};
  if (int rc = attention_params(who, p, q, q_stride_t, q_stride_h, k_pool, k_row_stride, k_head_stride, v_pool,
                                v_row_stride, v_head_stride, batch, total_q, q_heads, kv_heads, dim, scale, out,
                                out_stride_t, out_stride_h, lse, lse_stride_t))
    return rc;
  const int64_t most = (int64_t)max_q * p.group;  // rows of a request and KV head
  const int64_t need = 4 * workspace_rows(most) * (dim + 2);
  const int64_t keys = (int64_t)pt_cols * page_size;
  // a piece's end, its length rounded up to 64 keys in each of the pieces before it, stays below 2^31
  p.max_keys = (int32_t)(keys < 0x7ff00000 ? keys : 0x7ff00000);
  const Choice choice = choose(dim, batch, total_q, p.group, kv_heads, most, p.max_keys);
  if (!aligned(workspace, 16) || (workspace_bytes < need && (workspace != nullptr || choice.target > 0)))
    return api_error(MLA_ERR_INVALID_ARG, "%s: the workspace must be 16-byte aligned and hold %lld bytes, got %lld", who,
                     (long long)need, (long long)workspace_bytes);
  p.num_pages = num_pages;
  for (p.log2_ps = 0; (1 << p.log2_ps) < page_size;) ++p.log2_ps;
  p.page_table = page_table;
  p.pt_stride = pt_stride;
  p.cu_seqlens_q = cu_seqlens_q;
  p.seq_lens_k = seq_lens_k;
  p.max_q = max_q;
  if (workspace != nullptr) {
    p.ws_o = static_cast<float*>(workspace);
    p.ws_lse = reinterpret_cast<f32x2*>(p.ws_o + workspace_rows(most) * dim);
  }
  return launch(who, p, choice, dim, stream);
}

}  // namespace
}  // namespace mla

extern "C" {

int mla_gqa_workspace_bytes(int32_t max_q, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int64_t* bytes) {
  const char* who = "mla_gqa_workspace_bytes";
  if (bytes == nullptr || max_q < 0) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: bytes is null or max_q %d < 0", who, max_q);
  if (int rc = mla::check_heads(who, q_heads, kv_heads, head_dim)) return rc;
  *bytes = 4 * mla::workspace_rows((int64_t)max_q * (q_heads / kv_heads)) * (head_dim + 2);
  return mla::done(hipSuccess, who);
}

int mla_gqa_prompt_bf16(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_row_stride,
                        int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride,
                        const int32_t* cu_seqlens, int32_t batch, int32_t total_q, int32_t q_heads, int32_t kv_heads,
                        int32_t head_dim, float scale, void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
                        int64_t lse_stride_t, void* stream) {
  const char* who = "mla_gqa_prompt_bf16";
  if (batch < 0 || total_q < 0) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: batch %d, total_q %d", who, batch, total_q);
  if (int rc = mla::check_heads(who, q_heads, kv_heads, head_dim)) return rc;
  if (batch == 0 || total_q == 0) return mla::done(hipSuccess, who);
  if (cu_seqlens == nullptr) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  mla::GqaParams p = {};
  if (int rc = mla::attention_params(who, p, q, q_stride_t, q_stride_h, k, k_row_stride, k_head_stride, v, v_row_stride,
                                     v_head_stride, batch, total_q, q_heads, kv_heads, head_dim, scale, out,
                                     out_stride_t, out_stride_h, lse, lse_stride_t))
    return rc;
  p.max_keys = total_q;
  p.cu_seqlens_q = cu_seqlens;
  p.max_q = total_q;
  return mla::launch(who, p, mla::choose(head_dim, batch, total_q, p.group, kv_heads, (int64_t)total_q * p.group, 0), head_dim, stream);
}

int mla_gqa_chunk_bf16(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_pool, int64_t k_row_stride,
                       int64_t k_head_stride, const void* v_pool, int64_t v_row_stride, int64_t v_head_stride,
                       int32_t num_pages, int32_t page_size, const int32_t* page_table, int32_t pt_cols,
                       int64_t pt_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens_k, int32_t batch,
                       int32_t total_q, int32_t max_q, int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale,
                       void* workspace, int64_t workspace_bytes, void* out, int64_t out_stride_t, int64_t out_stride_h,
                       float* lse, int64_t lse_stride_t, void* stream) {
  const char* who = "mla_gqa_chunk_bf16";
  if (batch > 0 && total_q > 0 && max_q > 0 && cu_seqlens_q == nullptr)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  return mla::paged(who, q, q_stride_t, q_stride_h, k_pool, k_row_stride, k_head_stride, v_pool, v_row_stride,
                    v_head_stride, num_pages, page_size, page_table, pt_cols, pt_stride, cu_seqlens_q, seq_lens_k, batch,
                    total_q, max_q < total_q ? max_q : total_q, q_heads, kv_heads, head_dim, scale, workspace,
                    workspace_bytes, out, out_stride_t, out_stride_h, lse, lse_stride_t, stream);
}

int mla_gqa_decode_bf16(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_pool, int64_t k_row_stride,
                        int64_t k_head_stride, const void* v_pool, int64_t v_row_stride, int64_t v_head_stride,
                        int32_t num_pages, int32_t page_size, const int32_t* page_table, int32_t pt_cols,
                        int64_t pt_stride, const int32_t* seq_lens, int32_t batch, int32_t q_heads, int32_t kv_heads,
                        int32_t head_dim, float scale, void* workspace, int64_t workspace_bytes, void* out,
                        int64_t out_stride_b, int64_t out_stride_h, float* lse, int64_t lse_stride_b, void* stream) {
  return mla::paged("mla_gqa_decode_bf16", q, q_stride_b, q_stride_h, k_pool, k_row_stride, k_head_stride, v_pool,
                    v_row_stride, v_head_stride, num_pages, page_size, page_table, pt_cols, pt_stride, nullptr, seq_lens,
                    batch, batch, 1, q_heads, kv_heads, head_dim, scale, workspace, workspace_bytes, out, out_stride_b,
                    out_stride_h, lse, lse_stride_b, stream);
}

int mla_page_tables_from_lengths(int32_t* token_table, int32_t token_table_rows, int32_t token_table_cols,
                                 int64_t token_table_stride, const int32_t* table_idx, const int32_t* cached_lens,
                                 const int32_t* device_lens, int32_t batch, int32_t alloc_reqs,
                                 const int32_t* free_slots, int32_t num_free, int32_t page_size, int32_t max_extend,
                                 int32_t* page_table, int32_t pt_cols, int64_t pt_stride, int32_t* out_loc,
                                 int32_t* positions, int32_t total_new, int32_t* cu_seqlens_q, int32_t* pages_taken,
                                 void* stream) {
  const char* who = "mla_page_tables_from_lengths";
  if (batch < 1 || batch > 65535 || alloc_reqs < 0 || alloc_reqs > batch || num_free < 0 || max_extend < 0 || total_new < 0 || pt_cols < 0)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: batch %d (1 to 65535), alloc_reqs %d, num_free %d, max_extend %d, total_new %d, pt_cols %d",
                          who, batch, alloc_reqs, num_free, max_extend, total_new, pt_cols);
  if (page_size < 1 || page_size > (1 << 20)) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: page_size %d must be in [1, 2^20]", who, page_size);
  if (token_table == nullptr || table_idx == nullptr || cached_lens == nullptr || device_lens == nullptr ||
      cu_seqlens_q == nullptr || pages_taken == nullptr || (num_free > 0 && free_slots == nullptr) ||
      (pt_cols > 0 && page_table == nullptr) || (total_new > 0 && (out_loc == nullptr || positions == nullptr)))
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (token_table_rows < 1 || token_table_cols < 1 || token_table_cols > (1 << 30) || token_table_stride < token_table_cols)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: token table of %d x %d, stride %lld", who, token_table_rows,
                          token_table_cols, (long long)token_table_stride);
  if (batch > 1 && pt_stride < pt_cols)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: pt_stride %lld < %d columns", who, (long long)pt_stride, pt_cols);
  mla::PageTablesParams p;
  p.token_table = token_table;
  p.tt_rows = token_table_rows;
  p.tt_cols = token_table_cols;
  p.tt_stride = token_table_stride;
  p.table_idx = table_idx;
  p.cached_lens = cached_lens;
  p.device_lens = device_lens;
  p.batch = batch;
  p.alloc_reqs = alloc_reqs;
  p.free_slots = free_slots;
  p.num_free = num_free;
  p.page_size = page_size;
  p.log2_ps = -1;
  if (mla::is_pow2(page_size)) for (p.log2_ps = 0; (1 << p.log2_ps) < page_size;) ++p.log2_ps;
  p.page_table = page_table;
  p.pt_cols = pt_cols;
  p.pt_stride = pt_stride;
  p.out_loc = out_loc;
  p.positions = positions;
  p.total_new = total_new;
  p.cu_seqlens_q = cu_seqlens_q;
  p.pages_taken = pages_taken;
  return mla::done(mla::launch_page_tables(p, max_extend, (hipStream_t)stream), who);
}

}  // extern "C"
