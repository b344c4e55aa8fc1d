// extern "C" entry points of the grouped-head attention and of the step's tables (declared in include/mla_amd.h):
// argument checks, the choice of kernel, and launches.
#include <math.h>

#include <algorithm>

#include "mla_gqa.h"
#include "mla_gqa_mx4.h"

namespace mla {
namespace {

int done(hipError_t e, const char* who) {
  if (e != hipSuccess) return api_error(MLA_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
  api_error(MLA_OK, "%s", "");
  return MLA_OK;
}
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool is_pow2(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }
Mx4View mx4_view(const mla_mx4_pool& x) {
  return {static_cast<uint8_t*>(x.codes), static_cast<uint8_t*>(x.scales), x.code_stride_page, x.code_stride_token, x.code_stride_head,
          x.scale_stride_page, x.scale_stride_token, x.scale_stride_head};
}

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
// Of a cache of 4 bits joining costs more than reading. One piece / cut, us, of 4 heads a KV head, up to n keys (an eighth at
// least), head_dim 128: 320 CTAs of 16 rows 1600 21.6 / 25.5, 2400 30 / 28; 512 2400 32 / 37, 3200 40 / 44, 6000 70 / 67; 1024
// 3200 65 / 71, 6000 113 / 113; 2048 3200 112 / 129; 320 of 32 rows 1600 27 / 49, 3200 46 / 63, 6000 80 / 91; 512 2400 44 / 74,
// 6000 85 / 118; 1024 2400 90 / 119, 6000 200 / 212. Few long requests among many short ones would wait for the longest: not
// past 3200 and 6144.
int64_t one_piece_mx4(int rows, int64_t ctas) { return rows == 16 ? std::min<int64_t>(6 * ctas, 3200) : std::min<int64_t>(12 * ctas, 6144); }
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
//
// A cache of 4 bits costs instructions, as many at head_dim 64 as at 128, rather than bytes. One piece / cut, us, requests of
// one token of up to n keys (an eighth of it at least), head_dim 128: 8 CTAs 700 6.0 / 9.3, 1000 10.4 / 9.6; 32 900 8.9 / 9.9,
// 1200 10.8 / 9.9; 64 1200 10.4 / 11.9, 2000 12.9 / 13.0, 3000 20 / 15; 128 2000 15.6 / 16.4, 3000 20.5 / 19.8; 256 2000 17 / 21,
// 3000 23 / 29; 64: 8 1000 8.9 / 8.8; 32 1200 9.2 / 9.1; 128 2000 13.6 / 14.4, 3000 17.7 / 16.9; 256 3000 19 / 25.
// Four waves have a tile each by 128 keys, eight by 256: up to 200 keys 8 CTAs 4.8 / 5.0, 256 6.1 / 6.3, up to 400 5.5 / 5.8, 8.5 / 7.4.
// More than 16 rows, more CTAs than compute units: 16 rows of four waves / 32 of eight, 24 requests of 8 to 48 rows, 8 KV heads,
// up to 100 6.8 / 13.9, 500 10.6 / 16.1, 1000 16.2 / 17.7; at head_dim 64 5.9 / 11.4, 9.1 / 12.9, 13.7 / 14.5.
// More CTAs of 16 rows than run at once, 16 / 32 rows of four waves: 64 requests, up to 250 14.2 / 17.3, 750 25.9 / 24.6; 128, up to 250
// 24.8 / 27.2; requests of 64 rows, which fill 32: 200 of 4 KV heads on 190 42 / 38, at head_dim 64 30 / 25.
Choice choose(int dim, int32_t batch, int64_t total_q, int32_t group, int32_t kv_heads, int64_t most, int64_t keys, bool mx4 = false) {
  auto ctas = [&](int rows) { return std::max<int64_t>((total_q * group + rows - 1) / rows, batch) * kv_heads; };
  auto one_piece = [&](int64_t n) { return 2 * n <= kFit && (keys == 0 || (mx4 ? keys <= 850 + 10 * n : keys * dim <= (512 + 4 * n) * 128)); };
  const bool at_once = ctas(16) <= (dim == 64 ? kAtOnce64 : kAtOnce128);
  for (int rows : {16, 32}) {
    if (one_piece(ctas(rows))) return {rows, 0, false, !mx4 || keys > 256};
    if (most <= rows) break;
    if (mx4 && (at_once ? keys <= 1000 : keys <= 256 && total_q * group <= 32 * (int64_t)batch)) return {16, 0, false, false};
  }
  const int64_t blocks = (total_q * group + kBlock - 1) / kBlock * kv_heads;
  const int64_t avg = total_q / batch;
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
    return {rows, keys <= (mx4 ? one_piece_mx4(rows, ctas(rows)) : kOnePieceMany) ? 0 : kTarget, false, false};
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

// Whether rows of `width` elements do not overlap: `outer` of them outer_stride apart, each of `inner` inner_stride apart, in
// either order.
bool rows_apart(int64_t outer, int64_t outer_stride, int64_t inner, int64_t inner_stride, int64_t width) {
  const bool by_outer = (inner <= 1 || inner_stride >= width) && (outer <= 1 || outer_stride >= (inner - 1) * inner_stride + width);
  const bool by_inner = (outer <= 1 || outer_stride >= width) && (inner <= 1 || inner_stride >= (outer - 1) * outer_stride + width);
  return by_outer || by_inner;
}

// The same of a pool's rows, by dimensions of n and a stride each in any order: each lies outside all that those of smaller strides hold.
struct Steps {
  int64_t n, stride;
};
bool rows_apart(Steps a, Steps b, Steps c, int64_t width) {
  Steps x[] = {a, b, c};
  std::sort(x, x + 3, [](const Steps& p, const Steps& q) { return p.stride < q.stride; });
  __int128 held = width;
  for (const Steps& s : x) {
    if (s.n <= 1) continue;
    if (s.stride < held) return false;
    held += (__int128)(s.n - 1) * s.stride;
  }
  return true;
}

int check_heads(const char* who, int32_t q_heads, int32_t kv_heads, int32_t dim) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: %d query heads are no multiple of %d KV heads", who, q_heads, kv_heads);
  if (q_heads > 4096) return api_error(MLA_ERR_UNSUPPORTED, "%s: at most 4096 query heads, got %d", who, q_heads);
  if (dim != 64 && dim != 128) return api_error(MLA_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128, got %d", who, dim);
  return MLA_OK;
}

// What all attention entry points check of everything but keys and values.
int query_params(const char* who, GqaParams& p, const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t batch,
                 int32_t total_q, int32_t q_heads, int32_t kv_heads, int32_t dim, float scale, void* out,
                 int64_t out_stride_t, int64_t out_stride_h, float* lse, int64_t lse_stride_t) {
  if (q == nullptr || out == nullptr) return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!aligned(q, 16) || !aligned(out, 8)) return api_error(MLA_ERR_INVALID_ARG, "%s: q must be 16-byte and out 8-byte aligned", who);
  if (q_stride_t % 8 || q_stride_h % 8 || q_stride_t < 0 || q_stride_h < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: q strides (%lld, %lld) must be non-negative multiples of 8", who,
                     (long long)q_stride_t, (long long)q_stride_h);
  if (out_stride_t % 4 || out_stride_h % 4 || out_stride_t < 0 || out_stride_h < 0 ||
      !rows_apart(total_q, out_stride_t, q_heads, out_stride_h, dim))
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

// What the entry points over bf16 keys and values check; fills p but for the keys' addressing.
int attention_params(const char* who, GqaParams& p, const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                     int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                     int64_t v_head_stride, int32_t batch, int32_t total_q, int32_t q_heads, int32_t kv_heads,
                     int32_t dim, float scale, void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
                     int64_t lse_stride_t) {
  if (k == nullptr || v == nullptr) return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16)) return api_error(MLA_ERR_INVALID_ARG, "%s: k and v must be 16-byte aligned", who);
  if (k_row_stride > 0x7fffffff || v_row_stride > 0x7fffffff)
    return api_error(MLA_ERR_UNSUPPORTED, "%s: k and v rows lie more than 4 GiB apart", who);
  if (k_row_stride % 8 || k_head_stride % 8 || v_row_stride % 8 || v_head_stride % 8 || k_row_stride < 0 ||
      k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: k and v strides must be non-negative multiples of 8", who);
  p.k = static_cast<const __bf16*>(k);
  p.k_row_stride = k_row_stride;
  p.k_head_stride = k_head_stride;
  p.v = static_cast<const __bf16*>(v);
  p.v_row_stride = v_row_stride;
  p.v_head_stride = v_head_stride;
  return query_params(who, p, q, q_stride_t, q_stride_h, batch, total_q, q_heads, kv_heads, dim, scale, out, out_stride_t,
                      out_stride_h, lse, lse_stride_t);
}

int set_choice(const char* who, GqaParams& p, const Choice& c) {
  p.target = c.target;
  for (p.log2_target = 0; (1 << p.log2_target) < c.target;) ++p.log2_target;
  p.fit = c.fit;
  p.wide = c.wide;
  if (!gqa_grids_ok(p, c.rows))
    return api_error(MLA_ERR_UNSUPPORTED, "%s: %d rows of %d heads are more than a launch holds", who, p.total_q, p.kv_heads * p.group);
  return MLA_OK;
}

int launch(const char* who, GqaParams& p, const Choice& c, int dim, void* stream) {
  if (int rc = set_choice(who, p, c)) return rc;
  return done(c.rows >= kBlock ? launch_gqa_rows(p, dim, c.rows, (hipStream_t)stream) : launch_gqa_stream(p, dim, c.rows, (hipStream_t)stream), who);
}

int check_pages(const char* who, int32_t num_pages, int32_t page_size, const int32_t* page_table, int32_t pt_cols,
                int64_t pt_stride, const int32_t* seq_lens_k, int32_t batch, const void* workspace, int64_t workspace_bytes) {
  if (page_table == nullptr || seq_lens_k == nullptr || (workspace == nullptr && workspace_bytes != 0))
    return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!is_pow2(page_size)) return api_error(MLA_ERR_UNSUPPORTED, "%s: page_size %d must be a power of two", who, page_size);
  if (num_pages < 1 || pt_cols < 1 || (batch > 1 && pt_stride < pt_cols))
    return api_error(MLA_ERR_INVALID_ARG, "%s: num_pages %d, pt_cols %d, pt_stride %lld", who, num_pages, pt_cols, (long long)pt_stride);
  if ((int64_t)num_pages * page_size > 0x7fffffff)
    return api_error(MLA_ERR_UNSUPPORTED, "%s: a pool of %d pages of %d passes 2^31 rows", who, num_pages, page_size);
  return MLA_OK;
}

// The keys' addressing but for the pool's pointers.
void set_pages(GqaParams& p, int32_t num_pages, int32_t page_size, const int32_t* page_table, int64_t pt_stride,
               const int32_t* cu_seqlens_q, const int32_t* seq_lens_k, int32_t max_q) {
  p.num_pages = num_pages;
  for (p.log2_ps = 0; (1 << p.log2_ps) < page_size;) ++p.log2_ps;
  p.page_table = page_table;
  p.pt_stride = pt_stride;
  p.cu_seqlens_q = cu_seqlens_q;
  p.seq_lens_k = seq_lens_k;
  p.max_q = max_q;
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
  if (int rc = check_pages(who, num_pages, page_size, page_table, pt_cols, pt_stride, seq_lens_k, batch, workspace, workspace_bytes)) return rc;
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
  set_pages(p, num_pages, page_size, page_table, pt_stride, cu_seqlens_q, seq_lens_k, max_q);
  if (workspace != nullptr) {
    p.ws_o = static_cast<float*>(workspace);
    p.ws_lse = reinterpret_cast<f32x2*>(p.ws_o + workspace_rows(most) * dim);
  }
  return launch(who, p, choice, dim, stream);
}

// ---- over a cache of 4 bits

// Requests of up to this many rows are streamed from the codes, never laid out.
constexpr int64_t kStreamRows = 512;
// Bytes of a workspace: partial results (`split`), and for calls with requests of more rows, which may have them laid out, their keys'
// values in pages of 64 and the page table of these.
struct Mx4Space {
  int64_t split, table, rows, cols, bytes;
};
Mx4Space mx4_space(int64_t most, int32_t kv_heads, int32_t dim, int32_t batch, int64_t max_keys, int64_t total_keys) {
  Mx4Space s = {};
  s.split = 4 * workspace_rows(most) * (dim + 2);
  if (most > kStreamRows) {
    s.cols = (max_keys + 63) / 64;
    s.rows = std::min<int64_t>(64 * std::min(total_keys / 64 + batch, batch * s.cols), int64_t{1} << 31);  // (more are refused)
    s.table = (4 * batch * s.cols + 15) / 16 * 16;
  }
  s.bytes = s.split + s.table + 2 * s.rows * kv_heads * dim * 2;
  return s;
}

int check_mx4(const char* who, const Mx4View& k, const Mx4View& v, int32_t dim, int64_t num_pages, int64_t page_size, int32_t kv_heads) {
  if (k.codes == nullptr || k.scales == nullptr || v.codes == nullptr || v.scales == nullptr)
    return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!is_pow2(page_size)) return api_error(MLA_ERR_UNSUPPORTED, "%s: page_size %lld must be a power of two", who, (long long)page_size);
  if (num_pages < 1 || kv_heads < 1) return api_error(MLA_ERR_INVALID_ARG, "%s: num_pages %lld, kv_heads %d", who, (long long)num_pages, kv_heads);
  if (num_pages * page_size > 0x7fffffff)
    return api_error(MLA_ERR_UNSUPPORTED, "%s: a pool of %lld pages of %lld passes 2^31 rows", who, (long long)num_pages, (long long)page_size);
  const int64_t scale_row = dim / 32;
  if (!aligned(k.codes, 16) || !aligned(v.codes, 16) || !aligned(k.scales, scale_row) || !aligned(v.scales, scale_row))
    return api_error(MLA_ERR_INVALID_ARG, "%s: codes must be 16-byte aligned, scales by a row's %d bytes", who, dim / 32);
  for (const Mx4View* x : {&k, &v})
    if (x->c_page % 16 || x->c_tok % 16 || x->c_head % 16 || x->s_page % scale_row || x->s_tok % scale_row || x->s_head % scale_row ||
        x->c_page < 0 || x->c_tok < 0 || x->c_head < 0 || x->s_page < 0 || x->s_tok < 0 || x->s_head < 0)
      return api_error(MLA_ERR_INVALID_ARG, "%s: strides must be non-negative multiples of 16 bytes (codes) and of a row (scales)", who);
    else if (x->c_tok > (1 << 24) || x->s_tok > (1 << 24))
      return api_error(MLA_ERR_UNSUPPORTED, "%s: tokens lie more than 16 MiB apart", who);
    else if ((num_pages > 1 && (x->c_page < dim / 2 || x->s_page < scale_row)) || (page_size > 1 && (x->c_tok < dim / 2 || x->s_tok < scale_row)) ||
             (kv_heads > 1 && (x->c_head < dim / 2 || x->s_head < scale_row)))
      return api_error(MLA_ERR_INVALID_ARG, "%s: rows of a pool lie over one another: strides below a row", who);
  return MLA_OK;
}

int paged_mx4(const char* who, const void* q, int64_t q_stride_t, int64_t q_stride_h, const mla_mx4_pool* k_pool,
              const mla_mx4_pool* v_pool, int32_t num_pages, int32_t page_size, const int32_t* page_table, int32_t pt_cols,
              int64_t pt_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens_k, int32_t batch, int32_t total_q,
              int32_t max_q, int64_t total_keys, int32_t q_heads, int32_t kv_heads, int32_t dim, float scale, void* workspace,
              int64_t workspace_bytes, void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
              int64_t lse_stride_t, void* stream) {
  if (batch < 0 || total_q < 0 || max_q < 0 || total_keys < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: batch %d, total_q %d, max_q %d, total_keys %lld", who, batch, total_q, max_q, (long long)total_keys);
  if (int rc = check_heads(who, q_heads, kv_heads, dim)) return rc;
  if (batch == 0 || total_q == 0 || max_q == 0) return done(hipSuccess, who);
  if (k_pool == nullptr || v_pool == nullptr) return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  if (int rc = check_pages(who, num_pages, page_size, page_table, pt_cols, pt_stride, seq_lens_k, batch, workspace, workspace_bytes)) return rc;
  const Mx4View k = mx4_view(*k_pool), v = mx4_view(*v_pool);
  if (int rc = check_mx4(who, k, v, dim, num_pages, page_size, kv_heads)) return rc;
  if (k.c_page != v.c_page || k.c_tok != v.c_tok || k.c_head != v.c_head || k.s_page != v.s_page || k.s_tok != v.s_tok || k.s_head != v.s_head)
    return api_error(MLA_ERR_INVALID_ARG, "%s: the pools of keys and values must have the same strides", who);
  GqaMx4Params mp = {};
  GqaParams& p = mp.g;
  if (int rc = query_params(who, p, q, q_stride_t, q_stride_h, batch, total_q, q_heads, kv_heads, dim, scale, out, out_stride_t,
                            out_stride_h, lse, lse_stride_t))
    return rc;
  mp.k_codes = k.codes;
  mp.k_scales = k.scales;
  mp.v_codes = v.codes;
  mp.v_scales = v.scales;
  mp.c_page = k.c_page, mp.c_tok = k.c_tok, mp.c_head = k.c_head;
  mp.s_page = k.s_page, mp.s_tok = k.s_tok, mp.s_head = k.s_head;
  const int64_t most = (int64_t)max_q * p.group, keys = (int64_t)pt_cols * page_size;
  p.max_keys = (int32_t)(keys < 0x7ff00000 ? keys : 0x7ff00000);
  Choice choice = choose(dim, batch, total_q, p.group, kv_heads, most, p.max_keys, true);
  // Blocks read values that are laid out first, 512 bytes for every 136 of the cache: worth it where many rows read them. 32-row
  // CTAs / laid out, us, 64 and 8 heads of 128: six chunks of 32 on 8000 109 / 147, of 64 181 / 207, of 96 254 / 270, of 128 329 /
  // 288; four of 64 on 2000 64 / 54, on 500 15 / 28; 32 and 8 heads of 64, of 64 on 2000 16 / 16, of 128 51 / 48.
  // Where blocks are too few to fill the chip, more rows as well. 32-row CTAs / laid out, 512 CTAs, on 500, 2000, 4000, 6000 keys: a
  // chunk of 256, 64 and 8 heads 19 / 25, 41 / 52, 70 / 66, 128 / 82; of 1000, 16 and 2 24 / 43, 43 / 56, 68 / 72, 142 / 88; 320, four of
  // 160, 16 and 4 16 / 24, 29 / 40, 49 / 51; 960 31 / 28, 63 / 66, 108 / 108. (Up to 256 CTAs choose() streams what is short.)
  const int64_t ctas = std::max<int64_t>((total_q * (int64_t)p.group + 31) / 32, batch) * kv_heads;
  const bool few = 2 * ctas <= kFit;
  if (choice.rows >= kBlock && (most <= kStreamRows || (!few && ctas <= kFit && p.max_keys <= 4096)))
    choice = {32, few ? kFit : p.max_keys <= one_piece_mx4(32, ctas) || ctas >= kTarget ? 0 : kTarget, few, false};
  const bool laid_out = choice.rows >= kBlock;
  const Mx4Space space = mx4_space(most, kv_heads, dim, batch, p.max_keys, total_keys);
  const int64_t need = laid_out ? space.bytes : space.split;
  if (!aligned(workspace, 16) || (workspace_bytes < need && (workspace != nullptr || choice.target > 0 || laid_out)))
    return api_error(MLA_ERR_INVALID_ARG, "%s: the workspace must be 16-byte aligned and hold %lld bytes, got %lld", who,
                     (long long)need, (long long)workspace_bytes);
  set_pages(p, num_pages, page_size, page_table, pt_stride, cu_seqlens_q, seq_lens_k, max_q);
  if (workspace != nullptr) {
    p.ws_o = static_cast<float*>(workspace);
    p.ws_lse = reinterpret_cast<f32x2*>(p.ws_o + workspace_rows(most) * dim);
  }
  if (int rc = set_choice(who, p, choice)) return rc;
  if (!laid_out && (gqa_ctas(p, choice.rows) + 8 * kv_heads) * (choice.wide ? 512 : 256) > UINT32_MAX)  // in whole rounds of heads
    return api_error(MLA_ERR_UNSUPPORTED, "%s: %d rows of %d heads are more than a launch holds", who, total_q, q_heads);
  if (!laid_out) return done(launch_gqa_mx4(mp, dim, choice.rows, (hipStream_t)stream), who);
  char* at = static_cast<char*>(workspace) + space.split;
  mp.scratch_table = reinterpret_cast<int32_t*>(at);
  mp.scratch_cols = (int32_t)space.cols;
  mp.scratch_rows = space.rows;
  mp.scratch_k = reinterpret_cast<__bf16*>(at + space.table);
  mp.scratch_v = mp.scratch_k + space.rows * kv_heads * dim;
  if ((space.rows / 64 + 8) * kv_heads * 256 > UINT32_MAX || space.rows > 0x7fffffff)
    return api_error(MLA_ERR_UNSUPPORTED, "%s: %lld keys are more than a launch holds", who, (long long)space.rows);
  if (hipError_t e = launch_mx4_pages(mp, dim, (hipStream_t)stream); e != hipSuccess) return done(e, who);
  p.k = mp.scratch_k;
  p.v = mp.scratch_v;
  p.k_row_stride = p.v_row_stride = dim;
  p.k_head_stride = p.v_head_stride = space.rows * dim;
  p.num_pages = (int32_t)(space.rows / 64);
  p.log2_ps = 6;
  p.page_table = mp.scratch_table;
  p.pt_stride = space.cols;
  return done(launch_gqa_rows(p, dim, choice.rows, (hipStream_t)stream), who);
}

int mx4_rows(const char* who, bool load, const mla_mx4_pool* k_pool, const mla_mx4_pool* v_pool, int32_t num_pages, int32_t page_size,
             int32_t kv_heads, int32_t dim, const void* indices, int32_t index_bits, int32_t rows, const void* k,
             int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h, void* stream) {
  if (dim != 64 && dim != 128) return api_error(MLA_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128, got %d", who, dim);
  if (rows < 0 || (index_bits != 32 && index_bits != 64))
    return api_error(MLA_ERR_INVALID_ARG, "%s: rows %d, index_bits %d", who, rows, index_bits);
  if (rows == 0) return done(hipSuccess, who);
  if (k_pool == nullptr || v_pool == nullptr || indices == nullptr || k == nullptr || v == nullptr)
    return api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  Mx4Rows p = {};
  p.k_pool = mx4_view(*k_pool), p.v_pool = mx4_view(*v_pool);
  if (int rc = check_mx4(who, p.k_pool, p.v_pool, dim, num_pages, page_size, kv_heads)) return rc;
  if (!aligned(k, 16) || !aligned(v, 16) || k_stride_t % 8 || k_stride_h % 8 || v_stride_t % 8 || v_stride_h % 8 || k_stride_t < 0 ||
      k_stride_h < 0 || v_stride_t < 0 || v_stride_h < 0)
    return api_error(MLA_ERR_INVALID_ARG, "%s: k and v must be 16-byte aligned, with non-negative strides that are multiples of 8", who);
  if ((int64_t)rows * kv_heads * (dim / 8) > UINT32_MAX - 256)  // a thread for 8 dims of K and of V
    return api_error(MLA_ERR_UNSUPPORTED, "%s: %d rows of %d heads are more than a launch holds", who, rows, kv_heads);
  for (const Mx4View* x : {&p.k_pool, &p.v_pool})
    if (!load && (!rows_apart({num_pages, x->c_page}, {page_size, x->c_tok}, {kv_heads, x->c_head}, dim / 2) ||
                  !rows_apart({num_pages, x->s_page}, {page_size, x->s_tok}, {kv_heads, x->s_head}, dim / 32)))
      return api_error(MLA_ERR_INVALID_ARG, "%s: rows of a pool lie over one another", who);
  if (load && (!rows_apart(rows, k_stride_t, kv_heads, k_stride_h, dim) || !rows_apart(rows, v_stride_t, kv_heads, v_stride_h, dim)))
    return api_error(MLA_ERR_INVALID_ARG, "%s: rows of k or v overlap", who);
  if (load) {
    p.k_out = static_cast<__bf16*>(const_cast<void*>(k));
    p.v_out = static_cast<__bf16*>(const_cast<void*>(v));
  } else {
    p.k = static_cast<const __bf16*>(k);
    p.v = static_cast<const __bf16*>(v);
  }
  p.k_stride_t = k_stride_t, p.k_stride_h = k_stride_h, p.v_stride_t = v_stride_t, p.v_stride_h = v_stride_h;
  p.indices = indices;
  p.index_bits = index_bits;
  p.rows = rows;
  p.kv_heads = kv_heads;
  for (p.log2_ps = 0; (1 << p.log2_ps) < page_size;) ++p.log2_ps;
  p.pool_rows = (int64_t)num_pages * page_size;
  return done(launch_mx4_rows(p, dim, load, (hipStream_t)stream), who);
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

int mla_gqa_mx4_workspace_bytes(int32_t max_q, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t batch,
                                int64_t max_keys, int64_t total_keys, int64_t* bytes) {
  const char* who = "mla_gqa_mx4_workspace_bytes";
  if (bytes == nullptr || max_q < 0 || batch < 0 || max_keys < 0 || total_keys < 0)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: bytes is null, or max_q %d, batch %d, max_keys %lld or total_keys %lld < 0", who, max_q,
                          batch, (long long)max_keys, (long long)total_keys);
  if (batch > 65535) return mla::api_error(MLA_ERR_UNSUPPORTED, "%s: at most 65535 requests, got %d", who, batch);
  if (int rc = mla::check_heads(who, q_heads, kv_heads, head_dim)) return rc;
  *bytes = mla::mx4_space((int64_t)max_q * (q_heads / kv_heads), kv_heads, head_dim, batch, std::min<int64_t>(max_keys, 0x7ff00000), total_keys).bytes;
  return mla::done(hipSuccess, who);
}

int mla_gqa_chunk_mx4(const void* q, int64_t q_stride_t, int64_t q_stride_h, const mla_mx4_pool* k_pool,
                      const mla_mx4_pool* v_pool, int32_t num_pages, int32_t page_size, const int32_t* page_table,
                      int32_t pt_cols, int64_t pt_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens_k,
                      int32_t batch, int32_t total_q, int32_t max_q, int64_t total_keys, int32_t q_heads, int32_t kv_heads,
                      int32_t head_dim, float scale, void* workspace, int64_t workspace_bytes, void* out,
                      int64_t out_stride_t, int64_t out_stride_h, float* lse, int64_t lse_stride_t, void* stream) {
  const char* who = "mla_gqa_chunk_mx4";
  if (batch > 0 && total_q > 0 && max_q > 0 && cu_seqlens_q == nullptr)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  return mla::paged_mx4(who, q, q_stride_t, q_stride_h, k_pool, v_pool, num_pages, page_size, page_table, pt_cols, pt_stride,
                        cu_seqlens_q, seq_lens_k, batch, total_q, max_q < total_q ? max_q : total_q, total_keys, q_heads, kv_heads,
                        head_dim, scale, workspace, workspace_bytes, out, out_stride_t, out_stride_h, lse, lse_stride_t, stream);
}

int mla_gqa_decode_mx4(const void* q, int64_t q_stride_b, int64_t q_stride_h, const mla_mx4_pool* k_pool,
                       const mla_mx4_pool* v_pool, int32_t num_pages, int32_t page_size, const int32_t* page_table,
                       int32_t pt_cols, int64_t pt_stride, const int32_t* seq_lens, int32_t batch, int64_t total_keys,
                       int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale, void* workspace,
                       int64_t workspace_bytes, void* out, int64_t out_stride_b, int64_t out_stride_h, float* lse,
                       int64_t lse_stride_b, void* stream) {
  return mla::paged_mx4("mla_gqa_decode_mx4", q, q_stride_b, q_stride_h, k_pool, v_pool, num_pages, page_size, page_table, pt_cols,
                        pt_stride, nullptr, seq_lens, batch, batch, 1, total_keys, q_heads, kv_heads, head_dim, scale, workspace,
                        workspace_bytes, out, out_stride_b, out_stride_h, lse, lse_stride_b, stream);
}

int mla_mx4_store(const mla_mx4_pool* k_pool, const mla_mx4_pool* v_pool, int32_t num_pages, int32_t page_size,
                  int32_t kv_heads, int32_t head_dim, const void* indices, int32_t index_bits, int32_t rows, const void* k,
                  int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h, void* stream) {
  return mla::mx4_rows("mla_mx4_store", false, k_pool, v_pool, num_pages, page_size, kv_heads, head_dim, indices, index_bits, rows, k,
                       k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, stream);
}

int mla_mx4_load(const mla_mx4_pool* k_pool, const mla_mx4_pool* v_pool, int32_t num_pages, int32_t page_size, int32_t kv_heads,
                 int32_t head_dim, const void* indices, int32_t index_bits, int32_t rows, void* k, int64_t k_stride_t,
                 int64_t k_stride_h, void* v, int64_t v_stride_t, int64_t v_stride_h, void* stream) {
  return mla::mx4_rows("mla_mx4_load", true, k_pool, v_pool, num_pages, page_size, kv_heads, head_dim, indices, index_bits, rows, k,
                       k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, stream);
}

int mla_qk_norm_rope_bf16(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                          int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h, const void* q_weight,
                          const void* k_weight, float eps, const int32_t* positions, const float* cos_sin,
                          int32_t max_position, int32_t rotary_dim, int32_t interleaved, int32_t tokens, int32_t q_heads,
                          int32_t kv_heads, int32_t head_dim, void* q_out, int64_t q_out_stride_t, int64_t q_out_stride_h,
                          void* k_out, int64_t k_out_stride_row, int64_t k_out_stride_h, void* v_out,
                          int64_t v_out_stride_row, int64_t v_out_stride_h, const void* slots, int32_t index_bits,
                          int64_t out_rows, void* stream) {
  const char* who = "mla_qk_norm_rope_bf16";
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || q_heads > 4096 || kv_heads > 4096 || out_rows < 0)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: tokens %d, q_heads %d and kv_heads %d (0 to 4096), out_rows %lld", who, tokens, q_heads,
                          kv_heads, (long long)out_rows);
  if (head_dim != 64 && head_dim != 128) return mla::api_error(MLA_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128, got %d", who, head_dim);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 8 != 0 || (rotary_dim > 0 && max_position < 1))
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: rotary_dim %d must be a multiple of 8 in [0, %d], max_position %d positive", who,
                          rotary_dim, head_dim, max_position);
  if ((q_weight == nullptr) != (k_weight == nullptr) || (v == nullptr) != (v_out == nullptr))
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: both weights or none, v with v_out", who);
  if (!(eps >= 0.f) || !isfinite(eps)) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: bad eps", who);
  if (slots != nullptr && index_bits != 32 && index_bits != 64)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: index_bits %d", who, index_bits);
  if (slots == nullptr && out_rows < tokens)
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: %lld rows for %d tokens", who, (long long)out_rows, tokens);
  if (tokens == 0 || q_heads + kv_heads == 0) return mla::done(hipSuccess, who);
  if ((q_heads > 0 && (q == nullptr || q_out == nullptr)) || (kv_heads > 0 && (k == nullptr || k_out == nullptr)) ||
      (rotary_dim > 0 && (positions == nullptr || cos_sin == nullptr)))
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: null pointer", who);
  for (const void* x : {q, k, v, q_weight, k_weight, static_cast<const void*>(cos_sin), static_cast<const void*>(q_out),
                        static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    if (!mla::aligned(x, 16)) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: tensors must be 16-byte aligned", who);
  for (int64_t x : {q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h, q_out_stride_t, q_out_stride_h,
                    k_out_stride_row, k_out_stride_h, v_out_stride_row, v_out_stride_h})
    if (x % 8 || x < 0) return mla::api_error(MLA_ERR_INVALID_ARG, "%s: strides must be non-negative multiples of 8", who);
  if ((int64_t)tokens * (q_heads + 2 * kv_heads + 8) * (head_dim / 8) > UINT32_MAX - 256)
    return mla::api_error(MLA_ERR_UNSUPPORTED, "%s: %d tokens of %d heads are more than a launch holds", who, tokens, q_heads + 2 * kv_heads);
  if ((q_heads > 0 && !mla::rows_apart(tokens, q_out_stride_t, q_heads, q_out_stride_h, head_dim)) ||
      (kv_heads > 0 && !mla::rows_apart(out_rows, k_out_stride_row, kv_heads, k_out_stride_h, head_dim)) ||
      (kv_heads > 0 && v != nullptr && !mla::rows_apart(out_rows, v_out_stride_row, kv_heads, v_out_stride_h, head_dim)))
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: rows of q_out, k_out or v_out overlap", who);
  auto moved = [&](const void* in, int64_t in_t, int64_t in_h, const void* to, int64_t to_t, int64_t to_h, int32_t heads) {
    return heads > 0 && in == to && ((tokens > 1 && in_t != to_t) || (heads > 1 && in_h != to_h));
  };
  if (moved(q, q_stride_t, q_stride_h, q_out, q_out_stride_t, q_out_stride_h, q_heads) ||
      moved(k, k_stride_t, k_stride_h, k_out, k_out_stride_row, k_out_stride_h, kv_heads) ||
      (v != nullptr && moved(v, v_stride_t, v_stride_h, v_out, v_out_stride_row, v_out_stride_h, kv_heads)) ||
      (slots != nullptr && kv_heads > 0 && (k == k_out || (v != nullptr && v == v_out))))
    return mla::api_error(MLA_ERR_INVALID_ARG, "%s: outputs in the place of inputs take their strides, and no slots", who);
  mla::QkNormRopeParams p = {};
  p.q = static_cast<const __bf16*>(q);
  p.k = static_cast<const __bf16*>(k);
  p.v = static_cast<const __bf16*>(v);
  p.q_stride_t = q_stride_t, p.q_stride_h = q_stride_h, p.k_stride_t = k_stride_t, p.k_stride_h = k_stride_h;
  p.v_stride_t = v_stride_t, p.v_stride_h = v_stride_h;
  p.q_weight = static_cast<const __bf16*>(q_weight);
  p.k_weight = static_cast<const __bf16*>(k_weight);
  p.eps = eps;
  p.positions = positions;
  p.cos_sin = cos_sin;
  p.max_position = max_position;
  p.rotary_dim = rotary_dim;
  p.interleaved = interleaved != 0;
  p.tokens = tokens;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.q_out = static_cast<__bf16*>(q_out);
  p.k_out = static_cast<__bf16*>(k_out);
  p.v_out = static_cast<__bf16*>(v_out);
  p.qo_stride_t = q_out_stride_t, p.qo_stride_h = q_out_stride_h, p.ko_stride_row = k_out_stride_row, p.ko_stride_h = k_out_stride_h;
  p.vo_stride_row = v_out_stride_row, p.vo_stride_h = v_out_stride_h;
  p.slots = slots;
  p.index_bits = index_bits;
  p.out_rows = out_rows;
  return mla::done(mla::launch_qk_norm_rope(p, head_dim, (hipStream_t)stream), who);
}

}  // extern "C"
