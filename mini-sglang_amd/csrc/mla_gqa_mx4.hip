// Grouped-head attention over a cache of 4 bits (mla_mx4.h), with the items, pieces and joining of mla_gqa.h: single tokens
// and chunks of up to 512 rows read the codes here, and longer ones where their blocks would be too few to fill the chip; others have
// their keys' values laid out first (mx4_pages_kernel), for the bf16 kernels.
//
// As mla_gqa_stream.hip, one CTA per (request, rows, KV head, piece of the keys), whose waves take tiles of 32 keys in turn,
// load a tile ahead and share nothing until the end. A tile is 4.3 KB (head_dim 128): codes go through the wave's
// LDS, and become bf16 in the registers that the matrix instructions read:
//   scores   S^T = K Q^T: lane (key a16, g) reads the 16 bytes of the key's block g, and so the dims 32 g + 8 s + 0..7 for
//            step s; the queries lie alike. One scale a lane.
//   outputs  O^T = V^T P^T: lane (n, g) reads dims 8 n + 0..7 of keys 4 g + 0..3 and 16 + 4 g + 0..3, as the numerators lie;
//            a conversion gives dims (8 n + 2 c, + 1) of one key, two of them swap halves, and product m of 8 has dim
//            8 n + m in row n: lane (row a16, g) ends up with the 32 dims 32 g + 8 i + m.
// At head_dim 64 half as many of each.
// Bound: with 16 rows, reading (64 requests of 1k to 8k tokens, 64 and 8 heads of 128: 344 MB in 66 us, 5.2 TB/s; its loads alone, the
// rest left out, take 63, and a plain stream 49 with one CTA a compute unit, 54 to 77 with more); vector instructions, some 150 a
// tile, and the matrix instructions, which hardly overlap with them (measured: 1.8 ns and 7 ns each a SIMD, 9.5 for one of the
// latter with two of the former), take 45 us of it, hidden. With 32 rows they are the bound: 16 chunks of 1 to 8 tokens on 1k to
// 16k, 32 and 8 heads, 154 MB in 35 us. Below some 20 MB: dependent loads (lengths, page, tile) and the joining's launch: one
// request of 1500, 5.9 us and 4.2.
// What did not pay, us for the 64 requests: two tiles ahead in registers 77 for 75, in a ring of LDS tiles that loads fill by
// themselves 66 for 66 at any depth; more waves (128 registers) 72 for 66; pairs of dims in place of pairs of keys, without the
// swaps and with twice the matrix instructions, 66 for 66; equal shares of the batch's keys for as many CTAs as run at once
// 61 for 66, but 20 for 18.5 (8 of 32k to 128k) and 41 for 37 (the drafts).
#include <type_traits>

#include "mla_gqa.h"
#include "mla_gqa_mx4.h"

namespace mla {
namespace {

constexpr int kTileKeys = 32;
constexpr float kLowest = -3.4028234663852886e38f;
// Numerators are relative to a reference that a row's largest score (log2 domain) may pass by kLag before it follows: sums are
// rescaled seldom (16 drafts of 1 to 8 on 1k to 16k, 32 and 8 heads: 40.0 us with 0, 37.3).
constexpr float kLag = 6.f;
// A wave whose sums of values did not come out finite takes its keys again with numerators times 2^-room: numerators of at most
// 2^kLag of as many keys as the item has, of values of the largest size, 6 2^125, sum up within fp32's range then, and what is not finite
// now is the result. At least kRoom: up to 2^18 keys. (Smaller values would fall out of the range at the other end, and what tells large
// ones apart costs every tile 5 %.) The factor is kept beside the reference: a far score's spacing is more than kRoom.
constexpr int kRoom = 24;
// whether a byte of w is 253 or more
__device__ __forceinline__ uint32_t any_fd(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x03030303u) & w & 0x80808080u; }
// bit 2 of the codes of w that a scale of 253 or more puts past bf16's range: 4 and 6 2^126, 2 and more 2^127; all of 255
__device__ __forceinline__ uint32_t past_range(uint32_t w, uint32_t scale) {
  return (scale == 255 ? ~0u : scale == 254 ? w : scale == 253 ? w & w << 1 : 0) & 0x44444444u;
}

// The CTA's item, of which the heads come fastest: CTAs go to the chip's 8 dies in turn, and a round of 8 heads' CTAs takes 8 (block,
// piece)s with all their heads, a die each, since with small pages the heads of a token share cache lines. 64 requests of 1k
// to 8k, 64 and 8 heads of 128, us with / without: pages of 1 token 135 / 193, of 2 92 / 109, of 4 84 / 88, of 16 and 64 alike.
__device__ __forceinline__ int mx4_item(int heads) {
  const uint32_t per = 8 * heads, in = blockIdx.x % per;
  return (int)(blockIdx.x - in + in % 8 * heads + in / 8);
}
inline int64_t mx4_rounds(int64_t ctas, int heads) { return (ctas + 8 * heads - 1) / (8 * heads) * (8 * heads); }

// How a tile's codes are addressed: kPage, it lies in one page (of 32 tokens or more), by scalars of the wave's; kRow, a row a
// lane. kShared: as kRow, and a cache line holds codes of more than one head, so it should stay for the others; else codes
// are read once (non-temporal).
enum Mx4Tile { kPage, kRow, kShared };

// NB blocks of 16 rows, NW waves
template <int D, int NB, int NW, Mx4Tile kTile>
__global__ __launch_bounds__(64 * NW, 2) void gqa_mx4_kernel(const GqaMx4Params mp) {
  const GqaParams& p = mp.g;
  constexpr bool kBig = kTile == kPage;
  constexpr int kRows = 16 * NB, kRowB = D / 2, kKs = D / 32, kDb = D / 16;
  constexpr int kLoads = kTileKeys * kRowB / 1024;  // 16-byte loads of a lane per K or V tile
  constexpr int kLanes = kRowB / 16;                // lanes of a row in such a load
  using scale_t = std::conditional_t<D == 128, uint32_t, uint16_t>;
  using kword_t = std::conditional_t<D == 128, u32x4, u32x2>;
  using vword_t = std::conditional_t<D == 128, uint32_t, uint16_t>;
  struct Tile {
    char k[kTileKeys * kRowB], v[kTileKeys * kRowB];
    scale_t ks[kTileKeys], vs[kTileKeys];
  };
  union Own {
    Tile t;
    char o[16 * D * 4];  // a block's outputs at the end, fp32 [16 rows][D]
  };
  __shared__ __attribute__((aligned(16))) Own s_own[NW];
  __shared__ float s_m[NW][16], s_l[NW][16], s_room[NW];
  __shared__ __attribute__((aligned(NW))) uint8_t s_left_out[NW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  GqaItem it;
  const int item = mx4_item(p.kv_heads);
  // long requests first where items of a length differ in work (one block of rows or two): 16 drafts 37.3 -> 35.3 us; with one
  // block the order gains nothing and its search costs (64 requests of 1k to 8k 66.1 -> 68.4)
  if (!gqa_find<kRows, (NB > 1)>(p, item, it)) return;
  const int C = it.C;
  const int E = it.r.E, L = it.r.L, P = it.r.P, G = p.group;
  const int a16 = lane & 15, g = lane >> 4;
  int limit[NB];
  bf16x8 qf[NB][kKs];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = it.block * kRows + 16 * nb + a16, tok = r / G;
    const bool live = tok < E;
    limit[nb] = live ? P + tok : -1;
    const __bf16* q = p.q + (int64_t)(it.r.q0 + (live ? tok : 0)) * p.q_stride_t + (int64_t)(it.head * G + (live ? r % G : 0)) * p.q_stride_h;
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) qf[nb][ks] = *reinterpret_cast<const bf16x8*>(q + (8 * kKs) * g + 8 * ks);
  }
  const int last_tok = min(E - 1, (it.block * kRows + kRows - 1) / G);
  const int first_limit = P + it.block * kRows / G;  // of the item's first row: no key up to it is masked
  const int k0 = it.piece * C, k1 = min(it.pieces > 1 ? k0 + C : L, P + last_tok + 1);
  const int whole = min(k1, first_limit + 1);  // tiles that end past it have keys that some row does not attend
  const int masked0 = k0 + (max(whole - k0, 0) & -kTileKeys);

  f32x4 O[NB][kDb];
  float m[NB], l[NB];
  bool left_out = false;
  int room = 0;
  u32x4 kr[kLoads], vr[kLoads];
  scale_t sr{};
  // What a tile's addresses come from, read a tile ahead: the page's id (rows past the length in a page are read, and left
  // out), or the row of token t in lanes t and t + 32.
  auto rows = [&](int t0) __attribute__((always_inline)) {
    if constexpr (kBig) return p.page_table[(int64_t)it.b * p.pt_stride + (min(t0, L - 1) >> p.log2_ps)];
    else return gqa_row(p, it.b, it.r.q0, min(t0 + (lane & 31), L - 1));
  };
  // of the lane in a tile: codes by load, scales
  uint32_t code_at[kLoads], scale_off;
#pragma unroll
  for (int u = 0; u < kLoads; ++u) code_at[u] = (kBig ? (u * (64 / kLanes) + lane / kLanes) * (uint32_t)mp.c_tok : 0) + lane % kLanes * 16;
  scale_off = kBig ? (lane & 31) * (uint32_t)mp.s_tok : 0;
  const uint8_t *kh = mp.k_codes + (int64_t)it.head * mp.c_head, *vh = mp.v_codes + (int64_t)it.head * mp.c_head;
  const uint8_t *ksh = mp.k_scales + (int64_t)it.head * mp.s_head, *vsh = mp.v_scales + (int64_t)it.head * mp.s_head;
  auto codes = [&](const uint8_t* k, const uint8_t* v, int u) __attribute__((always_inline)) {
    const u32x4 *kp = reinterpret_cast<const u32x4*>(k), *vp = reinterpret_cast<const u32x4*>(v);
    if constexpr (kTile == kShared) {
      kr[u] = *kp;
      vr[u] = *vp;
    } else {
      kr[u] = __builtin_nontemporal_load(kp);
      vr[u] = __builtin_nontemporal_load(vp);
    }
  };
  auto load = [&](int t0, int row) __attribute__((always_inline)) {
    if constexpr (kBig) {
      const int64_t page = min(max(__builtin_amdgcn_readfirstlane(row), 0), p.num_pages - 1), tok = t0 & ((1 << p.log2_ps) - 1);
      const int64_t at = page * mp.c_page + tok * mp.c_tok, sat = page * mp.s_page + tok * mp.s_tok;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        codes(kh + at + code_at[u], vh + at + code_at[u], u);
      }
      sr = *reinterpret_cast<const scale_t*>((lane < 32 ? ksh : vsh) + sat + scale_off);
    } else {
      const int64_t page = row >> p.log2_ps, tok = row & ((1 << p.log2_ps) - 1);
      const int64_t at = page * mp.c_page + tok * mp.c_tok;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int64_t from = __shfl(at, u * (64 / kLanes) + lane / kLanes) + code_at[u];
        codes(kh + from, vh + from, u);
      }
      sr = *reinterpret_cast<const scale_t*>((lane < 32 ? ksh : vsh) + page * mp.s_page + tok * mp.s_tok);
    }
  };
  Tile& tile = s_own[wave].t;
  // K: 16-byte chunks of a key permuted (head_dim 128), so that the 16 keys of a read lie in different banks. V: key
  // 16 t + 4 g + i at row 16 t + 4 i + g, so that a read of one (t, i) is one run of bytes.
  auto kpos = [&](int t, int c) __attribute__((always_inline)) { return t * kRowB + (D == 128 ? c ^ ((t >> 2) & 3) : c) * 16; };
  auto vpos = [&](int t) __attribute__((always_inline)) { return ((t & 16) | (t & 3) << 2 | (t >> 2 & 3)) * kRowB; };
  // the byte of block b of a scale word, in bits 30..23; other bits are others'
  auto scale_at = [](uint32_t w, int b) __attribute__((always_inline)) { return D == 128 ? __builtin_amdgcn_alignbit(w, w, (8 * b + 9) & 31) : w >> 8 * b << 23; };
  constexpr int kLanesB = 32 / (D / 16);  // lanes n of a block of V

  // kMasked: some row does not attend some key of the tile. The item's first `active` blocks of rows have rows.
  auto step = [&](int t0, auto kMasked, auto active, auto roomy) __attribute__((always_inline)) {
    constexpr int kAct = decltype(active)::value;
    f32x4 sc[kAct][2];
    kword_t kw[2];
    uint32_t ks[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = 16 * h + a16;
      kw[h] = *reinterpret_cast<const kword_t*>(D == 128 ? tile.k + kpos(key, g) : tile.k + kpos(key, 0) + 8 * g);
      ks[h] = scale_at(tile.ks[key], D == 128 ? g : g >> 1);
    }
#pragma unroll
    for (int s = 0; s < kKs; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x8 kc = __builtin_bit_cast(bf16x8, mx4_values(kw[h][s], ks[h]));
#pragma unroll
        for (int nb = 0; nb < kAct; ++nb)
          sc[nb][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kc, qf[nb][s], s == 0 ? f32x4{} : sc[nb][h], 0, 0, 0);
      }
    // Numerators of a row, in pairs of keys, in bf16 as the matrix instruction takes them (their sum l is of the unrounded ones): each is
    // off by 2^-8 at most, independently, and results by 1.2 to 1.4 times what their own rounding costs. A second product with what
    // the rounding leaves out would be twice the matrix instructions.
    u32x4 pb[kAct];
#pragma unroll
    for (int nb = 0; nb < kAct; ++nb) {
      // the scaled scores are rounded before their maximum is taken from them: the largest numerator is 1 to 2^kLag at any size
#pragma clang fp contract(off)
      f32x4(&s)[2] = sc[nb];
      // score (h, i) of a lane: row a16, key t0 + 16 h + 4 g + i
      float top = kLowest;
      const int lim = min(limit[nb], k1 - 1) - t0 - 4 * g;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[h][i] *= p.scale_log2;
          if (decltype(kMasked)::value && 16 * h + i > lim) s[h][i] = -INFINITY;
          top = fmaxf(top, s[h][i]);
        }
      top = wave_max_g(top);
      if (__ballot(top - m[nb] > kLag) != 0) {  // (a sum of the two would round up where their spacing is more than kLag)
        const float m_new = fmaxf(m[nb], top), f = __builtin_amdgcn_exp2f(m[nb] - m_new);
        m[nb] = m_new;
        l[nb] *= f;
#pragma unroll
        for (int db = 0; db < kDb; ++db) O[nb][db] *= f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(s[h][i] - m[nb]);
          if constexpr (decltype(roomy)::value) e[i] *= __uint_as_float((uint32_t)(127 - room) << 23);
          l[nb] += e[i];
        }
        pb[nb][2 * h] = pack_bf16x2(e[0], e[1]);
        pb[nb][2 * h + 1] = pack_bf16x2(e[2], e[3]);
      }
    }
    vword_t vw[2][4];
    scale_t sw[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vw[h][i] = *reinterpret_cast<const vword_t*>(tile.v + (16 * h + 4 * i + g) * kRowB + sizeof(vword_t) * a16);
        sw[h][i] = tile.vs[16 * h + 4 * g + i];
      }
    if constexpr (decltype(kMasked)::value) {
      // What is not finite at a key that not every row attends, or past the item's keys (rows that nobody wrote): the product would
      // bring it to rows of weight zero. It is left out, and added to the rows that attend it at the end.
      uint32_t any = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) any |= any_fd(sw[h][i]);
      if (__ballot(any != 0) != 0) {
        uint32_t ours = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (16 * h + i < k1 - t0 - 4 * g) ours |= any_fd(sw[h][i]);
            const uint32_t scale = sw[h][i] >> (8 * (a16 / kLanesB)) & 255;
            vw[h][i] &= (vword_t)~((past_range(vw[h][i], scale) >> 2) * 15);
            if (scale == 255) sw[h][i] = 0;
          }
        left_out = left_out || __ballot(ours != 0) != 0;
      }
    }
    float vs[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) vs[h][i] = __uint_as_float(scale_at(sw[h][i], a16 / kLanesB));
    // two dims of V's word c of key (h, i)
    auto two = [&](auto c, int h, int i) __attribute__((always_inline)) {
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(vw[h][i], vs[h][i], decltype(c)::value));
    };
    auto mfma = [](u32x4 a, u32x4 b, f32x4& o) __attribute__((always_inline)) {
      o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), o, 0, 0, 0);
    };
    auto products = [&](auto c) __attribute__((always_inline)) {
      constexpr int kC = decltype(c)::value;
      if constexpr (kC < kDb / 2) {
        u32x4 lo, hi;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = two(c, h, 2 * i), y = two(c, h, 2 * i + 1);
            lo[2 * h + i] = __builtin_amdgcn_perm(y, x, 0x05040100);
            hi[2 * h + i] = __builtin_amdgcn_perm(y, x, 0x07060302);
          }
#pragma unroll
        for (int nb = 0; nb < kAct; ++nb) {
          mfma(lo, pb[nb], O[nb][2 * kC]);
          mfma(hi, pb[nb], O[nb][2 * kC + 1]);
        }
      }
    };
    products(std::integral_constant<int, 0>{});
    products(std::integral_constant<int, 1>{});
    products(std::integral_constant<int, 2>{});
    products(std::integral_constant<int, 3>{});
  };

  auto stream = [&](auto active, auto roomy) __attribute__((always_inline)) {
    constexpr int kStep = NW * kTileKeys;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = kLowest;
      l[nb] = 0.f;
#pragma unroll
      for (int db = 0; db < kDb; ++db) O[nb][db] = f32x4{};
    }
    int t0 = k0 + kTileKeys * wave, row_next = 0;
    if (t0 < k1) {
      const int row = rows(t0);
      row_next = rows(t0 + kStep);
      load(t0, row);
    }
    auto tiles = [&](int end, auto kMasked) __attribute__((always_inline)) {
      for (; t0 < end; t0 += kStep) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          const int t = u * (64 / kLanes) + lane / kLanes;
          *reinterpret_cast<u32x4*>(tile.k + kpos(t, lane % kLanes)) = kr[u];
          *reinterpret_cast<u32x4*>(tile.v + vpos(t) + lane % kLanes * 16) = vr[u];
        }
        (lane < 32 ? tile.ks : tile.vs)[lane & 31] = sr;
        if (t0 + kStep < k1) load(t0 + kStep, row_next);
        if (t0 + 2 * kStep < k1) row_next = rows(t0 + 2 * kStep);
        step(t0, kMasked, active, roomy);
      }
    };
    tiles(whole - kTileKeys + 1, std::false_type{});
    tiles(k1, std::true_type{});
  };
  if (NB == 1 || it.block * kRows + 16 < E * G) stream(std::integral_constant<int, NB>{}, std::false_type{});
  else stream(std::integral_constant<int, 1>{}, std::false_type{});
  float zero = 0.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) zero = fmaf(O[nb][db][i], 0.f, zero);  // finite sums times 0 are 0
  if (__builtin_expect(__ballot(zero != 0.f) != 0, 0)) {
    room = max(kRoom, (int)kLag + 32 - __builtin_clz(max(k1 - k0, 1)));
    stream(std::integral_constant<int, NB>{}, std::true_type{});
  }

  // ---- the waves' results joined, one block of 16 rows at a time
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float lw = wave_sum_g(l[nb]);
    if (nb > 0) __syncthreads();
    // lane: row a16, dims (kDb * 4) g + kDb i + m, 16-byte chunks rotated by the row
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < kDb / 4; ++c)
        *reinterpret_cast<f32x4*>(s_own[wave].o + a16 * (D * 4) + ((kDb * g + kDb / 4 * i + c + a16) % (D / 4)) * 16) =
            f32x4{O[nb][4 * c][i], O[nb][4 * c + 1][i], O[nb][4 * c + 2][i], O[nb][4 * c + 3][i]};
    if (g == 0) {
      s_m[wave][a16] = m[nb];
      s_l[wave][a16] = lw;
    }
    if (lane == 0) {
      s_room[wave] = (float)room;
      s_left_out[wave] = left_out;
    }
    __syncthreads();
    // kTpr threads a row, 4 dims each at a time
    constexpr int kTpr = 4 * NW;
    const int row = threadIdx.x / kTpr, x = threadIdx.x % kTpr;
    float mt = s_m[0][row], rt = s_room[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      mt = fmaxf(mt, s_m[w][row]);
      rt = fmaxf(rt, s_room[w]);
    }
    const bool add = *reinterpret_cast<const std::conditional_t<NW == 8, uint64_t, uint32_t>*>(s_left_out) != 0;
    float f[NW], lt = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = __builtin_amdgcn_exp2f(s_m[w][row] - mt) * __builtin_amdgcn_exp2f(s_room[w] - rt) * 0x1p-4f;  // their sum is finite too
      lt += f[w] * s_l[w][row];
    }
    const bool some = lt > 0.f || lt != lt;
    const float inv = some ? 1.f / lt : 0.f;
    const f32x2 lse2 = gqa_lse(some, mt, log2f(lt * (__builtin_amdgcn_exp2f(rt) * 0x1p4f)));
    const int r = it.block * kRows + 16 * nb + row, tok = r / G, head = it.head * G + r % G;
#pragma unroll
    for (int c = tok < E ? x : D; c < D / 4; c += kTpr) {
      f32x4 o = f32x4{};
#pragma unroll
      for (int w = 0; w < NW; ++w) o += *reinterpret_cast<const f32x4*>(s_own[w].o + row * (D * 4) + ((c + row) % (D / 4)) * 16) * f[w];
      o *= inv;
      if (__builtin_expect(add, 0)) {  // what the row attends of the masked tiles and their products left out
        for (int j = masked0; j < min(k1, P + tok + 1); ++j) {
          const int from = gqa_row(p, it.b, it.r.q0, j), in_page = from & ((1 << p.log2_ps) - 1);
          const int64_t page = from >> p.log2_ps;
          const uint32_t scale = vsh[page * mp.s_page + in_page * mp.s_tok + c / 8];
          if (scale < 253) continue;
          const uint32_t w = *reinterpret_cast<const uint16_t*>(vh + page * mp.c_page + in_page * mp.c_tok + 2 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (past_range(w, scale) >> (4 * i + 2) & 1) o[i] += scale == 255 ? __builtin_nanf("") : w >> (4 * i + 3) & 1 ? -INFINITY : INFINITY;
        }
      }
      if (it.slot >= 0) {
        *reinterpret_cast<f32x4*>(p.ws_o + ((int64_t)it.slot * kRows + 16 * nb + row) * D + 4 * c) = o;
      } else {
        u32x2 v{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
        *reinterpret_cast<u32x2*>(p.out + (int64_t)(it.r.q0 + tok) * p.out_stride_t + (int64_t)head * p.out_stride_h + 4 * c) = v;
      }
    }
    if (x == 0 && tok < E) {
      if (it.slot >= 0) p.ws_lse[(int64_t)it.slot * kRows + 16 * nb + row] = lse2;
      else if (p.lse != nullptr) p.lse[(int64_t)(it.r.q0 + tok) * p.lse_stride_t + head] = lse2[0] * 0.69314718055994531f;
    }
  }
}

// Values of every key of a batch, in pages of 64 rows for the bf16 kernels: request b's keys take the rows from 64 times the
// pages of the requests before it on. scratch: K and V [rows] of kv_heads * D each, and the page table.
template <int D>
__global__ __launch_bounds__(256) void mx4_pages_kernel(const GqaMx4Params mp) {
  const GqaParams& p = mp.g;
  constexpr int kLanes = D / 8;
  const int lane = threadIdx.x & 63;
  // the CTA's head and page of 64 keys: its request, by a scan of the pages
  const int item = mx4_item(p.kv_heads), head = item % p.kv_heads, to = item / p.kv_heads;
  int acc = 0, b = -1, first = 0, L = 0;
  for (int c0 = 0; c0 < p.batch && b < 0; c0 += 64) {
    int len = 0;
    if (c0 + lane < p.batch) len = gqa_request(p, c0 + lane).L;
    const int n = (len + 63) >> 6, incl = wave_iscan(n);
    const uint64_t hit = __ballot(to >= acc + incl - n && to < acc + incl);
    if (hit != 0) {
      const int fl = __builtin_ctzll(hit);
      b = c0 + fl;
      first = acc + __builtin_amdgcn_readlane(incl - n, fl);
      L = __builtin_amdgcn_readlane(len, fl);
    } else {
      acc += __builtin_amdgcn_readlane(incl, 63);
    }
  }
  if (b < 0 || to >= mp.scratch_rows / 64) return;
  const int page = to - first;
  if (threadIdx.x == 0 && head == 0) mp.scratch_table[(int64_t)b * mp.scratch_cols + page] = to;
  constexpr int kRowsAtOnce = 256 / kLanes, kN = 64 / kRowsAtOnce;
  const int x = threadIdx.x % kLanes, t0 = threadIdx.x / kLanes;
  int64_t pg[kN], tok[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int row = gqa_row(p, b, 0, min(64 * page + t0 + i * kRowsAtOnce, L - 1));
    pg[i] = row >> p.log2_ps;
    tok[i] = row & ((1 << p.log2_ps) - 1);
  }
  uint32_t codes[kN][2], scales[kN][2];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      codes[i][v] = *reinterpret_cast<const uint32_t*>((v ? mp.v_codes : mp.k_codes) + pg[i] * mp.c_page + tok[i] * mp.c_tok + head * mp.c_head + 4 * x);
      scales[i][v] = (v ? mp.v_scales : mp.k_scales)[pg[i] * mp.s_page + tok[i] * mp.s_tok + head * mp.s_head + x / 4];
    }
  // (rows past the request's last in its last page are its last again: nothing reads them)
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int64_t at = ((int64_t)head * mp.scratch_rows + (int64_t)to * 64 + t0 + i * kRowsAtOnce) * D + 8 * x;
      *reinterpret_cast<u32x4*>((v ? mp.scratch_v : mp.scratch_k) + at) = mx4_values(codes[i][v], scales[i][v] << 23);
    }
}

template <int D, int NB, Mx4Tile kTile>
void launch_stream(const GqaMx4Params& p, int64_t grid, hipStream_t stream) {
  if (p.g.wide) hipLaunchKernelGGL((gqa_mx4_kernel<D, NB, 8, kTile>), dim3((unsigned)grid), dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((gqa_mx4_kernel<D, NB, 4, kTile>), dim3((unsigned)grid), dim3(256), 0, stream, p);
}
template <int D, int NB>
void launch_stream(const GqaMx4Params& p, int64_t grid, hipStream_t stream) {
  // a head's run of codes in a page against a line of 128 bytes. us with temporal / non-temporal loads, 64 requests of 1k to 8k, 8 KV
  // heads: head_dim 128, pages of 1 token 112 / 135, of 2 (whole lines) 95 / 92; 64, of 1 81 / 116, of 2 67 / 74, of 4 59 / 58
  const int64_t run = p.c_tok == D / 2 ? (int64_t)(D / 2) << p.g.log2_ps : D / 2;
  if (run < 128 && p.g.kv_heads > 1) launch_stream<D, NB, kShared>(p, grid, stream);
  else if (p.g.log2_ps >= 5) launch_stream<D, NB, kPage>(p, grid, stream);
  else launch_stream<D, NB, kRow>(p, grid, stream);
}

}  // namespace

hipError_t launch_gqa_mx4(const GqaMx4Params& p, int dim, int rows, hipStream_t stream) {
  const int64_t grid = mx4_rounds(gqa_ctas(p.g, rows), p.g.kv_heads);
  if (dim == 128) rows == 16 ? launch_stream<128, 1>(p, grid, stream) : launch_stream<128, 2>(p, grid, stream);
  else rows == 16 ? launch_stream<64, 1>(p, grid, stream) : launch_stream<64, 2>(p, grid, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.g.target > 0) e = launch_gqa_merge(p.g, dim, rows, stream);
  return e;
}

hipError_t launch_mx4_pages(const GqaMx4Params& p, int dim, hipStream_t stream) {
  const dim3 grid((unsigned)mx4_rounds(p.scratch_rows / 64 * p.g.kv_heads, p.g.kv_heads));
  if (dim == 128) hipLaunchKernelGGL(mx4_pages_kernel<128>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(mx4_pages_kernel<64>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mla
