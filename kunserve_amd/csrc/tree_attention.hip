// Attention of drafted trees of tokens: a row's new tokens are the nodes of a tree
// (guesses of what follows its cache, verified in one step), of which each sees the
// row's cached tokens before them, its ancestors and itself. The reference decodes one
// token of a row in a step (kunserve/request.py:654-670).
//
//   o[i, h] = sum_t p[i, h, t] V[t, g],  p = softmax over t of (q[i, h] . K[t, g]) * scale,
//   t in the P cached tokens and {P + j : j an ancestor of i, or i}
//
// The (token, query head of a KV head) pairs of a row are the columns of a workgroup's
// products: column c is token c / ratio, head g ratio + c % ratio. K and V of the cached
// tokens are read once for all of them; the drafted tokens, whose mask is a bit per
// (token, drafted token), follow in rounds of their own, and with the step's new k
// and v their rows are read from there and written into their pages. Rows are split
// into runs of rounds where there is less to do than CUs; the partials are joined
// as those of decode rows are.
#include <algorithm>
#include <cmath>
#include <map>
#include <type_traits>
#include <vector>

#include "decode_tile.hpp"

namespace kunserve {
namespace {

constexpr int kTreeRecord = 16;   // ints of a work record
constexpr int kBlock = 32;        // tokens of a score tile

// A round is what the waves load at a time, LOADS loads of TPL token rows each, and its
// tokens are score tiles of 32. Element x of half h of a tile's scores (32x32: lane
// column, register x, lane half h) is token element e = x % 8 of lane group g = 2 (x / 8)
// + h: the 8 tokens of a group are those that one lane has of one wave's loads, or of two
// waves' (eight waves with 4 loads), so that V is transposed within a lane.
template <int D, int WC>
struct TreeTile {
  static constexpr int WAVES = WC > kWaves ? WC : kWaves;
  static constexpr int LOADS = 8 * kWaves / WAVES;
  static constexpr int CH = D / 8;              // 16-byte chunks of a token row
  static constexpr int TPL = kWave / CH;
  static constexpr int STEP = TPL * LOADS;      // tokens of a wave
  static constexpr int ROUND = WAVES * STEP;
  static constexpr int BLOCKS = ROUND / kBlock;
};
// Tile, element and lane group of a round's token u.
struct TilePlace {
  int tile, e, g;
};
__host__ __device__ __forceinline__ TilePlace tile_place(int head_dim, int u) {
  const int w = u & 31;
  if (head_dim == 64) return {2 * (u >> 6) + (u >> 2 & 1), u >> 3 & 7, u & 3};
  if (head_dim == 128) return {u >> 5, w >> 2, w & 3};
  return {u >> 5, w >> 1 & 7, 2 * (w >> 4) + (w & 1)};
}
__host__ __device__ __forceinline__ int mask_bit(const TilePlace& p) {
  return 16 * (p.g & 1) + 8 * (p.g >> 1) + p.e;
}

struct TreeArgs {
  DecodeArgs d;               // q, out, the pool, partials (work, group: unused)
  const int32_t* records;     // [num_work][kTreeRecord], as TreeItem has them
  const uint32_t* masks;      // [rows][T][rounds][BLOCKS]
};

// A work record: columns [c0, c0 + cols) of a row and KV head over rounds [rb, re) of
// its tokens: `np` rounds of cached ones, then those of the drafted ones.
struct TreeItem {
  int tokens;    // drafted tokens of the row; 0: padding
  int q_first;   // its first in q and out
  int prefix;    // cached tokens before them
  int page_at;   // where the row's pages start
  int c0, cols, head;
  int np, rb, re;
  int slot, parts, part;   // slot of the row's first partial (-1: none), of how many, which
  int mask_at, mask_words; // the row's masks, words of a token's
};
__device__ __forceinline__ TreeItem tree_item(const int32_t* r) {
  return {r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10], r[11], r[12], r[13], r[14]};
}

// A column's attention over the tokens [lo, hi) of every round of the item, in fp32 on
// the vector units, a load at a time (wave_rows, with the tree's mask). Masked tokens
// leave nothing, whatever K and V hold there.
template <typename T, int D, int WC>
__device__ __forceinline__ void tree_column(const TreeArgs& ta, const TreeItem& it, int c, int lo,
                                            int hi, float& m, float& l, float (&acc)[8]) {
  typedef TreeTile<D, WC> L;
  const DecodeArgs& a = ta.d;
  const int lane = threadIdx.x & (kWave - 1);
  const int lrow = lane / L::CH, lcol = lane % L::CH;
  const int token = c / a.ratio, hq = it.head * a.ratio + c % a.ratio;
  const auto q = load_v8<T>(a.q + int64_t(it.q_first + token) * a.q_tok + int64_t(hq) * a.q_head +
                            8 * lcol);
  const int64_t head = int64_t(it.head) * a.head_stride + 8 * lcol;
  const uint32_t* mask = ta.masks + it.mask_at + int64_t(token) * it.mask_words;
  m = kNegBig;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  for (int r = it.rb; r < it.re; ++r) {
    const bool drafted = r >= it.np;
    const int t0 = (drafted ? r - it.np : r) * L::ROUND;
    const int end = min(drafted ? it.tokens : it.prefix, t0 + hi);
#pragma unroll 1
    for (int u0 = t0 + lo; u0 < end; u0 += L::TPL) {
      const int u = u0 + lrow, pos = drafted ? it.prefix + u : u;
      bool seen = u < end;
      if (seen && drafted) {
        const TilePlace at = tile_place(D, u);
        seen = mask[at.tile] >> mask_bit(at) & 1;
      }
      int p = -1;
      if (seen) {
        p = a.indices[it.page_at + (pos >> a.page_shift)];
        seen = p >= 0 && p < a.num_pages;
      }
      const f16* kp = g_zero_row + 8 * lcol;
      const f16* vp = kp;
      if (seen && drafted && a.k_new) {
        kp = a.k_new + int64_t(it.q_first + u) * a.kn_tok + int64_t(it.head) * a.kn_head + 8 * lcol;
        vp = a.v_new + int64_t(it.q_first + u) * a.vn_tok + int64_t(it.head) * a.vn_head + 8 * lcol;
      } else if (seen) {
        const int64_t off = head + int64_t(p) * a.page_stride +
                            int64_t(pos & ((1 << a.page_shift) - 1)) * a.token_stride;
        kp = a.k + off;
        vp = a.v + off;
      }
      const auto k = load_v8<T>(kp);
      const auto v = load_v8<T>(vp);
      float s = group_sum<L::CH>(dot8(q, k, 0.f)) * a.scale_log2;
      s = seen ? s : -INFINITY;
      const float mx = fmaxf(m, s);
      const float alpha = fast_exp2(m - mx), pr = fast_exp2(s - mx);
      m = mx;
      l = fmaf(l, alpha, pr);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(pr, float(v[e]), acc[e] * alpha);
    }
  }
#pragma unroll
  for (int off = L::CH; off < kWave; off <<= 1) {
    const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
    const float mx = fmaxf(m, m2);
    const float f1 = fast_exp2(m - mx), f2 = fast_exp2(m2 - mx);
    m = mx;
    l = l * f1 + l2 * f2;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f1 + __shfl_xor(acc[e], off) * f2;
  }
}

// Two probabilities x, y as the sum of two 16-bit terms each: the first cut off, not
// rounded, so that it costs a byte move (bf16) or one conversion (fp16) for both; the second
// is the difference, rounded (2^-17 and 2^-22 of the value).
template <typename T>
__device__ __forceinline__ void two_terms(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, bf16>::value) {
    const uint32_t a = f32_to_bits(x), b = f32_to_bits(y);
    hi = __builtin_amdgcn_perm(b, a, 0x07060302u);
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 l = {__bf16(x - bits_to_f32(int(a & 0xffff0000u))),
                  __bf16(y - bits_to_f32(int(b & 0xffff0000u)))};
    lo = __builtin_bit_cast(uint32_t, l);
  } else {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x - float(h[0]), y - float(h[1])));
  }
}

// Where a column's result goes: a partial (fp32) or out.
__device__ __forceinline__ int64_t part_row(const TreeArgs& ta, const TreeItem& it, int c) {
  return int64_t(it.slot + c / ta.d.ratio * it.parts + it.part) * ta.d.num_qo_heads +
         it.head * ta.d.ratio + c % ta.d.ratio;
}

// The tokens' dwords x and y (2 dims each) to those of dim 2 d + odd.
__device__ __forceinline__ uint32_t dim_pair(uint32_t x, uint32_t y, int odd) {
  return __builtin_amdgcn_perm(y, x, odd ? 0x07060302u : 0x05040100u);
}

// A workgroup has 32 WC columns: wave w takes those of tile w % WC and, of each round,
// the tokens of its share w / WC of 4 / WC. All waves load: K goes to LDS by token rows, V
// as the 8 tokens of a lane for each dim. S^T = K Q^T and O^T = V^T P^T on 32x32 tiles,
// so that a column's scores are in the registers of its two lanes, where its
// probabilities are the second product's operand.
// Of the 24 products of a tile at head_dim 128 eight are the second terms of the
// probabilities. 64 rows of 4096 tokens (bf16, 32/8 heads of 128): 8 tokens each 172 us a
// layer, 6.25 TB/s, as fast as single tokens; 32 each 272 us, of which the products take
// 165 at a large product's rate; 64 each 446 us and 335.
template <typename T, int D, int WC>
__global__ __launch_bounds__((TreeTile<D, WC>::WAVES * kWave), D == 256 ? 1 : 2)
void tree_attention_kernel(TreeArgs ta) {
  typedef typename Vec<T>::v8 V8;
  typedef TreeTile<D, WC> L;
  constexpr int STEP = L::STEP, TPL = L::TPL, LOADS = L::LOADS, CH = L::CH;
  constexpr int KS = D / 16;           // products of a score tile
  constexpr int OT = D / 32;           // output tiles of a column tile
  constexpr int WAVES = L::WAVES;
  constexpr int WT = WAVES / WC;      // shares of a round's tokens
  constexpr int GB = L::BLOCKS / WT;   // score tiles of a share
  static_assert(GB >= 1, "a share has a tile at least");
  constexpr int KBYTES = L::ROUND * D * 2;
  constexpr int BUFS = WAVES > kWaves ? 2 : 1;
  const DecodeArgs& a = ta.d;
  __shared__ __attribute__((aligned(16))) char s_raw[BUFS * 2 * KBYTES];   // K, V; in the end O
  __shared__ uint32_t s_drop[BUFS][2 * WAVES];   // tokens of a round that nobody sees, by wave
  __shared__ float s_ml[WAVES][2][kWave];

  const TreeItem it = tree_item(ta.records + kTreeRecord * int64_t(blockIdx.x));
  if (it.tokens == 0) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int col = lane & 31, h = lane >> 5;   // column of a tile, half of its rows
  const int lrow = lane / CH, lcol = lane % CH;
  const int wc = wave % WC, wt = wave / WC;
  const bool active = 32 * wc < it.cols;      // uniform
  const int c = it.c0 + min(32 * wc + col, it.cols - 1);
  const int token = int(uint32_t(c) / uint32_t(a.ratio));
  const int hq = it.head * a.ratio + c - token * a.ratio;
  const int page_mask = (1 << a.page_shift) - 1;

  // (A copy of a lane's number that keeps what is made from it where it is made: what
  // seldom runs has its addresses to itself.)
  auto here = [](int x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  // ---- loads. A round's tokens of a wave are STEP; cached ones lie in pages whose ids a
  // register's lanes hold, one for `granule` tokens, a round ahead of the loads.
  const int gshift = min(a.page_shift, 4);
  const bool two = TPL == 8 && a.page_shift == 2;   // a load's rows in two pages
  const int last_page = max(it.prefix - 1, 0) >> a.page_shift;
  auto ids_of = [&](int r) {
    if (r < it.np) {   // uniform
      const int t = r * L::ROUND + wave * STEP + (lane << gshift);
      return a.indices[it.page_at + min(t >> a.page_shift, last_page)];
    }
    // Of drafted tokens page by page, from that of the wave's first.
    const int at = it.prefix + min((r - it.np) * L::ROUND + wave * STEP, it.tokens - 1);
    return a.indices[it.page_at + min((at >> a.page_shift) + lane,
                                      (it.prefix + it.tokens - 1) >> a.page_shift)];
  };
  const int64_t head_at = int64_t(it.head) * a.head_stride;
  const char* const kb = reinterpret_cast<const char*>(a.k + head_at);
  const char* const vb = reinterpret_cast<const char*>(a.v + head_at);
  const uint32_t lane_at =
      2 * (uint32_t(two ? lrow & 3 : lrow) * uint32_t(a.token_stride) + 8 * uint32_t(lcol));
  V8 k[LOADS], v[LOADS];
  uint32_t bad = 0;   // bit i: the lane's row of load i is no token that anybody sees
  // Page ids outside the pool, and tokens behind the cached ones, read page 0.
  auto load_cached = [&](int r, int ids, auto loads_per_page) __attribute__((always_inline)) {
    constexpr int P = decltype(loads_per_page)::value;   // 0: two pages to a load
    constexpr int G = P ? LOADS / (P ? P : 1) : 2 * LOADS;   // granules
    const int t0 = r * L::ROUND + wave * STEP;
    bad = 0;
    int64_t at[G];   // bytes from the head's base
    uint32_t gone = 0;
#pragma unroll
    for (int n = 0; n < G; ++n) {
      const int t = t0 + (P ? n * P * TPL : n * (TPL / 2));
      const int p = __builtin_amdgcn_readlane(ids, n);
      const bool ok = t < it.prefix && p >= 0 && p < a.num_pages;
      at[n] = ok ? 2 * (int64_t(p) * a.page_stride + int64_t(t & page_mask) * a.token_stride) : 0;
      gone |= ok ? 0u : 1u << n;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int64_t from;
      if constexpr (P)
        from = at[i / P] + i % P * (2 * TPL * a.token_stride);
      else
        from = at[2 * i] + (lrow & 4 ? at[2 * i + 1] - at[2 * i] : 0);
      // (Past the caches: 64 rows of 4096, 32 columns, 179 us a layer against 198; where four
      // workgroups read the same K and V 280 against 277.)
      k[i] = load_v8_nt<T>(kb + from + lane_at);
      v[i] = load_v8_nt<T>(vb + from + lane_at);
    }
    if (gone || t0 + STEP > it.prefix) {   // uniform
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int n = P ? i / (P ? P : 1) : 2 * i + (lrow >> 2);
        bad |= (gone >> n & 1) || t0 + i * TPL + lrow >= it.prefix ? 1u << i : 0u;
      }
    }
  };
  typedef std::integral_constant<int, 16 / TPL> Pages16;
  typedef std::integral_constant<int, TPL == 8 ? 0 : 4 / TPL> Pages4;
  typedef std::integral_constant<int, TPL == 8 ? 1 : 8 / TPL> Pages8;
  auto load_round = [&](int r, int ids) __attribute__((always_inline)) {
    if (r < it.np) {   // uniform
      if (a.page_shift >= 4)
        load_cached(r, ids, Pages16{});
      else if (a.page_shift == 3)
        load_cached(r, ids, Pages8{});
      else
        load_cached(r, ids, Pages4{});
    } else {
      const int u0 = (r - it.np) * L::ROUND + wave * STEP;
      bad = 0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int u = u0 + i * TPL + lrow, pos = it.prefix + u;
        const int p = __shfl(ids, (pos >> a.page_shift) - ((it.prefix + u0) >> a.page_shift));
        const bool ok = u < it.tokens && p >= 0 && p < a.num_pages;
        const f16* kp = g_zero_row;
        const f16* vp = g_zero_row;
        if (ok && a.k_new) {
          kp = a.k_new + int64_t(it.q_first + u) * a.kn_tok + int64_t(it.head) * a.kn_head;
          vp = a.v_new + int64_t(it.q_first + u) * a.vn_tok + int64_t(it.head) * a.vn_head;
        } else if (ok) {
          const int64_t at = head_at + int64_t(p) * a.page_stride + int64_t(pos & page_mask) * a.token_stride;
          kp = a.k + at;
          vp = a.v + at;
        }
        k[i] = load_v8<T>(kp + 8 * lcol);
        v[i] = load_v8<T>(vp + 8 * lcol);
        bad |= ok ? 0u : 1u << i;
      }
    }
  };

  // (The next round's ids are read without a branch, behind which the compiler would wait
  // for them, and so for the loads before them.)
  int ids = it.rb < it.re ? ids_of(it.rb) : 0;
  V8 q[KS];
  {
    const f16* qp = a.q + int64_t(it.q_first + token) * a.q_tok + int64_t(hq) * a.q_head + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = load_v8<T>(qp + 16 * s);
  }
  if (it.rb < it.re) {
    load_round(it.rb, ids);
    ids = ids_of(min(it.rb + 1, it.re - 1));
  }

  f32x16 o[OT];
#pragma unroll
  for (int d = 0; d < OT; ++d) o[d] = f32x16{};
  // Probabilities are 2^(s - m): m is the maximum, or up to 8 below it, and `lift` lower in
  // fp16, whose least value is 2^-24: many tokens far below the maximum do not vanish together.
  constexpr float lift = std::is_same<T, bf16>::value ? 0.f : 7.f;
  float m = kNegBig, lsum = 0.f;   // m the same in a column's two lanes

  // LDS addresses as one register each and constants: with one for each chunk they were
  // spilled, and their reloads waited for the loads on their way.
  // Row `col` of a score tile is element e of lane group g; its token's row in the round:
  const int e = ((col >> 3) & 1) * 4 + (col & 3), g = 2 * (col >> 4) + ((col >> 2) & 1);
  const int k_row = D == 64 ? 8 * e + g : D == 128 ? 4 * e + g : 16 * (g >> 1) + 2 * e + (g & 1);
  auto tile_row0 = [](int blk) { return D == 64 ? 64 * (blk >> 1) + 4 * (blk & 1) : 32 * blk; };
  // Chunk c of token row (e, g) lies at c ^ swz: the 16 rows that 16 lanes read differ in
  // it. A load's rows have one e.
  auto swz = [](int e, int g) { return D == 64 ? e : 2 * e + (g & 1); };
  auto moved = [](int base, int bits) {   // base ^ bits, made at each use
    asm volatile("v_xor_b32 %0, %1, %2" : "=v"(base) : "n"(bits), "v"(base));
    return base;
  };
  // What a lane loads: element own.e + i of lane group own.g of tile own.tile.
  const TilePlace own = tile_place(D, wave * STEP + lrow);
  // Dim i of lane group g's V lies at i ^ v_swz(i, g): so the dims 8 l + x of 16 lanes that
  // store for one x differ in their low four bits (at head_dim 64 two groups fill 16 lanes).
  auto v_swz = [](int i, int g) { return (i >> 4 & 3) ^ (D == 64 ? (g & 1) << 2 : i >> 4 & 4); };
  const int k_read = 16 * (k_row * CH + (h ^ swz(e, g)));
  const int v_read = KBYTES + 16 * (h * D + (col ^ v_swz(col, h)));   // dim `col`; 32 d + col
  auto v_tile = [](int d) { return 16 * (2 * (d & 1) + (D == 64 ? 0 : 4 * (d >> 1 & 1))); };   // more
  const int k_park = 16 * ((wave * STEP + lrow) * CH + (lcol ^ swz(own.e, own.g)));
  const int v_park = KBYTES +
                     16 * ((own.tile * 4 + own.g) * D + (8 * lcol ^ v_swz(8 * lcol, own.g))) + 2 * own.e;

  auto sync = [&] {
    // Where a share's tokens are those that its only wave has loaded, LDS order will do.
    if constexpr (WC == 1 && WT == WAVES)
      __builtin_amdgcn_wave_barrier();
    else
      __syncthreads();
  };

  // The loaded round r to LDS.
  auto stage = [&](int r, int buf) __attribute__((always_inline)) {
    const bool drafted = r >= it.np;   // uniform
    if (drafted && a.k_new) {   // rows whose first column is the workgroup's, to their pages
      const int lo = (it.c0 + a.ratio - 1) / a.ratio;
      const int hi = min(it.tokens, (it.c0 + it.cols + a.ratio - 1) / a.ratio);
      const int lr = here(lrow);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int u = (r - it.np) * L::ROUND + wave * STEP + i * TPL + lr, pos = it.prefix + u;
        if (u < lo || u >= hi || (bad >> i & 1)) continue;
        const int64_t at = head_at +
                           int64_t(a.indices[it.page_at + (pos >> a.page_shift)]) * a.page_stride +
                           int64_t(pos & page_mask) * a.token_stride + 8 * lcol;
        *reinterpret_cast<V8*>(const_cast<f16*>(a.k) + at) = k[i];
        *reinterpret_cast<V8*>(const_cast<f16*>(a.v) + at) = v[i];
      }
    }
    // V of a token that nobody sees has to be 0: 0 x V is.
    const bool any_bad = __any(bad != 0);
    if (any_bad) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (bad >> i & 1) v[i] = V8{};
    }
    char* const to = s_raw + buf * 2 * KBYTES;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *reinterpret_cast<V8*>(to + moved(k_park, 16 * (D == 64 ? i : 2 * i)) + 16 * i * TPL * CH) = k[i];
#pragma unroll
    for (int x = 0; x < 8; ++x) {   // dim 8 lcol + x of the lane's tokens
      char* const at = to + moved(v_park, 16 * x);
      uint32_t d[LOADS / 2];
#pragma unroll
      for (int y = 0; y < LOADS / 2; ++y)
        d[y] = dim_pair(__builtin_bit_cast(u32x4, v[2 * y])[x >> 1],
                        __builtin_bit_cast(u32x4, v[2 * y + 1])[x >> 1], x & 1);
      if constexpr (LOADS == 8)
        *reinterpret_cast<u32x4*>(at) = u32x4{d[0], d[1], d[2], d[3]};
      else
        *reinterpret_cast<uint64_t*>(at) = uint64_t(d[0]) | uint64_t(d[1]) << 32;
    }
    uint32_t word[2] = {0u, 0u};   // at head_dim 64 a wave's two tiles
    if (any_bad) {
      const uint32_t bits = bad << mask_bit(own);   // (elements own.e + i)
#pragma unroll
      for (int l = 0; l < TPL; ++l)
        word[D == 64 ? l >> 2 : 0] |= uint32_t(__builtin_amdgcn_readlane(int(bits), l * CH));
    }
    if (lane < 2) s_drop[buf][2 * wave + lane] = lane ? word[1] : word[0];
  };
  // Tokens of tile blk that nobody sees.
  auto dropped = [&](int buf, int blk) {
    constexpr int PER = 32 / (D == 64 ? STEP / 2 : STEP);   // waves that load a tile
    const int w0 = D == 64 ? (blk >> 1) * PER : blk * PER;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) w |= s_drop[buf][2 * (w0 + i) + (D == 64 ? blk & 1 : 0)];
    return w;
  };

  // This wave's tiles of round r.
  auto compute = [&](int r, int buf, int from, int to) __attribute__((always_inline)) {
    const bool drafted = r >= it.np;   // uniform
    const uint32_t* mask = ta.masks + it.mask_at + int64_t(token) * it.mask_words +
                           (r - it.np) * L::BLOCKS + wt * GB;
    const int left = drafted ? it.tokens - (r - it.np) * L::ROUND : it.prefix - r * L::ROUND;
#pragma unroll 1
    for (int b = from; b < to; ++b) {
      const int blk = wt * GB + b;
      if ((tile_row0(blk) & ~31) >= left) break;   // uniform: no tokens from here on
      const int k_at = k_read + buf * 2 * KBYTES + 16 * tile_row0(blk) * CH;
      const int v_at = v_read + buf * 2 * KBYTES + 16 * 4 * D * blk;
      // Operands are read together, V's while the scores become probabilities: read one
      // by one before its product, each waited for LDS.
      V8 ka[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) ka[s] = *reinterpret_cast<const V8*>(s_raw + moved(k_at, 32 * s));
      __builtin_amdgcn_sched_barrier(0);
      f32x16 sc = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) sc = mfma32(ka[s], q[s], sc);
      V8 va[2][OT];
#pragma unroll
      for (int d = 0; d < OT; ++d)
        va[0][d] = *reinterpret_cast<const V8*>(s_raw + moved(v_at, v_tile(d)) + 16 * 32 * d);
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t gone = __builtin_amdgcn_readfirstlane(dropped(buf, blk));
      if (drafted || gone) {   // uniform
        const uint32_t w = (drafted ? ~mask[b] | gone : gone) >> (16 * h);
#pragma unroll
        for (int x = 0; x < 16; ++x) sc[x] = w >> x & 1 ? -INFINITY : sc[x];
      }
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 16; ++x) mx = fmaxf(mx, sc[x]);
      if (__any(mx * a.scale_log2 > m + (8.f + lift))) {
        mx = fmaxf(mx, __shfl_xor(mx, 32)) * a.scale_log2;
        const float m_new = mx > m + (8.f + lift) ? mx - lift : m;
        const float alpha = fast_exp2(m - m_new);
        m = m_new;
        lsum *= alpha;
#pragma unroll
        for (int d = 0; d < OT; ++d)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[d][x] *= alpha;
      }
      // Probabilities in two 16-bit terms, as in every decode launch.
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 h4, l4;
#pragma unroll
        for (int x = 0; x < 8; x += 2) {
          const float p0 = fast_exp2(fmaf(sc[8 * s + x], a.scale_log2, -m));
          const float p1 = fast_exp2(fmaf(sc[8 * s + x + 1], a.scale_log2, -m));
          lsum += p0 + p1;
          uint32_t hi, lo;
          two_terms<T>(p0, p1, hi, lo);
          h4[x / 2] = hi;
          l4[x / 2] = lo;
        }
        const V8 ph = __builtin_bit_cast(V8, h4), pl = __builtin_bit_cast(V8, l4);
        if (s == 0) {
#pragma unroll
          for (int d = 0; d < OT; ++d)
            va[1][d] = *reinterpret_cast<const V8*>(s_raw + moved(v_at, v_tile(d)) + 16 * (2 * D + 32 * d));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < OT; ++d) o[d] = mfma32(va[s][d], ph, o[d]);
#pragma unroll
        for (int d = 0; d < OT; ++d) o[d] = mfma32(va[s][d], pl, o[d]);
      }
    }
  };

  auto next_round = [&](int r, int buf) __attribute__((always_inline)) {
    if (r >= it.re) return;
    stage(r, buf);
    if (r + 1 < it.re) {
      load_round(r + 1, ids);
      ids = ids_of(min(r + 2, it.re - 1));
    }
  };
  if constexpr (BUFS == 2) {
    // Eight waves are alone on their CU: half of them stage the next round, in the other
    // buffer, before their tiles, half between them, so that of a SIMD's two waves one
    // computes (after them instead: 262 us a layer against 255 for 8 rows of 4000 to 16000
    // with 512 columns). Four waves leave that to the CU's second workgroup: with two buffers
    // they took as long.
    const bool late = wave >= L::WAVES / 2;   // uniform
    next_round(it.rb, 0);
    __syncthreads();
    for (int r = it.rb; r < it.re; ++r) {
      const int buf = (r - it.rb) & 1;
      if (!late) next_round(r + 1, buf ^ 1);
      if (active) compute(r, buf, 0, GB / 2);
      if (late) next_round(r + 1, buf ^ 1);
      if (active) compute(r, buf, GB / 2, GB);
      __syncthreads();
    }
  } else {
    for (int r = it.rb; r < it.re; ++r) {
      next_round(r, 0);
      sync();
      if (active) compute(r, 0, 0, GB);
      sync();
    }
  }

  // Values that the products do not carry (0 x infinity of a token that a column does not
  // see, infinity in two terms): those columns once more on the vector units.
  f32x4 z = {};
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int x = 0; x < 16; ++x) z[x & 3] = fmaf(o[d][x], 0.f, z[x & 3]);
  if (active && __any(!(z[0] + z[1] + z[2] + z[3] == 0.f))) {
    const int n = min(32, it.cols - 32 * wc);
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      float m1, l1, acc[8];
      tree_column<T, D, WC>(ta, it, it.c0 + 32 * wc + j, wt * GB * kBlock, (wt + 1) * GB * kBlock, m1, l1, acc);
      const bool mine = col == j;
      if (mine) {
        m = m1;
        lsum = h ? 0.f : l1;
      }
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int from = 4 * d + (x >> 2);   // the chunk of dim 32 d + 8 (x / 4) + 4 h + x % 4
          const float y0 = __shfl(acc[x & 3], from), y1 = __shfl(acc[4 + (x & 3)], from);
          if (mine) o[d][x] = h ? y1 : y0;
        }
    }
  }
  lsum += __shfl_xor(lsum, 32);

  // The shares of a column tile joined: each wave has OWN of the units of 16 dims (8 of a
  // lane's values), the others' of which it reads from LDS, and writes them out. (As little
  // code as can be: a workgroup runs it once, and waits for most of it to be fetched. Halves
  // joined step by step, as single values in LDS, and written by one share's waves: one row of
  // 1500 12.4 us a layer against 11.8, 4 of 4096 with 256 columns at head_dim 256 67
  // against 64.)
  constexpr int U = 2 * OT, OWN = U / WT;
  float y[8 * OWN];
  if constexpr (WT > 1) {
    f32x4* const s_o = reinterpret_cast<f32x4*>(s_raw);
    auto place = [&](int owner, int from, int i) {   // unit i of the owner's, of share `from`
      return s_o + (((owner * (WT - 1) + from - (from > owner)) * WC + wc) * OWN + i) * 2 * kWave + lane;
    };
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u / OWN == wt) {   // uniform
#pragma unroll
        for (int x = 0; x < 8; ++x) y[8 * (u % OWN) + x] = o[u / 2][8 * (u % 2) + x];
      } else {
        f32x4* to = place(u / OWN, wt, u % OWN);
        const int at = 8 * (u % 2);
        to[0] = f32x4{o[u / 2][at], o[u / 2][at + 1], o[u / 2][at + 2], o[u / 2][at + 3]};
        to[kWave] = f32x4{o[u / 2][at + 4], o[u / 2][at + 5], o[u / 2][at + 6], o[u / 2][at + 7]};
      }
    }
    s_ml[wave][0][lane] = m;
    s_ml[wave][1][lane] = lsum;
    __syncthreads();
    float mx = m;
#pragma unroll
    for (int i = 0; i < WT; ++i) mx = fmaxf(mx, s_ml[i * WC + wc][0][lane]);
    const float f = fast_exp2(m - mx);
    m = mx;
    lsum *= f;
#pragma unroll
    for (int x = 0; x < 8 * OWN; ++x) y[x] *= f;
#pragma unroll 1
    for (int i = 1; i < WT; ++i) {
      const int from = (wt + i) % WT;
      const float f2 = fast_exp2(s_ml[from * WC + wc][0][lane] - mx);
      lsum += s_ml[from * WC + wc][1][lane] * f2;
#pragma unroll
      for (int n = 0; n < OWN; ++n) {
        const f32x4* p = place(wt, from, n);
        const f32x4 a0 = p[0], a1 = p[kWave];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          y[8 * n + x] = fmaf(a0[x], f2, y[8 * n + x]);
          y[8 * n + 4 + x] = fmaf(a1[x], f2, y[8 * n + 4 + x]);
        }
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int x = 0; x < 8; ++x) y[8 * u + x] = o[u / 2][8 * (u % 2) + x];
  }
  if (!active || 32 * wc + col >= it.cols) return;
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
  const int dim0 = 16 * OWN * wt + 4 * h;   // the lane's first dim, 8 apart from there
  if (it.slot < 0) {   // uniform
    f16* op = a.out + int64_t(it.q_first + token) * a.o_tok + int64_t(hq) * a.o_head + dim0;
    typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int n = 0; n < 2 * OWN; ++n) {
      const float* v4 = y + 4 * n;
      *reinterpret_cast<T4*>(op + 8 * n) = T4{T(v4[0] * inv), T(v4[1] * inv), T(v4[2] * inv), T(v4[3] * inv)};
    }
  } else {
    const int64_t prow = part_row(ta, it, c);
    float* po = a.part_o + prow * D + dim0;
#pragma unroll
    for (int n = 0; n < 2 * OWN; ++n) {
      const float* v4 = y + 4 * n;
      *reinterpret_cast<f32x4*>(po + 8 * n) = f32x4{v4[0] * inv, v4[1] * inv, v4[2] * inv, v4[3] * inv};
    }
    if (h == 0 && wt == 0) a.part_lse[prow] = partial_lse(m, lsum);
  }
}

// What a plan's workgroups can be: their columns, how many to a CU, and the time of a round
// where every place is taken, base + tile for each column tile (of 64 rows of 4096 tokens of
// 4 to 64, within a tenth; us). Four waves up to 128 columns; eight at head_dim 128 (at 64
// they gained nothing, at 256 a wave's registers are two waves').
struct TreeKind {
  int columns, per_cu;
  float base, tile;
};
constexpr TreeKind kKinds[3][4] = {
    {{32, 2, 4.0f, 0.8f}, {64, 2, 4.7f, 1.0f}, {128, 2, 6.0f, 1.0f}, {}},
    {{32, 2, 3.8f, 0.6f}, {64, 2, 4.6f, 0.6f}, {128, 2, 4.7f, 1.0f}, {256, 1, 4.1f, 0.36f}},
    {{64, 1, 3.6f, 0.1f}, {128, 1, 4.6f, 0.1f}, {}, {}},
};
const TreeKind* kinds_of(int head_dim) { return kKinds[head_dim / 128]; }
int round_tokens(int head_dim) { return kWaves * 8 * kWave / (head_dim / 8); }

template <typename T, int D>
int launch_tree_dim(int columns, const TreeArgs& ta, unsigned blocks, hipStream_t s) {
  if constexpr (D == 256) {
    if (columns == 64)
      tree_attention_kernel<T, D, 2><<<blocks, kThreads, 0, s>>>(ta);
    else
      tree_attention_kernel<T, D, 4><<<blocks, kThreads, 0, s>>>(ta);
  } else {
    if constexpr (D == 128) {
      if (columns == 256) tree_attention_kernel<T, D, 8><<<blocks, 2 * kThreads, 0, s>>>(ta);
    }
    switch (columns) {
      case 32: tree_attention_kernel<T, D, 1><<<blocks, kThreads, 0, s>>>(ta); break;
      case 64: tree_attention_kernel<T, D, 2><<<blocks, kThreads, 0, s>>>(ta); break;
      case 128: tree_attention_kernel<T, D, 4><<<blocks, kThreads, 0, s>>>(ta); break;
    }
  }
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

template <typename T>
int launch_tree(int head_dim, int columns, const TreeArgs& ta, unsigned blocks, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_tree_dim<T, 64>(columns, ta, blocks, s);
    case 128: return launch_tree_dim<T, 128>(columns, ta, blocks, s);
    default: return launch_tree_dim<T, 256>(columns, ta, blocks, s);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct TreeRow {
  int32_t tokens, q_first, prefix, page_at, mask_at, mask_words, np, rounds;
};

// The kind of workgroups that takes least time for all rows: the narrowest that hold a row's
// columns are its own best, but few rows wider than the others pay for several workgroups
// sooner than all for wider ones (63 rows of 8 tokens and one of 33, 4 heads: 222 us a layer,
// 322 in workgroups of 256 columns).
const TreeKind& best_kind(const int32_t* q_indptr, const int32_t* kv_len, int32_t num_seqs, int ratio,
                          int head_dim) {
  const TreeKind* const kinds = kinds_of(head_dim);
  int best = 0;
  double least = 0;
  for (int k = 0; k < 4 && kinds[k].columns; ++k) {
    double time = 0;
    for (int32_t b = 0; b < num_seqs; ++b) {
      const int64_t cols = (int64_t(q_indptr[b + 1]) - q_indptr[b]) * ratio;
      const double each = double(ceil_div(cols, kinds[k].columns)) * kinds[k].base +
                          double(ceil_div(cols, 32)) * kinds[k].tile;
      time += each * double(ceil_div(kv_len[b], round_tokens(head_dim)) + 1);
    }
    time /= kinds[k].per_cu;
    if (k == 0 || time < least) {
      best = k;
      least = time;
    }
  }
  return kinds[best];
}

// Rounds [rb, re) of a row to a workgroup for each KV head and column tile: of parts as
// long as one another, none longer than `run`.
int32_t part_rounds_of(const TreeRow& r, int64_t run) {
  return int32_t(ceil_div(r.rounds, ceil_div(r.rounds, run)));
}

// The run of rounds that ends first: workgroups go, longest first, to the place that is
// free first, of `places` on the device, and cost a round more than they have; joining
// partials costs a round and the time that their bytes take at the rate of a round's.
// (Against the time of every run, 13 shapes: the run taken 4% from the best at most, on
// average 0.5%; with work / places to each, as far as 20% off: 32 rows of 256 to 6000 tokens
// 115 us against 130, 4 of 4096 at head_dim 256 67 against 86, 21 whole rows of 40 to 1800 44
// against 50.)
int64_t best_run(const std::vector<TreeRow>& rows, int32_t longest, int64_t work, int cols, int ratio,
                 int32_t num_kv_heads, int round, int64_t places) {
  const int64_t even = std::max<int64_t>(1, ceil_div(work, places));
  int64_t best = std::max(longest, 1);
  double least = 0;
  auto attempt = [&](int64_t run) {
    std::map<int64_t, int64_t> items, load;   // workgroups by cost; places by when they are free
    int64_t slots = 0;
    for (const TreeRow& r : rows) {
      if (r.tokens == 0) continue;
      const int64_t len = part_rounds_of(r, run), parts = ceil_div(r.rounds, len);
      const int64_t each = num_kv_heads * ceil_div(int64_t(r.tokens) * ratio, cols);
      if (parts > 1) {
        items[len + 1] += (parts - 1) * each;
        slots += parts * r.tokens;
      }
      items[r.rounds - (parts - 1) * len + 1] += each;
    }
    load[0] = places;
    for (auto i = items.rbegin(); i != items.rend(); ++i) {
      for (int64_t left = i->second; left > 0;) {
        const auto first = load.begin();
        const int64_t at = first->first, n = std::min(left, first->second);
        if (n == first->second)
          load.erase(first);
        else
          first->second -= n;
        load[at + i->first] += n;
        left -= n;
      }
    }
    // (A partial of a head is 4 bytes a dim, written and read; a round's token 4 bytes a dim.)
    const double end = double(load.rbegin()->first) + (slots ? 1 : 0) +
                       2.0 * double(slots) * ratio * num_kv_heads / (double(places) * round);
    if (least == 0 || end < least) {
      least = end;
      best = run;
    }
  };
  attempt(best);
  // Equal parts of the longest row, down to half an even share.
  for (int64_t parts = 2, last = best; parts <= 64; ++parts) {
    const int64_t run = ceil_div(longest, parts);
    if (2 * run < even || run == last) break;
    last = run;
    attempt(run);
  }
  for (int64_t run : {even, even + (even + 3) / 4, even + (even + 1) / 2})
    if (run < longest) attempt(run);
  return best;
}

int tree_plan(const int32_t* indptr, const int32_t* q_indptr, const int32_t* q_first,
              const int32_t* kv_len, const int32_t* parents, int32_t num_seqs,
              int32_t num_qo_heads, int32_t num_kv_heads, int32_t page_size, int32_t head_dim,
              int32_t num_cus, int32_t part_rounds, std::vector<int32_t>& plan,
              kunserve_tree_plan_info* info) {
  const int ratio = num_qo_heads / num_kv_heads;
  const TreeKind& kind = best_kind(q_indptr, kv_len, num_seqs, ratio, head_dim);
  const int max_cols = kind.columns;
  const int round = round_tokens(head_dim), tiles = round / kBlock;
  const int64_t cus = num_cus > 0 ? num_cus : 256;
  std::vector<TreeRow> rows(num_seqs);
  std::vector<uint32_t> masks;
  int64_t work = 0;   // rounds of all workgroups
  int32_t longest = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    const int32_t n = q_indptr[b + 1] - q_indptr[b];
    TreeRow& r = rows[b];
    KSV_CHECK_ARG(n >= 0 && kv_len[b] >= n, "row %d: %d new tokens of %d", b, n, kv_len[b]);
    KSV_CHECK_ARG(indptr[b] >= 0, "row %d: its pages start at %d", b, indptr[b]);
    KSV_CHECK_ARG(int64_t(indptr[b + 1]) - indptr[b] >= ceil_div(kv_len[b], page_size),
                  "row %d: %lld pages for %d tokens", b, (long long)indptr[b + 1] - indptr[b],
                  kv_len[b]);
    r.tokens = n;
    r.q_first = q_first ? q_first[b] : q_indptr[b];
    KSV_CHECK_ARG(r.q_first >= 0 && int64_t(r.q_first) + n <= int64_t(1) << 31,
                  "row %d of %d tokens: its first token is %d", b, n, r.q_first);
    KSV_CHECK_ARG(int64_t(n) * ratio < (int64_t(1) << 31) - max_cols, "row %d: %d tokens of %d heads",
                  b, n, ratio);
    r.prefix = kv_len[b] - n;
    r.page_at = indptr[b];
    r.np = int32_t(ceil_div(r.prefix, round));
    r.rounds = r.np + int32_t(ceil_div(n, round));
    r.mask_words = int32_t(ceil_div(n, round)) * tiles;
    KSV_CHECK_ARG(int64_t(masks.size()) + int64_t(n) * r.mask_words < (int64_t(1) << 30),
                  "trees of too many tokens");
    r.mask_at = int32_t(masks.size());
    masks.resize(masks.size() + size_t(n) * r.mask_words, 0u);
    uint32_t* m = masks.data() + r.mask_at;
    const int32_t* up = parents + q_indptr[b];
    for (int32_t i = 0; i < n; ++i) {
      KSV_CHECK_ARG(up[i] >= -1 && up[i] < i, "row %d: token %d has parent %d", b, i, up[i]);
      uint32_t* own = m + size_t(i) * r.mask_words;
      if (up[i] >= 0) std::copy_n(m + size_t(up[i]) * r.mask_words, r.mask_words, own);
      const TilePlace at = tile_place(head_dim, i);
      own[at.tile] |= 1u << mask_bit(at);
    }
    work += n ? int64_t(r.rounds) * ceil_div(int64_t(n) * ratio, max_cols) * num_kv_heads : 0;
    if (n) longest = std::max(longest, r.rounds);
  }
  if (q_first) {   // rows write their tokens of out
    std::vector<int32_t> by_first;
    for (int32_t b = 0; b < num_seqs; ++b)
      if (rows[b].tokens) by_first.push_back(b);
    const auto before = [&](int32_t x, int32_t y) { return rows[x].q_first < rows[y].q_first; };
    if (!std::is_sorted(by_first.begin(), by_first.end(), before))
      std::sort(by_first.begin(), by_first.end(), before);
    for (size_t i = 1; i < by_first.size(); ++i) {
      const TreeRow &x = rows[by_first[i - 1]], &y = rows[by_first[i]];
      KSV_CHECK_ARG(int64_t(x.q_first) + x.tokens <= y.q_first, "rows %d and %d both have token %d",
                    by_first[i - 1], by_first[i], y.q_first);
    }
  }
  const int64_t slots_at_once = kind.per_cu * cus;
  const int64_t run = part_rounds > 0
                          ? std::min<int64_t>(part_rounds, std::max(longest, 1))
                          : best_run(rows, longest, work, max_cols, ratio, num_kv_heads, round,
                                     slots_at_once);

  struct Piece {
    int32_t row, part, rb, re;
  };
  std::vector<Piece> pieces;
  std::vector<int32_t> merges, slot(num_seqs, -1), parts(num_seqs, 1);
  int64_t slots = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    const TreeRow& r = rows[b];
    if (r.tokens == 0) continue;
    const int32_t len = part_rounds_of(r, run);
    parts[b] = int32_t(ceil_div(r.rounds, len));
    for (int32_t i = 0; i < parts[b]; ++i)
      pieces.push_back({b, i, i * len, std::min(r.rounds, (i + 1) * len)});
    if (parts[b] == 1) continue;
    slot[b] = int32_t(slots);
    for (int32_t i = 0; i < r.tokens; ++i, slots += parts[b])
      merges.insert(merges.end(), {r.q_first + i, int32_t(slots), parts[b], 0});
    KSV_CHECK_ARG(slots < (int64_t(1) << 31), "too many partial results");
  }
  // Longest first, to the XCD with least to do; the column tiles of a piece and KV
  // head, which read the same K and V, one after the other on one XCD.
  std::stable_sort(pieces.begin(), pieces.end(), [](const Piece& x, const Piece& y) {
    return x.re - x.rb > y.re - y.rb;
  });
  std::vector<int32_t> lanes[kXcds];
  int64_t load[kXcds] = {};
  size_t depth = 0;
  for (const Piece& p : pieces) {
    const TreeRow& r = rows[p.row];
    const int32_t cols = r.tokens * ratio;
    for (int32_t h = 0; h < num_kv_heads; ++h) {
      const int x = int(std::min_element(load, load + kXcds) - load);
      for (int32_t c = 0; c < cols; c += max_cols) {
        lanes[x].insert(lanes[x].end(),
                        {r.tokens, r.q_first, r.prefix, r.page_at, c, std::min(max_cols, cols - c),
                         h, r.np, p.rb, p.re, slot[p.row], parts[p.row], p.part, r.mask_at,
                         r.mask_words, 0});
        load[x] += p.re - p.rb + 1;
      }
      depth = std::max(depth, lanes[x].size() / kTreeRecord);
    }
  }
  for (size_t r = 0; r < depth; ++r)
    for (int x = 0; x < kXcds; ++x)
      for (int i = 0; i < kTreeRecord; ++i)
        plan.push_back(kTreeRecord * r + i < lanes[x].size() ? lanes[x][kTreeRecord * r + i] : 0);
  info->num_work = int32_t(kXcds * depth);
  info->num_merge = int32_t(merges.size() / 4);
  info->num_slots = int32_t(slots);
  info->columns = max_cols;
  info->num_seqs = num_seqs;
  info->head_dim = head_dim;
  info->page_size = page_size;
  info->num_qo_heads = num_qo_heads;
  info->num_kv_heads = num_kv_heads;
  plan.insert(plan.end(), merges.begin(), merges.end());
  plan.insert(plan.end(), masks.begin(), masks.end());
  KSV_CHECK_ARG(plan.size() < (size_t(1) << 31), "the plan is too long");
  info->plan_ints = int32_t(plan.size());
  return KUNSERVE_OK;
}

}  // namespace
}  // namespace kunserve

using namespace kunserve;

extern "C" int64_t kunserve_tree_plan_bound(const int32_t* q_indptr_host,
                                            const int32_t* kv_len_host, int32_t num_seqs,
                                            int32_t num_qo_heads, int32_t num_kv_heads,
                                            int32_t head_dim) {
  if (num_seqs < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 ||
      (num_seqs > 0 && (!q_indptr_host || !kv_len_host)) ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return -1;
  // (The fewest columns to a workgroup of any plan.)
  const int64_t round = round_tokens(head_dim), ratio = ceil_div(num_qo_heads, num_kv_heads);
  int64_t items = 0, rest = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    const int64_t n = std::max<int64_t>(0, int64_t(q_indptr_host[b + 1]) - q_indptr_host[b]);
    const int64_t rounds = ceil_div(std::max(kv_len_host[b], 0), round) + 1;
    items += rounds * num_kv_heads * ceil_div(n * ratio, 32);
    rest += n * (4 + ceil_div(n, 256) * (256 / kBlock));
  }
  return kTreeRecord * kXcds * items + rest;
}

extern "C" int kunserve_tree_plan(const int32_t* indptr_host, const int32_t* q_indptr_host,
                                  const int32_t* q_first_host, const int32_t* kv_len_host,
                                  const int32_t* parents_host, int32_t num_seqs,
                                  int32_t num_qo_heads, int32_t num_kv_heads, int32_t page_size,
                                  int32_t head_dim, int32_t num_cus, int32_t part_rounds,
                                  int32_t* plan_host, int64_t plan_capacity,
                                  kunserve_tree_plan_info* info) {
  clear_error();
  KSV_CHECK_ARG(info && plan_host, "null plan buffer or info");
  KSV_CHECK_ARG(num_seqs >= 0 && (num_seqs == 0 || (indptr_host && q_indptr_host && kv_len_host)),
                "bad table or num_seqs");
  KSV_CHECK_ARG(num_qo_heads > 0 && num_kv_heads > 0 && num_qo_heads % num_kv_heads == 0,
                "num_qo_heads %d not a multiple of num_kv_heads %d", num_qo_heads, num_kv_heads);
  KSV_CHECK_ARG(page_size >= kMinPageSize && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two >= %d", page_size, kMinPageSize);
  KSV_CHECK_ARG(part_rounds >= 0, "part_rounds %d is negative", part_rounds);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("head_dim %d not compiled", head_dim);
    return KUNSERVE_EUNSUPPORTED;
  }
  KSV_CHECK_ARG(num_seqs == 0 || q_indptr_host[0] == 0, "q_indptr starts at %d", q_indptr_host[0]);
  KSV_CHECK_ARG(num_seqs == 0 || q_indptr_host[num_seqs] == 0 || parents_host, "null parents");
  return no_throw([&] {
    std::vector<int32_t> plan;
    const int rc = tree_plan(indptr_host, q_indptr_host, q_first_host, kv_len_host, parents_host,
                             num_seqs, num_qo_heads, num_kv_heads, page_size, head_dim, num_cus,
                             part_rounds, plan, info);
    if (rc) return rc;
    if (int64_t(plan.size()) > plan_capacity) {
      set_error("plan needs %lld ints, capacity %lld", (long long)plan.size(),
                (long long)plan_capacity);
      return int(KUNSERVE_ENOSPC);
    }
    std::copy(plan.begin(), plan.end(), plan_host);
    return int(KUNSERVE_OK);
  });
}

extern "C" int64_t kunserve_tree_workspace_bytes(const kunserve_tree_plan_info* info) {
  if (!info) return -1;
  return int64_t(info->num_slots) * info->num_qo_heads * (info->head_dim + 1) * 4;
}

// The arguments of the launch and of the joining of its partials, which are the decode
// launch's; ta stays empty where there is no work.
static int tree_args(const kunserve_kv_pool* pool, int32_t layer, const kunserve_page_table* table,
                     const kunserve_tensor3* q, kunserve_tensor3* out, int32_t num_qo_heads,
                     float sm_scale, const int32_t* plan_dev, const kunserve_tree_plan_info* info,
                     void* workspace_dev, int64_t workspace_bytes, const StepFusion& fusion,
                     kunserve_decode_plan_info* parts, TreeArgs* ta) {
  clear_error();
  KSV_CHECK_ARG(pool && table && q && out && info, "null argument");
  KSV_CHECK_ARG(info->head_dim == pool->head_dim, "plan made for head_dim %d, pool has %d",
                info->head_dim, pool->head_dim);
  KSV_CHECK_ARG(info->page_size == pool->page_size, "plan made for pages of %d, pool has %d",
                info->page_size, pool->page_size);
  KSV_CHECK_ARG(info->num_qo_heads == num_qo_heads && info->num_kv_heads == pool->num_kv_heads,
                "plan made for %d query heads on %d, not %d on %d", info->num_qo_heads,
                info->num_kv_heads, num_qo_heads, pool->num_kv_heads);
  KSV_CHECK_ARG(info->num_seqs == table->num_seqs, "plan made for %d rows, not %d", info->num_seqs,
                table->num_seqs);
  KSV_CHECK_ARG(pool->token_stride < (int64_t(1) << 28),
                "tokens %lld elements apart: less than 2^28 here", (long long)pool->token_stride);
  KSV_CHECK_ARG(num_qo_heads < 65536, "%d query heads: at most 65535", num_qo_heads);
  *parts = kunserve_decode_plan_info{};
  parts->num_work = info->num_work;
  parts->num_merge = info->num_merge;
  parts->num_slots = info->num_slots;
  parts->group_size = decode_group(num_qo_heads, std::max(pool->num_kv_heads, 1));
  *ta = TreeArgs{};
  StepFusion append;
  append.k_new = fusion.k_new;
  append.v_new = fusion.v_new;
  const int rc = decode_args(pool, layer, table, nullptr, q, out, num_qo_heads, sm_scale, plan_dev,
                             parts, workspace_dev, workspace_bytes, append, &ta->d);
  if (rc || info->num_work == 0) return rc;
  bool known = false;   // (the pool's head_dim is one of three here)
  for (int k = 0; k < 4 && info->columns; ++k)
    known = known || kinds_of(info->head_dim)[k].columns == info->columns;
  KSV_CHECK_ARG(known, "plan of %d columns to a workgroup", info->columns);
  KSV_CHECK_ARG(aligned16(workspace_dev), "workspace must be 16-byte aligned");
  KSV_CHECK_ARG((reinterpret_cast<uintptr_t>(out->data) & 7) == 0 && out->token_stride % 4 == 0 &&
                    out->head_stride % 4 == 0,
                "q must be 16-byte aligned with strides that are multiples of 8, out 8-byte "
                "aligned with multiples of 4");
  ta->records = plan_dev;
  ta->masks = reinterpret_cast<const uint32_t*>(plan_dev + kTreeRecord * int64_t(info->num_work) +
                                                4 * int64_t(info->num_merge));
  return KUNSERVE_OK;
}

int kunserve::tree_check(const kunserve_kv_pool* pool, int32_t layer,
                         const kunserve_page_table* table, const kunserve_tensor3* q,
                         kunserve_tensor3* out, int32_t num_qo_heads, float sm_scale,
                         const int32_t* plan_dev, const kunserve_tree_plan_info* info,
                         void* workspace_dev, int64_t workspace_bytes) {
  kunserve_decode_plan_info parts;
  TreeArgs ta;
  return tree_args(pool, layer, table, q, out, num_qo_heads, sm_scale, plan_dev, info,
                   workspace_dev, workspace_bytes, StepFusion{}, &parts, &ta);
}

int kunserve::tree_attention(const kunserve_kv_pool* pool, int32_t layer,
                             const kunserve_page_table* table, const kunserve_tensor3* q,
                             kunserve_tensor3* out, int32_t num_qo_heads, float sm_scale,
                             const int32_t* plan_dev, const kunserve_tree_plan_info* info,
                             void* workspace_dev, int64_t workspace_bytes,
                             const StepFusion& fusion, kunserve_stream_t stream) {
  kunserve_decode_plan_info parts;
  TreeArgs ta;
  const int rc = tree_args(pool, layer, table, q, out, num_qo_heads, sm_scale, plan_dev, info,
                           workspace_dev, workspace_bytes, fusion, &parts, &ta);
  if (rc || info->num_work == 0) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int err = pool->dtype == KUNSERVE_DTYPE_BF16
                      ? launch_tree<bf16>(pool->head_dim, info->columns, ta, unsigned(info->num_work), s)
                      : launch_tree<f16>(pool->head_dim, info->columns, ta, unsigned(info->num_work), s);
  if (err) return err;
  parts.num_work = 0;   // the records behind which its merges are
  return decode_merge(pool, ta.d, &parts, plan_dev + kTreeRecord * int64_t(info->num_work), s);
}

extern "C" int kunserve_tree_attention(const kunserve_kv_pool* pool, int32_t layer,
                                       const kunserve_page_table* table,
                                       const kunserve_tensor3* q, kunserve_tensor3* out,
                                       int32_t num_qo_heads, float sm_scale,
                                       const int32_t* plan_dev,
                                       const kunserve_tree_plan_info* info, void* workspace_dev,
                                       int64_t workspace_bytes, kunserve_stream_t stream) {
  return kunserve::tree_attention(pool, layer, table, q, out, num_qo_heads, sm_scale, plan_dev,
                                  info, workspace_dev, workspace_bytes, StepFusion{}, stream);
}
