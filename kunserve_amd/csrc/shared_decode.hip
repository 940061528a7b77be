// Decode attention of rows whose page lists begin alike (requests behind one
// system prompt, samples of one prompt): K and V of the pages that several
// rows share are read once for all of them.
//
// The page lists of the rows form a prefix tree. A segment is a run of pages
// that the same rows, two or more, hold at the same place; a row's tokens are
// the segments on its path and a tail of its own (its new token among it). With
// o_i and lse_i of disjoint token ranges,
//   o = sum_i 2^(lse_i - lse) o_i,  lse = log2 sum_i 2^lse_i
// so segments and tails are attended apart and joined as the partitions of a
// split row are.
//
// One launch for both: the matrix units' work on segments hides behind the
// tails' bytes. The (row, query head of a KV head) pairs of a segment are the
// columns of a workgroup's products, up to 128; a tail is a segment of one row.
// K and V are read, parked and transposed as in paged_decode_mfma_kernel; a
// step's operands serve every 16-column tile, so a segment costs its bytes once
// and the matrix units 16 columns at a time.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "decode_tile.hpp"

namespace kunserve {
namespace {

constexpr int kMinSegmentTokens = 64;   // shorter runs of shared pages stay with their rows
// Bytes of K and V that sharing has to save in a layer: joining the partials in a
// launch of their own takes about 4 us. Per layer, shared against not: 3 rows
// behind 6917 tokens (4 KV heads of 64, 14 MB saved) 14.2 against 18.5 us, 7 behind
// 851 (8 of 128, 19 MB) 11.6 against 13.0; 5 behind 672 (11 MB) 11.5 against 9.9, 12
// behind 100 (4 MB) 11.6 against 8.7.
constexpr int64_t kMinSavedBytes = 13 << 20;
constexpr int kRecord = 8;              // ints of a work record
constexpr int kMinPieceTokens = 128;
// Columns, and us of the segments' work for each CU, from which workgroups are wide.
constexpr int kMinWideCols = 64;
constexpr double kMinWideShareUs = 24.0;

struct SharedArgs {
  DecodeArgs d;            // work: the tails'
  const int32_t* shared;   // [num_shared][kRecord]: rows (0: padding), their first pair,
                           // token begin, end, place among a row's partials, a row of them,
                           // head group, where that row's pages start in the table
  const int32_t* pairs;    // [...][2]: row, its first slot
  const int32_t* tail_pages;   // [work]: where its row's pages start
  const int32_t* first_ids;    // [work][waves][step_ids]: the pages of the waves' first steps
  int32_t step_ids;
  int32_t num_shared;
  uint32_t inv_group;          // 2^16 / group and 2^32 / head_groups, rounded up
  uint32_t inv_head_groups;
};

// Columns of a workgroup: 16, its waves taking the tokens in turn (narrow), or
// kWideCols, every wave with columns of its own (wide, at head_dim 128).
constexpr int kWideTiles = 2;                          // 16-column tiles of a wave
constexpr int kWideCols = kWaves * kWideTiles * 16;    // 128

// Where a workgroup's columns are in q and out: pairs of rows and their first
// partials, or one row (a tail: pairs null).
struct Columns {
  const int32_t* pairs;
  int seq, group, hq0;
  uint32_t inv_group;
  __device__ __forceinline__ int pair(int c) const { return int(uint32_t(c) * inv_group >> 16); }
  __device__ __forceinline__ int row(int c) const { return pairs ? pairs[2 * pair(c)] : seq; }
  __device__ __forceinline__ int token(const DecodeArgs& a, int c) const {
    return a.q_token ? a.q_token[row(c)] : row(c);
  }
  __device__ __forceinline__ int head(int c) const { return hq0 + c - pair(c) * group; }
  __device__ __forceinline__ const f16* q(const DecodeArgs& a, int c) const {
    return a.q + int64_t(token(a, c)) * a.q_tok + int64_t(head(c)) * a.q_head;
  }
};

// Scores of a step's 16-token tiles (masked where the step is not whole) to
// probabilities of a column tile, with the lazy running maximum of
// paged_decode_mfma_kernel (o: the column's accumulators): first its update, seldom
// made, for which alone the lanes' maxima are joined.
template <int D>
__device__ __forceinline__ void tile_max(const f32x4 (&sc)[DecodeTile<D>::PAIRS][2],
                                         float scale_log2, float& m, float& lsum,
                                         f32x4 (&o)[DecodeTile<D>::ACCS][8]) {
  typedef DecodeTile<D> L;
  float mx = -INFINITY;
#pragma unroll
  for (int p = 0; p < L::PAIRS; ++p)
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int x = 0; x < 4; ++x) mx = fmaxf(mx, sc[p][sub][x]);
  if (__any(mx * scale_log2 > m + 8.f)) {
    mx = groups_max(mx) * scale_log2;
    const float m_new = mx > m + 8.f ? mx : m;
    const float alpha = fast_exp2(m - m_new);
    m = m_new;
    lsum *= alpha;
#pragma unroll
    for (int x = 0; x < L::ACCS; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[x][e] *= alpha;
  }
}
// The probabilities, in two 16-bit terms (pl is left out by callers of one).
template <typename T, int D>
__device__ __forceinline__ void tile_exp(const f32x4 (&sc)[DecodeTile<D>::PAIRS][2],
                                         float scale_log2, float m, float& lsum,
                                         typename Vec<T>::v8 (&ph)[DecodeTile<D>::ACCS],
                                         typename Vec<T>::v8 (&pl)[DecodeTile<D>::ACCS]) {
  typedef DecodeTile<D> L;
  typedef typename Vec<T>::v8 V8;
#pragma unroll
  for (int p = 0; p < L::PAIRS; ++p)
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float pr = fast_exp2(fmaf(sc[p][sub][x], scale_log2, -m));
        lsum += pr;
        const T hi = T(pr);
        ph[p][4 * sub + x] = hi;
        pl[p][4 * sub + x] = T(pr - float(hi));
      }
  if constexpr (D == 256) {   // set x takes the lane groups of its half of the row
    const V8 zero = {};
    const bool odd = (threadIdx.x >> 4) & 1;
    ph[1] = odd ? ph[0] : zero;
    pl[1] = odd ? pl[0] : zero;
    ph[0] = odd ? zero : ph[0];
    pl[0] = odd ? zero : pl[0];
  }
}

// Step tokens past the partition, and those of page ids outside the pool.
template <int D>
__device__ __forceinline__ void mask_scores(f32x4 (&sc)[DecodeTile<D>::PAIRS][2], int t0, int te,
                                            int tg, bool any_bad, const int* s_pages,
                                            int page_shift, int pb) {
  typedef DecodeTile<D> L;
#pragma unroll
  for (int p = 0; p < L::PAIRS; ++p)
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int t = t0 + L::token(4 * sub + x, tg, p);
        bool drop = t >= te;
        if (any_bad) drop |= s_pages[min((min(t, te - 1) >> page_shift) - pb, kMaxPartPages - 1)] < 0;
        if (drop) sc[p][sub][x] = -INFINITY;
      }
}

// The same where whole loads are dropped.
template <int D>
__device__ __forceinline__ void mask_loads(f32x4 (&sc)[DecodeTile<D>::PAIRS][2], int t0, int te,
                                           int tg, int dropped) {
  typedef DecodeTile<D> L;
#pragma unroll
  for (int p = 0; p < L::PAIRS; ++p)
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int t = L::token(4 * sub + x, tg, p);
        if (t0 + t >= te || (dropped >> (t / L::TPL) & 1)) sc[p][sub][x] = -INFINITY;
      }
}

// vt[e]: dim 8 chunk + e of the lane's 8 tokens.
template <typename V8>
__device__ __forceinline__ void transpose8(const V8 (&v)[8], V8 (&vt)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    u32x4 d;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      d[x] = __builtin_amdgcn_perm(__builtin_bit_cast(u32x4, v[2 * x + 1])[e >> 1],
                                   __builtin_bit_cast(u32x4, v[2 * x])[e >> 1],
                                   (e & 1) ? 0x07060302u : 0x05040100u);
    vt[e] = __builtin_bit_cast(V8, d);
  }
}

// 0 x every sum: NaN where one is not finite (paged_decode_mfma_kernel).
template <int D>
__device__ __forceinline__ bool not_finite(const f32x4 (&o)[DecodeTile<D>::ACCS][8]) {
  float z[4] = {};
#pragma unroll
  for (int x = 0; x < (D == 256 ? 2 : 1); ++x)
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = fmaf(o[x][e][i], 0.f, z[i]);
  return __any(!(z[0] + z[1] + z[2] + z[3] == 0.f));
}

template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(kThreads, 2) void shared_decode_kernel(SharedArgs sa) {
  typedef typename Vec<T>::v8 V8;
  typedef DecodeTile<D> L;
  constexpr int STEP = L::STEP, TPL = L::TPL, LOADS = L::LOADS, PAIRS = L::PAIRS;
  constexpr int BLK = STEP * D;
  constexpr int KS = D / 32;
  constexpr int W = kWaves;

  const DecodeArgs& a = sa.d;
  __shared__ int s_pages[kMaxPartPages];
  __shared__ int s_bad[W];
  // The waves' K blocks and, where they share columns, their V; after the loop of
  // a narrow workgroup, the waves' O (fp32, 16 x D each).
  constexpr int kKBytes = (WIDE ? 2 : 1) * W * BLK * int(sizeof(T));
  constexpr int kOBytes = W * 16 * D * int(sizeof(float));
  __shared__ __attribute__((aligned(16))) char s_raw[kKBytes > kOBytes ? kKBytes : kOBytes];
  __shared__ __attribute__((aligned(16))) T s_new[2 * D];   // the new token's K and V row
  __shared__ float s_m[W][16];
  __shared__ float s_l[W][16];
  // Q of a narrow workgroup at head_dim 256 (column g's chunk c at c ^ (g & 7)):
  // in registers it would push the step's buffers out.
  constexpr bool kQInLds = D == 256;
  __shared__ __attribute__((aligned(16))) T s_q[kQInLds ? 16 * D : 8];

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = tid >> 6;
  const int j = lane & 15;
  const int tg = lane >> 4;
  const int lrow = lane / L::CH;
  const int lcol = lane % L::CH;

  // The segments' workgroups come first (a multiple of 8, so that those of the
  // tails are on the XCDs their plan has them on).
  int nrows = 1, hg, tb, te, place = 0, slot = -1;
  Columns columns{nullptr, 0, a.group, 0, sa.inv_group};
  int page_at, item = 0;
  const bool tail = int(blockIdx.x) >= sa.num_shared;   // uniform, as all of this
  if (!tail) {
    const int32_t* rec = sa.shared + kRecord * int(blockIdx.x);
    nrows = rec[0];
    if (nrows <= 0) return;
    columns.pairs = sa.pairs + 2 * rec[1];
    tb = rec[2];
    te = rec[3];
    place = rec[4];
    columns.seq = rec[5];
    hg = rec[6];
    page_at = rec[7];
  } else {
    const int b = int(blockIdx.x) - sa.num_shared;
    const int local = a.head_groups == 1 ? b >> 3 : int(__umulhi(uint32_t(b >> 3), sa.inv_head_groups));
    hg = (b >> 3) - local * a.head_groups;
    item = 8 * local + (b & 7);
    if (item >= a.num_work) return;
    const int32_t* w = a.work + 4 * item;
    page_at = sa.tail_pages[item];
    columns.seq = w[0];
    if (columns.seq < 0) return;
    tb = w[1];
    te = w[2];
    slot = w[3];
  }
  const int cols = nrows * a.group;
  const int hq0 = hg * a.group;
  columns.hq0 = hq0;
  const int hkv = a.group == a.ratio ? hg : hq0 / a.ratio;
  const int page_mask = (1 << a.page_shift) - 1;

  const int pb = tb >> a.page_shift;
  const int np = te > tb ? ((te - 1) >> a.page_shift) + 1 - pb : 0;
  const int32_t* seq_pages = a.indices + page_at;
  auto page_id = [&](int i) {   // -1: outside the pool
    const int p = seq_pages[pb + i];
    return p >= 0 && p < a.num_pages ? p : -1;
  };
  auto stage_pages = [&] {   // for all waves; whether one of the ids is bad
    bool bad_id = false;
    for (int i = tid; i < np; i += W * kWave) {
      const int p = page_id(i);
      s_pages[i] = p;
      bad_id |= p < 0;
    }
    const bool wave_bad = __any(bad_id);
    if (lane == 0) s_bad[wave] = wave_bad;
    __syncthreads();
    int bad_votes = 0;
#pragma unroll
    for (int wv = 0; wv < W; ++wv) bad_votes |= s_bad[wv];
    return __builtin_amdgcn_readfirstlane(bad_votes) != 0;
  };
  const bool wide = WIDE && cols > 16;   // uniform
  const f16* kb = a.k + int64_t(hkv) * a.head_stride + lcol * 8;
  const f16* vb = a.v + int64_t(hkv) * a.head_stride + lcol * 8;
  const int nsteps = (te - tb + STEP - 1) / STEP;
  T* const blocks = reinterpret_cast<T*>(s_raw);
  T* sk = blocks + wave * BLK;

  // Pages that hold a load's TPL token rows whole: the load's address is a scalar
  // and the lane's 32-bit offset (pieces begin at multiples of a page and of 64,
  // partitions of 128): all but pages of 4 tokens at head_dim 64. Looked up for each
  // lane's row instead, addresses were half of a tail's instructions.
  const bool scalar = TPL <= kMinPageSize || (1 << a.page_shift) >= TPL;   // uniform
  const char* const ks = reinterpret_cast<const char*>(a.k + int64_t(hkv) * a.head_stride);
  const char* const vs = reinterpret_cast<const char*>(a.v + int64_t(hkv) * a.head_stride);
  const uint32_t lane_at = 2 * (uint32_t(lrow) * uint32_t(a.token_stride) + 8 * uint32_t(lcol));
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);   // branches on it are scalar
  int64_t at[LOADS];   // bytes, of the loads of the step on its way
  int dropped = 0;     // those (bits) that lie past `te` or in a page outside the pool: from page 0
  // A step's pages: id(h) of its tokens from h * granule on.
  const int granule = a.page_shift >= 4 ? 16 : TPL;   // uniform
  auto find = [&](int c, auto loads_per_page, auto id) {
    constexpr int P = decltype(loads_per_page)::value;
    const int ts = tb + c * STEP;
    dropped = 0;
#pragma unroll
    for (int h = 0; h < LOADS / P; ++h) {
      const int t = ts + h * P * TPL;
      const int p = id(h);
      const bool drop = t >= te || p < 0;
      dropped |= drop ? ((1 << P) - 1) << (h * P) : 0;
      const int64_t off = drop ? 0 : 2 * (int64_t(p) * a.page_stride +
                                          int64_t(t & page_mask) * a.token_stride);
#pragma unroll
      for (int i = 0; i < P; ++i) at[h * P + i] = off + i * (2 * TPL * a.token_stride);
    }
  };
  typedef std::integral_constant<int, 16 / TPL> Granule16;
  typedef std::integral_constant<int, 1> Granule1;
  auto place_of = [&](int t) { return min(max((t >> a.page_shift) - pb, 0), np - 1); };
  // From LDS.
  auto find_step = [&](int c) {
    auto look = [&](auto loads_per_page) {
      constexpr int P = decltype(loads_per_page)::value;
      int page[LOADS / P];
#pragma unroll
      for (int h = 0; h < LOADS / P; ++h) page[h] = s_pages[place_of(tb + c * STEP + h * P * TPL)];
      find(c, loads_per_page, [&](int h) { return __builtin_amdgcn_readfirstlane(page[h]); });
    };
    if (a.page_shift >= 4)   // uniform
      look(Granule16{});
    else
      look(Granule1{});
  };
  // From the lanes of a register: lane h has id(h).
  auto ids_of = [&](int c) { return seq_pages[pb + place_of(tb + c * STEP + lane * granule)]; };
  auto find_ids = [&](int c, int ids) {
    auto id = [&](int h) {
      const int p = __builtin_amdgcn_readlane(ids, h);
      return p < a.num_pages ? p : -1;
    };
    if (a.page_shift >= 4)
      find(c, Granule16{}, id);
    else
      find(c, Granule1{}, id);
  };

  V8 k[LOADS], v[LOADS];
  auto load_rows = [&](int i) {
    k[i] = load_v8<T>(ks + at[i] + lane_at);
    v[i] = load_v8<T>(vs + at[i] + lane_at);
  };
  auto drop_rows = [&] {   // their scores are masked; 0 x V has to be 0
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (dropped >> i & 1) v[i] = V8{};
  };
  NewRow nr{-1, 0, 0};
  auto load_lanes = [&](int c) {   // each lane's row looked up in LDS
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = tb + c * STEP + TPL * i + lrow;
      const int pi = min((t >> a.page_shift) - pb, kMaxPartPages - 1);
      const int p = (c < nsteps && t < te) ? s_pages[pi] : -1;
      const int64_t off = int64_t(max(p, 0)) * a.page_stride + int64_t(t & page_mask) * a.token_stride;
      k[i] = load_v8<T>(p >= 0 ? kb + (t == nr.pos ? nr.k : off) : g_zero_row + lcol * 8);
      v[i] = load_v8<T>(p >= 0 ? vb + (t == nr.pos ? nr.v : off) : g_zero_row + lcol * 8);
    }
  };
  auto park = [&] {   // K in the wave's block
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = TPL * i + lrow;
      *reinterpret_cast<V8*>(&sk[t * D + ((lcol ^ L::swz(t)) << 3)]) = k[i];
    }
  };
  // Score tile row j of pair p, subtile sub: its token's chunks in a block.
  auto k_row = [&](const T* block, int p, int sub, int s) {
    const int t = L::token(4 * sub + (j & 3), j >> 2, p);
    return *reinterpret_cast<const V8*>(&block[t * D + (((4 * s + tg) ^ L::swz(t)) << 3)]);
  };

  if constexpr (WIDE) {
    static_assert(PAIRS == 1 && L::ACCS == 1 && kWideTiles == 2 && 2 * KS == 8);
    if (wide) {
      const bool any_bad = stage_pages();
      // Every wave has tiles of its own; a round of the loop is a step of each
      // wave's tokens, which all waves take from LDS.
      const int c0 = wave_s * kWideTiles * 16;
      V8 q[kWideTiles][KS];
#pragma unroll
      for (int ct = 0; ct < kWideTiles; ++ct) {
        const int c = c0 + 16 * ct + j;
        const f16* qp = columns.q(a, min(c, cols - 1)) + 8 * tg;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[ct][s] = c < cols ? load_v8<T>(qp + 32 * s) : V8{};
      }
      f32x4 o[kWideTiles][L::ACCS][8];
      float m[kWideTiles], lsum[kWideTiles];
#pragma unroll
      for (int ct = 0; ct < kWideTiles; ++ct) {
        m[ct] = kNegBig;
        lsum[ct] = 0.f;
#pragma unroll
        for (int x = 0; x < L::ACCS; ++x)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[ct][x][e] = f32x4{};
      }
      V8* const values = reinterpret_cast<V8*>(blocks + W * BLK);   // [wave][dim e][lane]
      // The blocks' places (k_row, park) differ by an XOR of bits 6 and 7 and by
      // constants: one register, and the XOR made at each use, so that none is kept.
      auto moved = [&](int base, int x) {
        asm volatile("v_xor_b32 %0, %1, %2" : "=v"(base) : "n"(x << 6), "v"(base));
        return base;
      };
      const int read_at = L::token(j & 3, j >> 2, 0) * D * 2 + ((tg ^ L::swz(L::token(j & 3, j >> 2, 0))) << 4);
      const int park_at = (wave * BLK + lrow * D) * 2 + ((lcol ^ lrow) << 4);
      find_step(wave_s);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load_rows(i);
      for (int c = 0; c < nsteps; c += W) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
          *reinterpret_cast<V8*>(s_raw + moved(park_at, i & 3) + i * TPL * D * 2) = k[i];
        if (dropped) drop_rows();   // uniform
        V8 vt[8];
        transpose8(v, vt);
#pragma unroll
        for (int e = 0; e < 8; ++e) values[(wave * 8 + e) * kWave + lane] = vt[e];
        find_step(c + W + wave_s);
        __syncthreads();
        // The next step's loads a few at a time between the products: together
        // they would wait for the CU's one path to the caches.
        auto load_some = [&](int blk) {
#pragma unroll
          for (int i = 0; i < LOADS / W; ++i) load_rows(blk * (LOADS / W) + i);
        };
        if (c0 >= cols) {   // uniform
#pragma unroll
          for (int blk = 0; blk < W; ++blk) load_some(blk);
        } else {
          // One wave to a SIMD: what overlaps does so within its instructions. A
          // tile's exponentials stand between the products of the other tile (scores of the
          // second, then P V of the first), and V and the next K are read into
          // the registers that the products are done with. Probabilities in two 16-bit terms, as in
          // every decode launch (bf16: 1.7e-3 off 64 bits, 2.1e-3 in one), though the
          // matrix units' work counts here. Steps past the piece are masked ones.
          // 128 rows behind 8192 tokens with tails of 20-100, 64 heads on 8: 79 us a layer
          // (65 with one term), whose products alone are 50 at the rate of a large
          // matrix product. The second term's products behind the first's, those of
          // the second tile unordered but for the reads: all in pairs 8 % more.
          V8 ka[2][KS], ve[8];
          auto read_k = [&](int blk, int i) {
            ka[i & 1][i >> 1] = *reinterpret_cast<const V8*>(
                s_raw + moved(read_at, i >> 1) + (blk * BLK + (i & 1) * 16 * D) * 2);
          };
#pragma unroll
          for (int i = 0; i < 2 * KS; ++i) read_k(0, i);
#pragma unroll
          for (int blk = 0; blk < W; ++blk) {
            load_some(blk);
            const int t0 = tb + (c + blk) * STEP;
            const bool edge = any_bad || t0 + STEP > te;   // uniform
            f32x4 sc[kWideTiles][PAIRS][2];
            V8 ph[kWideTiles][L::ACCS], pl[kWideTiles][L::ACCS];
            auto scores = [&](int ct, int s) {
#pragma unroll
              for (int sub = 0; sub < 2; ++sub)
                sc[ct][0][sub] = mfma16(ka[sub][s], q[ct][s], s == 0 ? f32x4{} : sc[ct][0][sub]);
            };
            auto maximum = [&](int ct) {
              if (edge) {
                int g = tg;
                asm volatile("" : "+v"(g));   // keeps the indexes' arithmetic in here
                mask_scores<D>(sc[ct], t0, te, g, any_bad, s_pages, a.page_shift, pb);
              }
              tile_max<D>(sc[ct], a.scale_log2, m[ct], lsum[ct], o[ct]);
            };
#pragma unroll
            for (int s = 0; s < KS; ++s) scores(0, s);
            __builtin_amdgcn_sched_barrier(0);
            maximum(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              scores(1, s);
              ve[2 * s] = values[(blk * 8 + 2 * s) * kWave + lane];
              ve[2 * s + 1] = values[(blk * 8 + 2 * s + 1) * kWave + lane];
            }
            tile_exp<T, D>(sc[0], a.scale_log2, m[0], lsum[0], ph[0], pl[0]);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // a product
              __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);   // vector operations
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // reads
              __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            maximum(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[0][0][e] = mfma16(ve[e], ph[0][0], o[0][0][e]);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[0][0][e] = mfma16(ve[e], pl[0][0], o[0][0][e]);
            tile_exp<T, D>(sc[1], a.scale_log2, m[1], lsum[1], ph[1], pl[1]);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[1][0][e] = mfma16(ve[e], ph[1][0], o[1][0][e]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              o[1][0][e] = mfma16(ve[e], pl[1][0], o[1][0][e]);
              if (blk + 1 < W) read_k(blk + 1, e);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        __syncthreads();   // the round's blocks are done with
      }
#pragma unroll
      for (int ct = 0; ct < kWideTiles; ++ct) {
        const int first = c0 + 16 * ct;
        if (first >= cols) break;   // uniform
        float sum = lsum[ct];
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        auto partial = [&](int c) {
          return int64_t(columns.pairs[2 * columns.pair(c) + 1] + place) * a.num_qo_heads +
                 columns.head(c);
        };
        if (not_finite<D>(o[ct])) {
#pragma unroll 1
          for (int c = first; c < min(first + 16, cols); ++c) {
            float m1, l1, acc[8];
            wave_rows<T, D>(a, load_v8<T>(columns.q(a, c) + 8 * lcol), kb, vb, tb, tb, STEP, te,
                            s_pages, nr, m1, l1, acc);
            const int64_t row = partial(c);
            if (lrow == 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                a.part_o[row * D + 8 * lcol + e] = l1 == 0.f ? 0.f : acc[e] / l1;
              if (lcol == 0) a.part_lse[row] = partial_lse(m1, l1);
            }
          }
        } else if (first + j < cols) {
          const int64_t row = partial(first + j);
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int half = 0; half < 2; ++half)   // dims 8 (4 tg + x) + 4 half ..
              *reinterpret_cast<f32x4*>(a.part_o + row * D + 8 * (4 * tg + x) + 4 * half) =
                  f32x4{o[ct][0][4 * half][x], o[ct][0][4 * half + 1][x],
                        o[ct][0][4 * half + 2][x], o[ct][0][4 * half + 3][x]} * inv;
          if (tg == 0) a.part_lse[row] = partial_lse(m[ct], sum);
        }
      }
      return;
    }
  }

  // What stands between a workgroup's start and its first K and V is all that
  // short tails wait for (2 us for each read that depends on another, while others
  // stream): the first steps' page ids come with the plan, later ones into a register,
  // a step ahead; q and the new row behind K and V; no barrier. 64 rows behind 2048
  // tokens with tails of 16 to 1500, 32 heads on 8: 47.5 us a layer against 50.
  bool any_bad = false;
  int ids = 0, ids_next = 0;   // lane h: the step's id(h)
  constexpr bool kIds = D != 256;   // there the registers are short, and q waits at a barrier
  if (!scalar || !kIds) {
    any_bad = stage_pages();
  } else if (wave_s < nsteps) {
    ids = tail ? sa.first_ids[(item * W + wave_s) * sa.step_ids + min(lane, sa.step_ids - 1)]
               : ids_of(wave_s);
    ids_next = ids_of(wave_s + W);
  }
  int token;
  if (tail) {   // uniform
    token = a.q_token ? a.q_token[columns.seq] : columns.seq;
    nr = new_row(a, columns.seq, token, hkv);
  } else {
    token = columns.token(a, min(j, cols - 1));
  }
  const bool has_new = nr.pos >= tb && nr.pos < te;   // uniform; then te - 1
  if (scalar && wave_s < nsteps) {
    if constexpr (kIds)
      find_ids(wave_s, ids);
    else
      find_step(wave_s);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_rows(i);
  }
  V8 qb[kQInLds ? 1 : KS];
  if constexpr (kQInLds) {
    for (int i = tid; i < 16 * L::CH; i += W * kWave) {
      const int g = i / L::CH, c = i % L::CH;
      *reinterpret_cast<V8*>(&s_q[g * D + 8 * (c ^ (g & 7))]) =
          g < cols ? load_v8<T>(columns.q(a, g) + 8 * c) : V8{};
    }
    __syncthreads();
  } else {
    const f16* qp = a.q + int64_t(token) * a.q_tok +
                    int64_t(columns.head(min(j, cols - 1))) * a.q_head + 8 * tg;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = j < cols ? load_v8<T>(qp + 32 * s) : V8{};
  }
  // The new row: to LDS and into its page by the wave that has the last step; lane
  // c chunk c, K's first.
  if (scalar && has_new && wave_s == (nsteps - 1) % W && lane < 2 * L::CH) {
    const bool of_v = lane >= L::CH;
    f16* base = const_cast<f16*>(of_v ? a.v : a.k) + int64_t(hkv) * a.head_stride + 8 * lcol;
    const V8 row = load_v8<T>(base + (of_v ? nr.v : nr.k));
    *reinterpret_cast<V8*>(&s_new[8 * lane]) = row;
    const int p = page_id(np - 1);
    if (p >= 0 && hq0 % a.ratio == 0)
      *reinterpret_cast<V8*>(base + int64_t(p) * a.page_stride +
                             int64_t(nr.pos & page_mask) * a.token_stride) = row;
  }
  __builtin_amdgcn_wave_barrier();
  f32x4 o[L::ACCS][8];
#pragma unroll
  for (int x = 0; x < L::ACCS; ++x)
#pragma unroll
    for (int e = 0; e < 8; ++e) o[x][e] = f32x4{};
  float m = kNegBig, lsum = 0.f;
  if (!scalar) {
    if (has_new && hq0 % a.ratio == 0)
      append_row<D>(a, nr, s_pages[(nr.pos >> a.page_shift) - pb], hkv);
    if (wave_s < nsteps) load_lanes(wave_s);
  }
  for (int c = wave_s; c < nsteps; c += W) {
    const int t0 = tb + c * STEP;
    const int gone = dropped;   // of this step
    if (scalar) {
      if (t0 + STEP >= te) {   // uniform, the last step: rows past the end, and the new one
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int t = t0 + TPL * i + lrow;
          if (t >= te) v[i] = V8{};
          if (has_new && t == nr.pos) {
            k[i] = *reinterpret_cast<const V8*>(&s_new[8 * lcol]);
            v[i] = *reinterpret_cast<const V8*>(&s_new[D + 8 * lcol]);
          }
        }
      }
      if (gone) drop_rows();   // uniform
    }
    park();
    V8 vt[8];
    transpose8(v, vt);
    if (!scalar) {
      load_lanes(c + W);
    } else if (c + W < nsteps) {
      if constexpr (kIds) {
        ids = ids_next;
        ids_next = ids_of(c + 2 * W);
        find_ids(c + W, ids);
      } else {
        find_step(c + W);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load_rows(i);
    }
    // LDS runs a wave's accesses in order; keep the compiler from moving them.
    f32x4 sc[PAIRS][2];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < PAIRS; ++p)
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        sc[p][sub] = f32x4{};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const V8 ka = k_row(sk, p, sub, s);
          V8 qs;
          if constexpr (kQInLds)
            qs = *reinterpret_cast<const V8*>(&s_q[j * D + 8 * ((4 * s + tg) ^ (j & 7))]);
          else
            qs = qb[s];
          sc[p][sub] = mfma16(ka, qs, sc[p][sub]);
        }
      }
    __builtin_amdgcn_wave_barrier();
    if (any_bad || (scalar && gone) || t0 + STEP > te) {   // uniform
      if (scalar)
        mask_loads<D>(sc, t0, te, tg, gone);
      else
        mask_scores<D>(sc, t0, te, tg, any_bad, s_pages, a.page_shift, pb);
    }
    V8 ph[L::ACCS], pl[L::ACCS];
    tile_max<D>(sc, a.scale_log2, m, lsum, o);
    tile_exp<T, D>(sc, a.scale_log2, m, lsum, ph, pl);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int x = 0; x < L::ACCS; ++x) o[x][e] = mfma16(vt[e], ph[x], o[x][e]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int x = 0; x < L::ACCS; ++x) o[x][e] = mfma16(vt[e], pl[x], o[x][e]);
  }

  // The waves' sums joined, and the columns' outputs or partials written.
  lsum += __shfl_xor(lsum, 16);
  lsum += __shfl_xor(lsum, 32);
  if constexpr (D == 256) lsum *= 0.5f;   // every token is in two of the groups
  // At 64 a group's rows are chunks 4 (tg % 2) + row of set tg / 2's tokens: add
  // the other set's, held by group tg ^ 2.
  if constexpr (D == 64) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float own = tg >> 1 ? o[1][e][x] : o[0][e][x];
        o[0][e][x] = own + __shfl_xor(own, 32);
      }
  }
  const bool again = not_finite<D>(o);
  __syncthreads();   // every wave is done with its K block
  float* s_o = reinterpret_cast<float*>(s_raw);
  auto unit_at = [&](int g, int unit) { return &s_o[(wave * 16 + g) * D + 4 * (unit ^ (g & 7))]; };
  if (again) {
    if (scalar)   // every wave that comes here the same
      for (int i = lane; i < np; i += kWave) s_pages[i] = page_id(i);
#pragma unroll 1
    for (int g = 0; g < cols; ++g) {
      float m1, l1, acc[8];
      wave_rows<T, D>(a, load_v8<T>(columns.q(a, g) + 8 * lcol), kb, vb, tb, tb + wave * STEP,
                      W * STEP, te, s_pages, nr, m1, l1, acc);
      if (lrow == 0) {
        if (lcol == 0) {
          s_m[wave][g] = m1;
          s_l[wave][g] = l1;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
          *reinterpret_cast<f32x4*>(unit_at(g, 2 * lcol + half)) =
              f32x4{acc[4 * half], acc[4 * half + 1], acc[4 * half + 2], acc[4 * half + 3]};
      }
    }
  } else if (j < cols) {
    if (tg == 0) {
      s_m[wave][j] = m;
      s_l[wave][j] = lsum;
    }
    if (D != 64 || tg < 2) {
#pragma unroll
      for (int x = 0; x < (D == 256 ? 2 : 1); ++x)
#pragma unroll
        for (int row = 0; row < 4; ++row)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // dims 8 (4 tg + row + 16 x) + 4 half ..
            const int unit = 2 * (4 * tg + row + 16 * x) + half;
            *reinterpret_cast<f32x4*>(unit_at(j, unit)) =
                f32x4{o[x][4 * half][row], o[x][4 * half + 1][row], o[x][4 * half + 2][row],
                      o[x][4 * half + 3][row]};
          }
    }
  }
  __syncthreads();
  for (int idx = tid; idx < cols * (D / 4); idx += W * kWave) {
    const int g = idx / (D / 4), unit = idx % (D / 4);
    float mxw = kNegBig;
#pragma unroll
    for (int wv = 0; wv < W; ++wv) mxw = fmaxf(mxw, s_m[wv][g]);
    float sum = 0.f;
    f32x4 x = {};
#pragma unroll
    for (int wv = 0; wv < W; ++wv) {
      const float f = fast_exp2(s_m[wv][g] - mxw);
      sum += s_l[wv][g] * f;
      x += *reinterpret_cast<const f32x4*>(&s_o[(wv * 16 + g) * D + 4 * (unit ^ (g & 7))]) * f;
    }
    x = sum == 0.f ? f32x4{} : x / sum;
    if (tail && slot < 0) {
      T* op = reinterpret_cast<T*>(a.out) + int64_t(columns.token(a, g)) * a.o_tok +
              int64_t(hq0 + g) * a.o_head + 4 * unit;
#pragma unroll
      for (int i = 0; i < 4; ++i) op[i] = T(x[i]);
      continue;
    }
    const int64_t row = int64_t(tail ? slot : columns.pairs[2 * columns.pair(g) + 1] + place) *
                            a.num_qo_heads + columns.head(g);
    *reinterpret_cast<f32x4*>(a.part_o + row * D + 4 * unit) = x;
    if (unit == 0) a.part_lse[row] = partial_lse(mxw, sum);
  }
}

template <typename T, int D>
int launch_shared(const SharedArgs& a, bool wide, unsigned blocks, hipStream_t s) {
  if (wide && D == 128)
    shared_decode_kernel<T, D, D == 128><<<blocks, kThreads, 0, s>>>(a);
  else
    shared_decode_kernel<T, D, false><<<blocks, kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

template <typename T>
int launch_shared_dim(int head_dim, const SharedArgs& a, bool wide, unsigned blocks,
                      hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_shared<T, 64>(a, wide, blocks, s);
    case 128: return launch_shared<T, 128>(a, wide, blocks, s);
    default: return launch_shared<T, 256>(a, wide, blocks, s);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Page ids that a step of a wave's tokens needs (shared_decode_kernel's `granule`); none
// where the kernel looks each row up.
struct StepIds {
  int32_t step, granule, count;
};
StepIds step_ids(int head_dim, int page_size) {
  const int32_t step = head_dim == 64 ? DecodeTile<64>::STEP
                       : head_dim == 128 ? DecodeTile<128>::STEP : DecodeTile<256>::STEP;
  const int32_t load = step / DecodeTile<64>::LOADS;
  if (page_size < load) return {step, 1, 0};
  const int32_t granule = page_size >= 16 ? 16 : load;
  return {step, granule, step / granule};
}

// Tokens [begin, end) that rows order[lo, hi) hold in the same pages.
struct Segment {
  int32_t lo, hi, begin, end;
};

// The prefix tree of rows whose lists (`pages[b]`, `count[b]` ids) may be
// shared, depth first; `order` lists the rows so that a segment's are together.
void find_segments(const std::vector<const int32_t*>& pages, const std::vector<int32_t>& count,
                   int32_t page_size, std::vector<int32_t>& order, std::vector<Segment>& segments) {
  order.resize(pages.size());
  for (size_t b = 0; b < order.size(); ++b) order[b] = int32_t(b);
  auto common = [&](int32_t x, int32_t y, int32_t from) {   // equal leading ids
    const int32_t n = std::min(count[x], count[y]);
    return int32_t(std::mismatch(pages[x] + std::min(from, n), pages[x] + n,
                                 pages[y] + std::min(from, n)).first - pages[x]);
  };
  std::stable_sort(order.begin(), order.end(), [&](int32_t x, int32_t y) {
    const int32_t n = common(x, y, 0);
    if (n == count[x] || n == count[y]) return count[x] < count[y];
    return pages[x][n] < pages[y][n];
  });
  struct Node {
    int32_t lo, hi, begin;   // rows order[lo, hi) agree on their first `known` pages and have
    int32_t known;           // had theirs up to `begin` taken
  };
  std::vector<Node> todo{{0, int32_t(order.size()), 0, 0}};
  while (!todo.empty()) {
    Node n = todo.back();
    todo.pop_back();
    if (n.hi - n.lo < 2) continue;
    const int32_t same = common(order[n.lo], order[n.hi - 1], n.known);
    if (int64_t(same - n.begin) * page_size >= kMinSegmentTokens) {
      segments.push_back({n.lo, n.hi, n.begin * page_size, same * page_size});
      n.begin = same;
    }
    // Children: rows by their next page; those that have none stand alone.
    int32_t at = n.lo;
    while (at < n.hi && count[order[at]] == same) ++at;
    while (at < n.hi) {
      int32_t end = at + 1;
      while (end < n.hi && pages[order[end]][same] == pages[order[at]][same]) ++end;
      if (end - at > 1) todo.push_back({at, end, n.begin, same + 1});
      at = end;
    }
  }
}

int shared_plan(const int32_t* indptr, const int32_t* indices, const int32_t* kv_len,
                int32_t num_seqs, int32_t num_qo_heads, int32_t num_kv_heads, int32_t page_size,
                int32_t head_dim, int32_t num_cus, int64_t min_bytes, std::vector<int32_t>& plan,
                kunserve_shared_plan_info* info) {
  const int group = decode_group(num_qo_heads, num_kv_heads);
  const int64_t head_groups = num_qo_heads / group;
  const int64_t cus = std::max(num_cus, 1);
  std::vector<const int32_t*> pages(num_seqs);
  std::vector<int32_t> count(num_seqs);
  for (int32_t b = 0; b < num_seqs; ++b) {
    const int64_t held = int64_t(indptr[b + 1]) - indptr[b];
    KSV_CHECK_ARG(kv_len[b] >= 0 && held >= ceil_div(kv_len[b], page_size),
                  "row %d: %lld pages for %d tokens", b, (long long)held, kv_len[b]);
    pages[b] = indices + indptr[b];
    // Whole pages before the new token's: a row always has a tail.
    count[b] = std::max(kv_len[b] - 1, 0) / page_size;
  }
  std::vector<int32_t> order;
  std::vector<Segment> segments;
  find_segments(pages, count, page_size, order, segments);
  int64_t saved = 0;   // K and V tokens that are not read again
  for (const Segment& s : segments) saved += int64_t(s.end - s.begin) * (s.hi - s.lo - 1);
  if (saved * num_kv_heads * head_dim * 4 < (min_bytes < 0 ? kMinSavedBytes * cus / 256 : min_bytes))
    segments.clear();

  // Segments in workgroups of whole rows (group is 16 at most). Wide ones where
  // narrow ones would keep the CUs busy for long: they read K and V once for
  // eight times as many columns, but take about 10 us to begin and end, and their
  // number is an eighth. Per layer, 8 KV heads of 128, tails of 20-100, narrow against
  // wide: 64 columns of 4000 tokens (a CU's share 6 us) 16.4 against 22.4, 160 of 3000
  // (11 us) 21.1 against 26.8, 320 of 3000 (22 us) 31.4 against 32.1, 256 of 8000 (46 us)
  // 41.6 against 34.8.
  double narrow_work = 0.0;
  // A token, of a workgroup (grouped_part_tokens: 11.5 ns at head_dim 128, 30 at 256).
  const double narrow_us = 0.0115 * std::pow(head_dim / 128.0, 1.4);
  int64_t tail_tokens = 0;
  for (int32_t b = 0; b < num_seqs; ++b) tail_tokens += kv_len[b];
  for (const Segment& s : segments) {
    narrow_work += narrow_us * double(s.end - s.begin) *
                   double(ceil_div(s.hi - s.lo, 16 / group) * head_groups);
    tail_tokens -= int64_t(s.end - s.begin) * (s.hi - s.lo);
  }
  auto is_wide = [&](const Segment& s) {
    return head_dim == 128 && (s.hi - s.lo) * group >= kMinWideCols &&
           narrow_work >= kMinWideShareUs * double(cus);
  };
  auto tile_rows = [&](const Segment& s) { return (is_wide(s) ? kWideCols : 16) / group; };
  auto token_us = [&](const Segment& s) { return is_wide(s) ? 0.035 : narrow_us; };
  double work = 0.0;   // of all segments' workgroups
  info->wide = 0;
  for (const Segment& s : segments) {
    work += token_us(s) * double(s.end - s.begin) *
            double(ceil_div(s.hi - s.lo, tile_rows(s)) * head_groups);
    info->wide |= is_wide(s);
  }
  // A piece takes at most a CU's share of the segments' work (of a long one of narrow
  // workgroups, which run two to a CU, 0.7 at head_dim 128: a few per cent either way.
  // 32 heads on 8 at 0.5, 0.7, 1.0 and 1.4 of a share: 24 rows behind 6000 tokens 24.5, 22.4,
  // 22.9 and 25.0 us, 48 behind 4096 28.1, 26.1, 26.7 and 29.8, 12 behind 12000 23.7, 22.8,
  // 22.5 and 25.5, 16 behind 4000 (6 us of share) 20.0, 17.5, 16.3 and 17.8; head_dim 64, 40
  // behind 3000 21.0, 20.4, 19.5 and 19.2, 32 behind 8000 25.6, 21.6, 23.2 and 24.6; head_dim
  // 256, 40 behind 3000 41.0, 36.3, 35.8 and 37.1), or what ends behind the tails' bytes:
  // fewer pieces are fewer partials. Wide, 128 rows behind 8192 tokens with
  // tails of up to 2000, 64 heads on 8: 110 us in pieces of 2048, 119 in 2752, 124 in 1600,
  // 137 in 1024.
  const double tails_us = double(tail_tokens) * num_kv_heads * head_dim * 4 / (6.6e6 * cus / 256);
  const double share_us = work / double(cus);
  auto pieces_of = [&](const Segment& s) {
    const double share = (is_wide(s) || head_dim != 128 || share_us < 12.0 ? 1.0 : 0.7) * share_us;
    const double most = std::min(double(kMaxPartTokens),
                                 std::max(double(kMinPieceTokens),
                                          std::max(share, 0.8 * tails_us) / token_us(s)));
    return int64_t(std::ceil(double(s.end - s.begin) / most));
  };

  // A row's partials: its segments' pieces, then its tail's partitions.
  std::vector<int32_t> partials(num_seqs, 0), covered(num_seqs, 0);
  struct Piece {
    int32_t segment, begin, end, place;
  };
  std::vector<Piece> pieces;
  for (size_t i = 0; i < segments.size(); ++i) {   // a parent comes before its children
    const Segment& s = segments[i];
    const int32_t len = int32_t(64 * ceil_div(s.end - s.begin, 64 * pieces_of(s)));
    const int32_t first = partials[order[s.lo]];
    int32_t made = 0;
    for (int32_t t = s.begin; t < s.end; t += len, ++made)
      pieces.push_back({int32_t(i), t, std::min(s.end, t + len), first + made});
    for (int32_t r = s.lo; r < s.hi; ++r) {
      partials[order[r]] += made;
      covered[order[r]] = s.end;
    }
  }
  std::vector<int32_t> tails(num_seqs);
  for (int32_t b = 0; b < num_seqs; ++b) tails[b] = kv_len[b] - covered[b];
  const int32_t part = decode_part_tokens(tails.data(), num_seqs, num_qo_heads, group, head_dim,
                                          int32_t(cus));
  std::vector<DecodeItem> items;
  std::vector<int32_t> merges, first_slot(num_seqs, -1);
  int64_t slots = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    const int32_t own = std::max<int32_t>(1, int32_t(ceil_div(tails[b], part)));
    if (partials[b] + own == 1) {
      items.push_back({b, covered[b], kv_len[b], -1});
      continue;
    }
    first_slot[b] = int32_t(slots);
    merges.insert(merges.end(), {b, int32_t(slots), partials[b] + own, 0});
    for (int32_t i = 0; i < own; ++i)
      items.push_back({b, covered[b] + i * part, std::min(kv_len[b], covered[b] + (i + 1) * part),
                       int32_t(slots) + partials[b] + i});
    slots += partials[b] + own;
    KSV_CHECK_ARG(slots < (int64_t(1) << 31), "too many partial results");
  }
  info->decode.num_work = decode_records(items, plan);
  plan.insert(plan.end(), merges.begin(), merges.end());
  info->decode.num_merge = int32_t(merges.size() / 4);
  info->decode.num_slots = int32_t(slots);
  info->decode.part_tokens = part;
  info->decode.group_size = group;
  info->decode.plan_ints = int32_t(plan.size());

  // Work records: the row tiles of a piece and head group, which read the same K
  // and V, on one XCD, one after the other; longest pieces first, to the XCD with
  // least to do.
  std::stable_sort(pieces.begin(), pieces.end(), [](const Piece& x, const Piece& y) {
    return x.end - x.begin > y.end - y.begin;
  });
  std::vector<int32_t> lanes[kXcds], pairs;
  std::vector<int32_t> pair_at(segments.size());
  for (size_t i = 0; i < segments.size(); ++i) {
    pair_at[i] = int32_t(pairs.size() / 2);
    for (int32_t r = segments[i].lo; r < segments[i].hi; ++r)
      pairs.insert(pairs.end(), {order[r], first_slot[order[r]]});
  }
  int64_t load[kXcds] = {};
  size_t depth = 0;
  for (const Piece& p : pieces) {
    const Segment& s = segments[p.segment];
    for (int32_t hg = 0; hg < head_groups; ++hg) {
      const int x = int(std::min_element(load, load + kXcds) - load);
      for (int32_t r = s.lo; r < s.hi; r += tile_rows(s)) {
        lanes[x].insert(lanes[x].end(),
                        {std::min(tile_rows(s), s.hi - r), pair_at[p.segment] + r - s.lo, p.begin,
                         p.end, p.place, order[s.lo], hg, indptr[order[s.lo]]});
        load[x] += p.end - p.begin;
      }
      depth = std::max(depth, lanes[x].size() / kRecord);
    }
  }
  for (size_t r = 0; r < depth; ++r)
    for (int x = 0; x < kXcds; ++x)
      for (int i = 0; i < kRecord; ++i)
        plan.push_back(kRecord * r + i < lanes[x].size() ? lanes[x][kRecord * r + i] : 0);
  plan.insert(plan.end(), pairs.begin(), pairs.end());
  for (int32_t i = 0; i < info->decode.num_work; ++i)
    plan.push_back(plan[4 * i] < 0 ? 0 : indptr[plan[4 * i]]);
  const StepIds ids = step_ids(head_dim, page_size);
  for (int32_t i = 0; i < info->decode.num_work; ++i)
    for (int32_t x = 0; x < kWaves * ids.count; ++x) {
      const int32_t b = plan[4 * i];
      const int32_t t = plan[4 * i + 1] + x / ids.count * ids.step + x % ids.count * ids.granule;
      plan.push_back(b < 0 || kv_len[b] == 0
                         ? -1
                         : pages[b][std::min(t, plan[4 * i + 2] - 1) / page_size]);
    }
  info->num_shared = int32_t(kXcds * depth);
  info->num_pairs = int32_t(pairs.size() / 2);
  info->num_segments = int32_t(segments.size());
  info->head_dim = head_dim;
  info->page_size = page_size;
  info->num_seqs = num_seqs;
  info->num_qo_heads = num_qo_heads;
  info->num_kv_heads = num_kv_heads;
  KSV_CHECK_ARG(plan.size() < (size_t(1) << 31), "the plan is too long");
  info->plan_ints = int32_t(plan.size());
  return KUNSERVE_OK;
}

}  // namespace
}  // namespace kunserve

using namespace kunserve;

extern "C" int64_t kunserve_shared_plan_bound(const int32_t* kv_len_host, int32_t num_seqs,
                                              int32_t num_qo_heads) {
  if (num_seqs < 0 || num_qo_heads <= 0 || (num_seqs > 0 && !kv_len_host)) return -1;
  // A row's partials: pieces and partitions of 64 tokens or more, but the last
  // of each of its segments, of which there is one to kMinSegmentTokens.
  int64_t partials = 0;
  for (int32_t b = 0; b < num_seqs; ++b)
    partials += 2 * ceil_div(std::max(kv_len_host[b], 0), kMinSegmentTokens) + 2;
  return ((5 + 8 * kWaves) * kXcds + kRecord * kXcds * int64_t(num_qo_heads) + 2) * partials +
         4 * int64_t(num_seqs);
}

extern "C" int kunserve_shared_plan(const int32_t* indptr_host, const int32_t* indices_host,
                                    const int32_t* kv_len_host, int32_t num_seqs,
                                    int32_t num_qo_heads, int32_t num_kv_heads, int32_t page_size,
                                    int32_t head_dim, int32_t num_cus, int64_t min_bytes,
                                    int32_t* plan_host, int64_t plan_capacity,
                                    kunserve_shared_plan_info* info) {
  clear_error();
  KSV_CHECK_ARG(info && plan_host, "null plan buffer or info");
  KSV_CHECK_ARG(num_seqs >= 0 && (num_seqs == 0 || (indptr_host && indices_host && kv_len_host)),
                "bad table or num_seqs");
  KSV_CHECK_ARG(num_qo_heads > 0 && num_kv_heads > 0 && num_qo_heads % num_kv_heads == 0,
                "num_qo_heads %d not a multiple of num_kv_heads %d", num_qo_heads, num_kv_heads);
  KSV_CHECK_ARG(page_size >= kMinPageSize && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two >= %d", page_size, kMinPageSize);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("head_dim %d not compiled", head_dim);
    return KUNSERVE_EUNSUPPORTED;
  }
  return no_throw([&] {
    std::vector<int32_t> plan;
    const int rc = shared_plan(indptr_host, indices_host, kv_len_host, num_seqs, num_qo_heads,
                               num_kv_heads, page_size, head_dim, num_cus, min_bytes, plan, info);
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

int kunserve::shared_decode(const kunserve_kv_pool* pool, int32_t layer,
                            const kunserve_page_table* table, const int32_t* q_token_dev,
                            const kunserve_tensor3* q, kunserve_tensor3* out, int32_t num_qo_heads,
                            float sm_scale, const int32_t* plan_dev,
                            const kunserve_shared_plan_info* info, void* workspace_dev,
                            int64_t workspace_bytes, const StepFusion& fusion,
                            kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  KSV_CHECK_ARG(table && q && out && info, "null argument");
  KSV_CHECK_ARG(layer >= 0 && layer < pool->num_layers, "layer %d outside [0, %d)", layer,
                pool->num_layers);
  KSV_CHECK_ARG(std::isfinite(sm_scale) && sm_scale > 0.f,
                "sm_scale %g must be finite and positive", double(sm_scale));
  KSV_CHECK_ARG(num_qo_heads > 0 && num_qo_heads % pool->num_kv_heads == 0,
                "num_qo_heads %d not a multiple of num_kv_heads %d", num_qo_heads,
                pool->num_kv_heads);
  KSV_CHECK_ARG(info->head_dim == pool->head_dim, "plan made for head_dim %d, pool has %d",
                info->head_dim, pool->head_dim);
  KSV_CHECK_ARG(info->page_size == pool->page_size, "plan made for pages of %d, pool has %d",
                info->page_size, pool->page_size);
  KSV_CHECK_ARG(pool->token_stride < (int64_t(1) << 28),
                "tokens %lld elements apart: less than 2^28 here", (long long)pool->token_stride);
  KSV_CHECK_ARG(info->decode.group_size == decode_group(num_qo_heads, pool->num_kv_heads),
                "plan group size %d is not that of %d query heads on %d", info->decode.group_size,
                num_qo_heads, pool->num_kv_heads);
  // The segments' records hold rows and head groups.
  KSV_CHECK_ARG(info->num_qo_heads == num_qo_heads && info->num_kv_heads == pool->num_kv_heads,
                "plan made for %d query heads on %d, not %d on %d", info->num_qo_heads,
                info->num_kv_heads, num_qo_heads, pool->num_kv_heads);
  KSV_CHECK_ARG(info->num_seqs == table->num_seqs, "plan made for %d rows, not %d", info->num_seqs,
                table->num_seqs);
  // Rows that share nothing run in the decode kernels.
  if (info->num_segments == 0)
    return paged_decode(pool, layer, table, q_token_dev, q, out, num_qo_heads, sm_scale, plan_dev,
                        &info->decode, workspace_dev, workspace_bytes, fusion, stream);
  SharedArgs sa{};
  rc = decode_args(pool, layer, table, q_token_dev, q, out, num_qo_heads, sm_scale, plan_dev,
                   &info->decode, workspace_dev, workspace_bytes, fusion, &sa.d);
  if (rc) return rc;
  KSV_CHECK_ARG(aligned16(workspace_dev), "workspace must be 16-byte aligned");
  sa.shared = plan_dev + info->decode.plan_ints;
  sa.pairs = sa.shared + kRecord * int64_t(info->num_shared);
  sa.tail_pages = sa.pairs + 2 * int64_t(info->num_pairs);
  sa.first_ids = sa.tail_pages + info->decode.num_work;
  sa.step_ids = step_ids(pool->head_dim, pool->page_size).count;
  sa.num_shared = info->num_shared;
  sa.inv_group = (65536u + sa.d.group - 1) / sa.d.group;
  sa.inv_head_groups = uint32_t((int64_t(1) << 32) / sa.d.head_groups + 1);
  const int64_t blocks = int64_t(info->num_shared) +
                         8 * ceil_div(info->decode.num_work, 8) * sa.d.head_groups;
  KSV_CHECK_ARG(blocks < (int64_t(1) << 31) && blocks / 8 * sa.d.head_groups < (int64_t(1) << 32),
                "grid of %lld workgroups is too large", (long long)blocks);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  rc = pool->dtype == KUNSERVE_DTYPE_BF16
           ? launch_shared_dim<bf16>(pool->head_dim, sa, info->wide != 0, unsigned(blocks), s)
           : launch_shared_dim<f16>(pool->head_dim, sa, info->wide != 0, unsigned(blocks), s);
  if (rc) return rc;
  return decode_merge(pool, sa.d, &info->decode, plan_dev, s);
}

extern "C" int kunserve_shared_decode(const kunserve_kv_pool* pool, int32_t layer,
                                      const kunserve_page_table* table,
                                      const int32_t* q_token_dev, const kunserve_tensor3* q,
                                      kunserve_tensor3* out, int32_t num_qo_heads, float sm_scale,
                                      const int32_t* plan_dev,
                                      const kunserve_shared_plan_info* info, void* workspace_dev,
                                      int64_t workspace_bytes, kunserve_stream_t stream) {
  return kunserve::shared_decode(pool, layer, table, q_token_dev, q, out, num_qo_heads, sm_scale,
                                 plan_dev, info, workspace_dev, workspace_bytes, StepFusion{},
                                 stream);
}
