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
// split row are. The tails run in the decode kernels (paged_decode); this
// file holds the plan and the kernel of the segments.
//
// The kernel has the (row, query head of a KV head) pairs of a segment as the
// columns of its products, up to 64 to a workgroup. K and V are read, parked
// and transposed as in paged_decode_mfma_kernel; a step's operands serve every
// 16-column tile, so a segment costs its bytes once and the matrix units
// 16 columns at a time.
#include <algorithm>
#include <cmath>
#include <vector>

#include "decode_tile.hpp"

namespace kunserve {
namespace {

constexpr int kMinSegmentTokens = 64;   // shorter runs of shared pages stay with their rows
constexpr int kRecord = 8;              // ints of a work record
constexpr int kMinPieceTokens = 128;

struct SharedArgs {
  DecodeArgs d;
  const int32_t* shared;   // [num_shared][kRecord]: rows (0: padding), their first pair,
                           // token begin, end, place among a row's partials, a row of them
  const int32_t* pairs;    // [...][2]: row, its first slot
  int32_t num_shared;
};

// Columns of a workgroup: 16-column tiles as the accumulators allow.
constexpr int max_tiles(int head_dim) { return head_dim == 128 ? 4 : 2; }

template <typename T, int D, int CT>
__global__ __launch_bounds__(kThreads, (CT == 4 || (CT == 2 && D == 256) ? 1 : 2)) void shared_decode_kernel(SharedArgs sa) {
  typedef typename Vec<T>::v8 V8;
  typedef DecodeTile<D> L;
  constexpr int STEP = L::STEP, TPL = L::TPL, LOADS = L::LOADS, PAIRS = L::PAIRS;
  constexpr int BLK = STEP * D;
  constexpr int KS = D / 32;
  constexpr int W = kWaves;
  constexpr int COLS = 16 * CT;

  const DecodeArgs& a = sa.d;
  __shared__ int s_pages[kMaxPartPages];
  __shared__ int s_bad[W];
  // The waves' K blocks; after the loop, their O of 16 columns (fp32).
  constexpr int kKBytes = W * BLK * int(sizeof(T)), kOBytes = W * 16 * D * int(sizeof(float));
  __shared__ __attribute__((aligned(16))) char s_raw[kKBytes > kOBytes ? kKBytes : kOBytes];
  __shared__ float s_m[W][16];
  __shared__ float s_l[W][16];
  __shared__ __attribute__((aligned(16))) T s_q[COLS * D];   // column g's chunk c at c ^ (g & 7)

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = tid >> 6;
  const int j = lane & 15;
  const int tg = lane >> 4;
  const int lrow = lane / L::CH;
  const int lcol = lane % L::CH;
  const int G = a.group;

  const int b = int(blockIdx.x);
  const int local = (b >> 3) / a.head_groups;
  const int hg = (b >> 3) - local * a.head_groups;
  const int item = 8 * local + (b & 7);
  if (item >= sa.num_shared) return;   // uniform, as the next
  const int32_t* rec = sa.shared + kRecord * item;
  const int nrows = rec[0];
  if (nrows <= 0) return;
  const int32_t* pairs = sa.pairs + 2 * rec[1];
  const int tb = rec[2], te = rec[3], place = rec[4], rep = rec[5];
  const int cols = nrows * G;
  const int ntiles = (cols + 15) >> 4;
  const int hq0 = hg * G;
  const int hkv = hq0 / a.ratio;
  const int page_mask = (1 << a.page_shift) - 1;
  auto q_row = [&](int c) {   // q of column c
    const int seq = pairs[2 * (c / G)];
    const int tok = a.q_token ? a.q_token[seq] : seq;
    return a.q + int64_t(tok) * a.q_tok + int64_t(hq0 + c % G) * a.q_head;
  };

  const int pb = tb >> a.page_shift;
  const int np = ((te - 1) >> a.page_shift) + 1 - pb;
  const int32_t* seq_pages = a.indices + a.indptr[rep];
  bool bad_id = false;
  for (int i = tid; i < np; i += W * kWave) {
    const int p = seq_pages[pb + i];
    const bool ok = p >= 0 && p < a.num_pages;
    s_pages[i] = ok ? p : -1;
    bad_id |= !ok;
  }
  const bool wave_bad = __any(bad_id);
  if (lane == 0) s_bad[wave] = wave_bad;
  for (int i = tid; i < COLS * L::CH; i += W * kWave) {
    const int g = i / L::CH, c = i % L::CH;
    *reinterpret_cast<V8*>(&s_q[g * D + 8 * (c ^ (g & 7))]) =
        g < cols ? load_v8<T>(q_row(g) + 8 * c) : V8{};
  }
  f32x4 o[CT][L::ACCS][8];
  float m[CT], lsum[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = kNegBig;
    lsum[ct] = 0.f;
#pragma unroll
    for (int x = 0; x < L::ACCS; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[ct][x][e] = f32x4{};
  }
  __syncthreads();
  int bad_votes = 0;
#pragma unroll
  for (int wv = 0; wv < W; ++wv) bad_votes |= s_bad[wv];
  const bool any_bad = __builtin_amdgcn_readfirstlane(bad_votes) != 0;

  const f16* kb = a.k + int64_t(hkv) * a.head_stride + lcol * 8;
  const f16* vb = a.v + int64_t(hkv) * a.head_stride + lcol * 8;
  const int nsteps = (te - tb + STEP - 1) / STEP;
  T* sk = reinterpret_cast<T*>(s_raw) + wave * BLK;

  V8 k[LOADS], v[LOADS];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = tb + c * STEP + TPL * i + lrow;
      const int pi = min((t >> a.page_shift) - pb, kMaxPartPages - 1);
      const int p = (c < nsteps && t < te) ? s_pages[pi] : -1;
      const int64_t off = int64_t(max(p, 0)) * a.page_stride + int64_t(t & page_mask) * a.token_stride;
      k[i] = load_v8<T>(p >= 0 ? kb + off : g_zero_row + lcol * 8);
      v[i] = load_v8<T>(p >= 0 ? vb + off : g_zero_row + lcol * 8);
    }
  };
  if (wave < nsteps) load(wave);
  for (int c = wave; c < nsteps; c += W) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = TPL * i + lrow;
      *reinterpret_cast<V8*>(&sk[t * D + ((lcol ^ L::swz(t)) << 3)]) = k[i];
    }
    V8 vt[8];   // vt[e]: dim 8 lcol + e of the lane's 8 tokens
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
    load(c + W);

    // LDS runs a wave's accesses in order; keep the compiler from moving them.
    __builtin_amdgcn_wave_barrier();
    V8 ka[PAIRS][2][KS];
#pragma unroll
    for (int p = 0; p < PAIRS; ++p)
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int t = L::token(4 * sub + (j & 3), j >> 2, p);   // tile row j
#pragma unroll
        for (int s = 0; s < KS; ++s)
          ka[p][sub][s] = *reinterpret_cast<const V8*>(&sk[t * D + (((4 * s + tg) ^ L::swz(t)) << 3)]);
      }
    __builtin_amdgcn_wave_barrier();
    const int t0 = tb + c * STEP;
    const bool whole = !any_bad && t0 + STEP <= te;   // uniform: nothing to mask
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if (ct >= ntiles) break;   // uniform
      V8 qs[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s)
        qs[s] = *reinterpret_cast<const V8*>(&s_q[(16 * ct + j) * D + 8 * ((4 * s + tg) ^ (j & 7))]);
      f32x4 sc[PAIRS][2];
      float mx = -INFINITY;
#pragma unroll
      for (int p = 0; p < PAIRS; ++p)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          sc[p][sub] = f32x4{};
#pragma unroll
          for (int s = 0; s < KS; ++s) sc[p][sub] = mfma16(ka[p][sub][s], qs[s], sc[p][sub]);
          if (!whole) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int t = t0 + L::token(4 * sub + x, tg, p);
              bool drop = t >= te;
              if (any_bad) drop |= s_pages[min((min(t, te - 1) >> a.page_shift) - pb, kMaxPartPages - 1)] < 0;
              if (drop) sc[p][sub][x] = -INFINITY;
            }
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) mx = fmaxf(mx, sc[p][sub][x]);
        }
      mx = groups_max(mx) * a.scale_log2;
      if (__any(mx > m[ct] + 8.f)) {
        const float m_new = mx > m[ct] + 8.f ? mx : m[ct];
        const float alpha = fast_exp2(m[ct] - m_new);
        m[ct] = m_new;
        lsum[ct] *= alpha;
#pragma unroll
        for (int x = 0; x < L::ACCS; ++x)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[ct][x][e] *= alpha;
      }
      V8 ph[L::ACCS], pl[L::ACCS];   // probabilities: rounded, and what rounding left
#pragma unroll
      for (int p = 0; p < PAIRS; ++p)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float pr = fast_exp2(fmaf(sc[p][sub][x], a.scale_log2, -m[ct]));
            lsum[ct] += pr;
            const T hi = T(pr);
            ph[p][4 * sub + x] = hi;
            pl[p][4 * sub + x] = T(pr - float(hi));
          }
      if constexpr (D == 256) {   // set x takes the lane groups of its half of the row
        const V8 zero = {};
        ph[1] = (tg & 1) ? ph[0] : zero;
        pl[1] = (tg & 1) ? pl[0] : zero;
        ph[0] = (tg & 1) ? zero : ph[0];
        pl[0] = (tg & 1) ? zero : pl[0];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < L::ACCS; ++x) {
          o[ct][x][e] = mfma16(vt[e], ph[x], o[ct][x][e]);
          o[ct][x][e] = mfma16(vt[e], pl[x], o[ct][x][e]);
        }
    }
  }

  // Tile by tile: the waves' sums joined, and the columns' partials written.
  float* s_o = reinterpret_cast<float*>(s_raw);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (ct >= ntiles) break;   // uniform
    float ls = lsum[ct];
    ls += __shfl_xor(ls, 16);
    ls += __shfl_xor(ls, 32);
    if constexpr (D == 256) ls *= 0.5f;   // every token is in two of the groups
    // At 64 a group's rows are chunks 4 (tg % 2) + row of set tg / 2's tokens:
    // add the other set's, held by group tg ^ 2.
    if constexpr (D == 64) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float own = tg >> 1 ? o[ct][1][e][x] : o[ct][0][e][x];
          o[ct][0][e][x] = own + __shfl_xor(own, 32);
        }
    }
    // Infinite and NaN values of V, as in paged_decode_mfma_kernel.
    float z[4] = {};
#pragma unroll
    for (int x = 0; x < (D == 256 ? 2 : 1); ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = fmaf(o[ct][x][e][i], 0.f, z[i]);
    const bool again = __any(!(z[0] + z[1] + z[2] + z[3] == 0.f));
    const int here = min(16, cols - 16 * ct);   // columns of this tile
    __syncthreads();   // the K blocks, or the tile before, are done with
    auto unit_at = [&](int g, int unit) { return &s_o[(wave * 16 + g) * D + 4 * (unit ^ (g & 7))]; };
    if (again) {
#pragma unroll 1
      for (int g = 0; g < here; ++g) {
        float m1, l1, acc[8];
        wave_rows<T, D, W>(a, load_v8<T>(q_row(16 * ct + g) + 8 * lcol), kb, vb, tb, te, s_pages,
                           NewRow{-1, 0, 0}, m1, l1, acc);
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
    } else if (j < here) {
      if (tg == 0) {
        s_m[wave][j] = m[ct];
        s_l[wave][j] = ls;
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
                  f32x4{o[ct][x][4 * half][row], o[ct][x][4 * half + 1][row],
                        o[ct][x][4 * half + 2][row], o[ct][x][4 * half + 3][row]};
            }
      }
    }
    __syncthreads();
    for (int idx = tid; idx < here * (D / 4); idx += W * kWave) {
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
      const int c = 16 * ct + g;
      const int64_t row = int64_t(pairs[2 * (c / G) + 1] + place) * a.num_qo_heads + hq0 + c % G;
      // A NaN score makes the columns' outputs NaN, at whatever weight.
      *reinterpret_cast<f32x4*>(a.part_o + row * D + 4 * unit) = sum == 0.f ? f32x4{} : x / sum;
      if (unit == 0)
        a.part_lse[row] = sum > 0.f ? mxw + __log2f(sum) : sum == 0.f ? -INFINITY : mxw;
    }
  }
}

template <typename T, int D>
int launch_shared(const SharedArgs& a, int tiles, unsigned blocks, hipStream_t s) {
  if (tiles == 1)
    shared_decode_kernel<T, D, 1><<<blocks, kThreads, 0, s>>>(a);
  else if (tiles == 2)
    shared_decode_kernel<T, D, 2><<<blocks, kThreads, 0, s>>>(a);
  else
    shared_decode_kernel<T, D, max_tiles(D)><<<blocks, kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

template <typename T>
int launch_shared_dim(int head_dim, const SharedArgs& a, int tiles, unsigned blocks,
                      hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_shared<T, 64>(a, tiles, blocks, s);
    case 128: return launch_shared<T, 128>(a, tiles, blocks, s);
    default: return launch_shared<T, 256>(a, tiles, blocks, s);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

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
                int32_t head_dim, int32_t num_cus, std::vector<int32_t>& plan,
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

  // Segments in workgroups of whole rows; pieces of their tokens so that the
  // device is filled once.
  int32_t tiles = 1;
  for (const Segment& s : segments)
    tiles = std::max<int64_t>(tiles, std::min<int64_t>(max_tiles(head_dim),
                                                       ceil_div(int64_t(s.hi - s.lo) * group, 16)));
  if (tiles == 3) tiles = 4;
  const int32_t tile_rows = 16 * tiles / group;   // group is 16 at most
  int64_t work = 0;
  for (const Segment& s : segments)
    work += int64_t(s.end - s.begin) * ceil_div(s.hi - s.lo, tile_rows) * head_groups;
  const int64_t piece = std::min<int64_t>(
      kMaxPartTokens, std::max<int64_t>(kMinPieceTokens, 64 * ceil_div(work, 64 * cus)));

  // A row's partials: its segments' pieces, then its tail's partitions.
  std::vector<int32_t> partials(num_seqs, 0), covered(num_seqs, 0);
  struct Piece {
    int32_t segment, begin, end, place;
  };
  std::vector<Piece> pieces;
  for (size_t i = 0; i < segments.size(); ++i) {   // a parent comes before its children
    const Segment& s = segments[i];
    const int32_t n = int32_t(ceil_div(s.end - s.begin, piece));
    const int32_t len = int32_t(64 * ceil_div(s.end - s.begin, 64 * int64_t(n)));
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

  // Work records: a piece's row tiles on one XCD, one after the other (they
  // read the same K and V), longest pieces first, to the XCD with least to do.
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
    const int x = int(std::min_element(load, load + kXcds) - load);
    for (int32_t r = s.lo; r < s.hi; r += tile_rows) {
      lanes[x].insert(lanes[x].end(), {std::min(tile_rows, s.hi - r), pair_at[p.segment] + r - s.lo,
                                       p.begin, p.end, p.place, order[s.lo], 0, 0});
      load[x] += p.end - p.begin;
    }
    depth = std::max(depth, lanes[x].size() / kRecord);
  }
  for (size_t r = 0; r < depth; ++r)
    for (int x = 0; x < kXcds; ++x)
      for (int i = 0; i < kRecord; ++i)
        plan.push_back(kRecord * r + i < lanes[x].size() ? lanes[x][kRecord * r + i] : 0);
  plan.insert(plan.end(), pairs.begin(), pairs.end());
  info->num_shared = int32_t(kXcds * depth);
  info->tiles = tiles;
  info->num_pairs = int32_t(pairs.size() / 2);
  info->num_segments = int32_t(segments.size());
  info->head_dim = head_dim;
  KSV_CHECK_ARG(plan.size() < (size_t(1) << 31), "the plan is too long");
  info->plan_ints = int32_t(plan.size());
  return KUNSERVE_OK;
}

}  // namespace
}  // namespace kunserve

using namespace kunserve;

extern "C" int64_t kunserve_shared_plan_bound(const int32_t* kv_len_host, int32_t num_seqs) {
  if (num_seqs < 0 || (num_seqs > 0 && !kv_len_host)) return -1;
  // A row's partials: pieces and partitions of 64 tokens or more, but the last
  // of each of its segments, of which there is one to kMinSegmentTokens.
  int64_t partials = 0;
  for (int32_t b = 0; b < num_seqs; ++b)
    partials += 2 * ceil_div(std::max(kv_len_host[b], 0), kMinSegmentTokens) + 2;
  return (4 * kXcds + kRecord * kXcds + 2) * partials + 4 * int64_t(num_seqs);
}

extern "C" int kunserve_shared_plan(const int32_t* indptr_host, const int32_t* indices_host,
                                    const int32_t* kv_len_host, int32_t num_seqs,
                                    int32_t num_qo_heads, int32_t num_kv_heads, int32_t page_size,
                                    int32_t head_dim, int32_t num_cus, int32_t* plan_host,
                                    int64_t plan_capacity, kunserve_shared_plan_info* info) {
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
                               num_kv_heads, page_size, head_dim, num_cus, plan, info);
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
  KSV_CHECK_ARG(info->decode.group_size == decode_group(num_qo_heads, pool->num_kv_heads),
                "plan group size %d is not that of %d query heads on %d", info->decode.group_size,
                num_qo_heads, pool->num_kv_heads);
  if (info->num_shared > 0) {
    KSV_CHECK_ARG(plan_dev && table->indptr_dev && table->indices_dev, "null plan or table");
    KSV_CHECK_ARG(q->data && aligned16(q->data) && q->token_stride % 8 == 0 &&
                      q->head_stride % 8 == 0,
                  "q must be 16-byte aligned with strides that are multiples of 8");
    const int64_t need =
        kunserve_decode_workspace_bytes(&info->decode, num_qo_heads, pool->head_dim);
    if (!workspace_dev || workspace_bytes < need) {
      set_error("decode workspace holds %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)need);
      return KUNSERVE_ENOSPC;
    }
    KSV_CHECK_ARG(aligned16(workspace_dev), "workspace must be 16-byte aligned");
    SharedArgs sa{};
    DecodeArgs& a = sa.d;
    a.q_token = q_token_dev;
    a.q = static_cast<const f16*>(q->data);
    a.q_tok = q->token_stride;
    a.q_head = q->head_stride;
    a.k = static_cast<const f16*>(pool->k) + int64_t(layer) * pool->layer_stride;
    a.v = static_cast<const f16*>(pool->v) + int64_t(layer) * pool->layer_stride;
    a.page_stride = pool->page_stride;
    a.head_stride = pool->head_stride;
    a.token_stride = pool->token_stride;
    a.num_pages = int32_t(pool->num_pages);
    a.page_shift = __builtin_ctz(pool->page_size);
    a.indptr = table->indptr_dev;
    a.indices = table->indices_dev;
    a.part_o = static_cast<float*>(workspace_dev);
    a.part_lse = a.part_o + int64_t(info->decode.num_slots) * num_qo_heads * pool->head_dim;
    a.num_qo_heads = num_qo_heads;
    a.group = info->decode.group_size;
    a.head_groups = num_qo_heads / a.group;
    a.ratio = num_qo_heads / pool->num_kv_heads;
    a.scale_log2 = sm_scale * 1.4426950408889634f;
    sa.shared = plan_dev + info->decode.plan_ints;
    sa.pairs = sa.shared + kRecord * int64_t(info->num_shared);
    sa.num_shared = info->num_shared;
    const int64_t blocks = 8 * ceil_div(info->num_shared, 8) * a.head_groups;
    KSV_CHECK_ARG(blocks < (int64_t(1) << 31), "grid of %lld workgroups is too large",
                  (long long)blocks);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    rc = pool->dtype == KUNSERVE_DTYPE_BF16
             ? launch_shared_dim<bf16>(pool->head_dim, sa, info->tiles, unsigned(blocks), s)
             : launch_shared_dim<f16>(pool->head_dim, sa, info->tiles, unsigned(blocks), s);
    if (rc) return rc;
  }
  StepFusion tails = fusion;
  tails.counters = nullptr;   // a row's partials are not its partitions alone
  return paged_decode(pool, layer, table, q_token_dev, q, out, num_qo_heads, sm_scale, plan_dev,
                      &info->decode, workspace_dev, workspace_bytes, tails, stream);
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
