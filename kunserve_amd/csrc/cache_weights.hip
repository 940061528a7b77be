// The attention weight that each cached token gets (what an eviction goes by).
//
// The observers of a row are the last min(q_len, window) of its new tokens.
// With p[i, h, t] = softmax over t <= pos(i) of q[i, h] . k[t] * sm_scale,
//   w[t] := (t new ? 0 : w[t]) + sum over observers i and the query heads h of
//           the KV head of p[i, h, t]
// for every cached token of the row and every KV head, in fp32. A new token's
// weight starts at 0 (clear_weights_kernel: in steps that add none).
//
// Columns: the row's observers times the query heads of a KV head. Two launches
// read K: the maximum and sum of every column over each partition of kPartTokens
// tokens, then the scores once more, this time as probabilities summed over the
// columns. The second combines the partitions' statistics itself; from rows of more
// than kMaxOwnParts partitions on, a launch between the two does. The sums run in one
// order, with no atomics, so results do not depend on timing. A workgroup keeps its
// partition of K in registers (64 tokens a wave, as MFMA operands) and takes the
// columns 16 at a time, so K is read once by each of the two. A step's decode rows need
// no second look at K: their decode launch leaves its scores.
#include <algorithm>
#include <cmath>
#include <vector>

#include "common.hpp"

namespace kunserve {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kSubs = 4;                            // 16-token tiles of a wave
constexpr int kPartTokens = kWaves * kSubs * 16;    // 256
constexpr int kCols = 64;                           // columns in LDS at a time
// Partitions up to which the last launch combines the columns itself.
constexpr int kMaxOwnParts = 64;
constexpr float kNegBig = -1.0e30f;                 // finite "minus infinity" for running maxima

struct WeightsArgs {
  const f16* q;
  int64_t q_tok, q_head;
  const f16* k;   // pool K at the layer
  int64_t page_stride, head_stride, token_stride;
  float* w;       // at the layer
  int64_t w_page, w_head;
  int32_t num_pages, page_shift;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* kv_len;
  const int32_t* q_indptr;
  const int32_t* items;      // [num_items][4]: row, first token, column offset, partitions
  const int32_t* combines;   // [num_combines][4]: row, first column, column offset, partitions
  float2* stats;             // per row: [partitions + 1][columns]; the last: combined
  int64_t num_columns;       // entries of stats
  int32_t num_qo_heads, num_kv_heads, ratio, window;
  float scale_log2;
};

// m and l of two disjoint sets of scores.
__device__ __forceinline__ float2 join(float2 x, float2 y) {
  const float m = fmaxf(x.x, y.x);
  return {m, x.y * fast_exp2(x.x - m) + y.y * fast_exp2(y.x - m)};
}
// What a probability is formed with: the maximum, and 1 / sum (a NaN sum stays).
__device__ __forceinline__ float2 normaliser(float2 s) {
  return {s.x, s.y > 0.f ? 1.f / s.y : s.y};
}

// ADD false: the partition's maxima and sums; true: its tokens' weights. COMBINE
// (with ADD): it combines the partitions' maxima and sums itself.
// Columns come kCols at a time: their q through LDS, the next ones' on the way
// meanwhile.
template <typename T, int D, bool ADD, bool COMBINE>
__global__ __launch_bounds__(kThreads) void weights_scores_kernel(WeightsArgs a) {
  typedef typename Vec<T>::v8 V8;
  constexpr int KS = D / 32;   // MFMAs of a 16-token tile
  constexpr int CH = D / 8;    // 16-byte chunks of a row
  constexpr int QL = kCols * CH / kThreads;
  __shared__ __attribute__((aligned(16))) T s_q[kCols * D];   // column g's chunk c at c ^ (g & 7)
  __shared__ float2 s_stat[kWaves][kCols];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int j = lane & 15, tg = lane >> 4;
  const int32_t* item = a.items + 4 * blockIdx.x;
  const int seq = item[0], part0 = item[1], hkv = blockIdx.y, parts = item[3];
  const int64_t offset = item[2];
  const int n = a.kv_len[seq], q0 = a.q_indptr[seq], q_len = a.q_indptr[seq + 1] - q0;
  const int obs = min(q_len, a.window);       // observers
  const int cols = obs * a.ratio;             // columns of this KV head
  const int all = cols * a.num_kv_heads;
  // A q_indptr that is not the plan's must not leave the workspace.
  if (offset + int64_t(parts + 1) * all > a.num_columns) return;   // uniform
  const int t0 = part0 + wave * kSubs * 16;   // first token of the wave
  const int mask = (1 << a.page_shift) - 1;
  const int32_t* pages = a.indices + a.indptr[seq];
  auto page_of = [&](int t) -> int {   // -1: past the row's end or outside the pool
    if (t >= n) return -1;
    const int p = pages[t >> a.page_shift];
    return p >= 0 && p < a.num_pages ? p : -1;
  };
  // Column c: observer c / ratio, query head c % ratio of the KV head's.
  V8 qn[QL];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int c = c0 + (tid + i * kThreads) / CH, chunk = (tid + i * kThreads) % CH;
      const int o = min(c, cols - 1) / a.ratio, h = hkv * a.ratio + min(c, cols - 1) % a.ratio;
      qn[i] = load_v8<T>(a.q + int64_t(q0 + q_len - obs + o) * a.q_tok + int64_t(h) * a.q_head +
                         8 * chunk);
    }
  };
  fetch(0);

  // K as the A operand: row j of tile `sub` is token t0 + 16 sub + j.
  V8 k[kSubs][KS];
  uint32_t ok = 0;   // of the lane's tokens in the result: bit 4 sub + x
#pragma unroll
  for (int sub = 0; sub < kSubs; ++sub) {
    const int t = t0 + 16 * sub + j;
    const int p = page_of(t);
    const f16* row = a.k + int64_t(hkv) * a.head_stride + int64_t(max(p, 0)) * a.page_stride +
                     int64_t(t & mask) * a.token_stride + 8 * tg;
#pragma unroll
    for (int s = 0; s < KS; ++s) k[sub][s] = p >= 0 ? load_v8<T>(row + 32 * s) : V8{};
    const uint64_t fine = __ballot(p >= 0);   // bit j: token t0 + 16 sub + j
    ok |= uint32_t((fine >> (4 * tg)) & 15u) << (4 * sub);
  }
  float mass[kSubs][4] = {};
  float2* stats = a.stats + offset;
  // Every token of the wave is there, and seen by every observer.
  const bool whole = __all(ok == 0xffffu) && t0 + kSubs * 16 <= n - obs + 1;
  for (int c0 = 0; c0 < cols; c0 += kCols) {
    __syncthreads();   // the columns before are done with
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int g = (tid + i * kThreads) / CH, chunk = (tid + i * kThreads) % CH;
      *reinterpret_cast<V8*>(&s_q[g * D + 8 * (chunk ^ (g & 7))]) = qn[i];
    }
    const int here = min(kCols, cols - c0);
    if constexpr (ADD) {
      // The columns' normalisers (columns past the last one: none gets anything).
      // A quarter of the partitions to each wave.
      float2 st = {kNegBig, 0.f};
      const float2* src = stats + int64_t(hkv) * cols + c0 + min(lane, here - 1);
      if constexpr (COMBINE) {
        for (int i0 = 0; i0 < parts; i0 += 4 * kWaves) {
          float2 x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            x[u] = src[int64_t(min(i0 + u * kWaves + wave, parts - 1)) * all];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (i0 + u * kWaves + wave < parts) st = join(st, x[u]);
        }
        s_stat[wave][lane] = st;
      } else if (wave == 0) {
        s_stat[0][lane] = lane < here ? src[int64_t(parts) * all] : float2{-kNegBig, 0.f};
      }
    }
    __syncthreads();
    if (c0 + kCols < cols) fetch(c0 + kCols);
    if constexpr (ADD && COMBINE) {
      if (wave == 0) {
        float2 st = s_stat[0][lane];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) st = join(st, s_stat[i][lane]);
        s_stat[0][lane] = lane < here ? normaliser(st) : float2{-kNegBig, 0.f};
      }
      __syncthreads();
    }
#pragma unroll
    for (int ct = 0; ct < kCols / 16; ++ct) {
      if (16 * ct >= here) break;   // uniform
      const int c = 16 * ct + j;
      const int last = n - obs + (c0 + c) / a.ratio;   // the last token that the observer sees
      V8 q[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s)
        q[s] = *reinterpret_cast<const V8*>(&s_q[c * D + 8 * ((4 * s + tg) ^ (c & 7))]);
      f32x4 sc[kSubs];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        sc[sub] = f32x4{};
#pragma unroll
        for (int s = 0; s < KS; ++s) sc[sub] = mfma16(k[sub][s], q[s], sc[sub]);
      }
      auto seen = [&](int sub, int x) {
        return ((ok >> (4 * sub + x)) & 1u) && t0 + 16 * sub + 4 * tg + x <= last;
      };
      if constexpr (ADD) {
        const float2 st = s_stat[0][c];
        auto add = [&](bool all_seen) {   // a NaN column gives nothing to what it does not see
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float p = fast_exp2(fmaf(sc[sub][x], a.scale_log2, -st.x)) * st.y;
              mass[sub][x] += all_seen || seen(sub, x) ? p : 0.f;
            }
        };
        if (whole)   // uniform
          add(true);
        else
          add(false);
      } else {
        if (!whole) {   // uniform; the scale is positive
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[sub][x] = seen(sub, x) ? sc[sub][x] : -INFINITY;
        }
        float m = -INFINITY;
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int x = 0; x < 4; ++x) m = fmaxf(m, sc[sub][x]);
        m = fmaxf(groups_max(m) * a.scale_log2, kNegBig);
        float l = 0.f;
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int x = 0; x < 4; ++x) l += fast_exp2(fmaf(sc[sub][x], a.scale_log2, -m));
        l = groups_sum(l);
        if (tg == 0) s_stat[wave][c] = float2{m, l};
      }
    }
    if constexpr (!ADD) {
      __syncthreads();
      if (tid < here) {
        float2 st = s_stat[0][tid];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) st = join(st, s_stat[i][tid]);
        stats[int64_t(part0 / kPartTokens) * all + int64_t(hkv) * cols + c0 + tid] = st;
      }
    }
  }
  if constexpr (ADD) {
    // Sums over the 16 columns of a lane row; lane j then takes result 4 sub
    // + x = j: token t0 + 16 (j / 4) + 4 tg + j % 4.
    float mine = 0.f;
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float s = row16_sum(mass[sub][x]);
        mine = j == 4 * sub + x ? s : mine;
      }
    const int t = t0 + 16 * (j >> 2) + 4 * tg + (j & 3);
    const int p = page_of(t);
    if (p >= 0) {
      float* w = a.w + int64_t(hkv) * a.w_head + int64_t(p) * a.w_page + (t & mask);
      *w = (t >= n - q_len ? 0.f : *w) + mine;
    }
  }
}

// A column's maximum and 1 / sum over the row's partitions.
__global__ __launch_bounds__(kThreads) void weights_combine_kernel(WeightsArgs a) {
  const int32_t* rec = a.combines + 4 * blockIdx.x;
  const int seq = rec[0], parts = rec[3];
  const int q_len = a.q_indptr[seq + 1] - a.q_indptr[seq];
  const int all = min(q_len, a.window) * a.num_qo_heads;
  const int c = rec[1] + threadIdx.x;
  if (c >= all || rec[2] + int64_t(parts + 1) * all > a.num_columns) return;
  float2* stats = a.stats + int64_t(rec[2]) + c;
  float2 st = {kNegBig, 0.f};
  int i = 0;
  for (; i + 8 <= parts; i += 8) {   // loads together, one order of joining
    float2 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = stats[int64_t(i + u) * all];
#pragma unroll
    for (int u = 0; u < 8; ++u) st = join(st, x[u]);
  }
  for (; i < parts; ++i) st = join(st, stats[int64_t(i) * all]);
  stats[int64_t(parts) * all] = normaliser(st);
}

// Decode rows: the decode launch left their scores and log-sum-exps (DecodeArgs::
// scores), so K is not read again: 4 bytes written and read per token and query
// head beside the 4 head_dim bytes of K and V that a KV head's token has. A thread
// per token, which looks its page up once for kScoreHeads KV heads; V scores to a
// load (V 4 where the group allows: lanes apart by more than their loads cost a line
// each).
constexpr int kScoreHeads = 4;

struct ScoreArgs {
  const int32_t* items;   // [..][4]: row, first token, the row's score_at
  const float* scores;
  const float* lse;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* kv_len;
  float* w;
  int64_t w_page, w_head;
  int32_t num_pages, page_shift, num_qo_heads, num_kv_heads, ratio, group;
};

template <int V>
__global__ __launch_bounds__(kThreads) void weights_from_scores_kernel(ScoreArgs a) {
  typedef float VecF __attribute__((ext_vector_type(V)));
  const int32_t* item = a.items + 4 * blockIdx.x;
  const int seq = item[0], t = item[1] + threadIdx.x, h0 = int(blockIdx.y) * kScoreHeads;
  const int n = a.kv_len[seq];
  if (t >= n) return;
  const int p = a.indices[a.indptr[seq] + (t >> a.page_shift)];
  const bool ok = p >= 0 && p < a.num_pages;
  float* w = a.w + int64_t(ok ? p : 0) * a.w_page + (t & ((1 << a.page_shift) - 1));
  const float* lse = a.lse + int64_t(seq) * a.num_qo_heads;
  // of KV head h: its head groups one after the other, [token][head of the group]
  const float* scores = a.scores + int64_t(item[2]) * a.num_qo_heads;
  float sum[kScoreHeads], old[kScoreHeads];
#pragma unroll
  for (int i = 0; i < kScoreHeads; ++i) {
    const int h = min(h0 + i, a.num_kv_heads - 1);
    old[i] = t < n - 1 ? w[int64_t(h) * a.w_head] : 0.f;   // the new token starts at 0
    sum[i] = 0.f;
    for (int q0 = h * a.ratio; q0 < (h + 1) * a.ratio; q0 += a.group) {
      const float* s = scores + (int64_t(q0 / a.group) * n + t) * a.group;
      for (int g = 0; g < a.group; g += V) {
        const VecF x = *reinterpret_cast<const VecF*>(s + g);
#pragma unroll
        for (int e = 0; e < V; ++e) sum[i] += fast_exp2(x[e] - lse[q0 + g + e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kScoreHeads; ++i)
    if (ok && h0 + i < a.num_kv_heads) w[int64_t(h0 + i) * a.w_head] = old[i] + sum[i];
}

// The weights of new tokens become 0 in every layer: a workgroup per token, whose
// (layer, KV head) pairs are a line each. For 32 layers of 8 heads, 64 tokens take 2.6 us,
// 4000 tokens 10: once for a step.
struct ClearArgs {
  float* w;
  int64_t w_page, w_layer, w_head;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* kv_len;
  const int32_t* q_indptr;
  int32_t num_seqs, num_pages, page_shift, num_layers, num_kv_heads;
};

__global__ __launch_bounds__(kThreads) void clear_weights_kernel(ClearArgs a) {
  const int tok = int(blockIdx.x);
  const int b = row_of_token(a.q_indptr, a.num_seqs, tok);
  if (b < 0) return;
  const int kvl = a.kv_len[b], at = kvl - a.q_indptr[b + 1] + tok;
  if (at < 0 || at >= kvl) return;
  const int p = a.indices[a.indptr[b] + (at >> a.page_shift)];
  if (p < 0 || p >= a.num_pages) return;
  float* w = a.w + int64_t(p) * a.w_page + (at & ((1 << a.page_shift) - 1));
  for (int64_t i = threadIdx.x; i < int64_t(a.num_layers) * a.num_kv_heads; i += kThreads)
    w[i / a.num_kv_heads * a.w_layer + i % a.num_kv_heads * a.w_head] = 0.f;
}

template <typename T, int D>
int run_weights(const WeightsArgs& a, const kunserve_weights_plan_info& info, hipStream_t s) {
  const dim3 grid(unsigned(info.num_items), unsigned(a.num_kv_heads));
  weights_scores_kernel<T, D, false, false><<<grid, kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  if (info.num_combines > 0) {
    weights_combine_kernel<<<dim3(unsigned(info.num_combines)), kThreads, 0, s>>>(a);
    KSV_CHECK_LAUNCH();
    weights_scores_kernel<T, D, true, false><<<grid, kThreads, 0, s>>>(a);
  } else {
    weights_scores_kernel<T, D, true, true><<<grid, kThreads, 0, s>>>(a);
  }
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

template <typename T>
int run_weights_dim(int head_dim, const WeightsArgs& a, const kunserve_weights_plan_info& info,
                    hipStream_t s) {
  switch (head_dim) {
    case 64: return run_weights<T, 64>(a, info, s);
    case 128: return run_weights<T, 128>(a, info, s);
    default: return run_weights<T, 256>(a, info, s);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int weights_plan(const int32_t* q_indptr, const int32_t* kv_len, int32_t num_seqs,
                 int32_t num_qo_heads, int32_t window, const int32_t* decodes,
                 std::vector<int32_t>& plan, kunserve_weights_plan_info* info) {
  std::vector<int32_t> items, combines, score_items, score_at;
  int64_t columns = 0, score_tokens = 0, most_parts = 0;
  KSV_CHECK_ARG(num_seqs == 0 || q_indptr[0] >= 0, "q_indptr begins at %d", q_indptr[0]);
  for (int32_t b = 0; b < num_seqs; ++b) {
    const int64_t q_len = int64_t(q_indptr[b + 1]) - q_indptr[b];
    KSV_CHECK_ARG(q_len >= 0 && kv_len[b] >= q_len, "row %d: kv_len %d for %lld new tokens", b,
                  kv_len[b], (long long)q_len);
    KSV_CHECK_ARG(!decodes || !decodes[b] || q_len == 1, "row %d decodes %lld tokens", b,
                  (long long)q_len);
    if (decodes && decodes[b] == 2) {   // leaves no scores: its K is read again
      score_at.push_back(-1);
    } else if (decodes && decodes[b]) {
      const int32_t row = int32_t(score_at.size());
      for (int32_t t = 0; t < kv_len[b]; t += kThreads)
        score_items.insert(score_items.end(), {row, t, int32_t(score_tokens), 0});
      score_at.push_back(int32_t(score_tokens));
      score_tokens += kv_len[b];
      KSV_CHECK_ARG(score_tokens < (int64_t(1) << 31), "too many cached tokens");
      continue;
    }
    if (q_len == 0) continue;
    const int64_t cols = std::min<int64_t>(q_len, window) * num_qo_heads;
    const int64_t parts = ceil_div(kv_len[b], kPartTokens);
    most_parts = std::max(most_parts, parts);
    KSV_CHECK_ARG(columns + (parts + 1) * cols < (int64_t(1) << 31),
                  "too many observed columns (%lld)", (long long)(columns + (parts + 1) * cols));
    for (int64_t p = 0; p < parts; ++p)
      items.insert(items.end(), {b, int32_t(p * kPartTokens), int32_t(columns), int32_t(parts)});
    for (int64_t c = 0; c < cols; c += kThreads)
      combines.insert(combines.end(), {b, int32_t(c), int32_t(columns), int32_t(parts)});
    columns += (parts + 1) * cols;
  }
  if (most_parts <= kMaxOwnParts) combines.clear();
  plan = std::move(items);
  info->num_items = int32_t(plan.size() / 4);
  plan.insert(plan.end(), combines.begin(), combines.end());
  info->num_combines = int32_t(combines.size() / 4);
  plan.insert(plan.end(), score_items.begin(), score_items.end());
  info->num_score_items = int32_t(score_items.size() / 4);
  plan.insert(plan.end(), score_at.begin(), score_at.end());
  info->num_score_rows = int32_t(score_at.size());
  info->score_tokens = score_tokens;
  info->num_seqs = num_seqs;
  info->window = window;
  info->num_qo_heads = num_qo_heads;
  info->plan_ints = int32_t(plan.size());
  info->num_columns = columns;
  return KUNSERVE_OK;
}

}  // namespace
}  // namespace kunserve

using namespace kunserve;

extern "C" int64_t kunserve_weights_plan_bound(const int32_t* q_indptr_host,
                                               const int32_t* kv_len_host, int32_t num_seqs,
                                               int32_t num_qo_heads, int32_t window) {
  if (num_seqs < 0 || num_qo_heads <= 0 || window <= 0 ||
      (num_seqs > 0 && (!q_indptr_host || !kv_len_host)))
    return -1;
  int64_t records = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    const int64_t q_len = std::max<int64_t>(0, int64_t(q_indptr_host[b + 1]) - q_indptr_host[b]);
    records += ceil_div(std::max(kv_len_host[b], 0), kPartTokens) +
               ceil_div(std::min<int64_t>(q_len, window) * num_qo_heads, kThreads) + 1;
  }
  return 4 * records;
}

extern "C" int kunserve_weights_plan(const int32_t* q_indptr_host, const int32_t* kv_len_host,
                                     int32_t num_seqs, int32_t num_qo_heads, int32_t window,
                                     const int32_t* decodes_host, int32_t* plan_host, int64_t plan_capacity,
                                     kunserve_weights_plan_info* info) {
  clear_error();
  KSV_CHECK_ARG(info && plan_host, "null plan buffer or info");
  KSV_CHECK_ARG(num_seqs >= 0 && (num_seqs == 0 || (q_indptr_host && kv_len_host)),
                "bad q_indptr, kv_len or num_seqs");
  KSV_CHECK_ARG(num_qo_heads > 0, "num_qo_heads %d", num_qo_heads);
  KSV_CHECK_ARG(window > 0, "window %d must be positive", window);
  return no_throw([&] {
    std::vector<int32_t> plan;
    const int rc = weights_plan(q_indptr_host, kv_len_host, num_seqs, num_qo_heads, window,
                                decodes_host, plan, info);
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

extern "C" int64_t kunserve_weights_workspace_bytes(const kunserve_weights_plan_info* info) {
  if (!info) return -1;
  if (info->num_columns == 0 && info->num_score_rows == 0) return 0;
  return 16 + info->num_columns * int64_t(sizeof(float2)) +
         (info->score_tokens + info->num_score_rows) * info->num_qo_heads * int64_t(sizeof(float));
}

void kunserve::weights_scores(const kunserve_weights_plan_info* info, const int32_t* plan_dev,
                              void* workspace_dev, StepFusion* fusion) {
  // 16-byte aligned, as the workspace is (an even number of columns)
  float* at = reinterpret_cast<float*>(static_cast<float2*>(workspace_dev) +
                                       (info->num_columns + 1) / 2 * 2);
  fusion->scores = at;
  fusion->lse = at + info->score_tokens * info->num_qo_heads;
  fusion->score_at = plan_dev + 4 * (int64_t(info->num_items) + info->num_combines +
                                     info->num_score_items);
}

int kunserve::weights_from_scores(const kunserve_kv_pool* pool, const kunserve_kv_weights* weights,
                                  int32_t layer, const kunserve_page_table* decode_table,
                                  int32_t num_qo_heads, const int32_t* plan_dev,
                                  const kunserve_weights_plan_info* info, void* workspace_dev,
                                  kunserve_stream_t stream) {
  if (info->num_score_items == 0) return KUNSERVE_OK;
  StepFusion f;
  weights_scores(info, plan_dev, workspace_dev, &f);
  ScoreArgs a{};
  a.items = plan_dev + 4 * (int64_t(info->num_items) + info->num_combines);
  a.scores = f.scores;
  a.lse = f.lse;
  a.indptr = decode_table->indptr_dev;
  a.indices = decode_table->indices_dev;
  a.kv_len = decode_table->kv_len_dev;
  a.w = weights->w + int64_t(layer) * weights->layer_stride;
  a.w_page = weights->page_stride;
  a.w_head = weights->head_stride;
  a.num_pages = int32_t(pool->num_pages);
  a.page_shift = __builtin_ctz(pool->page_size);
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = pool->num_kv_heads;
  a.ratio = num_qo_heads / pool->num_kv_heads;
  a.group = decode_group(num_qo_heads, pool->num_kv_heads);
  const dim3 grid(unsigned(info->num_score_items),
                  unsigned(ceil_div(pool->num_kv_heads, kScoreHeads)));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a.group % 4 == 0)
    weights_from_scores_kernel<4><<<grid, kThreads, 0, s>>>(a);
  else
    weights_from_scores_kernel<1><<<grid, kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

extern "C" int kunserve_cache_weights(const kunserve_kv_pool* pool,
                                      const kunserve_kv_weights* weights, int32_t layer,
                                      const kunserve_page_table* table,
                                      const int32_t* q_indptr_dev, const kunserve_tensor3* q,
                                      int32_t num_qo_heads, float sm_scale,
                                      const int32_t* plan_dev,
                                      const kunserve_weights_plan_info* info, void* workspace_dev,
                                      int64_t workspace_bytes, kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  rc = check_weights(weights, pool);
  if (rc) return rc;
  KSV_CHECK_ARG(table && q && info, "null argument");
  KSV_CHECK_ARG(layer >= 0 && layer < pool->num_layers, "layer %d outside [0, %d)", layer,
                pool->num_layers);
  KSV_CHECK_ARG(std::isfinite(sm_scale) && sm_scale > 0.f,
                "sm_scale %g must be finite and positive", double(sm_scale));
  KSV_CHECK_ARG(num_qo_heads > 0 && num_qo_heads % pool->num_kv_heads == 0,
                "num_qo_heads %d not a multiple of num_kv_heads %d", num_qo_heads,
                pool->num_kv_heads);
  KSV_CHECK_ARG(info->num_qo_heads == num_qo_heads, "plan made for %d query heads, not %d",
                info->num_qo_heads, num_qo_heads);
  KSV_CHECK_ARG(info->num_seqs == table->num_seqs, "plan made for %d rows, not %d", info->num_seqs,
                table->num_seqs);
  if (info->num_items == 0) return KUNSERVE_OK;
  KSV_CHECK_ARG(plan_dev && q_indptr_dev && table->indptr_dev && table->indices_dev &&
                    table->kv_len_dev,
                "null plan or table");
  KSV_CHECK_ARG(q->data && aligned16(q->data) && q->token_stride % 8 == 0 &&
                    q->head_stride % 8 == 0,
                "q must be 16-byte aligned with strides that are multiples of 8");
  KSV_CHECK_ARG(pool->num_kv_heads < 65536, "%d KV heads: at most 65535", pool->num_kv_heads);
  const int64_t need = kunserve_weights_workspace_bytes(info);
  if (!workspace_dev || workspace_bytes < need) {
    set_error("weights workspace holds %lld bytes, %lld needed", (long long)workspace_bytes,
              (long long)need);
    return KUNSERVE_ENOSPC;
  }
  KSV_CHECK_ARG(aligned16(workspace_dev), "workspace must be 16-byte aligned");
  WeightsArgs a{};
  a.q = static_cast<const f16*>(q->data);
  a.q_tok = q->token_stride;
  a.q_head = q->head_stride;
  a.k = static_cast<const f16*>(pool->k) + int64_t(layer) * pool->layer_stride;
  a.page_stride = pool->page_stride;
  a.head_stride = pool->head_stride;
  a.token_stride = pool->token_stride;
  a.w = weights->w + int64_t(layer) * weights->layer_stride;
  a.w_page = weights->page_stride;
  a.w_head = weights->head_stride;
  a.num_pages = int32_t(pool->num_pages);
  a.page_shift = __builtin_ctz(pool->page_size);
  a.indptr = table->indptr_dev;
  a.indices = table->indices_dev;
  a.kv_len = table->kv_len_dev;
  a.q_indptr = q_indptr_dev;
  a.items = plan_dev;
  a.combines = plan_dev + 4 * int64_t(info->num_items);
  a.stats = static_cast<float2*>(workspace_dev);
  a.num_columns = info->num_columns;
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = pool->num_kv_heads;
  a.ratio = num_qo_heads / pool->num_kv_heads;
  a.window = info->window;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (pool->dtype == KUNSERVE_DTYPE_BF16)
    return run_weights_dim<bf16>(pool->head_dim, a, *info, s);
  return run_weights_dim<f16>(pool->head_dim, a, *info, s);
}

extern "C" int kunserve_clear_weights(const kunserve_kv_pool* pool,
                                      const kunserve_kv_weights* weights,
                                      const kunserve_page_table* table,
                                      const int32_t* q_indptr_dev, int32_t num_tokens,
                                      kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  rc = check_weights(weights, pool);
  if (rc) return rc;
  KSV_CHECK_ARG(table && table->num_seqs >= 0 && num_tokens >= 0,
                "null table, num_seqs or num_tokens < 0");
  if (table->num_seqs == 0 || num_tokens == 0) return KUNSERVE_OK;
  KSV_CHECK_ARG(table->indptr_dev && table->indices_dev && table->kv_len_dev && q_indptr_dev,
                "null table array or q_indptr");
  ClearArgs a{};
  a.w = weights->w;
  a.w_page = weights->page_stride;
  a.w_layer = weights->layer_stride;
  a.w_head = weights->head_stride;
  a.indptr = table->indptr_dev;
  a.indices = table->indices_dev;
  a.kv_len = table->kv_len_dev;
  a.q_indptr = q_indptr_dev;
  a.num_seqs = table->num_seqs;
  a.num_pages = int32_t(pool->num_pages);
  a.page_shift = __builtin_ctz(pool->page_size);
  a.num_layers = pool->num_layers;
  a.num_kv_heads = pool->num_kv_heads;
  clear_weights_kernel<<<dim3(unsigned(num_tokens)), kThreads, 0,
                         reinterpret_cast<hipStream_t>(stream)>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}
