// What the decode kernels share: the launch's arguments, the order of its
// work, appending and combining rows, and the MFMA kernels' tile of K and V.
// Kernels, their constants and device helpers are local to the source that includes
// this.
#pragma once

#include "common.hpp"

namespace kunserve {

struct DecodeArgs {
  const int32_t* q_token;   // null, or [num_seqs]: token of q and out of each sequence
  const f16* q;
  int64_t q_tok, q_head;
  f16* out;
  int64_t o_tok, o_head;
  const f16* k;             // pool K at the layer
  const f16* v;
  int64_t page_stride, head_stride, token_stride;
  int32_t num_pages;
  int32_t page_shift;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* kv_len;    // for k_new and counters (null without them)
  // The step's new K/V rows of the same tokens as q, or null: they are then
  // in the pages already. With them the launch appends as well: the new
  // token's row (position kv_len - 1) is read from here instead of from its
  // page, and the workgroup that reads it writes it there. No other row's
  // table holds that page (the caller checks), so no other workgroup
  // reads what this launch writes.
  const f16* k_new;
  const f16* v_new;
  int64_t kn_tok, kn_head, vn_tok, vn_head;
  // null, or one zeroed counter per (first slot of a split row, head group):
  // the last of the row's workgroups to finish combines the partials.
  int32_t* counters;
  // null, or where the launch leaves its scores (in log2 units) and every row's
  // log-sum-exp: of row b, head group hg, token t and head g of the group at
  // scores[score_at[b] * num_qo_heads + (hg * kv_len[b] + t) * group + g], and
  // lse[b * num_qo_heads + head]. A NaN score makes a log-sum-exp NaN. score_at -1: the
  // row leaves no scores.
  float* scores;
  float* lse;
  const int32_t* score_at;
  int32_t part_tokens;
  const int32_t* work;      // [num_work][4]: seq (-1: padding), tok_begin, tok_end, slot (-1: direct)
  float* part_o;            // [slots][num_qo_heads][D]
  float* part_lse;          // [slots][num_qo_heads]
  int32_t num_qo_heads;
  int32_t group;            // G: query heads of a workgroup
  int32_t head_groups;      // num_qo_heads / G
  int32_t num_work;         // work items of the plan
  int32_t ratio;            // num_qo_heads / num_kv_heads
  float scale_log2;         // sm_scale * log2(e)
};

// The launch's arguments, checked, for a plan of DecodeItems (paged_decode);
// num_work 0: nothing to launch. And the launch that joins split rows.
int decode_args(const kunserve_kv_pool* pool, int32_t layer, const kunserve_page_table* table,
                const int32_t* q_token_dev, const kunserve_tensor3* q, kunserve_tensor3* out,
                int32_t num_qo_heads, float sm_scale, const int32_t* plan_dev,
                const kunserve_decode_plan_info* info, void* workspace_dev,
                int64_t workspace_bytes, const StepFusion& fusion, DecodeArgs* args);
int decode_merge(const kunserve_kv_pool* pool, const DecodeArgs& a,
                 const kunserve_decode_plan_info* info, const int32_t* plan_dev, hipStream_t s);

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kLoadsPerChunk = 4;        // 16-byte loads per lane per chunk (K and V each)
constexpr int kMaxPartTokens = 4096;
constexpr int kMinPageSize = 4;
constexpr int kMaxPartPages = kMaxPartTokens / kMinPageSize + 2;
constexpr int kMinPartTokens = 256;
constexpr int kMinAutoPartTokens = 128;  // shortest the grouped plan chooses by itself: a step of every wave
constexpr int kMaxCountedParts = 8;      // partitions a counting workgroup combines (one batch)
constexpr int kMaxGroup = 16;            // query heads of one workgroup (MFMA columns)
constexpr int kXcds = 8;                 // MI355X: workgroup b runs on XCD b % 8
constexpr float kNegBig = -1.0e30f;      // finite "minus infinity" for running maxima

// Source of the loads of lanes past a partition's end and of bad page ids:
// one zero K/V row (head_dim <= 256), so loaded data is never masked.
__device__ __attribute__((aligned(16))) f16 g_zero_row[256];

// Work record and head group of workgroup b. The hardware hands workgroup
// b to XCD b % 8. The plan's records are 8 lanes interleaved (record
// 8 r + x is entry r of XCD x's lane), and XCD x runs every head group of
// its lane's entries in order, an entry's head groups back to back, so the
// pages an XCD reads at a time are those of its own few items (measured
// 1-2% faster than spreading each item's head groups over all XCDs). A
// lane's padding records (seq -1) end the workgroup at once.
__device__ __forceinline__ bool decode_work(const DecodeArgs& a, int& item, int& hg) {
  const int b = int(blockIdx.x);
  const int j = b >> 3;
  const int local = j / a.head_groups;
  hg = j - local * a.head_groups;
  item = 8 * local + (b & 7);
  return item < a.num_work;
}

// Where an item's new K/V row is: its position (-1: not in this launch's
// care) and its distance in elements from the KV head's base in the pool, so
// that a lane's load address takes one select of two offsets.
struct NewRow {
  int pos;
  int64_t k, v;
};
__device__ __forceinline__ NewRow new_row(const DecodeArgs& a, int seq, int tok, int hkv) {
  if (!a.k_new) return {-1, 0, 0};
  auto distance = [&](const f16* row, const f16* pool) {   // both 16-byte aligned
    return (reinterpret_cast<intptr_t>(row) - reinterpret_cast<intptr_t>(pool + int64_t(hkv) * a.head_stride)) / 2;
  };
  return {a.kv_len[seq] - 1,
          distance(a.k_new + int64_t(tok) * a.kn_tok + int64_t(hkv) * a.kn_head, a.k),
          distance(a.v_new + int64_t(tok) * a.vn_tok + int64_t(hkv) * a.vn_head, a.v)};
}
// Writes the new row into its page (`page`, -1: outside the pool), by the
// workgroup of the KV head's first query heads whose partition holds it.
template <int D>
__device__ __forceinline__ void append_row(const DecodeArgs& a, const NewRow& nr, int page,
                                           int hkv) {
  constexpr int CH = D / 8;
  const int tid = threadIdx.x;
  if (page < 0 || tid >= 2 * CH) return;
  const int c = tid % CH;
  const int64_t off = int64_t(page) * a.page_stride +
                      int64_t(nr.pos & ((1 << a.page_shift) - 1)) * a.token_stride;
  const bool v = tid >= CH;
  f16* base = const_cast<f16*>(v ? a.v : a.k) + int64_t(hkv) * a.head_stride + 8 * c;
  store_f16x8(base + off, load_f16x8(base + (v ? nr.v : nr.k)));
}

__device__ __forceinline__ void store_agent(float* p, float x, float y) {
  const uint64_t w = uint64_t(uint32_t(f32_to_bits(x))) | uint64_t(uint32_t(f32_to_bits(y))) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Writes a workgroup's result, `result(g, d, x, y, lse)` giving head g's dims
// d, d + 1 and log-sum-exp (base 2): to out (slot -1), or as the partial of
// `slot`. With counters, the last workgroup of the row and head group to
// finish then combines the row's partials, in partition order, and no merge
// launch follows (about 3 us and the gap before it). A release/acquire pair
// at agent scope would write back and invalidate the XCD's whole L2 once per
// workgroup (10 times the launch's time). Instead the partials themselves are
// agent-scope atomic stores and loads, which do not stay in an L2: every
// wave waits for its stores (vmcnt counts stores on this part), the
// workgroup meets at a barrier, and only then is it counted.
template <typename T, int D, int THREADS, typename F>
__device__ __forceinline__ void decode_finish(const DecodeArgs& a, int seq, int tok, int tb,
                                              int slot, int hq0, int hg, int G, F result) {
  __shared__ int s_last;
  const int tid = threadIdx.x;
  const int pairs = G * (D / 2);
  auto write_out = [&](int g, int d, float x, float y) {
    T* op = reinterpret_cast<T*>(a.out) + int64_t(tok) * a.o_tok + int64_t(hq0 + g) * a.o_head + d;
    op[0] = T(x);
    op[1] = T(y);
  };
  for (int idx = tid; idx < pairs; idx += THREADS) {
    const int g = idx / (D / 2), d = 2 * (idx % (D / 2));
    float x, y, lse;
    result(g, d, x, y, lse);
    if (slot < 0) {
      write_out(g, d, x, y);
      if (d == 0 && a.lse) a.lse[int64_t(seq) * a.num_qo_heads + hq0 + g] = lse;
      continue;
    }
    const int64_t row = int64_t(slot) * a.num_qo_heads + hq0 + g;
    float* po = a.part_o + row * D + d;
    if (a.counters) {
      store_agent(po, x, y);
      if (d == 0)
        __hip_atomic_store(a.part_lse + row, lse, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      po[0] = x;
      po[1] = y;
      if (d == 0) a.part_lse[row] = lse;
    }
  }
  if (slot < 0 || !a.counters) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int s0 = slot - tb / a.part_tokens;   // the row's first slot
  const int n = (a.kv_len[seq] + a.part_tokens - 1) / a.part_tokens;
  if (tid == 0) {
    int32_t* counter = a.counters + int64_t(s0) * a.head_groups + hg;
    const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = before == n - 1;
    if (before == n - 1)   // zero again for the next layer
      __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();   // also keeps the compiler from moving the loads below before the count
  if (!s_last) return;
  for (int idx = tid; idx < pairs; idx += THREADS) {
    const int g = idx / (D / 2), d = 2 * (idx % (D / 2));
    const int64_t row0 = int64_t(s0) * a.num_qo_heads + hq0 + g;
    constexpr int kBatch = 8;   // partials read together, so their latencies overlap
    // The maximum from a number on: a row whose log-sum-exps are all NaN gets NaN
    // weights, one of no tokens (all -infinity) none.
    float mx = kNegBig, wsum = 0.f, x = 0.f, y = 0.f;
    for (int j = 0; j < n; j += kBatch) {
      float lse[kBatch];
      uint64_t po[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t row = row0 + int64_t(min(j + u, n - 1)) * a.num_qo_heads;
        lse[u] = __hip_atomic_load(a.part_lse + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        po[u] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(a.part_o + row * D + d),
                                  __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      float m2 = mx;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) m2 = j + u < n ? fmaxf(m2, lse[u]) : m2;
      const float keep = fast_exp2(mx - m2);
      mx = m2;
      wsum *= keep;
      x *= keep;
      y *= keep;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (j + u >= n) break;   // uniform: the last partial again, of no weight (0 x inf)
        const float w = fast_exp2(lse[u] - m2);
        wsum += w;
        x = fmaf(w, bits_to_f32(int(uint32_t(po[u]))), x);
        y = fmaf(w, bits_to_f32(int(uint32_t(po[u] >> 32))), y);
      }
    }
    const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
    write_out(g, d, x * inv, y * inv);
    if (d == 0 && a.lse)
      a.lse[int64_t(seq) * a.num_qo_heads + hq0 + g] = wsum == 0.f ? -INFINITY : mx + __log2f(wsum);
  }
}

// The MFMA kernels' step of K and V (paged_decode_mfma_kernel): which lane loads
// what, and which token is which row of the 16x16 score tiles.
template <int D>
struct DecodeTile {
  static constexpr int CH = D / 8;            // 16-byte chunks per token row
  static constexpr int TPL = kWave / CH;      // token rows per load instruction
  static constexpr int LOADS = 8;             // loads per lane per step (K and V each)
  static constexpr int STEP = TPL * LOADS;    // tokens per wave iteration
  static constexpr int PAIRS = D == 64 ? 2 : 1;   // pairs of 16-token score tiles per step
  static constexpr int ACCS = D == 128 ? 1 : 2;   // accumulator sets of 8
  // Step token of element i (0..7) of lane group g, score pair p.
  static __device__ __forceinline__ int token(int i, int g, int p) {
    return D == 64 ? 8 * i + 2 * g + p : D == 128 ? 4 * i + g : 2 * i + (g >> 1);
  }
  // XOR of token t's chunk index in the LDS block: the 8 rows that 8
  // consecutive lanes read differ in it.
  static __device__ __forceinline__ int swz(int t) {
    return D == 64 ? ((t >> 3) & 3) | ((t & 2) << 1) : D == 128 ? t & 15 : t & 7;
  }
};

// A partial's log-sum-exp from its maximum and sum. A NaN score makes the quotient of
// sums NaN, and with a weight that is a number, 0 at least, the row's output.
__device__ __forceinline__ float partial_lse(float m, float sum) {
  return sum > 0.f ? m + __log2f(sum) : sum == 0.f ? -INFINITY : m;
}

// A row's; for a launch that leaves its scores, NaN where a score is.
__device__ __forceinline__ float row_lse(const DecodeArgs& a, float m, float sum) {
  return sum > 0.f ? m + __log2f(sum) : a.lse && sum != sum ? sum : -INFINITY;
}

// One head's attention over the tokens of a wave's steps (from t0 on, every
// `stride`), in fp32 on the vector
// units and a load at a time: what the MFMA kernel falls back to for values
// that its products do not carry. Lane (row lane / CH, chunk lane % CH) holds
// dims 8 chunk .. + 7 in acc, the same in every row after the merge; kb and vb
// point at the lane's chunk.
template <typename T, int D>
__device__ __forceinline__ void wave_rows(const DecodeArgs& a, typename Vec<T>::v8 q, const f16* kb,
                                          const f16* vb, int tb, int t0, int stride, int te,
                                          const int* s_pages, const NewRow& nr, float& m, float& l,
                                          float (&acc)[8]) {
  typedef DecodeTile<D> L;
  const int lane = threadIdx.x & (kWave - 1);
  m = kNegBig;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  for (; t0 < te; t0 += stride)
#pragma unroll 1
    for (int i = 0; i < L::LOADS; ++i) {
      const int t = t0 + L::TPL * i + lane / L::CH;
      const int p = t < te ? s_pages[(t >> a.page_shift) - (tb >> a.page_shift)] : -1;
      const int64_t off = int64_t(max(p, 0)) * a.page_stride +
                          int64_t(t & ((1 << a.page_shift) - 1)) * a.token_stride;
      const f16* zero = g_zero_row + 8 * (lane % L::CH);
      const auto k = load_v8<T>(p >= 0 ? kb + (t == nr.pos ? nr.k : off) : zero);
      const auto v = load_v8<T>(p >= 0 ? vb + (t == nr.pos ? nr.v : off) : zero);
      float s = group_sum<L::CH>(dot8(q, k, 0.f)) * a.scale_log2;
      s = p >= 0 ? s : -INFINITY;
      const float mx = fmaxf(m, s);
      const float alpha = fast_exp2(m - mx), pr = fast_exp2(s - mx);
      m = mx;
      l = fmaf(l, alpha, pr);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(pr, float(v[e]), acc[e] * alpha);
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

}  // namespace
}  // namespace kunserve
