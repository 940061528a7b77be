// Eviction from the cache by accumulated attention weight: of each (row,
// layer, KV head) the first `sinks` tokens, the last `recent` ones and the
// heaviest of those between stay, in their order, in pages of their own.
//
// The heaviest are found by radix selection on the weights' bits (an order on
// unsigned integers that agrees with the order of fp32): the key of the last
// one that stays is built from the top, 8 bits at a time, from histograms of
// the tokens that agree with it so far. Tokens above it stay, and of those
// that equal it the first ones (the lowest indices).
//
// HBM-bound: 4 bytes per cached token and head are read to choose, and the K,
// V and weight of what stays are read and written once. Two launches: a
// workgroup per (row, layer, head) chooses; then workgroups of kMoveTokens
// kept tokens move them, so that a single row's move is spread over the device
// too.
#include "common.hpp"

namespace kunserve {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMoveTokens = 64;

struct EvictArgs {
  f16* k;
  f16* v;
  int64_t page_stride, layer_stride, head_stride, token_stride;
  float* w;
  int64_t w_page, w_layer, w_head;
  int32_t num_pages, page_shift, num_kv_heads, num_layers;
  const int32_t* indptr;       // the rows' pages
  const int32_t* indices;
  const int32_t* kv_len;
  const int32_t* out_indptr;   // the pages that are filled
  const int32_t* out_indices;
  const int32_t* keep;         // [num_seqs] tokens that stay (kv_len and max_keep at most)
  int32_t max_keep, sinks, recent;
  int32_t* kept;               // [num_seqs][layers][heads][kept_stride]
  int64_t kept_stride;
};

// Unsigned order of fp32 weights; both zeros are equal, NaN is below all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
  if (w != w) return 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of x over the workgroup; total: the sum.
__device__ __forceinline__ int block_scan(int x, int* s_sums, int& total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int y = __shfl_up(incl, off);
    if (lane >= off) incl += y;
  }
  __syncthreads();   // s_sums of the call before has been read
  if (lane == kWave - 1) s_sums[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave) before += s_sums[i];
    total += s_sums[i];
  }
  return before + incl - x;
}

__global__ __launch_bounds__(kThreads) void evict_choose_kernel(EvictArgs a) {
  __shared__ int s_hist[256];
  __shared__ int s_sums[kWaves];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x;
  const int head = blockIdx.x, layer = blockIdx.y, seq = blockIdx.z;
  const int n = a.kv_len[seq];
  const int keep = min(min(a.keep[seq], a.max_keep), n);
  int32_t* kept = a.kept + ((int64_t(seq) * a.num_layers + layer) * a.num_kv_heads + head) *
                               a.kept_stride;
  for (int64_t j = max(keep, 0) + tid; j < a.kept_stride; j += kThreads) kept[j] = -1;
  if (keep <= 0) return;   // uniform
  if (keep == n) {
    for (int j = tid; j < n; j += kThreads) kept[j] = j;
    return;
  }
  // The first ones come before the last ones where both are more than stay.
  // The middle [lo, hi) is longer than the tokens it keeps (n > keep).
  const int lo = min(a.sinks, keep), recent = min(a.recent, keep - lo), hi = n - recent;
  int need = keep - lo - recent;
  const int32_t* pages = a.indices + a.indptr[seq];
  const float* w = a.w + int64_t(layer) * a.w_layer + int64_t(head) * a.w_head;
  const int mask = (1 << a.page_shift) - 1;
  auto key_at = [&](int t) -> uint32_t {
    const int p = pages[t >> a.page_shift];
    return p >= 0 && p < a.num_pages ? weight_key(w[int64_t(p) * a.w_page + (t & mask)]) : 0u;
  };
  uint32_t prefix = 0;   // the key's bits so far
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_hist[tid] = 0;
      __syncthreads();
      const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int t = lo + tid; t < hi; t += kThreads) {
        const uint32_t key = key_at(t);
        if ((key & high) == prefix) atomicAdd(&s_hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      // Bin 255 - tid counted from above: the one in which the need-th falls.
      int total;
      const int mine = s_hist[255 - tid];
      const int above = block_scan(mine, s_sums, total);
      if (above < need && need <= above + mine) {
        s_prefix = prefix | uint32_t(255 - tid) << shift;
        s_need = need - above;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;   // tokens wanted among those that agree with prefix
    }
  }
  // In index order: the first ones, the middle's choice, the last ones.
  for (int j = tid; j < lo; j += kThreads) kept[j] = j;
  for (int j = tid; j < recent; j += kThreads) kept[keep - recent + j] = hi + j;
  if (keep == lo + recent) return;   // uniform
  int at = lo, equal = 0;
  for (int t0 = lo; t0 < hi; t0 += kThreads) {
    const int t = t0 + tid;
    const uint32_t key = t < hi ? key_at(t) : 0u;
    const bool tie = t < hi && key == prefix;
    int ties, chosen;
    const int rank = equal + block_scan(tie, s_sums, ties);
    const bool stays = t < hi && (key > prefix || (tie && rank < need));
    const int pos = at + block_scan(stays, s_sums, chosen);
    if (stays) kept[pos] = t;
    equal += ties;
    at += chosen;
  }
}

// Moves kept tokens: a 16-byte chunk of K and of V per thread and step.
template <int D>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int CH = D / 8;                   // 16-byte chunks per row
  constexpr int ROWS = kThreads / CH;         // tokens per step
  __shared__ int64_t s_src[kMoveTokens], s_dst[kMoveTokens];
  const int seq = blockIdx.z;
  const int head = int(blockIdx.y) % a.num_kv_heads, layer = int(blockIdx.y) / a.num_kv_heads;
  const int n = min(min(a.keep[seq], a.max_keep), a.kv_len[seq]);
  const int j0 = int(blockIdx.x) * kMoveTokens;
  if (j0 >= n) return;   // uniform
  const int cnt = min(kMoveTokens, n - j0);
  const int mask = (1 << a.page_shift) - 1;
  if (int(threadIdx.x) < cnt) {
    const int j = j0 + threadIdx.x;
    const int t = a.kept[((int64_t(seq) * a.num_layers + layer) * a.num_kv_heads + head) *
                             a.kept_stride + j];
    const int p = a.indices[a.indptr[seq] + (t >> a.page_shift)];
    const int d = a.out_indices[a.out_indptr[seq] + (j >> a.page_shift)];
    const bool src_ok = p >= 0 && p < a.num_pages, dst_ok = d >= 0 && d < a.num_pages;
    s_src[threadIdx.x] = src_ok ? int64_t(p) * a.page_stride + int64_t(t & mask) * a.token_stride : -1;
    s_dst[threadIdx.x] = dst_ok ? int64_t(d) * a.page_stride + int64_t(j & mask) * a.token_stride : -1;
    float* w = a.w + int64_t(layer) * a.w_layer + int64_t(head) * a.w_head;
    if (dst_ok)
      w[int64_t(d) * a.w_page + (j & mask)] = src_ok ? w[int64_t(p) * a.w_page + (t & mask)] : 0.f;
  }
  __syncthreads();
  const int64_t base = int64_t(layer) * a.layer_stride + int64_t(head) * a.head_stride +
                       8 * (threadIdx.x % CH);
  for (int i = threadIdx.x / CH; i < cnt; i += ROWS) {
    if (s_dst[i] < 0) continue;
    f16x8 x = {}, y = {};   // a token of no page of the pool: zeros
    if (s_src[i] >= 0) {
      x = load_f16x8_nt(a.k + base + s_src[i]);
      y = load_f16x8_nt(a.v + base + s_src[i]);
    }
    store_f16x8(a.k + base + s_dst[i], x);
    store_f16x8(a.v + base + s_dst[i], y);
  }
}

template <int D>
int launch_move(const EvictArgs& a, dim3 grid, hipStream_t s) {
  evict_move_kernel<D><<<grid, kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

}  // namespace

}  // namespace kunserve

using namespace kunserve;

extern "C" int kunserve_evict(const kunserve_kv_pool* pool, const kunserve_kv_weights* weights,
                              const kunserve_page_table* table, const int32_t* out_indptr_dev,
                              const int32_t* out_indices_dev, const int32_t* keep_dev,
                              int32_t max_keep, int32_t sinks, int32_t recent, int32_t* kept_dev,
                              int64_t kept_stride, kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  rc = check_weights(weights, pool);
  if (rc) return rc;
  KSV_CHECK_ARG(table && table->num_seqs >= 0, "null table or num_seqs < 0");
  KSV_CHECK_ARG(sinks >= 0 && recent >= 0, "sinks %d or recent %d < 0", sinks, recent);
  KSV_CHECK_ARG(max_keep >= 0 && kept_stride >= max_keep, "kept_stride %lld below max_keep %d",
                (long long)kept_stride, max_keep);
  if (table->num_seqs == 0 || max_keep == 0) return KUNSERVE_OK;
  KSV_CHECK_ARG(table->indptr_dev && table->indices_dev && table->kv_len_dev && out_indptr_dev &&
                    out_indices_dev && keep_dev && kept_dev,
                "null table array, keep or kept");
  KSV_CHECK_ARG(table->num_seqs < 65536, "%d rows: at most 65535", table->num_seqs);
  KSV_CHECK_ARG(pool->num_layers < 65536 &&
                    int64_t(pool->num_layers) * pool->num_kv_heads < 65536,
                "%d layers of %d heads: at most 65535 together", pool->num_layers,
                pool->num_kv_heads);
  EvictArgs a{};
  a.k = static_cast<f16*>(pool->k);
  a.v = static_cast<f16*>(pool->v);
  a.page_stride = pool->page_stride;
  a.layer_stride = pool->layer_stride;
  a.head_stride = pool->head_stride;
  a.token_stride = pool->token_stride;
  a.w = weights->w;
  a.w_page = weights->page_stride;
  a.w_layer = weights->layer_stride;
  a.w_head = weights->head_stride;
  a.num_pages = int32_t(pool->num_pages);
  a.page_shift = __builtin_ctz(pool->page_size);
  a.num_kv_heads = pool->num_kv_heads;
  a.num_layers = pool->num_layers;
  a.indptr = table->indptr_dev;
  a.indices = table->indices_dev;
  a.kv_len = table->kv_len_dev;
  a.out_indptr = out_indptr_dev;
  a.out_indices = out_indices_dev;
  a.keep = keep_dev;
  a.max_keep = max_keep;
  a.sinks = sinks;
  a.recent = recent;
  a.kept = kept_dev;
  a.kept_stride = kept_stride;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  evict_choose_kernel<<<dim3(unsigned(a.num_kv_heads), unsigned(a.num_layers),
                             unsigned(table->num_seqs)),
                        kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  const dim3 grid(unsigned((max_keep + kMoveTokens - 1) / kMoveTokens),
                  unsigned(a.num_layers * a.num_kv_heads), unsigned(table->num_seqs));
  switch (pool->head_dim) {
    case 64: return launch_move<64>(a, grid, s);
    case 128: return launch_move<128>(a, grid, s);
    default: return launch_move<256>(a, grid, s);
  }
}
