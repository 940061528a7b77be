// Eviction from the cache by accumulated attention weight: of each (row,
// layer, KV head) the first `sinks` tokens, the last `recent` ones and the
// heaviest of those between stay, in their order, in pages of their own.
//
// The heaviest are found by radix selection on the weights' bits (an order on
// unsigned integers that agrees with the order of fp32): the key of the last
// one that stays is built from the top, 11, 11 and 10 bits at a time, from
// histograms of the tokens that agree with it so far. Tokens above it stay, and
// of those that equal it the first ones (the lowest indices).
//
// HBM-bound: 4 bytes per cached token and head are read to choose, and the K,
// V and weight of what stays are read and written once. Two launches: a
// workgroup per (row, layer, head) chooses; then workgroups of kMoveTokens
// kept tokens move them, so that a single row's move is spread over the device
// too. The choice reads its weights once, into registers: the tokens of a wave are
// consecutive, 64 at a time, so a ballot gives a token's place among those that
// stay and only the waves' totals meet in LDS.
#include "common.hpp"

namespace kunserve {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveTokens = 64;
constexpr int kBins = 2048;   // of 11 bits

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
  int32_t max_keep, max_len, sinks, recent;
  int32_t* kept;               // [num_seqs][layers][heads][kept_stride]
  int64_t kept_stride;
};

// Unsigned order of fp32 weights; both zeros are equal, NaN is below all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
  if (w != w) return 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of x over the workgroup of W waves; total: the sum.
template <int W>
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
  for (int i = 0; i < W; ++i) {
    const int y = s_sums[i];
    if (i < wave) before += y;
    total += y;
  }
  return before + incl - x;
}

// KPT: keys a thread holds in registers (0: they are read again where they are
// needed; for middles longer than W * 64 * 32).
template <int W, int KPT>
__global__ __launch_bounds__(W * kWave) void evict_choose_kernel(EvictArgs a) {
  constexpr int THREADS = W * kWave, BPT = kBins / THREADS;
  __shared__ int s_hist[kBins];
  __shared__ int s_sums[W];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int head = blockIdx.x, layer = blockIdx.y, seq = blockIdx.z;
  const int n = min(a.kv_len[seq], a.max_len);
  const int keep = min(min(a.keep[seq], a.max_keep), n);
  int32_t* kept = a.kept + ((int64_t(seq) * a.num_layers + layer) * a.num_kv_heads + head) *
                               a.kept_stride;
  for (int64_t j = max(keep, 0) + tid; j < a.kept_stride; j += THREADS) kept[j] = -1;
  if (keep <= 0) return;   // uniform
  if (keep == n) {
    for (int j = tid; j < n; j += THREADS) kept[j] = j;
    return;
  }
  // The first ones come before the last ones where both are more than stay.
  // The middle [lo, hi) is longer than the tokens it keeps (n > keep).
  const int lo = min(a.sinks, keep), recent = min(a.recent, keep - lo), hi = n - recent;
  int need = keep - lo - recent;
  for (int j = tid; j < lo; j += THREADS) kept[j] = j;
  for (int j = tid; j < recent; j += THREADS) kept[keep - recent + j] = hi + j;
  if (need == 0) return;   // uniform
  const int32_t* pages = a.indices + a.indptr[seq];
  const float* w = a.w + int64_t(layer) * a.w_layer + int64_t(head) * a.w_head;
  const int mask = (1 << a.page_shift) - 1;
  // Round r of a wave: tokens lo + (wave * rounds + r) * 64 + lane.
  const int rounds = (hi - lo + THREADS - 1) / THREADS;
  const int first = lo + wave * rounds * kWave + lane;
  auto read_key = [&](int t) -> uint32_t {
    const int p = pages[t >> a.page_shift];
    return p >= 0 && p < a.num_pages ? weight_key(w[int64_t(p) * a.w_page + (t & mask)]) : 0u;
  };
  uint32_t keys[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int r = 0; r < KPT; ++r) {
      const int t = first + r * kWave;
      keys[r] = r < rounds && t < hi ? read_key(t) : 0u;
    }
  }
  // f(token, key) for the thread's tokens, by whole waves (token >= hi: none).
  auto each = [&](auto f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int r = 0; r < KPT; ++r)
        if (r < rounds) f(first + r * kWave, keys[r]);   // uniform
    } else {
      for (int r = 0; r < rounds; ++r) {
        const int t = first + r * kWave;
        f(t, t < hi ? read_key(t) : 0u);
      }
    }
  };

  uint32_t prefix = 0;   // the key's bits so far
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t high = pass == 0 ? 0u : ~0u << (pass == 1 ? 21 : 10);
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
#pragma unroll
    for (int i = 0; i < BPT; ++i) s_hist[tid + i * THREADS] = 0;
    __syncthreads();
    each([&](int t, uint32_t key) {
      const bool in = t < hi && (key & high) == prefix;
      const int bin = int((key >> shift) & digits);
      if (in) {
        // Tokens of equal weight are many where weights are few (zeros): one add.
        const int bin0 = __builtin_amdgcn_readfirstlane(bin);
        const uint64_t who = __ballot(true);
        if (__ballot(bin != bin0) != 0)
          atomicAdd(&s_hist[bin], 1);
        else if (lane == __builtin_ctzll(who))
          atomicAdd(&s_hist[bin0], __popcll(who));
      }
    });
    __syncthreads();
    // Bins from above, BPT to a thread: the one in which the need-th falls.
    int mine = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) mine += s_hist[kBins - 1 - tid * BPT - i];
    int total;
    int above = block_scan<W>(mine, s_sums, total);
    if (above < need && need <= above + mine) {
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        const int bin = kBins - 1 - tid * BPT - i, count = s_hist[bin];
        if (above < need && need <= above + count) {
          s_prefix = prefix | uint32_t(bin) << shift;
          s_need = need - above;
        }
        above += count;
      }
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;   // tokens wanted among those that agree with prefix
  }

  // The wave's tokens above the key, and its ties; then both before the wave.
  int over = 0, ties = 0, total;
  each([&](int t, uint32_t key) {
    over += __popcll(__ballot(t < hi && key > prefix));
    ties += __popcll(__ballot(t < hi && key == prefix));
  });
  int seen = block_scan<W>(lane == 0 ? ties : 0, s_sums, total);
  seen = __shfl(seen, 0);   // ties before
  const int staying = over + min(max(need - seen, 0), ties);
  int at = block_scan<W>(lane == 0 ? staying : 0, s_sums, total);
  at = lo + __shfl(at, 0);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  each([&](int t, uint32_t key) {
    const uint64_t tie = __ballot(t < hi && key == prefix);
    const bool stays = t < hi && (key > prefix || (key == prefix && seen + __popcll(tie & below) < need));
    seen += __popcll(tie);
    const uint64_t who = __ballot(stays);
    if (stays) kept[at + __popcll(who & below)] = t;
    at += __popcll(who);
  });
}

// Moves kept tokens: 16-byte chunks of K and of V, a thread's loads of all its
// tokens before their stores. Non-temporal both ways: 8 rows halved, 32 layers of 8
// heads of 128 (3.4 GB) 666 us against 688 with plain stores: 5.2 TB/s, what a
// large copy reaches.
template <int D>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int CH = D / 8;                       // 16-byte chunks per row
  constexpr int ROWS = kMoveThreads / CH;         // tokens per step
  constexpr int STEPS = kMoveTokens / ROWS;
  constexpr int BATCH = STEPS < 4 ? STEPS : 4;
  __shared__ int64_t s_src[kMoveTokens], s_dst[kMoveTokens];
  const int seq = blockIdx.z;
  const int head = int(blockIdx.y) % a.num_kv_heads, layer = int(blockIdx.y) / a.num_kv_heads;
  const int n = min(min(a.keep[seq], a.max_keep), min(a.kv_len[seq], a.max_len));
  const int j0 = int(blockIdx.x) * kMoveTokens;
  if (j0 >= n) return;   // uniform
  const int cnt = min(kMoveTokens, n - j0);
  const int mask = (1 << a.page_shift) - 1;
  if (int(threadIdx.x) < kMoveTokens) {
    int64_t from = -1, to = -1;
    if (int(threadIdx.x) < cnt) {
      const int j = j0 + threadIdx.x;
      const int t = a.kept[((int64_t(seq) * a.num_layers + layer) * a.num_kv_heads + head) *
                               a.kept_stride + j];
      const int p = a.indices[a.indptr[seq] + (t >> a.page_shift)];
      const int d = a.out_indices[a.out_indptr[seq] + (j >> a.page_shift)];
      const bool src_ok = p >= 0 && p < a.num_pages, dst_ok = d >= 0 && d < a.num_pages;
      if (src_ok) from = int64_t(p) * a.page_stride + int64_t(t & mask) * a.token_stride;
      if (dst_ok) to = int64_t(d) * a.page_stride + int64_t(j & mask) * a.token_stride;
      float* w = a.w + int64_t(layer) * a.w_layer + int64_t(head) * a.w_head;
      if (dst_ok)
        w[int64_t(d) * a.w_page + (j & mask)] = src_ok ? w[int64_t(p) * a.w_page + (t & mask)] : 0.f;
    }
    s_src[threadIdx.x] = from;
    s_dst[threadIdx.x] = to;
  }
  __syncthreads();
  const int64_t base = int64_t(layer) * a.layer_stride + int64_t(head) * a.head_stride +
                       8 * (threadIdx.x % CH);
  const int row = threadIdx.x / CH;
#pragma unroll
  for (int i0 = 0; i0 < STEPS; i0 += BATCH) {
    f16x8 x[BATCH], y[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int64_t from = s_src[row + (i0 + i) * ROWS];
      x[i] = y[i] = f16x8{};   // a token of no page of the pool: zeros
      if (from >= 0) {
        x[i] = load_f16x8_nt(a.k + base + from);
        y[i] = load_f16x8_nt(a.v + base + from);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int64_t to = s_dst[row + (i0 + i) * ROWS];
      if (to < 0) continue;
      __builtin_nontemporal_store(x[i], reinterpret_cast<f16x8*>(a.k + base + to));
      __builtin_nontemporal_store(y[i], reinterpret_cast<f16x8*>(a.v + base + to));
    }
  }
}

// How many waves choose, and what they hold. A workgroup waits at barriers most of
// its time: few of them take 16 waves each, many take 4 so that a CU holds more of
// them (2048 of up to 5000 tokens: 63 us against 96 with 16 waves; 56 and, for 64 of
// 5000 with 16 waves, 13 since ties and what is above them are counted in one pass).
void launch_choose(const EvictArgs& a, dim3 grid, int32_t max_len, hipStream_t s) {
  const int64_t workgroups = int64_t(grid.x) * grid.y * grid.z;
  if (max_len <= 4 * kWave * 16)
    evict_choose_kernel<4, 16><<<grid, 4 * kWave, 0, s>>>(a);
  else if (max_len <= 4 * kWave * 32 && workgroups >= 512)
    evict_choose_kernel<4, 32><<<grid, 4 * kWave, 0, s>>>(a);
  else if (max_len <= 16 * kWave * 16)
    evict_choose_kernel<16, 16><<<grid, 16 * kWave, 0, s>>>(a);
  else if (max_len <= 16 * kWave * 32)
    evict_choose_kernel<16, 32><<<grid, 16 * kWave, 0, s>>>(a);
  else
    evict_choose_kernel<16, 0><<<grid, 16 * kWave, 0, s>>>(a);
}

template <int D>
int launch_move(const EvictArgs& a, dim3 grid, hipStream_t s) {
  evict_move_kernel<D><<<grid, kMoveThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

}  // namespace

}  // namespace kunserve

using namespace kunserve;

extern "C" int kunserve_evict(const kunserve_kv_pool* pool, const kunserve_kv_weights* weights,
                              const kunserve_page_table* table, const int32_t* out_indptr_dev,
                              const int32_t* out_indices_dev, const int32_t* keep_dev,
                              int32_t max_keep, int32_t max_len, int32_t sinks, int32_t recent,
                              int32_t* kept_dev, int64_t kept_stride,
                              kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  rc = check_weights(weights, pool);
  if (rc) return rc;
  KSV_CHECK_ARG(table && table->num_seqs >= 0, "null table or num_seqs < 0");
  KSV_CHECK_ARG(sinks >= 0 && recent >= 0, "sinks %d or recent %d < 0", sinks, recent);
  KSV_CHECK_ARG(max_len >= 0, "max_len %d < 0", max_len);
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
  a.max_len = max_len;
  a.sinks = sinks;
  a.recent = recent;
  a.kept = kept_dev;
  a.kept_stride = kept_stride;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  launch_choose(a, dim3(unsigned(a.num_kv_heads), unsigned(a.num_layers),
                        unsigned(table->num_seqs)), max_len, s);
  KSV_CHECK_LAUNCH();
  const dim3 grid(unsigned((max_keep + kMoveTokens - 1) / kMoveTokens),
                  unsigned(a.num_layers * a.num_kv_heads), unsigned(table->num_seqs));
  switch (pool->head_dim) {
    case 64: return launch_move<64>(a, grid, s);
    case 128: return launch_move<128>(a, grid, s);
    default: return launch_move<256>(a, grid, s);
  }
}
