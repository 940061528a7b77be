// Cached tokens that change their place: of a row's tokens those that stay moved
// together (kunserve_keep_tokens), and rows continued in pages of their own
// (kunserve_copy_pages). The reference moves whole blocks alone
// (LlamaOp.local_copy_blocks, kunserve/worker.py:818-823).
//
// Both are HBM-bound copies of 16-byte chunks: what moves is read and written once.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "common.hpp"

namespace kunserve {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kLoads = 8;   // 16-byte loads of a lane that are under way together
constexpr int64_t kMaxBlocks = (int64_t(1) << 32) / kThreads;   // a launch's threads fit 32 bits

struct KeepArgs {
  f16* k;
  f16* v;
  int64_t page_stride, layer_stride, head_stride, token_stride;
  float* w;   // null, or the tokens' weights
  int64_t w_page, w_layer, w_head;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* kv_len;
  const int32_t* kept;
  int64_t kept_stride;
  int32_t max_kept;
  int32_t num_pages;
  int32_t page_shift;
  int32_t num_layers;
  int32_t num_heads;
  int64_t num_slabs;   // rows x layers x heads, x K and V where they are a workgroup's each
};

// [rows]: the rows' first places, which for few rows go with the launch's arguments (small rows
// cut short 15 us a call with the host's work, 29 with an upload and more of that).
struct FirstThere {
  const int32_t* at;
};
struct FirstHere {
  int32_t at[KUNSERVE_FIRST_BY_VALUE];
};

// A slab is a row's tokens of one layer and KV head, K and V for a wave (W 1), one of them
// for a workgroup. It moves chunk by chunk: slots [c, c + n) are written after the tokens
// kept[c], .. kept[c + n - 1] have been read, by the wave or by the workgroup, which meets
// between. A token moves down (kept[j] > j), so what a later chunk reads no earlier one has
// written. Accepted paths are short, and a wave waits for what it reads: rows, lists, page
// ids, tokens (64 rows, 32 layers of 8 heads: 17 us, 20 with a wave each for K and V).
template <int D, int W, typename First>
__global__ __launch_bounds__(kThreads) void keep_tokens_kernel(KeepArgs a, First from_place) {
  constexpr int CH = D / 8;
  constexpr int TPL = kWave / CH;                 // tokens of a load
  constexpr int KV = W == 1 ? 2 : 1;              // K and V of a wave's tokens, or one of them
  constexpr int N = kLoads / KV;                  // loads of either
  constexpr int CHUNK = N * TPL * W;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int64_t slab = W == 1 ? int64_t(blockIdx.x) * kWaves + wave : blockIdx.x;
  if (slab >= a.num_slabs) return;   // uniform in a wave; no barrier where W is 1
  const int head = int(slab % a.num_heads);
  const int64_t rest = slab / a.num_heads;
  const int layer = int(rest % a.num_layers);
  const bool of_v = KV == 1 && (rest / a.num_layers & 1);
  const int b = int(rest / a.num_layers / (KV == 1 ? 2 : 1));
  const int lrow = lane / CH, lcol = lane % CH;

  const int first = from_place.at[b], len = a.kv_len[b] - first;
  if (first < 0 || len <= 1) return;   // uniform
  const int32_t* pages = a.indices + a.indptr[b];
  const int32_t* kept = a.kept + int64_t(b) * a.kept_stride;
  const int mask = (1 << a.page_shift) - 1;
  const int64_t at = int64_t(layer) * a.layer_stride + int64_t(head) * a.head_stride + 8 * lcol;
  f16* const base[2] = {(of_v ? a.v : a.k) + at, a.v + at};
  float* weights = a.w && !of_v && lcol == 0
                       ? a.w + int64_t(layer) * a.w_layer + int64_t(head) * a.w_head
                       : nullptr;

  const int n = min(a.max_kept, len);
  for (int c = 0; c < n; c += CHUNK) {
    int from[N], src[N], dst[N];
    f16x8 x[KV][N];
    float w[N];
    auto place = [&](int i) { return c + ((W == 1 ? 0 : wave) + W * i) * TPL + lrow; };
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = place(i);
      from[i] = j < n ? kept[j] : -1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool moves = from[i] > place(i) && from[i] < len;
      src[i] = moves ? pages[(first + from[i]) >> a.page_shift] : -1;
      dst[i] = moves ? pages[(first + place(i)) >> a.page_shift] : -1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool ok = src[i] >= 0 && src[i] < a.num_pages;
      const int slot = (first + from[i]) & mask;
#pragma unroll
      for (int z = 0; z < KV; ++z)
        x[z][i] = ok ? load_f16x8(base[z] + int64_t(src[i]) * a.page_stride + int64_t(slot) * a.token_stride)
                     : f16x8{};
      if (a.w) w[i] = ok && weights ? weights[int64_t(src[i]) * a.w_page + slot] : 0.f;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // read before any of it is overwritten
    if constexpr (W > 1) __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (dst[i] < 0 || dst[i] >= a.num_pages) continue;
      const int slot = (first + place(i)) & mask;
#pragma unroll
      for (int z = 0; z < KV; ++z)
        store_f16x8(base[z] + int64_t(dst[i]) * a.page_stride + int64_t(slot) * a.token_stride, x[z][i]);
      if (weights) weights[int64_t(dst[i]) * a.w_page + slot] = w[i];
    }
  }
}

struct CopyArgs {
  f16* k;
  f16* v;
  int64_t page_stride, layer_stride, head_stride, token_stride;
  float* w;
  int64_t w_page, w_layer, w_head;
  int32_t num_pages;
  int32_t page_size;
  int32_t num_heads;
  int32_t heads, parts;   // heads of a workgroup, workgroups of all
};

// [n][3]: source page, destination page, tokens. Few of them go with the launch's
// arguments: an upload of their own takes longer than they do (8 samples' last pages, with
// building the table: 22 us against 30).
struct MovesThere {
  const int32_t* m;
};
struct MovesHere {
  int32_t m[3 * KUNSERVE_MOVES_BY_VALUE];
};

// Workgroup (move, layer and K or V, head group): the waves take the loads of its heads'
// tokens in turn. Moves are the slowest: those of one source read the same rows on one XCD
// where the groups are a multiple of eight, and neighbours in time are pages apart (eight
// pages of 76 tokens, 32 layers of 8 heads: 14 us from one source and 20 from eight; with the
// moves fastest 41 and 36). Past the caches only the writes: reads too 26 and 28.
template <int D, typename Moves>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a, Moves moves) {
  constexpr int CH = D / 8;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int slab = int(blockIdx.x);
  const int64_t at3 = 3 * int64_t(blockIdx.y);
  const int from = moves.m[at3], to = moves.m[at3 + 1], tokens = min(moves.m[at3 + 2], a.page_size);
  if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages || tokens <= 0) return;
  const int h0 = slab % a.parts * a.heads, layer = slab / a.parts >> 1;
  const bool of_v = slab / a.parts & 1;
  const int nh = min(a.heads, a.num_heads - h0);
  f16* base = (of_v ? a.v : a.k) + int64_t(layer) * a.layer_stride;
  const f16* src = base + int64_t(from) * a.page_stride;
  f16* dst = base + int64_t(to) * a.page_stride;
  const int per_head = (tokens * CH + kWave - 1) / kWave, total = per_head * nh;   // uniform
  for (int at = wave; at < total; at += kWaves * kLoads) {
    u32x4 x[kLoads];
    int64_t off[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int l = at + i * kWaves, h = l / per_head;   // uniform
      const int unit = (l - h * per_head) * kWave + lane;
      const bool in = l < total && unit < tokens * CH;
      off[i] = in ? int64_t(h0 + h) * a.head_stride + int64_t(unit / CH) * a.token_stride + 8 * (unit % CH)
                  : -1;
      if (in) x[i] = *reinterpret_cast<const u32x4*>(src + off[i]);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (off[i] >= 0) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(dst + off[i]));
  }
  if (a.w && !of_v) {
    float* w = a.w + int64_t(layer) * a.w_layer;
    for (int u = threadIdx.x; u < nh * a.page_size; u += kThreads) {
      const int h = h0 + u / a.page_size, t = u % a.page_size;
      if (t < tokens)
        w[int64_t(to) * a.w_page + int64_t(h) * a.w_head + t] =
            w[int64_t(from) * a.w_page + int64_t(h) * a.w_head + t];
    }
  }
}

template <int D>
void keep_tokens(dim3 grid, bool small, const KeepArgs& a, const int32_t* first_host,
                 const int32_t* first_dev, int32_t rows, hipStream_t s) {
  auto launch = [&](const auto& first) {
    typedef std::decay_t<decltype(first)> First;
    if (small)
      keep_tokens_kernel<D, 1, First><<<grid, kThreads, 0, s>>>(a, first);
    else
      keep_tokens_kernel<D, kWaves, First><<<grid, kThreads, 0, s>>>(a, first);
  };
  if (first_host) {
    FirstHere here;
    std::copy_n(first_host, rows, here.at);
    launch(here);
  } else {
    launch(FirstThere{first_dev});
  }
}

template <int D>
void copy_pages(dim3 grid, const CopyArgs& a, const int32_t* moves_host, const int32_t* moves_dev,
                hipStream_t s) {
  if (moves_host) {
    MovesHere here;
    std::copy_n(moves_host, 3 * grid.y, here.m);
    copy_pages_kernel<D><<<grid, kThreads, 0, s>>>(a, here);
  } else {
    copy_pages_kernel<D><<<grid, kThreads, 0, s>>>(a, MovesThere{moves_dev});
  }
}

}  // namespace
}  // namespace kunserve

using namespace kunserve;

extern "C" int kunserve_keep_tokens(const kunserve_kv_pool* pool,
                                    const kunserve_kv_weights* weights,
                                    const kunserve_page_table* table, const int32_t* first_host,
                                    const int32_t* first_dev, const int32_t* kept_dev,
                                    int64_t kept_stride, int32_t max_kept,
                                    kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  if (weights) {
    rc = check_weights(weights, pool);
    if (rc) return rc;
  }
  KSV_CHECK_ARG(table && table->num_seqs >= 0, "null table or num_seqs < 0");
  KSV_CHECK_ARG(max_kept >= 0 && kept_stride >= max_kept, "kept rows of %lld hold %d entries",
                (long long)kept_stride, max_kept);
  if (table->num_seqs == 0 || max_kept == 0) return KUNSERVE_OK;
  KSV_CHECK_ARG(table->indptr_dev && table->indices_dev && table->kv_len_dev && kept_dev,
                "null table array or kept");
  KSV_CHECK_ARG(!first_host != !first_dev, "first places are either on the host or on the device");
  KSV_CHECK_ARG(!first_host || table->num_seqs <= KUNSERVE_FIRST_BY_VALUE,
                "first places of %d rows on the host: %d at most", table->num_seqs,
                KUNSERVE_FIRST_BY_VALUE);
  KeepArgs a{};
  a.k = static_cast<f16*>(pool->k);
  a.v = static_cast<f16*>(pool->v);
  a.page_stride = pool->page_stride;
  a.layer_stride = pool->layer_stride;
  a.head_stride = pool->head_stride;
  a.token_stride = pool->token_stride;
  if (weights) {
    a.w = weights->w;
    a.w_page = weights->page_stride;
    a.w_layer = weights->layer_stride;
    a.w_head = weights->head_stride;
  }
  a.indptr = table->indptr_dev;
  a.indices = table->indices_dev;
  a.kv_len = table->kv_len_dev;
  a.kept = kept_dev;
  a.kept_stride = kept_stride;
  a.max_kept = max_kept;
  a.num_pages = int32_t(pool->num_pages);
  a.page_shift = __builtin_ctz(pool->page_size);
  a.num_layers = pool->num_layers;
  a.num_heads = pool->num_kv_heads;
  // A wave to a slab where two of its chunks hold the longest list: no barrier, and four slabs
  // to a workgroup. (8 layers of 8 heads of 128; 64 rows, all lists full: of 16 10 us against 19,
  // of 32 20 each, of 64 42 against 41; 4 rows: of 16 3.6 against 3.7, of 32 5.0 against 4.0, of
  // 64 8 against 5. Most lists are shorter than the longest.)
  const int chunk = kLoads * kWave / (pool->head_dim / 8);
  const bool small = max_kept <= chunk;
  a.num_slabs = (small ? 1 : 2) * int64_t(table->num_seqs) * pool->num_layers * pool->num_kv_heads;
  const int64_t blocks = small ? (a.num_slabs + kWaves - 1) / kWaves : a.num_slabs;
  KSV_CHECK_ARG(blocks < kMaxBlocks, "grid of %lld workgroups is too large",
                (long long)blocks);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (pool->head_dim) {
    case 64: keep_tokens<64>(grid, small, a, first_host, first_dev, table->num_seqs, s); break;
    case 128: keep_tokens<128>(grid, small, a, first_host, first_dev, table->num_seqs, s); break;
    default: keep_tokens<256>(grid, small, a, first_host, first_dev, table->num_seqs, s);
  }
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}

extern "C" int64_t kunserve_fork_moves(const int32_t* indptr_host, const int32_t* indices_host,
                                       const int32_t* kv_len_host, int32_t num_seqs,
                                       int32_t page_size, int64_t num_pages, int32_t* moves_host,
                                       int64_t capacity) {
  clear_error();
  KSV_CHECK_ARG(num_seqs >= 0 && page_size > 0 && num_pages >= 0 && num_pages < (int64_t(1) << 31),
                "bad num_seqs, page_size or num_pages");
  if (num_seqs == 0) return 0;
  KSV_CHECK_ARG(indptr_host && kv_len_host && indices_host && (moves_host || capacity == 0),
                "null table or moves");
  int64_t n = 0;
  const int rc = no_throw([&]() -> int {
    enum : uint8_t { kFree, kHeld, kTaken };
    std::vector<uint8_t> use(static_cast<size_t>(num_pages), kFree);
    auto pages = [&](int32_t b) { return indices_host + indptr_host[b]; };
    auto count = [&](int32_t b) { return (int64_t(kv_len_host[b]) + page_size - 1) / page_size; };
    for (int32_t b = 0; b < num_seqs; ++b) {
      KSV_CHECK_ARG(kv_len_host[b] >= 0, "row %d: %d tokens", b, kv_len_host[b]);
      for (int32_t list : {b, num_seqs + b}) {
        KSV_CHECK_ARG(indptr_host[list + 1] - int64_t(indptr_host[list]) >= count(b),
                      "row %d: %lld pages for %d tokens", b,
                      (long long)indptr_host[list + 1] - indptr_host[list], kv_len_host[b]);
        for (int64_t i = 0; i < count(b); ++i)
          KSV_CHECK_ARG(pages(list)[i] >= 0 && pages(list)[i] < num_pages,
                        "page id %d outside the pool [0, %lld)", pages(list)[i], (long long)num_pages);
      }
      for (int64_t i = 0; i < count(b); ++i) use[pages(b)[i]] = kHeld;   // (the kept ones too)
    }
    for (int32_t b = 0; b < num_seqs; ++b)
      for (int64_t i = 0; i < count(b); ++i) {
        const int32_t from = pages(b)[i], to = pages(num_seqs + b)[i];
        if (from == to) continue;
        KSV_CHECK_ARG(use[to] != kHeld, "page %d of pages_out holds tokens of the rows", to);
        KSV_CHECK_ARG(use[to] != kTaken, "page %d of pages_out is copied to twice", to);
        use[to] = kTaken;
        KSV_CHECK_ARG(n < capacity, "more than %lld moves", (long long)capacity);
        int32_t* m = moves_host + 3 * n++;
        m[0] = from;
        m[1] = to;
        m[2] = int32_t(std::min<int64_t>(page_size, kv_len_host[b] - i * page_size));
      }
    return KUNSERVE_OK;
  });
  return rc ? rc : n;
}

extern "C" int kunserve_copy_pages(const kunserve_kv_pool* pool, const kunserve_kv_weights* weights,
                                   const int32_t* moves_host, const int32_t* moves_dev, int64_t n,
                                   kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  if (weights) {
    rc = check_weights(weights, pool);
    if (rc) return rc;
  }
  KSV_CHECK_ARG(n >= 0 && n < (int64_t(1) << 31), "%lld moves", (long long)n);
  if (n == 0) return KUNSERVE_OK;
  KSV_CHECK_ARG(!moves_host != !moves_dev, "moves are either on the host or on the device");
  KSV_CHECK_ARG(!moves_host || n <= KUNSERVE_MOVES_BY_VALUE, "%lld moves on the host: %d at most",
                (long long)n, KUNSERVE_MOVES_BY_VALUE);
  KSV_CHECK_ARG(pool->num_layers < 32768 && pool->num_kv_heads < 65536,
                "%d layers of %d heads are too many", pool->num_layers, pool->num_kv_heads);
  CopyArgs a{};
  a.k = static_cast<f16*>(pool->k);
  a.v = static_cast<f16*>(pool->v);
  a.page_stride = pool->page_stride;
  a.layer_stride = pool->layer_stride;
  a.head_stride = pool->head_stride;
  a.token_stride = pool->token_stride;
  if (weights) {
    a.w = weights->w;
    a.w_page = weights->page_stride;
    a.w_layer = weights->layer_stride;
    a.w_head = weights->head_stride;
  }
  a.num_pages = int32_t(pool->num_pages);
  a.page_size = pool->page_size;
  a.num_heads = pool->num_kv_heads;
  // Heads of a workgroup: about 64 loads, two rounds of its waves.
  const int64_t per_head = (int64_t(pool->page_size) * (pool->head_dim / 8) + kWave - 1) / kWave;
  a.heads = int32_t(per_head >= 64 ? 1 : 64 / per_head);
  a.parts = (pool->num_kv_heads + a.heads - 1) / a.heads;
  const int64_t slabs = 2 * int64_t(pool->num_layers) * a.parts;   // workgroups of a move
  KSV_CHECK_ARG(slabs < kMaxBlocks, "moves of %lld workgroups", (long long)slabs);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  constexpr int64_t kMoves = 65535;   // of a launch
  for (int64_t from = 0; from < n; from += kMoves) {
    const dim3 grid(unsigned(slabs), unsigned(std::min(kMoves, n - from)));
    const int32_t* dev = moves_dev ? moves_dev + 3 * from : nullptr;
    switch (pool->head_dim) {
      case 64: copy_pages<64>(grid, a, moves_host, dev, s); break;
      case 128: copy_pages<128>(grid, a, moves_host, dev, s); break;
      default: copy_pages<256>(grid, a, moves_host, dev, s);
    }
  }
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}
