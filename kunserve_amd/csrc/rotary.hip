// Rotary embedding at positions of their own, fused with the K/V append
// (the prologue of LlamaOp.pforward's attention stage, kunserve/worker.py:
// 298-312; the append's slots kunserve/request.py:447-462).
//
// Token i of the step, at position p, has each rotated pair (a, b) of its q
// and k heads turned by the angle p * freq[j] (with axes, p its position on the
// pair's axis) and scaled:
//   a' = scale * (a cos - b sin),  b' = scale * (b cos + a sin).
// The first rotary_dim dims of a head are rotated, pair j being dims (j, j +
// rotary_dim / 2) or (2j, 2j + 1); the others pass. The angle is formed in 64
// bits: in 32 its product alone is off by up to p * freq * 2^-24, 0.06 rad at
// position 2^20. It is reduced to a fraction of a turn there, and sine and
// cosine are taken in 32 bits of a number that has 24 bits below half a turn.
// The rotation runs in fp32 with one rounding.
//
// HBM-bound: q read and written, k and v read and written once. One workgroup
// per token: its angles are evaluated once (rotary_dim / 2 of them, in 64 bits)
// and shared by its heads through LDS.
#include <cmath>

#include "common.hpp"

namespace kunserve {
namespace {

struct RotaryArgs {
  const f16* q;
  f16* q_out;
  const f16* k_new;
  const f16* v_new;
  int64_t q_tok, q_head, o_tok, o_head, k_tok, k_head, v_tok, v_head;
  f16* k;   // pool at the layer
  f16* v;
  int64_t page_stride, head_stride, token_stride;
  int32_t num_pages;
  int32_t page_shift;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* kv_len;
  const int32_t* q_indptr;
  const int32_t* positions;   // null, or [num_tokens]; with axes [num_axes][position_stride]
  const int32_t* axis;        // null, or [rotary_dim / 2]: the axis of each pair
  int32_t num_axes;
  int64_t position_stride;
  const double* freq;         // [rotary_dim / 2], radians per position
  float scale;
  int32_t num_seqs;
  int32_t num_qo_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t rotary_dim;
  int32_t interleave;
  int32_t copy_rest;          // q_out is not q: what is not rotated is copied
};

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;   // head_dim <= 256

template <typename T>
__global__ __launch_bounds__(kThreads) void rotary_append_kernel(RotaryArgs a) {
  typedef typename Vec<T>::v8 V8;
  __shared__ float s_cos[kMaxPairs], s_sin[kMaxPairs];
  const int tok = blockIdx.x;
  const int b = row_of_token(a.q_indptr, a.num_seqs, tok);
  if (b < 0) return;   // of no row: left as it is (uniform)
  const int kvl = a.kv_len[b];
  const int at = kvl - a.q_indptr[b + 1] + tok;   // the token's place in its row's cache
  if (at < 0 || at >= kvl) return;   // uniform
  const int pos = a.positions ? a.positions[tok] : at;
  const int half = a.rotary_dim / 2;
  for (int j = threadIdx.x; j < half; j += kThreads) {
    int at_axis = pos;
    if (a.axis) {
      const int x = a.axis[j];
      at_axis = a.positions[(x > 0 && x < a.num_axes ? x : 0) * a.position_stride + tok];
    }
    const double turns = double(at_axis) * a.freq[j] * 0.15915494309189535;   // 1 / 2 pi
    float s, c;
    sincospif(2.f * float(turns - rint(turns)), &s, &c);
    s_cos[j] = c * a.scale;
    s_sin[j] = s * a.scale;
  }
  __syncthreads();

  const int p = a.indices[a.indptr[b] + (at >> a.page_shift)];
  const bool page_ok = p >= 0 && p < a.num_pages;
  const int64_t dst = int64_t(page_ok ? p : 0) * a.page_stride +
                      int64_t(at & ((1 << a.page_shift) - 1)) * a.token_stride;
  // Units of 16 dims of a head: [0, rotary_dim / 16) are rotated (8 pairs),
  // the others pass.
  const int units = a.head_dim / 16, turned = a.rotary_dim / 16;
  const int n_units = (a.num_qo_heads + a.num_kv_heads) * units;
  for (int u = threadIdx.x; u < n_units; u += kThreads) {
    const int slot = u / units, c = u % units;
    const bool turn = c < turned;
    const int d0 = a.interleave || !turn ? 16 * c : 8 * c;
    const int d1 = a.interleave || !turn ? 16 * c + 8 : half + 8 * c;
    auto rotate = [&](V8& x0, V8& x1) {
      float w[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = float(x0[e]);
        w[8 + e] = float(x1[e]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int ia = a.interleave ? 2 * j : j, ib = a.interleave ? 2 * j + 1 : 8 + j;
        const float x = w[ia], y = w[ib], cs = s_cos[8 * c + j], sn = s_sin[8 * c + j];
        w[ia] = fmaf(x, cs, -y * sn);
        w[ib] = fmaf(y, cs, x * sn);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x0[e] = T(w[e]);
        x1[e] = T(w[8 + e]);
      }
    };
    if (slot < a.num_qo_heads) {
      if (!turn && !a.copy_rest) continue;
      const f16* qp = a.q + int64_t(tok) * a.q_tok + int64_t(slot) * a.q_head;
      f16* op = a.q_out + int64_t(tok) * a.o_tok + int64_t(slot) * a.o_head;
      V8 x0 = load_v8<T>(qp + d0), x1 = load_v8<T>(qp + d1);
      if (turn) rotate(x0, x1);
      *reinterpret_cast<V8*>(op + d0) = x0;
      *reinterpret_cast<V8*>(op + d1) = x1;
      continue;
    }
    if (!page_ok) continue;
    const int head = slot - a.num_qo_heads;
    const int64_t hd = dst + int64_t(head) * a.head_stride;
    const f16* kp = a.k_new + int64_t(tok) * a.k_tok + int64_t(head) * a.k_head;
    const f16* vp = a.v_new + int64_t(tok) * a.v_tok + int64_t(head) * a.v_head;
    V8 x0 = load_v8<T>(kp + d0), x1 = load_v8<T>(kp + d1);
    if (turn) rotate(x0, x1);
    *reinterpret_cast<V8*>(a.k + hd + d0) = x0;
    *reinterpret_cast<V8*>(a.k + hd + d1) = x1;
    store_f16x8(a.v + hd + d0, load_f16x8(vp + d0));
    store_f16x8(a.v + hd + d1, load_f16x8(vp + d1));
  }
}

}  // namespace
}  // namespace kunserve

using namespace kunserve;

extern "C" int kunserve_rotary_append_kv(const kunserve_kv_pool* pool, int32_t layer,
                                         const kunserve_page_table* table,
                                         const int32_t* q_indptr_dev, int32_t num_tokens,
                                         const kunserve_tensor3* q, kunserve_tensor3* q_out,
                                         int32_t num_qo_heads, const kunserve_tensor3* k_new,
                                         const kunserve_tensor3* v_new,
                                         const kunserve_rotary* rotary,
                                         const int32_t* positions_dev,
                                         kunserve_stream_t stream) {
  return kunserve_rotary_axes_append_kv(pool, layer, table, q_indptr_dev, num_tokens, q, q_out,
                                        num_qo_heads, k_new, v_new, rotary, nullptr,
                                        positions_dev, stream);
}

extern "C" int kunserve_rotary_axes_append_kv(const kunserve_kv_pool* pool, int32_t layer,
                                              const kunserve_page_table* table,
                                              const int32_t* q_indptr_dev, int32_t num_tokens,
                                              const kunserve_tensor3* q, kunserve_tensor3* q_out,
                                              int32_t num_qo_heads,
                                              const kunserve_tensor3* k_new,
                                              const kunserve_tensor3* v_new,
                                              const kunserve_rotary* rotary,
                                              const kunserve_rotary_axes* axes,
                                              const int32_t* positions_dev,
                                              kunserve_stream_t stream) {
  clear_error();
  int rc = check_pool(pool, true);
  if (rc) return rc;
  KSV_CHECK_ARG(table && q && q_out && k_new && v_new && rotary, "null argument");
  KSV_CHECK_ARG(layer >= 0 && layer < pool->num_layers, "layer %d outside [0, %d)", layer,
                pool->num_layers);
  KSV_CHECK_ARG(num_tokens >= 0 && table->num_seqs >= 0, "num_tokens or num_seqs < 0");
  KSV_CHECK_ARG(num_qo_heads > 0 && num_qo_heads % pool->num_kv_heads == 0,
                "num_qo_heads %d not a multiple of num_kv_heads %d", num_qo_heads,
                pool->num_kv_heads);
  KSV_CHECK_ARG(rotary->rotary_dim >= 16 && rotary->rotary_dim % 16 == 0 &&
                    rotary->rotary_dim <= pool->head_dim,
                "rotary_dim %d must be a multiple of 16 in [16, %d]", rotary->rotary_dim,
                pool->head_dim);
  KSV_CHECK_ARG(std::isfinite(rotary->scale), "rotary scale %g is not finite",
                double(rotary->scale));
  KSV_CHECK_ARG(!axes || (axes->num_axes > 0 && (axes->position_stride == 0 ||
                                                 axes->position_stride >= num_tokens)),
                "%d axes with positions %lld apart", axes ? axes->num_axes : 0,
                (long long)(axes ? axes->position_stride : 0));
  if (num_tokens == 0 || table->num_seqs == 0) return KUNSERVE_OK;
  KSV_CHECK_ARG(!axes || (axes->axis_dev && positions_dev), "axes need the pairs' and positions");
  KSV_CHECK_ARG(q_indptr_dev && table->indptr_dev && table->indices_dev && table->kv_len_dev &&
                    rotary->freq_dev,
                "null table array or frequencies");
  for (const kunserve_tensor3* t : {q, static_cast<const kunserve_tensor3*>(q_out), k_new, v_new})
    KSV_CHECK_ARG(t->data && aligned16(t->data) && t->token_stride % 8 == 0 &&
                      t->head_stride % 8 == 0,
                  "q / q_out / k_new / v_new must be 16-byte aligned with strides that are "
                  "multiples of 8");
  // A workgroup writes its token's q_out while others read theirs.
  const bool in_place = q_out->data == q->data && q_out->token_stride == q->token_stride &&
                        q_out->head_stride == q->head_stride;
  const int heads = pool->num_kv_heads, dim = pool->head_dim;
  const int64_t by_head = num_qo_heads > 1 ? q_out->head_stride : dim;
  const int64_t by_token = num_tokens > 1 ? q_out->token_stride : dim;
  KSV_CHECK_ARG(by_head >= dim && by_token >= dim &&
                    (num_qo_heads == 1 || num_tokens == 1 ||
                     by_token >= int64_t(num_qo_heads - 1) * by_head + dim ||
                     by_head >= int64_t(num_tokens - 1) * by_token + dim),
                "q_out's rows share memory");
  KSV_CHECK_ARG(in_place || !kunserve_tensors_overlap(q_out, num_qo_heads, q, num_qo_heads,
                                                      num_tokens, dim),
                "q_out overlaps q without being q");
  KSV_CHECK_ARG(!kunserve_tensors_overlap(q_out, num_qo_heads, k_new, heads, num_tokens, dim) &&
                    !kunserve_tensors_overlap(q_out, num_qo_heads, v_new, heads, num_tokens, dim),
                "q_out overlaps k_new or v_new");
  RotaryArgs a{};
  a.q = static_cast<const f16*>(q->data);
  a.q_out = static_cast<f16*>(q_out->data);
  a.k_new = static_cast<const f16*>(k_new->data);
  a.v_new = static_cast<const f16*>(v_new->data);
  a.q_tok = q->token_stride;
  a.q_head = q->head_stride;
  a.o_tok = q_out->token_stride;
  a.o_head = q_out->head_stride;
  a.k_tok = k_new->token_stride;
  a.k_head = k_new->head_stride;
  a.v_tok = v_new->token_stride;
  a.v_head = v_new->head_stride;
  a.k = static_cast<f16*>(pool->k) + int64_t(layer) * pool->layer_stride;
  a.v = static_cast<f16*>(pool->v) + int64_t(layer) * pool->layer_stride;
  a.page_stride = pool->page_stride;
  a.head_stride = pool->head_stride;
  a.token_stride = pool->token_stride;
  a.num_pages = int32_t(pool->num_pages);
  a.page_shift = __builtin_ctz(pool->page_size);
  a.indptr = table->indptr_dev;
  a.indices = table->indices_dev;
  a.kv_len = table->kv_len_dev;
  a.q_indptr = q_indptr_dev;
  a.positions = positions_dev;
  if (axes) {
    a.axis = axes->axis_dev;
    a.num_axes = axes->num_axes;
    a.position_stride = axes->position_stride;
  }
  a.freq = rotary->freq_dev;
  a.scale = rotary->scale;
  a.num_seqs = table->num_seqs;
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = heads;
  a.head_dim = dim;
  a.rotary_dim = rotary->rotary_dim;
  a.interleave = rotary->interleave != 0;
  a.copy_rest = !in_place;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (pool->dtype == KUNSERVE_DTYPE_BF16)
    rotary_append_kernel<bf16><<<dim3(unsigned(num_tokens)), kThreads, 0, s>>>(a);
  else
    rotary_append_kernel<f16><<<dim3(unsigned(num_tokens)), kThreads, 0, s>>>(a);
  KSV_CHECK_LAUNCH();
  return KUNSERVE_OK;
}
