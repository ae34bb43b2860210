// PyTorch operator registration of the C ABI: torch.ops.kiv.*
//
// Every operator is a thin adapter: it builds the POD descriptors of
// include/kiv_b200.h from tensors (data pointers, shapes, strides, dtype) and
// calls the `extern "C"` entry point on the current CUDA stream of the
// store's device.  The C ABI stays the boundary; this file only makes it
// visible to the dispatcher, so the operators show up in traces, run under
// torch.cuda.graph capture like any other CUDA op, and have Meta kernels
// (shape-only, no work) for tracing with fake tensors.
//
// A store is passed as two lists:
//   store = [cold_k, cold_v, summaries, hot_k, hot_v, state, host_k, host_v, page_sums]
//           (hot_*, host_* and page_sums may be empty tensors: no hot ring,
//           no host tier, no replicated summaries)
//   geom  = [page_size, shard_rank, shard_count, hot_hint, stage_pages, flags]
// and a query as (q [B, Hq, Q, D], scaling, top_pages, top_p, softcap).
// The operators that write return nothing and declare what they mutate in
// their schema.  Failures raise RuntimeError with the library's message.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <vector>

#include "../../include/kiv_b200.h"

namespace {

using at::Tensor;

void *ptr_or_null(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

int32_t dtype_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KIV_DTYPE_F32;
    case at::kBFloat16: return KIV_DTYPE_BF16;
    case at::kHalf: return KIV_DTYPE_F16;
    default: TORCH_CHECK(false, "kiv: store dtype must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
  return -1;
}

kiv_store make_store(at::TensorList s, at::IntArrayRef g) {
  TORCH_CHECK(s.size() == 9, "kiv: store list must hold 9 tensors (cold_k, cold_v, summaries, hot_k, hot_v, "
                             "state, host_k, host_v, page_sums), got ", s.size());
  TORCH_CHECK(g.size() == 6, "kiv: geom must hold 6 ints (page_size, shard_rank, shard_count, hot_hint, "
                             "stage_pages, flags), got ", g.size());
  const Tensor &ck = s[0], &hk = s[3], &st = s[5], &hok = s[6];
  TORCH_CHECK(ck.dim() == 4, "kiv: cold_k must be [B, Hkv, slots, D]");
  TORCH_CHECK(st.scalar_type() == at::kLong && st.numel() >= KIV_STATE_WORDS, "kiv: state must be int64[32]");
  kiv_store d = {};
  d.batch = (int32_t)ck.size(0);
  d.num_kv_heads = (int32_t)ck.size(1);
  d.head_dim = (int32_t)ck.size(3);
  d.page_size = (int32_t)g[0];
  d.dtype = dtype_code(ck);
  d.shard_rank = (int32_t)g[1];
  d.shard_count = (int32_t)g[2];
  d.hot_hint = (int32_t)g[3];
  d.cold_capacity = ck.size(2);
  d.hot_capacity = hk.defined() && hk.numel() > 0 ? hk.size(2) : 0;
  d.cold_k = ptr_or_null(s[0]);
  d.cold_v = ptr_or_null(s[1]);
  d.summaries = ptr_or_null(s[2]);
  d.hot_k = ptr_or_null(s[3]);
  d.hot_v = ptr_or_null(s[4]);
  d.state = static_cast<int64_t *>(st.data_ptr());
  d.host_capacity = hok.defined() && hok.numel() > 0 ? hok.size(2) : 0;
  d.host_k = ptr_or_null(s[6]);
  d.host_v = ptr_or_null(s[7]);
  d.stage_pages = (int32_t)g[4];
  d.flags = (int32_t)g[5];
  d.page_sums = static_cast<float *>(ptr_or_null(s[8]));
  return d;
}

kiv_query make_query(const Tensor &q, double scaling, int64_t top_pages, int64_t top_p, double softcap) {
  TORCH_CHECK(q.dim() == 4 && q.stride(3) == 1, "kiv: query must be [B, Hq, Q, D] with a contiguous last dim");
  kiv_query d = {};
  d.q = q.data_ptr();
  d.stride_b = q.stride(0);
  d.stride_h = q.stride(1);
  d.stride_t = q.stride(2);
  d.num_query_heads = (int32_t)q.size(1);
  d.query_len = (int32_t)q.size(2);
  d.scaling = (float)scaling;
  d.softcap = (float)softcap;
  d.top_pages = (int32_t)top_pages;
  d.top_p = (int32_t)top_p;
  return d;
}

kiv_mask make_mask(const c10::optional<Tensor> &add, bool causal) {
  kiv_mask m = {};
  m.causal = causal ? 1 : 0;
  if (add.has_value() && add->defined()) {
    const Tensor &a = *add;
    TORCH_CHECK(a.scalar_type() == at::kFloat && a.dim() == 4 && a.stride(3) == 1,
                "kiv: mask must be float32 [B, 1|Hq, Q, hot] with a contiguous last dim");
    m.add = a.data_ptr<float>();
    m.stride_b = a.size(0) == 1 ? 0 : a.stride(0);
    m.stride_h = a.size(1) == 1 ? 0 : a.stride(1);
    m.stride_t = a.stride(2);
  }
  return m;
}

kiv_exchange make_exchange(const kiv_store &st, at::IntArrayRef arenas, int64_t arena_bytes, int64_t wait_cycles) {
  TORCH_CHECK((int64_t)arenas.size() == st.shard_count && st.shard_count <= KIV_MAX_PEERS,
              "kiv: one arena address per rank expected");
  kiv_exchange x = {};
  x.world = st.shard_count;
  x.rank = st.shard_rank;
  for (size_t i = 0; i < arenas.size(); ++i) x.arena[i] = reinterpret_cast<void *>(arenas[i]);
  x.arena_bytes = arena_bytes;
  x.wait_cycles = wait_cycles;
  return x;
}

void check(kiv_status rc, const char *what) {
  TORCH_CHECK(rc == KIV_OK, "kiv.", what, ": ", kiv_status_string(rc), " (", rc, "): ", kiv_last_error());
}

void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ------------------------------------------------------------- CUDA kernels
void state_reset(at::TensorList store, at::IntArrayRef geom) {
  const kiv_store st = make_store(store, geom);
  c10::cuda::CUDAGuard g(store[5].device());
  check(kiv_state_reset(&st, stream_of(store[5])), "state_reset");
}

void append_evict(at::TensorList store, at::IntArrayRef geom, const c10::optional<Tensor> &k_new,
                  const c10::optional<Tensor> &v_new, int64_t keep, int64_t n_evict_max) {
  const kiv_store st = make_store(store, geom);
  c10::cuda::CUDAGuard g(store[5].device());
  const void *kp = nullptr, *vp = nullptr;
  int64_t sb = 0, sh = 0, stt = 0;
  int32_t n_new = 0;
  if (k_new.has_value() && k_new->defined()) {
    const Tensor &k = *k_new, &v = *v_new;
    TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes(), "kiv: new K/V rows must both be [B, Hkv, n, D]");
    // one set of strides serves both (a dimension of size 1 is never stepped)
    for (int d = 0; d < 4; ++d)
      TORCH_CHECK(k.size(d) == 1 || k.stride(d) == v.stride(d), "kiv: new K and V rows need the same strides");
    TORCH_CHECK(k.scalar_type() == store[0].scalar_type(), "kiv: new rows must have the store dtype");
    kp = k.data_ptr();
    vp = v.data_ptr();
    sb = k.stride(0);
    sh = k.stride(1);
    stt = k.stride(2);
    n_new = (int32_t)k.size(2);
  }
  check(kiv_append_evict(&st, kp, vp, sb, sh, stt, n_new, keep, n_evict_max, stream_of(store[5])), "append_evict");
}

void coarse_select(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                   int64_t top_p, double softcap, const Tensor &ws, const c10::optional<Tensor> &row_scores,
                   const c10::optional<Tensor> &row_pages) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  float *rs = row_scores.has_value() && row_scores->defined() ? row_scores->data_ptr<float>() : nullptr;
  int32_t *rp = row_pages.has_value() && row_pages->defined() ? row_pages->data_ptr<int32_t>() : nullptr;
  check(kiv_coarse_select(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), rs, rp, stream_of(q)), "coarse_select");
}

void coarse_merge(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                  int64_t top_p, double softcap, const Tensor &ws, const Tensor &lists_scores,
                  const Tensor &lists_pages) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_coarse_merge(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), lists_scores.data_ptr<float>(),
                         lists_pages.data_ptr<int32_t>(), (int32_t)lists_scores.size(0), stream_of(q)),
        "coarse_merge");
}

void fine_score(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                int64_t top_p, double softcap, const Tensor &ws) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_fine_score(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), stream_of(q)), "fine_score");
}

void fine_topk(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
               int64_t top_p, double softcap, const Tensor &ws, const Tensor &sel,
               const c10::optional<Tensor> &sel_scores) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  float *ss = sel_scores.has_value() && sel_scores->defined() ? sel_scores->data_ptr<float>() : nullptr;
  check(kiv_fine_topk(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), sel.data_ptr<int32_t>(), ss, stream_of(q)),
        "fine_topk");
}

void fine_select(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                 int64_t top_p, double softcap, const Tensor &ws, const Tensor &sel,
                 const c10::optional<Tensor> &sel_scores) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  float *ss = sel_scores.has_value() && sel_scores->defined() ? sel_scores->data_ptr<float>() : nullptr;
  check(kiv_fine_select(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), sel.data_ptr<int32_t>(), ss, stream_of(q)),
        "fine_select");
}

void fine_merge(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                int64_t top_p, double softcap, const Tensor &ws, const Tensor &lists_scores,
                const Tensor &lists_tokens, const Tensor &sel, const Tensor &sel_local) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_fine_merge(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), lists_scores.data_ptr<float>(),
                       lists_tokens.data_ptr<int32_t>(), (int32_t)lists_scores.size(0), sel.data_ptr<int32_t>(),
                       sel_local.data_ptr<int32_t>(), stream_of(q)),
        "fine_merge");
}

void gather_rows(at::TensorList store, at::IntArrayRef geom, const Tensor &sel, int64_t P, const Tensor &out_k,
                 const Tensor &out_v) {
  const kiv_store st = make_store(store, geom);
  c10::cuda::CUDAGuard g(sel.device());
  check(kiv_gather_rows(&st, sel.data_ptr<int32_t>(), (int32_t)sel.size(1), (int32_t)P, ptr_or_null(out_k),
                        ptr_or_null(out_v), stream_of(sel)),
        "gather_rows");
}

void attend(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
            int64_t top_p, double softcap, const Tensor &ws, const Tensor &sel, const c10::optional<Tensor> &mask_add,
            bool causal, int64_t hot_slice, int64_t hot_slices, const c10::optional<Tensor> &out,
            const c10::optional<Tensor> &partial_out) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_mask md = make_mask(mask_add, causal);
  c10::cuda::CUDAGuard g(q.device());
  void *o = out.has_value() && out->defined() ? out->data_ptr() : nullptr;
  float *po = partial_out.has_value() && partial_out->defined() ? partial_out->data_ptr<float>() : nullptr;
  check(kiv_attend(&st, &qd, &md, ws.data_ptr(), (size_t)ws.nbytes(), sel.data_ptr<int32_t>(), (int32_t)sel.size(1),
                   (int32_t)hot_slice, (int32_t)hot_slices, o, po, stream_of(q)),
        "attend");
}

void attend_peers(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                  int64_t top_p, double softcap, const Tensor &ws, const Tensor &sel,
                  const c10::optional<Tensor> &mask_add, bool causal, at::IntArrayRef peer_k, at::IntArrayRef peer_v,
                  const Tensor &out) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_mask md = make_mask(mask_add, causal);
  TORCH_CHECK(peer_k.size() == (size_t)st.shard_count && peer_v.size() == (size_t)st.shard_count &&
                  st.shard_count <= KIV_MAX_PEERS,
              "kiv: attend_peers needs one cold_k and cold_v address per shard");
  kiv_peer_rows pr = {};
  for (int r = 0; r < st.shard_count; ++r) {
    pr.cold_k[r] = reinterpret_cast<const void *>(static_cast<uintptr_t>(peer_k[r]));
    pr.cold_v[r] = reinterpret_cast<const void *>(static_cast<uintptr_t>(peer_v[r]));
  }
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_attend_peers(&st, &qd, &md, ws.data_ptr(), (size_t)ws.nbytes(), sel.data_ptr<int32_t>(),
                         (int32_t)sel.size(1), &pr, out.data_ptr(), stream_of(q)),
        "attend_peers");
}

void attend_merge(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                  int64_t top_p, double softcap, const Tensor &partials, const Tensor &out) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_attend_merge(&st, &qd, partials.data_ptr<float>(), (int32_t)partials.size(0), out.data_ptr(),
                         stream_of(q)),
        "attend_merge");
}

void retrieve_attend(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling, int64_t top_pages,
                     int64_t top_p, double softcap, const Tensor &ws, int64_t reuse, const Tensor &sel,
                     const c10::optional<Tensor> &mask_add, bool causal, const Tensor &out) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_mask md = make_mask(mask_add, causal);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_retrieve_attend(&st, &qd, &md, ws.data_ptr(), (size_t)ws.nbytes(), (int32_t)reuse,
                            sel.data_ptr<int32_t>(), out.data_ptr(), stream_of(q)),
        "retrieve_attend");
}

void coarse_exchange_merge(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling,
                           int64_t top_pages, int64_t top_p, double softcap, const Tensor &ws,
                           const Tensor &row_scores, const Tensor &row_pages, at::IntArrayRef arenas,
                           int64_t arena_bytes, int64_t wait_cycles) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_exchange x = make_exchange(st, arenas, arena_bytes, wait_cycles);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_coarse_exchange_merge(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), row_scores.data_ptr<float>(),
                                  row_pages.data_ptr<int32_t>(), &x, stream_of(q)),
        "coarse_exchange_merge");
}

void fine_exchange_merge(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling,
                         int64_t top_pages, int64_t top_p, double softcap, const Tensor &ws, const Tensor &scores,
                         const Tensor &tokens, at::IntArrayRef arenas, int64_t arena_bytes, int64_t wait_cycles,
                         const c10::optional<Tensor> &sel, const Tensor &sel_local) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_exchange x = make_exchange(st, arenas, arena_bytes, wait_cycles);
  c10::cuda::CUDAGuard g(q.device());
  int32_t *s = sel.has_value() && sel->defined() ? sel->data_ptr<int32_t>() : nullptr;
  check(kiv_fine_exchange_merge(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), scores.data_ptr<float>(),
                                tokens.data_ptr<int32_t>(), &x, s, sel_local.data_ptr<int32_t>(), stream_of(q)),
        "fine_exchange_merge");
}

void fine_exchange_select(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling,
                          int64_t top_pages, int64_t top_p, double softcap, const Tensor &ws, at::IntArrayRef arenas,
                          int64_t arena_bytes, int64_t wait_cycles, const Tensor &sel,
                          const c10::optional<Tensor> &sel_local) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_exchange x = make_exchange(st, arenas, arena_bytes, wait_cycles);
  c10::cuda::CUDAGuard g(q.device());
  int32_t *sl = sel_local.has_value() && sel_local->defined() ? sel_local->data_ptr<int32_t>() : nullptr;
  check(kiv_fine_exchange_select(&st, &qd, ws.data_ptr(), (size_t)ws.nbytes(), &x, sel.data_ptr<int32_t>(), sl,
                                 stream_of(q)),
        "fine_exchange_select");
}

void attend_exchange_merge(at::TensorList store, at::IntArrayRef geom, const Tensor &q, double scaling,
                           int64_t top_pages, int64_t top_p, double softcap, const Tensor &partial,
                           at::IntArrayRef arenas, int64_t arena_bytes, int64_t wait_cycles, const Tensor &out) {
  const kiv_store st = make_store(store, geom);
  const kiv_query qd = make_query(q, scaling, top_pages, top_p, softcap);
  const kiv_exchange x = make_exchange(st, arenas, arena_bytes, wait_cycles);
  c10::cuda::CUDAGuard g(q.device());
  check(kiv_attend_exchange_merge(&st, &qd, partial.data_ptr<float>(), &x, out.data_ptr(), stream_of(q)),
        "attend_exchange_merge");
}

// ------------------------------------------------- rotation and paged cache
void check_same(const Tensor &a, const Tensor &t, const char *what) {
  TORCH_CHECK(t.device() == a.device(), "kiv: ", what, " is on ", t.device(), ", the rows are on ", a.device());
}

int64_t *error_word(const Tensor &a, const c10::optional<Tensor> &errors) {
  if (!errors.has_value() || !errors->defined()) return nullptr;
  check_same(a, *errors, "errors");
  TORCH_CHECK(errors->scalar_type() == at::kLong && errors->numel() >= 1, "kiv: errors must be an int64 tensor");
  return errors->data_ptr<int64_t>();
}

// stride of a dimension; one of size 1 is never stepped, whatever its stride says
int64_t step(const Tensor &t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }

const Tensor *given(const c10::optional<Tensor> &t) { return t.has_value() && t->defined() ? &*t : nullptr; }

// lead: dimensions of positions behind the axes ([batch, tokens] or [num_tokens])
kiv_turn make_turn(const Tensor &rows, int64_t head_dim, const c10::optional<Tensor> &cos, const c10::optional<Tensor> &sin,
                   const c10::optional<Tensor> &positions, const c10::optional<Tensor> &pair_axes, bool interleaved,
                   c10::optional<double> eps, const c10::optional<Tensor> &q_weight, const c10::optional<Tensor> &k_weight,
                   double weight_offset, at::IntArrayRef lead, bool rows_given) {
  kiv_turn t = {};
  t.axes = 1;
  TORCH_CHECK((given(cos) != nullptr) == (given(sin) != nullptr), "kiv: cos and sin come together");
  if (const Tensor *c = given(cos)) {
    const Tensor &s = *given(sin);
    check_same(rows, *c, "cos");
    check_same(rows, s, "sin");
    TORCH_CHECK(c->dim() == 2 && s.sizes() == c->sizes() && s.strides() == c->strides() && c->stride(1) == 1,
                "kiv: cos and sin must be [rows, rot_dim / 2] alike, with a contiguous last dim");
    TORCH_CHECK(s.scalar_type() == c->scalar_type(), "kiv: cos and sin must have one dtype");
    t.cos = c->data_ptr();
    t.sin = s.data_ptr();
    t.cs_stride = c->stride(0);
    t.cs_rows = c->size(0);
    t.cs_dtype = dtype_code(*c);
    t.rot_dim = (int32_t)std::min<int64_t>(2 * c->size(1), 1 << 20);
    if (const Tensor *p = given(positions)) {
      check_same(rows, *p, "positions");
      TORCH_CHECK(p->scalar_type() == at::kLong || p->scalar_type() == at::kInt, "kiv: positions must be int32 or int64");
      const int64_t nl = (int64_t)lead.size();
      TORCH_CHECK(p->dim() == nl || p->dim() == nl + 1, "kiv: positions must have ", nl, " dimensions, or an axis in front");
      const int64_t o = p->dim() - nl;
      for (int64_t i = 0; i < nl; ++i)
        TORCH_CHECK(p->size(o + i) == lead[i], "kiv: positions do not match the tokens");
      TORCH_CHECK(o == 0 || p->size(0) >= 1, "kiv: positions without an axis");
      t.positions = p->data_ptr();
      t.pos_is_i64 = p->scalar_type() == at::kLong;
      t.axes = o ? (int32_t)p->size(0) : 1;
      t.pos_stride_a = o ? p->stride(0) : 0;
      t.pos_stride_b = nl == 2 ? p->stride(o) : 0;
      t.pos_stride_t = p->stride(o + nl - 1);
    }
    if (const Tensor *x = given(pair_axes)) {
      check_same(rows, *x, "pair_axes");
      TORCH_CHECK(x->scalar_type() == at::kInt && x->dim() == 1 && x->is_contiguous() && x->size(0) == c->size(1),
                  "kiv: pair_axes must be int32 [rot_dim / 2]");
      t.pair_axes = x->data_ptr<int32_t>();
    }
    TORCH_CHECK(t.axes == 1 || t.pair_axes, "kiv: positions of several axes need pair_axes");
    TORCH_CHECK(t.positions || rows_given || t.cs_rows == lead[0] * lead[lead.size() - 1],
                "kiv: without positions, cos and sin need a row for each token");
  } else {
    TORCH_CHECK(!given(positions) && !given(pair_axes), "kiv: positions without cos and sin");
  }
  t.interleaved = interleaved;
  t.norm = eps.has_value();
  t.eps = (float)eps.value_or(0.0);
  t.weight_offset = (float)weight_offset;
  const Tensor *ws[2] = {given(q_weight), given(k_weight)};
  for (int i = 0; i < 2; ++i) {
    if (!ws[i]) continue;
    TORCH_CHECK(t.norm, "kiv: a norm weight without eps");
    check_same(rows, *ws[i], "norm weight");
    TORCH_CHECK(ws[i]->dim() == 1 && ws[i]->size(0) == head_dim && ws[i]->is_contiguous(), "kiv: norm weights must be [head_dim]");
    TORCH_CHECK(!(ws[0] && ws[1]) || ws[0]->scalar_type() == ws[1]->scalar_type(), "kiv: norm weights must have one dtype");
    (i == 0 ? t.q_weight : t.k_weight) = ws[i]->data_ptr();
    t.weight_dtype = dtype_code(*ws[i]);
  }
  return t;
}

// Rows as the kernels read them: last dim contiguous, 16-byte aligned -- the
// tensor itself, or a copy.
Tensor readable(const Tensor &x) {
  const int64_t n = x.dim(), eb = x.element_size();
  bool ok = n > 0 && x.numel() > 0 && x.stride(n - 1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int64_t d = 0; ok && d + 1 < n; ++d) ok = x.size(d) == 1 || (x.stride(d) * eb) % 16 == 0;
  return ok || x.numel() == 0 ? x : x.clone(at::MemoryFormat::Contiguous);   // a contiguous one may be misaligned too
}

kiv_rows make_rows(const Tensor &x, const char *what) {
  TORCH_CHECK(x.dim() == 4 && x.stride(3) == 1, "kiv: ", what, " must be [B, H, Q, D] with a contiguous last dim");
  return kiv_rows{x.data_ptr(), step(x, 0), step(x, 1), step(x, 2), (int32_t)x.size(1), 0};
}

void qk_norm_rope(const Tensor &q_in, const c10::optional<Tensor> &k_in, const c10::optional<Tensor> &cos,
                  const c10::optional<Tensor> &sin, const c10::optional<Tensor> &positions,
                  const c10::optional<Tensor> &pair_axes, bool interleaved, c10::optional<double> eps,
                  const c10::optional<Tensor> &q_weight, const c10::optional<Tensor> &k_weight, double weight_offset,
                  const Tensor &q_out, const c10::optional<Tensor> &k_out, const c10::optional<Tensor> &errors) {
  c10::cuda::CUDAGuard g(q_in.device());
  const Tensor q = readable(q_in);
  Tensor k;
  if (const Tensor *t = given(k_in)) k = readable(*t);
  const kiv_rows qr = make_rows(q, "q"), qo = make_rows(q_out, "q_out");
  check_same(q, q_out, "q_out");
  TORCH_CHECK(q_out.sizes() == q.sizes() && q_out.scalar_type() == q.scalar_type(), "kiv: q_out must be like q");
  const Tensor *kt = k.defined() ? &k : nullptr, *kot = given(k_out);
  TORCH_CHECK((kt != nullptr) == (kot != nullptr), "kiv: k and k_out come together");
  kiv_rows kr = {}, ko = {};
  if (kt) {
    check_same(q, *kt, "k");
    check_same(q, *kot, "k_out");
    kr = make_rows(*kt, "k");
    ko = make_rows(*kot, "k_out");
    TORCH_CHECK(kot->sizes() == kt->sizes() && kt->scalar_type() == q.scalar_type() && kot->scalar_type() == q.scalar_type() &&
                    kt->size(0) == q.size(0) && kt->size(2) == q.size(2) && kt->size(3) == q.size(3),
                "kiv: k must match q in batch, tokens, head_dim and dtype, and k_out must be like k");
  }
  const int64_t lead[2] = {q.size(0), q.size(2)};
  const kiv_turn t = make_turn(q, q.size(3), cos, sin, positions, pair_axes, interleaved, eps, q_weight, k_weight,
                               weight_offset, lead, false);
  TORCH_CHECK(q.size(0) * q.size(2) <= 0x7fffffff && q.size(3) <= (1 << 20), "kiv: too many tokens");
  check(kiv_qk_norm_rope(dtype_code(q), (int32_t)q.size(0), (int32_t)q.size(2), (int32_t)q.size(3), &qr, kt ? &kr : nullptr,
                         &qo, kt ? &ko : nullptr, &t, error_word(q, errors), stream_of(q)),
        "qk_norm_rope");
}

kiv_paged make_paged(const Tensor &rows, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table,
                     const Tensor &seq_lens, const Tensor &q_starts, int64_t max_query_len,
                     const c10::optional<Tensor> &errors) {
  for (const Tensor *t : {&k_pages, &v_pages, &table, &seq_lens, &q_starts}) check_same(rows, *t, "the paged cache");
  TORCH_CHECK(rows.dim() == 3 && rows.stride(2) == 1, "kiv: rows must be [tokens, heads, D] with a contiguous last dim");
  TORCH_CHECK(k_pages.dim() == 4 && k_pages.stride(3) == 1 && v_pages.stride(3) == 1 && v_pages.sizes() == k_pages.sizes(),
              "kiv: pages must both be [num_pages, Hkv, page_size, D] with a contiguous last dim");
  TORCH_CHECK(k_pages.scalar_type() == rows.scalar_type() && v_pages.scalar_type() == rows.scalar_type(),
              "kiv: rows and pages must have one dtype");
  TORCH_CHECK(k_pages.size(3) == rows.size(2), "kiv: rows and pages must have one head_dim");
  for (const Tensor *t : {&table, &seq_lens, &q_starts})
    TORCH_CHECK(t->scalar_type() == at::kInt, "kiv: block_table, seq_lens and q_starts must be int32");
  TORCH_CHECK(table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), "kiv: block_table must be [batch, width]");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.is_contiguous() && seq_lens.size(0) == table.size(0) && q_starts.dim() == 1 &&
                  q_starts.is_contiguous() && q_starts.size(0) == table.size(0) + 1,
              "kiv: seq_lens must be [batch] and q_starts [batch + 1]");
  TORCH_CHECK(k_pages.size(1) <= 65536 && k_pages.size(2) <= (1 << 20) && k_pages.size(3) <= (1 << 20) &&
                  table.size(0) <= (1 << 20) && max_query_len <= 0x7fffffff,
              "kiv: paged cache too large");
  kiv_paged p = {};
  p.batch = (int32_t)table.size(0);
  p.num_kv_heads = (int32_t)k_pages.size(1);
  p.head_dim = (int32_t)k_pages.size(3);
  p.page_size = (int32_t)k_pages.size(2);
  p.dtype = dtype_code(rows);
  p.max_query_len = (int32_t)max_query_len;
  p.num_pages = k_pages.size(0);
  p.k = ptr_or_null(k_pages);
  p.v = ptr_or_null(v_pages);
  p.k_stride_p = step(k_pages, 0);
  p.k_stride_h = step(k_pages, 1);
  p.k_stride_t = step(k_pages, 2);
  p.v_stride_p = step(v_pages, 0);
  p.v_stride_h = step(v_pages, 1);
  p.v_stride_t = step(v_pages, 2);
  p.block_table = static_cast<const int32_t *>(ptr_or_null(table));
  p.table_stride = step(table, 0);
  p.table_width = table.size(1);
  p.seq_lens = static_cast<const int32_t *>(ptr_or_null(seq_lens));
  p.q_starts = static_cast<const int32_t *>(ptr_or_null(q_starts));
  p.num_tokens = rows.size(0);
  p.errors = error_word(rows, errors);
  return p;
}

void paged_append(const Tensor &k_in, const Tensor &v_in, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table,
                  const Tensor &seq_lens, const Tensor &q_starts, const c10::optional<Tensor> &cos,
                  const c10::optional<Tensor> &sin, const c10::optional<Tensor> &positions,
                  const c10::optional<Tensor> &pair_axes, bool interleaved, c10::optional<double> eps,
                  const c10::optional<Tensor> &k_weight, double weight_offset, const c10::optional<Tensor> &errors) {
  c10::cuda::CUDAGuard g(k_in.device());
  check_same(k_in, v_in, "v");
  const Tensor k = readable(k_in), v = readable(v_in);
  const kiv_paged p = make_paged(k, k_pages, v_pages, table, seq_lens, q_starts, 0, errors);
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.stride(2) == 1 && k.size(1) == p.num_kv_heads,
              "kiv: new K/V rows must both be [tokens, Hkv, D]");
  const int64_t lead[1] = {k.size(0)};
  const kiv_turn t = make_turn(k, k.size(2), cos, sin, positions, pair_axes, interleaved, eps, c10::nullopt, k_weight,
                               weight_offset, lead, true);
  check(kiv_paged_append(&p, k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1), &t, stream_of(k)),
        "paged_append");
}

void paged_attend(const Tensor &q_in, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &seq_lens,
                  const Tensor &q_starts, double scaling, bool causal, int64_t window, double softcap, int64_t max_query_len,
                  const Tensor &out, const c10::optional<Tensor> &lse, const c10::optional<Tensor> &errors) {
  c10::cuda::CUDAGuard g(q_in.device());
  const Tensor q = readable(q_in);
  const kiv_paged p = make_paged(q, k_pages, v_pages, table, seq_lens, q_starts, max_query_len, errors);
  check_same(q, out, "out");
  TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1, "kiv: out must be like q");
  TORCH_CHECK(window >= 0 && window <= 0x7fffffff, "kiv: bad window");
  kiv_paged_query d = {};
  d.q = q.data_ptr();
  d.stride_t = step(q, 0);
  d.stride_h = step(q, 1);
  d.out = out.data_ptr();
  d.out_stride_t = step(out, 0);
  d.out_stride_h = step(out, 1);
  if (const Tensor *l = given(lse)) {
    check_same(q, *l, "lse");
    TORCH_CHECK(l->scalar_type() == at::kFloat && l->dim() == 2 && l->size(0) == q.size(0) && l->size(1) == q.size(1) && l->is_contiguous(),
                "kiv: lse must be a contiguous float32 [tokens, Hq]");
    d.lse = l->data_ptr<float>();
  }
  d.num_query_heads = (int32_t)q.size(1);
  d.causal = causal;
  d.window = (int32_t)window;
  d.scaling = (float)scaling;
  d.softcap = (float)softcap;
  // scratch of this call alone, from the allocator of the stream (or graph) it runs in
  const size_t bytes = kiv_paged_workspace_bytes(&p, &d);
  Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(kiv_paged_attend(&p, &d, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)), "paged_attend");
}

// ------------------------------------------------------------ shape queries
// Workspace size and sub-buffer offsets: pure arithmetic on shapes (the data
// pointers are stand-ins), so the same kernel serves real and fake tensors.
std::vector<int64_t> workspace_layout(at::TensorList store, at::IntArrayRef geom, const Tensor &q,
                                      int64_t top_pages, int64_t top_p) {
  TORCH_CHECK(store.size() == 9 && geom.size() == 6, "kiv: bad store descriptor lists");
  const Tensor &ck = store[0], &hk = store[3], &hok = store[6];
  TORCH_CHECK(ck.dim() == 4 && q.dim() == 4, "kiv: bad store or query rank");
  char *fake = reinterpret_cast<char *>(uintptr_t(1) << 20);
  kiv_store st = {};
  st.batch = (int32_t)ck.size(0);
  st.num_kv_heads = (int32_t)ck.size(1);
  st.head_dim = (int32_t)ck.size(3);
  st.page_size = (int32_t)geom[0];
  st.dtype = dtype_code(ck);
  st.shard_rank = (int32_t)geom[1];
  st.shard_count = (int32_t)geom[2];
  st.hot_hint = (int32_t)geom[3];
  st.cold_capacity = ck.size(2);
  st.hot_capacity = hk.numel() > 0 ? hk.size(2) : 0;
  st.cold_k = st.cold_v = st.summaries = fake;
  st.hot_k = st.hot_v = st.hot_capacity > 0 ? fake : nullptr;
  st.state = reinterpret_cast<int64_t *>(fake);
  st.host_capacity = hok.numel() > 0 ? hok.size(2) : 0;
  st.host_k = st.host_v = st.host_capacity > 0 ? fake : nullptr;
  st.stage_pages = (int32_t)geom[4];
  st.flags = (int32_t)geom[5];
  st.page_sums = store[8].numel() > 0 ? reinterpret_cast<float *>(fake) : nullptr;
  kiv_query qd = {};
  qd.q = fake;
  // strides of a contiguous query (only their 16-byte alignment is checked)
  qd.stride_t = q.size(3);
  qd.stride_h = q.size(2) * q.size(3);
  qd.stride_b = q.size(1) * qd.stride_h;
  qd.num_query_heads = (int32_t)q.size(1);
  qd.query_len = (int32_t)q.size(2);
  qd.scaling = 1.f;
  qd.top_pages = (int32_t)top_pages;
  qd.top_p = (int32_t)top_p;
  std::vector<int64_t> out(11, 0);
  check(kiv_workspace_layout(&st, &qd, out.data()), "workspace_layout");
  out[10] = (int64_t)kiv_workspace_bytes(&st, &qd);
  return out;
}

// ------------------------------------------------------------- Meta kernels
// Shape-only: the writes go to caller-provided tensors, so tracing with fake
// tensors has nothing to compute.
void state_reset_meta(at::TensorList, at::IntArrayRef) {}
void append_evict_meta(at::TensorList, at::IntArrayRef, const c10::optional<Tensor> &, const c10::optional<Tensor> &,
                       int64_t, int64_t) {}
void coarse_select_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                        const Tensor &, const c10::optional<Tensor> &, const c10::optional<Tensor> &) {}
void coarse_merge_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                       const Tensor &, const Tensor &, const Tensor &) {}
void fine_score_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                     const Tensor &) {}
void fine_topk_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                    const Tensor &, const Tensor &, const c10::optional<Tensor> &) {}
void fine_select_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                      const Tensor &, const Tensor &, const c10::optional<Tensor> &) {}
void fine_merge_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                     const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &) {}
void gather_rows_meta(at::TensorList, at::IntArrayRef, const Tensor &, int64_t, const Tensor &, const Tensor &) {}
void attend_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double, const Tensor &,
                 const Tensor &, const c10::optional<Tensor> &, bool, int64_t, int64_t, const c10::optional<Tensor> &,
                 const c10::optional<Tensor> &) {}
void attend_merge_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                       const Tensor &, const Tensor &) {}
void retrieve_attend_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                          const Tensor &, int64_t, const Tensor &, const c10::optional<Tensor> &, bool,
                          const Tensor &) {}
void coarse_exchange_merge_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                                const Tensor &, const Tensor &, const Tensor &, at::IntArrayRef, int64_t, int64_t) {}
void fine_exchange_merge_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                              const Tensor &, const Tensor &, const Tensor &, at::IntArrayRef, int64_t, int64_t,
                              const c10::optional<Tensor> &, const Tensor &) {}
void fine_exchange_select_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                               const Tensor &, at::IntArrayRef, int64_t, int64_t, const Tensor &,
                               const c10::optional<Tensor> &) {}
void attend_peers_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                       const Tensor &, const Tensor &, const c10::optional<Tensor> &, bool, at::IntArrayRef,
                       at::IntArrayRef, const Tensor &) {}
void attend_exchange_merge_meta(at::TensorList, at::IntArrayRef, const Tensor &, double, int64_t, int64_t, double,
                                const Tensor &, at::IntArrayRef, int64_t, int64_t, const Tensor &) {}
void qk_norm_rope_meta(const Tensor &, const c10::optional<Tensor> &, const c10::optional<Tensor> &,
                       const c10::optional<Tensor> &, const c10::optional<Tensor> &, const c10::optional<Tensor> &, bool,
                       c10::optional<double>, const c10::optional<Tensor> &, const c10::optional<Tensor> &, double,
                       const Tensor &, const c10::optional<Tensor> &, const c10::optional<Tensor> &) {}
void paged_append_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                       const Tensor &, const c10::optional<Tensor> &, const c10::optional<Tensor> &,
                       const c10::optional<Tensor> &, const c10::optional<Tensor> &, bool, c10::optional<double>,
                       const c10::optional<Tensor> &, double, const c10::optional<Tensor> &) {}
void paged_attend_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                       double, bool, int64_t, double, int64_t, const Tensor &, const c10::optional<Tensor> &,
                       const c10::optional<Tensor> &) {}

}  // namespace

#define KIV_Q "Tensor q, float scaling, int top_pages, int top_p, float softcap"

TORCH_LIBRARY(kiv, m) {
  // Replaces: kiv/cold_store.py:142-184 (evict_from_hot), kiv/tiered_cache.py:55-72, :107-142
  m.def("state_reset(Tensor(a!)[] store, int[] geom) -> ()");
  m.def("append_evict(Tensor(a!)[] store, int[] geom, Tensor? k_new, Tensor? v_new, int keep, "
        "int n_evict_max) -> ()");
  m.def("workspace_layout(Tensor[] store, int[] geom, Tensor q, int top_pages, int top_p) -> int[]");
  // Replaces: kiv/cold_store.py:203-230 (coarse scoring, per-row top-k, union)
  m.def("coarse_select(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor(c!)? row_scores, "
        "Tensor(d!)? row_pages) -> ()");
  m.def("coarse_merge(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor lists_scores, "
        "Tensor lists_pages) -> ()");
  // Replaces: kiv/cold_store.py:227-262 (candidates), :301, :332-347 (fine scores, max, top-P)
  m.def("fine_score(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws) -> ()");
  m.def("fine_topk(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor(c!) sel, "
        "Tensor(d!)? sel_scores) -> ()");
  m.def("fine_select(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor(c!) sel, "
        "Tensor(d!)? sel_scores) -> ()");
  m.def("fine_merge(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor lists_scores, "
        "Tensor lists_tokens, Tensor(c!) sel, Tensor(d!) sel_local) -> ()");
  // Replaces: kiv/cold_store.py:357-362 (gather of the selected K/V rows)
  m.def("gather_rows(Tensor[] store, int[] geom, Tensor sel, int P, Tensor(b!) out_k, Tensor(c!) out_v) -> ()");
  // Replaces: kiv/middleware.py:330-352 and kiv/mask_utils.py:8-38 (attention over [cold ; hot])
  m.def("attend(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor sel, Tensor? mask_add, "
        "bool causal, int hot_slice, int hot_slices, Tensor(c!)? out, Tensor(d!)? partial_out) -> ()");
  m.def("attend_merge(Tensor[] store, int[] geom, " KIV_Q ", Tensor partials, Tensor(b!) out) -> ()");
  // Replaces: kiv/cold_store.py:283-371 + kiv/middleware.py:308-354 (one call)
  m.def("retrieve_attend(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, int reuse, Tensor(c!) sel, "
        "Tensor? mask_add, bool causal, Tensor(d!) out) -> ()");
  // Sharded layer-step exchanges (no reference counterpart: it has no multi-GPU code)
  m.def("coarse_exchange_merge(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor row_scores, "
        "Tensor row_pages, int[] arenas, int arena_bytes, int wait_cycles) -> ()");
  m.def("fine_exchange_merge(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor scores, "
        "Tensor tokens, int[] arenas, int arena_bytes, int wait_cycles, Tensor(c!)? sel, Tensor(d!) sel_local) -> ()");
  m.def("attend_exchange_merge(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor partial, int[] arenas, "
        "int arena_bytes, int wait_cycles, Tensor(b!) out) -> ()");
  // Replaces, for page-sharded stores: kiv/cold_store.py:283-371 steps 2-3 (fine pass over the whole union)
  m.def("fine_exchange_select(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, int[] arenas, "
        "int arena_bytes, int wait_cycles, Tensor(c!) sel, Tensor(d!)? sel_local) -> ()");
  // Replaces, for page-sharded stores: kiv/middleware.py:330-352, kiv/mask_utils.py:8-38 (rows read from
  // every shard's cold tier; peer addresses as int[])
  m.def("attend_peers(Tensor(a!)[] store, int[] geom, " KIV_Q ", Tensor(b!) ws, Tensor sel, Tensor? mask_add, "
        "bool causal, int[] peer_k, int[] peer_v, Tensor(c!) out) -> ()");
  // Rotation and paged cache (no reference counterpart: its caches are dense)
  m.def("qk_norm_rope(Tensor q, Tensor? k, Tensor? cos, Tensor? sin, Tensor? positions, Tensor? pair_axes, "
        "bool interleaved, float? eps, Tensor? q_weight, Tensor? k_weight, float weight_offset, Tensor(a!) q_out, "
        "Tensor(b!)? k_out, Tensor(c!)? errors) -> ()");
  m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor block_table, Tensor seq_lens, "
        "Tensor q_starts, Tensor? cos, Tensor? sin, Tensor? positions, Tensor? pair_axes, bool interleaved, float? eps, "
        "Tensor? k_weight, float weight_offset, Tensor(c!)? errors) -> ()");
  m.def("paged_attend(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor seq_lens, Tensor q_starts, "
        "float scaling, bool causal, int window, float softcap, int max_query_len, Tensor(a!) out, Tensor(b!)? lse, "
        "Tensor(c!)? errors) -> ()");
}

TORCH_LIBRARY_IMPL(kiv, CUDA, m) {
  m.impl("state_reset", &state_reset);
  m.impl("append_evict", &append_evict);
  m.impl("coarse_select", &coarse_select);
  m.impl("coarse_merge", &coarse_merge);
  m.impl("fine_score", &fine_score);
  m.impl("fine_topk", &fine_topk);
  m.impl("fine_select", &fine_select);
  m.impl("fine_merge", &fine_merge);
  m.impl("gather_rows", &gather_rows);
  m.impl("attend", &attend);
  m.impl("attend_merge", &attend_merge);
  m.impl("retrieve_attend", &retrieve_attend);
  m.impl("coarse_exchange_merge", &coarse_exchange_merge);
  m.impl("fine_exchange_merge", &fine_exchange_merge);
  m.impl("attend_exchange_merge", &attend_exchange_merge);
  m.impl("fine_exchange_select", &fine_exchange_select);
  m.impl("attend_peers", &attend_peers);
  m.impl("paged_attend", &paged_attend);
  m.impl("paged_append", &paged_append);
  m.impl("qk_norm_rope", &qk_norm_rope);
}

TORCH_LIBRARY_IMPL(kiv, Meta, m) {
  m.impl("state_reset", &state_reset_meta);
  m.impl("append_evict", &append_evict_meta);
  m.impl("coarse_select", &coarse_select_meta);
  m.impl("coarse_merge", &coarse_merge_meta);
  m.impl("fine_score", &fine_score_meta);
  m.impl("fine_topk", &fine_topk_meta);
  m.impl("fine_select", &fine_select_meta);
  m.impl("fine_merge", &fine_merge_meta);
  m.impl("gather_rows", &gather_rows_meta);
  m.impl("attend", &attend_meta);
  m.impl("attend_merge", &attend_merge_meta);
  m.impl("retrieve_attend", &retrieve_attend_meta);
  m.impl("coarse_exchange_merge", &coarse_exchange_merge_meta);
  m.impl("fine_exchange_merge", &fine_exchange_merge_meta);
  m.impl("attend_exchange_merge", &attend_exchange_merge_meta);
  m.impl("fine_exchange_select", &fine_exchange_select_meta);
  m.impl("attend_peers", &attend_peers_meta);
  m.impl("paged_attend", &paged_attend_meta);
  m.impl("paged_append", &paged_append_meta);
  m.impl("qk_norm_rope", &qk_norm_rope_meta);
}

TORCH_LIBRARY_IMPL(kiv, CompositeExplicitAutograd, m) { m.impl("workspace_layout", &workspace_layout); }
