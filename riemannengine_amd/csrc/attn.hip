// Attention over packed sequences: the entry points (riemann_hip.h). The
// passes are in attn_fwd.hip and attn_bwd.hip.
#include <climits>
#include <cmath>
#include <initializer_list>

#include "attn.hpp"

using namespace rhip;

namespace {

void check_attn_sizes(const rhip_attn *a) {
  RHIP_CHECK_ARG(a != nullptr, "descriptor is null");
  if (a->dtype != RHIP_F32 && a->dtype != RHIP_BF16)
    throw Error(RHIP_ERR_UNSUPPORTED, "dtype must be RHIP_F32 or RHIP_BF16");
  RHIP_CHECK_ARG(a->n_q >= 0 && a->n_k >= 0 && a->n_seq >= 0, "bad row or sequence count");
  if (a->n_q > INT32_MAX - 256 || a->n_k > INT32_MAX - 256)
    throw Error(RHIP_ERR_UNSUPPORTED, "row counts must stay below 2^31 - 256");
  RHIP_CHECK_ARG(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0,
                 "heads must be a positive multiple of kv_heads");
  if (a->n_q * (a->heads / a->kv_heads) > INT32_MAX - 256)
    throw Error(RHIP_ERR_UNSUPPORTED, "query rows of a group must stay below 2^31 - 256");
  RHIP_CHECK_ARG(a->dim >= 1, "head width must be positive");
  if (a->dim > kAttnMaxDim)
    throw Error(RHIP_ERR_UNSUPPORTED, "head width must not exceed 128");
  RHIP_CHECK_ARG(std::isfinite(a->scale) && a->scale > 0.f, "scale must be positive and finite");
}
void check_attn(const rhip_attn *a) {
  check_attn_sizes(a);
  RHIP_CHECK_ARG(a->n_seq == 0 || (a->q_offsets && a->k_offsets),
                 "sequence offsets are required");
}

AttnArgs make_args(const rhip_attn *a) {
  AttnArgs r{};
  r.q_off = a->q_offsets, r.k_off = a->k_offsets, r.k_len = a->k_lengths;
  r.q_row = a->q_row, r.q_head = a->q_head, r.k_row = a->k_row, r.k_head = a->k_head;
  r.v_row = a->v_row, r.v_head = a->v_head;
  r.n_q = static_cast<int32_t>(a->n_q), r.n_k = static_cast<int32_t>(a->n_k);
  r.n_seq = a->n_seq, r.heads = a->heads, r.kv_heads = a->kv_heads;
  r.group = a->heads / a->kv_heads;
  r.dim = a->dim, r.causal = a->causal;
  r.scale = a->scale, r.c = a->scale * kLog2e;
  return r;
}

// Whether every row starts 16-byte aligned and holds whole 16-byte chunks,
// and a tile's offsets fit the buffer loads.
bool vector_rows(const rhip_attn *a, std::initializer_list<const void *> ptrs,
                 std::initializer_list<int64_t> strides) {
  const int64_t e = a->dtype == RHIP_F32 ? 4 : 8;
  if (a->dim % e != 0)
    return false;
  for (const void *p : ptrs)
    if (p && !aligned16(p))
      return false;
  for (int64_t s : strides)
    if (s % e != 0 || s < 0 || s > (int64_t(1) << 22))
      return false;
  return true;
}

struct FwdWs {
  float *part_o, *part_ml;
};
FwdWs carve_forward(Carve &cv, const rhip_attn *a) {
  FwdWs w{};
  const int32_t splits = attn_forward_plan(*a).splits;
  if (splits > 1) {
    const size_t rows = static_cast<size_t>(splits) * a->n_q * a->heads;
    w.part_o = cv.take<float>(rows * a->dim);
    w.part_ml = cv.take<float>(rows * 2);
  }
  return w;
}

struct BwdWs {
  float2 *stat;
  float *part_k, *part_v;
};
BwdWs carve_backward(Carve &cv, const rhip_attn *a) {
  BwdWs w{};
  w.stat = cv.take<float2>(static_cast<size_t>(std::max<int64_t>(1, a->n_q)) * a->heads);
  const int32_t splits = attn_keys_plan(*a).splits;
  if (splits > 1) {
    const size_t n = static_cast<size_t>(splits) * a->n_k * a->kv_heads * a->dim;
    w.part_k = cv.take<float>(n);
    w.part_v = cv.take<float>(n);
  }
  return w;
}

} // namespace

extern "C" int rhip_attn_workspace_bytes(const rhip_attn *attn, int32_t backward,
                                         size_t *bytes) {
  return guarded([&] {
    check_attn(attn);
    RHIP_CHECK_ARG(bytes != nullptr, "bytes is null");
    Carve cv(nullptr, 0);
    if (backward)
      carve_backward(cv, attn);
    else
      carve_forward(cv, attn);
    *bytes = cv.used + 256;
  });
}

extern "C" int rhip_attn_plan(const rhip_attn *attn, int32_t pass, int32_t *blocks,
                              int32_t *splits) {
  return guarded([&] {
    check_attn_sizes(attn);
    RHIP_CHECK_ARG(blocks && splits, "blocks and splits are required");
    RHIP_CHECK_ARG(pass >= RHIP_ATTN_FORWARD && pass <= RHIP_ATTN_KEYS,
                   "pass must be one of RHIP_ATTN_");
    const AttnPlan p = pass == RHIP_ATTN_FORWARD   ? attn_forward_plan(*attn)
                       : pass == RHIP_ATTN_QUERIES ? attn_queries_plan(*attn)
                                                   : attn_keys_plan(*attn);
    *blocks = p.waves;
    *splits = p.splits;
  });
}

extern "C" int rhip_attn_forward(const rhip_attn *attn, const void *q, const void *k,
                                 const void *v, void *out, void *out_rest, float *lse,
                                 void *workspace, size_t ws_bytes, hipStream_t stream) {
  return guarded([&] {
    check_attn(attn);
    if (attn->n_q == 0)
      return;
    RHIP_CHECK_ARG(q && out, "q and out are required");
    RHIP_CHECK_ARG(attn->n_k == 0 || (k && v), "k and v are required");
    RHIP_CHECK_ARG(workspace != nullptr, "workspace is required");
    AttnArgs a = make_args(attn);
    Carve cv(workspace, ws_bytes);
    const FwdWs w = carve_forward(cv, attn);
    a.q = q, a.k = k, a.v = v, a.o = out, a.rest = out_rest, a.lse = lse;
    a.part_o = w.part_o, a.part_ml = w.part_ml;
    const bool vec = vector_rows(attn, {q, k, v, out, out_rest},
                                 {attn->q_row, attn->q_head, attn->k_row, attn->k_head,
                                  attn->v_row, attn->v_head});
    attn_forward_run(a, attn->dtype, vec, stream);
  });
}

extern "C" int rhip_attn_backward(const rhip_attn *attn, const void *grad_out,
                                  int64_t grad_out_row, int64_t grad_out_head, const void *q,
                                  const void *k, const void *v, const void *out,
                                  const void *out_rest, const float *lse, void *grad_q, void *grad_k, void *grad_v,
                                  void *workspace, size_t ws_bytes, hipStream_t stream) {
  return guarded([&] {
    check_attn(attn);
    if (attn->n_q == 0 && attn->n_k == 0)
      return;
    RHIP_CHECK_ARG(attn->n_q == 0 || (grad_out && q && out && lse),
                   "grad_out, q, out and lse are required");
    RHIP_CHECK_ARG(attn->n_k == 0 || (k && v), "k and v are required");
    RHIP_CHECK_ARG((grad_k == nullptr) == (grad_v == nullptr), "grad_k and grad_v go together");
    if (!grad_q && !grad_k)
      return;
    RHIP_CHECK_ARG(workspace != nullptr, "workspace is required");
    AttnArgs a = make_args(attn);
    Carve cv(workspace, ws_bytes);
    const BwdWs w = carve_backward(cv, attn);
    a.q = q, a.k = k, a.v = v, a.o = const_cast<void *>(out), a.lse = const_cast<float *>(lse);
    a.go = grad_out, a.go_row = grad_out_row, a.go_head = grad_out_head;
    a.rest = const_cast<void *>(out_rest);
    a.gq = grad_q, a.gk = grad_k, a.gv = grad_v;
    a.stat = w.stat, a.part_k = w.part_k, a.part_v = w.part_v;
    const bool vec = vector_rows(
        attn, {q, k, v, out, out_rest, grad_out, grad_q, grad_k, grad_v},
        {attn->q_row, attn->q_head, attn->k_row, attn->k_head, attn->v_row, attn->v_head,
         grad_out_row, grad_out_head});
    attn_backward_run(a, attn->dtype, vec, stream);
  });
}
