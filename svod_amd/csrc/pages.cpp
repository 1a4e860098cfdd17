// The op layer of a key/value cache in pages (svodk_pages), which has no counterpart in the reference: the same contract as
// ops.cpp, an op launches a kernel, or names why the caller's graph must run, or rejects its arguments.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>

#include "../../include/svodk.h"
#include "kernels.h"
#include "op_layer.h"

using namespace svodk::op;

namespace {

// A descriptor of a pool or its scales, whose types no other operand has.
bool pool_formed(const svodk_tensor *t) {
  if (t == nullptr || (t->dtype != SVODK_E4M3 && t->dtype != SVODK_E8M0)) return well_formed(t);
  svodk_tensor bytes = *t;
  bytes.dtype = SVODK_BOOL;
  return well_formed(&bytes);
}
size_t pool_bytes(const svodk_tensor *t) {
  return (size_t)numel(t) * (t->dtype == SVODK_E4M3 || t->dtype == SVODK_E8M0 ? 1 : dtype_bytes(t->dtype));
}

// The pages' descriptors checked and laid into `a`; `rows`: of the packed operands (with `starts` only).  0, a refusal, or a
// fallback that the caller answers when its own operands are checked.
int take_pages(const char *op, const svodk_pages *pages, bool starts, int64_t rows, svodk::PagesArgs &a, int &why) {
  why = 0;
  if (pages == nullptr || !pool_formed(pages->k) || !pool_formed(pages->v) || !well_formed(pages->table) ||
      !well_formed(pages->lens) || (starts && !well_formed(pages->starts)) ||
      (pages->k_scale != nullptr && !pool_formed(pages->k_scale)) || (pages->v_scale != nullptr && !pool_formed(pages->v_scale)))
    return fail(SVODK_ERR_ARGUMENT, "%s: a null or malformed tensor descriptor of the pages", op);
  const svodk_tensor *k = pages->k, *v = pages->v, *table = pages->table, *lens = pages->lens;
  if (k->rank != 4)
    return fail(SVODK_ERR_SHAPE, "%s: the key pool has shape %s, expected [pages, kv_heads, page, D]", op, fmt_shape(k).c_str());
  if (!same_shape(k, v))
    return fail(SVODK_ERR_SHAPE, "%s: the value pool has shape %s, expected %s", op, fmt_shape(v).c_str(), fmt_shape(k).c_str());
  if (k->dtype != v->dtype)
    return fail(SVODK_ERR_DTYPE, "%s: the value pool is %s, the key pool is %s", op, dtype_name(v->dtype), dtype_name(k->dtype));
  const bool coded = k->dtype == SVODK_E4M3;
  if (coded != (pages->k_scale != nullptr) || coded != (pages->v_scale != nullptr))
    return fail(SVODK_ERR_ARGUMENT, "%s: scales belong to pools of 8 bits, both of them", op);
  const svodk_tensor *scales[2] = {pages->k_scale, pages->v_scale};
  for (const svodk_tensor *x : scales) {
    if (x == nullptr) continue;
    if (!(x->rank == 3 && x->shape[0] == k->shape[0] && x->shape[1] == k->shape[1] && x->shape[2] == k->shape[2]))
      return fail(SVODK_ERR_SHAPE, "%s: scales have shape %s, expected [%lld, %lld, %lld]", op, fmt_shape(x).c_str(),
                  (long long)k->shape[0], (long long)k->shape[1], (long long)k->shape[2]);
    if (x->dtype != SVODK_E8M0) return fail(SVODK_ERR_DTYPE, "%s: scales are %s, expected Float8E8M0", op, dtype_name(x->dtype));
  }
  if (table->rank != 2)
    return fail(SVODK_ERR_SHAPE, "%s: the table has shape %s, expected [B, columns]", op, fmt_shape(table).c_str());
  if (table->dtype != SVODK_I32) return fail(SVODK_ERR_DTYPE, "%s: the table is %s, expected Int32", op, dtype_name(table->dtype));
  if (!(lens->rank == 1 && lens->shape[0] == table->shape[0]))
    return fail(SVODK_ERR_SHAPE, "%s: lens has shape %s, expected [%lld]", op, fmt_shape(lens).c_str(), (long long)table->shape[0]);
  if (!is_int(lens->dtype)) return fail(SVODK_ERR_DTYPE, "%s: lens is %s, expected an integer type", op, dtype_name(lens->dtype));
  if (starts) {
    const svodk_tensor *st = pages->starts;
    if (!(st->rank == 1 && st->shape[0] == table->shape[0] + 1))
      return fail(SVODK_ERR_SHAPE, "%s: starts has shape %s, expected [%lld]", op, fmt_shape(st).c_str(),
                  (long long)table->shape[0] + 1);
    if (!is_int(st->dtype)) return fail(SVODK_ERR_DTYPE, "%s: starts is %s, expected an integer type", op, dtype_name(st->dtype));
  }
  const int64_t page = k->shape[2], columns = table->shape[1];
  if (!coded && k->dtype != SVODK_BF16 && k->dtype != SVODK_F16)
    why = SVODK_GRAPH_DTYPE;
  else if (!svodk::pages_support(k->shape[3]) || page < svodk::kLeastPage || page > svodk::kMostPage || (page & (page - 1)) != 0)
    why = SVODK_GRAPH_SHAPE;
  else if (k->shape[0] == 0 || k->shape[1] == 0 || columns == 0 || table->shape[0] == 0 || rows == 0)
    why = SVODK_GRAPH_SHAPE;
  // Positions, sequences and rows are counted in 31 bits, a page's bytes in 32.
  else if (k->shape[0] > 0x7fffffff || k->shape[1] > 0xffff || columns > 0x3fffffff / page || table->shape[0] > 0xffffff || rows > 0x3fffffff)
    why = SVODK_GRAPH_SHAPE;
  if (why != 0) return 0;
  a.k = k->data, a.v = v->data;
  a.k_scale = coded ? pages->k_scale->data : nullptr, a.v_scale = coded ? pages->v_scale->data : nullptr;
  a.table = (const int32_t *)table->data, a.lens = lens->data;
  a.starts = starts ? pages->starts->data : nullptr;
  a.batch = (int32_t)table->shape[0], a.columns = (int32_t)columns, a.pages = (int32_t)k->shape[0];
  a.kv_heads = (int32_t)k->shape[1], a.d = (int32_t)k->shape[3], a.page_log2 = __builtin_ctzll((uint64_t)page);
  a.rows = (int32_t)rows;
  a.lens_i64 = lens->dtype == SVODK_I64, a.starts_i64 = starts && pages->starts->dtype == SVODK_I64;
  return 0;
}

// The addresses of a call's pages and of its operands beside them: none null, none off its alignment, nothing that is written
// shared.  `pools_written`: by the call.
int pages_addresses(const char *op, const svodk_pages *pages, bool starts, bool pools_written, const Span *operands, int n) {
  Span spans[12] = {{"key pool", pages->k->data, pool_bytes(pages->k), pools_written},
                    {"value pool", pages->v->data, pool_bytes(pages->v), pools_written},
                    {"table", pages->table->data, (size_t)numel(pages->table) * 4, false},
                    {"lens", pages->lens->data, (size_t)numel(pages->lens) * dtype_bytes(pages->lens->dtype), false}};
  size_t align[12] = {16, 16, 4, dtype_bytes(pages->lens->dtype)};
  int m = 4;
  if (starts) {
    align[m] = dtype_bytes(pages->starts->dtype);
    spans[m++] = {"starts", pages->starts->data, (size_t)numel(pages->starts) * dtype_bytes(pages->starts->dtype), false};
  }
  if (pages->k_scale != nullptr) {
    align[m] = 1;
    spans[m++] = {"key scales", pages->k_scale->data, pool_bytes(pages->k_scale), pools_written};
    align[m] = 1;
    spans[m++] = {"value scales", pages->v_scale->data, pool_bytes(pages->v_scale), pools_written};
  }
  for (int i = 0; i < n; i++) align[m] = 16, spans[m++] = operands[i];
  for (int i = 0; i < m; i++) {
    if (spans[i].data == nullptr) return fail(SVODK_ERR_ARGUMENT, "%s: a null device pointer", op);
    if (((uintptr_t)spans[i].data & (align[i] - 1)) != 0)
      return fail(SVODK_ERR_ARGUMENT, "%s: %s is not %zu-byte aligned", op, spans[i].name, align[i]);
  }
  return check_aliasing(op, spans, m);
}

// The 16-bit operands' type beside the pools'.
int pages_types(const char *op, const svodk_pages *pages, int32_t dtype, int &why) {
  if (why != 0) return 0;
  if (dtype != SVODK_BF16 && dtype != SVODK_F16)
    why = SVODK_GRAPH_DTYPE;
  else if (pages->k->dtype != SVODK_E4M3 && pages->k->dtype != dtype)
    return fail(SVODK_ERR_DTYPE, "%s: the pools are %s, the operands %s", op, dtype_name(pages->k->dtype), dtype_name(dtype));
  return 0;
}

// What both entry points of the attention over pages read off its operands: 0 and `a` filled in but for its addresses' checks and the
// workspace, a refusal, or `why` the graph runs.
int take_paged(const svodk_tensor *q, const svodk_pages *pages, const svodk_attn *opts, svodk::PagedArgs &a, int &why) {
  const char *op = "attention_paged";
  if (!well_formed(q) || opts == nullptr) return fail(SVODK_ERR_ARGUMENT, "%s: a null or malformed tensor descriptor", op);
  if (int rc = take_pages(op, pages, true, q->rank == 3 ? q->shape[0] : 0, a.pages, why)) return rc;
  const int64_t kv_heads = pages->k->shape[1], d = pages->k->shape[3];
  if (!(q->rank == 3 && q->shape[2] == d))
    return fail(SVODK_ERR_SHAPE, "%s: q has shape %s, expected [N, heads, %lld]", op, fmt_shape(q).c_str(), (long long)d);
  const int64_t heads = q->shape[1];
  if (kv_heads > 0 && (heads == 0 || heads % kv_heads != 0))
    return fail(SVODK_ERR_HEADS, "%s: %lld query heads over %lld key/value heads", op, (long long)heads, (long long)kv_heads);
  if (int rc = pages_types(op, pages, q->dtype, why)) return rc;
  if (opts->has_window && (opts->window_left < 0 || opts->window_right < 0))
    return fail(SVODK_ERR_ARGUMENT, "%s: a negative window reach", op);
  if (why != 0) return 0;
  if (opts->key_kind != SVODK_KEYS_NONE || opts->has_chunk || opts->seg_start != nullptr || opts->cache != nullptr ||
      opts->bias != nullptr || opts->batch_live > 0 || opts->row_order != nullptr)
    why = SVODK_GRAPH_CONFIG;
  // The merge counts (row, head)s in 31 bits.
  else if (heads / kv_heads > svodk::kMostPagedGroup || heads > 0xffff || q->shape[0] * heads > 0x7fffffff)
    why = SVODK_GRAPH_SHAPE;
  if (why != 0) return 0;
  a.q = q->data;
  a.heads = (int32_t)heads;
  a.causal = opts->causal != 0;
  a.win_left = -1;
  const int64_t far = (int64_t)a.pages.columns << a.pages.page_log2;  // a reach past which nothing is hidden
  if (opts->has_window) {
    a.win_left = (int32_t)std::min<int64_t>(opts->window_left, far);
    a.win_right = (int32_t)std::min<int64_t>(opts->window_right, far);
  }
  a.scale = opts->has_scale ? opts->scale : 1.0f / std::sqrt((float)d);
  a.pages.f16 = q->dtype == SVODK_F16;
  const int64_t blocks = (far + 63) / 64;
  a.splits = opts->splits <= 0 ? 0 : (int32_t)std::min<int64_t>(opts->splits, blocks);
  if (svodk::paged_slots(a) == 0) a.splits = 1;
  // A launch's threads are counted in 32 bits, 256 a workgroup.
  if (svodk::paged_workgroups(a) > 0xffffff) why = SVODK_GRAPH_SHAPE;
  // And the bytes of the states of a named count of splits in 32.
  if (a.splits > 1 && svodk::paged_workspace(a) > 0x7fffffff) why = SVODK_GRAPH_CONFIG;
  return 0;
}

}  // namespace

extern "C" {

int svodk_write_pages(const svodk_tensor *k, const svodk_tensor *v, const svodk_pages *pages, void *hip_stream) {
  const char *op = "write_pages";
  if (!well_formed(k) || !well_formed(v)) return fail(SVODK_ERR_ARGUMENT, "%s: a null or malformed tensor descriptor", op);
  svodk::PagesArgs a{};
  int why;
  if (int rc = take_pages(op, pages, true, k->rank == 3 ? k->shape[0] : 0, a, why)) return rc;
  if (!(k->rank == 3 && k->shape[1] == pages->k->shape[1] && k->shape[2] == pages->k->shape[3]))
    return fail(SVODK_ERR_SHAPE, "%s: k has shape %s, expected [N, %lld, %lld]", op, fmt_shape(k).c_str(),
                (long long)pages->k->shape[1], (long long)pages->k->shape[3]);
  if (!same_shape(k, v))
    return fail(SVODK_ERR_SHAPE, "%s: v has shape %s, expected %s", op, fmt_shape(v).c_str(), fmt_shape(k).c_str());
  if (k->dtype != v->dtype) return fail(SVODK_ERR_DTYPE, "%s: v is %s, k is %s", op, dtype_name(v->dtype), dtype_name(k->dtype));
  if (int rc = pages_types(op, pages, k->dtype, why)) return rc;
  const OnDeviceOf on(hip_stream);
  if (!current_device_has_kernels()) return ran_graph(op, SVODK_GRAPH_TARGET);
  if (why != 0) return ran_graph(op, why);
  const Span operands[2] = {{"k", k->data, (size_t)numel(k) * 2, false}, {"v", v->data, (size_t)numel(v) * 2, false}};
  if (int rc = pages_addresses(op, pages, true, true, operands, 2)) return rc;
  a.f16 = k->dtype == SVODK_F16;
  ran(op, op, pages->k->dtype == SVODK_E4M3 ? "e4m3" : "16 bits");
  const hipError_t e = svodk::launch_write_pages(a, k->data, v->data, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(SVODK_ERR_LAUNCH, "%s: %s", op, hipGetErrorString(e));
  return SVODK_KERNEL;
}

int svodk_read_pages(const svodk_pages *pages, const svodk_tensor *k, const svodk_tensor *v, void *hip_stream) {
  const char *op = "read_pages";
  if (!well_formed(k) || !well_formed(v)) return fail(SVODK_ERR_ARGUMENT, "%s: a null or malformed tensor descriptor", op);
  svodk::PagesArgs a{};
  int why;
  if (int rc = take_pages(op, pages, false, k->rank == 4 ? k->shape[1] : 0, a, why)) return rc;
  if (!(k->rank == 4 && k->shape[0] == pages->table->shape[0] && k->shape[2] == pages->k->shape[1] && k->shape[3] == pages->k->shape[3]))
    return fail(SVODK_ERR_SHAPE, "%s: k has shape %s, expected [%lld, T, %lld, %lld]", op, fmt_shape(k).c_str(),
                (long long)pages->table->shape[0], (long long)pages->k->shape[1], (long long)pages->k->shape[3]);
  if (!same_shape(k, v))
    return fail(SVODK_ERR_SHAPE, "%s: v has shape %s, expected %s", op, fmt_shape(v).c_str(), fmt_shape(k).c_str());
  if (k->dtype != v->dtype) return fail(SVODK_ERR_DTYPE, "%s: v is %s, k is %s", op, dtype_name(v->dtype), dtype_name(k->dtype));
  if (int rc = pages_types(op, pages, k->dtype, why)) return rc;
  const OnDeviceOf on(hip_stream);
  if (!current_device_has_kernels()) return ran_graph(op, SVODK_GRAPH_TARGET);
  if (why != 0) return ran_graph(op, why);
  const Span operands[2] = {{"k", k->data, (size_t)numel(k) * 2, true}, {"v", v->data, (size_t)numel(v) * 2, true}};
  if (int rc = pages_addresses(op, pages, false, false, operands, 2)) return rc;
  a.f16 = k->dtype == SVODK_F16;
  ran(op, op, pages->k->dtype == SVODK_E4M3 ? "e4m3" : "16 bits");
  const hipError_t e = svodk::launch_read_pages(a, (int32_t)k->shape[1], k->data, v->data, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(SVODK_ERR_LAUNCH, "%s: %s", op, hipGetErrorString(e));
  return SVODK_KERNEL;
}

int svodk_attention_paged(const svodk_tensor *q, const svodk_pages *pages, const svodk_attn *opts, const svodk_tensor *out,
                          void *hip_stream) {
  const char *op = "attention_paged";
  if (!well_formed(out)) return fail(SVODK_ERR_ARGUMENT, "%s: a null or malformed tensor descriptor", op);
  svodk::PagedArgs a{};
  int why;
  if (int rc = take_paged(q, pages, opts, a, why)) return rc;
  if (!same_shape(out, q))
    return fail(SVODK_ERR_SHAPE, "%s: out has shape %s, expected %s", op, fmt_shape(out).c_str(), fmt_shape(q).c_str());
  if (out->dtype != q->dtype)
    return fail(SVODK_ERR_DTYPE, "%s: out is %s, the input is %s", op, dtype_name(out->dtype), dtype_name(q->dtype));
  const OnDeviceOf on(hip_stream);
  if (!current_device_has_kernels()) return ran_graph(op, SVODK_GRAPH_TARGET);
  if (why != 0) return ran_graph(op, why);
  Span operands[3] = {{"q", q->data, (size_t)numel(q) * 2, false}, {"out", out->data, (size_t)numel(out) * 2, true}};
  int n = 2;
  if (a.splits != 1) {
    // Splits that the caller named need their workspace; the device's own are dropped without it.
    const int64_t need = svodk::paged_workspace(a);
    const bool lent = opts->workspace != nullptr && opts->workspace_bytes >= need;
    if (!lent && a.splits > 1) return ran_graph(op, SVODK_GRAPH_CONFIG);
    if (!lent) {
      a.splits = 1;
    } else {
      a.workspace = (float *)opts->workspace;
      operands[n++] = {"workspace", opts->workspace, (size_t)need, true};
    }
  }
  if (int rc = pages_addresses(op, pages, true, false, operands, n)) return rc;
  a.o = out->data;
  ran(op, "flash_attention", svodk::paged_config(a));
  const hipError_t e = svodk::launch_paged(a, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(SVODK_ERR_LAUNCH, "%s: %s", op, hipGetErrorString(e));
  return SVODK_KERNEL;
}

int64_t svodk_attention_paged_workspace(const svodk_tensor *q, const svodk_pages *pages, const svodk_attn *opts) {
  svodk::PagedArgs a{};
  int why;
  if (take_paged(q, pages, opts, a, why) != 0 || why != 0 || a.splits == 1) return 0;
  return svodk::paged_workspace(a);
}

}  // extern "C"
