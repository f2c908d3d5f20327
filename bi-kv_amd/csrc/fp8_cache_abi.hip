// C ABI of the 8-bit cache: the handle, argument checks, launches. Declarations: include/bikv_pagecopy.h.
#include "../../include/bikv_pagecopy.h"
#include "fp8_cache_kernels.h"
#include "pagecopy_internal.h"

#include <new>
#include <vector>

using namespace bikv;

struct bikv_fp8_cache {
  int device;
  int n_layers, heads, head_dim, page_tokens;
  int64_t n_pages, page_stride, token_stride, scale_stride;
  std::vector<char*> plane, scale;      // 2 * layer + (0 = K, 1 = V)
};

extern "C" int bikv_fp8_cache_create(const bikv_fp8_cache_desc* d, bikv_fp8_cache** out) {
  if (!d || !out) return fail(BIKV_EINVAL, "null argument");
  *out = nullptr;
  if (d->n_layers <= 0 || d->n_layers > 32768) return fail(BIKV_EINVAL, "n_layers %d out of range", d->n_layers);
  if (d->kv_heads <= 0 || d->kv_heads > 1024) return fail(BIKV_EINVAL, "kv_heads must be in [1, 1024], got %d", d->kv_heads);
  if (d->head_dim != 64 && d->head_dim != 128) return fail(BIKV_EINVAL, "head_dim must be 64 or 128, got %d", d->head_dim);
  if (d->page_tokens <= 0 || d->page_tokens > 65536) return fail(BIKV_EINVAL, "page_tokens must be in [1, 65536], got %d", d->page_tokens);
  if (d->n_pages <= 0) return fail(BIKV_EINVAL, "n_pages must be positive");
  const int64_t row = (int64_t)d->kv_heads * d->head_dim;
  if (d->token_stride_bytes < row || d->token_stride_bytes % 16 != 0 || d->token_stride_bytes >= (int64_t(1) << 31))
    return fail(BIKV_EINVAL, "token_stride_bytes must be a multiple of 16 from kv_heads*head_dim on, below 2 GiB (got %lld)", (long long)d->token_stride_bytes);
  if (d->page_stride_bytes < (d->page_tokens - 1) * d->token_stride_bytes + row || d->page_stride_bytes % 16 != 0)
    return fail(BIKV_EINVAL, "page_stride_bytes must be a multiple of 16 that holds page_tokens rows (got %lld)", (long long)d->page_stride_bytes);
  if (d->scale_page_stride_bytes < 4 * (int64_t)d->kv_heads || d->scale_page_stride_bytes % 4 != 0)
    return fail(BIKV_EINVAL, "scale_page_stride_bytes must be a multiple of 4 that holds kv_heads floats (got %lld)", (long long)d->scale_page_stride_bytes);
  if (!d->plane_base || !d->scale_plane_base) return fail(BIKV_EINVAL, "plane_base and scale_plane_base must be given");
  if (d->n_pages > (int64_t(1) << 62) / d->page_stride_bytes || d->n_pages > (int64_t(1) << 62) / d->scale_page_stride_bytes)
    return fail(BIKV_EINVAL, "n_pages %lld is more than an address range holds", (long long)d->n_pages);
  for (int q = 0; q < 2 * d->n_layers; ++q) {
    if (!d->plane_base[q] || (uintptr_t)d->plane_base[q] % 16 != 0) return fail(BIKV_EINVAL, "plane_base[%d] must be 16-byte aligned and not null", q);
    if (!d->scale_plane_base[q] || (uintptr_t)d->scale_plane_base[q] % 4 != 0) return fail(BIKV_EINVAL, "scale_plane_base[%d] must be 4-byte aligned and not null", q);
  }
  uint32_t* st = nullptr;
  const int rc = device_status(d->device, ST_BANK_SHARED, &st);
  if (rc) return rc;
  try {
    bikv_fp8_cache* c = new bikv_fp8_cache();
    *out = c;
    c->device = d->device;
    c->n_layers = d->n_layers;
    c->heads = d->kv_heads;
    c->head_dim = d->head_dim;
    c->page_tokens = d->page_tokens;
    c->n_pages = d->n_pages;
    c->page_stride = d->page_stride_bytes;
    c->token_stride = d->token_stride_bytes;
    c->scale_stride = d->scale_page_stride_bytes;
    c->plane.resize(2 * (size_t)d->n_layers);
    c->scale.resize(2 * (size_t)d->n_layers);
    for (int q = 0; q < 2 * d->n_layers; ++q) {
      c->plane[q] = static_cast<char*>(const_cast<void*>(d->plane_base[q]));
      c->scale[q] = static_cast<char*>(const_cast<void*>(d->scale_plane_base[q]));
    }
  } catch (const std::bad_alloc&) {
    delete *out;
    *out = nullptr;
    return fail(BIKV_ESYS, "out of host memory");
  }
  return BIKV_OK;
}

extern "C" int bikv_fp8_cache_destroy(bikv_fp8_cache* c) {
  delete c;
  return BIKV_OK;
}

namespace bikv {

static int check_batch(const bikv_fp8_cache* c, int32_t layer, const bikv_seq_batch* b, SeqArgs* seq, LayerArgs* l) {
  if (!c || !b) return fail(BIKV_EINVAL, "null cache or batch");
  if (layer < 0 || layer >= c->n_layers) return fail(BIKV_EINVAL, "layer %d outside [0, %d)", layer, c->n_layers);
  if (b->n_seqs < 0 || b->n_rows < 0 || b->max_pages < 0) return fail(BIKV_EINVAL, "negative n_seqs, n_rows or max_pages");
  if (b->dtype != BIKV_T_BF16 && b->dtype != BIKV_T_FP16) return fail(BIKV_EINVAL, "dtype must be BIKV_T_BF16 or BIKV_T_FP16, got %d", b->dtype);
  if (b->n_seqs == 0) return BIKV_OK;
  if (!b->kv_lens || (b->max_pages > 0 && !b->page_table)) return fail(BIKV_EINVAL, "page_table and kv_lens must be given");
  if (!b->q_starts && b->n_rows != b->n_seqs)
    return fail(BIKV_EINVAL, "without q_starts every sequence has one row: n_rows %lld, n_seqs %lld", (long long)b->n_rows, (long long)b->n_seqs);
  if (b->page_table_stride < b->max_pages) return fail(BIKV_EINVAL, "page_table_stride %lld is less than max_pages %lld", (long long)b->page_table_stride, (long long)b->max_pages);
  if (b->n_seqs >= (int64_t(1) << 24) || b->n_rows >= (int64_t(1) << 30)) return fail(BIKV_ERANGE, "more than 2^24 sequences or 2^30 rows");
  if (b->max_pages > (int64_t(1) << 30) / c->page_tokens)
    return fail(BIKV_ERANGE, "max_pages * page_tokens must not be more than 2^30 (got %lld * %d)", (long long)b->max_pages, c->page_tokens);
  seq->table = b->page_table;
  seq->table_stride = b->page_table_stride;
  seq->kv_lens = b->kv_lens;
  seq->q_starts = b->q_starts;
  seq->n_seqs = b->n_seqs;
  seq->n_rows = b->n_rows;
  seq->max_len = b->max_pages * c->page_tokens;
  l->k = c->plane[2 * (size_t)layer];
  l->v = c->plane[2 * (size_t)layer + 1];
  l->ks = c->scale[2 * (size_t)layer];
  l->vs = c->scale[2 * (size_t)layer + 1];
  l->n_pages = c->n_pages;
  l->page_stride = c->page_stride;
  l->token_stride = c->token_stride;
  l->scale_stride = c->scale_stride;
  l->page_tokens = fast_div((uint32_t)c->page_tokens);
  l->heads = c->heads;
  return BIKV_OK;
}

static int check_rows(const char* what, const void* p, int64_t row, int64_t head) {
  if (!p) return fail(BIKV_EINVAL, "%s is null", what);
  if ((uintptr_t)p % 16 != 0 || row % 8 != 0 || head % 8 != 0 || row < 0 || head < 0)
    return fail(BIKV_EINVAL, "%s: address and strides must be multiples of 16 bytes (8 elements) and not negative (strides %lld, %lld)", what, (long long)row, (long long)head);
  return BIKV_OK;
}

}  // namespace bikv

extern "C" int bikv_fp8_append(const bikv_fp8_cache* c, int32_t layer, const bikv_seq_batch* b, const void* k, int64_t k_row_stride,
                               int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, void* stream) {
  AppendArgs a = {};
  int rc = check_batch(c, layer, b, &a.seq, &a.layer);
  if (rc) return rc;
  if (b->n_seqs == 0 || b->n_rows == 0) return BIKV_OK;
  rc = check_rows("k", k, k_row_stride, k_head_stride);
  if (!rc) rc = check_rows("v", v, v_row_stride, v_head_stride);
  if (rc) return rc;
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.units = append_units(!b->q_starts, b->n_seqs, b->n_rows, c->page_tokens);
  if (!launch_fits(append_groups(a.units, c->heads), kAppendThreads)) return fail(BIKV_ERANGE, "too many pages times heads for one call");
  rc = device_status(c->device, ST_BANK_SHARED, &a.status);
  if (rc) return rc;
  BIKV_DEVICE(c->device);
  const hipError_t e = launch_fp8_append(c->head_dim, b->dtype, a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail_hip(e, "append launch");
  return BIKV_OK;
}

namespace bikv {

static int plan_call(const bikv_fp8_cache* c, const bikv_seq_batch* b, int32_t q_heads, AttendPlan* plan) {
  if (!c || !b) return fail(BIKV_EINVAL, "null cache or batch");
  if (q_heads <= 0 || q_heads % c->heads != 0) return fail(BIKV_EINVAL, "q_heads %d must be a positive multiple of kv_heads %d", q_heads, c->heads);
  if (b->n_seqs < 0 || b->n_rows < 0 || b->max_pages < 0) return fail(BIKV_EINVAL, "negative n_seqs, n_rows or max_pages");
  if (b->n_seqs >= (int64_t(1) << 24) || b->n_rows >= (int64_t(1) << 30) || b->n_rows * (q_heads / c->heads) >= (int64_t(1) << 31) ||
      b->max_pages > (int64_t(1) << 30) / c->page_tokens)
    return fail(BIKV_ERANGE, "too many sequences, rows or pages for one call");
  *plan = AttendPlan();
  if (b->n_seqs == 0 || b->n_rows == 0) return BIKV_OK;
  *plan = plan_fp8_attend(c->heads, q_heads / c->heads, !b->q_starts, b->n_seqs, b->n_rows, b->max_pages * c->page_tokens);
  if (!launch_fits(plan->groups, plan->threads))       // the joins' launches are smaller
    return fail(BIKV_ERANGE, "too many rows times heads for one call");
  return BIKV_OK;
}

// Parts' results, their (m, l), and the slots' words on joining them; part_rows is even, so the last are 8-byte aligned.
static int64_t workspace_bytes_of(const bikv_fp8_cache* c, const AttendPlan& p) {
  if (p.part_rows == 0) return 0;
  return p.part_rows * (c->head_dim + 2) * 4 + (p.form == ATTEND_MANY ? 0 : p.slots * (int64_t)sizeof(JoinHead));
}

}  // namespace bikv

extern "C" int64_t bikv_fp8_attend_workspace(const bikv_fp8_cache* c, const bikv_seq_batch* b, int32_t q_heads) {
  AttendPlan p;
  const int rc = plan_call(c, b, q_heads, &p);
  if (rc) return rc;
  return workspace_bytes_of(c, p);
}

extern "C" int bikv_fp8_attend(const bikv_fp8_cache* c, int32_t layer, const bikv_seq_batch* b, const void* q, int64_t q_row_stride,
                               int64_t q_head_stride, int32_t q_heads, int32_t causal, float softmax_scale, void* out,
                               int64_t out_row_stride, int64_t out_head_stride, float* lse, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  AttendArgs a = {};
  int rc = check_batch(c, layer, b, &a.seq, &a.layer);
  if (rc) return rc;
  AttendPlan p;
  rc = plan_call(c, b, q_heads, &p);
  if (rc) return rc;
  if (b->n_seqs == 0 || b->n_rows == 0) return BIKV_OK;
  rc = check_rows("q", q, q_row_stride, q_head_stride);
  if (!rc) rc = check_rows("out", out, out_row_stride, out_head_stride);
  if (rc) return rc;
  if ((uintptr_t)lse % 4 != 0) return fail(BIKV_EINVAL, "lse must be 4-byte aligned");
  const int64_t need = workspace_bytes_of(c, p);
  if (need > 0 && (!workspace || (uintptr_t)workspace % 16 != 0 || workspace_bytes < need))
    return fail(BIKV_EINVAL, "workspace must be 16-byte aligned and hold %lld bytes (got %lld)", (long long)need, (long long)workspace_bytes);
  if (!(softmax_scale == softmax_scale) || softmax_scale - softmax_scale != 0.f) return fail(BIKV_EINVAL, "softmax_scale must be finite");
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.o_row = out_row_stride;
  a.o_head = out_head_stride;
  a.group = fast_div((uint32_t)(q_heads / c->heads));
  a.causal = causal ? 1 : 0;
  a.scale_log2 = softmax_scale * 1.44269504088896340736f;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + p.part_rows * c->head_dim;
  a.part_join = reinterpret_cast<JoinHead*>(a.part_ml + 2 * p.part_rows);
  rc = device_status(c->device, ST_BANK_SHARED, &a.status);
  if (rc) return rc;
  BIKV_DEVICE(c->device);
  const hipError_t e = launch_fp8_attend(p, c->head_dim, b->dtype, a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail_hip(e, "attend launch");
  return BIKV_OK;
}
