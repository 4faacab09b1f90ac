// C ABI of the 8-bit key/value cache (include/ar_attn.h): argument checks and dispatch to the kernels in kv_cache_write.cu,
// kv_cache_attn.cu and kv_cache_attn_tc.cu.  What the page table, the lengths and the starts hold is checked by the kernels: it lies in device memory.
#include "../../include/ar_attn.h"
#include "ar_kernels.h"

namespace {

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

int check_pool(const ar_kv_pool* p, ar::KvPool* out) {
  if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) return AR_ERR_NULL;
  if (p->pages <= 0 || p->Hkv <= 0) return AR_ERR_SHAPE;
  if ((p->D != 64 && p->D != 128) || (p->format != AR_KV_INT8 && p->format != AR_KV_E4M3)) return AR_ERR_UNSUPPORTED;
  int log2 = 4;
  while (log2 < 8 && (1 << log2) != p->page) log2++;
  if (log2 == 8 || p->pages > INT32_MAX || p->Hkv > 65535) return AR_ERR_UNSUPPORTED;
  if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->k_scale, 4) || !aligned(p->v_scale, 4) || !aligned(p->k_mean, 16))
    return AR_ERR_ALIGNMENT;
  *out = ar::KvPool{(uint8_t*)p->k, (uint8_t*)p->v, p->k_scale, p->v_scale, p->k_mean, (int)p->pages, (int)p->Hkv, (int)p->D, log2,
                    p->format == AR_KV_E4M3};
  return AR_OK;
}
int check_batch(const ar_kv_batch* s, const ar::KvPool& pool, ar::KvBatch* out) {
  if (!s || !s->page_table || !s->lengths) return AR_ERR_NULL;
  if (s->B <= 0 || s->T < 0 || s->table_pages <= 0 || s->table_stride < 0 || (!s->starts && s->T != s->B)) return AR_ERR_SHAPE;
  if (s->B > 1 && s->table_stride < s->table_pages) return AR_ERR_SHAPE;
  // token positions, rows and grids are 32-bit numbers
  if (s->B > (1 << 24) || s->T > (1 << 28) || s->table_pages > (INT32_MAX >> pool.page_log2)) return AR_ERR_UNSUPPORTED;
  if (!aligned(s->page_table, 4) || !aligned(s->lengths, 4) || !aligned(s->starts, 4)) return AR_ERR_ALIGNMENT;
  *out = ar::KvBatch{s->page_table, s->lengths, s->starts, s->table_stride, (int)s->table_pages, (int)s->B, (int)s->T, nullptr};
  return AR_OK;
}
// A packed [T, H, D] tensor that is read (or, `written`, whose rows must not lie on one another).  The stride of an extent of
// one is not used and may be anything.
int check_rows(const void* p, const int64_t* strides, int64_t T, int64_t H, int dtype, bool written, ar::KvRows* out) {
  if (!p || !strides) return AR_ERR_NULL;
  const int64_t size = dtype == AR_DTYPE_F32 ? 4 : 2, extent[2] = {T, H};
  int64_t used[2];
  for (int i = 0; i < 2; i++) {
    used[i] = extent[i] == 1 ? 0 : strides[i];
    if (extent[i] == 1) continue;
    if (used[i] < 0 || (written && used[i] == 0)) return AR_ERR_SHAPE;
    if (used[i] * size % 16 != 0) return AR_ERR_ALIGNMENT;
  }
  if (!aligned(p, 16)) return AR_ERR_ALIGNMENT;
  *out = ar::KvRows{const_cast<void*>(p), used[0], used[1]};
  return AR_OK;
}
bool known(int dtype) { return dtype == AR_DTYPE_F32 || dtype == AR_DTYPE_BF16; }

int ready(ar::KvBatch* batch) {
  if (!ar::device_ok()) return AR_ERR_NO_DEVICE;
  uint32_t* word = nullptr;
  return ar::library_status_words(&word, &batch->sticky) ? AR_OK : AR_ERR_CUDA;
}

int move(bool write, const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, const void* k, const int64_t* k_strides,
         const void* v, const int64_t* v_strides, void* cu_stream) {
  ar::KvPool p;
  ar::KvBatch s;
  ar::KvRows kr, vr;
  int rc = check_pool(pool, &p);
  if (rc == AR_OK) rc = check_batch(batch, p, &s);
  if (rc == AR_OK && !known(dtype)) rc = AR_ERR_UNSUPPORTED;
  if (rc != AR_OK || s.T == 0) return rc;
  rc = check_rows(k, k_strides, s.T, p.Hkv, dtype, !write, &kr);
  if (rc == AR_OK) rc = check_rows(v, v_strides, s.T, p.Hkv, dtype, !write, &vr);
  if (rc != AR_OK) return rc;
  rc = ready(&s);
  if (rc != AR_OK) return rc;
  const cudaStream_t stream = (cudaStream_t)cu_stream;
  if ((write ? ar::launch_kv_append(p, s, dtype, kr, vr, stream) : ar::launch_kv_read(p, s, dtype, kr, vr, stream)) != cudaSuccess)
    return AR_ERR_CUDA;
  ar::count_launches(-1, 1);
  return AR_OK;
}

// The checks that the workspace's size depends on.
int check_attention(const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, int64_t Hq, int64_t max_length, ar::KvPool* p,
                    ar::KvBatch* s) {
  int rc = check_pool(pool, p);
  if (rc == AR_OK) rc = check_batch(batch, *p, s);
  if (rc != AR_OK) return rc;
  if (Hq <= 0 || Hq % p->Hkv != 0 || max_length <= 0) return AR_ERR_SHAPE;
  if (!known(dtype) || max_length > INT32_MAX - 256 || Hq > 65535 || batch->T * Hq > INT32_MAX) return AR_ERR_UNSUPPORTED;
  return AR_OK;
}

}  // namespace

extern "C" {

int ar_kv_cache_append(const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, const void* k, const int64_t* k_strides,
                       const void* v, const int64_t* v_strides, void* cu_stream) {
  return move(true, pool, batch, dtype, k, k_strides, v, v_strides, cu_stream);
}
int ar_kv_cache_read(const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, void* k_out, const int64_t* k_strides,
                     void* v_out, const int64_t* v_strides, void* cu_stream) {
  return move(false, pool, batch, dtype, k_out, k_strides, v_out, v_strides, cu_stream);
}

size_t ar_kv_cache_attention_workspace_bytes(const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, int64_t Hq,
                                             int64_t max_length, int causal) {
  ar::KvPool p;
  ar::KvBatch s;
  if (check_attention(pool, batch, dtype, Hq, max_length, &p, &s) != AR_OK || s.T == 0) return 0;
  return ar::kv_attn_plan(p, s, dtype, (int)Hq, (int)max_length, causal).workspace;
}

int ar_kv_cache_attention_plan(const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, int64_t Hq, int64_t max_length,
                               int causal, int32_t* plan) {
  ar::KvPool p;
  ar::KvBatch s;
  if (!plan) return AR_ERR_NULL;
  const int rc = check_attention(pool, batch, dtype, Hq, max_length, &p, &s);
  if (rc != AR_OK) return rc;
  const ar::KvAttnPlan found = s.T == 0 ? ar::KvAttnPlan{0, 0, 0, 0} : ar::kv_attn_plan(p, s, dtype, (int)Hq, (int)max_length, causal);
  plan[0] = found.rows;
  plan[1] = found.ctas;
  plan[2] = found.parts;
  return AR_OK;
}

int ar_kv_cache_attention(const ar_kv_pool* pool, const ar_kv_batch* batch, int dtype, const void* q,
                          const int64_t* q_strides, void* o, const int64_t* o_strides, int64_t Hq, int64_t max_length,
                          int causal, void* workspace, size_t workspace_bytes, void* cu_stream) {
  ar::KvAttnArgs a;
  int rc = check_attention(pool, batch, dtype, Hq, max_length, &a.pool, &a.batch);
  if (rc != AR_OK || a.batch.T == 0) return rc;
  rc = check_rows(q, q_strides, a.batch.T, Hq, dtype, false, &a.q);
  if (rc == AR_OK) rc = check_rows(o, o_strides, a.batch.T, Hq, dtype, true, &a.o);
  if (rc != AR_OK) return rc;
  a.dtype = dtype;
  a.Hq = (int)Hq;
  a.max_length = (int)max_length;
  a.causal = causal ? 1 : 0;
  a.partial = (float*)workspace;
  const ar::KvAttnPlan plan = ar::kv_attn_plan(a.pool, a.batch, dtype, a.Hq, a.max_length, a.causal);
  if (plan.workspace > 0) {
    if (!workspace || workspace_bytes < plan.workspace) return AR_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return AR_ERR_ALIGNMENT;
  }
  rc = ready(&a.batch);
  if (rc != AR_OK) return rc;
  int launches = 0;
  const cudaError_t e = ar::launch_kv_attention(a, plan, (cudaStream_t)cu_stream, &launches);
  ar::count_launches(-1, launches);
  return e == cudaSuccess ? AR_OK : AR_ERR_CUDA;
}

}  // extern "C"
