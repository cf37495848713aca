// C ABI of the token-by-token serving operators (include/esm_b200.h): checks
// of the arguments, then one call of the launcher API.  The arguments are
// checked before the context, so a refusal needs no device.
#include <cuda_runtime.h>

#include <cstdint>

#include "../kernels.cuh"
#include "context.h"
#include "esm_b200.h"

using namespace esmb200;

namespace {

// Leaves the calling thread's current device as it was.
class DeviceScope {
 public:
  DeviceScope() {
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
  }
  ~DeviceScope() {
    int now = -1;
    if (before_ >= 0 && (cudaGetDevice(&now) != cudaSuccess || now != before_)) cudaSetDevice(before_);
  }

 private:
  int before_ = -1;
};

int bad(const char* what) { return fail(ESMCU_ERR_INVALID_ARGUMENT, what); }

bool is_dtype(int t) { return t == ESMCU_F32 || t == ESMCU_F16 || t == ESMCU_BF16; }
int size_of(int t) { return t == ESMCU_F32 ? 4 : 2; }

// A pointer that is not on a boundary of its elements faults on the device.
bool off(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0; }

bool rows_on_16(const void* p, int size, int64_t a, int64_t b, int64_t c) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(a * size) |
                         static_cast<uintptr_t>(b * size) | static_cast<uintptr_t>(c * size);
  return (bits & 15) == 0;
}

int check_cache(const esmcu_paged_kv* c) {
  if (c == nullptr) return bad("cache is null");
  if (!is_dtype(c->dtype)) return bad("cache: bad dtype");
  if (c->num_pages < 0 || c->page_size <= 0 || c->num_kv_heads <= 0 || c->head_dim <= 0 || c->max_pages < 0)
    return bad("cache: need num_pages, max_pages >= 0 and page_size, num_kv_heads, head_dim > 0");
  if (c->k_stride_page < 0 || c->k_stride_slot < 0 || c->k_stride_head < 0 || c->v_stride_page < 0 ||
      c->v_stride_slot < 0 || c->v_stride_head < 0 || c->page_table_stride < 0)
    return bad("cache: negative stride");
  if ((c->num_pages > 1 && (c->k_stride_page == 0 || c->v_stride_page == 0)) ||
      (c->page_size > 1 && (c->k_stride_slot == 0 || c->v_stride_slot == 0)) ||
      (c->num_kv_heads > 1 && (c->k_stride_head == 0 || c->v_stride_head == 0)))
    return bad("cache: a stride of 0 would put several elements into one place");
  if (c->num_pages > 0 && (c->k == nullptr || c->v == nullptr)) return bad("cache: k or v is null");
  if (c->max_pages > 0 && c->page_table == nullptr) return bad("cache: page_table is null");
  if (off(c->k, size_of(c->dtype)) || off(c->v, size_of(c->dtype)) || off(c->page_table, 4))
    return bad("cache: k, v or page_table is not on a boundary of its elements");
  return ESMCU_OK;
}

PagedKV internal(const esmcu_paged_kv& c) {
  PagedKV kv;
  kv.k = c.k;
  kv.v = c.v;
  kv.type = c.dtype;
  kv.num_pages = c.num_pages;
  kv.page_size = c.page_size;
  kv.heads = c.num_kv_heads;
  kv.dh = c.head_dim;
  kv.k_page = c.k_stride_page;
  kv.k_slot = c.k_stride_slot;
  kv.k_head = c.k_stride_head;
  kv.v_page = c.v_stride_page;
  kv.v_slot = c.v_stride_slot;
  kv.v_head = c.v_stride_head;
  kv.table = c.page_table;
  kv.table_stride = c.page_table_stride;
  kv.max_pages = c.max_pages;
  return kv;
}

int check_decode(const esmcu_paged_kv* c, int num_q_heads) {
  const int rc = check_cache(c);
  if (rc != ESMCU_OK) return rc;
  if (num_q_heads <= 0 || num_q_heads % c->num_kv_heads != 0)
    return bad("num_q_heads must be a positive multiple of num_kv_heads");
  if (c->head_dim % 8 != 0 || c->head_dim > 256)
    return bad("head_dim must be a multiple of 8 and <= 256");
  const int size = size_of(c->dtype);
  if (!rows_on_16(c->k, size, c->k_stride_page, c->k_stride_slot, c->k_stride_head) ||
      !rows_on_16(c->v, size, c->v_stride_page, c->v_stride_slot, c->v_stride_head))
    return bad("cache: rows must start on 16-byte boundaries");
  return ESMCU_OK;
}

}  // namespace

extern "C" {

int esmcu_linear_w4_workspace(int dtype, int M, int K, int group, size_t* bytes) {
  if (bytes == nullptr) return bad("bytes is null");
  *bytes = 0;
  if (M < 0 || K < 0) return bad("negative shape");
  if (K > kLinearW4MaxK) return bad("K must be at most 131072");
  if (!is_dtype(dtype)) return bad("bad dtype");
  if (group != 32 && group != 64 && group != 128) return bad("group must be 32, 64 or 128");
  *bytes = linear_w4_workspace(dtype, M, K, group);
  return ESMCU_OK;
}

int esmcu_linear_w4(esmcu_context* ctx, const esmcu_linear_w4_args* p) {
  if (p == nullptr) return bad("args is null");
  const int M = p->M, N = p->N, K = p->K, group = p->group;
  if (M < 0 || N < 0 || K < 0) return bad("negative shape");
  if (K > kLinearW4MaxK) return bad("K must be at most 131072");
  if (!is_dtype(p->dtype) || !is_dtype(p->scales_dtype)) return bad("bad dtype");
  if (group != 32 && group != 64 && group != 128) return bad("group must be 32, 64 or 128");
  const int64_t groups = (static_cast<int64_t>(K) + group - 1) / group;
  if (p->ldx < K || p->ldw < (static_cast<int64_t>(K) + 1) / 2 || p->lds < groups ||
      (p->zeros != nullptr && p->ldz < groups) || p->ldo < N)
    return bad("a row stride is shorter than its row");
  if (M > 0 && N > 0 &&
      (p->out == nullptr || (K > 0 && (p->x == nullptr || p->wq == nullptr || p->scales == nullptr))))
    return bad("x, wq, scales or out is null");
  if (off(p->x, size_of(p->dtype)) || off(p->out, size_of(p->dtype)) || off(p->scales, size_of(p->scales_dtype)) ||
      off(p->bias, 4))
    return bad("x, scales, bias or out is not on a boundary of its elements");
  const size_t need = M > 0 && N > 0 ? linear_w4_workspace(p->dtype, M, K, group) : 0;
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(p->workspace) & 15)))
    return bad("workspace is null, too small or not 16-byte aligned");
  DeviceScope scope;
  const int rc = use_device(ctx);
  if (rc != ESMCU_OK) return rc;
  LinearW4Args a;
  a.x = p->x;
  a.ldx = p->ldx;
  a.type = p->dtype;
  a.W = p->wq;
  a.ldw = p->ldw;
  a.scales = p->scales;
  a.scale_type = p->scales_dtype;
  a.lds = p->lds;
  a.zeros = p->zeros;
  a.ldz = p->ldz;
  a.group = group;
  a.bias = p->bias;
  a.out = p->out;
  a.ldo = p->ldo;
  a.M = M;
  a.N = N;
  a.K = K;
  a.workspace = p->workspace;
  a.status = ctx->d_status;
  a.num_sms = ctx->num_sms;
  ESMCU_CUDA(launch_linear_w4(a, ctx->stream));
  return ESMCU_OK;
}

int esmcu_kv_append_paged(esmcu_context* ctx, const esmcu_paged_kv* cache, const esmcu_kv_append_args* p) {
  int rc = check_cache(cache);
  if (rc != ESMCU_OK) return rc;
  if (p == nullptr) return bad("args is null");
  if (p->B < 0 || p->T < 0 || p->num_q_heads < 0 || p->table_rows < 0) return bad("negative shape");
  if (p->dtype != cache->dtype && p->dtype != ESMCU_F32)
    return bad("dtype must be the cache's, or fp32 to be rounded to it");
  if (p->rot_dim < 0 || p->rot_dim % 2 != 0 || p->rot_dim > cache->head_dim)
    return bad("rot_dim must be even and at most head_dim");
  if (p->q_stride_token < 0 || p->q_stride_head < 0 || p->k_stride_token < 0 || p->k_stride_head < 0 ||
      p->v_stride_token < 0 || p->v_stride_head < 0)
    return bad("negative stride");
  const int size = size_of(p->dtype);
  if (off(p->q, size) || off(p->k, size) || off(p->v, size) || off(p->q_out, size_of(cache->dtype)) ||
      off(p->cos_t, 4) || off(p->sin_t, 4) || off(p->cu_seqlens, 4) || off(p->cache_lens, 4))
    return bad("q, k, v, q_out, cos_t, sin_t, cu_seqlens or cache_lens is not on a boundary of its elements");
  if (p->T > 0 && p->B > 0) {
    if (p->k == nullptr || p->v == nullptr || p->cu_seqlens == nullptr || p->cache_lens == nullptr)
      return bad("k, v, cu_seqlens or cache_lens is null");
    if ((p->num_q_heads > 0) != (p->q != nullptr) || (p->num_q_heads > 0) != (p->q_out != nullptr))
      return bad("q and q_out go with num_q_heads > 0");
    if (p->rot_dim > 0 && (p->cos_t == nullptr || p->sin_t == nullptr)) return bad("cos_t or sin_t is null");
  }
  DeviceScope scope;
  rc = use_device(ctx);
  if (rc != ESMCU_OK) return rc;
  KvAppendArgs a;
  a.kv = internal(*cache);
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.type = p->dtype;
  a.q_tok = p->q_stride_token;
  a.q_head = p->q_stride_head;
  a.k_tok = p->k_stride_token;
  a.k_head = p->k_stride_head;
  a.v_tok = p->v_stride_token;
  a.v_head = p->v_stride_head;
  a.q_heads = p->num_q_heads;
  a.q_out = p->q_out;
  a.cos_t = p->cos_t;
  a.sin_t = p->sin_t;
  a.table_len = p->table_rows;
  a.rot = p->rot_dim;
  a.cu = p->cu_seqlens;
  a.lens = p->cache_lens;
  a.B = p->B;
  a.T = p->T;
  a.status = ctx->d_status;
  a.num_sms = ctx->num_sms;
  ESMCU_CUDA(launch_kv_append(a, ctx->stream));
  return ESMCU_OK;
}

int esmcu_attention_decode_paged_workspace(esmcu_context* ctx, const esmcu_paged_kv* cache,
                                           int num_q_heads, size_t* bytes) {
  if (bytes == nullptr) return bad("bytes is null");
  *bytes = 0;
  const int rc = check_decode(cache, num_q_heads);
  if (rc != ESMCU_OK) return rc;
  if (ctx == nullptr) return bad("null context");
  *bytes = attention_decode_workspace(cache->dtype, num_q_heads, cache->num_kv_heads, cache->head_dim,
                                      ctx->num_sms);
  return ESMCU_OK;
}

int esmcu_attention_decode_paged(esmcu_context* ctx, const esmcu_paged_kv* cache,
                                 const esmcu_attention_decode_args* p) {
  if (p == nullptr) return bad("args is null");
  int rc = check_decode(cache, p->num_q_heads);
  if (rc != ESMCU_OK) return rc;
  if (p->B < 0 || p->window < 0) return bad("negative batch or window");
  if (p->q_stride_seq < 0 || p->q_stride_head < 0) return bad("negative stride");
  if (p->B > 0 && (p->q == nullptr || p->seq_lens == nullptr || p->out == nullptr))
    return bad("q, seq_lens or out is null");
  if (reinterpret_cast<uintptr_t>(p->out) & 15) return bad("out must be 16-byte aligned");
  if (off(p->q, size_of(cache->dtype)) || off(p->seq_lens, 4) || off(p->lse, 4))
    return bad("q, seq_lens or lse is not on a boundary of its elements");
  if (ctx == nullptr) return bad("null context");
  const size_t need = attention_decode_workspace(cache->dtype, p->num_q_heads, cache->num_kv_heads,
                                                 cache->head_dim, ctx->num_sms);
  if (p->B > 0 && (p->workspace == nullptr || p->workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(p->workspace) & 15)))
    return bad("workspace is null, too small or not 16-byte aligned");
  DeviceScope scope;
  rc = use_device(ctx);
  if (rc != ESMCU_OK) return rc;
  AttentionDecodeArgs a;
  a.kv = internal(*cache);
  a.q = p->q;
  a.q_seq = p->q_stride_seq;
  a.q_head = p->q_stride_head;
  a.q_heads = p->num_q_heads;
  a.lens = p->seq_lens;
  a.B = p->B;
  a.scale = p->scale;
  a.window = p->window;
  a.out = p->out;
  a.lse = p->lse;
  a.workspace = p->workspace;
  a.status = ctx->d_status;
  a.num_sms = ctx->num_sms;
  ESMCU_CUDA(launch_attention_decode(a, ctx->stream));
  return ESMCU_OK;
}

}  // extern "C"
