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

int esmcu_linear_w4(esmcu_context* ctx, const void* x, int64_t ldx, int dtype, const uint8_t* wq,
                    int64_t ldw, const void* scales, int scales_dtype, int64_t lds,
                    const uint8_t* zeros, int64_t ldz, int group, const float* bias, void* out,
                    int64_t ldo, int M, int N, int K, void* workspace, size_t workspace_bytes) {
  if (M < 0 || N < 0 || K < 0) return bad("negative shape");
  if (K > kLinearW4MaxK) return bad("K must be at most 131072");
  if (!is_dtype(dtype) || !is_dtype(scales_dtype)) return bad("bad dtype");
  if (group != 32 && group != 64 && group != 128) return bad("group must be 32, 64 or 128");
  const int64_t groups = (static_cast<int64_t>(K) + group - 1) / group;
  if (ldx < K || ldw < (static_cast<int64_t>(K) + 1) / 2 || lds < groups || (zeros != nullptr && ldz < groups) || ldo < N)
    return bad("a row stride is shorter than its row");
  if (M > 0 && N > 0 && (out == nullptr || (K > 0 && (x == nullptr || wq == nullptr || scales == nullptr))))
    return bad("x, wq, scales or out is null");
  const size_t need = M > 0 && N > 0 ? linear_w4_workspace(dtype, M, K, group) : 0;
  if (need > 0 &&
      (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return bad("workspace is null, too small or not 16-byte aligned");
  DeviceScope scope;
  const int rc = use_device(ctx);
  if (rc != ESMCU_OK) return rc;
  LinearW4Args a;
  a.x = x;
  a.ldx = ldx;
  a.type = dtype;
  a.W = wq;
  a.ldw = ldw;
  a.scales = scales;
  a.scale_type = scales_dtype;
  a.lds = lds;
  a.zeros = zeros;
  a.ldz = ldz;
  a.group = group;
  a.bias = bias;
  a.out = out;
  a.ldo = ldo;
  a.M = M;
  a.N = N;
  a.K = K;
  a.workspace = workspace;
  a.status = ctx->d_status;
  a.num_sms = ctx->num_sms;
  ESMCU_CUDA(launch_linear_w4(a, ctx->stream));
  return ESMCU_OK;
}

int esmcu_kv_append_paged(esmcu_context* ctx, const esmcu_paged_kv* cache, const void* q,
                          int64_t q_stride_token, int64_t q_stride_head, int num_q_heads,
                          const void* k, int64_t k_stride_token, int64_t k_stride_head,
                          const void* v, int64_t v_stride_token, int64_t v_stride_head, int dtype,
                          const float* cos_t, const float* sin_t, int table_rows, int rot_dim,
                          const int32_t* cu_seqlens, const int32_t* cache_lens, int B, int T,
                          void* q_out) {
  int rc = check_cache(cache);
  if (rc != ESMCU_OK) return rc;
  if (B < 0 || T < 0 || num_q_heads < 0 || table_rows < 0) return bad("negative shape");
  if (dtype != cache->dtype && dtype != ESMCU_F32)
    return bad("dtype must be the cache's, or fp32 to be rounded to it");
  if (!is_dtype(dtype)) return bad("bad dtype");
  if (rot_dim < 0 || rot_dim % 2 != 0 || rot_dim > cache->head_dim)
    return bad("rot_dim must be even and at most head_dim");
  if (q_stride_token < 0 || q_stride_head < 0 || k_stride_token < 0 || k_stride_head < 0 ||
      v_stride_token < 0 || v_stride_head < 0)
    return bad("negative stride");
  if (T > 0 && B > 0) {
    if (k == nullptr || v == nullptr || cu_seqlens == nullptr || cache_lens == nullptr)
      return bad("k, v, cu_seqlens or cache_lens is null");
    if ((num_q_heads > 0) != (q != nullptr) || (num_q_heads > 0) != (q_out != nullptr))
      return bad("q and q_out go with num_q_heads > 0");
    if (rot_dim > 0 && (cos_t == nullptr || sin_t == nullptr)) return bad("cos_t or sin_t is null");
  }
  DeviceScope scope;
  rc = use_device(ctx);
  if (rc != ESMCU_OK) return rc;
  KvAppendArgs a;
  a.kv = internal(*cache);
  a.q = q;
  a.k = k;
  a.v = v;
  a.type = dtype;
  a.q_tok = q_stride_token;
  a.q_head = q_stride_head;
  a.k_tok = k_stride_token;
  a.k_head = k_stride_head;
  a.v_tok = v_stride_token;
  a.v_head = v_stride_head;
  a.q_heads = num_q_heads;
  a.q_out = q_out;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.table_len = table_rows;
  a.rot = rot_dim;
  a.cu = cu_seqlens;
  a.lens = cache_lens;
  a.B = B;
  a.T = T;
  a.status = ctx->d_status;
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

int esmcu_attention_decode_paged(esmcu_context* ctx, const esmcu_paged_kv* cache, const void* q,
                                 int64_t q_stride_seq, int64_t q_stride_head, int num_q_heads,
                                 const int32_t* seq_lens, int B, float scale, int window, void* out,
                                 float* lse, void* workspace, size_t workspace_bytes) {
  int rc = check_decode(cache, num_q_heads);
  if (rc != ESMCU_OK) return rc;
  if (B < 0 || window < 0) return bad("negative batch or window");
  if (q_stride_seq < 0 || q_stride_head < 0) return bad("negative stride");
  if (B > 0 && (q == nullptr || seq_lens == nullptr || out == nullptr))
    return bad("q, seq_lens or out is null");
  if (reinterpret_cast<uintptr_t>(out) & 15) return bad("out must be 16-byte aligned");
  if (ctx == nullptr) return bad("null context");
  const size_t need = attention_decode_workspace(cache->dtype, num_q_heads, cache->num_kv_heads,
                                                 cache->head_dim, ctx->num_sms);
  if (B > 0 && need > 0 &&
      (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return bad("workspace is null, too small or not 16-byte aligned");
  DeviceScope scope;
  rc = use_device(ctx);
  if (rc != ESMCU_OK) return rc;
  AttentionDecodeArgs a;
  a.kv = internal(*cache);
  a.q = q;
  a.q_seq = q_stride_seq;
  a.q_head = q_stride_head;
  a.q_heads = num_q_heads;
  a.lens = seq_lens;
  a.B = B;
  a.scale = scale;
  a.window = window;
  a.out = out;
  a.lse = lse;
  a.workspace = workspace;
  a.status = ctx->d_status;
  a.num_sms = ctx->num_sms;
  ESMCU_CUDA(launch_attention_decode(a, ctx->stream));
  return ESMCU_OK;
}

}  // extern "C"
