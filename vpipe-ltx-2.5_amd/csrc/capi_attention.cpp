// The C ABI of attention and its cache (include/ltx25_attention.h): argument
// validation ahead of any HIP call, then the launch. No state: what a call
// needs is its own tensors and the caller's workspace.
#include "ltx25_block.h"

#include "block.h"
#include "checks.h"

#include <hip/hip_runtime.h>

#include <cmath>

namespace {

using namespace ltx25::checks;
using ltx25::set_error;

// The kernels form a 64-token tile's offsets in 32 bits.
constexpr int64_t kStrideMax = (int64_t)1 << 23;
// Tokens of a cached sequence; positions past them would not fit the kernels' 32-bit
// token numbers.
constexpr int kTokensMax = 1 << 30;

int check_stride(const char* name, int64_t stride, int heads, int head_dim)
{
  if (stride < (int64_t)heads * head_dim || stride >= kStrideMax || stride % 8 != 0) {
    return set_error(LTX25_E_INVAL,
                     "%s=%lld: a token's stride is a multiple of 8, at least %lld and below %lld",
                     name, (long long)stride, (long long)heads * head_dim, (long long)kStrideMax);
  }
  return LTX25_OK;
}

int check_heads(int heads, int kv_heads, int head_dim)
{
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) {
    return set_error(LTX25_E_INVAL, "heads=%d is not a positive multiple of kv_heads=%d", heads,
                     kv_heads);
  }
  if (head_dim != 64 && head_dim != 128) {
    return set_error(LTX25_E_UNSUPPORTED, "head_dim=%d: the kernels take 64 and 128", head_dim);
  }
  return LTX25_OK;
}

int check_attn(const ltx25_attn* a, float* scale)
{
  if (a == nullptr) { return set_error(LTX25_E_INVAL, "the attention's sizes are null"); }
  int rc = check_heads(a->heads, a->kv_heads, a->head_dim);
  if (rc != LTX25_OK) { return rc; }
  if (!(a->scale >= 0.0f) || !std::isfinite(a->scale)) {
    return set_error(LTX25_E_INVAL, "scale=%g is not a positive finite number (or 0)",
                     (double)a->scale);
  }
  *scale = a->scale > 0.0f ? a->scale : 1.0f / std::sqrt((float)a->head_dim);
  if ((rc = check_stride("q_stride", a->q_stride, a->heads, a->head_dim)) != LTX25_OK) {
    return rc;
  }
  return check_stride("out_stride", a->out_stride, a->heads, a->head_dim);
}

int check_cache(const ltx25_kv_cache* c, const int* table, int table_stride, int batch,
                ltx25::CacheArgs* out)
{
  if (c == nullptr) { return set_error(LTX25_E_INVAL, "the cache is null"); }
  int rc = check_heads(c->kv_heads, c->kv_heads, c->head_dim);
  if (rc != LTX25_OK) { return rc; }
  int log2 = 4;
  while (log2 < 7 && (1 << log2) != c->page_tokens) { ++log2; }
  if ((1 << log2) != c->page_tokens) {
    return set_error(LTX25_E_UNSUPPORTED, "page_tokens=%d: pages hold 16, 32, 64 or 128 tokens",
                     c->page_tokens);
  }
  if (c->pages <= 0 || table_stride <= 0 || batch < 0) {
    return set_error(LTX25_E_INVAL, "pages=%d table_stride=%d must be positive, batch=%d not below 0",
                     c->pages, table_stride, batch);
  }
  if ((rc = check_pointer("the cache's k", c->k, 16)) != LTX25_OK ||
      (rc = check_pointer("the cache's v", c->v, 16)) != LTX25_OK ||
      (rc = check_pointer("the cache's k_scale", c->k_scale, 4)) != LTX25_OK ||
      (rc = check_pointer("the cache's v_scale", c->v_scale, 4)) != LTX25_OK) {
    return rc;
  }
  if (batch > 0 && (rc = check_pointer("table", table, 4)) != LTX25_OK) { return rc; }
  out->k = (int8_t*)c->k;
  out->v = (int8_t*)c->v;
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->pages = c->pages;
  out->page_log2 = log2;
  out->kv_heads = c->kv_heads;
  out->head_dim = c->head_dim;
  out->table = table;
  out->table_stride = table_stride;
  return LTX25_OK;
}

// What append and read share.
int check_move(const ltx25_kv_cache* cache, const int* table, int table_stride, const void* k,
               const void* v, int64_t k_stride, int64_t v_stride, const int* cu, const int* start,
               int batch, int total, ltx25::CacheArgs* c)
{
  int rc = check_cache(cache, table, table_stride, batch, c);
  if (rc != LTX25_OK) { return rc; }
  if ((rc = check_tokens("total", total, kPackedMax)) != LTX25_OK ||
      (rc = check_stride("k_stride", k_stride, c->kv_heads, c->head_dim)) != LTX25_OK ||
      (rc = check_stride("v_stride", v_stride, c->kv_heads, c->head_dim)) != LTX25_OK) {
    return rc;
  }
  if (batch == 0 || total == 0) { return LTX25_OK; }
  if ((rc = check_pointer("k", k, 16)) != LTX25_OK ||
      (rc = check_pointer("v", v, 16)) != LTX25_OK ||
      (rc = check_pointer("cu", cu, 4)) != LTX25_OK ||
      (rc = check_pointer("start", start, 4)) != LTX25_OK) {
    return rc;
  }
  return LTX25_OK;
}

}  // namespace

namespace {

// `split`: the workspace is asked for and used where the plan has parts.
int attention(void* stream, const ltx25_attn* a, const void* q, const void* k, const void* v,
              void* out, float* lse, const int* cu_q, const int* cu_k, int batch, int total_q,
              int total_k, bool split, void* workspace, size_t workspace_bytes)
{
  float scale = 0.0f;
  int rc = check_attn(a, &scale);
  if (rc != LTX25_OK) { return rc; }
  if ((rc = check_stride("k_stride", a->k_stride, a->kv_heads, a->head_dim)) != LTX25_OK ||
      (rc = check_stride("v_stride", a->v_stride, a->kv_heads, a->head_dim)) != LTX25_OK ||
      (rc = check_tokens("total_q", total_q, kPackedMax)) != LTX25_OK ||
      (rc = check_tokens("total_k", total_k, kPackedMax)) != LTX25_OK) {
    return rc;
  }
  if (batch < 0) { return set_error(LTX25_E_INVAL, "batch=%d is negative", batch); }
  if ((cu_q == nullptr) != (cu_k == nullptr) || (cu_q == nullptr && batch > 1)) {
    return set_error(LTX25_E_INVAL,
                     "cu_q and cu_k: both, or neither with a batch of 1 (batch=%d)", batch);
  }
  if (batch == 0 || total_q == 0) { return LTX25_OK; }
  if ((rc = check_pointer("q", q, 16)) != LTX25_OK ||
      (rc = check_pointer("out", out, 16)) != LTX25_OK ||
      (total_k > 0 && (rc = check_pointer("k", k, 16)) != LTX25_OK) ||
      (total_k > 0 && (rc = check_pointer("v", v, 16)) != LTX25_OK)) {
    return rc;
  }
  if (!aligned(lse, 4) || !aligned(cu_q, 4) || !aligned(cu_k, 4)) {
    return set_error(LTX25_E_INVAL, "lse, cu_q or cu_k is not 4-byte aligned");
  }
  const size_t need = split ? ltx25_attention_workspace(a, batch, total_q, total_k) : 0;
  if (need > 0 && (rc = check_workspace(workspace, workspace_bytes, need)) != LTX25_OK) {
    return rc;
  }
  if ((rc = ltx25::check_device()) != LTX25_OK) { return rc; }
  ltx25::AttentionArgs p;
  p.workspace = need > 0 ? (float*)workspace : nullptr;
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.v = (const uint16_t*)v;
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.qs = a->q_stride;
  p.ks = a->k_stride;
  p.vs = a->v_stride;
  p.os = a->out_stride;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.causal = a->causal != 0;
  p.scale = scale;
  p.batch = batch;
  p.total_q = total_q;
  p.total_k = total_k;
  const hipError_t e = ltx25::launch_attention(p, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "attention launch");
}

}  // namespace

extern "C" {

int ltx25_attention(void* stream, const ltx25_attn* a, const void* q, const void* k, const void* v,
                    void* out, float* lse, const int* cu_q, const int* cu_k, int batch,
                    int total_q, int total_k)
{
  return attention(stream, a, q, k, v, out, lse, cu_q, cu_k, batch, total_q, total_k, false,
                   nullptr, 0);
}

size_t ltx25_attention_workspace(const ltx25_attn* a, int batch, int total_q, int total_k)
{
  if (a == nullptr || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads != 0 ||
      (a->head_dim != 64 && a->head_dim != 128) || batch <= 0 || total_q <= 0 || total_k <= 0 ||
      total_q > kPackedMax || total_k > kPackedMax) {
    return 0;
  }
  return ltx25::plan_prompt(a->heads, a->kv_heads, a->head_dim, batch, total_q, total_k)
      .workspace_bytes;
}

int ltx25_attention_split(void* stream, const ltx25_attn* a, const void* q, const void* k,
                          const void* v, void* out, float* lse, const int* cu_q, const int* cu_k,
                          int batch, int total_q, int total_k, void* workspace,
                          size_t workspace_bytes)
{
  return attention(stream, a, q, k, v, out, lse, cu_q, cu_k, batch, total_q, total_k, true,
                   workspace, workspace_bytes);
}

int ltx25_kv_append(void* stream, const ltx25_kv_cache* cache, const int* table, int table_stride,
                    const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                    const int* cu, const int* start, int batch, int total)
{
  ltx25::CacheArgs c;
  int rc = check_move(cache, table, table_stride, k, v, k_stride, v_stride, cu, start, batch, total,
                      &c);
  if (rc != LTX25_OK || batch == 0 || total == 0) { return rc; }
  if ((rc = ltx25::check_device()) != LTX25_OK) { return rc; }
  const hipError_t e =
      ltx25::launch_kv_append(c, (const uint16_t*)k, (const uint16_t*)v, k_stride, v_stride, cu,
                              start, batch, total, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "kv_append launch");
}

int ltx25_kv_append_rope(void* stream, const ltx25_kv_cache* cache, const int* table,
                         int table_stride, const void* k, const void* v, int64_t k_stride,
                         int64_t v_stride, const int* cu, const int* start,
                         const ltx25_rotation* r, int batch, int total)
{
  ltx25::CacheArgs c;
  ltx25::Rotation rot;
  int rc = check_move(cache, table, table_stride, k, v, k_stride, v_stride, cu, start, batch, total,
                      &c);
  if (rc != LTX25_OK) { return rc; }
  const bool work = batch > 0 && total > 0;
  if ((rc = ltx25::check_rotation(r, work, true, &rot)) != LTX25_OK) { return rc; }
  if (r->head_dim != c.head_dim) {
    return set_error(LTX25_E_INVAL, "the rotation is of heads of width %d, the cache's are of %d",
                     r->head_dim, c.head_dim);
  }
  if (r->freq_heads != 1 && r->freq_heads != c.kv_heads) {
    return set_error(LTX25_E_INVAL, "freq_heads=%d is neither 1 nor the cache's kv_heads=%d",
                     r->freq_heads, c.kv_heads);
  }
  if (!work) { return LTX25_OK; }
  if ((rc = ltx25::check_device()) != LTX25_OK) { return rc; }
  const hipError_t e =
      ltx25::launch_kv_append_rope(c, (const uint16_t*)k, (const uint16_t*)v, k_stride, v_stride,
                                   cu, start, rot, batch, total, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "kv_append_rope launch");
}

int ltx25_kv_read(void* stream, const ltx25_kv_cache* cache, const int* table, int table_stride,
                  void* k, void* v, int64_t k_stride, int64_t v_stride, const int* cu,
                  const int* start, int batch, int total)
{
  ltx25::CacheArgs c;
  int rc = check_move(cache, table, table_stride, k, v, k_stride, v_stride, cu, start, batch, total,
                      &c);
  if (rc != LTX25_OK || batch == 0 || total == 0) { return rc; }
  if ((rc = ltx25::check_device()) != LTX25_OK) { return rc; }
  const hipError_t e = ltx25::launch_kv_read(c, (uint16_t*)k, (uint16_t*)v, k_stride, v_stride, cu,
                                             start, batch, total, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "kv_read launch");
}

size_t ltx25_attention_cached_workspace(int batch, int q_len, int heads, int kv_heads, int head_dim,
                                        int max_len)
{
  if (batch <= 0 || q_len <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128) || max_len <= 0 || max_len > kTokensMax ||
      (long)batch * q_len > kPackedMax) {
    return 0;
  }
  return ltx25::plan_cached(batch, q_len, heads, kv_heads, head_dim, max_len).workspace_bytes;
}

int ltx25_attention_cached(void* stream, const ltx25_attn* a, const ltx25_kv_cache* cache,
                           const int* table, int table_stride, const int* lens, const void* q,
                           void* out, float* lse, int batch, int q_len, int max_len,
                           void* workspace, size_t workspace_bytes)
{
  float scale = 0.0f;
  int rc = check_attn(a, &scale);
  if (rc != LTX25_OK) { return rc; }
  ltx25::CachedArgs p;
  rc = check_cache(cache, table, table_stride, batch, &p.c);
  if (rc != LTX25_OK) { return rc; }
  if (a->kv_heads != cache->kv_heads || a->head_dim != cache->head_dim) {
    return set_error(LTX25_E_INVAL,
                     "the call has %d kv heads of width %d, the cache %d of width %d", a->kv_heads,
                     a->head_dim, cache->kv_heads, cache->head_dim);
  }
  if (q_len < 0 || max_len < 0) {
    return set_error(LTX25_E_INVAL, "q_len=%d max_len=%d must not be negative", q_len, max_len);
  }
  if ((rc = check_tokens("max_len", max_len, kTokensMax)) != LTX25_OK ||
      (rc = check_tokens("batch * q_len", (long)batch * q_len, kPackedMax)) != LTX25_OK) {
    return rc;
  }
  if (batch == 0 || q_len == 0) { return LTX25_OK; }
  if ((rc = check_pointer("lens", lens, 4)) != LTX25_OK ||
      (rc = check_pointer("q", q, 16)) != LTX25_OK ||
      (rc = check_pointer("out", out, 16)) != LTX25_OK) {
    return rc;
  }
  if (!aligned(lse, 4)) { return set_error(LTX25_E_INVAL, "lse is not 4-byte aligned"); }
  const size_t need = ltx25_attention_cached_workspace(batch, q_len, a->heads, a->kv_heads,
                                                       a->head_dim, max_len);
  if (need > 0 && (rc = check_workspace(workspace, workspace_bytes, need)) != LTX25_OK) {
    return rc;
  }
  if ((rc = ltx25::check_device()) != LTX25_OK) { return rc; }
  p.lens = lens;
  p.q = (const uint16_t*)q;
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.workspace = (float*)workspace;
  p.qs = a->q_stride;
  p.os = a->out_stride;
  p.heads = a->heads;
  p.causal = a->causal != 0;
  p.scale = scale;
  p.batch = batch;
  p.q_len = q_len;
  p.max_len = max_len;
  const hipError_t e = ltx25::launch_attention_cached(p, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "attention_cached launch");
}

}  // extern "C"
