// The C ABI of what a block does around its linears and its attention
// (include/ltx25_block.h; ltx25_kv_append_rope is in capi_attention.cpp, beside the
// cache's checks): argument validation ahead of any HIP call, then the launch. No state.
#include "ltx25_block.h"

#include "block.h"
#include "checks.h"

#include <cmath>

namespace {

using namespace ltx25::checks;
using ltx25::set_error;

constexpr int kNormWidthMax = 16384;

int check_stride(const char* name, int64_t stride, int64_t width)
{
  if (stride < width || stride >= (int64_t)1 << 31 || stride % 8 != 0) {
    return set_error(LTX25_E_INVAL,
                     "%s=%lld: a stride is a multiple of 8, at least %lld and below 2^31", name,
                     (long long)stride, (long long)width);
  }
  return LTX25_OK;
}

int check_float_type(const char* name, int type)
{
  if (type != LTX25_DT_BF16 && type != LTX25_DT_F32) {
    return set_error(LTX25_E_INVAL, "%s=%d is neither LTX25_DT_BF16 nor LTX25_DT_F32", name, type);
  }
  return LTX25_OK;
}

// An output in an input's place is there token for token, or one would be written over before
// it is read. `alike`: of one type.
int check_in_place(const char* name, const void* out, int64_t out_stride, const char* of,
                   const void* in, int64_t in_stride, bool alike, int tokens)
{
  if (out == nullptr || out != in || (alike && (tokens <= 1 || out_stride == in_stride))) {
    return LTX25_OK;
  }
  return set_error(LTX25_E_INVAL, "%s is %s but not of its type and stride", name, of);
}

// Everything but the output's own pointer and type. `out`: there is one.
int check_norm(const ltx25_norm* n, const void* x, const void* y, const void* x_out,
               const void* after, const void* gate, const void* weight, const void* scale,
               const void* shift, const int* rows, bool out, int step, int tokens,
               ltx25::NormArgs* a)
{
  if (n == nullptr) { return set_error(LTX25_E_INVAL, "the norm's sizes are null"); }
  if (n->width <= 0 || n->width > kNormWidthMax || n->width % step != 0) {
    return set_error(LTX25_E_INVAL, "width=%d is not a multiple of %d in %d .. %d", n->width, step,
                     step, kNormWidthMax);
  }
  if (n->layer != 0 && n->layer != 1) {
    return set_error(LTX25_E_INVAL, "layer=%d is neither 0 nor 1", n->layer);
  }
  if (!(n->eps >= 0x1p-80f) || !std::isfinite(n->eps)) {
    return set_error(LTX25_E_INVAL, "eps=%g is not a finite number of 2^-80 or more",
                     (double)n->eps);
  }
  if (!std::isfinite(n->residual_scale)) {
    return set_error(LTX25_E_INVAL, "residual_scale=%g is not finite", (double)n->residual_scale);
  }
  int rc = check_float_type("x_dtype", n->x_dtype);
  if (rc != LTX25_OK || (rc = check_tokens("tokens", tokens, kPackedMax)) != LTX25_OK ||
      (rc = check_stride("x_stride", n->x_stride, n->width)) != LTX25_OK) {
    return rc;
  }
  if (y == nullptr) {
    if (after != nullptr || gate != nullptr || x_out != nullptr) {
      return set_error(LTX25_E_INVAL, "post_weight, gate and x_out need a y");
    }
    if (!out && tokens > 0) { return set_error(LTX25_E_INVAL, "without y there must be an out"); }
  } else if ((rc = check_stride("y_stride", n->y_stride, n->width)) != LTX25_OK ||
             (rc = check_stride("x_out_stride", n->x_out_stride, n->width)) != LTX25_OK) {
    return rc;
  }
  const bool modulated = gate != nullptr || scale != nullptr || shift != nullptr;
  if (modulated) {
    if ((rc = check_float_type("mod_dtype", n->mod_dtype)) != LTX25_OK) { return rc; }
    if (n->mod_rows <= 0) {
      return set_error(LTX25_E_INVAL, "mod_rows=%d: gate, scale and shift have a row or more",
                       n->mod_rows);
    }
    if ((rc = check_stride("mod_stride", n->mod_stride, n->width)) != LTX25_OK) { return rc; }
    if (rows == nullptr && tokens % n->mod_rows != 0) {
      return set_error(LTX25_E_INVAL, "tokens=%d is no multiple of mod_rows=%d and rows is null",
                       tokens, n->mod_rows);
    }
  }
  if ((weight != nullptr || after != nullptr) &&
      (rc = check_float_type("weight_dtype", n->weight_dtype)) != LTX25_OK) {
    return rc;
  }
  if (tokens == 0) { return LTX25_OK; }
  if ((rc = check_pointer("x", x, 16)) != LTX25_OK ||
      (rc = check_aligned("y", y, 16)) != LTX25_OK ||
      (y != nullptr && (rc = check_pointer("x_out", x_out, 16)) != LTX25_OK) ||
      (rc = check_aligned("post_weight", after, 16)) != LTX25_OK ||
      (rc = check_aligned("gate", gate, 16)) != LTX25_OK ||
      (rc = check_aligned("weight", weight, 16)) != LTX25_OK ||
      (rc = check_aligned("scale", scale, 16)) != LTX25_OK ||
      (rc = check_aligned("shift", shift, 16)) != LTX25_OK ||
      (rc = check_aligned("rows", rows, 4)) != LTX25_OK ||
      (rc = check_in_place("x_out", x_out, n->x_out_stride, "x", x, n->x_stride, true, tokens)) !=
          LTX25_OK) {
    return rc;
  }
  if (x_out != nullptr && x_out == y) { return set_error(LTX25_E_INVAL, "x_out is y"); }
  a->x = x;
  a->y = (const uint16_t*)y;
  a->x_out = const_cast<void*>(x_out);
  a->after = after;
  a->gate = gate;
  a->weight = weight;
  a->scale = scale;
  a->shift = shift;
  a->rows = modulated ? rows : nullptr;
  a->xs = n->x_stride;
  a->xos = n->x_out_stride;
  a->ys = n->y_stride;
  a->ms = n->mod_stride;
  a->os = n->out_stride;
  a->width = n->width;
  a->tokens = tokens;
  a->mod_rows = modulated ? n->mod_rows : 0;
  a->run = modulated && rows == nullptr ? tokens / n->mod_rows : 1;
  a->layer = n->layer != 0;
  a->wide = n->x_dtype == LTX25_DT_F32;
  a->mod_wide = modulated && n->mod_dtype == LTX25_DT_F32;
  a->weight_wide = (weight != nullptr || after != nullptr) && n->weight_dtype == LTX25_DT_F32;
  a->eps = n->eps;
  a->alpha = n->residual_scale;
  return LTX25_OK;
}

int run_norm(void* stream, const ltx25::NormArgs& a)
{
  const int rc = ltx25::check_device();
  if (rc != LTX25_OK) { return rc; }
  const hipError_t e = ltx25::launch_norm(a, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "norm launch");
}

}  // namespace

namespace ltx25 {

int check_rotation(const ltx25_rotation* r, bool needed, bool place, Rotation* out)
{
  if (r == nullptr) { return set_error(LTX25_E_INVAL, "the rotation is null"); }
  if (r->head_dim < 16 || r->head_dim > 256 || r->head_dim % 16 != 0) {
    return set_error(LTX25_E_UNSUPPORTED, "head_dim=%d is not a multiple of 16 in 16 .. 256",
                     r->head_dim);
  }
  const int rot = r->rot_dim == 0 ? r->head_dim : r->rot_dim;
  if (rot < 16 || rot > r->head_dim || rot % 16 != 0) {
    return set_error(LTX25_E_INVAL, "rot_dim=%d is not a multiple of 16 in 16 .. %d (or 0)",
                     r->rot_dim, r->head_dim);
  }
  if (r->interleaved != 0 && r->interleaved != 1) {
    return set_error(LTX25_E_INVAL, "interleaved=%d is neither 0 nor 1", r->interleaved);
  }
  if (r->n_axes < 1 || r->n_axes > kAxesMax) {
    return set_error(LTX25_E_INVAL, "n_axes=%d is not in 1 .. %d", r->n_axes, kAxesMax);
  }
  const bool placed = place && r->positions == nullptr;
  if (!placed && r->pos_dtype != LTX25_DT_F32 && r->pos_dtype != LTX25_DT_I32) {
    return set_error(LTX25_E_INVAL, "pos_dtype=%d is neither LTX25_DT_F32 nor LTX25_DT_I32",
                     r->pos_dtype);
  }
  if (needed) {
    int rc = check_pointer("freqs", r->freqs, 16);
    if (rc != LTX25_OK || (rc = check_aligned("axes", r->axes, 16)) != LTX25_OK) { return rc; }
    if (!placed && (rc = check_pointer("positions", r->positions, 4)) != LTX25_OK) { return rc; }
  }
  out->freqs = r->freqs;
  out->axes = r->axes;
  out->positions = r->positions;
  out->pairs = rot / 2;
  out->n_axes = r->n_axes;
  out->whole = r->pos_dtype == LTX25_DT_I32;
  out->per_head = r->freq_heads != 1;
  out->interleaved = r->interleaved != 0;
  return LTX25_OK;
}

}  // namespace ltx25

extern "C" {

int ltx25_block_norm(void* stream, const ltx25_norm* n, const void* x, const void* y, void* x_out,
                     const void* post_weight, const void* gate, const void* weight,
                     const void* scale, const void* shift, const int* rows, void* out, int tokens)
{
  ltx25::NormArgs a;
  int rc = check_norm(n, x, y, x_out, post_weight, gate, weight, scale, shift, rows, out != nullptr,
                      8, tokens, &a);
  if (rc != LTX25_OK) { return rc; }
  if (out != nullptr && (rc = check_stride("out_stride", n->out_stride, n->width)) != LTX25_OK) {
    return rc;
  }
  if (tokens == 0) { return LTX25_OK; }
  if ((rc = check_aligned("out", out, 16)) != LTX25_OK ||
      (rc = check_in_place("out", out, n->out_stride, "x", x, n->x_stride,
                           n->x_dtype == LTX25_DT_BF16, tokens)) != LTX25_OK ||
      (rc = check_in_place("out", out, n->out_stride, "y", y, n->y_stride, true, tokens)) !=
          LTX25_OK) {
    return rc;
  }
  if (out != nullptr && (out == x_out || (out == x && y != nullptr))) {
    return set_error(LTX25_E_INVAL, "out is %s", out == x_out ? "x_out" : "x, and y is given");
  }
  a.out = (uint16_t*)out;
  return run_norm(stream, a);
}

int ltx25_block_norm_mx4(void* stream, const ltx25_norm* n, const void* x, const void* y,
                         void* x_out, const void* post_weight, const void* gate,
                         const void* weight, const void* scale, const void* shift,
                         const int* rows, const ltx25_mx4* q, int tokens)
{
  ltx25::NormArgs a;
  int rc = check_norm(n, x, y, x_out, post_weight, gate, weight, scale, shift, rows, true, 32,
                      tokens, &a);
  if (rc != LTX25_OK) { return rc; }
  if (q == nullptr || q->rows != tokens || q->K != n->width) {
    return set_error(LTX25_E_INVAL, "q must have the call's %d rows of %d values", tokens, n->width);
  }
  if (tokens == 0) { return LTX25_OK; }
  if ((rc = check_pointer("q's codes", q->codes, 16)) != LTX25_OK ||
      (rc = check_pointer("q's scales", q->scales, 4)) != LTX25_OK) {
    return rc;
  }
  a.q.codes = (uint8_t*)q->codes;
  a.q.scales = (uint8_t*)q->scales;
  a.q.rows = q->rows;
  a.q.K = q->K;
  return run_norm(stream, a);
}

int ltx25_rope(void* stream, const ltx25_rotation* r, const void* q, void* q_out, int heads,
               int64_t q_stride, int64_t q_out_stride, const void* k, void* k_out, int kv_heads,
               int64_t k_stride, int64_t k_out_stride, int tokens)
{
  ltx25::RopeArgs a;
  int rc = check_tokens("tokens", tokens, kPackedMax);
  if (rc != LTX25_OK ||
      (rc = ltx25::check_rotation(r, tokens > 0, tokens == 0, &a.r)) != LTX25_OK) {
    return rc;
  }
  // the kernel's divisions are exact below 2^16 pieces of a token
  constexpr int kHeadsMax = 1024;
  if (heads < 0 || kv_heads < 0 || heads + (long)kv_heads < 1 || heads + (long)kv_heads > kHeadsMax) {
    return set_error(LTX25_E_INVAL, "heads=%d and kv_heads=%d are not 1 .. %d together", heads,
                     kv_heads, kHeadsMax);
  }
  if (r->freq_heads != 1 && ((heads > 0 && r->freq_heads != heads) ||
                             (kv_heads > 0 && r->freq_heads != kv_heads))) {
    return set_error(LTX25_E_INVAL, "freq_heads=%d is neither 1 nor heads=%d and kv_heads=%d",
                     r->freq_heads, heads, kv_heads);
  }
  const void* const in[2] = {q, k};
  void* const out[2] = {q_out, k_out};
  const int64_t strides[2][2] = {{q_stride, q_out_stride}, {k_stride, k_out_stride}};
  const int counts[2] = {heads, kv_heads};
  const char* const names[2][4] = {{"q", "q_out", "q_stride", "q_out_stride"},
                                   {"k", "k_out", "k_stride", "k_out_stride"}};
  for (int i = 0; i < 2; ++i) {
    if (counts[i] == 0) {
      if (in[i] != nullptr || out[i] != nullptr) {
        return set_error(LTX25_E_INVAL, "%s is given but has no heads", names[i][0]);
      }
      continue;
    }
    const int64_t width = (int64_t)counts[i] * r->head_dim;
    if ((rc = check_stride(names[i][2], strides[i][0], width)) != LTX25_OK ||
        (rc = check_stride(names[i][3], strides[i][1], width)) != LTX25_OK) {
      return rc;
    }
    if (tokens == 0) { continue; }
    if ((rc = check_pointer(names[i][0], in[i], 16)) != LTX25_OK ||
        (rc = check_pointer(names[i][1], out[i], 16)) != LTX25_OK ||
        (rc = check_in_place(names[i][1], out[i], strides[i][1], names[i][0], in[i], strides[i][0],
                             true, tokens)) != LTX25_OK) {
      return rc;
    }
    a.in[i] = (const uint16_t*)in[i];
    a.out[i] = (uint16_t*)out[i];
    a.in_stride[i] = strides[i][0];
    a.out_stride[i] = strides[i][1];
    a.heads[i] = counts[i];
  }
  if (tokens == 0) { return LTX25_OK; }
  if (heads > 0 && kv_heads > 0 && (q_out == k_out || q_out == k || k_out == q)) {
    return set_error(LTX25_E_INVAL, "%s: one tensor turned as queries and as keys",
                     q_out == k_out ? "q_out is k_out" : q_out == k ? "q_out is k" : "k_out is q");
  }
  if ((rc = ltx25::check_device()) != LTX25_OK) { return rc; }
  a.head_dim = r->head_dim;
  a.tokens = tokens;
  const hipError_t e = ltx25::launch_rope(a, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "rope launch");
}

}  // extern "C"
