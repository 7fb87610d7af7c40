// The C ABI of the microscaled 4-bit tier (include/ltx25_mx4.h): argument validation
// ahead of any HIP call, then the launch. No state.
#include "ltx25_mx4.h"

#include "attention.h"
#include "checks.h"
#include "mx4.h"

#include <initializer_list>

namespace {

using namespace ltx25::checks;
using ltx25::set_error;

// Rows of an operand, and values of a row: a tile's rows then lie within 32-bit offsets
// past a 2 GiB operand's end.
constexpr int kRowsMax = 1 << 27;
constexpr int kWidthMax = 1 << 20;

bool sizes_fit(long rows, long K)
{
  return rows > 0 && rows <= kRowsMax && K > 0 && K <= kWidthMax && K % 32 == 0;
}

// No rows are an empty call rather than a mistake
int check_operand(const char* name, const ltx25_mx4* q, ltx25::Mx4Args* out)
{
  if (q == nullptr) { return set_error(LTX25_E_INVAL, "%s is null", name); }
  if (q->rows < 0 || q->rows > kRowsMax) {
    return set_error(LTX25_E_INVAL, "%s has %d rows: 0 .. %d are taken", name, q->rows, kRowsMax);
  }
  if (q->K <= 0 || q->K > kWidthMax || q->K % 32 != 0) {
    return set_error(LTX25_E_INVAL, "%s: K=%d is not a multiple of 32 in 32 .. %d", name, q->K,
                     kWidthMax);
  }
  out->codes = (uint8_t*)q->codes;
  out->scales = (uint8_t*)q->scales;
  out->rows = q->rows;
  out->K = q->K;
  if (q->rows == 0) { return LTX25_OK; }
  if (q->codes == nullptr || q->scales == nullptr) {
    return set_error(LTX25_E_INVAL, "%s: codes or scales is null", name);
  }
  if (!aligned(q->codes, 16) || !aligned(q->scales, 4)) {
    return set_error(LTX25_E_INVAL, "%s: codes (%p) must be 16-byte and scales (%p) 4-byte aligned",
                     name, q->codes, q->scales);
  }
  return LTX25_OK;
}

int check_row_stride(const char* name, int64_t stride, int K, int multiple)
{
  if (stride < K || stride >= (int64_t)1 << 31 || stride % multiple != 0) {
    return set_error(LTX25_E_INVAL,
                     "%s=%lld: a row's stride is a multiple of %d, at least %d and below 2^31", name,
                     (long long)stride, multiple, K);
  }
  return LTX25_OK;
}

// What the two products share, after their operands' own checks. `need`: the workspace's
// bytes.
int check_product(const ltx25::Mx4Args& w, int M, const void* bias, int bias_dtype, const void* y,
                  int epilogue, const void* workspace, size_t workspace_bytes, size_t need)
{
  if (bias_dtype < LTX25_DT_NONE || bias_dtype > LTX25_DT_F32) {
    return set_error(LTX25_E_INVAL, "bias_dtype=%d is none of LTX25_DT_NONE, BF16 and F32",
                     bias_dtype);
  }
  if ((bias == nullptr) != (bias_dtype == LTX25_DT_NONE)) {
    return set_error(LTX25_E_INVAL, "bias and bias_dtype=%d do not go together", bias_dtype);
  }
  if (epilogue != LTX25_EPI_NONE && epilogue != LTX25_EPI_GELU_TANH) {
    return set_error(LTX25_E_INVAL, "epilogue=%d is none of LTX25_EPI_*", epilogue);
  }
  if (ltx25::mx4_code_bytes(w.rows, w.K) >= (size_t)1 << 31) {
    return set_error(LTX25_E_UNSUPPORTED, "the weight's %zu bytes of codes are 2 GiB or more",
                     ltx25::mx4_code_bytes(w.rows, w.K));
  }
  if (M == 0 || w.rows == 0) { return LTX25_OK; }
  int rc = check_pointer("y", y, 16);
  if (rc != LTX25_OK) { return rc; }
  if ((rc = check_aligned("bias", bias, bias_dtype == LTX25_DT_F32 ? 4 : 2)) != LTX25_OK) {
    return rc;
  }
  return need > 0 ? check_workspace(workspace, workspace_bytes, need) : LTX25_OK;
}

// An output that begins where another tensor of the call does would be written while that is
// still read.
struct Named {
  const char* name;
  const void* at;
};
int check_apart(Named out, std::initializer_list<Named> others)
{
  for (const Named& o : others) {
    if (o.at == out.at) {
      return set_error(LTX25_E_INVAL, "%s is %s: not in place", out.name, o.name);
    }
  }
  return LTX25_OK;
}

// Rows and the library's order of them
int check_orders(const void* codes, const void* scales, const ltx25_mx4* q)
{
  int rc = check_pointer("codes", codes, 16);
  if (rc != LTX25_OK || (rc = check_pointer("scales", scales, 16)) != LTX25_OK) { return rc; }
  rc = check_apart({"codes", codes}, {{"q's codes", q->codes}, {"q's scales", q->scales}});
  return rc != LTX25_OK
             ? rc
             : check_apart({"scales", scales}, {{"q's codes", q->codes}, {"q's scales", q->scales}});
}

int check_source(const char* name, const void* x, int64_t stride, int K, bool wide)
{
  const int rc = check_row_stride(name, stride, K, wide ? 4 : 8);
  return rc != LTX25_OK ? rc : check_pointer("x", x, 16);
}

// Where the activations' scales lie in linear_mx4's workspace, behind their codes
size_t scales_at(int M, int K) { return (ltx25::mx4_code_bytes(M, K) + 255) & ~(size_t)255; }

int run(void* stream, ltx25::Mx4Gemm& g, const ltx25::Mx4Plan& plan, const void* bias,
        int bias_dtype, void* y, int epilogue)
{
  int rc = ltx25::check_device();
  if (rc != LTX25_OK) { return rc; }
  g.bias = bias;
  g.bias_type = bias_dtype == LTX25_DT_BF16   ? ltx25::kBiasBf16
                : bias_dtype == LTX25_DT_F32 ? ltx25::kBiasF32
                                             : ltx25::kBiasNone;
  g.epilogue = epilogue == LTX25_EPI_GELU_TANH ? ltx25::kEpiGelu : ltx25::kEpiNone;
  g.y = (uint16_t*)y;
  const hipError_t e = ltx25::launch_mx4_gemm(g, plan, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "4-bit product launch");
}

}  // namespace

extern "C" {

size_t ltx25_mx4_code_bytes(int rows, int K)
{
  return sizes_fit(rows, K) ? ltx25::mx4_code_bytes(rows, K) : 0;
}

size_t ltx25_mx4_scale_bytes(int rows, int K)
{
  return sizes_fit(rows, K) ? ltx25::mx4_scale_bytes(rows, K) : 0;
}

int ltx25_mx4_quantize_rows(void* stream, const void* x, int x_dtype, int64_t x_stride,
                            const ltx25_mx4* q)
{
  ltx25::Mx4Args a;
  int rc = check_operand("q", q, &a);
  if (rc != LTX25_OK) { return rc; }
  if (x_dtype != LTX25_DT_BF16 && x_dtype != LTX25_DT_F32) {
    return set_error(LTX25_E_INVAL, "x_dtype=%d is neither LTX25_DT_BF16 nor LTX25_DT_F32", x_dtype);
  }
  if (a.rows == 0) { return LTX25_OK; }
  const bool wide = x_dtype == LTX25_DT_F32;
  if ((rc = check_source("x_stride", x, x_stride, a.K, wide)) != LTX25_OK ||
      (rc = ltx25::check_device()) != LTX25_OK) {
    return rc;
  }
  const hipError_t e = ltx25::launch_mx4_quantize(x, wide, x_stride, a, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "4-bit coding launch");
}

int ltx25_mx4_dequant(void* stream, const ltx25_mx4* q, void* out, int64_t out_stride)
{
  ltx25::Mx4Args a;
  int rc = check_operand("q", q, &a);
  if (rc != LTX25_OK || a.rows == 0) { return rc; }
  if ((rc = check_row_stride("out_stride", out_stride, a.K, 8)) != LTX25_OK ||
      (rc = check_pointer("out", out, 16)) != LTX25_OK || (rc = ltx25::check_device()) != LTX25_OK) {
    return rc;
  }
  const hipError_t e = ltx25::launch_mx4_dequant(a, (uint16_t*)out, out_stride, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "4-bit expansion launch");
}

int ltx25_mx4_pack(void* stream, const void* codes, const void* scales, const ltx25_mx4* q)
{
  ltx25::Mx4Args a;
  int rc = check_operand("q", q, &a);
  if (rc != LTX25_OK || a.rows == 0) { return rc; }
  if ((rc = check_orders(codes, scales, q)) != LTX25_OK ||
      (rc = ltx25::check_device()) != LTX25_OK) {
    return rc;
  }
  const hipError_t e = ltx25::launch_mx4_pack((const uint8_t*)codes, (const uint8_t*)scales, a,
                                              (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "4-bit packing launch");
}

int ltx25_mx4_unpack(void* stream, const ltx25_mx4* q, void* codes, void* scales)
{
  ltx25::Mx4Args a;
  int rc = check_operand("q", q, &a);
  if (rc != LTX25_OK || a.rows == 0) { return rc; }
  if ((rc = check_orders(codes, scales, q)) != LTX25_OK ||
      (rc = ltx25::check_device()) != LTX25_OK) {
    return rc;
  }
  const hipError_t e =
      ltx25::launch_mx4_unpack(a, (uint8_t*)codes, (uint8_t*)scales, (hipStream_t)stream);
  return e == hipSuccess ? LTX25_OK : hip_error(e, "4-bit unpacking launch");
}

// The waves' sums meet in LDS
size_t ltx25_mx4_gemm_workspace(int, int, int) { return 0; }

int ltx25_mx4_gemm(void* stream, const ltx25_mx4* x, const ltx25_mx4* w, const void* bias,
                   int bias_dtype, void* y, int epilogue, void* workspace, size_t workspace_bytes)
{
  ltx25::Mx4Gemm g;
  int rc = check_operand("x", x, &g.x);
  if (rc != LTX25_OK || (rc = check_operand("w", w, &g.w)) != LTX25_OK) { return rc; }
  if (g.x.K != g.w.K) {
    return set_error(LTX25_E_INVAL, "x has rows of %d values, w of %d", g.x.K, g.w.K);
  }
  const size_t need = ltx25_mx4_gemm_workspace(g.x.rows, g.x.K, g.w.rows);
  rc = check_product(g.w, g.x.rows, bias, bias_dtype, y, epilogue, workspace, workspace_bytes, need);
  if (rc != LTX25_OK || g.x.rows == 0 || g.w.rows == 0) { return rc; }
  rc = check_apart({"y", y}, {{"x's codes", x->codes}, {"x's scales", x->scales},
                              {"w's codes", w->codes}, {"w's scales", w->scales}, {"bias", bias}});
  if (rc != LTX25_OK) { return rc; }
  return run(stream, g, ltx25::plan_mx4(g.x.rows, g.x.K, g.w.rows, false), bias, bias_dtype, y,
             epilogue);
}

size_t ltx25_linear_mx4_workspace(int M, int K, int N)
{
  if (!sizes_fit(M, K) || !sizes_fit(N, K)) { return 0; }
  if (!ltx25::plan_mx4(M, K, N, true).codes_ahead) { return 0; }
  return scales_at(M, K) + ltx25::mx4_scale_bytes(M, K);
}

int ltx25_linear_mx4(void* stream, const void* x, int64_t x_stride, int M, const ltx25_mx4* w,
                     const void* bias, int bias_dtype, void* y, int epilogue, void* workspace,
                     size_t workspace_bytes)
{
  ltx25::Mx4Gemm g;
  int rc = check_operand("w", w, &g.w);
  if (rc != LTX25_OK || (rc = check_tokens("M", M, kRowsMax)) != LTX25_OK) { return rc; }
  const size_t need = ltx25_linear_mx4_workspace(M, g.w.K, g.w.rows);
  rc = check_product(g.w, M, bias, bias_dtype, y, epilogue, workspace, workspace_bytes, need);
  if (rc != LTX25_OK || M == 0 || g.w.rows == 0) { return rc; }
  if ((rc = check_source("x_stride", x, x_stride, g.w.K, false)) != LTX25_OK ||
      (rc = check_apart({"y", y}, {{"x", x}, {"w's codes", w->codes}, {"w's scales", w->scales},
                                   {"bias", bias}, {"the workspace", workspace}})) != LTX25_OK) {
    return rc;
  }
  const ltx25::Mx4Plan plan = ltx25::plan_mx4(M, g.w.K, g.w.rows, true);
  g.x.codes = (uint8_t*)workspace;
  g.x.scales = (uint8_t*)workspace + scales_at(M, g.w.K);
  g.x.rows = M;
  g.x.K = g.w.K;
  g.xb = (const uint16_t*)x;
  g.xb_stride = x_stride;
  return run(stream, g, plan, bias, bias_dtype, y, epilogue);
}

}  // extern "C"
