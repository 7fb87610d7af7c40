// ltx25::Ops' 4-bit, norm and position members as a C++ program calls them: a norm into
// 4-bit activations, their product with a packed weight, the same of bf16 rows in one
// call, keys rotated in place and on their way into the cache, and a refused call that
// wait_ok reports. Outputs against double sums on the host.
#include "ltx25_ops.h"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <string>
#include <vector>

namespace {

constexpr int kTokens = 70, kWidth = 160, kOut = 50;
constexpr int kHeads = 4, kKv = 2, kDim = 64, kPage = 32, kPages = 4;

float value_of(uint16_t b)
{
  const uint32_t u = (uint32_t)b << 16;
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
uint16_t bf16_of(float f)
{
  uint32_t u;
  std::memcpy(&u, &f, 4);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <typename T>
T* upload(const std::vector<T>& v)
{
  T* p = nullptr;
  if (hipMalloc((void**)&p, v.size() * sizeof(T)) != hipSuccess ||
      hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) {
    std::printf("upload failed\n");
    std::exit(1);
  }
  return p;
}
template <typename T>
T* room(size_t n)
{
  return upload(std::vector<T>(n));
}
template <typename T>
std::vector<T> download(const void* p, size_t n)
{
  std::vector<T> v(n);
  if (hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess) {
    std::printf("download failed\n");
    std::exit(1);
  }
  return v;
}

bool near(const char* what, int row, int at, double got, double want, double allowed)
{
  if (std::fabs(got - want) <= allowed) { return true; }
  std::printf("%s, row %d, %d: %g, not %g\n", what, row, at, got, want);
  return false;
}

ltx25_mx4 mx4(int rows, int K)
{
  return {room<uint8_t>(ltx25_mx4_code_bytes(rows, K)), room<uint8_t>(ltx25_mx4_scale_bytes(rows, K)),
          rows, K};
}

constexpr double kMagnitudes[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};

}  // namespace

int main()
{
  ltx25::Ops ops;
  std::string err;
  if (!ops.init(&err)) {
    std::printf("NODEV: %s\n", err.c_str());
    return 3;
  }
  hipStream_t st = nullptr;
  std::mt19937 gen(11);
  std::normal_distribution<float> normal;
  auto random_bf16 = [&](size_t n) {
    std::vector<uint16_t> v(n);
    for (uint16_t& x : v) { x = bf16_of(normal(gen)); }
    return v;
  };

  // ---- a norm, in bf16 and in 4 bits, and products of it
  const auto x = random_bf16((size_t)kTokens * kWidth), weight = random_bf16(kWidth);
  uint16_t* const d_x = upload(x);
  uint16_t* const d_weight = upload(weight);
  uint16_t* const d_normed = room<uint16_t>((size_t)kTokens * kWidth);
  uint16_t* const d_values = room<uint16_t>((size_t)kTokens * kWidth);
  ltx25_norm n = {};
  n.width = kWidth;
  n.eps = 1e-6f;
  n.residual_scale = 1.0f;
  n.x_dtype = n.mod_dtype = n.weight_dtype = LTX25_DT_BF16;
  n.x_stride = n.x_out_stride = n.y_stride = n.mod_stride = n.out_stride = kWidth;
  const ltx25_mx4 q = mx4(kTokens, kWidth), w = mx4(kOut, kWidth);
  std::vector<uint8_t> wcodes((size_t)kOut * kWidth / 2), wscales((size_t)kOut * kWidth / 32);
  for (uint8_t& b : wcodes) { b = (uint8_t)gen(); }
  for (uint8_t& b : wscales) { b = (uint8_t)(122 + gen() % 6); }
  uint8_t* const d_wcodes = upload(wcodes);
  uint8_t* const d_wscales = upload(wscales);
  uint8_t* const d_codes_back = room<uint8_t>(wcodes.size());
  uint8_t* const d_scales_back = room<uint8_t>(wscales.size());
  const auto bias = random_bf16(kOut);
  uint16_t* const d_bias = upload(bias);
  uint16_t* const d_y = room<uint16_t>((size_t)kTokens * kOut);
  uint16_t* const d_y2 = room<uint16_t>((size_t)kTokens * kOut);
  uint16_t* const d_y3 = room<uint16_t>((size_t)kTokens * kOut);

  ops.block_norm(st, n, d_x, nullptr, nullptr, nullptr, nullptr, d_weight, nullptr, nullptr,
                 nullptr, d_normed, kTokens);
  ops.block_norm_mx4(st, n, d_x, nullptr, nullptr, nullptr, nullptr, d_weight, nullptr, nullptr,
                     nullptr, q, kTokens);
  ops.mx4_dequant(st, q, d_values, kWidth);
  ops.mx4_pack(st, d_wcodes, d_wscales, w);
  ops.mx4_unpack(st, w, d_codes_back, d_scales_back);
  const size_t bytes = ltx25::Ops::mx4_gemm_workspace(kTokens, kWidth, kOut);
  void* const ws = bytes > 0 ? (void*)room<uint8_t>(bytes) : nullptr;
  ops.mx4_gemm(st, q, w, d_bias, d_y, false, ws, bytes);
  // the activations' codes by two calls and by one
  ops.mx4_quantize_rows(st, d_normed, LTX25_DT_BF16, kWidth, q);
  ops.mx4_gemm(st, q, w, nullptr, d_y2, true, ws, bytes);
  const size_t bytes3 = ltx25::Ops::linear_mx4_workspace(kTokens, kWidth, kOut);
  void* const ws3 = bytes3 > 0 ? (void*)room<uint8_t>(bytes3) : nullptr;
  ops.linear_mx4(st, d_normed, kWidth, kTokens, w, nullptr, d_y3, true, ws3, bytes3);
  if (!ops.wait_ok(st, &err)) {
    std::printf("norm and products: %s\n", err.c_str());
    return 1;
  }
  const auto normed = download<uint16_t>(d_normed, (size_t)kTokens * kWidth);
  const auto values = download<uint16_t>(d_values, (size_t)kTokens * kWidth);
  const auto y = download<uint16_t>(d_y, (size_t)kTokens * kOut);
  if (download<uint8_t>(d_codes_back, wcodes.size()) != wcodes ||
      download<uint8_t>(d_scales_back, wscales.size()) != wscales) {
    std::printf("packed and unpacked again the weight is another\n");
    return 1;
  }
  if (download<uint16_t>(d_y2, (size_t)kTokens * kOut) !=
      download<uint16_t>(d_y3, (size_t)kTokens * kOut)) {
    std::printf("linear_mx4 is not the two calls\n");
    return 1;
  }
  auto w_at = [&](int r, int k) {
    const int code = wcodes[((size_t)r * kWidth + k) / 2] >> (4 * (k & 1)) & 15;
    const double v = std::ldexp(kMagnitudes[code & 7], wscales[((size_t)r * kWidth + k) / 32] - 127);
    return code & 8 ? -v : v;
  };
  for (int t = 0; t < kTokens; ++t) {
    double sum = 0, want[kWidth];
    for (int k = 0; k < kWidth; ++k) { sum += std::pow((double)value_of(x[t * kWidth + k]), 2); }
    for (int k = 0; k < kWidth; ++k) {
      want[k] = value_of(x[t * kWidth + k]) / std::sqrt(sum / kWidth + 1e-6) * value_of(weight[k]);
      // one rounding to bf16, and a few to f32
      if (!near("norm", t, k, value_of(normed[t * kWidth + k]), want[k],
                std::fabs(want[k]) * (1.0 / 256 + 1e-6))) {
        return 1;
      }
    }
    for (int b = 0; b < kWidth; b += 32) {
      double top = 0;
      for (int k = b; k < b + 32; ++k) { top = std::fmax(top, std::fabs(want[k])); }
      // magnitudes of 6 to 8 units of the block's, of which the largest is at least as much, lose
      // up to 2 of them, those of 4 to 6 (the largest 4 or more) up to 1
      for (int k = b; k < b + 32; ++k) {
        if (!near("codes", t, k, value_of(values[t * kWidth + k]), want[k], top * 0.3334)) { return 1; }
      }
    }
    for (int c = 0; c < kOut; ++c) {
      double v = value_of(bias[c]), mag = std::fabs(v);
      for (int k = 0; k < kWidth; ++k) {
        const double p = value_of(values[t * kWidth + k]) * w_at(c, k);
        v += p;
        mag += std::fabs(p);
      }
      // one rounding to bf16, and f32 sums of kWidth products
      if (!near("product", t, c, value_of(y[t * kOut + c]), v,
                std::fabs(v) / 256 + mag * kWidth / (1 << 24))) {
        return 1;
      }
    }
  }

  // ---- keys rotated in place, and on their way into the cache
  constexpr int kPitch = (kHeads + 2 * kKv) * kDim;   // q | k | v of one projection
  const auto qkv = random_bf16((size_t)kTokens * kPitch);
  uint16_t* const d_qkv = upload(qkv);
  uint16_t* const d_turned = upload(qkv);
  std::vector<float> freqs(kDim / 2);
  for (int p = 0; p < kDim / 2; ++p) { freqs[p] = (float)std::pow(10000.0, -2.0 * p / kDim); }
  std::vector<int> places(kTokens);
  for (int i = 0; i < kTokens; ++i) { places[i] = i; }
  const ltx25_attn a = {kHeads, kKv, kDim, 1, 0.0f, kPitch, kPitch, kPitch, kHeads * kDim};
  ltx25_rotation r = {};
  r.head_dim = kDim;
  r.n_axes = 1;
  r.freq_heads = 1;
  r.pos_dtype = LTX25_DT_I32;
  r.freqs = upload(freqs);
  r.positions = upload(places);
  ltx25_kv_cache caches[2] = {};
  for (ltx25_kv_cache& c : caches) {
    c.k = room<int8_t>((size_t)kPages * kKv * kPage * kDim);
    c.v = room<int8_t>((size_t)kPages * kKv * kPage * kDim);
    c.k_scale = room<float>(kPages * kKv);
    c.v_scale = room<float>(kPages * kKv);
    c.pages = kPages;
    c.page_tokens = kPage;
    c.kv_heads = kKv;
    c.head_dim = kDim;
  }
  int* const d_table = upload(std::vector<int>{2, 0, 3});
  int* const d_cu = upload(std::vector<int>{0, kTokens});
  int* const d_start = upload(std::vector<int>{0});
  uint16_t* const d_tk = d_turned + kHeads * kDim;
  const uint16_t* const d_k = d_qkv + kHeads * kDim;
  const uint16_t* const d_v = d_k + kKv * kDim;
  ops.rope(st, r, a, d_turned, d_tk, kTokens);
  ops.kv_append(st, a, caches[0], d_table, 3, d_tk, d_v, d_cu, d_start, 1, kTokens);
  r.positions = nullptr;
  ops.kv_append_rope(st, a, caches[1], d_table, 3, d_k, d_v, d_cu, d_start, r, 1, kTokens);
  if (!ops.wait_ok(st, &err)) {
    std::printf("rotations: %s\n", err.c_str());
    return 1;
  }
  const auto turned = download<uint16_t>(d_turned, qkv.size());
  for (int t = 0; t < kTokens; ++t) {
    for (int c = 0; c < kPitch; ++c) {
      const size_t at = (size_t)t * kPitch + c;
      if (c >= (kHeads + kKv) * kDim) {   // v
        if (turned[at] == qkv[at]) { continue; }
        std::printf("rope wrote behind the keys\n");
        return 1;
      }
      const int p = c % (kDim / 2);
      const bool first = c % kDim < kDim / 2;
      const double me = value_of(qkv[at]);
      const double other = value_of(qkv[first ? at + kDim / 2 : at - kDim / 2]);
      const double angle = (double)freqs[p] * t;
      const double want = me * std::cos(angle) + (first ? -other : other) * std::sin(angle);
      if (!near("rotation", t, c, value_of(turned[at]), want,
                std::fabs(want) * (1.0 / 256 + 1e-6) +
                    (std::fabs(me) + std::fabs(other)) / (1 << 20))) {
        return 1;
      }
    }
  }
  const size_t codes = (size_t)kPages * kKv * kPage * kDim;
  if (download<int8_t>(caches[0].k, codes) != download<int8_t>(caches[1].k, codes) ||
      download<int8_t>(caches[0].v, codes) != download<int8_t>(caches[1].v, codes) ||
      download<float>(caches[0].k_scale, kPages * kKv) !=
          download<float>(caches[1].k_scale, kPages * kKv)) {
    std::printf("kv_append_rope is not the two calls\n");
    return 1;
  }

  n.width = kWidth + 4;
  ops.block_norm(st, n, d_x, nullptr, nullptr, nullptr, nullptr, d_weight, nullptr, nullptr,
                 nullptr, d_normed, kTokens);
  if (ops.wait_ok(st, &err) || err.find("width") == std::string::npos) {
    std::printf("a refused call was not reported: %s\n", err.c_str());
    return 1;
  }
  std::printf("OK\n");
  return 0;
}
