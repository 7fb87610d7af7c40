// ltx25::Ops' attention members as a C++ program calls them: a prompt, its keys
// and values into the cache, the newest token over the cache, and a refused call
// that wait_ok reports. Outputs against double sums on the host.
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

constexpr int kTokens = 150, kHeads = 4, kKv = 2, kDim = 64, kPage = 32, kPages = 6;

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
std::vector<T> download(const void* p, size_t n)
{
  std::vector<T> v(n);
  if (hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess) {
    std::printf("download failed\n");
    std::exit(1);
  }
  return v;
}

// One query over `n` keys: each weight and the output are rounded to bf16, 2^-8 of
// themselves each, and a tenth is left for what is done in f32.
template <typename K, typename V>
bool row_is_right(const uint16_t* q, int n, K key, V val, const uint16_t* got)
{
  std::vector<double> s(n);
  double top = -1e300, sum = 0;
  for (int j = 0; j < n; ++j) {
    double x = 0;
    for (int d = 0; d < kDim; ++d) { x += (double)value_of(q[d]) * key(j, d); }
    s[j] = x / 8.0;
    top = std::fmax(top, s[j]);
  }
  for (double& x : s) { sum += x = std::exp(x - top); }
  for (int d = 0; d < kDim; ++d) {
    double want = 0, mag = 0;
    for (int j = 0; j < n; ++j) {
      want += s[j] / sum * val(j, d);
      mag += s[j] / sum * std::fabs(val(j, d));
    }
    if (!(std::fabs(value_of(got[d]) - want) <= 1.1 / 128 * mag)) {
      std::printf("channel %d: %g, not %g\n", d, value_of(got[d]), want);
      return false;
    }
  }
  return true;
}

}  // namespace

int main()
{
  ltx25::Ops ops;
  std::string err;
  if (!ops.init(&err)) {
    std::printf("NODEV: %s\n", err.c_str());
    return 3;
  }
  std::mt19937 gen(7);
  std::normal_distribution<float> normal;
  constexpr int kWidth = (kHeads + 2 * kKv) * kDim;   // q | k | v of one projection
  std::vector<uint16_t> qkv((size_t)kTokens * kWidth);
  for (uint16_t& x : qkv) { x = bf16_of(normal(gen)); }
  uint16_t* const d_qkv = upload(qkv);
  uint16_t* const d_out = upload(std::vector<uint16_t>((size_t)kTokens * kHeads * kDim));
  hipStream_t st = nullptr;

  const ltx25_attn a = {kHeads, kKv, kDim, 1, 0.0f, kWidth, kWidth, kWidth, kHeads * kDim};
  const uint16_t* const d_k = d_qkv + kHeads * kDim;
  const uint16_t* const d_v = d_k + kKv * kDim;
  ops.attention(st, a, d_qkv, d_k, d_v, d_out, nullptr, nullptr, nullptr, 1, kTokens, kTokens);
  if (!ops.wait_ok(st, &err)) {
    std::printf("attention: %s\n", err.c_str());
    return 1;
  }
  auto out = download<uint16_t>(d_out, (size_t)kTokens * kHeads * kDim);
  for (int i = 0; i < kTokens; ++i) {
    for (int h = 0; h < kHeads; ++h) {
      const int g = h / (kHeads / kKv);
      auto at = [&](int part, int j, int d) {
        return (double)value_of(qkv[(size_t)j * kWidth + (kHeads + part * kKv + g) * kDim + d]);
      };
      if (!row_is_right(&qkv[(size_t)i * kWidth + h * kDim], i + 1,
                        [&](int j, int d) { return at(0, j, d); },
                        [&](int j, int d) { return at(1, j, d); },
                        &out[((size_t)i * kHeads + h) * kDim])) {
        std::printf("token %d head %d\n", i, h);
        return 1;
      }
    }
  }

  const size_t codes = (size_t)kPages * kKv * kPage * kDim;
  ltx25_kv_cache cache = {};
  cache.k = upload(std::vector<int8_t>(codes));
  cache.v = upload(std::vector<int8_t>(codes));
  cache.k_scale = upload(std::vector<float>(kPages * kKv));
  cache.v_scale = upload(std::vector<float>(kPages * kKv));
  cache.pages = kPages;
  cache.page_tokens = kPage;
  cache.kv_heads = kKv;
  cache.head_dim = kDim;
  const std::vector<int> table = {3, 0, 5, 1, 4};
  int* const d_table = upload(table);
  int* const d_cu = upload(std::vector<int>{0, kTokens});
  int* const d_start = upload(std::vector<int>{0});
  int* const d_len = upload(std::vector<int>{kTokens});
  ops.kv_append(st, a, cache, d_table, (int)table.size(), d_k, d_v, d_cu, d_start, 1, kTokens);
  const size_t bytes = ltx25::Ops::attention_cached_workspace(a, 1, 1, kTokens);
  void* const ws = bytes > 0 ? (void*)upload(std::vector<uint8_t>(bytes)) : nullptr;
  const uint16_t* const q1 = d_qkv + (size_t)(kTokens - 1) * kWidth;
  ops.attention_cached(st, a, cache, d_table, (int)table.size(), d_len, q1, d_out, nullptr, 1, 1,
                       kTokens, ws, bytes);
  uint16_t* const d_back = upload(std::vector<uint16_t>((size_t)kTokens * kWidth));
  ops.kv_read(st, a, cache, d_table, (int)table.size(), d_back, d_back + kKv * kDim, d_cu, d_start,
              1, kTokens);
  if (!ops.wait_ok(st, &err)) {
    std::printf("cache: %s\n", err.c_str());
    return 1;
  }
  const auto kc = download<int8_t>(cache.k, codes), vc = download<int8_t>(cache.v, codes);
  const auto ks = download<float>(cache.k_scale, kPages * kKv);
  const auto vs = download<float>(cache.v_scale, kPages * kKv);
  const auto back = download<uint16_t>(d_back, (size_t)kTokens * kWidth);
  out = download<uint16_t>(d_out, (size_t)kHeads * kDim);
  for (int h = 0; h < kHeads; ++h) {
    const int g = h / (kHeads / kKv);
    auto key = [&](int j, int d) {
      const int b = table[j / kPage] * kKv + g;
      return (double)kc[((size_t)b * kPage + j % kPage) * kDim + d] * ks[b];
    };
    auto val = [&](int j, int d) {
      const int b = table[j / kPage] * kKv + g;
      return (double)vc[((size_t)b * kDim + d) * kPage + j % kPage] * vs[b];
    };
    if (!row_is_right(&qkv[(size_t)(kTokens - 1) * kWidth + h * kDim], kTokens, key, val,
                      &out[(size_t)h * kDim])) {
      std::printf("cached, head %d\n", h);
      return 1;
    }
    for (int j = 0; j < kTokens; ++j) {
      for (int d = 0; d < kDim; ++d) {
        const uint16_t* const row = &back[(size_t)j * kWidth + g * kDim + d];
        if (row[0] != bf16_of((float)key(j, d)) || row[kKv * kDim] != bf16_of((float)val(j, d))) {
          std::printf("read back: token %d head %d channel %d\n", j, g, d);
          return 1;
        }
      }
    }
  }

  ltx25_attn bad = a;
  bad.head_dim = 96;
  ops.attention(st, bad, d_qkv, d_k, d_v, d_out, nullptr, nullptr, nullptr, 1, kTokens, kTokens);
  if (ops.wait_ok(st, &err) || err.find("head_dim") == std::string::npos) {
    std::printf("a refused call was not reported: %s\n", err.c_str());
    return 1;
  }
  std::printf("OK\n");
  return 0;
}
