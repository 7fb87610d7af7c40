// Positions rotated into queries and keys (ltx25_rope).
#include "block.h"

#include <algorithm>
#include <climits>

namespace ltx25 {
namespace {

constexpr int kThreads = 256;

struct RopeParams {
  Rotation r;
  const uint16_t* in[2];
  uint16_t* out[2];
  long in_stride[2], out_stride[2];
  int heads[2];
  int dim, tokens;
  int chunks;        // 16-byte pieces, or pairs of them, of a head
  int units;         // of a token
  uint32_t by_chunks, by_units;   // ceil(2^32 / .)
  int per_group;     // tokens of a workgroup
};

// n / d for n < 2^16, m = ceil(2^32 / d) (d > 1; d = 1: m = 0)
__device__ __forceinline__ int divide(int n, uint32_t m) { return m == 0 ? n : (int)__umulhi(n, m); }

// A thread turns eight channels (pairs side by side) or twice eight, half of the rotated
// channels apart, and computes its pairs' sines itself.
//
// Bound by memory.
template <bool SIDE>
__global__ void __launch_bounds__(kThreads) rope_kernel(RopeParams p, long first)
{
  const long token0 = first + (long)blockIdx.x * p.per_group;
  const int count = min((long)p.per_group, p.tokens - token0) * p.units;
  for (int u = threadIdx.x; u < count; u += kThreads) {
    const int t = divide(u, p.by_units);
    const int unit = u - t * p.units;
    int head = divide(unit, p.by_chunks);
    const int chunk = unit - head * p.chunks;
    const int which = head >= p.heads[0] ? 1 : 0;
    head -= which ? p.heads[0] : 0;
    const long token = token0 + t;
    const uint16_t* const in =
        (which ? p.in[1] + token * p.in_stride[1] : p.in[0] + token * p.in_stride[0]) + head * p.dim;
    uint16_t* const out =
        (which ? p.out[1] + token * p.out_stride[1] : p.out[0] + token * p.out_stride[0]) + head * p.dim;
    if constexpr (SIDE) {
      uint4 x = *(const uint4*)(in + chunk * 8);
      if (chunk * 4 < p.r.pairs) {
        x = rotate_side(x, turns_of(p.r, token), pairs_of<4>(p.r, head, chunk * 4));
      }
      *(uint4*)(out + chunk * 8) = x;
    } else {
      const bool turn = chunk * 8 < p.r.pairs;
      // chunks past the pairs' are those of the channels that are not rotated
      const int at = turn ? chunk * 8 : chunk * 8 + p.r.pairs;
      uint4 a = *(const uint4*)(in + at);
      if (turn) {
        uint4 b = *(const uint4*)(in + at + p.r.pairs);
        rotate_halves(a, b, turns_of(p.r, token), pairs_of<8>(p.r, head, chunk * 8));
        *(uint4*)(out + at + p.r.pairs) = b;
      }
      *(uint4*)(out + at) = a;
    }
  }
}

uint32_t magic(int d) { return d <= 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / (unsigned)d); }

}  // namespace

hipError_t launch_rope(const RopeArgs& a, hipStream_t stream)
{
  RopeParams p;
  p.r = a.r;
  for (int i = 0; i < 2; ++i) {
    p.in[i] = a.in[i];
    p.out[i] = a.out[i];
    p.in_stride[i] = (long)a.in_stride[i];
    p.out_stride[i] = (long)a.out_stride[i];
    p.heads[i] = a.heads[i];
  }
  p.dim = a.head_dim;
  p.tokens = a.tokens;
  p.chunks = a.r.interleaved ? a.head_dim / 8 : (a.head_dim - a.r.pairs) / 8;
  p.units = (a.heads[0] + a.heads[1]) * p.chunks;
  p.by_chunks = magic(p.chunks);
  p.by_units = magic(p.units);
  p.per_group = std::max(1, 2 * kThreads / p.units);
  // a launch has fewer than 2^32 threads
  const long most = ((1L << 32) / kThreads - 1) * p.per_group;
  for (long first = 0; first < a.tokens; first += most) {
    const long n = std::min(most, a.tokens - first);
    const unsigned groups = (unsigned)((n + p.per_group - 1) / p.per_group);
    if (a.r.interleaved) {
      rope_kernel<true><<<groups, kThreads, 0, stream>>>(p, first);
    } else {
      rope_kernel<false><<<groups, kThreads, 0, stream>>>(p, first);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { return e; }
  }
  return hipSuccess;
}

}  // namespace ltx25
