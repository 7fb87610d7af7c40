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
  int dim;
  long tokens;
  int chunks;        // a head's pieces of work
  int units;         // a token's
  int blocks;        // workgroups over a token's
  uint32_t by_chunks;   // ceil(2^32 / chunks)
};

// n / d for n < 2^16, m = ceil(2^32 / d) (d = 1: m = 0)
__device__ __forceinline__ uint32_t divide(uint32_t n, uint32_t m) { return m == 0 ? n : __umulhi(n, m); }

// A thread turns eight channels (SIDE: pairs side by side) or twice eight, half of the rotated
// channels apart, of TOKENS tokens one after another, for which it reads their frequencies and axes
// once, and computes its pairs' sines itself.
//
// Bound by memory.
template <bool SIDE, bool MANY, int TOKENS>
__global__ void __launch_bounds__(kThreads) rope_kernel(RopeParams p, long first)
{
  const long group = first + (long)(blockIdx.x / (unsigned)p.blocks);
  const uint32_t unit = blockIdx.x % (unsigned)p.blocks * kThreads + threadIdx.x;
  if (unit >= (uint32_t)p.units) { return; }
  int head = (int)divide(unit, p.by_chunks);
  const int chunk = (int)unit - head * p.chunks;
  const int which = head >= p.heads[0] ? 1 : 0;
  head -= which ? p.heads[0] : 0;
  const uint16_t* const in = (which ? p.in[1] : p.in[0]) + head * p.dim;
  uint16_t* const out = (which ? p.out[1] : p.out[0]) + head * p.dim;
  const long in_stride = which ? p.in_stride[1] : p.in_stride[0];
  const long out_stride = which ? p.out_stride[1] : p.out_stride[0];
  const bool turn = chunk * (SIDE ? 4 : 8) < p.r.pairs;
  // halves: chunks past the pairs' are those of the channels that are not rotated
  const int at = SIDE || turn ? chunk * 8 : chunk * 8 + p.r.pairs;
  const long token0 = group * TOKENS;
  uint4 a[TOKENS], b[SIDE ? 1 : TOKENS];
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    const long token = min(token0 + t, p.tokens - 1);
    a[t] = *(const uint4*)(in + token * in_stride + at);
    if constexpr (!SIDE) {
      if (turn) { b[t] = *(const uint4*)(in + token * in_stride + at + p.r.pairs); }
    }
  }
  if (turn) {
    const Pairs<SIDE ? 4 : 8> pairs = pairs_of<MANY, SIDE ? 4 : 8>(p.r, head, chunk * (SIDE ? 4 : 8));
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      const Turns<MANY> turns = turns_of<MANY>(p.r, min(token0 + t, p.tokens - 1));
      if constexpr (SIDE) {
        a[t] = rotate_side<MANY>(a[t], turns, pairs);
      } else {
        rotate_halves<MANY>(a[t], b[t], turns, pairs);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    if (token0 + t >= p.tokens) { break; }
    uint16_t* const to = out + (token0 + t) * out_stride + at;
    *(uint4*)to = a[t];
    if constexpr (!SIDE) {
      if (turn) { *(uint4*)(to + p.r.pairs) = b[t]; }
    }
  }
}

uint32_t magic(int d) { return d <= 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / (unsigned)d); }

template <bool SIDE, bool MANY, int TOKENS>
hipError_t run(const RopeParams& p, hipStream_t stream)
{
  // a launch has fewer than 2^32 threads
  const long groups = (p.tokens + TOKENS - 1) / TOKENS;
  const long most = ((1L << 32) / kThreads - 1) / p.blocks;
  for (long first = 0; first < groups; first += most) {
    const long n = std::min(most, groups - first);
    rope_kernel<SIDE, MANY, TOKENS><<<(unsigned)(n * p.blocks), kThreads, 0, stream>>>(p, first);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { return e; }
  }
  return hipSuccess;
}

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
  p.blocks = (p.units + kThreads - 1) / kThreads;
  p.by_chunks = magic(p.chunks);
  const bool side = a.r.interleaved, many = a.r.n_axes > 1;
  // Four tokens a thread where that leaves enough workgroups for the CUs
  if ((long)a.tokens * p.blocks >= 8192) {
    return side ? many ? run<true, true, 4>(p, stream) : run<true, false, 4>(p, stream)
                : many ? run<false, true, 4>(p, stream) : run<false, false, 4>(p, stream);
  }
  return side ? many ? run<true, true, 1>(p, stream) : run<true, false, 1>(p, stream)
              : many ? run<false, true, 1>(p, stream) : run<false, false, 1>(p, stream);
}

}  // namespace ltx25
