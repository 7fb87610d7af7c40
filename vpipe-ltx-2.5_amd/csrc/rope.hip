// Positions rotated into queries and keys (ltx25_rope).
#include "block.h"

#include <algorithm>

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
  long tokens;       // the launch's end
  int chunks;        // a head's pieces of work
  int units;         // a token's
  uint32_t by_chunks, by_units;   // ceil(2^32 / them)
};

// n / d for n < 2^16, m = ceil(2^32 / d) (d = 1: m = 0)
__device__ __forceinline__ uint32_t divide(uint32_t n, uint32_t m) { return m == 0 ? n : __umulhi(n, m); }

// A thread turns eight channels (SIDE: pairs side by side) or twice eight, half of the rotated
// channels apart, of one token, and computes its pairs' sines itself; threads are dealt out over
// the tokens' pieces one after another, so that few heads fill waves too.
//
// Bound by memory: 8160 tokens of 32 + 32 heads of 128 by three axes, 267 MB, 54.5 us (4.9 TB/s),
// 2048 of 32 + 8 by one 8.8, changing tensors. Two and four tokens a thread, which share their
// frequencies, were no faster (50.0 and 52.4 us where one token's were 50.5; 9.2 and 10.0 for 8.6).
template <bool SIDE, bool MANY>
__global__ void __launch_bounds__(kThreads) rope_kernel(RopeParams p, long first)
{
  // the workgroup's first token and unit, and the thread's
  const uint32_t base = blockIdx.x * kThreads, units = (uint32_t)p.units;
  const uint32_t token0 = base / units, at0 = base - token0 * units + threadIdx.x;
  const uint32_t more = divide(at0, p.by_units);
  const uint32_t unit = at0 - more * units;
  const long token = first + token0 + more;
  if (token >= p.tokens) { return; }
  int head = (int)divide(unit, p.by_chunks);
  const int chunk = (int)unit - head * p.chunks;
  const int which = head >= p.heads[0] ? 1 : 0;
  head -= which ? p.heads[0] : 0;
  const bool turn = chunk * (SIDE ? 4 : 8) < p.r.pairs;
  // halves: chunks past the pairs' are those of the channels that are not rotated
  const int at = head * p.dim + (SIDE || turn ? chunk * 8 : chunk * 8 + p.r.pairs);
  const uint16_t* const in =
      (which ? p.in[1] : p.in[0]) + token * (which ? p.in_stride[1] : p.in_stride[0]) + at;
  uint16_t* const out =
      (which ? p.out[1] : p.out[0]) + token * (which ? p.out_stride[1] : p.out_stride[0]) + at;
  uint4 a = *(const uint4*)in, b;
  if (turn) {
    if constexpr (!SIDE) { b = *(const uint4*)(in + p.r.pairs); }
    const Words words = words_of<MANY>(p.r, token);
    const Pairs<SIDE ? 4 : 8> pairs = pairs_of<MANY, SIDE ? 4 : 8>(p.r, head, chunk * (SIDE ? 4 : 8));
    const Places places = places_of<MANY>(p.r, words);
    if constexpr (SIDE) {
      a = rotate_side<MANY>(a, places, pairs);
    } else {
      rotate_halves<MANY>(a, b, places, pairs);
      *(uint4*)(out + p.r.pairs) = b;
    }
  }
  *(uint4*)out = a;
}

uint32_t magic(int d) { return d <= 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / (unsigned)d); }

template <bool SIDE, bool MANY>
hipError_t run(const RopeParams& p, hipStream_t stream)
{
  // a launch has fewer than 2^32 threads
  const long most = ((1L << 32) - 2 * kThreads) / p.units;
  for (long first = 0; first < p.tokens; first += most) {
    RopeParams part = p;   // a launch's last workgroup ends with its tokens, not with all
    part.tokens = std::min(p.tokens, first + most);
    const long n = part.tokens - first;
    const unsigned blocks = (unsigned)((n * p.units + kThreads - 1) / kThreads);
    rope_kernel<SIDE, MANY><<<blocks, kThreads, 0, stream>>>(part, first);
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
  p.by_chunks = magic(p.chunks);
  p.by_units = magic(p.units);
  const bool side = a.r.interleaved, many = a.r.n_axes > 1;
  return side ? many ? run<true, true>(p, stream) : run<true, false>(p, stream)
              : many ? run<false, true>(p, stream) : run<false, false>(p, stream);
}

}  // namespace ltx25
