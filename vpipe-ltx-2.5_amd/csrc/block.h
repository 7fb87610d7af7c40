// Rotations on the device, and the launchers of the norms and rotations
// (norm.hip, rope.hip, kv_cache.hip) that their C ABI layer (capi_block.cpp) calls.
#pragma once

#include "attention.h"
#include "mx4.h"

namespace ltx25 {

constexpr int kAxesMax = 4;

// ltx25_rotation as the kernels take it
struct Rotation {
  const float* freqs = nullptr;
  const int* axes = nullptr;         // null: axis 0
  const void* positions = nullptr;   // null: a token's place in its sequence
  int pairs = 0;                     // rot_dim / 2
  int n_axes = 1;
  bool whole = false;                // positions are int32
  bool per_head = false;
  bool interleaved = false;
};

// 1 / (2 pi), and what 64 bits leave of it
constexpr double kInv2Pi = 0x1.45f306dc9c883p-3;
constexpr double kInv2PiRest = -0x1.6b01ec5417056p-57;

// A token's positions as they lie in memory, the last one again past the axes; b, c and d with
// MANY (more than one axis) alone: asked for before anything waits.
struct Words {
  uint32_t a = 0, b = 0, c = 0, d = 0;
};
template <bool MANY>
__device__ __forceinline__ Words words_of(const Rotation& r, long token)
{
  const uint32_t* const at = (const uint32_t*)r.positions + token * r.n_axes;
  Words w;
  w.a = at[0];
  if constexpr (MANY) {
    const int last = r.n_axes - 1;
    w.b = at[min(1, last)];
    w.c = at[min(2, last)];
    w.d = at[min(3, last)];
  }
  return w;
}

// The same as numbers, which 64 bits hold exactly
struct Places {
  double a = 0.0, b = 0.0, c = 0.0, d = 0.0;
};
template <bool MANY>
__device__ __forceinline__ Places places_of(const Rotation& r, const Words& w)
{
  auto number = [&](uint32_t v) { return r.whole ? (double)(int)v : (double)__uint_as_float(v); };
  Places t;
  t.a = number(w.a);
  if constexpr (MANY) {
    t.b = number(w.b);
    t.c = number(w.c);
    t.d = number(w.d);
  }
  return t;
}

// A pair's frequency in turns (divided by 2 pi): a number of 64 bits and what that leaves. One
// alone is off by 2^-53 of the turns: 2^-18 radians at position 2^20 of a frequency of 15708.
struct Freq {
  double turns;
  float rest;
};
__device__ __forceinline__ Freq freq_of(float f)
{
  const double freq = (double)f, turns = freq * kInv2Pi;
  return {turns, (float)fma(freq, kInv2PiRest, fma(freq, kInv2Pi, -turns))};
}

// The sine and cosine of one pair's angle. Whole turns are taken off the product of position and
// frequency in 64 bits before it is rounded; what is left, and the share of the frequency's rest (a
// sixteenth of a turn at 2^52 radians), are good to 2^-25 turns in 32. They go to the hardware's sine
// and cosine, whose argument is in turns (off by at most 2^-22.9).
template <bool MANY>
__device__ __forceinline__ void sin_cos(const Places& t, const Freq& freq, int axis, float& sn,
                                        float& cs)
{
  double at = t.a;
  if constexpr (MANY) {
    // As values: of members the compiler selects the addresses and keeps them in LDS, or in
    // scratch memory, and reads the workgroup's shape from the dispatch packet, which lies in the
    // host's memory (128 tokens by three axes 13 us, so 3.1).
    const double a = +t.a, b = +t.b, c = +t.c, d = +t.d;
    const double low = axis == 1 ? +b : +a, high = axis == 2 ? +c : +d;
    at = axis <= 1 ? +low : +high;
  }
  const double whole = rint(at * freq.turns);
  const float left = fmaf((float)at, freq.rest, (float)fma(at, freq.turns, -whole));
  sn = __builtin_amdgcn_sinf(left);
  cs = __builtin_amdgcn_cosf(left);
}

// N consecutive pairs' frequencies and axes (N 4 or 8, the first a multiple of 4)
template <int N>
struct Pairs {
  Freq freq[N];
  int axis[N];
};
template <bool MANY, int N>
__device__ __forceinline__ Pairs<N> pairs_of(const Rotation& r, int head, int first)
{
  Pairs<N> p;
  const long at = (long)(r.per_head ? head : 0) * r.pairs + first;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const f32x4 f = *(const f32x4*)(r.freqs + at + i);
    const i32x4 a = MANY && r.axes != nullptr ? *(const i32x4*)(r.axes + at + i) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      p.freq[i + k] = freq_of(f[k]);
      p.axis[i + k] = min(a[k], r.n_axes - 1);
    }
  }
  return p;
}

// Two bf16 (low, high half) as floats
__device__ __forceinline__ float low_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_f32(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// A pair (a, b) turned: a cos - b sin, b cos + a sin
__device__ __forceinline__ float turned_a(float a, float b, float sn, float cs)
{
  return fmaf(a, cs, -(b * sn));
}
__device__ __forceinline__ float turned_b(float a, float b, float sn, float cs)
{
  return fmaf(b, cs, a * sn);
}

// Eight channels of pairs side by side, turned by four frequencies
template <bool MANY, int N>
__device__ __forceinline__ uint4 rotate_side(uint4 x, const Places& t, const Pairs<N>& p)
{
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float sn, cs;
    sin_cos<MANY>(t, p.freq[i], p.axis[i], sn, cs);
    const float a = low_f32(w[i]), b = high_f32(w[i]);
    w[i] = pack_bf16x2(turned_a(a, b, sn, cs), turned_b(a, b, sn, cs));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight pairs, their first channels in xa and their second in xb
template <bool MANY>
__device__ __forceinline__ void rotate_halves(uint4& xa, uint4& xb, const Places& t,
                                              const Pairs<8>& p)
{
  uint32_t a[4] = {xa.x, xa.y, xa.z, xa.w}, b[4] = {xb.x, xb.y, xb.z, xb.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float s0, c0, s1, c1;
    sin_cos<MANY>(t, p.freq[2 * i], p.axis[2 * i], s0, c0);
    sin_cos<MANY>(t, p.freq[2 * i + 1], p.axis[2 * i + 1], s1, c1);
    const float a0 = low_f32(a[i]), a1 = high_f32(a[i]), b0 = low_f32(b[i]), b1 = high_f32(b[i]);
    a[i] = pack_bf16x2(turned_a(a0, b0, s0, c0), turned_a(a1, b1, s1, c1));
    b[i] = pack_bf16x2(turned_b(a0, b0, s0, c0), turned_b(a1, b1, s1, c1));
  }
  xa = make_uint4(a[0], a[1], a[2], a[3]);
  xb = make_uint4(b[0], b[1], b[2], b[3]);
}

// The same where one lane has eight pairs' first channels and another, `from`, their second (or
// the other way round, `second`): the first takes four of the pairs and the second the other
// four (`p`, theirs), and each gives the other what is its. Every lane takes part; `there`, which
// both agree on: x is turned.
template <bool MANY>
__device__ __forceinline__ uint4 rotate_half(uint4 x, int from, bool second, bool there,
                                             const Places& t, const Pairs<4>& p)
{
  const uint32_t given[2] = {second ? x.x : x.z, second ? x.y : x.w};
  const uint32_t kept[2] = {second ? x.z : x.x, second ? x.w : x.y};
  uint32_t first_w[2], second_w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t got = (uint32_t)__shfl((int)given[i], from);
    first_w[i] = second ? got : kept[i];
    second_w[i] = second ? kept[i] : got;
  }
  if (there) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s0, c0, s1, c1;
      sin_cos<MANY>(t, p.freq[2 * i], p.axis[2 * i], s0, c0);
      sin_cos<MANY>(t, p.freq[2 * i + 1], p.axis[2 * i + 1], s1, c1);
      const float a0 = low_f32(first_w[i]), a1 = high_f32(first_w[i]);
      const float b0 = low_f32(second_w[i]), b1 = high_f32(second_w[i]);
      first_w[i] = pack_bf16x2(turned_a(a0, b0, s0, c0), turned_a(a1, b1, s1, c1));
      second_w[i] = pack_bf16x2(turned_b(a0, b0, s0, c0), turned_b(a1, b1, s1, c1));
    }
  }
  uint32_t mine[2], his[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    mine[i] = second ? second_w[i] : first_w[i];
    his[i] = (uint32_t)__shfl((int)(second ? first_w[i] : second_w[i]), from);
  }
  return second ? make_uint4(his[0], his[1], mine[0], mine[1])
                : make_uint4(mine[0], mine[1], his[0], his[1]);
}

// ---- launchers --------------------------------------------------------------

struct RopeArgs {
  Rotation r;
  const uint16_t* in[2] = {nullptr, nullptr};   // queries, keys
  uint16_t* out[2] = {nullptr, nullptr};
  int64_t in_stride[2] = {0, 0}, out_stride[2] = {0, 0};
  int heads[2] = {0, 0};
  int head_dim = 0, tokens = 0;
};
hipError_t launch_rope(const RopeArgs& a, hipStream_t stream);

hipError_t launch_kv_append_rope(const CacheArgs& c, const uint16_t* k, const uint16_t* v,
                                 int64_t ks, int64_t vs, const int* cu, const int* start,
                                 const Rotation& r, int batch, int total, hipStream_t stream);

struct NormArgs {
  const void* x = nullptr;
  const uint16_t* y = nullptr;
  void* x_out = nullptr;
  const void* after = nullptr;    // post_weight
  const void* gate = nullptr;
  const void* weight = nullptr;
  const void* scale = nullptr;
  const void* shift = nullptr;
  const int* rows = nullptr;
  uint16_t* out = nullptr;
  Mx4Args q;                      // codes null: out is bf16 (or none)
  int64_t xs = 0, xos = 0, ys = 0, ms = 0, os = 0;
  int width = 0, tokens = 0, mod_rows = 0, run = 1;   // run: tokens of a modulation row
  bool layer = false, wide = false, mod_wide = false, weight_wide = false;
  float eps = 0.0f, alpha = 1.0f;
};
hipError_t launch_norm(const NormArgs& a, hipStream_t stream);

}  // namespace ltx25
