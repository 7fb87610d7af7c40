// Norms fused with the gate, the residual and the modulation (ltx25_block_norm,
// ltx25_block_norm_mx4).
#include "block.h"

#include <algorithm>
#include <type_traits>

namespace ltx25 {
namespace {

// 8 values of a tensor as they lie in memory: 16 bytes of bf16, 32 of f32
template <bool WIDE>
struct Raw {
  uint4 w[WIDE ? 2 : 1];
};
template <bool WIDE>
__device__ __forceinline__ Raw<WIDE> fetch8(const void* p, long at)
{
  const uint4* const q = (const uint4*)((const char*)p + at * (WIDE ? 4 : 2));
  Raw<WIDE> r;
  r.w[0] = q[0];
  if constexpr (WIDE) { r.w[1] = q[1]; }
  return r;
}
template <bool WIDE>
__device__ __forceinline__ void values8(const Raw<WIDE>& r, float (&v)[8])
{
#pragma unroll
  for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
    const uint32_t a[4] = {r.w[h].x, r.w[h].y, r.w[h].z, r.w[h].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (WIDE) {
        v[4 * h + i] = __uint_as_float(a[i]);
      } else {
        v[2 * i] = low_f32(a[i]);
        v[2 * i + 1] = high_f32(a[i]);
      }
    }
  }
}
__device__ __forceinline__ void load8(const void* p, bool wide, long at, float (&v)[8])
{
  if (wide) {
    values8(fetch8<true>(p, at), v);
  } else {
    values8(fetch8<false>(p, at), v);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8])
{
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}

// WAVES waves hold a token, CH chunks of eight values a lane: lane l of wave w has the
// chunks w * 64 + l + i * 64 * WAVES. A single wave's tokens share a workgroup of four, and
// of narrow ones, of LANES lanes each (a head's channels), several share a wave.
//
// Sums in f32, the mean taken off before the squares are added; where a sum leaves f32's
// range the values are taken 2^-80 times as large, which leaves every square that counts
// inside it.
//
// WIDE: x is f32. EARLY: what multiplies and shifts is bf16 and asked for before the sums. LONE:
// there is no y, whose registers let more tokens be in flight (8160 x 4096 into 4 bits 22 us and, as
// with one, 25; 4096 x 12288 45 and 51).
//
// Bound by memory: 8192 tokens of 4096 with a branch, gate and modulation 48.9 us (268 MB, 5.5
// TB/s), post-normed and with means 53.7, 4-bit output 47.4 (219 MB).
template <int WAVES, int CH, bool WIDE, bool EARLY, int LANES, bool LONE>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) norm_kernel(NormArgs p, long first)
{
  static_assert(LANES == 64 || WAVES == 1, "lanes of a wave");
  __shared__ float part[4][WAVES];
  const int lane = threadIdx.x & (LANES - 1);
  const int wave = WAVES == 1 ? 0 : (int)(threadIdx.x >> 6);
  // Coded rows lie four to 64 bytes and 16 to a tile: 16 tokens go to workgroups of one XCD
  // (every eighth), whose cache puts their lines together.
  long place = blockIdx.x;
  if (p.q.codes != nullptr && (place | 127) < (long)gridDim.x) {
    place = (place & ~127L) + (place & 7) * 16 + ((place >> 3) & 15);
  }
  const long token = first + (WAVES == 1 ? place * (256 / LANES) + threadIdx.x / LANES : place);
  if (token >= p.tokens) { return; }
  int turn = 0;
  auto total = [&](float v) {
#pragma unroll
    for (int i = 1; i < LANES; i *= 2) { v += __shfl_xor(v, i); }
    if constexpr (WAVES > 1) {
      // the next sum's slots are others: its writers do not meet this one's readers
      float* const at = part[turn & 3];
      ++turn;
      if (lane == 0) { at[wave] = v; }
      __syncthreads();
      v = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) { v += at[w]; }
    }
    return v;
  };
  int col[CH];
  bool in[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    col[i] = (i * 64 * WAVES + wave * 64 + lane) * 8;
    in[i] = col[i] < p.width;
  }
  const float over = 1.0f / (float)p.width;
  // v -> (v - mean) / sqrt(mean square + eps), zeros past the width kept
  auto normalise = [&](float (&v)[CH][8]) {
    auto mean_of = [&](float unit) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) { s = fmaf(v[i][k], unit, s); }
      }
      return total(s) * over;
    };
    // The values times `unit` less `mean`, and their mean square
    auto square_of = [&](float unit, float mean) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (!in[i]) { continue; }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float d = fmaf(v[i][k], unit, -mean);
          s = fmaf(d, d, s);
        }
      }
      return total(s) * over;
    };
    float mean = 0.0f, unit = 1.0f, square;
    if (p.layer) {
      mean = mean_of(1.0f);
      square = square_of(1.0f, mean) + p.eps;
    } else {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) { s = fmaf(v[i][k], v[i][k], s); }
      }
      square = total(s) * over + p.eps;
    }
    if (!(square < INFINITY)) {
      unit = 0x1p-80f;
      mean = p.layer ? mean_of(unit) : 0.0f;
      square = square_of(unit, mean) + fmaxf(p.eps * 0x1p-80f * 0x1p-80f, 0x1p-126f);
    }
    const float rs = 1.0f / sqrtf(square);
    if (p.layer || unit != 1.0f) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) { v[i][k] = fmaf(v[i][k], unit, -mean) * rs; }
      }
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) { v[i][k] *= rs; }
      }
    }
  };

  long row = 0;
  if (p.mod_rows > 0) {
    row = p.rows != nullptr ? clampi(p.rows[token], 0, p.mod_rows - 1) : token / p.run;
    row *= p.ms;
  }
  // lanes past the width read its last values again
  int from[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) { from[i] = min(col[i], p.width - 8); }
  Raw<WIDE> rx[CH];
  Raw<false> ry[CH], after[CH], gate[CH], weight[CH], scale[CH], shift[CH];
  auto fetch = [&](auto& to, const void* t, long at) {
    constexpr bool kWide = std::is_same_v<decltype(to), Raw<true>(&)[CH]>;
    if (t == nullptr) { return; }
#pragma unroll
    for (int i = 0; i < CH; ++i) { to[i] = fetch8<kWide>(t, at + from[i]); }
  };
  fetch(rx, p.x, token * p.xs);
  if constexpr (!LONE) { fetch(ry, p.y, token * p.ys); }
  if constexpr (EARLY && !LONE) {
    fetch(after, p.after, 0);
    fetch(gate, p.gate, row);
  }
  if constexpr (EARLY) {
    fetch(weight, p.weight, 0);
    fetch(scale, p.scale, row);
    fetch(shift, p.shift, row);
  }
  // chunk i of one of them
  auto values = [&](const Raw<false>& early, const void* t, bool wide, long at, float (&m)[8]) {
    if constexpr (EARLY) {
      values8(early, m);
    } else {
      load8(t, wide, at, m);
    }
  };
  float x[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) { x[i][k] = 0.0f; }
    if (in[i]) { values8(rx[i], x[i]); }
  }
  if (!LONE && p.y != nullptr) {
    float y[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) { y[i][k] = 0.0f; }
      if (in[i]) { values8(ry[i], y[i]); }
    }
    if (p.after != nullptr) { normalise(y); }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (!in[i]) { continue; }
      float m[8];
      if (p.after != nullptr) {
        values(after[i], p.after, p.weight_wide, col[i], m);
#pragma unroll
        for (int k = 0; k < 8; ++k) { y[i][k] *= m[k]; }
      }
      if (p.gate != nullptr) {
        values(gate[i], p.gate, p.mod_wide, row + col[i], m);
#pragma unroll
        for (int k = 0; k < 8; ++k) { y[i][k] *= m[k]; }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) { x[i][k] = fmaf(p.alpha, x[i][k], y[i][k]); }
      if constexpr (WIDE) {
        f32x4* const o = (f32x4*)((float*)p.x_out + token * p.xos + col[i]);
        o[0] = f32x4{x[i][0], x[i][1], x[i][2], x[i][3]};
        o[1] = f32x4{x[i][4], x[i][5], x[i][6], x[i][7]};
      } else {
        *(uint4*)((uint16_t*)p.x_out + token * p.xos + col[i]) = pack8(x[i]);
      }
    }
  }
  if (p.out == nullptr && p.q.codes == nullptr) { return; }
  normalise(x);
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (in[i]) {
      float m[8];
      if (p.weight != nullptr) {
        values(weight[i], p.weight, p.weight_wide, col[i], m);
#pragma unroll
        for (int k = 0; k < 8; ++k) { x[i][k] *= m[k]; }
      }
      if (p.scale != nullptr) {
        values(scale[i], p.scale, p.mod_wide, row + col[i], m);
#pragma unroll
        for (int k = 0; k < 8; ++k) { x[i][k] = fmaf(x[i][k], m[k], x[i][k]); }
      }
      if (p.shift != nullptr) {
        values(shift[i], p.shift, p.mod_wide, row + col[i], m);
#pragma unroll
        for (int k = 0; k < 8; ++k) { x[i][k] += m[k]; }
      }
      if (p.out != nullptr) { *(uint4*)(p.out + token * p.os + col[i]) = pack8(x[i]); }
    }
    if (p.q.codes != nullptr) {
      // a block's four lanes are in or out together: the width is a multiple of 32; blocks past
      // it in the row's last tiles are zeros
      const int block = col[i] >> 5, slices = mx4_slices(p.width), spans = mx4_spans(p.width);
      uint32_t scale = 0, codes = 0;
      if (in[i]) { codes = mx4_code_quad(x[i], scale); }
      if (block < slices * 4) {
        *(uint32_t*)(p.q.codes + ((token >> 4) * slices + (block >> 2)) * kMx4CodeTile +
                     mx4_code_at((int)(token & 15), block) + (lane & 3) * 4) = codes;
      }
      if ((lane & 3) == 0 && block < spans * 16) {
        p.q.scales[((token >> 4) * spans + (block >> 4)) * kMx4Tile +
                   mx4_scale_at((int)(token & 15), block)] = (uint8_t)scale;
      }
    }
  }
}

template <int WAVES, int CH, bool WIDE, bool EARLY, int LANES, bool LONE>
hipError_t run(const NormArgs& a, hipStream_t stream)
{
  // a launch has fewer than 2^32 threads; whole runs of 128 workgroups
  constexpr int kThreads = WAVES == 1 ? 256 : 64 * WAVES, kTokens = WAVES == 1 ? 256 / LANES : 1;
  constexpr long kMost = (((1L << 32) / kThreads - 1) & ~127L) * kTokens;
  // LDS that nothing uses, for four workgroups a CU and no fifth: where a token has much to move and
  // one sum, more of them at once take the memory longer. By the bytes of its x and y, 16 KB or more
  // (with gate and modulation; in fours, and in fives): 8160 x 4096 48.2 us and 48.6, into 4 bits
  // 46.4 and 46.5, 32768 tokens 178 and 182; of f32 x 72.1 and 73.4, 32768 tokens 273 and 280, 3080
  // wide 57.1 and 60.9, into 4 bits 3584 wide 59.9 and 64.9 (2048 x 3080 18.1 and 16.0). Below:
  // 3584 wide 45.1 and 44.2, into 4 bits 43.6 and 41.8, f32 modulations 53.4 and 51.2; 3840 wide
  // 47.8 and 47.7, 45.6 and 45.0, 57.6 and 55.3. Post-normed with means, four sums, 8160 x 4096 55.2
  // and 53.9.
  const bool four = WAVES == 4 && CH == 2 && !LONE && a.after == nullptr && !a.layer &&
                    (WIDE ? 6 : 4) * a.width >= 16 << 10;
  const size_t spare = four ? 36 << 10 : 0;
  for (long first = 0; first < a.tokens; first += kMost) {
    const long n = std::min(kMost, a.tokens - first);
    norm_kernel<WAVES, CH, WIDE, EARLY, LANES, LONE>
        <<<(unsigned)((n + kTokens - 1) / kTokens), kThreads, spare, stream>>>(a, first);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { return e; }
  }
  return hipSuccess;
}

template <int WAVES, int CH, int LANES = 64>
hipError_t run(const NormArgs& a, hipStream_t stream)
{
  constexpr bool kEarly = WAVES * CH < 24;   // wider ones with a y: 10240 72.8 us, late 57.9
  const bool narrow = !a.mod_wide && !a.weight_wide;
  if (narrow && a.y == nullptr) {
    return a.wide ? run<WAVES, CH, true, true, LANES, true>(a, stream)
                  : run<WAVES, CH, false, true, LANES, true>(a, stream);
  }
  if (narrow && kEarly) {
    return a.wide ? run<WAVES, CH, true, kEarly, LANES, false>(a, stream)
                  : run<WAVES, CH, false, kEarly, LANES, false>(a, stream);
  }
  return a.wide ? run<WAVES, CH, true, false, LANES, false>(a, stream)
                : run<WAVES, CH, false, false, LANES, false>(a, stream);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, hipStream_t stream)
{
  const bool coded = a.q.codes != nullptr;
  // the padded blocks of a 4-bit output's last span are the lanes' past the width, too
  const int width = coded ? (a.width + 511) / 512 * 512 : a.width;
  // Few idle lanes, then few waves to wait for (with a branch, gate and modulation, in the form
  // taken and in the next larger: 65536 tokens of 128 13 us for 27, 30840 of 1088 50 for 57, 13107
  // of 2560 52 for 57, 6553 of 5120 52 for 60).
  auto fits = [&](int waves, int chunks, int lanes = 64) {
    return width <= 8 * lanes * waves * chunks;
  };
  if (fits(1, 1, 8)) { return run<1, 1, 8>(a, stream); }
  if (fits(1, 1, 16)) { return run<1, 1, 16>(a, stream); }
  if (fits(1, 1, 32)) { return run<1, 1, 32>(a, stream); }
  if (fits(1, 1)) { return run<1, 1>(a, stream); }
  if (fits(1, 2)) { return run<1, 2>(a, stream); }
  if (fits(3, 1)) { return run<3, 1>(a, stream); }
  if (fits(4, 1)) { return run<4, 1>(a, stream); }
  if (fits(3, 2)) { return run<3, 2>(a, stream); }
  if (fits(4, 2)) { return run<4, 2>(a, stream); }
  if (fits(4, 3)) { return run<4, 3>(a, stream); }
  if (fits(8, 2)) { return run<8, 2>(a, stream); }
  if (fits(8, 3)) { return run<8, 3>(a, stream); }
  return run<8, 4>(a, stream);
}

}  // namespace ltx25
