// The paged cache of 8-bit keys and values: appending to it, reading it back,
// and attention over it (ltx25_kv_append, ltx25_kv_read,
// ltx25_attention_cached).
#include "block.h"

#include <algorithm>
#include <climits>

namespace ltx25 {
namespace {

constexpr int kThreads = 256;

struct CacheView {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  const int* table;
  int pages, pl, kv_heads, table_stride;   // pl: log2 of a page's tokens
};

// 8 codes -> 8 bf16, exactly
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t a, uint32_t b)
{
  auto f = [](uint32_t w, int i) { return (float)(int8_t)((w >> (8 * i)) & 0xffu); };
  uint4 r;
  r.x = pack_bf16x2(f(a, 0), f(a, 1));
  r.y = pack_bf16x2(f(a, 2), f(a, 3));
  r.z = pack_bf16x2(f(b, 0), f(b, 1));
  r.w = pack_bf16x2(f(b, 2), f(b, 3));
  return as_bf16x8(r);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f16x8 as_f16x8(uint4 v) { return __builtin_bit_cast(f16x8, v); }
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b)
{
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// 8 codes -> 8 f16, exactly: 0x64 before a byte u makes 1024 + u
__device__ __forceinline__ f16x8 codes_f16(uint32_t a, uint32_t b)
{
  auto two = [](uint32_t w, uint32_t bytes) {
    const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, bytes);
    const f16x2 y = __builtin_bit_cast(f16x2, x) - f16x2{1152, 1152};
    return __builtin_bit_cast(uint32_t, y);
  };
  return as_f16x8(make_uint4(two(a, 0x04010400u), two(a, 0x04030402u), two(b, 0x04010400u),
                             two(b, 0x04030402u)));
}

// rint(x / s) within +-127; 0 for s = 0 and for a NaN
__device__ __forceinline__ int quantize(float x, float s)
{
  const float r = rintf(x / s);
  return s > 0.0f && r == r ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0;
}

// Four codes as bytes. `rs` > 0 is 1 / s, correctly rounded, for s well inside the
// normal range and |x| at most 127 s: the quotient is x rs made better twice by its
// exact remainder, after which it is the correctly rounded one (after the first
// step it is off by less than a unit of its last place, from where the second is
// Markstein's), in five operations for the division's ten; quotients too small for
// an exact remainder are far below 1/2. Adding 3 * 2^22 rounds to even with the
// code in the low byte. rs 0: any s and x.
__device__ __forceinline__ uint32_t quantize4(const float (&x)[4], float s, float rs)
{
  uint32_t c[4];
  if (rs > 0.0f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float q = x[i] * rs;
      q = fmaf(fmaf(-q, s, x[i]), rs, q);
      q = fmaf(fmaf(-q, s, x[i]), rs, q);
      c[i] = __float_as_uint(q + 12582912.0f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = (uint32_t)quantize(x[i], s); }
  }
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
  return lo | hi;
}

// Four words of four bytes each, turned: word i of the result is byte i of the four
__device__ __forceinline__ void turn4(uint32_t (&w)[4])
{
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);   // 0.0 1.0 0.1 1.1
  const uint32_t b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);   // 0.2 1.2 0.3 1.3
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// ---- append, read -----------------------------------------------------------

struct MoveParams {
  CacheView c;
  const uint16_t* k_in;
  const uint16_t* v_in;
  uint16_t* k_out;
  uint16_t* v_out;
  long kstride, vstride;
  const int* cu;
  const int* start;
  int batch, total;
};

// One page of one sequence that a call touches: tokens lo .. hi - 1 of it are
// packed tokens first + lo ...
struct Span {
  const int* id;   // where the page's id is; null past the table
  int lo, hi;
  long first;
  long place;      // of the page's token 0 in its sequence
};

// The unit blockIdx.x of all sequences' touched pages; false past the last.
__device__ __forceinline__ bool find_span(const MoveParams& p, Span& s)
{
  constexpr int kFar = 1 << 30;
  int c0 = 0, n = 0, at = 0;
  auto count = [&](int b) {
    c0 = clampi(p.cu[b], 0, p.total);
    n = clampi(p.cu[b + 1], c0, p.total) - c0;
    at = clampi(p.start[b], 0, kFar);
    return n > 0 ? ((at + (n - 1)) >> p.c.pl) - (at >> p.c.pl) + 1 : 0;
  };
  int seq = 0, place = 0, from = 0;
  if (!find_unit((int)blockIdx.x, p.batch, count, seq, place, from)) { return false; }
  c0 = __builtin_amdgcn_readlane(c0, from);
  n = __builtin_amdgcn_readlane(n, from);
  at = __builtin_amdgcn_readlane(at, from);
  const int page = (at >> p.c.pl) + place;
  const long t0 = (long)page << p.c.pl;   // the page's first token
  s.lo = (int)(max((long)at, t0) - t0);
  s.hi = (int)(min((long)at + n, t0 + (1 << p.c.pl)) - t0);
  s.first = c0 + (t0 - at);
  s.place = t0;
  s.id = page < p.c.table_stride ? p.c.table + (long)seq * p.c.table_stride + page : nullptr;
  return true;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u16x2 max_magnitudes(u16x2 top, uint4 v)
{
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  }
  return top;
}

// The largest finite magnitude of 8 values, as the bits of a bf16
__device__ __forceinline__ uint32_t max_finite(uint32_t top, uint4 v)
{
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = (w[i >> 1] >> (16 * (i & 1))) & 0x7fffu;
    top = a < 0x7f80u ? max(top, a) : top;
  }
  return top;
}

// 8 values' codes
__device__ __forceinline__ uint2 quantize8(uint4 x, float s, float rs)
{
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = bf16_to_f32((uint16_t)(w[2 * h + (k >> 1)] >> (16 * (k & 1))));
    }
    c[h] = quantize4(v, s, rs);
  }
  return make_uint2(c[0], c[1]);
}

// A workgroup quantizes one page's new tokens of one kv head: their keys
// (blockIdx.z 0) or their values (1). A thread holds four tokens of 8 channels, so
// that its codes are whole words both by token and, turned, by channel; of a few
// tokens (a decode step's one) it holds one token's 8 channels, since a quarter or
// less of that work is then there to do (one token each of 64 sequences, 8 heads of
// 128: 5.7 us, 8.4 by fours).
//
// Bound by memory where there is much to do: 8192 tokens of 8 heads of 128, 50 MB read
// and written, 17.0 us on changing tensors (3.0 TB/s; a page's first code waits for all its
// values), 13.4 on the same ones again.
//
// ROPE: the keys are turned in registers as they arrive and rounded to bf16, and from there on
// are the keys of a plain append. Pairs half of the rotated channels apart meet by exchanges
// between two lanes of one token, each of which turns half of their pairs (all of them, its own
// channels alone: half a microsecond more). 8192 tokens of 8 heads of 128 19.3 us on changing
// tensors (pairs side by side 18.1, by three axes 21.0), 17.5 on the same ones again (15.6, 18.2):
// every head's workgroup computes its tokens' sines.
// ROPE 2: positions of several axes.
template <int D, int ROPE = 0>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(MoveParams p, Rotation rot)
{
  constexpr int kMaxP = 128;
  constexpr int kPer = D / 8;   // 16-byte pieces of a token
  constexpr int kHeld = kMaxP / 4 * kPer / kThreads;
  constexpr int kFew = kThreads / kPer;
  __shared__ uint32_t wave_top[kThreads / 64];
  __shared__ __attribute__((aligned(16))) uint8_t turned[D * (kMaxP + 4)];

  Span sp;
  if (!find_span(p, sp) || sp.id == nullptr) { return; }
  const int tid = threadIdx.x;
  const int g = blockIdx.y;
  const bool values = blockIdx.z != 0;
  const int P = 1 << p.c.pl;
  const uint16_t* const x = (values ? p.v_in : p.k_in) + g * D;
  const long stride = values ? p.vstride : p.kstride;
  const bool few = sp.hi - sp.lo <= kFew;

  // the tokens are asked for beside the page's id
  const int pid = *sp.id;
  const int quad0 = sp.lo >> 2;
  const int pieces = few ? (sp.hi - sp.lo) * kPer : (((sp.hi + 3) >> 2) - quad0) * kPer;
  // The lane's piece of a key is the same in all its tokens, so are its pairs. A key of the
  // page's token `tok`: every lane of a wave takes part.
  constexpr bool kMany = ROPE == 2;
  const int piece = tid % kPer;
  const int apart = ROPE && !rot.interleaved ? rot.pairs / 8 : 0;   // pieces between a pair's two
  const bool second = apart > 0 && piece >= apart;
  const bool turning = ROPE && piece * 8 < 2 * rot.pairs;
  // four of the pairs: those of the piece's channels, or half of those that it shares
  Pairs<4> pairs;
  if (ROPE && !values && turning) {
    const int first = rot.interleaved ? piece * 4 : (piece - (second ? apart : 0)) * 8 + second * 4;
    pairs = pairs_of<kMany, 4>(rot, g, first);
  }
  const bool given = kMany || rot.positions != nullptr;
  auto there = [&](int tok) { return turning && tok >= sp.lo && tok < sp.hi; };
  auto words = [&](int tok) {
    return given && there(tok) ? words_of<kMany>(rot, sp.first + tok) : Words();
  };
  auto rotate = [&](uint4& w, int tok, const Words& at) {
    const bool on = there(tok);
    Places t;
    if (given) {
      t = places_of<kMany>(rot, at);
    } else {
      t.a = (double)(uint32_t)(sp.place + tok);   // below 2^31 (find_span)
    }
    if (!rot.interleaved) {
      const int from = (tid & 63) + (second ? -apart : apart);
      // (of a channel that is not turned the partner may be any lane)
      const uint4 r = rotate_half<kMany>(w, from & 63, second, on, t, pairs);
      if (turning) { w = r; }
    } else if (on) {
      w = rotate_side<kMany>(w, t, pairs);
    }
  };
  uint4 held[kHeld][4];
  Words at_words[ROPE ? kHeld : 1][4];
  uint32_t top = 0;
  bool odd = false;   // an infinity or a NaN among the lane's values
  if (few) {
    held[0][0] = make_uint4(0, 0, 0, 0);
    if (ROPE && !values) { at_words[0][0] = words(sp.lo + tid / kPer); }
    if (tid < pieces) {
      held[0][0] = *(const uint4*)(x + (sp.first + sp.lo + tid / kPer) * stride + (tid % kPer) * 8);
    }
    if constexpr (ROPE) {
      if (!values) { rotate(held[0][0], sp.lo + tid / kPer, at_words[0][0]); }
    }
    const u16x2 tops = max_magnitudes(u16x2{0, 0}, held[0][0]);
    top = max((uint32_t)tops[0], (uint32_t)tops[1]);
    odd = top >= 0x7f80u;
    if (odd) { top = max_finite(0, held[0][0]); }
  } else {
    u16x2 tops = {0, 0};
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = tid + i * kThreads;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = (quad0 + at / kPer) * 4 + j;
        held[i][j] = make_uint4(0, 0, 0, 0);
        if (at < pieces && tok >= sp.lo && tok < sp.hi) {
          held[i][j] = *(const uint4*)(x + (sp.first + tok) * stride + (at % kPer) * 8);
        }
        if (ROPE && !values) { at_words[i][j] = words(tok); }
      }
    }
    if constexpr (ROPE) {
      if (!values) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            rotate(held[i][j], (quad0 + (tid + i * kThreads) / kPer) * 4 + j, at_words[i][j]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) { tops = max_magnitudes(tops, held[i][j]); }
    }
    top = max((uint32_t)tops[0], (uint32_t)tops[1]);
    odd = top >= 0x7f80u;
    if (odd) {
      top = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { top = max_finite(top, held[i][j]); }
      }
    }
  }
  if (pid < 0 || pid >= p.c.pages) { return; }
  int8_t* const codes = (values ? p.c.v : p.c.k) + (((long)pid * p.c.kv_heads + g) << p.c.pl) * D;
  float* const scale = (values ? p.c.vs : p.c.ks) + (long)pid * p.c.kv_heads + g;
  const float s0 = sp.lo > 0 ? *scale : 0.0f;
  top = wave_max(top);
  if ((tid & 63) == 0) { wave_top[tid >> 6] = top; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) { top = max(top, wave_top[w]); }
  const float s1 = fmaxf(s0, bf16_to_f32((uint16_t)top) / 127.0f);
  const bool again = sp.lo > 0 && s1 > s0;   // the tokens before these: new codes
  if (tid == 0) { *scale = s1; }
  const bool easy = s1 >= 0x1p-90f && s1 <= 0x1p90f;
  const float rs = easy ? 1.0f / s1 : 0.0f;
  const float my_rs = odd ? 0.0f : rs;

  // an old code's value is at most 127 s0, so quantize4's bound holds for it too
  auto requantize = [&](uint32_t w) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = (float)(int8_t)((w >> (8 * j)) & 0xffu) * s0; }
    return quantize4(v, s1, rs);
  };
  if (few) {
    if (tid < pieces) {
      const int tok = sp.lo + tid / kPer, d0 = (tid % kPer) * 8;
      const uint2 c = quantize8(held[0][0], s1, my_rs);
      if (values) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          turned[(d0 + k) * (P + 4) + tok] = (uint8_t)((k < 4 ? c.x : c.y) >> (8 * (k & 3)));
        }
      } else {
        *(uint2*)(codes + tok * D + d0) = c;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = tid + i * kThreads;
      if (at < pieces) {
        const int tok0 = (quad0 + at / kPer) * 4, d0 = (at % kPer) * 8;
        uint32_t c[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint2 q = quantize8(held[i][j], s1, my_rs);
          c[0][j] = q.x;
          c[1][j] = q.y;
        }
        if (values) {
          turn4(c[0]);
          turn4(c[1]);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            *(uint32_t*)(turned + (d0 + k) * (P + 4) + tok0) = c[k >> 2][k & 3];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (tok0 + j >= sp.lo && tok0 + j < sp.hi) {
              *(uint2*)(codes + (tok0 + j) * D + d0) = make_uint2(c[0][j], c[1][j]);
            }
          }
        }
      }
    }
  }
  if (!values) {
    if (again) {
      for (int at = tid; at < sp.lo * D / 16; at += kThreads) {
        uint4 w = *(const uint4*)(codes + at * 16);
        w = make_uint4(requantize(w.x), requantize(w.y), requantize(w.z), requantize(w.w));
        *(uint4*)(codes + at * 16) = w;
      }
    }
    return;
  }
  __syncthreads();
  // values: a channel's 16 tokens at a time, from the first that changes
  const int t0 = again ? 0 : sp.lo & ~15;
  const int runs = (sp.hi - t0 + 15) / 16;
  for (int at = tid; at < D * runs; at += kThreads) {
    const int d = at / runs, tok = t0 + (at % runs) * 16;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (tok < sp.lo) {
      w = *(const uint4*)(codes + d * P + tok);
      if (again) {
        w = make_uint4(requantize(w.x), requantize(w.y), requantize(w.z), requantize(w.w));
      }
    }
    uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int first = tok + 4 * j;
      if (first + 3 >= sp.lo && first < sp.hi) {
        const uint32_t n = *(const uint32_t*)(turned + d * (P + 4) + first);
        // bytes of tokens lo .. hi - 1 are the new ones
        const int skip = max(sp.lo - first, 0), end = min(sp.hi - first, 4);
        const uint32_t mask = (0xffffffffu << (8 * skip)) & (0xffffffffu >> (8 * (4 - end)));
        r[j] = (r[j] & ~mask) | (n & mask);
      }
    }
    *(uint4*)(codes + d * P + tok) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// A workgroup reads one page's span of one kv head back as bf16; values are turned in
// LDS. Bound by memory: 8192 tokens of 8 heads of 128, 50 MB, 11 us (4.6 TB/s).
template <int D>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(MoveParams p)
{
  constexpr int kMaxP = 128;
  constexpr int kPer = D / 8;
  __shared__ __attribute__((aligned(16))) uint8_t turned[kMaxP * (D + 4)];
  Span sp;
  if (!find_span(p, sp)) { return; }
  int pid = sp.id == nullptr ? -1 : *sp.id;
  if (pid >= p.c.pages) { pid = -1; }
  const int tid = threadIdx.x;
  const int g = blockIdx.y;
  const bool values = blockIdx.z != 0;
  const int P = 1 << p.c.pl;
  uint16_t* const y = (values ? p.v_out : p.k_out) + g * D;
  const long stride = values ? p.vstride : p.kstride;
  const long block = (long)(pid < 0 ? 0 : pid) * p.c.kv_heads + g;
  const int8_t* const codes = (values ? p.c.v : p.c.k) + (block << p.c.pl) * D;
  const float s = pid < 0 ? 0.0f : (values ? p.c.vs : p.c.ks)[block];
  if (values && pid >= 0) {
    const int t0 = sp.lo & ~15;
    const int runs = (sp.hi - t0 + 15) / 16;
    for (int at = tid; at < D * runs; at += kThreads) {
      const int d = at / runs, tok = t0 + (at % runs) * 16;
      const uint4 q = *(const uint4*)(codes + d * P + tok);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        turned[(tok + j) * (D + 4) + d] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
      }
    }
  }
  __syncthreads();
  for (int at = tid; at < (sp.hi - sp.lo) * kPer; at += kThreads) {
    const int tok = sp.lo + at / kPer, d0 = (at % kPer) * 8;
    uint2 q = make_uint2(0, 0);
    if (pid >= 0) {
      if (values) {
        const uint32_t* const w = (const uint32_t*)(turned + tok * (D + 4) + d0);
        q = make_uint2(w[0], w[1]);
      } else {
        q = *(const uint2*)(codes + tok * D + d0);
      }
    }
    auto value = [&](uint32_t w, int i) { return (float)(int8_t)((w >> (8 * i)) & 0xffu) * s; };
    uint4 r = make_uint4(0, 0, 0, 0);
    if (pid >= 0) {
      r.x = pack_bf16x2(value(q.x, 0), value(q.x, 1));
      r.y = pack_bf16x2(value(q.x, 2), value(q.x, 3));
      r.z = pack_bf16x2(value(q.y, 0), value(q.y, 1));
      r.w = pack_bf16x2(value(q.y, 2), value(q.y, 3));
    }
    *(uint4*)(y + (sp.first + tok) * stride + d0) = r;
  }
}

// ---- attention over the cache -------------------------------------------------

struct CachedParams {
  CacheView c;
  const int* lens;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  float* part;       // [rows][splits][D] means, then [rows][splits][2] maximum and sum
  long qs, os;
  int heads, share, causal;
  float scale2;      // scale log2(e)
  int batch, q_len, max_len;
  int row_blocks, splits, chunk;
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c)
{
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c)
{
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float xor16_max(float v)
{
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float v)
{
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int visible_len(const CachedParams& p, int b)
{
  const long most = min((long)p.max_len, (long)p.c.table_stride << p.c.pl);
  return (int)min((long)max(p.lens[b], 0), most);
}

// A workgroup takes 16 RT rows (query token x head of the kv head) of one
// sequence and kv head over one split of the tokens; its four waves take tiles
// of 64 tokens in turn and join at the end.
//
// A wave multiplies S^T = K Q^T with v_mfma_f32_16x16x32_bf16. Row r of the
// tile's 16-token block t is token 16 (r / 4) + 4 t + r % 4, so that the lanes
// 16 j .. 16 j + 15 end up with the logits of tokens 16 j .. 16 j + 15: in
// order, they are the right operand of O^T = V^T P^T, whose left one is 16 bytes
// of a channel's tokens. Keys and values so go from memory to the matrix
// instructions through registers alone.
//
// The second product's weights w = exp(s - m) times the page's scale lie in f16
// under a running power of two of their own, 2^mw: the largest has 2^12 to 2^15, so
// that weights 2^26 times smaller keep all their 11 bits, and the output's own
// rounding is all of its error (0.00166 of its norm; with weights in bf16 0.0024,
// 0.0030 where few keys count). The sums stay as they are while no row's largest
// weight grows four times over, which pays for the second maximum: 64 sequences of
// 200 to 4000 tokens 64.1 us, 65 with bf16 weights and sums rescaled for every tile.
// (The weights as two bf16 each are as exact and took 66; 57 us for 52 at head width
// 64, 16 sequences of 8000 tokens.)
//
// Bound by memory: 4 x 8 kv heads of 99991 to 131072 tokens, 988 MB, 171 us (5.8 TB/s); 64
// sequences of 200 to 4000 tokens, 275 MB, 55 us (5.0 TB/s).
//
// Held to registers: two row tiles to two waves a SIMD (8 queries of 16 sequences of
// 4000 tokens 37.7 us, 42.6 with the registers it would take), one of head width 64
// to four (16 sequences of 8000 tokens 52.3 us, 55.2 with three).
template <int D, int RT>
__global__ void __launch_bounds__(kThreads, RT == 2 ? 2 : D == 64 && RT == 1 ? 4 : 1)
attention_cached_kernel(CachedParams p)
{
  constexpr int NW = kThreads / 64;
  constexpr int kL = D / 64;    // 16-byte loads of a token's key for each lane
  constexpr int kDT = D / 16;   // 16-channel tiles
  constexpr int kRows = 16 * RT;
  // of w, log2; a lane's weights count as 2^kFaint times the row's largest one or more where
  // mw is chosen, which keeps 2^-mw times any seen scale inside f32
  constexpr float kRoom = 13.0f, kLag = 2.0f, kFaint = -110.0f;
  __shared__ __attribute__((aligned(16))) float join[NW][16][D + 4];
  __shared__ float2 stat[NW][16];

  // Workgroups go round-robin to the 8 XCDs. The kv heads are innermost, so that
  // every XCD gets its share of each sequence, however long; the blocks of rows
  // of one part of the tokens stay on one XCD, side by side.
  const int units = p.splits * p.batch * p.c.kv_heads, whole = units & ~7;
  int u, rb;
  if ((int)blockIdx.x < whole * p.row_blocks) {
    const int at = blockIdx.x % (8 * p.row_blocks);
    u = blockIdx.x / (8 * p.row_blocks) * 8 + at % 8;
    rb = at / 8;
  } else {
    const int at = blockIdx.x - whole * p.row_blocks;
    u = whole + at % (units - whole);
    rb = at / (units - whole);
  }
  const int g = u % p.c.kv_heads;
  const int b = u / p.c.kv_heads % p.batch;
  const int split = u / p.c.kv_heads / p.batch;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kg = lane >> 4;
  const int first = split * p.chunk;
  const int* const table = p.c.table + (long)b * p.c.table_stride;
  // pages of the tokens of which the lane loads the keys (16 (n / 4) ..), and of
  // those of which it loads the values and holds the logits (16 kg ..); the first
  // ones are asked for together with the length
  const int last_page = p.c.table_stride - 1;
  auto page_of = [&](int t) { return table[min(t >> p.c.pl, last_page)]; };
  int t0 = first + wave * 64;
  int id_k = page_of(t0 + 16 * (n >> 2)), id_v = page_of(t0 + 16 * kg);
  const int len = __builtin_amdgcn_readfirstlane(visible_len(p, b));
  if (first >= len && split > 0) { return; }
  const int end = min(len, first + p.chunk);

  // rows of the lane's column of each row tile
  int limit[RT];
  bf16x8 qf[RT][2 * kL];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = min(rb * kRows + rt * 16 + n, p.q_len * p.share - 1);
    const int qi = r / p.share;
    limit[rt] = p.causal ? len - p.q_len + qi : len - 1;
    const uint16_t* const qp = p.q + ((long)b * p.q_len + qi) * p.qs +
                               (long)(g * p.share + r % p.share) * D + kg * 16;
#pragma unroll
    for (int i = 0; i < 2 * kL; ++i) {
      qf[rt][i] = as_bf16x8(*(const uint4*)(qp + (i >> 1) * 64 + (i & 1) * 8));
    }
  }
  f32x4 o[RT][kDT];
  float m[RT], l[RT];
  float mw[RT];   // log2 of what w is counted in, over 2^m
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = mw[rt] = -INFINITY;
    l[rt] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDT; ++d) { o[rt][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
  }
  const int pmask = (1 << p.c.pl) - 1;

  uint4 kc[4][kL];
  auto load_keys = [&](int t0, int id) {
    const int tk = t0 + 16 * (n >> 2);
    const long bk = (long)clampi(id, 0, p.c.pages - 1) * p.c.kv_heads + g;
    const int8_t* const kp = p.c.k + ((bk << p.c.pl) + (tk & pmask) + (n & 3)) * D + kg * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < kL; ++i) { kc[t][i] = *(const uint4*)(kp + t * 4 * D + i * 64); }
    }
  };
  // A tile's keys are asked for as soon as the keys of the tile before have been
  // used, its scales and the next pages' ids behind them, its values as soon as those
  // of the tile before have been: one tile of each in registers, and always loads in
  // flight.
  uint4 vc[kDT];
  auto load_values = [&](int t0, int id) {
    const long bv = (long)clampi(id, 0, p.c.pages - 1) * p.c.kv_heads + g;
    const int8_t* const vp =
        p.c.v + (bv << p.c.pl) * D + ((long)n << p.c.pl) + ((t0 + 16 * kg) & pmask);
#pragma unroll
    for (int d = 0; d < kDT; ++d) { vc[d] = *(const uint4*)(vp + ((long)d << (p.c.pl + 4))); }
  };
  float next_k = 0.0f, next_v = 0.0f;
  auto load_scales = [&](int id) {
    const long bv = (long)clampi(id, 0, p.c.pages - 1) * p.c.kv_heads + g;
    next_k = p.c.ks[bv];
    next_v = p.c.vs[bv];
  };
  int id_v1 = id_v;
  if (t0 < end) {
    load_keys(t0, id_k);
    load_scales(id_v);
    const int t1 = t0 + 64 * NW;
    if (t1 < end) {
      id_k = page_of(t1 + 16 * (n >> 2));
      id_v1 = page_of(t1 + 16 * kg);
    }
    load_values(t0, id_v);
  }
  for (; t0 < end; t0 += 64 * NW) {
    const int tv = t0 + 16 * kg;
    const bool held = id_v >= 0 && id_v < p.c.pages;
    const int t1 = t0 + 64 * NW;

    f32x4 s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) { s[rt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
#pragma unroll
      for (int i = 0; i < kL; ++i) {
        const bf16x8 a = codes_bf16(kc[t][i].x, kc[t][i].y);
        const bf16x8 c = codes_bf16(kc[t][i].z, kc[t][i].w);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          s[rt][t] = mfma16(a, qf[rt][2 * i], s[rt][t]);
          s[rt][t] = mfma16(c, qf[rt][2 * i + 1], s[rt][t]);
        }
      }
    }
    const float sk = next_k * p.scale2, sv = next_v;
    id_v = id_v1;
    if (t1 < end) {
      load_keys(t1, id_k);
      load_scales(id_v);
      const int t2 = t1 + 64 * NW;
      if (t2 < end) {
        id_k = page_of(t2 + 16 * (n >> 2));
        id_v1 = page_of(t2 + 16 * kg);
      }
    }
    // the scale in two parts, since 1 / sv may be past f32's end: a logarithm and a reciprocal
    // lose scales below 2^-113, which appending makes of values below 2^-106
    const float sv_m = __builtin_amdgcn_frexp_mantf(sv);
    const float sv_e = (float)__builtin_amdgcn_frexp_expf(sv);
    f16x8 pf[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int lim = held ? min(limit[rt], end - 1) : -1;
      // the scale of a page without a token that the row sees may be anything: not counted
      const bool seen = tv <= lim;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { s[rt][t][i] *= sk; }
      }
      if (any_lane(lim < tv + 15)) {   // else the tile is seen whole
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[rt][t][i] = tv + 4 * t + i <= lim ? s[rt][t][i] : -INFINITY;
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { top = fmaxf(top, s[rt][t][i]); }
      }
      const float m_new = fmaxf(m[rt], xor32_max(xor16_max(top)));
      const float ms = m_new == -INFINITY ? 0.0f : m_new;
      const float lag = m[rt] - ms, keep = __builtin_amdgcn_exp2f(lag);
      m[rt] = m_new;
      // the row's largest w: the 16 tokens of a lane are of one page
      const float lane_w = seen && sv != 0.0f ? fmaxf(top - ms, kFaint) + sv_e : -INFINITY;
      const float top_w = xor32_max(xor16_max(lane_w)) - kRoom;
      mw[rt] += lag;
      if (any_lane(top_w > mw[rt] + kLag)) {
        const float mw_new = fmaxf(mw[rt], top_w);
        const float keep_o = mw_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw[rt] - mw_new);
        mw[rt] = mw_new;
#pragma unroll
        for (int d = 0; d < kDT; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i) { o[rt][d][i] *= keep_o; }
        }
      }
      const float f =
          (seen ? sv_m : 0.0f) * __builtin_amdgcn_exp2f(fminf(sv_e - mw[rt], 127.0f));
      float sum = 0.0f;
      float w[16];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(s[rt][t][i] - ms);
          sum += e;
          w[4 * t + i] = e * f;
        }
      }
      l[rt] = fmaf(l[rt], keep, sum);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 pw;
        pw.x = pack_f16x2(w[8 * j + 0], w[8 * j + 1]);
        pw.y = pack_f16x2(w[8 * j + 2], w[8 * j + 3]);
        pw.z = pack_f16x2(w[8 * j + 4], w[8 * j + 5]);
        pw.w = pack_f16x2(w[8 * j + 6], w[8 * j + 7]);
        pf[rt][j] = as_f16x8(pw);
      }
    }
#pragma unroll
    for (int d = 0; d < kDT; ++d) {
      const f16x8 a = codes_f16(vc[d].x, vc[d].y);
      const f16x8 c = codes_f16(vc[d].z, vc[d].w);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        o[rt][d] = mfma16(a, pf[rt][0], o[rt][d]);
        o[rt][d] = mfma16(c, pf[rt][1], o[rt][d]);
      }
    }
    if (t1 < end) { load_values(t1, id_v); }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] = xor32_sum(xor16_sum(l[rt]));
    // means from here on: they stay in range where sums of large values would not. 2^mw in
    // two steps: it may be below f32's range where the mean is not
    const float half = __builtin_amdgcn_exp2f(0.5f * mw[rt]);
    const float f = l[rt] == 0.0f ? 0.0f : half / l[rt];
#pragma unroll
    for (int d = 0; d < kDT; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) { o[rt][d][i] = o[rt][d][i] * half * f; }
    }
  }

  // ---- the waves join through LDS, 16 rows at a time: a thread takes kPer
  // channels of one row
  constexpr int kPer = D * 16 / (NW * 64);
  static_assert(kPer % 4 == 0, "a thread's channels are whole stores");
  const int jr = threadIdx.x / (4 * NW), jd = threadIdx.x % (4 * NW) * kPer;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (rt > 0) { __syncthreads(); }
#pragma unroll
    for (int d = 0; d < kDT; ++d) { *(f32x4*)&join[wave][n][16 * d + 4 * kg] = o[rt][d]; }
    if (kg == 0) { stat[wave][n] = make_float2(m[rt], l[rt]); }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) { top = fmaxf(top, stat[w][jr].x); }
    const float ms = top == -INFINITY ? 0.0f : top;
    float part[NW], sum = 0.0f, acc[kPer];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 x = stat[w][jr];
      part[w] = __builtin_amdgcn_exp2f(x.x - ms) * x.y;
      sum += part[w];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { acc[i] = 0.0f; }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) { acc[i] = fmaf(part[w] * inv, join[w][jr][jd + i], acc[i]); }
    }
    const int r = rb * kRows + rt * 16 + jr;
    if (r >= p.q_len * p.share) { continue; }
    const long token = (long)b * p.q_len + r / p.share;
    const int head = g * p.share + r % p.share;
    const long at = token * p.heads + head;
    if (p.splits > 1) {
      const long rows = (long)p.batch * p.q_len * p.heads;
      float* const op = p.part + (at * p.splits + split) * D + jd;
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        *(f32x4*)(op + i) = f32x4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
      }
      if (jd == 0) {
        *(float2*)(p.part + rows * p.splits * D + (at * p.splits + split) * 2) =
            make_float2(top, sum);
      }
    } else {
      uint32_t* const op = (uint32_t*)(p.out + token * p.os + (long)head * D + jd);
#pragma unroll
      for (int i = 0; i < kPer; i += 2) { op[i / 2] = pack_bf16x2(acc[i], acc[i + 1]); }
      if (p.lse != nullptr && jd == 0) {
        p.lse[at] = sum == 0.0f ? -INFINITY : (ms + log2f(sum)) * 0.69314718055994531f;
      }
    }
  }
}

// The parts of a row joined; a wave for each row. Bound by the latency of its loads,
// one after another: 4.8 us.
template <int D>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(CachedParams p)
{
  const long rows = (long)p.batch * p.q_len * p.heads;
  const long at = (long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (at >= rows) { return; }
  const long token = at / p.heads;
  const int head = (int)(at % p.heads);
  const int len = visible_len(p, (int)(token / p.q_len));
  join_parts<D>(p.part + at * p.splits * D,
                (const float2*)(p.part + rows * p.splits * D) + at * p.splits,
                min((len + p.chunk - 1) / p.chunk, p.splits), p.out + token * p.os + (long)head * D,
                p.lse == nullptr ? nullptr : p.lse + at);
}

CacheView view_of(const CacheArgs& c)
{
  CacheView v;
  v.k = c.k;
  v.v = c.v;
  v.ks = c.ks;
  v.vs = c.vs;
  v.table = c.table;
  v.pages = c.pages;
  v.pl = c.page_log2;
  v.kv_heads = c.kv_heads;
  v.table_stride = c.table_stride;
  return v;
}

// Pages that `total` tokens of `batch` sequences can touch: a sequence's n
// tokens lie in at most n / P + 2.
bool move_grid(const MoveParams& p, dim3& grid)
{
  const long units = ((long)p.total >> p.c.pl) + 2L * p.batch;
  if (units > INT_MAX || p.c.kv_heads > 65535) { return false; }
  grid = dim3((unsigned)units, (unsigned)p.c.kv_heads, 2);
  return true;
}

template <int D, int RT>
hipError_t run_cached(const CachedParams& p, hipStream_t stream)
{
  const long grid = (long)p.batch * p.c.kv_heads * p.splits * p.row_blocks;
  const long rows = (long)p.batch * p.q_len * p.heads;
  if (grid > INT_MAX || rows > INT_MAX) { return hipErrorInvalidConfiguration; }
  attention_cached_kernel<D, RT><<<(int)grid, kThreads, 0, stream>>>(p);
  if (p.splits > 1) {
    constexpr int kWaves = kThreads / 64;
    attention_join_kernel<D><<<(int)((rows + kWaves - 1) / kWaves), kThreads, 0, stream>>>(p);
  }
  return hipGetLastError();
}

template <int D>
hipError_t run_cached(const CachedParams& p, const CachedPlan& plan, hipStream_t stream)
{
  if (plan.row_tiles == 1) { return run_cached<D, 1>(p, stream); }
  if (plan.row_tiles == 2) { return run_cached<D, 2>(p, stream); }
  return run_cached<D, 4>(p, stream);
}

}  // namespace

hipError_t launch_kv_append(const CacheArgs& c, const uint16_t* k, const uint16_t* v, int64_t ks,
                            int64_t vs, const int* cu, const int* start, int batch, int total,
                            hipStream_t stream)
{
  const MoveParams p = {view_of(c), k, v, nullptr, nullptr, (long)ks, (long)vs, cu, start, batch,
                        total};
  dim3 grid;
  if (!move_grid(p, grid)) { return hipErrorInvalidConfiguration; }
  if (c.head_dim == 128) {
    kv_append_kernel<128><<<grid, kThreads, 0, stream>>>(p, Rotation());
  } else {
    kv_append_kernel<64><<<grid, kThreads, 0, stream>>>(p, Rotation());
  }
  return hipGetLastError();
}

hipError_t launch_kv_append_rope(const CacheArgs& c, const uint16_t* k, const uint16_t* v,
                                 int64_t ks, int64_t vs, const int* cu, const int* start,
                                 const Rotation& r, int batch, int total, hipStream_t stream)
{
  const MoveParams p = {view_of(c), k, v, nullptr, nullptr, (long)ks, (long)vs, cu, start, batch,
                        total};
  dim3 grid;
  if (!move_grid(p, grid)) { return hipErrorInvalidConfiguration; }
  // (a token's place is the same on every axis)
  const bool many = r.positions != nullptr && r.n_axes > 1;
  if (c.head_dim == 128) {
    (many ? kv_append_kernel<128, 2> : kv_append_kernel<128, 1>)<<<grid, kThreads, 0, stream>>>(p, r);
  } else {
    (many ? kv_append_kernel<64, 2> : kv_append_kernel<64, 1>)<<<grid, kThreads, 0, stream>>>(p, r);
  }
  return hipGetLastError();
}

hipError_t launch_kv_read(const CacheArgs& c, uint16_t* k, uint16_t* v, int64_t ks, int64_t vs,
                          const int* cu, const int* start, int batch, int total,
                          hipStream_t stream)
{
  const MoveParams p = {view_of(c), nullptr, nullptr, k, v, (long)ks, (long)vs, cu, start, batch,
                        total};
  dim3 grid;
  if (!move_grid(p, grid)) { return hipErrorInvalidConfiguration; }
  if (c.head_dim == 128) {
    kv_read_kernel<128><<<grid, kThreads, 0, stream>>>(p);
  } else {
    kv_read_kernel<64><<<grid, kThreads, 0, stream>>>(p);
  }
  return hipGetLastError();
}

CachedPlan plan_cached(int batch, int q_len, int heads, int kv_heads, int head_dim, int max_len)
{
  CachedPlan r;
  const long rows = (long)q_len * (heads / kv_heads);
  r.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  r.row_blocks = (int)((rows + 16 * r.row_tiles - 1) / (16 * r.row_tiles));
  // Parts of whole rounds of the four waves (256 tokens). Up to 3 rounds: one part. A
  // round more takes 2 us where the GPU is not full, the join's launch 3 on the GPU and
  // 3 on the host (700 tokens, 8 kv heads: 9.1 us a call, 11.4 in 3 parts; replayed in a
  // graph 8.6 and 7.7). Else two workgroups for each CU, which hold enough loads in
  // flight (4 x 8 kv heads of 99991 to 131072 tokens: 175 us, 180 with four workgroups, 185 with
  // eight) -- but past 20 rounds no part longer than 8 rounds or a 16th of the tokens,
  // since the lengths may be very uneven and only the longest is known here (63
  // sequences of 200 tokens beside one of 30000: 52 us for 78 in parts of 20 rounds; from how
  // many rounds on that pays has not been measured).
  const long units = (long)batch * kv_heads * r.row_blocks;
  const long rounds = ((long)max_len + 255) / 256;
  long per = std::max(rounds, 1L);
  if (rounds > 3) {
    const long want = (512 + units - 1) / units;
    const long cap = rounds <= 20 ? rounds : std::max(8L, rounds / 16);
    per = std::min((rounds + want - 1) / want, cap);
    per = (rounds + (rounds + per - 1) / per - 1) / ((rounds + per - 1) / per);
  }
  r.chunk = (int)std::min(per * 256, (long)(INT_MAX & ~255));
  r.splits = (int)std::max(1L, (rounds + per - 1) / per);
  if (r.splits > 1) {
    r.workspace_bytes = (size_t)batch * q_len * heads * r.splits * (head_dim + 2) * sizeof(float);
  }
  return r;
}

hipError_t launch_attention_cached(const CachedArgs& a, hipStream_t stream)
{
  const CachedPlan plan =
      plan_cached(a.batch, a.q_len, a.heads, a.c.kv_heads, a.c.head_dim, a.max_len);
  CachedParams p;
  p.c = view_of(a.c);
  p.lens = a.lens;
  p.q = a.q;
  p.out = a.out;
  p.lse = a.lse;
  p.part = a.workspace;
  p.qs = (long)a.qs;
  p.os = (long)a.os;
  p.heads = a.heads;
  p.share = a.heads / a.c.kv_heads;
  p.causal = a.causal;
  p.scale2 = a.scale * 1.4426950408889634f;
  p.batch = a.batch;
  p.q_len = a.q_len;
  p.max_len = a.max_len;
  p.row_blocks = plan.row_blocks;
  p.splits = plan.splits;
  p.chunk = plan.chunk;
  return a.c.head_dim == 128 ? run_cached<128>(p, plan, stream)
                             : run_cached<64>(p, plan, stream);
}

}  // namespace ltx25
