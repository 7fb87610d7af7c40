// Device helpers and launchers of the attention kernels (attention.hip,
// kv_cache.hip), and the launcher interface their C ABI layer
// (capi_attention.cpp) calls.
#pragma once

#include "common.h"

#include <cmath>

namespace ltx25 {

typedef __attribute__((address_space(3))) uint32_t lds_word;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

__device__ __forceinline__ float xor32_max(float v)
{
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float xor32_sum(float v)
{
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ bool any_lane(bool b) { return __any(b) != 0; }
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// v of the lane that the DPP control names, 0 where there is none or the row is
// masked off
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp_or_zero(int v)
{
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}

// The sum over the lanes up to the lane's own: within rows of 16, then the rows'
// last lanes on (DPP moves take a VALU operation's time, a shuffle an LDS access's)
__device__ __forceinline__ int scan_sum(int v)
{
  v += dpp_or_zero<0x111>(v);
  v += dpp_or_zero<0x112>(v);
  v += dpp_or_zero<0x114>(v);
  v += dpp_or_zero<0x118>(v);
  v += dpp_or_zero<0x142, 0xa>(v);
  v += dpp_or_zero<0x143, 0xc>(v);
  return v;
}

// The largest over the wave
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
  v = max(v, (uint32_t)dpp_or_zero<0x111>((int)v));
  v = max(v, (uint32_t)dpp_or_zero<0x112>((int)v));
  v = max(v, (uint32_t)dpp_or_zero<0x114>((int)v));
  v = max(v, (uint32_t)dpp_or_zero<0x118>((int)v));
  v = max(v, (uint32_t)dpp_or_zero<0x142, 0xa>((int)v));
  v = max(v, (uint32_t)dpp_or_zero<0x143, 0xc>((int)v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// A list of units, count(b) for each sequence b in order: the sequence, the
// place within it of unit u, and the lane whose last count(b) was the sequence's
// (what else that call read is there). Every lane of a wave takes part and all get
// the same answer; false when there are fewer units. The counts come from device
// memory that the caller has not checked: each is cut to [0, 2^24] and the sums
// kept in 64 bits.
//
// More than 64 sequences are looked at 256 at a time, whose reads are then in
// flight together, and the unit's own is read again at the end.
template <typename Count>
__device__ __forceinline__ bool find_unit(int u, int batch, Count&& count, int& seq, int& place,
                                          int& from)
{
  const int lane = threadIdx.x & 63;
  auto count_of = [&](int b) { return b < batch ? clampi(count(b), 0, 1 << 24) : 0; };
  if (batch <= 64) {
    const int n = count_of(lane);
    const int sum = scan_sum(n);
    const unsigned long long past = __ballot(sum > u);
    if (past == 0) { return false; }
    from = seq = __builtin_ctzll(past);
    place = u - __builtin_amdgcn_readlane(sum - n, from);
    return true;
  }
  long base = 0;
  for (int b0 = 0; b0 < batch; b0 += 256) {
    int n[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { n[j] = count_of(b0 + 64 * j + lane); }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int sum = scan_sum(n[j]);
      const unsigned long long past = __ballot(base + sum > (long)u);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        seq = b0 + 64 * j + at;
        place = (int)(u - base) - __builtin_amdgcn_readlane(sum - n[j], at);
        (void)count(seq);   // in every lane
        from = 0;
        return true;
      }
      base += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  return false;
}

// One row's parts joined by a wave: `used` means of D channels at `means`, a maximum
// (log2) and a sum each at `ml`. D / 4 lanes take 4 channels each of one part, so that
// 64 / (D / 4) parts are read side by side, and four of those in flight; always added in
// the same order. No parts at all, or none with a sum: zeros. A mean that is not finite
// comes from a token that the row sees, whose weight is positive however small: it counts
// whole, where a weight below f32's range would make a NaN of an infinity.
template <int D>
__device__ __forceinline__ void join_parts(const float* means, const float2* ml, int used,
                                           uint16_t* out, float* lse)
{
  constexpr int kLanes = D / 4, kSide = 64 / kLanes;
  const int lane = threadIdx.x & 63;
  const int part = lane / kLanes, d = (lane % kLanes) * 4;
  f32x4 x[4];
  float2 st[4];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = max(min(s0 + j * kSide, used - 1), 0);
      x[j] = *(const f32x4*)(means + (long)s * D + d);
      st[j] = ml[s];
    }
  };
  fetch(part);   // beside the maxima
  float top = -INFINITY;
  for (int s = lane; s < used; s += 64) { top = fmaxf(top, ml[s].x); }
#pragma unroll
  for (int i = 1; i < 64; i *= 2) { top = fmaxf(top, __shfl_xor(top, i)); }
  const float ms = top == -INFINITY ? 0.0f : top;
  float l = 0.0f;
  for (int s = lane; s < used; s += 64) { l = fmaf(__builtin_amdgcn_exp2f(ml[s].x - ms), ml[s].y, l); }
#pragma unroll
  for (int i = 1; i < 64; i *= 2) { l += __shfl_xor(l, i); }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = part; s0 < used; s0 += 4 * kSide) {
    if (s0 != part) { fetch(s0); }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // past the last part x is that part's again; selected rather than branched over, so that
      // the loads stay in flight together (32 parts: 21 us a call, 25 with branches)
      const bool there = s0 + j * kSide < used;
      const float w = __builtin_amdgcn_exp2f(st[j].x - ms) * st[j].y * inv;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = there ? x[j][i] : 0.0f;
        acc[i] = fmaf(!there ? 0.0f : fabsf(v) < INFINITY ? w : 1.0f, v, acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = kLanes; i < 64; i *= 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) { acc[j] += __shfl_xor(acc[j], i); }
  }
  if (part != 0) { return; }
  *(uint2*)(out + d) = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
  if (lse != nullptr && d == 0) {
    *lse = l == 0.0f ? -INFINITY : (ms + log2f(l)) * 0.69314718055994531f;
  }
}

// ---- launchers --------------------------------------------------------------

struct AttentionArgs {
  const uint16_t* q = nullptr;
  const uint16_t* k = nullptr;
  const uint16_t* v = nullptr;
  uint16_t* out = nullptr;
  float* lse = nullptr;
  const int* cu_q = nullptr;
  const int* cu_k = nullptr;
  int64_t qs = 0, ks = 0, vs = 0, os = 0;
  int heads = 0, kv_heads = 0, head_dim = 0;
  int causal = 0;
  float scale = 0.0f;
  int batch = 0, total_q = 0, total_k = 0;
  float* workspace = nullptr;   // null: every row in one part
};
// How a call's work is cut; a function of the sizes alone, so that the workspace can be
// asked for ahead.
struct PromptPlan {
  bool turns = false;         // the form of 8 waves
  int hp_log2 = 0, tb_log2 = 0;   // a workgroup's rows: 2^hp heads x 2^tb tokens
  int head_groups = 1;
  long units = 0;             // units of 2^tb tokens, at most
  int splits = 1;             // parts of the keys, with a workspace
  size_t workspace_bytes = 0;
};
PromptPlan plan_prompt(int heads, int kv_heads, int head_dim, int batch, int total_q, int total_k);
hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream);

struct CacheArgs {
  int8_t* k = nullptr;
  int8_t* v = nullptr;
  float* ks = nullptr;
  float* vs = nullptr;
  int pages = 0, page_log2 = 0, kv_heads = 0, head_dim = 0;
  const int* table = nullptr;
  int table_stride = 0;
};
hipError_t launch_kv_append(const CacheArgs& c, const uint16_t* k, const uint16_t* v, int64_t ks,
                            int64_t vs, const int* cu, const int* start, int batch, int total,
                            hipStream_t stream);
hipError_t launch_kv_read(const CacheArgs& c, uint16_t* k, uint16_t* v, int64_t ks, int64_t vs,
                          const int* cu, const int* start, int batch, int total,
                          hipStream_t stream);

struct CachedArgs {
  CacheArgs c;
  const int* lens = nullptr;
  const uint16_t* q = nullptr;
  uint16_t* out = nullptr;
  float* lse = nullptr;
  float* workspace = nullptr;
  int64_t qs = 0, os = 0;
  int heads = 0, causal = 0;
  float scale = 0.0f;
  int batch = 0, q_len = 0, max_len = 0;
};
// How the cached attention's tokens are split; a function of the sizes alone,
// so that the workspace can be asked for ahead.
struct CachedPlan {
  int row_tiles = 1;    // 16-row tiles of a workgroup
  int row_blocks = 1;   // workgroups over a kv head's rows
  int splits = 1;
  int chunk = 0;        // tokens of a split
  size_t workspace_bytes = 0;
};
CachedPlan plan_cached(int batch, int q_len, int heads, int kv_heads, int head_dim, int max_len);
hipError_t launch_attention_cached(const CachedArgs& a, hipStream_t stream);

// The current device is one that the kernels are built for (LTX25_OK, or the
// code of the error that was set); capi.cpp.
int check_device();

}  // namespace ltx25
