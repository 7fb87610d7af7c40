// The product of two microscaled 4-bit operands (ltx25_mx4_gemm, ltx25_linear_mx4) on
// v_mfma_scale_f32_16x16x128_f8f6f4: a lane's 16 bytes of an operand are one block of 32
// and its scale is one byte of a register of the lane's, so the scales cost no arithmetic.
#include "mx4.h"

#include <algorithm>
#include <type_traits>

namespace ltx25 {
namespace {

typedef uint32_t __attribute__((address_space(3))) lds_u32;

struct GemmParams {
  const uint8_t* x;
  const uint8_t* xs;
  const uint8_t* w;
  const uint8_t* ws;
  const void* bias;
  uint16_t* y;
  float* partial;   // null: y is written
  int M, N, K;
  int bias_type, epilogue;
  int tiles_m, tiles_n;
  int span_chunk;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, size_t bytes)
{
  // loads past `bytes` return zeros
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)(uint32_t)bytes,
                                           0x00020000);
}

// acc += w . x over 128 values, scales in byte J of the lanes' registers
template <int J>
__device__ __forceinline__ f32x4 mfma_mx4(i32x4 w, i32x4 x, f32x4 acc, int ws, int xs)
{
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(w), mx4_operand(x), acc,
                                                          kMfmaFp4, kMfmaFp4, J, ws, J, xs);
}

// 32 RB x 32 CB outputs of a workgroup of four waves, 2 x 2; a wave has RB x CB blocks of
// 16 x 16. A step is 256 values of K: 128 bytes of a row, which go from memory straight into
// one of two LDS stages, 8 rows an instruction, the row's 16-byte pieces at slot piece ^ (row
// % 8), so that a fragment's reads (16 rows x 4 pieces) are free of bank conflicts. Scales go
// to registers, a dword of a lane for each block of rows and two steps.
template <int RB, int CB>
__global__ void __launch_bounds__(256, 2) mx4_tile_kernel(GemmParams p)
{
  constexpr int BM = 32 * RB, BN = 32 * CB;
  constexpr int kStage = (BM + BN) * 128;
  constexpr int kEP = BN + 8;   // staged output row
  static_assert(BM * kEP * 2 <= 2 * kStage, "the staged tile fits the stages");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  map_tile(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;

  const int spans = mx4_spans(p.K);
  const int span0 = (int)blockIdx.y * p.span_chunk;
  const int span1 = min(span0 + p.span_chunk, spans);
  const int blocks = p.K >> 5;
  const int step1 = min(2 * span1, (blocks + 7) >> 3);
  const uint32_t pitch = (uint32_t)p.K >> 1;

  const size_t xbytes = (size_t)p.M * pitch, wbytes = (size_t)p.N * pitch;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x, xbytes), wr = make_rsrc(p.w, wbytes);
  const __amdgpu_buffer_rsrc_t xsr = make_rsrc(p.xs, mx4_scale_bytes(p.M, p.K));
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(p.ws, mx4_scale_bytes(p.N, p.K));

  // wave w issues instructions RB w + i of X and CB w + i of W
  const int piece = (lane & 7) ^ (lane >> 3);
  const uint32_t xoff = (uint32_t)(m0 + 8 * RB * wave + (lane >> 3)) * pitch + piece * 16;
  const uint32_t woff = (uint32_t)(n0 + 8 * CB * wave + (lane >> 3)) * pitch + piece * 16;
  auto load = [&](int s) {
    uint8_t* const xd = lds + (s & 1) * kStage + RB * wave * 1024;
    uint8_t* const wd = lds + (s & 1) * kStage + BM * 128 + CB * wave * 1024;
    // pieces past the row's end would be the next row's: an offset past the operand gives zeros
    const bool in = 8 * s + piece < blocks;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (lds_u32*)(xd + i * 1024), 16, (int)(in ? xoff + 8u * i * pitch : (uint32_t)xbytes),
          s * 128, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr, (lds_u32*)(wd + i * 1024), 16, (int)(in ? woff + 8u * i * pitch : (uint32_t)wbytes),
          s * 128, 0, 0);
    }
  };
  int xs[RB], ws[CB];
  auto load_scales = [&](int span) {
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const uint32_t at = (uint32_t)((m0 + wm * 16 * RB) / 16 + i) * spans * kMx4Tile + lane * 4;
      xs[i] = __builtin_amdgcn_raw_buffer_load_b32(xsr, (int)at, span * kMx4Tile, 0);
    }
#pragma unroll
    for (int j = 0; j < CB; ++j) {
      const uint32_t at = (uint32_t)((n0 + wn * 16 * CB) / 16 + j) * spans * kMx4Tile + lane * 4;
      ws[j] = __builtin_amdgcn_raw_buffer_load_b32(wsr, (int)at, span * kMx4Tile, 0);
    }
  };
  const int fo0 = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16);
  const int fo1 = (lane & 15) * 128 + (((4 + (lane >> 4)) ^ (lane & 7)) * 16);
  f32x4 acc[RB][CB] = {};
  int cxs[RB], cws[CB];
  auto step = [&](int s, auto half) {
    constexpr int H = decltype(half)::value;
    const uint8_t* const xb = lds + (s & 1) * kStage + wm * 16 * RB * 128;
    const uint8_t* const wb = lds + (s & 1) * kStage + BM * 128 + wn * 16 * CB * 128;
    auto slice = [&](auto sl) {
      constexpr int J = 2 * H + decltype(sl)::value;
      const int fo = decltype(sl)::value ? fo1 : fo0;
      i32x4 a[RB], b[CB];
#pragma unroll
      for (int i = 0; i < RB; ++i) { a[i] = *(const i32x4*)(xb + fo + i * 16 * 128); }
#pragma unroll
      for (int j = 0; j < CB; ++j) { b[j] = *(const i32x4*)(wb + fo + j * 16 * 128); }
#pragma unroll
      for (int i = 0; i < RB; ++i) {
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          acc[i][j] = mfma_mx4<J>(b[j], a[i], acc[i][j], cws[j], cxs[i]);
        }
      }
    };
    slice(std::integral_constant<int, 0>{});
    slice(std::integral_constant<int, 1>{});
  };
  // every load in flight has landed, in all waves
  auto landed = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
  };

  load(2 * span0);
  load_scales(span0);
  for (int s = 2 * span0; s < step1; s += 2) {
    landed();
#pragma unroll
    for (int i = 0; i < RB; ++i) { cxs[i] = xs[i]; }
#pragma unroll
    for (int j = 0; j < CB; ++j) { cws[j] = ws[j]; }
    if (s + 1 < step1) { load(s + 1); }
    if (s + 2 < step1) { load_scales((s + 2) / 2); }
    step(s, std::integral_constant<int, 0>{});
    landed();
    if (s + 1 >= step1) { break; }
    if (s + 2 < step1) { load(s + 2); }
    step(s + 1, std::integral_constant<int, 1>{});
  }
  __syncthreads();

  // block (i, j), lane l, register r: row 16 i + l % 16, column 16 j + 4 (l / 16) + r
  const int lrow = lane & 15, lcol = (lane >> 4) * 4;
  if (p.partial != nullptr) {
    float* const out = p.partial + (size_t)blockIdx.y * p.M * p.N;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int m = m0 + (wm * RB + i) * 16 + lrow;
      if (m >= p.M) { continue; }
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        const int n = n0 + (wn * CB + j) * 16 + lcol;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (n + r < p.N) { out[(size_t)m * p.N + n + r] = acc[i][j][r]; }
        }
      }
    }
    return;
  }
  uint16_t* const stage = (uint16_t*)lds;
#pragma unroll
  for (int j = 0; j < CB; ++j) {
    const int c = (wn * CB + j) * 16 + lcol;
    float bias[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) { bias[r] = load_bias(p.bias, p.bias_type, min(n0 + c + r, p.N - 1)); }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = acc[i][j][r] + bias[r];
        if (p.epilogue == kEpiGelu) { v[r] = gelu_tanh(v[r]); }
      }
      *(uint2*)(stage + ((wm * RB + i) * 16 + lrow) * kEP + c) =
          make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  }
  __syncthreads();
  if (p.N % 8 == 0) {
    for (int q = tid; q < BM * BN / 8; q += 256) {
      const int r = q / (BN / 8), c = (q % (BN / 8)) * 8;
      if (m0 + r < p.M && n0 + c < p.N) {
        *(uint4*)(p.y + (size_t)(m0 + r) * p.N + n0 + c) = *(const uint4*)(stage + r * kEP + c);
      }
    }
  } else {
    for (int q = tid; q < BM * BN; q += 256) {
      const int r = q / BN, c = q % BN;
      if (m0 + r < p.M && n0 + c < p.N) {
        p.y[(size_t)(m0 + r) * p.N + n0 + c] = stage[r * kEP + c];
      }
    }
  }
}

template <int RB, int CB>
hipError_t run_tile(GemmParams& p, const Mx4Plan& plan, hipStream_t stream)
{
  p.tiles_m = (p.M + 32 * RB - 1) / (32 * RB);
  p.tiles_n = (p.N + 32 * CB - 1) / (32 * CB);
  const long tiles = (long)p.tiles_m * p.tiles_n;
  if (tiles * 256 >= 1L << 32) { return hipErrorInvalidConfiguration; }
  mx4_tile_kernel<RB, CB><<<dim3((unsigned)tiles, (unsigned)plan.splits), 256, 0, stream>>>(p);
  return hipGetLastError();
}

// Rows of x below 2 GiB of codes and scales
constexpr size_t kSlabBytes = (size_t)1 << 31;

}  // namespace

Mx4Plan plan_mx4(int M, int K, int N, bool bf16)
{
  Mx4Plan r;
  r.codes_ahead = bf16;
  const int spans = mx4_spans(K);
  const long big = (long)((M + 127) / 128) * ((N + 127) / 128);
  const long small = (long)((M + 63) / 64) * ((N + 63) / 64);
  r.tile = big >= 256 ? 0 : 1;
  const long tiles = r.tile == 0 ? big : small;
  r.splits = (int)std::max(1L, std::min((long)spans, 512 / std::max(1L, tiles)));
  r.span_chunk = (spans + r.splits - 1) / r.splits;
  r.splits = (spans + r.span_chunk - 1) / r.span_chunk;
  r.partial_bytes = r.splits > 1 ? (size_t)r.splits * M * N * sizeof(float) : 0;
  return r;
}

hipError_t launch_mx4_gemm(const Mx4Gemm& g, const Mx4Plan& plan, hipStream_t stream)
{
  if (plan.codes_ahead) {
    const hipError_t e = launch_mx4_quantize(g.xb, false, g.xb_stride, g.x, stream);
    if (e != hipSuccess) { return e; }
  }
  const int K = g.w.K, M = g.x.rows, N = g.w.rows;
  // rows of a launch: whole tiles, operands that 32-bit offsets reach
  const long most = (long)((kSlabBytes - 1) / (size_t)(K / 2)) & ~255L;
  for (long m = 0; m < M; m += most) {
    GemmParams p;
    p.x = g.x.codes + (size_t)m * (K / 2);
    p.xs = g.x.scales + (size_t)(m / 16) * mx4_spans(K) * kMx4Tile;
    p.w = g.w.codes;
    p.ws = g.w.scales;
    p.bias = g.bias;
    p.y = g.y + (size_t)m * N;
    p.partial = plan.splits > 1 ? g.partial : nullptr;
    p.M = (int)std::min(most, M - m);
    p.N = N;
    p.K = K;
    p.bias_type = g.bias_type;
    p.epilogue = g.epilogue;
    p.span_chunk = plan.span_chunk;
    hipError_t e = plan.tile == 0 ? run_tile<4, 4>(p, plan, stream) : run_tile<2, 2>(p, plan, stream);
    if (e == hipSuccess && p.partial != nullptr) {
      e = launch_splitk_reduce(p.partial, plan.splits, g.bias, g.bias_type, g.epilogue, nullptr,
                               p.y, p.M, N, stream);
    }
    if (e != hipSuccess) { return e; }
  }
  return hipSuccess;
}

}  // namespace ltx25
