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

// An offset past every operand, whose soffset still adds up within 32 bits
constexpr uint32_t kPast = 0xc0000000u;

// acc += w . x over 128 values, scales in byte J of the lanes' registers
template <int J>
__device__ __forceinline__ f32x4 mfma_mx4(i32x4 w, i32x4 x, f32x4 acc, int ws, int xs)
{
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(w), mx4_operand(x), acc,
                                                          kMfmaFp4, kMfmaFp4, J, ws, J, xs);
}

// 64 RB x 16 CB outputs of a workgroup of four waves, one below the other: a wave has RB x CB
// blocks of 16 x 16. The weight's rows, which all four read, go through LDS; a wave's rows of x
// are its own and go from memory straight to its registers, two slices of 128 values ahead: LDS
// then carries (16 CB rows x 5) bytes of K where both operands through LDS and 2 x 2 waves of
// the same size carry (32 RB + 16 CB) x 3.
//
// A span is 512 values: two LDS stages of CB tiles x 4 slices take turns, filled a span ahead
// by loads that go straight into LDS, one barrier a span. Tiles lie in LDS as in memory, and a
// fragment's read is the tile's 1 KB in the order of the lanes.
template <int RB, int CB>
__global__ void __launch_bounds__(256, 2) mx4_wide_kernel(GemmParams p)
{
  constexpr int BM = 64 * RB, BN = 16 * CB;
  constexpr int kStage = 4 * CB * kMx4CodeTile;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  map_tile(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int n0 = tn * BN, row0 = tm * BM + wave * 16 * RB;   // the wave's rows

  const int spans = mx4_spans(p.K);
  const int span0 = (int)blockIdx.y * p.span_chunk;
  const int span1 = min(span0 + p.span_chunk, spans);
  const int slices = mx4_slices(p.K);
  const uint32_t pitch = (uint32_t)slices * kMx4CodeTile;   // of 16 rows
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x, mx4_code_bytes(p.M, p.K));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.w, mx4_code_bytes(p.N, p.K));
  const __amdgpu_buffer_rsrc_t xsr = make_rsrc(p.xs, mx4_scale_bytes(p.M, p.K));
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(p.ws, mx4_scale_bytes(p.N, p.K));

  // Stage: [tile row][slice]. Wave w loads slice w of every tile row. Slices past the rows' end
  // would be the next rows': an offset past the operand gives zeros.
  const uint32_t woff = (uint32_t)(n0 / 16) * pitch + lane * 16;
  auto load_w = [&](int span) {
    const int t = 4 * span + wave;
    uint8_t* const at = lds + (span & 1) * kStage + wave * kMx4CodeTile;
#pragma unroll
    for (int j = 0; j < CB; ++j) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_u32*)(at + j * 4 * kMx4CodeTile), 16,
                                               (int)(t < slices ? woff + j * pitch : kPast),
                                               t * kMx4CodeTile, 0, 0);
    }
  };
  const uint32_t xoff = (uint32_t)(row0 / 16) * pitch + lane * 16;
  i32x4 x[4][RB];
  auto load_x = [&](int t, int buf) {
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      x[buf][i] = __builtin_bit_cast(
          i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                     xr, (int)(t < slices ? xoff + i * pitch : kPast), t * kMx4CodeTile, 0));
    }
  };
  int xs[RB], ws[CB], nxs[RB], nws[CB];
  auto load_scales = [&](int span) {
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      nxs[i] = __builtin_amdgcn_raw_buffer_load_b32(
          xsr, (int)((uint32_t)(row0 / 16 + i) * spans * kMx4Tile + lane * 4), span * kMx4Tile, 0);
    }
#pragma unroll
    for (int j = 0; j < CB; ++j) {
      nws[j] = __builtin_amdgcn_raw_buffer_load_b32(
          wsr, (int)((uint32_t)(n0 / 16 + j) * spans * kMx4Tile + lane * 4), span * kMx4Tile, 0);
    }
  };
  f32x4 acc[RB][CB] = {};
  auto slice = [&](int span, auto sl) {
    constexpr int J = decltype(sl)::value;
    const uint8_t* const wb = lds + (span & 1) * kStage + J * kMx4CodeTile + lane * 16;
    i32x4 w[CB];
#pragma unroll
    for (int j = 0; j < CB; ++j) { w[j] = *(const i32x4*)(wb + j * 4 * kMx4CodeTile); }
#pragma unroll
    for (int j = 0; j < CB; ++j) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        acc[i][j] = mfma_mx4<J>(w[j], x[J][i], acc[i][j], ws[j], xs[i]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J & 1) {
      load_x(4 * span + J + 3, J - 1);
      load_x(4 * span + J + 4, J);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  load_w(span0);
  load_scales(span0);
  load_x(4 * span0, 0);
  load_x(4 * span0 + 1, 1);
  load_x(4 * span0 + 2, 2);
  load_x(4 * span0 + 3, 3);
  for (int span = span0; span < span1; ++span) {
    // this span's weight loads have landed: two slices of x and no more came after them
    __builtin_amdgcn_s_waitcnt(0x0f70 | (2 * RB));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < RB; ++i) { xs[i] = nxs[i]; }
#pragma unroll
    for (int j = 0; j < CB; ++j) { ws[j] = nws[j]; }
    // Unconditionally, so that the compiler knows how many loads there are behind a slice of x;
    // past the row's end they give zeros.
    load_w(span + 1);
    load_scales(span + 1);
    __builtin_amdgcn_sched_barrier(0);
    slice(span, std::integral_constant<int, 0>{});
    slice(span, std::integral_constant<int, 1>{});
    slice(span, std::integral_constant<int, 2>{});
    slice(span, std::integral_constant<int, 3>{});
  }

  __builtin_amdgcn_s_waitcnt(0x0f70);   // no load into LDS outlives the wave

  // block (i, j), lane l, register r: row 16 i + l % 16, column 16 j + 4 (l / 16) + r
  const int g = lane >> 4;
  if (p.partial != nullptr || p.N % 8 != 0) {
    float* const part = p.partial == nullptr ? nullptr : p.partial + (size_t)blockIdx.y * p.M * p.N;
#pragma unroll
    for (int j = 0; j < CB; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + 16 * j + 4 * g + r;
        const float bias = load_bias(p.bias, p.bias_type, min(n, p.N - 1));
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const int m = row0 + 16 * i + (lane & 15);
          if (m >= p.M || n >= p.N) { continue; }
          if (part != nullptr) {
            part[(size_t)m * p.N + n] = acc[i][j][r];
          } else {
            const float v = acc[i][j][r] + bias;
            p.y[(size_t)m * p.N + n] = f32_to_bf16(p.epilogue == kEpiGelu ? gelu_tanh(v) : v);
          }
        }
      }
    }
    return;
  }
  // Two blocks side by side: the lanes' rows of 16 are exchanged so that each lane has eight
  // columns of one of them, 16 bytes.
  auto store = [&](auto gelu) {
#pragma unroll
    for (int j = 0; j < CB; j += 2) {
      float bias[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bias[h][r] =
              load_bias(p.bias, p.bias_type, min(n0 + 16 * (j + h) + 4 * g + r, p.N - 1));
        }
      }
      const int n = n0 + 16 * (j + (g & 1)) + 8 * (g >> 1);
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        uint32_t w[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v[r] = acc[i][j + h][r] + bias[h][r];
            if constexpr (decltype(gelu)::value) { v[r] = gelu_tanh(v[r]); }
          }
          w[h][0] = pack_bf16x2(v[0], v[1]);
          w[h][1] = pack_bf16x2(v[2], v[3]);
        }
        const auto a = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
        const auto b = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
        const int m = row0 + 16 * i + (lane & 15);
        if (m < p.M && n < p.N) {
          const i32x4 v = {(int)a[0], (int)b[0], (int)a[1], (int)b[1]};
          __builtin_nontemporal_store(v, (i32x4*)(p.y + (size_t)m * p.N + n));
        }
      }
    }
  };
  if (p.epilogue == kEpiGelu) {
    store(std::true_type{});
  } else {
    store(std::false_type{});
  }
}

template <int RB, int CB>
hipError_t run_wide(GemmParams& p, const Mx4Plan& plan, hipStream_t stream)
{
  p.tiles_m = (p.M + 64 * RB - 1) / (64 * RB);
  p.tiles_n = (p.N + 16 * CB - 1) / (16 * CB);
  const long tiles = (long)p.tiles_m * p.tiles_n;
  if (tiles * 256 >= 1L << 32) { return hipErrorInvalidConfiguration; }
  mx4_wide_kernel<RB, CB><<<dim3((unsigned)tiles, (unsigned)plan.splits), 256, 0, stream>>>(p);
  return hipGetLastError();
}

// Bytes of a launch's rows of x
constexpr size_t kSlabBytes = (size_t)1 << 30;

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
  const long most = (long)(kSlabBytes / ((size_t)mx4_slices(K) * (kMx4CodeTile / 16))) & ~255L;
  for (long m = 0; m < M; m += most) {
    GemmParams p;
    p.x = g.x.codes + (size_t)(m / 16) * mx4_slices(K) * kMx4CodeTile;
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
    hipError_t e = plan.tile == 0 ? run_wide<4, 8>(p, plan, stream) : run_wide<1, 4>(p, plan, stream);
    if (e == hipSuccess && p.partial != nullptr) {
      e = launch_splitk_reduce(p.partial, plan.splits, g.bias, g.bias_type, g.epilogue, nullptr,
                               p.y, p.M, N, stream);
    }
    if (e != hipSuccess) { return e; }
  }
  return hipSuccess;
}

}  // namespace ltx25
