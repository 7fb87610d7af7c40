// The product of two microscaled 4-bit operands (ltx25_mx4_gemm, ltx25_linear_mx4) on
// v_mfma_scale_f32_16x16x128_f8f6f4: a lane's 16 bytes of an operand are one block of 32
// and its scale is one byte of a register of the lane's, so the scales cost no arithmetic.
#include "mx4.h"

#include <algorithm>
#include <type_traits>
#include <utility>

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
  int M, N, K;
  int bias_type, epilogue;
  int tiles_m, tiles_n, group;
  bool whole;   // rows of y lie in whole pieces of 64 bytes
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, size_t bytes)
{
  // loads past `bytes` return zeros
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)(uint32_t)bytes,
                                           0x00020000);
}

// 2 W bf16 to columns n .. of a row of N, of which those past N are left alone. Rows of an
// odd N begin anywhere: the store is one all the same. `whole`: a wave's stores are whole
// pieces of 64 aligned bytes, and pass the cache by (others go through it, which puts their
// lines together: 5304 x 608 -> 11000 56 us, past it 118; 8160 x 512 -> 16376 122 and 261).
template <int W>
struct Words {
  uint32_t w[W];
};
template <int W>
__device__ __forceinline__ void store_bf16(uint16_t* row, int n, int N, bool whole,
                                           const Words<W>& v)
{
  typedef uint32_t words __attribute__((ext_vector_type(W), aligned(2)));
  if (n + 2 * W <= N) {
    words x;
#pragma unroll
    for (int i = 0; i < W; ++i) { x[i] = v.w[i]; }
    if (whole) {
      __builtin_nontemporal_store(x, (words*)(row + n));
    } else {
      // (The empty statement keeps the compiler from making one ordinary store of the two:
      // 8160 x 4096 -> 16384 340 us for 267.)
      asm volatile("" ::: "memory");
      *(words*)(row + n) = x;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) {
      if (n + i < N) { row[n + i] = (uint16_t)(v.w[i >> 1] >> (16 * (i & 1))); }
    }
  }
}

// f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>)
template <typename F, int... I>
__device__ __forceinline__ void unroll_seq(F&& f, std::integer_sequence<int, I...>)
{
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unroll(F&& f)
{
  unroll_seq(f, std::make_integer_sequence<int, N>{});
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

// Tile id -> (tile_m, tile_n): ids are dealt to the eight XCDs in turn, so each XCD gets a run of
// tiles, walked in groups of p.group rows of tiles. Few, so that a group's rows of x stay in the
// XCD's cache from one round to the next and the stores run along the output's rows: 8160 x 4096
// -> 16384 288 us in groups of 4, 292 of 8 and 302 of 16; 8160 x 512 -> 16384, bound by its
// stores, 75 of 2, 86 of 4, 101 of 8.
__device__ __forceinline__ void tile_at(int id, const GemmParams& p, int& tm, int& tn)
{
  const int total8 = p.tiles_m * p.tiles_n & ~7;
  const int at = id < total8 ? (id & 7) * (total8 >> 3) + (id >> 3) : id;
  const int per_group = p.group * p.tiles_n;
  const int first = at / per_group * p.group;
  const int rows = min(p.tiles_m - first, p.group);
  const int r = at % per_group;
  tm = first + r % rows;
  tn = r / rows;
}

// 64 RB x 16 CB outputs of a workgroup of four waves, one below the other: a wave has RB x CB
// blocks of 16 x 16. The weight's rows, which all four read, go through LDS; a wave's rows of x
// are its own and go from memory straight to its registers, DEPTH slices of 128 values ahead: LDS
// then carries 5 x 16 CB rows of K where both operands through LDS and 2 x 2 waves of the same
// size carry 3 x (64 RB + 16 CB).
//
// 8160 x 4096 -> 16384 in 272 us one after another, 4.0 PFLOP/s (250 to 305 one at a time, as power
// allows: 4.45e5 cycles, at 1.76 GHz 250 us): address units are busy in 84% of the cycles, matrix
// cores in 59, LDS in 18; on zeros as many cycles at 2.2 GHz. The instructions alone reach 7.2
// PFLOP/s on random operands.
//
// A span is 512 values: STAGES LDS stages of CB x 4 tiles of codes and all the workgroup's scales
// take turns, filled STAGES - 1 spans ahead by loads that go straight into LDS, one barrier a
// span. Tiles lie in LDS as in memory, and a fragment's read is the tile's 1 KB in the order of
// the lanes.
template <int RB, int CB, int STAGES, int DEPTH>
__global__ void __launch_bounds__(256, 2) mx4_wide_kernel(GemmParams p)
{
  static_assert(DEPTH == 4 || (DEPTH == 8 && STAGES > 2), "slices of x in flight: a span's or two");
  constexpr int kCodes = 4 * CB * kMx4CodeTile;
  constexpr int kScaleTiles = 4 * RB + CB, kScaleLoads = (kScaleTiles + 15) / 16;
  constexpr int kScaleRoom = (kScaleTiles + 3) / 4 * 4;   // four tiles a load
  constexpr int kStage = kCodes + kScaleRoom * kMx4Tile;
  // behind the stages: where loads of no tile go, and a tile's bias, a copy a wave
  constexpr int kNowhere = STAGES * kStage, kBias = kNowhere + 4 * kMx4Tile;
  constexpr int kBiases = (CB + 3) / 4;   // of 64 columns
  constexpr int kLds = kBias + 4 * 256 * kBiases;
  static_assert(kLds <= 80 * 1024, "two workgroups a CU");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.tiles_m * p.tiles_n;
  const int slices = mx4_slices(p.K), spans = mx4_spans(p.K);
  const uint32_t pitch = (uint32_t)slices * kMx4CodeTile;   // of 16 rows
  const uint32_t spitch = (uint32_t)spans * kMx4Tile;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x, mx4_code_bytes(p.M, p.K));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.w, mx4_code_bytes(p.N, p.K));
  const __amdgpu_buffer_rsrc_t xsr = make_rsrc(p.xs, mx4_scale_bytes(p.M, p.K));
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(p.ws, mx4_scale_bytes(p.N, p.K));

  // The loads run ahead of the products, those into LDS STAGES - 1 spans, those of x one; with
  // two stages over the end of a tile to the workgroup's next. Past the last tile, and in slices
  // past the rows' end (which would be the next rows'), offsets lie past the operands and give
  // zeros.
  //
  // Codes of a stage: [tile row][slice], wave w loads slice w of every tile row. Scales: tiles of
  // x, then of w, four a load; wave w has loads w, w + 4 (those past the last tile zeros).
  struct Place {
    uint32_t w, x, s[kScaleLoads];
  };
  auto place_of = [&](int tile) {
    int tm, tn;
    const bool in = tile < tiles;
    tile_at(in ? tile : 0, p, tm, tn);
    Place at;
    at.w = in ? (uint32_t)(tn * CB) * pitch + lane * 16 : kPast;
    at.x = in ? (uint32_t)((tm * 4 + wave) * RB) * pitch + lane * 16 : kPast;
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
      const int q = wave + 4 * i, t = 4 * q + g;
      const uint32_t r = q < RB ? (uint32_t)(tm * 4 * RB + t) : (uint32_t)(tn * CB + t - 4 * RB);
      at.s[i] = in && t < kScaleTiles ? r * spitch + (lane & 15) * 16 : kPast;
    }
    return at;
  };
  Place here = place_of(blockIdx.x), then = place_of(STAGES == 2 ? blockIdx.x + gridDim.x : tiles);
  constexpr int kW = CB + kScaleLoads;   // loads of a wave into a stage
  auto load_w = [&](int span, int stage, int k) {   // the k-th of them
    const bool on = span >= spans;
    const int from = on ? span - spans : span;
    uint8_t* const at = lds + stage * kStage;
    if (k < CB) {
      const int t = 4 * from + wave;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr, (lds_u32*)(at + (4 * k + wave) * kMx4CodeTile), 16,
          (int)(t < slices ? (on ? then.w : here.w) + k * pitch : kPast), t * kMx4CodeTile, 0, 0);
    } else {
      const int q = wave + 4 * (k - CB);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          q < RB ? xsr : wsr,
          (lds_u32*)(4 * q < kScaleTiles ? at + kCodes + q * 4 * kMx4Tile : lds + kNowhere), 16,
          (int)(on ? then.s[k - CB] : here.s[k - CB]), from * kMx4Tile, 0, 0);
    }
  };
  i32x4 x[DEPTH][RB];
  auto load_x = [&](int span, int slice, int buf, int i) {
    const bool on = span >= spans;
    const int t = 4 * (on ? span - spans : span) + slice;
    x[buf][i] = __builtin_bit_cast(
        i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                   xr, (int)(t < slices ? (on ? then.x : here.x) + i * pitch : kPast),
                   t * kMx4CodeTile, 0));
  };
  // A span is 4 CB fragments of w, RB matrix instructions each. Its loads go out one by one among
  // them, since a wave waits until the address unit has taken its load (all of a span's loads to
  // LDS at its start and a slice's of x behind the slice: 2.5 us a span of one workgroup a CU;
  // without those of x 1.9, without those to LDS 2.1): the k-th load to LDS at fragment 2 k,
  // and slice J - 1's registers are filled anew during slice J.
  static_assert(2 * (kW - 1) < 4 * CB && CB >= RB, "a span has room for its loads");
  // loads of x before the slice's fragment j, and those of a span behind its last one to LDS
  constexpr auto x_before = [](int j) { return j * RB / CB; };
  constexpr int kLast = 2 * (kW - 1);
  constexpr int kXBehind = 4 * RB - (kLast / CB * RB + x_before(kLast % CB));
  f32x4 acc[RB][CB];
  int stage = 0;   // of the span
  auto step = [&](int span, auto parity) {
    constexpr int B = DEPTH == 8 ? 4 * decltype(parity)::value : 0;
    // The span's loads into LDS have landed: behind them came those of x of the span that issued
    // them, and STAGES - 2 spans' since (an epilogue's accesses only add to the count). Then the
    // stage that the last span used is free.
    constexpr int kBehind = kXBehind + (STAGES - 2) * (kW + 4 * RB);
    constexpr int kWait = kBehind < 63 ? kBehind : 63;
    __builtin_amdgcn_s_waitcnt(0x0f70 | (kWait & 15) | ((kWait >> 4) << 14));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const int next = stage == 0 ? STAGES - 1 : stage - 1;
    const uint8_t* const at = lds + stage * kStage + lane * 16;
    const uint8_t* const sat = lds + stage * kStage + kCodes + lane * 4;
    int xs[RB], ws[CB];
#pragma unroll
    for (int i = 0; i < RB; ++i) { xs[i] = *(const int*)(sat + (wave * RB + i) * kMx4Tile); }
#pragma unroll
    for (int j = 0; j < CB; ++j) { ws[j] = *(const int*)(sat + (4 * RB + j) * kMx4Tile); }
    // Fragment f is slice f / CB of tile row f % CB; three are on their way from LDS while one
    // is multiplied (left to itself the compiler asks for two and waits for them).
    auto fragment = [&](int f) { return *(const i32x4*)(at + (4 * (f % CB) + f / CB) * kMx4CodeTile); };
    i32x4 w[4] = {fragment(0), fragment(1), fragment(2)};
    __builtin_amdgcn_sched_barrier(0);
    unroll<4 * CB>([&](auto ff) {
      constexpr int f = decltype(ff)::value, J = f / CB, j = f % CB;
      if constexpr (f + 3 < 4 * CB) { w[(f + 3) % 4] = fragment(f + 3); }
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        acc[i][j] = mfma_mx4<J>(w[f % 4], x[B + J][i], acc[i][j], ws[j], xs[i]);
      }
      // Unconditionally and in this order, so that the number of loads behind others is known: a
      // load of x that came before the span's last one to LDS would let the wait end before that.
      if constexpr (f % 2 == 0 && f / 2 < kW) {
        load_w(span + STAGES - 1, next, f / 2);
        if constexpr (f == kLast) { __builtin_amdgcn_sched_barrier(0); }
      }
      if constexpr (x_before(j + 1) > x_before(j)) {
        constexpr int kBuf = J > 0 ? B + J - 1 : DEPTH == 8 ? 7 - B : 3;
        load_x(span + DEPTH / 4 - (J == 0 ? 1 : 0), (J + 3) % 4, kBuf, x_before(j));
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
#pragma unroll
    for (int k = 0; k < kW; ++k) { load_w(i, i, k); }
  }
#pragma unroll
  for (int t = 0; t < DEPTH - 1; ++t) {
#pragma unroll
    for (int i = 0; i < RB; ++i) { load_x(t / 4, t % 4, t, i); }
  }
  // With more than a workgroup a CU the whole weight is asked for at the start, a word of each 64
  // bytes over all workgroups, so that later spans find it beside the memory: with each span's
  // loads the first to see their lines, a span waits for the memory behind the stores. On weights
  // not read for a while, and just read: 8160 x 4096 -> 16384 275 us for 360, and 257 for 246;
  // 4096 x 4096 -> 4096 39 for 43, 35 both; 2048 rows, one workgroup a CU, 25 for 24; tiles of
  // 128 x 64, 300 x 16384 -> 4096, 34 for 31. Up to half of what is kept.
  auto touch = [&](__amdgpu_buffer_rsrc_t r, size_t bytes) {
    const uint32_t end = (uint32_t)min(bytes, (size_t)128 << 20);
    for (uint32_t at = (blockIdx.x * 4 + wave) * 4096; at < end; at += gridDim.x * 4 * 4096) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_u32*)(lds + kNowhere), 4, (int)(at + lane * 64),
                                               0, 0, 0);
    }
  };
  if (STAGES == 2 && tiles > 256) {
    touch(wr, mx4_code_bytes(p.N, p.K));
    touch(wsr, mx4_scale_bytes(p.N, p.K));
  }
  // the first stages have landed, for what the count above does not see
  constexpr int kFirst = (DEPTH - 1) * RB;
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kFirst < 15 ? kFirst : 15));

  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
#pragma unroll
    for (int i = 0; i < RB; ++i) {
#pragma unroll
      for (int j = 0; j < CB; ++j) { acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
    }
    // The tile's bias, a column or two a lane, which has landed long before the tile is done
    int tm, tn;
    tile_at(tile, p, tm, tn);
    const int n0 = tn * 16 * CB, row0 = (tm * 4 + wave) * 16 * RB;   // the wave's rows
    float bias[kBiases];
#pragma unroll
    for (int i = 0; i < kBiases; ++i) {
      bias[i] = load_bias(p.bias, p.bias_type, min(n0 + 64 * i + lane, p.N - 1));
    }
    if constexpr (DEPTH == 8) {
      int span = 0;
      for (; span + 1 < spans; span += 2) {
        step(span, std::integral_constant<int, 0>{});
        step(span + 1, std::integral_constant<int, 1>{});
      }
      if (span < spans) { step(span, std::integral_constant<int, 0>{}); }
    } else {
      for (int span = 0; span < spans; ++span) { step(span, std::integral_constant<int, 0>{}); }
    }
    here = then;
    then = place_of(tile + 2 * (int)gridDim.x);

    // Block (i, j), lane l, register r: row 16 i + l % 16, column 16 j + 4 (l / 16) + r. The
    // loads of x that are in flight, the next tile's, have landed before anything is stored.
    float* const biases = (float*)(lds + kBias) + wave * 64 * kBiases;
#pragma unroll
    for (int i = 0; i < kBiases; ++i) { biases[64 * i + lane] = bias[i]; }
    // Two blocks side by side: the lanes' rows of 16 are exchanged so that each lane has eight
    // columns of one of them, 16 bytes.
    auto store = [&](auto gelu) {
      unroll<CB / 2>([&](auto jj) {
        constexpr int j = 2 * decltype(jj)::value;
        __builtin_amdgcn_sched_barrier(0);
        const f32x4 bias[2] = {*(const f32x4*)(biases + 16 * j + 4 * g),
                               *(const f32x4*)(biases + 16 * j + 16 + 4 * g)};
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
          if constexpr (j == 0) {
            if (i == 0) { __builtin_amdgcn_s_waitcnt(0x0f70); }
          }
          const int m = row0 + 16 * i + (lane & 15);
          if (m < p.M) {
            store_bf16<4>(p.y + (size_t)m * p.N, n, p.N, p.whole, {a[0], b[0], a[1], b[1]});
          }
        }
      });
    };
    if (p.epilogue == kEpiGelu) {
      store(std::true_type{});
    } else {
      store(std::false_type{});
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);   // no load into LDS outlives the wave
}

template <int RB, int CB, int STAGES, int DEPTH>
hipError_t run_wide(GemmParams& p, hipStream_t stream)
{
  p.tiles_m = (p.M + 64 * RB - 1) / (64 * RB);
  p.tiles_n = (p.N + 16 * CB - 1) / (16 * CB);
  p.group = p.K <= 1024 ? 2 : 4;
  const long tiles = (long)p.tiles_m * p.tiles_n;
  if (tiles * 256 >= 1L << 32) { return hipErrorInvalidConfiguration; }
  // two workgroups on each of the 256 CUs; a multiple of the XCDs, so that a workgroup's tiles
  // are its XCD's (tile_at)
  const long grid = STAGES == 2 ? std::min(tiles, 512L) : tiles;
  mx4_wide_kernel<RB, CB, STAGES, DEPTH><<<(unsigned)grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

// ---- panels: few outputs -------------------------------------------------------

// 16 RB x 16 CB outputs of a workgroup whose waves deal the spans of K among themselves: both
// operands go from memory straight to registers, a tile's 1 KB an instruction, with four slices
// in flight (the next span's slice is asked for when this span's has been multiplied), no
// barrier before the waves' sums meet in LDS. For outputs of few tiles, where a workgroup that
// walks all of K is a chain of its loads' latencies. 1 x 4096 -> 4096 5.0 us, latency; 16 x 15072
// -> 15872, 127 MB, 27.9 us, memory.
//
// CODED false: bf16 activations, up to 16 rows. A wave codes what it multiplies: four lanes
// have a block and find its largest value, and the codes change to the matrix instruction's
// lanes through LDS of the wave's own.
template <int RB, int CB, int WAVES, bool CODED>
__global__ void __launch_bounds__(64 * WAVES, WAVES >= 8 ? 2 : 1)
mx4_panel_kernel(GemmParams p, const uint16_t* xb, long stride)
{
  static_assert(CODED || (RB == 1 && CB == 1), "more rows are coded ahead");
  constexpr int kOut = 256 * RB * CB;
  constexpr int kBuf = 5 * kMx4CodeTile;   // four slices' codes, and scales
  __shared__ __attribute__((aligned(16))) uint8_t
      lds[WAVES * (CODED ? kOut * 4 : (kOut * 4 > kBuf ? kOut * 4 : kBuf))];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  const int tn = (int)(blockIdx.x % (unsigned)p.tiles_n), tm = (int)(blockIdx.x / (unsigned)p.tiles_n);
  const int slices = mx4_slices(p.K), spans = mx4_spans(p.K);
  const uint32_t pitch = (uint32_t)slices * kMx4CodeTile, spitch = (uint32_t)spans * kMx4Tile;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x, CODED ? mx4_code_bytes(p.M, p.K) : 0);
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.w, mx4_code_bytes(p.N, p.K));
  const __amdgpu_buffer_rsrc_t xsr = make_rsrc(p.xs, CODED ? mx4_scale_bytes(p.M, p.K) : 0);
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(p.ws, mx4_scale_bytes(p.N, p.K));
  const uint32_t xoff = (uint32_t)(tm * RB) * pitch + lane * 16;
  const uint32_t woff = (uint32_t)(tn * CB) * pitch + lane * 16;
  const uint32_t xsoff = (uint32_t)(tm * RB) * spitch + lane * 4;
  const uint32_t wsoff = (uint32_t)(tn * CB) * spitch + lane * 4;

  i32x4 w[4][CB], x[4][RB];
  uint4 raw[4][CODED ? 1 : 4];
  int ws[CB], xs[RB], nws[CB], nxs[RB];
  auto load = [&](int t, int j) {   // slice t; past the rows' end zeros
    const bool in = t < slices;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      w[j][c] = __builtin_bit_cast(
          i32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, (int)(in ? woff + c * pitch : kPast),
                                                       t * kMx4CodeTile, 0));
    }
    if constexpr (CODED) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        x[j][i] = __builtin_bit_cast(
            i32x4, __builtin_amdgcn_raw_buffer_load_b128(xr, (int)(in ? xoff + i * pitch : kPast),
                                                         t * kMx4CodeTile, 0));
      }
    } else {
      // lane l: values 8 (l % 16) .. of row 4 i + l / 16; past K the row's first ones, unused
      const int at = t * 128 + row * 8;
      const uint16_t* const from = xb + (at < p.K ? at : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (4 * i < p.M) { raw[j][i] = *(const uint4*)(from + min(4 * i + g, p.M - 1) * stride); }
      }
    }
  };
  auto load_scales = [&](int span) {
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      nws[c] = __builtin_amdgcn_raw_buffer_load_b32(wsr, (int)(wsoff + c * spitch), span * kMx4Tile, 0);
    }
    if constexpr (CODED) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        nxs[i] = __builtin_amdgcn_raw_buffer_load_b32(xsr, (int)(xsoff + i * spitch), span * kMx4Tile, 0);
      }
    }
  };
  f32x4 acc[RB][CB] = {};
  auto multiply = [&](auto sl) {
    constexpr int J = decltype(sl)::value;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        acc[i][c] = mfma_mx4<J>(w[J][c], x[J][i], acc[i][c], ws[c], xs[i]);
      }
    }
  };
  // the wave's rows of x coded, from raw to x and xs
  uint8_t* const own = lds + wave * kBuf;
  auto code = [&](int span) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = (4 * span + j) * 128 + row * 8 < p.K;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (4 * i >= p.M) { break; }
        uint32_t scale;
        const uint32_t codes = mx4_code_bf16_quad(raw[j][i], scale);
        // row / 4 is the block of the slice, row % 4 the lane's place in it
        const int at = (row >> 2) * 16 + 4 * i + g;
        *(uint32_t*)(own + j * kMx4CodeTile + at * 16 + (row & 3) * 4) = in ? codes : 0u;
        if ((row & 3) == 0) { own[4 * kMx4CodeTile + at * 4 + j] = in ? (uint8_t)scale : 0; }
      }
    }
    xs[0] = *(const int*)(own + 4 * kMx4CodeTile + lane * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[j][0] = *(const i32x4*)(own + j * kMx4CodeTile + lane * 16); }
  };

  if (wave < spans) {
    load_scales(wave);
#pragma unroll
    for (int j = 0; j < 4; ++j) { load(4 * wave + j, j); }
  }
  for (int span = wave; span < spans; span += WAVES) {
    __builtin_amdgcn_sched_barrier(0);   // every load is asked for before the first is used
#pragma unroll
    for (int c = 0; c < CB; ++c) { ws[c] = nws[c]; }
    if constexpr (CODED) {
#pragma unroll
      for (int i = 0; i < RB; ++i) { xs[i] = nxs[i]; }
    } else {
      code(span);
    }
    const bool more = span + WAVES < spans;
    if (more) { load_scales(span + WAVES); }
    auto slice = [&](auto sl) {
      multiply(sl);
      if (more) {
        __builtin_amdgcn_sched_barrier(0);
        load(4 * (span + WAVES) + decltype(sl)::value, decltype(sl)::value);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    slice(std::integral_constant<int, 0>{});
    slice(std::integral_constant<int, 1>{});
    slice(std::integral_constant<int, 2>{});
    slice(std::integral_constant<int, 3>{});
  }

  // the waves' sums, in one order; block (i, c), lane l: row 16 i + l % 16, columns 16 c +
  // 4 (l / 16) .. of it
  float* const red = (float*)lds;
  if constexpr (!CODED) { __syncthreads(); }   // the codes' LDS is free
#pragma unroll
  for (int i = 0; i < RB; ++i) {
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      *(f32x4*)(red + wave * kOut + (i * 16 + row) * 16 * CB + c * 16 + g * 4) = acc[i][c];
    }
  }
  __syncthreads();
  const int used = min(WAVES, spans);
  for (int t = threadIdx.x * 4; t < kOut; t += 256 * WAVES) {
    const int m = tm * 16 * RB + t / (16 * CB), n = (tn * 16 * CB) + t % (16 * CB);
    if (m >= p.M || n >= p.N) { continue; }
    f32x4 v = *(const f32x4*)(red + t);
    for (int k = 1; k < used; ++k) { v += *(const f32x4*)(red + k * kOut + t); }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] += load_bias(p.bias, p.bias_type, min(n + r, p.N - 1));
      if (p.epilogue == kEpiGelu) { v[r] = gelu_tanh(v[r]); }
    }
    store_bf16<2>(p.y + (size_t)m * p.N, n, p.N, false,
                  {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
  }
}

template <int RB, int CB, int WAVES, bool CODED = true>
hipError_t run_panel(GemmParams& p, hipStream_t stream, const uint16_t* xb = nullptr,
                     int64_t stride = 0)
{
  p.tiles_m = (p.M + 16 * RB - 1) / (16 * RB);
  p.tiles_n = (p.N + 16 * CB - 1) / (16 * CB);
  const long tiles = (long)p.tiles_m * p.tiles_n;
  if (tiles * 64 * WAVES >= 1L << 32) { return hipErrorInvalidConfiguration; }
  mx4_panel_kernel<RB, CB, WAVES, CODED>
      <<<(unsigned)tiles, 64 * WAVES, 0, stream>>>(p, xb, (long)stride);
  return hipGetLastError();
}

// Bytes of a launch's rows of x
constexpr size_t kSlabBytes = (size_t)1 << 30;

}  // namespace

// Tiles of a wide workgroup, 64 RB x 16 CB, and of a panel, 16 RB x 16 CB
enum Tile : int { kWide48, kWide46, kWide44, kWide24, kWide14, kPanel22, kPanel22x8, kPanel21, kPanel11 };

Mx4Plan plan_mx4(int M, int K, int N, bool bf16)
{
  auto groups = [&](int rows, int columns) {
    return (long)((M + rows - 1) / rows) * ((N + columns - 1) / columns);
  };
  Mx4Plan r;
  // Rows that every workgroup of panels would code again cost 0.7 us for each time around the
  // CUs, step of a wave's and four rows (1 x 15072 -> 15872, 16 of them: 37.5 us; 16 x 4096 ->
  // 4096, 4: 6.8), a launch ahead 2.6 (26.1 + 2.6; 5.8 + 2.6).
  const long coding = (groups(16, 16) + 255) / 256 * ((mx4_spans(K) + 7) / 8) * ((M + 3) / 4);
  r.codes_ahead = bf16 && (M > 16 || coding > 4);
  // The largest tile whose rows are half there and that still gives three CUs of four a workgroup,
  // wide ones first (us; M x K -> N, replayed in a graph). Columns are not asked for: with few of
  // them many rows take tiles that are mostly empty (16384 x 4096 -> 8 9.2 us, by panels 7.4; 50000
  // 21.9 and 21.3, 200000 87 and 78; at 32 columns 9.2 and 7.8, 21.4 and 21.7).
  //                         256 x 128  256 x 64  128 x 64  64 x 64  32 x 32  32 x 16 (8 waves)
  //   8160 x 4096 -> 4096        64        81        92      128      173
  //   1024 x 4096 -> 4096        17.4      12.8      13.7     18.9     26.3
  //    512 x 4096 -> 4096        17.2      12.0       9.8     11.4     16.0
  //    256 x 4096 -> 4096        16.8      11.0       8.1      6.2      9.7
  //    333 x 2080 -> 1001        21.0      12.7       8.5      6.7      4.7      5.7
  //     64 x 4096 -> 4096                                      7.1      4.5      4.9
  //     32 x 4096 -> 4096                                      7.0      4.0      3.8
  //    128 x 16384 -> 64                                      19.1      6.7      5.6
  // A panel of one block has the most workgroups (128 x 16384 -> 64: 4.6).
  constexpr long kEnough = 192;
  r.tile = M <= 16                                    ? kPanel11
           : M > 128 && groups(256, 128) >= kEnough ? kWide48
           : M > 128 && groups(256, 64) >= kEnough  ? kWide44
           : M > 64 && groups(128, 64) >= kEnough   ? kWide24
           : groups(64, 64) >= kEnough              ? kWide14
           : groups(32, 32) > 256                   ? kPanel22
           : groups(32, 32) >= kEnough              ? kPanel22x8
           : groups(32, 16) >= kEnough              ? kPanel21
                                                    : kPanel11;
  // Columns of blocks that a CU multiplies, in tiles of 256 x 128 and of 256 x 96 (a CU has one tile
  // of up to 256, two of more): the narrower ones read more of x for each, and are taken for four
  // fifths or less. 1024 x 4096 -> 12288 35.6 us and 33.3, 640 33.1 and 28.8, 1024 x 2048 -> 6144
  // 13.8 and 12.1; of as many columns, 8160 x 4096 -> 12288, 209 and 220.
  auto columns = [&](int cb) {
    const long tiles = groups(256, 16 * cb);
    return tiles <= 256 ? cb : (tiles + 511) / 512 * 2 * cb;
  };
  if (r.tile == kWide48 && 5 * columns(6) <= 4 * columns(8)) { r.tile = kWide46; }
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
    p.M = (int)std::min(most, M - m);
    p.N = N;
    p.K = K;
    p.bias_type = g.bias_type;
    p.epilogue = g.epilogue;
    p.whole = N % 32 == 0 && (uintptr_t)g.y % 64 == 0;
    hipError_t e = hipSuccess;
    switch (plan.tile) {
      case kWide48: e = run_wide<4, 8, 2, 4>(p, stream); break;
      case kWide46: e = run_wide<4, 6, 2, 4>(p, stream); break;
      case kWide44: e = run_wide<4, 4, 3, 4>(p, stream); break;
      case kWide24: e = run_wide<2, 4, 4, 8>(p, stream); break;
      case kWide14: e = run_wide<1, 4, 4, 8>(p, stream); break;
      case kPanel22: e = run_panel<2, 2, 4>(p, stream); break;
      case kPanel22x8: e = run_panel<2, 2, 8>(p, stream); break;
      case kPanel21: e = run_panel<2, 1, 8>(p, stream); break;
      default:
        e = g.xb != nullptr && !plan.codes_ahead
                ? run_panel<1, 1, 8, false>(p, stream, g.xb, g.xb_stride)
                : run_panel<1, 1, 8>(p, stream);
        break;
    }
    if (e != hipSuccess) { return e; }
  }
  return hipSuccess;
}

}  // namespace ltx25
