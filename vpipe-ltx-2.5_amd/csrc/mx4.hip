// Coding rows in microscaled 4 bits and back (ltx25_mx4_quantize_rows,
// ltx25_mx4_dequant, ltx25_mx4_pack, ltx25_mx4_unpack).
#include "mx4.h"

namespace ltx25 {
namespace {

constexpr int kThreads = 256;

// The workgroup blockIdx.x's span of 512 values of 16 rows: four tiles of codes and one of
// scales, in LDS on their way to or from memory.
struct Span {
  int row0, span, slices;   // slices: tiles of codes that the span has, 1 to 4
  uint8_t* codes;
  uint32_t* scales;
};
__device__ __forceinline__ Span span_of(const Mx4Args& q)
{
  const int spans = mx4_spans(q.K), slices = mx4_slices(q.K);
  Span s;
  s.span = (int)(blockIdx.x % (unsigned)spans);
  const int block = (int)(blockIdx.x / (unsigned)spans);
  s.row0 = block * 16;
  s.slices = min(4, slices - 4 * s.span);
  s.codes = q.codes + ((long)block * slices + 4 * s.span) * kMx4CodeTile;
  s.scales = (uint32_t*)(q.scales + (long)blockIdx.x * kMx4Tile);
  return s;
}
// Thread t's 16 bytes of the codes and word of the scales
__device__ __forceinline__ void store_span(const Span& s, const uint4* codes, const uint32_t* scales)
{
  __syncthreads();
  const int t = threadIdx.x;
  if (t < s.slices * 64) { ((uint4*)s.codes)[t] = codes[t]; }
  if (t < kMx4Tile / 4) { s.scales[t] = scales[t]; }
}
__device__ __forceinline__ void load_span(const Span& s, uint4* codes, uint32_t* scales)
{
  const int t = threadIdx.x;
  if (t < s.slices * 64) { codes[t] = ((const uint4*)s.codes)[t]; }
  if (t < kMx4Tile / 4) { scales[t] = s.scales[t]; }
  __syncthreads();
}
// Where eight codes from value 8 `lane` of the span lie in LDS
__device__ __forceinline__ int codes_at(int row, int lane)
{
  return (lane >> 4) * kMx4CodeTile + mx4_code_at(row, lane >> 2) + (lane & 3) * 4;
}

// A wave takes a row at a time, eight values a lane, so that a block's largest value is found
// among four lanes and every load is whole lines; the codes change to their tiles' order in LDS,
// which is written out whole. Bound by memory: 16384 x 4096 f32 65 us (304 MB, 4.7 TB/s), 8160 x
// 4096 bf16 15.2 (85 MB, 5.6 TB/s, partly beside the memory).
template <bool WIDE>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(const void* x, long stride,
                                                                Mx4Args q)
{
  __shared__ uint4 held[4 * kMx4CodeTile / 16];
  __shared__ uint32_t tile[kMx4Tile / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Span s = span_of(q);
  const int row0 = s.row0, col = s.span * 512 + lane * 8;
  const bool in = col < q.K;   // K is a multiple of 32: a block's four lanes agree
  uint4 raw[4][WIDE ? 2 : 1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + wave + 4 * i;
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
      raw[i][h] = make_uint4(0, 0, 0, 0);
      if (in && row < q.rows) {
        raw[i][h] = ((const uint4*)((const char*)x + ((long)row * stride + col) * (WIDE ? 4 : 2)))[h];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = wave + 4 * i;
    uint32_t scale, codes;
    if constexpr (WIDE) {
      const uint32_t w[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                             raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) { v[k] = __uint_as_float(w[k]); }
      codes = mx4_code_quad(v, scale);
    } else {
      codes = mx4_code_bf16_quad(raw[i][0], scale);
    }
    // zeros in blocks past K (and in rows past the last, which nothing reads)
    *(uint32_t*)((uint8_t*)held + codes_at(r, lane)) = codes;
    if ((lane & 3) == 0) { ((uint8_t*)tile)[mx4_scale_at(r, lane >> 2)] = in ? (uint8_t)scale : 0; }
  }
  store_span(s, held, tile);
}

// A workgroup expands a span: 16384 x 4096 28 us (170 MB, 6 TB/s; the codes are beside the memory).
__global__ void __launch_bounds__(kThreads) mx4_dequant_kernel(Mx4Args q, uint16_t* out, long stride)
{
  __shared__ uint4 held[4 * kMx4CodeTile / 16];
  __shared__ uint32_t tile[kMx4Tile / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Span sp = span_of(q);
  const int row0 = sp.row0, col = sp.span * 512 + lane * 8;
  const bool in = col < q.K;
  load_span(sp, held, tile);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = wave + 4 * i;
    if (!in || row0 + r >= q.rows) { continue; }
    const int s = ((const uint8_t*)tile)[mx4_scale_at(r, lane >> 2)];
    const uint32_t codes = *(const uint32_t*)((const uint8_t*)held + codes_at(r, lane));
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t c = codes >> (4 * k);
      // magnitudes m / 2: 0 1 2 3 4 6 8 12, a nibble each
      const float m = (float)((0xc8643210u >> (4 * (c & 7u))) & 15u);
      v[k] = s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(c & 8u ? -m : m, s - 128);
    }
    *(uint4*)(out + (long)(row0 + r) * stride + col) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                   pack_bf16x2(v[6], v[7]));
  }
}

// Between rows and a span's tiles: thread t has block t % 16 of row t / 16.
template <bool PACK>
__global__ void __launch_bounds__(kThreads) mx4_order_kernel(Mx4Args q, uint8_t* codes,
                                                             uint8_t* scales)
{
  __shared__ uint4 held[4 * kMx4CodeTile / 16];
  __shared__ uint32_t tile[kMx4Tile / 4];
  const Span s = span_of(q);
  const int r = (int)threadIdx.x >> 4, b = (int)threadIdx.x & 15, blocks = q.K >> 5;
  const int row = s.row0 + r, block = s.span * 16 + b;
  const bool in = row < q.rows && block < blocks;
  uint4* const code = (uint4*)codes + (long)row * blocks + block;
  uint8_t* const scale = scales + (long)row * blocks + block;
  uint4* const here = (uint4*)((uint8_t*)held + (b >> 2) * kMx4CodeTile + mx4_code_at(r, b));
  uint8_t* const exponent = (uint8_t*)tile + mx4_scale_at(r, b);
  if (PACK) {
    *here = in ? *code : make_uint4(0, 0, 0, 0);
    *exponent = in ? *scale : 0;
    store_span(s, held, tile);
  } else {
    load_span(s, held, tile);
    if (in) {
      *code = *here;
      *scale = *exponent;
    }
  }
}

// One workgroup for each span of 16 rows
bool tiles_of(int rows, int K, int& grid)
{
  const long n = (long)((rows + 15) / 16) * mx4_spans(K);
  grid = (int)n;
  return n < (1L << 32) / kThreads;   // threads of a launch
}

}  // namespace

hipError_t launch_mx4_quantize(const void* x, bool wide, int64_t stride, const Mx4Args& q,
                               hipStream_t stream)
{
  int grid;
  if (!tiles_of(q.rows, q.K, grid)) { return hipErrorInvalidConfiguration; }
  if (wide) {
    mx4_quantize_kernel<true><<<grid, kThreads, 0, stream>>>(x, (long)stride, q);
  } else {
    mx4_quantize_kernel<false><<<grid, kThreads, 0, stream>>>(x, (long)stride, q);
  }
  return hipGetLastError();
}

hipError_t launch_mx4_dequant(const Mx4Args& q, uint16_t* out, int64_t stride, hipStream_t stream)
{
  int grid;
  if (!tiles_of(q.rows, q.K, grid)) { return hipErrorInvalidConfiguration; }
  mx4_dequant_kernel<<<grid, kThreads, 0, stream>>>(q, out, (long)stride);
  return hipGetLastError();
}

hipError_t launch_mx4_pack(const uint8_t* codes, const uint8_t* scales, const Mx4Args& q,
                           hipStream_t stream)
{
  int grid;
  if (!tiles_of(q.rows, q.K, grid)) { return hipErrorInvalidConfiguration; }
  mx4_order_kernel<true><<<grid, kThreads, 0, stream>>>(q, const_cast<uint8_t*>(codes),
                                                        const_cast<uint8_t*>(scales));
  return hipGetLastError();
}

hipError_t launch_mx4_unpack(const Mx4Args& q, uint8_t* codes, uint8_t* scales, hipStream_t stream)
{
  int grid;
  if (!tiles_of(q.rows, q.K, grid)) { return hipErrorInvalidConfiguration; }
  mx4_order_kernel<false><<<grid, kThreads, 0, stream>>>(q, codes, scales);
  return hipGetLastError();
}

}  // namespace ltx25
