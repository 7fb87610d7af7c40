// Coding rows in microscaled 4 bits and back (ltx25_mx4_quantize_rows,
// ltx25_mx4_dequant, ltx25_mx4_pack_scales, ltx25_mx4_unpack_scales).
#include "mx4.h"

namespace ltx25 {
namespace {

constexpr int kThreads = 256;

// A workgroup codes one tile of scales, 16 rows x 512 values. A wave takes a row at a
// time, eight values a lane, so that a block's largest value is found among four lanes
// and every load and store is a whole line; the tile's 256 scales go out together.
template <bool WIDE>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(const void* x, long stride,
                                                                Mx4Args q, int spans)
{
  __shared__ uint32_t tile[kMx4Tile / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int span = (int)(blockIdx.x % (unsigned)spans);
  const int row0 = (int)(blockIdx.x / (unsigned)spans) * 16;
  const int col = span * 512 + lane * 8;
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
    float v[8];
    if constexpr (WIDE) {
      const uint32_t w[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                             raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
#pragma unroll
      for (int k = 0; k < 8; ++k) { v[k] = __uint_as_float(w[k]); }
    } else {
      const uint32_t w[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
      }
    }
    uint32_t scale;
    const uint32_t codes = mx4_code_quad(v, scale);
    if (in && row0 + r < q.rows) {
      *(uint32_t*)(q.codes + (long)(row0 + r) * (q.K >> 1) + (col >> 1)) = codes;
    }
    // zeros in blocks past K (and in rows past the last, which nothing reads)
    if ((lane & 3) == 0) { ((uint8_t*)tile)[mx4_scale_at(r, lane >> 2)] = in ? (uint8_t)scale : 0; }
  }
  __syncthreads();
  if (threadIdx.x < kMx4Tile / 4) {
    ((uint32_t*)(q.scales + (long)blockIdx.x * kMx4Tile))[threadIdx.x] = tile[threadIdx.x];
  }
}

// A workgroup expands the codes of one tile of scales.
__global__ void __launch_bounds__(kThreads) mx4_dequant_kernel(Mx4Args q, uint16_t* out, long stride,
                                                               int spans)
{
  __shared__ uint32_t tile[kMx4Tile / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int span = (int)(blockIdx.x % (unsigned)spans);
  const int row0 = (int)(blockIdx.x / (unsigned)spans) * 16;
  const int col = span * 512 + lane * 8;
  const bool in = col < q.K;
  uint32_t codes[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + wave + 4 * i;
    codes[i] = 0;
    if (in && row < q.rows) {
      codes[i] = *(const uint32_t*)(q.codes + (long)row * (q.K >> 1) + (col >> 1));
    }
  }
  if (threadIdx.x < kMx4Tile / 4) {
    tile[threadIdx.x] = ((const uint32_t*)(q.scales + (long)blockIdx.x * kMx4Tile))[threadIdx.x];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = wave + 4 * i;
    if (!in || row0 + r >= q.rows) { continue; }
    const int s = ((const uint8_t*)tile)[mx4_scale_at(r, lane >> 2)];
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t c = codes[i] >> (4 * k);
      // magnitudes m / 2: 0 1 2 3 4 6 8 12, a nibble each
      const float m = (float)((0xc8643210u >> (4 * (c & 7u))) & 15u);
      v[k] = s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(c & 8u ? -m : m, s - 128);
    }
    *(uint4*)(out + (long)(row0 + r) * stride + col) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                   pack_bf16x2(v[6], v[7]));
  }
}

// Scales between rows of K / 32 bytes and tiles; a thread moves one byte of a tile.
__global__ void __launch_bounds__(kThreads) mx4_scales_kernel(const uint8_t* in, uint8_t* out,
                                                              int rows, int blocks, int spans,
                                                              bool pack)
{
  const int row = (int)(blockIdx.x / (unsigned)spans) * 16 + (int)(threadIdx.x >> 4);
  const int block = (int)(blockIdx.x % (unsigned)spans) * 16 + (int)(threadIdx.x & 15);
  const long at = (long)blockIdx.x * kMx4Tile + mx4_scale_at(row, block);
  const bool there = row < rows && block < blocks;
  const long flat = (long)row * blocks + block;
  if (pack) {
    out[at] = there ? in[flat] : 0;
  } else if (there) {
    out[flat] = in[at];
  }
}

// One workgroup for each tile of scales
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
    mx4_quantize_kernel<true><<<grid, kThreads, 0, stream>>>(x, (long)stride, q, mx4_spans(q.K));
  } else {
    mx4_quantize_kernel<false><<<grid, kThreads, 0, stream>>>(x, (long)stride, q, mx4_spans(q.K));
  }
  return hipGetLastError();
}

hipError_t launch_mx4_dequant(const Mx4Args& q, uint16_t* out, int64_t stride, hipStream_t stream)
{
  int grid;
  if (!tiles_of(q.rows, q.K, grid)) { return hipErrorInvalidConfiguration; }
  mx4_dequant_kernel<<<grid, kThreads, 0, stream>>>(q, out, (long)stride, mx4_spans(q.K));
  return hipGetLastError();
}

hipError_t launch_mx4_scales(const uint8_t* in, uint8_t* out, int rows, int K, bool pack,
                             hipStream_t stream)
{
  int grid;
  if (!tiles_of(rows, K, grid)) { return hipErrorInvalidConfiguration; }
  mx4_scales_kernel<<<grid, kThreads, 0, stream>>>(in, out, rows, K / 32, mx4_spans(K), pack);
  return hipGetLastError();
}

}  // namespace ltx25
