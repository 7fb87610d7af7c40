// Attention of packed prompts: out = softmax(scale q k^T) v per sequence and
// head, in one pass over the keys with a running maximum and sum.
//
// A workgroup holds 32 query rows in each of its waves and walks the keys in
// tiles of 64 tokens. A wave computes the tile's logits transposed,
// S^T = K Q^T on v_mfma_f32_32x32x16_bf16, so that a lane holds half of one
// row's 64 logits: the row's maximum and sum are the lane's own and one swap
// with the other half's lane. exp(S^T - m) rounded to bf16 is then, register
// for register, the right operand of O^T = V^T P^T on the same instruction: its
// k index runs over the tokens in the order in which the first product's
// registers hold them, and V^T's fragments are read from LDS in that order by
// the transposing LDS read (4 tokens x 16 channels for each 16 lanes).
//
// K and V tiles go from global memory straight into LDS (16 bytes a lane), the
// loads in flight counted by hand. Their rows' 16-byte pieces are swizzled on the
// way in (the source address is permuted, the LDS side of such a load is linear)
// so that the fragment reads meet no bank twice (the conflicts counted, 250 cycles a
// workgroup however many its tiles, are the output's on its way through LDS).
//
// What bounds it: a tile takes a wave 32 products of 32 cycles on the matrix
// cores and about 120 operations for the weights, 32 of them exponentials at 9
// cycles and the rest at 4 to 5 each. Two waves a SIMD overlap them only in part, since
// a product also takes about 16 cycles of the other wave's issue: of long prompts'
// cycles the matrix cores are busy in 66%, at head width 64 in 50 to 55%, where vector
// operations take 69 to 76%. The instructions' energy counts as well: 17% fewer cycles
// (attention_turns_kernel against attention_kernel) came at 10% less clock. The weights
// are rounded to bf16 as the values are; the sums and statistics are f32.
// Two forms:
//   attention_kernel: 4 waves, 128 rows; two to four such workgroups share a CU
//   and one computes while another waits.
//   attention_turns_kernel (head width 128): 8 waves, 256 rows, in two groups
//   that take turns with the matrix cores.
// The second is the faster one from two rounds of workgroups on and for sequences
// that are long on average; whole calls of 32 heads (8 of keys), first and second form:
//   one causal prompt of 333 tokens      12.6 us   14.7
//                        2048              52        56
//                        4096             148       130
//                       16384            2032      1890 (1163 TFLOP/s)
//   eight of 1024                          95        98
//   four of 2048                          156       149
//   8000 tokens beside 200, 100 and 60    495       471
//   8160 that all see each other, 32 heads of keys  1015  918 (1188 TFLOP/s)
// on a card whose power allowed 3% less than another's.
#include "attention.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace ltx25 {
namespace {

constexpr int kBN = 64;   // tokens of a tile

// A bit for each of a lane's D / 2 elements
template <int D>
using Bits = std::conditional_t<D == 64, uint32_t, uint64_t>;

// The weights are 2^(logit - maximum - kShift). With 8, 16 and 32 a long prompt takes 0.6 to
// 1% less time than with 0, 4 and 12, at the same instructions (16384 causal tokens: 1771, 1768
// and 1765 us for 1782, 1787 and 1789). 8, since a product with the smallest normal value,
// 2^-126, then keeps 15 bits, and with 32 none.
constexpr float kShift = 8.0f, kOne = 256.0f;
constexpr float kMost = 4096.0f / kOne;   // what a lane's weights may sum to under an old maximum

struct PromptParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* lse;
  const int* cu_q;
  const int* cu_k;
  long qs, ks, vs, os;
  int heads, share;       // share: query heads of a kv head
  int batch, total_q, total_k;
  int causal;
  float c;                // scale log2(e): the softmax runs on powers of two
  int hp_log2, tb_log2;   // a workgroup's rows: 2^hp heads x 2^tb tokens
  int head_groups;
  int splits;             // parts of a row's keys
  float* part;            // [total_q][heads][splits][D] means, then [total_q][heads][splits][2]
};                        // maximum and sum

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c)
{
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Where the 16-byte piece `c` of a tile's row lies. K rows are read 16 bytes a
// lane, lane = row: 16 rows in a run take 16 different pieces. V rows are read
// 4 rows x 64 bytes (for each half of the wave): the 4 take different quarters.
template <int D>
__device__ __forceinline__ int k_piece(int row, int c)
{
  return D == 128 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_piece(int row, int c)
{
  return D == 128 ? c ^ ((row & 3) << 2) : c ^ (((row >> 1) & 1) << 2);
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes a lane from the buffer straight into LDS, lane after lane from the LDS
// address `to`. In asm, so that the compiler does not make every LDS read wait for
// it; the kernel counts the loads in flight itself. Nothing else in these kernels
// uses m0.
__device__ __forceinline__ void load_lds(i32x4 from, uint32_t to, int offset)
{
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(to), "v"(offset), "s"(from)
               : "memory");
}

// A buffer over `bytes` bytes at p, as the asm takes it
__device__ __forceinline__ i32x4 words_of(const void* p, uint32_t bytes)
{
  const uint64_t a = (uint64_t)p;
  return i32x4{(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xffffu), (int)bytes, 0x00020000};
}

// A barrier that the scheduler moves nothing across
__device__ __forceinline__ void meet()
{
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
template <int P>
__device__ __forceinline__ void prio() { __builtin_amdgcn_s_setprio(P); }

// At most N of the wave's loads are still in flight, and every wave has come here
template <int N>
__device__ __forceinline__ void landed()
{
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
  __syncthreads();
}

// V^T's fragment: 4 tokens at a, 4 at b, of the lane's channel
__device__ __forceinline__ bf16x8 turned(const uint8_t* a, const uint8_t* b)
{
  union { s16x4 h[2]; bf16x8 f; } r;
  r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
  r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)b);
  return r.f;
}

// The compiler's scheduler moves nothing across: the order of the steps below is
// the one that overlaps the two products with the weights' arithmetic
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// The order of a block: AHEAD fragments (READS reads each) first, then product
// after product with the reads of the fragment AHEAD on
template <int N, int AHEAD, int READS>
__device__ __forceinline__ void ahead()
{
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if (i + AHEAD < N) { __builtin_amdgcn_sched_group_barrier(0x100, READS, 0); }
  }
}

// What a workgroup works on: sequence `seq`, its unit of rows counted from the
// sequence's end, and the sequence's place in the tensors.
struct Unit {
  int from_end;
  int q0, lq, k0, lk;
};

// Unit u of all sequences' units of 2^tb queries; false past the last. One
// sequence: the last unit first, which under a causal mask has the most keys. Up
// to 64 sequences: in the order of their keys, most first, so that the longest
// work does not start last; a lane holds a sequence, and the key count L where
// unit u lies is found by quartering (three sums of 6 DPP additions side by side a
// step; halving took 0.7 us longer on 12 sequences of up to 2047 tokens). More sequences: one
// after another.
__device__ __forceinline__ bool find_rows(const PromptParams& p, int u, Unit& r)
{
  const int lane = threadIdx.x & 63;
  const int tb = 1 << p.tb_log2;
  if (p.cu_q == nullptr) {
    r = {u, 0, p.total_q, 0, p.total_k};
    return u < (p.total_q + tb - 1) >> p.tb_log2;
  }
  int q0 = 0, lq = 0, k0 = 0, lk = 0;
  auto read = [&](int b) {
    const int qa = p.cu_q[b], qb = p.cu_q[b + 1], ka = p.cu_k[b], kb = p.cu_k[b + 1];
    q0 = clampi(qa, 0, p.total_q);
    lq = clampi(qb, q0, p.total_q) - q0;
    k0 = clampi(ka, 0, p.total_k);
    lk = clampi(kb, k0, p.total_k) - k0;
    return (lq + tb - 1) >> p.tb_log2;
  };
  int at = 0;
  if (p.batch == 1) {
    if (u >= read(0)) { return false; }
    r.from_end = u;
  } else if (p.batch > 64) {
    int seq;
    if (!find_unit(u, p.batch, read, seq, r.from_end, at)) { return false; }
  } else {
    const int n = lane < p.batch ? read(lane) : 0;
    const int most = (lk + tb - 1) >> p.tb_log2;   // the last unit's keys, in units
    // units of the lane's sequence with at least L keys
    auto with = [&](int L) { return p.causal ? clampi(most - L + 1, 0, n) : most >= L ? n : 0; };
    auto total = [&](int v) { return __builtin_amdgcn_readlane(scan_sum(v), 63); };
    // units that see no key count as having none or less: they come last
    const bool blind = __any(lq > lk);
    int lo = blind ? -(p.total_q >> p.tb_log2) - 1 : 0, hi = (int)wave_max((uint32_t)most) + 1;
    if (total(n) <= u) { return false; }
    while (hi - lo > 1) {   // with(lo) > u >= with(hi), which falls from lo to hi
      const int q = (hi - lo + 3) >> 2;
      const int x = total(with(lo + q)), y = total(with(lo + 2 * q)), z = total(with(lo + 3 * q));
      lo += q * ((x > u) + (y > u) + (z > u));
      hi = min(hi, lo + q);
    }
    const int before = with(lo + 1);
    const int here = with(lo) - before;
    const int place = u - total(before);
    const int sum = scan_sum(here);
    at = __builtin_ctzll(__ballot(sum > place));
    r.from_end = __builtin_amdgcn_readlane(before, at) + place -
                 __builtin_amdgcn_readlane(sum - here, at);
  }
  r.q0 = __builtin_amdgcn_readlane(q0, at);
  r.lq = __builtin_amdgcn_readlane(lq, at);
  r.k0 = __builtin_amdgcn_readlane(k0, at);
  r.lk = __builtin_amdgcn_readlane(lk, at);
  return true;
}

// A wave's rows and the workgroup's tiles.
template <int D, int NW>
struct Rows {
  int q0, lq, k0, lk;   // the sequence
  int tok0, head0, g;   // first token and head of the workgroup, kv head
  int tok, head;        // of the lane's row
  bool valid;
  int limit;            // the last key that the lane's row sees
  int wave_lo, wave_hi; // and that the wave's first and last rows see
  int first, end;       // the workgroup's tiles
};

// The row of the workgroup's rows that the lane holds
template <int D, int NW>
__device__ __forceinline__ void find_row(const PromptParams& p, Rows<D, NW>& r, int lane)
{
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = wave * 32 + (lane & 31);
  r.head = r.head0 + (row >> p.tb_log2);
  r.tok = r.tok0 + (row & ((1 << p.tb_log2) - 1));
  r.valid = r.tok < r.lq;
  r.limit = p.causal ? min(min(r.tok, r.lq - 1) + r.lk - r.lq, r.lk - 1) : r.lk - 1;
}

template <int D, int NW>
__device__ __forceinline__ bool find(const PromptParams& p, Rows<D, NW>& r, bool split)
{
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tb = 1 << p.tb_log2;
  int hg, u;
  if (p.head_groups % 8 == 0) {
    // workgroups go round-robin to the 8 XCDs: a kv head's stay on one, in
    // whose L2 its keys and values then are
    const int per = p.head_groups >> 3;
    const int i = blockIdx.x >> 3;
    hg = (blockIdx.x & 7) * per + i % per;
    u = i / per;
  } else {
    hg = blockIdx.x % p.head_groups;
    u = blockIdx.x / p.head_groups;
  }
  Unit un;
  if (!find_rows(p, u, un)) { return false; }
  r.q0 = un.q0;
  r.lq = un.lq;
  r.k0 = un.k0;
  r.lk = un.lk;
  r.tok0 = (((un.lq + tb - 1) >> p.tb_log2) - 1 - un.from_end) << p.tb_log2;
  r.head0 = hg << p.hp_log2;
  r.g = r.head0 / p.share;
  find_row(p, r, lane);
  const int shift = p.causal ? r.lk - r.lq : 0;
  auto last_key = [&](int t) { return p.causal ? min(t + shift, un.lk - 1) : un.lk - 1; };
  const int lo = r.tok0 + (p.tb_log2 >= 5 ? (wave * 32) & (tb - 1) : 0);
  const int hi = min(lo + min(tb, 32), r.lq) - 1;
  r.wave_lo = lo < r.lq ? last_key(lo) : -1;
  r.wave_hi = lo < r.lq ? last_key(hi) : -1;
  const int last = last_key(min(r.tok0 + tb, r.lq) - 1);
  const int n_tiles = last < 0 ? 0 : last / kBN + 1;
  r.first = 0;
  r.end = n_tiles;
  if (split) {
    const int per = (n_tiles + p.splits - 1) / p.splits;
    r.first = min((int)blockIdx.y * per, n_tiles);
    r.end = min(r.first + per, n_tiles);
  }
  return true;
}

// The lane's row's queries, 8 channels of each 16
template <int D, int NW>
__device__ __forceinline__ void load_queries(const PromptParams& p, const Rows<D, NW>& r,
                                             bf16x8 (&qf)[D / 16])
{
  const int half = (threadIdx.x >> 5) & 1;
  const uint16_t* const qp =
      p.q + (long)(r.q0 + min(r.tok, r.lq - 1)) * p.qs + r.head * D + half * 8;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) { qf[i] = as_bf16x8(*(const uint4*)(qp + i * 16)); }
}

// The loads of K and V into LDS, tile after tile: instruction i of a wave fills 1
// KB, kRowsPer rows. Every tile is asked for by the same number of instructions,
// past the last one too (of no bytes), so that the counts of loads in flight hold
// everywhere.
template <int D, int NW>
struct Loader {
  static constexpr int kRow = D * 2;             // bytes of a row
  static constexpr int kTile = kBN * kRow;       // bytes of a stage
  static constexpr int kPieces = kRow / 16;
  static constexpr int kRowsPer = 64 / kPieces;  // rows of one instruction
  static constexpr int kLoads = kBN / kRowsPer / NW;   // of K, and of V, per wave
  static_assert(kLoads >= 1 && kLoads * NW * kRowsPer == kBN, "the waves load whole tiles");

  uint32_t lds0, k_bytes, v_bytes;
  int koff[kLoads], voff[kLoads];
  const uint16_t* kp;   // the next tile of K, the next of V, and the rows left
  const uint16_t* vp;
  long k_step, v_step;
  int k_left, v_left;

  __device__ __forceinline__ Loader(const PromptParams& p, const Rows<D, NW>& r, uint8_t* lds)
  {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    k_bytes = (uint32_t)p.ks * 2u;
    v_bytes = (uint32_t)p.vs * 2u;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (wave * kLoads + i) * kRowsPer + lane / kPieces;
      koff[i] = (int)(row * k_bytes + k_piece<D>(row, lane % kPieces) * 16);
      voff[i] = (int)(row * v_bytes + v_piece<D>(row, lane % kPieces) * 16);
    }
    lds0 = (uint32_t)(uintptr_t)(lds_word*)lds + wave * kLoads * 1024;
    kp = p.k + (long)(r.k0 + r.first * kBN) * p.ks + r.g * D;
    vp = p.v + (long)(r.k0 + r.first * kBN) * p.vs + r.g * D;
    k_step = (long)kBN * p.ks;
    v_step = (long)kBN * p.vs;
    k_left = v_left = min(r.end * kBN, r.lk) - r.first * kBN;
  }
  // the next tile into stage `st`, of the stages of K, then those of V
  __device__ __forceinline__ void keys(int st)
  {
    const int rows = min(k_left, kBN);
    const i32x4 from = words_of(kp, rows > 0 ? (uint32_t)(rows - 1) * k_bytes + kRow : 0u);
    kp += k_step;
    k_left -= kBN;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) { load_lds(from, lds0 + st * kTile + i * 1024, koff[i]); }
  }
  __device__ __forceinline__ void values(int st)
  {
    const int rows = min(v_left, kBN);
    const i32x4 from = words_of(vp, rows > 0 ? (uint32_t)(rows - 1) * v_bytes + kRow : 0u);
    vp += v_step;
    v_left -= kBN;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) { load_lds(from, lds0 + st * kTile + i * 1024, voff[i]); }
  }
};

// Fragments, by the order in which the products take them: the first product's
// step i is k chunk i / 2 of tokens 32 (i % 2) .., the second's 16 tokens i / (D /
// 32) of channels 32 (i % (D / 32)) ..
template <int D>
__device__ __forceinline__ bf16x8 k_frag(const uint8_t* kt, int i)
{
  const int lane = threadIdx.x & 63;
  const int r = (i & 1) * 32 + (lane & 31);
  return as_bf16x8(*(const uint4*)(kt + r * D * 2 + k_piece<D>(r, (i & ~1) + (lane >> 5)) * 16));
}
template <int D>
__device__ __forceinline__ bf16x8 v_frag(const uint8_t* vt, int i)
{
  const int lane = threadIdx.x & 63;
  const int r = i / (D / 32) * 16 + (lane >> 5) * 4 + ((lane & 15) >> 2);
  const int piece = i % (D / 32) * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  const int low = (lane & 1) * 8;
  return turned(vt + r * D * 2 + v_piece<D>(r, piece) * 16 + low,
                vt + (r + 8) * D * 2 + v_piece<D>(r + 8, piece) * 16 + low);
}

// -infinity for what a row does not see of tile t, of which s[b][i] is token
// 32 b + (i & 3) + 8 (i >> 2) + 4 half
template <int D, int NW>
__device__ __forceinline__ void mask(const Rows<D, NW>& r, int t, f32x16 (&s)[2])
{
  if (t * kBN + kBN - 1 > r.wave_lo) {
    const int lim = r.limit - t * kBN - 4 * (int)((threadIdx.x >> 5) & 1);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = b * 32 + (i & 3) + 8 * (i >> 2) > lim ? -INFINITY : s[b][i];
      }
    }
  }
}

// Whether one of 8 bf16 is an infinity or a NaN
__device__ __forceinline__ bool not_finite(uint4 v)
{
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    any = any || (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  }
  return any;
}

// 8 bf16, each as pick() makes it of its bits
template <typename Pick>
__device__ __forceinline__ bf16x8 each_bf16(bf16x8 f, Pick&& pick)
{
  const uint4 v = __builtin_bit_cast(uint4, f);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[i] = pick(w[i] & 0xffffu) | pick(w[i] >> 16) << 16; }
  return as_bf16x8(make_uint4(x[0], x[1], x[2], x[3]));
}

// The wave's rows' means again, for the elements whose bits are set in `open`: those that
// the sums left not finite (bit 16 d + i: register i of o[d]), `was_nan` those that are a NaN.
// A sum of weights up to 2^12 times values near f32's end passes it though the mean does not.
// A weight of zero times a value that is not finite is a NaN, and a causal tile's masked
// tokens take part in the second product, so that a row can show what it does not see.
//
// First the values alone, 32 tokens at a time, for infinities and NaN that the rows do see: a
// block that has any is multiplied as indicators of each kind. Weights are positive, so an
// element that sees infinities of one sign is that infinity; one that sees a NaN, both signs,
// or an infinity under a logit of -infinity, whose weight is zero, is a NaN. An element that has
// shown itself a NaN is settled, as is an infinity of one that was no NaN, and where all are,
// the wave is done. What is then left saw finite values alone: its mean is taken over the keys
// once more, with every value that is not finite as 0. It is kept as a mean, halved, that each
// block moves: no sum leaves f32's range.
//
// `mine`: the wave's own 32 rows of LDS. Rare, and no faster than that asks for: one value that
// is not finite in the last of 8192 causal tokens, 32 / 8 heads of 128, makes the call 1.6 ms
// for 0.5 (117 ms when the rows were taken one at a time), values that are all infinite 4.6 (239).
// What rows do see costs them the values up to it once more: an infinity in the last of 16384
// tokens that all see each other 8.6 ms for 3.5, a NaN in the middle of a causal prompt 3.2 for 1.9.
template <bool SPLIT, int D, int NW>
__device__ __forceinline__ void again(const PromptParams& p, const Rows<D, NW>& r, uint8_t* mine,
                                      Bits<D> open, Bits<D> was_nan)
{
  constexpr int kRow = D * 2, kPieces = kRow / 16, kRowsPer = 64 / kPieces, kDT = D / 32;
  constexpr int kKC = D / 16, kBlock = 32;
  const int begin = r.first * kBN, end = min(r.end * kBN, r.wave_hi + 1);
  // the lane's row found anew, so that the loops before this hold no registers for it
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int half = lane >> 5;
  Rows<D, NW> x = r;
  find_row(p, x, lane);
  const int tok = x.tok, head = x.head, limit = x.limit;
  const int row0 = lane / kPieces, piece = lane % kPieces;   // of the values that the lane fetches

  // s[i]: token t0 + (i & 3) + 8 (i >> 2) + 4 half
  f32x16 s;
  auto logits = [&](int t0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { s[i] = 0.0f; }
    const uint16_t* const kp = p.k + (long)(r.k0 + min(t0 + (lane & 31), r.lk - 1)) * p.ks +
                               r.g * D + half * 8;
    const uint16_t* const qp =
        p.q + (long)(r.q0 + min(tok, r.lq - 1)) * p.qs + head * D + half * 8;
    fence();
#pragma unroll
    for (int c = 0; c < kKC; ++c) {
      s = mfma32(as_bf16x8(*(const uint4*)(kp + c * 16)),
                 as_bf16x8(*(const uint4*)(qp + c * 16)), s);
    }
    fence();
  };
  // the block's values into LDS, if any is not finite (which is the answer) or `all`
  auto fetch = [&](int t0, bool all) {
    uint4 v[kBlock / kRowsPer];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kBlock / kRowsPer; ++i) {
      const int row = i * kRowsPer + row0;
      v[i] = *(const uint4*)(p.v + (long)(r.k0 + min(t0 + row, r.lk - 1)) * p.vs + r.g * D +
                             piece * 8);
    }
#pragma unroll
    for (int i = 0; i < kBlock / kRowsPer; ++i) { bad = bad || not_finite(v[i]); }
    bad = any_lane(bad);
    if (bad || all) {
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");   // the reads of the block before
#pragma unroll
      for (int i = 0; i < kBlock / kRowsPer; ++i) {
        const int row = i * kRowsPer + row0;
        *(uint4*)(mine + row * kRow + v_piece<D>(row, piece) * 16) = v[i];
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    }
    return bad;
  };
  // v_frag of 16 tokens from 16 c on and channels from 32 d on, of the lane found anew
  auto frag = [&](int c, int d) {
    const int row = c * 16 + half * 4 + ((lane & 15) >> 2);
    const int at = v_piece<D>(row, d * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1));
    const uint8_t* const x = mine + row * kRow + at * 16 + (lane & 1) * 8;
    return turned(x, x + 8 * kRow);   // 8 rows on the pieces lie alike
  };
  uint32_t pw[8];   // weights, two of bf16 each
  auto part = [&](int c) {
    return as_bf16x8(make_uint4(pw[4 * c], pw[4 * c + 1], pw[4 * c + 2], pw[4 * c + 3]));
  };

  Bits<D> plus = 0, minus = 0, nans = 0;
  for (int t0 = begin; t0 < end; t0 += kBlock) {
    if (!any_lane((open & ~(nans | (~was_nan & (plus | minus)))) != 0)) { break; }
    if (!fetch(t0, false)) { continue; }
    logits(t0);
    // 1 for a token that the row sees, 2^10 for one whose weight is zero
    const int lim = limit - t0 - 4 * half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      auto of = [&](int j) {
        return (j & 3) + 8 * (j >> 2) > lim ? 0u : s[j] == -INFINITY ? 0x4480u : 0x3f80u;
      };
      pw[i] = of(2 * i) | of(2 * i + 1) << 16;
    }
#pragma unroll 1
    for (int d = 0; d < kDT; ++d) {
      // how often the row sees values whose bits under the mask lie in lo .. hi
      auto count = [&](uint32_t mask, uint32_t lo, uint32_t hi, Bits<D>& kind) {
        f32x16 n;
#pragma unroll
        for (int i = 0; i < 16; ++i) { n[i] = 0.0f; }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          n = mfma32(each_bf16(frag(c, d),
                               [&](uint32_t x) { return (x & mask) - lo <= hi - lo ? 0x3f80u : 0u; }),
                     part(c), n);
        }
        uint32_t some = 0, none = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          some |= n[i] > 0.0f ? 1u << i : 0u;
          none |= n[i] >= 1024.0f ? 1u << i : 0u;
        }
        kind |= (Bits<D>)some << (16 * d);
        nans |= (Bits<D>)none << (16 * d);
      };
      count(0xffffu, 0x7f80u, 0x7f80u, plus);
      count(0xffffu, 0xff80u, 0xff80u, minus);
      count(0x7fffu, 0x7f81u, 0x7fffu, nans);
    }
    nans |= plus & minus;
  }
  open &= ~nans;

  f32x16 o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { o[d][i] = 0.0f; }
  }
  if (any_lane((open & ~(plus | minus)) != 0)) {
    float m = -INFINITY, l = 0.0f;
    for (int t0 = begin; t0 < end; t0 += kBlock) {
      (void)fetch(t0, true);
      logits(t0);
      const int lim = limit - t0 - 4 * half;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = (i & 3) + 8 * (i >> 2) > lim ? -INFINITY : s[i];
        top = fmaxf(top, s[i]);
      }
      const float m_new = fmaxf(m, xor32_max(top));
      const float mz = m_new == -INFINITY ? 0.0f : m_new;
      const float before = l * exp2_of((m - mz) * p.c);
      m = m_new;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = exp2_of((s[i] - mz) * p.c);
        sum += s[i];
      }
      l = before + xor32_sum(sum);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l, keep = before * inv;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        pw[i] = pack_bf16x2(s[2 * i] * (0.5f * inv), s[2 * i + 1] * (0.5f * inv));
      }
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { o[d][i] *= keep; }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          o[d] = mfma32(each_bf16(frag(c, d),
                                  [](uint32_t x) { return (x & 0x7f80u) == 0x7f80u ? 0u : x; }),
                        part(c), o[d]);
        }
        fence();
      }
    }
  }

  // behind the wave's own stores of the same elements
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  const long token = r.q0 + tok;
  uint16_t* const op = p.out + token * p.os + head * D + 4 * half;
  float* const pp =
      p.part + ((token * p.heads + head) * p.splits + blockIdx.y) * D + 4 * half;
#pragma unroll
  for (int d = 0; d < kDT; ++d) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const Bits<D> bit = (Bits<D>)1 << (16 * d + i);
      if ((open & bit) != 0) {
        // rounding may not make an infinity of a mean of finite values
        const float mean = fminf(fmaxf(o[d][i] * 2.0f, -0x1.fep127f), 0x1.fep127f);
        const float x = (plus & bit) != 0 ? INFINITY : (minus & bit) != 0 ? -INFINITY : mean;
        const int channel = d * 32 + (i & 3) + 8 * (i >> 2);
        if (SPLIT) {
          pp[channel] = x;
        } else {
          op[channel] = f32_to_bf16(x);
        }
      }
    }
  }
}

// The sums and statistics of the wave's rows out: through LDS, each wave its own
// part of it, so that a store has whole rows' pieces side by side. SPLIT: a part's means,
// maximum (log2) and sum into the workspace instead.
template <bool SPLIT, int D, int NW>
__device__ __forceinline__ void finish(const PromptParams& p, const Rows<D, NW>& r, uint8_t* lds,
                                       f32x16 (&o)[D / 32], float m, float l)
{
  constexpr int kRow = D * 2, kPieces = kRow / 16, kRowsPer = 64 / kPieces, kDT = D / 32;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  const int tb = 1 << p.tb_log2;
  l = xor32_sum(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  landed<0>();
  uint8_t* const mine = lds + wave * 32 * kRow;
  float odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // a NaN where any is not finite
#pragma unroll
  for (int d = 0; d < kDT; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = o[d][4 * i + j] * inv;
        odd[j] = fmaf(x[j], 0.0f, odd[j]);
      }
      *(uint2*)(mine + (lane & 31) * kRow + k_piece<D>(lane & 31, d * 4 + i) * 16 + half * 8) =
          make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    }
  }
#pragma unroll
  for (int i = 0; i < 32 / kRowsPer; ++i) {
    const int at = i * kRowsPer + lane / kPieces, wr = wave * 32 + at;
    const int t = r.tok0 + (wr & (tb - 1)), c = lane % kPieces;
    const uint4 v = *(const uint4*)(mine + at * kRow + k_piece<D>(at, c) * 16);
    if (!SPLIT && t < r.lq) {
      *(uint4*)(p.out + (long)(r.q0 + t) * p.os + (r.head0 + (wr >> p.tb_log2)) * D + c * 8) = v;
    }
  }
  const long row = ((long)(r.q0 + r.tok) * p.heads + r.head) * p.splits + blockIdx.y;
  if (SPLIT) {
    if (r.valid) {
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *(f32x4*)(p.part + row * D + d * 32 + i * 8 + half * 4) =
              f32x4{o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv,
                    o[d][4 * i + 3] * inv};
        }
      }
      if (half == 0) {
        *(float2*)(p.part + (long)p.total_q * p.heads * p.splits * D + row * 2) =
            make_float2(l == 0.0f ? -INFINITY : m * p.c, l * kOne);
      }
    }
  } else if (p.lse != nullptr && half == 0 && r.valid) {
    p.lse[(long)(r.q0 + r.tok) * p.heads + r.head] =
        l == 0.0f ? -INFINITY : fmaf(m, p.c, log2f(l * kOne)) * 0.69314718055994531f;
  }
  // A sum of weights that is a NaN has seen one itself
  const float any = (odd[0] + odd[1]) + (odd[2] + odd[3]);
  const bool bad = r.valid && l == l && any != any;
  if (__builtin_expect(any_lane(bad), 0)) {
    Bits<D> open = 0, nans = 0;
#pragma unroll
    for (int d = 0; d < kDT; ++d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = o[d][i] * inv;
        const Bits<D> bit = (Bits<D>)1 << (16 * d + i);
        open |= fabsf(x) < INFINITY ? 0 : bit;
        nans |= x != x ? bit : 0;
      }
    }
    again<SPLIT>(p, r, mine, bad ? open : 0, nans);
  }
}

// 4 waves, two stages of tiles: the next tile lands while this one is multiplied.
// SPLIT: few rows see many keys; a workgroup takes part blockIdx.y of its rows' tiles, and
// attention_parts_kernel joins the parts.
template <int D, bool SPLIT>
__global__ void __launch_bounds__(256, D == 64 && !SPLIT ? 4 : 2) attention_kernel(PromptParams p)
{
  constexpr int kNW = 4;
  using Load = Loader<D, kNW>;
  constexpr int kTile = Load::kTile;
  constexpr int kKC = D / 16;   // k chunks of the first product
  constexpr int kDT = D / 32;   // 32-channel tiles of the second
  static_assert(kNW * 32 * Load::kRow <= 4 * kTile, "the staged output fits the stages");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kTile];   // K 0, 1, V 0, 1

  Rows<D, kNW> r;
  if (!find(p, r, SPLIT)) { return; }
  Load load(p, r, lds);
  bf16x8 qf[kKC];
  load_queries(p, r, qf);
  load.keys(0);
  load.values(2);
  // the queries are waited for here: inside the loop the compiler's wait for them
  // would be one for the tiles under way, in every round
#pragma unroll
  for (int i = 0; i < kKC; ++i) { asm volatile("" : "+v"(qf[i])); }

  f32x16 o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { o[d][i] = 0.0f; }
  }
  // the row's maximum so far and, with c and shifted, what the weights are taken from;
  // -infinity: nothing seen yet
  float m = -INFINITY, mc = -INFINITY, l = 0.0f;

  for (int t = r.first; t < r.end; ++t) {
    // this tile is there, every wave's share of it, and no wave reads tile t - 1,
    // whose stage the next one takes
    const int st = (t - r.first) & 1;
    landed<0>();
    load.keys(st ^ 1);
    load.values(2 + (st ^ 1));
    if (t * kBN > r.wave_hi) { continue; }
    const uint8_t* const kt = lds + st * kTile;
    const uint8_t* const vt = lds + (2 + st) * kTile;

    f32x16 s[2];
    auto logits = [&]() {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[b][i] = 0.0f; }
      }
#pragma unroll
      for (int i = 0; i < 2 * kKC; ++i) { s[i & 1] = mfma32(k_frag<D>(kt, i), qf[i >> 1], s[i & 1]); }
      ahead<2 * kKC, 8, 1>();
      mask(r, t, s);
    };
    uint32_t pw[16];
    auto weigh = [&]() {
      float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = exp2_of(fmaf(s[i >> 3][2 * (i & 7)], p.c, -mc));
        const float b = exp2_of(fmaf(s[i >> 3][2 * (i & 7) + 1], p.c, -mc));
        sums[2 * (i & 1)] += a;
        sums[2 * (i & 1) + 1] += b;
        pw[i] = pack_bf16x2(a, b);
      }
      return (sums[0] + sums[1]) + (sums[2] + sums[3]);
    };
    // The weights are taken from the maximum so far, and only if a lane's sum of 32
    // passes 2^12 -- a logit that much above the maximum, a first look at any key, a
    // NaN -- the maximum is brought up to date, the sums with it, and the weights are
    // taken again, of logits multiplied again, since the registers have room for one of
    // the two: most tiles need no maximum at all (5% of the time at head width 64), and
    // weights up to 2^12 are as exact as others in floating point.
    logits();
    float sum = 0.0f;
    bool settle = t == r.first;
    if (!settle) {
      sum = weigh();
      settle = any_lane(!(sum <= kMost));
      if (settle) { logits(); }
    }
    if (settle) {
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) { top = fmaxf(top, s[i >> 4][i & 15]); }
      const float m_new = fmaxf(m, xor32_max(top));
      const float mz = m_new == -INFINITY ? 0.0f : m_new;
      const float keep = exp2_of((m - mz) * p.c);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { o[d][i] *= keep; }
      }
      mc = fmaf(mz, p.c, kShift);
      sum = weigh();
      mc = m == -INFINITY ? -INFINITY : mc;
    }
    l += sum;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bf16x8 pf = as_bf16x8(make_uint4(pw[4 * c], pw[4 * c + 1], pw[4 * c + 2], pw[4 * c + 3]));
#pragma unroll
      for (int d = 0; d < kDT; ++d) { o[d] = mfma32(v_frag<D>(vt, c * kDT + d), pf, o[d]); }
    }
  }
  finish<SPLIT>(p, r, lds, o, m, l);
}

// The parts of attention_kernel's rows joined, a row a wave. The grid's x is the other
// kernel's, so that rows of no sequence stay as they are.
template <int D>
__global__ void __launch_bounds__(256) attention_parts_kernel(PromptParams p)
{
  Rows<D, 4> r;
  if (!find(p, r, false)) { return; }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at = blockIdx.y * 4 + wave;
  const int tok = r.tok0 + (at & ((1 << p.tb_log2) - 1)), head = r.head0 + (at >> p.tb_log2);
  if (tok >= r.lq) { return; }
  const long row = (long)(r.q0 + tok) * p.heads + head;
  join_parts<D>(p.part + row * p.splits * D,
                (const float2*)(p.part + (long)p.total_q * p.heads * p.splits * D) + row * p.splits,
                p.splits, p.out + (long)(r.q0 + tok) * p.os + head * D,
                p.lse == nullptr ? nullptr : p.lse + row);
}

// 8 waves in two groups of four, one wave of each on every SIMD, that take turns:
// while one group multiplies (its tile's logits, and the weights of the tile before
// with their values), the other takes its tile's weights; a barrier ends each turn,
// and the second group runs a turn behind. What a wave asks for in its weights' turn
// -- keys two tiles on, values one on -- has the turns until the end of its next
// products to land, and goes where no group reads any more: three stages.
__global__ void __launch_bounds__(512, 2) attention_turns_kernel(PromptParams p)
{
  constexpr int D = 128, kNW = 8;
  using Load = Loader<D, kNW>;
  constexpr int kTile = Load::kTile;
  constexpr int kKC = D / 16;   // k chunks of the first product
  constexpr int kDT = D / 32;   // 32-channel tiles of the second
  constexpr int kStages = 3;
  constexpr int kAhead = 6;     // fragments read ahead
  static_assert(kNW * 32 * Load::kRow <= 2 * kStages * kTile, "the staged output fits");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStages * kTile];

  Rows<D, kNW> r;
  if (!find(p, r, false)) { return; }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Load load(p, r, lds);
  bf16x8 qf[kKC];
  load_queries(p, r, qf);
  load.keys(0);
  load.keys(1);
  load.values(kStages);
  // as in attention_kernel
#pragma unroll
  for (int i = 0; i < kKC; ++i) { asm volatile("" : "+v"(qf[i])); }

  const f32x16 zero = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f,
                       0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  f32x16 o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d) { o[d] = zero; }
  float m = -INFINITY, mc = -INFINITY, l = 0.0f;   // as in attention_kernel

  constexpr int kQK = 2 * kKC, kPV = 4 * kDT;   // products of a tile

  // s[b] holds the logits of tokens 32 b + (i & 3) + 8 (i >> 2) + 4 half of a tile,
  // pw the weights of the tile before
  f32x16 s[2];
  uint32_t pw[16];
  auto part = [&](int c) {
    return as_bf16x8(make_uint4(pw[4 * c], pw[4 * c + 1], pw[4 * c + 2], pw[4 * c + 3]));
  };
  auto first_product = [&](const uint8_t* kt) {
    bf16x8 f[kQK];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) { f[i] = k_frag<D>(kt, i); }
    fence();
#pragma unroll
    for (int i = 0; i < kQK; ++i) {
      s[i & 1] = mfma32(f[i], qf[i >> 1], i < 2 ? zero : s[i & 1]);
      if (i + kAhead < kQK) { f[i + kAhead] = k_frag<D>(kt, i + kAhead); }
      fence();
    }
  };
  auto second_product = [&](const uint8_t* vt) {
    bf16x8 f[kPV];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) { f[i] = v_frag<D>(vt, i); }
    fence();
#pragma unroll
    for (int i = 0; i < kPV; ++i) {
      o[i % kDT] = mfma32(f[i], part(i / kDT), o[i % kDT]);
      if (i + kAhead < kPV) { f[i + kAhead] = v_frag<D>(vt, i + kAhead); }
      fence();
    }
  };
  auto both_products = [&](const uint8_t* vt, const uint8_t* kt) {
    bf16x8 f[kPV + kQK];
    auto frag = [&](int i) { return i < kPV ? v_frag<D>(vt, i) : k_frag<D>(kt, i - kPV); };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) { f[i] = frag(i); }
    fence();
#pragma unroll
    for (int i = 0; i < kPV + kQK; ++i) {
      if (i < kPV) {
        o[i % kDT] = mfma32(f[i], part(i / kDT), o[i % kDT]);
      } else {
        const int j = i - kPV;
        s[j & 1] = mfma32(f[i], qf[j >> 1], j < 2 ? zero : s[j & 1]);
      }
      if (i + kAhead < kPV + kQK) { f[i + kAhead] = frag(i + kAhead); }
      fence();
    }
  };
  auto softmax = [&](int t) {
    mask(r, t, s);
    float sums[4];
    auto weigh = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j) { sums[j] = 0.0f; }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = exp2_of(fmaf(s[i >> 3][2 * (i & 7)], p.c, -mc));
        const float b = exp2_of(fmaf(s[i >> 3][2 * (i & 7) + 1], p.c, -mc));
        sums[2 * (i & 1)] += a;
        sums[2 * (i & 1) + 1] += b;
        pw[i] = pack_bf16x2(a, b);
      }
      return (sums[0] + sums[1]) + (sums[2] + sums[3]);
    };
    // as in attention_kernel, with the logits still there
    float sum = weigh();
    if (any_lane(!(sum <= kMost))) {
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) { top = fmaxf(top, s[i >> 4][i & 15]); }
      const float m_new = fmaxf(m, xor32_max(top));
      const float mz = m_new == -INFINITY ? 0.0f : m_new;
      const float keep = exp2_of((m - mz) * p.c);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { o[d][i] *= keep; }
      }
      mc = fmaf(mz, p.c, kShift);
      sum = weigh();
      mc = m == -INFINITY ? -INFINITY : mc;
    }
    l += sum;
  };

  if (r.end > 0) {
    landed<2 * Load::kLoads>();
    if (wave >= kNW / 2) { meet(); }
    int at = 0, prev = 2;   // stages of tile t, and of tile t - 1
    for (int t = 0; t < r.end; ++t) {
      const uint8_t* const kt = lds + at * kTile;
      const uint8_t* const vt = lds + (kStages + prev) * kTile;
      const int next = at == 2 ? 0 : at + 1;
      prio<1>();
      // past its last tile a wave's next logits are not used: a path without them would
      // cost registers that the loop does not have
      if (t == 0) {
        first_product(kt);
      } else if ((t - 1) * kBN <= r.wave_hi) {
        both_products(vt, kt);
      }
      prio<0>();
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
      meet();
      load.keys(prev);                // of tile t + 2
      load.values(kStages + next);    // of tile t + 1
      if (t * kBN <= r.wave_hi) { softmax(t); }
      meet();
      prev = at;
      at = next;
    }
    if (wave < kNW / 2) { meet(); }
    if ((r.end - 1) * kBN <= r.wave_hi) { second_product(lds + (kStages + prev) * kTile); }
  }

  finish<false>(p, r, lds, o, m, l);
}

template <int D>
hipError_t run(const PromptParams& p, const PromptPlan& plan, int grid, hipStream_t st)
{
  if (p.splits > 1) {
    attention_kernel<D, true><<<dim3(grid, p.splits), 256, 0, st>>>(p);
    attention_parts_kernel<D><<<dim3(grid, 32), 256, 0, st>>>(p);
  } else if (D == 128 && plan.turns) {
    attention_turns_kernel<<<grid, 512, 0, st>>>(p);
  } else {
    attention_kernel<D, false><<<grid, 256, 0, st>>>(p);
  }
  return hipGetLastError();
}

}  // namespace

PromptPlan plan_prompt(int heads, int kv_heads, int head_dim, int batch, int total_q, int total_k)
{
  PromptPlan r;
  const int share = heads / kv_heads;
  // The form that takes turns, from two rounds of its workgroups on and for sequences
  // that are long on average (the figures at the top of this file).
  r.turns = head_dim == 128 && (long)total_q * heads >= 2L * 256 * 256 && total_k / batch >= 2048;
  // rows: heads of one kv head side by side first, so that a workgroup spans few
  // tokens and little of its last tile is masked, 32 tokens of a head at least
  const int rows_log2 = r.turns ? 8 : 7;
  while (share % (2 << r.hp_log2) == 0 && r.hp_log2 < rows_log2 - 5) { ++r.hp_log2; }
  r.tb_log2 = rows_log2 - r.hp_log2;
  r.head_groups = heads >> r.hp_log2;
  r.units = (long)(total_q >> r.tb_log2) + batch;
  // Parts of the keys, for few rows: as many as make the call's time least. A tile takes
  // a workgroup 1.1 us (0.76 at head width 64), half as long again where two share a CU;
  // the join 6 us, a tenth more for each part, and the means' bytes at 4 TB/s. Measured, in
  // one part and in those chosen: 5 queries of 32 heads over 4000 keys 71 and 14 us, over
  // 16000 269 and 22; 500 over 16000 277 and 143; 2048 causal tokens of 4 heads 40 and 26.
  // Where it says one: 1200 causal tokens of 16 heads 26, 31 in two.
  const long grid = r.units * r.head_groups, tiles = (total_k / batch + kBN - 1) / kBN;
  const float rows = (float)total_q * heads, tile_us = head_dim == 128 ? 1.1f : 0.76f;
  const long most = std::min({512 / std::max(grid, 1L), tiles / 2, 64L});
  float best = tiles * tile_us;
  for (int n = 2; n <= most; ++n) {
    const float us = tiles * tile_us / n * (grid * n > 256 ? 1.55f : 1.0f) + 6.0f + 0.1f * n +
                     rows * n * (head_dim + 2) * 8 / 4e6f;
    if (us < best) {
      best = us;
      r.splits = n;
    }
  }
  if (r.splits > 1) {
    r.workspace_bytes = (size_t)total_q * heads * r.splits * (head_dim + 2) * sizeof(float);
  }
  return r;
}

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream)
{
  const PromptPlan plan =
      plan_prompt(a.heads, a.kv_heads, a.head_dim, a.batch, a.total_q, a.total_k);
  PromptParams p;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.out = a.out;
  p.lse = a.lse;
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.qs = (long)a.qs;
  p.ks = (long)a.ks;
  p.vs = (long)a.vs;
  p.os = (long)a.os;
  p.heads = a.heads;
  p.share = a.heads / a.kv_heads;
  p.batch = a.batch;
  p.total_q = a.total_q;
  p.total_k = a.total_k;
  p.causal = a.causal;
  p.c = a.scale * 1.4426950408889634f;
  p.hp_log2 = plan.hp_log2;
  p.tb_log2 = plan.tb_log2;
  p.head_groups = plan.head_groups;
  p.splits = a.workspace != nullptr ? plan.splits : 1;
  p.part = a.workspace;
  const long grid = plan.units * plan.head_groups;
  if (grid > INT_MAX) { return hipErrorInvalidConfiguration; }
  return a.head_dim == 128 ? run<128>(p, plan, (int)grid, stream)
                           : run<64>(p, plan, (int)grid, stream);
}

}  // namespace ltx25
