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
// K and V tiles go from global memory straight into LDS (16 bytes a lane), two
// stages. Their rows' 16-byte pieces are swizzled on the way in (the source
// address is permuted, the LDS side of such a load is linear) so that the
// fragment reads meet no bank twice.
#include "attention.h"

#include <climits>

namespace ltx25 {
namespace {

constexpr int kBN = 64;     // tokens of a tile
constexpr int kWaves = 8;   // of a workgroup

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
};

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

template <int D, int NW>
__global__ void __launch_bounds__(NW * 64) attention_kernel(PromptParams p)
{
  constexpr int kRow = D * 2;             // bytes of a row
  constexpr int kTile = kBN * kRow;       // bytes of a stage of K or V
  constexpr int kPieces = kRow / 16;
  constexpr int kRowsPer = 64 / kPieces;  // rows of one load instruction
  constexpr int kLoads = kBN / kRowsPer / NW;   // of K, and of V, per wave
  constexpr int kKC = D / 16;             // k chunks of the first product
  constexpr int kDT = D / 32;             // 32-channel tiles of the second
  static_assert(kLoads >= 1 && kLoads * NW * kRowsPer == kBN, "the waves load whole tiles");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kTile];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  const int tb = 1 << p.tb_log2;

  // ---- this workgroup's rows
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
  int seq = 0, place = 0, from = 0;
  auto len_q = [&](int b, int& q0) {
    if (p.cu_q == nullptr) { q0 = 0; return p.total_q; }
    q0 = clampi(p.cu_q[b], 0, p.total_q);
    return clampi(p.cu_q[b + 1], q0, p.total_q) - q0;
  };
  auto tiles = [&](int b) {
    int q0;
    return (len_q(b, q0) + tb - 1) >> p.tb_log2;
  };
  if (!find_unit(u, p.batch, tiles, seq, place, from)) { return; }
  int q0, k0;
  const int lq = __builtin_amdgcn_readfirstlane(len_q(seq, q0));
  q0 = __builtin_amdgcn_readfirstlane(q0);
  int lk = p.total_k;
  k0 = 0;
  if (p.cu_k != nullptr) {
    k0 = clampi(p.cu_k[seq], 0, p.total_k);
    lk = clampi(p.cu_k[seq + 1], k0, p.total_k) - k0;
    k0 = __builtin_amdgcn_readfirstlane(k0);
    lk = __builtin_amdgcn_readfirstlane(lk);
  }
  // a causal sequence's long tiles first
  const int n_units = (lq + tb - 1) >> p.tb_log2;
  const int tok0 = (n_units - 1 - place) << p.tb_log2;
  const int head0 = hg << p.hp_log2;
  const int g = head0 / p.share;

  const int row = wave * 32 + (lane & 31);
  const int head = head0 + (row >> p.tb_log2);
  const int tok = tok0 + (row & (tb - 1));
  const bool valid = tok < lq;
  // the first and last token of the wave's rows; the last key that a query sees
  const int wlo = tok0 + (p.tb_log2 >= 5 ? (wave * 32) & (tb - 1) : 0);
  const int whi = min(wlo + min(tb, 32), lq) - 1;
  const int shift = p.causal ? lk - lq : 0;
  auto last_key = [&](int t) { return p.causal ? min(t + shift, lk - 1) : lk - 1; };
  const int limit = last_key(min(tok, lq - 1));
  const int wave_lo = wlo < lq ? last_key(wlo) : -1;
  const int wave_hi = wlo < lq ? last_key(whi) : -1;
  const int wg_hi = last_key(min(tok0 + tb, lq) - 1);
  const int n_tiles = wg_hi < 0 ? 0 : wg_hi / kBN + 1;

  // ---- queries: lane's row, 8 channels of each 16
  bf16x8 qf[kKC];
  {
    const uint16_t* const qp = p.q + (long)(q0 + min(tok, lq - 1)) * p.qs + head * D + half * 8;
#pragma unroll
    for (int i = 0; i < kKC; ++i) { qf[i] = as_bf16x8(*(const uint4*)(qp + i * 16)); }
  }

  // ---- loads into LDS: instruction i of a wave fills 1 KB, kRowsPer rows
  const int lrow = lane / kPieces;
  const uint32_t ks_bytes = (uint32_t)p.ks * 2u, vs_bytes = (uint32_t)p.vs * 2u;
  auto load_tile = [&](int t, int st) {
    const int rows = min(lk - t * kBN, kBN);
    const long at = (long)k0 + (long)t * kBN;
    const __amdgpu_buffer_rsrc_t kr =
        buffer_of(p.k + at * p.ks + g * D, (uint32_t)(rows - 1) * ks_bytes + kRow);
    const __amdgpu_buffer_rsrc_t vr =
        buffer_of(p.v + at * p.vs + g * D, (uint32_t)(rows - 1) * vs_bytes + kRow);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (wave * kLoads + i) * kRowsPer + lrow;
      const int piece = k_piece<D>(r, lane % kPieces);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          kr, (lds_word*)(lds + st * kTile + (wave * kLoads + i) * 1024), 16,
          (int)(r * ks_bytes + piece * 16), 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (wave * kLoads + i) * kRowsPer + lrow;
      const int piece = v_piece<D>(r, lane % kPieces);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          vr, (lds_word*)(lds + (2 + st) * kTile + (wave * kLoads + i) * 1024), 16,
          (int)(r * vs_bytes + piece * 16), 0, 0, 0);
    }
  };

  f32x16 o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { o[d][i] = 0.0f; }
  }
  float m = -INFINITY, l = 0.0f;

  if (n_tiles > 0) { load_tile(0, 0); }
  for (int t = 0; t < n_tiles; ++t) {
    // this tile has landed (every wave's share), and no wave reads the other stage
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): the loads into LDS are counted by hand
    __syncthreads();
    const int st = t & 1;
    if (t + 1 < n_tiles) { load_tile(t + 1, st ^ 1); }
    if (t * kBN > wave_hi) { continue; }

    // ---- logits: s[b] holds tokens 32 b + (i & 3) + 8 (i >> 2) + 4 half
    const uint8_t* const kt = lds + st * kTile;
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[b][i] = 0.0f; }
      const int r = b * 32 + (lane & 31);
#pragma unroll
      for (int i = 0; i < kKC; ++i) {
        const uint4 kf = *(const uint4*)(kt + r * kRow + k_piece<D>(r, 2 * i + half) * 16);
        s[b] = mfma32(as_bf16x8(kf), qf[i], s[b]);
      }
    }
    if (t * kBN + kBN - 1 > wave_lo) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int token = t * kBN + b * 32 + (i & 3) + 8 * (i >> 2) + 4 * half;
          if (token > limit) { s[b][i] = -INFINITY; }
        }
      }
    }
    // ---- running maximum and sum
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) { top = fmaxf(top, s[b][i]); }
    }
    const float m_new = fmaxf(m, xor32_max(top));
    const float mc = m_new == -INFINITY ? 0.0f : m_new * p.c;   // nothing seen yet
    const float keep = __builtin_amdgcn_exp2f(fmaf(m, p.c, -mc));
    m = m_new;
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], p.c, -mc));
        sum += s[b][i];
      }
    }
    l = fmaf(l, keep, sum);
#pragma unroll
    for (int d = 0; d < kDT; ++d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) { o[d][i] *= keep; }
    }
    // ---- O^T += V^T P^T, 16 tokens a step
    const uint8_t* const vt = lds + (2 + st) * kTile;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4 pw;
      const f32x16& sc = s[c >> 1];
      const int e = (c & 1) * 8;
      pw.x = pack_bf16x2(sc[e + 0], sc[e + 1]);
      pw.y = pack_bf16x2(sc[e + 2], sc[e + 3]);
      pw.z = pack_bf16x2(sc[e + 4], sc[e + 5]);
      pw.w = pack_bf16x2(sc[e + 6], sc[e + 7]);
      const bf16x8 pf = as_bf16x8(pw);
      const int r = c * 16 + half * 4 + ((lane & 15) >> 2);
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        const int piece = d * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        const uint8_t* const a = vt + r * kRow + v_piece<D>(r, piece) * 16 + (lane & 1) * 8;
        const uint8_t* const b = vt + (r + 8) * kRow + v_piece<D>(r + 8, piece) * 16 + (lane & 1) * 8;
        union { s16x4 h[2]; bf16x8 f; } vf;
        vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
        vf.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)b);
        o[d] = mfma32(vf.f, pf, o[d]);
      }
    }
  }

  // ---- out, lse
  l = xor32_sum(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  bool bad = false;
#pragma unroll
  for (int d = 0; d < kDT; ++d) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      o[d][i] *= inv;
      bad = bad || __builtin_isnan(o[d][i]);
    }
  }
  if (valid) {
    uint16_t* const op = p.out + (long)(q0 + tok) * p.os + head * D + half * 4;
#pragma unroll
    for (int d = 0; d < kDT; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2 w;
        w.x = pack_bf16x2(o[d][4 * i], o[d][4 * i + 1]);
        w.y = pack_bf16x2(o[d][4 * i + 2], o[d][4 * i + 3]);
        *(uint2*)(op + d * 32 + i * 8) = w;
      }
    }
    if (p.lse != nullptr && half == 0) {
      p.lse[(long)(q0 + tok) * p.heads + head] =
          l == 0.0f ? -INFINITY : fmaf(m, p.c, __builtin_log2f(l)) * 0.69314718055994531f;
    }
  }
  // A NaN in a row: a weight of zero times an infinite or NaN value that the
  // row does not see (a tile's masked tokens take part in the second product)
  // gives one too. Such rows are computed again over the tokens they see alone,
  // one at a time, by the whole wave: a rare case whose speed does not matter.
  unsigned long long again = __ballot(bad && valid);
  again = (again | (again >> 32)) & 0xffffffffull;
  while (again != 0) {
    const int r = __builtin_ctzll(again);
    again &= again - 1;
    const int rtok = __shfl(tok, r), rhead = __shfl(head, r), rlimit = __shfl(limit, r);
    constexpr int kPer = D / 64;
    const uint16_t* const qp = p.q + (long)(q0 + rtok) * p.qs + rhead * D + lane * kPer;
    float qv[kPer], acc[kPer], rm = -INFINITY, rl = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { qv[i] = bf16_to_f32(qp[i]); acc[i] = 0.0f; }
    for (int j = 0; j <= rlimit; ++j) {
      const uint16_t* const kp = p.k + (long)(k0 + j) * p.ks + g * D + lane * kPer;
      const uint16_t* const vp = p.v + (long)(k0 + j) * p.vs + g * D + lane * kPer;
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) { x = fmaf(qv[i], bf16_to_f32(kp[i]), x); }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) { x += __shfl_xor(x, d); }
      const float n = fmaxf(rm, x);
      const float nc = n == -INFINITY ? 0.0f : n * p.c;
      const float kept = __builtin_amdgcn_exp2f(fmaf(rm, p.c, -nc));
      const float w = __builtin_amdgcn_exp2f(fmaf(x, p.c, -nc));
      rm = n;
      rl = fmaf(rl, kept, w);
#pragma unroll
      for (int i = 0; i < kPer; ++i) { acc[i] = fmaf(acc[i], kept, w * bf16_to_f32(vp[i])); }
    }
    const float rinv = rl == 0.0f ? 0.0f : 1.0f / rl;
    uint16_t* const op = p.out + (long)(q0 + rtok) * p.os + rhead * D + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { op[i] = f32_to_bf16(acc[i] * rinv); }
  }
}

template <int D>
hipError_t run(const PromptParams& p, int grid, hipStream_t st)
{
  attention_kernel<D, kWaves><<<grid, kWaves * 64, 0, st>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream)
{
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
  // rows: heads of one kv head side by side first, so that a tile spans few
  // tokens and little of it is masked
  p.hp_log2 = 0;
  while (p.share % (2 << p.hp_log2) == 0 && p.hp_log2 < 3) { ++p.hp_log2; }
  p.tb_log2 = 8 - p.hp_log2;
  p.head_groups = a.heads >> p.hp_log2;
  const long units = (long)(a.total_q >> p.tb_log2) + a.batch;
  const long grid = units * p.head_groups;
  if (grid > INT_MAX) { return hipErrorInvalidConfiguration; }
  return a.head_dim == 128 ? run<128>(p, (int)grid, stream)
                           : run<64>(p, (int)grid, stream);
}

}  // namespace ltx25
