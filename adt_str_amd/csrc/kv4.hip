// kv4.hip -- a K/V cache held in 4 bits, and the attention that reads it (gfx950).
//
// Every 64 channels of a K or V row (one token, one head) share a scale and a minimum:
//   lo = min x, hi = max x, s = bf16(max((hi - lo) / 15, 2^-100)), m = lo, c = the integer nearest to (x - lo) / s (ties to even, at most 15)
//   and the row stands for c s + m.  A group with an infinity or a NaN (or a range past fp32): s = m = NaN.
//
// Layout: per (sequence, head) a run of tiles of 32 tokens, per tile of head_dim D one record
//   K codes 32 D / 2 | V codes 32 D / 2 | K parameters [D/64][32] | V parameters [D/64][32]        4608 bytes at D = 128 (16384 in bf16)
// laid out as the matrix instructions of the attention consume it, so that a code is unpacked where it lies and nothing is transposed:
//   K: a token's row is D/2 bytes; channel 32 g + 8 u + j is in the dword (D/32) u + g of the row: a lane's 4 D/32 bytes (token lane & 15, u = lane >> 4)
//      are its operands of the row's D/32 products over 32 channels each.
//   V: channel 16 b + i and the eight tokens 4 u + {0..3}, 16 + 4 u + {0..3} are one dword, number ((b / 4) 64 + 16 u + i) 4 + (b & 3): a lane's
//      (i = lane & 15, u = lane >> 4) 16-byte pieces are its operands of four products over 32 tokens; the token order is the one in which a lane
//      holds the scores.
//   A dword's element j is at bits 4 (j / 2) + 16 (j & 1): (w << 3), (w >> 1), (w >> 5), (w >> 9), masked to 0x00780078 and joined with 0x41804180,
//   are four pairs of the bf16 numbers 16 + c.
//   A parameter dword is the bf16 scale (low half) and the bf16 minimum (high half).
#include <hip/hip_runtime.h>

#include <cstdio>

#include "adt_common.h"

namespace adt {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kKvTile = 32;
constexpr float kKvTiny = 7.888609052210118e-31f;      // 2^-100
template <int D> struct KvRec {
  static constexpr int kG = D / 64;                    // scale groups of a row
  static constexpr int kRow = D / 2;                   // bytes of a K row's codes
  static constexpr int kV = kKvTile * kRow;            // byte offset of the V codes
  static constexpr int kKp = 2 * kV;                   // ... of the K parameters
  static constexpr int kVp = kKp + kG * kKvTile * 4;
  static constexpr int kBytes = kVp + kG * kKvTile * 4;
};
static_assert(KvRec<128>::kBytes == 4608 && KvRec<64>::kBytes == 2304, "record sizes of include/adt_hip.h");

__device__ __forceinline__ float kv_bf2f(unsigned v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ unsigned kv_f2bf(float f) { return __builtin_bit_cast(unsigned short, static_cast<__bf16>(f)); }
__device__ __forceinline__ unsigned kv_pack_bf2(float lo, float hi) {
  typedef __bf16 bf16x2_ __attribute__((ext_vector_type(2)));
  typedef float f32x2_ __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2_{lo, hi}, bf16x2_));
}

struct KvArgs {
  unsigned char* cache; int B, H, cap, tiles;          // tiles = ceil(cap / 32)
  const unsigned short *k, *v; long ldk, ldv;          // [B * n, H * D] bf16, row strides in elements
  const int *end, *count; int n;
  void *ko, *vo; long ldko, ldvo; int out32;           // read only: rows of n per sequence
};
// rows i in [0, cnt) of sequence b go to (or come from) positions end - cnt + i; positions outside [0, cap) are left out
struct KvRange { int first, lo, hi; };                 // position of row 0, and the positions touched: [lo, hi)
__device__ __forceinline__ KvRange kv_range(const KvArgs& a, int b) {
  int cnt = a.count ? a.count[b] : a.n;
  cnt = cnt < 0 ? 0 : (cnt > a.n ? a.n : cnt);
  const int end = a.end ? a.end[b] : a.cap;
  // (in 64 bits: end is the caller's word)
  const long first = static_cast<long>(end) - cnt;
  const long lo = first < 0 ? 0 : (first > a.cap ? a.cap : first), hi = end < 0 ? 0 : (end > a.cap ? a.cap : end);
  return KvRange{static_cast<int>(first < -(1L << 30) ? -(1L << 30) : first), static_cast<int>(lo), static_cast<int>(hi > lo ? hi : lo)};
}

// ------------------------------------------------------------------------------------ append
// One wave per (32-token tile, head, sequence) and side (K or V).  A lane holds eight channels of a row: D/8 lanes per row, 512 / D rows at a
// time; eight lanes share a group, whose extrema are three exchanges.  (x - lo) / s is a correctly rounded quotient: q0 = d y, y = 1 / s,
// corrected by the exact remainder fma(-q0, s, d).
// The K codes of a lane are one dword of the record.  The V codes go through LDS as bytes [token][channel] and leave as the dwords of
// eight tokens; a tile that is not written whole keeps its other tokens' codes (the wave is the only writer of its record half).
template <int D>
__global__ __launch_bounds__(128) void kv4_append_kernel(KvArgs a) {
  using R = KvRec<D>;
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;   // lanes per row, rows per pass
  __shared__ unsigned char vb[kKvTile][D + 4];
  const int lane = threadIdx.x & 63, side = threadIdx.x >> 6;      // side 0: K, 1: V
  const int b = blockIdx.z, h = blockIdx.y;
  const KvRange r = kv_range(a, b);
  const int tile = (r.lo >> 5) + static_cast<int>(blockIdx.x);
  if (tile * kKvTile >= r.hi || r.lo >= r.hi) return;  // block-uniform
  unsigned char* rec = a.cache + (static_cast<long>(b * a.H + h) * a.tiles + tile) * R::kBytes;
  const int t0 = max(r.lo - tile * kKvTile, 0), t1 = min(r.hi - tile * kKvTile, kKvTile);      // tokens of the tile that are written
  const int c8 = lane % kLanes, sub = lane / kLanes;
  const unsigned short* src = side ? a.v : a.k;
  const long ld = side ? a.ldv : a.ldk;
  unsigned* par = reinterpret_cast<unsigned*>(rec + (side ? R::kVp : R::kKp)) + (c8 >> 3) * kKvTile;
  for (int t = sub; t < kKvTile; t += kRows) {
    const bool live = t >= t0 && t < t1;
    const int tt = live ? t : t0;                      // (every lane takes part in the exchanges)
    const unsigned short* p = src + (static_cast<long>(b) * a.n + (tile * kKvTile + tt - r.first)) * ld + h * D + 8 * c8;
    float x[8];
    if (((reinterpret_cast<uintptr_t>(src) & 15) | (ld & 7)) == 0) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = kv_bf2f(p[j]);
    }
    float lo = x[0], hi = x[0];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo = fminf(lo, x[j]); hi = fmaxf(hi, x[j]);
      bad |= !(fabsf(x[j]) < INFINITY);
    }
    unsigned bb = bad ? 1u : 0u;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) { lo = fminf(lo, __shfl_xor(lo, o)); hi = fmaxf(hi, __shfl_xor(hi, o)); bb |= __shfl_xor(bb, o); }
    const float range = hi - lo;
    bad = bb != 0 || !(range < INFINITY);
    const unsigned sb = kv_f2bf(fmaxf(range / 15.0f, kKvTiny));
    const float s = kv_bf2f(sb), y = 1.0f / s;
    unsigned code[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = x[j] - lo;
      const float q0 = d * y;
      const float q = fmaf(fmaf(-q0, s, d), y, q0);
      code[j] = bad ? 0u : __float_as_uint(fminf(q, 15.0f) + 12582912.0f) & 15u;
    }
    if (live) {
      if ((c8 & 7) == 0) par[t] = bad ? 0x7fc07fc0u : (sb | (__float_as_uint(lo) & 0xffff0000u));
      if (side == 0) {
        unsigned w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= code[j] << (4 * (j >> 1) + 16 * (j & 1));
        // channels 8 c8 .. + 7 = 32 g + 8 u with g = c8 / 4, u = c8 & 3
        reinterpret_cast<unsigned*>(rec + t * R::kRow)[(D / 32) * (c8 & 3) + (c8 >> 2)] = w;
      } else {
        *reinterpret_cast<unsigned*>(&vb[t][8 * c8]) = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        *reinterpret_cast<unsigned*>(&vb[t][8 * c8 + 4]) = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
      }
    }
  }
  if (side == 0) return;
  __builtin_amdgcn_wave_barrier();                     // one wave wrote vb and reads it back: its LDS operations are in order
  unsigned* vw = reinterpret_cast<unsigned*>(rec + R::kV);
  const int i = lane & 15, u = lane >> 4;
#pragma unroll
  for (int blk = 0; blk < D / 16; ++blk) {
    unsigned w = 0, mask = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = (j < 4 ? 0 : 16) + 4 * u + (j & 3), sh = 4 * (j >> 1) + 16 * (j & 1);
      if (t >= t0 && t < t1) { w |= static_cast<unsigned>(vb[t][16 * blk + i]) << sh; mask |= 15u << sh; }
    }
    unsigned* p = vw + ((blk >> 2) * 64 + lane) * 4 + (blk & 3);
    if (mask == 0xffffffffu) *p = w;
    else if (mask) *p = (*p & ~mask) | w;
  }
}

// ------------------------------------------------------------------------------------ read
// Rows i < count of every sequence as the numbers they stand for (bf16 or fp32), the other rows of the output zeros.
template <int D, bool k32>
__global__ __launch_bounds__(128) void kv4_read_kernel(KvArgs a) {
  using R = KvRec<D>;
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;
  const int lane = threadIdx.x & 63, side = threadIdx.x >> 6;
  const int b = blockIdx.z, h = blockIdx.y;
  const KvRange r = kv_range(a, b);
  const int c8 = lane % kLanes, sub = lane / kLanes;
  void* out = side ? a.vo : a.ko;
  const long ld = side ? a.ldvo : a.ldko;
  for (int t = sub; t < kKvTile; t += kRows) {
    const int i = blockIdx.x * kKvTile + t;
    if (i >= a.n) break;
    const long pos = static_cast<long>(r.first) + i;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (pos >= r.lo && pos < r.hi) {
      const unsigned char* rec = a.cache + (static_cast<long>(b * a.H + h) * a.tiles + (pos >> 5)) * R::kBytes;
      const int tt = pos & 31;
      const unsigned par = reinterpret_cast<const unsigned*>(rec + (side ? R::kVp : R::kKp))[(c8 >> 3) * kKvTile + tt];
      const float s = kv_bf2f(par & 0xffffu), m = __uint_as_float(par & 0xffff0000u);
      if (side == 0) {
        const unsigned w = reinterpret_cast<const unsigned*>(rec + tt * R::kRow)[(D / 32) * (c8 & 3) + (c8 >> 2)];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = static_cast<float>((w >> (4 * (j >> 1) + 16 * (j & 1))) & 15u) * s + m;
      } else {
        const int u = (tt & 15) >> 2, j8 = (tt & 3) + (tt & 16 ? 4 : 0), sh = 4 * (j8 >> 1) + 16 * (j8 & 1);
        const unsigned* vw = reinterpret_cast<const unsigned*>(rec + R::kV);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = 8 * c8 + j, blk = d >> 4;
          x[j] = static_cast<float>((vw[((blk >> 2) * 64 + 16 * u + (d & 15)) * 4 + (blk & 3)] >> sh) & 15u) * s + m;
        }
      }
    }
    const long row = static_cast<long>(b) * a.n + i;
    if (k32) {
      float* p = static_cast<float*>(out) + row * ld + h * D + 8 * c8;
      reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
      reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      unsigned short* p = static_cast<unsigned short*>(out) + row * ld + h * D + 8 * c8;
      *reinterpret_cast<u32x4*>(p) = u32x4{kv_pack_bf2(x[0], x[1]), kv_pack_bf2(x[2], x[3]), kv_pack_bf2(x[4], x[5]), kv_pack_bf2(x[6], x[7])};
    }
  }
}

// ------------------------------------------------------------------------------------ attention
// A workgroup = four waves on one (sequence, K/V head, block of 16 rows, span of tiles); a row is a (query position, query head of the group)
// pair, row = position * group + head.  A wave takes every fourth tile of the span:
//   scores  S[token][row] = sum_g s_g (K codes . q)_g + m_g (sum of q)_g    two 16 x 16 x 32 bf16 products per group and 16 tokens; the codes enter as
//           16 + c, and the accumulator starts at -16 (sum of q)_g, so it ends at the sum of c q: q and the codes are exact in bf16, the sums fp32
//   softmax over the tokens: a lane holds eight tokens of one row; one running maximum per row, raised only when a score exceeds it by more
//           than 2^8 (the probabilities are then at most 2^8 and the sums stay exact to fp32), so the cross-lane exchange is rare
//   output  O[row][channel] += (p s_g) (16 + c)   the weight p s_g goes in as two bf16 numbers, upper and lower half (2^-17 of it is lost);
//           p (m_g - 16 s_g) is added up per row and group in fp32 on the side.
// The waves' (max, sum, O) join through LDS; with more than one span per head they go to the workspace and a second kernel joins them.
struct KvAttnArgs {
  const unsigned short* q; long ldq; bool qvec;        // qvec: 16-byte loads of q
  const unsigned char* cache; int B, Hk, group, cap, tiles;
  const int* key_len;
  unsigned short* out; long ldo; float* lse;
  int q_len, causal; float sl2;                        // scale * log2 e
  int rows, row_blocks, spans, span_tiles;             // rows = q_len * group
  float* part;                                         // spans > 1: [B][Hk][rows][spans][D + 2]
};
constexpr float kKvNegBig = -3.0e38f;               // below every score: the running maximum of a row that has seen no token
constexpr float kKvThr = 8.0f;

__device__ __forceinline__ float kv_max_over_groups(float v) {      // over the four lanes that share lane & 15
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float kv_sum_over_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
union KvFrag { unsigned u[4]; bf16x8 v; };
__device__ __forceinline__ KvFrag kv_unpack(unsigned w) {            // eight codes -> the bf16 numbers 16 + c
  KvFrag f;
  f.u[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
  f.u[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
  f.u[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
  f.u[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
  return f;
}

template <int D>
__global__ __launch_bounds__(256) void attn_kv4_kernel(KvAttnArgs a) {
  using R = KvRec<D>;
  constexpr int kG = R::kG, kNB = D / 16, kPieces = D / 64;          // V pieces (16 bytes) per lane and tile; K: D/64 dword pairs per 16 tokens
  __shared__ float sm[4][16], sl[4][16], sc[4][kG][16];
  __shared__ float so[4][16][D + 4];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, u = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = blockIdx.x;
  const int span = id % a.spans; id /= a.spans;
  const int rb = id % a.row_blocks; id /= a.row_blocks;
  const int hk = id % a.Hk, b = id / a.Hk;
  int klen = a.key_len ? a.key_len[b] : a.cap;
  klen = klen < 0 ? 0 : (klen > a.cap ? a.cap : klen);
  // this lane's row (as a column of the score product)
  const int row = rb * 16 + li;
  const bool live = row < a.rows;
  const int qi = live ? row / a.group : 0, qh = live ? row % a.group : 0;
  const unsigned short* qp = a.q + (static_cast<long>(b) * a.q_len + qi) * a.ldq + (hk * a.group + qh) * D + 8 * u;
  KvFrag qf[D / 32];
  float qs[kG];
#pragma unroll
  for (int g = 0; g < kG; ++g) qs[g] = 0.f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    if (a.qvec) {
      const u32x4 w = live ? *reinterpret_cast<const u32x4*>(qp + 32 * s) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[s].u[j] = w[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned lo = live ? qp[32 * s + 2 * j] : 0u, hi = live ? qp[32 * s + 2 * j + 1] : 0u;
        qf[s].u[j] = lo | hi << 16;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) qs[s / 2] += kv_bf2f(qf[s].u[j] & 0xffffu) + __uint_as_float(qf[s].u[j] & 0xffff0000u);
  }
#pragma unroll
  for (int g = 0; g < kG; ++g) qs[g] = kv_sum_over_groups(qs[g]);
  const int limit = a.causal ? klen - (a.q_len - 1 - qi) : klen;      // tokens [0, limit) are this row's
  // the tiles any row of this block can see
  const int qlast = min(rb * 16 + 15, a.rows - 1) / a.group;
  const int most = a.causal ? klen - (a.q_len - 1 - qlast) : klen;
  const int tile_end = min((max(most, 0) + kKvTile - 1) / kKvTile, (span + 1) * a.span_tiles);

  float m = kKvNegBig, l = 0.f, cb[kG];
  f32x4 o[kNB];
#pragma unroll
  for (int i = 0; i < kNB; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < kG; ++g) cb[g] = 0.f;

  const unsigned char* base = a.cache + static_cast<long>(b * a.Hk + hk) * a.tiles * R::kBytes;
  for (int tile = span * a.span_tiles + wave; tile < tile_end; tile += 4) {
    const unsigned char* rec = base + static_cast<long>(tile) * R::kBytes;
    unsigned kw[2][D / 32];
    u32x4 vw[kPieces], kp[2][kG], vp[2][kG];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const unsigned* p = reinterpret_cast<const unsigned*>(rec + (16 * hb + li) * R::kRow) + (D / 32) * u;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) kw[hb][s] = p[s];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        kp[hb][g] = *reinterpret_cast<const u32x4*>(rec + R::kKp + (g * kKvTile + 16 * hb + 4 * u) * 4);
        vp[hb][g] = *reinterpret_cast<const u32x4*>(rec + R::kVp + (g * kKvTile + 16 * hb + 4 * u) * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) vw[i] = *reinterpret_cast<const u32x4*>(rec + R::kV + (i * 64 + lane) * 16);
    // ---- scores (log2 units)
    float z[8];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      f32x4 acc[kG];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const float c0 = -16.0f * qs[g];
        acc[g] = f32x4{c0, c0, c0, c0};
#pragma unroll
        for (int s = 2 * g; s < 2 * g + 2; ++s) acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv_unpack(kw[hb][s]).v, qf[s].v, acc[g], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < kG; ++g) t += __uint_as_float(kp[hb][g][r] << 16) * acc[g][r] + __uint_as_float(kp[hb][g][r] & 0xffff0000u) * qs[g];
        z[4 * hb + r] = t * a.sl2;
      }
    }
    const int key0 = tile * kKvTile + 4 * u;
    const bool edge = (tile + 1) * kKvTile > (a.causal ? klen - (a.q_len - 1) : klen);      // block-uniform: some row does not see all of it
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = key0 + (j < 4 ? j : 12 + j);
        if (key >= limit) z[j] = kKvNegBig;
      }
    }
    float mx = z[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, z[j]);
    if (__ballot(mx > m + kKvThr) != 0) {
      const float m_new = fmaxf(m, kv_max_over_groups(mx));
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int g = 0; g < kG; ++g) cb[g] *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ar = __shfl(alpha, 4 * u + r);                    // the output's rows are 4 u + r
#pragma unroll
        for (int i = 0; i < kNB; ++i) o[i][r] *= ar;
      }
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(z[j] - m);
      if (edge && key0 + (j < 4 ? j : 12 + j) >= limit) p[j] = 0.f;
      l += p[j];
    }
    // ---- output
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      KvFrag hi, lo;
      float ps[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        unsigned par = vp[j >> 2][g][j & 3];
        if (edge && key0 + (j < 4 ? j : 12 + j) >= limit) par = 0;    // what a row does not see may be anything
        const float s = __uint_as_float(par << 16), mn = __uint_as_float(par & 0xffff0000u);
        ps[j] = p[j] * s;
        cb[g] += p[j] * mn - 16.0f * ps[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned a0 = __float_as_uint(ps[2 * j]) & 0xffff0000u, a1 = __float_as_uint(ps[2 * j + 1]) & 0xffff0000u;
        hi.u[j] = a0 >> 16 | a1;
        lo.u[j] = kv_pack_bf2(ps[2 * j] - __uint_as_float(a0), ps[2 * j + 1] - __uint_as_float(a1));
      }
#pragma unroll
      for (int i = 4 * g; i < 4 * g + 4; ++i) {
        const KvFrag vf = kv_unpack(vw[i >> 2][i & 3]);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi.v, vf.v, o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo.v, vf.v, o[i], 0, 0, 0);
      }
    }
  }
  // ---- the waves join
  l = kv_sum_over_groups(l);
#pragma unroll
  for (int g = 0; g < kG; ++g) cb[g] = kv_sum_over_groups(cb[g]);
  if (u == 0) {
    sm[wave][li] = m; sl[wave][li] = l;
#pragma unroll
    for (int g = 0; g < kG; ++g) sc[wave][g][li] = cb[g];
  }
#pragma unroll
  for (int i = 0; i < kNB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) so[wave][4 * u + r][16 * i + li] = o[i][r];
  __syncthreads();
  const int n_rows = min(16, a.rows - rb * 16);
  for (int e = tid; e < n_rows * D; e += 256) {
    const int rr = e / D, d = e % D;
    const float mm = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr]));
    float lt = 0.f, ot = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][rr] - mm);
      lt += f * sl[w][rr];
      ot += f * (so[w][rr][d] + sc[w][d >> 6][rr]);
    }
    const int orow = rb * 16 + rr, oi = orow / a.group, oh = hk * a.group + orow % a.group;
    if (a.spans == 1) {
      a.out[(static_cast<long>(b) * a.q_len + oi) * a.ldo + oh * D + d] = static_cast<unsigned short>(kv_f2bf(lt > 0.f || lt != lt ? ot / lt : 0.f));
      if (d == 0 && a.lse) a.lse[(static_cast<long>(b) * (a.Hk * a.group) + oh) * a.q_len + oi] = lt > 0.f || lt != lt ? (mm + log2f(lt)) * 0.6931471805599453f : -INFINITY;
    } else {
      float* part = a.part + (((static_cast<long>(b) * a.Hk + hk) * a.rows + orow) * a.spans + span) * (D + 2);
      part[d] = ot;
      if (d == 0) { part[D] = mm; part[D + 1] = lt; }
    }
  }
}

template <int D>
__global__ __launch_bounds__(64) void attn_kv4_join_kernel(KvAttnArgs a) {
  const int orow = blockIdx.x % a.rows, bh = blockIdx.x / a.rows, hk = bh % a.Hk, b = bh / a.Hk;
  const float* part = a.part + (static_cast<long>(bh) * a.rows + orow) * a.spans * (D + 2);
  float mm = kKvNegBig;
  for (int s = 0; s < a.spans; ++s) mm = fmaxf(mm, part[s * (D + 2) + D]);
  float lt = 0.f, ot[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) ot[i] = 0.f;
  for (int s = 0; s < a.spans; ++s) {
    const float f = __builtin_amdgcn_exp2f(part[s * (D + 2) + D] - mm);
    lt += f * part[s * (D + 2) + D + 1];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) ot[i] += f * part[s * (D + 2) + 64 * i + threadIdx.x];
  }
  const int oi = orow / a.group, oh = hk * a.group + orow % a.group;
  const bool any = lt > 0.f || lt != lt;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    a.out[(static_cast<long>(b) * a.q_len + oi) * a.ldo + oh * D + 64 * i + threadIdx.x] = static_cast<unsigned short>(kv_f2bf(any ? ot[i] / lt : 0.f));
  if (threadIdx.x == 0 && a.lse) a.lse[(static_cast<long>(b) * (a.Hk * a.group) + oh) * a.q_len + oi] = any ? (mm + log2f(lt)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace adt

using namespace adt;

namespace adt {
static int kv_check(const char* who, const void* cache, int64_t B, int64_t H, int64_t D, int64_t cap) {
  static thread_local char msg[160];
  auto fail = [&](int code, const char* what) {
    snprintf(msg, sizeof(msg), "%s: %s", who, what);
    return set_error(code, msg);
  };
  if (B < 0 || H <= 0 || cap <= 0) return fail(ADT_EINVAL, "negative batch, or no heads or no capacity");
  if (D != 64 && D != 128) return fail(ADT_ESHAPE, "head_dim must be 64 or 128");
  if (B > 65535 || H > 65535 || cap > (1LL << 30)) return fail(ADT_ESHAPE, "at most 65535 sequences and heads and 2^30 positions");
  if (B > 0 && (!cache || !aligned16(cache))) return fail(ADT_EINVAL, "the cache is null or not 16-byte aligned");
  return ADT_OK;
}
static int kv_rows_check(const char* who, int64_t B, int64_t H, int64_t D, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t n) {
  static thread_local char msg[160];
  const char* what = nullptr;
  if (n < 0 || n > (1LL << 30)) what = "bad number of rows";
  else if (B > 0 && n > 0 && (!k || !v)) what = "null pointer";
  else if (ldk < H * D || ldv < H * D) what = "a row holds kv_heads * head_dim elements";
  if (!what) return ADT_OK;
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  return set_error(ADT_EINVAL, msg);
}
struct KvPlan { int rows, row_blocks, tiles, spans, span_tiles; };
// Spans per head: a workgroup's four waves want two tiles each at least, and below three workgroups per CU the chip is not full.
static int kv_plan(const adt_attn_kv4_desc* d, KvPlan* p) {
  int n_cu = 256;
  (void)device_cu_count(&n_cu);
  p->rows = d->q_len * (d->heads / d->kv_heads);
  p->row_blocks = (p->rows + 15) / 16;
  p->tiles = (d->capacity + kKvTile - 1) / kKvTile;
  const long wgs = static_cast<long>(d->batch) * d->kv_heads * p->row_blocks;
  long want = wgs > 0 ? (3L * n_cu + wgs - 1) / wgs : 1;
  const long most = (p->tiles + 7) / 8;
  want = want < 1 ? 1 : (want > most ? most : want);
  p->span_tiles = static_cast<int>((p->tiles + want - 1) / want);
  p->spans = (p->tiles + p->span_tiles - 1) / p->span_tiles;
  return ADT_OK;
}
static int kv_desc_check(const adt_attn_kv4_desc* d, const void* cache) {
  if (!d) return set_error(ADT_EINVAL, "adt_attn_kv4: null descriptor");
  if (int rc = kv_check("adt_attn_kv4", cache, d->batch, d->kv_heads, d->head_dim, d->capacity)) return rc;
  if (d->heads <= 0 || d->heads % d->kv_heads) return set_error(ADT_ESHAPE, "adt_attn_kv4: heads must be a multiple of kv_heads");
  if (d->q_len <= 0) return set_error(ADT_EINVAL, "adt_attn_kv4: q_len must be positive");
  if (static_cast<int64_t>(d->q_len) * (d->heads / d->kv_heads) > (1 << 24)) return set_error(ADT_ESHAPE, "adt_attn_kv4: too many query rows");
  const int64_t width = static_cast<int64_t>(d->heads) * d->head_dim;
  if (d->ldq < width || d->ldo < width) return set_error(ADT_EINVAL, "adt_attn_kv4: a row of q and o holds heads * head_dim elements");
  return ADT_OK;
}
}  // namespace adt

extern "C" size_t adt_kv4_bytes(int64_t batch, int32_t kv_heads, int32_t head_dim, int64_t capacity) {
  if (batch <= 0 || kv_heads <= 0 || capacity <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return static_cast<size_t>(batch) * kv_heads * ((capacity + kKvTile - 1) / kKvTile) * (head_dim == 128 ? KvRec<128>::kBytes : KvRec<64>::kBytes);
}

extern "C" int adt_kv4_append(void* cache, int64_t batch, int32_t kv_heads, int32_t head_dim, int64_t capacity, const void* k, int64_t ldk, const void* v,
                              int64_t ldv, int64_t n, const int32_t* end, const int32_t* count, void* stream) {
  if (int rc = kv_check("adt_kv4_append", cache, batch, kv_heads, head_dim, capacity)) return rc;
  if (int rc = kv_rows_check("adt_kv4_append", batch, kv_heads, head_dim, k, ldk, v, ldv, n)) return rc;
  if (batch == 0 || n == 0) return ADT_OK;
  KvArgs a{};
  a.cache = static_cast<unsigned char*>(cache); a.B = static_cast<int>(batch); a.H = kv_heads; a.cap = static_cast<int>(capacity);
  a.tiles = static_cast<int>((capacity + kKvTile - 1) / kKvTile);
  a.k = static_cast<const unsigned short*>(k); a.ldk = ldk; a.v = static_cast<const unsigned short*>(v); a.ldv = ldv;
  a.end = end; a.count = count; a.n = static_cast<int>(n);
  const int64_t span = n < capacity ? n : capacity;
  const dim3 grid(static_cast<unsigned>((span + kKvTile - 2) / kKvTile + 1), static_cast<unsigned>(kv_heads), static_cast<unsigned>(batch));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (head_dim == 128) hipLaunchKernelGGL(kv4_append_kernel<128>, grid, dim3(128), 0, st, a);
  else hipLaunchKernelGGL(kv4_append_kernel<64>, grid, dim3(128), 0, st, a);
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

extern "C" int adt_kv4_read(const void* cache, int64_t batch, int32_t kv_heads, int32_t head_dim, int64_t capacity, void* k, int64_t ldk, void* v, int64_t ldv,
                            int32_t out_fp32, int64_t n, const int32_t* end, const int32_t* count, void* stream) {
  if (int rc = kv_check("adt_kv4_read", cache, batch, kv_heads, head_dim, capacity)) return rc;
  if (int rc = kv_rows_check("adt_kv4_read", batch, kv_heads, head_dim, k, ldk, v, ldv, n)) return rc;
  if (batch > 0 && n > 0 && (!aligned16(k) || !aligned16(v) || (ldk * (out_fp32 ? 4 : 2)) % 16 || (ldv * (out_fp32 ? 4 : 2)) % 16))
    return set_error(ADT_EINVAL, "adt_kv4_read: output rows are 16-byte aligned");
  if (batch == 0 || n == 0) return ADT_OK;
  KvArgs a{};
  a.cache = static_cast<unsigned char*>(const_cast<void*>(cache)); a.B = static_cast<int>(batch); a.H = kv_heads; a.cap = static_cast<int>(capacity);
  a.tiles = static_cast<int>((capacity + kKvTile - 1) / kKvTile);
  a.ko = k; a.ldko = ldk; a.vo = v; a.ldvo = ldv; a.out32 = out_fp32;
  a.end = end; a.count = count; a.n = static_cast<int>(n);
  const dim3 grid(static_cast<unsigned>((n + kKvTile - 1) / kKvTile), static_cast<unsigned>(kv_heads), static_cast<unsigned>(batch));
  const auto fn = head_dim == 128 ? (out_fp32 ? kv4_read_kernel<128, true> : kv4_read_kernel<128, false>)
                                  : (out_fp32 ? kv4_read_kernel<64, true> : kv4_read_kernel<64, false>);
  hipLaunchKernelGGL(fn, grid, dim3(128), 0, static_cast<hipStream_t>(stream), a);
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

extern "C" size_t adt_attn_kv4_workspace_bytes(const adt_attn_kv4_desc* d) {
  if (!d || d->batch <= 0 || d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads || d->q_len <= 0 || d->capacity <= 0) return 0;
  KvPlan p;
  (void)kv_plan(d, &p);
  return p.spans > 1 ? static_cast<size_t>(d->batch) * d->kv_heads * p.rows * p.spans * (d->head_dim + 2) * 4 : 0;
}

extern "C" int adt_attn_kv4(const adt_attn_kv4_desc* d, const void* q, const void* cache, void* o, float* lse, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = kv_desc_check(d, cache)) return rc;
  if (d->batch == 0) return ADT_OK;
  if (!q || !o) return set_error(ADT_EINVAL, "adt_attn_kv4: null pointer");
  KvPlan p;
  if (int rc = kv_plan(d, &p)) return rc;
  if (p.spans > 1 && (!ws || ws_bytes < adt_attn_kv4_workspace_bytes(d))) return set_error(ADT_EINVAL, "adt_attn_kv4: workspace too small");
  KvAttnArgs a{};
  a.q = static_cast<const unsigned short*>(q); a.ldq = d->ldq; a.qvec = aligned16(q) && d->ldq % 8 == 0;
  a.cache = static_cast<const unsigned char*>(cache); a.B = d->batch; a.Hk = d->kv_heads; a.group = d->heads / d->kv_heads; a.cap = d->capacity;
  a.tiles = p.tiles; a.key_len = d->key_len; a.out = static_cast<unsigned short*>(o); a.ldo = d->ldo; a.lse = lse;
  a.q_len = d->q_len; a.causal = d->causal; a.sl2 = d->scale * 1.4426950408889634f;
  a.rows = p.rows; a.row_blocks = p.row_blocks; a.spans = p.spans; a.span_tiles = p.span_tiles; a.part = static_cast<float*>(ws);
  const int64_t wgs = static_cast<int64_t>(d->batch) * d->kv_heads * p.row_blocks * p.spans, joins = static_cast<int64_t>(d->batch) * d->kv_heads * p.rows;
  if (wgs > (1LL << 31) - 1 || joins > (1LL << 31) - 1) return set_error(ADT_ESHAPE, "adt_attn_kv4: too many workgroups");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->head_dim == 128) hipLaunchKernelGGL(attn_kv4_kernel<128>, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(attn_kv4_kernel<64>, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, st, a);
  ADT_HIP_TRY(hipGetLastError());
  if (p.spans > 1) {
    if (d->head_dim == 128) hipLaunchKernelGGL(attn_kv4_join_kernel<128>, dim3(static_cast<unsigned>(joins)), dim3(64), 0, st, a);
    else hipLaunchKernelGGL(attn_kv4_join_kernel<64>, dim3(static_cast<unsigned>(joins)), dim3(64), 0, st, a);
    ADT_HIP_TRY(hipGetLastError());
  }
  return ADT_OK;
}
