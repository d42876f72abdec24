// kv4.hip -- a K/V cache held in 4 bits, and the attention that reads it (gfx950).
//
// Every 64 channels of a K or V row (one token, one head) share a scale and a minimum:
//   lo = min x, hi = max x, s = bf16(max((hi - lo) / 15, 2^-100)), m = lo, c = the integer nearest to (x - lo) / s (ties to even, at most 15)
//   and the row stands for c s + m.  A group with an infinity or a NaN (or a range past fp32): s = m = NaN.  The differences are fp32's: exact unless two
//   values of the group are more than 2^16 apart; the quotients of them are decided as real numbers are.
//
// Layout: per (sequence, head) a run of tiles of 32 tokens, per tile of head_dim D one record
//   K codes 32 D / 2 | V codes 32 D / 2 | K parameters [D/64][32] | V parameters [D/64][32]        4608 bytes at D = 128 (16384 in bf16)
// laid out as the matrix instructions of the attention consume it, so that a code is unpacked where it lies and nothing is transposed:
//   K: a token's row is D/2 bytes; channel 32 g + 8 u + j is in the dword (D/32) u + g of the row: a lane's 4 D/32 bytes (token lane & 15, u = lane >> 4)
//      are its operands of the row's D/32 products over 32 channels each.
//   V: channel 16 b + i and the eight tokens 4 u + {0..3}, 16 + 4 u + {0..3} are one dword, number ((b / 4) 64 + 16 u + i) 4 + (b & 3): a lane's
//      (i = lane & 15, u = lane >> 4) 16-byte pieces are its operands of four products over 32 tokens; the token order is the one in which a lane
//      holds the scores.
//   A dword's element j is at bits 4 (j / 2) + 16 (j & 1): w, w >> 4, w >> 8 and w >> 12, masked to 0x000f000f and joined with 0x43004300, are four pairs
//   of the bf16 numbers 128 + c.
//   A parameter dword is the bf16 scale (low half) and the bf16 minimum (high half).
#include <hip/hip_runtime.h>

#include <cmath>
#include <algorithm>
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
// One wave per (32-token tile, head, sequence) and side (K or V).  A lane holds eight channels of a row, D/8 lanes a row, and goes through the
// tokens whose codes share a dword of the V record, 4 u + {0..3} and 16 + 4 u + {0..3} (at 64 channels one half of them): its eight channels' dwords
// then fill up in its registers, and the K codes of a row are one dword per lane anyway.  All rows are requested before the first is used.
//   extrema: bf16 numbers, sign-folded, order like 16-bit integers (NaNs at the ends, so that they and infinities show in the range), two per
//            instruction; eight lanes share a group and exchange in the DPP network
//   codes: (x - lo) / s is a correctly rounded quotient, q0 = d y, y = 1 / s, corrected by the exact remainder fma(-q0, s, d); rounding to the integer is the
//            addition of 2^23, whose low half is then the code.  It is 15 at most: s is (hi - lo) / 15 to 2^-9.
// The V dwords pass through LDS once to leave as 16-byte pieces; a tile that is not written whole keeps its other tokens' codes (the wave is
// the only writer of its record half).
// Bound: vector instructions, 110 per eight values, about the time of the memory traffic (63104 rows of 768, K and V).
typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned kv_fold(unsigned w) {             // two bf16 numbers <-> 16-bit integers of the same order
  const s16x2 x = __builtin_bit_cast(s16x2, w);
  return w ^ (__builtin_bit_cast(unsigned, x >> static_cast<short>(15)) & 0x7fff7fffu);
}
__device__ __forceinline__ unsigned kv_pk_min(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
__device__ __forceinline__ unsigned kv_pk_max(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
template <int kCtrl>
__device__ __forceinline__ unsigned kv_dpp(unsigned v) { return __builtin_amdgcn_update_dpp(v, v, kCtrl, 0xf, 0xf, false); }
__device__ __forceinline__ unsigned kv_halves(unsigned hi, unsigned lo) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }      // lo & 0xffff | hi << 16

template <int D>
__global__ __launch_bounds__(128) void kv4_append_kernel(KvArgs a) {
  using R = KvRec<D>;
  constexpr int kLanes = D / 8, kJ = D == 128 ? 8 : 4;             // lanes per row, rows per lane
  __shared__ __attribute__((aligned(16))) unsigned vl[D / 64][4][72];      // [piece][u][16 channels x 4 blocks + 8: the four u on different banks]
  const int lane = threadIdx.x & 63, side = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);      // side 0: K, 1: V
  const int b = blockIdx.z, h = blockIdx.y;
  const KvRange r = kv_range(a, b);
  const int tile = (r.lo >> 5) + static_cast<int>(blockIdx.x);
  if (tile * kKvTile >= r.hi || r.lo >= r.hi) return;  // block-uniform
  unsigned char* rec = a.cache + (static_cast<long>(b * a.H + h) * a.tiles + tile) * R::kBytes;
  const int t0 = max(r.lo - tile * kKvTile, 0), t1 = min(r.hi - tile * kKvTile, kKvTile);      // tokens of the tile that are written
  const int c8 = lane % kLanes, sub = lane / kLanes, u = sub & 3, half = sub >> 2;            // (half: 64 channels only)
  const unsigned short* src = side ? a.v : a.k;
  const long ld = side ? a.ldv : a.ldk;
  const unsigned short* row0 = src + (static_cast<long>(b) * a.n + (tile * kKvTile - r.first)) * ld + h * D + 8 * c8;      // (of token 0, which need not exist)
  const bool vec = ((reinterpret_cast<uintptr_t>(src) & 15) | (ld & 7)) == 0;
  auto token_of = [&](int j) { return 16 * (D == 128 ? j >> 2 : half) + 4 * u + (j & 3); };
  unsigned any = 0;                                    // bit j: some lane's row j is written (uniform)
#pragma unroll
  for (int t = 0; t < kKvTile; ++t)
    if (t >= t0 && t < t1) any |= 1u << (D == 128 ? (t & 3) + 4 * (t >> 4) : t & 3);
  u32x4 raw[kJ];
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    if (!(any >> j & 1u)) continue;
    const int t = token_of(j);
    const unsigned short* p = row0 + (t >= t0 && t < t1 ? t : t0) * ld;      // (every lane takes part in the exchanges)
    if (vec) {
      raw[j] = *reinterpret_cast<const u32x4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[j][i] = p[2 * i] | static_cast<unsigned>(p[2 * i + 1]) << 16;
    }
  }
  unsigned* par = reinterpret_cast<unsigned*>(rec + (side ? R::kVp : R::kKp)) + (c8 >> 3) * kKvTile;
  unsigned vw[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};   // channel i's dword
  unsigned even[8];
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    unsigned bits[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
    if (any >> j & 1u) {
      const int t = token_of(j);
      const bool live = t >= t0 && t < t1;
      unsigned f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = kv_fold(raw[j][i]);
      unsigned lo2 = kv_pk_min(kv_pk_min(f[0], f[1]), kv_pk_min(f[2], f[3])), hi2 = kv_pk_max(kv_pk_max(f[0], f[1]), kv_pk_max(f[2], f[3]));
      lo2 = kv_pk_min(lo2, kv_dpp<0xB1>(lo2)); hi2 = kv_pk_max(hi2, kv_dpp<0xB1>(hi2));          // lane ^ 1
      lo2 = kv_pk_min(lo2, kv_dpp<0x4E>(lo2)); hi2 = kv_pk_max(hi2, kv_dpp<0x4E>(hi2));          // lane ^ 2
      lo2 = kv_pk_min(lo2, kv_dpp<0x141>(lo2)); hi2 = kv_pk_max(hi2, kv_dpp<0x141>(hi2));        // mirrored in eight lanes: the other four
      lo2 = kv_pk_min(lo2, lo2 >> 16);                 // (the low half)
      hi2 = kv_pk_max(hi2, hi2 << 16);                 // (the high half)
      const unsigned both = kv_fold((lo2 & 0xffffu) | (hi2 & 0xffff0000u));
      const float lo = kv_bf2f(both & 0xffffu), hi = __uint_as_float(both & 0xffff0000u);
      const float range = hi - lo;
      const bool bad = !(range < INFINITY);
      constexpr float y15 = 1.0f / 15.0f;
      const float s0 = range * y15;                    // a correctly rounded range / 15, as the codes are
      const unsigned sb = kv_f2bf(fmaxf(fmaf(fmaf(-s0, 15.0f, range), y15, s0), kKvTiny));
      const float s = kv_bf2f(sb);
      const float y0 = __builtin_amdgcn_rcpf(s), y = fmaf(fmaf(-s, y0, 1.0f), y0, y0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = i & 1 ? __uint_as_float(raw[j][i >> 1] & 0xffff0000u) : __uint_as_float(raw[j][i >> 1] << 16);
        const float d = x - lo;
        const float q0 = d * y;
        bits[i] = __float_as_uint(fmaf(fmaf(-q0, s, d), y, q0) + 8388608.0f);
      }
      if (__builtin_amdgcn_ballot_w64(bad || !live) != 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) bits[i] = bad || !live ? 0u : bits[i];
      }
      if (live && (c8 & 7) == 0) par[t] = bad ? 0x7fc07fc0u : (sb | both << 16);
      if (side == 0 && live) {
        const unsigned w = kv_halves(bits[1], bits[0]) | kv_halves(bits[3], bits[2]) << 4 | kv_halves(bits[5], bits[4]) << 8 | kv_halves(bits[7], bits[6]) << 12;
        // channels 8 c8 .. + 7 = 32 g + 8 v with g = c8 / 4, v = c8 & 3
        reinterpret_cast<unsigned*>(rec + t * R::kRow)[(D / 32) * (c8 & 3) + (c8 >> 2)] = w;
      }
    }
    if (side) {                                        // rows 2 k and 2 k + 1: nibble k of the dword's halves
      if (j & 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vw[i] |= kv_halves(bits[i], even[i]) << (4 * (j >> 1));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) even[i] = bits[i];
      }
    }
  }
  if (side == 0) return;
  unsigned keep = 0;                                   // of lane (channel lane & 15, u = lane >> 4) of the pieces: the nibbles of tokens that stay
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int t = (j < 4 ? 0 : 16) + 4 * (lane >> 4) + (j & 3);
    if (t < t0 || t >= t1) keep |= 15u << (4 * (j >> 1) + 16 * (j & 1));
  }
  if constexpr (D == 64) {                             // the other half's tokens: lane ^ 32; each of the two writes four channels
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (half) vw[i] <<= 8;
      vw[i] |= __shfl_xor(vw[i], 32);
    }
  }
  // channel 8 c8 + i: block c8 / 2, its channel 8 (c8 & 1) + i
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (D == 128 || (i >> 2) == half) vl[c8 >> 3][u][(8 * (c8 & 1) + i) * 4 + ((c8 >> 1) & 3)] = vw[i];
  __builtin_amdgcn_wave_barrier();                     // one wave wrote vl and reads it back: its LDS operations are in order
  u32x4* out = reinterpret_cast<u32x4*>(rec + R::kV);
#pragma unroll
  for (int piece = 0; piece < D / 64; ++piece) {
    u32x4 w = *reinterpret_cast<const u32x4*>(&vl[piece][lane >> 4][(lane & 15) * 4]);
    u32x4* p = out + piece * 64 + lane;
    if (keep == 0u) {
      *p = w;
    } else if (keep != 0xffffffffu) {
      const u32x4 old = *p;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] |= old[k] & keep;
      *p = w;
    }
  }
}

// ------------------------------------------------------------------------------------ read
// Rows i < count of every sequence as the numbers they stand for (bf16 or fp32), the other rows of the output zeros.  One wave per 32 output
// rows and side; where those lie in a tile (or two) a wave holds the tile's V codes in LDS, as they come.
template <int D, bool k32>
__global__ __launch_bounds__(128) void kv4_read_kernel(KvArgs a) {
  using R = KvRec<D>;
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;
  __shared__ unsigned vl[2][32 * D / 8];               // the V codes of the one or two tiles that the 32 rows lie in
  const int lane = threadIdx.x & 63, side = threadIdx.x >> 6;
  const int b = blockIdx.z, h = blockIdx.y;
  const KvRange r = kv_range(a, b);
  const int c8 = lane % kLanes, sub = lane / kLanes;
  void* out = side ? a.vo : a.ko;
  const long ld = side ? a.ldvo : a.ldko;
  const int i0 = blockIdx.x * kKvTile;
  const long first = static_cast<long>(r.first) + i0;                  // the position of row i0
  const long lo = max(first, static_cast<long>(r.lo)), hi = min(first + kKvTile, static_cast<long>(r.hi));
  const unsigned char* recs = a.cache + static_cast<long>(b * a.H + h) * a.tiles * R::kBytes;
  const int tile0 = static_cast<int>(lo >> 5);
  if (side && lo < hi) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (tile0 + k > static_cast<int>((hi - 1) >> 5)) break;
      const u32x4* p = reinterpret_cast<const u32x4*>(recs + static_cast<long>(tile0 + k) * R::kBytes + R::kV);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) reinterpret_cast<u32x4*>(vl[k])[i * 64 + lane] = p[i * 64 + lane];
    }
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int t = sub; t < kKvTile; t += kRows) {
    const int i = i0 + t;
    if (i >= a.n) break;
    const long pos = first + t;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (pos >= lo && pos < hi) {
      const int tile = static_cast<int>(pos >> 5), tt = static_cast<int>(pos & 31);
      const unsigned char* rec = recs + static_cast<long>(tile) * R::kBytes;
      const unsigned par = reinterpret_cast<const unsigned*>(rec + (side ? R::kVp : R::kKp))[(c8 >> 3) * kKvTile + tt];
      const float s = kv_bf2f(par & 0xffffu), m = __uint_as_float(par & 0xffff0000u);
      if (side == 0) {
        const unsigned w = reinterpret_cast<const unsigned*>(rec + tt * R::kRow)[(D / 32) * (c8 & 3) + (c8 >> 2)];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = static_cast<float>((w >> (4 * (j >> 1) + 16 * (j & 1))) & 15u) * s + m;
      } else {
        const int u = (tt & 15) >> 2, j8 = (tt & 3) + (tt & 16 ? 4 : 0), sh = 4 * (j8 >> 1) + 16 * (j8 & 1);
        const unsigned* vw = vl[tile - tile0];
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
// A workgroup = kW waves on one (sequence, K/V head, block of 16 rows, span of tiles); a row is a (query position, query head of the group)
// pair, row = position * group + head.  A wave takes every kW-th tile of the span:
//   scores  S[token][row] = sum_g s_g (K codes . q)_g + m_g (sum of q)_g    two 16 x 16 x 32 bf16 products per group and 16 tokens; the codes enter as
//           128 + c, and the accumulator starts at -128 (sum of q)_g, so it ends at the sum of c q: q and the codes are exact in bf16, the sums fp32
//   softmax over the tokens: a lane holds eight tokens of one row; one running maximum per row, raised only when a score exceeds it by more
//           than 2^8 (the probabilities are then at most 2^8 and the sums stay exact to fp32), so the cross-lane exchange is rare
//   output  O[row][channel] += (p s_g) (128 + c) - 128 (p s_g)    the weight p s_g goes in as two bf16 numbers, upper and lower half (2^-17 of it is
//           lost), and the subtrahend is a product of the same two with ones, so that the offset costs no accuracy; p m_g is added up per
//           row and group in fp32 on the side.
// The waves' (max, sum, O) join through LDS; with more than one span per head they go to the workspace and a second kernel joins them.
// Bound: the instructions beside the products (340 per wave and tile at D = 128, 56 + 56 of them unpacking codes), about 8 TB/s of cache on the
// whole chip, then the memory.  The next tile's K (V) is requested as soon as this tile's K (V) is used up.
struct KvAttnArgs {
  const unsigned short* q; long ldq; bool qvec;        // qvec: 16-byte loads of q
  const unsigned char* cache; int B, Hk, group, cap, tiles;
  const int* key_len;
  unsigned short* out; long ldo; float* lse;
  int q_len, causal; float sl2; bool negate;           // |scale| * log2 e, and q enters negated for a negative scale
  int rows, row_blocks, spans, span_tiles;             // rows = q_len * group
  float* part;                                         // spans > 1: [B][Hk][rows][spans][D + 2]
};
constexpr float kKvNegBig = -3.0e38f;               // below every score: the running maximum of a row that has seen no token
constexpr float kKvThr = 8.0f;
constexpr int kKvMaxSpans = 64, kKvFewSpans = 8;

__device__ __forceinline__ float kv_max_over_groups(float v) {      // over the four lanes that share lane & 15
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float kv_sum_over_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
union KvFrag { unsigned u[4]; bf16x8 v; };
// eight codes -> the bf16 numbers 128 + c; mask and bits are 0x000f000f and 0x43004300 in registers (one instruction takes one literal at most)
__device__ __forceinline__ KvFrag kv_unpack(unsigned w, unsigned mask, unsigned bits) {
  KvFrag f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.u[i] = ((w >> (4 * i)) & mask) | bits;
  return f;
}
__device__ __forceinline__ float kv_scale_of(unsigned par) { return __uint_as_float(par << 16); }
__device__ __forceinline__ float kv_min_of(unsigned par) { return __uint_as_float(par & 0xffff0000u); }

template <int D, int kW>
__global__ __launch_bounds__(64 * kW, kW < 8 ? 3 : 1) void attn_kv4_kernel(KvAttnArgs a, int n_max) {      // n_max = min(16, rows)
  using R = KvRec<D>;
  constexpr int kG = R::kG, kNB = D / 16, kPieces = D / 64;          // V pieces (16 bytes) per lane and tile
  constexpr int kPitch = D + 4;
  constexpr int kQ = (2 * D + 64 * kW - 1) / (64 * kW);              // sixteen-byte pieces of q per thread
  extern __shared__ __attribute__((aligned(16))) float so[];         // [kW][n_max][kPitch] at the end; the rows of q at the start
  __shared__ float sm[kW][16], sl[kW][16], sc[kW][kG][16];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, u = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = blockIdx.x;
  const int slot = id % a.spans; id /= a.spans;
  const int span = (slot + id) % a.spans;      // (blocks b and b + 8 share an XCD: the late spans, empty in short sequences, are spread over them)
  const int rb = id % a.row_blocks; id /= a.row_blocks;
  const int hk = id % a.Hk, b = id / a.Hk;
  // ---- everything the first tile needs is asked for at once: the length, this block's rows of q (sixteen bytes per thread, two-byte loads where
  // the rows are not aligned), the tile itself (the span's last one at most, whatever the length is)
  int klen = a.key_len ? a.key_len[b] : a.cap;
  u32x4 qw[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    qw[i] = u32x4{0u, 0u, 0u, 0u};
    const int piece = tid + 64 * kW * i, row = rb * 16 + piece / (D / 8), c = 8 * (piece % (D / 8));
    if (piece >= 2 * D || row >= a.rows) continue;
    const unsigned short* p = a.q + (static_cast<long>(b) * a.q_len + row / a.group) * a.ldq + (hk * a.group + row % a.group) * D + c;
    if (a.qvec) {
      qw[i] = *reinterpret_cast<const u32x4*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) qw[i][j] = p[2 * j] | static_cast<unsigned>(p[2 * j + 1]) << 16;
    }
  }
  const unsigned char* const base = a.cache + static_cast<long>(b * a.Hk + hk) * a.tiles * R::kBytes;
  unsigned kw[2][D / 32];
  u32x4 vw[kPieces], kp[2][kG], vp[2][kG];
  auto load_k = [&](int t) __attribute__((always_inline)) {
    const unsigned char* rec = base + static_cast<long>(t) * R::kBytes;
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const unsigned* p = reinterpret_cast<const unsigned*>(rec + (16 * hb + li) * R::kRow + 4 * (D / 32) * u);
      if constexpr (D == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int s = 0; s < 4; ++s) kw[hb][s] = w[s];
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        kw[hb][0] = w.x; kw[hb][1] = w.y;
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) kp[hb][g] = *reinterpret_cast<const u32x4*>(rec + R::kKp + (g * kKvTile + 16 * hb + 4 * u) * 4);
    }
  };
  auto load_v = [&](int t) __attribute__((always_inline)) {
    const unsigned char* rec = base + static_cast<long>(t) * R::kBytes;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) vw[i] = *reinterpret_cast<const u32x4*>(rec + R::kV + (i * 64 + lane) * 16);
#pragma unroll
    for (int hb = 0; hb < 2; ++hb)
#pragma unroll
      for (int g = 0; g < kG; ++g) vp[hb][g] = *reinterpret_cast<const u32x4*>(rec + R::kVp + (g * kKvTile + 16 * hb + 4 * u) * 4);
  };
  int tile = span * a.span_tiles + wave;
  load_k(min(tile, a.tiles - 1));
  load_v(min(tile, a.tiles - 1));
  // Query i of a causal call sees klen - (q_len - 1 - i) positions, of which the cache has the first cap: a length past the capacity is taken to the
  // capacity behind the subtraction, not in front of it.
  klen = max(klen, 0);
  auto seen = [&](int row) { return min(a.causal ? klen - (a.q_len - 1 - row / a.group) : klen, a.cap); };
  const int most = seen(min(rb * 16 + 15, a.rows - 1));              // the tokens that some row of this block sees
  const int tile_end = min((max(most, 0) + kKvTile - 1) / kKvTile, (span + 1) * a.span_tiles);

  unsigned short* const ql = reinterpret_cast<unsigned short*>(so);  // [16][D + 8]
  constexpr int kQPitch = D + 8;
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const int piece = tid + 64 * kW * i;
    if (a.negate) qw[i] ^= 0x80008000u;
    if (piece < 2 * D) *reinterpret_cast<u32x4*>(ql + (piece / (D / 8)) * kQPitch + 8 * (piece % (D / 8))) = qw[i];
  }
  __syncthreads();
  KvFrag qf[D / 32];
  float qs[kG];
#pragma unroll
  for (int g = 0; g < kG; ++g) qs[g] = 0.f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(ql + li * kQPitch + 32 * s + 8 * u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      qf[s].u[j] = w[j];
      qs[s / 2] += kv_scale_of(w[j]) + kv_min_of(w[j]);              // (the two halves as numbers)
    }
  }
#pragma unroll
  for (int g = 0; g < kG; ++g) qs[g] = kv_sum_over_groups(qs[g]);
  __syncthreads();                                                   // ql becomes so
  // this lane's row (as a column of the score product) sees the tokens [0, limit)
  const int limit = seen(min(rb * 16 + li, a.rows - 1));
  const int least = seen(0);

  unsigned mask = 0x000f000fu, bits = 0x43004300u;
  asm volatile("" : "+v"(mask), "+s"(bits));
  float m = kKvNegBig, l = 0.f, cb[kG];
  f32x4 o[kNB], os[kG];
#pragma unroll
  for (int i = 0; i < kNB; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < kG; ++g) { cb[g] = 0.f; os[g] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  KvFrag ones;
#pragma unroll
  for (int j = 0; j < 4; ++j) ones.u[j] = 0x3f803f80u;

  for (; tile < tile_end; tile += kW) {
    const int next = min(tile + kW, tile_end - 1);                   // (past the end: a tile that is there, for nothing)
    float z[8];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      f32x4 acc[kG];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const float c0 = -128.0f * qs[g];
        acc[g] = f32x4{c0, c0, c0, c0};
#pragma unroll
        for (int s = 2 * g; s < 2 * g + 2; ++s) acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv_unpack(kw[hb][s], mask, bits).v, qf[s].v, acc[g], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float t = kv_min_of(kp[hb][0][r]) * qs[0];
        t = fmaf(kv_scale_of(kp[hb][0][r]), acc[0][r], t);
#pragma unroll
        for (int g = 1; g < kG; ++g) t = fmaf(kv_scale_of(kp[hb][g][r]), acc[g][r], fmaf(kv_min_of(kp[hb][g][r]), qs[g], t));
        z[4 * hb + r] = t;
      }
    }
    load_k(next);
    const int key0 = tile * kKvTile + 4 * u;
    const bool edge = (tile + 1) * kKvTile > least;                  // block-uniform: some row does not see all of the tile
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key0 + (j < 4 ? j : 12 + j) >= limit) z[j] = kKvNegBig;
    }
    float mx = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))) * a.sl2;
    if (__builtin_amdgcn_ballot_w64(mx > m + kKvThr) != 0) {
      const float m_new = fmaxf(m, kv_max_over_groups(mx));
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int g = 0; g < kG; ++g) cb[g] *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ar = __shfl(alpha, 4 * u + r);                   // the output's rows are 4 u + r
#pragma unroll
        for (int i = 0; i < kNB; ++i) o[i][r] *= ar;
#pragma unroll
        for (int g = 0; g < kG; ++g) os[g][r] *= ar;
      }
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(z[j], a.sl2, -m));
    if (edge) {                                                      // what a row does not see may be anything
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key0 + (j < 4 ? j : 12 + j) >= limit) {
          p[j] = 0.f;
#pragma unroll
          for (int g = 0; g < kG; ++g) vp[j >> 2][g][j & 3] = 0u;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) l += p[j];
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      KvFrag hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned p0 = vp[j >> 1][g][(2 * j) & 3], p1 = vp[j >> 1][g][(2 * j + 1) & 3];
        const float w0 = p[2 * j] * kv_scale_of(p0), w1 = p[2 * j + 1] * kv_scale_of(p1);
        cb[g] = fmaf(p[2 * j], kv_min_of(p0), cb[g]);
        cb[g] = fmaf(p[2 * j + 1], kv_min_of(p1), cb[g]);
        hi.u[j] = __builtin_amdgcn_perm(__float_as_uint(w1), __float_as_uint(w0), 0x07060302u);
        lo.u[j] = kv_pack_bf2(w0 - kv_min_of(__float_as_uint(w0)), w1 - kv_min_of(__float_as_uint(w1)));
      }
      os[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi.v, ones.v, os[g], 0, 0, 0);
      os[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo.v, ones.v, os[g], 0, 0, 0);
#pragma unroll
      for (int i = 4 * g; i < 4 * g + 4; ++i) {
        const KvFrag vf = kv_unpack(vw[i >> 2][i & 3], mask, bits);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi.v, vf.v, o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo.v, vf.v, o[i], 0, 0, 0);
      }
    }
    load_v(next);
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
  for (int r = 0; r < 4; ++r) {
    if (4 * u + r >= n_max) continue;
#pragma unroll
    for (int i = 0; i < kNB; ++i) so[(wave * n_max + 4 * u + r) * kPitch + 16 * i + li] = fmaf(-128.0f, os[i / 4][r], o[i][r]);
  }
  __syncthreads();
  const int n_rows = min(16, a.rows - rb * 16);
  for (int e = tid; e < n_rows * D; e += 64 * kW) {
    const int rr = e / D, d = e % D;
    float mm = sm[0][rr];
#pragma unroll
    for (int w = 1; w < kW; ++w) mm = fmaxf(mm, sm[w][rr]);
    float lt = 0.f, ot = 0.f;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][rr] - mm);
      lt = fmaf(f, sl[w][rr], lt);
      ot = fmaf(f, so[(w * n_max + rr) * kPitch + d] + sc[w][d >> 6][rr], ot);
    }
    const int orow = rb * 16 + rr, oi = orow / a.group, oh = hk * a.group + orow % a.group;
    const bool any = lt > 0.f || lt != lt;
    if (a.spans == 1) {
      a.out[(static_cast<long>(b) * a.q_len + oi) * a.ldo + oh * D + d] = static_cast<unsigned short>(kv_f2bf(any ? ot / lt : 0.f));
      if (d == 0 && a.lse) a.lse[(static_cast<long>(b) * (a.Hk * a.group) + oh) * a.q_len + oi] = any ? (mm + log2f(lt)) * 0.6931471805599453f : -INFINITY;
    } else {
      float* part = a.part + (((static_cast<long>(b) * a.Hk + hk) * a.rows + orow) * a.spans + span) * (D + 2);
      part[d] = ot;
      if (d == 0) { part[D] = mm; part[D + 1] = lt; }
    }
  }
}

// 512 / D / kS rows per workgroup, kS threads a channel: lane s weighs span s (at most 64 of them); the spans' outputs are dealt to the threads of a
// channel, all loads at once.  kS = 512 / D past eight spans (a thread a channel: 37 spans 4 us more), 1 up to there (1680 rows of 2 spans, 64 channels,
// 2.2 to 3.9 us; with a workgroup a row 5.0).
template <int D, int kS>
__global__ __launch_bounds__(512) void attn_kv4_join_kernel(KvAttnArgs a, int n_rows) {
  constexpr int kEach = (kS == 1 ? kKvFewSpans : kKvMaxSpans) / kS, kRows = 512 / D / kS;
  __shared__ float so[kS][D];
  const int lane = threadIdx.x & 63, d = threadIdx.x % D;
  const int own = __builtin_amdgcn_readfirstlane(threadIdx.x / D), part_of = kS == 1 ? 0 : own;
  const int row = blockIdx.x * kRows + (kS == 1 ? own : 0);
  if (row >= n_rows) return;                     // (kS == 1: no barrier below)
  const int orow = row % a.rows, bh = row / a.rows, hk = bh % a.Hk, b = bh / a.Hk;
  const float* part = a.part + static_cast<long>(row) * a.spans * (D + 2);
  float ms = kKvNegBig, ls = 0.f, ov[kEach];
  if (lane < a.spans) { ms = part[lane * (D + 2) + D]; ls = part[lane * (D + 2) + D + 1]; }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = part_of + kS * i;
    ov[i] = s < a.spans ? part[s * (D + 2) + d] : 0.f;
  }
  float mm = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
  const float f = __builtin_amdgcn_exp2f(ms - mm);
  float lt = f * ls, ot = 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) lt += __shfl_xor(lt, o);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const float fs = __shfl(f, part_of + kS * i);
    if (part_of + kS * i < a.spans) ot = fmaf(fs, ov[i], ot);
  }
  if constexpr (kS > 1) {
    so[part_of][d] = ot;
    __syncthreads();
    if (part_of) return;
#pragma unroll
    for (int s = 1; s < kS; ++s) ot += so[s][d];
  }
  const int oi = orow / a.group, oh = hk * a.group + orow % a.group;
  const bool any = lt > 0.f || lt != lt;
  a.out[(static_cast<long>(b) * a.q_len + oi) * a.ldo + oh * D + d] = static_cast<unsigned short>(kv_f2bf(any ? ot / lt : 0.f));
  if (d == 0 && a.lse) a.lse[(static_cast<long>(b) * (a.Hk * a.group) + oh) * a.q_len + oi] = any ? (mm + log2f(lt)) * 0.6931471805599453f : -INFINITY;
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
struct KvPlan { int rows, row_blocks, tiles, spans, span_tiles, waves; };
// How a call is cut.  A wave's tile costs 1 us when it has its SIMD to itself (420 instructions), a call 5 us around its tiles and 2 us more for the
// join of spans.  A workgroup of eight waves fills half a CU or more, of four a third.  us with waves / spans, heads x positions:
//   at most one workgroup a CU and 26 tiles, three a wave and a fourth in two of them: eight waves, one span.  The border is a compromise between few and many
//   heads (one query, 128 channels; 6 heads x 24 tiles 8/1 8.0, 4/4 7.7, 4/8 7.0, 27 tiles 8.5, 7.8, 6.9; 192 heads x 24 tiles 8/1 8.3, 4/2 10.7, 4/4
//   10.6, 27 tiles 8.9, 12.3, 11.2: one span is as good or better to 20 tiles everywhere, and to 34 for 192 heads);
//   one to four rows: four waves, and spans until the card is full, or of 32 tiles, as short sequences leave theirs empty and the late
//   ones even that out (6 x 986 4/8 7.3, 8/4 8.3, 8/1 9.6; 64 x 32000 in four rows, ragged, 4/24 39, 4/12 53, 8/4 55; 174 x 21483 4/24 41, 4/4 59, 8/2 74);
//   more rows, whose joins weigh more: eight waves, spans for one workgroup a CU, or of 64 tiles (60 x 2359 in 16 rows 8/4 13.6, 4/12 15.1; 108 x 4271
//   in 8 rows 8/2 14.8, 4/6 15.8);
//   more workgroups than CUs: four waves, spans of 32 tiles (1536 x 986 4/1 40, 4/2 50, 8/1 52; 384 x 500 4/1 10.2, 4/2 12.4), and two waves where a sequence
//   is five tiles at most (1440 x 85 2/1 8.0, 4/1 10.6).
// Sixteen workgroups a CU are the most that spans make: past that nothing is left to even out, and the workspace stays under 35 MB.
static int kv_plan(const adt_attn_kv4_desc* d, KvPlan* p) {
  int n_cu = 256;
  (void)device_cu_count(&n_cu);
  p->rows = d->q_len * (d->heads / d->kv_heads);
  p->row_blocks = (p->rows + 15) / 16;
  p->tiles = (d->capacity + kKvTile - 1) / kKvTile;
  const int64_t wgs = static_cast<int64_t>(d->batch) * d->kv_heads * p->row_blocks;
  int64_t want = 1;
  if (wgs > n_cu) {
    p->waves = wgs > 2 * n_cu && p->tiles <= 5 ? 2 : 4;
    want = (p->tiles + 16) / 32;
  } else if (p->tiles <= 26) {
    p->waves = 8;
  } else if (p->rows <= 4) {
    p->waves = 4;
    want = std::max<int64_t>(3 * n_cu / std::max<int64_t>(wgs, 1), (p->tiles + 16) / 32);
  } else {
    p->waves = 8;
    want = std::max<int64_t>(n_cu / std::max<int64_t>(wgs, 1), (p->tiles + 32) / 64);
  }
  const int64_t most = std::min({static_cast<int64_t>((p->tiles + p->waves - 1) / p->waves), static_cast<int64_t>(kKvMaxSpans), 16 * n_cu / std::max<int64_t>(wgs, 1)});
  want = std::max<int64_t>(1, std::min(want, most));
  p->span_tiles = static_cast<int>((p->tiles + want - 1) / want);
  p->spans = (p->tiles + p->span_tiles - 1) / p->span_tiles;
  return ADT_OK;
}
template <int D, int kW>
static int launch_attn_kv4(const KvAttnArgs& a, unsigned wgs, hipStream_t st) {
  const int n_max = a.rows < 16 ? a.rows : 16;
  const int q_bytes = 16 * (D + 8) * 2, o_bytes = kW * n_max * (D + 4) * 4, lds = o_bytes > q_bytes ? o_bytes : q_bytes;
  if (lds > 64 * 1024 - 4096)
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(attn_kv4_kernel<D, kW>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL((attn_kv4_kernel<D, kW>), dim3(wgs), dim3(64 * kW), lds, st, a, n_max);
  ADT_HIP_TRY(hipGetLastError());
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
  a.q_len = d->q_len; a.causal = d->causal; a.sl2 = fabsf(d->scale) * 1.4426950408889634f; a.negate = d->scale < 0.f;
  a.rows = p.rows; a.row_blocks = p.row_blocks; a.spans = p.spans; a.span_tiles = p.span_tiles; a.part = static_cast<float*>(ws);
  const int64_t wgs = static_cast<int64_t>(d->batch) * d->kv_heads * p.row_blocks * p.spans;
  if (wgs >= 1LL << 23) return set_error(ADT_ESHAPE, "adt_attn_kv4: too many workgroups");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  typedef int (*Launch)(const KvAttnArgs&, unsigned, hipStream_t);
  static const Launch launches[2][3] = {{launch_attn_kv4<64, 2>, launch_attn_kv4<64, 4>, launch_attn_kv4<64, 8>},
                                        {launch_attn_kv4<128, 2>, launch_attn_kv4<128, 4>, launch_attn_kv4<128, 8>}};
  const Launch launch = launches[d->head_dim == 128][p.waves >> 2];
  if (int rc = launch(a, static_cast<unsigned>(wgs), st)) return rc;
  if (p.spans > 1) {
    typedef void (*Join)(KvAttnArgs, int);
    static const Join join[2][2] = {{attn_kv4_join_kernel<64, 1>, attn_kv4_join_kernel<64, 8>}, {attn_kv4_join_kernel<128, 1>, attn_kv4_join_kernel<128, 4>}};
    const bool many = p.spans > kKvFewSpans;
    const int n_rows = static_cast<int>(static_cast<int64_t>(d->batch) * d->kv_heads * p.rows), per_wg = many ? 1 : 512 / d->head_dim;      // (spans: 2^16 rows at most)
    hipLaunchKernelGGL(join[d->head_dim == 128][many], dim3((n_rows + per_wg - 1) / per_wg), dim3(512), 0, st, a, n_rows);
    ADT_HIP_TRY(hipGetLastError());
  }
  return ADT_OK;
}
