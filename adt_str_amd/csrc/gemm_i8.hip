// gemm_i8.hip -- matrix product in 8-bit integers with one scale per row of each operand (token / output channel), and the quantiser
// of the activations in front of it (gfx950).
//
//   quant_rows   a_m = max(max_k |x_mk|, 2^-100);  q_mk = the integer nearest to 127 x_mk / a_m (ties to even);  scale_m = a_m / 127
//   gemm_i8      acc_mn = sum_k a_mk b_nk (exact, int32);  z = acc * a_scale_m * b_scale_n + bias_n; activation; + residual_mn
//
// The int8 matrix instruction (v_mfma_i32_16x16x64_i8) does twice the products of the bf16 one per cycle on the same operand bytes.
// Four kernels, by how many tiles a call has: 16 channels a workgroup for few tokens, 64 x 64, 128 x 128 and 256 x 256 tiles (launch_i8).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>

#include "adt_common.h"

namespace adt {
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float i8_bf2f(unsigned short v) { return __uint_as_float(static_cast<unsigned>(v) << 16); }
__device__ __forceinline__ unsigned short i8_f2bf(float f) { return __builtin_bit_cast(unsigned short, static_cast<__bf16>(f)); }
__device__ __forceinline__ unsigned i8_pack_bf2(float lo, float hi) {
  typedef __bf16 bf16x2_ __attribute__((ext_vector_type(2)));
  typedef float f32x2_ __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2_{lo, hi}, bf16x2_));
}

// GELU(x) = max(x, 0) - |x| Q(|x|), Q(a) = erfc(a / sqrt 2) / 2 = 2^P8(a): a polynomial fitted to log2 Q with Q as the weight, so that the error of |x| Q is
// 4.1e-8 at most (at 1.54), fp32 rounding included, 4.8e-8 with an exponential that is off by its last place, and for every a (the leading coefficient is
// negative: past the fit's 5.5, where Q is 2e-8, 2^P8 falls faster than Q).  Relative to the tail itself that is 1 % at -5, 12 % at -6, 56 % at -7, where
// GELU is -1.4e-6, -6e-9 and -9e-12.  One v_exp and eleven plain instructions on scalars, as packed fp32 ones are off; with erfc as t P5(t) exp(-a^2 / 2), t = 1 / (1 + c a), 63104 x 2304
// x 768 took 178 us, with this 170.  (The factor is held below infinity: infinity times zero is no number.)
__device__ __forceinline__ float i8_gelu(float x) {
  const float a = fabsf(x);
  float p = fmaf(-2.7720532216e-06f, a, 3.8620797568e-05f);
  p = fmaf(p, a, -1.8254783936e-04f);
  p = fmaf(p, a, -1.4586953330e-04f);
  p = fmaf(p, a, 7.0754708722e-03f);
  p = fmaf(p, a, -5.2505027503e-02f);
  p = fmaf(p, a, -4.5920491219e-01f);
  p = fmaf(p, a, -1.1511057615e+00f);
  p = fmaf(p, a, -1.0f);
  return fmaf(-fminf(a, 3.0e38f), __builtin_amdgcn_exp2f(p), fmaxf(x, 0.f));
}

__device__ __forceinline__ float i8_relu(float x) { return x < 0.f ? 0.f : x; }      // (a row without numbers stays one)

// ------------------------------------------------------------------------------------ row quantiser
// 16 to 256 lanes per row.  The codes are those of real arithmetic: with e the exponent of a, n = x 127 2^-e is exact for bf16 x (and carried with
// its rounding error for fp32 x), b = a 2^-e lies in [1, 2), and n / b is formed as r0 = n y, y = 1 / b, corrected by the exact remainder
// fma(-r0, b, n): a correctly rounded quotient, so that x = a / 2 is 63.5 and not a neighbour of it.  Rounding to the integer is the
// addition of 1.5 2^23, whose low byte is then the code.  A bf16 x has no quotient within 2^-16 of a half that is none (2 n and an odd multiple of b are
// multiples of 2^-14 at least); an fp32 x has, and its quotient as a float may be a half that it is not.  An element with a quotient that near a half
// in one of the wave's rows is therefore coded again by the sign of an exact difference (quant_code_exact): about one in a thousand (4096 x 4096 in
// fp32 14.2 us, without the second look 13.9 and 1.2e-6 of normal rows' codes wrong by one).
// Bound: the memory, a row is read once and held (63104 x 768 bf16 24.5 us, 6 TB/s with the codes, part of it from the last-level cache).
struct QuantArgs { const void* x; long ldx; signed char* q; long ldq; float* scale; int M, K, Kp; };
constexpr float kQuantTiny = 7.888609052210118e-31f;      // 2^-100

struct RowScale { float c, b, y; bool bad; };
__device__ __forceinline__ RowScale row_scale(unsigned abits, float* scale) {      // abits: the row's largest |x| as fp32 bits
  RowScale s;
  s.bad = abits >= 0x7f800000u;                                // an infinity or a NaN: integer order puts them above every number
  const unsigned tiny = __float_as_uint(kQuantTiny);
  const unsigned a = s.bad ? 0x3f800000u : (abits > tiny ? abits : tiny);
  const unsigned e = a >> 23;                                  // biased exponent, 27 .. 254
  s.b = __uint_as_float((a & 0x007fffffu) | 0x3f800000u);
  s.c = 127.0f * __uint_as_float((254u - e + (e == 254u)) << 23) * (e == 254u ? 0.5f : 1.0f);      // 127 2^-e (2^-127 is formed in two factors)
  s.y = 1.0f / s.b;
  *scale = s.bad ? __uint_as_float(0x7fc00000u) : __uint_as_float(a) / 127.0f;
  return s;
}
constexpr float kQuantRound = 12582912.0f;                     // 1.5 2^23
// k = an integer within one half and a few roundings of the quotient: n - k b is then a float (a multiple of 2^-23 below 1 + 2^-14), and so is its distance
// from b / 2 where that is small; with n's rounding error e1 added, the sum's sign is the sign of |x 127 / a - k| - 1/2.
__device__ __forceinline__ unsigned quant_code_exact(float x, const RowScale& s) {
  const float n = x * s.c, e1 = fmaf(x, s.c, -n);
  const float t = fmaf(n, s.y, kQuantRound);
  const float d = fmaf(-(t - kQuantRound), s.b, n);
  const float past = (fabsf(d) - 0.5f * s.b) + (d < 0.f ? -e1 : e1);
  const unsigned k = __float_as_uint(t);
  return past > 0.f || (past == 0.f && (k & 1u)) ? k + (d < 0.f ? -1 : 1) : k;
}
template <bool kF32, int kN>
__device__ __forceinline__ void quant_codes(const float (&x)[kN], const RowScale& s, unsigned (&q)[kN]) {
  float off[kN], most = 0.f;                                   // distances of the quotients from their integers
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const float n = x[j] * s.c;
    const float r0 = n * s.y;
    float rem = fmaf(-r0, s.b, n);
    if (kF32) rem += fmaf(x[j], s.c, -n);
    const float r = fmaf(rem, s.y, r0), t = r + kQuantRound;
    q[j] = __float_as_uint(t);
    if (kF32) {
      off[j] = fabsf(r - (t - kQuantRound));
      most = fmaxf(most, off[j]);
    }
  }
  if constexpr (kF32) {
    constexpr float kNear = 0.5f - 0x1p-17f;                   // (a quotient is off by half of 2^-17, its last rounding, and 2^-38)
    if (__builtin_amdgcn_ballot_w64(most > kNear) != 0) {
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (__builtin_amdgcn_ballot_w64(off[j] > kNear) != 0) q[j] = quant_code_exact(x[j], s);
    }
  }
}
__device__ __forceinline__ unsigned pack_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {      // the low bytes
  const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// eight elements of a row from column k on, zeros past K
template <bool kF32>
__device__ __forceinline__ void load8(const QuantArgs& a, long row, int k, bool vec, float (&v)[8]) {
  if (kF32) {
    const float* p = static_cast<const float*>(a.x) + row * a.ldx + k;
    if (vec && k + 8 <= a.K) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = lo[j]; v[4 + j] = hi[j]; }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < a.K ? p[j] : 0.f;
    }
  } else {
    const unsigned short* p = static_cast<const unsigned short*>(a.x) + row * a.ldx + k;
    if (vec && k + 8 <= a.K) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < a.K ? i8_bf2f(p[j]) : 0.f;
    }
  }
}
template <int kLanes>
__device__ __forceinline__ unsigned lanes_max_u32(unsigned v) {
#pragma unroll
  for (int o = (kLanes < 64 ? kLanes : 64) / 2; o > 0; o >>= 1) { const unsigned t = __shfl_xor(v, o); v = t > v ? t : v; }
  if constexpr (kLanes == 256) {                 // the workgroup's four waves share a row
    __shared__ unsigned part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) v = part[w] > v ? part[w] : v;
  }
  return v;
}
__device__ __forceinline__ unsigned widest8(const float (&v)[8], unsigned mx) {
#pragma unroll
  for (int j = 0; j < 8; ++j) { const unsigned t = __float_as_uint(v[j]) & 0x7fffffffu; mx = t > mx ? t : mx; }
  return mx;
}
template <bool kF32>
__device__ __forceinline__ uint2 quant8(const float (&v)[8], const RowScale& s) {
  unsigned q[8];
  quant_codes<kF32>(v, s, q);
  return s.bad ? make_uint2(0u, 0u) : make_uint2(pack_bytes(q[0], q[1], q[2], q[3]), pack_bytes(q[4], q[5], q[6], q[7]));
}
// kLanes lanes per row, kP pieces of eight elements per lane held in registers from the maximum to the codes: one read of x.  kP = 0: any K,
// the row is read twice.
template <bool kF32, int kLanes, int kP>
__global__ __launch_bounds__(256) void quant_rows_i8_kernel(QuantArgs a, bool vec) {
  const int sub = threadIdx.x % kLanes;
  const long row = static_cast<long>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const bool live = row < a.M;
  const long r = live ? row : a.M - 1;           // (lanes of rows past the last one take part in the exchanges)
  float v[kP > 0 ? kP : 1][8];
  unsigned mx = 0;
  if constexpr (kP > 0) {
#pragma unroll
    for (int p = 0; p < kP; ++p) load8<kF32>(a, r, 8 * (sub + kLanes * p), vec, v[p]);
#pragma unroll
    for (int p = 0; p < kP; ++p) mx = widest8(v[p], mx);
  } else {
    for (int k = 8 * sub; k < a.Kp; k += 8 * kLanes) {
      load8<kF32>(a, r, k, vec, v[0]);
      mx = widest8(v[0], mx);
    }
  }
  float sc;
  const RowScale s = row_scale(lanes_max_u32<kLanes>(mx), &sc);
  if (!live) return;
  if (sub == 0) a.scale[row] = sc;
  if constexpr (kP > 0) {
#pragma unroll
    for (int p = 0; p < kP; ++p) {
      const int k = 8 * (sub + kLanes * p);
      if (k < a.Kp) *reinterpret_cast<uint2*>(a.q + row * a.ldq + k) = quant8<kF32>(v[p], s);
    }
  } else {
    for (int k = 8 * sub; k < a.Kp; k += 8 * kLanes) {
      load8<kF32>(a, r, k, vec, v[0]);
      *reinterpret_cast<uint2*>(a.q + row * a.ldq + k) = quant8<kF32>(v[0], s);
    }
  }
}

// ------------------------------------------------------------------------------------ products
// The weight rows are the matrix instruction's rows and the token rows its columns, so a lane's four accumulators are four neighbouring
// output channels of one token.  Which weight row an instruction's row i of block j stands for is free, and is chosen so that the lane's
// blocks join: bf16 outputs n = 32 (j / 2) + 8 (i / 4) + 4 (j & 1) + (i & 3), eight neighbours = 16 bytes per lane and store; fp32 outputs
// n = 16 j + i, four neighbours = 16 bytes.  The result leaves the registers without a trip through LDS.
struct GemmI8Args {
  const signed char* A; long lda; const float* a_scale;
  const signed char* B; long ldb; const float* b_scale;
  void* C; long ldc;
  const float* bias; const float* residual; long ld_res; int res_row_mod; unsigned short* aux; long ld_aux;
  int M, N, K, act;
  bool stream;                  // the rows of C are whole 128-byte lines
};
// Rows of the outputs and the residual begin wherever the caller's strides put them, so their 16-byte pieces are typed by their elements' alignment;
// the hardware takes wide accesses there: 17297 x 2602 x 1190 in bf16 takes 70 us, one element at a time it took 150.
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ int w_row_bf16(int j, int i) { return 32 * (j >> 1) + 8 * (i >> 2) + 4 * (j & 1) + (i & 3); }

// What a call's epilogue is made of, as far as it is known when the kernel is compiled: everything at run time costs the 256 x 256 kernel 80 KB of
// code, more than an instruction cache holds.
__device__ __forceinline__ const float* i8_residual(const GemmI8Args& g, long m, int n) {
  return g.residual + (g.res_row_mod ? static_cast<unsigned>(m) % static_cast<unsigned>(g.res_row_mod) : m) * g.ld_res + n;
}
constexpr int kI8Plain = 0, kI8Gelu = 1, kI8Residual = 2, kI8Any = 3;      // no activation / GELU, and no residual / copy; residual and / or copy, no activation; whatever the call says
__device__ __forceinline__ f32x4 i8_residual4(const GemmI8Args& g, long m, int n) {
  const float* r = i8_residual(g, m, n);
  if (n + 4 <= g.N) return *reinterpret_cast<const f32x4_any*>(r);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < g.N) v[e] = r[e];
  return v;
}
// A piece of a row, channels n ..: eight bf16 results or four fp32 ones.  Where rows are whole 128-byte lines the 256 x 256 kernel's leave
// nontemporal (63104 x 2304 x 768: 132 / 155 us with and without, fp32 169 / 210; 16384 x 2312 x 768, where they are not, 52.6 / 42.0, fp32 96 / 59).
template <bool kStream>
__device__ __forceinline__ void i8_put_bf16(unsigned short* row, int n, int n_end, u32x4 v, bool stream) {
  if (n + 8 <= n_end) {
    u32x4_any* c = reinterpret_cast<u32x4_any*>(row + n);
    if (kStream && stream) {                     // (the empty statements keep the two stores two: joined, they lose the hint)
      asm volatile("" ::: "memory");
      __builtin_nontemporal_store(v, c);
      asm volatile("" ::: "memory");
    } else {
      *c = v;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (n + e < n_end) row[n + e] = static_cast<unsigned short>(v[e >> 1] >> (16 * (e & 1)));
}
template <bool kStream>
__device__ __forceinline__ void i8_put_f32(float* row, int n, int n_end, f32x4 v, bool stream) {
  if (n + 4 <= n_end) {
    f32x4_any* c = reinterpret_cast<f32x4_any*>(row + n);
    if (kStream && stream) {                     // (the empty statements keep the two stores two: joined, they lose the hint)
      asm volatile("" ::: "memory");
      __builtin_nontemporal_store(v, c);
      asm volatile("" ::: "memory");
    } else {
      *c = v;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < n_end) row[n + e] = v[e];
}
__device__ __forceinline__ void i8_put_copy(unsigned short* row, int n, int n_end, f32x4 v) {      // four bf16 results
  const unsigned lo = i8_pack_bf2(v[0], v[1]), hi = i8_pack_bf2(v[2], v[3]);
  if (n + 4 <= n_end) {
    *reinterpret_cast<u32x2_any*>(row + n) = u32x2_any{lo, hi};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < n_end) row[n + e] = static_cast<unsigned short>((e < 2 ? lo : hi) >> (16 * (e & 1)));
}

// The results of a wave's kT token blocks (16 tokens each, rows m0 ..) x 64 channels (n0 ..).  acc_of(j, t) is the lane's accumulator quad of channel
// block j and token block t, as_of(t) its token's scale; bs_of(c) and bias_of(c) give a channel's scale and bias.
//
// A lane holds two 16-byte pieces of one row that lie half a 128-byte line apart (bf16: channels 8 lg and 32 + 8 lg; fp32: 4 lg and 16 + 4 lg of each half).
// Lanes li and li ^ 8 trade one for the other, so that a store covers whole lines of eight rows instead of half lines of sixteen: 63104 x 2304
// bf16 results wrote 345 MB with half lines for their 291 MB (139 -> 133 us).  All residual rows of a group of blocks are requested at once.
template <bool kOut32, int kForm, int kT, bool kStream, typename AccOf, typename AsOf, typename BsOf, typename BiasOf>
__device__ __forceinline__ void i8_store_tile(const GemmI8Args& g, long m0, int n0, int li, int lg, AccOf acc_of, AsOf as_of, BsOf bs_of, BiasOf bias_of) {
  constexpr int kN = kOut32 ? 4 : 8, kGap = kOut32 ? 16 : 32;
  const bool low = li < 8;
  constexpr int kMost = kForm >= kI8Residual && !kOut32 ? (kT == 8 ? 1 : 2) : 4, kGroup = kT < kMost ? kT : kMost;      // token blocks whose residual rows are in flight together
#pragma unroll
  for (int b = 0; b < 8 / kN; ++b) {             // pairs of pieces
    const int nl = kOut32 ? 32 * b + 4 * lg : 8 * lg;
    if (n0 + nl >= g.N) continue;
    float bs[2][kN], bias[2][kN];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < kN; ++e) { bs[h][e] = bs_of(nl + h * kGap + e); bias[h][e] = bias_of(nl + h * kGap + e); }
    const int n = n0 + nl + (low ? 0 : kGap);    // of the two pieces that this lane stores, in rows li & 7 and 8 + (li & 7)
    const bool in = n < g.N;
#pragma unroll
    for (int t0 = 0; t0 < kT; t0 += kGroup) {
      f32x4 ahead[kForm >= kI8Residual ? kGroup : 1][kOut32 ? 2 : 4];
      if constexpr (kForm >= kI8Residual) {
#pragma unroll
        for (int t = 0; t < kGroup; ++t) {
#pragma unroll
          for (int q = 0; q < (kOut32 ? 2 : 4); ++q) {        // fp32: the two pieces as they are stored; bf16: four quads as they are computed
            const long m = min(m0 + 16 * (t0 + t) + (kOut32 ? 8 * q + (li & 7) : li), static_cast<long>(g.M) - 1);
            const int c = kOut32 ? n : n0 + nl + (q >> 1) * kGap + 4 * (q & 1);
            ahead[t][q] = g.residual && c < g.N ? i8_residual4(g, m, c) : f32x4{0.f, 0.f, 0.f, 0.f};
          }
        }
      }
#pragma unroll
      for (int t = 0; t < kGroup; ++t) {
        const float as = as_of(t0 + t);
        unsigned w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float z[kN];
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            const int a = kOut32 ? acc_of(2 * b + h, t0 + t)[e & 3] : acc_of(2 * h + (e >> 2), t0 + t)[e & 3];
            z[e] = static_cast<float>(a) * as * bs[h][e] + bias[h][e];
            if (kForm == kI8Gelu) z[e] = i8_gelu(z[e]);
            if (kForm == kI8Any) z[e] = g.act == 1 ? i8_gelu(z[e]) : (g.act == 2 ? i8_relu(z[e]) : z[e]);
            if (kForm >= kI8Residual && !kOut32) z[e] += ahead[t][(2 * h + (e >> 2)) & (kOut32 ? 1 : 3)][e & 3];
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) w[h][q] = kOut32 ? __float_as_uint(z[q]) : i8_pack_bf2(z[(2 * q) % kN], z[(2 * q + 1) % kN]);
        }
        u32x4 s[2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          s[0][q] = __builtin_amdgcn_update_dpp(w[0][q], w[1][q], 0x128, 0xf, 0xc, false);            // row_ror:8: lane li ^ 8; lanes 8 .. 15 take
          s[1][q] = __builtin_amdgcn_update_dpp(w[1][q], w[0][q], 0x128, 0xf, 0x3, false);            // lanes 0 .. 7 take
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const long m = m0 + 16 * (t0 + t) + 8 * r + (li & 7);
          if (!in || m >= g.M) continue;
          if constexpr (kOut32) {
            f32x4 v = __builtin_bit_cast(f32x4, s[r]);
            if (kForm >= kI8Residual) v += ahead[t][r];
            i8_put_f32<kStream>(static_cast<float*>(g.C) + m * g.ldc, n, g.N, v, g.stream);
            if (kForm >= kI8Residual && g.aux) i8_put_copy(g.aux + m * g.ld_aux, n, g.N, v);
          } else {
            i8_put_bf16<kStream>(static_cast<unsigned short*>(g.C) + m * g.ldc, n, g.N, s[r], g.stream);
          }
        }
      }
    }
  }
}

// ---- kTile x kTile tiles, K in steps of 128 bytes through a ring of kStages LDS stages filled by LDS-DMA
//
// 128: 2 x 2 waves of 64 tokens x 64 channels.  64: four pairs of waves of 16 tokens x 64 channels, half of every step each, which join at the end
// (1000 x 1000 x 4800 in bf16 15.6 us with one wave each, 13.3 with two).  kStages - 1 steps are on their way while one is multiplied: a
// call whose tiles leave CUs idle is bound by the time of a step's round trip, and the ring divides that by its depth.
// One barrier a step: behind it step s has landed for every wave, and every wave has read what step s + kStages - 1 is fetched over.
__device__ __attribute__((aligned(16))) unsigned g_i8_zero[4];
// position p of LDS row r holds the row's 16-byte piece p ^ f(r); f makes the 16 rows of a fragment read fall on all eight positions twice
__device__ __forceinline__ int i8_swz_natural(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int i8_swz_bf16(int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); }

// LDS-DMA as inline asm without results: through the builtin the compiler takes every later LDS read to depend on it and waits for all
// fetches in front of it.  The waits are the explicit ones of the schedule.
__device__ __forceinline__ unsigned i8_lds_addr(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}
__device__ __forceinline__ void i8_dma16(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(src), "s"(lds) : "memory");
}
__device__ __forceinline__ void i8_dma4(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(src), "s"(lds) : "memory");
}

constexpr int i8_tile_lds(int tile, int stages) { return stages * 2 * tile * 128; }
template <bool kOut32, int kForm, int kTile, int kStages>
__global__ __launch_bounds__(kTile == 64 ? 512 : 256) void gemm_i8_kernel(GemmI8Args g, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // [stage][token tile | weight tile]
  constexpr int kOp = kTile * 128, kTok = kTile == 128 ? 4 : 1, kDma = kTile == 128 ? 4 : 1;      // bytes of an operand's stage; a wave's token blocks; its fetches of an operand
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = kTile == 128 ? wave >> 1 : wave & 3, wn = kTile == 128 ? wave & 1 : 0;
  constexpr int kKs = kTile == 128 ? 2 : 1;      // of a step's two halves, those that a wave multiplies
  const int ks0 = kTile == 128 ? 0 : wave >> 2;
  // blocks b and b + 8 share an XCD and its L2: every XCD gets a contiguous range of tiles, the tiles of a token panel side by side
  const int nwg = tiles_m * tiles_n, bid = blockIdx.x;
  const int q8 = nwg >> 3, r8 = nwg & 7, xcd = bid & 7;
  const int logical = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (bid >> 3);
  const int m0 = (logical / tiles_n) * kTile, n0 = (logical % tiles_n) * kTile;
  const int steps = (g.K + 127) >> 7;

  // fetch i of this wave fills rows 8 (kDma wave + i) .. + 7 of a tile, 16 bytes per lane; rows past the matrix are the last one's
  const signed char *pa[kDma], *pb[kDma];
  int ka[kDma], kb[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int row = 8 * (kDma * wave + i) + (lane >> 3);
    ka[i] = ((lane & 7) ^ i8_swz_natural(row)) * 16;
    kb[i] = ((lane & 7) ^ (kOut32 ? i8_swz_natural(row) : i8_swz_bf16(row))) * 16;
    const int ar = min(m0 + row, g.M - 1), br = min(n0 + row, g.N - 1);
    pa[i] = g.A + static_cast<long>(ar) * g.lda + ka[i];
    pb[i] = g.B + static_cast<long>(br) * g.ldb + kb[i];
  }
  const unsigned lds0 = i8_lds_addr(smem);
  auto dma = [&](int step, int stage) {          // steps past the end fetch zeros into stages that nobody reads, so that the counts stay exact
    const unsigned st = lds0 + stage * 2 * kOp + kDma * wave * 1024;
    const int k0 = step * 128;
#pragma unroll
    for (int i = 0; i < kDma; ++i) {             // pieces past K are zeros on both sides
      i8_dma16(k0 + ka[i] < g.K ? static_cast<const void*>(pa[i] + k0) : static_cast<const void*>(g_i8_zero), st + i * 1024);
      i8_dma16(k0 + kb[i] < g.K ? static_cast<const void*>(pb[i] + k0) : static_cast<const void*>(g_i8_zero), st + kOp + i * 1024);
    }
  };
  const int li = lane & 15, lg = lane >> 4, sw = (li >> 1) & 7;
  int xr[kTok], wr[4];
#pragma unroll
  for (int t = 0; t < kTok; ++t) xr[t] = (wm * 16 * kTok + 16 * t + li) * 128;
#pragma unroll
  for (int t = 0; t < 4; ++t) wr[t] = kOp + (wn * 64 + (kOut32 ? 16 * t + li : w_row_bf16(t, li))) * 128;
  i32x4 acc[4][kTok];                            // [weight block][token block]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kTok; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) dma(s, s);
  int stage = 0;
  for (int s = 0; s < steps; ++s) {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"((kStages - 2) * 2 * kDma) : "memory");
    asm volatile("s_barrier" ::: "memory");
    const int last = stage == 0 ? kStages - 1 : stage - 1;
    dma(s + kStages - 1, last);
    const unsigned char* st = smem + stage * 2 * kOp;
    i32x4 xf[kKs][kTok], wf[kKs][4];
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) {
      const int c = ((4 * (ks0 + ks) + lg) ^ sw) * 16;
#pragma unroll
      for (int t = 0; t < kTok; ++t) xf[ks][t] = *reinterpret_cast<const i32x4*>(st + xr[t] + c);
#pragma unroll
      for (int t = 0; t < 4; ++t) wf[ks][t] = *reinterpret_cast<const i32x4*>(st + wr[t] + c);
    }
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kTok; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[ks][i], xf[ks][j], acc[i][j], 0, 0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // (the reads are done in front of the next barrier)
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // no fetch outlives its workgroup's LDS
  if constexpr (kTile == 64) {                   // the two waves of a block join, one integer sum
    __syncthreads();
    i32x4* const part = reinterpret_cast<i32x4*>(smem) + wm * 256 + lane;
    if (wave >= 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[64 * i] = acc[i][0];
    }
    __syncthreads();
    if (wave >= 4) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][0] += part[64 * i];
  }
  float as[kTok];
#pragma unroll
  for (int j = 0; j < kTok; ++j) as[j] = g.a_scale[min(m0 + wm * 16 * kTok + 16 * j + li, g.M - 1)];
  const int nw = n0 + wn * 64;
  i8_store_tile<kOut32, kForm, kTok, false>(g, m0 + wm * 16 * kTok, nw, li, lg, [&](int i, int j) { return acc[i][j]; }, [&](int j) { return as[j]; },
                                            [&](int c) { return g.b_scale[min(nw + c, g.N - 1)]; }, [&](int c) { return g.bias ? g.bias[min(nw + c, g.N - 1)] : 0.f; });
}

// ---- few tokens: 16 kMT tokens x 16 channels per workgroup, K dealt in steps of 64 bytes over its eight waves, which join through LDS
//
// What bounds such a call is the time of a memory round trip, not its bytes, so a wave asks for the operands of several steps at once and there
// is one launch where the rows still have to be quantised (kX: x is bf16 or fp32): every workgroup then quantises its 16 rows for itself,
// 7 instructions a code, from the registers that hold its share of them (K up to 2048).
constexpr int kI8SkinnyDepth = 4, kI8SkinnyWaves = 8;
struct LinearX { const void* x; long ldx; int K; bool vec; };      // K columns of x; GemmI8Args::K is K rounded up to 16
enum { kXInt8 = 0, kXBf16 = 1, kXF32 = 2 };
template <bool kOut32, int kMT, int kX>
__global__ __launch_bounds__(64 * kI8SkinnyWaves) void gemm_i8_skinny_kernel(GemmI8Args g, LinearX lx) {
  static_assert(kX == kXInt8 || kMT == 1, "rows are quantised here for one block of tokens");
  constexpr int kW = kI8SkinnyWaves;
  __shared__ int part[kW][16 * kMT][20];
  __shared__ unsigned smax[kW][16];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * kMT;
  const int steps = (g.K + 63) >> 6;
  // what the end needs is asked for at the start: four channels of one token per thread
  const int er = tid >> 2, en = n0 + 4 * (tid & 3);
  const long em = m0 + er;
  const bool mine = tid < 64 * kMT && em < g.M && en < g.N;
  float ebs[4], ebias[4], eas = 0.f;
  if (mine) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = min(en + j, g.N - 1);
      ebs[j] = g.b_scale[c];
      ebias[j] = g.bias ? g.bias[c] : 0.f;
    }
    if (kX == kXInt8) eas = g.a_scale[em];
  }
  const signed char* pb = g.B + static_cast<long>(min(n0 + li, g.N - 1)) * g.ldb + 16 * lg;
  const i32x4 zero = {0, 0, 0, 0};
  i32x4 acc[kMT];
#pragma unroll
  for (int t = 0; t < kMT; ++t) acc[t] = zero;
  float a_own = 0.f;                             // kX: the scale of this lane's token
  if constexpr (kX == kXInt8) {
    const signed char* pa[kMT];
#pragma unroll
    for (int t = 0; t < kMT; ++t) pa[t] = g.A + static_cast<long>(min(m0 + 16 * t + li, g.M - 1)) * g.lda + 16 * lg;
    for (int s0 = wave; s0 < steps; s0 += kW * kI8SkinnyDepth) {
      i32x4 fb[kI8SkinnyDepth], fa[kMT][kI8SkinnyDepth];
#pragma unroll
      for (int i = 0; i < kI8SkinnyDepth; ++i) {
        const int k = 64 * (s0 + kW * i);
        const bool in = k + 16 * lg < g.K;         // the last step's pieces past K, and steps past the last one
        fb[i] = in ? *reinterpret_cast<const i32x4*>(pb + k) : zero;
#pragma unroll
        for (int t = 0; t < kMT; ++t) fa[t][i] = in ? *reinterpret_cast<const i32x4*>(pa[t] + k) : zero;
      }
#pragma unroll
      for (int i = 0; i < kI8SkinnyDepth; ++i)
#pragma unroll
        for (int t = 0; t < kMT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[i], fa[t][i], acc[t], 0, 0, 0);
    }
  } else {
    const QuantArgs qa{lx.x, lx.ldx, nullptr, 0, nullptr, g.M, lx.K, g.K};
    const long row = min(m0 + li, g.M - 1);
    float held[kI8SkinnyDepth][16];
    i32x4 fb[kI8SkinnyDepth];
    auto load16 = [&](int s, float (&v)[16]) {
      float lo[8], hi[8];
      load8<kX == kXF32>(qa, row, 64 * s + 16 * lg, lx.vec, lo);
      load8<kX == kXF32>(qa, row, 64 * s + 16 * lg + 8, lx.vec, hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) { v[j] = lo[j]; v[8 + j] = hi[j]; }
    };
    unsigned mx = 0;
    auto widen = [&](const float (&v)[16]) {
#pragma unroll
      for (int j = 0; j < 16; ++j) { const unsigned t = __float_as_uint(v[j]) & 0x7fffffffu; mx = t > mx ? t : mx; }
    };
#pragma unroll
    for (int i = 0; i < kI8SkinnyDepth; ++i) {     // (past K: zeros)
      const int s = wave + kW * i, k = 64 * s;
      fb[i] = k + 16 * lg < g.K ? *reinterpret_cast<const i32x4*>(pb + k) : zero;
      if (s < steps) load16(s, held[i]);         // (wave-uniform)
    }
#pragma unroll
    for (int i = 0; i < kI8SkinnyDepth; ++i)
      if (wave + kW * i < steps) widen(held[i]);
    { const unsigned a = __shfl_xor(mx, 16); mx = a > mx ? a : mx; }
    { const unsigned a = __shfl_xor(mx, 32); mx = a > mx ? a : mx; }
    if (lg == 0) smax[wave][li] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kW; ++w) mx = smax[w][li] > mx ? smax[w][li] : mx;
    const RowScale rs = row_scale(mx, &a_own);
    auto codes = [&](const float (&v)[16]) {
      i32x4 f;
      unsigned c[16];
      quant_codes<kX == kXF32>(v, rs, c);
#pragma unroll
      for (int q = 0; q < 4; ++q) f[q] = rs.bad ? 0 : static_cast<int>(pack_bytes(c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]));
      return f;
    };
#pragma unroll
    for (int i = 0; i < kI8SkinnyDepth; ++i)
      if (wave + kW * i < steps) acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[i], codes(held[i]), acc[0], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < kMT; ++t) *reinterpret_cast<i32x4*>(&part[wave][16 * t + li][4 * lg]) = acc[t];
  __shared__ float srow[16];
  if (kX != kXInt8 && wave == 0 && lg == 0) srow[li] = a_own;
  __syncthreads();
  if (!mine) return;
  int z[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = 4 * (tid & 3) + j;
    z[j] = 0;
#pragma unroll
    for (int w = 0; w < kW; ++w) z[j] += part[w][er][c];
  }
  const float as = kX == kXInt8 ? eas : srow[er & 15];
  f32x4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = static_cast<float>(z[j]) * as * ebs[j] + ebias[j];
    if (g.act == 1) y[j] = i8_gelu(y[j]);
    else if (g.act == 2) y[j] = i8_relu(y[j]);
  }
  if (g.residual) y += i8_residual4(g, em, en);
  if (kOut32) {
    i8_put_f32<false>(static_cast<float*>(g.C) + em * g.ldc, en, g.N, y, false);
    if (g.aux) i8_put_copy(g.aux + em * g.ld_aux, en, g.N, y);
  } else {
    i8_put_copy(static_cast<unsigned short*>(g.C) + em * g.ldc, en, g.N, y);
  }
}

// ---- 256 x 256 tile, eight waves (2 x 4, 128 tokens x 64 channels each), K in steps of 128 bytes, one persistent workgroup per CU
//
// LDS: two buffers of four half-tiles of 128 rows x 128 bytes,
//     A_h: token rows wr 128 + 64 h + 0..63 of the tile for the wave rows wr = 0, 1;  B_h: weight rows wc 64 + 32 h + 0..31 for the wave columns wc = 0..3
// so that a half-tile is consumed in one phase by all waves.  A K-step is four phases of 16 products per wave:
//     phase 1: read B_0, A_0   products (A_0, B_0)   fetch A_1 of step t + 1
//     phase 2: read B_1        products (A_0, B_1)   fetch B_0 of step t + 2
//     phase 3: read A_1        products (A_1, B_1)   fetch A_0 of step t + 2
//     phase 4:                 products (A_1, B_0)   fetch B_1 of step t + 2
// In front of its first barrier a phase waits for what the next one reads and for no more: five half-tiles (80 KB) stay in flight, which
// is what the loop's rate hangs on (the latency of a loaded L2 is more than a microsecond).
// The wave rows run one barrier apart, so that one row's LDS reads and fetches lie under the other row's products on the same SIMDs.
// A fetched half is read at least a phase after the wait that retires it; it is fetched into again two phases after its last read, or one
// phase after where those reads were retired in front of that phase's barrier (B_0).  Barriers are raw, a __syncthreads would drain the
// fetches.  Steps past the end fetch the last one again into halves that nobody reads, so that the counts stay exact.
// Tiles are dealt statically: the workgroups of an XCD (block index modulo 8) walk one contiguous eighth of the tiles, in groups of a few tile
// columns; no counters, so a captured launch is like any other.  The next tile's first fetches, its scales among them, are issued before this
// tile's results are scaled and stored, which needs no LDS tile of its own.
constexpr int kI8Half = 128 * 128;
constexpr int kI8Buf = 4 * kI8Half;              // A_0 | A_1 | B_0 | B_1
constexpr int kI8Scales = 3 * 256 * 4;           // a_scale | b_scale | bias of a tile
constexpr int kI8BigLds = 2 * kI8Buf + 2 * kI8Scales;

template <bool kOut32, int kForm, bool kTail>
__global__ __launch_bounds__(512) void gemm_i8_256_kernel(GemmI8Args g, int tiles_m, int tiles_n, int group_n) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 2, wc = wave & 3;
  const int k_steps = (g.K + 127) >> 7;
  const int n_tiles = tiles_m * tiles_n, xg = blockIdx.x & 7;
  const int q8 = n_tiles >> 3, r8 = n_tiles & 7;
  const int slice0 = xg < r8 ? xg * (q8 + 1) : r8 * (q8 + 1) + (xg - r8) * q8, slice_n = q8 + (xg < r8 ? 1 : 0);
  const int stride = (static_cast<int>(gridDim.x) + 7 - xg) >> 3;
  int v = blockIdx.x >> 3;
  if (v >= slice_n) return;

  // fetch j of this wave fills LDS rows 8 (2 wave + j) + (lane >> 3) of a half-tile, position p of row r holding the piece p ^ f(r)
  const signed char *pa[2][2], *pb[2][2];        // [half][j]
  int kca[2], kcb[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 8 * (2 * wave + j) + (lane >> 3);
    kca[j] = ((lane & 7) ^ i8_swz_natural(r)) * 16;
    kcb[j] = ((lane & 7) ^ (kOut32 ? i8_swz_natural(r) : i8_swz_bf16(r))) * 16;
  }
  const unsigned lds0 = i8_lds_addr(smem);
  auto set_tile = [&](int v_, int& m0, int& n0) {
    const int logical = slice0 + v_;
    const int per_group = tiles_m * group_n;
    const int cg = logical / per_group, rem = logical - cg * per_group;
    const int gw = min(group_n, tiles_n - cg * group_n);
    m0 = (rem / gw) * 256;
    n0 = (cg * group_n + rem % gw) * 256;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 8 * (2 * wave + j) + (lane >> 3);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int ar = min(m0 + (r >> 6) * 128 + h * 64 + (r & 63), g.M - 1);
        pa[h][j] = g.A + static_cast<long>(ar) * g.lda + kca[j];
        const int br = min(n0 + (r >> 5) * 64 + h * 32 + (r & 31), g.N - 1);
        pb[h][j] = g.B + static_cast<long>(br) * g.ldb + kcb[j];
      }
    }
  };
  auto dma = [&](const signed char* const (&p)[2], const int (&kc)[2], int step, int buf, int half) {
    const int s = step < k_steps ? step : k_steps - 1;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const void* src = p[j] + static_cast<long>(s) * 128;
      if (kTail) src = s * 128 + kc[j] < g.K ? src : static_cast<const void*>(g_i8_zero);      // (else K is a multiple of 128)
      i8_dma16(src, lds0 + buf * kI8Buf + half * kI8Half + (2 * wave + j) * 1024);
    }
  };
  auto prologue = [&](int m0, int n0, int sbuf) {      // the tile's scales; step 0 whole; B_0, A_0, B_1 of step 1
    const unsigned sl = lds0 + 2 * kI8Buf + sbuf * kI8Scales + (wave & 3) * 256;
    if (wave < 4) {
      i8_dma4(g.a_scale + min(m0 + 64 * wave + lane, g.M - 1), sl);
    } else {
      const int n = min(n0 + 64 * (wave - 4) + lane, g.N - 1);
      i8_dma4(g.b_scale + n, sl + 1024);
      if (g.bias) i8_dma4(g.bias + n, sl + 2048);
    }
    dma(pb[0], kcb, 0, 0, 2); dma(pa[0], kca, 0, 0, 0); dma(pb[1], kcb, 0, 0, 3); dma(pa[1], kca, 0, 0, 1);
    dma(pb[0], kcb, 1, 1, 2); dma(pa[0], kca, 1, 1, 0); dma(pb[1], kcb, 1, 1, 3);
  };
  // fragment reads (byte offsets in a half-tile): token rows wr 64 + 16 i + li; weight rows wc 32 + (bf16 outputs: 8 (li / 4) + 4 j + (li & 3), fp32: 16 j + li)
  const int sw = (li >> 1) & 7;
  const int c0 = (lg ^ sw) * 16, c1 = c0 ^ 64;
  const int a_off = (wr * 64 + li) * 128;
  const int b_off = 2 * kI8Half + (wc * 32 + (kOut32 ? li : 8 * (li >> 2) + (li & 3))) * 128;
  constexpr int kBj = kOut32 ? 16 * 128 : 4 * 128;
  i32x4 fa[4][2], fb0[2][2], fb1[2][2];
#define ADT_I8_READ_A(H)                                                                                   \
  _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                          \
    fa[i][0] = *reinterpret_cast<const i32x4*>(st + a_off + c0 + (H) * kI8Half + i * 2048);                 \
    fa[i][1] = *reinterpret_cast<const i32x4*>(st + a_off + c1 + (H) * kI8Half + i * 2048);                 \
  }
#define ADT_I8_READ_B(F, H)                                                                                \
  _Pragma("unroll") for (int j = 0; j < 2; ++j) {                                                          \
    F[j][0] = *reinterpret_cast<const i32x4*>(st + b_off + c0 + (H) * kI8Half + j * kBj);                   \
    F[j][1] = *reinterpret_cast<const i32x4*>(st + b_off + c1 + (H) * kI8Half + j * kBj);                   \
  }
// What the next phase reads has landed when the five half-tiles asked for after it, ten fetches of this wave, are all that is in flight -- or those
// and the stores that stand between them in the order of issue (a tile's first phases after an interior tile).
#define ADT_I8_LANDED(BEHIND_STORES)                                                                       \
  do {                                                                                                     \
    if (stored && (BEHIND_STORES)) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(10 + kStores) : "memory");     \
    else asm volatile("s_waitcnt vmcnt(10)" ::: "memory");                                                 \
  } while (0)
#define ADT_I8_QUAD(I0, FB, J0)                                                                            \
  do {                                                                                                     \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                     \
    __builtin_amdgcn_sched_barrier(0);                                                                     \
    __builtin_amdgcn_s_setprio(1);                                                                         \
    _Pragma("unroll") for (int ks = 0; ks < 2; ++ks)                                                       \
      _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                        \
        _Pragma("unroll") for (int j = 0; j < 2; ++j)                                                      \
          acc[I0 + i][J0 + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(FB[j][ks], fa[i][ks], acc[I0 + i][J0 + j], 0, 0, 0); \
    __builtin_amdgcn_s_setprio(0);                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                     \
    asm volatile("s_barrier" ::: "memory");                                                                \
  } while (0)

  constexpr int kStores = kOut32 ? 32 : 16;      // 16-byte stores of a wave's 128 x 64 results
  int m0, n0, sbuf = 0;
  set_tile(v, m0, n0);
  prologue(m0, n0, 0);
  asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
  bool stored = false;                           // the tile before left its last stores in flight
  asm volatile("s_barrier" ::: "memory");
  while (true) {
    i32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    if (wr == 1) asm volatile("s_barrier" ::: "memory");
    for (int t = 0; t < k_steps; ++t) {
      const int buf = t & 1;
      const unsigned char* st = smem + buf * kI8Buf;
      ADT_I8_READ_B(fb0, 0)
      __builtin_amdgcn_sched_barrier(0);
      ADT_I8_READ_A(0)
      dma(pa[1], kca, t + 1, buf ^ 1, 1);
      asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");           // the B_0 reads: B_0 is fetched into in phase 2
      ADT_I8_LANDED(t <= 1);
      asm volatile("s_barrier" ::: "memory");
      ADT_I8_QUAD(0, fb0, 0);
      ADT_I8_READ_B(fb1, 1)
      dma(pb[0], kcb, t + 2, buf, 2);
      ADT_I8_LANDED(t == 0);
      asm volatile("s_barrier" ::: "memory");
      ADT_I8_QUAD(0, fb1, 2);
      ADT_I8_READ_A(1)
      dma(pa[0], kca, t + 2, buf, 0);
      asm volatile("s_barrier" ::: "memory");
      ADT_I8_QUAD(4, fb1, 2);
      dma(pb[1], kcb, t + 2, buf, 3);
      ADT_I8_LANDED(t == 0);
      asm volatile("s_barrier" ::: "memory");
      ADT_I8_QUAD(4, fb0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (wr == 0) asm volatile("s_barrier" ::: "memory");
    asm volatile("s_barrier" ::: "memory");        // every fetch has landed and every fragment is read: the buffers are free
    const int em0 = m0, en0 = n0;
    const float* const scales = reinterpret_cast<const float*>(smem + 2 * kI8Buf + sbuf * kI8Scales);
    v += stride;
    const bool more = v < slice_n;                 // block-uniform
    if (more) {
      sbuf ^= 1;
      set_tile(v, m0, n0);
      prologue(m0, n0, sbuf);
    }
    float as[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) as[i] = scales[wr * 128 + 16 * i + li];
    i8_store_tile<kOut32, kForm, 8, true>(g, em0 + wr * 128, en0 + wc * 64, li, lg, [&](int j, int i) { return acc[i][j]; }, [&](int i) { return as[i]; },
                                          [&](int c) { return scales[256 + wc * 64 + c]; }, [&](int c) { return g.bias ? scales[512 + wc * 64 + c] : 0.f; });
    if (!more) break;
    // The next tile's first fetches are older than this tile's stores, and a wave of an interior tile has just issued kStores of those at least: they
    // may stay in flight under the next tile's first steps.  A wave of an edge tile may have issued none.
    stored = em0 + 256 <= g.M && en0 + 256 <= g.N;
    if (stored) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(10 + kStores) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_barrier" ::: "memory");
  }
#undef ADT_I8_READ_A
#undef ADT_I8_READ_B
#undef ADT_I8_QUAD
#undef ADT_I8_LANDED
}

}  // namespace adt

using namespace adt;

namespace adt {
// Lanes per row: the fewest that hold the row in at most three pieces each, so that no lane idles (768 columns: 32 lanes, three pieces); a whole
// workgroup past 2048 columns (us with 64 / 256 lanes, fp32: 4096 x 4096 17.2 / 14.0, 2048 x 8192 23.1 / 13.9, 1 x 3400 4.1 / 2.6)
template <bool kF32, int kLanes, int kP>
static void launch_quant_as(const QuantArgs& a, bool vec, hipStream_t st) {
  constexpr int64_t kRows = 256 / kLanes, kMost = kRows << 23;      // (a grid holds fewer than 2^32 threads)
  for (int64_t m0 = 0; m0 < a.M; m0 += kMost) {
    QuantArgs c = a;
    c.M = static_cast<int>(std::min(a.M - m0, kMost));
    c.x = static_cast<const char*>(a.x) + m0 * a.ldx * (kF32 ? 4 : 2);
    c.q = a.q + m0 * a.ldq;
    c.scale = a.scale + m0;
    hipLaunchKernelGGL((quant_rows_i8_kernel<kF32, kLanes, kP>), dim3(static_cast<unsigned>((c.M + kRows - 1) / kRows)), dim3(256), 0, st, c, vec);
  }
}
template <bool kF32>
static void launch_quant(const QuantArgs& a, bool vec, hipStream_t st) {
  const int pieces = (a.Kp + 7) / 8;
  if (pieces <= 16) launch_quant_as<kF32, 16, 1>(a, vec, st);
  else if (pieces <= 32) launch_quant_as<kF32, 16, 2>(a, vec, st);
  else if (pieces <= 48) launch_quant_as<kF32, 16, 3>(a, vec, st);
  else if (pieces <= 64) launch_quant_as<kF32, 32, 2>(a, vec, st);
  else if (pieces <= 96) launch_quant_as<kF32, 32, 3>(a, vec, st);
  else if (pieces <= 128) launch_quant_as<kF32, 64, 2>(a, vec, st);
  else if (pieces <= 192) launch_quant_as<kF32, 64, 3>(a, vec, st);
  else if (pieces <= 256) launch_quant_as<kF32, 64, 4>(a, vec, st);
  else if (pieces <= 512) launch_quant_as<kF32, 256, 2>(a, vec, st);
  else if (pieces <= 1024) launch_quant_as<kF32, 256, 4>(a, vec, st);
  else launch_quant_as<kF32, 256, 0>(a, vec, st);
}
}  // namespace adt

extern "C" int adt_quant_rows_i8(const void* x, int32_t x_fp32, int64_t ldx, int64_t M, int64_t K, void* q, int64_t ldq, float* scale, void* stream) {
  if (!x || !q || !scale) return set_error(ADT_EINVAL, "adt_quant_rows_i8: null pointer");
  if (M < 0 || K <= 0 || M > (1LL << 31) - 1 || K > (1LL << 17)) return set_error(ADT_ESHAPE, "adt_quant_rows_i8: M must fit 31 bits, 1 <= K <= 131072");
  const int64_t Kp = (K + 15) / 16 * 16;
  if (ldx < K || ldq < Kp || (ldq & 15) || !aligned16(q)) return set_error(ADT_EINVAL, "adt_quant_rows_i8: q rows are 16-byte aligned and hold K rounded up to 16 bytes");
  if (M == 0) return ADT_OK;
  QuantArgs a{x, static_cast<long>(ldx), static_cast<signed char*>(q), static_cast<long>(ldq), scale, static_cast<int>(M), static_cast<int>(K), static_cast<int>(Kp)};
  const bool vec = aligned16(x) && (ldx * (x_fp32 ? 4 : 2)) % 16 == 0;
  if (x_fp32) launch_quant<true>(a, vec, static_cast<hipStream_t>(stream));
  else launch_quant<false>(a, vec, static_cast<hipStream_t>(stream));
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

namespace adt {
static int gemm_i8_check(const char* who, int64_t M, int64_t N, int64_t K, const void* B, int64_t ldb, const float* b_scale, const void* C, int64_t ldc,
                         const adt_gemm_epilogue* ep) {
  static thread_local char msg[200];
  auto fail = [&](int code, const char* what) {
    snprintf(msg, sizeof(msg), "%s: %s", who, what);
    return set_error(code, msg);
  };
  if (!B || !C || !b_scale || !ep) return fail(ADT_EINVAL, "null pointer");
  if (M < 0 || N < 0 || K <= 0 || M > (1LL << 30) || N > (1LL << 30) || K > (1LL << 17)) return fail(ADT_ESHAPE, "M and N fit 30 bits, 1 <= K <= 131072 (the int32 sums stay exact)");
  if (ldb < (K + 15) / 16 * 16 || ldc < N || (ldb & 15) || !aligned16(B)) return fail(ADT_EINVAL, "weight rows are 16-byte aligned and hold K rounded up to 16; ldc >= N");
  if (ep->act < 0 || ep->act > 2 || ep->alpha != 1.0f) return fail(ADT_EINVAL, "act is 0, 1 or 2 and alpha 1");
  if (ep->gelu_grad_of || ep->pre_act_out || ep->colsum_out || ep->res_ln_mean || ep->drop.p > 0.f || ep->act_grad_mode || ep->side_fp32)
    return fail(ADT_EINVAL, "an inference product (bias, activation, residual, bf16 copy); the training epilogues are not its own");
  if (ep->aux_bf16_out && !ep->out_fp32) return fail(ADT_EINVAL, "aux_bf16_out goes with an fp32 C");
  if (ep->residual && (ep->res_row_mod < 0 || ep->ld_res < N)) return fail(ADT_EINVAL, "residual rows hold N floats");
  if (ep->aux_bf16_out && ep->ld_aux < N) return fail(ADT_EINVAL, "aux rows hold N elements");
  return ADT_OK;
}
// What the results may lie on.  In place every element of the residual is read and written by one lane, which needs it to be the same element in both; x: the
// rows, in either form.
static int gemm_i8_places_check(int64_t M, const void* x, const void* B, const void* C, int64_t ldc, const adt_gemm_epilogue* ep) {
  if (ep->residual == C && (!ep->out_fp32 || ep->res_row_mod || (M > 1 && ep->ld_res != ldc)))
    return set_error(ADT_EINVAL, "adt_gemm_i8: a residual in place is fp32, of C's row stride and without res_row_mod");
  const void* aux = ep->aux_bf16_out;
  if (C == x || C == B || (aux && (aux == x || aux == B || aux == C || aux == ep->residual)))
    return set_error(ADT_EINVAL, "adt_gemm_i8: C and aux_bf16_out share no memory with the operands or each other");
  return ADT_OK;
}
static GemmI8Args gemm_i8_args(int64_t M, int64_t N, int64_t Kp, const void* B, int64_t ldb, const float* b_scale, void* C, int64_t ldc, const adt_gemm_epilogue* ep) {
  GemmI8Args g{};
  g.B = static_cast<const signed char*>(B); g.ldb = ldb; g.b_scale = b_scale;
  g.C = C; g.ldc = ldc; g.bias = ep->bias; g.residual = static_cast<const float*>(ep->residual); g.ld_res = ep->ld_res; g.res_row_mod = ep->res_row_mod;
  g.aux = static_cast<unsigned short*>(ep->aux_bf16_out); g.ld_aux = ep->ld_aux;
  g.M = static_cast<int>(M); g.N = static_cast<int>(N); g.K = static_cast<int>(Kp); g.act = ep->act; 
  g.stream = (reinterpret_cast<uintptr_t>(C) & 127) == 0 && (ldc * (ep->out_fp32 ? 4 : 2)) % 128 == 0;
  return g;
}
template <bool kOut32, int kMT, int kX>
static int launch_i8_skinny(const GemmI8Args& g, const LinearX& lx, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((g.N + 15) / 16), static_cast<unsigned>((g.M + 16 * kMT - 1) / (16 * kMT)));
  hipLaunchKernelGGL((gemm_i8_skinny_kernel<kOut32, kMT, kX>), grid, dim3(64 * kI8SkinnyWaves), 0, st, g, lx);
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}
template <bool kOut32, int kTile, int kStages>
static int launch_i8_tile(const GemmI8Args& g, int form, int64_t tm, int64_t tn, hipStream_t st) {
  typedef void (*Fn)(GemmI8Args, int, int);
  static const Fn fns[4] = {gemm_i8_kernel<kOut32, 0, kTile, kStages>, gemm_i8_kernel<kOut32, 1, kTile, kStages>, gemm_i8_kernel<kOut32, 2, kTile, kStages>,
                            gemm_i8_kernel<kOut32, 3, kTile, kStages>};
  if (tm * tn >= 1LL << 24) return set_error(ADT_ESHAPE, "adt_gemm_i8: too many tiles");      // (a grid holds fewer than 2^32 threads; 2^30 x 128 results are 2^23)
  constexpr int kLds = i8_tile_lds(kTile, kStages);
  if (kLds > 65536) ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(fns[form]), hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  hipLaunchKernelGGL(fns[form], dim3(static_cast<unsigned>(tm * tn)), dim3(kTile == 64 ? 512 : 256), kLds, st, g, static_cast<int>(tm), static_cast<int>(tn));
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}
template <bool kOut32>
static int launch_i8(const GemmI8Args& g, hipStream_t st) {
  typedef void (*BigFn)(GemmI8Args, int, int, int);
  static const BigFn big[2][4] = {{gemm_i8_256_kernel<kOut32, 0, false>, gemm_i8_256_kernel<kOut32, 1, false>, gemm_i8_256_kernel<kOut32, 2, false>, gemm_i8_256_kernel<kOut32, 3, false>},
                                  {gemm_i8_256_kernel<kOut32, 0, true>, gemm_i8_256_kernel<kOut32, 1, true>, gemm_i8_256_kernel<kOut32, 2, true>, gemm_i8_256_kernel<kOut32, 3, true>}};
  int n_cu = 0;
  if (int rc = device_cu_count(&n_cu)) return rc;
  const bool extra = g.residual || g.aux;
  const int form = g.act == 0 ? (extra ? kI8Residual : kI8Plain) : (g.act == 1 && !extra ? kI8Gelu : kI8Any);
  const int64_t tm = (g.M + 127) / 128, tn = (g.N + 127) / 128, bm = (g.M + 255) / 256, bn = (g.N + 255) / 256, sm = (g.M + 63) / 64, sn = (g.N + 63) / 64;
  // Few tokens: the kernel that asks for everything at once, with 16, 32 or 64 tokens a workgroup, the fewest that leave one workgroup of 16 channels a CU,
  // or two where 32 are all there are; then 64 x 64 tiles while they are two a CU at most (us with 16 tokens / 32 / 64 / 64 x 64 tiles / 128 x 128:
  // 64 x 768 x 768 3.0 / 3.4 / 4.2 / -, 128 x 768 x 3000 5.7 / 5.0 / 6.7 / -, 64 x 4096 x 4096 17 / 13.4 / 11.9 / 10.5, 16 x 8000 x 768 3.7 / - / - / 4.7 / 7.5,
  // 32 x 16000 x 768 - / 7.3 / - / 4.8 / 7.7, 128 x 2304 x 768 - / - / 6.2 / 4.7 / 8.0, 256 x 4096 x 4096 - / - / 40 / 13.3 / 25.6;
  // three 64 x 64 tiles a CU, 1282 x 2263 x 137, 8.6 / 7.6).
  const int64_t cols = (g.N + 15) / 16;
  if ((g.M + 15) / 16 * cols <= (g.M <= 16 ? 2 : 1) * n_cu) return launch_i8_skinny<kOut32, 1, kXInt8>(g, LinearX{}, st);
  if ((g.M + 31) / 32 * cols <= (g.M <= 32 ? 2 : 1) * n_cu) return launch_i8_skinny<kOut32, 2, kXInt8>(g, LinearX{}, st);
  if (sm * cols <= n_cu) return launch_i8_skinny<kOut32, 4, kXInt8>(g, LinearX{}, st);
  if (sm * sn <= 2 * n_cu) return launch_i8_tile<kOut32, 64, 4>(g, form, sm, sn, st);
  // 256 x 256 tiles run one per CU and twice as efficiently, but in whole rounds: a round of them costs 1.6 of 128 x 128 ones at two per CU (us with
  // 256 / 128: 4096 x 2304 x 768 16.4 / 18.9, 7747 x 768 x 768 14.6 / 11.2, 8192 x 2304 x 768 29.4 / 29.3, 16384 x 2304 x 768 43.6 / 53.1,
  // 63104 x 2304 x 768 140 / 240, 2048 x 4096 x 4096 43.8 / 45.1, 4096^3 55.2 / 85.3).
  if (8 * ((bm * bn + n_cu - 1) / n_cu) <= 5 * ((tm * tn + 2 * n_cu - 1) / (2 * n_cu))) {
    const BigFn fn = big[(g.K & 127) != 0][form];
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, kI8BigLds));
    const int64_t wgs = bm * bn < n_cu ? bm * bn : n_cu;
    // tile columns walked together: as many as 2 MB of weights (half an XCD's L2) are, three at least; the token panels are then read once
    // (63104 x 2304 x 768, nine columns in one group or in threes: 137.6 / 142.0 us; 16384 x 2304 x 768 41.9 / 43.5)
    const int group_n = static_cast<int>(std::max<int64_t>(3, std::min<int64_t>(bn, (2 << 20) / (256LL * g.K))));
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(wgs)), dim3(512), kI8BigLds, st, g, static_cast<int>(bm), static_cast<int>(bn), group_n);
  } else {
    return launch_i8_tile<kOut32, 128, 2>(g, form, tm, tn, st);
  }
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}
}  // namespace adt

extern "C" int adt_gemm_i8(int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const float* a_scale, const void* B, int64_t ldb,
                           const float* b_scale, void* C, int64_t ldc, const adt_gemm_epilogue* ep, void* stream) {
  if (!A || !a_scale) return set_error(ADT_EINVAL, "adt_gemm_i8: null pointer");
  if (int rc = gemm_i8_check("adt_gemm_i8", M, N, K, B, ldb, b_scale, C, ldc, ep)) return rc;
  if (K & 15) return set_error(ADT_ESHAPE, "adt_gemm_i8: K must be a multiple of 16");
  if (lda < K || (lda & 15) || !aligned16(A)) return set_error(ADT_EINVAL, "adt_gemm_i8: operand rows are 16-byte aligned and hold K");
  if (M == 0 || N == 0) return ADT_OK;
  if (int rc = gemm_i8_places_check(M, A, B, C, ldc, ep)) return rc;
  GemmI8Args g = gemm_i8_args(M, N, K, B, ldb, b_scale, C, ldc, ep);
  g.A = static_cast<const signed char*>(A); g.lda = lda; g.a_scale = a_scale;
  return ep->out_fp32 ? launch_i8<true>(g, static_cast<hipStream_t>(stream)) : launch_i8<false>(g, static_cast<hipStream_t>(stream));
}

// Rows quantised inside the product: as long as a workgroup holds its 16 of them in registers, and every workgroup of the card is there for the repeated
// work of the next 16 channels (us in one launch / in two, bf16 rows: 1 x 2304 x 768 4.0 / 5.4, 64 x 768 x 768 4.2 / 7.0, 64 x 768 x 2048 6.5 / 10.1,
// 64 x 1400 x 768 5.5 / 7.1, 16 x 8000 x 768 5.8 / 6.4; past two workgroups a CU 64 x 2304 x 768 7.9 / 7.1, 16 x 30000 x 768 17.3 / 8.9).
static bool linear_i8_fused(int64_t M, int64_t N, int64_t K) {
  int n_cu = 256;
  (void)device_cu_count(&n_cu);
  return K <= 64 * kI8SkinnyDepth * kI8SkinnyWaves && M <= 16 * n_cu && (M + 15) / 16 * ((N + 15) / 16) <= 2 * n_cu;
}

extern "C" size_t adt_linear_i8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || linear_i8_fused(M, N, K)) return 0;
  return static_cast<size_t>(M) * ((K + 15) / 16 * 16) + static_cast<size_t>(M) * 4;
}

extern "C" int adt_linear_i8(int64_t M, int64_t N, int64_t K, const void* x, int32_t x_fp32, int64_t ldx, const void* W, int64_t ldw, const float* w_scale,
                             void* C, int64_t ldc, const adt_gemm_epilogue* ep, void* ws, size_t ws_bytes, void* stream) {
  if (!x) return set_error(ADT_EINVAL, "adt_linear_i8: null pointer");
  if (int rc = gemm_i8_check("adt_linear_i8", M, N, K, W, ldw, w_scale, C, ldc, ep)) return rc;
  if (ldx < K) return set_error(ADT_EINVAL, "adt_linear_i8: rows of x hold K elements");
  if (M == 0 || N == 0) return ADT_OK;
  if (int rc = gemm_i8_places_check(M, x, W, C, ldc, ep)) return rc;
  const int64_t Kp = (K + 15) / 16 * 16;
  GemmI8Args g = gemm_i8_args(M, N, Kp, W, ldw, w_scale, C, ldc, ep);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (linear_i8_fused(M, N, K)) {
    const LinearX lx{x, static_cast<long>(ldx), static_cast<int>(K), aligned16(x) && (ldx * (x_fp32 ? 4 : 2)) % 16 == 0};
    if (ep->out_fp32) return x_fp32 ? launch_i8_skinny<true, 1, kXF32>(g, lx, st) : launch_i8_skinny<true, 1, kXBf16>(g, lx, st);
    return x_fp32 ? launch_i8_skinny<false, 1, kXF32>(g, lx, st) : launch_i8_skinny<false, 1, kXBf16>(g, lx, st);
  }
  if (!ws || ws_bytes < adt_linear_i8_workspace_bytes(M, N, K) || !aligned16(ws)) return set_error(ADT_EINVAL, "adt_linear_i8: workspace too small or not 16-byte aligned");
  float* scale = reinterpret_cast<float*>(static_cast<char*>(ws) + M * Kp);
  if (int rc = adt_quant_rows_i8(x, x_fp32, ldx, M, K, ws, Kp, scale, stream)) return rc;
  g.A = static_cast<const signed char*>(ws); g.lda = Kp; g.a_scale = scale;
  return ep->out_fp32 ? launch_i8<true>(g, st) : launch_i8<false>(g, st);
}
