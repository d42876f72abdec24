// gemm_i8.hip -- matrix product in 8-bit integers with one scale per row of each operand (token / output channel), and the quantiser
// of the activations in front of it (gfx950).
//
//   quant_rows   a_m = max(max_k |x_mk|, 2^-100);  q_mk = the integer nearest to 127 x_mk / a_m (ties to even);  scale_m = a_m / 127
//   gemm_i8      acc_mn = sum_k a_mk b_nk (exact, int32);  z = acc * a_scale_m * b_scale_n + bias_n; activation; + residual_mn
//
// The int8 matrix instruction (v_mfma_i32_16x16x64_i8) does twice the products of the bf16 one per cycle on the same operand bytes.
#include <hip/hip_runtime.h>

#include "adt_common.h"

namespace adt {
#include "gelu.h"

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

// ------------------------------------------------------------------------------------ row quantiser
// One wave per row.  The codes are those of real arithmetic: with e the exponent of a, n = x 127 2^-e is exact for bf16 x (and carried with
// its rounding error for fp32 x), b = a 2^-e lies in [1, 2), and n / b is formed as r0 = n y, y = 1 / b, corrected by the exact remainder
// fma(-r0, b, n): a correctly rounded quotient, so that x = a / 2 is 63.5 and not a neighbour of it.  Rounding to the integer is the
// addition of 1.5 2^23, whose low byte is then the code.
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
template <bool kF32>
__device__ __forceinline__ unsigned quant_code(float x, const RowScale& s) {
  const float n = x * s.c;
  const float r0 = n * s.y;
  float rem = fmaf(-r0, s.b, n);
  if (kF32) rem += fmaf(x, s.c, -n);
  const float r = fmaf(rem, s.y, r0);
  return __float_as_uint(r + 12582912.0f);
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
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const unsigned t = __shfl_xor(v, o); v = t > v ? t : v; }
  return v;
}
template <bool kF32>
__global__ __launch_bounds__(256) void quant_rows_i8_kernel(QuantArgs a, bool vec) {
  const int lane = threadIdx.x & 63;
  const long row = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= a.M) return;
  unsigned mx = 0;
  for (int k = 8 * lane; k < a.Kp; k += 512) {
    float v[8];
    load8<kF32>(a, row, k, vec, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) { const unsigned t = __float_as_uint(v[j]) & 0x7fffffffu; mx = t > mx ? t : mx; }
  }
  float sc;
  const RowScale s = row_scale(wave_max_u32(mx), &sc);
  if (lane == 0) a.scale[row] = sc;
  for (int k = 8 * lane; k < a.Kp; k += 512) {
    float v[8];
    load8<kF32>(a, row, k, vec, v);
    unsigned q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = s.bad ? 0u : quant_code<kF32>(v[j], s);
    *reinterpret_cast<uint2*>(a.q + row * a.ldq + k) = make_uint2(pack_bytes(q[0], q[1], q[2], q[3]), pack_bytes(q[4], q[5], q[6], q[7]));
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
  bool vec;                     // N % 8 == 0 and every row of C, bias, b_scale, residual and aux 16-byte aligned
};
__device__ __forceinline__ int w_row_bf16(int j, int i) { return 32 * (j >> 1) + 8 * (i >> 2) + 4 * (j & 1) + (i & 3); }

template <bool kOut32, int kN>
__device__ __forceinline__ void i8_store(const GemmI8Args& g, long m, int n, const int (&acc)[kN], float as, const float (&bs)[kN], const float (&bias)[kN]) {
  float z[kN];
  const float* res = nullptr;
  if (g.residual) res = g.residual + (g.res_row_mod ? m % g.res_row_mod : m) * g.ld_res + n;
  const bool whole = g.vec && n + kN <= g.N;
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    z[e] = static_cast<float>(acc[e]) * as * bs[e] + bias[e];
    if (g.act == 1) z[e] = gelu_erf(z[e]);
    else if (g.act == 2) z[e] = fmaxf(z[e], 0.f);
  }
  if (whole) {
    if (res) {
#pragma unroll
      for (int e = 0; e < kN; e += 4) {
        const f32x4 r = *reinterpret_cast<const f32x4*>(res + e);
        z[e] += r[0]; z[e + 1] += r[1]; z[e + 2] += r[2]; z[e + 3] += r[3];
      }
    }
    if (kOut32) {
      float* c = static_cast<float*>(g.C) + m * g.ldc + n;
#pragma unroll
      for (int e = 0; e < kN; e += 4) *reinterpret_cast<f32x4*>(c + e) = f32x4{z[e], z[e + 1], z[e + 2], z[e + 3]};
    }
    unsigned p[kN / 2];
#pragma unroll
    for (int e = 0; e < kN / 2; ++e) p[e] = i8_pack_bf2(z[2 * e], z[2 * e + 1]);
    unsigned short* h = kOut32 ? g.aux : static_cast<unsigned short*>(g.C);
    const long ldh = kOut32 ? g.ld_aux : g.ldc;
    if (!kOut32 || h) {
      if constexpr (kN == 8) *reinterpret_cast<u32x4*>(h + m * ldh + n) = u32x4{p[0], p[1], p[2], p[3]};
      else *reinterpret_cast<uint2*>(h + m * ldh + n) = make_uint2(p[0], p[1]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    if (n + e >= g.N) continue;
    const float v = res ? z[e] + res[e] : z[e];
    if (kOut32) static_cast<float*>(g.C)[m * g.ldc + n + e] = v;
    else static_cast<unsigned short*>(g.C)[m * g.ldc + n + e] = i8_f2bf(v);
    if (kOut32 && g.aux) g.aux[m * g.ld_aux + n + e] = i8_f2bf(v);
  }
}

// ---- 128 x 128 tile, four waves (2 x 2, 64 x 64 each), K in steps of 128 bytes, two LDS stages filled by LDS-DMA
constexpr int kI8Tile = 128 * 128;               // one operand's stage: 128 rows x 128 bytes
constexpr int kI8Lds = 4 * kI8Tile;
__device__ __attribute__((aligned(16))) unsigned g_i8_zero[4];
// position p of LDS row r holds the row's 16-byte piece p ^ f(r); f makes the 16 rows of a fragment read fall on all eight positions twice
__device__ __forceinline__ int i8_swz_natural(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int i8_swz_bf16(int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); }

template <bool kOut32>
__global__ __launch_bounds__(256) void gemm_i8_kernel(GemmI8Args g, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // [2 stages][token tile | weight tile]
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  // blocks b and b + 8 share an XCD and its L2: every XCD gets a contiguous range of tiles, the tiles of a token panel side by side
  const int nwg = tiles_m * tiles_n, bid = blockIdx.x;
  const int q8 = nwg >> 3, r8 = nwg & 7, xcd = bid & 7;
  const int logical = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (bid >> 3);
  const int m0 = (logical / tiles_n) * 128, n0 = (logical % tiles_n) * 128;
  const int steps = (g.K + 127) >> 7;

  // DMA instruction i of this wave fills rows 8 (4 wave + i) .. + 7 of a tile, 16 bytes per lane; rows past the matrix are the last one's
  const signed char *pa[4], *pb[4];
  int ka[4], kb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * (4 * wave + i) + (lane >> 3);
    ka[i] = ((lane & 7) ^ i8_swz_natural(row)) * 16;
    kb[i] = ((lane & 7) ^ (kOut32 ? i8_swz_natural(row) : i8_swz_bf16(row))) * 16;
    const int ar = min(m0 + row, g.M - 1), br = min(n0 + row, g.N - 1);
    pa[i] = g.A + static_cast<long>(ar) * g.lda + ka[i];
    pb[i] = g.B + static_cast<long>(br) * g.ldb + kb[i];
  }
  auto dma = [&](int step) {
    unsigned char* st = smem + (step & 1) * 2 * kI8Tile;
    const int k0 = step * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {                // pieces past K are zeros on both sides
      const void* sa = k0 + ka[i] < g.K ? static_cast<const void*>(pa[i] + k0) : static_cast<const void*>(g_i8_zero);
      const void* sb = k0 + kb[i] < g.K ? static_cast<const void*>(pb[i] + k0) : static_cast<const void*>(g_i8_zero);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)sa, (__attribute__((address_space(3))) void*)(st + (4 * wave + i) * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)sb, (__attribute__((address_space(3))) void*)(st + kI8Tile + (4 * wave + i) * 1024), 16, 0, 0);
    }
  };
  const int li = lane & 15, lg = lane >> 4, sw = (li >> 1) & 7;
  int xr[4], wr[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    xr[t] = (wm * 64 + 16 * t + li) * 128;
    wr[t] = kI8Tile + (wn * 64 + (kOut32 ? 16 * t + li : w_row_bf16(t, li))) * 128;
  }
  i32x4 acc[4][4];                               // [weight block][token block]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  dma(0);
  __syncthreads();
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) dma(s + 1);
    const unsigned char* st = smem + (s & 1) * 2 * kI8Tile;
    i32x4 xf[2][4], wf[2][4];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int c = ((4 * ks + lg) ^ sw) * 16;
        xf[ks][t] = *reinterpret_cast<const i32x4*>(st + xr[t] + c);
        wf[ks][t] = *reinterpret_cast<const i32x4*>(st + wr[t] + c);
      }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[ks][i], xf[ks][j], acc[i][j], 0, 0, 0);
    __syncthreads();
  }
  constexpr int kN = kOut32 ? 4 : 8;
#pragma unroll
  for (int b = 0; b < 16 / kN; ++b) {            // the lane's groups of kN channels
    const int n = n0 + wn * 64 + (kOut32 ? 16 * b + 4 * lg : 32 * b + 8 * lg);
    if (n >= g.N) continue;
    float bs[kN], bias[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const int c = min(n + e, g.N - 1);
      bs[e] = g.b_scale[c];
      bias[e] = g.bias ? g.bias[c] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long m = m0 + wm * 64 + 16 * j + li;
      if (m >= g.M) continue;
      int v[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = kOut32 ? acc[b][j][e & 3] : acc[2 * b + (e >> 2)][j][e & 3];
      i8_store<kOut32, kN>(g, m, n, v, g.a_scale[m], bs, bias);
    }
  }
}

}  // namespace adt

using namespace adt;

extern "C" int adt_quant_rows_i8(const void* x, int32_t x_fp32, int64_t ldx, int64_t M, int64_t K, void* q, int64_t ldq, float* scale, void* stream) {
  if (!x || !q || !scale) return set_error(ADT_EINVAL, "adt_quant_rows_i8: null pointer");
  if (M < 0 || K <= 0 || M > (1LL << 31) - 1 || K > (1LL << 17)) return set_error(ADT_ESHAPE, "adt_quant_rows_i8: M must fit 31 bits, 1 <= K <= 131072");
  const int64_t Kp = (K + 15) / 16 * 16;
  if (ldx < K || ldq < Kp || (ldq & 15) || !aligned16(q)) return set_error(ADT_EINVAL, "adt_quant_rows_i8: q rows are 16-byte aligned and hold K rounded up to 16 bytes");
  if (M == 0) return ADT_OK;
  QuantArgs a{x, static_cast<long>(ldx), static_cast<signed char*>(q), static_cast<long>(ldq), scale, static_cast<int>(M), static_cast<int>(K), static_cast<int>(Kp)};
  const bool vec = aligned16(x) && (ldx * (x_fp32 ? 4 : 2)) % 16 == 0;
  const dim3 grid(static_cast<unsigned>((M + 3) / 4));
  if (x_fp32) hipLaunchKernelGGL(quant_rows_i8_kernel<true>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a, vec);
  else hipLaunchKernelGGL(quant_rows_i8_kernel<false>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a, vec);
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

extern "C" int adt_gemm_i8(int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const float* a_scale, const void* B, int64_t ldb,
                           const float* b_scale, void* C, int64_t ldc, const adt_gemm_epilogue* ep, void* stream) {
  if (!A || !B || !C || !a_scale || !b_scale || !ep) return set_error(ADT_EINVAL, "adt_gemm_i8: null pointer");
  if (M < 0 || N < 0 || K <= 0 || M > (1LL << 30) || N > (1LL << 30) || K > (1LL << 17) || (K & 15))
    return set_error(ADT_ESHAPE, "adt_gemm_i8: K must be a multiple of 16, at most 131072 (the int32 sums stay exact)");
  if (lda < K || ldb < K || ldc < N || (lda & 15) || (ldb & 15) || !aligned16(A) || !aligned16(B))
    return set_error(ADT_EINVAL, "adt_gemm_i8: operand rows are 16-byte aligned; lda, ldb >= K, ldc >= N");
  if (ep->act < 0 || ep->act > 2 || ep->alpha != 1.0f) return set_error(ADT_EINVAL, "adt_gemm_i8: act is 0, 1 or 2 and alpha 1");
  if (ep->gelu_grad_of || ep->pre_act_out || ep->colsum_out || ep->res_ln_mean || ep->drop.p > 0.f || ep->act_grad_mode || ep->side_fp32)
    return set_error(ADT_EINVAL, "adt_gemm_i8: an inference product (bias, activation, residual, bf16 copy); the training epilogues are not its own");
  if (ep->aux_bf16_out && !ep->out_fp32) return set_error(ADT_EINVAL, "adt_gemm_i8: aux_bf16_out goes with an fp32 C");
  if (ep->residual && (ep->res_row_mod < 0 || ep->ld_res < N)) return set_error(ADT_EINVAL, "adt_gemm_i8: residual rows hold N floats");
  if (ep->aux_bf16_out && ep->ld_aux < N) return set_error(ADT_EINVAL, "adt_gemm_i8: aux rows hold N elements");
  if (M == 0 || N == 0) return ADT_OK;
  GemmI8Args g{};
  g.A = static_cast<const signed char*>(A); g.lda = lda; g.a_scale = a_scale;
  g.B = static_cast<const signed char*>(B); g.ldb = ldb; g.b_scale = b_scale;
  g.C = C; g.ldc = ldc; g.bias = ep->bias; g.residual = static_cast<const float*>(ep->residual); g.ld_res = ep->ld_res; g.res_row_mod = ep->res_row_mod;
  g.aux = static_cast<unsigned short*>(ep->aux_bf16_out); g.ld_aux = ep->ld_aux;
  g.M = static_cast<int>(M); g.N = static_cast<int>(N); g.K = static_cast<int>(K); g.act = ep->act;
  auto ok = [](const void* p, int64_t ld, int elem) { return !p || (aligned16(p) && (ld * elem) % 16 == 0); };
  g.vec = (N % 8) == 0 && ok(C, ldc, ep->out_fp32 ? 4 : 2) && ok(g.bias, 4, 4) && ok(b_scale, 4, 4) && ok(g.residual, g.ld_res, 4) && ok(g.aux, g.ld_aux, 2);
  const int64_t tm = (M + 127) / 128, tn = (N + 127) / 128;
  if (tm * tn > (1LL << 31) - 1) return set_error(ADT_ESHAPE, "adt_gemm_i8: too many tiles");
  const auto fn = ep->out_fp32 ? gemm_i8_kernel<true> : gemm_i8_kernel<false>;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(tm * tn)), dim3(256), kI8Lds, static_cast<hipStream_t>(stream), g, static_cast<int>(tm), static_cast<int>(tn));
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}
