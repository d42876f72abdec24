// htsat_fused.hip -- K15: fused row-block kernels for the HBM-bound stages of the CLAP HTSAT audio encoder (gfx950).
//
// Stands behind the two halves of transformers' ClapAudioLayer.forward as the reference reaches it through
// ClapWrapper._get_audio_features (modules/clap_encoder.py:45-49 -> modeling_clap.py ClapAudioLayer: layernorm_before -> q/k/v ->
// window attention -> attention.output.dense -> + shortcut;  layernorm_after -> intermediate.dense -> GELU -> output.dense -> +).
// In the first two stages (C = 96 / 192 channels, 4096 / 1024 tokens per clip) these layers are bandwidth problems: at 512 clips
// the residual stream of stage 0 alone is 805 MB, and run as separate LayerNorm / GEMM launches a layer moves ~14 GB.  Here a
// wave owns 32 token rows from the first load to the last store:
//
//   mode LN_GEMM   (q/k/v):      x fp32 -> LayerNorm -> bf16 operand in registers -> W[3C, C] -> + bias -> bf16 qkv
//   mode GEMM_RES  (attn. out):  ctx bf16 -> W[C, C] -> + bias + x -> x            (in place)
//   mode MERGE_GEMM (patch merging): the 2x2 neighbourhood of a token, four rows of C/4 channels in ClapAudioPatchMerging's order ->
//                                LayerNorm(C) -> W[C/2, C] -> fp32 rows of the next stage's residual stream (the gathered, normalised
//                                bf16 tensor of adt_patch_merge_ln + GEMM never exists)
//   mode MLP:                    x fp32 -> LayerNorm -> W1[4C, C] -> + bias, GELU (erf form, gelu.h) -> W2[C, 4C] -> + bias + x -> x   (in place;
//                                the 4C-wide hidden activation never leaves the registers)
//
// MFMA orientation (v_mfma_f32_32x32x16_bf16): the TOKEN is the lane.  A operand = 32 weight rows, B operand = the lane's token row,
// so the accumulator tile is [32 output units][32 tokens] with a token's outputs in its own lane -- bias / GELU are per-lane
// arithmetic, and accumulator registers 8s .. 8s+7 ARE the bf16 B operand of k-step s of the next product (the hidden unit order
// 16s + 8(j>>2) + 4h + (j&3) they come in is baked into the packing of W2).  Activations therefore never touch LDS.
// Weights are pre-packed on the host into the order the kernel consumes them, one 1 KiB MFMA fragment (64 lanes x 16 bytes) after the
// other, and streamed global -> LDS by LDS-DMA in chunks through a ring shared by the 4 waves (128 tokens) of a workgroup: one
// barrier per chunk, two chunks ahead in flight; two workgroups share a CU.  LDS reads of the loop are inline asm (a compiler-generated LDS access
// would be ordered behind the DMA in flight with a vmcnt(0)).
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <type_traits>

#include "adt_common.h"

namespace adt {

typedef __attribute__((ext_vector_type(8))) short bf16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
#include "gelu.h"

constexpr int kRbThreads = 256;           // 4 waves x 32 tokens; two workgroups per CU (<= 80 KiB of LDS, <= 256 registers): one loads /
constexpr int kRbRows = 128;              // stores its rows while the other computes
constexpr int kRbWaves = kRbThreads / 64;
enum { kRbLnGemm = 0, kRbGemmRes = 1, kRbMlp = 2, kRbLnGemmGelu = 4, kRbMergeGemm = 5 };   // (3: the MLP phase by phase, an A/B arm of 2)

struct RbArgs {
  float* x;                      // [M, C] fp32 residual stream (read; written by GEMM_RES / MLP)
  const unsigned short* a16;     // GEMM_RES: bf16 input [M, lda]
  long lda;
  const float *gamma, *beta;     // LayerNorm (LN_GEMM, MLP)
  float eps;
  const unsigned char* wpk;      // packed weight stream, n_chunks * chunk bytes
  const float* bias1;            // [32 * n_tiles]: qkv bias / out-proj bias / fc1 bias
  const float* bias2;            // MLP: fc2 bias [C]
  unsigned short* out16;         // LN_GEMM: bf16 output [M, ldo]
  long ldo;
  long M;
  int n_tiles;                   // 32-unit output tiles of the (first) product
  float* out32;                  // MERGE_GEMM: fp32 output [M, ldo]
  int merge_R;                   // MERGE_GEMM: side of the SOURCE token grid (x is [B * R * R, C / 4]; M = B * (R / 2)^2)
};

__device__ __forceinline__ unsigned lds_off_f(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) const void*)p));
}
__device__ __forceinline__ unsigned pack2_f(float lo, float hi) {
  unsigned r;
  asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi));
  return r;
}
__device__ __forceinline__ void zero_acc(f32x16& x) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
}
// compile-time loop: body(std::integral_constant<int, I>{}) for I = I0 .. N - 1 (a `#pragma unroll` over 48 large iterations is refused by
// the unroller's size limit, and a rolled loop indexes the register arrays dynamically)
template <int I, int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<I + 1, N>(f);
  }
}
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void wait_lgkm() { asm volatile("s_waitcnt lgkmcnt(%0)" :: "n"(N) : "memory"); }

template <int C, int MODE, int TPC>
__global__ __launch_bounds__(kRbThreads, 2) void htsat_rowblock_kernel(RbArgs a) {
  constexpr int KS = C / 16;                                  // k-steps of the product over the C input channels
  constexpr int CT = C / 32;                                  // 32-channel tiles of the MLP's second product
  constexpr int kTileFrags = MODE == kRbMlp ? 2 * KS : KS;    // KiB of packed weights per 32-unit tile
  constexpr int kChunkKb = TPC * kTileFrags;
  constexpr int kChunkBytes = kChunkKb * 1024;
  constexpr int kRing = 3;
  constexpr int kDepth = kRing - 1;                           // chunks in flight ahead of the one being consumed
  // LDS-DMA work split: every participating wave issues IPW instructions per chunk (uniform counts keep vmcnt arithmetic uniform;
  // a wave that issues none passes the counted waits trivially)
  constexpr int IPW = kChunkKb % kRbWaves == 0 ? kChunkKb / kRbWaves : 6;
  constexpr int kDmaWaves = kChunkKb / IPW;
  static_assert(kDmaWaves * IPW == kChunkKb && kDmaWaves <= kRbWaves, "chunk size must split evenly over the waves");
  static_assert(kRing * kChunkBytes <= 76 * 1024, "two workgroups per CU");
  static_assert(KS % 6 == 0, "C must be a multiple of 96");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];   // [ring][chunk] | bias1 [32 * n_tiles] fp32
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long row0 = static_cast<long>(blockIdx.x) * kRbRows + wave * 32;
  long tok = row0 + r;
  const bool row_ok = tok < a.M;
  if (!row_ok) tok = a.M - 1;                                  // clamped loads, predicated stores
  float* bias_lds = reinterpret_cast<float*>(smem + kRing * kChunkBytes);
  const int n_chunks = a.n_tiles / TPC;

  auto issue_chunk = [&](int c) {
    if (wave < kDmaWaves) {
      const unsigned char* src = a.wpk + static_cast<long>(c) * kChunkBytes + (wave * IPW) * 1024 + lane * 16;
      unsigned char* dst = smem + (c % kRing) * kChunkBytes + (wave * IPW) * 1024;
#pragma unroll
      for (int i = 0; i < IPW; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + i * 1024),
                                         (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, 0, 0);
    }
  };

  // the weight stream starts first: its latency hides under the row loads and the LayerNorm
#pragma unroll
  for (int c = 0; c < kDepth; ++c)
    if (c < n_chunks) issue_chunk(c);

  // ---- prologue: the token row -> bf16 B operands b[s] (lane holds channels 16s + 8h .. + 7 of its token)
  bf16x8 b[KS];
  if (MODE == kRbGemmRes) {
    const unsigned short* ap = a.a16 + tok * a.lda + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 v = *reinterpret_cast<const uint4*>(ap + 16 * s);
      b[s] = *reinterpret_cast<const bf16x8*>(&v);
    }
  } else {
    const float* xp = a.x + tok * C + 8 * h;
    long mbase = 0;                                            // MERGE_GEMM: source row of the neighbourhood's (even, even) token
    if (MODE == kRbMergeGemm) {
      const int R2 = a.merge_R >> 1;
      const long per = static_cast<long>(R2) * R2, bb = tok / per;
      const int rem = static_cast<int>(tok - bb * per), i = rem / R2, j = rem - i * R2;
      mbase = (bb * a.merge_R + 2 * i) * a.merge_R + 2 * j;
    }
    float xv[KS][8];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (MODE == kRbMergeGemm) {                              // channels [q C/4, (q + 1) C/4) come from source (2i + (q & 1), 2j + (q >> 1))
        constexpr int SPQ = KS / 4;
        const int q = s / SPQ;
        xp = a.x + (mbase + (q & 1) * a.merge_R + (q >> 1)) * (C / 4) + 8 * h - 16 * (q * SPQ);
      }
      const float4 v0 = *reinterpret_cast<const float4*>(xp + 16 * s), v1 = *reinterpret_cast<const float4*>(xp + 16 * s + 4);
      xv[s][0] = v0.x; xv[s][1] = v0.y; xv[s][2] = v0.z; xv[s][3] = v0.w; xv[s][4] = v1.x; xv[s][5] = v1.y; xv[s][6] = v1.z; xv[s][7] = v1.w;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += xv[s][e];
    }
    sum += __shfl_xor(sum, 32);                                // the other half of the row lives in lane ^ 32
    const float mean = sum * (1.0f / C);
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float d = xv[s][e] - mean; ss = fmaf(d, d, ss); }
    ss += __shfl_xor(ss, 32);
    const float rstd = rsqrtf(ss * (1.0f / C) + a.eps);
    // gamma == nullptr: plain normalisation -- the caller folded gamma into the columns of the following weight and W beta into its bias (the
    // fused tower does: 4 KS loads of gamma / beta cost a lone wave ~10 k cycles of issue per workgroup, profiles/r06/clap_residual_ab.txt)
    auto ln_pack = [&](auto affine_tag, int s) {
      union { unsigned u[4]; bf16x8 v; } pk;
      if constexpr (decltype(affine_tag)::value) {
        const float4 g0 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h), g1 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h + 4);
        const float4 e0 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h), e1 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h + 4);
        const float ga[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w}, be[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pk.u[e] = pack2_f(fmaf((xv[s][2 * e] - mean) * rstd, ga[2 * e], be[2 * e]), fmaf((xv[s][2 * e + 1] - mean) * rstd, ga[2 * e + 1], be[2 * e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) pk.u[e] = pack2_f((xv[s][2 * e] - mean) * rstd, (xv[s][2 * e + 1] - mean) * rstd);
      }
      b[s] = pk.v;
    };
#pragma unroll
    for (int s = 0; s < KS; ++s) ln_pack(std::true_type{}, s);
  }
  // GEMM_RES: the residual in the accumulator layout (channel 32n + 8g + 4h + e of the lane's token), loaded before any DMA is in flight
  constexpr bool kPreloadRes = MODE == kRbGemmRes && CT * 16 <= 96;       // C = 384: 192 registers -- loaded per tile instead
  f32x4 res[kPreloadRes ? CT * 4 : 1];
  if (kPreloadRes) {
#pragma unroll
    for (int n = 0; n < CT; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) res[n * 4 + g] = *reinterpret_cast<const f32x4*>(a.x + tok * C + 32 * n + 8 * g + 4 * h);
  }
  for (int i = tid; i < 32 * a.n_tiles; i += kRbThreads) bias_lds[i] = a.bias1[i];       // (read after the loop's first barrier)
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" :: "v"(b[s]));

  f32x16 acc2[MODE == kRbMlp ? CT : 1];
  if (MODE == kRbMlp) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc2[ct][i] = 0.f;
  }
  const unsigned ring_base = lds_off_f(smem) + lane * 16;
  const unsigned bias_base = lds_off_f(bias_lds) + 16 * h;     // + 4 * (32 n + 8 g): four consecutive units 8g + 4h .. + 3

  auto do_chunk = [&](const int c) {
    // chunk c has landed once at most the DMAs of the chunks behind it remain in flight (in-order counters; the stores of the
    // previous chunk's epilogue are younger still, so the count only errs on the safe side)
    const int behind = n_chunks - 1 - c;
    if (behind >= kDepth - 1) wait_vm<(kDepth - 1) * IPW>();
    else if (kDepth >= 3 && behind == 1) wait_vm<IPW>();
    else wait_vm<0>();
    asm volatile("s_barrier" ::: "memory");
    if (c + kDepth < n_chunks) issue_chunk(c + kDepth);
    const unsigned chunk_a = ring_base + static_cast<unsigned>((c % kRing) * kChunkBytes);
#pragma unroll
    for (int tl = 0; tl < TPC; ++tl) {
      const int n = c * TPC + tl;
      const unsigned ta = chunk_a + static_cast<unsigned>(tl * kTileFrags * 1024);
      // ---- first product: acc[32 units][32 tokens]
      f32x16 acc;
      zero_acc(acc);
      f32x4 bv[4];
#pragma unroll
      for (int g0 = 0; g0 < KS; g0 += 6) {
        bf16x8 f[6];
        asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:1024\n\tds_read_b128 %2, %6 offset:2048\n\t"
                     "ds_read_b128 %3, %6 offset:3072\n\tds_read_b128 %4, %6 offset:4096\n\tds_read_b128 %5, %6 offset:5120"
                     : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5])
                     : "v"(ta + static_cast<unsigned>(g0 * 1024)) : "memory");
        if (g0 + 6 >= KS) {                                    // the bias of the tile's 16 units per lane, queued behind the last fragments
          const unsigned ba = bias_base + static_cast<unsigned>(n * 128);
          asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:32\n\tds_read_b128 %2, %4 offset:64\n\tds_read_b128 %3, %4 offset:96"
                       : "=&v"(bv[0]), "=&v"(bv[1]), "=&v"(bv[2]), "=&v"(bv[3]) : "v"(ba) : "memory");
        }
        const bool last = g0 + 6 >= KS;
#pragma unroll
        for (int j = 0; j < 6; ++j) {
          if (last) {
            if (j == 0) wait_lgkm<9>(); else if (j == 1) wait_lgkm<8>(); else if (j == 2) wait_lgkm<7>();
            else if (j == 3) wait_lgkm<6>(); else if (j == 4) wait_lgkm<5>(); else wait_lgkm<4>();
          } else {
            if (j == 0) wait_lgkm<5>(); else if (j == 1) wait_lgkm<4>(); else if (j == 2) wait_lgkm<3>();
            else if (j == 3) wait_lgkm<2>(); else if (j == 4) wait_lgkm<1>(); else wait_lgkm<0>();
          }
          __builtin_amdgcn_sched_barrier(0);
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], b[g0 + j], acc, 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      wait_lgkm<0>();
      __builtin_amdgcn_sched_barrier(0);
      if (MODE == kRbLnGemm || MODE == kRbLnGemmGelu) {
        // unit 32n + 8g + 4h + e of the lane's token -> bf16, four consecutive columns per group (the two halves of a wave interleave to
        // whole 16-byte pieces of the row)
        // The natural store is 4 x 8 bytes per lane (lanes r and r + 32 share a row: 16 x 8-byte pieces per row and tile), and with 32 rows per
        // wave-instruction that is 64 partial-line requests each: the L2's request rate, not its bandwidth, bounded these launches (without
        // the stores: 274 -> 162 us for LN -> fc1 -> GELU at C = 384, profiles/r06/clap_rowblock_stores_ab.txt).  One v_permlane32_swap per dword
        // and pair of groups (g, g + 1) hands the upper half's group g to the lower lanes and the lower half's group g + 1 to the upper
        // lanes (as attn_common.h: store_transposed): 2 x 16-byte stores of the same bytes to the same addresses, a quarter of the requests.
        {
          float z[16];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x2 z0 = {acc[4 * g] + bv[g][0], acc[4 * g + 1] + bv[g][1]}, z1 = {acc[4 * g + 2] + bv[g][2], acc[4 * g + 3] + bv[g][3]};
#ifndef ADT_RB_NOGELU
            if (MODE == kRbLnGemmGelu) gelu_bf16_4(z0, z1, z0, z1);
#endif
            z[4 * g] = z0[0]; z[4 * g + 1] = z0[1]; z[4 * g + 2] = z1[0]; z[4 * g + 3] = z1[1];
          }
          unsigned short* op = a.out16 + tok * a.ldo + 32 * n + 8 * h;
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            const unsigned ax = pack2_f(z[4 * g], z[4 * g + 1]), ay = pack2_f(z[4 * g + 2], z[4 * g + 3]);
            const unsigned bx = pack2_f(z[4 * g + 4], z[4 * g + 5]), by = pack2_f(z[4 * g + 6], z[4 * g + 7]);
            const auto rx = __builtin_amdgcn_permlane32_swap(ax, bx, false, false);
            const auto ry = __builtin_amdgcn_permlane32_swap(ay, by, false, false);
            // lower lanes: [own g | upper's g] = units 8g .. 8g+7; upper lanes: [lower's g+1 | own g+1] = units 8g+8 .. 8g+15
#ifdef ADT_RB_NOSTORE      // timing experiment: the outputs are formed and (all but a never-true case) not stored
            if (row_ok && acc[0] == 123456.789f)
#else
            if (row_ok)
#endif
              *reinterpret_cast<uint4*>(op + 8 * g) = make_uint4(rx[0], ry[0], rx[1], ry[1]);
          }
        }
      } else if (MODE == kRbMergeGemm) {
        if (row_ok) {
          float* op = a.out32 + tok * a.ldo + 32 * n + 4 * h;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(op + 8 * g) = f32x4{acc[4 * g] + bv[g][0], acc[4 * g + 1] + bv[g][1], acc[4 * g + 2] + bv[g][2], acc[4 * g + 3] + bv[g][3]};
        }
      } else if (MODE == kRbGemmRes) {
        if (row_ok) {
          float* op = a.x + tok * C + 32 * n + 4 * h;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 rv = kPreloadRes ? res[(kPreloadRes ? n : 0) * 4 + g] : *reinterpret_cast<const f32x4*>(op + 8 * g);
            *reinterpret_cast<f32x4*>(op + 8 * g) = f32x4{acc[4 * g] + bv[g][0] + rv[0], acc[4 * g + 1] + bv[g][1] + rv[1],
                                                          acc[4 * g + 2] + bv[g][2] + rv[2], acc[4 * g + 3] + bv[g][3] + rv[3]};
          }
        }
      } else {
        // ---- MLP: hidden = gelu(acc + bias) stays in registers as the B operands of the second product (k-step s2 = registers 8 s2 ..)
        union { unsigned u[4]; bf16x8 v; } hb[2];
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          const f32x2 z = {acc[2 * m] + bv[m >> 1][2 * (m & 1)], acc[2 * m + 1] + bv[m >> 1][2 * (m & 1) + 1]};
          const f32x2 gv = gelu_bf16_2(z);
          hb[m >> 2].u[m & 3] = pack2_f(gv[0], gv[1]);
        }
        const unsigned wa = ta + static_cast<unsigned>(KS * 1024);       // [s2][ct] fragments of W2 for this hidden tile
#pragma unroll
        for (int g0 = 0; g0 < 2 * CT; g0 += 6) {
          bf16x8 f[6];
          asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:1024\n\tds_read_b128 %2, %6 offset:2048\n\t"
                       "ds_read_b128 %3, %6 offset:3072\n\tds_read_b128 %4, %6 offset:4096\n\tds_read_b128 %5, %6 offset:5120"
                       : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5])
                       : "v"(wa + static_cast<unsigned>(g0 * 1024)) : "memory");
#pragma unroll
          for (int j = 0; j < 6; ++j) {
            if (j == 0) wait_lgkm<5>(); else if (j == 1) wait_lgkm<4>(); else if (j == 2) wait_lgkm<3>();
            else if (j == 3) wait_lgkm<2>(); else if (j == 4) wait_lgkm<1>(); else wait_lgkm<0>();
            __builtin_amdgcn_sched_barrier(0);
            const int fi = g0 + j, s2 = fi / CT, ct = fi % CT;
            acc2[ct] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], hb[s2].v, acc2[ct], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  };
  if constexpr (MODE == kRbGemmRes) {                     // CT / TPC chunks, known at compile time: the residual registers are indexed statically
#pragma unroll
    for (int c = 0; c < CT / TPC; ++c) do_chunk(c);
  } else {
    for (int c = 0; c < n_chunks; ++c) do_chunk(c);
  }
  if (MODE == kRbMlp) {
    // y = acc2 (x went in at the start) + fc2 bias, channel 32 ct + 8g + 4h + e of the lane's token
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (row_ok) {
      float* xp = a.x + tok * C + 4 * h;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 xr = *reinterpret_cast<const f32x4*>(xp + 32 * ct + 8 * g);
          const f32x4 b2 = *reinterpret_cast<const f32x4*>(a.bias2 + 32 * ct + 8 * g + 4 * h);
          *reinterpret_cast<f32x4*>(xp + 32 * ct + 8 * g) = f32x4{acc2[ct][4 * g] + b2[0] + xr[0], acc2[ct][4 * g + 1] + b2[1] + xr[1],
                                                                 acc2[ct][4 * g + 2] + b2[2] + xr[2], acc2[ct][4 * g + 3] + b2[3] + xr[3]};
        }
    }
  }
}

// ---- MLP, software pipelined.  A 32-unit hidden tile costs 2 C/16 MFMAs and ~150 vector instructions (exact-erf GELU of 16 values per
// lane), and run phase by phase (product, GELU, product) the two waves of a SIMD want the matrix pipe together and the vector
// pipe together.  So the three phases of consecutive tiles share a STEP: step k issues the MFMAs of fc1(tile k) and of
// fc2(tile k - 2), one at a time, with a slice of GELU(tile k - 1) behind each (an MFMA runs 32 cycles; the five or six vector
// instructions behind it issue meanwhile), fc1 and fc2 MFMAs alternating so that the fc1 accumulation chain never waits for itself.
// The weight stream is packed in exactly this order, one step after the
// other -- [fc1(k) fragment s, fc2(k-2) fragment (s2, ct)] interleaved, zero fragments where k or k - 2 is out of range -- so the
// LDS-DMA ring protocol is the one above; fragments go through a ring of six registers refilled as each MFMA issues.
// C = 384 (round 6): kOcc = 1 -- ONE workgroup per CU, a wave alone on its SIMD with the whole 512-register file (the token's 96 operand
// registers + 192 fc2 accumulators do not fit 256) and a 3 x 48 KiB weight ring; what it buys is bytes: the hidden activation (403 MB
// written by LN -> fc1 -> GELU and read back by the fc2 GEMM per third-stage layer at 512 clips) never exists.
#ifdef ADT_MLP_STAMPS
__device__ unsigned long long g_mlp_stamps[8];
#endif
#ifdef ADT_MLP_PHASES      // experiment build: where a workgroup's time goes outside the step loop (workgroups 40 and 300: first and second round)
__device__ unsigned long long g_mlp_phases[16];
#define ADT_MLP_PHASE(K) do { if ((blockIdx.x == 40 || blockIdx.x == 300) && wave == 0) { const unsigned long long tn = __builtin_amdgcn_s_memtime(); if (lane == 0) g_mlp_phases[(blockIdx.x == 300 ? 8 : 0) + K] = tn; } } while (0)
#else
#define ADT_MLP_PHASE(K) do { } while (0)
#endif
// The step loop of the fused MLP (fc1 of hidden tile k, GELU of k - 1, fc2 of k - 2 per step; see htsat_mlp_kernel) on a wave's 32 token rows:
// b = the rows' LayerNorm'd operands, acc2 = the fc2 accumulators (in: the residual; out: residual + MLP without the fc2 bias).  Expects chunks
// 0 .. kDepth-1 of the weight stream issued by mlp_issue_chunk and the fc1 bias in bias_lds (ordered by the first chunk's barrier).
struct MlpStream { const unsigned char* wpk; int n_tiles; };
template <int C, int SPC>
__device__ __forceinline__ void mlp_issue_chunk(const MlpStream& a, unsigned char* smem, int c, int wave, int lane) {
  constexpr int kChunkKb = SPC * 2 * (C / 16), kChunkBytes = kChunkKb * 1024, IPW = kChunkKb / kRbWaves;
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const unsigned char* src = a.wpk + static_cast<long>(c) * kChunkBytes + (wave * IPW + i) * 1024 + lane * 16;
    unsigned char* dst = smem + (c % 3) * kChunkBytes + (wave * IPW + i) * 1024;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
  }
}
template <int C, int SPC, int kOcc>
__device__ __forceinline__ void mlp_steps(const MlpStream& a, unsigned char* smem, float* bias_lds, bf16x8 (&b)[C / 16], f32x16 (&acc2)[C / 32],
                                          const int wave, const int lane, const int h) {
  constexpr int KS = C / 16, CT = C / 32, NM = 2 * KS;
  constexpr int kChunkKb = SPC * NM;
  constexpr int kChunkBytes = kChunkKb * 1024;
  constexpr int kRing = 3;
  constexpr int kDepth = 2;
  constexpr int IPW = kChunkKb / kRbWaves;
  const int n_tiles = a.n_tiles;
  const int n_steps = n_tiles + 2;
  const int n_chunks = n_steps / SPC;
  auto issue_chunk = [&](int c) { mlp_issue_chunk<C, SPC>(a, smem, c, wave, lane); };
  f32x16 acc1[2];                                              // [k & 1]: being accumulated by fc1(k); [1 - (k & 1)]: fc1(k - 1), being GELU'd
  union HB { unsigned u[4]; bf16x8 v; };
  HB hb[2][2];                                                 // [(k - 1) & 1][s2]: written by GELU(k - 1); [k & 1][s2]: GELU(k - 2), read by fc2(k - 2)
#pragma unroll
  for (int i = 0; i < 16; ++i) { acc1[0][i] = 0.f; acc1[1][i] = 0.f; }
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int e = 0; e < 4; ++e) hb[p][s2].u[e] = 0u;
  const unsigned ring_base = lds_off_f(smem) + lane * 16;
  const unsigned bias_base = lds_off_f(bias_lds) + 16 * h;

  auto pre_chunk = [&](int c) {                                // chunk c landed everywhere; its predecessor's slot is free again
    if (kOcc == 1 || c + 1 < n_chunks) wait_vm<IPW>();           // (kOcc == 1: a chunk -- real or re-fetched -- is always in flight behind c)
    else wait_vm<0>();
    asm volatile("s_barrier" ::: "memory");
    // kOcc == 1 (a wave alone on its SIMD): a block of IPW vector-memory instructions costs the wave ~50-100 issue cycles each with nobody to
    // cover them -- they are issued one at a time behind the products of the step instead (step(), below; htsat_attn_big_kernel)
    if (kOcc != 1 && c + kDepth < n_chunks) issue_chunk(c + kDepth);
  };
  auto step = [&](const int k, auto ph_tag) {
    constexpr int PH = decltype(ph_tag)::value;
    // kOcc == 1: where this step's DMA instructions read and write (chunk k + kDepth, clamped to the last one)
    const int dma_c = k + kDepth < n_chunks ? k + kDepth : n_chunks - 1;
    const unsigned char* dma_src = a.wpk + static_cast<long>(dma_c) * kChunkBytes + (wave * IPW) * 1024 + lane * 16;
    unsigned char* dma_dst = smem + ((k + kDepth) % kRing) * kChunkBytes + (wave * IPW) * 1024;
    (void)dma_src; (void)dma_dst;
    const unsigned ta = ring_base + static_cast<unsigned>(((k / SPC) % kRing) * kChunkBytes + (k % SPC) * NM * 1024);
    // bias of tile k - 1, whose GELU runs in this step (index clamped: the out-of-range steps at either end are never used)
    const int bt = k < 1 ? 0 : (k - 1 < n_tiles ? k - 1 : n_tiles - 1);
    const unsigned ba = bias_base + static_cast<unsigned>(bt * 128);
    f32x4 bq[4];
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:32\n\tds_read_b128 %2, %4 offset:64\n\tds_read_b128 %3, %4 offset:96"
                 : "=&v"(bq[0]), "=&v"(bq[1]), "=&v"(bq[2]), "=&v"(bq[3]) : "v"(ba) : "memory");
    bf16x8 f[6];
    asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:1024\n\tds_read_b128 %2, %6 offset:2048\n\t"
                 "ds_read_b128 %3, %6 offset:3072\n\tds_read_b128 %4, %6 offset:4096\n\tds_read_b128 %5, %6 offset:5120"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]) : "v"(ta) : "memory");
    zero_acc(acc1[PH]);
    wait_lgkm<6>();                                            // the bias (older than the six fragments) is back: it goes into fc1(k - 1)
    __builtin_amdgcn_sched_barrier(0);                         // right away, so that its 16 registers are free during the loop
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc1[1 - PH][4 * g + e] += bq[g][e];
    __builtin_amdgcn_sched_barrier(0);
    static_for<0, NM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      // fragment i is the oldest of the (at most six) reads in flight
      if (i + 6 <= NM) wait_lgkm<5>();
      else if (i + 5 == NM) wait_lgkm<4>();
      else if (i + 4 == NM) wait_lgkm<3>();
      else if (i + 3 == NM) wait_lgkm<2>();
      else if (i + 2 == NM) wait_lgkm<1>();
      else wait_lgkm<0>();
      __builtin_amdgcn_sched_barrier(0);
      if ((i & 1) == 0) {
        acc1[PH] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i % 6], b[i >> 1], acc1[PH], 0, 0, 0);
      } else {
        const int fi = i >> 1, s2 = fi / CT, ct = fi % CT;
        acc2[ct] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i % 6], hb[PH][s2].v, acc2[ct], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i + 6 < NM)                                          // the register of fragment i takes fragment i + 6
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f[i % 6]) : "v"(ta), "n"((i + 6) * 1024) : "memory");      // (immediate offset: no address add per read)
      if constexpr (kOcc == 1 && SPC == 1) {                   // one instruction of chunk k + kDepth behind every (NM / IPW)-th product
        constexpr int kEvery = NM / IPW;
        if constexpr (i % kEvery == 1 && i / kEvery < IPW) {
          // instruction q of the chunk: 4 KiB groups from one address each, the instruction's immediate offset (added to the global AND the LDS
          // address) steps through the group -- three address computations per step instead of twelve, no branch (past the end the last chunk
          // is fetched again into a slot nobody reads: the counted waits stay exact)
          constexpr int q = i / kEvery;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(dma_src + (q / 4) * 4096),
                                           (__attribute__((address_space(3))) void*)(dma_dst + (q / 4) * 4096), 16, (q % 4) * 1024, 0);
        }
      }
      // a slice of GELU(k - 1): the 8 register pairs go two at a time (two independent polynomial chains: a single chain of dependent
      // packed FMAs costs a wait state per instruction), i.e. four slices spread over the NM MFMAs
#pragma unroll
      for (int q = (i * 4) / NM; q < ((i + 1) * 4) / NM; ++q) {
        f32x2 g0, g1;
        gelu_bf16_4(f32x2{acc1[1 - PH][4 * q], acc1[1 - PH][4 * q + 1]}, f32x2{acc1[1 - PH][4 * q + 2], acc1[1 - PH][4 * q + 3]}, g0, g1);
        hb[1 - PH][q >> 1].u[2 * (q & 1)] = pack2_f(g0[0], g0[1]);
        hb[1 - PH][q >> 1].u[2 * (q & 1) + 1] = pack2_f(g1[0], g1[1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
#ifdef ADT_MLP_STAMPS      // experiment build: cycle stamps of wave 0 of workgroup 300 around steps 10 / 11 (tools/probe/rowblock384.py prints them)
#define ADT_MLP_STAMP(K) do { if (blockIdx.x == 300 && wave == 0 && k == 10) { const unsigned long long tn = __builtin_amdgcn_s_memtime(); if (lane == 0) g_mlp_stamps[K] = tn; } } while (0)
#else
#define ADT_MLP_STAMP(K) do { } while (0)
#endif
  ADT_MLP_PHASE(2);
  for (int k = 0; k < n_steps; k += 2) {                       // n_steps is even (4C / 32 + 2)
    ADT_MLP_STAMP(0);
    if (k % SPC == 0) pre_chunk(k / SPC);
    ADT_MLP_STAMP(1);
    step(k, std::integral_constant<int, 0>{});
    ADT_MLP_STAMP(2);
    if ((k + 1) % SPC == 0) pre_chunk((k + 1) / SPC);
    ADT_MLP_STAMP(3);
    step(k + 1, std::integral_constant<int, 1>{});
    ADT_MLP_STAMP(4);
  }
}

template <int C, int SPC, int kOcc = 2, bool kAffine = true>      // SPC: steps per LDS-DMA chunk; kAffine = false: LayerNorm without gamma / beta (folded by the caller)
__global__ __launch_bounds__(kRbThreads, kOcc) void htsat_mlp_kernel(RbArgs a) {
  constexpr int KS = C / 16, CT = C / 32, NM = 2 * KS;         // MFMAs (= fragments, KiB) per step
  constexpr int kChunkKb = SPC * NM;
  constexpr int kChunkBytes = kChunkKb * 1024;
  constexpr int kRing = 3;
  constexpr int kDepth = 2;
  constexpr int IPW = kChunkKb / kRbWaves;
  static_assert(kChunkKb % kRbWaves == 0 && kRing * kChunkBytes <= (kOcc == 2 ? 76 : 152) * 1024, "chunks split over the waves; two workgroups per CU (one at kOcc = 1)");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];   // [ring][chunk] | fc1 bias [4C] | fc2 bias [C] fp32
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  long tok = static_cast<long>(blockIdx.x) * kRbRows + wave * 32 + r;
  const bool row_ok = tok < a.M;
  if (!row_ok) tok = a.M - 1;
  float* bias_lds = reinterpret_cast<float*>(smem + kRing * kChunkBytes);
  const int n_tiles = a.n_tiles;                               // hidden tiles (4C / 32)
  const int n_steps = n_tiles + 2;
  const int n_chunks = n_steps / SPC;
  ADT_MLP_PHASE(0);

  auto issue_chunk_i = [&](int c, int i) {
    const unsigned char* src = a.wpk + static_cast<long>(c) * kChunkBytes + (wave * IPW + i) * 1024 + lane * 16;
    unsigned char* dst = smem + (c % kRing) * kChunkBytes + (wave * IPW + i) * 1024;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
  };
  auto issue_chunk = [&](int c) {
#pragma unroll
    for (int i = 0; i < IPW; ++i) issue_chunk_i(c, i);
  };
  // the weight stream starts first: its latency hides under the row loads and the LayerNorm
#pragma unroll
  for (int c = 0; c < kDepth; ++c)
    if (c < n_chunks) issue_chunk(c);

  bf16x8 b[KS];
  f32x16 acc2[CT];
  {
    const float* xp = a.x + tok * C + 8 * h;
    float xv[KS][8];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float4 v0 = *reinterpret_cast<const float4*>(xp + 16 * s), v1 = *reinterpret_cast<const float4*>(xp + 16 * s + 4);
      xv[s][0] = v0.x; xv[s][1] = v0.y; xv[s][2] = v0.z; xv[s][3] = v0.w; xv[s][4] = v1.x; xv[s][5] = v1.y; xv[s][6] = v1.z; xv[s][7] = v1.w;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += xv[s][e];
    }
    sum += __shfl_xor(sum, 32);
    ADT_MLP_PHASE(1);
    const float mean = sum * (1.0f / C);
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float d = xv[s][e] - mean; ss = fmaf(d, d, ss); }
    ss += __shfl_xor(ss, 32);
    const float rstd = rsqrtf(ss * (1.0f / C) + a.eps);
    // gamma == nullptr: plain normalisation -- the caller folded gamma into the columns of the following weight and W beta into its bias (the
    // fused tower does: 4 KS loads of gamma / beta cost a lone wave ~10 k cycles of issue per workgroup, profiles/r06/clap_residual_ab.txt)
    auto ln_pack = [&](auto affine_tag, int s) {
      union { unsigned u[4]; bf16x8 v; } pk;
      if constexpr (decltype(affine_tag)::value) {
        const float4 g0 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h), g1 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h + 4);
        const float4 e0 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h), e1 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h + 4);
        const float ga[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w}, be[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pk.u[e] = pack2_f(fmaf((xv[s][2 * e] - mean) * rstd, ga[2 * e], be[2 * e]), fmaf((xv[s][2 * e + 1] - mean) * rstd, ga[2 * e + 1], be[2 * e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) pk.u[e] = pack2_f((xv[s][2 * e] - mean) * rstd, (xv[s][2 * e + 1] - mean) * rstd);
      }
      b[s] = pk.v;
      // The residual rides in the fc2 accumulators from the start (acc2 = x; the fc2 bias joins from LDS at the end) instead of being read again at the end: a third of the
      // kernel's HBM bytes, and the exposed end of a workgroup is stores only.  The lane holds channels 16s + 8h + 0..7 of its token (operand
      // layout); the accumulator of output tile ct holds channels 32ct + 8g + 4h + 0..3: with s = 2ct + j, groups g = 2j and 2j + 1 are the
      // lower / upper lanes' halves of the same 16 channels, exchanged by one v_permlane32_swap per register pair.
      const int ct = s >> 1, j = s & 1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(xv[s][e]), __float_as_uint(xv[s][4 + e]), false, false);
        acc2[ct][8 * j + e] = __uint_as_float(sw[0]);
        acc2[ct][8 * j + 4 + e] = __uint_as_float(sw[1]);
      }
    };
#pragma unroll
    for (int s = 0; s < KS; ++s) ln_pack(std::integral_constant<bool, kAffine>{}, s);
  }
  // fc1 bias | fc2 bias -> LDS.  (Compiler-generated LDS stores: they wait for the DMAs above, which chunk 0 needs anyway.)
  for (int i = tid; i < 32 * n_tiles; i += kRbThreads) bias_lds[i] = a.bias1[i];
  for (int i = tid; i < C; i += kRbThreads) bias_lds[32 * n_tiles + i] = a.bias2[i];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" :: "v"(b[s]));

  mlp_steps<C, SPC, kOcc>(MlpStream{a.wpk, a.n_tiles}, smem, bias_lds, b, acc2, wave, lane, h);
  // y = acc2 (x went in at the start) + fc2 bias, channel 32 ct + 8g + 4h + e of the lane's token
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  ADT_MLP_PHASE(3);
  if (row_ok) {
    float* xp = a.x + tok * C + 4 * h;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 b2 = *reinterpret_cast<const f32x4*>(bias_lds + 32 * n_tiles + 32 * ct + 8 * g + 4 * h);
        *reinterpret_cast<f32x4*>(xp + 32 * ct + 8 * g) = f32x4{acc2[ct][4 * g] + b2[0], acc2[ct][4 * g + 1] + b2[1], acc2[ct][4 * g + 2] + b2[2], acc2[ct][4 * g + 3] + b2[3]};
      }
  }
  ADT_MLP_PHASE(4);
#ifdef ADT_MLP_PHASES
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  ADT_MLP_PHASE(5);
#endif
}

template <int C, int SPC, int kOcc, bool kAffine>
static int launch_mlp_(const RbArgs& a, hipStream_t st) {
  constexpr int kChunkBytes = SPC * 2 * (C / 16) * 1024;
  const int lds = 3 * kChunkBytes + 32 * a.n_tiles * 4 + C * 4;
  if ((a.n_tiles + 2) % SPC || (a.n_tiles & 1)) return set_error(ADT_ESHAPE, "htsat MLP kernel: step count must be even and a multiple of the chunk size");
  static thread_local int done_for = -1;
  int dev = 0;
  ADT_HIP_TRY(hipGetDevice(&dev));
  if (done_for != dev) {
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_mlp_kernel<C, SPC, kOcc, kAffine>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    done_for = dev;
  }
  const unsigned grid = static_cast<unsigned>((a.M + kRbRows - 1) / kRbRows);
  hipLaunchKernelGGL((htsat_mlp_kernel<C, SPC, kOcc, kAffine>), dim3(grid), dim3(kRbThreads), lds, st, a);
#ifdef ADT_MLP_STAMPS
  if (getenv("ADT_MLP_PRINT") && C == 384) {
    unsigned long long h[8];
    ADT_HIP_TRY(hipStreamSynchronize(st));
    ADT_HIP_TRY(hipMemcpyFromSymbol(h, HIP_SYMBOL(g_mlp_stamps), sizeof(h)));
    fprintf(stderr, "mlp384 stamps (cycles): pre_chunk %lld, step %lld, pre_chunk %lld, step %lld\n", static_cast<long long>(h[1] - h[0]),
            static_cast<long long>(h[2] - h[1]), static_cast<long long>(h[3] - h[2]), static_cast<long long>(h[4] - h[3]));
  }
#endif
#ifdef ADT_MLP_PHASES
  if (getenv("ADT_MLP_PRINT") && C == 384) {
    unsigned long long h[16];
    ADT_HIP_TRY(hipStreamSynchronize(st));
    ADT_HIP_TRY(hipMemcpyFromSymbol(h, HIP_SYMBOL(g_mlp_phases), sizeof(h)));
    for (int w = 0; w < 2; ++w)
      fprintf(stderr, "mlp384 phases, workgroup %d (ticks of s_memtime, 100 MHz): rows loaded +%lld, LN + bias + first chunks +%lld, step loop +%lld, epilogue issued +%lld, "
              "stores done +%lld; start relative to workgroup 40: %lld\n", w ? 300 : 40, static_cast<long long>(h[8 * w + 1] - h[8 * w]), static_cast<long long>(h[8 * w + 2] - h[8 * w + 1]),
              static_cast<long long>(h[8 * w + 3] - h[8 * w + 2]), static_cast<long long>(h[8 * w + 4] - h[8 * w + 3]), static_cast<long long>(h[8 * w + 5] - h[8 * w + 4]),
              static_cast<long long>(h[8 * w] - h[0]));
  }
#endif
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

template <int C, int SPC, int kOcc = 2>
static int launch_mlp(const RbArgs& a, hipStream_t st) {
  return a.gamma ? launch_mlp_<C, SPC, kOcc, true>(a, st) : launch_mlp_<C, SPC, kOcc, false>(a, st);
}

// ---- the whole attention half of a layer in one launch (C = 96: four heads of 24): x -> LayerNorm -> q | k | v -> window attention with
// the relative-position bias (and the shifted-window mask) -> output projection -> + x, in place.  Unfused, this half moves the
// residual stream twice and the bf16 q | k | v and context tensors in between (5.6 GB per stage-0 layer at 512 clips); here
// only x is read and written (1.6 GB).  The token stays on the lane from the first load to the last store:
//   * workgroup = 4 waves = 2 windows x 2 token tiles; wave (window wi, tile tt) owns tokens 32 tt .. 32 tt + 31 of its window;
//   * per head: q, k, v = three 32-unit tiles (24 real units + 8 of zero weights) of the row-block product; q and k are packed
//     straight from the accumulators into MFMA operands (B operand of S^T = K Q^T, and -- the same register layout -- A operand),
//     k and v cross to the window's other wave through LDS (2 KiB of operands, a 4 KiB [key][d] tile read back transposed);
//     softmax in registers (query on the lane), P^T from the accumulator as the next B operand, and the head's context tile goes --
//     again from the accumulator -- into the output projection, whose accumulators run over the heads;
//   * weights: one 24 KiB chunk per head [Wq | Wk | Wv fragments, then Wo's for this head's 24 (+8 zero) inputs in accumulator order],
//     a ring of two chunks filled by LDS-DMA one head ahead.
struct AtArgs {
  float* x; const float *gamma, *beta; float eps;
  const unsigned char* wpk;      // [heads] chunks of (3 C/16 + 2 C/32) KiB
  const float* qkv_bias;         // [heads][3][32]  (units 24..31 zero)
  const float* out_bias;         // [C]
  const float* rel_bias; int n_bias_windows;       // lane-linear, as adt_window_attn_fwd
  int B, R, shift; float scale;
  // htsat_attn_big_kernel<C, false, true> (the whole layer in one launch): the MLP half's stream, as adt_htsat_rowblock mode 2 with a folded LayerNorm
  const unsigned char* mlp_wpk; const float* mlp_b1; const float* mlp_b2; int mlp_tiles;
  // htsat_attn_big_kernel<192, false, true>: rel_bias as bf16, [.., query tile 2, key tile 2, group pair 2, lane 64, group 2, e 4] (clap_encoder.py:window_bias_layout_bf16)
  const unsigned short* rel_bias16;
};
__device__ __forceinline__ long at_token_row(const AtArgs& a, int b, int wy, int wx, int t) {
  const int y = (wy * 8 + (t >> 3) + a.shift) % a.R, x = (wx * 8 + (t & 7) + a.shift) % a.R;
  return (static_cast<long>(b) * a.R + y) * a.R + x;
}

// ---- the MLP half of a layer on the rows an attention kernel still holds (round 6: the one-launch layer): x' = acc_out + bias stays in the
// accumulators -- it is the MLP's residual AND, back in operand layout, the input of its LayerNorm -- so one store and one load of the rows, a
// launch and the lock-step row phases of a second kernel go.  (Both LayerNorms folded into the weights by the caller.)
template <int C, int kOcc>
__device__ __forceinline__ void layer_mlp_tail(const AtArgs& a, unsigned char* smem, bf16x8 (&b)[C / 16], f32x16 (&acc_out)[C / 32], const int wave, const int lane,
                                               const int h, const int tid, const bool win_ok, const long row) {
  constexpr int KS = C / 16, CT = C / 32;
  constexpr int kMlpChunk = 2 * KS * 1024;
  float* bias_lds = reinterpret_cast<float*>(smem + 3 * kMlpChunk);
  const MlpStream ms{a.mlp_wpk, a.mlp_tiles};
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // the attention half's DMAs (the re-fetched tail included) have landed ...
  asm volatile("s_barrier" ::: "memory");                          // ... and nobody reads its LDS any more: the MLP's ring takes it over
  mlp_issue_chunk<C, 1>(ms, smem, 0, wave, lane);
  mlp_issue_chunk<C, 1>(ms, smem, 1, wave, lane);
  float sum = 0.f;
  {
    const float* __restrict__ ob = a.out_bias + 4 * h;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 b2 = *reinterpret_cast<const f32x4*>(ob + 32 * ct + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) { acc_out[ct][4 * g + e] += b2[e]; sum += acc_out[ct][4 * g + e]; }
      }
  }
  sum += __shfl_xor(sum, 32);
  const float mean = sum * (1.0f / C);
  float ss = 0.f;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int i = 0; i < 16; ++i) { const float d = acc_out[ct][i] - mean; ss = fmaf(d, d, ss); }
  ss += __shfl_xor(ss, 32);
  const float rstd = rsqrtf(ss * (1.0f / C) + a.eps);
#pragma unroll
  for (int s = 0; s < KS; ++s) {                                   // accumulator layout -> operand layout: the swap is its own inverse
    float xv[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc_out[s >> 1][8 * (s & 1) + e]), __float_as_uint(acc_out[s >> 1][8 * (s & 1) + 4 + e]), false, false);
      xv[e] = __uint_as_float(sw[0]);
      xv[4 + e] = __uint_as_float(sw[1]);
    }
    union { unsigned u[4]; bf16x8 v; } pk;
#pragma unroll
    for (int e = 0; e < 4; ++e) pk.u[e] = pack2_f((xv[2 * e] - mean) * rstd, (xv[2 * e + 1] - mean) * rstd);
    b[s] = pk.v;
  }
  for (int i = tid; i < 32 * a.mlp_tiles; i += 256) bias_lds[i] = a.mlp_b1[i];
  for (int i = tid; i < C; i += 256) bias_lds[32 * a.mlp_tiles + i] = a.mlp_b2[i];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" :: "v"(b[s]));
  mlp_steps<C, 1, kOcc>(ms, smem, bias_lds, b, acc_out, wave, lane, h);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (win_ok) {
    float* xp = a.x + row * C + 4 * h;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 b2 = *reinterpret_cast<const f32x4*>(bias_lds + 32 * a.mlp_tiles + 32 * ct + 8 * g + 4 * h);
        *reinterpret_cast<f32x4*>(xp + 32 * ct + 8 * g) = f32x4{acc_out[ct][4 * g] + b2[0], acc_out[ct][4 * g + 1] + b2[1], acc_out[ct][4 * g + 2] + b2[2], acc_out[ct][4 * g + 3] + b2[3]};
      }
  }
}

// (compiler-visible conversion, NOT the inline-asm pack2_f: these read MFMA results, and an asm statement gets none of the wait
// states the hazard recognizer puts between an MFMA and a vector instruction that reads its destination -- packed by asm right
// behind the P V chain, the context tile went into the projection without its last product)
__device__ __forceinline__ unsigned pack2_c(float lo, float hi) {
  typedef __bf16 bf16x2_ __attribute__((ext_vector_type(2)));
  typedef float f32x2_ __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2_{lo, hi}, bf16x2_));
}
// p = 2^(s - mx) over a wave's 2 x 16 scores, and their sum: the subtraction and the sums in pairs, four independent partial sums instead of one chain of 32 dependent adds
__device__ __forceinline__ float softmax_exp_sum(f32x16 (&st)[2], float mx) {
  const f32x2 m2 = {mx, mx};
  f32x2 ps[2][2] = {{{0.f, 0.f}, {0.f, 0.f}}, {{0.f, 0.f}, {0.f, 0.f}}};
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f32x2 d = f32x2{st[kt][2 * i], st[kt][2 * i + 1]} - m2;
      const f32x2 pp = {__builtin_amdgcn_exp2f(d[0]), __builtin_amdgcn_exp2f(d[1])};
      st[kt][2 * i] = pp[0]; st[kt][2 * i + 1] = pp[1];
      ps[kt][i & 1] += pp;
    }
  const f32x2 t = (ps[0][0] + ps[0][1]) + (ps[1][0] + ps[1][1]);
  return t[0] + t[1];
}
__device__ __forceinline__ bf16x8 acc_to_b_f(const f32x16& x, int s) {
  union { unsigned u[4]; bf16x8 v; } r;
  r.u[0] = pack2_c(x[8 * s + 0], x[8 * s + 1]); r.u[1] = pack2_c(x[8 * s + 2], x[8 * s + 3]);
  r.u[2] = pack2_c(x[8 * s + 4], x[8 * s + 5]); r.u[3] = pack2_c(x[8 * s + 6], x[8 * s + 7]);
  return r.v;
}

template <int C, bool kAffine = true, bool kMlp = false>      // kAffine = false: LayerNorm without gamma / beta (folded into Wq|k|v and their bias by the caller); kMlp: the MLP half follows (layer_mlp_tail)
__global__ __launch_bounds__(256, 2) void htsat_attn_kernel(AtArgs a) {
  constexpr int KS = C / 16, CT = C / 32, NH = C / 24;
  constexpr int kChunkKb = 3 * KS + 2 * CT, kChunkBytes = kChunkKb * 1024;
  constexpr int IPW = kChunkKb / 4;
  static_assert(kChunkKb % 4 == 0 && KS == 6, "built for C = 96");
  constexpr int kKx = 2 * kChunkBytes, kVt = kKx + 2 * 2 * 2 * 1024, kQb = kVt + 2 * 4096;     // ring | K operands | V tiles | q|k|v bias
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave >> 1, tt = wave & 1;
  const int nw = a.R / 8;
  long widx = static_cast<long>(blockIdx.x) * 2 + wi;                                  // (b, wy, wx)
  const long n_windows = static_cast<long>(a.B) * nw * nw;
  const bool win_ok = widx < n_windows;
  if (!win_ok) widx = n_windows - 1;
  const int wx = static_cast<int>(widx % nw), wy = static_cast<int>((widx / nw) % nw), bi = static_cast<int>(widx / (nw * nw));
  const long row = at_token_row(a, bi, wy, wx, 32 * tt + r);
  const unsigned smem_base = lds_off_f(smem);

  auto issue_chunk = [&](int c) {
    const unsigned char* src = a.wpk + static_cast<long>(c) * kChunkBytes + (wave * IPW) * 1024 + lane * 16;
    unsigned char* dst = smem + (c & 1) * kChunkBytes + (wave * IPW) * 1024;
#pragma unroll
    for (int i = 0; i < IPW; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + i * 1024),
                                       (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, 0, 0);
  };
  issue_chunk(0);

  // ---- the token row -> LayerNorm -> bf16 B operands
  bf16x8 b[KS];
  f32x16 acc_out[CT];                                          // starts as the residual x (see htsat_mlp_kernel): no second read of the rows at the end
  {
    const float* xp = a.x + row * C + 8 * h;
    float xv[KS][8];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float4 v0 = *reinterpret_cast<const float4*>(xp + 16 * s), v1 = *reinterpret_cast<const float4*>(xp + 16 * s + 4);
      xv[s][0] = v0.x; xv[s][1] = v0.y; xv[s][2] = v0.z; xv[s][3] = v0.w; xv[s][4] = v1.x; xv[s][5] = v1.y; xv[s][6] = v1.z; xv[s][7] = v1.w;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += xv[s][e];
    }
    sum += __shfl_xor(sum, 32);
    const float mean = sum * (1.0f / C);
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float d = xv[s][e] - mean; ss = fmaf(d, d, ss); }
    ss += __shfl_xor(ss, 32);
    const float rstd = rsqrtf(ss * (1.0f / C) + a.eps);
    // gamma == nullptr: plain normalisation -- the caller folded gamma into the columns of the following weight and W beta into its bias (the
    // fused tower does: 4 KS loads of gamma / beta cost a lone wave ~10 k cycles of issue per workgroup, profiles/r06/clap_residual_ab.txt)
    auto ln_pack = [&](auto affine_tag, int s) {
      union { unsigned u[4]; bf16x8 v; } pk;
      if constexpr (decltype(affine_tag)::value) {
        const float4 g0 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h), g1 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h + 4);
        const float4 e0 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h), e1 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h + 4);
        const float ga[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w}, be[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pk.u[e] = pack2_f(fmaf((xv[s][2 * e] - mean) * rstd, ga[2 * e], be[2 * e]), fmaf((xv[s][2 * e + 1] - mean) * rstd, ga[2 * e + 1], be[2 * e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) pk.u[e] = pack2_f((xv[s][2 * e] - mean) * rstd, (xv[s][2 * e + 1] - mean) * rstd);
      }
      b[s] = pk.v;
      // operand layout (channels 16s + 8h + 0..7) -> accumulator layout (32ct + 8g + 4h + 0..3): s = 2ct + j, groups 2j / 2j + 1, one swap per pair
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(xv[s][e]), __float_as_uint(xv[s][4 + e]), false, false);
        acc_out[s >> 1][8 * (s & 1) + e] = __uint_as_float(sw[0]);
        acc_out[s >> 1][8 * (s & 1) + 4 + e] = __uint_as_float(sw[1]);
      }
    };
#pragma unroll
    for (int s = 0; s < KS; ++s) ln_pack(std::integral_constant<bool, kAffine>{}, s);
  }
  float* qb_lds = reinterpret_cast<float*>(smem + kQb);
  for (int i = tid; i < NH * 96; i += 256) qb_lds[i] = a.qkv_bias[i];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" :: "v"(b[s]));

  const unsigned kx_w = smem_base + kKx + static_cast<unsigned>(((wi * 2 + tt) * 2) * 1024 + lane * 16);       // this wave's K operands (k-step s: + s KiB)
  const unsigned kx_r = smem_base + kKx + static_cast<unsigned>((wi * 2 * 2) * 1024 + lane * 16);              // the window's: + (kt * 2 + s) KiB
  const unsigned vt_b = smem_base + kVt + static_cast<unsigned>(wi * 4096);
  const unsigned vt_w = vt_b + static_cast<unsigned>((32 * tt + r) * 64 + 8 * h);                               // d = 8g + 4h .. + 3: + 16 g bytes
  const unsigned qb_a = smem_base + kQb + static_cast<unsigned>(16 * h);                                         // + (head * 96 + which * 32 + 8g) * 4
  const int wsel = a.n_bias_windows > 1 ? (wy * nw + wx) : 0;
  const float sl2 = a.scale * 1.4426950408889634f;

  // one 32-unit tile of the row-block product + its bias: acc[unit 8g + 4h + e][token]
  auto tile = [&](unsigned ta, unsigned bias_a, f32x16& acc) {
    bf16x8 f[6];
    f32x4 bv[4];
    asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:1024\n\tds_read_b128 %2, %6 offset:2048\n\t"
                 "ds_read_b128 %3, %6 offset:3072\n\tds_read_b128 %4, %6 offset:4096\n\tds_read_b128 %5, %6 offset:5120"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]) : "v"(ta) : "memory");
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:32\n\tds_read_b128 %2, %4 offset:64\n\tds_read_b128 %3, %4 offset:96"
                 : "=&v"(bv[0]), "=&v"(bv[1]), "=&v"(bv[2]), "=&v"(bv[3]) : "v"(bias_a) : "memory");
    zero_acc(acc);
#pragma unroll
    for (int j = 0; j < 6; ++j) {
      if (j == 0) wait_lgkm<9>(); else if (j == 1) wait_lgkm<8>(); else if (j == 2) wait_lgkm<7>();
      else if (j == 3) wait_lgkm<6>(); else if (j == 4) wait_lgkm<5>(); else wait_lgkm<4>();
      __builtin_amdgcn_sched_barrier(0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], b[j], acc, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_lgkm<0>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * g + e] += bv[g][e];
  };

  for (int hd = 0; hd < NH; ++hd) {
    // chunk hd landed (this wave's share; the barrier makes it everyone's); every wave is past head hd - 1, so the other ring slot and
    // the K / V buffers are free
    wait_vm<0>();
    asm volatile("s_barrier" ::: "memory");
    // relative-position bias (+ shift mask) of (query tile tt, key tile kt, group g): lane-linear table, plain loads, requested BEFORE the
    // next chunk's DMA so that waiting for them does not wait for it (in-order counters)
    const float* rb = a.rel_bias + (static_cast<long>(wsel) * NH + hd) * 4096 + tt * 2048 + lane * 4;
    float4 rbv[2][4];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int g = 0; g < 4; ++g) rbv[kt][g] = *reinterpret_cast<const float4*>(rb + (kt * 4 + g) * 256);
    if (hd + 1 < NH) issue_chunk(hd + 1);
    const unsigned ta = smem_base + static_cast<unsigned>((hd & 1) * kChunkBytes + lane * 16);
    const unsigned ba = qb_a + static_cast<unsigned>(hd * 96 * 4);
    f32x16 acc;
    bf16x8 qop[2];
    tile(ta, ba, acc);                                        // q
    qop[0] = acc_to_b_f(acc, 0); qop[1] = acc_to_b_f(acc, 1);
    tile(ta + KS * 1024, ba + 128, acc);                      // k -> the window's K operands
    {
      const bf16x8 k0 = acc_to_b_f(acc, 0), k1 = acc_to_b_f(acc, 1);
      asm volatile("ds_write_b128 %0, %1\n\tds_write_b128 %0, %2 offset:1024" :: "v"(kx_w), "v"(k0), "v"(k1) : "memory");
    }
    tile(ta + 2 * KS * 1024, ba + 256, acc);                  // v -> the window's [key][d] tile
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const unsigned lo = pack2_f(acc[4 * g], acc[4 * g + 1]), hi = pack2_f(acc[4 * g + 2], acc[4 * g + 3]);
      typedef unsigned u32x2_ __attribute__((ext_vector_type(2)));
      const u32x2_ pr = {lo, hi};
      asm volatile("ds_write_b64 %0, %1" :: "v"(vt_w + static_cast<unsigned>(16 * g)), "v"(pr) : "memory");
    }
    wait_lgkm<0>();
    asm volatile("s_barrier" ::: "memory");
    // ---- S^T[key][query] for this wave's 32 queries and the window's 64 keys
    bf16x8 kf[4];
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %4 offset:3072"
                 : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3]) : "v"(kx_r) : "memory");
    f32x16 st[2];
    wait_lgkm<0>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      zero_acc(st[kt]);
      st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[2 * kt], qop[0], st[kt], 0, 0, 0);
      st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[2 * kt + 1], qop[1], st[kt], 0, 0, 0);
    }
    float mx = -3.0e38f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float bb[4] = {rbv[kt][g].x, rbv[kt][g].y, rbv[kt][g].z, rbv[kt][g].w};
#pragma unroll
        for (int e = 0; e < 4; e += 2) {                             // log2 domain: the bias table comes pre-multiplied by log2 e
          const f32x2 v = f32x2{st[kt][4 * g + e], st[kt][4 * g + e + 1]} * sl2 + f32x2{bb[e], bb[e + 1]};
          st[kt][4 * g + e] = v[0]; st[kt][4 * g + e + 1] = v[1];
          mx = fmaxf(mx, fmaxf(v[0], v[1]));
        }
      }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    float sum = softmax_exp_sum(st, mx);
    sum += __shfl_xor(sum, 32);
    const float inv = 1.0f / sum;
    // ---- O^T[d][query] = sum over keys of V^T P^T
    f32x16 o;
    zero_acc(o);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const int i16 = lane & 15, g4 = (lane >> 4) & 1;
        const unsigned base = vt_b + static_cast<unsigned>((kt * 32 + 16 * s2 + 4 * h + (i16 >> 2)) * 64 + (16 * g4 + 4 * (i16 & 3)) * 2);
        typedef __attribute__((ext_vector_type(4))) short bf16x4_;
        bf16x4_ lo, hi;
        bf16x8 af;
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:512\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(lo), "=&v"(hi) : "v"(base) : "memory");
        af[0] = lo[0]; af[1] = lo[1]; af[2] = lo[2]; af[3] = lo[3]; af[4] = hi[0]; af[5] = hi[1]; af[6] = hi[2]; af[7] = hi[3];
        union { unsigned u[4]; bf16x8 v; } pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf.u[e] = pack2_f(st[kt][8 * s2 + 2 * e], st[kt][8 * s2 + 2 * e + 1]);       // un-normalised: O is scaled by 1 / sum below
        o = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, pf.v, o, 0, 0, 0);
      }
    // ---- output projection: this head's 24 (+ 8 zero) context values are k-steps 0, 1 of Wo's slice
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] *= inv;              // the softmax denominator, once per output instead of once per probability
    const bf16x8 ob0 = acc_to_b_f(o, 0), ob1 = acc_to_b_f(o, 1);
    {
      bf16x8 f[6];
      asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:1024\n\tds_read_b128 %2, %6 offset:2048\n\t"
                   "ds_read_b128 %3, %6 offset:3072\n\tds_read_b128 %4, %6 offset:4096\n\tds_read_b128 %5, %6 offset:5120"
                   : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]) : "v"(ta + 3 * KS * 1024) : "memory");
      wait_lgkm<0>();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 6; ++j) acc_out[j % CT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], j < CT ? ob0 : ob1, acc_out[j % CT], 0, 0, 0);
    }
  }
  if constexpr (kMlp) {
    static_assert(!kAffine, "the one-launch layer is built with both LayerNorms folded into the weights");
    layer_mlp_tail<C, 2>(a, smem, b, acc_out, wave, lane, h, tid, win_ok, row);
    return;
  }
  // ---- x = acc_out (x went in at the start) + bias: stores only
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (win_ok) {
    float* __restrict__ xp = a.x + row * C + 4 * h;
    const float* __restrict__ ob = a.out_bias + 4 * h;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      f32x4 b2[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) b2[g] = *reinterpret_cast<const f32x4*>(ob + 32 * ct + 8 * g);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(xp + 32 * ct + 8 * g) = f32x4{acc_out[ct][4 * g] + b2[g][0], acc_out[ct][4 * g + 1] + b2[g][1],
                                                               acc_out[ct][4 * g + 2] + b2[g][2], acc_out[ct][4 * g + 3] + b2[g][3]};
    }
  }
}

// ---- the same attention half for C = 192 / 384 (stages 1 and 2; round 6): ONE workgroup per CU, a wave alone on its SIMD with the 512-register
// file (the token's C/16 operand registers + C/2 output-projection accumulators do not fit 256).  Unfused, a third-stage layer's attention
// half moves x twice and the bf16 q | k | v / context tensors in between (1.4 GB per layer at 512 clips, at the ~3.2 TB/s every launch of
// this tower is bound by); here x is read and written once (0.4 GB).  The head's weights no longer fit LDS twice (96 KiB per head at
// C = 384), so the stream is cut into SUB-chunks of C/16 KiB -- per head [Wq_h | Wk_h | Wv_h | Wo_h], each exactly C/16 fragments, the order
// pack_attn_block_weights already writes -- through a FOUR-slot ring, two sub-chunks ahead: sub-chunk n is waited for with a counted vmcnt
// that leaves n + 1 (and, where they are younger, the next head's relative-position bias pieces, which travel by LDS-DMA into per-wave
// staging slots) outstanding, one barrier per sub-chunk, and the DMA instructions of sub-chunk n + 2 are issued one at a time BEHIND
// products of the tile that reads sub-chunk n.  Sub-chunks past the end re-fetch the last one into slots nobody reads again, so that the
// counts stay exact.  Measured (profiles/r06/clap_attn_big.txt): same bits as the three launches' bf16 roundings to 5e-4 of the update;
// alone 395 vs 405-440 us (C = 384) and 602-627 vs 664-677 us (C = 192) per layer; inside the tower 37.8 k vs 36.8 k embeds/s.
#ifdef ADT_ATB_STAMPS      // experiment build: cycle stamps of wave 0 of workgroup 300 for head 2 (tools/probe/attn_big.py prints them)
__device__ unsigned long long g_atb_stamps[16];
#define ADT_ATB_STAMP(K) do { if (blockIdx.x == 300 && wave == 0 && hd == 2) { const unsigned long long tn = __builtin_amdgcn_s_memtime(); if (lane == 0) g_atb_stamps[K] = tn; } } while (0)
#else
#define ADT_ATB_STAMP(K) do { } while (0)
#endif
// C = 192 is built for 256 registers (two workgroups per CU): its fragments go through a ring of SIX registers refilled as each product issues
// (kRing6, as mlp_steps), not through two sets of six -- under that budget the allocator spilled a prefetched set right behind the asm statement
// that had requested it, before the data had landed (DESIGN 8.6.9 e; tools/probe/check_pending_lds_regs.py guards it).
template <int C, bool kAffine = true, bool kMlp = false>      // kMlp: the layer's MLP half follows in the same launch, on the rows still in the accumulators
__global__ __launch_bounds__(256, C == 192 ? 2 : 1) void htsat_attn_big_kernel(AtArgs a) {
  constexpr int KS = C / 16, CT = C / 32, NH = C / 24;
  constexpr bool kRing6 = C == 192;
  constexpr int kSubBytes = KS * 1024;
  constexpr int IPW = KS / 4;                                  // DMA instructions per wave and sub-chunk
  constexpr int kSubs = 4 * NH;
  static_assert(KS % 12 == 0 && IPW * 4 == KS, "C = 192 or 384");
  // The C = 192 layer (two workgroups per CU: 80 KiB each) runs a THREE-slot ring -- sub-chunk n + 2 goes into the slot of n - 1, which everybody has
  // read before the barrier of n -- and stages the relative-position bias as bf16 (4 KiB per wave and head, 4 DMA instructions instead of 8): 71 KiB
  // for the attention half, 76 for the MLP half.  (bf16 on a bias of a few units: 0.4 % of a logit's bias, the rounding the probabilities get anyway.)
  constexpr bool kRb16 = C == 192 && kMlp;
  constexpr int kSlots = kRb16 ? 3 : 4;
  constexpr int kRbN = kRb16 ? 4 : 8, kRbWave = kRbN * 1024;                                   // bias DMA instructions / staging bytes per wave and head
  constexpr int kKx = kSlots * kSubBytes, kVt = kKx + 2 * 2 * 2 * 1024, kQb = kVt + 2 * 4096;     // ring | K operands | V tiles | q|k|v bias | bias staging
  constexpr int kRb = kQb + NH * 96 * 4;                                                     // per wave: the head's relative-position bias pieces
  static_assert(kRb + 4 * kRbWave <= (kRb16 ? 80 : 160) * 1024, "LDS budget");
  auto slot = [](int n) { return kSlots == 4 ? (n & 3) : n % 3; };
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave >> 1, tt = wave & 1;
  const int nw = a.R / 8;
  long widx = static_cast<long>(blockIdx.x) * 2 + wi;                                  // (b, wy, wx)
  const long n_windows = static_cast<long>(a.B) * nw * nw;
  const bool win_ok = widx < n_windows;
  if (!win_ok) widx = n_windows - 1;
  const int wx = static_cast<int>(widx % nw), wy = static_cast<int>((widx / nw) % nw), bi = static_cast<int>(widx / (nw * nw));
  const long row = at_token_row(a, bi, wy, wx, 32 * tt + r);
  const unsigned smem_base = lds_off_f(smem);

  // one LDS-DMA instruction (1 KiB) of sub-chunk n: a wave's vector-memory instruction costs it ~50-100 issue cycles, and a wave alone on its
  // SIMD has nobody to cover them -- so inside the head loop they are issued one at a time BETWEEN the products of a tile (the matrix pipe
  // works meanwhile), not as a block in front of it (cycle stamps: a tile's segment 1 300 cycles without a single product, profiles/r06/clap_attn_big.txt)
  auto issue_sub_i = [&](int n, int i) {
    const int nn = n < kSubs ? n : kSubs - 1;
    const unsigned char* src = a.wpk + static_cast<long>(nn) * kSubBytes + (wave * IPW + i) * 1024 + lane * 16;
    unsigned char* dst = smem + slot(n) * kSubBytes + (wave * IPW + i) * 1024;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
  };
  auto issue_sub = [&](int n) {
#pragma unroll
    for (int i = 0; i < IPW; ++i) issue_sub_i(n, i);
  };
  // piece i (of 8) of head hd's relative-position bias (+ shift mask) for (query tile tt; key tile, group): lane-linear table -> the wave's own
  // staging slots (read back by the wave that fetched them: no barrier)
  const int wsel_ = a.n_bias_windows > 1 ? (wy * nw + wx) : 0;
  auto issue_rb_i = [&](int hd, int i) {
    const int hh = hd < NH ? hd : NH - 1;
    if constexpr (kRb16) {       // piece i = (key tile i >> 1, group pair i & 1): 16 bytes = 8 bf16 per lane
      const unsigned short* rb = a.rel_bias16 + (static_cast<long>(wsel_) * NH + hh) * 4096 + tt * 2048 + lane * 8;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(rb + i * 512),
                                       (__attribute__((address_space(3))) void*)(smem + kRb + wave * kRbWave + i * 1024), 16, 0, 0);
    } else {
      const float* rb = a.rel_bias + (static_cast<long>(wsel_) * NH + hh) * 4096 + tt * 2048 + lane * 4;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(rb + i * 256),
                                       (__attribute__((address_space(3))) void*)(smem + kRb + wave * kRbWave + i * 1024), 16, 0, 0);
    }
  };
  // ---- the token row -> LayerNorm -> bf16 B operands (before any DMA is in flight: these are plain loads)
  bf16x8 b[KS];
  f32x16 acc_out[CT];                                          // starts as the residual x (see htsat_mlp_kernel): no second read of the rows at the end
  {
    const float* xp = a.x + row * C + 8 * h;
    float xv[KS][8];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float4 v0 = *reinterpret_cast<const float4*>(xp + 16 * s), v1 = *reinterpret_cast<const float4*>(xp + 16 * s + 4);
      xv[s][0] = v0.x; xv[s][1] = v0.y; xv[s][2] = v0.z; xv[s][3] = v0.w; xv[s][4] = v1.x; xv[s][5] = v1.y; xv[s][6] = v1.z; xv[s][7] = v1.w;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += xv[s][e];
    }
    sum += __shfl_xor(sum, 32);
    const float mean = sum * (1.0f / C);
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float d = xv[s][e] - mean; ss = fmaf(d, d, ss); }
    ss += __shfl_xor(ss, 32);
    const float rstd = rsqrtf(ss * (1.0f / C) + a.eps);
    // gamma == nullptr: plain normalisation -- the caller folded gamma into the columns of the following weight and W beta into its bias (the
    // fused tower does: 4 KS loads of gamma / beta cost a lone wave ~10 k cycles of issue per workgroup, profiles/r06/clap_residual_ab.txt)
    auto ln_pack = [&](auto affine_tag, int s) {
      union { unsigned u[4]; bf16x8 v; } pk;
      if constexpr (decltype(affine_tag)::value) {
        const float4 g0 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h), g1 = *reinterpret_cast<const float4*>(a.gamma + 16 * s + 8 * h + 4);
        const float4 e0 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h), e1 = *reinterpret_cast<const float4*>(a.beta + 16 * s + 8 * h + 4);
        const float ga[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w}, be[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pk.u[e] = pack2_f(fmaf((xv[s][2 * e] - mean) * rstd, ga[2 * e], be[2 * e]), fmaf((xv[s][2 * e + 1] - mean) * rstd, ga[2 * e + 1], be[2 * e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) pk.u[e] = pack2_f((xv[s][2 * e] - mean) * rstd, (xv[s][2 * e + 1] - mean) * rstd);
      }
      b[s] = pk.v;
      // operand layout (channels 16s + 8h + 0..7) -> accumulator layout (32ct + 8g + 4h + 0..3): s = 2ct + j, groups 2j / 2j + 1, one swap per pair
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(xv[s][e]), __float_as_uint(xv[s][4 + e]), false, false);
        acc_out[s >> 1][8 * (s & 1) + e] = __uint_as_float(sw[0]);
        acc_out[s >> 1][8 * (s & 1) + 4 + e] = __uint_as_float(sw[1]);
      }
    };
#pragma unroll
    for (int s = 0; s < KS; ++s) ln_pack(std::integral_constant<bool, kAffine>{}, s);
  }
  float* qb_lds = reinterpret_cast<float*>(smem + kQb);
  for (int i = tid; i < NH * 96; i += 256) qb_lds[i] = a.qkv_bias[i];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" :: "v"(b[s]));
  // (two sub-chunks ahead, not three: with three plus the bias pieces a wave had up to 26 vector-memory operations outstanding, and past ~16 the
  //  issue of the next one waits for the oldest to retire -- a hidden wait inside the tiles)
  issue_sub(0);
#pragma unroll
  for (int i = 0; i < kRbN; ++i) issue_rb_i(0, i);
  issue_sub(1);

  const unsigned kx_w = smem_base + kKx + static_cast<unsigned>(((wi * 2 + tt) * 2) * 1024 + lane * 16);       // this wave's K operands (k-step s: + s KiB)
  const unsigned kx_r = smem_base + kKx + static_cast<unsigned>((wi * 2 * 2) * 1024 + lane * 16);              // the window's: + (kt * 2 + s) KiB
  const unsigned vt_b = smem_base + kVt + static_cast<unsigned>(wi * 4096);
  const unsigned vt_w = vt_b + static_cast<unsigned>((32 * tt + r) * 64 + 8 * h);                               // d = 8g + 4h .. + 3: + 16 g bytes
  const unsigned qb_a = smem_base + kQb + static_cast<unsigned>(16 * h);                                         // + (head * 96 + which * 32 + 8g) * 4
  const float sl2 = a.scale * 1.4426950408889634f;

  auto frag6 = [&](bf16x8 (&f)[6], unsigned addr) {
    asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:1024\n\tds_read_b128 %2, %6 offset:2048\n\t"
                 "ds_read_b128 %3, %6 offset:3072\n\tds_read_b128 %4, %6 offset:4096\n\tds_read_b128 %5, %6 offset:5120"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]) : "v"(addr) : "memory");
  };
  // one 32-unit tile of the row-block product + its bias: acc[unit 8g + 4h + e][token]; ta = the sub-chunk's first fragment (+ lane * 16)
  // N products over consecutive fragments at ta through a ring of six registers: fragment i is the oldest of the (at most six) reads in flight,
  // its register takes fragment i + 6 as soon as its product has issued; prod(i, fragment) issues product i, between(i) what goes behind it
  auto ring6 = [&](auto n_tag, unsigned ta, auto&& prod, auto&& between) {
    constexpr int N = decltype(n_tag)::value;
    bf16x8 f[6];
    frag6(f, ta);
    static_for<0, N>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i + 6 <= N) wait_lgkm<5>();
      else wait_lgkm<N - 1 - i>();
      __builtin_amdgcn_sched_barrier(0);
      prod(ic, f[i % 6]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i + 6 < N)
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f[i % 6]) : "v"(ta), "n"((i + 6) * 1024) : "memory");
      between(ic);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto tile = [&](unsigned ta, unsigned bias_a, f32x16& acc, auto&& between) {
    f32x4 bv[4];
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:32\n\tds_read_b128 %2, %4 offset:64\n\tds_read_b128 %3, %4 offset:96"
                 : "=&v"(bv[0]), "=&v"(bv[1]), "=&v"(bv[2]), "=&v"(bv[3]) : "v"(bias_a) : "memory");
    zero_acc(acc);
    // (The token's operand registers b[] must STAY in arch VGPRs: with more than ~250 live values the allocator parks them in AGPRs and moves
    // all C/4 dwords back in front of every tile -- profiles/r06/clap_attn_big.txt.)
    // fragments in two sets of six: group g + 1 is requested before group g's products, so that only the tile's first group waits for the LDS
    if constexpr (kRing6) {
      ring6(std::integral_constant<int, KS>{}, ta,
            [&](auto ic, const bf16x8& fr) { acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr, b[decltype(ic)::value], acc, 0, 0, 0); }, between);
    } else {
    bf16x8 f[2][6];
    frag6(f[0], ta);
    static_for<0, KS / 6>([&](auto gc) {
      constexpr int g = decltype(gc)::value;
      constexpr bool more = g + 1 < KS / 6;
      if constexpr (more) frag6(f[(g + 1) & 1], ta + static_cast<unsigned>((g + 1) * 6 * 1024));
      static_for<0, 6>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        wait_lgkm<(5 - j) + (more ? 6 : 0)>();
        __builtin_amdgcn_sched_barrier(0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[g & 1][j], b[6 * g + j], acc, 0, 0, 0);      // (one chain: two were measured, twice, +-0)
        __builtin_amdgcn_sched_barrier(0);
        between(std::integral_constant<int, 6 * g + j>{});
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * g + e] += bv[g][e];
  };
  // sub-chunk n has landed for everybody (and n - 1 has been read by everybody): counted wait (kExtra = other vector-memory operations of
  // this wave that are younger than sub-chunk n and may stay outstanding), barrier, then n + 3 goes into the slot of n - 1
  auto sub_ready = [&](int n, auto extra_tag) {
    constexpr int kExtra = decltype(extra_tag)::value;
    wait_vm<IPW + kExtra>();
    asm volatile("s_barrier" ::: "memory");
    (void)n;
  };

  for (int hd = 0; hd < NH; ++hd) {
    const int n0 = 4 * hd;
    ADT_ATB_STAMP(0);
    // in-order list of this wave's vector-memory operations here: sub-chunk n0, the 8 bias pieces of this head, sub-chunk n0 + 1
    sub_ready(n0, std::integral_constant<int, kRbN>{});
    ADT_ATB_STAMP(1);
    const unsigned ba = qb_a + static_cast<unsigned>(hd * 96 * 4);
    // sub-chunk n + 2 is issued one instruction behind every (KS / IPW)-th product of the tile that reads sub-chunk n
    constexpr int kEvery = KS / IPW;
    auto dma_q = [&](auto mc) { constexpr int m = decltype(mc)::value; if constexpr (m % kEvery == 1) issue_sub_i(n0 + 2, m / kEvery); };
    auto dma_k = [&](auto mc) { constexpr int m = decltype(mc)::value; if constexpr (m % kEvery == 1) issue_sub_i(n0 + 3, m / kEvery); };
    auto dma_v = [&](auto mc) { constexpr int m = decltype(mc)::value; if constexpr (m % kEvery == 1) issue_sub_i(n0 + 4, m / kEvery); };
    f32x16 acc;
    bf16x8 qop[2];
    tile(smem_base + static_cast<unsigned>(slot(n0) * kSubBytes + lane * 16), ba, acc, dma_q);                    // q
    qop[0] = acc_to_b_f(acc, 0); qop[1] = acc_to_b_f(acc, 1);
    ADT_ATB_STAMP(2);
    sub_ready(n0 + 1, std::integral_constant<int, 0>{});
    ADT_ATB_STAMP(3);          // (younger than sub-chunk n0 + 1: n0 + 2; the bias pieces are OLDER than n0 + 1: landed with it)
    tile(smem_base + static_cast<unsigned>(slot(n0 + 1) * kSubBytes + lane * 16), ba + 128, acc, dma_k);        // k -> the window's K operands
    {
      const bf16x8 k0 = acc_to_b_f(acc, 0), k1 = acc_to_b_f(acc, 1);
      asm volatile("ds_write_b128 %0, %1\n\tds_write_b128 %0, %2 offset:1024" :: "v"(kx_w), "v"(k0), "v"(k1) : "memory");
    }
    ADT_ATB_STAMP(4);
    sub_ready(n0 + 2, std::integral_constant<int, 0>{});          // (younger: n0 + 3)
    ADT_ATB_STAMP(5);
    tile(smem_base + static_cast<unsigned>(slot(n0 + 2) * kSubBytes + lane * 16), ba + 256, acc, dma_v);        // v -> the window's [key][d] tile
    ADT_ATB_STAMP(14);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const unsigned lo = pack2_c(acc[4 * g], acc[4 * g + 1]), hi = pack2_c(acc[4 * g + 2], acc[4 * g + 3]);
      typedef unsigned u32x2_ __attribute__((ext_vector_type(2)));
      const u32x2_ pr = {lo, hi};
      asm volatile("ds_write_b64 %0, %1" :: "v"(vt_w + static_cast<unsigned>(16 * g)), "v"(pr) : "memory");
    }
    ADT_ATB_STAMP(15);
    wait_lgkm<0>();
    ADT_ATB_STAMP(6);
    asm volatile("s_barrier" ::: "memory");
    ADT_ATB_STAMP(7);
    // ---- S^T[key][query] for this wave's 32 queries and the window's 64 keys
    bf16x8 kf[4];
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %4 offset:3072"
                 : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3]) : "v"(kx_r) : "memory");
    f32x16 st[2];
    wait_lgkm<0>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      zero_acc(st[kt]);
      st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[2 * kt], qop[0], st[kt], 0, 0, 0);
      st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[2 * kt + 1], qop[1], st[kt], 0, 0, 0);
    }
    ADT_ATB_STAMP(8);          // (the bias pieces landed before sub-chunk n0 + 1 did)
    ADT_ATB_STAMP(9);
    float mx = -3.0e38f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {                      // (one key tile's bias at a time: 16 registers live instead of 32)
      f32x4 rbv[4];
      if constexpr (kRb16) {
        typedef unsigned u32x4_ __attribute__((ext_vector_type(4)));
        u32x4_ rq[2];                                      // [group pair]: groups 2gp, 2gp + 1, four bf16 each
        const unsigned ra = smem_base + static_cast<unsigned>(kRb + wave * kRbWave + kt * 2048 + lane * 16);
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)" : "=&v"(rq[0]), "=&v"(rq[1]) : "v"(ra) : "memory");
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned w = rq[g >> 1][(g & 1) * 2 + (e >> 1)];
            rbv[g][e] = __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
          }
      } else {
      const unsigned ra = smem_base + static_cast<unsigned>(kRb + wave * kRbWave + kt * 4096 + lane * 16);
      asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %4 offset:3072\n\t"
                   "s_waitcnt lgkmcnt(0)"
                   : "=&v"(rbv[0]), "=&v"(rbv[1]), "=&v"(rbv[2]), "=&v"(rbv[3]) : "v"(ra) : "memory");
      }
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {                               // log2 domain: the bias table comes pre-multiplied by log2 e
          const f32x2 v = f32x2{st[kt][4 * g + e], st[kt][4 * g + e + 1]} * sl2 + f32x2{rbv[g][e], rbv[g][e + 1]};
          st[kt][4 * g + e] = v[0]; st[kt][4 * g + e + 1] = v[1];
          mx = fmaxf(mx, fmaxf(v[0], v[1]));
        }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    float sum = softmax_exp_sum(st, mx);
    sum += __shfl_xor(sum, 32);
    const float inv = 1.0f / sum;
    ADT_ATB_STAMP(10);
    // ---- O^T[d][query] = sum over keys of V^T P^T
    f32x16 o;
    zero_acc(o);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const int i16 = lane & 15, g4 = (lane >> 4) & 1;
        const unsigned base = vt_b + static_cast<unsigned>((kt * 32 + 16 * s2 + 4 * h + (i16 >> 2)) * 64 + (16 * g4 + 4 * (i16 & 3)) * 2);
        typedef __attribute__((ext_vector_type(4))) short bf16x4_;
        bf16x4_ lo, hi;
        bf16x8 af;
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:512\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(lo), "=&v"(hi) : "v"(base) : "memory");
        af[0] = lo[0]; af[1] = lo[1]; af[2] = lo[2]; af[3] = lo[3]; af[4] = hi[0]; af[5] = hi[1]; af[6] = hi[2]; af[7] = hi[3];
        union { unsigned u[4]; bf16x8 v; } pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf.u[e] = pack2_c(st[kt][8 * s2 + 2 * e], st[kt][8 * s2 + 2 * e + 1]);       // un-normalised: O is scaled by 1 / sum below
        o = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, pf.v, o, 0, 0, 0);
      }
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] *= inv;              // the softmax denominator, once per output instead of once per probability
    const bf16x8 ob0 = acc_to_b_f(o, 0), ob1 = acc_to_b_f(o, 1);
    // ---- output projection: this head's 24 (+ 8 zero) context values are k-steps 0, 1 of Wo's slice (fragment s2 * CT + ct)
    ADT_ATB_STAMP(11);
    sub_ready(n0 + 3, std::integral_constant<int, 0>{});
    ADT_ATB_STAMP(12);
    {
      const unsigned ta = smem_base + static_cast<unsigned>(slot(n0 + 3) * kSubBytes + lane * 16);
      if constexpr (kRing6) {
        ring6(std::integral_constant<int, 2 * CT>{}, ta,
              [&](auto ic, const bf16x8& fr) {
                constexpr int fi = decltype(ic)::value;
                acc_out[fi % CT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr, fi < CT ? ob0 : ob1, acc_out[fi % CT], 0, 0, 0);
              },
              [&](auto ic) {
                constexpr int fi = decltype(ic)::value;
                if constexpr (fi < kRbN) issue_rb_i(hd + 1, fi);
                else if constexpr (fi - kRbN < IPW) issue_sub_i(n0 + 5, fi - kRbN);
              });
      } else {
      bf16x8 f[2][6];
      frag6(f[0], ta);
      static_for<0, 2 * CT / 6>([&](auto gc) {
        constexpr int g = decltype(gc)::value;
        constexpr bool more = g + 1 < 2 * CT / 6;
        if constexpr (more) frag6(f[(g + 1) & 1], ta + static_cast<unsigned>((g + 1) * 6 * 1024));
        static_for<0, 6>([&](auto jc) {
          constexpr int j = decltype(jc)::value;
          constexpr int fi = 6 * g + j;
          wait_lgkm<(5 - j) + (more ? 6 : 0)>();
          __builtin_amdgcn_sched_barrier(0);
          acc_out[fi % CT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[g & 1][j], fi < CT ? ob0 : ob1, acc_out[fi % CT], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          // behind the products: the NEXT head's 8 bias pieces (their staging slots were read in this head's softmax), then sub-chunk n0 + 5
          if constexpr (fi < kRbN) issue_rb_i(hd + 1, fi);
          else if constexpr (fi - kRbN < IPW) issue_sub_i(n0 + 5, fi - kRbN);
          __builtin_amdgcn_sched_barrier(0);
        });
      });
      }
    }
    ADT_ATB_STAMP(13);
  }
  if constexpr (kMlp) {
    static_assert(!kAffine, "the one-launch layer is built with both LayerNorms folded into the weights");
    layer_mlp_tail<C, 1>(a, smem, b, acc_out, wave, lane, h, tid, win_ok, row);
    return;
  }
  // ---- x = acc_out (x went in at the start) + bias: stores only
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (win_ok) {
    float* __restrict__ xp = a.x + row * C + 4 * h;
    const float* __restrict__ ob = a.out_bias + 4 * h;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      f32x4 b2[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) b2[g] = *reinterpret_cast<const f32x4*>(ob + 32 * ct + 8 * g);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(xp + 32 * ct + 8 * g) = f32x4{acc_out[ct][4 * g] + b2[g][0], acc_out[ct][4 * g + 1] + b2[g][1],
                                                               acc_out[ct][4 * g + 2] + b2[g][2], acc_out[ct][4 * g + 3] + b2[g][3]};
    }
  }
}

template <int C, int MODE, int TPC>
static int launch_rb(const RbArgs& a, hipStream_t st) {
  constexpr int KS = C / 16;
  constexpr int kTileFrags = MODE == kRbMlp ? 2 * KS : KS;
  constexpr int kChunkBytes = TPC * kTileFrags * 1024;
  constexpr int kRing = 3;
  const int lds = kRing * kChunkBytes + 32 * a.n_tiles * 4;
  if (a.n_tiles % TPC) return set_error(ADT_ESHAPE, "htsat row-block kernel: tile count is not a multiple of the chunk size");
  static thread_local int done_for = -1;
  int dev = 0;
  ADT_HIP_TRY(hipGetDevice(&dev));
  if (done_for != dev) {
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_rowblock_kernel<C, MODE, TPC>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    done_for = dev;
  }
  const unsigned grid = static_cast<unsigned>((a.M + kRbRows - 1) / kRbRows);
  hipLaunchKernelGGL((htsat_rowblock_kernel<C, MODE, TPC>), dim3(grid), dim3(kRbThreads), lds, st, a);
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

}  // namespace adt

using namespace adt;

// Tiles per chunk of each (mode, C): chunks of 12-24 KiB.  The host packs the weight stream with the same numbers
// (adt_htsat_rowblock_chunk_tiles).
static int chunk_tiles(int mode, int C) {
  if (C == 96) return mode == kRbMlp ? 2 : 3;       // tiles of 12 / 6 KiB -> 24 / 18 KiB chunks (q/k/v: 9 tiles, out-proj: 3)
  if (C == 192) return mode == kRbMlp ? 1 : 2;      // tiles of 24 / 12 KiB -> 24 KiB chunks
  if (C == 384) return mode == kRbMlp ? 0 : 1;      // tiles of 24 KiB (no fused MLP: its 12 accumulator tiles do not fit the registers)
  return 0;
}
extern "C" int adt_htsat_rowblock_chunk_tiles(int32_t mode, int32_t C) { return chunk_tiles(mode, C); }

extern "C" int adt_htsat_rowblock(int32_t mode, float* x, int64_t M, int32_t C, const void* a16, int64_t lda, const float* ln_gamma,
                                  const float* ln_beta, float eps, const void* w_packed, int32_t n_tiles, const float* bias1,
                                  const float* bias2, void* out16, int64_t ldo, void* stream) {
  // mode 3: the MLP phase by phase (no software pipeline; its own weight order) -- the A/B arm of mode 2
  if (mode < 0 || mode > 4) return set_error(ADT_EINVAL, "adt_htsat_rowblock: mode must be 0 (LN + GEMM), 1 (GEMM + residual), 2 (MLP) or 4 (LN + GEMM + GELU)");
  if (C != 96 && C != 192 && C != 384) return set_error(ADT_ESHAPE, "adt_htsat_rowblock: built for C = 96, 192 and 384");
  if (C == 384 && mode == 3) return set_error(ADT_ESHAPE, "adt_htsat_rowblock: the phase-by-phase MLP (mode 3) is built for C = 96 and 192");
  if (M < 0 || n_tiles <= 0 || !x || !w_packed || !bias1) return set_error(ADT_EINVAL, "adt_htsat_rowblock: bad arguments");
  // (gamma and beta both NULL: plain normalisation, the caller folded the affine part into w_packed / bias1)
  if (mode != kRbGemmRes && ((ln_gamma == nullptr) != (ln_beta == nullptr))) return set_error(ADT_EINVAL, "adt_htsat_rowblock: give both LayerNorm parameters or neither");
  if (mode == kRbGemmRes && (!a16 || lda < C || (lda & 7) || n_tiles != C / 32)) return set_error(ADT_ESHAPE, "adt_htsat_rowblock: bad bf16 input / tile count");
  if ((mode == kRbLnGemm || mode == kRbLnGemmGelu) && (!out16 || ldo < 32 * n_tiles || (ldo & 3))) return set_error(ADT_ESHAPE, "adt_htsat_rowblock: bad bf16 output");
  if ((mode == 2 || mode == 3) && (!bias2 || n_tiles != C / 8)) return set_error(ADT_ESHAPE, "adt_htsat_rowblock: the MLP has 4C hidden units");
  if (!ln_gamma && mode != kRbGemmRes && mode != kRbMlp) return set_error(ADT_EINVAL, "adt_htsat_rowblock: the folded LayerNorm (NULL gamma / beta) is built for mode 2");
  if (!aligned16(x) || !aligned16(w_packed) || (a16 && !aligned16(a16)) || (out16 && (reinterpret_cast<uintptr_t>(out16) & 7)))
    return set_error(ADT_EINVAL, "adt_htsat_rowblock: misaligned pointer");
  if (M == 0) return ADT_OK;
  RbArgs a{};
  a.x = x; a.a16 = static_cast<const unsigned short*>(a16); a.lda = lda; a.gamma = ln_gamma; a.beta = ln_beta; a.eps = eps;
  a.wpk = static_cast<const unsigned char*>(w_packed); a.bias1 = bias1; a.bias2 = bias2; a.out16 = static_cast<unsigned short*>(out16);
  a.ldo = ldo; a.M = M; a.n_tiles = n_tiles;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (C == 384) {
    if (mode == kRbMlp) return launch_mlp<384, 1, 1>(a, st);
    if (mode == kRbLnGemm) return launch_rb<384, kRbLnGemm, 1>(a, st);
    if (mode == kRbLnGemmGelu) return launch_rb<384, kRbLnGemmGelu, 1>(a, st);
    return launch_rb<384, kRbGemmRes, 1>(a, st);
  }
  if (C == 96) {
    if (mode == kRbLnGemm) return launch_rb<96, kRbLnGemm, 3>(a, st);
    if (mode == kRbLnGemmGelu) return launch_rb<96, kRbLnGemmGelu, 3>(a, st);
    if (mode == kRbGemmRes) return launch_rb<96, kRbGemmRes, 3>(a, st);
    if (mode == 3) return launch_rb<96, kRbMlp, 2>(a, st);
    // one step (12 KiB) per LDS-DMA chunk: 37 KiB of LDS, three workgroups per CU (two with 24 KiB chunks; -4 % on the launch).
    static const bool spc2 = [] { const char* v = getenv("ADT_HTSAT_MLP96_SPC"); return v && v[0] == '2'; }();
    if (spc2) return launch_mlp<96, 2>(a, st);
    return launch_mlp<96, 1>(a, st);
  }
  if (mode == kRbLnGemm) return launch_rb<192, kRbLnGemm, 2>(a, st);
  if (mode == kRbLnGemmGelu) return launch_rb<192, kRbLnGemmGelu, 2>(a, st);
  if (mode == kRbGemmRes) return launch_rb<192, kRbGemmRes, 2>(a, st);
  if (mode == 3) return launch_rb<192, kRbMlp, 1>(a, st);
  return launch_mlp<192, 1>(a, st);
}

extern "C" int adt_htsat_merge_rowblock(const float* x, int64_t B, int32_t R, int32_t C_src, const float* ln_gamma, const float* ln_beta, float eps,
                                        const void* w_packed, int32_t n_tiles, const float* bias, float* out32, int64_t ldo, void* stream) {
  if (!x || !ln_gamma || !ln_beta || !w_packed || !bias || !out32) return set_error(ADT_EINVAL, "adt_htsat_merge_rowblock: null pointer");
  if (C_src != 96) return set_error(ADT_ESHAPE, "adt_htsat_merge_rowblock: built for 96 source channels (LayerNorm over 384)");
  if (B < 0 || R <= 0 || (R & 1) || n_tiles <= 0 || ldo < 32 * n_tiles || (ldo & 3)) return set_error(ADT_ESHAPE, "adt_htsat_merge_rowblock: bad shape");
  if (!aligned16(x) || !aligned16(w_packed) || !aligned16(out32)) return set_error(ADT_EINVAL, "adt_htsat_merge_rowblock: misaligned pointer");
  const long M = B * static_cast<long>(R / 2) * (R / 2);
  if (M == 0) return ADT_OK;
  RbArgs a{};
  a.x = const_cast<float*>(x); a.gamma = ln_gamma; a.beta = ln_beta; a.eps = eps; a.wpk = static_cast<const unsigned char*>(w_packed);
  a.bias1 = bias; a.out32 = out32; a.ldo = ldo; a.M = M; a.n_tiles = n_tiles; a.merge_R = R;
  return launch_rb<384, kRbMergeGemm, 1>(a, static_cast<hipStream_t>(stream));
}

extern "C" int adt_htsat_attn_block(float* x, int64_t B, int32_t R, int32_t C, int32_t heads, int32_t shift, const float* ln_gamma,
                                    const float* ln_beta, float eps, const void* w_packed, const float* qkv_bias, const float* out_bias,
                                    const float* rel_bias, int32_t n_bias_windows, float scale, void* stream) {
  if (!x || !w_packed || !qkv_bias || !out_bias || !rel_bias) return set_error(ADT_EINVAL, "adt_htsat_attn_block: null pointer");
  if ((ln_gamma == nullptr) != (ln_beta == nullptr)) return set_error(ADT_EINVAL, "adt_htsat_attn_block: give both LayerNorm parameters or neither (folded into the weights)");
  if (!((C == 96 && heads == 4) || (C == 192 && heads == 8) || (C == 384 && heads == 16)))
    return set_error(ADT_ESHAPE, "adt_htsat_attn_block: built for C = 96 / 192 / 384 with heads of 24");
  if (B < 0 || R <= 0 || (R & 7) || shift < 0 || shift >= 8) return set_error(ADT_ESHAPE, "adt_htsat_attn_block: window 8, R % 8 == 0");
  const int nw = R / 8;
  if (n_bias_windows != 1 && n_bias_windows != nw * nw) return set_error(ADT_EINVAL, "adt_htsat_attn_block: n_bias_windows must be 1 or (R/8)^2");
  if (!aligned16(x) || !aligned16(w_packed) || !aligned16(rel_bias)) return set_error(ADT_EINVAL, "adt_htsat_attn_block: misaligned pointer");
  const long n_windows = B * nw * nw;
  if (n_windows == 0) return ADT_OK;
  AtArgs a{x, ln_gamma, ln_beta, eps, static_cast<const unsigned char*>(w_packed), qkv_bias, out_bias, rel_bias, n_bias_windows,
           static_cast<int>(B), R, shift, scale};
  static thread_local int done_for = -1;
  int dev = 0;
  ADT_HIP_TRY(hipGetDevice(&dev));
  if (done_for != dev) {
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_kernel<96, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_kernel<96, false>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_big_kernel<192, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_big_kernel<192, false>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_big_kernel<384, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_big_kernel<384, false>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    done_for = dev;
  }
  const dim3 grid(static_cast<unsigned>((n_windows + 1) / 2));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool affine = ln_gamma != nullptr;
  if (C == 96) {
    constexpr int kChunk = (3 * 6 + 2 * 3) * 1024;
    const int lds = 2 * kChunk + 8 * 1024 + 2 * 4096 + 4 * 96 * 4;
    if (affine) hipLaunchKernelGGL((htsat_attn_kernel<96, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((htsat_attn_kernel<96, false>), grid, dim3(256), lds, st, a);
  } else {
    // ring of four C/16-KiB sub-chunks | K operands 8 KiB | V tiles 8 KiB | q|k|v bias | per-wave relative-bias staging 4 x 8 KiB
    const int lds = 4 * (C / 16) * 1024 + 8 * 1024 + 2 * 4096 + heads * 96 * 4 + 4 * 8192;
    if (C == 192 && affine) hipLaunchKernelGGL((htsat_attn_big_kernel<192, true>), grid, dim3(256), lds, st, a);
    else if (C == 192) hipLaunchKernelGGL((htsat_attn_big_kernel<192, false>), grid, dim3(256), lds, st, a);
    else if (affine) hipLaunchKernelGGL((htsat_attn_big_kernel<384, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((htsat_attn_big_kernel<384, false>), grid, dim3(256), lds, st, a);
#ifdef ADT_ATB_STAMPS
    if (getenv("ADT_ATB_PRINT")) {
      unsigned long long h[16];
      ADT_HIP_TRY(hipStreamSynchronize(static_cast<hipStream_t>(stream)));
      ADT_HIP_TRY(hipMemcpyFromSymbol(h, HIP_SYMBOL(g_atb_stamps), sizeof(h)));
      fprintf(stderr, "attn_big stamps C=%d (ticks of s_memtime, 100 MHz): ", C);
      for (int i = 1; i < 14; ++i) fprintf(stderr, "%d:+%lld ", i, static_cast<long long>(h[i] - h[i - 1]));
      fprintf(stderr, "| head total %lld | v segment: tile %lld, packs + writes %lld, write wait %lld\n", static_cast<long long>(h[13] - h[0]),
              static_cast<long long>(h[14] - h[5]), static_cast<long long>(h[15] - h[14]), static_cast<long long>(h[6] - h[15]));
    }
#endif
  }
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}

// One ClapAudioLayer in ONE launch (C = 96 / 192 / 384; round 6): the attention half as adt_htsat_attn_block, then the MLP half as adt_htsat_rowblock
// mode 2 on the rows still in the accumulators.  Both LayerNorms folded into the weights by the caller (no gamma / beta arguments).
extern "C" int adt_htsat_layer_block(float* x, int64_t B, int32_t R, int32_t C, int32_t heads, int32_t shift, float eps, const void* attn_w_packed,
                                     const float* qkv_bias, const float* out_bias, const float* rel_bias, int32_t n_bias_windows, float scale,
                                     const void* mlp_w_packed, int32_t n_tiles, const float* fc1_bias, const float* fc2_bias, const void* rel_bias_bf16,
                                     void* stream) {
  if (!x || !attn_w_packed || !qkv_bias || !out_bias || !rel_bias || !mlp_w_packed || !fc1_bias || !fc2_bias) return set_error(ADT_EINVAL, "adt_htsat_layer_block: null pointer");
  if (!((C == 384 && heads == 16) || (C == 192 && heads == 8) || (C == 96 && heads == 4))) return set_error(ADT_ESHAPE, "adt_htsat_layer_block: built for C = 96 / 192 / 384 with heads of 24");
  if (B < 0 || R <= 0 || (R & 7) || shift < 0 || shift >= 8 || n_tiles != C / 8) return set_error(ADT_ESHAPE, "adt_htsat_layer_block: window 8, R % 8 == 0, 4C hidden units");
  const int nw = R / 8;
  if (n_bias_windows != 1 && n_bias_windows != nw * nw) return set_error(ADT_EINVAL, "adt_htsat_layer_block: n_bias_windows must be 1 or (R/8)^2");
  if (!aligned16(x) || !aligned16(attn_w_packed) || !aligned16(rel_bias) || !aligned16(mlp_w_packed) || !aligned16(out_bias))
    return set_error(ADT_EINVAL, "adt_htsat_layer_block: misaligned pointer");
  if (C == 192 && (!rel_bias_bf16 || !aligned16(rel_bias_bf16)))
    return set_error(ADT_EINVAL, "adt_htsat_layer_block: C = 192 stages the relative-position bias as bf16 (rel_bias_bf16, 16-byte aligned)");
  const long n_windows = B * nw * nw;
  if (n_windows == 0) return ADT_OK;
  AtArgs a{x, nullptr, nullptr, eps, static_cast<const unsigned char*>(attn_w_packed), qkv_bias, out_bias, rel_bias, n_bias_windows,
           static_cast<int>(B), R, shift, scale, static_cast<const unsigned char*>(mlp_w_packed), fc1_bias, fc2_bias, n_tiles,
           static_cast<const unsigned short*>(rel_bias_bf16)};
  static thread_local int done_for = -1;
  int dev = 0;
  ADT_HIP_TRY(hipGetDevice(&dev));
  if (done_for != dev) {
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_big_kernel<384, false, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_big_kernel<192, false, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    ADT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(htsat_attn_kernel<96, false, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    done_for = dev;
  }
  const int lds_attn = C == 96 ? 2 * (3 * 6 + 2 * 3) * 1024 + 8 * 1024 + 2 * 4096 + 4 * 96 * 4
                     : C == 192 ? 3 * (C / 16) * 1024 + 8 * 1024 + 2 * 4096 + heads * 96 * 4 + 4 * 4096       // three-slot ring, bf16 bias staging: two workgroups per CU
                                : 4 * (C / 16) * 1024 + 8 * 1024 + 2 * 4096 + heads * 96 * 4 + 4 * 8192;
  const int lds_mlp = 3 * 2 * (C / 16) * 1024 + 32 * n_tiles * 4 + C * 4;
  const dim3 grid(static_cast<unsigned>((n_windows + 1) / 2));
  const int lds = lds_attn > lds_mlp ? lds_attn : lds_mlp;
  if (C == 384) hipLaunchKernelGGL((htsat_attn_big_kernel<384, false, true>), grid, dim3(256), lds, static_cast<hipStream_t>(stream), a);
  else if (C == 96) hipLaunchKernelGGL((htsat_attn_kernel<96, false, true>), grid, dim3(256), lds, static_cast<hipStream_t>(stream), a);
  else hipLaunchKernelGGL((htsat_attn_big_kernel<192, false, true>), grid, dim3(256), lds, static_cast<hipStream_t>(stream), a);
  ADT_HIP_TRY(hipGetLastError());
  return ADT_OK;
}
