// sesa_linear_i8: out[m, n] = act(x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] + bias[n]) on 8-bit integers.
//
// v_mfma_i32_16x16x64_i8 with the weights as the first operand: a lane's accumulators are then consecutive output
// channels of one token.  The sums are exact 32-bit integers; scales, bias and activation are fp32, one rounding.  The
// token's scale goes to the sum first: the two scales' own product may leave the range of fp32 where the result does not.
// Measured: one token, 4096 -> 16384 (64 MB of weights) 17.2 us, 3.9 TB/s; 8192 tokens 485 us, 2.27 POP/s (542 us back to
// back on the same inputs: the clock sinks).
//
// Two kernels:
//  * tile_kernel: BM tokens x BN channels per workgroup, K in 128-byte steps through a ring of LDS stages.
//  * few_kernel (m <= 16, and to 64 with few channels): 16 channels per workgroup, the waves split K and read both operands straight into the
//    matrix instruction's registers; joined in LDS.
#include "sesa_tokens.hpp"

namespace sesa {
namespace {

struct LinArgs {
  const int8_t* x;
  int64_t x_ld;
  const float* x_scale;
  const int8_t* w;
  int64_t w_ld;
  const float* w_scale;
  const float* bias;
  int act;
  int m, n, k;
  void* out;
  int64_t o_ld;
};

__device__ __forceinline__ i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// TO: fp32 results show what gelu_f's polynomial leaves (1.5e-7 of |v| / 2, more than the value itself below -5); 16-bit ones
// do not, and their epilogue is bound by the VALU.
template <int ACT, class TO>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == SESA_ACT_GELU && sizeof(TO) == 4) return gelu_fine_f(v);
  if constexpr (ACT == SESA_ACT_GELU) return gelu_f(v);
  if constexpr (ACT == SESA_ACT_TANH) return tanh_f(v);
  if constexpr (ACT == SESA_ACT_RELU) return v > 0.f || v != v ? v : 0.f;   // (keeps NaN)
  return v;
}

// body(activation as a constant): one copy of an epilogue per activation and one branch around them, where a branch per
// element made the epilogue 12000 instructions and slower than the product (m 49662, k 512, n 2048: 130 us of 164)
template <class F>
__device__ __forceinline__ void with_act(int act, F body) {
  if (act == SESA_ACT_NONE) body(std::integral_constant<int, SESA_ACT_NONE>{});
  else if (act == SESA_ACT_GELU) body(std::integral_constant<int, SESA_ACT_GELU>{});
  else if (act == SESA_ACT_TANH) body(std::integral_constant<int, SESA_ACT_TANH>{});
  else body(std::integral_constant<int, SESA_ACT_RELU>{});
}

// 16 bytes of a row from byte k on, zero from byte K on
__device__ __forceinline__ i32x4 load_k(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return __builtin_bit_cast(i32x4, load16(row + k));
  i32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (k + e < K) v[e >> 2] |= (int)((uint32_t)(uint8_t)row[k + e] << (8 * (e & 3)));
  return v;
}

// ---------------------------------------------------------------------------------------------
// LDS image of a stage: rows of BK bytes, 16-byte piece c of row r at position c ^ key(r), so that the 8 rows whose pieces
// a fragment read takes together lie in 8 different 16-byte columns of 128 B.  Token fragments take 16 consecutive rows;
// weight fragments rows {0..3, 16..19, 32..35, 48..51} + 4 j of a 64-row group (see tile_kernel).
template <int BK>
__device__ __forceinline__ int key_x(int r) { return BK == 128 ? r & 7 : (r >> 1) & 3; }
template <int BK>
__device__ __forceinline__ int key_w(int r) { return BK == 128 ? (r & 3) | ((r >> 2) & 4) : ((r >> 1) & 1) | ((r >> 3) & 2); }

// WAN x WAM waves, each GN groups of 64 channels x GM blocks of 16 tokens.
// Channel order: accumulator block j (0..3) of a 64-channel group holds, in row 4 g + i of the matrix instruction,
// channel 16 g + 4 j + i, so lane group g owns 16 consecutive channels (32 B of fp16 a lane, 128 B a token and
// group) and the epilogue stores straight from registers.
// DMA: rows 16-byte aligned and K % 16 == 0 -- a ring of S stages filled by global_load_lds_dwordx4 (the swizzle on the
// source address), S - 1 of them in flight.  Otherwise two stages filled through S - 1 sets of registers, where the last
// partial piece of a row is completed with zeros.
template <class TO, int WAN, int WAM, int GN, int GM, int BK, int S, int OCC, bool DMA>
__global__ void __launch_bounds__(WAN* WAM * 64, OCC) tile_kernel(LinArgs a) {
  constexpr int NW = WAN * WAM, BN = WAN * GN * 64, BM = WAM * GM * 16;
  constexpr int STAGE = (BN + BM) * BK, PIECES = STAGE / 1024 / NW, WP = BN * BK / 1024 / NW;   // per wave
  constexpr int LPR = BK / 16, RPP = 64 / LPR;   // lanes per row, rows per piece
  static_assert(STAGE % (1024 * NW) == 0 && BN * BK % (1024 * NW) == 0, "whole pieces per wave");
  constexpr int SLOTS = DMA ? S : 2;
  static_assert(S >= 2 && S <= 4 && 2 * PIECES <= 63, "counted waits");
  __shared__ __attribute__((aligned(16))) char smem[SLOTS * STAGE];
  float* xs_l = reinterpret_cast<float*>(smem);   // the tile's scales and bias, once the stages are done
  float* ws_l = xs_l + BM;
  float* b_l = ws_l + BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wn = wave % WAN, wm = wave / WAN;
  const int tiles_n = (a.n + BN - 1) / BN, tiles_m = (a.m + BM - 1) / BM;
  const int steps = (a.k + BK - 1) / BK;
  // within a die's range of tiles: strips of 4 token tiles, channels along the strip
  const int nb = tiles_m * tiles_n;
  if (long_block() >= nb) return;
  const int t = die_tile((int)long_block(), nb);
  constexpr int STRIP = 4;
  const int strip = t / (STRIP * tiles_n), in = t - strip * STRIP * tiles_n;
  const int sm = min(STRIP, tiles_m - strip * STRIP);
  const int m0 = (strip * STRIP + in % sm) * BM, n0 = in / sm * BN;

  // piece p of this wave: RPP rows from RPP (wave + NW p) on of the weight (p < WP) or token image
  const int8_t* src[PIECES];
  int piece[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const bool is_w = p < WP;
    const int r = RPP * (wave + NW * (is_w ? p : p - WP)) + lane / LPR;
    piece[p] = 16 * (lane % LPR ^ (is_w ? key_w<BK>(r) : key_x<BK>(r)));
    src[p] = is_w ? a.w + (int64_t)min(n0 + r, a.n - 1) * a.w_ld : a.x + (int64_t)min(m0 + r, a.m - 1) * a.x_ld;
  }
  constexpr int SETS = DMA ? 1 : S - 1;
  u32x4 held[SETS][DMA ? 1 : PIECES];
  auto lds_at = [&](int p) { return (p < WP ? 0 : BN * BK) + (wave + NW * (p < WP ? p : p - WP)) * 1024; };
  auto fetch = [&](int s, char* stage, u32x4* set) {
    const bool whole = (s + 1) * BK <= a.k;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int k = s * BK + piece[p];
      if constexpr (DMA)   // pieces past K: any valid address (their products are masked in the last step)
        dma16(src[p] + (whole || k < a.k ? k : 0), stage + lds_at(p));
      else
        set[p] = whole ? load16(src[p] + k) : __builtin_bit_cast(u32x4, load_k(src[p], k, a.k));
    }
  };
  auto put = [&](char* stage, const u32x4* set) {
    if constexpr (!DMA) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) *reinterpret_cast<u32x4*>(stage + lds_at(p) + lane * 16) = set[p];
    }
  };

  i32x4 acc[GN][4][GM];
  const int l16 = lane & 15, g = lane >> 4;
  // All fragment reads of ONCE 64-byte halves stand before their products: left to itself the compiler reuses one
  // register set and waits out an LDS round trip per product, which a small tile has no other waves to hide.
  constexpr int HALVES = BK / 64, ONCE = GN * GM <= 4 ? HALVES : 1;
  auto compute = [&](const char* stage, int s) {
#pragma unroll
    for (int h0 = 0; h0 < HALVES; h0 += ONCE) {
      i32x4 wf[ONCE][GN][4], xf[ONCE][GM];
#pragma unroll
      for (int q = 0; q < ONCE; ++q) {
        const int h = h0 + q;
#pragma unroll
        for (int i = 0; i < GM; ++i) {
          const int r = (wm * GM + i) * 16 + l16;
          xf[q][i] = *reinterpret_cast<const i32x4*>(stage + BN * BK + r * BK + 16 * ((h * 4 + g) ^ key_x<BK>(r)));
        }
#pragma unroll
        for (int u = 0; u < GN; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = (wn * GN + u) * 64 + (l16 >> 2) * 16 + j * 4 + (l16 & 3);
            wf[q][u][j] = *reinterpret_cast<const i32x4*>(stage + r * BK + 16 * ((h * 4 + g) ^ key_w<BK>(r)));
          }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < ONCE; ++q) {
        // the last step: pieces from K on hold anything (DMA; K % 16 == 0, so they lie whole inside or outside)
        const int k0 = s * BK + (h0 + q) * 64;
        if (DMA && k0 + 64 > a.k) {
          const bool out = k0 + 16 * g >= a.k;
#pragma unroll
          for (int i = 0; i < GM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) xf[q][i][e] = out ? 0 : xf[q][i][e];
        }
#pragma unroll
        for (int i = 0; i < GM; ++i)
#pragma unroll
          for (int u = 0; u < GN; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[u][j][i] = mfma_i8(wf[q][u][j], xf[q][i], acc[u][j][i]);
      }
    }
  };

#pragma unroll
  for (int u = 0; u < GN; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < GM; ++i) acc[u][j][i] = i32x4{0, 0, 0, 0};
  if constexpr (DMA) {
#pragma unroll
    for (int s = 0; s < S - 1; ++s)
      if (s < steps) fetch(s, smem + s * STAGE, nullptr);
    int slot = 0;
    for (int s = 0; s < steps; ++s) {
      // this wave's part of stage s has landed (at most the pieces of the stages behind it are on the way); behind the
      // barrier everyone's has, and everyone is done with stage s - 1, whose slot stage s + S - 1 takes
      const int behind = min(S - 2, steps - 1 - s);
      if (S > 3 && behind == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PIECES) : "memory");
      else if (S > 2 && behind == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      stage_sync();
      const int ahead = slot ? slot - 1 : S - 1;   // (slot + S - 1) % S
      if (s + S - 1 < steps) fetch(s + S - 1, smem + ahead * STAGE, nullptr);
      compute(smem + slot * STAGE, s);
      slot = slot + 1 < S ? slot + 1 : 0;
    }
  } else {
    // stage s + 1 waits in registers while stage s is computed, and goes to the other slot behind it; set j holds the
    // stages j, j + SETS, ...
#pragma unroll
    for (int j = 0; j < SETS; ++j)
      if (j < steps) fetch(j, nullptr, held[j]);
    put(smem, held[0]);
    for (int s0 = 0; s0 < steps; s0 += SETS) {
#pragma unroll
      for (int j = 0; j < SETS; ++j) {
        const int s = s0 + j;
        if (s >= steps) break;
        stage_sync();
        if (s + SETS < steps) fetch(s + SETS, nullptr, held[j]);
        compute(smem + (s & 1) * STAGE, s);
        if (s + 1 < steps) put(smem + ((s + 1) & 1) * STAGE, held[(j + 1) % SETS]);
      }
    }
  }

  sesa_sync();
  for (int e = tid; e < BM; e += NW * 64) xs_l[e] = a.x_scale[min(m0 + e, a.m - 1)];
  for (int e = tid; e < BN; e += NW * 64) {
    const int n = min(n0 + e, a.n - 1);
    ws_l[e] = a.w_scale[n];
    b_l[e] = a.bias ? a.bias[n] : 0.f;
  }
  sesa_sync();
  TO* out = reinterpret_cast<TO*>(a.out);
  with_act(a.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
#pragma unroll
    for (int u = 0; u < GN; ++u) {
      const int c0 = (wn * GN + u) * 64 + 16 * g, n = n0 + c0, left = a.n - n;
#pragma unroll
      for (int i = 0; i < GM; ++i) {
        const int r = (wm * GM + i) * 16 + l16, m = m0 + r;
        const float xs = xs_l[r];
        float v[2][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 w4 = *reinterpret_cast<const f32x4*>(ws_l + c0 + 4 * j);
          const f32x4 b4 = *reinterpret_cast<const f32x4*>(b_l + c0 + 4 * j);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[j >> 1][4 * (j & 1) + e] = activate<ACT, TO>(fmaf((float)acc[u][j][i][e] * xs, w4[e], b4[e]));
        }
        if (m < a.m && left > 0) {
          TO* o = out + (int64_t)m * a.o_ld + n;
          store8(o, left, v[0]);
          store8(o + 8, left - 8, v[1]);
        }
      }
    }
  });
}

// ---------------------------------------------------------------------------------------------
// Few tokens: bound by reading the weights once.  Workgroup = 16 channels x all (16 MI) tokens; NW waves take every
// NW-th 64-byte step of K, U steps' loads in flight.
template <class TO, int MI>
__global__ void __launch_bounds__(512) few_kernel(LinArgs a) {
  constexpr int NW = 8, U = 4;   // (one token, 64 MB of weights: 17.0 us; 4 waves of 8 steps 17.9)
  __shared__ i32x4 part[NW][MI][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  if (long_block() * 16 >= a.n) return;
  const int n0 = (int)long_block() * 16;
  const int8_t* wr = a.w + (int64_t)min(n0 + l16, a.n - 1) * a.w_ld + 16 * g;
  const int8_t* xr[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) xr[i] = a.x + (int64_t)min(i * 16 + l16, a.m - 1) * a.x_ld + 16 * g;
  i32x4 acc[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) acc[i] = i32x4{0, 0, 0, 0};
  const int whole = a.k / 64;   // steps that lie inside every row
  int s = wave;
  for (; s + (U - 1) * NW < whole; s += U * NW) {
    i32x4 wf[U], xf[U][MI];
#pragma unroll
    for (int q = 0; q < U; ++q) wf[q] = __builtin_bit_cast(i32x4, load16(wr + (s + q * NW) * 64));
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        // up to 16 tokens: only the rows there are (repeats of the last one would cost as many loads as the weights)
        if (MI > 1 || l16 < a.m) xf[q][i] = __builtin_bit_cast(i32x4, load16(xr[i] + (s + q * NW) * 64));
        else xf[q][i] = i32x4{0, 0, 0, 0};
      }
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[i] = mfma_i8(wf[q], xf[q][i], acc[i]);
  }
  for (; s * 64 < a.k; s += NW) {
    const i32x4 wf = load_k(wr, s * 64, a.k - 16 * g);
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[i] = mfma_i8(wf, load_k(xr[i], s * 64, a.k - 16 * g), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) part[wave][i][lane] = acc[i];
  sesa_sync();
  TO* out = reinterpret_cast<TO*>(a.out);
  with_act(a.act, [&](auto act) {
    for (int i = wave; i < MI; i += NW) {
      i32x4 v = part[0][i][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += part[w][i][lane];
      const int m = i * 16 + l16, n = n0 + 4 * g;
      if (m >= a.m) continue;
      const float xs = a.x_scale[m];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.n)
          out[(int64_t)m * a.o_ld + n + e] = (TO)activate<decltype(act)::value, TO>(
              fmaf((float)v[e] * xs, a.w_scale[n + e], a.bias ? a.bias[n + e] : 0.f));
    }
  });
}

template <class TO, int WAN, int WAM, int GN, int GM, int BK, int S, int OCC>
void launch_tile(const LinArgs& a, bool dma, hipStream_t st) {
  constexpr int BN = WAN * GN * 64, BM = WAM * GM * 16, NT = WAN * WAM * 64;
  const dim3 grid = long_grid((int64_t)((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN));
  if (dma) hipLaunchKernelGGL((tile_kernel<TO, WAN, WAM, GN, GM, BK, S, OCC, true>), grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((tile_kernel<TO, WAN, WAM, GN, GM, BK, S, OCC, false>), grid, dim3(NT), 0, st, a);
}

template <class TO>
int launch_linear(const LinArgs& a, hipStream_t st) {
  // Few tokens: the weights' reading counts, and splitting K over waves covers it.  From about 1536 blocks of 16 tokens x
  // 16 channels on the same operands are re-read so often that the 64 x 64 tile takes less (us, few | tile, k = 4096:
  // 17 x 8192 12.5 | 16.7, 17 x 16384 20.9 | 17.2, 32 x 8192 14.8 | 16.7, 64 x 4096 12.4 | 16.7, 64 x 8192 21.6 | 16.8).
  if (a.m <= 16 || (a.m <= 64 && (int64_t)((a.m + 15) / 16) * ((a.n + 15) / 16) <= 1536)) {
    const dim3 grid = long_grid((a.n + 15) / 16);
    if (a.m <= 16) hipLaunchKernelGGL((few_kernel<TO, 1>), grid, dim3(512), 0, st, a);
    else if (a.m <= 32) hipLaunchKernelGGL((few_kernel<TO, 2>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((few_kernel<TO, 4>), grid, dim3(512), 0, st, a);
    SESA_CHECK_LAUNCH();
    return SESA_OK;
  }
  const bool dma = a.k % 16 == 0 && a.x_ld % 16 == 0 && a.w_ld % 16 == 0 && (uintptr_t)a.x % 16 == 0 &&
                   (uintptr_t)a.w % 16 == 0;
  auto tiles = [&](int bm, int bn) { return (int64_t)((a.m + bm - 1) / bm) * ((a.n + bn - 1) / bn); };
  // The largest tile that still gives every compute unit a workgroup: operands are read from LDS 0.75 (256 x 256), 1
  // (128 x 128) and 2.5 (64 x 64) times per 16-deep product.  Up to K = 640 a tile has so few steps that its
  // epilogue and first loads take longer than its products: 128 x 128 in 64-byte steps leaves room for more workgroups
  // a CU, which hide each other's.  That border, many tokens (us, fp16 out; 256 | 128 | 128 at 64 bytes):
  //   49662 x K x 2048 GELU   K 512  130 | 112 | 102   576  142 | 130 | 112   640  138 | 125 | 119   1024  169 | 168 | 161
  //   49662 x K x 2048        K 512   96 |  91 |  87   576  111 | 104 |  96   640  108 | 103 | 103    768  118 | 116 | 122
  //   20000 x K x 1024 GELU   K 512   36 |  27 |  26   576   40 |  31 |  28   640   39 |  31 |  29   1024   47 |  38 |  38
  // Sizes apart (256 | 128 | 128 at 64 bytes | 64):
  //   8192 x 4096 x 16384     495 | 575 | 675 | 878    4096 x 1024 x 4096    22 |  28 |  29 |  36
  //   2048 x 2048 x 2048       30 |  15 |  20 |  18    256 x 4096 x 4096     51 |  24 |  33 |  17
  //   777 x 1008 x 1537 GELU   25 |  12 |  14 | 9.4
  // The large ones run at the rate the chip sustains on int8 products (8192^3: 2.38 PFLOP/s; MFMA busy 49 % of the
  // cycles at about 2.06 GHz); a ring deeper than two stages helps only the 64 x 64 tile (19 -> 17 us at 256 x 4096^2).
  if (a.k <= 640 && tiles(128, 128) >= 1024) launch_tile<TO, 2, 2, 1, 4, 64, 2, 3>(a, dma, st);
  else if (tiles(256, 256) >= 256) launch_tile<TO, 2, 4, 2, 4, 128, 2, 2>(a, dma, st);
  else if (tiles(128, 128) >= 256) launch_tile<TO, 2, 2, 1, 4, 128, 2, 2>(a, dma, st);
  else launch_tile<TO, 1, 4, 1, 1, 128, 4, 2>(a, dma, st);
  SESA_CHECK_LAUNCH();
  return SESA_OK;
}

}  // namespace
}  // namespace sesa

using namespace sesa;

extern "C" int sesa_linear_i8(const int8_t* x, int64_t x_ld, const float* x_scale, const int8_t* w, int64_t w_ld,
                              const float* w_scale, const float* bias, int act, int64_t m, int n, int k, void* out,
                              int out_dtype, int64_t o_ld, void* stream) {
  clear_error();
  SESA_REQUIRE(m >= 0 && m < (1ll << 31) - 256 && n >= 1 && n < (1 << 27) && k >= 1 && k <= 131071, SESA_ERR_INVALID,
               "linear_i8: m %lld, n %d, k %d (0 <= m < 2^31 - 256, 1 <= n < 2^27, 1 <= k <= 131071)", (long long)m, n, k);
  SESA_REQUIRE(act >= SESA_ACT_NONE && act <= SESA_ACT_RELU, SESA_ERR_INVALID, "linear_i8: act %d", act);
  SESA_REQUIRE(out_dtype >= SESA_DTYPE_F32 && out_dtype <= SESA_DTYPE_BF16, SESA_ERR_INVALID, "linear_i8: out_dtype %d",
               out_dtype);
  if (m == 0) return SESA_OK;
  SESA_REQUIRE(x && x_scale && w && w_scale && out, SESA_ERR_INVALID, "linear_i8: null operand");
  SESA_REQUIRE(m == 1 || o_ld >= n, SESA_ERR_INVALID, "linear_i8: o_ld %lld is below n %d", (long long)o_ld, n);
  // (no tile is smaller than 64 x 64 where m > 64: tile numbers fit 32 bits)
  SESA_REQUIRE((m + 63) / 64 * ((n + 63) / 64) < (1ll << 31), SESA_ERR_INVALID, "linear_i8: m x n too large");
  const LinArgs a{x, x_ld, x_scale, w, w_ld, w_scale, bias, act, (int)m, n, k, out, o_ld};
  hipStream_t st = as_stream(stream);
  if (out_dtype == SESA_DTYPE_F32) return launch_linear<float>(a, st);
  if (out_dtype == SESA_DTYPE_F16) return launch_linear<f16>(a, st);
  return launch_linear<__bf16>(a, st);
}
