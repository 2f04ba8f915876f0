// sesa_linear_i8: out[m, n] = act(x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] + bias[n]) on 8-bit integers.
//
// v_mfma_i32_16x16x64_i8 with the weights as the first operand: a lane's accumulators are then consecutive output
// channels of one token.  The sums are exact 32-bit integers; scales, bias and activation are fp32, one rounding.
//
// Two kernels:
//  * tile_kernel: BM tokens x BN channels per workgroup, K in 128-byte steps through a ring of LDS stages.
//  * few_kernel (m <= 64): 16 channels per workgroup, the waves split K and read both operands straight into the
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

__device__ __forceinline__ float activate(float v, int act) {
  if (act == SESA_ACT_GELU) return gelu_erf(v);
  if (act == SESA_ACT_TANH) return tanh_f(v);
  if (act == SESA_ACT_RELU) return v > 0.f || v != v ? v : 0.f;   // (keeps NaN)
  return v;
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
constexpr int kBK = 128;   // K bytes per stage: one row is 8 16-byte pieces

// LDS image of a stage: rows of 128 B, piece c of row r at position c ^ key(r), so that the 8 rows whose pieces a
// fragment read takes together lie in 8 different piece columns.  Token fragments take 16 consecutive rows; weight
// fragments rows {0..3, 16..19, 32..35, 48..51} + 4 j of a 64-row group (see tile_kernel).
__device__ __forceinline__ int key_x(int r) { return r & 7; }
__device__ __forceinline__ int key_w(int r) { return (r & 3) | ((r >> 2) & 4); }

// WAN x WAM waves, each GN groups of 64 channels x GM blocks of 16 tokens.
// Channel order: accumulator block j (0..3) of a 64-channel group holds, in row 4 g + i of the matrix instruction,
// channel 16 g + 4 j + i, so lane group g owns 16 consecutive channels (32 B of fp16 a lane, 128 B a token and
// group) and the epilogue stores straight from registers.
// DMA: rows 16-byte aligned and K % 16 == 0 -- stages filled by global_load_lds_dwordx4 (the swizzle on the source
// address).  Otherwise through registers, where the last partial piece of a row is completed with zeros.
template <class TO, int WAN, int WAM, int GN, int GM, bool DMA>
__global__ void __launch_bounds__(WAN* WAM * 64, 2) tile_kernel(LinArgs a) {
  constexpr int NW = WAN * WAM, BN = WAN * GN * 64, BM = WAM * GM * 16;
  constexpr int STAGE = (BN + BM) * kBK, PIECES = STAGE / 1024 / NW, WP = BN * kBK / 1024 / NW;   // per wave
  static_assert(STAGE % (1024 * NW) == 0 && BN * kBK % (1024 * NW) == 0, "whole pieces per wave");
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wn = wave % WAN, wm = wave / WAN;
  const int tiles_n = (a.n + BN - 1) / BN, tiles_m = (a.m + BM - 1) / BM;
  // within a die's range: strips of 4 token tiles, channels along the strip
  const int t = die_tile(blockIdx.x, gridDim.x);
  constexpr int STRIP = 4;
  const int strip = t / (STRIP * tiles_n), in = t - strip * STRIP * tiles_n;
  const int sm = min(STRIP, tiles_m - strip * STRIP);
  const int m0 = (strip * STRIP + in % sm) * BM, n0 = in / sm * BN;
  const int steps = (a.k + kBK - 1) / kBK;

  // piece p of this wave: rows 8 (wave + NW p) .. + 7 of the weight (p < WP) or token image, 8 lanes a row
  const int8_t* src[PIECES];
  int piece[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const bool is_w = p < WP;
    const int r = 8 * (wave + NW * (is_w ? p : p - WP)) + (lane >> 3);
    piece[p] = 16 * ((lane & 7) ^ (is_w ? key_w(r) : key_x(r)));
    src[p] = is_w ? a.w + (int64_t)min(n0 + r, a.n - 1) * a.w_ld : a.x + (int64_t)min(m0 + r, a.m - 1) * a.x_ld;
  }
  u32x4 held[DMA ? 1 : PIECES];
  auto lds_at = [&](int p) { return (p < WP ? 0 : BN * kBK) + (wave + NW * (p < WP ? p : p - WP)) * 1024; };
  auto fetch = [&](int s, char* stage) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int k = s * kBK + piece[p];
      if constexpr (DMA) {   // pieces past K: any valid address (their products are masked in the last step)
        dma16(src[p] + (k < a.k ? k : 0), stage + lds_at(p));
      } else {
        held[p] = __builtin_bit_cast(u32x4, load_k(src[p], k, a.k));
      }
    }
  };
  auto put = [&](char* stage) {
    if constexpr (!DMA) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) *reinterpret_cast<u32x4*>(stage + lds_at(p) + lane * 16) = held[p];
    }
  };

  i32x4 acc[GN][4][GM];
#pragma unroll
  for (int u = 0; u < GN; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < GM; ++i) acc[u][j][i] = i32x4{0, 0, 0, 0};

  const int l16 = lane & 15, g = lane >> 4;
  auto compute = [&](const char* stage, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k0 = s * kBK + h * 64;
      if (k0 >= a.k) break;
      i32x4 wf[GN][4], xf[GM];
#pragma unroll
      for (int i = 0; i < GM; ++i) {
        const int r = (wm * GM + i) * 16 + l16;
        xf[i] = *reinterpret_cast<const i32x4*>(stage + BN * kBK + r * kBK + 16 * ((h * 4 + g) ^ key_x(r)));
      }
#pragma unroll
      for (int u = 0; u < GN; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = (wn * GN + u) * 64 + (l16 >> 2) * 16 + j * 4 + (l16 & 3);
          wf[u][j] = *reinterpret_cast<const i32x4*>(stage + r * kBK + 16 * ((h * 4 + g) ^ key_w(r)));
        }
      if (DMA && k0 + 64 > a.k && k0 + 16 * g >= a.k) {   // (K % 16 == 0: whole pieces lie inside or outside)
#pragma unroll
        for (int i = 0; i < GM; ++i) xf[i] = i32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < GM; ++i)
#pragma unroll
        for (int u = 0; u < GN; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[u][j][i] = mfma_i8(wf[u][j], xf[i], acc[u][j][i]);
    }
  };

  fetch(0, smem);
  put(smem);
  for (int s = 0; s < steps; ++s) {
    char* cur = smem + (s & 1) * STAGE;
    char* next = smem + ((s + 1) & 1) * STAGE;
    // this wave's part of stage s has landed; after the barrier everyone's has, and everyone is done reading stage
    // s - 1, whose place stage s + 1 takes
    if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    sesa_sync();
    if (s + 1 < steps) fetch(s + 1, next);
    compute(cur, s);
    if (s + 1 < steps) put(next);
  }

  TO* out = reinterpret_cast<TO*>(a.out);
#pragma unroll
  for (int u = 0; u < GN; ++u) {
    const int n = n0 + (wn * GN + u) * 64 + 16 * g, left = a.n - n;
    float ws[16], b[16];
    {
      float lo[8], hi[8];
      load8(a.w_scale + n, left, lo);
      load8(a.w_scale + n + 8, left - 8, hi);
#pragma unroll
      for (int e = 0; e < 8; ++e) { ws[e] = lo[e]; ws[8 + e] = hi[e]; }
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.f;
      if (a.bias) {
        load8(a.bias + n, left, lo);
        load8(a.bias + n + 8, left - 8, hi);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) { b[e] = lo[e]; b[8 + e] = hi[e]; }
    }
#pragma unroll
    for (int i = 0; i < GM; ++i) {
      const int m = m0 + (wm * GM + i) * 16 + l16;
      const float xs = a.x_scale[min(m, a.m - 1)];
      float lo[8], hi[8];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 4 * j + e;
          const float v = activate(fmaf((float)acc[u][j][i][e], xs * ws[c], b[c]), a.act);
          if (c < 8) lo[c] = v;
          else hi[c - 8] = v;
        }
      if (m < a.m && left > 0) {
        TO* o = out + (int64_t)m * a.o_ld + n;
        store8(o, left, lo);
        store8(o + 8, left - 8, hi);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Few tokens: bound by reading the weights once.  Workgroup = 16 channels x all (16 MI) tokens; NW waves take every
// NW-th 64-byte step of K, kUnroll steps' loads in flight.
template <class TO, int MI>
__global__ void __launch_bounds__(256) few_kernel(LinArgs a) {
  constexpr int NW = 4, U = MI == 1 ? 8 : 4;
  __shared__ i32x4 part[NW][MI][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
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
      for (int i = 0; i < MI; ++i) xf[q][i] = __builtin_bit_cast(i32x4, load16(xr[i] + (s + q * NW) * 64));
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
        out[(int64_t)m * a.o_ld + n + e] =
            (TO)activate(fmaf((float)v[e], xs * a.w_scale[n + e], a.bias ? a.bias[n + e] : 0.f), a.act);
  }
}

template <class TO, int WAN, int WAM, int GN, int GM>
void launch_tile(const LinArgs& a, bool dma, hipStream_t st) {
  constexpr int BN = WAN * GN * 64, BM = WAM * GM * 16, NT = WAN * WAM * 64;
  const dim3 grid((unsigned)((int64_t)((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN)));
  if (dma) hipLaunchKernelGGL((tile_kernel<TO, WAN, WAM, GN, GM, true>), grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((tile_kernel<TO, WAN, WAM, GN, GM, false>), grid, dim3(NT), 0, st, a);
}

template <class TO>
int launch_linear(const LinArgs& a, hipStream_t st) {
  if (a.m <= 64) {
    const dim3 grid((unsigned)((a.n + 15) / 16));
    if (a.m <= 16) hipLaunchKernelGGL((few_kernel<TO, 1>), grid, dim3(256), 0, st, a);
    else if (a.m <= 32) hipLaunchKernelGGL((few_kernel<TO, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((few_kernel<TO, 4>), grid, dim3(256), 0, st, a);
    SESA_CHECK_LAUNCH();
    return SESA_OK;
  }
  const bool dma = a.k % 16 == 0 && a.x_ld % 16 == 0 && a.w_ld % 16 == 0 && (uintptr_t)a.x % 16 == 0 &&
                   (uintptr_t)a.w % 16 == 0;
  auto tiles = [&](int bm, int bn) { return (int64_t)((a.m + bm - 1) / bm) * ((a.n + bn - 1) / bn); };
  // the largest tile that still gives every compute unit a workgroup
  if (tiles(256, 256) >= 256) launch_tile<TO, 2, 4, 2, 4>(a, dma, st);
  else if (tiles(128, 128) >= 256) launch_tile<TO, 2, 2, 1, 4>(a, dma, st);
  else launch_tile<TO, 1, 4, 1, 1>(a, dma, st);
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
  SESA_REQUIRE(m >= 0 && m < (1ll << 31) - 256 && n >= 1 && n < (1 << 30) && k >= 1 && k <= 131071, SESA_ERR_INVALID,
               "linear_i8: m %lld, n %d, k %d (0 <= m < 2^31 - 256, 1 <= n < 2^30, 1 <= k <= 131071)", (long long)m, n, k);
  SESA_REQUIRE(act >= SESA_ACT_NONE && act <= SESA_ACT_RELU, SESA_ERR_INVALID, "linear_i8: act %d", act);
  SESA_REQUIRE(out_dtype >= SESA_DTYPE_F32 && out_dtype <= SESA_DTYPE_BF16, SESA_ERR_INVALID, "linear_i8: out_dtype %d",
               out_dtype);
  if (m == 0) return SESA_OK;
  SESA_REQUIRE(x && x_scale && w && w_scale && out, SESA_ERR_INVALID, "linear_i8: null operand");
  SESA_REQUIRE(m == 1 || o_ld >= n, SESA_ERR_INVALID, "linear_i8: o_ld %lld is below n %d", (long long)o_ld, n);
  SESA_REQUIRE((m + 63) / 64 * ((n + 63) / 64) < (1ll << 31), SESA_ERR_INVALID, "linear_i8: m x n too large");
  const LinArgs a{x, x_ld, x_scale, w, w_ld, w_scale, bias, act, (int)m, n, k, out, o_ld};
  hipStream_t st = as_stream(stream);
  if (out_dtype == SESA_DTYPE_F32) return launch_linear<float>(a, st);
  if (out_dtype == SESA_DTYPE_F16) return launch_linear<f16>(a, st);
  return launch_linear<__bf16>(a, st);
}
