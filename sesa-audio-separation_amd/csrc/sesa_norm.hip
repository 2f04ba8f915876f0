// sesa_norm_residual: y = residual + scale * gate_act(gate) * post_norm(x), n = pre_norm(y) (fp or 8 bits), one pass.
//
// Memory bound: x, residual (and a per-row gate) are read once, y and n written once, and every value of a row stays
// in registers between the reductions.  One wave per row up to dim 1024 (no LDS, no barrier), 256 threads up to 4096,
// 1024 above: a thread keeps at most 32 values and enough rows are in flight to cover the loads (16384 x 8192 bf16,
// sandwich norms and gate: 334 us at 256 threads, 278 at 512, 275 at 1024; 16384 x 4096: 134, 139, -).  Statistics are
// two-pass over the registers (mean, then squared deviations), so LayerNorm does not cancel.
#include "sesa_tokens.hpp"

namespace sesa {
namespace {

constexpr int kMaxDim = 32768;

// Sum or unsigned max over the TPR threads of a row; `slot` is this reduction's own LDS row, so one barrier is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    sesa_sync();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += slot[w];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* slot) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = __builtin_bit_cast(float, v);
    sesa_sync();
    v = 0;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v = max(v, __builtin_bit_cast(uint32_t, slot[w]));
  }
  return v;
}

template <int TPR, int NCH>
__device__ __forceinline__ void normalise(float (&v)[NCH][8], int kind, int dim, int t, float eps,
                                          const float* __restrict__ w, const float* __restrict__ b, float* slot) {
  float mean = 0.f;
  if (kind == SESA_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[c][e];
    mean = row_sum<TPR>(s, slot) / (float)dim;
  }
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int left = dim - (c * TPR + t) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] = e < left ? v[c][e] - mean : 0.f;
      s = fmaf(v[c][e], v[c][e], s);
    }
  }
  const float r = 1.f / sqrtf(row_sum<TPR>(s, slot + 16) / (float)dim + eps);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * TPR + t) * 8;
    float p[8];
    if (w) {
      load8(w + at, dim - at, p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] *= r * p[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] *= r;
    }
    if (b) {
      load8(b + at, dim - at, p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] += p[e];
    }
  }
}

// TPR threads per row, NCH groups of 8 elements per thread (group c of thread t: elements 8 (c TPR + t) ..).
template <class TX, class TR, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_residual_kernel(sesa_norm_args a) {
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[TPR > 64 ? 5 * 16 : 1];
  const int t = threadIdx.x % TPR;
  const int64_t row = long_block() * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;   // (whole waves; with TPR > 64 a block has one row, so its waves go together)
  const int dim = a.dim;
  float x[NCH][8], y[NCH][8], g[NCH][8];
  const TX* xr = reinterpret_cast<const TX*>(a.x) + row * a.x_ld;
  const TR* rr = reinterpret_cast<const TR*>(a.residual) + row * a.r_ld;
  const TX* gr = reinterpret_cast<const TX*>(a.gate) + (a.gate ? row / a.rows_per_gate : 0) * a.gate_ld;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * TPR + t) * 8;
    load8(xr + at, dim - at, x[c]);
    if (a.residual) load8(rr + at, dim - at, y[c]);
    if (a.gate) load8(gr + at, dim - at, g[c]);
  }
  if (a.post != SESA_NORM_NONE)
    normalise<TPR, NCH>(x, a.post, dim, t, a.eps, a.post_weight, a.post_bias, red);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * TPR + t) * 8;
    if (a.gate) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float s = g[c][e];
        if (a.gate_act == SESA_GATE_SIGMOID) s = sigmoid_f(s);
        else if (a.gate_act == SESA_GATE_SILU) s = s * sigmoid_f(s);
        else if (a.gate_act == SESA_GATE_TANH) s = tanh_f(s);
        x[c][e] *= s;
      }
    }
    if (a.scale) {
      float p[8];
      load8(a.scale + at, dim - at, p);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] *= p[e];
    }
    if (a.residual) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[c][e] += x[c][e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[c][e] = x[c][e];
    }
    if (a.y) store8(reinterpret_cast<TR*>(a.y) + row * a.y_ld + at, dim - at, y[c]);
  }
  if (!a.n && !a.q) return;
  if (a.pre != SESA_NORM_NONE)
    normalise<TPR, NCH>(y, a.pre, dim, t, a.eps, a.pre_weight, a.pre_bias, red + 32);
  if (a.n) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int at = (c * TPR + t) * 8;
      store8(reinterpret_cast<TX*>(a.n) + row * a.n_ld + at, dim - at, y[c]);
    }
    return;
  }
  // |n| as integers: a NaN or an infinity compares above every finite value, so one maximum finds both the scale and
  // the rows that have none
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int left = dim - (c * TPR + t) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) top = max(top, __builtin_bit_cast(uint32_t, y[c][e]) & 0x7fffffffu);
  }
  top = row_max<TPR>(top, red + 64);
  float amax = __builtin_bit_cast(float, top), down = 1.f;
  const bool fine = top < 0x7f800000u, some = amax >= 1.6e-36f;   // (below: the scale would be subnormal; counts as 0)
  // amax / 127 and 1 / scale, each rounded to nearest: an estimate and one correction by its exact remainder (Markstein).
  float scale = 0.f, inv = 0.f;
  if (fine && some) {
    if (amax < 0x1p-90f) {   // (rare: the remainders would be subnormal)
      amax *= 0x1p64f;
      down = 0x1p-64f;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[c][e] *= 0x1p64f;
    }
    scale = amax * (1.f / 127.f);
    scale = fmaf(fmaf(-127.f, scale, amax), 1.f / 127.f, scale);
    inv = __builtin_amdgcn_rcpf(scale);
    inv = fmaf(fmaf(-inv, scale, 1.f), inv, inv);
  }
  if (t == 0) a.q_scale[row] = fine ? scale * down : __builtin_nanf("");
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * TPR + t) * 8, left = dim - at;
    if (left <= 0) continue;
    int8_t* qp = a.q + row * a.q_ld + at;
    uint32_t w[2] = {0, 0};   // (a row without a scale stores 0)
    if (inv > 0.f) {
      uint32_t k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // y / scale rounded to nearest, the same way; at most 127 (1 + 2^-23) in size: no clamp needed.  1.5 * 2^23 on top
        // rounds it to a whole number, half to even, whose two's complement is the sum's low byte.
        const float g = y[c][e] * inv;
        k[e] = __builtin_bit_cast(uint32_t, fmaf(fmaf(-g, scale, y[c][e]), inv, g) + 12582912.f);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)   // the four low bytes: two and two, then all
        w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(k[4 * h + 3], k[4 * h + 2], 0x0c0c0400u),
                                     __builtin_amdgcn_perm(k[4 * h + 1], k[4 * h], 0x0c0c0400u), 0x05040100u);
    }
    if (left >= 8) {
      struct __attribute__((packed)) B8 { uint32_t a, b; };
      *reinterpret_cast<B8*>(qp) = B8{w[0], w[1]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) qp[e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  }
}

template <class TX, class TR>
int launch_norm(const sesa_norm_args& a, hipStream_t st) {
  auto go = [&](auto tpr, auto nch) {
    constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value, NT = TPR < 256 ? 256 : TPR;
    const int64_t blocks = (a.rows + NT / TPR - 1) / (NT / TPR);
    hipLaunchKernelGGL((norm_residual_kernel<TX, TR, TPR, NCH>), long_grid(blocks), dim3(NT), 0, st, a);
  };
  using std::integral_constant;
  if (a.dim <= 512) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (a.dim <= 1024) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (a.dim <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (a.dim <= 4096) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (a.dim <= 8192) go(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
  else if (a.dim <= 16384) go(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  else go(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
  SESA_CHECK_LAUNCH();
  return SESA_OK;
}

}  // namespace
}  // namespace sesa

using namespace sesa;

extern "C" int sesa_norm_residual(const sesa_norm_args* args, void* stream) {
  clear_error();
  SESA_REQUIRE(args, SESA_ERR_INVALID, "norm_residual: null arguments");
  const sesa_norm_args& a = *args;
  SESA_REQUIRE(a.rows >= 0 && a.rows < (1ll << 31) && a.dim >= 1 && a.dim <= kMaxDim, SESA_ERR_INVALID,
               "norm_residual: rows %lld, dim %d (0 <= rows < 2^31, 1 <= dim <= %d)", (long long)a.rows, a.dim, kMaxDim);
  const bool x16 = a.x_dtype == SESA_DTYPE_F16 || a.x_dtype == SESA_DTYPE_BF16;
  SESA_REQUIRE(x16 || a.x_dtype == SESA_DTYPE_F32, SESA_ERR_INVALID, "norm_residual: x_dtype %d", a.x_dtype);
  SESA_REQUIRE(a.r_dtype == a.x_dtype || a.r_dtype == SESA_DTYPE_F32, SESA_ERR_INVALID,
               "norm_residual: r_dtype %d is neither x's type nor fp32", a.r_dtype);
  SESA_REQUIRE(a.post >= SESA_NORM_NONE && a.post <= SESA_NORM_LAYER && a.pre >= SESA_NORM_NONE &&
                   a.pre <= SESA_NORM_LAYER, SESA_ERR_INVALID, "norm_residual: norm kinds %d, %d", a.post, a.pre);
  SESA_REQUIRE(a.gate_act >= SESA_GATE_NONE && a.gate_act <= SESA_GATE_TANH, SESA_ERR_INVALID,
               "norm_residual: gate_act %d", a.gate_act);
  SESA_REQUIRE(a.eps >= 0.f && a.eps < INFINITY, SESA_ERR_INVALID, "norm_residual: eps %g", (double)a.eps);
  if (a.rows == 0) return SESA_OK;
  SESA_REQUIRE(!(a.n && a.q) && (a.y || a.n || a.q), SESA_ERR_INVALID,
               "norm_residual: at most one of n and q, at least one of y, n and q");
  SESA_REQUIRE(a.x, SESA_ERR_INVALID, "norm_residual: null x");
  SESA_REQUIRE(!a.q || a.q_scale, SESA_ERR_INVALID, "norm_residual: q without q_scale");
  SESA_REQUIRE(!a.gate || a.rows_per_gate >= 1, SESA_ERR_INVALID, "norm_residual: rows_per_gate %lld",
               (long long)a.rows_per_gate);
  // a row of an output may not reach into the next one (one row: any ld)
  SESA_REQUIRE(a.rows == 1 || ((!a.y || a.y_ld >= a.dim) && (!a.n || a.n_ld >= a.dim) && (!a.q || a.q_ld >= a.dim)),
               SESA_ERR_INVALID, "norm_residual: an output's ld is below dim %d", a.dim);
  hipStream_t st = as_stream(stream);
  if (a.x_dtype == SESA_DTYPE_F32) return launch_norm<float, float>(a, st);
  if (a.x_dtype == SESA_DTYPE_F16)
    return a.r_dtype == SESA_DTYPE_F32 ? launch_norm<f16, float>(a, st) : launch_norm<f16, f16>(a, st);
  return a.r_dtype == SESA_DTYPE_F32 ? launch_norm<__bf16, float>(a, st) : launch_norm<__bf16, __bf16>(a, st);
}
