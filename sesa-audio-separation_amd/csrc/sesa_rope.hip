// sesa_rope_axes: rotary positions of several axes on one or two tensors (q and k) of the same tokens, one launch.
//
// Memory bound (each element read once and written once).  A thread owns up to 8 pairs of one token (16-byte loads and
// stores of 16-bit types), takes their sines and cosines once and applies them to its share of the heads of every tensor;
// heads are dealt to more threads only where the tokens alone do not fill the chip.  24001 tokens, 32 + 8 heads x 128,
// bf16: 109 us, 4.5 TB/s of the copy's 5.1; three tokens: 5.6 us on the device.
// Angle: one turn is 2^64.  freqs / (2 pi), with 1 / (2 pi) in two doubles, is reduced to a fraction of a turn and held as
// a 64-bit integer, so position * freq wraps modulo one turn in integer arithmetic: the phase is off by at most |position|
// 2^-63 turns for |freq| up to 2^40 (one double: |position| max(1, |freq| / pi) 2^-54; an fp32 product is off by half a
// radian at position 10^7).  The phase's top 32 bits then go to sin / cos as fp32 half-turns, off by at most 2^-25 of one.
#include "sesa_tokens.hpp"

namespace sesa {
namespace {

constexpr int kPairs = 8;   // pairs per thread: 16 B of 16-bit elements per load in the split layout

struct RopePlan {
  int P;        // rotated pairs per head
  int n_rot;    // threads per token that rotate
  int n_all;    // ... and that copy the elements behind the pairs
  int hsplit;   // heads of each tensor are dealt round-robin to this many threads
};

// freq / (2 pi) modulo one turn in units of 2^-64 turns, rounded to an even number of them
__device__ __forceinline__ uint64_t turn_step(float freq) {
#pragma clang fp contract(off)   // (f as rounded: a product fused into f - rint(f) would count the remainder twice)
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57, kTurn = 0x1p63;   // 1 / (2 pi) = kHi + kLo
  const double f = (double)freq * kHi, rem = fma((double)freq, kHi, -f) + (double)freq * kLo;
  const double top = (f - rint(f)) * kTurn, whole = trunc(top);   // [-1/2, 1/2] turns: times 2^63 it fits with room
  const double low = rint((rem - rint(rem)) * kTurn + (top - whole));
  return ((uint64_t)(int64_t)whole + (uint64_t)(int64_t)low) << 1;
}

template <class T, bool PAIRS>
__global__ void __launch_bounds__(256) rope_axes_kernel(sesa_rope_args a, RopePlan pl) {
  const int64_t per_token = (int64_t)pl.n_all * pl.hsplit;
  const int64_t id = long_block() * 256 + threadIdx.x;
  const int64_t token = id / per_token;
  if (token >= a.tokens) return;
  const int rest = (int)(id - token * per_token);
  const int h0 = rest / pl.n_all, c = rest - h0 * pl.n_all;
  if (c >= pl.n_rot) {   // 16 pass-through elements
    const int at = 2 * pl.P + (c - pl.n_rot) * 16, left = a.head_dim - at;
    for (int k = 0; k < a.n_tensors; ++k) {
      const sesa_rope_tensor& r = a.t[k];
      for (int h = h0; h < r.heads; h += pl.hsplit) {
        const T* xp = reinterpret_cast<const T*>(r.x) + token * r.x_t + h * r.x_h + at;
        T* op = reinterpret_cast<T*>(r.out) + token * r.o_t + h * r.o_h + at;
        float u[8], v[8];
        load8(xp, left, u);
        load8(xp + 8, left - 8, v);
        store8(op, left, u);
        store8(op + 8, left - 8, v);
      }
    }
    return;
  }
  const int p0 = c * kPairs, np = pl.P - p0;   // pairs from here on
  float cs[kPairs], sn[kPairs];
  const int e1 = a.sections[0], e2 = e1 + a.sections[1], e3 = e2 + a.sections[2];   // (unused sections are 0)
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int p = p0 + i;
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (i < np) {
      const int axis = (p >= e1) + (p >= e2) + (p >= e3);
      const int64_t at = token * a.positions_ld + min(axis, a.n_axes - 1);
      const int64_t pos = a.positions_i64 ? reinterpret_cast<const int64_t*>(a.positions)[at]
                                          : reinterpret_cast<const int32_t*>(a.positions)[at];
      const float freq = a.freqs[p];
      const bool fine = fabsf(freq) < INFINITY;   // (anything else has no integer; it turns its pair into NaN)
      const int32_t phase = (int32_t)((turn_step(fine ? freq : 0.f) * (uint64_t)pos) >> 32);
      sincospif((float)phase * 4.656612873077392578125e-10f, &sn[i], &cs[i]);   // phase 2^-31 half-turns
      if (!fine) cs[i] = sn[i] = __builtin_nanf("");
    }
  }
  for (int k = 0; k < a.n_tensors; ++k) {
    const sesa_rope_tensor& r = a.t[k];
#pragma unroll 4
    for (int h = h0; h < r.heads; h += pl.hsplit) {
      const T* xp = reinterpret_cast<const T*>(r.x) + token * r.x_t + h * r.x_h;
      T* op = reinterpret_cast<T*>(r.out) + token * r.o_t + h * r.o_h;
      float u[8], v[8], s[8], d[8];
      if constexpr (PAIRS) {
        load8(xp + 2 * p0, 2 * np, u);
        load8(xp + 2 * p0 + 8, 2 * np - 8, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[2 * i] = u[2 * i] * cs[i] - u[2 * i + 1] * sn[i];
          s[2 * i + 1] = u[2 * i] * sn[i] + u[2 * i + 1] * cs[i];
          d[2 * i] = v[2 * i] * cs[4 + i] - v[2 * i + 1] * sn[4 + i];
          d[2 * i + 1] = v[2 * i] * sn[4 + i] + v[2 * i + 1] * cs[4 + i];
        }
        store8(op + 2 * p0, 2 * np, s);
        store8(op + 2 * p0 + 8, 2 * np - 8, d);
      } else {
        load8(xp + p0, np, u);
        load8(xp + pl.P + p0, np, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[i] = u[i] * cs[i] - v[i] * sn[i];
          d[i] = u[i] * sn[i] + v[i] * cs[i];
        }
        store8(op + p0, np, s);
        store8(op + pl.P + p0, np, d);
      }
    }
  }
}

template <class T>
int launch_rope(const sesa_rope_args& a, const RopePlan& pl, hipStream_t st) {
  const int64_t blocks = (a.tokens * pl.n_all * pl.hsplit + 255) / 256;
  SESA_REQUIRE(blocks < (1ll << 33), SESA_ERR_INVALID, "rope_axes: too many tokens");
  if (a.layout == SESA_ROPE_PAIRS)
    hipLaunchKernelGGL((rope_axes_kernel<T, true>), long_grid(blocks), dim3(256), 0, st, a, pl);
  else
    hipLaunchKernelGGL((rope_axes_kernel<T, false>), long_grid(blocks), dim3(256), 0, st, a, pl);
  SESA_CHECK_LAUNCH();
  return SESA_OK;
}

}  // namespace
}  // namespace sesa

using namespace sesa;

extern "C" int sesa_rope_axes(const sesa_rope_args* args, void* stream) {
  clear_error();
  SESA_REQUIRE(args, SESA_ERR_INVALID, "rope_axes: null arguments");
  const sesa_rope_args& a = *args;
  SESA_REQUIRE(a.tokens >= 0 && a.tokens < (1ll << 31), SESA_ERR_INVALID, "rope_axes: tokens %lld", (long long)a.tokens);
  SESA_REQUIRE(a.head_dim >= 2 && a.head_dim <= 4096, SESA_ERR_INVALID, "rope_axes: head_dim %d (2..4096)", a.head_dim);
  SESA_REQUIRE(a.layout == SESA_ROPE_HALVES || a.layout == SESA_ROPE_PAIRS, SESA_ERR_INVALID, "rope_axes: layout %d",
               a.layout);
  SESA_REQUIRE(a.n_axes >= 1 && a.n_axes <= 4, SESA_ERR_INVALID, "rope_axes: n_axes %d (1..4)", a.n_axes);
  SESA_REQUIRE(a.n_tensors == 1 || a.n_tensors == 2, SESA_ERR_INVALID, "rope_axes: n_tensors %d", a.n_tensors);
  int64_t P = 0;
  for (int i = 0; i < a.n_axes; ++i) {
    SESA_REQUIRE(a.sections[i] >= 0, SESA_ERR_INVALID, "rope_axes: sections[%d] = %d", i, a.sections[i]);
    P += a.sections[i];
  }
  SESA_REQUIRE(P >= 1 && 2 * P <= a.head_dim, SESA_ERR_INVALID, "rope_axes: %lld pairs in a head of %d", (long long)P,
               a.head_dim);
  int heads = 0;
  for (int k = 0; k < a.n_tensors; ++k) {
    SESA_REQUIRE(a.t[k].heads >= 1 && a.t[k].heads <= 65536, SESA_ERR_INVALID, "rope_axes: tensor %d has %d heads", k,
                 a.t[k].heads);
    SESA_REQUIRE(a.tokens == 0 || (a.t[k].x && a.t[k].out), SESA_ERR_INVALID, "rope_axes: tensor %d is null", k);
    heads = std::max(heads, a.t[k].heads);
  }
  if (a.tokens == 0) return SESA_OK;
  SESA_REQUIRE(a.positions && a.freqs, SESA_ERR_INVALID, "rope_axes: null positions or freqs");
  sesa_rope_args b = a;
  for (int i = a.n_axes; i < 4; ++i) b.sections[i] = 0;
  RopePlan pl{};
  pl.P = (int)P;
  pl.n_rot = (pl.P + kPairs - 1) / kPairs;
  pl.n_all = pl.n_rot + (a.head_dim - 2 * pl.P + 15) / 16;
  // heads over enough threads that the chip is busy (256 CUs x 2048 threads), no more than there are
  const int64_t want = (256 * 2048 + a.tokens * pl.n_all - 1) / (a.tokens * pl.n_all);
  pl.hsplit = (int)std::min<int64_t>(heads, std::max<int64_t>(1, want));
  hipStream_t st = as_stream(stream);
  if (a.dtype == SESA_DTYPE_F32) return launch_rope<float>(b, pl, st);
  if (a.dtype == SESA_DTYPE_F16) return launch_rope<f16>(b, pl, st);
  SESA_REQUIRE(a.dtype == SESA_DTYPE_BF16, SESA_ERR_INVALID, "rope_axes: dtype %d", a.dtype);
  return launch_rope<__bf16>(b, pl, st);
}
