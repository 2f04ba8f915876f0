// Shared device helpers of the transformer operators (sesa_norm / sesa_rope / sesa_linear_i8 / sesa_attn_packed).
#pragma once
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdint>

#include "sesa_common.hpp"

namespace sesa {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any address: the rows of the public operators start where the caller's strides put them, and gfx950
// loads and stores a dwordx4 at any byte (one instruction; only the cache lines it touches count).
struct __attribute__((packed)) Bytes16 {
  u32x4 v;
};

__device__ __forceinline__ u32x4 load16(const void* p) { return reinterpret_cast<const Bytes16*>(p)->v; }
__device__ __forceinline__ void store16(void* p, u32x4 v) { reinterpret_cast<Bytes16*>(p)->v = v; }

// Eight consecutive elements of a row as fp32; `left` = elements of the row from here on (<= 0: none).  Whole groups
// take vector loads, a row's last partial group goes element by element (zero past its end).
template <class T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      // (whole vectors: a bit cast of one vector element reads element 0 whatever the index is)
      const f32x4 a = __builtin_bit_cast(f32x4, load16(p)), b = __builtin_bit_cast(f32x4, load16(p + 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
      const u32x4 a = load16(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = (float)__builtin_bit_cast(T, (uint16_t)(a[e] & 0xffffu));
        v[2 * e + 1] = (float)__builtin_bit_cast(T, (uint16_t)(a[e] >> 16));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? (float)p[e] : 0.f;
  }
}

// two fp32 values rounded to nearest even in one 32-bit word (one v_cvt_pk on gfx950)
template <class T>
__device__ __forceinline__ uint32_t pack2t(float a, float b) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, t2));
}

template <class T>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      u32x4 a, b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = __builtin_bit_cast(uint32_t, v[e]);
        b[e] = __builtin_bit_cast(uint32_t, v[4 + e]);
      }
      store16(p, a);
      store16(p + 4, b);
    } else {
      store16(p, u32x4{pack2t<T>(v[0], v[1]), pack2t<T>(v[2], v[3]), pack2t<T>(v[4], v[5]), pack2t<T>(v[6], v[7])});
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) p[e] = (T)v[e];
  }
}

// 16 bytes a lane from anywhere to LDS at the (wave-uniform) base + 16 * lane, counted by vmcnt.  A function of its own:
// inside a template's lambda the host pass drops the kernel's launch stub over the builtin.
__device__ __forceinline__ void dma16(const void* src, char* base) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)base, 16, 0, 0);
}

// The same by an asm statement, for kernels that also use the transposing LDS reads: the compiler takes those for stores
// too and would wait for every load in flight before each.  No registers are written; the kernel waits on vmcnt itself.
__device__ __forceinline__ void dma16_asm(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

// Exact (erf) GELU as max(v, 0) - |v| erfc(|v| / sqrt 2) / 2 -- both signs in one expression, no select --
// with erfc(z) = t P4(t) exp(-z^2), t = 1 / (1 + p z) (Abramowitz & Stegun 7.1.26, |error| < 1.5e-7, the 1 / 2 in the
// coefficients).  19 VALU slots where Phi(v) by a select takes 24: the 8-bit Linear's epilogue is bound by them.
__device__ __forceinline__ float gelu_f(float v) {
  const float z = fabsf(v);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752440f, z, 1.0f));
  float p = 0.5f * 1.061405429f;
  p = fmaf(p, t, 0.5f * -1.453152027f);
  p = fmaf(p, t, 0.5f * 1.421413741f);
  p = fmaf(p, t, 0.5f * -0.284496736f);
  p = fmaf(p, t, 0.5f * 0.254829592f);
  const float w = v * 0.84932180028801904272f;   // sqrt(log2(e) / 2): exp(-v^2 / 2) = exp2(-w^2)
  const float q = p * t * __builtin_amdgcn_exp2f(-(w * w));
  return fmaf(-fminf(z, 1e30f), q, fmaxf(v, 0.f));   // (the minimum: an infinity times its tail of 0)
}

// The same to fp32: erfc(z) = t P7(t) exp(-z^2), t = 1 / (1 + 0.44 z), P fitted here to the least relative error on z in
// [0, 10], 1.8e-7 (the 1 / 2 in the coefficients).  rms error on [-8, 8] 5.2e-8, which is the result's own rounding; three
// operations more than gelu_f.
__device__ __forceinline__ float gelu_fine_f(float v) {
  const float z = fabsf(v);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.44f * 0.70710678118654752440f, z, 1.0f));
  float p = 0.0356115793f;
  p = fmaf(p, t, -0.13897336f);
  p = fmaf(p, t, 0.148342622f);
  p = fmaf(p, t, -0.0100893122f);
  p = fmaf(p, t, 0.107905584f);
  p = fmaf(p, t, 0.108656933f);
  p = fmaf(p, t, 0.124435566f);
  p = fmaf(p, t, 0.124110478f);
  const float w = v * 0.84932180028801904272f;
  const float q = p * t * __builtin_amdgcn_exp2f(-(w * w));
  return fmaf(-fminf(z, 1e30f), q, fmaxf(v, 0.f));
}

// Workgroup barrier behind this wave's own LDS operations that leaves loads to LDS in flight: __syncthreads() would wait
// for all of them, whatever stage they are for.  A kernel that uses it waits on vmcnt for the stage it is about to read.
__device__ __forceinline__ void stage_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Larger of the two values that lanes l and l ^ 32 hold
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

__device__ __forceinline__ float sigmoid_f(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}
// tanh(v) = (1 - e) / (1 + e), e = exp(-2 |v|); below 0.09 the odd series to v^7 (next term 2^-26 relative there),
// where the quotient would cancel.
__device__ __forceinline__ float tanh_f(float v) {
  const float z = fabsf(v), e = __builtin_amdgcn_exp2f(-2.f * 1.4426950408889634f * z), s = v * v;
  const float big = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), v);
  const float small = v * fmaf(s, fmaf(s, fmaf(s, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  return z < 0.09f ? small : big;
}

// A 1-D grid of nb workgroups as a launch takes it (a dimension holds less than 2^32 threads): rows of 2^18 workgroups,
// and its workgroup number (nb and above: nothing to do).  The row length is a multiple of 8, so numbers keep their die.
inline dim3 long_grid(int64_t nb) {
  constexpr int64_t kRow = 1 << 18;
  return nb <= kRow ? dim3((unsigned)nb) : dim3((unsigned)kRow, (unsigned)((nb + kRow - 1) / kRow));
}
__device__ __forceinline__ int64_t long_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// Tile order of a 1-D grid: workgroup b of nb runs on die b % 8, so give each die one contiguous range of tiles (its
// own L2 then sees neighbouring tiles' operands).
__device__ __forceinline__ int die_tile(int b, int nb) {
  const int q = nb >> 3, r = nb & 7, x = b & 7, i = b >> 3;
  return x * q + min(x, r) + i;
}

}  // namespace sesa
