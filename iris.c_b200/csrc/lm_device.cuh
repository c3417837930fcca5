// What the kernels of the language-model operators share: conversions, matrix
// and copy instructions, the order of a row's values, guarded loads of a row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include "iris_cuda.h"

namespace {

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void mma_bf16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same onto nothing
__device__ __forceinline__ void mma_bf16_first(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void mma_f16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// an 8 x 8 matrix of 16-bit values over the warp, rows in the lanes' fours, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint32_t pack2h(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// four e4m3 as two pairs of f16, exactly
__device__ __forceinline__ void e4m3_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// 2^(e - 127) for a scale's exponent e, which is held to the range that the formats here have
__device__ __forceinline__ int exp8(uint32_t e) { return min(max((int)e, IRIS_EXP8_MIN), IRIS_EXP8_MAX); }
__device__ __forceinline__ float scale8(int e) { return __int_as_float(e << 23); }

// 16 bytes, or zeros where `bytes` is 0 (nothing is read then)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Order of the alternatives: larger values first, equal ones by id, NaN before
// all; as one whole number a value, larger first, 0 for none.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  if (x != x) return 0xFF800001u;  // one above +inf
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float rank_value(uint32_t r) { return __uint_as_float(r & 0x80000000u ? r & 0x7FFFFFFFu : ~r); }
__device__ __forceinline__ uint64_t place(uint32_t rank, uint32_t id) { return (uint64_t)rank << 32 | (uint32_t)~id; }

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The values at [e, e + kVec) of a row of `vocab` <= 2^30 values, 16-byte
// aligned; -inf where the row has none.  Nothing outside the row is read.
template <typename In>
__device__ __forceinline__ uint4 row_vec(const In* x, int e, int vocab) {
  constexpr int VEC = 16 / sizeof(In);
  if (e >= 0 && e + VEC <= vocab) return __ldg(reinterpret_cast<const uint4*>(x + e));
  uint32_t w[4];
  if (e >= vocab || e + VEC <= 0) {
    w[0] = sizeof(In) == 4 ? 0xFF800000u : 0xFF80FF80u;
    return make_uint4(w[0], w[0], w[0], w[0]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(In) == 4) {
      w[i] = e + i >= 0 && e + i < vocab ? __float_as_uint(x[e + i]) : 0xFF800000u;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
      const uint32_t lo = e + 2 * i >= 0 && e + 2 * i < vocab ? h[e + 2 * i] : 0xFF80u;
      const uint32_t hi = e + 2 * i + 1 >= 0 && e + 2 * i + 1 < vocab ? h[e + 2 * i + 1] : 0xFF80u;
      w[i] = lo | hi << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename In>
__device__ __forceinline__ void vec_values(uint4 u, float x[16 / sizeof(In)]) {
  if constexpr (sizeof(In) == 4) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  } else {
    const float2 a = unpack2(u.x), b = unpack2(u.y), c = unpack2(u.z), d = unpack2(u.w);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
  }
}

// The largest of the values, NaN if one is.
template <typename In>
__device__ __forceinline__ float vec_max(uint4 u) {
  if constexpr (sizeof(In) == 4) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)),
                   max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else {
    auto h = [](uint32_t v) { return *reinterpret_cast<__nv_bfloat162*>(&v); };
    const __nv_bfloat162 v = __hmax2_nan(__hmax2_nan(h(u.x), h(u.y)), __hmax2_nan(h(u.z), h(u.w)));
    return max_nan(__low2float(v), __high2float(v));
  }
}

// First value of block 0 before the row's first one: blocks are cut at 16-byte boundaries.
template <typename In>
__device__ __forceinline__ int row_offset(const In* x) {
  return (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(In));
}

}  // namespace
