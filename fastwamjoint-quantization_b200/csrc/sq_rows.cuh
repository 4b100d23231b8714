// Row helpers shared by the block-norm, e4m3 quantizer and rotary kernels: 8-element vectors of bf16 / fp16 / fp32, e4m3
// conversion with the scale of a run of 128, GELU.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sq {

constexpr float kE4M3Max = 448.0f;      // largest finite e4m3 value
constexpr float kSmallestScale = 1e-8f; // floor of a scale: an all-zero run gets zero codes, not 0 / 0

__device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8], const __half*) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8], const __nv_bfloat16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8], const __half*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// data read once: past the L1, so that the parameter rows every token rereads stay there
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// 8 parameters, in the rows' type or in fp32: 32 bytes in one load, which the host checks the alignment for (two loads of 16
// bytes: 237 us instead of 227 for the norms of 32768 x 4096 with fp32 modulation)
template <typename T>
__device__ __forceinline__ void load_params(const void* base, int64_t index, bool f32, float (&v)[8]) {
  if (f32) {
    asm("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
        : "l"(static_cast<const float*>(base) + index));
  } else {
    unpack8(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(base) + index)), v, static_cast<const T*>(nullptr));
  }
}

// Largest magnitude as an integer: magnitudes order like their bit patterns, and - unlike fmaxf - a NaN stays on top,
// so a run that holds one gets a NaN scale and its row comes out NaN instead of silently finite.
__device__ __forceinline__ uint32_t magnitude8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// Scale of a run of 128 from its largest magnitude: amax / 448, both divisions IEEE.  NaN stays NaN.
__device__ __forceinline__ float e4m3_scale(uint32_t magnitude) {
  const float s = __fdiv_rn(__uint_as_float(magnitude), kE4M3Max);
  return s < kSmallestScale ? kSmallestScale : s;
}

// Four floats -> four e4m3 codes, round to nearest even, saturating (NaN gives the NaN code).
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// Codes of 8 elements given the run's scale: x * (1 / s), one reciprocal per run.
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float inverse) {
  return make_uint2(pack_e4m3x4(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                    pack_e4m3x4(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse));
}

// Largest magnitude over the 16 lanes (8 elements each) that hold a run of 128.
__device__ __forceinline__ uint32_t run_max(uint32_t m) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}

// Two fp32 values in one register pair: one instruction for both products or sums.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  return static_cast<uint64_t>(__float_as_uint(lo)) | (static_cast<uint64_t>(__float_as_uint(hi)) << 32);
}
__device__ __forceinline__ float low2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, float c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(pack2(c, c)));
  return d;
}

// erf GELU, x * Phi(x), of 8 values.  With a = |x| and t = 1 / (1 + 0.306 a):
//   x * Phi(x) = (x < 0 ? 0 : x) - a * Phi(-a),   a * Phi(-a) = a * t * exp(-a^2 / 2) * P(t)
// Phi(-a) exp(a^2 / 2) is smooth in t over all of 0 .. 1, so one polynomial serves every x; P was fitted to the function in
// 64 bits for the least relative error (1.1e-7).  In fp32 the whole is within 5e-7 of its value down to x = -3 and 2e-6
// to -8: unlike x / 2 * (1 + erf(x / sqrt 2)) nothing cancels where x is negative.  The quantizer is bound by its issue
// slots with the activation (20.0 us for 1592 x 12288, 11.6 without): with erff it took 28.7, with this one value at a time
// 22.0, with one reciprocal for four values 21.3.
__device__ __forceinline__ void gelu8(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t a = pack2(fminf(fabsf(v[i]), 64.0f), fminf(fabsf(v[i + 1]), 64.0f));  // 64: infinity times zero stays out
    const uint64_t d = fma2(a, pack2(0.306f, 0.306f), 1.0f);
    const uint64_t power = mul2(mul2(a, a), pack2(-0.72134752044448170f, -0.72134752044448170f));  // -log2(e) / 2
    float t0, t1, e0, e1;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(low2(d)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(high2(d)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(low2(power)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(high2(power)));
    const uint64_t t = pack2(t0, t1);
    uint64_t p = fma2(t, pack2(0.036538217f, 0.036538217f), -0.15070112f);
    p = fma2(p, t, 0.17938644f);
    p = fma2(p, t, -0.033036616f);
    p = fma2(p, t, 0.11862919f);
    p = fma2(p, t, 0.10436764f);
    p = fma2(p, t, 0.122772194f);
    p = fma2(p, t, 0.1220441f);
    const uint64_t h = mul2(mul2(mul2(a, t), pack2(e0, e1)), p);
    v[i] = fmaf(v[i], v[i] < 0.0f ? 0.0f : 1.0f, -low2(h));  // x * 0, not 0: -infinity gives NaN as the formula does
    v[i + 1] = fmaf(v[i + 1], v[i + 1] < 0.0f ? 0.0f : 1.0f, -high2(h));
  }
}

inline bool aligned16_host(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// a vector of 8 parameters: 16 bytes, 32 in fp32
inline bool aligned_param_host(const void* p, bool f32) { return (reinterpret_cast<uintptr_t>(p) & (f32 ? 31u : 15u)) == 0; }

}  // namespace sq
