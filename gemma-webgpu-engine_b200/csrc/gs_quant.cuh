// Row loads and stores, and the 8-bit codes of the norm's output and the key/value cache.
#pragma once
#include <type_traits>

#include "gs_device.cuh"

namespace gs {

constexpr float kE4m3Max = 448.0f;
constexpr float kInt8Max = 127.0f;
// Floor of a group's largest magnitude: a group of zeros gets this scale and zero codes.
constexpr float kQuantTiny = 5.421010862427522e-20f;  // 2^-64

// max(a, tiny) that keeps a NaN, then the scale a / M and the factor M / a of the codes.
__device__ __forceinline__ float quant_floor(float a) { return max_nan(a, kQuantTiny); }
__device__ __forceinline__ float quant_scale(float a, float most) { return __fdiv_rn(quant_floor(a), most); }
__device__ __forceinline__ float quant_inv(float a, float most) { return __fdiv_rn(most, quant_floor(a)); }

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// Two values as e4m3 codes, lo in the low byte (round to nearest even, saturating).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
// Two e4m3 codes (low 16 bits) as a half pair, exact.
__device__ __forceinline__ uint32_t e4m3x2_half2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(codes)));
  return r;
}
__device__ __forceinline__ float2 half2_float2(uint32_t h) {
  float2 f;
  asm("{\n .reg .b16 l, u;\n mov.b32 {l, u}, %2;\n cvt.f32.f16 %0, l;\n cvt.f32.f16 %1, u;\n}\n"
      : "=f"(f.x), "=f"(f.y)
      : "r"(h));
  return f;
}
// Four int8 codes, a in the low byte (round to nearest even; NaN gives 0).
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
  const uint32_t x = static_cast<uint32_t>(__float2int_rn(a)) & 0xffu, y = static_cast<uint32_t>(__float2int_rn(b)) & 0xffu;
  const uint32_t z = static_cast<uint32_t>(__float2int_rn(c)) & 0xffu, w = static_cast<uint32_t>(__float2int_rn(d)) & 0xffu;
  return x | (y << 8) | (z << 16) | (w << 24);
}
// bf16 pair of two floats (round to nearest even), lo in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// V consecutive elements (float32, or bf16 as unsigned short) as float32.
template <int V, bool BF16>
__device__ __forceinline__ void load_row(const void* p, float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (BF16) v[0] = __uint_as_float(static_cast<uint32_t>(*static_cast<const unsigned short*>(p)) << 16);
    else v[0] = *static_cast<const float*>(p);
  } else if constexpr (BF16) {
    static_assert(V == 8, "one 16-byte access");
    const uint4 u = *static_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    }
  } else {
    static_assert(V == 8, "two 16-byte accesses");
    const float4 a = static_cast<const float4*>(p)[0], b = static_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}
template <int V, bool BF16>
__device__ __forceinline__ void store_row(void* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (BF16) *static_cast<unsigned short*>(p) = static_cast<unsigned short>(bf16x2(v[0], 0.0f) & 0xffffu);
    else *static_cast<float*>(p) = v[0];
  } else if constexpr (BF16) {
    *static_cast<uint4*>(p) = make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
  } else {
    static_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    static_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// Makes `d` the current device for the scope of a host call.
struct DeviceScope {
  int prev = -1, dev;
  explicit DeviceScope(int d) : dev(d) {
    cudaGetDevice(&prev);
    if (prev != d) cudaSetDevice(d);
  }
  ~DeviceScope() {
    if (prev >= 0 && prev != dev) cudaSetDevice(prev);
  }
};

}  // namespace gs
