// Device helpers shared by the sampler kernels.
//
// Everything here that decides an ordering or a token is exact IEEE arithmetic written
// with explicit round-to-nearest intrinsics (__fmul_rn, __dadd_rn, ...), so nvcc's
// default FMA contraction cannot change a rounding the reference's JavaScript performs.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>

namespace gs {

constexpr uint32_t kFullMask = 0xffffffffu;

// ----------------------------------------------------------------------------------
// Logit soft cap: c·tanh(x/c) in float32, stated as a fixed sequence of IEEE single
// operations so that host and device produce identical bits.  The reference runtime
// declares the Gemma final-logit cap (30) but never applies it; the benchmark inputs
// are specified with it applied, so it is an option of the streaming pass (0 = off).
// Method: y = x·fl(1/c), z = fl(y²).  z < 1 (|y| < 1, so |x| < c): odd polynomial
// c·(y + y·z·Q(z)) on the signed y, Q of degree 6 (least-squares / Lawson minimax fit of
// tanh, csrc/derive_softcap.py; 0.93 ulp against tanh(y)).  Otherwise
// t = 1 − 2/(e^{2|y|} + 1) for |y| < 9 (e^z by Cody–Waite reduction z = n·ln2 + r and a
// degree-6 polynomial for e^r), t = 1 above, and the result is c·copysign(t, y).  Over
// every float32 input the result is monotone and within 3.2 ulp of c·tanh(x/c) (most of
// it from rounding x·fl(1/c)); the oracle's tests check both exhaustively.
// ----------------------------------------------------------------------------------
__device__ __forceinline__ float softcap_exp_reduced(float z) {
  const float n = rintf(__fmul_rn(z, 1.44269502162933349609375f));
  float r = __fmaf_rn(-n, 0.693145751953125f, z);
  r = __fmaf_rn(-n, 1.428606765330187e-06f, r);
  float p = 0.00138142f;
  p = __fmaf_rn(p, r, 0.00836891f);
  p = __fmaf_rn(p, r, 0.04166841f);
  p = __fmaf_rn(p, r, 0.1666652f);
  p = __fmaf_rn(p, r, 0.49999994f);
  const float r2 = __fmul_rn(r, r);
  const float e = __fadd_rn(__fmaf_rn(p, r2, r), 1.0f);
  const int ni = static_cast<int>(n);
  const float scale = __uint_as_float(static_cast<uint32_t>(ni + 127) << 23);
  return __fmul_rn(e, scale);
}

// |y| >= 1 branch of softcap (|x| >= c), kept out of line so the streaming loops stay small.
static __device__ __noinline__ float softcap_tail(float a) {
  if (a < 9.0f) {
    const float e = softcap_exp_reduced(__fadd_rn(a, a));
    return __fsub_rn(1.0f, __fdiv_rn(2.0f, __fadd_rn(e, 1.0f)));
  }
  return 1.0f;
}

// Polynomial branch, evaluated on the signed y: c·fma(y·z, Q(z), y) with z = fl(y²)
// (a zero y gives +0).  z < 1 exactly when |y| < 1 (the largest float below 1 squares
// to 1 − 2^-23).
constexpr float kSoftcapPolyZ = 1.0f;

// log2(e) as a float pair (hi + lo): e^d = 2^(d·hi + d·lo) with the product's error
// carried by the second term.
constexpr float kL2eHi = 1.44269502162933349609375f;
constexpr float kL2eLo = 1.925963033500011e-08f;
#define GS_SOFTCAP_Q6 -0.00035845203f
#define GS_SOFTCAP_Q5 0.0023013647f
#define GS_SOFTCAP_Q4 -0.007946107f
#define GS_SOFTCAP_Q3 0.021486657f
#define GS_SOFTCAP_Q2 -0.0538798f
#define GS_SOFTCAP_Q1 0.13332345f
#define GS_SOFTCAP_Q0 -0.33333296f
__device__ __forceinline__ float softcap_poly_q(float z) {
  float q = GS_SOFTCAP_Q6;
  q = __fmaf_rn(q, z, GS_SOFTCAP_Q5);
  q = __fmaf_rn(q, z, GS_SOFTCAP_Q4);
  q = __fmaf_rn(q, z, GS_SOFTCAP_Q3);
  q = __fmaf_rn(q, z, GS_SOFTCAP_Q2);
  q = __fmaf_rn(q, z, GS_SOFTCAP_Q1);
  return __fmaf_rn(q, z, GS_SOFTCAP_Q0);
}

__device__ __forceinline__ float softcap(float x, float cap, float inv_cap) {
  const float y = __fmul_rn(x, inv_cap);
  const float z = __fmul_rn(y, y);
  if (z < kSoftcapPolyZ) return __fmul_rn(cap, __fmaf_rn(__fmul_rn(y, z), softcap_poly_q(z), y));
  if (x != x) return x;
  return __fmul_rn(cap, copysignf(softcap_tail(fabsf(y)), y));
}

// Polynomial branch for two values at once with packed float32 arithmetic (sm_100
// f32x2), the same IEEE operations as softcap() per component.  Returns the squares in
// *z so the caller can check the range (z < kSoftcapPolyZ) for a whole tile at once and
// redo the values outside it with softcap().
__device__ __forceinline__ float2 softcap2_poly(float2 x, float cap, float inv_cap, float2* zout) {
  const float2 y = __fmul2_rn(x, make_float2(inv_cap, inv_cap));
  const float2 z = __fmul2_rn(y, y);
  float2 q = make_float2(GS_SOFTCAP_Q6, GS_SOFTCAP_Q6);
  q = __ffma2_rn(q, z, make_float2(GS_SOFTCAP_Q5, GS_SOFTCAP_Q5));
  q = __ffma2_rn(q, z, make_float2(GS_SOFTCAP_Q4, GS_SOFTCAP_Q4));
  q = __ffma2_rn(q, z, make_float2(GS_SOFTCAP_Q3, GS_SOFTCAP_Q3));
  q = __ffma2_rn(q, z, make_float2(GS_SOFTCAP_Q2, GS_SOFTCAP_Q2));
  q = __ffma2_rn(q, z, make_float2(GS_SOFTCAP_Q1, GS_SOFTCAP_Q1));
  q = __ffma2_rn(q, z, make_float2(GS_SOFTCAP_Q0, GS_SOFTCAP_Q0));
  const float2 t = __ffma2_rn(__fmul2_rn(y, z), q, y);
  *zout = z;
  return __fmul2_rn(make_float2(cap, cap), t);
}

// Two soft caps at once; components outside the polynomial range take softcap().
__device__ __forceinline__ float2 softcap2(float2 x, float cap, float inv_cap) {
  float2 z;
  const float2 r = softcap2_poly(x, cap, inv_cap, &z);
  if (!(z.x < kSoftcapPolyZ && z.y < kSoftcapPolyZ)) return make_float2(softcap(x.x, cap, inv_cap), softcap(x.y, cap, inv_cap));
  return r;
}

// max that propagates NaN (PTX max.NaN)
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// ----------------------------------------------------------------------------------
// Ordered keys.  key32(x) is monotone in the float value (−inf lowest, NaN excluded by
// the callers).  A candidate "pack" puts key32 in the high word and ~id in the low word,
// so larger pack == earlier in the reference's sort order (logit descending, lower id
// first on ties: Array.prototype.sort is stable over ids in ascending order,
// src/runtime/sampling.ts:33-35).
// ----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t key32(float x) {
  // -0 and +0 compare equal in the reference's comparator (ties then go by id): +0 both
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key32_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ uint64_t make_pack(float x, uint32_t id) {
  return (static_cast<uint64_t>(key32(x)) << 32) | static_cast<uint64_t>(~id);
}
__device__ __forceinline__ uint32_t pack_id(uint64_t p) { return ~static_cast<uint32_t>(p); }
__device__ __forceinline__ float pack_value(uint64_t p) { return key32_value(static_cast<uint32_t>(p >> 32)); }

// Monotone map of a double onto uint64 (used to sort exact double keys).
__device__ __forceinline__ uint64_t key64(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x));
  return (b & 0x8000000000000000ull) ? ~b : (b | 0x8000000000000000ull);
}

// ----------------------------------------------------------------------------------
// SeededRandom (src/runtime/sampling.ts:3-16).  The reference keeps its state in a JS
// number that grows by 0x6d2b79f5 per draw without wrapping; every use converts it with
// ToUint32.  The state is kept as that same double here, so the stream matches the
// reference for any number of draws (the double stops being exact after ~4.9e6 draws
// in both).
// ----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t js_to_uint32(double v) {
  const double m = fmod(v, 4294967296.0);
  const double w = m < 0 ? __dadd_rn(m, 4294967296.0) : m;
  return static_cast<uint32_t>(static_cast<unsigned long long>(w));
}
__device__ __forceinline__ double seeded_next(double* state) {
  *state = __dadd_rn(*state, 1831565813.0);
  uint32_t v = js_to_uint32(*state);
  v = (v ^ (v >> 15)) * (v | 1u);
  v ^= v + (v ^ (v >> 7)) * (v | 61u);
  return __ddiv_rn(static_cast<double>(v ^ (v >> 14)), 4294967296.0);
}

// ----------------------------------------------------------------------------------
// Streaming loads (read once: do not keep in L1).
// ----------------------------------------------------------------------------------
__device__ __forceinline__ float4 ld_stream_f4(const float4* p) {
  float4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ld_stream_u4(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ float load_logit(const void* base, int dtype, int64_t idx) {
  if (dtype == 0) return __ldg(static_cast<const float*>(base) + idx);
  const uint16_t h = __ldg(static_cast<const unsigned short*>(base) + idx);
  return __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// 2^x (hardware approximation, flush-to-zero; 2^-inf = 0).
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ----------------------------------------------------------------------------------
// TMA bulk copy global -> shared (no multicast) completing on an mbarrier.
// ----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count));
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_g2s(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void bulk_g2s_addr(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
      "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ uint64_t globaltimer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
constexpr uint64_t kWaitNs = 1000000000ull;  // 1 s bound on every device-side wait
// Bounded wait on phase `parity`; returns false when `limit_ns` of wall time ran out.
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    if (mbar_try(bar, parity)) return true;
    if (globaltimer_ns() - t0 > limit_ns) return false;
  }
}

// Warp / block reductions.
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __dadd_rn(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}
__device__ __forceinline__ int warp_sum_i(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

}  // namespace gs
