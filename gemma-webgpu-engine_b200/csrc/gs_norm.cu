// Residual + RMS norm with an 8-bit output (gs_rms_norm).
//
//   h = x + residual,  y = h · (Σh²/n + eps)^-1/2 · (offset + w),
//   e4m3: a = max(max|y|, 2^-64) per group, code = round(y · (448 / a)), scale = a / 448.
//
// One pass over the data: a row's threads keep its float32 h in registers between the sum
// of squares, the group maxima and the store, so each input is read once and each output
// written once (bf16 -> e4m3 with residual: 7 bytes an element; HBM-bound for many rows,
// launch latency for few).  Sums and maxima are float32; h is rounded only where it is
// stored to residual_out.
//
// Measured (8192 rows of 4096 bf16 with a residual, e4m3 by groups of 128): 47 us a call, 44 us on the device in a row, 5.0
// TB/s and more (0.76 of a copy's rate; the issue slots are the other bound); one row of 1536 1.8 us on the device, on the LM
// head's grid 2.3 us; 8192 rows of 1536 f32 to that grid 36.5 us, 5.5 TB/s.
#include <cmath>

#include "gs_device.cuh"
#include "gs_internal.cuh"
#include "gs_quant.cuh"
#include "../../include/gsampler.h"

namespace gs {
namespace {

struct NormArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* residual_out;
  void* out;
  float* out_scale;
  float* row_sum;
  int64_t rows;
  int64_t ld_x, ld_residual, ld_residual_out, ld_out;
  int32_t hidden;
  int32_t group;   // columns per scale (hidden when one scale a row)
  int32_t shift;   // log2(group) where a row has several scales
  int32_t groups;  // scales per row
  int32_t weight_bf16;
  float eps, offset, srq_scale, inv_hidden;
};

enum { kOutF32 = 0, kOutBf16 = 1, kOutE4m3 = 2, kOutSrq = 3 };

// Rows of V values by packed float32 pairs (the kernel is bound by issue slots, not by HBM, when its
// inputs are bf16).
template <int V>
__device__ __forceinline__ void add_row(float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) a[0] += b[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = __fadd2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      a[i] = r.x, a[i + 1] = r.y;
    }
}
template <int V>
__device__ __forceinline__ void mul_row(float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) a[0] *= b[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      a[i] = r.x, a[i + 1] = r.y;
    }
}
template <int V>
__device__ __forceinline__ void scale_row(float (&a)[V], float f) {
  float b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = f;
  mul_row(a, b);
}
template <int V>
__device__ __forceinline__ void square_row(const float (&a)[V], float2& s) {
  if constexpr (V == 1) s.x = fmaf(a[0], a[0], s.x);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 x = make_float2(a[i], a[i + 1]);
      s = __ffma2_rn(x, x, s);
    }
}
// x within [lo, hi]; a NaN stays one (fminf and fmaxf alone would make it a code like any other).
__device__ __forceinline__ float clamp_nan(float x, float lo, float hi) { return x != x ? x : fminf(fmaxf(x, lo), hi); }

template <int V>
__device__ __forceinline__ void load_weight(const NormArgs& A, int col, float (&w)[V]) {
  if (!A.weight) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 1.0f;
    return;
  }
  if (A.weight_bf16) load_row<V, true>(static_cast<const unsigned short*>(A.weight) + col, w);
  else load_row<V, false>(static_cast<const float*>(A.weight) + col, w);
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = A.offset;
  add_row(w, o);
}

// max of non-negative values over the warp: their bits in integer order are in value order, NaN above all.
__device__ __forceinline__ float warp_max_bits(float v) {
  return __int_as_float(__reduce_max_sync(kFullMask, __float_as_int(v) & 0x7fffffff));
}

// TPR = blockDim.x threads per row (a multiple of 32), blockDim.y rows per block; thread t
// holds the row's V-element pieces t, t + TPR, ...  V = 8: 16-byte (bf16) or two 16-byte
// (f32) accesses, all pointers and strides 16-byte aligned and hidden % 8 == 0; V = 1:
// any alignment and width.
template <bool BF16, int OUT, int V, int PIECES, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_kernel(const __grid_constant__ NormArgs A) {
  __shared__ float red[32];
  __shared__ float red2[32];
  extern __shared__ int gmax[];  // V = 1, several groups: [blockDim.y][groups] bits of max|y|
  const int t = threadIdx.x, tpr = blockDim.x, warps = tpr >> 5;
  const int wid = threadIdx.y * warps + (t >> 5), lane = t & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool live = row < A.rows;
  bool in[PIECES];  // whether this thread's pieces lie in the row
#pragma unroll
  for (int p = 0; p < PIECES; ++p) in[p] = live && (t + p * tpr) * V < A.hidden;
  using T = typename std::conditional<BF16, unsigned short, float>::type;
  float h[PIECES][V];
  float2 sq2 = make_float2(0.0f, 0.0f);
  if (live) {
    const T* x = static_cast<const T*>(A.x) + row * A.ld_x;
    const T* r = A.residual ? static_cast<const T*>(A.residual) + row * A.ld_residual : nullptr;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (t + p * tpr) * V;
      if (in[p]) load_row<V, BF16>(x + col, h[p]);
    }
    if (r) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int col = (t + p * tpr) * V;
        if (in[p]) {
          float b[V];
          load_row<V, BF16>(r + col, b);
          add_row(h[p], b);
        }
      }
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (t + p * tpr) * V;
      if (in[p]) {
        if (A.residual_out) store_row<V, BF16>(static_cast<T*>(A.residual_out) + row * A.ld_residual_out + col, h[p]);
        square_row(h[p], sq2);
      }
    }
  }
  float sq = warp_sum_f(sq2.x + sq2.y);
  if (warps > 1) {
    if (lane == 0) red[wid] = sq;
    __syncthreads();
    sq = warp_sum_f(lane < warps ? red[threadIdx.y * warps + lane] : 0.0f);
  }
  const float rstd = rsqrtf(sq * A.inv_hidden + A.eps);
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int col = (t + p * tpr) * V;
    if (in[p]) {
      float w[V];
      load_weight<V>(A, col, w);
      scale_row(h[p], rstd);
      mul_row(h[p], w);
    }
  }
  if constexpr (OUT == kOutF32 || OUT == kOutBf16) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (t + p * tpr) * V;
      if (in[p]) {
        using O = typename std::conditional<OUT == kOutBf16, unsigned short, float>::type;
        store_row<V, OUT == kOutBf16>(static_cast<O*>(A.out) + row * A.ld_out + col, h[p]);
      }
    }
  } else if constexpr (OUT == kOutSrq) {
    // (The sum of codes in float32: at most 2^15 codes of at most 2^7, exact in any order, and a NaN stays one.)
    float qs = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (t + p * tpr) * V;
      if (in[p]) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float q = clamp_nan(rintf(__fdiv_rn(h[p][i], A.srq_scale)), -128.0f, 127.0f);
          qs += q;
          o[i] = __fmul_rn(q, A.srq_scale);
        }
        store_row<V, false>(static_cast<float*>(A.out) + row * A.ld_out + col, o);
      }
    }
    qs = warp_sum_f(qs);
    if (warps > 1) {
      if (lane == 0) red2[wid] = qs;
      __syncthreads();
      qs = warp_sum_f(lane < warps ? red2[threadIdx.y * warps + lane] : 0.0f);
    }
    if (t == 0 && live && A.row_sum) A.row_sum[row] = __fmul_rn(qs, A.srq_scale);
  } else {
    unsigned char* out = static_cast<unsigned char*>(A.out) + row * A.ld_out;
    float* scales = A.out_scale + row * A.groups;
    float gm[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      gm[p] = 0.0f;
      const int col = (t + p * tpr) * V;
      if (in[p])
#pragma unroll
        for (int i = 0; i < V; ++i) gm[p] = max_nan(gm[p], fabsf(h[p][i]));
    }
    if (A.groups == 1) {
      float m = 0.0f;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) m = max_nan(m, gm[p]);
      m = warp_max_bits(m);
      if (warps > 1) {
        if (lane == 0) red2[wid] = m;
        __syncthreads();
        m = warp_max_bits(lane < warps ? red2[threadIdx.y * warps + lane] : 0.0f);
      }
#pragma unroll
      for (int p = 0; p < PIECES; ++p) gm[p] = m;
      if (t == 0 && live) scales[0] = quant_scale(m, kE4m3Max);
    } else if (V == 8) {
      // a group is group / 8 consecutive pieces, so as many neighbouring lanes (4, 8 or 16)
      const int span = A.group >> 3;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        gm[p] = max_nan(gm[p], __shfl_xor_sync(kFullMask, gm[p], 1));
        gm[p] = max_nan(gm[p], __shfl_xor_sync(kFullMask, gm[p], 2));
        if (span > 4) gm[p] = max_nan(gm[p], __shfl_xor_sync(kFullMask, gm[p], 4));
        if (span > 8) gm[p] = max_nan(gm[p], __shfl_xor_sync(kFullMask, gm[p], 8));
        const int col = (t + p * tpr) * V;
        if (col < A.hidden && live && (lane & (span - 1)) == 0)
          scales[col >> A.shift] = quant_scale(gm[p], kE4m3Max);
      }
    } else {
      int* gr = gmax + threadIdx.y * A.groups;
      for (int g = t; g < A.groups; g += tpr) gr[g] = 0;
      __syncthreads();
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        // a warp's 32 columns lie in one group (groups are multiples of 32 columns)
        const int col = t + p * tpr;
        const int m = __float_as_int(warp_max_bits(gm[p]));
        if (lane == 0 && col < A.hidden) atomicMax(gr + (col >> A.shift), m);
      }
      __syncthreads();
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int col = (t + p * tpr) * V;
        if (in[p]) gm[p] = __int_as_float(gr[col >> A.shift]);
      }
      if (live)
        for (int g = t; g < A.groups; g += tpr) scales[g] = quant_scale(__int_as_float(gr[g]), kE4m3Max);
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (t + p * tpr) * V;
      if (in[p]) {
        const float inv = quant_inv(gm[p], kE4m3Max);
        if constexpr (V == 8) {
          uint2 c;
          scale_row(h[p], inv);
          c.x = e4m3x4(h[p][0], h[p][1], h[p][2], h[p][3]);
          c.y = e4m3x4(h[p][4], h[p][5], h[p][6], h[p][7]);
          *reinterpret_cast<uint2*>(out + col) = c;
        } else {
          out[col] = static_cast<unsigned char>(e4m3x2(h[p][0] * inv, 0.0f) & 0xffu);
        }
      }
    }
  }
}

template <bool BF16, int OUT, int V>
cudaError_t launch_norm_v(const NormArgs& a, cudaStream_t st) {
  const int pieces = (a.hidden + V - 1) / V;
  int tpr = 32;
  // (one element a piece: blocks of 512 threads overlap better than of 1024: 4118 rows of 3834 f32 by groups of 128 22% less time,
  // 92 us, 8000 of 1111 9% less, but 20000 of 333 7% more)
  const int want = a.rows <= 296 ? 1 : V == 8 ? 2 : pieces > 512 ? 8 : 4;
  while (tpr < 1024 && tpr * want < pieces) tpr <<= 1;
  const int rpb = tpr >= 256 ? 1 : 256 / tpr;
  const int per = (pieces + tpr - 1) / tpr;
  const dim3 block(tpr, rpb);
  const unsigned grid = static_cast<unsigned>((a.rows + rpb - 1) / rpb);
  const size_t smem = (OUT == kOutE4m3 && V == 1 && a.groups > 1) ? sizeof(int) * rpb * a.groups : 0;
  const bool wide = tpr > 256;
  // (V = 8: at most 4096 pieces, so at most 2 a thread but for rows of 1024 threads; V = 1: at most 32768)
  auto run = [&](auto pieces_, auto threads_) {
    norm_kernel<BF16, OUT, V, decltype(pieces_)::value, decltype(threads_)::value><<<grid, block, smem, st>>>(a);
  };
  using std::integral_constant;
  constexpr integral_constant<int, 256> narrow{};
  constexpr integral_constant<int, 1024> most{};
  if (per <= 1 && !wide) run(integral_constant<int, 1>{}, narrow);
  else if (per <= 1) run(integral_constant<int, 1>{}, most);
  else if (per <= 2 && !wide) run(integral_constant<int, 2>{}, narrow);
  else if (per <= 2) run(integral_constant<int, 2>{}, most);
  else if constexpr (V == 8) run(integral_constant<int, 4>{}, most);
  else if (per <= 4 && !wide) run(integral_constant<int, 4>{}, narrow);
  else if (per <= 4) run(integral_constant<int, 4>{}, most);
  else if (per <= 8) run(integral_constant<int, 8>{}, most);
  else if (per <= 16) run(integral_constant<int, 16>{}, most);
  else run(integral_constant<int, 32>{}, most);
  return cudaGetLastError();
}

template <bool BF16, int OUT>
cudaError_t launch_norm_o(const NormArgs& a, bool vec, cudaStream_t st) {
  return vec ? launch_norm_v<BF16, OUT, 8>(a, st) : launch_norm_v<BF16, OUT, 1>(a, st);
}

template <bool BF16>
cudaError_t launch_norm(const NormArgs& a, int out, bool vec, cudaStream_t st) {
  switch (out) {
    case kOutF32: return launch_norm_o<BF16, kOutF32>(a, vec, st);
    case kOutBf16: return launch_norm_o<BF16, kOutBf16>(a, vec, st);
    case kOutE4m3: return launch_norm_o<BF16, kOutE4m3>(a, vec, st);
    default: return launch_norm_o<BF16, kOutSrq>(a, vec, st);
  }
}

gs_status nfail(gs_ctx* c, gs_status s, const char* m) {
  ctx_set_error(c, m);
  return s;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" gs_status gs_rms_norm(gs_ctx* ctx, const gs_rms_norm_args* p, void* stream) {
  if (!ctx || !p) return GS_EINVAL;
  if (p->rows < 0 || p->hidden <= 0) return nfail(ctx, GS_EINVAL, "RMS norm: rows >= 0 and hidden >= 1 are required");
  if (p->hidden > GS_MAX_NORM_HIDDEN) return nfail(ctx, GS_EUNSUPPORTED, "RMS norm: hidden is at most 32768");
  if (p->rows == 0) return GS_OK;
  if (p->rows > 0x7fffffffll) return nfail(ctx, GS_EUNSUPPORTED, "RMS norm: at most 2^31 - 1 rows");
  const bool in_ok = (p->dtype == GS_DTYPE_F32 || p->dtype == GS_DTYPE_BF16) &&
                     (!p->weight || p->weight_dtype == GS_DTYPE_F32 || p->weight_dtype == GS_DTYPE_BF16);
  if (!in_ok || (p->out_dtype != GS_DTYPE_F32 && p->out_dtype != GS_DTYPE_BF16 && p->out_dtype != GS_DTYPE_E4M3))
    return nfail(ctx, GS_EINVAL, "RMS norm: float32 or bfloat16 inputs and float32, bfloat16 or e4m3 output");
  if (!p->x || !p->out) return nfail(ctx, GS_EINVAL, "RMS norm: x and out are required");
  if (p->ld_x < p->hidden || p->ld_out < p->hidden || (p->residual && p->ld_residual < p->hidden) ||
      (p->residual_out && p->ld_residual_out < p->hidden))
    return nfail(ctx, GS_EINVAL, "RMS norm: row strides must be at least hidden");
  if (!(p->eps >= 0.0f) || !std::isfinite(p->eps) || !std::isfinite(p->weight_offset) || !(p->srq_scale >= 0.0f) ||
      !std::isfinite(p->srq_scale))
    return nfail(ctx, GS_EINVAL, "RMS norm: eps and srq_scale must be finite and >= 0, weight_offset finite");
  if (p->srq_scale != 0.0f && p->out_dtype != GS_DTYPE_F32)
    return nfail(ctx, GS_EINVAL, "RMS norm: srq_scale goes with a float32 output");
  if (p->group != 0 && p->group != 32 && p->group != 64 && p->group != 128)
    return nfail(ctx, GS_EINVAL, "RMS norm: group must be 0, 32, 64 or 128");
  if (p->out_dtype == GS_DTYPE_E4M3 && !p->out_scale) return nfail(ctx, GS_EINVAL, "RMS norm: out_scale is required");
  if (p->out_dtype != GS_DTYPE_E4M3 && p->group != 0)
    return nfail(ctx, GS_EINVAL, "RMS norm: groups go with an e4m3 output");
  NormArgs a{};
  a.x = p->x;
  a.residual = p->residual;
  a.weight = p->weight;
  a.residual_out = p->residual_out;
  a.out = p->out;
  a.out_scale = p->out_scale;
  a.row_sum = p->row_sum;
  a.rows = p->rows;
  a.ld_x = p->ld_x;
  a.ld_residual = p->ld_residual;
  a.ld_residual_out = p->ld_residual_out;
  a.ld_out = p->ld_out;
  a.hidden = static_cast<int32_t>(p->hidden);
  a.group = p->group ? p->group : a.hidden;
  a.groups = (a.hidden + a.group - 1) / a.group;
  a.shift = p->group == 32 ? 5 : p->group == 64 ? 6 : 7;
  a.weight_bf16 = p->weight_dtype == GS_DTYPE_BF16;
  a.eps = p->eps;
  a.offset = p->weight_offset;
  a.srq_scale = p->srq_scale;
  a.inv_hidden = static_cast<float>(1.0 / static_cast<double>(p->hidden));
  // 16-byte accesses need every row to start on 16 bytes (8 for codes) and whole pieces
  auto fits = [&](const void* ptr, int64_t ld, int dtype) {
    if (!ptr) return true;
    const int64_t e = dtype == GS_DTYPE_F32 ? 4 : dtype == GS_DTYPE_BF16 ? 2 : 1;
    const uintptr_t al = dtype == GS_DTYPE_E4M3 ? 8 : 16;
    return reinterpret_cast<uintptr_t>(ptr) % al == 0 && (p->rows == 1 || (ld * e) % static_cast<int64_t>(al) == 0);
  };
  const bool vec = p->hidden % 8 == 0 && fits(p->x, p->ld_x, p->dtype) && fits(p->residual, p->ld_residual, p->dtype) &&
                   fits(p->residual_out, p->ld_residual_out, p->dtype) && fits(p->out, p->ld_out, p->out_dtype) &&
                   fits(p->weight, p->hidden, p->weight_dtype);
  const int out = p->srq_scale != 0.0f ? kOutSrq : p->out_dtype == GS_DTYPE_E4M3 ? kOutE4m3
                  : p->out_dtype == GS_DTYPE_BF16 ? kOutBf16 : kOutF32;
  DeviceScope scope(ctx_device(ctx));
  const cudaError_t e = p->dtype == GS_DTYPE_BF16 ? launch_norm<true>(a, out, vec, static_cast<cudaStream_t>(stream))
                                                  : launch_norm<false>(a, out, vec, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return nfail(ctx, GS_ECUDA, cudaGetErrorString(e));
  return GS_OK;
}
