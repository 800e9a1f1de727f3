// Paged key/value cache: handle, quantising write, read back, and the attention entry.
//
// write  a = max(max|x|, 2^-64) over head_dim, code = round(x · (M / a)), scale = a / M
// read   value = code · scale, rounded once
// A row (one token and head) is a few neighbouring lanes of 8 or 16 elements each, so its
// maximum is a shuffle reduction and every access is 16 bytes; one launch
// covers keys and values.  Both directions move 3 bytes an element (bf16 beside codes) and
// are bound by HBM for long chunks, by launch latency for one step.
//
// Measured (calls in a row, 16384 tokens of 8 heads of 128, bf16 outside): e4m3 or int8 22.5 us written, 20.5 us read back
// (4.5 and 5.0 TB/s, 0.69 and 0.76 of a copy's rate), bf16 25.1 and 25.2 us (5.3 TB/s, 0.82); 32768 tokens of 4 heads of 256
// read from e4m3: 35 us, 5.8 TB/s.  What holds the write back is the bytes in flight: two tokens a thread in 64 registers keep 42 % of
// the warps active.
#include <cmath>
#include <new>

#include "gs_attn.cuh"
#include "gs_overlap.h"

namespace gs {
namespace {

struct KvRowsArgs {
  KvPool kv;
  unsigned char* k;  // the caller's rows
  unsigned char* v;
  uint32_t k_token, k_head, v_token, v_head;  // elements
  const int32_t* slots;
  int64_t tokens;
  int64_t slots_end; // pages · page_size
  int32_t* flag;
};

struct SlotAt {
  int32_t page;
  int32_t off;
  bool ok;
};

__device__ __forceinline__ SlotAt slot_at(const KvRowsArgs& A, uint32_t token) {
  const int32_t s = __ldg(A.slots + token);
  SlotAt r;
  r.ok = s >= 0 && s < A.slots_end;
  if (s >= A.slots_end) atomicOr(A.flag, GS_KV_ERR_SLOT);
  r.page = r.ok ? s >> A.kv.page_shift : 0;
  r.off = r.ok ? s & ((1 << A.kv.page_shift) - 1) : 0;
  return r;
}

// Element offset of (token, head) in the caller's rows.
__device__ __forceinline__ uint64_t row_at(const KvRowsArgs& A, bool value, uint32_t token, uint32_t head) {
  return static_cast<uint64_t>(token) * (value ? A.v_token : A.k_token) + static_cast<uint64_t>(head) * (value ? A.v_head : A.k_head);
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
  if constexpr (VEC) {
    store_row<8, BF16>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y[1] = {x[i]};
      store_row<1, BF16>(static_cast<unsigned char*>(p) + i * (BF16 ? 2 : 4), y);
    }
  }
}

// Elements of a row per lane: eight beside a bf16 pool, else twice eight, half a row apart, so that neighbouring
// lanes' 16-byte pieces (8 of codes) are neighbours.
template <int FMT, bool VEC>
constexpr int row_piece() {
  return FMT == GS_DTYPE_BF16 || !VEC ? 8 : 16;
}

// A group of lanes takes the key and the value of U tokens (`step` apart) of one head, all loads together: one
// row keeps too few bytes in flight for a long chunk, and a step's few rows are better spread.  (The kernels
// are bound by issue slots about as much as by HBM: what a row costs beside its data is shared where it can be.)
template <int D, int FMT, bool BF16, bool VEC, int U>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvRowsArgs A, uint32_t step) {
  constexpr int E = row_piece<FMT, VEC>(), kLanes = D / E, kWords = E / (BF16 ? 8 : 4);
  const uint32_t row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const uint32_t token0 = row / static_cast<uint32_t>(A.kv.kv_heads);
  const int head = static_cast<int>(row - token0 * A.kv.kv_heads);
  const int at = (threadIdx.x % kLanes) * 8;
  uint4 raw[U][2][kWords];
  SlotAt s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t token = token0 + u * step;
    s[u] = SlotAt{0, 0, false};
    if (token0 < step && token < A.tokens) s[u] = slot_at(A, token);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) raw[u][v][i] = make_uint4(0u, 0u, 0u, 0u);
      if (!s[u].ok) continue;
      const unsigned char* src = (v ? A.v : A.k) + (row_at(A, v, token0 + u * step, head) + at) * (BF16 ? 2 : 4);
      if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          constexpr int kPer = BF16 ? 1 : 2;  // words of eight elements
          raw[u][v][i] = ld_stream_u4(reinterpret_cast<const uint4*>(src + (i / kPer) * (D / 2) * (BF16 ? 2 : 4)) + i % kPer);
        }
      } else if constexpr (BF16) {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(src);
        raw[u][v][0] = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
      } else {
        const uint32_t* h = reinterpret_cast<const uint32_t*>(src);
        raw[u][v][0] = make_uint4(h[0], h[1], h[2], h[3]);
        raw[u][v][kWords - 1] = make_uint4(h[4], h[5], h[6], h[7]);
      }
    }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float x[E];
#pragma unroll
      for (int i = 0; i < E / 8; ++i) load_row<8, BF16>(&raw[u][v][i * (BF16 ? 1 : 2)], *reinterpret_cast<float(*)[8]>(x + 8 * i));
      unsigned char* pool = const_cast<unsigned char*>(A.kv.at(v, s[u].page, head, s[u].off));
      if constexpr (FMT == GS_DTYPE_BF16) {
        if (s[u].ok) store_row<8, true>(pool + at * 2, *reinterpret_cast<float(*)[8]>(x));
      } else {
        constexpr float kMax = FMT == GS_DTYPE_E4M3 ? kE4m3Max : kInt8Max;
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) m = max_nan(m, fabsf(x[i]));
#pragma unroll
        for (int o = kLanes >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFullMask, m, o));
        const float inv = quant_inv(m, kMax);
        if (!s[u].ok) continue;
        uint32_t c[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          const float y0 = x[4 * i] * inv, y1 = x[4 * i + 1] * inv, y2 = x[4 * i + 2] * inv, y3 = x[4 * i + 3] * inv;
          c[i] = FMT == GS_DTYPE_E4M3 ? e4m3x4(y0, y1, y2, y3) : int8x4(y0, y1, y2, y3);
        }
#pragma unroll
        for (int i = 0; i < E / 8; ++i) *reinterpret_cast<uint2*>(pool + at + i * (D / 2)) = make_uint2(c[2 * i], c[2 * i + 1]);
        if (at == 0) *const_cast<float*>(A.kv.scale_at(v, s[u].page, head, s[u].off)) = quant_scale(m, kMax);
      }
    }
}

template <int D, int FMT, bool BF16, bool VEC, int U>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvRowsArgs A, uint32_t step) {
  constexpr int E = row_piece<FMT, VEC>(), kLanes = D / E;
  const uint32_t row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const uint32_t token0 = row / static_cast<uint32_t>(A.kv.kv_heads);
  const int head = static_cast<int>(row - token0 * A.kv.kv_heads);
  if (token0 >= step) return;
  const int at = (threadIdx.x % kLanes) * 8;
  uint4 raw[U][2];  // the piece as it lies in the pool
  float sc[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t token = token0 + u * step;
    SlotAt s{0, 0, false};
    if (token < A.tokens) s = slot_at(A, token);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      raw[u][v] = make_uint4(0u, 0u, 0u, 0u);
      sc[u][v] = 0.0f;
      if (!s.ok) continue;
      const unsigned char* pool = A.kv.at(v, s.page, head, s.off);
      if constexpr (FMT == GS_DTYPE_BF16) {
        raw[u][v] = ld_stream_u4(reinterpret_cast<const uint4*>(pool + at * 2));
      } else {
        const uint2 c = *reinterpret_cast<const uint2*>(pool + at);
        raw[u][v].x = c.x, raw[u][v].y = c.y;
        if constexpr (E == 16) {
          const uint2 d = *reinterpret_cast<const uint2*>(pool + at + D / 2);
          raw[u][v].z = d.x, raw[u][v].w = d.y;
        }
        sc[u][v] = *A.kv.scale_at(v, s.page, head, s.off);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t token = token0 + u * step;
    if (token >= A.tokens) continue;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      unsigned char* dst = (v ? A.v : A.k) + (row_at(A, v, token, head) + at) * (BF16 ? 2 : 4);
      const uint32_t w[4] = {raw[u][v].x, raw[u][v].y, raw[u][v].z, raw[u][v].w};
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        float x[8];
        if constexpr (FMT == GS_DTYPE_BF16) {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[2 * k] = bf16_lo(w[k]), x[2 * k + 1] = bf16_hi(w[k]);
        } else {
          const float2 f = make_float2(sc[u][v], sc[u][v]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t c = w[2 * i + k];
            float2 a, b;
            if constexpr (FMT == GS_DTYPE_E4M3) {
              a = half2_float2(e4m3x2_half2(c & 0xffffu)), b = half2_float2(e4m3x2_half2(c >> 16));
            } else {
              a = make_float2(static_cast<float>(static_cast<int8_t>(c & 0xffu)), static_cast<float>(static_cast<int8_t>((c >> 8) & 0xffu)));
              b = make_float2(static_cast<float>(static_cast<int8_t>((c >> 16) & 0xffu)), static_cast<float>(static_cast<int8_t>(c >> 24)));
            }
            a = __fmul2_rn(a, f), b = __fmul2_rn(b, f);
            x[4 * k] = a.x, x[4 * k + 1] = a.y, x[4 * k + 2] = b.x, x[4 * k + 3] = b.y;
          }
        }
        store8<BF16, VEC>(dst + i * (D / 2) * (BF16 ? 2 : 4), x);
      }
    }
  }
}

template <int D, int FMT, bool BF16, bool VEC>
cudaError_t launch_rows3(const KvRowsArgs& a, bool write, cudaStream_t st) {
  constexpr int64_t per = 256 / (D / row_piece<FMT, VEC>());
  constexpr int U = 2;
  // (two tokens a thread from about two blocks an SM on)
  const bool many = VEC && a.tokens * a.kv.kv_heads >= 148 * 2 * per * U;
  const uint32_t step = static_cast<uint32_t>(many ? (a.tokens + U - 1) / U : a.tokens);
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(step) * a.kv.kv_heads + per - 1) / per);
  if (write) {
    if (VEC && many) kv_write_kernel<D, FMT, BF16, VEC, VEC ? U : 1><<<grid, 256, 0, st>>>(a, step);
    else kv_write_kernel<D, FMT, BF16, VEC, 1><<<grid, 256, 0, st>>>(a, step);
  } else {
    if (VEC && many) kv_read_kernel<D, FMT, BF16, VEC, VEC ? U : 1><<<grid, 256, 0, st>>>(a, step);
    else kv_read_kernel<D, FMT, BF16, VEC, 1><<<grid, 256, 0, st>>>(a, step);
  }
  return cudaGetLastError();
}
template <int D, int FMT, bool BF16>
cudaError_t launch_rows2(const KvRowsArgs& a, bool write, bool vec, cudaStream_t st) {
  return vec ? launch_rows3<D, FMT, BF16, true>(a, write, st) : launch_rows3<D, FMT, BF16, false>(a, write, st);
}
template <int D, int FMT>
cudaError_t launch_rows1(const KvRowsArgs& a, bool write, bool bf16, bool vec, cudaStream_t st) {
  return bf16 ? launch_rows2<D, FMT, true>(a, write, vec, st) : launch_rows2<D, FMT, false>(a, write, vec, st);
}
template <int D>
cudaError_t launch_rows(const KvRowsArgs& a, int fmt, bool write, bool bf16, bool vec, cudaStream_t st) {
  switch (fmt) {
    case GS_DTYPE_BF16: return launch_rows1<D, GS_DTYPE_BF16>(a, write, bf16, vec, st);
    case GS_DTYPE_E4M3: return launch_rows1<D, GS_DTYPE_E4M3>(a, write, bf16, vec, st);
    default: return launch_rows1<D, GS_DTYPE_INT8>(a, write, bf16, vec, st);
  }
}

// Rows (new tokens × heads of a group) up to which the few-row kernel is taken (8 sequences of 4000 tokens, 8
// heads, few rows against many: 64 rows of 128 50 and 59 us bf16, 61 and 69 int8, 96 rows 81 and 62, 104 and 72;
// 32 rows of 256 62 and 74 us bf16, 66 and 80 int8, 64 rows 100 and 78, 111 and 84.  Where contexts fill the device the lines cross
// earlier: 26 sequences of 4000, 55 rows of 128, 158 and 120 us bf16, 198 and 178 int8).
int64_t few_rows(int head_dim) { return head_dim == 256 ? 32 : 64; }

gs_status kfail(gs_kv_cache* c, gs_status s, const char* m) {
  c->err = m;
  return s;
}

KvPool pool_of(const gs_kv_cache* c) {
  const gs_kv_cache_desc& d = c->d;
  const int64_t e = d.format == GS_DTYPE_BF16 ? 2 : 1;
  KvPool p{};
  p.k = static_cast<const unsigned char*>(d.k);
  p.v = static_cast<const unsigned char*>(d.v);
  p.k_scale = d.k_scale;
  p.v_scale = d.v_scale;
  auto pieces = [&](int64_t stride) { return static_cast<uint32_t>(stride * e / 16); };
  p.k_page = pieces(d.k_page_stride), p.k_head = pieces(d.k_head_stride), p.k_token = pieces(d.k_token_stride);
  p.v_page = pieces(d.v_page_stride), p.v_head = pieces(d.v_head_stride), p.v_token = pieces(d.v_token_stride);
  p.pages = static_cast<int32_t>(d.pages);
  p.page_shift = c->page_shift;
  p.kv_heads = d.kv_heads;
  return p;
}

gs_status move_rows(gs_kv_cache* c, const gs_kv_rows* r, void* stream, bool write) {
  if (!c) return GS_EINVAL;
  if (!r) return kfail(c, GS_EINVAL, "rows are required");
  if (r->tokens < 0) return kfail(c, GS_EINVAL, "tokens must be >= 0");
  if (r->tokens == 0) return GS_OK;
  if (!r->k || !r->v || !r->slots) return kfail(c, GS_EINVAL, "k, v and slots are required");
  if (r->dtype != GS_DTYPE_F32 && r->dtype != GS_DTYPE_BF16) return kfail(c, GS_EINVAL, "k and v must be float32 or bfloat16");
  if (r->tokens > (1ll << 30)) return kfail(c, GS_EUNSUPPORTED, "at most 2^30 tokens per call");
  const int64_t e = r->dtype == GS_DTYPE_F32 ? 4 : 2;
  const int64_t st[4] = {r->k_token_stride, r->k_head_stride, r->v_token_stride, r->v_head_stride};
  for (int64_t s : st)
    if (s < 0 || s >= (1ll << 32)) return kfail(c, GS_EUNSUPPORTED, "strides of k and v must be in [0, 2^32)");
  if (!write) {
    const int64_t D = c->d.head_dim;
    if ((c->d.kv_heads > 1 && (st[1] < D || st[3] < D)) || (r->tokens > 1 && (st[0] < D || st[2] < D)))
      return kfail(c, GS_EINVAL, "output strides must not make rows overlap");
    const RowGrid k{reinterpret_cast<uintptr_t>(r->k), r->tokens, c->d.kv_heads, st[0] * e, st[1] * e, D * e};
    const RowGrid v{reinterpret_cast<uintptr_t>(r->v), r->tokens, c->d.kv_heads, st[2] * e, st[3] * e, D * e};
    if (rows_overlap(k) || rows_overlap(v) || rows_overlap(k, v)) return kfail(c, GS_EINVAL, "output rows must not overlap");
  }
  KvRowsArgs a{};
  a.kv = pool_of(c);
  a.k = static_cast<unsigned char*>(r->k);
  a.v = static_cast<unsigned char*>(r->v);
  a.k_token = static_cast<uint32_t>(st[0]), a.k_head = static_cast<uint32_t>(st[1]);
  a.v_token = static_cast<uint32_t>(st[2]), a.v_head = static_cast<uint32_t>(st[3]);
  a.slots = r->slots;
  a.tokens = r->tokens;
  a.slots_end = c->d.pages * c->d.page_size;
  a.flag = c->flag;
  if (r->tokens * c->d.kv_heads > 0x7fffffffll) return kfail(c, GS_EUNSUPPORTED, "tokens * kv_heads is at most 2^31 - 1");
  bool vec = reinterpret_cast<uintptr_t>(r->k) % 16 == 0 && reinterpret_cast<uintptr_t>(r->v) % 16 == 0;
  for (int64_t s : st) vec = vec && (s * e) % 16 == 0;
  DeviceScope scope(c->device);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const bool bf16 = r->dtype == GS_DTYPE_BF16;
  const cudaError_t er = c->d.head_dim == 64    ? launch_rows<64>(a, c->d.format, write, bf16, vec, cs)
                         : c->d.head_dim == 128 ? launch_rows<128>(a, c->d.format, write, bf16, vec, cs)
                                                : launch_rows<256>(a, c->d.format, write, bf16, vec, cs);
  if (er != cudaSuccess) return kfail(c, GS_ECUDA, cudaGetErrorString(er));
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

gs_status gs_kv_cache_create(gs_ctx* ctx, const gs_kv_cache_desc* d, gs_kv_cache** out) {
  if (!out) return GS_EINVAL;
  *out = nullptr;
  if (!ctx || !d) return GS_EINVAL;
  auto bad = [&](gs_status s, const char* m) {
    ctx_set_error(ctx, m);
    return s;
  };
  if (d->format != GS_DTYPE_BF16 && d->format != GS_DTYPE_E4M3 && d->format != GS_DTYPE_INT8)
    return bad(GS_EINVAL, "KV cache: format must be bfloat16, e4m3 or int8");
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return bad(GS_EUNSUPPORTED, "KV cache: head_dim must be 64, 128 or 256");
  int shift = 0;
  while (shift < 9 && (1 << shift) != d->page_size) ++shift;
  if (shift < 4 || shift > 8) return bad(GS_EUNSUPPORTED, "KV cache: page_size must be 16, 32, 64, 128 or 256");
  if (d->pages < 1 || d->pages > 0x7fffffffll / d->page_size)
    return bad(GS_EINVAL, "KV cache: pages must be >= 1 and pages * page_size below 2^31");
  if (d->kv_heads < 1 || d->kv_heads > 1024) return bad(GS_EINVAL, "KV cache: kv_heads must be in [1, 1024]");
  if (!d->k || !d->v) return bad(GS_EINVAL, "KV cache: k and v are required");
  if (d->format != GS_DTYPE_BF16 && (!d->k_scale || !d->v_scale))
    return bad(GS_EINVAL, "KV cache: 8-bit formats need k_scale and v_scale");
  if (reinterpret_cast<uintptr_t>(d->k_scale) % 16 || reinterpret_cast<uintptr_t>(d->v_scale) % 16)
    return bad(GS_EINVAL, "KV cache: scales must be 16-byte aligned");
  const int64_t e = d->format == GS_DTYPE_BF16 ? 2 : 1;
  const int64_t strides[6] = {d->k_page_stride, d->k_head_stride, d->k_token_stride,
                              d->v_page_stride, d->v_head_stride, d->v_token_stride};
  for (int64_t s : strides)
    if (s < d->head_dim || (s * e) % 16 != 0 || s >= (1ll << 35))
      return bad(GS_EINVAL, "KV cache: strides must be at least head_dim, whole 16-byte pieces and below 2^35 elements");
  if (reinterpret_cast<uintptr_t>(d->k) % 16 || reinterpret_cast<uintptr_t>(d->v) % 16)
    return bad(GS_EINVAL, "KV cache: k and v must be 16-byte aligned");
  auto* c = new (std::nothrow) gs_kv_cache();
  if (!c) return bad(GS_ENOMEM, "KV cache: host allocation failed");
  c->ctx = ctx;
  c->device = ctx_device(ctx);
  c->d = *d;
  c->page_shift = shift;
  DeviceScope scope(c->device);
  cudaError_t er = cudaMalloc(&c->flag, 4);
  if (er == cudaSuccess) er = clear_now(c->flag, 4);
  if (er == cudaSuccess) er = ctx_attn_workspace(ctx, kAttnWsBytes + kAttnTicketBytes + kAttnMendBytes, kAttnTicketBytes + kAttnMendBytes, &c->ws);
  if (er == cudaSuccess) er = cudaDeviceGetAttribute(&c->num_sms, cudaDevAttrMultiProcessorCount, c->device);
  if (er != cudaSuccess) {
    ctx_set_error(ctx, cudaGetErrorString(er));
    cudaFree(c->flag);
    delete c;
    return er == cudaErrorMemoryAllocation ? GS_ENOMEM : GS_ECUDA;
  }
  if (const char* m = make_attn_maps(c)) {
    ctx_set_error(ctx, m);
    cudaFree(c->flag);
    delete c;
    return GS_EUNSUPPORTED;
  }
  *out = c;
  return GS_OK;
}

gs_status gs_kv_cache_destroy(gs_kv_cache* c) {
  if (!c) return GS_OK;
  DeviceScope scope(c->device);
  cudaDeviceSynchronize();
  cudaFree(c->flag);
  delete c;
  return GS_OK;
}

const char* gs_kv_cache_last_error(const gs_kv_cache* c) { return c ? c->err.c_str() : ""; }

gs_status gs_kv_cache_check(gs_kv_cache* c, int32_t* bits) {
  if (!c || !bits) return GS_EINVAL;
  DeviceScope scope(c->device);
  int32_t f = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(&f, c->flag, 4, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && f) e = clear_now(c->flag, 4);
  if (e == cudaSuccess && (f & GS_KV_ERR_TIMEOUT)) e = clear_now(c->ws + kAttnWsBytes, kAttnTicketBytes + kAttnMendBytes);  // (a piece may not have counted)
  if (e != cudaSuccess) return kfail(c, GS_ECUDA, cudaGetErrorString(e));
  *bits = f;
  if (f & GS_KV_ERR_TIMEOUT) return kfail(c, GS_ETIMEOUT, "a bounded wait inside the attention kernel ran out");
  if (f & GS_KV_ERR_SLOT) return kfail(c, GS_EINVAL, "a slot lies past the cache");
  if (f & GS_KV_ERR_PAGE) return kfail(c, GS_EINVAL, "a page-table entry is outside the cache");
  if (f & GS_KV_ERR_LENGTH) return kfail(c, GS_EINVAL, "a sequence is longer than max_q or max_kv, or outside the tokens");
  return GS_OK;
}

gs_status gs_kv_write(gs_kv_cache* c, const gs_kv_rows* rows, void* stream) { return move_rows(c, rows, stream, true); }
gs_status gs_kv_read(gs_kv_cache* c, const gs_kv_rows* rows, void* stream) { return move_rows(c, rows, stream, false); }

gs_status gs_attention(gs_kv_cache* c, const gs_attention_args* p, void* stream) {
  if (!c) return GS_EINVAL;
  if (!p) return kfail(c, GS_EINVAL, "arguments are required");
  if (p->seqs < 0 || p->tokens < 0) return kfail(c, GS_EINVAL, "seqs and tokens must be >= 0");
  if (p->seqs == 0 || p->tokens == 0) return GS_OK;
  if (!p->q || !p->out || !p->kv_len || !p->page_table)
    return kfail(c, GS_EINVAL, "q, out, kv_len and page_table are required");
  if (p->q == p->out) return kfail(c, GS_EINVAL, "out must not be q");
  if (!p->q_start && p->tokens != p->seqs) return kfail(c, GS_EINVAL, "without q_start every sequence has one token");
  if (p->q_heads < 1 || p->q_heads > (1 << 20) || p->q_heads % c->d.kv_heads != 0)
    return kfail(c, GS_EINVAL, "q_heads must be a multiple of the cache's kv_heads");
  if (p->max_q < 1 || p->max_kv < 0) return kfail(c, GS_EINVAL, "max_q >= 1 and max_kv >= 0 are required");
  if (!p->q_start && p->max_q != 1) return kfail(c, GS_EINVAL, "without q_start max_q is 1");
  if (p->window < 0 || p->sinks < 0 || (p->sinks > 0 && p->window == 0))
    return kfail(c, GS_EINVAL, "window and sinks must be >= 0, sinks only beside a window");
  if (!std::isfinite(p->scale)) return kfail(c, GS_EINVAL, "scale must be finite");
  if (p->page_table_cols < 0 || p->page_table_stride < p->page_table_cols ||
      p->page_table_cols * c->d.page_size < p->max_kv)
    return kfail(c, GS_EINVAL, "the page table must have columns for max_kv tokens");
  if (p->page_table_cols > 0x7fffffffll || p->tokens > 0x7fffffffll)
    return kfail(c, GS_EUNSUPPORTED, "tokens and page table columns are at most 2^31 - 1");
  const int64_t st[4] = {p->q_token_stride, p->q_head_stride, p->out_token_stride, p->out_head_stride};
  for (int64_t s : st)
    if (s < c->d.head_dim || s % 8 != 0 || s > 0x7fffffffll)
      return kfail(c, GS_EINVAL, "q and out strides must be >= head_dim, multiples of 8 and below 2^31");
  if (reinterpret_cast<uintptr_t>(p->q) % 16 || reinterpret_cast<uintptr_t>(p->out) % 16)
    return kfail(c, GS_EINVAL, "q and out must be 16-byte aligned");
  const RowGrid q{reinterpret_cast<uintptr_t>(p->q), p->tokens, p->q_heads, st[0] * 2, st[1] * 2, c->d.head_dim * 2};
  const RowGrid o{reinterpret_cast<uintptr_t>(p->out), p->tokens, p->q_heads, st[2] * 2, st[3] * 2, c->d.head_dim * 2};
  if (rows_overlap(o)) return kfail(c, GS_EINVAL, "out rows must not overlap");
  if (rows_overlap(q, o)) return kfail(c, GS_EINVAL, "out must not overlap q");
  const int64_t group = p->q_heads / c->d.kv_heads;
  const int64_t most_rows = static_cast<int64_t>(p->max_q) * group;
  // (the many-row grid's second dimension holds blocks of at least 128 rows for every head)
  if (most_rows > (1ll << 23) || (most_rows + 127) / 128 * c->d.kv_heads > 65535)
    return kfail(c, GS_EUNSUPPORTED, "max_q * q_heads has to stay below 2^23 - 2^17");
  if (p->seqs > 65535) return kfail(c, GS_EUNSUPPORTED, "at most 65535 sequences per call");
  AttnArgs a{};
  a.kv = pool_of(c);
  a.q = static_cast<const __nv_bfloat16*>(p->q);
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.lse = p->lse;
  a.q_start = p->q_start;
  a.kv_len = p->kv_len;
  a.table = p->page_table;
  a.q_token = static_cast<int32_t>(st[0]), a.q_head = static_cast<int32_t>(st[1]);
  a.o_token = static_cast<int32_t>(st[2]), a.o_head = static_cast<int32_t>(st[3]);
  a.table_stride = p->page_table_stride;
  a.table_cols = static_cast<int32_t>(p->page_table_cols);
  a.tokens = p->tokens;
  a.seqs = p->seqs;
  a.q_heads = p->q_heads;
  a.group = static_cast<int32_t>(group);
  a.inv_group = 1.0f / static_cast<float>(group);
  a.max_q = p->max_q;
  a.max_kv = p->max_kv;
  // (a window that covers max_kv tokens hides nothing)
  a.window = p->window >= p->max_kv ? 0 : p->window;
  a.sinks = a.window ? (p->sinks < p->max_kv ? p->sinks : p->max_kv) : 0;
  a.scale_log2 = static_cast<float>(static_cast<double>(p->scale) * 1.4426950408889634);
  a.flag = c->flag;
  a.mend = reinterpret_cast<unsigned*>(c->ws + kAttnWsBytes + kAttnTicketBytes);
  DeviceScope scope(c->device);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const cudaError_t e = most_rows > few_rows(c->d.head_dim) ? launch_attn_tile(c, a, cs) : launch_attn_rows(c, a, cs);
  if (e != cudaSuccess) return kfail(c, GS_ECUDA, cudaGetErrorString(e));
  return GS_OK;
}

}  // extern "C"
