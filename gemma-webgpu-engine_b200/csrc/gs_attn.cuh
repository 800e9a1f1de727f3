// Shared types of the paged key/value cache and its attention kernels.
#pragma once
#include <string>

#include "gs_device.cuh"
#include "gs_internal.cuh"
#include "gs_quant.cuh"
#include "../../include/gsampler.h"

struct gs_kv_cache {
  gs_ctx* ctx = nullptr;
  int device = 0;
  int num_sms = 0;
  gs_kv_cache_desc d{};
  int page_shift = 0;
  int32_t* flag = nullptr;       // device: GS_KV_ERR_* bits
  unsigned char* ws = nullptr;   // the context's attention workspace (kAttnWsBytes)
  alignas(64) unsigned char maps[768] = {};  // tensor maps of the pools: many-row kernel's, few-row kernel's, two-block kernel's
  std::string err;
};

namespace gs {

// Workspace of split-context partial results, float32 outputs and their maxima and sums.  The planners never
// ask for more.
constexpr size_t kAttnWsBytes = 64u << 20;
constexpr size_t kAttnTicketBytes = 16u << 10;  // behind it, zero between calls
constexpr size_t kAttnMendBytes = 64;           // and behind that, zero between calls (many-row kernel)

struct KvPool {
  const unsigned char* k;
  const unsigned char* v;
  const float* k_scale;
  const float* v_scale;
  // strides in 16-byte pieces: each product below is one 32 x 32 -> 64-bit multiply-add
  uint32_t k_page, k_head, k_token;
  uint32_t v_page, v_head, v_token;
  int32_t pages;
  int32_t page_shift;
  int32_t kv_heads;
  __device__ __forceinline__ const unsigned char* at(bool value, int page, int head, int off) const {
    const uint64_t e = static_cast<uint64_t>(static_cast<uint32_t>(page)) * (value ? v_page : k_page) +
                       static_cast<uint64_t>(static_cast<uint32_t>(head)) * (value ? v_head : k_head) +
                       static_cast<uint64_t>(static_cast<uint32_t>(off)) * (value ? v_token : k_token);
    return (value ? v : k) + (e << 4);
  }
  __device__ __forceinline__ const float* scale_at(bool value, int page, int head, int off) const {
    const uint64_t e = static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(kv_heads) + static_cast<uint32_t>(head);
    return (value ? v_scale : k_scale) + (e << page_shift) + off;
  }
};

struct AttnArgs {
  KvPool kv;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* table;
  int32_t q_token, q_head, o_token, o_head;  // element strides
  int64_t table_stride;
  int64_t tokens;
  int32_t table_cols;
  int32_t seqs, q_heads, group;
  float inv_group;      // 1 / group
  int32_t max_q, max_kv;
  int32_t window, sinks;
  float scale_log2;     // scale · log2(e): scores in log2 units
  int32_t chunk_tiles;  // (many-row kernel) context tiles per split
  int32_t splits;       // partial results per (sequence, head, row block)
  int32_t cluster;      // blocks per partial result (few-row kernel)
  int32_t row_blocks;   // (many-row kernel) blocks of query rows per sequence and head
  int32_t units;        // (many-row kernel, balanced) sequences times row blocks
  unsigned* tickets;    // finished parts of a context, per warp that holds the same rows of each; zero between calls
  unsigned* mend;       // (many-row kernel) whether a result is not finite; blocks that have mended theirs
  float* part_o;        // partial results: outputs
  float* part_ml;       // and running maxima (log2 units) and sums
  int32_t* flag;
};

// What one block of query rows of a sequence sees: rows are (new token, head of the
// group), row = token · group + head.
struct RowRange {
  int32_t q0;       // first new token of the sequence
  int32_t nq;       // its new tokens
  int32_t len;      // its cached tokens
  int32_t rows;     // rows of this block
  int32_t p0;       // position of new token 0
  int32_t hi;       // tokens >= hi are hidden from every row
  int32_t lo;       // tokens in [sink, lo) are hidden from every row (0 without a window)
  int32_t sink;     // tokens below stay visible (0 without a window)
  int32_t t0, g0;   // new token and head of the block's row 0
  int32_t sink_tiles, first_tile, tiles;  // context tiles: [0, sink_tiles), then from first_tile
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : first_tile + i - sink_tiles; }
  // New token and head of the group of row i of the block.  (g0 + i + 1/2) / group stays 1 / (2 group) away from
  // every whole number, which the float product's error does not reach below 2^21.
  __device__ __forceinline__ int token_of(const AttnArgs& A, int i, int& g) const {
    const int x = g0 + i, t = static_cast<int>((static_cast<float>(x) + 0.5f) * A.inv_group);
    g = x - t * A.group;
    return t0 + t;
  }
  __device__ __forceinline__ bool seen_by_any(int j) const { return j < hi && (j >= lo || j < sink); }
};

__device__ __forceinline__ const __nv_bfloat16* q_row(const AttnArgs& A, const RowRange& R, int head, int t, int g) {
  return A.q + static_cast<int64_t>(R.q0 + t) * A.q_token + static_cast<int64_t>(head * A.group + g) * A.q_head;
}
__device__ __forceinline__ __nv_bfloat16* o_row(const AttnArgs& A, const RowRange& R, int head, int t, int g) {
  return A.out + static_cast<int64_t>(R.q0 + t) * A.o_token + static_cast<int64_t>(head * A.group + g) * A.o_head;
}
// Power of two that brings a row into [1, 2) at its largest component (all bits of `top`, the largest
// magnitude's bf16 pattern), as the factor down and the factor back; 1 for a row of zeros or not finite.
__device__ __forceinline__ void row_power(uint32_t top, float& down, float& up) {
  int e = static_cast<int>(top >> 7) - 127;
  e = top == 0u || e > 127 ? 0 : min(max(e, -120), 120);
  down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
// Larger magnitudes of two bf16 pairs, and of a pair's halves (patterns without sign order as values do).
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); }

// Rows [r0, r0 + cap) of sequence b, context tiles of kTile tokens.
template <int kTile>
__device__ __forceinline__ RowRange row_range(const AttnArgs& A, int b, int r0, int cap) {
  RowRange R;
  R.q0 = A.q_start ? A.q_start[b] : b;
  int q1 = A.q_start ? A.q_start[b + 1] : b + 1;
  R.len = A.kv_len[b];
  bool bad = R.len > A.max_kv || R.len < 0 || R.q0 < 0 || q1 > A.tokens || q1 - R.q0 > A.max_q;
  R.len = min(max(R.len, 0), A.max_kv);
  R.q0 = max(R.q0, 0);
  q1 = static_cast<int>(min(static_cast<int64_t>(q1), A.tokens));
  R.nq = max(q1 - R.q0, 0);
  R.p0 = R.len - R.nq;
  R.nq = min(R.nq, A.max_q);
  R.rows = min(cap, R.nq * A.group - r0);
  R.t0 = r0 / A.group;
  R.g0 = r0 - R.t0 * A.group;
  if (R.rows <= 0) {
    R.rows = 0;
    R.tiles = 0;
    if (bad && r0 == 0 && threadIdx.x == 0) atomicOr(A.flag, GS_KV_ERR_LENGTH);
    return R;
  }
  if (bad && threadIdx.x == 0) atomicOr(A.flag, GS_KV_ERR_LENGTH);
  const int pf = R.p0 + R.t0, pl = R.p0 + (r0 + R.rows - 1) / A.group;
  R.hi = max(pl + 1, 0);
  R.lo = A.window ? max(pf - A.window + 1, 0) : 0;
  R.lo = min(R.lo, R.hi);
  R.sink = A.window ? min(A.sinks, R.hi) : 0;
  R.sink_tiles = (R.sink + kTile - 1) / kTile;
  R.first_tile = max(R.lo / kTile, R.sink_tiles);
  R.tiles = R.sink_tiles + max((R.hi + kTile - 1) / kTile - R.first_tile, 0);
  return R;
}

// Context tiles of kTile tokens the widest row block of a call can see (host side).
inline int64_t most_tiles(const AttnArgs& a, int tile, int rows_per_block) {
  const int64_t all = (static_cast<int64_t>(a.max_kv) + tile - 1) / tile;
  if (!a.window) return all;
  const int64_t span = static_cast<int64_t>(a.window) + (rows_per_block + a.group - 1) / a.group + 1;
  const int64_t w = (static_cast<int64_t>(a.sinks) + tile - 1) / tile + (span + tile - 1) / tile + 2;
  return w < all ? w : all;
}

__device__ __forceinline__ float ex2(float x) { return ex2_approx(x); }

__device__ __forceinline__ bool finite4(float4 x) {
  return fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY && fabsf(x.z) < INFINITY && fabsf(x.w) < INFINITY;
}

// Values d .. d + 3 of one row's result by the formula, token by token over what the row sees, in float32 by one
// thread: (O, not yet divided by the sum) and (m in log2 units, sum).  The kernels' second product runs over whole tiles, where a
// hidden token's weight is 0; when its value is an infinity or a NaN, 0 times that is a NaN in rows that never see
// the token.  So a result that is not finite is computed again here, which the sums of finite values never pay for.
template <int FMT>
__device__ __noinline__ void attn_by_row(const AttnArgs& A, int b, int head, const __nv_bfloat16* q, int pos, int head_dim, int d, float4* o,
                                         float2* ml) {
  constexpr int kEl = FMT == GS_DTYPE_BF16 ? 2 : 1;
  const int32_t* table = A.table + b * A.table_stride;
  const int lo = A.window ? max(pos - A.window + 1, 0) : 0, mask = (1 << A.kv.page_shift) - 1;
  auto four = [](const unsigned char* p) {
    if constexpr (FMT == GS_DTYPE_BF16) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
      if constexpr (FMT == GS_DTYPE_E4M3) {
        const float2 x = half2_float2(e4m3x2_half2(w & 0xffffu)), y = half2_float2(e4m3x2_half2(w >> 16));
        return make_float4(x.x, x.y, y.x, y.y);
      } else {
        return make_float4(static_cast<float>(static_cast<signed char>(w)), static_cast<float>(static_cast<signed char>(w >> 8)),
                           static_cast<float>(static_cast<signed char>(w >> 16)), static_cast<float>(static_cast<signed char>(w >> 24)));
      }
    }
  };
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int j = A.sinks > 0 ? 0 : lo; j <= pos; ++j) {
    if (j >= A.sinks && j < lo) j = lo;
    const int col = j >> A.kv.page_shift, off = j & mask;
    int page = col < A.table_cols ? __ldg(table + col) : 0;
    if (page < 0 || page >= A.kv.pages) page = 0;  // (noted by the kernel that came here)
    const unsigned char* k = A.kv.at(false, page, head, off);
    float s = 0.0f;
    for (int i = 0; i < head_dim; i += 4) {
      const float4 x = four(k + i * kEl);
      const uint2 w = *reinterpret_cast<const uint2*>(q + i);
      s += bf16_lo(w.x) * x.x, s += bf16_hi(w.x) * x.y, s += bf16_lo(w.y) * x.z, s += bf16_hi(w.y) * x.w;
    }
    s *= A.scale_log2;
    float vs = 1.0f;
    if constexpr (FMT != GS_DTYPE_BF16) {
      s *= *A.kv.scale_at(false, page, head, off);
      vs = *A.kv.scale_at(true, page, head, off);
    }
    const float mx = max_nan(M, s), at = mx == -INFINITY ? 0.0f : mx, back = ex2(M - at), p = ex2(s - at);
    const float4 x = four(A.kv.at(true, page, head, off) + d * kEl);
    M = mx;
    L = L * back + p;
    acc.x = acc.x * back + p * (x.x * vs), acc.y = acc.y * back + p * (x.y * vs);
    acc.z = acc.z * back + p * (x.z * vs), acc.w = acc.w * back + p * (x.w * vs);
    if (L != L) break;  // (a score that is no number: all of the row is none)
  }
  if (L != L) acc = make_float4(L, L, L, L);
  *o = acc;
  *ml = make_float2(M, L);
}

// Few-row kernel (mma.sync, one 16-token tile per warp): any number of rows in blocks.
cudaError_t launch_attn_rows(const gs_kv_cache* c, AttnArgs a, cudaStream_t st);
// Many-row kernel (tcgen05), and the tensor maps both read a cache by (an error text, or nullptr).
cudaError_t launch_attn_tile(const gs_kv_cache* c, AttnArgs a, cudaStream_t st);
const char* make_attn_maps(gs_kv_cache* c);
}  // namespace gs
