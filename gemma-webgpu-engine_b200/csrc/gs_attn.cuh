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
  unsigned* mend;       // (many-row kernel) whether values were left out of a product; blocks that have seen to it
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
  // Tokens that some rows see and others do not: from ahead0 to hi (some row's position is before them), and from left0 to left1
  // (some row's window has left them).
  __device__ __forceinline__ int ahead0() const { return max(p0 + t0 + 1, 0); }
  __device__ __forceinline__ int left0() const { return max(sink, lo); }
  __device__ __forceinline__ int left1(const AttnArgs& A) const { return min(hi - A.window, p0 + t0 + 1); }
  // Whether every row sees the tokens j .. j + n - 1.
  __device__ __forceinline__ bool seen_by_all(const AttnArgs& A, int j, int n = 1) const {
    return j + n - 1 <= p0 + t0 && (!A.window || j > hi - 1 - A.window || j + n <= sink);
  }
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

// Rows [r0, r0 + cap) of sequence b, context tiles of kTile tokens.  note: whether this thread reports what is wrong with the
// sequence's entries.
template <int kTile>
__device__ __forceinline__ RowRange row_range(const AttnArgs& A, int b, int r0, int cap, bool note) {
  RowRange R;
  R.q0 = A.q_start ? A.q_start[b] : b;
  int q1 = A.q_start ? A.q_start[b + 1] : b + 1;
  R.len = A.kv_len[b];
  const bool bad = R.len > A.max_kv || R.len < 0 || R.q0 < 0 || q1 > A.tokens || q1 < R.q0 || q1 - R.q0 > A.max_q;
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
    if (bad && r0 == 0 && note) atomicOr(A.flag, GS_KV_ERR_LENGTH);
    return R;
  }
  if (bad && note) atomicOr(A.flag, GS_KV_ERR_LENGTH);
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

// Values that are not finite.  The kernels' second product runs over whole tiles, where a token hidden from a row has the weight
// 0 in it, and 0 times an infinity is a NaN.  Tokens that no row of a block sees are zeroed before the product.  Of tokens that
// some rows see and others do not (at the causal edge and at the window's, as many as a block has new tokens) the elements
// that are not finite are zeroed, and the rows that see them get what is not finite apart from the product (few rows: a NaN; many: the
// value).  Beside an 8-bit cache a scale that is not finite counts for all of its row.  Tokens that all rows see go through
// the product as they are.
//
// The elements of a word of a cached row that are not finite, all bits of each.
template <int FMT>
__device__ __forceinline__ uint32_t not_finite_in(uint32_t w) {
  if constexpr (FMT == GS_DTYPE_BF16) return __vcmpeq2(w & 0x7f807f80u, 0x7f807f80u);
  else if constexpr (FMT == GS_DTYPE_E4M3) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
  else return 0u;
}
template <int FMT>
__device__ __forceinline__ uint4 not_finite_in(uint4 w) {
  return make_uint4(not_finite_in<FMT>(w.x), not_finite_in<FMT>(w.y), not_finite_in<FMT>(w.z), not_finite_in<FMT>(w.w));
}
// Looks for them in four words: `found`, zero at first, tells later whether there was one (bf16: an infinity or a NaN times zero
// is a NaN, all else adds zero; e4m3: the code after the largest finite one carries into the sign's place).
template <int FMT>
__device__ __forceinline__ void look_for_not_finite(uint4 w, uint32_t& found) {
  if constexpr (FMT == GS_DTYPE_BF16) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(found) : "r"(x[i]), "r"(0u));
  } else if constexpr (FMT == GS_DTYPE_E4M3) {
    constexpr uint32_t kCode = 0x7f7f7f7fu, kOne = 0x01010101u;
    found |= ((w.x & kCode) + kOne) | ((w.y & kCode) + kOne) | ((w.z & kCode) + kOne) | ((w.w & kCode) + kOne);
  }
}
template <int FMT>
__device__ __forceinline__ bool found_not_finite(uint32_t found) {
  return FMT == GS_DTYPE_BF16 ? (found & 0x7fff7fffu) != 0u : FMT == GS_DTYPE_E4M3 ? (found & 0x80808080u) != 0u : false;
}
template <int FMT>
__device__ __forceinline__ bool any_not_finite(uint4 w) {
  uint32_t found = 0u;
  look_for_not_finite<FMT>(w, found);
  return found_not_finite<FMT>(found);
}
__device__ __forceinline__ uint4 without4(uint4 w, uint4 m) { return make_uint4(w.x & ~m.x, w.y & ~m.y, w.z & ~m.z, w.w & ~m.w); }

// Few-row kernel (mma.sync, one 16-token tile per warp): any number of rows in blocks.
cudaError_t launch_attn_rows(const gs_kv_cache* c, AttnArgs a, cudaStream_t st);
// Many-row kernel (tcgen05), and the tensor maps both read a cache by (an error text, or nullptr).
cudaError_t launch_attn_tile(const gs_kv_cache* c, AttnArgs a, cudaStream_t st);
const char* make_attn_maps(gs_kv_cache* c);
}  // namespace gs
