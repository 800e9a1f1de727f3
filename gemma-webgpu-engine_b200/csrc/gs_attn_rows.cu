// Attention of few query rows over the paged cache (one decoded token, a few drafted ones).
//
// Per row, over the visible tokens j in tiles of 16, with the running maximum m and sum l
// (log2 units, s_j = scale · log2(e) · q·k_j):
//   m' = max(m, max s_j);  l = l · 2^(m - m') + Σ 2^(s_j - m');  O = O · 2^(m - m') + Σ 2^(s_j - m') v_j
//   out = O / l,  lse = (m + log2 l) / log2(e)
// Bound by HBM: each cached byte is used for 2 · rows multiply-adds an element, so all the
// rows of a key/value head (new tokens × heads of the group) share one pass over its tokens.
//
// The products run transposed, S^T = K Q^T and O^T = V^T P^T (mma m16n8k16): the 16 tokens
// (or 16 values of head_dim) are the M side, so 8 rows fill the N side and a group of 1 to 8
// heads wastes no registers on padding; O^T takes head_dim / 4 registers a lane per 8 rows.
// S^T's accumulators become the B operand of the second product by one 8x8 transpose each.
//
// Every warp walks its own tiles (every fourth of the block's share) through a private ring of
// shared-memory stages that one lane fills by TMA boxes of 16 tokens in the swizzled layout
// ldmatrix reads without bank conflicts: the loop has no block barrier, and 100 to 190 KB are in flight per SM.
// A row's reference point m moves only when a score passes it by 2^8 (as V's reference scale does
// when a larger one comes), so the usual tile needs one vote instead of reductions and rescaling.
// Values of tokens hidden from every row of the block are set to zero before they are used, and so is what is not finite in
// tokens hidden from some rows, whose columns are then a NaN in the rows that see them.
//
// A context is shared evenly by the blocks of a cluster (up to 8), which join their (m, l, O) through
// distributed shared memory; of several clusters per context the last to finish joins their partial
// results.
//
// Measured (calls in a row; one token a sequence, 32 query heads on 8 of 128): 64 sequences of 8192 tokens bf16 313 us,
// 6.9 TB/s, e4m3 188 us, 5.9 TB/s, ragged 187 and 123 us; two of 131072 tokens (4 heads) 91 us, 5.9 TB/s;
// one of 777 tokens (2 heads of 256) 7 us on the device: launch, table and query loads, one round of tiles, join.
// Beside 8-bit codes the widening keeps the issue slots half busy and the ragged last round is the
// other loss; 20 rows of 256 (16 windows of 1028 tokens, int8, 27 us) take two passes of 16 rows at 1.5 us
// a tile and warp: bound by the products' latency, not by bytes.
//
// 8-bit codes are widened to float16 (exact for e4m3 and int8) in registers, K's scale
// multiplies the finished score, V's scale the weight: 2^(s - m) · (scale / largest magnitude of one so
// far) · 2^7, at most 2^15, which float16 holds to 11 bits down to 2^-21 of the largest; the factor is
// taken out of O at the end.  q is brought into float16's range by a power of two per row
// (bfloat16 has fewer mantissa bits: exact except for components below 2^-17 of the row's
// largest).  Beside a bf16 cache the weights are bf16, as q and v are.
#include <cuda.h>

#include "gs_attn.cuh"

namespace gs {
namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr int kRT = 16;  // tokens per warp tile
constexpr float kPScale = 128.0f;
constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100: reference of V scales below it (its reciprocal is finite)
constexpr float kSlack = 8.0f;  // log2 units a score may pass the reference by

template <int D, int FMT>
struct RowsPlan {
  static constexpr bool kBf = FMT == GS_DTYPE_BF16;
  static constexpr int kEl = kBf ? 2 : 1;
  static constexpr int kRow = D * kEl;                       // bytes of one token's K (or V) row
  static constexpr int kInner = kRow < 128 ? kRow : 128;     // bytes of a row in one TMA box
  static constexpr int kCols = kRow / kInner;                // boxes across a row
  static constexpr int kTileBytes = kRT * kRow;              // K or V of one tile
  static constexpr int kSub = kTileBytes <= 1024 ? 2 : 1;    // tiles per stage
  // A stage holds K and V of its tiles, or, where those are 16 KB, one of them, in turn: three stages of 8 KB a warp
  // then leave room for a second block on the SM (32 rows, 8 sequences of 4000 tokens, 8 heads of 256: 38% less time), at the
  // price of two waits and two fetches a tile (narrower rows lose by it: heads of 64 16%).
  static constexpr bool kHalves = kTileBytes >= 8192;
  static constexpr int kParts = kHalves ? 1 : 2;
  static constexpr int kStage = kSub * kParts * kTileBytes;
  static constexpr int kStages = 3;
  static constexpr int kRing = kRowsWarps * kStages * kStage;
  static constexpr int kScale = kBf ? 0 : kSub * 2 * kRT * 4;  // scales of a stage
};

template <int D, int FMT, int NB>
struct RowsSmem {
  using P = RowsPlan<D, FMT>;
  static constexpr int kRows = 8 * NB;
  static constexpr int kJoin = kRowsWarps * kRows * (D + 4) * 4;
  static constexpr int kMain = P::kRing > kJoin ? P::kRing : kJoin;
  static constexpr int kOffScale = kMain;
  static constexpr int kOffQ = kOffScale + kRowsWarps * P::kStages * P::kScale;
  static constexpr int kTotal = kOffQ + NB * (D / 16) * 32 * 8 + 1024;  // Q fragments, alignment slack
};

__device__ __forceinline__ void box_in(uint32_t dst, const CUtensorMap* map, int x, int tok, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(tok), "r"(head), "r"(page), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint4 ld_shared4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared1(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <bool BF16>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes in the low bytes of each 16-bit half order (b0, b1) -> half pair, exact.
// int8: byte + 128 becomes the low mantissa of 1024, minus 1152.
template <int FMT>
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& lo, uint32_t& hi) {  // bytes (0,1) and (2,3)
  if constexpr (FMT == GS_DTYPE_E4M3) {
    lo = e4m3x2_half2(codes & 0xffffu);
    hi = e4m3x2_half2(codes >> 16);
  } else {
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(l), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(h), "r"(0x64806480u));
  }
}

// Byte offset of 16-byte piece c of row r in a tile as the TMA boxes lay it: blocks of kInner bytes of
// all 16 rows, pieces permuted by the row (128-byte swizzle; 64-byte for the narrowest rows).
template <int INNER>
__device__ __forceinline__ uint32_t piece(int r, int c) {
  if constexpr (INNER == 64) return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  else return static_cast<uint32_t>((c >> 3) * (kRT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

struct RowsMaps {
  CUtensorMap k, v;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_rank4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float2 ld_rank2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
  return v;
}

// Blocks per SM the register budget leaves room for (the rings' sizes allow as many).
template <int D, int FMT, int NB>
constexpr int rows_occupancy() {
  const int by_smem = 227 * 1024 / (RowsSmem<D, FMT, NB>::kTotal + 1024);
  const int by_regs = D * NB <= 128 ? 4 : D * NB <= 256 ? 3 : 2;
  return by_smem < by_regs ? (by_smem < 1 ? 1 : by_smem) : by_regs;
}

// What is not finite in the V tile at vs (tokens j0 ..) and in tokens that some rows of the block see and others do not: set to
// zero, and its columns marked in the rows that see it (odd: words of 32 columns; scale_odd: tokens whose scale is not finite, all of
// their columns).  By a warp; whether this lane wrote to the tile.  (R lies in shared memory: the main loop has no registers for it.  With
// and without this: 20 rows of 256 25.4 and 25.3 us bf16, 25.4 and 25.1 e4m3, 32 rows of 256 59 and 57 e4m3, 64 rows of 128 50 and 49 bf16.)
template <int D, int FMT>
__device__ __forceinline__ bool leave_odd_out(const AttnArgs& A, const RowRange& R, uint32_t vs, int j0, unsigned scale_odd, uint32_t* odd, int* any) {
  using P = RowsPlan<D, FMT>;
  constexpr int kPc = P::kRow / 16;
  const int lane = threadIdx.x & 31;
  uint32_t all = 0u;
#pragma unroll
  for (int id = lane; id < kRT * kPc; id += 32) {
    uint32_t found = 0u;
    look_for_not_finite<FMT>(ld_shared4(vs + piece<P::kInner>(id / kPc, id % kPc)), found);
    all |= found;
  }
  if (!__any_sync(kFullMask, found_not_finite<FMT>(all)) && scale_odd == 0u) return false;
  bool wrote = false;
  for (int t = 0; t < kRT; ++t) {
    const int j = j0 + t;
    if (!R.seen_by_any(j) || R.seen_by_all(A, j)) continue;
    for (int at = lane * 4; at < P::kRow; at += 128) {  // a word of the token's row
      const uint32_t w = vs + piece<P::kInner>(t, at / 16) + (at & 12), x = ld_shared1(w), m = scale_odd >> t & 1u ? ~0u : not_finite_in<FMT>(x);
      if (m == 0u) continue;
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(w), "r"(x & ~m) : "memory");
      wrote = true;
      *any = 1;
      for (int r = 0, g = R.g0, p = R.p0 + R.t0; r < R.rows; ++r, ++g) {
        if (g == A.group) g = 0, ++p;
        if (j > p || (A.window && j <= p - A.window && j >= A.sinks)) continue;
        for (int b = 0; b < 4; b += P::kEl)
          if (m >> (8 * b) & 1u) atomicOr(odd + (r * D + (at + b) / P::kEl) / 32, 1u << ((at + b) / P::kEl & 31));
      }
    }
  }
  return wrote;
}

// TOKENS: a sequence may have more than one new token, so that the rows of a block need not see the same ones (the code for that costs the
// main loop registers and time: 64 sequences of 8192 tokens, one token each, e4m3 188 -> 194 us with it, int8 211 -> 216).
template <int D, int FMT, int NB, bool TOKENS>
__global__ void __launch_bounds__(kRowsThreads, (rows_occupancy<D, FMT, NB>()))
    attn_rows_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ RowsMaps maps) {
  using P = RowsPlan<D, FMT>;
  using S = RowsSmem<D, FMT, NB>;
  constexpr bool kBf = P::kBf;
  constexpr int kRows = 8 * NB;
  constexpr int KS = D / 16;  // k-steps of the first product, 16-wide value blocks of the second
  constexpr bool kQRegs = D * NB <= 128;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint2* qfrag = reinterpret_cast<uint2*>(smem + S::kOffQ);  // [NB][KS][32]
  __shared__ float s_m[kRowsWarps][kRows], s_l[kRowsWarps][kRows], s_f[kRowsWarps];
  __shared__ float s_qf[kRows];
  __shared__ __align__(8) float s_ml[kRows][2];  // the block's joined maximum and sum
  // (TOKENS) columns of rows that have a value which is not finite and was left out of the product; whether there are any
  __shared__ uint32_t s_odd[TOKENS ? kRows : 1][D / 32];
  __shared__ int s_any;
  __shared__ RowRange s_range;
  __shared__ __align__(8) uint64_t s_bar[kRowsWarps][P::kStages];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int b = blockIdx.z;
  const int head = blockIdx.y % A.kv.kv_heads, rb = blockIdx.y / A.kv.kv_heads;
  const int r0 = rb * kRows;
  const RowRange R = row_range<kRT>(A, b, r0, kRows, tid == 0);
  if (R.rows == 0) return;  // (the whole cluster)
  // this block's tiles: an even share of the context's
  const int share = (R.tiles + A.splits * A.cluster - 1) / (A.splits * A.cluster);
  const int i_begin = min(static_cast<int>(blockIdx.x) * share, R.tiles);
  const int i_end = min(i_begin + share, R.tiles);
  if (lane < P::kStages) mbar_init(&s_bar[warp][lane], 1);
  if constexpr (TOKENS) {
    for (int i = tid; i < kRows * (D / 32); i += kRowsThreads) s_odd[0][i] = 0u;
    if (tid == 0) s_any = 0, s_range = R;
  }
  __syncwarp();

  // ---- the warp's ring: stage i holds the warp's step i, tiles i_begin + (i · 4 + warp) · kSub .., or (halves)
  // K (i even) or V of step i / 2
  const uint32_t ring = smem_addr(smem) + warp * (P::kStages * P::kStage);
  const uint32_t scales = smem_addr(smem + S::kOffScale) + warp * (P::kStages * P::kScale);
  const int32_t* table = A.table + b * A.table_stride;
  const int per_page = A.kv.page_shift - 4;  // log2 of tiles per page
  const int page_mask = (1 << A.kv.page_shift) - 1;
  const int first = i_begin + warp * P::kSub;
  constexpr int kStep = kRowsWarps * P::kSub;
  const int n_steps = i_end > first ? (i_end - first + kStep - 1) / kStep : 0;
  int pages = 0;       // table entries of the warp's next 32 tiles
  int pages_at = -1;   // which 32
  auto fetch = [&](int i, int slot) {
    const int n = P::kHalves ? i >> 1 : i, t = n * P::kSub;  // step, the warp's tile number
    if ((t >> 5) != pages_at) {
      pages_at = t >> 5;
      const int tl = (pages_at << 5) + lane;
      const int il = first + tl / P::kSub * kStep + tl % P::kSub;
      pages = -1;
      if (il < i_end) {
        const int col = R.tile(il) >> per_page;
        if (col < A.table_cols) pages = __ldg(table + col);
        if (pages < 0 || pages >= A.kv.pages) {
          pages = 0;
          atomicOr(A.flag, GS_KV_ERR_PAGE);
        }
      }
    }
    int pg[P::kSub];
#pragma unroll
    for (int u = 0; u < P::kSub; ++u) pg[u] = __shfl_sync(kFullMask, pages, (t + u) & 31);
    if (lane == 0 && n < n_steps) {
      uint64_t* bar = &s_bar[warp][slot];
      const int i0 = first + n * kStep;
      const int live = P::kSub == 1 || i0 + 1 < i_end ? P::kSub : 1;
      mbar_expect_tx(bar, live * (P::kParts * P::kTileBytes + (kBf ? 0 : 2 * kRT * 4)));
#pragma unroll
      for (int u = 0; u < P::kSub; ++u) {
        if (u >= live) break;
        const int off = (R.tile(i0 + u) * kRT) & page_mask;
        const uint32_t at = ring + slot * P::kStage + u * P::kParts * P::kTileBytes;
#pragma unroll
        for (int cb = 0; cb < P::kCols; ++cb) {
          const int x = cb * (P::kInner / P::kEl);
          const uint32_t to = at + cb * (kRT * P::kInner);
          if constexpr (P::kHalves) {
            box_in(to, i & 1 ? &maps.v : &maps.k, x, off, head, pg[u], bar);
          } else {
            box_in(to, &maps.k, x, off, head, pg[u], bar);
            box_in(to + P::kTileBytes, &maps.v, x, off, head, pg[u], bar);
          }
        }
        if constexpr (!kBf) {
          static_assert(kBf || !P::kHalves, "scales come with both");
          const uint32_t sd = scales + slot * P::kScale + u * (2 * kRT * 4);
          bulk_g2s_addr(sd, A.kv.scale_at(false, pg[u], head, off), kRT * 4, bar);
          bulk_g2s_addr(sd + kRT * 4, A.kv.scale_at(true, pg[u], head, off), kRT * 4, bar);
        }
      }
    }
    __syncwarp();
  };
#pragma unroll
  for (int i = 0; i < P::kStages; ++i) fetch(i, i);

  // ---- Q fragments (B operand: k = 2c.. of row n = g), once
  for (int nb = warp; nb < NB; nb += kRowsWarps) {
    const int r = 8 * nb + g;
    const bool live = r < R.rows;
    int gq;
    const int tq = R.token_of(A, live ? r : 0, gq);
    const __nv_bfloat16* q = q_row(A, R, head, tq, gq);
    uint32_t w[KS][2];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      // bf16: elements 16k + 2c, + 8; codes: the k order of a byte-wise K fragment, 16k + 4c, + 2
      const int e0 = kBf ? 16 * k + 2 * c : 16 * k + 4 * c, e1 = kBf ? e0 + 8 : e0 + 2;
      w[k][0] = live ? *reinterpret_cast<const uint32_t*>(q + e0) : 0u;
      w[k][1] = live ? *reinterpret_cast<const uint32_t*>(q + e1) : 0u;
    }
    float f = 1.0f;
    if constexpr (!kBf) {
      uint32_t mx = 0;
#pragma unroll
      for (int k = 0; k < KS; ++k) mx = __vmaxu2(mx, pair_max(w[k][0], w[k][1]));
      mx = __vmaxu2(mx, __shfl_xor_sync(kFullMask, mx, 1));
      mx = __vmaxu2(mx, __shfl_xor_sync(kFullMask, mx, 2));
      float down;
      row_power(max(mx & 0xffffu, mx >> 16), down, f);
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[k][h] = half2_of(bf16_lo(w[k][h]) * down, bf16_hi(w[k][h]) * down);
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) qfrag[(nb * KS + k) * 32 + lane] = make_uint2(w[k][0], w[k][1]);
    if (c == 0) s_qf[r] = f * A.scale_log2;
  }
  __syncthreads();
  uint2 qreg[kQRegs ? NB * KS : 1];
  if constexpr (kQRegs) {
#pragma unroll
    for (int k = 0; k < NB * KS; ++k) qreg[k] = qfrag[k * 32 + lane];
  }
  auto qf_at = [&](int nb, int k) {
    if constexpr (kQRegs) return qreg[nb * KS + k];
    else return qfrag[(nb * KS + k) * 32 + lane];
  };

  float qf[NB][2];
  int pos[NB][2];  // position of the lane's two rows
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * nb + 2 * c + h;
      qf[nb][h] = s_qf[r];
      int gq;
      pos[nb][h] = R.p0 + R.token_of(A, min(r, R.rows - 1), gq);
    }
  const int p_min = R.p0 + R.t0, p_max = R.hi - 1;

  float o[NB][KS][4];
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = -INFINITY;
    l[nb][0] = l[nb][1] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int u = 0; u < 4; ++u) o[nb][k][u] = 0.0f;
  }
  float vref = 0.0f, vinv = 0.0f;  // (8-bit) largest V scale's magnitude so far, kPScale over it

  int slot = 0;  // of the next stage
  uint32_t phase = 0;
  auto wait = [&](int s_, uint32_t p_) {
    const bool ok = mbar_wait(&s_bar[warp][s_], p_, kWaitNs);
    if (!ok) atomicOr(A.flag, GS_KV_ERR_TIMEOUT);
    return __all_sync(kFullMask, ok);
  };
  bool ok = true;
  for (int n = 0; n < n_steps; ++n) {
    const int k_slot = slot;
    const uint32_t k_phase = phase;
    if (++slot == P::kStages) slot = 0, phase ^= 1;
    const int v_slot = P::kHalves ? slot : k_slot;
    const uint32_t v_phase = phase;  // (halves)
    if constexpr (P::kHalves) {
      if (++slot == P::kStages) slot = 0, phase ^= 1;
    }
    const int i0 = first + n * kStep;
    ok = wait(k_slot, k_phase);
    if (!ok) break;
#pragma unroll
    for (int sub = 0; sub < P::kSub; ++sub) {
      const bool last = sub == P::kSub - 1 || (P::kSub > 1 && i0 + sub + 1 >= i_end);
      const uint32_t ks = ring + k_slot * P::kStage + sub * P::kParts * P::kTileBytes;
      const uint32_t vs = P::kHalves ? ring + v_slot * P::kStage : ks + P::kTileBytes;
      const int j0 = R.tile(i0 + sub) * kRT;
      const bool whole = j0 + kRT - 1 <= p_min && (!A.window || j0 > p_max - A.window || j0 + kRT <= A.sinks);
      // ---- S^T = K Q^T
      float s[NB][4];
      {
        float s2[NB][4];  // a second chain halves the dependent products
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int u = 0; u < 4; ++u) s[nb][u] = s2[nb][u] = 0.0f;
        const int mr = lane & 15, mh = lane >> 4;  // matrix row and half of this lane's address
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          if constexpr (kBf) {
            uint32_t a[4], a2[4];
            ldsm4(ks + piece<P::kInner>(mr, 2 * k + mh), a);
            ldsm4(ks + piece<P::kInner>(mr, 2 * k + 2 + mh), a2);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const uint2 q0 = qf_at(nb, k), q1 = qf_at(nb, k + 1);
              mma16<true>(s[nb], a[0], a[1], a[2], a[3], q0.x, q0.y);
              mma16<true>(s2[nb], a2[0], a2[1], a2[2], a2[3], q1.x, q1.y);
            }
          } else {
            uint32_t x[4];  // rows g / g + 8 of pieces k, k + 1: bytes 4c .. 4c + 3
            ldsm4(ks + piece<P::kInner>(mr, k + mh), x);
            uint32_t a0, a1, a2, a3, e0, e1, e2, e3;
            widen4<FMT>(x[0], a0, a2);
            widen4<FMT>(x[1], a1, a3);
            widen4<FMT>(x[2], e0, e2);
            widen4<FMT>(x[3], e1, e3);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const uint2 q0 = qf_at(nb, k), q1 = qf_at(nb, k + 1);
              mma16<false>(s[nb], a0, a1, a2, a3, q0.x, q0.y);
              mma16<false>(s2[nb], e0, e1, e2, e3, q1.x, q1.y);
            }
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int u = 0; u < 4; ++u) s[nb][u] += s2[nb][u];
      }
      // ---- scores in log2 units; lane: tokens j0 + g, j0 + g + 8, rows 2c, 2c + 1
      float ksc[2] = {1.0f, 1.0f}, vsc[2] = {1.0f, 1.0f};
      if constexpr (!kBf) {
        const float* sc = reinterpret_cast<const float*>(smem + S::kOffScale) + ((warp * P::kStages + k_slot) * P::kSub + sub) * 2 * kRT;
        ksc[0] = sc[g], ksc[1] = sc[g + 8], vsc[0] = sc[16 + g], vsc[1] = sc[24 + g];
        if (!whole) {
          if (!R.seen_by_any(j0 + g)) vsc[0] = 0.0f;
          if (!R.seen_by_any(j0 + g + 8)) vsc[1] = 0.0f;
        }
      }
      if constexpr (P::kHalves) {
        __syncwarp();  // (every lane has read the stage)
        fetch(2 * n + P::kStages, k_slot);
        ok = wait(v_slot, v_phase);
        if (!ok) break;
      }
      if (!whole) {
        // tokens no row sees (past the context, before every window): their pages may hold anything
        constexpr int kPc = P::kRow / 16;
        bool wrote = false;
        for (int id = lane; id < kRT * kPc; id += 32) {
          const int r = id / kPc, ch = id % kPc;
          if (!R.seen_by_any(j0 + r)) {
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vs + piece<P::kInner>(r, ch)), "r"(0u) : "memory");
            wrote = true;
          }
        }
        if constexpr (TOKENS) {
          unsigned scale_odd = 0u;
          if constexpr (!kBf) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!(fabsf(vsc[h]) < INFINITY) && !s_range.seen_by_all(A, j0 + g + 8 * h)) scale_odd |= 1u << (g + 8 * h), vsc[h] = 0.0f;
            scale_odd = __reduce_or_sync(kFullMask, scale_odd);
          }
          if (FMT != GS_DTYPE_INT8 || scale_odd) wrote |= leave_odd_out<D, FMT>(A, s_range, vs, j0, scale_odd, &s_odd[0][0], &s_any);
        }
        if (wrote) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before the stage's next copy)
        __syncwarp();
      }
      bool move = !kBf && fmaxf(fabsf(vsc[0]), fabsf(vsc[1])) > vref;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int u = 0; u < 4; ++u) s[nb][u] *= kBf ? qf[nb][u & 1] : qf[nb][u & 1] * ksc[u >> 1];
        if (!whole) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int j = j0 + g + 8 * (u >> 1), p = pos[nb][u & 1];
            const bool seen = j <= p && (!A.window || j > p - A.window || j < A.sinks);
            s[nb][u] = seen ? s[nb][u] : -INFINITY;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) move = move || fmaxf(s[nb][h], s[nb][2 + h]) > m[nb][h] + kSlack;
      }
      if (__any_sync(kFullMask, move)) {
        // new references: every row's largest score so far, the largest V scale so far
        float vfac = 1.0f;
        if constexpr (!kBf) {
          float vm = fmaxf(fmaxf(vref, kLeastScale), fmaxf(fabsf(vsc[0]), fabsf(vsc[1])));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) vm = fmaxf(vm, __shfl_xor_sync(kFullMask, vm, d));
          vfac = vm > vref ? vref / vm : 1.0f;
          vref = vm;
          vinv = kPScale / vref;
        }
        float al[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mx = fmaxf(s[nb][h], s[nb][2 + h]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, d));
            mx = fmaxf(m[nb][h], mx);
            const float f = m[nb][h] == mx ? 1.0f : ex2(m[nb][h] - mx);
            m[nb][h] = mx;
            l[nb][h] *= f;
            al[nb][h] = f * vfac;
          }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[nb][k][u] *= al[nb][u & 1];
      }
      uint32_t pb[NB][2];
      const float vmul0 = vsc[0] * vinv, vmul1 = vsc[1] * vinv;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ref = m[nb][h] == -INFINITY ? 0.0f : m[nb][h];
          s[nb][h] = ex2(s[nb][h] - ref);
          s[nb][2 + h] = ex2(s[nb][2 + h] - ref);
          l[nb][h] += s[nb][h] + s[nb][2 + h];
        }
        if constexpr (kBf) {
          pb[nb][0] = transpose8(bf16x2(s[nb][0], s[nb][1]));
          pb[nb][1] = transpose8(bf16x2(s[nb][2], s[nb][3]));
        } else {
          pb[nb][0] = transpose8(half2_of(s[nb][0] * vmul0, s[nb][1] * vmul0));
          pb[nb][1] = transpose8(half2_of(s[nb][2] * vmul1, s[nb][3] * vmul1));
        }
      }
      // ---- O^T += V^T P^T
      if constexpr (kBf) {
        // address lane: token (lane & 7) + 8 · (lane >> 4), 8-value block (lane >> 3) & 1
        const int vt = (lane & 7) + ((lane >> 4) << 3), vh = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t a[4];
          ldsm4t(vs + piece<P::kInner>(vt, 2 * k + vh), a);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16<true>(o[nb][k], a[0], a[1], a[2], a[3], pb[nb][0], pb[nb][1]);
        }
      } else {
        // pairs of codes as 16-bit units: values 2g, 2g + 1 of a 16-value block for tokens 2c, 2c + 1
        const int vt = (lane & 7) + (((lane >> 3) & 1) << 3), vh = lane >> 4;
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t x[4];
          ldsm4t(vs + piece<P::kInner>(vt, k + vh), x);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t a0, a1, a2, a3;
            widen4<FMT>(__byte_perm(x[2 * w], 0u, 0x3120), a0, a1);
            widen4<FMT>(__byte_perm(x[2 * w + 1], 0u, 0x3120), a2, a3);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma16<false>(o[nb][k + w], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
          }
        }
      }
      if (last) {
        __syncwarp();
        fetch((P::kHalves ? 2 * n + 1 : n) + P::kStages, v_slot);
        break;
      }
    }
    if (!ok) break;
  }
  if (!ok) {
    // (bounded: what is in flight gets the same limit once more before the block ends)
    for (int s_ = 0; s_ < P::kStages; ++s_)
      for (uint32_t p_ = 0; p_ < 2; ++p_) mbar_wait(&s_bar[warp][s_], p_, kWaitNs / 8);
  }
  __syncthreads();  // (the rings are done with)

  // ---- join the warps
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[nb][h] += __shfl_xor_sync(kFullMask, l[nb][h], d);
      if (g == 0) {
        s_m[warp][8 * nb + 2 * c + h] = m[nb][h];
        s_l[warp][8 * nb + 2 * c + h] = l[nb][h];
      }
    }
  if (lane == 0) s_f[warp] = kBf ? 1.0f : vref / kPScale;
  float* os = reinterpret_cast<float*>(smem) + warp * kRows * (D + 4);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = kBf ? 16 * k + g + 8 * (u >> 1) : 16 * k + 2 * g + (u >> 1);
        os[(8 * nb + 2 * c + (u & 1)) * (D + 4) + d] = o[nb][k][u];
      }
  __syncthreads();
  float* oj = reinterpret_cast<float*>(smem);
  if (TOKENS && s_any) {  // (into warp 0's part: whatever is added to it is a NaN)
    for (int i = tid; i < R.rows * D; i += kRowsThreads)
      if (s_odd[i / D][i % D / 32] >> (i % 32) & 1u) oj[i / D * (D + 4) + i % D] = NAN;
    __syncthreads();
  }
  const bool alone = A.cluster == 1;
  // the (m, l, O) of a row's four values as the result
  auto put = [&](int r, int d, float M, float L, float4 acc) {
    int gq;
    const int t = R.token_of(A, r, gq);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const uint2 w = make_uint2(bf16x2(acc.x * inv, acc.y * inv), bf16x2(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(o_row(A, R, head, t, gq) + d) = w;
    if (A.lse && d == 0)
      A.lse[static_cast<int64_t>(R.q0 + t) * A.q_heads + head * A.group + gq] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  };
  for (int e = tid; e < R.rows * (D / 4); e += kRowsThreads) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) M = max_nan(M, s_m[w][r]);
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float f = ex2(s_m[w][r] - ref);
      L += f * s_l[w][r];
      const float fo = f * s_f[w];
      const float4 x = *reinterpret_cast<const float4*>(oj + (w * kRows + r) * (D + 4) + d);
      acc.x += fo * x.x, acc.y += fo * x.y, acc.z += fo * x.z, acc.w += fo * x.w;
    }
    if (alone) {
      put(r, d, M, L, acc);
    } else {
      // (into warp 0's part, whose same four values this thread has just read)
      *reinterpret_cast<float4*>(oj + r * (D + 4) + d) = acc;
      if (d == 0) s_ml[r][0] = M, s_ml[r][1] = L;
    }
  }
  if (alone) return;
  // ---- join the cluster: four values of a row per thread of its blocks (8 blocks have one for each)
  cluster_sync();
  const uint32_t rank = cluster_rank();
  const uint32_t o_at = smem_addr(oj), ml_at = smem_addr(&s_ml[0][0]);
  for (int e = static_cast<int>(rank) * kRowsThreads + tid; e - lane < R.rows * (D / 4); e += A.cluster * kRowsThreads) {
    const bool has = e < R.rows * (D / 4);
    const int r = has ? e / (D / 4) : 0, d = (e % (D / 4)) * 4;
    float2 ml[8];
    float4 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < A.cluster) {
        ml[k] = ld_rank2(in_rank(ml_at + r * 8, k));
        x[k] = ld_rank4(in_rank(o_at + (r * (D + 4) + d) * 4, k));
      }
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < A.cluster) M = max_nan(M, ml[k].x);
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < A.cluster) {
        const float f = ex2(ml[k].x - ref);
        L += f * ml[k].y;
        acc.x += f * x[k].x, acc.y += f * x[k].y, acc.z += f * x[k].z, acc.w += f * x[k].w;
      }
    if (A.splits == 1) {
      if (has) put(r, d, M, L, acc);
      continue;
    }
    // ---- several clusters (of 8: one turn of this loop): partial results to the workspace, each thread's
    // four values with their row's maximum and sum.  The same values are the same thread's in every cluster,
    // so a counter per warp tells which cluster's is last (nothing waits), and that one joins them.
    const int item = b * gridDim.y + blockIdx.y;
    auto part = [&](int k) { return (static_cast<int64_t>(item * A.splits + k) * kRows + r) * (D / 4) + d / 4; };
    if (has) {
      const int64_t at = part(blockIdx.x / A.cluster);
      __stcg(reinterpret_cast<float4*>(A.part_o) + at, acc);
      __stcg(reinterpret_cast<float2*>(A.part_ml) + at, make_float2(M, L));
    }
    __threadfence();
    __syncwarp();
    unsigned* ticket = A.tickets + item * 32 + static_cast<int>(rank) * kRowsWarps + warp;
    unsigned old = 0;
    if (lane == 0) old = atomicAdd(ticket, 1u);
    if (__shfl_sync(kFullMask, old, 0) != static_cast<unsigned>(A.splits - 1)) continue;
    __threadfence();
    if (lane == 0) *ticket = 0u;  // (for the next call)
    if (!has) continue;
    // (eight parts' loads together)
    M = -INFINITY;
    L = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = 0; k0 < A.splits; k0 += 8) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < A.splits) {
          ml[k] = __ldcg(reinterpret_cast<const float2*>(A.part_ml) + part(k0 + k));
          x[k] = __ldcg(reinterpret_cast<const float4*>(A.part_o) + part(k0 + k));
        }
      float mx = M;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < A.splits) mx = max_nan(mx, ml[k].x);
      const float at = mx == -INFINITY ? 0.0f : mx, back = ex2(M - at);
      L *= back;
      acc.x *= back, acc.y *= back, acc.z *= back, acc.w *= back;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < A.splits) {
          const float f = ex2(ml[k].x - at);
          L += f * ml[k].y;
          acc.x += f * x[k].x, acc.y += f * x[k].y, acc.z += f * x[k].z, acc.w += f * x[k].w;
        }
      M = mx;
    }
    put(r, d, M, L, acc);
  }
  cluster_sync();  // (no block leaves while its shared memory is read)
}

template <int D, int FMT, int NB, bool TOKENS>
cudaError_t go(const gs_kv_cache* c, AttnArgs a, cudaStream_t st) {
  constexpr int kRows = 8 * NB;
  using P = RowsPlan<D, FMT>;
  constexpr int smem = RowsSmem<D, FMT, NB>::kTotal;
  const int blocks = static_cast<int>((static_cast<int64_t>(a.max_q) * a.group + kRows - 1) / kRows);
  const int64_t items = static_cast<int64_t>(a.seqs) * a.kv.kv_heads * blocks;
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> held{0};  // clusters of 8 that the device holds at once (a GPU process runs on one kind of device)
  if (device_todo(done)) {
    cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<D, FMT, NB, TOKENS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t q{};
    cudaLaunchAttribute at{};
    q.gridDim = dim3(8 * 1024);
    q.blockDim = dim3(kRowsThreads);
    q.dynamicSmemBytes = smem;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 8, at.val.clusterDim.y = at.val.clusterDim.z = 1;
    q.attrs = &at;
    q.numAttrs = 1;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, attn_rows_kernel<D, FMT, NB, TOKENS>, &q);
    if (e != cudaSuccess) return e;
    held.store(n > 0 ? n : 1);
    mark_device_done(done);
  }
  // Blocks per context: one round of what the device holds (in clusters of 8, which have to find their SMs
  // in one GPC: fewer than the SMs alone would), each block with at least a stage a warp.  (Two sequences of 131072 tokens, 4 heads
  // of 128, bf16: two rounds take 19% longer.)  Up to 8 blocks are one cluster; more are
  // clusters of 8 whose partial results are joined.
  const int64_t tiles = most_tiles(a, kRT, kRows);
  int64_t want = 8ll * held.load() / items;
  const int64_t by_len = (tiles + kRowsWarps * P::kSub - 1) / (kRowsWarps * P::kSub);
  want = want > by_len ? by_len : want;
  int cluster = 1;
  while (cluster < 8 && cluster * 2 <= want) cluster *= 2;
  // More contexts than blocks at once: two blocks each all the same where a warp still has 32 tiles, since shorter blocks
  // leave a shorter last round (64 sequences of up to 8192 tokens, 8 heads, ragged: 2% less time at 128, 3% bf16 and 6% e4m3
  // at 256; all alike 1% and 4% less at 128, 1% and 5% more at 256; 128 sequences of 2000 tokens 6% more).
  if (cluster < 2 && tiles >= 2 * kRowsWarps * 32) cluster = 2;
  int64_t splits = want / cluster;
  const int64_t by_ws = static_cast<int64_t>(kAttnWsBytes) / (items * kRows * (D / 4) * 24);
  splits = splits > by_ws ? by_ws : splits;
  // (8 blocks of 128 threads have a thread for each four values of a block's rows)
  static_assert(kRows * (D / 4) <= 8 * kRowsThreads, "one turn of the join");
  if (splits < 1 || cluster < 8 || items * 32 * 4 > static_cast<int64_t>(kAttnTicketBytes)) splits = 1;
  a.cluster = cluster;
  a.splits = static_cast<int32_t>(splits);
  a.part_o = reinterpret_cast<float*>(c->ws);
  a.part_ml = a.part_o + items * splits * kRows * D;
  a.tickets = reinterpret_cast<unsigned*>(c->ws + kAttnWsBytes);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(splits * cluster), static_cast<unsigned>(a.kv.kv_heads * blocks), static_cast<unsigned>(a.seqs));
  if (cfg.gridDim.y > 65535) return cudaErrorInvalidConfiguration;
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(cluster);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attn_rows_kernel<D, FMT, NB, TOKENS>, a, *reinterpret_cast<const RowsMaps*>(c->maps + 256));
}

template <int D, int FMT, bool TOKENS>
cudaError_t go_nb(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
  if (rows <= 8) return go<D, FMT, 1, TOKENS>(c, a, st);
  // (32 rows of head_dim 256 would need 256 registers a thread for O alone: two passes of 16)
  if (rows <= 16 || D == 256) return go<D, FMT, 2, TOKENS>(c, a, st);
  return go<D, FMT, D == 256 ? 2 : 4, TOKENS>(c, a, st);
}
template <int D, int FMT>
cudaError_t go_tokens(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  return a.max_q > 1 ? go_nb<D, FMT, true>(c, a, st) : go_nb<D, FMT, false>(c, a, st);
}
template <int D>
cudaError_t go_fmt(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  switch (c->d.format) {
    case GS_DTYPE_BF16: return go_tokens<D, GS_DTYPE_BF16>(c, a, st);
    case GS_DTYPE_E4M3: return go_tokens<D, GS_DTYPE_E4M3>(c, a, st);
    default: return go_tokens<D, GS_DTYPE_INT8>(c, a, st);
  }
}

}  // namespace

cudaError_t launch_attn_rows(const gs_kv_cache* c, AttnArgs a, cudaStream_t st) {
  return c->d.head_dim == 64 ? go_fmt<64>(c, a, st) : c->d.head_dim == 128 ? go_fmt<128>(c, a, st) : go_fmt<256>(c, a, st);
}

}  // namespace gs
