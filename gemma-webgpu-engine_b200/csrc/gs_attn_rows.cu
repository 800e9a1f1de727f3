// Attention of few query rows over the paged cache (one decoded token, a few drafted ones),
// and the join of split contexts.
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
// Every warp walks its own tiles (every fourth of the block's split) through a private ring of
// shared-memory stages filled by 16-byte cp.async, so the loop has no block barrier and
// 96 to 128 KB are in flight per SM; warps meet once, at the end, to join their (m, l, O).
// Tokens hidden from every row of the block are filled with zeros instead of read.
//
// 8-bit codes are widened to float16 (exact for e4m3 and int8) in registers, K's scale
// multiplies the finished score, V's scale the weight: 2^(s - m) · (scale / largest scale so
// far) · 1024, which float16 holds to 11 bits down to 2^-24 of the largest; the factor is
// taken out of O at the end.  q is brought into float16's range by a power of two per row
// (bfloat16 has fewer mantissa bits: exact except for components below 2^-17 of the row's
// largest).  Beside a bf16 cache the weights are bf16, as q and v are.
#include "gs_attn.cuh"

namespace gs {
namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr int kRT = 16;  // tokens per warp tile
constexpr float kPScale = 1024.0f;

template <int D, int FMT>
struct RowsPlan {
  static constexpr int kEl = FMT == GS_DTYPE_BF16 ? 2 : 1;
  static constexpr int kRow = D * kEl;                         // bytes of one token's K (or V) row
  static constexpr int kChunks = kRow / 16;                    // 16-byte pieces per row: 4 .. 32
  static constexpr int kTileBytes = kRT * kRow;                // K or V of one tile
  static constexpr int kStage = 2 * kTileBytes + (FMT == GS_DTYPE_BF16 ? 0 : 2 * kRT * 4);
  static constexpr int kWant = 96 * 1024 / (kRowsWarps * kStage);
  static constexpr int kStages = kWant < 3 ? 3 : kWant > 6 ? 6 : kWant;
  static constexpr int kRing = kRowsWarps * kStages * kStage;
};

template <int D, int FMT, int NB>
constexpr int rows_smem() {
  constexpr int ring = RowsPlan<D, FMT>::kRing;
  constexpr int join = kRowsWarps * 8 * NB * (D + 4) * 4;
  return (ring > join ? ring : join) + NB * (D / 16) * 32 * 8;  // + Q fragments
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// Byte offset of 16-byte piece c of row r in a tile, pieces permuted so that 8 rows'
// equal pieces lie in different banks (rows of 64 bytes: two rows share 128 bytes).
template <int CH>
__device__ __forceinline__ uint32_t piece(int r, int c) {
  if constexpr (CH == 4) return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  else return static_cast<uint32_t>(r * CH * 16 + ((c ^ (r & 7)) << 4));
}

template <int D, int FMT, int NB>
__global__ void __launch_bounds__(kRowsThreads) attn_rows_kernel(const __grid_constant__ AttnArgs A) {
  using P = RowsPlan<D, FMT>;
  constexpr bool kBf = FMT == GS_DTYPE_BF16;
  constexpr int kRows = 8 * NB;
  constexpr int KS = D / 16;  // k-steps of the first product, 16-wide value blocks of the second
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int kQOff = rows_smem<D, FMT, NB>() - NB * KS * 32 * 8;
  uint2* qfrag = reinterpret_cast<uint2*>(smem + kQOff);  // [NB][KS][32]
  __shared__ float s_m[kRowsWarps][kRows], s_l[kRowsWarps][kRows], s_f[kRowsWarps];
  __shared__ float s_qf[kRows];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int b = blockIdx.z;
  const int head = blockIdx.y % A.kv.kv_heads, rb = blockIdx.y / A.kv.kv_heads;
  const int r0 = rb * kRows;
  const RowRange R = row_range<kRT>(A, b, r0, kRows);
  if (R.rows == 0) return;
  int nsplit = (R.tiles + A.chunk_tiles - 1) / A.chunk_tiles;
  nsplit = nsplit < 1 ? 1 : nsplit > A.splits ? A.splits : nsplit;
  const int split = blockIdx.x;
  if (split >= nsplit) return;
  const int i_end = split == nsplit - 1 ? R.tiles : (split + 1) * A.chunk_tiles;

  // ---- Q fragments (B operand: k = 2c.. of row n = g), once
  for (int nb = warp; nb < NB; nb += kRowsWarps) {
    const int r = 8 * nb + g;
    const bool live = r < R.rows;
    const int row = r0 + (live ? r : 0);
    const __nv_bfloat16* q = A.q + (R.q0 + row / A.group) * A.q_token + (head * A.group + row % A.group) * A.q_head;
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
      float mx = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(w[k][h])), fabsf(bf16_hi(w[k][h]))));
      mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 2));
      // 2^-e with 2^e <= mx < 2^(e + 1); exponents clamped so that both factors are normal
      int e = static_cast<int>((__float_as_uint(mx) >> 23) & 0xffu) - 127;
      e = mx == 0.0f || e > 127 ? 0 : max(e, -120);
      e = min(e, 120);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      f = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
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

  float qf[NB][2];
  int pos[NB][2];  // position of the lane's two rows
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * nb + 2 * c + h;
      qf[nb][h] = s_qf[r];
      pos[nb][h] = R.p0 + (r0 + min(r, R.rows - 1)) / A.group;
    }
  const int p_min = R.p0 + r0 / A.group, p_max = R.hi - 1;

  // ---- the warp's ring
  unsigned char* ring = smem + warp * (P::kStages * P::kStage);
  const uint32_t ring_s = smem_addr(ring);
  const int32_t* table = A.table + b * A.table_stride;
  const int per_page = A.kv.page_shift - 4;  // log2 of tiles per page
  int pages = 0;       // table entries of 32 consecutive tiles of this warp
  int pages_at = -1;   // which 32
  auto fetch = [&](int n, int stage) {  // the warp's n-th tile
    const int i = split * A.chunk_tiles + warp + n * kRowsWarps;
    if ((n >> 5) != pages_at) {
      pages_at = n >> 5;
      const int il = split * A.chunk_tiles + warp + ((pages_at << 5) + lane) * kRowsWarps;
      pages = -1;
      if (il < i_end) {
        const int col = R.tile(il) >> per_page;
        if (col < A.table_cols) pages = __ldg(table + col);
        if (pages < 0 || pages >= A.kv.pages) {
          pages = -1;
          atomicOr(A.flag, GS_KV_ERR_PAGE);
        }
      }
    }
    const int page = __shfl_sync(kFullMask, pages, n & 31);
    if (i < i_end) {
      const int j0 = R.tile(i) * kRT;
      const int off = j0 & ((1 << A.kv.page_shift) - 1);
      const int pg = page < 0 ? 0 : page;
      const unsigned char* kp = A.kv.at(false, pg, head, off);
      const unsigned char* vp = A.kv.at(true, pg, head, off);
      const uint32_t ks = ring_s + stage * P::kStage, vs = ks + P::kTileBytes;
#pragma unroll
      for (int u = 0; u < P::kChunks / 2; ++u) {
        const int id = lane + 32 * u, r = id / P::kChunks, ch = id % P::kChunks;
        const bool real = page >= 0 && R.seen_by_any(j0 + r);
        const uint32_t at = piece<P::kChunks>(r, ch);
        cp_async16(ks + at, kp + (static_cast<uint64_t>(static_cast<uint32_t>(r)) * A.kv.k_token + ch) * 16, real);
        cp_async16(vs + at, vp + (static_cast<uint64_t>(static_cast<uint32_t>(r)) * A.kv.v_token + ch) * 16, real);
      }
      if constexpr (!kBf) {
        const int r = lane & 15;
        const float* sc = A.kv.scale_at(lane >= 16, pg, head, off + r);
        cp_async4(ks + 2 * P::kTileBytes + lane * 4, sc, page >= 0 && R.seen_by_any(j0 + r));
      }
    }
    cp_commit();
  };

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
  float vref = 0.0f;  // largest V scale so far (8-bit)

  const int first = split * A.chunk_tiles + warp;
  const int n_tiles = i_end > first ? (i_end - first + kRowsWarps - 1) / kRowsWarps : 0;
#pragma unroll
  for (int s = 0; s < P::kStages - 1; ++s) fetch(s, s);
  int stage = 0;
  for (int n = 0; n < n_tiles; ++n) {
    cp_wait<P::kStages - 2>();
    __syncwarp();
    {
      int ns = stage + P::kStages - 1;
      ns = ns >= P::kStages ? ns - P::kStages : ns;
      fetch(n + P::kStages - 1, ns);
    }
    const uint32_t ks = ring_s + stage * P::kStage, vs = ks + P::kTileBytes;
    const int j0 = R.tile(first + n * kRowsWarps) * kRT;
    // ---- S^T = K Q^T
    float s[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[nb][u] = 0.0f;
    {
      float s2[NB][4];  // a second chain halves the dependent products
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int u = 0; u < 4; ++u) s2[nb][u] = 0.0f;
      const int mr = lane & 15, mh = lane >> 4;  // matrix row and half of this lane's address
#pragma unroll
      for (int k = 0; k < KS; k += 2) {
        if constexpr (kBf) {
          uint32_t a[4], a2[4];
          ldsm4(ks + piece<P::kChunks>(mr, 2 * k + mh), a);
          ldsm4(ks + piece<P::kChunks>(mr, 2 * k + 2 + mh), a2);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const uint2 q0 = qfrag[(nb * KS + k) * 32 + lane], q1 = qfrag[(nb * KS + k + 1) * 32 + lane];
            mma16<true>(s[nb], a[0], a[1], a[2], a[3], q0.x, q0.y);
            mma16<true>(s2[nb], a2[0], a2[1], a2[2], a2[3], q1.x, q1.y);
          }
        } else {
          uint32_t x[4];  // rows g / g + 8 of pieces k, k + 1: bytes 4c .. 4c + 3
          ldsm4(ks + piece<P::kChunks>(mr, k + mh), x);
          uint32_t a0, a1, a2, a3, e0, e1, e2, e3;
          widen4<FMT>(x[0], a0, a2);
          widen4<FMT>(x[1], a1, a3);
          widen4<FMT>(x[2], e0, e2);
          widen4<FMT>(x[3], e1, e3);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const uint2 q0 = qfrag[(nb * KS + k) * 32 + lane], q1 = qfrag[(nb * KS + k + 1) * 32 + lane];
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
      const float* sc = reinterpret_cast<const float*>(ring + stage * P::kStage + 2 * P::kTileBytes);
      ksc[0] = sc[g], ksc[1] = sc[g + 8], vsc[0] = sc[16 + g], vsc[1] = sc[24 + g];
    }
    const bool whole = j0 + kRT - 1 <= p_min && (!A.window || j0 > p_max - A.window || j0 + kRT <= A.sinks);
    float mx[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s[nb][u] *= qf[nb][u & 1] * ksc[u >> 1];
      if (!whole) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + g + 8 * (u >> 1), p = pos[nb][u & 1];
          const bool seen = j <= p && (!A.window || j > p - A.window || j < A.sinks);
          s[nb][u] = seen ? s[nb][u] : -INFINITY;
        }
      }
      mx[nb][0] = max_nan(s[nb][0], s[nb][2]);
      mx[nb][1] = max_nan(s[nb][1], s[nb][3]);
    }
    float vmx = vsc[0];
    if constexpr (!kBf) vmx = fmaxf(vsc[0], vsc[1]);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) mx[nb][h] = max_nan(mx[nb][h], __shfl_xor_sync(kFullMask, mx[nb][h], d));
      if constexpr (!kBf) vmx = fmaxf(vmx, __shfl_xor_sync(kFullMask, vmx, d));
    }
    float vfac = 1.0f, vmul0 = 1.0f, vmul1 = 1.0f;
    if constexpr (!kBf) {
      const float vnew = fmaxf(vref, vmx);
      if (vnew > vref) {
        vfac = vref / vnew;
        vref = vnew;
      }
      const float inv = vref > 0.0f ? kPScale / vref : 0.0f;
      vmul0 = vsc[0] * inv;
      vmul1 = vsc[1] * inv;
    }
    uint32_t pb[NB][2];
    float al[NB][2];
    bool same = vfac == 1.0f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mn = max_nan(m[nb][h], mx[nb][h]);
        const float ref = mn == -INFINITY ? 0.0f : mn;
        al[nb][h] = ex2(m[nb][h] - ref);
        m[nb][h] = mn;
        s[nb][h] = ex2(s[nb][h] - ref);
        s[nb][2 + h] = ex2(s[nb][2 + h] - ref);
        l[nb][h] = l[nb][h] * al[nb][h] + (s[nb][h] + s[nb][2 + h]);
        same = same && al[nb][h] == 1.0f;
        al[nb][h] *= vfac;
      }
      if constexpr (kBf) {
        pb[nb][0] = transpose8(bf16x2(s[nb][0], s[nb][1]));
        pb[nb][1] = transpose8(bf16x2(s[nb][2], s[nb][3]));
      } else {
        pb[nb][0] = transpose8(half2_of(s[nb][0] * vmul0, s[nb][1] * vmul0));
        pb[nb][1] = transpose8(half2_of(s[nb][2] * vmul1, s[nb][3] * vmul1));
      }
    }
    if (!__all_sync(kFullMask, same)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int u = 0; u < 4; ++u) o[nb][k][u] *= al[nb][u & 1];
    }
    // ---- O^T += V^T P^T
    if constexpr (kBf) {
      // address lane: token (lane & 7) + 8 · (lane >> 4), 8-value block (lane >> 3) & 1
      const int vt = (lane & 7) + ((lane >> 4) << 3), vh = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t a[4];
        ldsm4t(vs + piece<P::kChunks>(vt, 2 * k + vh), a);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16<true>(o[nb][k], a[0], a[1], a[2], a[3], pb[nb][0], pb[nb][1]);
      }
    } else {
      // pairs of codes as 16-bit units: values 2g, 2g + 1 of a 16-value block for tokens 2c, 2c + 1
      const int vt = (lane & 7) + (((lane >> 3) & 1) << 3), vh = lane >> 4;
#pragma unroll
      for (int k = 0; k < KS; k += 2) {
        uint32_t x[4];
        ldsm4t(vs + piece<P::kChunks>(vt, k + vh), x);
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
    stage = stage + 1 == P::kStages ? 0 : stage + 1;
    __syncwarp();  // the stage just read is the next fetch's
  }
  cp_wait<0>();
  __syncthreads();

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
  const float* oj = reinterpret_cast<const float*>(smem);
  const bool whole_context = nsplit == 1;
  const int64_t part = (static_cast<int64_t>(b) * gridDim.y + blockIdx.y) * A.splits + split;
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
    if (whole_context) {
      const int row = r0 + r;
      const int64_t t = R.q0 + row / A.group;
      const int hq = head * A.group + row % A.group;
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      const uint2 w = make_uint2(bf16x2(acc.x * inv, acc.y * inv), bf16x2(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2*>(A.out + t * A.o_token + hq * A.o_head + d) = w;
      if (A.lse && d == 0) A.lse[t * A.q_heads + hq] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    } else {
      *reinterpret_cast<float4*>(A.part_o + (part * kRows + r) * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(A.part_ml + (part * kRows + r) * 2) = make_float2(M, L);
    }
  }
}

// One block per query row: its splits' (m, l, O) joined as the warps' are above.  kTile and
// rows per block as in the kernel that wrote them, so that the number of splits agrees.
template <int D, int kTile>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs A, int rows_per_block) {
  constexpr int kVec = D / 4, kParts = 128 / kVec;  // threads across head_dim, splits in parallel
  __shared__ float4 s_acc[128];
  __shared__ float s_red[4], s_lse[4];
  const int b = blockIdx.z, head = blockIdx.y % A.kv.kv_heads, rb = blockIdx.y / A.kv.kv_heads;
  const int r = blockIdx.x, r0 = rb * rows_per_block, tid = threadIdx.x;
  const RowRange R = row_range<kTile>(A, b, r0, rows_per_block);
  if (r >= R.rows) return;
  int nsplit = (R.tiles + A.chunk_tiles - 1) / A.chunk_tiles;
  nsplit = nsplit < 1 ? 1 : nsplit > A.splits ? A.splits : nsplit;
  if (nsplit == 1) return;
  const int64_t part0 = (static_cast<int64_t>(b) * gridDim.y + blockIdx.y) * A.splits;
  const float* ml = A.part_ml + (part0 * rows_per_block + r) * 2;
  const int64_t step = static_cast<int64_t>(rows_per_block);
  float M = -INFINITY;
  for (int s = tid; s < nsplit; s += 128) M = max_nan(M, ml[s * step * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(kFullMask, M, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = M;
  __syncthreads();
  M = max_nan(max_nan(s_red[0], s_red[1]), max_nan(s_red[2], s_red[3]));
  const float ref = M == -INFINITY ? 0.0f : M;
  float L = 0.0f;
  for (int s = tid; s < nsplit; s += 128) {
    const float2 v = *reinterpret_cast<const float2*>(ml + s * step * 2);
    L += ex2(v.x - ref) * v.y;
  }
  L = warp_sum_f(L);
  if ((tid & 31) == 0) s_lse[tid >> 5] = L;
  const int pv = tid / kVec, d = (tid % kVec) * 4;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s = pv; s < nsplit; s += kParts) {
    const float f = ex2(ml[s * step * 2] - ref);
    const float4 x = *reinterpret_cast<const float4*>(A.part_o + ((part0 + s) * rows_per_block + r) * D + d);
    acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid >= kVec) return;
#pragma unroll
  for (int p = 1; p < kParts; ++p) {
    const float4 x = s_acc[p * kVec + tid];
    acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
  }
  L = s_lse[0] + s_lse[1] + s_lse[2] + s_lse[3];
  const int row = r0 + r;
  const int64_t t = R.q0 + row / A.group;
  const int hq = head * A.group + row % A.group;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint2*>(A.out + t * A.o_token + hq * A.o_head + d) =
      make_uint2(bf16x2(acc.x * inv, acc.y * inv), bf16x2(acc.z * inv, acc.w * inv));
  if (A.lse && d == 0) A.lse[t * A.q_heads + hq] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

template <int D, int FMT, int NB>
cudaError_t go(const gs_kv_cache* c, AttnArgs a, cudaStream_t st) {
  constexpr int kRows = 8 * NB;
  const int blocks = static_cast<int>((static_cast<int64_t>(a.max_q) * a.group + kRows - 1) / kRows);
  const int64_t items = static_cast<int64_t>(a.seqs) * a.kv.kv_heads * blocks;
  // Splits: enough blocks to fill the SMs about four times over (contexts are ragged), each
  // at least 16 tiles (256 tokens, four a warp), within the workspace.
  const int64_t tiles = most_tiles(a, kRT, kRows);
  int64_t splits = (4ll * c->num_sms + items - 1) / items;
  const int64_t by_len = (tiles + 15) / 16;
  splits = splits > by_len ? by_len : splits;
  const int64_t slot = static_cast<int64_t>(kRows) * (D + 2) * 4;
  const int64_t by_ws = static_cast<int64_t>(kAttnWsBytes) / (items * slot);
  splits = splits > by_ws ? by_ws : splits;
  if (splits < 1) splits = 1;
  int64_t chunk = tiles > 0 ? (tiles + splits - 1) / splits : 1;
  chunk = (chunk + kRowsWarps - 1) / kRowsWarps * kRowsWarps;
  a.chunk_tiles = static_cast<int32_t>(chunk);
  a.splits = static_cast<int32_t>(tiles > 0 ? (tiles + chunk - 1) / chunk : 1);
  a.part_o = reinterpret_cast<float*>(c->ws);
  a.part_ml = a.part_o + items * a.splits * kRows * D;
  constexpr int smem = rows_smem<D, FMT, NB>();
  static std::atomic<uint64_t> done{0};
  if (device_todo(done)) {
    const cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<D, FMT, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    mark_device_done(done);
  }
  const dim3 grid(static_cast<unsigned>(a.splits), static_cast<unsigned>(a.kv.kv_heads * blocks), static_cast<unsigned>(a.seqs));
  if (grid.y > 65535) return cudaErrorInvalidConfiguration;
  attn_rows_kernel<D, FMT, NB><<<grid, kRowsThreads, smem, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || a.splits == 1) return e;
  return launch_attn_join(a, D, kRows, blocks, kRT, st);
}

template <int D, int FMT>
cudaError_t go_nb(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
  return rows <= 8 ? go<D, FMT, 1>(c, a, st) : go<D, FMT, 2>(c, a, st);
}
template <int D>
cudaError_t go_fmt(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  switch (c->d.format) {
    case GS_DTYPE_BF16: return go_nb<D, GS_DTYPE_BF16>(c, a, st);
    case GS_DTYPE_E4M3: return go_nb<D, GS_DTYPE_E4M3>(c, a, st);
    default: return go_nb<D, GS_DTYPE_INT8>(c, a, st);
  }
}

}  // namespace

cudaError_t launch_attn_rows(const gs_kv_cache* c, AttnArgs a, cudaStream_t st) {
  return c->d.head_dim == 64 ? go_fmt<64>(c, a, st) : c->d.head_dim == 128 ? go_fmt<128>(c, a, st) : go_fmt<256>(c, a, st);
}

cudaError_t launch_attn_join(const AttnArgs& a, int head_dim, int rows_per_block, int row_blocks, int tile, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows_per_block), static_cast<unsigned>(a.kv.kv_heads * row_blocks),
                  static_cast<unsigned>(a.seqs));
  auto run = [&](auto kern) {
    kern<<<grid, 128, 0, st>>>(a, rows_per_block);
    return cudaGetLastError();
  };
  if (tile == 16) {
    return head_dim == 64 ? run(attn_join_kernel<64, 16>) : head_dim == 128 ? run(attn_join_kernel<128, 16>) : run(attn_join_kernel<256, 16>);
  }
  return head_dim == 64 ? run(attn_join_kernel<64, 128>) : head_dim == 128 ? run(attn_join_kernel<128, 128>) : run(attn_join_kernel<256, 128>);
}

}  // namespace gs
