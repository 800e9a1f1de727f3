// Attention of many query rows over the paged cache (prompt chunks) on the tcgen05 tensor cores.
//
// A block owns kTileRows query rows of one key/value head (new tokens × heads of the group,
// so the group shares every cached byte) and walks its context in tiles of 128 tokens:
//   S = Q K^T (128 x 128, float32 in tensor memory), weights P = 2^(c S - c m) in bf16 written
//   over S, O += P V (A operand from tensor memory), one row per softmax thread, so that the
//   row's maximum and sum need no shuffles.
// The reference point m is moved only when a tile's maximum passes it by 2^8: float32 sums and
// bf16 weights hold 2^8 as well as 1, and rescaling O (128 x D in tensor memory) then happens a
// few times a row instead of once a tile.
//
// Bound: 4 D multiply-adds a score at 4096 a clock and SM, against one 2^x a score at 16 a
// clock: at D = 128 both take 1024 clocks per 128 x 128 tile, so two query tiles take turns
// (D <= 128): one tile's products run under the other's softmax.  At D = 256 the products take twice
// as long as the softmax and the output alone fills half of tensor memory: one query tile, two
// score buffers.
//
// Measured (2048 new tokens over 16384, calls in a row, the clock at 1.7 GHz under the 1000 W cap): 32 / 8 heads of 128 bf16
// 516 us, 1.0 PFLOP/s, both the tensor pipe and the 2^x unit 55 % busy (starting the second product at three quarters of P
// gained nothing: 1% more time); of 64 377 us; 16 / 8 heads of 256 510 us, 1.0 PFLOP/s, bound by what L2 delivers of K and V;
// e4m3 of 64 518, of 128 661, of 256 500 us, int8 530, 704, 532 us: widening and softmax share the issue slots and shared
// memory.  Six ragged chunks of up to 1500 tokens, windows of 1024, heads of 256: e4m3 223 us, bf16 200 us; an
// item's 11 tiles take 25 of its 38 us, query loads from HBM 4, output 3.
//
// Tensor memory (512 columns): S0 at 0, S1 at 128, O0 at 256, O1 at 256 + D.
// Warps: softmax warpgroup(s) first (warp % 4 = its tensor-memory lanes), then the MMA issuer and the
// loader (TMA boxes; bf16 pages go straight to the swizzled operand layout), then, beside an 8-bit
// cache, four warps that widen the loaded codes to float16 operands (exact).  K's scale multiplies the
// float32 score, V's the float16 weight.  Q is brought into float16 by a power of two per row.
// Order of products and of shared-memory stages: K(0) .. K(SB-1), then V(j), K(j + SB) for each j:
// P(j) overlays S(j), and the tensor core takes one thread's products in order, so S(j + SB) is
// issued right behind the product that reads P(j).
// Every wait is bounded (1 s); a wait that runs out sets GS_KV_ERR_TIMEOUT, ends the block's loops,
// waits (bounded) for copies and products in flight and frees tensor memory.
#include <cuda.h>

#include "gs_attn.cuh"

namespace gs {
namespace {

constexpr int kTT = 128;        // context tokens per tile
constexpr int kMostRows = 256;  // query rows of a group of blocks, at most

// CG: blocks that share a context's tiles (tcgen05 cta_group).  Two blocks of a cluster each hold half of
// every K tile (tokens) and V tile (columns), and one product covers the query rows of both: half the L2
// reads, shared memory traffic and widening per row.
template <int D, int FMT, int CG>
struct TilePlan {
  static constexpr bool kBf = FMT == GS_DTYPE_BF16;
  static constexpr int NQ = D == 256 ? 1 : 2;   // query tiles of 128 rows
  static constexpr int SB = D == 256 ? 2 : 1;   // score buffers per query tile
  static constexpr int kRows = 128 * NQ;        // query rows of a block
  static constexpr int kPer = D == 256 && CG == 1 ? 2 : 1;                   // stages per K or V tile
  static constexpr int kKTok = kTT / CG, kKCols = kPer == 2 ? 128 : D;       // one K stage: tokens x columns
  static constexpr int kVTok = kPer == 2 ? 64 : kTT, kVCols = D / CG;        // one V stage
  static constexpr int kStage = kKTok * kKCols * 2;
  static constexpr int kStages = kBf ? (D == 64 ? 8 : kStage == 16384 ? 10 : 5) : (D == 64 ? 6 : kStage == 16384 ? 5 : 3);
  static constexpr int kEl = kBf ? 2 : 1;
  static constexpr int kKInner = kKCols * kEl < 128 ? kKCols * kEl : 128;  // bytes of a row in one TMA box
  static constexpr int kVInner = kVCols * kEl < 128 ? kVCols * kEl : 128;
  static constexpr int kRawStage = kBf ? 0 : kStage / 2;        // codes of one stage
  static constexpr int kRawStages = kBf ? 0 : kStage == 16384 ? 6 : 3;
  // Tiles whose scales are held: K(j + 8) is loaded only after the codes of an earlier V were taken
  // (raw and operand stages reach at most 6 tiles ahead of the products).
  static constexpr int kScaleSlots = 8;
  static constexpr int kQ = NQ * 128 * D * 2;
  static constexpr int kOffStage = kQ;
  static constexpr int kOffRaw = kOffStage + kStages * kStage;
  static constexpr int kOffScale = kOffRaw + kRawStages * kRawStage;       // [slot][K, V][kTT] float
  static constexpr int kOffQf = kOffScale + (kBf ? 0 : kScaleSlots * 2 * kTT * 4);  // [kRows] float
  static constexpr int kOffRef = kOffQf + (kBf ? 0 : kRows * 4);           // [slot][widening warp] float
  static constexpr int kOffBar = kOffRef + (kBf ? 0 : 128);
  static constexpr int kOffWalk = kOffBar + 512;                           // (balanced) a Walk per warp
  static constexpr bool kBalance = NQ == 2 && (kBf || D == 64);
  static constexpr int kWalks = !kBalance ? 0 : kBf ? 1536 : 2304;
  static constexpr int kSmem = kOffWalk + kWalks + 1024;         // alignment slack
  // Warpgroups: softmax (NQ), then the MMA issuer with the TMA loader beside it, then the widening
  // loaders.  Registers a thread: a row of 128 scores lives in its softmax thread; the shares add
  // up to what the block is launched with.
  static constexpr int kSoftWarps = 4 * NQ, kMmaWarp = kSoftWarps, kLoadWarp = kSoftWarps + 1, kWidenWarp = kSoftWarps + 4;
  // (At head_dim 256 eight warps widen: four take 1400 cycles a stage and the products wait for them.)
  static constexpr int kWidenGroups = kBf ? 0 : NQ == 1 ? 2 : 1, kWideners = kBf ? 128 : 128 * kWidenGroups;
  static constexpr int kGroups = NQ + 1 + kWidenGroups;
  static constexpr int kThreads = 128 * kGroups;
  static constexpr int kRegs = kGroups == 2 ? 248 : kGroups == 3 ? 168 : 128;
  static constexpr int kSoftRegs = kGroups == 2 ? 248 : kBf ? 216 : NQ == 1 ? 224 : 200;
  static constexpr int kMmaRegs = kGroups == 2 ? 248 : kBf ? 72 : NQ == 1 ? 64 : 40;
  static constexpr int kLoadRegs = kBf ? 0 : NQ == 1 ? 112 : 72;  // (widening warps)
  static_assert(NQ * kSoftRegs + kMmaRegs + kWidenGroups * kLoadRegs == kGroups * kRegs, "register shares");
  static_assert(kVTok * kVCols * 2 == kStage, "K and V stages are one size");
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// tcgen05.mma kind::f16: f32 accumulators, bf16 or f16 operands (both the same), M = 128
// rows a block.
template <bool BF16, int CG>
constexpr uint32_t kIdescQK = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((128u >> 3) << 17) | ((128u * CG >> 4) << 24);
template <int D, bool BF16, int CG>
constexpr uint32_t kIdescPV = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) |
                              ((static_cast<uint32_t>(D) >> 3) << 17) | ((128u * CG >> 4) << 24);  // bit 16: B MN-major (V's token rows)

// 128-byte swizzled operands.  K-major: 8-row groups 1024 bytes apart (stride offset).  MN-major:
// blocks of 64 columns `lead` bytes apart (leading offset), 8-token groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lead) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
#define GS_TC_MMA(GROUP, A_OPERAND)                                                                                   \
  "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], " A_OPERAND    \
  ", %2, %3, p;\n\t}\n"
template <int CG>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1) asm volatile(GS_TC_MMA("1", "%1")::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
  else asm volatile(GS_TC_MMA("2", "%1")::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1) asm volatile(GS_TC_MMA("1", "[%1]")::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
  else asm volatile(GS_TC_MMA("2", "[%1]")::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// Completion of the products issued so far, on the barrier of every block of the group.
template <int CG>
__device__ __forceinline__ void commit_to(uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}
__device__ __forceinline__ void arrive_on(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Arrival on the first block's barrier (the one that issues the products).  It releases at block scope: what the products
// read lies in the arriving block's own shared memory, handed to the async proxy by its writers before, or in tensor
// memory, ordered by the tcgen05 fences.  At cluster scope each arrival waits for all of the thread's memory traffic, 1000
// clocks a tile (2048 x 16384 tokens, heads of 256: 19% more time).
template <int CG>
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
  if constexpr (CG == 1) {
    arrive_on(bar);
  } else {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(bar)));
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
  }
}
// Bounded wait on a barrier that the other block may have arrived on.
template <int CG>
__device__ __forceinline__ bool wait_group(uint64_t* bar, uint32_t parity) {
  if constexpr (CG == 1) {
    return mbar_wait(bar, parity, kWaitNs);
  } else {
    uint64_t t0 = 0;
    for (;;) {
      uint32_t done;
      asm volatile(
          "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
          : "=r"(done)
          : "r"(smem_addr(bar)), "r"(parity)
          : "memory");
      if (done) return true;
      const uint64_t t = globaltimer_ns();
      if (t0 == 0) t0 = t;
      else if (t - t0 > kWaitNs) return false;
    }
  }
}
template <int CG>
__device__ __forceinline__ void group_sync() {
  if constexpr (CG == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool elected() {
  uint32_t p = 0;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.b32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int tok, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(tok), "r"(head), "r"(page), "r"(smem_addr(bar))
      : "memory");
}
// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tm_ld32(uint32_t a, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// This warpgroup's registers a thread, from `From` at launch.
template <int From, int To>
__device__ __forceinline__ void set_regs() {
  if constexpr (To > From) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(To));
  if constexpr (To < From) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(To));
}

// Four 8-bit codes as two float16 pairs, exact.  int8: byte + 128 becomes the low mantissa of
// 1024, minus 1152.
template <int FMT>
__device__ __forceinline__ uint2 widen_half(uint32_t codes) {
  uint2 r;
  if constexpr (FMT == GS_DTYPE_E4M3) {
    r.x = e4m3x2_half2(codes & 0xffffu);
    r.y = e4m3x2_half2(codes >> 16);
  } else {
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(l), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(h), "r"(0x64806480u));
  }
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
struct TileMaps {
  CUtensorMap k, v;
};

// One stretch of context tiles of one item (sequence, key/value head, query rows of a group of blocks).
struct Piece {
  RowRange R;
  int b, head;
  int t_begin, n;  // context tiles
  int part;        // partial-result slot, or -1: the whole context is here
  int first, pieces;  // (balanced, pieces > 0) first group with a piece of the item, and how many have one
};

// The pieces of a group of blocks.  Fixed: grid (split, head and row block, sequence), one
// piece.  Balanced: the items in a row (head by head, sequence by sequence), measured in tiles, are cut into as many equal stretches as there are groups; a group walks its stretch, and an
// item cut in two or more is joined by whoever finishes its last piece.
struct Cursor {
  int64_t x, x1, total;
  int head, b, rb, off;
  int me, groups, blocks;
  __device__ __forceinline__ int group_of(int64_t at) const { return static_cast<int>(((at + 1) * groups - 1) / total); }
};

// Cursor and piece of a warp lie in shared memory (a softmax thread has no registers for them); the whole warp
// takes the step and one lane writes it down.
struct Walk {
  Cursor cursor;
  Piece piece;
};

template <int ROWS, bool BAL>
__device__ __forceinline__ bool next_piece(const AttnArgs& A, Cursor& c, Piece& p) {
  if constexpr (!BAL) {
    if (c.x >= c.x1) return false;
    c.x = c.x1;
    p.R = row_range<kTT>(A, c.b, c.rb * ROWS, ROWS, threadIdx.x == 0);
    int nsplit = (p.R.tiles + A.chunk_tiles - 1) / A.chunk_tiles;
    nsplit = nsplit < 1 ? 1 : nsplit > A.splits ? A.splits : nsplit;
    if (p.R.rows == 0 || c.off >= nsplit) return false;
    p.b = c.b, p.head = c.head;
    p.t_begin = c.off * A.chunk_tiles;
    p.n = (c.off == nsplit - 1 ? p.R.tiles : p.t_begin + A.chunk_tiles) - p.t_begin;
    p.part = nsplit == 1 ? -1 : ((c.b * c.blocks + c.rb) * A.kv.kv_heads + c.head) * A.splits + c.off;
    p.pieces = 0;
    return true;
  }
  while (c.x < c.x1 && c.head < A.kv.kv_heads) {
    p.R = row_range<kTT>(A, c.b, c.rb * ROWS, ROWS, false);  // (noted when the tiles were counted)
    const int w = p.R.rows == 0 ? 0 : max(p.R.tiles, 1);
    const int take = static_cast<int>(min(static_cast<int64_t>(w - c.off), c.x1 - c.x));
    const bool got = take > 0;
    if (got) {
      p.b = c.b, p.head = c.head;
      p.t_begin = c.off;
      p.n = min(take, p.R.tiles);
      p.part = -1;
      p.pieces = 0;
      if (take < w) {
        const int64_t start = c.x - c.off;
        p.first = c.group_of(start);
        p.pieces = c.group_of(start + w - 1) - p.first + 1;
        p.part = 2 * c.me + (c.me == p.first ? 1 : 0);  // the stretch's last item, or its first
      }
      c.x += take;
      c.off += take;
    }
    if (c.off >= w) {
      c.off = 0;
      if (++c.rb == c.blocks) {
        c.rb = 0;
        if (++c.b == A.seqs) c.b = 0, ++c.head;
      }
    }
    if (got) return true;
  }
  return false;
}

template <int ROWS>
__device__ __forceinline__ bool next_piece(const AttnArgs& A, Walk* walk, int lane) {
  __syncwarp();
  Cursor c = walk->cursor;
  Piece p;
  const bool got = next_piece<ROWS, true>(A, c, p);
  __syncwarp();
  if (lane == 0) {
    walk->cursor = c;
    if (got) walk->piece = p;
  }
  __syncwarp();
  return got;
}

// Row of its query tile that warp `quad` brings as its i-th of 32: a few neighbouring rows at a time (as many as the
// 32 lanes hold 16-byte pieces of), the four warps in turn.
template <int D>
__device__ __forceinline__ constexpr int q_slot(int quad, int i) {
  constexpr int kPerWarp = 256 / D;
  return i / kPerWarp * (4 * kPerWarp) + quad * kPerWarp + i % kPerWarp;
}

// Item i of the stage order of n tiles: K(0) .. K(SB - 1), then V(j), K(j + SB) in turn.
template <int SB>
__device__ __forceinline__ void stage_item(int i, int n, bool& value, int& j) {
  const int lead = SB < n ? SB : n;
  if (i < lead) {
    value = false, j = i;
    return;
  }
  const int k = i - lead;
  if (k < 2 * (n - SB)) value = (k & 1) == 0, j = value ? k >> 1 : (k >> 1) + SB;
  else value = true, j = k - (n - SB > 0 ? n - SB : 0);
}

template <int D, int FMT, int CG, bool BAL>
__global__ void __launch_bounds__(TilePlan<D, FMT, CG>::kThreads, 1)
    attn_tile_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TileMaps maps) {
  using P = TilePlan<D, FMT, CG>;
  constexpr int NQ = P::NQ, SB = P::SB;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + P::kOffBar);
  uint64_t* full = bars;                   // [kStages]
  uint64_t* freeb = full + P::kStages;     // [kStages]
  uint64_t* s_full = freeb + P::kStages;   // [2]: score buffer (query tile, or tile parity)
  uint64_t* p_full = s_full + 2;           // [2]
  uint64_t* o_done = p_full + 2;           // [NQ]
  uint64_t* m_done = o_done + 2;
  uint64_t* q_full = m_done + 2;                    // every query tile of the group is in shared memory
  uint64_t* raw_full = q_full + 1;                  // [kRawStages]
  uint64_t* raw_free = raw_full + P::kRawStages;    // [kRawStages]
  uint64_t* peer_full = raw_free + P::kRawStages;   // [kStages] (CG 2, first block): the other block's stage is there
  uint64_t* looked = peer_full + (CG == 2 ? P::kStages : 0);  // [2] (fixed, bf16): V of the tokens that some rows' windows have left, or
  int* odd_v = reinterpret_cast<int*>(looked + 2);            // that some rows do not reach, has been looked at; whether there is what is not finite
  static_assert(8 * (2 * P::kStages + 2 * P::kRawStages + (CG == 2 ? P::kStages : 0) + 12) <= 512, "barriers");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(m_done + 1);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kGroupRows = CG * P::kRows;
  const int rank = CG == 1 ? 0 : static_cast<int>(blockIdx.x) & 1;  // (clusters of CG blocks along x)
  Cursor start;
  start.blocks = A.row_blocks;
  start.me = static_cast<int>(blockIdx.x) / CG;
  start.groups = static_cast<int>(gridDim.x) / CG;
  if constexpr (!BAL) {
    start.b = blockIdx.z;
    start.head = blockIdx.y / A.row_blocks;
    start.rb = A.row_blocks - 1 - static_cast<int>(blockIdx.y % A.row_blocks);  // longest contexts first
    start.off = start.me;  // (the split)
    start.x = 0, start.x1 = 1, start.total = 1;
  } else {
    // every unit's (sequence, row block) tiles, their running sum, and where this group's stretch begins
    int* sums = reinterpret_cast<int*>(sm + P::kOffStage);  // [units + 1]
    for (int u = tid; u < A.units; u += P::kThreads) {
      const RowRange R = row_range<kTT>(A, u / A.row_blocks, u % A.row_blocks * kGroupRows, kGroupRows, blockIdx.x == 0);
      sums[u] = R.rows == 0 ? 0 : max(R.tiles, 1);
    }
    __syncthreads();
    if (warp == 0) {
      int carry = 0;
      for (int u0 = 0; u0 < A.units; u0 += 32) {
        const int v = u0 + lane < A.units ? sums[u0 + lane] : 0;
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(kFullMask, x, o);
          if (lane >= o) x += y;
        }
        if (u0 + lane < A.units) sums[u0 + lane] = carry + x - v;
        carry += __shfl_sync(kFullMask, x, 31);
      }
      if (lane == 0) sums[A.units] = carry;
    }
    __syncthreads();
    const int per_head = sums[A.units];
    start.total = static_cast<int64_t>(per_head) * A.kv.kv_heads;
    // (The host chose the path by the bounds max_q and max_kv.  Of fewer tiles than groups each goes to one group and the
    // groups past them have nothing: a group in between without a tile would be counted among an item's pieces.)
    start.groups = static_cast<int>(min(static_cast<int64_t>(start.groups), max(start.total, static_cast<int64_t>(1))));
    start.x = start.me * start.total / start.groups;
    start.x1 = start.me < start.groups ? (start.me + 1) * start.total / start.groups : start.x;
    int at = 0;
    start.head = 0;
    start.off = 0;
    if (start.x < start.x1) {
      start.head = static_cast<int>(start.x / per_head);
      const int rem = static_cast<int>(start.x - static_cast<int64_t>(start.head) * per_head);
      int lo = 0, hi = A.units;  // the last unit whose sum is at most rem
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= rem) lo = mid;
        else hi = mid;
      }
      at = lo;
      start.off = rem - sums[at];
    }
    start.b = at / A.row_blocks;
    start.rb = at % A.row_blocks;
    fence_async();  // (the loads that overwrite the sums)
  }
  // (balanced: a Walk per warp in shared memory, two warps idle; fixed: the one piece in registers)
  Walk* walk = reinterpret_cast<Walk*>(sm + P::kOffWalk) + (warp <= P::kLoadWarp ? warp : warp - 2);
  Piece only;
  {
    Cursor c = start;
    if (!next_piece<kGroupRows, BAL>(A, c, only)) return;  // (the whole group)
    if constexpr (BAL) {
      static_assert(static_cast<int>(sizeof(Walk)) * (P::kThreads / 32 - 2) <= P::kWalks, "a Walk per warp");
      if (lane == 0 && (warp <= P::kLoadWarp || warp >= P::kWidenWarp)) {
        walk->cursor = c;
        walk->piece = only;
      }
      __syncwarp();
    }
  }
  const Piece& pc = BAL ? walk->piece : only;
  // (A piece of at most 128 rows leaves the second query tile out: 8 sequences of 4000 tokens, 128 rows of 128, 9% less time
  // bf16, 18% int8; the counting costs chunks over 8-bit caches with heads of 64 3%.)
  auto query_tiles = [&]() { return NQ == 2 && pc.R.rows <= 128 ? 1 : NQ; };  // (with rows of the piece)
  auto another = [&]() {  // the next piece, once a warp is done with this one
    if constexpr (BAL) return *stop == 0 && next_piece<kGroupRows>(A, walk, lane);
    else return false;
  };

  if (tid == 0) {
    for (int s = 0; s < P::kStages; ++s) {
      mbar_init(full + s, P::kBf ? 1 : P::kWideners);
      mbar_init(freeb + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, 4 * CG);
      mbar_init(o_done + s, 1);
    }
    mbar_init(m_done, 1);
    mbar_init(q_full, 4 * NQ * CG);
    if constexpr (CG == 2)
      for (int s = 0; s < P::kStages; ++s) mbar_init(peer_full + s, 1);
    for (int s = 0; s < P::kRawStages; ++s) {
      mbar_init(raw_full + s, 1);
      mbar_init(raw_free + s, P::kWideners);
    }
    mbar_init(looked, 2);
    mbar_init(looked + 1, 2);
    *odd_v = 0;
    *stop = 0;
  }
  if (warp == P::kMmaWarp) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  fence_before();
  group_sync<CG>();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  auto give_up = [&]() {
    *stop = 1;
    atomicOr(A.flag, GS_KV_ERR_TIMEOUT);
  };

  const int shift = A.kv.page_shift, page_mask = (1 << shift) - 1;
  auto page_of = [&](int b, int tok) {  // the page of a context token, checked
    const int col = tok >> shift;
    int pg = col < A.table_cols ? __ldg(A.table + b * A.table_stride + col) : -1;
    if (pg < 0 || pg >= A.kv.pages) {
      atomicOr(A.flag, GS_KV_ERR_PAGE);
      pg = 0;
    }
    return pg;
  };

  // ---------------- loaders ----------------
  auto load = [&]() {
    // The stages of a bf16 cache are the operands themselves; of an 8-bit one the codes, which the
    // widening warps turn into operands.
    constexpr int kRing = P::kBf ? P::kStages : P::kRawStages;
    constexpr int kRingStage = P::kBf ? P::kStage : P::kRawStage;
    uint64_t* ring_full = P::kBf ? full : raw_full;
    uint64_t* ring_free = P::kBf ? freeb : raw_free;
    unsigned char* ring = sm + (P::kBf ? P::kOffStage : P::kOffRaw);
    int issued = 0;
    bool ok = true;
    do {
     const RowRange& R = pc.R;
     const int head = pc.head;
     for (int i = 0; i < 2 * pc.n && ok && !*stop; ++i) {
      bool value;
      int j;
      stage_item<SB>(i, pc.n, value, j);
      for (int h = 0; h < P::kPer; ++h) {
        const int at = issued % kRing, round = issued / kRing;
        const int toks = value ? P::kVTok : P::kKTok;
        const int inner = value ? P::kVInner : P::kKInner;
        const int box = min(1 << shift, toks);  // tokens per box
        const int groups = toks / box;
        const int cols = (value ? P::kVCols : P::kKCols) * P::kEl / inner;
        const int j0 = R.tile(pc.t_begin + j) * kTT + (value ? h * P::kVTok : rank * P::kKTok);
        // lane g: token group g (at most 8), of one page.  A group that no row sees a token of stays as it is, and so does its table
        // entry: past the last position, or behind the window, where a server may have freed the page.  (K's scores there
        // are masked, V's rows set to zero.)
        const int tok = j0 + lane * box;
        const bool real = lane < groups && tok < R.hi && (tok + box > R.lo || tok < R.sink);
        const int pg = real ? page_of(pc.b, tok) : 0;  // (on its way while the stage is awaited)
        if (round > 0) ok = __all_sync(kFullMask, mbar_wait(ring_free + at, static_cast<uint32_t>((round - 1) & 1), kWaitNs));
        if (!ok) break;
        const unsigned live = __ballot_sync(kFullMask, real);
        const uint32_t bytes = static_cast<uint32_t>(__popc(live) * box * cols * inner);
        if (lane == 0) {
          if (bytes) mbar_expect_tx(ring_full + at, bytes);
          else arrive_on(ring_full + at);
        }
        __syncwarp();
        if (real) {
          const uint32_t dst = smem_addr(ring + at * kRingStage) + lane * box * inner;
          const int x0 = value ? rank * P::kVCols : h * P::kKCols;
          for (int cb = 0; cb < cols; ++cb)
            tma_box(dst + cb * toks * inner, value ? &maps.v : &maps.k, x0 + cb * (inner / P::kEl), tok & page_mask, head, pg,
                    ring_full + at);
        }
        __syncwarp();
        ++issued;
      }
     }
    } while (ok && another());
    if (!ok) give_up();
    if (*stop)  // copies in flight land before the block ends
      for (int k = max(0, issued - kRing); k < issued; ++k)
        mbar_wait(ring_full + k % kRing, static_cast<uint32_t>((k / kRing) & 1), kWaitNs);
    __syncwarp();
  };

  // ---------------- widening warps (8-bit): codes -> float16 operands ----------------
  // The softmax multiplies V's scales into its weights; so that float16 holds the products, it takes its
  // reference point relative to vref, a power of two at or above every V scale's magnitude so far (from 2^-60 up).
  auto widen = [&]() {
    const int lt = tid - 32 * P::kWidenWarp;
    constexpr int kPieces = P::kRawStage / 16 / P::kWideners;  // 16-byte pieces of codes per thread and stage
    int k0 = 0, g0 = 0;  // stages and tiles of the pieces before
    do {
    const RowRange& R = pc.R;
    const int head = pc.head, n = pc.n, t_begin = pc.t_begin;
    float vref = 8.673617379884035e-19f;
    // the scales of token lt of the tile after this one, in flight
    float next_k = 0.0f, next_v = 0.0f;
    auto fetch_scales = [&](int j) {
      const int tok = R.tile(t_begin + j) * kTT + lt;
      next_k = next_v = 0.0f;  // (a hidden token's weight is 0; its page may hold a NaN)
      if (R.seen_by_any(tok)) {
        const int pg = page_of(pc.b, tok), off = tok & page_mask;
        next_k = __ldg(A.kv.scale_at(false, pg, head, off));
        next_v = __ldg(A.kv.scale_at(true, pg, head, off));
      }
    };
    const bool scales = lt < kTT;  // (a token each)
    if (scales && n > 0) fetch_scales(0);
    const int total = 2 * n * P::kPer;
    for (int k = 0; k < total && !*stop; ++k) {
      bool value;
      int j;
      stage_item<SB>(k / P::kPer, n, value, j);
      const int h = k % P::kPer, kk = k0 + k;
      const int rs = kk % P::kRawStages, at = kk % P::kStages;
      bool ok = mbar_wait(raw_full + rs, static_cast<uint32_t>((kk / P::kRawStages) & 1), kWaitNs);
      if (kk >= P::kStages) ok = ok && mbar_wait(freeb + at, static_cast<uint32_t>((kk / P::kStages - 1) & 1), kWaitNs);
      if (!__all_sync(kFullMask, ok)) {
        give_up();
        break;
      }
      const int j0 = R.tile(t_begin + j) * kTT;
      float* sc = reinterpret_cast<float*>(sm + P::kOffScale) + ((g0 + j) % P::kScaleSlots) * (2 * kTT);
      if (scales && !value && h == 0) {
        // The tile's largest magnitude of a V scale (bits of positive floats in order), by way of this warp's maximum of
        // the 32 tokens it holds: vref only has to be at or above the scales that were seen with it, so each
        // warp keeps one of its own.
        sc[lt] = next_k;
        sc[kTT + lt] = next_v;
        uint32_t mag = __float_as_uint(next_v) & 0x7fffffffu;
        if (mag >= 0x7f800000u) {
          if (!R.seen_by_all(A, j0 + lt)) sc[kTT + lt] = 0.0f, A.mend[0] = 1u;  // (attn_mend_kernel)
          mag = 0u;
        }
        const uint32_t mx = __reduce_max_sync(kFullMask, mag);
        const float top = __uint_as_float(mx > 0x7e800000u ? 0x7f000000u : (mx + 0x7fffffu) & 0x7f800000u);  // up to a power of two
        if (top > vref) vref = fminf(2.0f * top, 1.7014118346046923e38f);  // (a power of two of room: each move costs a pass over O)
        if (lane == 0) reinterpret_cast<float*>(sm + P::kOffRef)[((g0 + j) % P::kScaleSlots) * 4 + (warp & 3)] = vref;
        if (j + 1 < n) fetch_scales(j + 1);
      }
      const int toks = value ? P::kVTok : P::kKTok;
      const int jt = j0 + (value ? h * P::kVTok : rank * P::kKTok);
      const unsigned char* src = sm + P::kOffRaw + rs * P::kRawStage;
      unsigned char* dst = sm + P::kOffStage + at * P::kStage;
      // TOKS tokens in column blocks of INNER codes.  MIXED: a V stage with tokens that not every row sees: those that no row sees are
      // zeros, and codes that are not finite are left out of the others.
      auto turn = [&](auto mixed_, auto toks_, auto inner_) {
        constexpr bool MIXED = decltype(mixed_)::value;
        constexpr int TOKS = decltype(toks_)::value, INNER = decltype(inner_)::value;
        auto put = [&](int id, uint4 x, bool hide) {
          const int ch = id % (INNER / 16), rowid = id / (INNER / 16);
          const int cb = rowid / TOKS, tr = rowid % TOKS;  // column block, token
          uint2 q[4] = {widen_half<FMT>(x.x), widen_half<FMT>(x.y), widen_half<FMT>(x.z), widen_half<FMT>(x.w)};
          if (MIXED && hide) q[0] = q[1] = q[2] = q[3] = make_uint2(0u, 0u);
          const int hc = (cb * INNER + ch * 16) / 64;  // 64-column operand block
          const int c0 = (ch & 3) * 2, odd = INNER == 64 ? (tr >> 1) & 1 : hc & 1;
          unsigned char* rowp = dst + hc * (TOKS * 128) + tr * 128;
          // (the lanes of a store's quarter warp take their halves in opposite orders: no two in one bank)
          const uint4 lo = make_uint4(q[0].x, q[0].y, q[1].x, q[1].y), hi = make_uint4(q[2].x, q[2].y, q[3].x, q[3].y);
          *reinterpret_cast<uint4*>(rowp + (((c0 + odd) ^ (tr & 7)) << 4)) = odd ? hi : lo;
          *reinterpret_cast<uint4*>(rowp + (((c0 + 1 - odd) ^ (tr & 7)) << 4)) = odd ? lo : hi;
        };
        if constexpr (!MIXED) {
#pragma unroll
          for (int u = 0; u < kPieces; ++u) put(lt + P::kWideners * u, *reinterpret_cast<const uint4*>(src + (lt + P::kWideners * u) * 16), false);
        } else {
#pragma unroll 1
          for (int u = 0; u < kPieces; ++u) {
            const int id = lt + P::kWideners * u, tok = jt + id / (INNER / 16) % TOKS;
            uint4 x = *reinterpret_cast<const uint4*>(src + id * 16);
            const bool hide = !R.seen_by_any(tok);
            if (any_not_finite<FMT>(x) && !hide && !R.seen_by_all(A, tok)) {
              x = without4(x, not_finite_in<FMT>(x));
              A.mend[0] = 1u;  // (attn_mend_kernel)
            }
            put(id, x, hide);
          }
        }
      };
      if (!value) turn(std::false_type{}, std::integral_constant<int, P::kKTok>{}, std::integral_constant<int, P::kKInner>{});
      else if (R.seen_by_all(A, jt, toks)) turn(std::false_type{}, std::integral_constant<int, P::kVTok>{}, std::integral_constant<int, P::kVInner>{});
      else turn(std::true_type{}, std::integral_constant<int, P::kVTok>{}, std::integral_constant<int, P::kVInner>{});
      fence_async();
      arrive_on(raw_free + rs);
      arrive_on(full + at);
    }
    k0 += total;
    g0 += n;
    } while (another());
    __syncwarp();
  };

  if (warp < P::kSoftWarps) {
    // ---------------- softmax: one query row per thread ----------------
    set_regs<P::kRegs, P::kSoftRegs>();
    const int s = NQ == 2 ? warp >> 2 : 0;  // query tile
    const int quad = warp & 3;
    const int r = s * 128 + quad * 32 + lane;
    const int gr = rank * P::kRows + r;  // row of the group
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t o_at = lane_base + 256u + static_cast<uint32_t>(s * D);
    uint32_t q_turn = 0;
    int g0 = 0, gp = 0;  // tiles of the pieces before, and those of them this query tile had a part in
    do {
    const RowRange& R = pc.R;
    const int head = pc.head, n = pc.n;
    // ---- Q: [query tile][64-column block][128 rows][128 bytes], swizzled; rows past the group zero.  Each
    // warpgroup brings its own tile, sixteen bytes a lane, all its loads at once, while the loaders start.  A lane works
    // out the address of one of the warp's rows for all (an item of 10 tiles spends 6 us here at head_dim 256
    // where every lane does so for each piece).
    if (n > 0) {
      constexpr int kCh = D / 8;          // pieces of a row
      constexpr int kPerWarp = 32 / kCh;  // rows a warp covers at once
      const uint32_t flip = A.scale_log2 < 0.0f ? 0x80008000u : 0u;  // (a negative scale: -q and |scale|)
      const int ch = lane % kCh;
      unsigned char* tile = sm + s * (D / 64) * 16384 + (ch >> 3) * 16384;
      const uint4* mine = nullptr;
      {
        const int gq = rank * P::kRows + s * 128 + q_slot<D>(quad, lane);
        int g;
        const int t = R.token_of(A, gq, g);
        if (gq < R.rows) mine = reinterpret_cast<const uint4*>(q_row(A, R, head, t, g));
      }
      uint4 x[kCh];
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        const uint4* row = reinterpret_cast<const uint4*>(__shfl_sync(kFullMask, reinterpret_cast<uint64_t>(mine), i * kPerWarp + lane / kCh));
        x[i] = row ? row[ch] : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        const int rr = q_slot<D>(quad, i * kPerWarp + lane / kCh);
        uint32_t w[4] = {x[i].x ^ flip, x[i].y ^ flip, x[i].z ^ flip, x[i].w ^ flip};
        if constexpr (!P::kBf) {
          // float16 by a power of two per row (bf16 has fewer mantissa bits: exact except for components
          // below 2^-17 of the row's largest); the lanes of a row are neighbours
          uint32_t mx = pair_max(pair_max(w[0], w[1]), pair_max(w[2], w[3]));
          if constexpr (kCh == 32) {
            mx = __reduce_max_sync(kFullMask, max(mx & 0xffffu, mx >> 16));
          } else {
#pragma unroll
            for (int o = kCh >> 1; o > 0; o >>= 1) mx = __vmaxu2(mx, __shfl_xor_sync(kFullMask, mx, o));
          }
          float down, up;
          row_power(max(mx & 0xffffu, mx >> 16), down, up);
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = half2_of(bf16_lo(w[u]) * down, bf16_hi(w[u]) * down);
          if (ch == 0) reinterpret_cast<float*>(sm + P::kOffQf)[s * 128 + rr] = up;
        }
        *reinterpret_cast<uint4*>(tile + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_async();
      __syncwarp();
      if (lane == 0) arrive_first<CG>(q_full);
    }
    q_turn ^= n > 0 ? 1u : 0u;
    if (s >= query_tiles()) {
      // No rows of the piece.  (Its barrier has to be through: arrivals of the next piece would count in it.)
      if (BAL && n > 0 && !__all_sync(kFullMask, mbar_wait(q_full, q_turn ^ 1u, kWaitNs))) give_up();
      g0 += n;
      continue;
    }
    int hq;
    const int tq = R.token_of(A, min(gr, R.rows - 1), hq);
    hq += head * A.group;
    const int p = R.p0 + tq;
    const int lo = A.window ? max(p - A.window + 1, 0) : 0;
    float c = fmaxf(fabsf(A.scale_log2), 1e-30f);  // (0 would turn a hidden score's -inf into NaN)
    float slack = 8.0f / c;
    float m = -INFINITY;
    float2 l2 = make_float2(0.0f, 0.0f);
    float vref = 1.0f;  // (8-bit) weights, sums and O are in units of vref / 2^7
    float unit = 0.0f;  // log2 of 1 over that
    for (int j = 0; j < n && !*stop; ++j) {
      const int gt = g0 + j;  // tile number of this block
      const int buf = NQ == 2 ? s : (gt & 1);
      const uint32_t ph = static_cast<uint32_t>(((gp + j) / SB) & 1);
      const uint32_t s_at = lane_base + static_cast<uint32_t>(buf * 128);
      const int j0 = R.tile(pc.t_begin + j) * kTT;
      if (!__all_sync(kFullMask, mbar_wait(s_full + buf, ph, kWaitNs))) {
        give_up();
        break;
      }
      fence_after();
      if constexpr (!P::kBf) {
        if (j == 0) {  // (every warp's Q is in place: the products have read it)
          c = fmaxf(fabsf(A.scale_log2) * reinterpret_cast<const float*>(sm + P::kOffQf)[r], 1e-30f);
          slack = 8.0f / c;
        }
      }
      float x[128];
#pragma unroll
      for (int q = 0; q < 4; ++q) tm_ld32(s_at + 32 * q, x + 32 * q);
      tm_wait_ld();
      const float* sc = reinterpret_cast<const float*>(sm + P::kOffScale) + (gt % P::kScaleSlots) * (2 * kTT);
      if constexpr (!P::kBf) {
#pragma unroll
        for (int i = 0; i < 128; i += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(sc + i);
          const float2 a = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(k4.x, k4.y));
          const float2 b2 = __fmul2_rn(make_float2(x[i + 2], x[i + 3]), make_float2(k4.z, k4.w));
          x[i] = a.x, x[i + 1] = a.y, x[i + 2] = b2.x, x[i + 3] = b2.y;
        }
      }
      const bool whole = j0 + kTT - 1 <= p && (j0 >= lo || j0 + kTT <= R.sink);
      if (!__all_sync(kFullMask, whole)) {
        // One bound where one is enough: a causal edge, a window's edge past the sinks (6 sequences of windows of
        // 1024 at head_dim 256, e4m3: 2% less time; not with two query tiles beside an 8-bit cache, whose
        // softmax has no registers left for it: 8% more at head_dim 128).
        constexpr bool kEdges = P::kBf || NQ == 1;
        const int hi_c = p + 1 - j0, lo_c = lo - j0, sk_c = R.sink - j0;
        if (kEdges && __all_sync(kFullMask, lo_c <= 0)) {
#pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = i < hi_c ? x[i] : -INFINITY;
        } else if (kEdges && sk_c <= 0 && __all_sync(kFullMask, hi_c >= kTT)) {
#pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = i >= lo_c ? x[i] : -INFINITY;
        } else {
#pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = (i < hi_c && (i >= lo_c || i < sk_c)) ? x[i] : -INFINITY;
        }
      }
      float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < 128; i += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = i + 4 + u < 128 ? fmaxf(fmaxf(mx[u], x[i + u]), x[i + 4 + u]) : fmaxf(mx[u], x[i + u]);
      }
      const float tm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool move = tm > m + slack || (m == -INFINITY && tm > m);
      float vnew = vref;
      if constexpr (!P::kBf) {
        const float4 v4 = reinterpret_cast<const float4*>(sm + P::kOffRef)[gt % P::kScaleSlots];
        vnew = fmaxf(fmaxf(v4.x, v4.y), fmaxf(v4.z, v4.w));
      }
      if (__any_sync(kFullMask, move || vnew != vref)) {
        const float mn = move ? tm : m;
        float al = m == -INFINITY ? 0.0f : ex2((m - mn) * c);
        m = mn;
        l2.x *= al, l2.y *= al;
        if constexpr (!P::kBf) {
          al *= vref / vnew;
          l2.x *= vref / vnew, l2.y *= vref / vnew;
          vref = vnew;
          unit = 7.0f - log2f(vref);
        }
        if (j > 0) {
          bool ok = true;
          if constexpr (SB == 2) ok = mbar_wait(o_done, static_cast<uint32_t>((gt - 1) & 1), kWaitNs);
          if (!__all_sync(kFullMask, ok)) {
            give_up();
            break;
          }
          fence_after();
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            float o[32];
            tm_ld32(o_at + 32 * q, o);
            tm_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= al;
            tm_st32(o_at + 32 * q, reinterpret_cast<uint32_t*>(o));
          }
        }
      }
      const float mc = (m == -INFINITY ? 0.0f : -m * c) + unit;
      uint32_t* w = reinterpret_cast<uint32_t*>(x);
      float2 l3 = make_float2(0.0f, 0.0f);  // (two chains of the sum)
#pragma unroll
      for (int i = 0; i < 128; i += 4) {
        float2 t = __ffma2_rn(make_float2(x[i], x[i + 1]), make_float2(c, c), make_float2(mc, mc));
        float2 u = __ffma2_rn(make_float2(x[i + 2], x[i + 3]), make_float2(c, c), make_float2(mc, mc));
        t.x = ex2(t.x), t.y = ex2(t.y), u.x = ex2(u.x), u.y = ex2(u.y);
        l2 = __fadd2_rn(l2, t);
        l3 = __fadd2_rn(l3, u);
        if constexpr (P::kBf) {
          w[i >> 1] = bf16x2(t.x, t.y);
          w[(i >> 1) + 1] = bf16x2(u.x, u.y);
        } else {
          const float4 v4 = *reinterpret_cast<const float4*>(sc + kTT + i);
          t = __fmul2_rn(t, make_float2(v4.x, v4.y));
          u = __fmul2_rn(u, make_float2(v4.z, v4.w));
          w[i >> 1] = half2_of(t.x, t.y);
          w[(i >> 1) + 1] = half2_of(u.x, u.y);
        }
      }
      l2 = __fadd2_rn(l2, l3);
      tm_st32(s_at, w);
      tm_st32(s_at + 32, w + 32);
      tm_wait_st();
      fence_before();
      if (SB == 2 && j > 0 && j == n - 1) {
        // (the product before the last has to be over before the last one may start: a wait by parity that
        // finds two phases passed would never end)
        if (!__all_sync(kFullMask, mbar_wait(o_done, static_cast<uint32_t>((gt - 1) & 1), kWaitNs))) {
          give_up();
          break;
        }
      }
      __syncwarp();
      if (lane == 0) arrive_first<CG>(p_full + buf);
    }
    // ---- epilogue
    float l = l2.x + l2.y;
    float ml = m == -INFINITY ? m : m * c - unit;  // (log2 units)
    bool ok = *stop == 0;
    if (n > 0 && ok) {
      ok = mbar_wait(o_done + s, static_cast<uint32_t>((gp + n - 1) & 1), kWaitNs);
      if (!ok) give_up();
    }
    ok = __all_sync(kFullMask, ok);
    bool finish = pc.part < 0;  // whether the result leaves from here
    if (BAL && ok && pc.pieces > 0) {
      // A piece of an item that other groups have the rest of: its (m, l, O) to the workspace, warp by warp,
      // column quads of the 32 rows side by side.  The same 32 rows are the same warp's in every piece, so a
      // counter per warp tells who is last (nothing waits), and the last one adds them up, its own too, in
      // the pieces' order: which of them came last changes no bit of the result.
      fence_after();
      const int64_t warp_at = static_cast<int64_t>(rank * P::kRows + s * 128 + quad * 32);
      auto part_o = [&](int slot) { return reinterpret_cast<float4*>(A.part_o) + (static_cast<int64_t>(slot) * kGroupRows + warp_at) * (D / 4) + lane; };
      auto part_ml = [&](int slot) { return reinterpret_cast<float2*>(A.part_ml) + static_cast<int64_t>(slot) * kGroupRows + warp_at + lane; };
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        float o[32];
        tm_ld32(o_at + 32 * q, o);
        tm_wait_ld();
        float4* dst = part_o(pc.part) + q * 8 * 32;
#pragma unroll
        for (int i = 0; i < 8; ++i) __stcg(dst + i * 32, make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
      }
      __stcg(part_ml(pc.part), make_float2(ml, l));
      __threadfence();
      __syncwarp();
      unsigned* ticket = A.tickets + pc.first * 8 + static_cast<int>(warp_at / 32);
      unsigned old = 0;
      if (lane == 0) old = atomicAdd(ticket, 1u);
      finish = __shfl_sync(kFullMask, old, 0) == static_cast<unsigned>(pc.pieces - 1);
      if (finish) {
        __threadfence();
        if (lane == 0) *ticket = 0u;  // (for the next call)
        auto slot = [&](int k) { return k == 0 ? 2 * pc.first + 1 : 2 * (pc.first + k); };
        float M = -INFINITY, L = 0.0f;
        for (int k = 0; k < pc.pieces; ++k) M = max_nan(M, __ldcg(part_ml(slot(k))).x);
        const float ref = M == -INFINITY ? 0.0f : M;
        for (int k = 0; k < pc.pieces; ++k) {
          const float2 v = __ldcg(part_ml(slot(k)));
          L += ex2(v.x - ref) * v.y;
        }
        for (int k = 0; k < pc.pieces; ++k) {
          const float f = ex2(__ldcg(part_ml(slot(k))).x - ref);
          const float4* src = part_o(slot(k));
          float4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = __ldcg(src + i * 32);
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            float4 y[8];  // (the next columns, in flight)
            if (q + 1 < D / 32) {
#pragma unroll
              for (int i = 0; i < 8; ++i) y[i] = __ldcg(src + ((q + 1) * 8 + i) * 32);
            }
            float o[32];
            if (k == 0) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0.0f;
            } else {
              tm_ld32(o_at + 32 * q, o);
              tm_wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[4 * i] += f * x[i].x, o[4 * i + 1] += f * x[i].y;
              o[4 * i + 2] += f * x[i].z, o[4 * i + 3] += f * x[i].w;
            }
            tm_st32(o_at + 32 * q, reinterpret_cast<uint32_t*>(o));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = y[i];
          }
          tm_wait_st();
        }
        ml = M;
        l = L;
      }
    }
    if (ok && (finish || pc.pieces == 0)) {
      fence_after();
      const bool live = gr < R.rows;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t part = static_cast<int64_t>(pc.part) * kGroupRows + gr;
      if (finish) {
        // by way of shared memory (the query tile's, which no product reads any more): whole rows leave in
        // 16-byte pieces of neighbouring lanes.  A warp stages its 32 rows where it brings its 32 rows of the next
        // item's Q (q_slot), and no other warp of the tile writes there: the four are not ordered between one item and the next.
        constexpr int kCh = D / 8;
        unsigned char* st = sm + s * (D / 64) * 16384;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          float o[32];
          if (n > 0) {
            tm_ld32(o_at + 32 * q, o);
            tm_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 w = make_uint4(bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv), bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                       bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
            *reinterpret_cast<uint4*>(st + q_slot<D>(quad, lane) * 128 + ((4 * q + i) >> 3) * 16384 + ((((4 * q + i) ^ lane) & 7) << 4)) = w;
          }
        }
        __syncwarp();
        uint4* mine = live ? reinterpret_cast<uint4*>(o_row(A, R, head, tq, hq - head * A.group)) : nullptr;  // (lane = row)
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
          const int rr = (i * 32 + lane) / kCh, ch = (i * 32 + lane) % kCh;
          uint4* row = reinterpret_cast<uint4*>(__shfl_sync(kFullMask, reinterpret_cast<uint64_t>(mine), rr));
          if (row) row[ch] = *reinterpret_cast<const uint4*>(st + q_slot<D>(quad, rr) * 128 + (ch >> 3) * 16384 + (((ch ^ rr) & 7) << 4));
        }
      } else {
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          float o[32];
          if (n > 0) {
            tm_ld32(o_at + 32 * q, o);
            tm_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
          }
          if (live) {
            float4* dst = reinterpret_cast<float4*>(A.part_o + part * D + 32 * q);
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
      }
      if (live) {
        if (finish) {
          if (A.lse) A.lse[static_cast<int64_t>(R.q0 + tq) * A.q_heads + hq] = l == 0.0f ? -INFINITY : (ml + log2f(l)) * 0.6931471805599453f;
        } else {
          *reinterpret_cast<float2*>(A.part_ml + part * 2) = make_float2(ml, l);
        }
      }
    }
    fence_before();
    g0 += n;
    gp += n;
    } while (another());
  } else if (warp < P::kMmaWarp + 4) {
   set_regs<P::kRegs, P::kMmaRegs>();
   if (warp == P::kMmaWarp) {
    // ---------------- MMA issuer ----------------
    const bool leader = elected();
    int cnt = 0;  // stages consumed
    int g0 = 0;   // tiles of the pieces before
    int g1 = 0;   // those of them with a second query tile
    uint32_t q_phase = 0;
    auto stage_ready = [&](int at) {  // this block's half
      return __all_sync(kFullMask, mbar_wait(full + at % P::kStages, static_cast<uint32_t>((at / P::kStages) & 1), kWaitNs));
    };
    auto peer_ready = [&](int at) {  // the other's
      return CG == 1 || __all_sync(kFullMask, wait_group<CG>(peer_full + at % P::kStages, static_cast<uint32_t>((at / P::kStages) & 1)));
    };
    // S(query tile s, buffer buf) = Q K^T over stages at .. at + kPer - 1
    auto scores = [&](int s, int buf, int at) {
      if (leader) {
#pragma unroll
        for (int h = 0; h < P::kPer; ++h) {
          const uint32_t ka = smem_addr(sm + P::kOffStage + ((at + h) % P::kStages) * P::kStage);
          const uint32_t qa = smem_addr(sm + s * (D / 64) * 16384 + h * (P::kKCols / 64) * 16384);
#pragma unroll
          for (int k = 0; k < P::kKCols / 16; ++k)
            mma_ss<CG>(tmem + buf * 128, desc_sw128(qa + (k >> 2) * 16384 + (k & 3) * 32, 16),
                       desc_sw128(ka + (k >> 2) * (P::kKTok * 128) + (k & 3) * 32, 16), kIdescQK<P::kBf, CG>, (h | k) != 0 ? 1u : 0u);
        }
      }
      __syncwarp();
    };
    // Zeros in the rows of a V stage that no query row of the block sees (their weights are 0, and what the pages hold there may
    // be a NaN), and in place of what is not finite in rows that only some see (attn_mend_kernel adds it to those).
    int have_looked = 0;
    auto clean = [&](int at, int j, int h) {
      const RowRange& R = pc.R;
      const int j0 = R.tile(pc.t_begin + j) * kTT + h * P::kVTok;
      if (!P::kBf || R.seen_by_all(A, j0, P::kVTok)) return true;
      unsigned char* st = sm + P::kOffStage + (at % P::kStages) * P::kStage;
      constexpr int kCh = P::kVCols / 8;
      bool odd = false, wrote = false;
      auto piece = [&](int id) {
        const int tr = id / kCh, ch = id % kCh;
        return reinterpret_cast<uint4*>(st + (ch >> 3) * (P::kVTok * 128) + tr * 128 + ((ch & 7) << 4));
      };
      // (context tokens t0 .. t1 - 1, as far as the stage has them)
      auto zero = [&](int t0, int t1) {
        for (int id = max(t0 - j0, 0) * kCh + lane; id < min(t1 - j0, P::kVTok) * kCh; id += 32) *piece(id) = make_uint4(0u, 0u, 0u, 0u), wrote = true;
      };
      auto sift = [&](int t0, int t1) {
        const int end = min(t1 - j0, P::kVTok) * kCh;
        for (int id0 = max(t0 - j0, 0) * kCh + lane; id0 < end; id0 += 256) {
          uint4 w[8];
          uint32_t found = 0u;
#pragma unroll
          for (int u = 0; u < 8; ++u) w[u] = *piece(min(id0 + 32 * u, end - 1));
#pragma unroll
          for (int u = 0; u < 8; ++u) look_for_not_finite<FMT>(w[u], found);
          if (!found_not_finite<FMT>(found)) continue;
          for (int id = id0; id < end && id < id0 + 256; id += 32) *piece(id) = without4(*piece(id), not_finite_in<FMT>(*piece(id)));
          odd = true;
        }
      };
      if (A.window) zero(R.sink, R.lo);
      zero(R.hi, j0 + P::kVTok);
      auto range = [&](int k, int t0, int t1) {
        if (t0 >= min(t1, j0 + P::kVTok) || t1 <= j0) return true;
        if (!BAL) {
          if (!(have_looked >> k & 1) && !__all_sync(kFullMask, mbar_wait(looked + k, 0, kWaitNs))) return false;
          have_looked |= 1 << k;
          if (!(*reinterpret_cast<volatile int*>(odd_v) >> k & 1)) return true;
        }
        sift(t0, t1);
        return true;
      };
      if (A.window && !range(0, R.left0(), R.left1(A))) return false;
      if (!range(1, R.ahead0(), R.hi)) return false;
      if (odd) A.mend[0] = 1u;
      if (odd || wrote) fence_async();
      __syncwarp();
      return true;
    };
    bool ok = true;
    const bool issues = CG == 1 || rank == 0;
    do {
    const int n = pc.n, nq = query_tiles();
    if (CG == 2 && rank == 1) {
      // second block: tells the first when a stage of its own is there (and clean)
      for (int i = 0; ok && i < 2 * n && !*stop; ++i) {
        bool value;
        int j;
        stage_item<SB>(i, n, value, j);
        for (int h = 0; ok && h < P::kPer; ++h, ++cnt) {
          ok = stage_ready(cnt);
          if (!ok) break;
          if (value) ok = clean(cnt, j, h);
          if (!ok) break;
          if (lane == 0) arrive_first<CG>(peer_full + cnt % P::kStages);
          __syncwarp();
        }
      }
    }
    if (issues && n > 0) {
      ok = ok && __all_sync(kFullMask, wait_group<CG>(q_full, q_phase));
      q_phase ^= 1;
    }
    for (int i = 0; issues && ok && i < SB && i < n; ++i) {
      for (int h = 0; ok && h < P::kPer; ++h) ok = stage_ready(cnt + h) && peer_ready(cnt + h);
      if (!ok) break;
      fence_after();
      for (int s = 0; s < nq; ++s) {
        scores(s, NQ == 2 ? s : (g0 + i) & 1, cnt);
        if (leader) {
          commit_to<CG>(s_full + (NQ == 2 ? s : (g0 + i) & 1));
          if (s == nq - 1)
            for (int h = 0; h < P::kPer; ++h) commit_to<CG>(freeb + (cnt + h) % P::kStages);
        }
        __syncwarp();
      }
      cnt += P::kPer;
    }
    for (int j = 0; issues && ok && j < n && !*stop; ++j) {
      const int v_at = cnt, k_at = cnt + P::kPer;
      const bool more = j + SB < n;
      for (int s = 0; ok && s < nq; ++s) {
        const int buf = NQ == 2 ? s : ((g0 + j) & 1);
        if (s == 0)
          for (int h = 0; ok && h < P::kPer; ++h) {
            ok = stage_ready(v_at + h);
            ok = ok && clean(v_at + h, j, h);
            ok = ok && peer_ready(v_at + h);
          }
        ok = ok && __all_sync(kFullMask, wait_group<CG>(p_full + buf, static_cast<uint32_t>((((s == 0 ? g0 : g1) + j) / SB) & 1)));
        if (!ok) break;
        fence_after();
        if (leader) {
#pragma unroll
          for (int h = 0; h < P::kPer; ++h) {
            const uint32_t va = smem_addr(sm + P::kOffStage + ((v_at + h) % P::kStages) * P::kStage);
#pragma unroll
            for (int k = 0; k < P::kVTok / 16; ++k)
              mma_ts<CG>(tmem + 256 + s * D, tmem + buf * 128 + (h * P::kVTok + k * 16) / 2, desc_sw128(va + k * 2048, P::kVTok * 128),
                         kIdescPV<D, P::kBf, CG>, (j | h | k) != 0 ? 1u : 0u);
          }
          commit_to<CG>(o_done + s);
          if (s == nq - 1)
            for (int h = 0; h < P::kPer; ++h) commit_to<CG>(freeb + (v_at + h) % P::kStages);
        }
        __syncwarp();
        if (more) {
          if (s == 0)
            for (int h = 0; ok && h < P::kPer; ++h) ok = stage_ready(k_at + h) && peer_ready(k_at + h);
          if (!ok) break;
          fence_after();
          scores(s, buf, k_at);
          if (leader) {
            commit_to<CG>(s_full + buf);
            if (s == nq - 1)
              for (int h = 0; h < P::kPer; ++h) commit_to<CG>(freeb + (k_at + h) % P::kStages);
          }
          __syncwarp();
        }
      }
      cnt += more ? 2 * P::kPer : P::kPer;
    }
    g0 += n;
    if (nq == 2) g1 += n;
    } while (ok && another());
    if (!ok) give_up();
    // every product has completed before tensor memory is freed
    if (leader && issues) commit_to<CG>(m_done);
    __syncwarp();
    if (!__all_sync(kFullMask, mbar_wait(m_done, 0, kWaitNs))) give_up();
   } else if (warp == P::kLoadWarp) {
    load();
   } else if (P::kBf && !BAL) {
    // ---------------- the two warps left: a look at V ahead of the products ----------------
    // (A call of short windows waits for V: 6 chunks of up to 1500 tokens, windows of 1024, heads of 256, without a look 192 us, with
    // one in the stages 205, with this 200.  Blocks that walk several items have time for it in the stages: 2048 tokens over 16384,
    // heads of 128, 516 us with and without.)
    const RowRange& R = pc.R;
    constexpr int kCh = P::kVCols / 8, kBatch = NQ == 1 ? 16 : 8;
    auto look = [&](int k, int t0, int t1) {
      uint32_t found = 0u;
      const int n = (t1 - t0) * kCh;
      for (int id0 = (warp & 1) * 32 + lane; id0 < n; id0 += 64 * kBatch) {
        uint4 w[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int id = min(id0 + 64 * u, n - 1), tok = t0 + id / kCh;
          w[u] = __ldg(reinterpret_cast<const uint4*>(A.kv.at(true, page_of(pc.b, tok), pc.head, tok & page_mask)) + rank * kCh + id % kCh);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) look_for_not_finite<FMT>(w[u], found);
      }
      if (found_not_finite<FMT>(found)) atomicOr(odd_v, 1 << k);
      __syncwarp();
      if (lane == 0) arrive_on(looked + k);
    };
    if (A.window) look(0, R.left0(), R.left1(A));
    look(1, R.ahead0(), R.hi);
   }
  } else if constexpr (!P::kBf) {
   set_regs<P::kRegs, P::kLoadRegs>();
   widen();
  }
  fence_before();
  group_sync<CG>();  // (no block leaves while the other's products may read its shared memory)
  if (warp == P::kMmaWarp) {
    fence_after();
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// One block per query row of a split context: the splits' (m, l, O) joined.
template <int D>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs A, int rows_per_block) {
  constexpr int kVec = D / 4, kParts = 128 / kVec;  // threads across head_dim, splits in parallel
  __shared__ float4 s_acc[128];
  __shared__ float s_red[4], s_lse[4];
  const int b = blockIdx.z, head = blockIdx.y % A.kv.kv_heads, rb = blockIdx.y / A.kv.kv_heads;
  const int r = blockIdx.x, r0 = rb * rows_per_block, tid = threadIdx.x;
  const RowRange R = row_range<kTT>(A, b, r0, rows_per_block, false);
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
  int gq;
  const int t = R.token_of(A, r, gq);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint2*>(o_row(A, R, head, t, gq) + d) =
      make_uint2(bf16x2(acc.x * inv, acc.y * inv), bf16x2(acc.z * inv, acc.w * inv));
  if (A.lse && d == 0) A.lse[static_cast<int64_t>(R.q0 + t) * A.q_heads + head * A.group + gq] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// After the many-row kernel, and nothing to do unless that left values out of a product: tokens that some rows of a
// block see and others do not, and whose values are not finite.  A row that sees such a token lies at most a block's new tokens
// behind it, or the token lies as little behind the beginning of the row's window: those tokens are asked, four columns a
// thread, and what is not finite is added to the result.  (Where a token was not left out it is in the result
// already, which adding it again does not change.)  Launched while the kernel before it still runs and waiting for its end on the
// device, it costs a call about a microsecond.
template <int FMT>
__global__ void __launch_bounds__(128) attn_mend_kernel(const __grid_constant__ AttnArgs A, int head_dim) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (__ldcg(A.mend) == 0u) return;
  constexpr int kEl = FMT == GS_DTYPE_BF16 ? 2 : 1;
  const int pieces = head_dim / 4, mask = (1 << A.kv.page_shift) - 1;
  const int span = (kMostRows + A.group - 2) / A.group + 1;  // tokens that a block's rows are of, at most
  for (int u = blockIdx.x; u < A.seqs * A.kv.kv_heads; u += gridDim.x) {
    const int b = u / A.kv.kv_heads, head = u % A.kv.kv_heads;
    const RowRange R = row_range<kTT>(A, b, 0, 0x7fffffff, false);
    const int32_t* table = A.table + b * A.table_stride;
    for (int64_t e = threadIdx.x + static_cast<int64_t>(blockIdx.y) * 128; e < static_cast<int64_t>(R.rows) * pieces; e += gridDim.y * 128) {
      const int r = static_cast<int>(e / pieces), d = static_cast<int>(e % pieces) * 4, t = r / A.group, g = r % A.group;
      const int pos = R.p0 + t, lo = A.window ? max(pos - A.window + 1, 0) : 0;
      float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      auto ask = [&](int j0, int end) {
#pragma unroll 8
        for (int j = j0; j < end; ++j) {
          const int col = j >> A.kv.page_shift, off = j & mask;
          int page = col < A.table_cols ? __ldg(table + col) : 0;
          if (page < 0 || page >= A.kv.pages) page = 0;  // (noted by the kernel that came here)
          const unsigned char* v = A.kv.at(true, page, head, off) + d * kEl;
          if constexpr (FMT == GS_DTYPE_BF16) {
            const uint2 w = *reinterpret_cast<const uint2*>(v);
            const float x[4] = {bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
#pragma unroll
            for (int i = 0; i < 4; ++i) add[i] += fabsf(x[i]) < INFINITY ? 0.0f : x[i];
          } else {
            const uint32_t m = fabsf(*A.kv.scale_at(true, page, head, off)) < INFINITY ? not_finite_in<FMT>(*reinterpret_cast<const uint32_t*>(v)) : ~0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) add[i] = m >> (8 * i) & 1u ? NAN : add[i];
          }
        }
      };
      const int recent = max(max(pos - span + 1, lo), 0);
      ask(recent, pos + 1);
      if (A.window) {
        ask(max(recent - span, 0), min(recent, min(A.sinks, lo)));  // (a sink among them that the window has left behind)
        ask(lo, min(lo + span, recent));
      }
      if (add[0] == 0.0f && add[1] == 0.0f && add[2] == 0.0f && add[3] == 0.0f) continue;
      uint2* at = reinterpret_cast<uint2*>(o_row(A, R, head, t, g) + d);
      const uint2 w = *at;
      *at = make_uint2(bf16x2(bf16_lo(w.x) + add[0], bf16_hi(w.x) + add[1]), bf16x2(bf16_lo(w.y) + add[2], bf16_hi(w.y) + add[3]));
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    // (all have read the flag when the last one comes here)
    if (atomicAdd(A.mend + 1, 1u) == gridDim.x * gridDim.y - 1u) A.mend[0] = 0u, A.mend[1] = 0u;
  }
}

template <int FMT>
cudaError_t mend(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  const int64_t heads = static_cast<int64_t>(a.seqs) * a.kv.kv_heads, most = 4ll * c->num_sms;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim.x = static_cast<unsigned>(heads < most ? heads : most);
  cfg.gridDim.y = static_cast<unsigned>((most + heads - 1) / heads);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_mend_kernel<FMT>, a, c->d.head_dim);
}

// Units (sequence, row block) whose tile counts a block sums up at the start of a balanced call, and the
// blocks whose partial results the workspace holds.
constexpr int64_t kBalancedUnits = 2048;
constexpr int64_t kMaxGroups = 240;

template <int D, int FMT, int CG, bool BAL>
cudaError_t run(const gs_kv_cache* c, const AttnArgs& a, dim3 grid, cudaStream_t st) {
  using P = TilePlan<D, FMT, CG>;
  auto kern = attn_tile_kernel<D, FMT, CG, BAL>;
  static std::atomic<uint64_t> done{0};
  if (device_todo(done)) {
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, kern);
    // (the warpgroups' shares must not exceed what the block is launched with)
    if (e == cudaSuccess && P::kSoftRegs != P::kRegs && at.numRegs != P::kRegs) e = cudaErrorInvalidKernelImage;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kSmem);
    if (e != cudaSuccess) return e;
    mark_device_done(done);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(P::kThreads);
  cfg.dynamicSmemBytes = P::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = CG;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, a, *reinterpret_cast<const TileMaps*>(c->maps + (CG == 1 ? 0 : 512)));
}

template <int D, int FMT, int CG>
cudaError_t go(const gs_kv_cache* c, AttnArgs a, cudaStream_t st) {
  using P = TilePlan<D, FMT, CG>;
  constexpr int kRows = CG * P::kRows;  // rows of a group of blocks
  static_assert(kRows <= kMostRows, "rows by which attn_mend_kernel asks");
  const int blocks = static_cast<int>((static_cast<int64_t>(a.max_q) * a.group + kRows - 1) / kRows);
  const int64_t items = static_cast<int64_t>(a.seqs) * a.kv.kv_heads * blocks;
  const int64_t tiles = most_tiles(a, kTT, kRows);
  const int64_t groups = c->num_sms / CG;
  const int64_t units = static_cast<int64_t>(a.seqs) * blocks;
  a.row_blocks = blocks;
  a.part_o = reinterpret_cast<float*>(c->ws);
  if constexpr (P::kBalance) {
    // Balanced: every block takes an equal stretch of all items' tiles.  Against the rounds of a fixed grid
    // this saves the last round's idle blocks and costs a block about one more beginning and end (about 5
    // tiles' time) and the joining of what is cut (as much again): 2048 tokens over 16384 in 1.73 rounds take 6% less time
    // at head_dim 128, 8% at 64, 1024-token windows (10 tiles) 23% more, so not there.  (8-bit caches: at head_dim 64 7% less; at 128
    // the softmax spills for it, 23% more; at head_dim 256 there are half as many groups, 5% more.)
    const int64_t rounds = (items + groups - 1) / groups;
    const bool gains = rounds * groups * (tiles + 5) > items * tiles + (items + 2 * groups) * 5;
    if (2 * items > groups && gains && units <= kBalancedUnits && groups <= kMaxGroups) {
      static_assert(2 * kMaxGroups * static_cast<int64_t>(kRows) * (D + 2) * 4 <= static_cast<int64_t>(kAttnWsBytes), "partial results");
      a.tickets = reinterpret_cast<unsigned*>(c->ws + kAttnWsBytes);
      a.units = static_cast<int32_t>(units);
      a.part_ml = a.part_o + 2 * groups * kRows * D;
      return run<D, FMT, CG, true>(c, a, dim3(static_cast<unsigned>(groups)), st);
    }
  }
  // Fixed: a block (or two) an item.  Where the items do not fill the SMs each is split evenly, in pieces of at
  // least 8 tiles, and a second launch joins them.
  int64_t splits = groups / items;
  const int64_t by_len = tiles / 8;
  splits = splits > by_len ? by_len : splits;
  const int64_t slot = static_cast<int64_t>(kRows) * (D + 2) * 4;
  const int64_t by_ws = static_cast<int64_t>(kAttnWsBytes) / (items * slot);
  splits = splits > by_ws ? by_ws : splits;
  if (splits < 1) splits = 1;
  const int64_t chunk = tiles > 0 ? (tiles + splits - 1) / splits : 1;
  a.chunk_tiles = static_cast<int32_t>(chunk);
  a.splits = static_cast<int32_t>(tiles > 0 ? (tiles + chunk - 1) / chunk : 1);
  a.part_ml = a.part_o + items * a.splits * kRows * D;
  const dim3 grid(static_cast<unsigned>(a.splits * CG), static_cast<unsigned>(a.kv.kv_heads * blocks), static_cast<unsigned>(a.seqs));
  if (grid.y > 65535) return cudaErrorInvalidConfiguration;
  const cudaError_t e = run<D, FMT, CG, false>(c, a, grid, st);
  if (e != cudaSuccess || a.splits == 1) return e;
  attn_join_kernel<D><<<dim3(kRows, static_cast<unsigned>(a.kv.kv_heads * blocks), static_cast<unsigned>(a.seqs)), 128, 0, st>>>(a, kRows);
  return cudaGetLastError();
}

template <int D, int FMT>
cudaError_t go_cg(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  // Two blocks a group at head_dim 256, where one block's 128 rows read K and V faster than L2 gives them
  // (2048 x 16384 tokens, 16 / 8 heads: bf16 36% less time, e4m3 44%).  At head_dim 128 a block has
  // 256 rows of its own, and two of them gain nothing (32 / 8 heads: e4m3 1% more, int8 3% less).
  if constexpr (D == 256) {
    if (static_cast<int64_t>(a.max_q) * a.group > TilePlan<D, FMT, 1>::kRows) return go<D, FMT, 2>(c, a, st);
  }
  return go<D, FMT, 1>(c, a, st);
}

template <int D>
cudaError_t go_fmt(const gs_kv_cache* c, const AttnArgs& a, cudaStream_t st) {
  switch (c->d.format) {
    case GS_DTYPE_BF16: return go_cg<D, GS_DTYPE_BF16>(c, a, st);
    case GS_DTYPE_E4M3: return go_cg<D, GS_DTYPE_E4M3>(c, a, st);
    default: return go_cg<D, GS_DTYPE_INT8>(c, a, st);
  }
}

}  // namespace

cudaError_t launch_attn_tile(const gs_kv_cache* c, AttnArgs a, cudaStream_t st) {
  const cudaError_t e = c->d.head_dim == 64 ? go_fmt<64>(c, a, st) : c->d.head_dim == 128 ? go_fmt<128>(c, a, st) : go_fmt<256>(c, a, st);
  if (e != cudaSuccess) return e;
  return c->d.format == GS_DTYPE_BF16   ? mend<GS_DTYPE_BF16>(c, a, st)
         : c->d.format == GS_DTYPE_E4M3 ? mend<GS_DTYPE_E4M3>(c, a, st) : mend<GS_DTYPE_INT8>(c, a, st);
}

// The pools as (head_dim, page token, head, page) tensors, boxes of at most 128 bytes of a row (bf16:
// one swizzle row) by as many tokens as a page and a stage share.
const char* make_attn_maps(gs_kv_cache* c) {
  static_assert(6 * sizeof(CUtensorMap) <= sizeof(c->maps), "room for the tensor maps");
  const gs_kv_cache_desc& d = c->d;
  const bool bf16 = d.format == GS_DTYPE_BF16;
  const cuuint64_t el = bf16 ? 2 : 1;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult res;
  if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res) != cudaSuccess ||
      res != cudaDriverEntryPointSuccess || !fn)
    return "cuTensorMapEncodeTiled is not available";
  auto encode = reinterpret_cast<CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill)>(fn);
  CUtensorMap* maps = reinterpret_cast<CUtensorMap*>(c->maps);
  for (int i = 0; i < 6; ++i) {  // K and V of the one-block kernel, the few-row kernel, the two-block kernel
    const bool v = (i & 1) != 0, rows = i / 2 == 1, two = i / 2 == 2;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d.head_dim), static_cast<cuuint64_t>(d.page_size),
                                static_cast<cuuint64_t>(d.kv_heads), static_cast<cuuint64_t>(d.pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(v ? d.v_token_stride : d.k_token_stride) * el,
                                   static_cast<cuuint64_t>(v ? d.v_head_stride : d.k_head_stride) * el,
                                   static_cast<cuuint64_t>(v ? d.v_page_stride : d.k_page_stride) * el};
    // a box row: 128 bytes, or the whole (half) row where that is less
    const int row = v && two ? d.head_dim / 2 : d.head_dim;
    const int inner = row * static_cast<int>(el) < 128 ? row : 128 / static_cast<int>(el);
    const int most = rows ? 16 : two ? (v ? kTT : kTT / 2) : v && d.head_dim == 256 ? 64 : kTT;
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(inner), static_cast<cuuint32_t>(d.page_size < most ? d.page_size : most), 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    if (two && d.head_dim != 256) break;
    // operands of the tensor cores and of ldmatrix are swizzled; codes to be widened are read row by row
    const CUtensorMapSwizzle swizzle = !rows && !bf16 ? CU_TENSOR_MAP_SWIZZLE_NONE
                                       : inner * el == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    const CUresult r = encode(maps + i, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, v ? d.v : d.k,
                              dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return "KV cache: these strides do not make a tensor map";
  }
  return nullptr;
}

}  // namespace gs
