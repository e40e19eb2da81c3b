// Products of row groups: rows [offsets[g], offsets[g+1]) of A meet the weight B[g] of their group.
//
//   forward   D[i]  = alpha * A[i] . B[g]^T + beta * D[i]         A (rows, K), B (G, N, K), D (rows, N)
//             (B seen as (G, K, N) with its last two modes swapped gives dA = dD . B, the gradient of the rows)
//   gradient  dB[g] = alpha * sum_{i in g} dD[i]^T A[i] + beta * dB[g]
//
// The group borders are read on the device: nothing waits for the host, and a captured launch follows new borders.
// The reference has no counterpart; the arithmetic per group is its `gemm!` (src/algorithm/blas.jl:39-88).
//
// The accumulator is turned against the dense kernels': the tensor-memory lanes (the M of the instruction, always full)
// run along the output's contiguous mode -- the weight's rows in the forward product, the features of A in the
// gradient -- and the columns (its N, a multiple of 32 up to 256, chosen per tile) along the rows of the group or of the
// weight.  A group of a few rows then costs a narrow instruction instead of a 128-row tile that is mostly padding, the
// last tile of a group simply has fewer columns, and a warp's 32 lanes are 32 neighbouring elements of an output row.
//
// Persistent CTA pairs (tcgen05 cta_group::2, see gemm_pair.cu): 256 lanes x up to 256 columns, each CTA holds 128 lanes
// and half of the column operand.  Per CTA: warp 0 TMA producer, warp 1 tcgen05.mma issuer (leader), warp 2
// clears, in the gradient, the rows behind a group's end, warp 3 reads the borders and deals the tiles, warps 4-11
// epilogue; accumulators double-buffered.
//
// The tensor cores cut the sum after every instruction's 16 products instead of rounding it, always towards zero: for a
// 16-bit output far below its step, but a Float32 output loses precision in proportion to the length of the sum (1.2e-6
// at 1000, plain fp32 sums 6e-7).  Float32 outputs are therefore summed in runs of 512 that the epilogue adds up in
// registers, rounding to nearest (`PROMOTE`).
//
// Bound by memory where groups are short (128 rows in 64 groups, 2048 x 2048 bf16: 66 us captured, 6.5 TB/s), by the tensor
// cores where they are long.  32768 rows, 4096 x 2048, in a burst / for seconds at the power cap of 1000 W: one group 386 /
// 452 us (the dense pair kernel 382 / 446), 32 equal groups 413 / 482, 32 uneven ones 448 / 522 (1227 / 1054 TFLOP/s); the
// gradient of their rows 466 / 551, of the weights 479 / 569.  Equal groups pay for 32 weights from memory.  What uneven
// groups lose are last tiles that are too narrow for the operand loads (256 + N cycles a block against 2 N of arithmetic)
// and a partly filled last wave.
#include <cstring>

#include "gemm_common.cuh"

namespace moye {

constexpr int kMaxGemmGroups = 1024;
constexpr int kMaxGroupedExtent = 1 << 27;  // a sum this long ends well inside the limit of a bounded wait
enum : int { SITEG_PROD_EMPTY = 161, SITEG_MMA_ACC = 162, SITEG_MMA_FULL = 163, SITEG_EPI_ACC = 164, SITEG_FIX_TAIL = 165, SITEG_RING = 166 };
enum : int { GROUPED_K_MAJOR = 0, GROUPED_MN_MAJOR = 1, GROUPED_GRAD = 2 };

// Columns of a tile.  The instruction's N and the loads follow the tile's own width, so a group of a few rows pays nothing
// for the size; narrower tiles for small groups gained at most 2 % (64 groups of 1 to 128 rows, 2048 x 2048) and lost 20 %
// where groups are uneven and a weight is streamed for each of their tiles.
constexpr int BT = 256;
constexpr int kColBox = 32;  // rows of one load of a K-major column operand in a narrow tile
constexpr int kPromoteBlocks = 8;  // blocks of 64 summed in tensor memory before registers take over

struct GroupedArgs {
  int rows, groups;
  int lanes;            // extent of the output's contiguous mode (N forward, K gradient)
  int cols;             // gradient: extent of the other mode (N)
  int k_blocks;         // forward: blocks of 64 along K
  int lane_tiles, col_tiles;
  int vec_out;          // D has a 16-byte base and pitches (and, for 16-bit outputs, beta is 0: one rounding)
  int tma_out;          // ... and TMA too: beta is 0 (or, for Float32 outputs, 1), rows are whole 16-byte units
  const int* offsets;
  uint32_t idesc;       // without N
  float alpha, beta;
  void* D;
  long long ld, group_stride;  // elements
  int* status;
};

struct alignas(16) GroupedTile {
  int g, row0, nrows;  // the group, its first row here and the rows of it this tile reads (gradient: all of them)
  int lane0, col0;     // first output element along the two modes (forward: col0 = row0)
  int ncols, width;    // columns to store; the instruction's N, a multiple of 32
  int k_blocks;        // blocks of 64 summed; -1: no tile left
};

// Tiles are worked out by a warp of their own and handed to the others through a ring in shared memory: finding a tile's
// group takes hundreds of cycles, which the producer and the MMA issuer spent between tiles (32768 rows, 32 groups,
// 4096 x 2048, equal groups: 411 us with the search in every role, 391 with the ring).
constexpr int kTileRing = 4;
struct TileRing {
  GroupedTile* slots;
  uint64_t *full, *empty;
  int* status;
  int n;
  __device__ __forceinline__ bool take(GroupedTile& t) {  // one reader; `leave` gives the slot back
    if (!mbar_wait(&full[n % kTileRing], (n / kTileRing) & 1, status, SITEG_RING)) return false;
    const int4* p = reinterpret_cast<const int4*>(&slots[n % kTileRing]);
    *reinterpret_cast<int4*>(&t) = p[0];
    *(reinterpret_cast<int4*>(&t) + 1) = p[1];
    return t.k_blocks >= 0;
  }
  __device__ __forceinline__ void leave() {
    mbar_arrive(&empty[n % kTileRing]);
    ++n;
  }
};

// Deals this CTA's tiles to the ring; one warp.  The groups come 32 at a time, a lane each: clamped borders, tiles, and a
// prefix over the lanes; the group of a tile is then found with one ballot.  Borders outside the arrays or running
// backwards are a caller's mistake that must not become a bad address: they are clamped, such groups come out empty.
template <int MODE>
__device__ __forceinline__ void deal_tiles(const GroupedArgs& a, TileRing& ring, int first_tile, int tile_step, int lane) {
  int next = first_tile, before = 0, last = 0;
  bool ok = true;
  auto deal = [&](const GroupedTile& t) {
    if (lane == 0) {
      const int slot = ring.n % kTileRing;
      // debug build: a tile inside the arrays, columns inside the accumulator
      ok = MOYE_DBG_OK(t.k_blocks < 0 || (t.row0 >= 0 && t.nrows >= 0 && t.row0 + t.nrows <= a.rows && t.lane0 >= 0 && t.lane0 < a.lanes &&
                                          t.ncols > 0 && t.width <= BT && t.g < a.groups), a.status, 983) &&
           mbar_wait(&ring.empty[slot], ((ring.n / kTileRing) & 1) ^ 1, a.status, SITEG_RING);
      if (ok) {
        ring.slots[slot] = t;
        mbar_arrive(&ring.full[slot]);
      }
    }
    ++ring.n;
    ok = __shfl_sync(~0u, ok, 0);
  };
  for (int g0 = 0; g0 < a.groups && ok; g0 += 32) {
    const int g = g0 + lane;
    auto border = [&](int i) { return min(max(__ldg(a.offsets + i), 0), a.rows); };
    int lo = g < a.groups ? border(g) : 0, hi = g < a.groups ? border(g + 1) : 0;
    if (lane == 0 && g0 == 0) last = lo;
    last = __shfl_sync(~0u, last, 0);
    hi = max(hi, max(lo, last));  // not decreasing: the running maximum
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, hi, d);
      if (lane >= d) hi = max(hi, up);
    }
    lo = __shfl_up_sync(~0u, hi, 1);
    if (lane == 0) lo = last;
    last = __shfl_sync(~0u, hi, 31);
    const int count = hi - lo;
    const int col_tiles = MODE == GROUPED_GRAD ? a.col_tiles : (count + BT - 1) / BT;
    const int mine = g < a.groups ? col_tiles * a.lane_tiles : 0;
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, incl, d);
      if (lane >= d) incl += up;
    }
    const int total = __shfl_sync(~0u, incl, 31);
    while (next < before + total && ok) {
      const int l = __ffs(__ballot_sync(~0u, before + incl > next)) - 1;
      const int tiles = __shfl_sync(~0u, col_tiles, l), rows = __shfl_sync(~0u, count, l), start = __shfl_sync(~0u, lo, l);
      const int q = next - before - __shfl_sync(~0u, incl - mine, l);
      // bands of 8 column tiles, whose operand stays in L2 while the lane tiles pass
      const int band = q / (a.lane_tiles * 8), w = min(8, tiles - band * 8), r = q - band * a.lane_tiles * 8;
      const int ct = band * 8 + r % w;
      GroupedTile t;
      t.g = g0 + l;
      t.lane0 = r / w * 256;
      if (MODE == GROUPED_GRAD) {
        t.col0 = ct * BT;
        t.row0 = start;
        t.nrows = rows;
        t.ncols = min(BT, a.cols - t.col0);
        t.k_blocks = (rows + 63) >> 6;
      } else {
        // a few tiles share a group's rows evenly; of many only the last is narrow
        const int step = tiles <= 4 ? ((rows + tiles - 1) / tiles + 31) & ~31 : BT;
        t.row0 = start + ct * step;
        t.nrows = min(step, start + rows - t.row0);
        t.col0 = t.row0;
        t.ncols = t.nrows;
        t.k_blocks = a.k_blocks;
      }
      t.width = (t.ncols + 31) & ~31;
      deal(t);
      next += tile_step;
    }
    before += total;
  }
  GroupedTile end = {};
  end.k_blocks = -1;
  if (ok) deal(end);
}

__device__ __forceinline__ void tma_reduce_add_3d(const CUtensorMap* m, const void* smem_src, int32_t x, int32_t y, int32_t z) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// Tensor memory -> registers in the order of matrix fragments: 16 lanes x 32 columns, of which thread T receives, for the
// columns 8 b + 2 (T % 4) and the next one, lane T / 4 in v[4 b], v[4 b + 1] and lane T / 4 + 8 in v[4 b + 2], v[4 b + 3].
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// Four transposed 8 x 8 fragments of 16-bit elements to shared memory; thread T gives the address of row T % 8 of fragment T / 8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
// Float32 tiles leave through two staging tiles a warp in turn (those gradients in Float32: 193 -> 184 us), 16-bit ones
// through one a warp, two for the pair.  What is left of shared memory holds 5 stages of operands, or 6 (16-bit with 5: 1 to
// 2 % slower on long sums).
template <typename OutT>
__host__ __device__ constexpr int grouped_epi_bufs() { return sizeof(OutT) == 4 ? 2 : 1; }

template <int MODE, typename OutT, int STAGES>
__global__ void __launch_bounds__(384, 1)
gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmL, const __grid_constant__ CUtensorMap tmC,
                    const __grid_constant__ CUtensorMap tmN, const __grid_constant__ CUtensorMap tmD, const GroupedArgs a) {
  // tmL: the operand along the lanes (weights / A), tmC: the one along the columns (rows of A / dD), tmN: the same in
  // boxes of 32 rows for narrow tiles, tmD: the output (swizzled boxes of 64 lanes, or plain ones of 32 for Float32)
  constexpr int BK = 64, UMMA_K = 16;
  constexpr int L_BYTES = 128 * 128;
  constexpr int C_BYTES = BT / 2 * 128;  // this CTA's half of the columns
  constexpr int STAGE_BYTES = L_BYTES + C_BYTES;
  constexpr uint32_t TMEM_COLS = 2 * BT;
  constexpr bool L_MN = MODE != GROUPED_K_MAJOR, C_MN = MODE == GROUPED_GRAD;
  constexpr bool PROMOTE = sizeof(OutT) == 4;
  constexpr int EPI_BUF = 32 * 128;            // a staging tile: 32 columns of 128 bytes
  constexpr int EPI_BUFS = grouped_epi_bufs<OutT>();  // staging tiles of each epilogue warp
  constexpr int EPI_BYTES = 8 * EPI_BUFS * EPI_BUF;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + STAGES * STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + EPI_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* tail = bars + 2 * STAGES;  // gradient: a group's last block has landed, its rows are not cleared yet
  uint64_t* acc_full = bars + 3 * STAGES;
  uint64_t* acc_empty = bars + 3 * STAGES + 2;
  uint64_t* ring_full = bars + 3 * STAGES + 4;
  uint64_t* ring_empty = ring_full + kTileRing;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(ring_empty + kTileRing);
  GroupedTile* ring_slots = reinterpret_cast<GroupedTile*>(ring_empty + kTileRing + 2 - (3 * STAGES & 1));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();  // 0 = leader
  const int first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
      mbar_init(&tail[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16);
    }
    for (int i = 0; i < kTileRing; ++i) {
      mbar_init(&ring_full[i], 1);
      mbar_init(&ring_empty[i], 9 + (rank == 0 ? 1 : 0) + (MODE == GROUPED_GRAD ? 1 : 0));  // readers of this CTA
    }
    fence_mbar_init();
    if (a.rows > 0) {  // without rows the operands' maps are not set up, and nothing is loaded
      prefetch_tensormap(&tmL);
      prefetch_tensormap(&tmC);
      if (!C_MN) prefetch_tensormap(&tmN);
    }
    if (a.tma_out) prefetch_tensormap(&tmD);
  }
  if (warp == 1) {
    tmem_alloc2(tmem_holder, TMEM_COLS);
    tmem_relinquish2();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive();
  cluster_wait();  // both CTAs' barriers are initialised and both halves of the TMEM pair are allocated
  tc_fence_after_sync();
  griddep_launch();  // programmatic dependent launch, after the tensor-memory allocation; nothing above touches global memory
  griddep_wait();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_holder);
  TileRing ring{ring_slots, ring_full, ring_empty, a.status, 0};
  GroupedTile tile;

  // Float32 tiles of 256 columns keep 128 sums a thread: the eight epilogue warps take registers over from the other four
  // (4 x 32 x 40 + 8 x 32 x 232 = 12 x 32 x 168).
  constexpr bool SHIFT_REGS = PROMOTE;
  if (warp < 4) {
    if (SHIFT_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer (both CTAs)
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint32_t leader_full0 = mapa_shared(smem_u32(&full[0]), 0);
        while (ok && ring.take(tile)) {
          ring.leave();
          const int kbs = tile.k_blocks;
          const int l0 = tile.lane0 + rank * 128, half = tile.width / 2, c0 = tile.col0 + rank * half;
          // only the columns that the instruction reads: narrow tiles are bound by these loads
          const int loads = C_MN ? (half + 63) / 64 : (half + kColBox - 1) / kColBox;
          const bool whole = !C_MN && loads * kColBox == BT / 2;  // one large box is faster than four small ones: 452 us against 479
          const uint32_t bytes = L_BYTES + loads * (C_MN ? BK * 128 : kColBox * 128);
          for (int kb = 0; kb < kbs; ++kb) {
            if (!mbar_wait(&empty[stage], phase ^ 1, a.status, SITEG_PROD_EMPTY)) { ok = false; break; }
            uint8_t* sl = smem + stage * STAGE_BYTES;
            uint8_t* sc = sl + L_BYTES;
            auto load = [&](auto&& load2, auto&& load3) {
              if constexpr (MODE == GROUPED_K_MAJOR) {
                load3(sl, &tmL, kb * BK, l0, tile.g);
              } else if constexpr (MODE == GROUPED_MN_MAJOR) {
                for (int c = 0; c < 2; ++c) load3(sl + c * (BK * 128), &tmL, l0 + c * 64, kb * BK, tile.g);
              } else {
                for (int c = 0; c < 2; ++c) load2(sl + c * (BK * 128), &tmL, l0 + c * 64, tile.row0 + kb * BK);
              }
              if constexpr (C_MN) {
                for (int c = 0; c < loads; ++c) load2(sc + c * (BK * 128), &tmC, c0 + c * 64, tile.row0 + kb * BK);
              } else if (whole) {
                load2(sc, &tmC, kb * BK, c0);
              } else {
                for (int c = 0; c < loads; ++c) load2(sc + c * (kColBox * 128), &tmN, kb * BK, c0 + c * kColBox);
              }
            };
            const bool cleared = MODE == GROUPED_GRAD && tile.nrows - kb * BK < BK;  // warp 2 passes this block on
            if (rank == 0 || cleared) {
              uint64_t* bar = cleared ? &tail[stage] : &full[stage];
              mbar_arrive_expect_tx(bar, bytes);
              load([&](uint8_t* d, const CUtensorMap* m, int x, int y) { tma_load_2d(d, m, bar, x, y); },
                   [&](uint8_t* d, const CUtensorMap* m, int x, int y, int z) { tma_load_3d(d, m, bar, x, y, z); });
            } else {
              const uint32_t bar = leader_full0 + stage * 8;
              mbar_arrive_expect_tx_remote(bar, bytes);
              load([&](uint8_t* d, const CUtensorMap* m, int x, int y) { tma_load_2d_pair(d, m, bar, x, y); },
                   [&](uint8_t* d, const CUtensorMap* m, int x, int y, int z) { tma_load_3d_pair(d, m, bar, x, y, z); });
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer (leader CTA only)
      if (lane == 0 && rank == 0) {
        int stage = 0;
        uint32_t phase = 0;
        int lt = 0;
        bool ok = true;
        const OperandDesc dl = make_operand_desc<BK, UMMA_K>(L_MN), dc = make_operand_desc<BK, UMMA_K>(C_MN);
        const uint32_t empty_local = smem_u32(&empty[0]), empty_peer = mapa_shared(empty_local, 1);
        while (ok && ring.take(tile)) {
          ring.leave();
          const int kbs = tile.k_blocks;
          const uint32_t idesc = a.idesc | ((uint32_t)(tile.width >> 3) << 17);
          for (int seg = 0; seg < kbs && ok; seg += PROMOTE ? kPromoteBlocks : kbs, ++lt) {
            const int buf = lt & 1, end = PROMOTE ? min(seg + kPromoteBlocks, kbs) : kbs;
            const uint32_t aphase = (lt >> 1) & 1;
            ok = mbar_wait(&acc_empty[buf], aphase ^ 1, a.status, SITEG_MMA_ACC);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t d_tmem = tmem_base + buf * BT;
            for (int kb = seg; kb < end; ++kb) {
              // a cleared block was written by threads of both CTAs
              ok = MODE == GROUPED_GRAD ? mbar_wait_cluster(&full[stage], phase, a.status, SITEG_MMA_FULL)
                                        : mbar_wait(&full[stage], phase, a.status, SITEG_MMA_FULL);
              if (!ok) break;
              tc_fence_after_sync();
              const uint32_t s = smem_u32(smem + stage * STAGE_BYTES);
              const uint64_t ld = dl.base + (s >> 4), cd = dc.base + ((s + L_BYTES) >> 4);
#pragma unroll
              for (int k = 0; k < BK / UMMA_K; ++k)
                tc_mma_ss2<KIND_F16>(d_tmem, ld + k * dl.kstep, cd + k * dc.kstep, idesc, (kb > seg || k > 0) ? 1u : 0u);
              tc_commit2(empty_local + stage * 8);
              tc_commit2(empty_peer + stage * 8);
              if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
            if (ok) {
              const uint32_t f_local = smem_u32(&acc_full[buf]);
              tc_commit2(f_local);
              tc_commit2(mapa_shared(f_local, 1));
            }
          }
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // ------------------------------------------------------------ rows behind a group's end (gradient, both CTAs)
      // The last block of a group reaches into the next group's rows, or past the last one, where anything may lie: those K
      // rows are zeroed in both operands.  A K row is 128 bytes in every chunk, swizzled within itself.
      if constexpr (MODE == GROUPED_GRAD) {
        int pos = 0;            // stages used before this tile
        uint32_t phases = 0;    // one bit per stage
        while (__all_sync(~0u, ring.take(tile))) {
          __syncwarp();
          if (lane == 0) ring.leave();
          else ++ring.n;
          const int kbs = tile.k_blocks, valid = tile.nrows - (kbs - 1) * BK;
          if (kbs > 0 && valid < BK) {
            const int stage = (pos + kbs - 1) % STAGES;
            // every lane waits: it is the wait that orders a lane's stores behind the loads that they overwrite
            if (!__all_sync(~0u, mbar_wait(&tail[stage], (phases >> stage) & 1, a.status, SITEG_FIX_TAIL))) break;
            phases ^= 1u << stage;
            uint8_t* sl = smem + stage * STAGE_BYTES;
            for (int c = 0; c < 2 + (tile.width / 2 + 63) / 64; ++c)
              for (int off = valid * 128 + lane * 16; off < BK * 128; off += 512)
                *reinterpret_cast<uint4*>(sl + c * (BK * 128) + off) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote_release(mapa_shared(smem_u32(&full[stage]), 0));
          }
          pos = (pos + kbs) % STAGES;
        }
      }
    } else if (warp == 3) {
      // ------------------------------------------------------------ tile scheduler (each CTA for itself, the same tiles)
      deal_tiles<MODE>(a, ring, first_tile, tile_step, lane);
    }
  } else {
    if (SHIFT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ------------------------------------------------------------ epilogue (warps 4..11, both CTAs)
    // Four warps read the tensor memory's four quarters of 32 lanes; two such sets share the blocks of 32 columns.
    const int q = warp & 3;
    const int set = (warp - 4) >> 2;
    uint8_t* my_epi = epi + (PROMOTE ? warp - 4 : (warp - 4) >> 1 << 1) * (EPI_BUFS * EPI_BUF);
    int buf = 0, lt = 0;
    bool ok = true;
    while (ok && all_of<128>(1 + set, ring.take(tile))) {
      if (lane == 0) ring.leave();
      else ++ring.n;
      const int kbs = tile.k_blocks;
      const int l0 = tile.lane0 + rank * 128, m = l0 + q * 32 + lane;
      OutT* row0 = static_cast<OutT*>(a.D) + (MODE == GROUPED_GRAD ? tile.g * a.group_stride : 0ll) + tile.col0 * a.ld;
      auto store_elements = [&](int c, const uint32_t (&v)[32]) {
        if (m < a.lanes) {
          OutT* p = row0 + c * a.ld + m;
          const int live = tile.ncols - c;
          float old[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) old[j] = 0.f;
          if (a.beta != 0.f) {  // all requests under way at once: rows behind the last read that one again
#pragma unroll
            for (int j = 0; j < 32; ++j) old[j] = load_c_as_float<OutT>(p, min(j, live - 1) * a.ld);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float x = __uint_as_float(v[j]) * a.alpha;
            if (j < live) p[j * a.ld] = cvt_out<OutT>(a.beta != 0.f ? x + a.beta * old[j] : x);
          }
        }
      };
      auto arrived = [&]() {  // waits for the accumulator of the next run
        // the four warps of a set go on or give up together: they meet again at the barriers of the stores
        ok = all_of<128>(1 + set, mbar_wait(&acc_full[lt & 1], (lt >> 1) & 1, a.status, SITEG_EPI_ACC));
        tc_fence_after_sync();
        return ok;
      };
      auto release = [&]() {  // hands the accumulator back after its last read
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) mbar_arrive(&acc_empty[lt & 1]);
          else mbar_arrive_remote(mapa_shared(smem_u32(&acc_empty[lt & 1]), 0));
        }
        ++lt;
      };
      const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      if constexpr (PROMOTE) {
        constexpr int MINE = (BT + 63) / 64;  // this set's blocks of 32 columns, from 64 i + 32 set on
        float acc[MINE * 32];
#pragma unroll
        for (int j = 0; j < MINE * 32; ++j) acc[j] = 0.f;
        for (int seg = 0; seg < kbs; seg += kPromoteBlocks) {
          if (!arrived()) break;
#pragma unroll
          for (int i = 0; i < MINE; ++i) {
            const int c = i * 64 + set * 32;
            if (c < tile.width) {
              uint32_t v[32];
              tmem_ld_x32(t_lane + (lt & 1) * BT + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) acc[i * 32 + j] += __uint_as_float(v[j]);
            }
          }
          release();
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int c = i * 64 + set * 32;
          if (c < tile.width) {
            uint32_t v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(acc[i * 32 + j]);
            if (a.vec_out) {
              // [32 columns][32 lanes] per warp, stored as rows of 128 bytes
              float* sb = reinterpret_cast<float*>(my_epi + buf * EPI_BUF);
              buf ^= 1;
              const bool add = a.beta == 1.f;  // the memory adds: nothing is read
              const bool whole = a.tma_out && (MODE == GROUPED_GRAD || c + 32 <= tile.ncols);
              if (lane == 0) tma_store_wait_read<1>();
              __syncwarp();  // the block that was here has left
#pragma unroll
              for (int j = 0; j < 32; ++j) sb[j * 32 + lane] = __uint_as_float(v[j]) * a.alpha;
              if (whole) {
                fence_proxy_async_smem();
                __syncwarp();
                const int x = l0 + q * 32;
                if (lane == 0 && x < a.lanes) {
                  if constexpr (MODE == GROUPED_GRAD) {
                    if (add) tma_reduce_add_3d(&tmD, sb, x, tile.col0 + c, tile.g);
                    else tma_store_3d(&tmD, sb, x, tile.col0 + c, tile.g);
                  } else {
                    if (add) tma_reduce_add_2d(&tmD, sb, x, tile.col0 + c);
                    else tma_store_2d(&tmD, sb, x, tile.col0 + c);
                  }
                }
                if (lane == 0) tma_store_commit();
                continue;
              }
              if (lane == 0) tma_store_commit();  // an empty group: every block counts as one
              __syncwarp();
              const int x = l0 + q * 32 + (lane & 7) * 4, j0 = lane >> 3;
              float4 w[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) w[k] = *reinterpret_cast<const float4*>(sb + (k * 4 + j0) * 32 + (lane & 7) * 4);
              float* p = reinterpret_cast<float*>(row0) + c * a.ld + x;
              const int live = x < a.lanes ? tile.ncols - c : 0;  // rows k * 4 + j0 < live are stored
              if (x + 4 <= a.lanes) {
                if (a.beta != 0.f) {
                  float4 old[8];
#pragma unroll
                  for (int k = 0; k < 8; ++k) old[k] = *reinterpret_cast<const float4*>(p + min(k * 4 + j0, live - 1) * a.ld);
#pragma unroll
                  for (int k = 0; k < 8; ++k)
                    w[k] = make_float4(w[k].x + a.beta * old[k].x, w[k].y + a.beta * old[k].y, w[k].z + a.beta * old[k].z, w[k].w + a.beta * old[k].w);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  if (k * 4 + j0 < live) *reinterpret_cast<float4*>(p + (k * 4 + j0) * a.ld) = w[k];
              } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  if (k * 4 + j0 < live) {
                    const float e[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
                    float* to = p + (k * 4 + j0) * a.ld;
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                      if (x + i < a.lanes) to[i] = a.beta != 0.f ? e[i] + a.beta * to[i] : e[i];
                  }
                }
              }
            } else {
              store_elements(c, v);
            }
          }
        }
      } else {
        if (kbs > 0 && !arrived()) break;
        const int t_buf = (lt & 1) * BT;
        const int blocks = tile.width / 32, last = (blocks - 1 - set) / 2 * 2 + set;  // this set's last block (below 0: none)
        if (kbs > 0 && blocks <= set) release();
        // Two blocks at a time: short sums are bound by a block's latencies (tensor-memory load, conversion, proxy fence,
        // barriers; 0.8 us of them), which two have in common (64 weight gradients of 2048 x 2048, one row each: 163 -> 128 us).
#pragma unroll 1
        for (int blk = set; blk < blocks; blk += 4) {
          const int both = blk + 2 < blocks ? 2 : 1;
          if (a.vec_out) {
            // Two warps share two staging tiles [32 columns][128 bytes of 64 lanes] in the 128-byte swizzle.  Whole 8 x 8
            // fragments are staged transposed: single 16-bit elements would take twice the shared-memory cycles, which the tensor
            // cores need for their operands.
            uint32_t f[2][4][4];
            {
              uint32_t v[4][16];
              if (kbs > 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (h < both) {
                    tmem_ld_16x32(t_lane + t_buf + (blk + 2 * h) * 32, v[2 * h]);
                    tmem_ld_16x32(t_lane + t_buf + (blk + 2 * h) * 32 + (16u << 16), v[2 * h + 1]);
                  }
                tmem_ld_wait();
                if (blk + 2 * both - 2 == last) release();
              } else {
#pragma unroll
                for (int j = 0; j < 64; ++j) v[j >> 4][j & 15] = 0u;
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const int h = j >> 4, b = (j >> 2) & 3, i = j & 3;
                f[h][b][i] = pack_pair<OutT>(__uint_as_float(v[2 * h + (i >> 1)][4 * b + 2 * (i & 1)]) * a.alpha,
                                             __uint_as_float(v[2 * h + (i >> 1)][4 * b + 2 * (i & 1) + 1]) * a.alpha);
              }
            }
            // the tiles are free when the stores of the last step have read them, and both warps are done with it
            const bool storer = (q & 1) == 0 && lane == 0;
            auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(3 + ((warp - 4) >> 1)) : "memory"); };  // barriers 3..6
            if (storer) tma_store_wait_read<0>();
            meet();
            const int row = lane & 7, unit = (q & 1) * 4 + (lane >> 3);  // this thread's row and fragment of every group of four
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (h < both) {
#pragma unroll
                for (int b = 0; b < 4; ++b)
                  stmatrix_x4_trans(smem_u32(my_epi + h * EPI_BUF) + (b * 8 + row) * 128 + ((unit ^ row) << 4), f[h][b][0], f[h][b][1],
                                    f[h][b][2], f[h][b][3]);
              }
            fence_proxy_async_smem();
            meet();
            // A block that belongs to this tile as a whole goes out by TMA, the last rows of a group by vector stores.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h >= both) break;
              const int c = (blk + 2 * h) * 32;
              const uint8_t* from = my_epi + h * EPI_BUF;
              if (a.tma_out && (MODE == GROUPED_GRAD || c + 32 <= tile.ncols)) {
                const int x = l0 + (q >> 1) * 64;
                if (storer && x < a.lanes) {
                  if constexpr (MODE == GROUPED_GRAD) tma_store_3d(&tmD, from, x, tile.col0 + c, tile.g);
                  else tma_store_2d(&tmD, from, x, tile.col0 + c);
                  tma_store_commit();
                }
                continue;
              }
              const int x = l0 + (q >> 1) * 64 + (lane & 7) * 8, j0 = (q & 1) * 16 + (lane >> 3);
              uint4 w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = *reinterpret_cast<const uint4*>(from + (j0 + i * 4) * 128 + (((lane & 7) ^ ((j0 + i * 4) & 7)) << 4));
              OutT* p = row0 + (c + j0) * a.ld + x;
              const int live = x < a.lanes ? tile.ncols - c - j0 : 0;  // rows i * 4 < live are stored
              if (x + 8 <= a.lanes) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (i * 4 < live) *reinterpret_cast<uint4*>(p + i * 4 * a.ld) = w[i];
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                  for (int k = 0; k < 7; ++k)  // constant indices: `w` stays in registers
                    if (i * 4 < live && x + k < a.lanes) p[i * 4 * a.ld + k] = reinterpret_cast<const OutT*>(&w[i])[k];
              }
            }
          } else {
            for (int h = 0; h < both; ++h) {
              const int c = (blk + 2 * h) * 32;
              uint32_t v[32];
              if (kbs > 0) {
                tmem_ld_x32(t_lane + t_buf + c, v);
                tmem_ld_wait();
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0u;
              }
              if (kbs > 0 && blk + 2 * h == last) release();
              store_elements(c, v);
            }
          }
        }
      }
    }
  }

  if (warp >= 4) tma_store_wait_all<0>();

  // ---------------------------------------------------------------- teardown
  if (*reinterpret_cast<volatile int*>(a.status) != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // a wait gave up: copies in flight get time to land
  }
  tc_fence_before_sync();
  __syncthreads();
  // neither CTA may leave while its partner can still signal its barriers or read its operands
  cluster_arrive();
  cluster_wait();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc2(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------- host side
template <int MODE, typename OutT>
static int launch_grouped_inst(moye_b200_ctx* h, const CUtensorMap& tl, const CUtensorMap& tc, const CUtensorMap& tn, const CUtensorMap& td,
                               const GroupedArgs& a, long long tiles, cudaStream_t stream) {
  constexpr int EXTRA = 1024 + 1024 + 8 * grouped_epi_bufs<OutT>() * 32 * 128;
  constexpr int STAGE = 128 * 128 + BT / 2 * 128;
  constexpr int STAGES = (227 * 1024 - EXTRA) / STAGE;
  constexpr int SMEM = STAGES * STAGE + EXTRA;
  auto kern = gemm_grouped_kernel<MODE, OutT, STAGES>;
  if (int rc = configure_once(h, kern, SMEM)) return rc;
  if (sizeof(OutT) == 4) {  // what the epilogue takes over has to be there, or it would wait for it
    static const int regs = [&] {
      cudaFuncAttributes attr = {};
      return cudaFuncGetAttributes(&attr, kern) == cudaSuccess ? attr.numRegs : 0;
    }();
    if (regs < 168) MOYE_FAIL(MOYE_ERR_CUDA, "the Float32 kernel was built with %d registers a thread, 168 are needed", regs);
  }
  const long long pairs = tiles < h->num_sms / 2 ? tiles : h->num_sms / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = launch_without_pdl() ? 1 : 2;
  MOYE_CUDA(cudaLaunchKernelEx(&cfg, kern, tl, tc, tn, td, a));
  return MOYE_OK;
}

template <int MODE>
static int launch_grouped(int out, moye_b200_ctx* h, const CUtensorMap& tl, const CUtensorMap& tc, const CUtensorMap& tn, const CUtensorMap& td,
                          const GroupedArgs& a, long long tiles, cudaStream_t stream) {
  if (out == MOYE_F32) return launch_grouped_inst<MODE, float>(h, tl, tc, tn, td, a, tiles, stream);
  if (out == MOYE_F16) return launch_grouped_inst<MODE, __half>(h, tl, tc, tn, td, a, tiles, stream);
  return launch_grouped_inst<MODE, __nv_bfloat16>(h, tl, tc, tn, td, a, tiles, stream);
}

static int check_grouped_types(const char* who, const moye_tensor_t* x, const moye_tensor_t* y, const moye_tensor_t* out) {
  if ((x->dtype != MOYE_F16 && x->dtype != MOYE_BF16) || y->dtype != x->dtype)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "%s: operands must both be f16 or both bf16 (got %d, %d)", who, x->dtype, y->dtype);
  if (out->dtype != MOYE_F32 && out->dtype != x->dtype)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "%s: the output must be f32 or the operands' type (got %d)", who, out->dtype);
  return MOYE_OK;
}

// A matrix of rows read by TMA: contiguous rows, base and pitch on 16 bytes.
static int check_row_operand(const char* who, const char* what, const moye_tensor_t* t) {
  if (t->shape[1] > 1 && t->stride[1] != 1) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows of %s must be contiguous", who, what);
  if (t->shape[0] > 1 && t->stride[0] < t->shape[1]) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows of %s overlap", who, what);
  if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) != 0 || (t->shape[0] > 1 && (t->stride[0] * 2) % 16 != 0))
    MOYE_FAIL(MOYE_ERR_MISALIGNED, "%s: %s needs a base and a row pitch that are multiples of 16 bytes", who, what);
  return MOYE_OK;
}

// Bytes from row to row, of any tensor map's liking where there is but one row, whose pitch says nothing.
static uint64_t row_pitch(const moye_tensor_t* t) {
  const uint64_t eb = dtype_bytes(t->dtype);
  return t->shape[0] > 1 ? t->stride[0] * eb : (t->shape[1] * eb + 15) / 16 * 16;
}

// Weights of all groups as one matrix of rows, for `rows_overlap`: exact where the groups follow one another in the rows'
// own pitch, else a row is all that lies between a group's ends.
static moye_tensor_t weight_rows(const moye_tensor_t* t, int64_t inner, int64_t outer, int64_t pitch) {
  moye_tensor_t m = *t;
  m.rank = 2;
  const bool even = t->shape[0] == 1 || t->stride[0] == outer * pitch;
  m.shape[0] = even ? t->shape[0] * outer : t->shape[0];
  m.shape[1] = even ? inner : (outer - 1) * pitch + inner;
  m.stride[0] = even ? pitch : t->stride[0];
  m.stride[1] = 1;
  return m;
}

static int check_borders(const char* who, const int* offsets, int groups) {
  if (groups < 1 || groups > kMaxGemmGroups)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: 1 to %d groups (got %d)", who, kMaxGemmGroups, groups);
  if (!offsets) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "%s: null offsets", who);
  return MOYE_OK;
}

int launch_gemm_grouped(moye_b200_ctx* h, const moye_tensor_t* D, const moye_tensor_t* A, const moye_tensor_t* B, const int* offsets,
                        float alpha, float beta, cudaStream_t stream) {
  const char* who = "gemm_grouped";
  if (D->rank != 2 || A->rank != 2 || B->rank != 3) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: D and A must be rank 2, B rank 3", who);
  const int64_t R = A->shape[0], K = A->shape[1], G = B->shape[0], N = B->shape[1];
  if (B->shape[2] != K || D->shape[0] != R || D->shape[1] != N)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: shape mismatch: A (%lld,%lld) B (%lld,%lld,%lld) D (%lld,%lld)", who, (long long)R,
              (long long)K, (long long)G, (long long)N, (long long)B->shape[2], (long long)D->shape[0], (long long)D->shape[1]);
  if (int rc = check_grouped_types(who, A, B, D)) return rc;
  if (R < 0 || N <= 0 || K <= 0) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: empty product", who);
  if (R > kMaxGroupedExtent || N > kMaxGroupedExtent || K > kMaxGroupedExtent) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "%s: extent too large", who);
  if (int rc = check_borders(who, offsets, (int)(G > INT32_MAX ? INT32_MAX : G))) return rc;
  if (R == 0) return MOYE_OK;
  if (!A->ptr || !B->ptr || !D->ptr) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "%s: null data pointer", who);
  if (int rc = check_row_operand(who, "A", A)) return rc;
  if ((N > 1 && D->stride[1] != 1) || (R > 1 && D->stride[0] < N))
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows of D must be contiguous and must not overlap", who);
  const bool mn = K > 1 ? B->stride[2] != 1 : (B->stride[1] == 1 && N > 1);
  const int64_t inner = mn ? N : K, outer = mn ? K : N, pitch = mn ? B->stride[2] : B->stride[1];
  if (mn && N > 1 && B->stride[1] != 1) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: B needs a unit stride along K or along N", who);
  if ((outer > 1 && pitch < inner) || (G > 1 && B->stride[0] < (outer - 1) * pitch + inner))
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows or groups of B overlap", who);
  if ((reinterpret_cast<uintptr_t>(B->ptr) & 15) != 0 || (outer > 1 && pitch % 8 != 0) || (G > 1 && B->stride[0] % 8 != 0))
    MOYE_FAIL(MOYE_ERR_MISALIGNED, "%s: B needs a base, a row pitch and a group pitch that are multiples of 16 bytes", who);
  const moye_tensor_t weights = weight_rows(B, inner, outer, outer > 1 ? pitch : inner);
  if (rows_overlap(D, A) || rows_overlap(D, &weights)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "%s: D overlaps an operand", who);
  const int ob = dtype_bytes(D->dtype);
  GroupedArgs a = {};
  a.rows = (int)R;
  a.groups = (int)G;
  a.lanes = (int)N;
  a.k_blocks = (int)((K + 63) / 64);
  a.lane_tiles = (int)((N + 255) / 256);
  a.vec_out = (beta == 0.f || ob == 4) && (reinterpret_cast<uintptr_t>(D->ptr) & 15) == 0 && (R == 1 || (D->stride[0] * ob) % 16 == 0);
  a.offsets = offsets;
  const uint32_t fmt = A->dtype == MOYE_BF16 ? 1u : 0u;
  a.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((mn ? 1u : 0u) << 15) | (16u << 24);
  a.alpha = alpha;
  a.beta = beta;
  a.D = D->ptr;
  a.ld = D->stride[0];
  a.status = h->d_status;
  const long long live = G < R ? G : R, tiles = (live + (R - live) / BT) * a.lane_tiles;  // at most
  if (tiles > INT32_MAX / 2) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "%s: too many tiles", who);
  CUtensorMap tl, tc, tn, td;
  std::memset(&td, 0, sizeof(td));
  if (int rc = encode_tmap_3d(&tl, B->ptr, B->dtype, inner, outer, G, (outer > 1 ? pitch : (inner + 7) / 8 * 8) * 2,
                              (G > 1 ? B->stride[0] : (inner + 7) / 8 * 8) * 2, 64, mn ? 64 : 128, true))
    return rc;
  if (int rc = encode_tmap_2d_uncached(&tc, A->ptr, A->dtype, K, R, row_pitch(A), 64, BT / 2, true)) return rc;
  if (int rc = encode_tmap_2d_uncached(&tn, A->ptr, A->dtype, K, R, row_pitch(A), 64, kColBox, true)) return rc;
  a.tma_out = a.vec_out && (beta == 0.f || beta == 1.f) && (a.lanes * ob) % 16 == 0;  // TMA writes whole 16-byte units, past an odd extent too
  if (a.tma_out)
    if (int rc = encode_tmap_2d_uncached(&td, D->ptr, D->dtype, N, R, row_pitch(D), ob == 2 ? 64 : 32, 32, ob == 2)) return rc;
  log_line("gemm_grouped %lld rows, %lld groups, %lld x %lld  in %d", (long long)R, (long long)G, (long long)N,
           (long long)K, A->dtype);
  if (mn) return launch_grouped<GROUPED_MN_MAJOR>(D->dtype, h, tl, tc, tn, td, a, tiles, stream);
  return launch_grouped<GROUPED_K_MAJOR>(D->dtype, h, tl, tc, tn, td, a, tiles, stream);
}

int launch_gemm_grouped_grad(moye_b200_ctx* h, const moye_tensor_t* dB, const moye_tensor_t* dD, const moye_tensor_t* A,
                             const int* offsets, float alpha, float beta, cudaStream_t stream) {
  const char* who = "gemm_grouped_grad";
  if (dB->rank != 3 || dD->rank != 2 || A->rank != 2) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: dD and A must be rank 2, dB rank 3", who);
  const int64_t R = A->shape[0], K = A->shape[1], G = dB->shape[0], N = dB->shape[1];
  if (dB->shape[2] != K || dD->shape[0] != R || dD->shape[1] != N)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: shape mismatch: A (%lld,%lld) dD (%lld,%lld) dB (%lld,%lld,%lld)", who, (long long)R,
              (long long)K, (long long)dD->shape[0], (long long)dD->shape[1], (long long)G, (long long)N, (long long)dB->shape[2]);
  if (int rc = check_grouped_types(who, A, dD, dB)) return rc;
  if (R < 0 || N <= 0 || K <= 0) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: empty product", who);
  if (R > kMaxGroupedExtent || N > kMaxGroupedExtent || K > kMaxGroupedExtent) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "%s: extent too large", who);
  if (int rc = check_borders(who, offsets, (int)(G > INT32_MAX ? INT32_MAX : G))) return rc;
  if (!dB->ptr || (R > 0 && (!A->ptr || !dD->ptr))) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "%s: null data pointer", who);
  if (int rc = check_row_operand(who, "A", A)) return rc;
  if (int rc = check_row_operand(who, "dD", dD)) return rc;
  if ((K > 1 && dB->stride[2] != 1) || (N > 1 && dB->stride[1] < K) || (G > 1 && dB->stride[0] < (N - 1) * dB->stride[1] + K))
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: dB needs contiguous rows, and rows and groups that do not overlap", who);
  const moye_tensor_t weights = weight_rows(dB, K, N, N > 1 ? dB->stride[1] : K);
  if (rows_overlap(&weights, dD) || rows_overlap(&weights, A)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "%s: dB overlaps an operand", who);
  const int ob = dtype_bytes(dB->dtype);
  GroupedArgs a = {};
  a.rows = (int)R;
  a.groups = (int)G;
  a.lanes = (int)K;
  a.cols = (int)N;
  a.lane_tiles = (int)((K + 255) / 256);
  a.col_tiles = (int)((N + BT - 1) / BT);
  a.vec_out = (beta == 0.f || ob == 4) && (reinterpret_cast<uintptr_t>(dB->ptr) & 15) == 0 && (N == 1 || (dB->stride[1] * ob) % 16 == 0) &&
              (G == 1 || (dB->stride[0] * ob) % 16 == 0);
  a.offsets = offsets;
  const uint32_t fmt = A->dtype == MOYE_BF16 ? 1u : 0u;
  a.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (3u << 15) | (16u << 24);
  a.alpha = alpha;
  a.beta = beta;
  a.D = dB->ptr;
  a.ld = dB->stride[1];
  a.group_stride = dB->stride[0];
  a.status = h->d_status;
  const long long tiles = (long long)G * a.lane_tiles * a.col_tiles;
  if (tiles > INT32_MAX / 2) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "%s: too many tiles", who);
  CUtensorMap tl, tc, tn, td;
  std::memset(&td, 0, sizeof(td));
  std::memset(&tn, 0, sizeof(tn));
  std::memset(&tl, 0, sizeof(tl));
  std::memset(&tc, 0, sizeof(tc));
  if (R > 0) {  // without rows the kernel loads nothing, every group's sum is empty
    if (int rc = encode_tmap_2d_uncached(&tl, A->ptr, A->dtype, K, R, row_pitch(A), 64, 64, true)) return rc;
    if (int rc = encode_tmap_2d_uncached(&tc, dD->ptr, dD->dtype, N, R, row_pitch(dD), 64, 64, true)) return rc;
  }
  a.tma_out = a.vec_out && (beta == 0.f || beta == 1.f) && (a.lanes * ob) % 16 == 0;  // TMA writes whole 16-byte units, past an odd extent too
  if (a.tma_out) {
    const uint64_t row = N > 1 ? (uint64_t)dB->stride[1] * ob : ((uint64_t)K * ob + 15) / 16 * 16;
    const uint64_t group = G > 1 ? (uint64_t)dB->stride[0] * ob : (uint64_t)N * row;
    if (int rc = encode_tmap_3d(&td, dB->ptr, dB->dtype, K, N, G, row, group, ob == 2 ? 64 : 32, 32, ob == 2)) return rc;
  }
  log_line("gemm_grouped_grad %lld rows, %lld groups, %lld x %lld  in %d", (long long)R, (long long)G,
           (long long)N, (long long)K, A->dtype);
  return launch_grouped<GROUPED_GRAD>(dB->dtype, h, tl, tc, tn, td, a, tiles, stream);
}

}  // namespace moye
