// Products grouped by expert, and products of 4-bit microscaled operands (sm_100a).
//
// Rows 0..T-1 of a token matrix belong to E groups: group e owns rows offsets[e] .. offsets[e+1]-1
// (offsets lie in device memory; the host never reads them).  One kernel body, four modes:
//
//   kFwd  out[r, n]    = sum_k x[r, k]  * w[e(r), n, k]
//   kDx   dx[r, k]     = sum_n dy[r, n] * w[e(r), n, k]
//   kDw   dw[e, n, k]  = sum_{r in e} dy[r, n] * x[r, k]        (zeros for a group without rows)
//   kMx   kFwd with both operands in MXFP4; with offsets == nullptr one group of all T rows, which is
//         the dense product C = A * B^T
//
// All are D[m, c] = sum_j A[m, j] * B[c, j] with D's M axis on the 128 TMEM lanes.  The M axis is
// always the contiguous axis of the output (a feature), never the ragged one: a tile's columns are
// tokens, and the width of an MMA is chosen per tile in steps of 16 (N of tcgen05.mma), so a group of
// five rows costs a 128 x 16 product and not a 128 x 128 one.  With the roles the other way round a
// group's last tile would always be computed 128 rows high.  The epilogue stores output rows: 32 lanes of
// fp32 are 128 consecutive bytes; 16-bit values go through shared memory to 16-byte pieces, or one by one
// where a row is no multiple of 16 bytes, so no output extent has an alignment rule.
//
//   mode   A (M axis)                     B (columns)              reduction
//   kFwd   w, K-major                     x, K-major               K
//   kDx    w, MN-major (k contiguous)     dy, K-major              N
//   kDw    x, MN-major (k contiguous)     dy, MN-major             the group's rows (ragged)
//   kMx    w codes, K-major               x codes, K-major         K
//
// Operand layouts, the ring of TMA stages, the roles of the warps and the bounded waits are those of
// hb_umma_kernel (hb_kernel.cuh).  In kDw a group's last block of 64 rows usually reaches into the
// next group: a warp writes zeros over those rows of both operands (another group's infinity times zero
// would be NaN) up to the next multiple of 16, and no MMA is issued beyond it.
//
// Tiles are listed on the device: every CTA reads the offsets, keeps the groups that have rows (all
// of them in kDw) with a running count of tiles in shared memory, and walks tiles blockIdx.x,
// blockIdx.x + gridDim.x, ...  A group's rows are cut into equal tiles, not full ones and a rest, so
// that the tiles of a wave cost about the same.  (Dealing the groups out by falling cost of their tiles made
// no difference: 8192 rows over 32 experts 85.6 - 88.4 us sorted, 82.8 - 90.5 in order.  Taking half of the lists
// backwards, so that wide and narrow tiles meet, cost 7 %: neighbours then share fewer operands in L2.)
//
// A CTA pair (CG = 2) shares tiles of 256 features as in hb_umma_kernel; in kMx each CTA brings the scales of its
// own features and of all the tile's rows.  SPLIT: the 2, 4 or 8 CTAs of a cluster share a tile's reduction
// and join their sums through distributed shared memory, in the order of the shares.
//
// What bounds it (B200; loops of 0.15 s, in brackets loops of some 10 ms, whose clocks are higher): 8192 rows over 32
// experts of 2048 x 2048 bf16 88 us (73), 335 MB of traffic at 3.8 TB/s (4.6), tensor cores active 62 %; dx and dw of 8192
// rows, 16 groups of 2048 x 1024, 96 us (41 + 44): dx has 160 tiles for 74 pairs, 2.2 rounds paid as three; in dw the tensor
// cores are active 48 % and the operands' path 41 %, and what it waits for is not known (CTA pairs, which halve B's way
// through shared memory, were level); 4096^3 in 4 bits 39.5 us (34.9): 256 tiles for 74 pairs are 3.46 rounds paid as four,
// each with one accumulator, and a block's scale copies and MMAs take their issuing thread about as long (460 cycles)
// as the tensor core (512).
// Offsets are clamped to [0, T] and a group whose end
// lies before its start counts as empty: wrong offsets give wrong rows, never an access out of range.
#pragma once
#include "hb_kernel.cuh"
#include <cuda_bf16.h>

namespace hb {

enum { kFwd = 0, kDx = 1, kDw = 2, kMx = 3 };

constexpr int kMaxGroups = 1024;
// A producer, MMA, the epilogue warps, B producer; kDw: the zeros behind a group; kMx: the scales' producer.
// Eight epilogue warps, two to each quarter of the TMEM lanes (with four the weight gradient waited for its
// accumulators); four in the narrow form, of which two CTAs share an SM.
__host__ __device__ constexpr int group_epi(bool narrow) { return narrow ? 4 : 8; }
__host__ __device__ constexpr int group_threads(int mode, bool narrow) {
  return 32 * (3 + group_epi(narrow) + (mode == kMx || mode == kDw ? 1 : 0));
}
// epilogue staging of a warp: 32 columns x 32 16-bit values, twice in the wide form
__host__ __device__ constexpr int group_staging(bool narrow) { return narrow ? 2048 : 4096; }
constexpr int kSpan = 128;             // bytes of the reduction axis in a ring stage (TMA swizzle span)
constexpr int kAtomBytes = 512;        // scales of 128 rows x 128 elements

struct GroupParams {
  const int* offsets;   // E + 1; nullptr: one group of T rows
  int E, T;
  int M;                // extent of the M axis (the output's contiguous extent)
  int C;                // kDw: extent of the column axis; otherwise unused (columns are a group's rows)
  int R;                // extent of the reduction axis; kDw: unused (a group's rows)
  int BN;               // widest tile, a multiple of 64
  int stages, acc_stages, tmem_cols, tiles_m;
  int out_type;         // 0: fp32, 1: fp16, 2: bf16
  int wide_rows;        // 16-bit output whose rows are multiples of 16 bytes
  int ksplit;           // SPLIT: CTAs of a cluster that share a tile's reduction
  uint32_t idesc;       // without the N field
  void* out;
  long long ldc;        // elements between consecutive output rows
  long long out_group;  // kDw: elements between the outputs of consecutive groups
  const uint8_t* sfa;   // kMx: scales of w (per expert) and of the token matrix
  const uint8_t* sfb;
  int silent_producer;  // test hook, see hb_knobs
  long long wait_limit_cycles;
};

// One group as the walkers see it.
struct GroupEntry {
  int e, start, n, end_tile;  // index, first row, rows, one past its last tile
};

struct GroupTile {
  int e, start, n;  // group
  int m0;           // first M index of the (pair) tile
  int c0, ncols;    // first column within the group (kDw: of the column axis) and valid columns
  int nmma;         // columns the MMA computes
  int blocks;       // reduction blocks
  int kb0, kb1;     // those of this CTA
};

__host__ __device__ __forceinline__ int round_up(int v, int step) { return (v + step - 1) / step * step; }

// Column tiles of a group with n rows and the width of all but its last.  Widths are multiples of the
// MMA's column step; in kMx a tile starts at a multiple of 64 rows of its group (128 where the widest
// tile is a multiple of 128), because scales lie in tiles of 128 rows.
template <int MODE, int CG>
__host__ __device__ __forceinline__ int group_width(int n, int tiles, int BN) {
  if (tiles <= 1) return BN;
  const int step = MODE == kMx ? (BN % 128 ? 64 : 128) : 16 * CG;
  return round_up((n + tiles - 1) / tiles, step);
}

template <int MODE, int CG>
__device__ __forceinline__ bool group_tile(const GroupParams& p, const GroupEntry* g, int& at, int t, int total,
                                           GroupTile& o) {
  if (t >= total) return false;
  while (g[at].end_tile <= t) ++at;  // (tiles are taken in ascending order)
  const GroupEntry ge = g[at];
  const int first = at ? g[at - 1].end_tile : 0;
  o.e = ge.e;
  o.start = ge.start;
  o.n = ge.n;
  const int cols = MODE == kDw ? p.C : ge.n;
  const int ct = (cols + p.BN - 1) / p.BN;
  const int r = t - first;
  const int mt = r / ct;
  o.m0 = mt * kTileM * CG;
  const int w = group_width<MODE, CG>(cols, ct, p.BN);
  o.c0 = (r - mt * ct) * w;
  o.ncols = min(w, cols - o.c0);
  o.nmma = round_up(o.ncols, 16 * CG);
  constexpr int kElems = MODE == kMx ? 256 : 64;  // reduction elements of a stage
  const int red = MODE == kDw ? ge.n : p.R;
  o.blocks = (red + kElems - 1) / kElems;
  return true;
}

// Fills the group list; called by all threads, ends behind a barrier.  Returns the tile count.
template <int MODE, int CG>
__device__ __forceinline__ int group_list(const GroupParams& p, GroupEntry* g, int* total) {
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int s = 0, t = p.T;
    if (p.offsets) {
      s = min(max(p.offsets[e], 0), p.T);
      t = min(max(p.offsets[e + 1], s), p.T);
    }
    g[e].start = s;
    g[e].n = t - s;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int kept = 0;
    // (in 64 bits and cut at 2^30, which no ascending offsets reach: a row in many groups at once must not make
    // the counts wrap and a walker run past the list)
    long long sum = 0;
    constexpr long long kMost = 1LL << 30;
    for (int base = 0; base < p.E; base += 32) {
      const int e = base + lane;
      const int start = e < p.E ? g[e].start : 0, n = e < p.E ? g[e].n : 0;
      const int cols = MODE == kDw ? (e < p.E ? p.C : 0) : n;
      const int tiles = (cols + p.BN - 1) / p.BN * p.tiles_m;
      const uint32_t has = __ballot_sync(0xffffffffu, tiles > 0);
      long long incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      // (every lane holds its group in registers: the entries written below are at or before these)
      if (tiles > 0) {
        const int slot = kept + __popc(has & ((1u << lane) - 1u));
        g[slot] = GroupEntry{e, start, n, static_cast<int>(min(sum + incl, kMost))};
      }
      __syncwarp();
      kept += __popc(has);
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) *total = static_cast<int>(min(sum, kMost));
  }
  __syncthreads();
  return *total;
}

struct GroupBars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t edge[kMaxStages];  // kDw: the stage's edge is zero
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint64_t red_full, red_empty;  // SPLIT: a share's partial sums are here; are read
  uint32_t tmem_base;
  int abort_flag;
  int total;
};

// Bytes of a ring stage of one CTA: operands, and in kMx the scales of 256 elements: one tile row of
// scales for A, up to two for B's columns.
__host__ __device__ __forceinline__ int group_sf_rows(int BN) { return BN <= 64 ? 1 : (BN + 127) / 128; }
template <int MODE, int CG>
__host__ __device__ __forceinline__ int group_stage_bytes(int BN) {
  return (kTileM + BN / CG) * kSpan + (MODE == kMx ? (1 + group_sf_rows(BN)) * 2 * kAtomBytes : 0);
}

// Two accumulators rounded to the 16-bit output type (one rounding, to nearest even).
__device__ __forceinline__ uint32_t pack16(int out_type, uint32_t a, uint32_t b) {
  if (out_type == 1) {
    const __half2 h = __floats2half2_rn(__uint_as_float(a), __uint_as_float(b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(a), __uint_as_float(b));
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int MODE, int CG, bool SPLIT = false, bool NARROW = false>
__global__ void __launch_bounds__(group_threads(MODE, NARROW), NARROW ? 2 : 1)
hb_group_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmB16, const __grid_constant__ CUtensorMap tmBw,
                const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const GroupParams p) {
  constexpr bool A_MN = MODE == kDx || MODE == kDw;
  constexpr bool B_MN = MODE == kDw;
  constexpr int kElems = MODE == kMx ? 256 : 64;
  constexpr int kGroupEpi = group_epi(NARROW), kGroupStage = group_staging(NARROW);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  static_assert(!NARROW || (CG == 1 && !SPLIT && MODE != kDw), "the narrow form is one of single CTAs");
  static_assert(!SPLIT || (CG == 1 && (MODE == kFwd || MODE == kMx)), "the joined form is that of the forward products");
  const uint32_t cta_rank = (CG == 2) ? cluster_ctarank() : 0u;
  const bool leader = cta_rank == 0u;
  constexpr int a_bytes = kTileM * kSpan;
  const int b_bytes = p.BN / CG * kSpan;
  const int sf_rows = group_sf_rows(p.BN);
  const int sf_bytes = MODE == kMx ? (1 + sf_rows) * 2 * kAtomBytes : 0;  // A's tile row first, then B's
  const uint32_t sA = smem_base;
  const uint32_t sB = sA + p.stages * a_bytes;
  const uint32_t sSF = sB + p.stages * b_bytes;
  const uint32_t sEpi = sSF + p.stages * sf_bytes;
  uint8_t* after = smem + (sEpi - smem_base) + kGroupEpi * kGroupStage;
  GroupBars* bars = reinterpret_cast<GroupBars*>(after);
  GroupEntry* groups = reinterpret_cast<GroupEntry*>(after + ((sizeof(GroupBars) + 15) & ~15));
  // SPLIT: partial sums of this CTA's share of the lanes, [source][column][lane]
  const int ks = SPLIT ? p.ksplit : 1;
  const int ks_rank = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  float* const red = reinterpret_cast<float*>(groups + p.E);
  volatile int* abort_flag = &bars->abort_flag;
  const WaitCtx wctx{abort_flag, p.wait_limit_cycles > 0 ? p.wait_limit_cycles : HB_WAIT_LIMIT_CYCLES};
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), MODE == kDw ? 2 : 1);
      mbar_init(smem_u32(&bars->edge[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bars->tmem_full[a]), 1);
      mbar_init(smem_u32(&bars->tmem_empty[a]), kGroupEpi * CG);
    }
    mbar_init(smem_u32(&bars->drain), 1);
    if (SPLIT) {
      mbar_init(smem_u32(&bars->red_full), ks * 2 * max(4 / ks, 1));  // two warps of each quarter of the lanes in a share
      mbar_init(smem_u32(&bars->red_empty), ks * kGroupEpi);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmB16);
    prefetch_tmap(&tmBw);
    if (MODE == kMx && CG == 2) {
      prefetch_tmap(&tmSA);
      prefetch_tmap(&tmSB);
    }
  }
  if (warp == 1) tmem_alloc_cg<CG>(smem_u32(&bars->tmem_base), static_cast<uint32_t>(p.tmem_cols));
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || SPLIT) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  griddep_wait();  // (the offsets too may come from the kernel before)
  griddep_launch_dependents();
  const int total = group_list<MODE, CG>(p, groups, &bars->total);
  const int first_tile = blockIdx.x / (CG * ks);
  const int tile_step = gridDim.x / (CG * ks);

  // the i-th tile of this CTA (pair, cluster)
  auto take = [&](int& at, int i, GroupTile& tl) {
    if (!group_tile<MODE, CG>(p, groups, at, first_tile + i * tile_step, total, tl)) return false;
    tl.kb0 = SPLIT ? ks_rank * tl.blocks / ks : 0;
    tl.kb1 = SPLIT ? (ks_rank + 1) * tl.blocks / ks : tl.blocks;
    return true;
  };

  // B rows (K-major) or columns (MN-major) of a tile that this CTA stages, and how they are fetched: boxes
  // of 16 rows for narrow tiles, one box of the widest tile where that reads at most a third too much (a
  // load costs its issuing thread 85 cycles: with boxes of 64 throughout, that thread bounded the 4-bit
  // product of 192-row tiles), of 64 otherwise
  auto b_boxes = [&](int nmma, int& box) {
    const int mine = nmma / CG;
    const int cap = p.BN / CG;  // rows that a stage has room for
    if (B_MN) box = 64;
    else box = mine <= 48 ? 16 : (4 * mine >= 3 * cap || round_up(mine, 64) > cap ? cap : 64);
    return (mine + box - 1) / box;
  };
  auto sf_b_rows = [&](const GroupTile& tl) { return ((tl.c0 & 127) + tl.nmma + 127) >> 7; };

  // part bit 0: A (and the barrier's byte count); bit 1: B; bit 2: kMx's scales
  auto produce = [&](int part) {
    int stage = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    int at = 0;
    GroupTile tl;
    const int kt = MODE == kMx ? (p.R + 127) / 128 : 0;  // scale tiles along the reduction
    for (int i = 0; ok && !p.silent_producer && take(at, i, tl); ++i) {
      int box;
      const int boxes = b_boxes(tl.nmma, box);
      const uint32_t tx_ab = static_cast<uint32_t>(a_bytes + boxes * box * kSpan) * CG;
      const int nb_sf = MODE == kMx ? sf_b_rows(tl) : 0;
      const int m0 = tl.m0 + static_cast<int>(cta_rank) * kTileM;
      const int mine0 = tl.c0 + static_cast<int>(cta_rank) * (tl.nmma / CG);  // first B row / column
      // tile rows of the scales
      const int sf_row_a = tl.e * ((p.M + 127) / 128) + m0 / 128;
      const int sf_row_b = tl.start / 128 + tl.e + tl.c0 / 128;
      for (int kb = tl.kb0; kb < tl.kb1; ++kb) {
        const uint32_t full_local = smem_u32(&bars->full[stage]);
        const uint32_t full = (CG == 2) ? mapa(full_local, 0) : full_local;
        if (!mbar_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, wctx)) {
          ok = false;
          break;
        }
        // (an untiled copy completes in its own CTA: the pair's scales come by tensor map, whole boxes)
        const uint32_t sf_tile = MODE == kMx && CG == 1 ? min(2, kt - 2 * kb) * kAtomBytes : 0;
        const uint32_t sf_tx = MODE != kMx ? 0 : (CG == 1 ? (1 + nb_sf) * sf_tile : (1 + sf_rows) * 4 * kAtomBytes);
        if (leader && (part & 1)) mbar_arrive_expect_tx(full_local, tx_ab + sf_tx);
        const uint32_t dA = sA + stage * a_bytes, dB = sB + stage * b_bytes, dSF = sSF + stage * sf_bytes;
        // first index of this block on the reduction axis (in bytes of packed codes for kMx)
        const int red = MODE == kMx ? kb * kSpan : kb * kElems;
        if (part & 1) {
          if (MODE == kFwd || MODE == kMx) {
            tma_load_3d_cg<CG>(dA, &tmA, full, red, m0, tl.e);
          } else {
            const int row = MODE == kDw ? tl.start + red : red;
            const int z = MODE == kDw ? 0 : tl.e;
            tma_load_3d_cg<CG>(dA, &tmA, full, m0, row, z);
            tma_load_3d_cg<CG>(dA + a_bytes / 2, &tmA, full, m0 + 64, row, z);
          }
        }
        if (part & 2) {
          if (B_MN) {
            for (int b = 0; b < boxes; ++b)
              tma_load_3d_cg<CG>(dB + b * 64 * kSpan, &tmB, full, mine0 + b * 64, tl.start + red, 0);
          } else if (boxes == 1 && box > 64) {
            tma_load_3d_cg<CG>(dB, &tmBw, full, red, tl.start + mine0, 0);
          } else if (box == 16) {
            for (int b = 0; b < boxes; ++b)
              tma_load_3d_cg<CG>(dB + b * 16 * kSpan, &tmB16, full, red, tl.start + mine0 + b * 16, 0);
          } else {
            for (int b = 0; b < boxes; ++b)
              tma_load_3d_cg<CG>(dB + b * 64 * kSpan, &tmB, full, red, tl.start + mine0 + b * 64, 0);
          }
        }
        if (MODE == kMx && (part & 4)) {
          if (CG == 1) {
            bulk_load(dSF, p.sfa + (static_cast<long long>(sf_row_a) * kt + 2 * kb) * kAtomBytes, sf_tile, full);
            for (int b = 0; b < nb_sf; ++b)
              bulk_load(dSF + (1 + b) * 2 * kAtomBytes,
                        p.sfb + (static_cast<long long>(sf_row_b + b) * kt + 2 * kb) * kAtomBytes, sf_tile, full);
          } else {
            tma_load_3d_cg<CG>(dSF, &tmSA, full, kb * 256, sf_row_a, 0);
            tma_load_3d_cg<CG>(dSF + 2 * kAtomBytes, &tmSB, full, kb * 256, sf_row_b, 0);
          }
        }
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {  // wait (bounded) for the copies in flight; see hb_umma_kernel
      if (leader) {
        const int pending = issued < p.stages ? static_cast<int>(issued) : p.stages;
        for (int i = 0; i < pending; ++i) {
          if (--stage < 0) {
            stage = p.stages - 1;
            phase ^= 1u;
          }
          mbar_wait_drain(smem_u32(&bars->full[stage]), phase);
        }
      } else {
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) {
        }
      }
    }
  };

  // The MMA role, one elected lane.
  auto multiply = [&]() {
    int stage = 0;
    uint32_t phase = 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    uint32_t edges = 0;  // kDw: parity of each stage's next wait for its edge's zeros
    constexpr uint32_t layout_type = 2u;  // 128-byte swizzle
    constexpr uint64_t desc_hi = static_cast<uint64_t>(((8u * kSpan) >> 4) | (1u << 14) | (layout_type << 29)) << 32;
    // MN-major: 64 x 64 chunks of 8 KB, 16 reduction rows (2 KB) per MMA; K-major: 32 bytes per MMA
    constexpr uint32_t chunk16 = 64u * kSpan >> 4;
    constexpr uint32_t a_lo_fixed = (A_MN ? chunk16 : 1u) << 16, b_lo_fixed = (B_MN ? chunk16 : 1u) << 16;
    constexpr uint32_t a_step = A_MN ? 16u * kSpan >> 4 : 2u, b_step = B_MN ? 16u * kSpan >> 4 : 2u;
    const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
    const uint32_t edge0 = smem_u32(&bars->edge[0]);
    const uint32_t sf_cols = static_cast<uint32_t>(8 * (1 + sf_rows));  // TMEM columns of a stage's scales
    const uint32_t sf_tmem = tmem_base + static_cast<uint32_t>(p.acc_stages * p.BN);
    int at = 0;
    GroupTile tl;
    for (int i = 0; ok && take(at, i, tl); ++i) {
      if ((MODE == kDw || SPLIT) && tl.kb0 == tl.kb1) continue;  // (the epilogue writes zeros without an accumulator)
      ok = mbar_wait(smem_u32(&bars->tmem_empty[acc]), acc_phase ^ 1u, wctx);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * p.BN);
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(tl.nmma >> 3) << 17);
      uint32_t accum = 0u;
      const int nb_sf = MODE == kMx ? sf_b_rows(tl) : 0;
      for (int kb = tl.kb0; kb < tl.kb1; ++kb) {
        ok = mbar_wait(full0 + 8u * stage, phase, wctx);
        if (!ok) break;
        tc_fence_after();
        const uint32_t stA = sA + stage * a_bytes, stB = sB + stage * b_bytes;
        // MMAs of this stage: 16 (kMx: 64) reduction elements each
        int steps = 4;
        if (MODE == kMx) steps = min(4, (p.R - kb * kElems + 63) / 64);
        if (MODE == kDw) {
          const int valid = tl.n - kb * 64;
          if (valid < 64) {
            steps = (valid + 15) / 16;
            if (valid & 15) {  // (the rows behind the group's last one are zero when this barrier says so)
              if (!mbar_wait(edge0 + 8u * stage, (edges >> stage) & 1u, wctx)) {
                ok = false;
                break;
              }
              edges ^= 1u << stage;
            }
          }
        }
        {
          const uint32_t a_lo = ((stA >> 4) & 0x3FFFu) | a_lo_fixed, b_lo = ((stB >> 4) & 0x3FFFu) | b_lo_fixed;
          uint32_t ta = 0, tb = 0;
          if constexpr (MODE == kMx) {
            // Scales into TMEM, in order before the MMAs of this thread.  A stage has its own columns: they
            // are written again only after the MMAs that read them have freed the stage.  Columns: A's two
            // tiles of 128 elements, then per tile of 128 elements B's tile rows side by side (column j
            // holds rows 32 j ...).  (Copied by another thread, with a barrier between, a stage waits for
            // the copies' completion: 4096^3 took 43.7 us so and 39.4 this way, when it was tried.)
            ta = sf_tmem + stage * sf_cols;
            tb = ta + 8u;
            const uint32_t sf = sSF + stage * sf_bytes;
#pragma unroll
            for (int ka = 0; ka < 2; ++ka) {
              if (2 * ka < steps) {
                tmem_cp_scales<CG>(ta + 4u * ka, sf + ka * kAtomBytes);
                tmem_cp_scales<CG>(tb + static_cast<uint32_t>(4 * ka * sf_rows), sf + (2 + ka) * kAtomBytes);
                if (nb_sf > 1)
                  tmem_cp_scales<CG>(tb + static_cast<uint32_t>(4 * ka * sf_rows + 4), sf + (4 + ka) * kAtomBytes);
              }
            }
            tb += static_cast<uint32_t>((tl.c0 & 127) >> 5);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k < steps) {
              const uint64_t ad = desc_hi | (a_lo + a_step * k), bd = desc_hi | (b_lo + b_step * k);
              if constexpr (MODE == kMx)
                umma_mxf4<CG>(d_tmem, ad, bd, idesc | (k & 1 ? (2u << 4) | (2u << 29) : 0u), ta + 4u * (k >> 1),
                          tb + static_cast<uint32_t>(4 * sf_rows * (k >> 1)), accum);
              else
                umma_cg<CG, 0>(d_tmem, ad, bd, idesc, accum);
              accum = 1u;
            }
          }
          umma_commit_cg<CG>(empty0 + 8u * stage);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      umma_commit_cg<CG>(smem_u32(&bars->tmem_full[acc]));
      if (++acc == p.acc_stages) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (!ok) {
      umma_commit_local<CG>(smem_u32(&bars->drain));
      mbar_wait_drain(smem_u32(&bars->drain), 0u);
    }
  };

  // kDw: the rows behind a group's last one in its last block, up to the next multiple of 16, set to zero in
  // both operands as soon as the block has landed.  A warp of its own: done by the MMA warp it held up
  // every tile by some 2500 cycles.
  auto clear_edges = [&]() {
    int stage = 0, at = 0;
    uint32_t phase = 0;
    GroupTile tl;
    for (int i = 0; take(at, i, tl); ++i) {
      const int valid = tl.n & 15 ? tl.n & 63 : 64;
      for (int kb = tl.kb0; kb < tl.kb1; ++kb) {
        // (lanes may disagree only once a wait has run out)
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->full[stage]), phase, wctx))) return;
        if (kb + 1 == tl.blocks && valid < 64) {
          const int vecs = (16 - (valid & 15)) * 8;  // 16-byte vectors of a 64-column chunk
          const int chunks = 2 + (tl.nmma + 63) / 64;
          for (int c = 0; c < chunks; ++c) {
            const uint32_t base = (c < 2 ? sA + stage * a_bytes + c * 64 * kSpan : sB + stage * b_bytes + (c - 2) * 64 * kSpan) +
                                  valid * kSpan;
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (lane + 32 * v < vecs)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + (lane + 32 * v) * 16), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars->edge[stage]));
        }
        // (a stage is refilled only when this warp has passed it too: its waits never fall a turn behind)
        if (lane == 0) mbar_arrive(smem_u32(&bars->empty[stage]));
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  };

  if (warp == 0) {
    if (elect_one()) produce(1);
    __syncwarp();
  } else if (warp == 1) {
    if (leader && elect_one()) multiply();
    __syncwarp();
  } else if (warp == 2 + kGroupEpi) {
    if (elect_one()) produce(2);
    __syncwarp();
  } else if (MODE == kDw && warp == 3 + kGroupEpi) {
    clear_edges();
    __syncwarp();
  } else if (MODE == kMx && warp == 3 + kGroupEpi) {
    if (elect_one()) produce(4);
    __syncwarp();
  } else {
    // this warp's quarter of the TMEM lanes; of two warps of a quarter each takes every second chunk of 32 columns
    constexpr int kStride = NARROW ? 32 : 64, kChunks = NARROW ? 2 : 4, kAtOnce = NARROW ? 1 : 2;
    const int q = warp & 3;
    const int half = NARROW ? 0 : warp >= 6;
    const uint32_t stage_base = sEpi + (warp - 2) * kGroupStage;
    // gives an accumulator back to the MMA warp
    auto hand_back = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2)
          mbar_arrive_cluster(mapa(smem_u32(&bars->tmem_empty[acc]), 0));
        else
          mbar_arrive(smem_u32(&bars->tmem_empty[acc]));
      }
    };
    int acc = 0;
    uint32_t acc_phase = 0;
    int at = 0;
    GroupTile tl;
    uint32_t red_phase = 0;
    for (int i = 0; take(at, i, tl); ++i) {
      const bool empty = (MODE == kDw || SPLIT) && tl.kb0 == tl.kb1;
      const int m = tl.m0 + static_cast<int>(cta_rank) * kTileM + q * 32 + lane;
      const bool mine = m < p.M;
      const long long row0 = MODE == kDw ? tl.c0 : static_cast<long long>(tl.start) + tl.c0;
      const long long first = (MODE == kDw ? tl.e * p.out_group : 0) + row0 * p.ldc + m;
      if (!empty) {
        // (a whole reduction's wait, its bound by the blocks: 2^24 of them, the most there are, take 4.3 s, and what goes
        // wrong in one ends at the ring's waits)
        const WaitCtx whole{abort_flag, wctx.limit_cycles + (tl.kb1 - tl.kb0) * 8192LL};
        if (!mbar_wait_relaxed(smem_u32(&bars->tmem_full[acc]), acc_phase, whole)) break;
        tc_fence_after();
      }
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * p.BN);
      if constexpr (SPLIT) {
        // Every CTA of the cluster has the sums over its share of the reduction.  CTA j joins lanes
        // [j L, (j + 1) L), L = 128 / ks: the others write theirs into its buffer, it adds them in the order
        // of the shares and stores the result.
        const int share = kTileM / ks;
        uint32_t v[32];
        if (empty) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        } else {
          tmem_ld_32x32(t_addr + half * 32, v);
          tmem_ld_wait();
          hand_back(acc);
          if (++acc == p.acc_stages) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
        // (the buffers are free again once every share of the tile before has been read)
        if (!mbar_wait_cluster(smem_u32(&bars->red_empty), red_phase ^ 1u, wctx)) break;
        const int at_lane = q * 32 + lane, owner = at_lane / share;
        const uint32_t dst = mapa(smem_u32(red), owner) +
                             ((ks_rank * 64 + half * 32) * share + at_lane - owner * share) * 4;
        const int mine_cols = min(tl.ncols - half * 32, 32);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < mine_cols) st_cluster_u32(dst + j * share * 4, v[j]);
        __syncwarp();
        const int first_owner = q * 32 / share, last_owner = (q * 32 + 31) / share;
        if (lane <= last_owner - first_owner)
          mbar_arrive_cluster(mapa(smem_u32(&bars->red_full), first_owner + lane));
        if (!mbar_wait_cluster(smem_u32(&bars->red_full), red_phase, wctx)) break;
        const int m0 = tl.m0 + ks_rank * share;
        for (int u = threadIdx.x - 64; u < share * tl.ncols; u += kGroupEpi * 32) {
          const int col = u / share, l = u - col * share;
          float sum = 0.f;
          for (int k = 0; k < ks; ++k) sum += red[(k * 64 + col) * share + l];
          if (m0 + l < p.M) {
            const long long o = (static_cast<long long>(tl.start) + tl.c0 + col) * p.ldc + m0 + l;
            if (p.out_type == 0)
              static_cast<float*>(p.out)[o] = sum;
            else
              static_cast<uint16_t*>(p.out)[o] = static_cast<uint16_t>(pack16(p.out_type, __float_as_uint(sum), 0u));
          }
        }
        __syncwarp();
        if (lane < ks) mbar_arrive_cluster(mapa(smem_u32(&bars->red_empty), lane));
        red_phase ^= 1u;
        continue;
      }
      if (half && tl.ncols <= 32) {  // nothing for this warp
        if (!empty) {
          hand_back(acc);
          if (++acc == p.acc_stages) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
        continue;
      }
      if (!empty && tl.ncols <= 8) {
        // few rows: the wide path's code would be fetched for eight columns (1.1 us a call of one token)
        uint32_t v[8];
        tmem_ld_32x8(t_addr, v);
        tmem_ld_wait();
        hand_back(acc);
        if (mine) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < tl.ncols) {
              if (p.out_type == 0)
                static_cast<uint32_t*>(p.out)[first + j * p.ldc] = v[j];
              else
                static_cast<uint16_t*>(p.out)[first + j * p.ldc] = static_cast<uint16_t>(pack16(p.out_type, v[j], 0u));
            }
        }
        if (++acc == p.acc_stages) {
          acc = 0;
          acc_phase ^= 1u;
        }
        continue;
      }
      // this warp's chunks of 32 columns start at half * 32 + kStride i, i < kChunks
      // (the row pitch is opaque here: its multiples, computed once for all tiles, would take 64 registers
      // and spill)
      long long ldc = p.ldc;
      asm volatile("" : "+l"(ldc));
      if (p.out_type == 0) {
        for (int c = half * 32; c < tl.ncols; c += kStride) {
          uint32_t v[32];
          if (empty) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          } else {
            tmem_ld_32x32(t_addr + c, v);
            tmem_ld_wait();
            if (c + kStride >= tl.ncols) hand_back(acc);  // last read of this accumulator
          }
          if (mine) {
            uint32_t* out = static_cast<uint32_t*>(p.out) + first + c * ldc;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < tl.ncols - c) out[j * ldc] = v[j];
          }
        }
      } else {
        // All of them to registers, rounded and in pairs (columns 2 j and 2 j + 1 of a chunk in word j), and the
        // accumulator back, before anything is stored: a tile of 256 columns has no second accumulator beside
        // the scales, and the MMA warp would wait for the stores (4096^3 in 4 bits 37.8 us, 34.6 so, in short loops).
        uint32_t h[kChunks][16];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const int c = half * 32 + kStride * i;
          if (c >= tl.ncols) break;
          uint32_t v[32];
          if (empty) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          } else {
            tmem_ld_32x32(t_addr + c, v);
            tmem_ld_wait();
          }
          if (p.out_type == 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) h[i][j] = pack16(1, v[2 * j], v[2 * j + 1]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) h[i][j] = pack16(2, v[2 * j], v[2 * j + 1]);
          }
        }
        if (!empty) hand_back(acc);
        // Through shared memory to 16-byte stores, kAtOnce chunks at a time: a chunk as 32 rows (columns) of 64
        // bytes, 16-byte pieces xor-swizzled by row pair.  Neighbouring lanes exchange halves first, so that
        // a lane stores the values of two features of one column (even lanes the even column): 128 bytes a
        // store without a bank conflict.  The MMA's operands come through the same shared memory.  (Two-byte
        // stores to shared memory took 39.4 us, this 37.3, two-byte stores to memory 45, when they were tried.)
        const uint32_t pick = lane & 1 ? 0x3276u : 0x5410u;
        const uint32_t pair_base = stage_base + (lane & 1) * 64 + ((lane >> 1) & 3) * 4;
        const int piece = lane & 3;
        const int mp = m - lane + piece * 8;  // (the extent is a multiple of 8: all of a piece or none)
#pragma unroll
        for (int i = 0; i < kChunks; i += kAtOnce) {
          const int c = half * 32 + kStride * i;
          if (c >= tl.ncols) break;
#pragma unroll
          for (int b = 0; b < kAtOnce; ++b) {
            if (b == 1 && c + kStride >= tl.ncols) break;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, h[i + b][j], 1);
              const uint32_t a = pair_base + b * 2048 + j * 128 + (((lane >> 3) ^ (j & 3)) << 4);
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(__byte_perm(h[i + b][j], other, pick)) : "memory");
            }
          }
          __syncwarp();
          if (p.wide_rows) {
            uint4 d[4 * kAtOnce];
#pragma unroll
            for (int u = 0; u < 4 * kAtOnce; ++u) {
              const int row = (u & 3) * 8 + (lane >> 2);
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(d[u].x), "=r"(d[u].y), "=r"(d[u].z), "=r"(d[u].w)
                           : "r"(stage_base + (u >> 2) * 2048 + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4))
                           : "memory");
            }
            if (mp < p.M) {
              uint16_t* out = static_cast<uint16_t*>(p.out) + first - lane + piece * 8 + (c + (lane >> 2)) * ldc;
              const int left = tl.ncols - c - (lane >> 2);
#pragma unroll
              for (int u = 0; u < 4 * kAtOnce; ++u) {
                const int row = (u >> 2) * kStride + (u & 3) * 8;
                if (row < left) *reinterpret_cast<uint4*>(out + row * ldc) = d[u];
              }
            }
          } else {
            // rows of any length and alignment: a value a lane.  (Rolled: 32 stores a chunk written out, straight
            // from the registers, cost 1003 rows of 1001 features 4250 cycles a tile, mostly instruction fetch.)
            for (int b = 0; b < kAtOnce; ++b) {
              const int rows = min(tl.ncols - c - kStride * b, 32);
              uint16_t* out = static_cast<uint16_t*>(p.out) + first + (c + kStride * b) * ldc;
#pragma unroll 4
              for (int row = 0; row < rows; ++row, out += ldc) {
                uint16_t d;
                asm volatile("ld.shared.u16 %0, [%1];"
                             : "=h"(d)
                             : "r"(stage_base + b * 2048 + row * 64 + (((lane >> 3) ^ ((row >> 1) & 3)) << 4) + (lane & 7) * 2)
                             : "memory");
                if (mine) *out = d;
              }
            }
          }
          __syncwarp();
        }
      }
      if (!empty && ++acc == p.acc_stages) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (CG == 2 || SPLIT) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_cg<CG>(tmem_base, static_cast<uint32_t>(p.tmem_cols));
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_hb_status, kErrTimeout);
}

}  // namespace hb
