// Plans for the products grouped by expert and the 4-bit products (hb_group.cuh), and the launches of
// the quantisation kernels (hb_mx.cuh).  Times at the rules are of loops of some 10 ms where nothing else is said.
#pragma once
#include "hb_plan.cuh"

namespace {

int out_type_of(hb_dtype t) { return t == HB_F32 ? 0 : (t == HB_F16 ? 1 : (t == HB_BF16 ? 2 : -1)); }

struct GroupProblem {
  int mode;  // hb::kFwd ...
  int T, E;  // rows of the token matrix, groups
  int M, C, R;  // see hb::GroupParams
  hb_dtype in, out;  // in: unused for kMx
};

// (split: the buffer in which the CTAs of a cluster join their sums, 128 lanes x 64 columns)
int group_fixed_smem(int E, bool split = false, bool narrow = false) {
  return (split ? hb::kTileM * 64 * 4 : 0) + 1024 /*alignment of the ring*/ +
         hb::group_epi(narrow) * hb::group_staging(narrow) + static_cast<int>((sizeof(hb::GroupBars) + 15) & ~15) +
         E * static_cast<int>(sizeof(hb::GroupEntry));
}

// Most tiles that the offsets can ask for.
long long most_tiles(const GroupProblem& g, const hb_knobs& k) {
  const int rows_m = hb::kTileM * k.cta_group;
  const long long ct = g.mode == hb::kDw ? static_cast<long long>(g.E) * ((g.C + k.tile_n - 1) / k.tile_n)
                                         : (g.T < g.T / k.tile_n + g.E ? g.T : g.T / k.tile_n + g.E);
  return ct * ((g.M + rows_m - 1) / rows_m);
}

int group_stage(const GroupProblem& g, int BN, int cg) {
  if (g.mode == hb::kMx) return cg == 2 ? hb::group_stage_bytes<hb::kMx, 2>(BN) : hb::group_stage_bytes<hb::kMx, 1>(BN);
  return cg == 2 ? hb::group_stage_bytes<hb::kFwd, 2>(BN) : hb::group_stage_bytes<hb::kFwd, 1>(BN);
}

int group_tmem(const GroupProblem& g, const hb_knobs& k) {
  int c = k.acc_stages * k.tile_n;
  if (g.mode == hb::kMx) c += k.stages * 8 * (1 + hb::group_sf_rows(k.tile_n));
  return c;
}

// The narrow form, two CTAs to an SM (tiles of 64 columns, four epilogue warps, rings half as deep): one's
// set-up, epilogue and issuing pass under the other's loads, and twice as many tiles find a place at once.
// Measured, wide / narrow: MXFP4 16 rows over 32 experts of 2048 x 2048 10.8 / 8.5 us, 256 rows 19.0 / 16.1, 1024 rows over
// 128 of 1024 x 2048 31.7 / 29.1; fp16 1003 rows over 24 experts of 1001 x 712 13.0 / 12.1, bf16 256 rows over 32 of
// 2048 x 2048 45.0 / 43.7.  16-bit operands lose where all tiles find an SM of their own (256 rows over 8 experts 15.2 / 16.5,
// unless the reduction is short: dx with 328 features 6.1 / 5.8) and where there are many rounds (1024 rows over 128
// experts 82.4 / 83.8): the deeper ring is worth more there.
constexpr int kNarrowSmem = (233472 - 2 * 1024) / 2;  // an SM's shared memory less what the system keeps of a CTA's
bool is_narrow(const GroupProblem& g, const hb_knobs& k, int sms) {
  if (g.mode == hb::kDw || k.tile_n != 64 || k.cta_group != 1 || k.split_k != 1 || k.max_ctas != 0) return false;
  const int elems = g.mode == hb::kMx ? 256 : 64;
  // (tiles to expect: a row in every group, or as many groups as rows)
  const long long tiles = static_cast<long long>(g.T < g.E ? g.T : g.E) * ((g.M + hb::kTileM - 1) / hb::kTileM);
  if (tiles <= sms && (g.R + elems - 1) / elems > 8) return false;
  if (g.mode != hb::kMx && tiles > 6LL * sms) return false;
  return group_fixed_smem(g.E, false, true) + (k.stages > 0 ? k.stages : 2) * group_stage(g, 64, 1) <= kNarrowSmem;
}

void group_knobs(const GroupProblem& g, const hb_knobs* in, int sms, hb_knobs* out) {
  hb_knobs k;
  if (in) k = *in; else std::memset(&k, 0, sizeof(k));
  const int avg = g.T / g.E;  // mean rows of a group
  // CTA pairs: half of B to each CTA.  Measured, single CTAs against pairs, both with their best tile, in a loop
  // of half a second: 8192 rows, 32 groups of 2048 x 2048 bf16 94 / 84 us; dx of 16 groups of 512 rows 47.7 / 42.1;
  // MXFP4 4096^3 43.7 / 39.5, 187 rows a group 31.8 / 29.8.  dw by pairs (its edge rows cleared in both CTAs)
  // was level, 49.4 / 49.2, and is not built.
  if (k.cta_group == 0)
    k.cta_group = (g.mode != hb::kDw && avg >= (g.mode == hb::kMx ? 128 : 256) && g.M >= 256 && (k.tile_n == 0 || k.tile_n >= 128)) ? 2 : 1;
  if (k.tile_n == 0) {
    if (g.mode == hb::kDw)
      // (up to 64 rows a group a tile is one block and its time the epilogue's, which narrower tiles spread
      // better: 777 rows, 20 groups of 328 x 520 8.9 us with 128 columns, 9.7 with 256; 512 rows a group 57 / 48)
      k.tile_n = g.C > 128 && avg > 64 ? 256 : (g.C > 64 ? 128 : 64);
    else if (g.mode == hb::kMx)
      // (two accumulators and the scales fit TMEM beside 192 columns; pairs take 256 and one accumulator: 4096^3
      // 37.5 us with 192, 34.6 with 256; single CTAs 37.3 with 192, 46 with 128)
      k.tile_n = k.cta_group == 2 ? 256 : (avg > 128 ? 192 : (avg > 48 ? 128 : 64));
    else
      k.tile_n = k.cta_group == 2 || avg > 96 ? 256 : (avg > 48 ? 128 : 64);
  }
  if (k.split_k == 0) {
    // A product of few tiles: the reduction of a tile over a cluster of 2 or 4 CTAs, as long as all of them
    // find an SM.  A tile's time is that of its operands through one SM's ring; the cluster costs about 2 us.
    // Measured, one / two / four CTAs a tile, 32 rows x 4096 features in one group: bf16, K 4096 18.8 / 15.2 / 12.6 us;
    // MXFP4, K 8192 14.3 / 13.4 / 11.4, K 4096 (16 blocks) 8.9 / 10.0 / 9.0.  (Clusters of eight: 128 CTAs did not all run
    // at once, 12.3 us where four took 7.8.)  49 to 64 rows take tiles of 128 columns and no cluster, 18.0 us for 64 rows
    // bf16, K 4096, although 64 columns and four CTAs take 14.7: most_tiles has to hold for all offsets and counts two
    // tiles there.
    k.split_k = 1;
    if ((g.mode == hb::kFwd || g.mode == hb::kMx) && k.cta_group == 1 && k.tile_n == 64) {
      const int elems = g.mode == hb::kMx ? 256 : 64;
      const int most = k.max_ctas > 0 && k.max_ctas < sms ? k.max_ctas : sms;
      if ((g.R + elems - 1) / elems >= 32)
        while (k.split_k < 4 && most_tiles(g, k) * k.split_k * 2 <= most) k.split_k *= 2;
    }
  }
  const bool narrow = is_narrow(g, k, sms);
  const int room = (narrow ? kNarrowSmem : kSmemLimit) - group_fixed_smem(g.E, k.split_k > 1, narrow);
  if (k.stages == 0) {
    k.stages = room / group_stage(g, k.tile_n, k.cta_group);
    // (kMx: TMEM columns of the scales beside two accumulators, or one where two leave none)
    const int sf = 8 * (1 + hb::group_sf_rows(k.tile_n));
    const int most = g.mode == hb::kMx ? (512 - (2 * k.tile_n + 2 * sf <= 512 ? 2 : 1) * k.tile_n) / sf : hb::kMaxStages;
    if (k.stages > most) k.stages = most;
    if (k.stages > hb::kMaxStages) k.stages = hb::kMaxStages;
    if (k.stages < 1) k.stages = 1;
  }
  if (k.acc_stages == 0) {
    k.acc_stages = 2;
    if (group_tmem(g, k) > 512) k.acc_stages = 1;
  }
  *out = k;
}

// What the caller gave, before defaults are worked out from it (sizes of a ring stage are divided by).
bool group_knobs_in_range(const hb_knobs& k) {
  return k.tile_n >= 0 && k.tile_n <= 256 && k.tile_n % 64 == 0 && k.cta_group >= 0 && k.cta_group <= 2 && k.split_k >= 0 &&
         k.split_k <= 8 && k.stages >= 0 && k.stages <= hb::kMaxStages && k.acc_stages >= 0 && k.acc_stages <= 2 &&
         k.max_ctas >= 0;
}

int check_group_knobs(const GroupProblem& g, const hb_knobs& k) {
  if (k.cta_group != 1 && k.cta_group != 2) return HB_ERR_KNOB;
  if (k.cta_group == 2 && g.mode == hb::kDw) return HB_ERR_KNOB;
  if (k.tile_n < 64 * k.cta_group || k.tile_n > 256 || k.tile_n % 64 != 0) return HB_ERR_KNOB;
  if (k.stages < 1 || k.stages > hb::kMaxStages) return HB_ERR_KNOB;
  if (k.acc_stages < 1 || k.acc_stages > 2) return HB_ERR_KNOB;
  if (k.max_ctas < 0) return HB_ERR_KNOB;
  if (group_tmem(g, k) > 512) return HB_ERR_KNOB;
  if (k.split_k != 1 && k.split_k != 2 && k.split_k != 4 && k.split_k != 8) return HB_ERR_KNOB;
  if (k.split_k > 1 && (k.cta_group != 1 || k.tile_n != 64 || (g.mode != hb::kFwd && g.mode != hb::kMx))) return HB_ERR_KNOB;
  if (group_fixed_smem(g.E, k.split_k > 1) + k.stages * group_stage(g, k.tile_n, k.cta_group) > kSmemLimit) return HB_ERR_KNOB;
  return HB_OK;
}

// Whether a product is left to the kernels that stream the weights (hb_rows.cuh): by the weights that all their passes
// read (one pass for eight rows of a group, so one for up to eight rows of a single group, and at worst one for every row
// where there are more groups), and by the blocks that a launch has, T * N / 16, of which those without rows leave at
// once: with short reductions the blocks' start is the time.  Measured, streaming / tiles of 64 columns (with a cluster or
// two CTAs to an SM where those are chosen), us, rows x features x reduction; more groups: rows spread at random:
//   bf16, one group.  Up to 8 rows of 4096 features: K 64 2.2 - 2.9 / 3.1, K 1024 5.7 / 6.5 - 6.8, K 4096 8.3 - 10.3 / 11.2 -
//   11.5, K 16384 25.4 - 25.9 / 28.0 - 28.5.  64 x 512 x 256 4.5 / 5.8, 16 x 2048 x 2048 6.3 / 7.7.  Between 2^15 and 2^16 rows x
//   features (8 rows at least): K 1024 8 x 8192 7.2 / 7.6, 32 x 2048 6.4 / 7.8, 64 x 1024 6.8 / 7.5; K 512 6.5 / 5.7, 5.8 /
//   5.4 (16 x 4096); K 256 32 x 2048 6.0 / 4.8.  Beyond: 1 x 16384 x 512 10.2 / 6.7, 8 x 65536 x 128 44.7 / 6.8, 64 x 2048 x
//   512 10.4 / 6.8.  More than 8.4 million weights in all passes: 32 x 2048 x 2048 8.5 / 8.2, 24 x 4096 x 2048 11.7 / 9.6
//   bf16, more groups.  K 2048: 2 rows x 2048 3.7 / 7.8, 4 rows 7.8 / 10.7, 8 rows 11.0 - 14.1 / 11.5 - 12.9, 24 rows over 32
//   25.6 / 26.5, 48 over 48 44.2 / 41.5 (the memory's time either way).  Shorter ones: 8 x 1024 x 1024 6.0 / 6.8, 10 x 1024 x
//   1024 6.2 / 7.0, 16 x 512 x 512 5.5 / 5.4, 8 x 2048 x 1024 7.5 - 10.4 / 7.5 - 8.2, 16 x 1024 x 1024 9.2 / 8.1, 32 x 2048 x 256
//   17.6 / 7.4, 64 x 512 x 512 11.4 / 7.7
//   MXFP4, bound by widening elements.  One group: 1 row x 4096 x 512 2.6 / 3.8, x 4096 7.5 / 8.8; x 6144 x 2048 6.6 / 6.2,
//   x 8192 x 1024 5.6 / 5.0, 4 rows 7.0 / 5.0; x 4096 x 8192 12.8 / 10.5; two passes, 16 x 2048 x 1024, 5.5 / 5.0.  More
//   groups: 4 x 1024 x 1024 3.3 / 4.5, 2 x 2048 x 2048 4.4 / 5.8, 4 x 2048 x 1024 5.6 / 5.0, 8 x 1024 x 512 4.3 / 4.2, 16 x 512 x
//   512 4.2 / 4.2, 8 x 2048 x 256 6.7 / 4.1, 64 x 512 x 512 11.5 / 5.7; 4 x 2048 x 2048 7.8 / 6.4
bool few_rows(const GroupProblem& g) {
  if ((g.mode != hb::kFwd && g.mode != hb::kMx) || g.T > 64) return false;
  const long long weights = static_cast<long long>(g.M) * g.R, T = g.T;
  if (g.mode == hb::kMx)
    return g.R <= 8192 && (g.E == 1 ? T <= 8 && g.M <= 4096 && weights <= (1LL << 24)
                                    : T * weights <= (1LL << 23) && T * g.M <= 8192);
  if (g.E == 1) {
    const long long outputs = (T < 8 ? 8 : T) * g.M;
    if (outputs > 65536 || (outputs > 32768 && g.R < 1024)) return false;
    return (T <= 8 && outputs <= 32768) || (T + 7) / 8 * weights <= (1LL << 23);
  }
  return T <= (g.E > 8 ? g.E : 8) && (g.R >= 2048 || T * g.M <= 10240);
}

// Knobs of the tile kernel, given by the caller: then that kernel is meant.
bool knob_names_tiles(const hb_knobs& k) {
  return k.tile_n || k.split_k || k.stages || k.acc_stages || k.max_ctas || k.cta_group || k.silent_producer;
}

// Scale tiles (512 bytes, kt to a tile row) as rows of words: boxes of two tiles and `rows` tile rows, dense in
// shared memory.
int encode_scales(Driver& d, CUtensorMap* m, const void* ptr, uint64_t kt, uint64_t tile_rows, uint32_t rows) {
  cuuint64_t dims[3] = {kt * 128, tile_rows, 1};
  cuuint64_t strides[2] = {kt * hb::kAtomBytes, kt * hb::kAtomBytes * tile_rows};
  cuuint32_t box[3] = {256, rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = d.tiled(m, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? HB_OK : HB_ERR_LAUNCH;
}

// A: w (kFwd, kDx, kMx) or x (kDw); B: the token matrix (kDw: dy).
int plan_group(const GroupProblem& g, const void* A, const void* B, void* out, const void* sfa, const void* sfb,
               const int* offsets, const hb_knobs* knobs, hb_plan* plan) {
  std::memset(plan, 0, sizeof(*plan));
  plan->group = true;
  plan->group_mode = g.mode;
  const int eo = esize(g.out);
  const bool dw = g.mode == hb::kDw, mx = g.mode == hb::kMx;
  if (g.T == 0) {  // no rows: nothing to compute, and the gradient of every weight is zero
    if (!dw) return HB_OK;
    if (!out || !aligned16(out)) return HB_ERR_ALIGN;
    Driver& d0 = driver();
    if (d0.status != HB_OK) return d0.status;
    plan->gp.out = out;
    plan->group_zero_bytes = static_cast<size_t>(g.E) * g.M * g.C * eo;
    return HB_OK;
  }
  if (!A || !B || !out || !aligned16(A) || !aligned16(B) || !aligned16(out)) return HB_ERR_ALIGN;
  if (mx && (!sfa || !sfb || !aligned16(sfa) || !aligned16(sfb))) return HB_ERR_ALIGN;
  if (!offsets && !(mx && g.E == 1)) return HB_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(offsets) & 3u) != 0) return HB_ERR_ALIGN;
  if (knobs && !group_knobs_in_range(*knobs)) return HB_ERR_KNOB;
  Driver& d = driver();
  if (d.status != HB_OK) return d.status;
  hb_knobs k;
  group_knobs(g, knobs, d.sm_count, &k);
  int rc = check_group_knobs(g, k);
  if (rc != HB_OK) return rc;
  if ((!knobs || !knob_names_tiles(*knobs)) && few_rows(g)) {
    hb::RowsParams& r = plan->rp;
    r.w = A; r.x = B; r.out = out; r.offsets = offsets;
    r.w_sf = static_cast<const uint8_t*>(sfa);
    r.x_sf = static_cast<const uint8_t*>(sfb);
    r.E = g.E; r.T = g.T; r.N = g.M; r.K = g.R;
    r.out_type = out_type_of(g.out);
    r.w_matrix_sf = mx ? (g.M + 127LL) / 128 * ((g.R + 127LL) / 128) * hb::kAtomBytes : 0;
    plan->group_rows = true;
    plan->group_mode = mx ? hb::kMx : (g.in == HB_F16 ? 1 : 2);  // (no knobs: they are the tile kernel's)
    // (4-bit: 16 features to a block within a tile of 128)
    plan->grid = mx ? (g.M + 127) / 128 * 8 : (g.M + hb::kRowsFeatures - 1) / hb::kRowsFeatures;
    return HB_OK;
  }

  hb::GroupParams& p = plan->gp;
  p.offsets = offsets;
  p.E = g.E; p.T = g.T; p.M = g.M; p.C = g.C; p.R = g.R;
  p.BN = k.tile_n; p.stages = k.stages; p.acc_stages = k.acc_stages;
  p.tmem_cols = next_pow2_cols(group_tmem(g, k));
  const int rows_m = hb::kTileM * k.cta_group;
  p.tiles_m = (g.M + rows_m - 1) / rows_m;
  p.out = out;
  p.out_type = out_type_of(g.out);
  p.ldc = g.M;
  p.wide_rows = eo == 2 && g.M % 8 == 0;
  p.out_group = static_cast<long long>(g.C) * g.M;
  p.sfa = static_cast<const uint8_t*>(sfa);
  p.sfb = static_cast<const uint8_t*>(sfb);
  p.silent_producer = k.silent_producer ? 1 : 0;
  if (p.silent_producer) p.wait_limit_cycles = 200000000LL;
  // instruction descriptor: M / 16 in bits 24..28, the majors in bits 15 and 16, formats in 7..9 and 10..12
  p.idesc = static_cast<uint32_t>(rows_m >> 4) << 24;
  if (mx) {
    p.idesc |= (1u << 7) | (1u << 10) | (1u << 23);  // E2M1 both, scales E8M0
  } else {
    const uint32_t f = g.in == HB_BF16 ? 1u : 0u;
    p.idesc |= (1u << 4) | (f << 7) | (f << 10);  // fp32 accumulator
    if (g.mode != hb::kFwd) p.idesc |= 1u << 15;
    if (dw) p.idesc |= 1u << 16;
  }
  const long long tiles = most_tiles(g, k);
  if (tiles > 0x3fffffffLL) return HB_ERR_SHAPE;
  const bool narrow = is_narrow(g, k, d.sm_count);
  plan->group_narrow = narrow;
  const int together = k.cta_group * k.split_k;  // CTAs of a cluster
  int units = d.sm_count * (narrow ? 2 : 1) / together;
  if (k.max_ctas > 0 && k.max_ctas / together < units) units = k.max_ctas / together;
  if (units < 1) units = 1;
  plan->grid = static_cast<int>(tiles < units ? tiles : units) * together;
  p.ksplit = k.split_k;
  plan->smem = group_fixed_smem(g.E, k.split_k > 1, narrow) + k.stages * group_stage(g, k.tile_n, k.cta_group);
  // CTA pairs have their SMs for themselves, also with few stages: of two pairs (of calls on two streams) that share SMs
  // each could hold the tensor memory of one SM and wait, without a bound, for that of the other.
  if (k.cta_group == 2 && plan->smem <= kNarrowSmem) plan->smem = kNarrowSmem + 1024;
  plan->knobs = k;

  const uint64_t T = g.T, E = g.E, M = g.M, R = g.R, C = g.C;
  if (mx) {
    const uint64_t row = R / 2;
    rc = encode_tiled3(d, &plan->tmA, HB_U8, A, row, M, E, row, row * M, 128, hb::kTileM, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmB, HB_U8, B, row, T, 1, row, row * T, 128, 64, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmB2, HB_U8, B, row, T, 1, row, row * T, 128, 16, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmC, HB_U8, B, row, T, 1, row, row * T, 128, k.tile_n / k.cta_group, 128);
    if (rc == HB_OK && k.cta_group == 2) {
      const uint64_t kt = (R + 127) / 128;
      rc = encode_scales(d, &plan->tmSA, sfa, kt, E * ((M + 127) / 128), 1);
      const uint64_t rows_b = offsets ? T / 128 + E : (T + 127) / 128;
      if (rc == HB_OK) rc = encode_scales(d, &plan->tmSB, sfb, kt, rows_b, hb::group_sf_rows(k.tile_n));
    }
  } else if (dw) {
    rc = encode_tiled3(d, &plan->tmA, g.in, A, M, T, 1, M * 2, M * 2 * T, 64, 64, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmB, g.in, B, C, T, 1, C * 2, C * 2 * T, 64, 64, 128);
    plan->tmC = plan->tmB2 = plan->tmB;
  } else {
    rc = g.mode == hb::kFwd ? encode_tiled3(d, &plan->tmA, g.in, A, R, M, E, R * 2, R * 2 * M, 64, hb::kTileM, 128)
                            : encode_tiled3(d, &plan->tmA, g.in, A, M, R, E, M * 2, M * 2 * R, 64, 64, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmB, g.in, B, R, T, 1, R * 2, R * 2 * T, 64, 64, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmB2, g.in, B, R, T, 1, R * 2, R * 2 * T, 64, 16, 128);
    if (rc == HB_OK) rc = encode_tiled3(d, &plan->tmC, g.in, B, R, T, 1, R * 2, R * 2 * T, 64, k.tile_n / k.cta_group, 128);
  }
  return rc;
}

// The kernels round sizes up to whole tiles in 32 bits.
constexpr int kMostSize = 1 << 30;
bool sizes_ok(int T, int K, int N, int E) {
  return T >= 0 && T <= kMostSize && K > 0 && K <= kMostSize && N > 0 && N <= kMostSize && E > 0 && E <= hb::kMaxGroups;
}

int plan_grouped(int mode, const void* A, const void* B, void* out, const int* offsets, int T, int K, int N, int E,
                 hb_dtype in, hb_dtype out_t, const hb_knobs* knobs, hb_plan* plan) {
  std::memset(plan, 0, sizeof(*plan));
  if (!sizes_ok(T, K, N, E)) return HB_ERR_SHAPE;
  if ((in != HB_F16 && in != HB_BF16) || out_type_of(out_t) < 0) return HB_ERR_DTYPE;
  // row pitches of the operands are multiples of 16 bytes (the output's need not be)
  if (K % 8 != 0 || (mode != hb::kFwd && N % 8 != 0)) return HB_ERR_SHAPE;
  GroupProblem g;
  g.mode = mode; g.T = T; g.E = E; g.in = in; g.out = out_t;
  g.M = mode == hb::kFwd ? N : K;
  g.C = N;
  g.R = mode == hb::kFwd ? K : N;
  return plan_group(g, A, B, out, nullptr, nullptr, offsets, knobs, plan);
}

int plan_mx(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, const int* offsets,
            int T, int K, int N, int E, hb_dtype out_t, const hb_knobs* knobs, hb_plan* plan) {
  std::memset(plan, 0, sizeof(*plan));
  if (!sizes_ok(T, K, N, E) || K % 32 != 0) return HB_ERR_SHAPE;
  if (out_type_of(out_t) < 0) return HB_ERR_DTYPE;
  GroupProblem g;
  g.mode = hb::kMx; g.T = T; g.E = E; g.in = HB_U8; g.out = out_t;
  g.M = N; g.C = 0; g.R = K;
  return plan_group(g, w, x, out, w_scales, x_scales, offsets, knobs, plan);
}

template <int MODE, int CG, bool SPLIT = false, bool NARROW = false>
int launch_group(const hb_plan* plan, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(plan->grid);
  cfg.blockDim = dim3(hb::group_threads(MODE, NARROW));
  cfg.dynamicSmemBytes = plan->smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLIT ? plan->gp.ksplit : CG; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, hb::hb_group_kernel<MODE, CG, SPLIT, NARROW>, plan->tmA, plan->tmB, plan->tmB2, plan->tmC, plan->tmSA, plan->tmSB, plan->gp);
  return e == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
}

int launch_rows(const hb_plan* plan, cudaStream_t stream) {
  const bool mx = plan->group_mode == hb::kMx;
  const int warps = !mx && plan->rp.K > 2048 ? 16 : hb::kRowsWarps;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(plan->grid, plan->rp.T);
  cfg.blockDim = dim3(warps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  void (*kernel)(const hb::RowsParams) =
      mx ? hb::hb_mx_rows_kernel
         : (plan->group_mode == 1 ? (warps == 16 ? hb::hb_group_rows_kernel<1, 16> : hb::hb_group_rows_kernel<1, 8>)
                                  : (warps == 16 ? hb::hb_group_rows_kernel<2, 16> : hb::hb_group_rows_kernel<2, 8>));
  return cudaLaunchKernelEx(&cfg, kernel, plan->rp) == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
}

int run_group(const hb_plan* plan, cudaStream_t stream) {
  if (plan->group_rows) return launch_rows(plan, stream);
  if (plan->group_zero_bytes)
    return cudaMemsetAsync(plan->gp.out, 0, plan->group_zero_bytes, stream) == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
  if (plan->grid == 0) return HB_OK;  // no rows
  const bool pair = plan->knobs.cta_group == 2;
  if (plan->gp.ksplit > 1)
    return plan->group_mode == hb::kFwd ? launch_group<hb::kFwd, 1, true>(plan, stream)
                                        : launch_group<hb::kMx, 1, true>(plan, stream);
  if (plan->group_narrow) {
    switch (plan->group_mode) {
      case hb::kFwd: return launch_group<hb::kFwd, 1, false, true>(plan, stream);
      case hb::kDx: return launch_group<hb::kDx, 1, false, true>(plan, stream);
      default: return launch_group<hb::kMx, 1, false, true>(plan, stream);
    }
  }
  switch (plan->group_mode) {
    case hb::kFwd: return pair ? launch_group<hb::kFwd, 2>(plan, stream) : launch_group<hb::kFwd, 1>(plan, stream);
    case hb::kDx: return pair ? launch_group<hb::kDx, 2>(plan, stream) : launch_group<hb::kDx, 1>(plan, stream);
    case hb::kDw: return launch_group<hb::kDw, 1>(plan, stream);
    default: return pair ? launch_group<hb::kMx, 2>(plan, stream) : launch_group<hb::kMx, 1>(plan, stream);
  }
}

// ---- MXFP4 quantisation -----------------------------------------------------------------------
size_t mx_scale_bytes(int batch, int rows, int K, int groups) {
  if (batch <= 0 || rows < 0 || K <= 0 || K % 32 != 0 || groups < 0 || groups > hb::kMaxGroups) return 0;
  if (groups > 0 && batch != 1) return 0;
  const long long tile_rows = groups > 0 ? rows / 128 + groups : (rows + 127LL) / 128;
  size_t bytes;  // (one matrix has at most 2^57)
  return __builtin_mul_overflow(static_cast<size_t>(batch), static_cast<size_t>(tile_rows * ((K + 127LL) / 128) * hb::kAtomBytes), &bytes)
             ? 0 : bytes;
}

// Both directions: `values` is the input of the quantisation or the output of the way back.
int run_mx(bool back, const void* values, const void* codes, const void* scales, const int* offsets, int batch,
           int rows, int K, int groups, hb_dtype type, cudaStream_t stream) {
  if (batch <= 0 || rows < 0 || K <= 0 || K % 32 != 0 || groups < 0 || groups > hb::kMaxGroups) return HB_ERR_SHAPE;
  if (groups > 0 && batch != 1) return HB_ERR_SHAPE;
  const int t = out_type_of(type);
  if (t < 0) return HB_ERR_DTYPE;
  if (rows == 0) return HB_OK;
  if (!values || !codes || !scales || !aligned16(values) || !aligned16(codes) || !aligned16(scales)) return HB_ERR_ALIGN;
  if ((groups > 0) != (offsets != nullptr) || (reinterpret_cast<uintptr_t>(offsets) & 3u) != 0) return HB_ERR_ALIGN;
  if (static_cast<long long>(batch) * rows > 0x7fffffffLL) return HB_ERR_SHAPE;
  // 16 blocks of eight rows to a tile row of scales
  const long long row_blocks = 16LL * batch * (groups > 0 ? rows / 128 + groups : (rows + 127LL) / 128);
  const int segments = (K - 1) / hb::kMxSegment + 1;
  if (segments > 65535 || row_blocks > 0x7fffffffLL) return HB_ERR_SHAPE;
  Driver& d = driver();
  if (d.status != HB_OK) return d.status;
  hb::MxParams p;
  std::memset(&p, 0, sizeof(p));
  p.x = values;
  p.out = const_cast<void*>(values);
  p.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  p.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  p.offsets = offsets;
  p.batch = batch; p.rows = rows; p.K = K; p.groups = groups;
  p.matrix_scales = static_cast<long long>(mx_scale_bytes(1, rows, K, groups));
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(row_blocks), segments);
  cfg.blockDim = dim3(hb::kMxThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e;
  if (back)
    e = t == 0 ? cudaLaunchKernelEx(&cfg, hb::hb_dequantize_mxfp4_kernel<0>, p)
               : (t == 1 ? cudaLaunchKernelEx(&cfg, hb::hb_dequantize_mxfp4_kernel<1>, p)
                         : cudaLaunchKernelEx(&cfg, hb::hb_dequantize_mxfp4_kernel<2>, p));
  else
    e = t == 0 ? cudaLaunchKernelEx(&cfg, hb::hb_quantize_mxfp4_kernel<0>, p)
               : (t == 1 ? cudaLaunchKernelEx(&cfg, hb::hb_quantize_mxfp4_kernel<1>, p)
                         : cudaLaunchKernelEx(&cfg, hb::hb_quantize_mxfp4_kernel<2>, p));
  return e == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
}

}  // namespace
