// Products of few rows: grouped_gemm and the 4-bit products where every weight meets only a row or two (a
// decoding step).  Such a product is one pass over the weights, 2 K N bytes an expert (16-bit) or K N (1/2 +
// 1/32) (MXFP4), and the time is the memory's.  The tile kernel (hb_group.cuh) gives a tile of 128 features to
// one SM, which draws at most about 50 bytes a cycle through its ring: with fewer tiles than SMs most of
// the memory's bandwidth is idle (one token, 2048 features x 1024, bf16: 6.4 us by tiles, 3.2 here).  Here a block takes 16
// features and up to eight rows of a group, its eight warps a share of the reduction each: every lane
// loads its operands straight from memory in 16-byte pieces, many in flight before the first is used, and
// the partial sums are joined in shared memory in the order of the warps.
//
// The arithmetic is mma.sync m16n8k16 with the weights as its 16 rows and the tokens as its 8 columns: a
// lane's 16 bytes of a weight row and of a token row are the same stretch of the reduction, and since the
// order of a sum's terms is free, that stretch is what the lane contributes as its "k" indexes of the
// instruction, without any exchange.  (tcgen05 would need the operands in shared memory first.  The tensor
// rate does not matter here: a weight takes part in one such instruction.  With fp32 multiply-adds in
// their place four rows took twice the time of one.)
//
//   block (x, y): 16 features, and row y; the block of a group's rows 8 i, of which it takes up to eight,
//   works, the others leave at once (see rows_taken).  The grid depends on T, not on E or the offsets.
#pragma once
#include "hb_mx.cuh"

namespace hb {

constexpr int kRowsWarps = 8;  // (MXFP4; 16-bit operands: 8 or 16)
constexpr int kRowsFeatures = 16;
constexpr int kRowsAtOnce = 8;

struct RowsParams {
  const void* w;         // (E, N, K) values, or codes (E, N, K / 2)
  const void* x;         // (T, K) values, or codes (T, K / 2)
  const uint8_t* w_sf;   // MXFP4 only
  const uint8_t* x_sf;
  const int* offsets;    // nullptr (MXFP4 only): one group of T rows
  int E, T, N, K;
  int out_type;
  void* out;
  long long w_matrix_sf;  // scale bytes of one expert
};

// The rows r .. r + rows - 1 that the block of row r takes, all of group e (by clamped ranges, the first group
// that claims r); 0 for a block that leaves.  All lanes take part and get the answer.  A block works for a group's
// rows 0, 8, ..., and for a group's row behind one that another group claims first, up to the group's next
// multiple of eight: with offsets out of order, [0, 6, 2, 8], rows 6 and 7 are the third group's alone, whose row 2
// goes to the first.  So every row that some group claims is taken.
__device__ __forceinline__ int rows_taken(const RowsParams& p, int r, int& e, int& start) {
  e = 0;
  start = 0;
  if (!p.offsets) return (r & (kRowsAtOnce - 1)) == 0 ? min(kRowsAtOnce, p.T - r) : 0;
  const int lane = threadIdx.x & 31;
  bool other = false;  // row r - 1 is claimed by a group before this one
  for (int base = 0; base < p.E; base += 32) {
    const int g = base + lane;
    int s = 0, t = 0;
    if (g < p.E) {
      s = min(max(p.offsets[g], 0), p.T);
      t = min(max(p.offsets[g + 1], s), p.T);
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, s <= r && r < t);
    const uint32_t above = __ballot_sync(0xffffffffu, s < r && r <= t);
    if (hit) {
      const int src = __ffs(hit) - 1;
      e = base + src;
      start = __shfl_sync(0xffffffffu, s, src);
      const int end = __shfl_sync(0xffffffffu, t, src);
      const int into = (r - start) & (kRowsAtOnce - 1);
      other |= (above & ((1u << src) - 1u)) != 0u;
      return into == 0 || other ? min(kRowsAtOnce - into, end - r) : 0;
    }
    other |= above != 0u;
  }
  return 0;
}

// d (16 x 8, fp32) += a (16 x 16) * b (16 x 8).  TYPE: 1 fp16, 2 bf16
template <int TYPE>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  if constexpr (TYPE == 1)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Joins the warps' sums (lane (g, c): features g and g + 8 of tokens 2 c and 2 c + 1) and stores them.
// feature(j): the j-th feature of the block.
template <int WARPS, class Feature>
__device__ __forceinline__ void rows_join(const RowsParams& p, const float (&acc)[4], int rows, int r, Feature feature) {
  __shared__ float sums[WARPS][kRowsFeatures][kRowsAtOnce];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  sums[warp][g][2 * c] = acc[0];
  sums[warp][g][2 * c + 1] = acc[1];
  sums[warp][g + 8][2 * c] = acc[2];
  sums[warp][g + 8][2 * c + 1] = acc[3];
  __syncthreads();
  const int j = threadIdx.x & 15, t = threadIdx.x >> 4;  // feature of the block, token
  if (t >= rows) return;
  const int n = feature(j);
  if (n >= p.N) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v += sums[w][j][t];
  const long long o = static_cast<long long>(r + t) * p.N + n;
  if (p.out_type == 0)
    static_cast<float*>(p.out)[o] = v;
  else if (p.out_type == 1)
    static_cast<__half*>(p.out)[o] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(v);
}

// (volatile: the loads stay together, ahead of the arithmetic; left to the compiler, four are in flight)
__device__ __forceinline__ uint4 load_or_zero(const uint4* p, bool in) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (in)
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// 16-bit operands.  A warp takes stretches of 256 elements (512 bytes of every row), WARPS stretches apart: 16
// warps where the reduction has that many.
template <int TYPE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) hb_group_rows_kernel(const RowsParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int r = blockIdx.y;
  int e, start;
  const int rows = rows_taken(p, r, e, start);
  if (rows == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * kRowsFeatures;
  // (rows behind the last feature read the last one and are not stored)
  const uint16_t* w = static_cast<const uint16_t*>(p.w) + static_cast<long long>(e) * p.N * p.K;
  const uint4* w0 = reinterpret_cast<const uint4*>(w + static_cast<long long>(min(n0 + g, p.N - 1)) * p.K);
  const uint4* w1 = reinterpret_cast<const uint4*>(w + static_cast<long long>(min(n0 + g + 8, p.N - 1)) * p.K);
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) +
                                                  static_cast<long long>(r + min(g, rows - 1)) * p.K);  // (columns behind the last row are not stored)
  const int pieces = p.K / 8;  // 16-byte pieces of a row
  constexpr int kAhead = 8;    // pieces of 32 elements a stretch
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  auto stretch = [&](int q0, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;  // all of the stretch lies within the row
    uint4 a[kAhead], b[kAhead], t[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int q = q0 + u * 4 + c;
      a[u] = load_or_zero(w0 + q, kWhole || q < pieces);
      b[u] = load_or_zero(w1 + q, kWhole || q < pieces);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int q = q0 + u * 4 + c;
      t[u] = load_or_zero(x + q, kWhole || q < pieces);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      mma_16x8x16<TYPE>(acc, a[u].x, b[u].x, a[u].y, b[u].y, t[u].x, t[u].y);
      mma_16x8x16<TYPE>(acc, a[u].z, b[u].z, a[u].w, b[u].w, t[u].z, t[u].w);
    }
  };
  for (int q0 = warp * kAhead * 4; q0 < pieces; q0 += WARPS * kAhead * 4) {
    if (q0 + kAhead * 4 <= pieces)
      stretch(q0, std::true_type{});
    else
      stretch(q0, std::false_type{});
  }
  rows_join<WARPS>(p, acc, rows, r, [&](int j) { return n0 + j; });
}

// Lane c of four holds word i of M[c][i]; afterwards word i of lane c is M[i][c].
__device__ __forceinline__ void transpose4(uint4& q, int c) {
  uint32_t s = c & 1 ? q.x : q.y, t = c & 1 ? q.z : q.w;
  s = __shfl_xor_sync(0xffffffffu, s, 1);
  t = __shfl_xor_sync(0xffffffffu, t, 1);
  if (c & 1) { q.x = s; q.z = t; } else { q.y = s; q.w = t; }
  s = c & 2 ? q.x : q.z;
  t = c & 2 ? q.y : q.w;
  s = __shfl_xor_sync(0xffffffffu, s, 2);
  t = __shfl_xor_sync(0xffffffffu, t, 2);
  if (c & 2) { q.x = s; q.y = t; } else { q.z = s; q.w = t; }
}

// 8 E2M1 elements as four pairs of fp16, elements j and j + 4 of the word in pair j.  With sign, exponent
// and mantissa bit in place both formats' values, the subnormal included, differ by the factor 2^14.
__device__ __forceinline__ void widen_e2m1x8(uint32_t w, uint32_t (&h)[4]) {
  h[0] = ((w << 12) & 0x80008000u) | ((w << 9) & 0x0e000e00u);
  h[1] = ((w << 8) & 0x80008000u) | ((w << 5) & 0x0e000e00u);
  h[2] = ((w << 4) & 0x80008000u) | ((w << 1) & 0x0e000e00u);
  h[3] = (w & 0x80008000u) | ((w >> 3) & 0x0e000e00u);
}

// Whether one of four scale bytes (E8M0) is 160 or more: 2^33 on, and NaN.
__device__ __forceinline__ bool e8m0_far(uint32_t word) { return (word & ((word << 1) | (word << 2)) & 0x80808080u) != 0u; }

// The values of four scale bytes that are not far, times 2^14 (so that byte 0, 2^-127, is a normal number too).
__device__ __forceinline__ void e8m0_values(uint32_t word, float (&v)[4]) {
  constexpr uint32_t k14 = 14u << 23;
  v[0] = __uint_as_float(((word << 23) & 0x7f800000u) + k14);
  v[1] = __uint_as_float(((word << 15) & 0x7f800000u) + k14);
  v[2] = __uint_as_float(((word << 7) & 0x7f800000u) + k14);
  v[3] = __uint_as_float(((word >> 1) & 0x7f800000u) + k14);
}

// sum + d 2^28 2^(a - 127) 2^(b - 127) for any two scale bytes, 255 being NaN.  d 2^28 is a multiple of 1/4 with 13 bits;
// the exponents are added as integers and half of their sum is applied at a time (2^-127 is subnormal), so that nothing
// leaves fp32 on the way unless the result does, and the only rounding is that of the sum.
__device__ __forceinline__ float add_far(float d, uint32_t a, uint32_t b, float sum) {
  const int e = static_cast<int>(a + b) - 254, h = e >> 1;
  auto power = [](int n) { return __uint_as_float(n > -127 ? static_cast<uint32_t>(n + 127) << 23 : 0x00400000u); };
  const float s = a == 255u || b == 255u ? __uint_as_float(0x7fc00000u) : power(e - h);
  return fmaf(d * 268435456.f * power(h), s, sum);
}

// d (16 x 8, fp32) = a (16 x 16, fp16) * b (16 x 8, fp16)
__device__ __forceinline__ void mma_16x8x16_from_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                      uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// MXFP4 operands.  A lane's 16 bytes are one block of 32 elements; four lanes exchange them so that each
// holds a quarter of every block, and a block is two instructions in fp16 from zero: the elements' products
// are multiples of 1/4 up to 36 (times 2^-28), so the block's sum has 13 bits and is exact.  It is
// multiplied by the product of the two scales, each times 2^14, and added in fp32.  That product is below 2^93 as long
// as no scale passes 2^32, and it is exact down to 2^-149, below which a block's true sum is under 2^-166 and lost in any
// fp32 sum.  A warp that meets a larger scale takes the longer way of add_far for the tile: scales of 2^64 would meet
// in an infinity where the sum is 2^126 or 0.  (2^28 put back at the end kept sums below 2^-98 in subnormals.)
// The instructions bound the kernel (about 400 for 16 x 128 weights), not the memory: one row of 4096 x 4096
// 7.0 us, eight 7.6 (with the choice made inside the loop over blocks 7.4 and 7.9); the conversion
// instruction for two elements and E4M3 operands for the 32-deep instruction were no faster than the bit operations here.  A warp takes tiles of 128 elements, kRowsWarps tiles apart.
// The 16 features are four lines of the scale tile in each of its four bands: their scales of 128 elements
// are 64 consecutive bytes (16 features in a row would use a quarter of every sector).
__global__ void __launch_bounds__(kRowsWarps * 32) hb_mx_rows_kernel(const RowsParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int r = blockIdx.y;
  int e, start;
  const int rows = rows_taken(p, r, e, start);
  if (rows == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int kt = (p.K + 127) / 128, blocks = p.K / 32;
  const int line0 = (blockIdx.x & 7) * 4, tile_n = blockIdx.x >> 3;
  auto feature = [&](int j) { return tile_n * 128 + (j & 3) * 32 + line0 + (j >> 2); };
  const uint4* w = static_cast<const uint4*>(p.w) + static_cast<long long>(e) * p.N * blocks;
  const uint4* w0 = w + static_cast<long long>(min(feature(g), p.N - 1)) * blocks;
  const uint4* w1 = w + static_cast<long long>(min(feature(g + 8), p.N - 1)) * blocks;
  const uint32_t* wsf = reinterpret_cast<const uint32_t*>(p.w_sf + e * p.w_matrix_sf + static_cast<long long>(tile_n) * kt * kAtomBytes) +
                        (line0 + (g >> 2)) * 4 + (g & 3);
  const uint4* x = static_cast<const uint4*>(p.x) + static_cast<long long>(r + min(g, rows - 1)) * blocks;
  // (a group's rows start at tile row start / 128 + e; rows up to the next multiple of eight share a band)
  const int local = r - start;
  const uint32_t* xsf = reinterpret_cast<const uint32_t*>(
                            p.x_sf + static_cast<long long>((p.offsets ? start / 128 + e : 0) + local / 128) * kt * kAtomBytes) +
                        (local % 32) * 4 + (local % 128) / 32;
  constexpr int kAhead = 4;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = warp; i0 < kt; i0 += kRowsWarps * kAhead) {
    uint4 a[kAhead], b[kAhead], t[kAhead];
    uint32_t sa[kAhead], sb[kAhead], s0[kAhead], s1[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kRowsWarps, q = i * 4 + c;
      a[u] = load_or_zero(w0 + q, q < blocks);
      b[u] = load_or_zero(w1 + q, q < blocks);
      t[u] = load_or_zero(x + q, q < blocks);
      const bool in = i < kt;
      sa[u] = in ? wsf[i * (kAtomBytes / 4)] : 0u;
      sb[u] = in ? wsf[i * (kAtomBytes / 4) + 8] : 0u;  // (feature g + 8: two lines on)
      // (columns without a row: scales of 1, which are not far)
      s0[u] = in && 2 * c < rows ? xsf[i * (kAtomBytes / 4) + 8 * c] : 0x7f7f7f7fu;
      s1[u] = in && 2 * c + 1 < rows ? xsf[i * (kAtomBytes / 4) + 8 * c + 4] : 0x7f7f7f7fu;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u * kRowsWarps >= kt) break;
      transpose4(a[u], c);
      transpose4(b[u], c);
      transpose4(t[u], c);
      const uint32_t wa[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, wb[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
      const uint32_t wt[4] = {t[u].x, t[u].y, t[u].z, t[u].w};
      const bool far = __any_sync(0xffffffffu, e8m0_far(sa[u]) || e8m0_far(sb[u]) || e8m0_far(s0[u]) || e8m0_far(s1[u]));
      // block k of the tile: its sum over each pair of a feature and a token, times 2^-28
      auto block_sums = [&](int k, float (&d)[4]) {
        uint32_t ha[4], hb[4], ht[4];
        widen_e2m1x8(wa[k], ha);
        widen_e2m1x8(wb[k], hb);
        widen_e2m1x8(wt[k], ht);
        mma_16x8x16_from_zero(d, ha[0], hb[0], ha[1], hb[1], ht[0], ht[1]);
        mma_16x8x16<1>(d, ha[2], hb[2], ha[3], hb[3], ht[2], ht[3]);
      };
      if (!far) {
        float fa[4], fb[4], f0[4], f1[4];
        e8m0_values(sa[u], fa);
        e8m0_values(sb[u], fb);
        e8m0_values(s0[u], f0);
        e8m0_values(s1[u], f1);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float d[4];
          block_sums(k, d);
          acc[0] = fmaf(d[0], fa[k] * f0[k], acc[0]);
          acc[1] = fmaf(d[1], fa[k] * f1[k], acc[1]);
          acc[2] = fmaf(d[2], fb[k] * f0[k], acc[2]);
          acc[3] = fmaf(d[3], fb[k] * f1[k], acc[3]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float d[4];
          block_sums(k, d);
          const uint32_t a0 = (sa[u] >> (8 * k)) & 255u, b0 = (sb[u] >> (8 * k)) & 255u;
          const uint32_t t0 = (s0[u] >> (8 * k)) & 255u, t1 = (s1[u] >> (8 * k)) & 255u;
          acc[0] = add_far(d[0], a0, t0, acc[0]);
          acc[1] = add_far(d[1], a0, t1, acc[1]);
          acc[2] = add_far(d[2], b0, t0, acc[2]);
          acc[3] = add_far(d[3], b0, t1, acc[3]);
        }
      }
    }
  }
  rows_join<kRowsWarps>(p, acc, rows, r, feature);
}

}  // namespace hb
