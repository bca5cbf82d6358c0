// Microscaled 4-bit floating point (MXFP4): quantisation and the way back.
//
// 32 consecutive elements of a row share one power-of-two scale 2^s:
//   s = max(floor(log2(max |x|)) - 2, -127),   q = round_e2m1(x * 2^-s)
// with E2M1 the values 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives, round to nearest even, and what is
// above 6 (x * 2^-s is below 8) set to 6.  x * 2^-s is a multiplication by a power of two, so it rounds
// only where the result is far below the smallest element: q is exact from the definition.  The scale
// byte is s + 127 (E8M0).  A block with an infinity or a NaN has no such scale: its byte is 255, its
// elements are 0, and it reads back as NaN.
//
// Memory.  Codes: two to a byte, even element in the low half, rows dense (K / 2 bytes).  Scales: tiles
// of 128 rows x 4 blocks (128 elements), 512 bytes each, the tiles of a tile row side by side; in a tile
// the byte of row r, block b is (r % 32) * 16 + r / 32 * 4 + b: what one copy brings to tensor memory.
// Rows grouped by expert start a new tile row per group: group g's first tile row is
// offsets[g] / 128 + g, which leaves room for every group before it.  Bytes of a row behind its last
// block are written as 0; bytes of rows that a tile has and the matrix has not are never written.
//
// Both kernels move each byte once and are bound by memory.
#pragma once
#include "hb_group.cuh"

namespace hb {

struct MxParams {
  const void* x;         // quantise: input values; dequantise: unused
  uint8_t* codes;
  uint8_t* scales;
  void* out;             // dequantise: output values
  const int* offsets;    // groups of rows, or nullptr
  int batch, rows, K, groups;
  long long matrix_scales;  // scale bytes of one matrix of the batch
};

// Tile row and row within it of row r of matrix b; false for a row of no group.
__device__ __forceinline__ bool mx_place(const MxParams& p, const int* off, int r, int& tile_row, int& local) {
  if (!off) {
    tile_row = r >> 7;
    local = r & 127;
    return true;
  }
  // the last group that starts at or before r (of groups that start at the same row only the last
  // has rows); wrong offsets give some group, and a tile row of at most r / 128 + groups - 1
  int lo = 0, hi = p.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= r) lo = mid; else hi = mid;
  }
  if (off[lo] > r || r >= off[lo + 1]) return false;
  const int first = max(off[lo], 0);
  tile_row = (first >> 7) + lo + ((r - first) >> 7);
  local = (r - first) & 127;
  return true;
}

__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// TYPE: 0 fp32, 1 fp16, 2 bf16
template <int TYPE>
__device__ __forceinline__ void load8(const void* src, long long i, float (&v)[8]) {
  if constexpr (TYPE == 0) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(src) + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (TYPE == 1) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  }
}

constexpr int kMxThreads = 256;

// 16 lanes take 128 elements of a row: 8 elements a lane, four lanes a block.
template <int TYPE>
__global__ void __launch_bounds__(kMxThreads) hb_quantize_mxfp4_kernel(const MxParams p) {
  extern __shared__ int s_off[];
  griddep_wait();
  griddep_launch_dependents();
  const int* off = nullptr;
  if (p.offsets) {
    for (int i = threadIdx.x; i <= p.groups; i += kMxThreads) s_off[i] = p.offsets[i];
    __syncthreads();
    off = s_off;
  }
  const int kt = (p.K + 127) / 128;
  const int lane16 = threadIdx.x & 15;
  const long long units = static_cast<long long>(p.batch) * p.rows * kt;
  for (long long base = (static_cast<long long>(blockIdx.x) * kMxThreads + threadIdx.x - lane16) >> 4; ;
       base += static_cast<long long>(gridDim.x) * (kMxThreads / 16)) {
    // (whole warps leave together: the shuffles below name all lanes)
    if (!__any_sync(0xffffffffu, base < units)) break;
    const bool live = base < units;
    const long long row_all = live ? base / kt : 0;
    const int tile_k = live ? static_cast<int>(base - row_all * kt) : 0;
    const int mat = static_cast<int>(row_all / p.rows), r = static_cast<int>(row_all - static_cast<long long>(mat) * p.rows);
    int tile_row = 0, local = 0;
    const bool placed = live && mx_place(p, off, r, tile_row, local);
    const int col = tile_k * 128 + lane16 * 8;
    const bool has = placed && col < p.K;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (has) load8<TYPE>(p.x, row_all * p.K + col, v);
    // the largest magnitude as bits: the order of non-negative floats, with infinity and NaN on top
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = static_cast<int>(top >> 23);
    const bool bad = ex == 255;
    const uint32_t code = bad ? 255u : static_cast<uint32_t>(max(ex - 2, 0));  // s + 127
    const float inv = __uint_as_float((254u - (bad ? 127u : code)) << 23);     // 2^-s
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bad ? 0.f : v[j] * inv;
    const uint32_t packed = pack_e2m1x8(v);
    // four blocks' scale bytes of these 128 elements as one word
    uint32_t word = has ? code << (8 * (lane16 >> 2)) : 0u;
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if (has) *reinterpret_cast<uint32_t*>(p.codes + ((row_all * p.K + col) >> 1)) = packed;
    if (placed && lane16 == 0)
      *reinterpret_cast<uint32_t*>(p.scales + mat * p.matrix_scales +
                                   (static_cast<long long>(tile_row) * kt + tile_k) * kAtomBytes + (local & 31) * 16 +
                                   (local >> 5) * 4) = word;
  }
}

template <int TYPE>
__global__ void __launch_bounds__(kMxThreads) hb_dequantize_mxfp4_kernel(const MxParams p) {
  extern __shared__ int s_off[];
  griddep_wait();
  griddep_launch_dependents();
  const int* off = nullptr;
  if (p.offsets) {
    for (int i = threadIdx.x; i <= p.groups; i += kMxThreads) s_off[i] = p.offsets[i];
    __syncthreads();
    off = s_off;
  }
  const int kt = (p.K + 127) / 128;
  const int lane16 = threadIdx.x & 15;
  const long long units = static_cast<long long>(p.batch) * p.rows * kt;
  for (long long base = (static_cast<long long>(blockIdx.x) * kMxThreads + threadIdx.x) >> 4; base < units;
       base += static_cast<long long>(gridDim.x) * (kMxThreads / 16)) {
    const long long row_all = base / kt;
    const int tile_k = static_cast<int>(base - row_all * kt);
    const int mat = static_cast<int>(row_all / p.rows), r = static_cast<int>(row_all - static_cast<long long>(mat) * p.rows);
    int tile_row = 0, local = 0;
    const int col = tile_k * 128 + lane16 * 8;
    if (col >= p.K || !mx_place(p, off, r, tile_row, local)) continue;
    const uint32_t packed = *reinterpret_cast<const uint32_t*>(p.codes + ((row_all * p.K + col) >> 1));
    const uint32_t code = p.scales[mat * p.matrix_scales + (static_cast<long long>(tile_row) * kt + tile_k) * kAtomBytes +
                                   (local & 31) * 16 + (local >> 5) * 4 + (lane16 >> 2)];
    // 2^(code - 127): the smallest is subnormal, 255 stands for NaN
    const float scale = __uint_as_float(code == 0 ? 0x00400000u : (code == 255u ? 0x7fc00000u : code << 23));
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t h2;
      asm("{\n\t"
          ".reg .b8 b, z;\n\t"
          "mov.b16 {b, z}, %1;\n\t"
          "cvt.rn.f16x2.e2m1x2 %0, b;\n\t"
          "}"
          : "=r"(h2)
          : "h"(static_cast<uint16_t>((packed >> (8 * j)) & 255u)));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      v[2 * j] = f.x * scale;
      v[2 * j + 1] = f.y * scale;
    }
    const long long o = row_all * p.K + col;
    if constexpr (TYPE == 0) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p.out) + o);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (TYPE == 1) {
          const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + o) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

}  // namespace hb
