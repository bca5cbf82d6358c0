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

// Eight values as they lie in memory.  TYPE: 0 fp32, 1 fp16, 2 bf16
template <int TYPE>
struct Eight {
  uint4 w[TYPE == 0 ? 2 : 1];

  __device__ __forceinline__ void load(const void* src, long long i) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(src) + i * (TYPE == 0 ? 4 : 2));
    w[0] = q[0];
    if constexpr (TYPE == 0) w[1] = q[1];
  }
  __device__ __forceinline__ void clear() {
    w[0] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (TYPE == 0) w[1] = w[0];
  }
  // The largest magnitude as the bits of a float: the order of non-negative floats, infinity and NaN on
  // top.  16-bit values are compared in pairs (a maximum that keeps NaN) and widened once.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (TYPE == 0) {
      const uint32_t b[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
      uint32_t t = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) t = max(t, b[j] & 0x7fffffffu);
      return t;
    } else {
      const uint32_t b[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
      if constexpr (TYPE == 1) {
        const __half2* h = reinterpret_cast<const __half2*>(b);
        const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
        return __float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))) & 0x7fffffffu;
      } else {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(b);
        const __nv_bfloat162 m =
            __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
        return __float_as_uint(__bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)))) & 0x7fffffffu;
      }
    }
  }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
    if constexpr (TYPE == 0) {
      const uint32_t b[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(b[j]);
    } else {
      const uint32_t b[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (TYPE == 1) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b[j]));
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        } else {
          v[2 * j] = __uint_as_float(b[j] << 16);
          v[2 * j + 1] = __uint_as_float(b[j] & 0xffff0000u);
        }
      }
    }
  }
};

constexpr int kMxThreads = 256;
constexpr int kMxSegment = 1024;  // elements of a row that a block takes

// Block (x, y): tile row x / 16 of the scales, segment y of its rows.  A warp takes 256 elements of one
// row in each of the tile's four bands of 32 rows, because the scales of those four rows and 128 elements
// are 16 consecutive bytes: four 16-byte loads of values a lane in flight, one 16-byte store of scales.
// 16 lanes take 128 elements, four a block of 32.  The grid names rows and segments, so that the index
// costs no division.  8192 x 4096 bf16: a flat index with two divisions per 128 elements 33.8 us, a warp
// per row and four-byte scale stores 19.0 us, the four rows collected in shared memory 22.9 us.
struct MxLane {
  long long row[4];  // of the batch's rows one after the other
  bool placed[4];
  long long sf;  // the four rows' scale words of the lane's 128 elements
  int col;       // the lane's first element
};
__device__ __forceinline__ MxLane mx_lane(const MxParams& p, int kt) {
  MxLane l;
  const int* off = p.offsets;
  const int warp = threadIdx.x >> 5;
  int tile_row = blockIdx.x >> 4;
  const int local = 2 * (blockIdx.x & 15) + (warp & 1);
  l.col = blockIdx.y * kMxSegment + (warp >> 1) * 256 + (threadIdx.x & 31) * 8;
  l.sf = (static_cast<long long>(tile_row) * kt + (l.col >> 7)) * kAtomBytes + local * 16;
  long long first, end, base = 0;  // row of the tile's first line, one past the last row, and of the matrix
  if (off) {
    // The last group whose first tile row, offsets[g] / 128 + g, is not behind this one (those rise with
    // g); wrong offsets give some group, and the rows stay within the matrix all the same.  A warp looks at
    // 32 groups at once, in two rounds beyond 32 groups: one or two loads' latency ahead of the data's
    // (a binary search in shared memory behind a barrier: 22.3 us for 8192 x 4096 bf16 in 32 groups, 16.8
    // without groups).
    const int lane = threadIdx.x & 31;
    auto last_at = [&](int from, int step, int count) {
      const int g = from + lane * step;
      const bool in = lane < count && g < p.groups;
      const bool before = in && (min(max(off[in ? g : 0], 0), p.rows) >> 7) + g <= tile_row;
      return from + max(__popc(__ballot_sync(0xffffffffu, before)) - 1, 0) * step;
    };
    const int step = (p.groups + 31) / 32;
    int lo = last_at(0, step, 32);
    if (step > 1) lo = last_at(lo, 1, step);
    const int start = min(max(off[lo], 0), p.rows);
    const int behind = tile_row - (start >> 7) - lo;
    first = start + behind * 128LL;
    end = behind < 0 ? 0 : min(off[lo + 1], p.rows);
  } else {
    if (p.batch > 1) {
      const int per = (p.rows - 1) / 128 + 1;
      const int mat = tile_row / per;
      tile_row -= mat * per;
      base = static_cast<long long>(mat) * p.rows;
    }
    first = tile_row * 128LL;
    end = p.rows;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    l.row[i] = base + first + local + 32 * i;
    l.placed[i] = first + local + 32 * i < end && l.col < p.K;
  }
  return l;
}

template <int TYPE>
__global__ void __launch_bounds__(kMxThreads, TYPE == 0 ? 4 : 6) hb_quantize_mxfp4_kernel(const MxParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const MxLane l = mx_lane(p, (p.K + 127) / 128);
  if (!__any_sync(0xffffffffu, l.placed[0])) return;  // (the first band's row exists wherever another does)
  const int lane16 = threadIdx.x & 15;
  Eight<TYPE> in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (l.placed[i]) in[i].load(p.x, l.row[i] * p.K + l.col); else in[i].clear();
  }
  uint32_t word[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t top = in[i].top();
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = static_cast<int>(top >> 23);
    const bool bad = ex == 255;
    const uint32_t code = bad ? 255u : static_cast<uint32_t>(max(ex - 2, 0));  // s + 127
    const float inv = __uint_as_float((254u - (bad ? 127u : code)) << 23);     // 2^-s
    float v[8];
    in[i].widen(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    const uint32_t packed = bad ? 0u : pack_e2m1x8(v);
    if (l.placed[i]) *reinterpret_cast<uint32_t*>(p.codes + ((l.row[i] * p.K + l.col) >> 1)) = packed;
    // four blocks' scale bytes of these 128 elements as one word, zeros behind the row's last block
    word[i] = l.placed[i] ? code << (8 * (lane16 >> 2)) : 0u;
    word[i] |= __shfl_xor_sync(0xffffffffu, word[i], 4);
    word[i] |= __shfl_xor_sync(0xffffffffu, word[i], 8);
  }
  if (lane16 != 0) return;
  uint32_t* sf = reinterpret_cast<uint32_t*>(p.scales + l.sf);
  if (l.placed[3]) {
    *reinterpret_cast<uint4*>(sf) = make_uint4(word[0], word[1], word[2], word[3]);
  } else {  // not all four rows exist
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (l.placed[i]) sf[i] = word[i];
  }
}

template <int TYPE>
__global__ void __launch_bounds__(kMxThreads) hb_dequantize_mxfp4_kernel(const MxParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const MxLane l = mx_lane(p, (p.K + 127) / 128);
  if (!l.placed[0]) return;
  const int block = (threadIdx.x & 15) >> 2;  // of the four in a scale word
  // (bytes of rows that do not exist belong to the same 16 bytes of the array; they are not used)
  const uint4 words = *reinterpret_cast<const uint4*>(p.scales + l.sf);
  const uint32_t word[4] = {words.x, words.y, words.z, words.w};
  uint32_t packed[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    packed[i] = l.placed[i] ? *reinterpret_cast<const uint32_t*>(p.codes + ((l.row[i] * p.K + l.col) >> 1)) : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!l.placed[i]) break;
    const uint32_t code = (word[i] >> (8 * block)) & 255u;
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
          : "h"(static_cast<uint16_t>((packed[i] >> (8 * j)) & 255u)));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      v[2 * j] = f.x * scale;
      v[2 * j + 1] = f.y * scale;
    }
    const long long o = l.row[i] * p.K + l.col;
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
