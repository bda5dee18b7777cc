// Quantisers to E4M3 with FP32 scales, for the block-scaled products (gemm_grouped.cuh):
//   rows:  one scale for 128 consecutive values of a row       (activations)
//   tiles: one scale for a 128 x 128 tile of a matrix          (weights)
// amax = max |x| of the block, at least 2^-100 (a block of zeros then has a finite inverse);
// scale = amax / 448, q = e4m3(x * (448 / amax)), both quotients and the product rounded to FP32
// once, q to nearest even and clamped to +-448 (the product can pass it by an ulp). The amax is
// taken on the sign-cleared bits, whose order as integers is the order of the values with infinity
// and then NaN on top, so a NaN or an infinity in a block makes its scale one as well.
//
// Bound: HBM, 3 bytes a value. One pass: a block's values stay in registers between the maximum and
// the conversion. Rows: a half-warp holds a block as 16 bytes a lane, each thread loads four blocks
// before it uses the first, and a CTA takes 8 rows x 8 blocks, so that the scales, stored by blocks,
// go out as 32-byte sectors. Tiles: a CTA of 256 threads holds the 32 KB tile as eight 16-byte loads a
// thread.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace hst {

constexpr int kQuantThreads = 256;
constexpr int kQuantRows = 8, kQuantBlocks = 8;  // rows and 128-value blocks of a CTA
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 7.8886090522101181e-31f;  // 2^-100

struct QuantizeArgs {
  const void* x;
  int64_t x_batch, x_row, x_col;  // strides, elements
  uint8_t* q;
  int64_t q_batch, q_row;
  float* scales;
  int64_t s_batch, s_row, s_col;
  int rows, cols, col_blocks;
};

template <typename T>
__device__ __forceinline__ float bits_to_f32(uint32_t b);
template <>
__device__ __forceinline__ float bits_to_f32<__half>(uint32_t b) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
}
template <>
__device__ __forceinline__ float bits_to_f32<__nv_bfloat16>(uint32_t b) {
  return __uint_as_float(b << 16);
}

__device__ __forceinline__ uint32_t absmax2(uint32_t m, uint32_t v) { return __vmaxu2(m, v & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t absmax8(uint32_t m, const uint4& v) {
  return absmax2(absmax2(absmax2(absmax2(m, v.x), v.y), v.z), v.w);
}

// The block's amax from its bits (two 16-bit maxima packed).
template <typename T>
__device__ __forceinline__ float amax_of(uint32_t m) {
  const float a = bits_to_f32<T>(max(m & 0xffffu, m >> 16));
  return a < kAmaxFloor ? kAmaxFloor : a;  // keeps NaN
}

template <typename T>
__device__ __forceinline__ uint32_t quantize4(uint32_t a, uint32_t b, float inv) {
  const float2 lo = make_float2(bits_to_f32<T>(a & 0xffffu) * inv, bits_to_f32<T>(a >> 16) * inv);
  const float2 hi = make_float2(bits_to_f32<T>(b & 0xffffu) * inv, bits_to_f32<T>(b >> 16) * inv);
  const uint32_t l = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3);
  const uint32_t h = __nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3);
  return l | (h << 16);
}

template <typename T>
__device__ __forceinline__ uint8_t quantize1(uint32_t bits, float inv) {
  return __nv_cvt_float_to_fp8(bits_to_f32<T>(bits) * inv, __NV_SATFINITE, __NV_E4M3);
}

// Rows whose values come 16 bytes at a time: unit column stride, rows and base 16-byte aligned, a
// multiple of 8 columns; q's rows 8-byte aligned.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const QuantizeArgs a) {
  __shared__ float staged[kQuantRows * kQuantBlocks];
  const int half_lane = threadIdx.x & 15, half_warp = threadIdx.x >> 4;
  const int block_tiles = (a.col_blocks + kQuantBlocks - 1) / kQuantBlocks;
  const int row_tile = static_cast<int>(blockIdx.x) / block_tiles;
  const int row0 = row_tile * kQuantRows, cb0 = (static_cast<int>(blockIdx.x) - row_tile * block_tiles) * kQuantBlocks;
  const int cb = half_warp % kQuantBlocks;  // this half-warp's block of four rows
  const int col = (cb0 + cb) * 128 + half_lane * 8;
  constexpr int kStep = kQuantThreads / 16 / kQuantBlocks;
  const int first = half_warp / kQuantBlocks;
  const uint16_t* x = static_cast<const uint16_t*>(a.x);
  uint4 v[kQuantRows / kStep];
#pragma unroll
  for (int i = 0; i < kQuantRows / kStep; ++i) {
    const int row = row0 + first + i * kStep;
    v[i] = make_uint4(0, 0, 0, 0);
    if (row < a.rows && col < a.cols) v[i] = __ldcs(reinterpret_cast<const uint4*>(x + row * a.x_row + col));
  }
#pragma unroll
  for (int i = 0; i < kQuantRows / kStep; ++i) {
    const int r = first + i * kStep;
    uint32_t m = absmax8(0, v[i]);
#pragma unroll
    for (int d = 8; d >= 1; d /= 2) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float amax = amax_of<T>(m);
    const float inv = kE4m3Max / amax;
    if (row0 + r < a.rows && col < a.cols) {
      *reinterpret_cast<uint2*>(a.q + (row0 + r) * a.q_row + col) =
          make_uint2(quantize4<T>(v[i].x, v[i].y, inv), quantize4<T>(v[i].z, v[i].w, inv));
    }
    if (half_lane == 0) staged[cb * kQuantRows + r] = amax / kE4m3Max;
  }
  __syncthreads();
  const int t = static_cast<int>(threadIdx.x);
  if (t < kQuantRows * kQuantBlocks) {
    const int r = row0 + t % kQuantRows, c = cb0 + t / kQuantRows;
    if (r < a.rows && c < a.col_blocks) a.scales[r * a.s_row + c * a.s_col] = staged[t];
  }
}

// Any strides and extents: one warp per block of 128 values.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_any_kernel(const QuantizeArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t units = static_cast<int64_t>(a.rows) * a.col_blocks;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (u >= units) return;
  const int64_t row = u / a.col_blocks;
  const int cb = static_cast<int>(u - row * a.col_blocks);
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.x_row;
  uint32_t v[4], m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = cb * 128 + i * 32 + lane;
    v[i] = col < a.cols ? x[col * a.x_col] : 0u;
    m = max(m, v[i] & 0x7fffu);
  }
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  const float amax = amax_of<T>(m);
  const float inv = kE4m3Max / amax;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = cb * 128 + i * 32 + lane;
    if (col < a.cols) a.q[row * a.q_row + col] = quantize1<T>(v[i], inv);
  }
  if (lane == 0) a.scales[row * a.s_row + cb * a.s_col] = amax / kE4m3Max;
}

__device__ __forceinline__ uint32_t block_absmax(uint32_t m) {
  __shared__ uint32_t part[kQuantThreads / 32];
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) m = __vmaxu2(m, part[i]);
  return m;
}

// One 128 x 128 tile per CTA (x: column tile, y: row tile, z: matrix), with the alignment of
// quantize_rows_kernel.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_tiles_kernel(const QuantizeArgs a) {
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + blockIdx.z * a.x_batch;
  uint8_t* q = a.q + blockIdx.z * a.q_batch;
  const int col = blockIdx.x * 128 + (threadIdx.x & 15) * 8;
  const int row0 = blockIdx.y * 128 + (threadIdx.x >> 4);
  uint4 v[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + i * 16;
    v[i] = make_uint4(0, 0, 0, 0);
    if (row < a.rows && col < a.cols) v[i] = __ldcs(reinterpret_cast<const uint4*>(x + row * a.x_row + col));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = absmax8(m, v[i]);
  const float amax = amax_of<T>(block_absmax(m));
  const float inv = kE4m3Max / amax;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + i * 16;
    if (row < a.rows && col < a.cols) {
      *reinterpret_cast<uint2*>(q + row * a.q_row + col) =
          make_uint2(quantize4<T>(v[i].x, v[i].y, inv), quantize4<T>(v[i].z, v[i].w, inv));
    }
  }
  if (threadIdx.x == 0)
    a.scales[blockIdx.z * a.s_batch + blockIdx.y * a.s_row + blockIdx.x * a.s_col] = amax / kE4m3Max;
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_tiles_any_kernel(const QuantizeArgs a) {
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + blockIdx.z * a.x_batch;
  uint8_t* q = a.q + blockIdx.z * a.q_batch;
  const int col = blockIdx.x * 128 + (threadIdx.x & 127);
  const int row0 = blockIdx.y * 128 + (threadIdx.x >> 7);
  uint32_t m = 0;
  for (int i = 0; i < 128; i += 2) {
    if (row0 + i < a.rows && col < a.cols) m = max(m, x[(row0 + i) * a.x_row + col * a.x_col] & 0x7fffu);
  }
  const float amax = amax_of<T>(block_absmax(m));
  const float inv = kE4m3Max / amax;
  for (int i = 0; i < 128; i += 2) {
    if (row0 + i < a.rows && col < a.cols)
      q[(row0 + i) * a.q_row + col] = quantize1<T>(x[(row0 + i) * a.x_row + col * a.x_col], inv);
  }
  if (threadIdx.x == 0)
    a.scales[blockIdx.z * a.s_batch + blockIdx.y * a.s_row + blockIdx.x * a.s_col] = amax / kE4m3Max;
}

}  // namespace hst
