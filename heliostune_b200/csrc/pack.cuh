// Copies of operands whose layout a TMA tensor map cannot describe, into rows of a multiple of 16
// bytes. A stack of weights is copied for the groups that have rows alone: what a call does not read it
// does not copy (one token among 49 experts: one weight instead of 49).
//
// Bound: HBM, each byte read and written once. A thread makes 16 bytes of the copy, from the widest
// loads the source's alignment allows.
#pragma once

#include <stdint.h>

namespace hst {

constexpr int kPackThreads = 256;
constexpr int kPackPerThread = 4;

struct PackArgs {
  const uint8_t* src;
  int64_t s_group, s_row, s_col;  // bytes
  uint8_t* dst;
  int64_t d_group, d_row;  // bytes, multiples of 16
  const int32_t* ends;     // null: every group
  int total_rows;          // of the row matrix `ends` is about
  int64_t rows;            // of one matrix
  int chunks;              // 16-byte chunks of a row
  int64_t row_bytes;
};

// Whether group g has no rows, its ends taken as build_group_rows takes them. All threads.
__device__ inline bool group_is_empty(const PackArgs& a, int g) {
  if (a.ends == nullptr) return false;
  int before = 0;
  for (int i = static_cast<int>(threadIdx.x); i < g; i += static_cast<int>(blockDim.x)) before = max(before, a.ends[i]);
  const int end = min(a.ends[g], a.total_rows);
  return __syncthreads_or(before >= end || end <= 0) != 0;
}

// U: the widest type the source's rows are aligned to (unit column stride).
template <typename U>
__global__ void __launch_bounds__(kPackThreads) pack_rows_kernel(const PackArgs a) {
  const int g = static_cast<int>(blockIdx.y);
  if (group_is_empty(a, g)) return;
  const int64_t total = a.rows * a.chunks;
  constexpr int kParts = 16 / sizeof(U);
#pragma unroll
  for (int j = 0; j < kPackPerThread; ++j) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * kPackPerThread + j) * kPackThreads + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / a.chunks;
    const int64_t at = (i - row * a.chunks) * 16;
    const uint8_t* src = a.src + g * a.s_group + row * a.s_row + at;
    union {
      U part[kParts];
      uint4 all;
    } v;
    v.all = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      if (at + p * static_cast<int64_t>(sizeof(U)) < a.row_bytes) v.part[p] = reinterpret_cast<const U*>(src)[p];
    }
    *reinterpret_cast<uint4*>(a.dst + g * a.d_group + row * a.d_row + at) = v.all;
  }
}

// Any column stride: U is one value. A block takes 32 x 32 values through shared memory, so that both
// sides of a transposing copy are read and written along their contiguous dimension.
template <typename U>
__global__ void __launch_bounds__(kPackThreads) pack_any_kernel(const PackArgs a) {
  __shared__ U tile[32][33];
  const int g = static_cast<int>(blockIdx.y);
  if (group_is_empty(a, g)) return;
  const int cols = static_cast<int>(a.row_bytes / sizeof(U));
  const int col_tiles = (cols + 31) / 32;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) / col_tiles * 32;
  const int col0 = static_cast<int>(static_cast<int64_t>(blockIdx.x) % col_tiles) * 32;
  const uint8_t* src = a.src + g * a.s_group;
  const bool by_column = a.s_row < a.s_col;  // the rows are the closer dimension of the source
  const int fast = threadIdx.x & 31;
  for (int slow = threadIdx.x >> 5; slow < 32; slow += kPackThreads / 32) {
    const int r = by_column ? fast : slow, c = by_column ? slow : fast;
    if (row0 + r < a.rows && col0 + c < cols) {
      tile[r][c] = *reinterpret_cast<const U*>(src + (row0 + r) * a.s_row + (col0 + c) * a.s_col);
    }
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < 32; r += kPackThreads / 32) {
    if (row0 + r < a.rows && col0 + fast < cols) {
      *reinterpret_cast<U*>(a.dst + g * a.d_group + (row0 + r) * a.d_row + (col0 + fast) * static_cast<int64_t>(sizeof(U))) =
          tile[r][fast];
    }
  }
}

}  // namespace hst
