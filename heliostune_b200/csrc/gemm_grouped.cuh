// Matrix products over rows grouped by expert, on CTA pairs (tcgen05.mma.cta_group::2).
//
// Group e owns rows [ends[e - 1], ends[e]) of a row matrix; `ends` lives on the GPU, so nothing
// about the sizes is known on the host. Four products share this kernel:
//   kForward       y[t, :] = x[t, :] W[e(t)]          16-bit x [T, K], W [E, K, N] (either of its
//                                                     two inner dimensions contiguous)
//   kWeightGrad    D[e] = L[rows of e]^T R[rows of e]  16-bit L [T, Lc], R [T, Rc]
//   kScaledWide    y[t, n] = sum_b sa[t, b] sb[e, n/128, b] sum_{k in block b} a[t, k] b[e, n, k]
//   kScaledStream  the same                            E4M3 a [T, K], b [E, N, K], FP32 scales of
//                                                     128 (a) and 128 x 128 (b) values
//
// One pair of CTAs computes a 256 x width tile: CTA r owns 128 rows of the L operand and half of
// the R operand's `width` columns. Which side the rows are on decides what raggedness costs:
//   * kForward and kScaledStream put the weights on the L side (M = 256 output columns) and the
//     rows on the R side, whose width is a run-time field of the UMMA descriptor (32..256). A
//     group's rows are cut into equal widths, so a group of r rows costs round_up(r / tiles, 32)
//     columns of tensor-core time per tile instead of the next multiple of 256, and each weight is
//     read once for up to 256 rows;
//   * kScaledWide keeps the rows on the L side, where one row is one TMEM lane: its scale is one
//     register, and the promotion below costs one FMA per element;
//   * kWeightGrad reduces over the rows, 64 at a time. Rows past the group's end in its last block
//     belong to other groups: a fourth kind of warp zeroes those of the last 16-row UMMA step in
//     shared memory (both operands, so that NaN or infinity there stays out), and the UMMA steps
//     past them are not issued.
//
// The scaled products accumulate each 128-deep block in a TMEM buffer of its own; the epilogue
// warps read it, multiply by the block's scales and add it to FP32 registers, while the next
// block's UMMAs fill another buffer.
//
// Schedule: all (tile, K block) iterations of all groups in one line, cut into one equal share per
// pair (contiguous, so neighbours in a share use the same weights out of L2). A tile cut by a
// share's end leaves FP32 pieces in the workspace, which a second small kernel
// (grouped_finish_kernel, a programmatic dependent) adds in K order. No CTA ever waits for another
// pair, no atomics: results are bitwise reproducible, and the two kernels can be captured and
// replayed. The second kernel also writes the zeros of rows past the last group and of the weight
// gradients of empty groups.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "gemm_tile.cuh"
#include "ptx.cuh"

namespace hst {

enum class GroupMode { kForward, kWeightGrad, kScaledWide, kScaledStream };

constexpr int kMaxGroups = 1024;
constexpr int kGroupLBytes = 16384;  // 128 L rows x 128 bytes of K (or 2 boxes of 64 x 64)
constexpr int kGroupRaster = 8;      // row tiles before the next column tile

__host__ __device__ constexpr bool group_scaled(GroupMode m) { return m == GroupMode::kScaledWide || m == GroupMode::kScaledStream; }
// Rows of the row matrix on the R side (their count is the tile's width).
__host__ __device__ constexpr bool group_rows_on_r(GroupMode m) { return m == GroupMode::kForward || m == GroupMode::kScaledStream; }
__host__ __device__ constexpr int group_epilogue_warps(GroupMode m) { return m == GroupMode::kScaledWide ? 8 : 4; }
__host__ __device__ constexpr int group_threads(GroupMode m) {
  return 64 + 32 * group_epilogue_warps(m) + (m == GroupMode::kWeightGrad ? 32 : 0);
}
__host__ __device__ constexpr int group_tmem_bufs(GroupMode m) { return m == GroupMode::kScaledStream ? 8 : 2; }

struct GroupedMaps {
  CUtensorMap l;
  CUtensorMap r[4];  // R boxes of 128, 64, 32 and 16 rows (kWeightGrad: r[0], 64 x 64)
};

struct GroupedArgs {
  const int32_t* ends;  // [groups]; null: one group of all rows
  int groups;
  int rows;             // T
  int cols;             // columns of the output
  int lrows;            // kWeightGrad: rows of one group's output
  int k_blocks;         // K blocks of a tile (kWeightGrad: by group)
  int width_cap;        // rows on the R side: most of them in a tile (a multiple of 32)
  int stages;
  int r_bytes;          // bytes of the R operand's part of a stage
  int pairs;            // CTA pairs launched
  int min_blocks;       // iterations a share has at least
  int vec;              // output rows allow 32-byte stores
  int* status;
  void* out;            // [rows, cols], or [groups, lrows, cols], contiguous
  float* partials;      // [pairs][2 pieces][2 CTAs][piece_floats]
  int piece_floats;
  const float* row_scales;  // sa: strides below, in elements
  int64_t rs_row, rs_k;
  const float* tile_scales;  // sb
  int64_t ts_group, ts_n, ts_k;
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Width of a group's tiles when its rows are on the R side: equal parts of at most `cap`, rounded
// up to the UMMA's step of 32.
__host__ __device__ inline int group_width(int rows, int cap) {
  const int tiles = ceil_div(rows, cap);
  return ceil_div(ceil_div(rows, tiles), 32) * 32;
}

// Index among the R boxes (128, 64, 32, 16 rows) of the smallest that holds half a tile's width.
__host__ __device__ inline int group_box(int half) { return half > 64 ? 0 : (half > 32 ? 1 : (half > 16 ? 2 : 3)); }

template <GroupMode MODE>
__host__ __device__ inline int group_row_tiles(const GroupedArgs& a, int rows) {
  if (rows <= 0) return 0;
  if (group_rows_on_r(MODE)) return ceil_div(rows, group_width(rows, a.width_cap));
  return ceil_div(MODE == GroupMode::kWeightGrad ? a.lrows : rows, 256);
}

template <GroupMode MODE>
__host__ __device__ inline int group_blocks(const GroupedArgs& a, int rows) {
  return MODE == GroupMode::kWeightGrad ? ceil_div(rows, 64) : a.k_blocks;
}

template <GroupMode MODE>
__host__ __device__ inline int group_iterations(const GroupedArgs& a, int rows) {
  return group_row_tiles<MODE>(a, rows) * ceil_div(a.cols, 256) * group_blocks<MODE>(a, rows);
}

// start[e]: first row of group e; base[e]: first iteration of group e; both with an entry past the
// last group. Ends are taken as they would be if clamped to [previous end, rows], so no value of
// `ends` leads out of the matrices. One warp.
template <GroupMode MODE>
__device__ inline void build_group_table(const GroupedArgs& a, int* start, int* base) {
  const int lane = static_cast<int>(lane_id());
  int row = 0, it = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    int end = 0;
    if (g < a.groups) end = a.ends == nullptr ? a.rows : min(max(a.ends[g], 0), a.rows);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end = max(end, o);
    }
    end = max(end, row);
    int begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = row;
    const int its = g < a.groups ? group_iterations<MODE>(a, end - begin) : 0;
    int sum = its;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (g < a.groups) {
      start[g] = begin;
      base[g] = it + sum - its;
    }
    row = __shfl_sync(0xffffffffu, end, 31);
    it += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) {
    start[a.groups] = row;
    base[a.groups] = it;
  }
}

// Pairs that get a share, and the first iteration of share p.
__device__ inline int group_shares(const GroupedArgs& a, int total) {
  return max(1, min(a.pairs, total / a.min_blocks));
}
__device__ inline int share_begin(int total, int shares, int p) {
  return static_cast<int>(int64_t(total) * p / shares);
}

// One run of K blocks of one tile.
struct GroupSegment {
  int group;
  int row0, row_end;  // the group's rows
  int l0, r0;         // first L row / R column of the tile (row side: rows of the whole matrix)
  int width;          // R columns the UMMA takes
  int kb0, kb1, blocks;
  bool first;         // the share's first segment
};

// Tile `q` of group `e`: where it lies.
template <GroupMode MODE>
__device__ inline void group_tile(const GroupedArgs& a, const int* start, int e, int q, GroupSegment& s) {
  s.group = e;
  s.row0 = start[e];
  s.row_end = start[e + 1];
  const int rows = s.row_end - s.row0;
  const int row_tiles = group_row_tiles<MODE>(a, rows);
  int pr, pc;
  grouped_tile(q, row_tiles, ceil_div(a.cols, 256), kGroupRaster, pr, pc);
  if (group_rows_on_r(MODE)) {
    s.width = group_width(rows, a.width_cap);
    s.r0 = s.row0 + pr * s.width;
    s.l0 = pc * 256;
  } else {
    s.l0 = (MODE == GroupMode::kWeightGrad ? 0 : s.row0) + pr * 256;
    s.r0 = pc * 256;
    s.width = a.cols - s.r0 <= 128 ? 128 : 256;
  }
}

template <GroupMode MODE>
struct GroupWalk {
  int it, lo, hi, e;
  __device__ GroupWalk(const GroupedArgs& a, const int* base, int pair) {
    const int total = base[a.groups];
    const int shares = group_shares(a, total);
    lo = pair < shares ? share_begin(total, shares, pair) : total;
    hi = pair < shares ? share_begin(total, shares, pair + 1) : total;
    it = lo;
    e = 0;
    int top = a.groups - 1;  // last group whose base is <= lo
    while (e < top) {
      const int mid = (e + top + 1) >> 1;
      if (base[mid] <= lo) {
        e = mid;
      } else {
        top = mid - 1;
      }
    }
  }
  __device__ bool next(const GroupedArgs& a, const int* start, const int* base, GroupSegment& s) {
    if (it >= hi) return false;
    while (it >= base[e + 1]) ++e;  // past groups without rows
    const int blocks = group_blocks<MODE>(a, start[e + 1] - start[e]);
    const int q = (it - base[e]) / blocks;
    group_tile<MODE>(a, start, e, q, s);
    s.blocks = blocks;
    s.kb0 = it - base[e] - q * blocks;
    s.kb1 = min(blocks, s.kb0 + hi - it);
    s.first = it == lo;
    it += s.kb1 - s.kb0;
    return true;
  }
};

__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster_addr,
                                                 int32_t x, int32_t y, int32_t z, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}

// D (TMEM of both CTAs) (+)= A * B, E4M3 inputs, FP32 accumulator. Issued by one thread of the leader.
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Lets the finish kernel launch as soon as every CTA of this grid runs; it waits for the grid's
// memory itself.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// acc (two FP32 values) += p * s, both halves by the same pair of scales.
__device__ __forceinline__ void fma_f32x2(uint64_t& acc, uint64_t p, uint64_t s) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(p), "l"(s));
}
__device__ __forceinline__ uint64_t pack_b32x2(uint32_t lo, uint32_t hi) {
  return static_cast<uint64_t>(hi) << 32 | lo;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <typename T>
__device__ __forceinline__ uint32_t pack_f32(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_f32<__half>(float lo, float hi) {
  return pack_half2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack_f32<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// One warp's lanes are 32 consecutive output columns, v[j] the value of row `row + j`: 2-byte
// stores, 64 consecutive bytes per row and warp.
template <typename T, int N>
__device__ __forceinline__ void store_rows_across(T* out, int64_t ldo, const float (&v)[N], int row, int row_end,
                                                  int col, int cols) {
  if (col >= cols) return;
  T* p = out + static_cast<int64_t>(row) * ldo + col;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (row + j < row_end) p[static_cast<int64_t>(j) * ldo] = from_f32<T>(v[j]);
  }
}

// One lane's 16 consecutive output columns of its own row (32 bytes).
template <typename T>
__device__ __forceinline__ void store_cols_16(T* p, const float (&v)[16], int left, bool vec) {
  if (vec && left >= 16) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p),
                 "r"(pack_f32<T>(v[0], v[1])), "r"(pack_f32<T>(v[2], v[3])), "r"(pack_f32<T>(v[4], v[5])),
                 "r"(pack_f32<T>(v[6], v[7])), "r"(pack_f32<T>(v[8], v[9])), "r"(pack_f32<T>(v[10], v[11])),
                 "r"(pack_f32<T>(v[12], v[13])), "r"(pack_f32<T>(v[14], v[15]))
                 : "memory");
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (j < left) p[j] = from_f32<T>(v[j]);
    }
  }
}

template <GroupMode MODE>
struct GroupedShape {
  static constexpr int kBarriers = 3 * kMaxStages + 2 * 8 + 1;
  static constexpr int kBarrierBytes = kBarriers * 8 + 16;
  __host__ __device__ static constexpr int stage_bytes(int r_bytes) { return kGroupLBytes + r_bytes; }
  __host__ __device__ static constexpr int smem_bytes(int stages, int r_bytes, int groups) {
    return 1024 + stages * stage_bytes(r_bytes) + kBarrierBytes + (groups + 1) * 8;
  }
};

// L_MN: the L operand's rows are its contiguous dimension (kForward with W [E, K, N] row-major, and
// kWeightGrad); otherwise K is.
template <GroupMode MODE, bool L_MN, typename T>
__global__ void __launch_bounds__(group_threads(MODE), 1)
    grouped_gemm_kernel(const __grid_constant__ GroupedMaps maps, const __grid_constant__ GroupedArgs args) {
  using S = GroupedShape<MODE>;
  constexpr bool kScaled = group_scaled(MODE);
  constexpr bool kGrad = MODE == GroupMode::kWeightGrad;
  constexpr int kEpilogueWarps = group_epilogue_warps(MODE);
  constexpr int kBufs = group_tmem_bufs(MODE);
  constexpr int kBufCols = 512 / kBufs;
  constexpr int kSteps = 4;                       // UMMA K steps of a block: 128 bytes of K
  constexpr int kBlockK = kScaled ? 128 : 64;     // K values of a block
  constexpr bool kBf16 = sizeof(T) == 2 && !kScaled && std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescBase = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (L_MN ? 1u << 15 : 0u) |
                                  (kGrad ? 1u << 16 : 0u) | ((256u >> 4) << 24);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = args.stages;
  const int stage_bytes = S::stage_bytes(args.r_bytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + stages * stage_bytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tail_full = empty + kMaxStages;  // kWeightGrad: this CTA's own part of a block to be masked
  uint64_t* tmem_full = tail_full + kMaxStages;
  uint64_t* tmem_empty = tmem_full + 8;
  uint64_t* mma_done = tmem_empty + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 4);
  int* base = start + args.groups + 1;

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(cluster_id_x());

  launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], kGrad ? 2 : 1);  // kWeightGrad: both CTAs report each stage
      mbar_init(&empty[s], 1);
      mbar_init(&tail_full[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&tmem_full[b], 1);
      mbar_init(&tmem_empty[b], 2 * kEpilogueWarps);  // the epilogue warps of both CTAs (leader's copy)
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_map(&maps.l);
    for (int i = 0; i < (kGrad ? 1 : 4); ++i) tma_prefetch_map(&maps.r[i]);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  if (warp == 2) build_group_table<MODE>(args, start, base);
  tc_fence_before_sync();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    const uint64_t policy = l2_policy_evict_normal();
    int stage = 0;
    uint32_t phase = 0;
    uint32_t armed_mask = 0, armed_parity = 0;  // stages this thread has armed (leader)
    uint32_t tail_mask = 0, tail_parity = 0;    // tail barriers used; parity of their next use
    bool ok = true;
    GroupWalk<MODE> walk(args, base, pair);
    GroupSegment s;
    while (ok && walk.next(args, start, base, s)) {
      const int half = s.width / 2;
      const int box = kGrad ? 0 : group_box(half);
      const uint32_t r_bytes = kGrad ? static_cast<uint32_t>(half) * 128u : (128u >> box) * 128u;
      const int tail = kGrad ? (s.row_end - s.row0) - (s.blocks - 1) * 64 : 0;
      const int l0 = s.l0 + static_cast<int>(rank) * 128;
      const int r0 = s.r0 + static_cast<int>(rank) * half;
      for (int kb = s.kb0; kb < s.kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) {
          raise_abort(args.status, abort_flag, kStatusProducerTimeout);
          ok = false;
          break;
        }
        uint8_t* l_dst = ring + stage * stage_bytes;
        uint8_t* r_dst = l_dst + kGroupLBytes;
        const uint32_t leader_full = map_to_rank(smem_addr(&full[stage]), 0);
        if (kGrad && kb == s.blocks - 1 && (tail & 15) != 0) {
          // The group's last rows: into this CTA's own barrier, for the masking warp.
          mbar_arrive_expect_tx(&tail_full[stage], kGroupLBytes + r_bytes);
          tail_mask |= 1u << stage;
          tail_parity ^= 1u << stage;
          armed_mask &= ~(1u << stage);
          const int y = s.row0 + kb * 64;
          for (int i = 0; i < 2; ++i) tma_load_2d(l_dst + i * 8192, &maps.l, &tail_full[stage], l0 + 64 * i, y, policy);
          for (int i = 0; i < half / 64; ++i) {
            tma_load_2d(r_dst + i * 8192, &maps.r[0], &tail_full[stage], r0 + 64 * i, y, policy);
          }
        } else {
          if (rank == 0) {
            mbar_arrive_expect_tx(&full[stage], 2 * (kGroupLBytes + r_bytes));
            armed_mask |= 1u << stage;
            armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
          } else if (kGrad) {
            mbar_arrive_cluster(leader_full);
          }
          if constexpr (kGrad) {
            const int y = s.row0 + kb * 64;
            for (int i = 0; i < 2; ++i) tma_load_2d_pair(l_dst + i * 8192, &maps.l, leader_full, l0 + 64 * i, y, policy);
            for (int i = 0; i < half / 64; ++i) {
              tma_load_2d_pair(r_dst + i * 8192, &maps.r[0], leader_full, r0 + 64 * i, y, policy);
            }
          } else {
            const int k0 = kb * kBlockK;
            if constexpr (MODE == GroupMode::kScaledWide) {
              tma_load_2d_pair(l_dst, &maps.l, leader_full, k0, l0, policy);
              tma_load_3d_pair(r_dst, &maps.r[box], leader_full, k0, r0, s.group, policy);
            } else {
              if constexpr (L_MN) {
                for (int i = 0; i < 2; ++i) {
                  tma_load_3d_pair(l_dst + i * 8192, &maps.l, leader_full, l0 + 64 * i, k0, s.group, policy);
                }
              } else {
                tma_load_3d_pair(l_dst, &maps.l, leader_full, k0, l0, s.group, policy);
              }
              tma_load_2d_pair(r_dst, &maps.r[box], leader_full, k0, r0, policy);
            }
          }
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {  // drain the copies in flight before the pair can exit
      for (int st = 0; st < stages; ++st) {
        if (rank == 0 && (armed_mask & (1u << st)) &&
            !mbar_wait(&full[st], (armed_parity >> st) & 1u, nullptr, 200000000ull)) {
          atomicOr(args.status, kStatusDrainTimeout);
        }
        if ((tail_mask & (1u << st)) &&
            !mbar_wait(&tail_full[st], ((tail_parity >> st) & 1u) ^ 1u, nullptr, 200000000ull)) {
          atomicOr(args.status, kStatusDrainTimeout);
        }
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------- UMMA issuer (leader only) ----------------
    int stage = 0;
    uint32_t phase = 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    const uint64_t l_desc0 = smem_desc(smem_addr(ring), L_MN ? 8192 : 16, 1024);
    const uint64_t r_desc0 = smem_desc(smem_addr(ring) + kGroupLBytes, kGrad ? 8192 : 16, 1024);
    constexpr uint32_t kLStep = (L_MN ? 2048 : 32) >> 4, kRStep = (kGrad ? 2048 : 32) >> 4;
    GroupWalk<MODE> walk(args, base, pair);
    GroupSegment s;
    while (ok && walk.next(args, start, base, s)) {
      const uint32_t idesc = kIdescBase | (static_cast<uint32_t>(s.width >> 3) << 17);
      const int tail = kGrad ? (s.row_end - s.row0) - (s.blocks - 1) * 64 : 0;
      for (int kb = s.kb0; kb < s.kb1; ++kb) {
        if (kScaled || kb == s.kb0) {
          if (!mbar_wait(&tmem_empty[buf], buf_phase ^ 1u, abort_flag)) {
            raise_abort(args.status, abort_flag, kStatusMmaTimeout);
            ok = false;
            break;
          }
          tc_fence_after_sync();
        }
        // kWeightGrad: the peer's masking warp wrote its shared memory (cluster-scope acquire).
        if (!(kGrad ? mbar_wait_cluster(&full[stage], phase, abort_flag) : mbar_wait(&full[stage], phase, abort_flag))) {
          raise_abort(args.status, abort_flag, kStatusMmaTimeout);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint64_t off = static_cast<uint64_t>(stage * (stage_bytes >> 4));
        const int steps = kGrad && kb == s.blocks - 1 ? (tail + 15) / 16 : kSteps;
        const uint32_t d = tmem_base + static_cast<uint32_t>(buf * kBufCols);
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
          if (kk < steps) {
            const uint32_t accumulate = kScaled ? (kk != 0) : (kb != s.kb0 || kk != 0);
            if constexpr (kScaled) {
              umma_f8_pair(d, l_desc0 + off + kk * kLStep, r_desc0 + off + kk * kRStep, idesc, accumulate);
            } else {
              umma_f16_pair(d, l_desc0 + off + kk * kLStep, r_desc0 + off + kk * kRStep, idesc, accumulate);
            }
          }
        }
        umma_commit_pair_multicast(smem_addr(&empty[stage]), 3);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (kScaled || kb + 1 == s.kb1) {
          umma_commit_pair_multicast(smem_addr(&tmem_full[buf]), 3);
          if (++buf == kBufs) {
            buf = 0;
            buf_phase ^= 1u;
          }
        }
      }
    }
    umma_commit_pair(smem_addr(mma_done));
    if (!mbar_wait(mma_done, 0, nullptr, 200000000ull)) atomicOr(args.status, kStatusDrainTimeout);
  } else if (kGrad && warp == 6) {
    // ---------------- masking warp (both CTAs): rows past the group in its last block ----------
    int stage = 0;
    uint32_t parity = 0;  // bit s: parity of the next use of tail_full[s]
    GroupWalk<MODE> walk(args, base, pair);
    GroupSegment s;
    bool ok = true;
    while (ok && walk.next(args, start, base, s)) {
      const int blocks = s.kb1 - s.kb0;
      const int tail = (s.row_end - s.row0) - (s.blocks - 1) * 64;
      if (s.kb1 == s.blocks && (tail & 15) != 0) {
        const int st = (stage + blocks - 1) % stages;
        ok = __all_sync(0xffffffffu, mbar_wait(&tail_full[st], (parity >> st) & 1u, abort_flag));
        if (!ok) {
          if (lane == 0) raise_abort(args.status, abort_flag, kStatusEpilogueTimeout);
          break;
        }
        parity ^= 1u << st;
        // A box is 64 rows of 128 bytes; the swizzle moves 16-byte chunks within a row only.
        const int from = tail, count = ((tail + 15) & ~15) - tail;
        const int boxes = 2 + s.width / 128;
        const uint32_t st_addr = smem_addr(ring + st * stage_bytes);
        for (int i = static_cast<int>(lane); i < boxes * count * 8; i += 32) {
          const int chunk = i & 7, r = (i >> 3) % count, b = (i >> 3) / count;
          st_shared_v4(st_addr + b * 8192 + (from + r) * 128 + chunk * 16, 0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_addr(&full[st]), 0));
      }
      stage = (stage + blocks) % stages;
    }
  } else if (warp >= 2 && warp < 2 + kEpilogueWarps) {
    // ---------------- epilogue (both CTAs, own 128 TMEM lanes) ----------------
    const int quarter = warp & 3;
    const int row = quarter * 32 + static_cast<int>(lane);  // TMEM lane
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    T* out = static_cast<T*>(args.out);
    int buf = 0;
    uint32_t buf_phase = 0;
    auto wait_buf = [&]() {
      const bool ready = __all_sync(0xffffffffu, mbar_wait(&tmem_full[buf], buf_phase, abort_flag));
      if (!ready && lane == 0) raise_abort(args.status, abort_flag, kStatusEpilogueTimeout);
      if (ready) tc_fence_after_sync();
      return ready;
    };
    auto release_buf = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) {
          mbar_arrive_relaxed(&tmem_empty[buf]);
        } else {
          mbar_arrive_cluster_relaxed(map_to_rank(smem_addr(&tmem_empty[buf]), 0));
        }
      }
      if (++buf == kBufs) {
        buf = 0;
        buf_phase ^= 1u;
      }
    };
    auto piece_of = [&](const GroupSegment& s) {
      return args.partials +
             (static_cast<size_t>(pair * 2 + (s.first ? 0 : 1)) * 2 + rank) * static_cast<size_t>(args.piece_floats);
    };
    GroupWalk<MODE> walk(args, base, pair);
    GroupSegment s;
    if constexpr (!kScaled) {
      while (walk.next(args, start, base, s)) {
        if (!wait_buf()) break;
        const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols);
        const int l = s.l0 + static_cast<int>(rank) * 128 + row;
        const bool whole = s.kb0 == 0 && s.kb1 == s.blocks;
#pragma unroll 1
        for (int c = 0; c < s.width; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + c, v);
          tmem_ld_wait();
          if (!whole) {
            float* dst = piece_of(s) + (static_cast<size_t>(c / 4) * 128 + row) * 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              st_global_v4(dst + static_cast<size_t>(j) * 512, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
          } else if constexpr (kGrad) {
            if (l < args.lrows) {
              T* p = out + (static_cast<int64_t>(s.group) * args.lrows + l) * args.cols + s.r0 + c;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float f[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(v[16 * h + j]);
                store_cols_16(p + 16 * h, f, args.cols - (s.r0 + c + 16 * h), args.vec != 0);
              }
            }
          } else {
            float f[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
            store_rows_across(out, args.cols, f, s.r0 + c, min(s.row_end, s.r0 + s.width), l, args.cols);
          }
        }
        release_buf();
      }
    } else if constexpr (MODE == GroupMode::kScaledWide) {
      const int half = (warp - 2) / 4;  // 128 of the tile's 256 columns
      while (walk.next(args, start, base, s)) {
        const int t = s.l0 + static_cast<int>(rank) * 128 + row;
        const bool live = half * 128 < s.width && s.r0 + half * 128 < args.cols;
        const float* sa = args.row_scales + static_cast<int64_t>(min(t, args.rows - 1)) * args.rs_row;
        const float* sb = args.tile_scales + s.group * args.ts_group + ((s.r0 >> 7) + (live ? half : 0)) * args.ts_n;
        uint64_t acc[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = 0;
        float scale = sa[s.kb0 * args.rs_k] * sb[s.kb0 * args.ts_k];
        bool ready = true;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          const int ahead = min(kb + 1, s.kb1 - 1);
          const float next_a = sa[ahead * args.rs_k], next_b = sb[ahead * args.ts_k];
          ready = wait_buf();
          if (!ready) break;
          if (live) {
            const uint64_t scale2 = pack_b32x2(__float_as_uint(scale), __float_as_uint(scale));
            const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols + half * 128);
            uint32_t v[2][16];
            tmem_ld_32x32b_x16(taddr, v[0]);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              tmem_ld_wait();
              tmem_ld_fence_regs(v[c & 1]);
              if (c < 7) tmem_ld_32x32b_x16(taddr + (c + 1) * 16, v[(c + 1) & 1]);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                fma_f32x2(acc[8 * c + j], pack_b32x2(v[c & 1][2 * j], v[c & 1][2 * j + 1]), scale2);
              }
            }
          }
          release_buf();
          scale = next_a * next_b;
        }
        if (!ready) break;
        if (!live) continue;
        if (s.kb0 == 0 && s.kb1 == s.blocks) {
          if (t < s.row_end) {
            T* p = out + static_cast<int64_t>(t) * args.cols + s.r0 + half * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              float f[16];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                f[2 * j] = __uint_as_float(static_cast<uint32_t>(acc[8 * c + j]));
                f[2 * j + 1] = __uint_as_float(static_cast<uint32_t>(acc[8 * c + j] >> 32));
              }
              store_cols_16(p + 16 * c, f, args.cols - (s.r0 + half * 128 + 16 * c), args.vec != 0);
            }
          }
        } else {
          float* dst = piece_of(s) + (static_cast<size_t>(half * 32) * 128 + row) * 4;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            st_global_v4(dst + static_cast<size_t>(j) * 512, static_cast<uint32_t>(acc[2 * j]),
                         static_cast<uint32_t>(acc[2 * j] >> 32), static_cast<uint32_t>(acc[2 * j + 1]),
                         static_cast<uint32_t>(acc[2 * j + 1] >> 32));
          }
        }
      }
    } else {
      while (walk.next(args, start, base, s)) {
        const int l = s.l0 + static_cast<int>(rank) * 128 + row;
        const int valid = min(s.row_end - s.r0, s.width);  // rows of the tile
        // This CTA's 128 output columns share one weight scale per block.
        const int nb = min((s.l0 >> 7) + static_cast<int>(rank), (args.cols - 1) >> 7);
        const float* sb = args.tile_scales + s.group * args.ts_group + nb * args.ts_n;
        // Lane j holds the scales of rows j and j + 32.
        const float* sa0 = args.row_scales + static_cast<int64_t>(min(s.r0 + static_cast<int>(lane), args.rows - 1)) * args.rs_row;
        const float* sa1 =
            args.row_scales + static_cast<int64_t>(min(s.r0 + 32 + static_cast<int>(lane), args.rows - 1)) * args.rs_row;
        float acc[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = 0.f;
        float a0 = sa0[s.kb0 * args.rs_k], a1 = sa1[s.kb0 * args.rs_k], b = sb[s.kb0 * args.ts_k];
        bool ready = true;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          const int ahead = min(kb + 1, s.kb1 - 1);
          const float next_a0 = sa0[ahead * args.rs_k], next_a1 = sa1[ahead * args.rs_k], next_b = sb[ahead * args.ts_k];
          ready = wait_buf();
          if (!ready) break;
          const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols);
          const float s0 = a0 * b, s1 = a1 * b;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c * 16 < valid) {  // warp-uniform
              uint32_t v[16];
              tmem_ld_32x32b_x16(taddr + c * 16, v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float sc = __shfl_sync(0xffffffffu, c < 2 ? s0 : s1, (c & 1) * 16 + j);
                acc[16 * c + j] = fmaf(__uint_as_float(v[j]), sc, acc[16 * c + j]);
              }
            }
          }
          release_buf();
          a0 = next_a0;
          a1 = next_a1;
          b = next_b;
        }
        if (!ready) break;
        if (s.kb0 == 0 && s.kb1 == s.blocks) {
          store_rows_across(out, args.cols, acc, s.r0, s.r0 + valid, l, args.cols);
        } else {
          float* dst = piece_of(s) + static_cast<size_t>(row) * 4;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (4 * j < s.width) {
              st_global_v4(dst + static_cast<size_t>(j) * 512, __float_as_uint(acc[4 * j]), __float_as_uint(acc[4 * j + 1]),
                           __float_as_uint(acc[4 * j + 2]), __float_as_uint(acc[4 * j + 3]));
            }
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  cluster_sync();  // the leader's UMMAs read the peer's shared memory until here
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

constexpr int kFinishThreads = 128;
constexpr int kFinishChunks = 4;  // blocks along a piece's columns

// Joins the tiles that shares cut: block (p, CTA half, chunk) takes the tile in which share p + 1
// begins, if that is the first share to begin inside it, and adds its FP32 pieces in K order. Then
// all blocks write the zeros nobody else writes.
template <GroupMode MODE, typename T>
__global__ void __launch_bounds__(kFinishThreads) grouped_finish_kernel(const __grid_constant__ GroupedArgs args) {
  extern __shared__ int finish_table[];
  int* start = finish_table;
  int* base = start + args.groups + 1;
  if (threadIdx.x < 32) build_group_table<MODE>(args, start, base);
  __syncthreads();
  wait_for_primary();
  T* out = static_cast<T*>(args.out);
  const int total = base[args.groups];
  const int shares = group_shares(args, total);
  const int p = static_cast<int>(blockIdx.x) + 1;
  const int rank = static_cast<int>(blockIdx.y);
  if (p < shares) {
    const int cut = share_begin(total, shares, p);
    int e = 0;
    while (cut >= base[e + 1]) ++e;
    const int blocks = group_blocks<MODE>(args, start[e + 1] - start[e]);
    const int q = (cut - base[e]) / blocks;
    const int tile_begin = base[e] + q * blocks;
    const int tile_end = tile_begin + blocks;
    const int before = share_begin(total, shares, p - 1);
    if (cut > tile_begin && before <= tile_begin) {
      GroupSegment s;
      group_tile<MODE>(args, start, e, q, s);
      const int row = static_cast<int>(threadIdx.x);
      for (int c = static_cast<int>(blockIdx.z) * 4; c < s.width; c += kFinishChunks * 4) {
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int o = p - 1; o < shares && share_begin(total, shares, o) < tile_end; ++o) {
          const int piece = share_begin(total, shares, o) >= tile_begin ? 0 : 1;
          const float* src = args.partials +
                             (static_cast<size_t>(o * 2 + piece) * 2 + rank) * static_cast<size_t>(args.piece_floats) +
                             (static_cast<size_t>(c / 4) * 128 + row) * 4;
          const float4 v = *reinterpret_cast<const float4*>(src);
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        const int l = s.l0 + rank * 128 + row;
        if constexpr (group_rows_on_r(MODE)) {
          store_rows_across(out, args.cols, v, s.r0 + c, min(s.row_end, s.r0 + s.width), l, args.cols);
        } else {
          const bool inside = MODE == GroupMode::kWeightGrad ? l < args.lrows : l < s.row_end;
          const int64_t line = MODE == GroupMode::kWeightGrad ? static_cast<int64_t>(e) * args.lrows + l : l;
          if (inside) {
            for (int j = 0; j < 4; ++j) {
              if (s.r0 + c + j < args.cols) out[line * args.cols + s.r0 + c + j] = from_f32<T>(v[j]);
            }
          }
        }
      }
    }
  }
  // Zeros: rows past the last group, or the outputs of groups without rows.
  const int64_t step = static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z * kFinishThreads;
  const int64_t mine =
      ((static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * kFinishThreads + threadIdx.x;
  auto zero = [&](T* p, int64_t count) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && count % 8 == 0) {
      for (int64_t i = mine; i < count / 8; i += step) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
    } else {
      for (int64_t i = mine; i < count; i += step) p[i] = from_f32<T>(0.f);
    }
  };
  if constexpr (MODE == GroupMode::kWeightGrad) {
    const int64_t size = static_cast<int64_t>(args.lrows) * args.cols;
    for (int g = 0; g < args.groups; ++g) {
      if (start[g + 1] == start[g]) zero(out + g * size, size);
    }
  } else {
    const int64_t from = start[args.groups];
    if (from < args.rows) zero(out + from * args.cols, (args.rows - from) * args.cols);
  }
}

}  // namespace hst
