// Matrix products over rows grouped by expert, on CTA pairs (tcgen05.mma.cta_group::2).
//
// Group e owns rows [ends[e - 1], ends[e]) of a row matrix; `ends` lives on the GPU, so nothing
// about the sizes is known on the host. Three products, in four forms, share this kernel:
//   kForward     y[t, :] = x[t, :] W[e(t)]           16-bit x [T, K], W [E, K, N] (either of its two
//                                                    inner dimensions contiguous)
//   kWeightGrad  D[e] = L[rows of e]^T R[rows of e]   16-bit L [T, Lc], R [T, Rc]
//   kScaled and  y[t, n] = sum_b sa[t, b] sb[e, n/128, b] sum_{k in block b} a[t, k] b[e, n, k]
//   kScaledFew                                       E4M3 a [T, K], b [E, N, K], FP32 scales of 128
//                                                    (a) and 128 x 128 (b) values
//
// One pair of CTAs computes a 256 x width tile: CTA r owns 128 rows of the L operand and half of
// the R operand's `width` columns. Each weight is read once for up to 256 rows, so few rows a group
// are bound by HBM, many by the tensor cores.
//   * kForward puts the weights on the L side (M = 256 output columns) and the rows on the R side,
//     whose width is a run-time field of the UMMA descriptor (32..256): a group's rows, rounded up to
//     a multiple of 32, are cut into widths that differ by at most one 32, so raggedness costs up to
//     31 columns of tensor-core time a group instead of the next multiple of 256.
//   * kWeightGrad reduces over the rows, 64 at a time. Rows past the group's end in its last block
//     belong to other groups: one more warp zeroes those of the last 16-row UMMA step in shared
//     memory (both operands, so that NaN or infinity there stays out), and the steps past them are
//     not issued.
//   * kScaled accumulates each 128-deep block in a TMEM buffer of its own; the epilogue warps read
//     it, multiply by the block's scales and add it to FP32 registers, while the next block's UMMAs
//     fill the other buffer. The rows are on the L side, where a row is a TMEM lane and its scale one
//     register: on the R side the scales of 256 rows are 128 a thread and block, and their broadcast
//     loads from shared memory, beside the UMMAs' operands, took three times the UMMAs' time. Bound now
//     by the way of a block through the two buffers (UMMAs 512 cycles, hand-over, 128 columns a thread
//     read and added, hand-back): 8192 x 14336 x 4096 in 481 us, 350 without the reading and adding.
//   * kScaledFew is for few rows a group: as kForward, weights on the L side and at most 64 rows on
//     the R side, in eight TMEM buffers. A block then costs 64 to 128 UMMA cycles instead of 512 and
//     keeps all lanes busy, and the weights stream at the rate of HBM.
//
// Schedule: all (tile, K block) iterations of all groups in one line, cut into one equal share per
// pair (GroupTable). A tile cut by a share's end leaves FP32 pieces in the workspace, which a second
// small kernel (grouped_finish_kernel, a programmatic dependent) adds in K order. Where ending the
// shares at tiles idles the last pairs for a few K blocks only (GroupedArgs::idle_limit), they end there
// instead: writing, reading and adding the pieces costs more (8192 x 2048 x 2048 over 16 groups: 72 us
// cut, 63 whole; 421 x 520 x 1000 over 8: 16 and 10).
// No CTA ever waits for another pair, no atomics: results are bitwise reproducible, and the kernels can
// be captured and replayed. Whichever kernel is last also writes the zeros of rows past the last group
// and of the weight gradients of empty groups.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "gemm_tile.cuh"
#include "ptx.cuh"

namespace hst {

enum class GroupMode { kForward, kWeightGrad, kScaled, kScaledFew };
__host__ __device__ constexpr bool group_scaled(GroupMode m) { return m == GroupMode::kScaled || m == GroupMode::kScaledFew; }
// The rows are on the R side.
__host__ __device__ constexpr bool group_rows_right(GroupMode m) { return m == GroupMode::kForward || m == GroupMode::kScaledFew; }

constexpr int kMaxGroups = 1024;
constexpr int kGroupLBytes = 16384;  // 128 L rows x 128 bytes of K (or 2 boxes of 64 x 64)
constexpr int kGroupRaster = 8;      // row tiles before the next column tile

// Warps: 0 loads, 1 issues the UMMAs; then the epilogue, and for kWeightGrad the masking warp. kScaled
// holds 128 x 256 FP32 sums in the registers of 8 epilogue warps, which therefore form warpgroups of
// their own (2 and 3 idle); kWeightGrad has 8 because a group of few
// rows is little but epilogue (32 groups of 64 rows, 2048 x 2816: 102 us against 108 with four).
__host__ __device__ constexpr int group_first_epilogue_warp(GroupMode m) { return m == GroupMode::kScaled ? 4 : 2; }
__host__ __device__ constexpr int group_epilogue_warps(GroupMode m) { return m == GroupMode::kScaled || m == GroupMode::kWeightGrad ? 8 : 4; }
__host__ __device__ constexpr int group_threads(GroupMode m) {
  return 32 * (group_first_epilogue_warp(m) + group_epilogue_warps(m) + (m == GroupMode::kWeightGrad ? 1 : 0));
}

// Boxes of 128, 64, 32 and 16 rows on the side that has the rows (kForward, kScaledFew: R; kScaled: L), else one in
// [0] (kScaled's R: 128 rows and, in [1], 64; kWeightGrad: 64 x 64).
struct GroupedMaps {
  CUtensorMap l[4];
  CUtensorMap r[4];
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
  int idle_limit;       // shares end at tiles if that idles a pair for at most so many K blocks (GroupTable)
  int whole;            // they do whatever the ends are: no finish kernel follows
  int vec;              // bytes of a store the output rows' alignment allows: 32, 16, 8, 4 or 2
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

// Rows on the R side: units of 32 rows (the UMMA's step) in a group, and tiles of at most `cap` rows.
__host__ __device__ inline int group_units(int rows) { return ceil_div(rows, 32); }
__host__ __device__ inline int group_tiles_right(int rows, int cap) { return ceil_div(group_units(rows), cap / 32); }

// Index among the boxes (128, 64, 32, 16 rows) of the smallest that holds `rows`.
__host__ __device__ inline int group_box(int rows) { return rows > 64 ? 0 : (rows > 32 ? 1 : (rows > 16 ? 2 : 3)); }

template <GroupMode MODE>
__host__ __device__ inline int group_row_tiles(const GroupedArgs& a, int rows) {
  if (rows <= 0) return 0;
  if (group_rows_right(MODE)) return group_tiles_right(rows, a.width_cap);
  return ceil_div(MODE == GroupMode::kWeightGrad ? a.lrows : rows, 256);
}

template <GroupMode MODE>
__host__ __device__ inline int group_blocks(const GroupedArgs& a, int rows) {
  return MODE == GroupMode::kWeightGrad ? ceil_div(rows, 64) : a.k_blocks;
}

// The tiles of all groups, numbered group by group, and how the pairs share them.
//
// kForward and the scaled products (every tile has the same K blocks): the tiles are dealt to `shares`
// columns like cards (tile t * shares + c is number t of column c; the last, part-filled row is spread
// evenly over the columns), the columns are put end to end into one line of (tile, K block)
// iterations, and the line is cut into equal shares (or every pair takes its column, GroupShares). Share
// c then runs along column c, give or take a part of a tile, so at any moment the pairs work on
// neighbouring tiles: with contiguous runs of the group-by-group order instead, the 74 weight panels in
// use passed L2's size (8194 x 14336 x 4096 over 8 groups: 1007 us against 811, before the steps that
// followed).
//
// kWeightGrad (K blocks by group, the same number of tiles in each): of every group with rows, each
// pair takes its tiles / pairs whole tiles, all pairs at the same group at the same time; what remains
// of the groups, put end to end, is the line that is cut into equal shares. (Dealt as above, heavy and
// light columns put the pairs into different groups, whose rows together do not stay in L2: 823 MB
// read from DRAM for 160 MB of operands, 16384 x 2048 x 2816 over 32 ragged groups.)
//
// In shared memory: eight integers (below), then [groups + 1] of first row and three more (below), then
// [pairs + 1] first tile of each column along the line and its first iteration. The view keeps one
// address: the issuing warps have no registers for six.
constexpr int kTableHead = 8;
struct GroupTable {
  int* mem;
  int groups, pairs;

  __device__ int& tiles() const { return mem[0]; }       // kWeightGrad: of the line
  __device__ int& shares() const { return mem[1]; }
  __device__ int& total() const { return mem[2]; }       // iterations of the line
  __device__ int& per_column() const { return mem[3]; }  // tiles / shares
  __device__ int& per_share() const { return mem[4]; }   // total / shares, and what remains
  __device__ int& more_share() const { return mem[5]; }
  __device__ int& used() const { return mem[6]; }        // kWeightGrad: groups with rows
  __device__ int& whole() const { return mem[7]; }       // the shares end at tiles
  __device__ int& start(int e) const { return mem[kTableHead + e]; }
  // First tile of a group, tiles in a column of its output, and the units of 32 rows of its smaller
  // tiles (rows on the R side: the first group_units mod tiles of them have one more).
  __device__ int& tile_base(int e) const { return mem[kTableHead + groups + 1 + e]; }
  __device__ int& row_tiles(int e) const { return mem[kTableHead + 2 * (groups + 1) + e]; }
  __device__ int& units(int e) const { return mem[kTableHead + 3 * (groups + 1) + e]; }
  // kWeightGrad, in their place: the r-th group with rows, and the K blocks of a tile of those before it.
  __device__ int& used_group(int r) const { return tile_base(r); }
  __device__ int& blocks_before(int r) const { return row_tiles(r); }
  __device__ int& col_tile(int c) const { return mem[kTableHead + 4 * (groups + 1) + c]; }
  __device__ int& col_base(int c) const { return mem[kTableHead + 4 * (groups + 1) + pairs + 1 + c]; }

  // Column c gets tiles / shares tiles, and the part-filled row's are spread over the columns.
  __device__ static int column_first(int c, int tiles, int shares) {
    return c * (tiles / shares) + c * (tiles % shares) / shares;
  }
  __device__ int share_begin(int p) const {
    return whole() ? col_base(p) : p * per_share() + min(p, more_share());  // kWeightGrad: never whole here
  }
  // The column of the line's tile v: the last c with column_first(c) = floor(c * tiles / shares) <= v.
  __device__ int column_of(int v) const { return ((v + 1) * shares() - 1) / tiles(); }
  __device__ int tile_of(int c, int t) const {
    const int high = per_column(), wide = shares();
    return t < high ? t * wide + c : high * wide + col_tile(c) - c * high;
  }
  __device__ int group_of(int tile) const {
    int e = 0, top = groups - 1;  // last group whose first tile is <= tile; groups without tiles come before it
    while (e < top) {
      const int mid = (e + top + 1) >> 1;
      if (tile_base(mid) <= tile) {
        e = mid;
      } else {
        top = mid - 1;
      }
    }
    return e;
  }
};

constexpr __host__ __device__ int group_table_ints(int groups, int pairs) {
  return kTableHead + 4 * (groups + 1) + 2 * (pairs + 1);
}

// Tiles of a group's weight gradient, and those each pair takes of it; what is over goes to the line.
struct GradTiles {
  int all, each, over;
  __device__ explicit GradTiles(const GroupedArgs& a) {
    all = ceil_div(a.lrows, 256) * ceil_div(a.cols, 256);
    each = all / a.pairs;
    over = all - each * a.pairs;
  }
};

// How the line is shared: by whole tiles or by K blocks, and among how many pairs (the first ones; the
// others have what precedes the line alone: cut into a share for every pair, the one tile left over of 75 cost
// 4096 rows of 1280 x 3840 137 us, and 68 in shares of at least min_blocks).
struct GroupShares {
  int shares;
  bool whole;
  __host__ __device__ GroupShares(const GroupedArgs& a, int tiles, int total, int deepest) {
    const int by_tiles = at_least_one(a.pairs, tiles);
    const int by_blocks = at_least_one(a.pairs, total / a.min_blocks);
    const int64_t idle = static_cast<int64_t>(ceil_div(tiles, by_tiles)) * deepest - total / by_blocks;
    whole = a.whole != 0 || idle <= a.idle_limit;
    shares = whole ? by_tiles : by_blocks;
  }
  __host__ __device__ static int at_least_one(int pairs, int work) { return work < 1 ? 1 : (work < pairs ? work : pairs); }
};

// Builds the groups' part. Ends are taken as they would be if clamped to [previous end, rows], so no
// value of `ends` leads out of the matrices. One warp; a barrier before the second step.
template <GroupMode MODE>
__device__ inline void build_group_rows(const GroupedArgs& a, const GroupTable& t) {
  constexpr bool kGrad = MODE == GroupMode::kWeightGrad;
  const int lane = static_cast<int>(lane_id());
  const int col_tiles = ceil_div(a.cols, 256);
  int row = 0, tiles = 0, total = 0;  // kGrad: groups with rows, and K blocks of a tile of each
  int deepest = kGrad ? 0 : a.k_blocks;
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
    const int rows = g < a.groups ? end - begin : 0;
    const int high = kGrad ? (rows > 0 ? 1 : 0) : group_row_tiles<MODE>(a, rows);
    const int mine = kGrad ? group_blocks<MODE>(a, rows) : high * col_tiles;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (g < a.groups) t.start(g) = begin;
    if constexpr (kGrad) {
      const uint32_t with_rows = __ballot_sync(0xffffffffu, high != 0);
      if (high != 0) {
        const int r = tiles + __popc(with_rows & ((1u << lane) - 1));
        t.used_group(r) = g;
        t.blocks_before(r) = total + sum - mine;
      }
      tiles += __popc(with_rows);
      deepest = max(deepest, __reduce_max_sync(0xffffffffu, mine));
      total += __shfl_sync(0xffffffffu, sum, 31);
    } else {
      if (g < a.groups) {
        t.tile_base(g) = tiles + sum - mine;
        t.row_tiles(g) = high;
        t.units(g) = group_rows_right(MODE) && high > 0 ? group_units(rows) / high : 0;
      }
      tiles += __shfl_sync(0xffffffffu, sum, 31);
    }
    row = __shfl_sync(0xffffffffu, end, 31);
  }
  if (lane == 0) {
    t.start(a.groups) = row;
    if constexpr (kGrad) {
      const GradTiles n(a);
      t.blocks_before(tiles) = total;
      t.used() = tiles;
      tiles *= n.over;
      total *= n.over;
    } else {
      t.tile_base(a.groups) = tiles;
      total = tiles * a.k_blocks;
    }
    const GroupShares plan(a, tiles, total, deepest);
    const int shares = plan.shares;
    t.whole() = plan.whole;
    t.shares() = shares;
    t.tiles() = tiles;
    t.total() = total;
    t.per_column() = tiles / shares;
    t.per_share() = total / shares;
    t.more_share() = total % shares;
  }
}

// Second step, the columns' part: all threads, and a barrier before the table is used.
template <GroupMode MODE>
__device__ inline void build_group_columns(const GroupedArgs& a, const GroupTable& t) {
  if constexpr (MODE != GroupMode::kWeightGrad) {
    const int shares = t.shares(), tiles = t.tiles();
    for (int c = static_cast<int>(threadIdx.x); c <= shares; c += static_cast<int>(blockDim.x)) {
      const int first = GroupTable::column_first(c, tiles, shares);
      t.col_tile(c) = first;
      t.col_base(c) = first * a.k_blocks;
    }
  }
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

// Tiles of group e, rows on the R side, that have a unit more than the others.
__device__ inline int larger_tiles(const GroupTable& t, int e) {
  return group_units(t.start(e + 1) - t.start(e)) - t.units(e) * t.row_tiles(e);
}

// Width of a tile of group e whose first R column is r0.
template <GroupMode MODE>
__device__ inline int tile_width(const GroupedArgs& a, const GroupTable& t, int e, int r0) {
  if (!group_rows_right(MODE)) return a.cols - r0 <= 128 ? 128 : 256;
  const int units = t.units(e);
  return 32 * (r0 - t.start(e) < 32 * (units + 1) * larger_tiles(t, e) ? units + 1 : units);
}

// First L row and R column of tile `tile` of group `e`.
template <GroupMode MODE>
__device__ inline void tile_origin(const GroupedArgs& a, const GroupTable& t, int e, int tile, int& l0, int& r0) {
  const int row0 = t.start(e);
  const bool grad = MODE == GroupMode::kWeightGrad;  // `tile` counts within the group
  int pr, pc;
  grouped_tile(grad ? tile : tile - t.tile_base(e), grad ? ceil_div(a.lrows, 256) : t.row_tiles(e), ceil_div(a.cols, 256),
               kGroupRaster, pr, pc);
  if (group_rows_right(MODE)) {
    r0 = row0 + 32 * (pr * t.units(e) + min(pr, larger_tiles(t, e)));
    l0 = pc * 256;
  } else {
    l0 = (grad ? 0 : row0) + pr * 256;
    r0 = pc * 256;
  }
}

// The tiles of one share, or of one stretch [lo, hi) of the line, in order, by a whole warp: each lane
// works out one tile of a batch of 32, since a tile's place takes about a dozen divisions (one at a
// time, they cost the UMMA issuer half a microsecond a tile).
template <GroupMode MODE>
struct GroupWalk {
  int lo, hi;
  int v, v_end;    // first tile of the next batch, counted along the line, and the end
  int ahead;       // kWeightGrad: whole tiles still to come before those of the line,
  int done;        // and those behind
  int cur, count;  // the batch's next lane, and the end of its live lanes
  // This lane's tile: its group (negative, ~group, if it begins the stretch), origin and K blocks.
  int group, l0, r0, kb0, kb1;

  // A stretch of the line; `guess`: a column near lo.
  __device__ GroupWalk(const GroupedArgs& a, const GroupTable& t, int lo_, int hi_, int guess)
      : lo(lo_), hi(hi_), v(0), v_end(0), ahead(0), done(0), cur(0), count(0) {
    if (lo >= hi) return;
    if constexpr (MODE == GroupMode::kWeightGrad) {
      const int over = GradTiles(a).over;
      int r = 0, top = t.used() - 1;  // last group with rows that begins at or before lo
      while (r < top) {
        const int mid = (r + top + 1) >> 1;
        if (over * t.blocks_before(mid) <= lo) {
          r = mid;
        } else {
          top = mid - 1;
        }
      }
      v = r * over + (lo - over * t.blocks_before(r)) / (t.blocks_before(r + 1) - t.blocks_before(r));
    } else {
      int c = guess;
      while (t.col_base(c) > lo) --c;
      while (t.col_base(c + 1) <= lo) ++c;
      v = t.col_tile(c) + (lo - t.col_base(c)) / a.k_blocks;
    }
    v_end = t.tiles();
  }
  // The share of `pair`.
  __device__ GroupWalk(const GroupedArgs& a, const GroupTable& t, int pair)
      : GroupWalk(a, t, line_begin(a, t, pair), line_begin(a, t, pair + 1), min(pair, t.shares() - 1)) {
    if constexpr (MODE == GroupMode::kWeightGrad) {
      ahead = t.used() * GradTiles(a).each;
      if (t.whole()) {  // shares of whole tiles
        const int per = t.per_column(), more = t.tiles() - per * t.shares();
        lo = 0;
        hi = t.total();
        v = pair * per + min(pair, more);
        v_end = pair < t.shares() ? v + per + (pair < more ? 1 : 0) : v;
      }
    }
  }
  __device__ static int line_begin(const GroupedArgs& a, const GroupTable& t, int p) {
    if (MODE == GroupMode::kWeightGrad && t.whole()) return 0;
    return p <= t.shares() ? t.share_begin(p) : t.total();
  }

  __device__ void refill(const GroupedArgs& a, const GroupTable& t, int pair) {
    const int lane = static_cast<int>(lane_id());
    bool live = false;
    int e = 0, tile = 0, begin = 0, blocks = 0;
    if constexpr (MODE == GroupMode::kWeightGrad) {
      const GradTiles n(a);
      const int i = done + lane;
      if (i < ahead) {  // whole tiles: number i % each of the pair's in a group
        const int r = i / n.each;
        e = t.used_group(r);
        tile = (i - r * n.each) * a.pairs + pair;
        blocks = group_blocks<MODE>(a, t.start(e + 1) - t.start(e));
        begin = lo;
        live = true;
      } else if (v + i - ahead < v_end) {
        const int at = v + i - ahead, r = at / n.over;
        e = t.used_group(r);
        tile = n.each * a.pairs + at - r * n.over;
        blocks = group_blocks<MODE>(a, t.start(e + 1) - t.start(e));
        begin = n.over * t.blocks_before(r) + (at - r * n.over) * blocks;
        live = begin < hi;
      }
      if (live) {
        const bool line = i >= ahead;
        group = line && begin <= lo ? ~e : e;
        kb0 = line ? max(lo - begin, 0) : 0;
        kb1 = line ? min(blocks, hi - begin) : blocks;
      }
      done += 32;
    } else {
      const int at = v + done + lane;
      if (at < v_end) {
        const int c = t.column_of(at);
        tile = t.tile_of(c, at - t.col_tile(c));
        e = t.group_of(tile);
        blocks = a.k_blocks;
        begin = at * blocks;
        live = begin < hi;
      }
      if (live) {
        group = begin <= lo ? ~e : e;
        kb0 = max(lo - begin, 0);
        kb1 = min(blocks, hi - begin);
      }
      done += 32;
    }
    if (live) tile_origin<MODE>(a, t, e, tile, l0, r0);
    cur = 0;
    count = __popc(__ballot_sync(0xffffffffu, live));  // the live lanes come first
  }

  __device__ bool next(const GroupedArgs& a, const GroupTable& t, int pair, GroupSegment& s) {
    if (cur >= count) {
      if (done > 0 && count < 32) return false;
      refill(a, t, pair);
      if (count == 0) return false;
    }
    const int from = cur++;
    const int g = __shfl_sync(0xffffffffu, group, from);
    s.first = g < 0;
    s.group = s.first ? ~g : g;
    s.l0 = __shfl_sync(0xffffffffu, l0, from);
    s.r0 = __shfl_sync(0xffffffffu, r0, from);
    s.kb0 = __shfl_sync(0xffffffffu, kb0, from);
    s.kb1 = __shfl_sync(0xffffffffu, kb1, from);
    s.row0 = t.start(s.group);
    s.row_end = t.start(s.group + 1);
    s.blocks = group_blocks<MODE>(a, s.row_end - s.row0);
    s.width = tile_width<MODE>(a, t, s.group, s.r0);
    return true;
  }
};

// Forms of the loads and of the barrier arrivals for a whole, converged warp: one elected lane
// performs them. Their operands then come from code all lanes share and stay in uniform registers,
// which TMA takes: from a branch of one lane a load cost about 130 cycles.
__device__ __forceinline__ void elected_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster,
                                                     int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];\n\t}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void elected_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster,
                                                     int32_t x, int32_t y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];\n\t}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y)
      : "memory");
}
// Into this CTA, completing on its own barrier.
__device__ __forceinline__ void elected_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];\n\t}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void elected_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}\n" ::"r"(bar),
      "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void elected_arrive_cluster_relaxed(uint32_t bar_cluster) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}\n" ::"r"(bar_cluster)
      : "memory");
}

// The `steps` (1..4) UMMAs of one K block: D (TMEM of both CTAs) (+)= A * B, operands advancing by
// LSTEP and RSTEP in descriptor units. A whole, converged warp calls it and one elected lane
// issues: with the operands' arithmetic in code all lanes share, it stays in uniform registers,
// which the instruction takes (issued from a branch of one lane, each UMMA cost 66 cycles).
template <bool F8, int LSTEP, int RSTEP>
__device__ __forceinline__ void umma_block_pair(uint32_t d, uint64_t l, uint64_t r, uint32_t idesc, uint32_t accumulate,
                                                int steps) {
#define HST_UMMA_BLOCK(KIND)                                                                             \
  asm volatile(                                                                                          \
      "{\n\t.reg .pred e, p, q;\n\t.reg .b64 l, r;\n\t"                                                  \
      "elect.sync _|e, 0xffffffff;\n\t"                                                                  \
      "setp.ne.b32 p, %4, 0;\n\t"                                                                        \
      "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], %1, %2, %3, p;\n\t"                              \
      "setp.gt.and.s32 q, %5, 1, e;\n\tadd.s64 l, %1, %6;\n\tadd.s64 r, %2, %7;\n\tsetp.eq.b32 p, 0, 0;\n\t" \
      "@q tcgen05.mma.cta_group::2.kind::" KIND " [%0], l, r, %3, p;\n\t"                                \
      "setp.gt.and.s32 q, %5, 2, e;\n\tadd.s64 l, l, %6;\n\tadd.s64 r, r, %7;\n\t"                       \
      "@q tcgen05.mma.cta_group::2.kind::" KIND " [%0], l, r, %3, p;\n\t"                                \
      "setp.gt.and.s32 q, %5, 3, e;\n\tadd.s64 l, l, %6;\n\tadd.s64 r, r, %7;\n\t"                       \
      "@q tcgen05.mma.cta_group::2.kind::" KIND " [%0], l, r, %3, p;\n\t}\n" ::"r"(d),                   \
      "l"(l), "l"(r), "r"(idesc), "r"(accumulate), "r"(steps), "n"(LSTEP), "n"(RSTEP)                    \
      : "memory")
  if constexpr (F8) {
    HST_UMMA_BLOCK("f8f6f4");
  } else {
    HST_UMMA_BLOCK("f16");
  }
#undef HST_UMMA_BLOCK
}

// umma_commit_pair_multicast by the lane that umma_block_pair elects.
__device__ __forceinline__ void umma_commit_elected(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}\n" ::"r"(
          bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// Lets the finish kernel launch as soon as every CTA of this grid runs; it waits for the grid's memory
// itself. (This kernel is no dependent of what precedes it: that gained 2% and would have the finish
// kernel read `ends` before they are written.)
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// (a0, a1) += (p0, p1) * s, as one operation on a pair of FP32 values.
__device__ __forceinline__ void fma_pair(float& a0, float& a1, uint32_t p0, uint32_t p1, float s) {
  asm("{\n\t.reg .b64 a, p, s;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 p, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\t"
      "fma.rn.f32x2 a, p, s, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(p0), "r"(p1), "f"(s));
}

// The scale a * b of a block's sums, which are up to 2^25, may leave FP32's normal range where what it scales does
// not (BF16's ends reach it: 2^100 x 2^60 with sums of zero, or 2^-109 x 2^-20). The sums then take one factor
// at a time: the smaller first where the product is too large, the larger first where it is too small, so that
// no step leaves the range before the result does.
__device__ __forceinline__ bool is_normal(float v) {
  return (__float_as_uint(v) << 1) - 0x01000000u < 0xfe000000u;  // neither zero, subnormal, infinite nor NaN
}
__device__ __forceinline__ void split_scale(float a, float b, float& before, float& scale) {
  scale = a * b;
  before = 1.f;
  if (is_normal(scale) || a == 0.f || b == 0.f) return;
  const bool a_first = (fabsf(a) < fabsf(b)) != (fabsf(scale) < 1.f);
  before = a_first ? a : b;
  scale = a_first ? b : a;
}
__device__ __forceinline__ uint32_t scaled_bits(uint32_t v, float s) { return __float_as_uint(__uint_as_float(v) * s); }

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

// One warp's lanes are 32 consecutive output columns from `col` on, v[j] the value of row `row + j`. With
// rows of an even length neighbouring lanes trade every second row's value, so that each stores two
// columns of one row (64 consecutive bytes per row and warp, half the stores). The whole warp.
template <typename T, int N>
__device__ __forceinline__ void store_rows_across(T* out, const GroupedArgs& a, const float (&v)[N], int row,
                                                  int row_end, int col) {
  const int lane = static_cast<int>(lane_id());
  if (a.vec >= 4) {
    const bool odd = (lane & 1) != 0;
    uint32_t* p = reinterpret_cast<uint32_t*>(out + static_cast<int64_t>(row + (odd ? 1 : 0)) * a.cols + col + (lane & ~1));
    const bool inside = col + (lane & ~1) < a.cols;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float got = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
      const uint32_t w = odd ? pack_f32<T>(got, v[j + 1]) : pack_f32<T>(v[j], got);
      if (inside && row + j + (odd ? 1 : 0) < row_end) p[static_cast<int64_t>(j) * (a.cols / 2)] = w;
    }
  } else if (col + lane < a.cols) {
    T* p = out + static_cast<int64_t>(row) * a.cols + col + lane;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (row + j < row_end) p[static_cast<int64_t>(j) * a.cols] = from_f32<T>(v[j]);
    }
  }
}

// Transposes the warp's 32 x 32 matrix: v[i] of lane j becomes v[j] of lane i.
__device__ __forceinline__ void warp_transpose(float (&v)[32]) {
  const uint32_t lane = lane_id();
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) {
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if ((i & d) == 0) {
        const float give = upper ? v[i] : v[i + d];
        const float got = __shfl_xor_sync(0xffffffffu, give, d);
        if (upper) {
          v[i] = got;
        } else {
          v[i + d] = got;
        }
      }
    }
  }
}

// The warp's 32 rows x 64 output columns from column `col` on, one row a lane: `first` is the warp's
// first row in the output, `rows` how many of the 32 exist. Rows of 16-byte alignment go through
// 4 KB of the warp's shared memory (16-byte chunks, XORed with the row against bank conflicts), so that
// a store covers four whole 128-byte lines: with one row a lane, a store touches 32 lines, and a
// 128 x 256 tile took 6000 cycles. Other rows are transposed in registers and stored two bytes a lane.
constexpr int kStageOutBytes = 4096;
template <typename T>
__device__ __forceinline__ void store_cols_64(T* out, int64_t first, int rows, int col, const GroupedArgs& a, uint32_t stage,
                                              float (&lo)[32], float (&hi)[32]) {
  const int lane = static_cast<int>(lane_id());
  if (a.vec >= 16) {
    const uint32_t mine = stage + lane * 128;
    __syncwarp();  // the warp has read what was staged before
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float* f = j < 4 ? &lo[8 * j] : &hi[8 * (j - 4)];
      st_shared_v4(mine + ((j ^ (lane & 7)) << 4), pack_f32<T>(f[0], f[1]), pack_f32<T>(f[2], f[3]), pack_f32<T>(f[4], f[5]),
                   pack_f32<T>(f[6], f[7]));
    }
    __syncwarp();
    const int ch = lane & 7;
    const bool inside = col + ch * 8 < a.cols;  // rows are whole chunks: none is ragged
    T* p = out + (first + (lane >> 3)) * a.cols + col + ch * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3);
      const float4 v = ld_shared_f32x4(stage + r * 128 + ((ch ^ (r & 7)) << 4));
      if (inside && r < rows) *reinterpret_cast<float4*>(p + static_cast<int64_t>(4 * i) * a.cols) = v;
    }
  } else {
    T* p = out + first * a.cols + col + lane;
    warp_transpose(lo);
    warp_transpose(hi);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i < rows && col + lane < a.cols) p[static_cast<int64_t>(i) * a.cols] = from_f32<T>(lo[i]);
      if (i < rows && col + lane + 32 < a.cols) p[static_cast<int64_t>(i) * a.cols + 32] = from_f32<T>(hi[i]);
    }
  }
}

// What no tile covers: rows past the last group, or the outputs of groups without rows. Thread `mine`
// of `step`.
template <GroupMode MODE, typename T>
__device__ inline void write_zeros(const GroupedArgs& a, const GroupTable& t, T* out, int64_t mine, int64_t step) {
  auto zero = [&](T* p, int64_t count) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && count % 8 == 0) {
      for (int64_t i = mine; i < count / 8; i += step) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
    } else {
      for (int64_t i = mine; i < count; i += step) p[i] = from_f32<T>(0.f);
    }
  };
  if constexpr (MODE == GroupMode::kWeightGrad) {
    const int64_t size = static_cast<int64_t>(a.lrows) * a.cols;
    for (int g = 0; g < a.groups; ++g) {
      if (t.start(g + 1) == t.start(g)) zero(out + g * size, size);
    }
  } else {
    const int64_t from = t.start(a.groups);
    if (from < a.rows) zero(out + from * a.cols, (a.rows - from) * a.cols);
  }
}

// Takes registers from, or gives them to, the calling warpgroup: REGS a thread then. The kernel is
// launched with 384 x 168 = 64512; 128 x 80 + 256 x 208 are 63488, and neither side spills (with 40 and
// 232, or 56 and 224, the issuing warps did: 46 us against 43 for 257 x 12800 x 4096).
template <int REGS>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}

// Shared memory: the ring, the staged output rows, the barriers and the table.
template <GroupMode MODE>
struct GroupedShape {
  static constexpr int kBarriers = 3 * kMaxStages + 2 * 8 + 1;
  static constexpr int kBarrierBytes = kBarriers * 8 + 16;
  static constexpr int kOutBytes = group_rows_right(MODE) ? 0 : group_epilogue_warps(MODE) * kStageOutBytes;
  __host__ __device__ static constexpr int stage_bytes(int r_bytes) { return kGroupLBytes + r_bytes; }
  __host__ __device__ static constexpr int smem_bytes(int stages, int r_bytes, int groups, int pairs) {
    return 1024 + stages * stage_bytes(r_bytes) + kOutBytes + kBarrierBytes + group_table_ints(groups, pairs) * 4;
  }
};

// L_MN: the L operand's rows are its contiguous dimension (kForward with W [E, K, N] row-major, and
// kWeightGrad); otherwise K is.
template <GroupMode MODE, bool L_MN, typename T>
__global__ void __launch_bounds__(group_threads(MODE), 1)
    grouped_gemm_kernel(const __grid_constant__ GroupedMaps maps, const __grid_constant__ GroupedArgs args) {
  using S = GroupedShape<MODE>;
  constexpr bool kScaled = group_scaled(MODE);
  constexpr bool kWide = MODE == GroupMode::kScaled;
  constexpr bool kFew = MODE == GroupMode::kScaledFew;
  constexpr bool kGrad = MODE == GroupMode::kWeightGrad;
  constexpr int kFirstEpilogue = group_first_epilogue_warp(MODE);
  constexpr int kEpilogueWarps = group_epilogue_warps(MODE);
  constexpr int kSteps = 4;                    // UMMA K steps of a block: 128 bytes of K
  constexpr int kBlockK = kScaled ? 128 : 64;  // K values of a block
  constexpr bool kBf16 = !kScaled && std::is_same<T, __nv_bfloat16>::value;
  constexpr int kBufs = kFew ? 8 : 2;  // TMEM buffers
  constexpr int kBufCols = 512 / kBufs;
  constexpr uint32_t kIdescBase = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (L_MN ? 1u << 15 : 0u) |
                                  (kGrad ? 1u << 16 : 0u) | ((256u >> 4) << 24);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = args.stages;
  const int stage_bytes = S::stage_bytes(args.r_bytes);
  uint8_t* out_stage = ring + stages * stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_stage + S::kOutBytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tail_full = empty + kMaxStages;  // kWeightGrad: this CTA's own part of a block to be masked
  uint64_t* tmem_full = tail_full + kMaxStages;
  uint64_t* tmem_empty = tmem_full + 8;
  uint64_t* mma_done = tmem_empty + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const GroupTable table = {reinterpret_cast<int*>(tmem_slot + 4), args.groups, args.pairs};

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
    tma_prefetch_map(&maps.l[0]);
    tma_prefetch_map(&maps.r[0]);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  if (warp == 2) build_group_rows<MODE>(args, table);
  __syncthreads();
  build_group_columns<MODE>(args, table);
  tc_fence_before_sync();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  if constexpr (kWide) {
    if (warp < kFirstEpilogue) registers_down<80>();
  }

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    int stage = 0;
    uint32_t phase = 0;
    uint32_t armed_mask = 0, armed_parity = 0;  // stages this warp has armed (leader)
    uint32_t tail_mask = 0, tail_parity = 0;    // tail barriers used; parity of their next use
    bool ok = true;
    GroupWalk<MODE> walk(args, table, pair);
    GroupSegment s;
    while (ok && walk.next(args, table, pair, s)) {
      const int half = s.width / 2;
      const int tail = kGrad ? (s.row_end - s.row0) - (s.blocks - 1) * 64 : 0;
      const int l0 = s.l0 + static_cast<int>(rank) * 128;
      const int r0 = s.r0 + static_cast<int>(rank) * half;
      // kScaled: rows the tile has in this CTA, and in both; what a box of them leaves of the stage
      // holds what it held (those lanes are not stored).
      const int left = s.row_end - s.l0;
      const int mine = min(128, left - static_cast<int>(rank) * 128);
      auto box_bytes = [](int rows) { return rows <= 0 ? 0u : (128u >> group_box(rows)) * 128u; };
      const CUtensorMap* l_map = &maps.l[kWide ? group_box(mine) : 0];
      const CUtensorMap* r_map = &maps.r[kGrad ? 0 : group_box(half)];
      const uint32_t r_bytes = group_rows_right(MODE) ? box_bytes(half) : static_cast<uint32_t>(half) * 128u;
      const uint32_t both_bytes = 2 * r_bytes + (kWide ? box_bytes(left) + box_bytes(left - 128) : 2 * kGroupLBytes);
      for (int kb = s.kb0; kb < s.kb1; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, abort_flag));
        if (!ok) break;
        const uint32_t l_dst = smem_addr(ring) + static_cast<uint32_t>(stage * stage_bytes);
        const uint32_t r_dst = l_dst + kGroupLBytes;
        const uint32_t leader_full = map_to_rank(smem_addr(&full[stage]), 0);
        if (kGrad && kb == s.blocks - 1 && (tail & 15) != 0) {
          // The group's last rows: into this CTA's own barrier, for the masking warp.
          const uint32_t bar = smem_addr(&tail_full[stage]);
          elected_expect_tx(bar, kGroupLBytes + r_bytes);
          tail_mask |= 1u << stage;
          tail_parity ^= 1u << stage;
          armed_mask &= ~(1u << stage);
          const int y = s.row0 + kb * 64;
          for (int i = 0; i < 2; ++i) elected_load_2d(l_dst + i * 8192, l_map, bar, l0 + 64 * i, y);
          for (int i = 0; i < half / 64; ++i) elected_load_2d(r_dst + i * 8192, r_map, bar, r0 + 64 * i, y);
        } else {
          if (rank == 0) {
            elected_expect_tx(smem_addr(&full[stage]), both_bytes);
            armed_mask |= 1u << stage;
            armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
          } else if (kGrad) {
            elected_arrive_cluster_relaxed(leader_full);
          }
          if constexpr (kGrad) {
            const int y = s.row0 + kb * 64;
            for (int i = 0; i < 2; ++i) elected_load_2d_pair(l_dst + i * 8192, l_map, leader_full, l0 + 64 * i, y);
            for (int i = 0; i < half / 64; ++i) elected_load_2d_pair(r_dst + i * 8192, r_map, leader_full, r0 + 64 * i, y);
          } else {
            const int k0 = kb * kBlockK;
            if constexpr (kWide) {
              if (mine > 0) elected_load_2d_pair(l_dst, l_map, leader_full, k0, l0);
              elected_load_3d_pair(r_dst, r_map, leader_full, k0, r0, s.group);
            } else {
              if constexpr (L_MN) {
                for (int i = 0; i < 2; ++i) elected_load_3d_pair(l_dst + i * 8192, l_map, leader_full, l0 + 64 * i, k0, s.group);
              } else {
                elected_load_3d_pair(l_dst, l_map, leader_full, k0, l0, s.group);
              }
              elected_load_2d_pair(r_dst, r_map, leader_full, k0, r0);
            }
          }
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && lane == 0) {
      raise_abort(args.status, abort_flag, kStatusProducerTimeout);
      for (int st = 0; st < stages; ++st) {  // drain the copies in flight before the pair can exit
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
  } else if (warp == 1 && rank == 0) {
    // ---------------- UMMA issuer (leader only) ----------------
    int stage = 0;
    uint32_t phase = 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    const uint64_t l_desc0 = smem_desc(smem_addr(ring), L_MN ? 8192 : 16, 1024);
    const uint64_t r_desc0 = smem_desc(smem_addr(ring) + kGroupLBytes, kGrad ? 8192 : 16, 1024);
    constexpr int kLStep = (L_MN ? 2048 : 32) >> 4, kRStep = (kGrad ? 2048 : 32) >> 4;
    GroupWalk<MODE> walk(args, table, pair);
    GroupSegment s;
    while (ok && walk.next(args, table, pair, s)) {
      const uint32_t idesc = kIdescBase | (static_cast<uint32_t>(s.width >> 3) << 17);
      const int tail = kGrad ? (s.row_end - s.row0) - (s.blocks - 1) * 64 : 0;
      for (int kb = s.kb0; kb < s.kb1; ++kb) {
        if (kScaled || kb == s.kb0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&tmem_empty[buf], buf_phase ^ 1u, abort_flag));
          if (!ok) break;
          tc_fence_after_sync();
        }
        // A masked block: the peer's masking warp wrote its shared memory, which takes an acquire at
        // cluster scope (1.0 us a block when every wait was one, against 0.5).
        const bool masked = kGrad && kb == s.blocks - 1 && (tail & 15) != 0;
        ok = __all_sync(0xffffffffu, masked ? mbar_wait_cluster(&full[stage], phase, abort_flag)
                                            : mbar_wait(&full[stage], phase, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t off = static_cast<uint64_t>(stage * (stage_bytes >> 4));
        const int steps = kGrad && kb == s.blocks - 1 ? (tail + 15) / 16 : kSteps;
        umma_block_pair<kScaled, kLStep, kRStep>(tmem_base + static_cast<uint32_t>(buf * kBufCols), l_desc0 + off, r_desc0 + off,
                                                 idesc, !kScaled && kb != s.kb0, steps);
        umma_commit_elected(smem_addr(&empty[stage]));
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (kScaled || kb + 1 == s.kb1) {
          umma_commit_elected(smem_addr(&tmem_full[buf]));
          if (++buf == kBufs) {
            buf = 0;
            buf_phase ^= 1u;
          }
        }
      }
    }
    if (!ok && lane == 0) raise_abort(args.status, abort_flag, kStatusMmaTimeout);
    umma_commit_elected(smem_addr(mma_done));
    if (!mbar_wait(mma_done, 0, nullptr, 200000000ull) && lane == 0) atomicOr(args.status, kStatusDrainTimeout);
  } else if (kGrad && warp == kFirstEpilogue + kEpilogueWarps) {
    // ---------------- masking warp (both CTAs): rows past the group in its last block ----------
    int stage = 0;
    uint32_t parity = 0;  // bit s: parity of the next use of tail_full[s]
    GroupWalk<MODE> walk(args, table, pair);
    GroupSegment s;
    while (walk.next(args, table, pair, s)) {
      const int blocks = s.kb1 - s.kb0;
      const int tail = (s.row_end - s.row0) - (s.blocks - 1) * 64;
      if (s.kb1 == s.blocks && (tail & 15) != 0) {
        const int st = (stage + blocks - 1) % stages;
        if (!__all_sync(0xffffffffu, mbar_wait(&tail_full[st], (parity >> st) & 1u, abort_flag))) {
          if (lane == 0) raise_abort(args.status, abort_flag, kStatusEpilogueTimeout);
          break;
        }
        parity ^= 1u << st;
        // A box is 64 rows of 128 bytes; the swizzle moves 16-byte chunks within a row only. One
        // 512-byte store of the warp clears four rows.
        const int end = (tail + 15) & ~15;
        const uint32_t st_addr = smem_addr(ring + st * stage_bytes) + (lane & 7u) * 16;
        for (int b = 0; b < 2 + s.width / 128; ++b) {
          for (int r = tail + static_cast<int>(lane >> 3); r < end; r += 4) {
            st_shared_v4(st_addr + b * 8192 + r * 128, 0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_addr(&full[st]), 0));
      }
      stage = (stage + blocks) % stages;
    }
  } else if (warp >= kFirstEpilogue && warp < kFirstEpilogue + kEpilogueWarps) {
    // ---------------- epilogue (both CTAs, own 128 TMEM lanes) ----------------
    if constexpr (kWide) registers_up<208>();
    const int quarter = warp & 3;
    const int row = quarter * 32 + static_cast<int>(lane);  // TMEM lane
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    T* out = static_cast<T*>(args.out);
    const int half = kEpilogueWarps == 8 ? (warp - kFirstEpilogue) / 4 : 0;  // of the tile's columns
    int buf = 0;
    uint32_t buf_phase = 0;
    auto wait_buf = [&]() {
      const bool ready = __all_sync(0xffffffffu, mbar_wait(&tmem_full[buf], buf_phase, abort_flag));
      if (!ready && lane == 0) raise_abort(args.status, abort_flag, kStatusEpilogueTimeout);
      if (ready) tc_fence_after_sync();
      return ready;
    };
    const uint32_t leader_empty = map_to_rank(smem_addr(tmem_empty), 0);
    auto release_buf = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      elected_arrive_cluster_relaxed(leader_empty + static_cast<uint32_t>(buf) * 8);
      if (++buf == kBufs) {
        buf = 0;
        buf_phase ^= 1u;
      }
    };
    auto piece_of = [&](const GroupSegment& s) {
      return args.partials +
             (static_cast<size_t>(pair * 2 + (s.first ? 0 : 1)) * 2 + rank) * static_cast<size_t>(args.piece_floats);
    };
    GroupWalk<MODE> walk(args, table, pair);
    GroupSegment s;
    if constexpr (!kScaled) {
      while (walk.next(args, table, pair, s)) {
        if (!wait_buf()) break;
        const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols);
        const int l32 = s.l0 + static_cast<int>(rank) * 128 + quarter * 32;  // the warp's first L row
        const bool whole = s.kb0 == 0 && s.kb1 == s.blocks;
        const int c_begin = kGrad ? half * (s.width / 2) : 0, c_end = kGrad ? c_begin + s.width / 2 : s.width;
        if (!whole) {
#pragma unroll 1
          for (int c = c_begin; c < c_end; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(taddr + c, v);
            tmem_ld_wait();
            float* dst = piece_of(s) + (static_cast<size_t>(c / 4) * 128 + row) * 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              st_global_v4(dst + static_cast<size_t>(j) * 512, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
          }
        } else if constexpr (kGrad) {
          const uint32_t stage_out = smem_addr(out_stage) + static_cast<uint32_t>(warp - kFirstEpilogue) * kStageOutBytes;
#pragma unroll 1
          for (int c = c_begin; c < c_end; c += 64) {
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(taddr + c, v[0]);
            tmem_ld_32x32b_x32(taddr + c + 32, v[1]);
            tmem_ld_wait();
            float f[2][32];
#pragma unroll
            for (int j = 0; j < 64; ++j) f[j / 32][j % 32] = __uint_as_float(v[j / 32][j % 32]);
            store_cols_64(out, static_cast<int64_t>(s.group) * args.lrows + l32, args.lrows - l32, s.r0 + c, args, stage_out,
                          f[0], f[1]);
          }
        } else {
          // 32 columns at a time, the next ones in flight while these are stored.
          uint32_t v[2][32];
          tmem_ld_32x32b_x32(taddr, v[0]);
          tmem_ld_wait();
          tmem_ld_fence_regs(v[0]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (32 * i >= s.width) break;
            if (32 * i + 32 < s.width) tmem_ld_32x32b_x32(taddr + 32 * i + 32, v[(i & 1) ^ 1]);
            float f[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[i & 1][j]);
            store_rows_across(out, args, f, s.r0 + 32 * i, min(s.row_end, s.r0 + s.width), l32);
            tmem_ld_wait();
            tmem_ld_fence_regs(v[(i & 1) ^ 1]);
          }
        }
        release_buf();
      }
    } else if constexpr (kWide) {
      // One weight scale a block for the 128 columns of a half; both scales are loaded a block ahead.
      while (walk.next(args, table, pair, s)) {
        const int l32 = s.l0 + static_cast<int>(rank) * 128 + quarter * 32;
        const int col = s.r0 + half * 128;
        const bool live = l32 < s.row_end && col < args.cols;  // warp-uniform
        const float* sa = args.row_scales + static_cast<int64_t>(min(l32 + static_cast<int>(lane), args.rows - 1)) * args.rs_row +
                          s.kb0 * args.rs_k;
        const float* sb = args.tile_scales + s.group * args.ts_group + (min(col, args.cols - 1) >> 7) * args.ts_n + s.kb0 * args.ts_k;
        float next_a = *sa, next_b = *sb;
        float acc[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] = 0.f;
        bool ready = true;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          const float a = next_a, b = next_b;
          if (kb + 1 < s.kb1) {
            sa += args.rs_k;
            sb += args.ts_k;
            next_a = *sa;
            next_b = *sb;
          }
          ready = wait_buf();
          if (!ready) break;
          float now = a * b;
          const bool split = !__all_sync(0xffffffffu, is_normal(now));
          // Rare: the block's sums take the first factor in TMEM, so that the loop below stays as it is (with a copy of the
          // loop for this, 8192 x 14336 x 4096 took 487 to 502 us). The vote itself costs 481 against 470 us there, and
          // 42.7 against 41.3 for 257 x 12800 x 4096.
          if (live && split) {
            float before;
            split_scale(a, b, before, now);
#pragma unroll 1
            for (int c = 0; c < 128; c += 16) {
              const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols + half * 128 + c);
              uint32_t v[16];
              tmem_ld_32x32b_x16(taddr, v);
              tmem_ld_wait();
              tmem_ld_fence_regs(v);
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = scaled_bits(v[j], before);
              tmem_st_32x32b_x16(taddr, v);
            }
            tmem_st_wait();
          }
          if (live) {
            const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols + half * 128);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t v[2][32];
              tmem_ld_32x32b_x32(taddr + 64 * h, v[0]);
              tmem_ld_32x32b_x32(taddr + 64 * h + 32, v[1]);
              tmem_ld_wait();
              tmem_ld_fence_regs(v[0]);
              tmem_ld_fence_regs(v[1]);
              if (h == 1) release_buf();
#pragma unroll
              for (int j = 0; j < 64; j += 2) {
                fma_pair(acc[64 * h + j], acc[64 * h + j + 1], v[j / 32][j % 32], v[j / 32][j % 32 + 1], now);
              }
            }
          } else {
            release_buf();
          }
        }
        if (!ready) break;
        if (!live) continue;
        const bool whole = s.kb0 == 0 && s.kb1 == s.blocks;
        if (whole) {
          const uint32_t stage_out = smem_addr(out_stage) + static_cast<uint32_t>(warp - kFirstEpilogue) * kStageOutBytes;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float f[2][32];
#pragma unroll
            for (int j = 0; j < 64; ++j) f[j / 32][j % 32] = acc[64 * h + j];
            store_cols_64(out, l32, s.row_end - l32, col + 64 * h, args, stage_out, f[0], f[1]);
          }
        } else {
          float* dst = piece_of(s) + (static_cast<size_t>(half * 32) * 128 + row) * 4;
          if (l32 + static_cast<int>(lane) < s.row_end) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              st_global_v4(dst + static_cast<size_t>(j) * 512, __float_as_uint(acc[4 * j]), __float_as_uint(acc[4 * j + 1]),
                           __float_as_uint(acc[4 * j + 2]), __float_as_uint(acc[4 * j + 3]));
            }
          }
        }
      }
    } else {
      // kScaledFew: lane j holds the scales of rows j and j + 32, times this CTA's weight scale.
      while (walk.next(args, table, pair, s)) {
        const int l32 = s.l0 + static_cast<int>(rank) * 128 + quarter * 32;
        const int nb = min((s.l0 >> 7) + static_cast<int>(rank), (args.cols - 1) >> 7);
        const float* sb = args.tile_scales + s.group * args.ts_group + nb * args.ts_n + s.kb0 * args.ts_k;
        const float* sa = args.row_scales + static_cast<int64_t>(min(s.r0 + static_cast<int>(lane), args.rows - 1)) * args.rs_row +
                          s.kb0 * args.rs_k;
        const float* sa32 =
            args.row_scales + static_cast<int64_t>(min(s.r0 + 32 + static_cast<int>(lane), args.rows - 1)) * args.rs_row +
            s.kb0 * args.rs_k;
        const bool second = s.width > 32;
        float acc[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = 0.f;
        float next_a = *sa, next_a32 = second ? *sa32 : 0.f, next_b = *sb;
        bool ready = true;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          const float a = next_a, a32 = next_a32, b = next_b;
          if (kb + 1 < s.kb1) {
            sa += args.rs_k;
            sb += args.ts_k;
            next_a = *sa;
            next_b = *sb;
            if (second) {
              sa32 += args.rs_k;
              next_a32 = *sa32;
            }
          }
          ready = wait_buf();
          if (!ready) break;
          const uint32_t taddr = lane_base + static_cast<uint32_t>(buf * kBufCols);
          uint32_t v[2][32];
          tmem_ld_32x32b_x32(taddr, v[0]);
          if (second) tmem_ld_32x32b_x32(taddr + 32, v[1]);
          float now = a * b, now32 = a32 * b;
          const bool split = !__all_sync(0xffffffffu, is_normal(now) & is_normal(second ? now32 : 1.f));
          tmem_ld_wait();
          // Rare: as in the wide form, and loaded again. The vote costs 23.8 against 23.3 us for 1 x 18944 x 3584, 43.4
          // against 41.9 for 128 rows over 32 groups of 2816 x 2048 (24.5 and 46.2 where it comes before the loads).
          if (split) {
            float before, before32;
            split_scale(a, b, before, now);
            split_scale(a32, b, before32, now32);
#pragma unroll 1
            for (int c = 0; c < s.width; c += 16) {
              uint32_t w[16];
              tmem_ld_32x32b_x16(taddr + c, w);
              tmem_ld_wait();
              tmem_ld_fence_regs(w);
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = scaled_bits(w[j], __shfl_sync(0xffffffffu, c < 32 ? before : before32, (c & 31) + j));
              tmem_st_32x32b_x16(taddr + c, w);
            }
            tmem_st_wait();
            tmem_ld_32x32b_x32(taddr, v[0]);
            if (second) tmem_ld_32x32b_x32(taddr + 32, v[1]);
            tmem_ld_wait();
          }
          tmem_ld_fence_regs(v[0]);
          tmem_ld_fence_regs(v[1]);
          release_buf();
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[j] = fmaf(__uint_as_float(v[0][j]), __shfl_sync(0xffffffffu, now, j), acc[j]);
          if (second) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              acc[32 + j] = fmaf(__uint_as_float(v[1][j]), __shfl_sync(0xffffffffu, now32, j), acc[32 + j]);
            }
          }
        }
        if (!ready) break;
        const int row_end = min(s.row_end, s.r0 + s.width);
        if (s.kb0 == 0 && s.kb1 == s.blocks) {
          store_rows_across(out, args, acc, s.r0, row_end, l32);
        } else {
          float* dst = piece_of(s) + static_cast<size_t>(row) * 4;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (s.r0 + 4 * j < row_end) {
              st_global_v4(dst + static_cast<size_t>(j) * 512, __float_as_uint(acc[4 * j]), __float_as_uint(acc[4 * j + 1]),
                           __float_as_uint(acc[4 * j + 2]), __float_as_uint(acc[4 * j + 3]));
            }
          }
        }
      }
    }
    if (args.whole) {
      const int64_t thread = (warp - kFirstEpilogue) * 32 + static_cast<int>(lane);
      write_zeros<MODE>(args, table, out, blockIdx.x * (kEpilogueWarps * 32) + thread,
                        static_cast<int64_t>(gridDim.x) * (kEpilogueWarps * 32));
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
constexpr int kFinishCols = 32;  // columns of a piece one block joins (kWeightGrad, kScaled: 64)
template <GroupMode MODE>
__host__ __device__ constexpr int finish_cols() {
  return group_rows_right(MODE) ? kFinishCols : 2 * kFinishCols;
}

// Joins the tiles that shares cut: block (p, CTA half, chunk of columns) takes the tile in which share
// p + 1 begins, if that is the first share to begin inside it, and adds its FP32 pieces in K order.
// Then all blocks write the zeros nobody else writes.
template <GroupMode MODE, typename T>
__global__ void __launch_bounds__(kFinishThreads) grouped_finish_kernel(const __grid_constant__ GroupedArgs args) {
  constexpr int kCols = finish_cols<MODE>();
  __shared__ __align__(128) uint8_t out_stage[group_rows_right(MODE) ? 16 : kFinishThreads / 32 * kStageOutBytes];
  extern __shared__ int finish_table[];
  const GroupTable table = {finish_table, args.groups, args.pairs};
  if (threadIdx.x < 32) build_group_rows<MODE>(args, table);
  __syncthreads();
  build_group_columns<MODE>(args, table);
  __syncthreads();
  T* out = static_cast<T*>(args.out);
  const int p = static_cast<int>(blockIdx.x) + 1;
  const int rank = static_cast<int>(blockIdx.y);
  GroupSegment s = {};
  int cut = 0;
  const bool joins = !table.whole() && p < table.shares() && table.share_begin(p) < table.total();
  if (joins) {
    cut = table.share_begin(p);
    GroupWalk<MODE> walk(args, table, cut, cut + 1, p);
    walk.next(args, table, 0, s);
  }
  wait_for_primary();  // the pieces; all before it comes from `ends` alone
  if (joins) {
    const int begin = cut - s.kb0, end = begin + s.blocks;
    const int c = static_cast<int>(blockIdx.z) * kCols;
    if (cut > begin && table.share_begin(p - 1) <= begin && c < s.width) {
      const int row = static_cast<int>(threadIdx.x);
      float v[kCols / 32][32];
#pragma unroll
      for (int j = 0; j < kCols; ++j) v[j / 32][j % 32] = 0.f;
      // Columns and rows that hold values of the output (what else a piece has was not written).
      const bool mine = MODE != GroupMode::kScaled || s.l0 + rank * 128 + row < s.row_end;
      const int live_cols = group_rows_right(MODE) ? min(s.width, s.row_end - s.r0) : min(s.width, args.cols - s.r0);
      // The pieces' shares: p - 1 to last, of which the first may have the tile as its second piece. Loads
      // of kBatch pieces are in flight together: few rows are cut into many pieces (1 x 18944 x 3584 in 8 bits, six a
      // tile: 26.2 us one after the other, 24.9 so). Where the pieces are large the blocks that fit on an SM count
      // for more (four of 32 columns in the forward: 1000 x 8192 x 4096 from 57.8 to 61.5 us).
      constexpr int kBatch = MODE == GroupMode::kScaledFew ? 4 : (kCols == 32 ? 2 : 1);
      int last = p;
      while (last + 1 < table.shares() && table.share_begin(last + 1) < end) ++last;
      const int64_t piece = 2 * static_cast<int64_t>(args.piece_floats);
      const float* src = args.partials + (2 * (p - 1) + (table.share_begin(p - 1) >= begin ? 0 : 1)) * piece +
                         static_cast<int64_t>(rank) * args.piece_floats + (static_cast<int64_t>(c / 4) * 128 + row) * 4;
      const float* next = args.partials + 2 * p * piece + static_cast<int64_t>(rank) * args.piece_floats +
                          (static_cast<int64_t>(c / 4) * 128 + row) * 4;
      for (int o = p - 1; mine && o <= last; o += kBatch) {
        float4 f[kBatch][kCols / 4];
        auto add = [&](const float4& g, int j) {
          float* sum = &v[j / 8][4 * (j % 8)];
          sum[0] += g.x;
          sum[1] += g.y;
          sum[2] += g.z;
          sum[3] += g.w;
        };
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (o + i <= last) {
#pragma unroll
            for (int j = 0; j < kCols / 4; ++j) {
              if (c + 4 * j < live_cols) {
                f[i][j] = *reinterpret_cast<const float4*>(src + j * 512);
                if (kBatch == 1) add(f[i][j], j);
              }
            }
            src = next;
            next += 2 * piece;
          }
        }
        if constexpr (kBatch > 1) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            if (o + i <= last) {
#pragma unroll
              for (int j = 0; j < kCols / 4; ++j) {
                if (c + 4 * j < live_cols) add(f[i][j], j);
              }
            }
          }
        }
      }
      const int l32 = s.l0 + rank * 128 + (row & ~31);
      if constexpr (group_rows_right(MODE)) {
        store_rows_across(out, args, v[0], s.r0 + c, min(s.row_end, s.r0 + s.width), l32);
      } else {
        const bool grad = MODE == GroupMode::kWeightGrad;
        store_cols_64(out, grad ? static_cast<int64_t>(s.group) * args.lrows + l32 : l32,
                      (grad ? args.lrows : s.row_end) - l32, s.r0 + c, args,
                      smem_addr(out_stage) + (threadIdx.x >> 5) * kStageOutBytes, v[0], v[kCols / 32 - 1]);
      }
    }
  }
  write_zeros<MODE>(args, table, out,
                    ((static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * kFinishThreads + threadIdx.x,
                    static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z * kFinishThreads);
}

}  // namespace hst
