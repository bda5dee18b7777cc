// C ABI of the grouped and block-scaled products and of the quantisers: argument checks, tensor
// maps, workspace sizes and the choice of kernel. See include/heliostune_b200.h.
#include <algorithm>

#include "gemm_grouped.cuh"
#include "host.h"
#include "pack.cuh"
#include "quantize.cuh"

namespace hst {
namespace {

constexpr int64_t kMaxExtent = INT32_MAX / 2;

// What the host knows of one grouped product.
struct GroupedProblem {
  int64_t rows;      // T
  int groups;
  int64_t cols;      // output columns
  int64_t lrows;     // kWeightGrad: rows of one output
  int64_t k_blocks;  // forward, scaled
  int width_cap;     // columns of a piece; rows on the R side: most of them in a tile
};

int check_groups(const char* what, int64_t rows, int32_t groups, const void* ends) {
  if (groups < 1 || groups > kMaxGroups)
    return fail(HST_ERR_INVALID, "%s serves 1 to %d groups, got %d", what, kMaxGroups, groups);
  if (ends == nullptr && groups != 1) return fail(HST_ERR_INVALID, "group ends are null");
  if (rows < 0 || rows > kMaxExtent) return fail(HST_ERR_INVALID, "%s: bad row count %lld", what, (long long)rows);
  return HST_OK;
}

int check_extents(const char* what, int64_t a, int64_t b) {
  if (a < 0 || b < 0 || a > kMaxExtent || b > kMaxExtent)
    return fail(HST_ERR_INVALID, "%s: bad extents %lld, %lld", what, (long long)a, (long long)b);
  return HST_OK;
}

// Whether a pointer starts on a multiple of its values' size; what does not would fault on the GPU.
int check_aligned(const char* name, const void* ptr, int bytes) {
  if (reinterpret_cast<uintptr_t>(ptr) % bytes != 0)
    return fail(HST_ERR_INVALID, "%s must be aligned to %d bytes", name, bytes);
  return HST_OK;
}

// A stack of matrices [groups, rows, cols] with strides in values.
struct Stack {
  const void* ptr;
  int64_t elem;  // bytes of a value
  int64_t groups, rows, cols;
  int64_t s_group, s_row, s_col;

  int64_t unit() const { return 16 / elem; }
  int64_t packed_row() const { return round_up(cols, unit()); }
  size_t packed_bytes() const { return static_cast<size_t>(round_up(groups * rows * packed_row() * elem, 256)); }
  // Strides of dimensions of one entry do not matter; a tensor map wants some.
  void settle() {
    if (cols == 1) s_col = 1;
    if (rows == 1) s_row = packed_row();
    if (groups == 1) s_group = s_row * rows;
  }
  // Whether a tensor map can describe it: unit column stride, and the base, the rows (at least as long as
  // the columns) and the groups aligned to 16 bytes, none overlapping the next.
  bool readable() const {
    return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && s_col == 1 && s_row % unit() == 0 && s_row >= cols &&
           s_group % unit() == 0 && s_group >= s_row * rows;
  }
};

Stack make_stack(const void* ptr, int64_t elem, int64_t groups, int64_t rows, int64_t cols, int64_t s_group, int64_t s_row,
                 int64_t s_col) {
  Stack s = {ptr, elem, groups, rows, cols, s_group, s_row, s_col};
  s.settle();
  return s;
}

// Whether the copies a product needs can be counted in 64 bits and made by one grid; no GPU holds more. (Extents of
// broadcast operands are not bound by the memory behind them.)
constexpr int64_t kMaxCopyBytes = int64_t(1) << 44;
int check_copies(const char* what, const Stack& a, const Stack& b) {
  for (const Stack* s : {&a, &b}) {
    if (!s->readable() && s->groups > kMaxCopyBytes / (s->rows * s->packed_row() * s->elem))
      return fail(HST_ERR_UNSUPPORTED, "%s: an operand to be copied is too large", what);
  }
  return HST_OK;
}

size_t pack_bytes(const Stack& s) { return s.readable() ? 0 : s.packed_bytes(); }

// Copies a stack that is not readable to `dst`, the weights of empty groups left out where `ends` tells
// of them, and describes the copy.
int pack(Stack* s, void* dst, const int32_t* ends, int64_t total_rows, cudaStream_t stream) {
  const int64_t e = s->elem;
  PackArgs a = {static_cast<const uint8_t*>(s->ptr), s->s_group * e, s->s_row * e, s->s_col * e, static_cast<uint8_t*>(dst),
                s->rows * s->packed_row() * e, s->packed_row() * e, ends, static_cast<int>(total_rows), s->rows,
                static_cast<int>(cdiv(s->cols * e, 16)), s->cols * e};
  if (s->s_col == 1) {
    const dim3 grid(static_cast<unsigned>(cdiv(s->rows * a.chunks, kPackThreads * kPackPerThread)), static_cast<unsigned>(s->groups));
    // The common alignment of every row's start and of its length.
    const uint64_t bits = reinterpret_cast<uintptr_t>(s->ptr) | static_cast<uint64_t>(a.row_bytes) |
                          static_cast<uint64_t>(a.s_row) | static_cast<uint64_t>(a.s_group);
    if (bits % 16 == 0) pack_rows_kernel<uint4><<<grid, kPackThreads, 0, stream>>>(a);
    else if (bits % 8 == 0) pack_rows_kernel<uint2><<<grid, kPackThreads, 0, stream>>>(a);
    else if (bits % 4 == 0) pack_rows_kernel<uint32_t><<<grid, kPackThreads, 0, stream>>>(a);
    else if (bits % 2 == 0) pack_rows_kernel<uint16_t><<<grid, kPackThreads, 0, stream>>>(a);
    else pack_rows_kernel<uint8_t><<<grid, kPackThreads, 0, stream>>>(a);
  } else {
    const int64_t tiles = cdiv(s->rows, 32) * cdiv(s->cols, 32);
    if (tiles > INT32_MAX) return fail(HST_ERR_UNSUPPORTED, "an operand to be copied is too large");
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(s->groups));
    if (e == 2) pack_any_kernel<uint16_t><<<grid, kPackThreads, 0, stream>>>(a);
    else pack_any_kernel<uint8_t><<<grid, kPackThreads, 0, stream>>>(a);
  }
  HST_CUDA(cudaGetLastError());
  s->ptr = dst;
  s->s_col = 1;
  s->s_row = s->packed_row();
  s->s_group = s->s_row * s->rows;
  return HST_OK;
}

template <GroupMode MODE>
int64_t max_iterations(const GroupedProblem& p) {
  const int64_t cols = cdiv(p.cols, 256);
  if (MODE == GroupMode::kWeightGrad) return cols * cdiv(p.lrows, 256) * (p.rows / 64 + p.groups);
  return cols * std::min(p.rows / (group_rows_right(MODE) ? p.width_cap : 256) + p.groups, p.rows) * p.k_blocks;
}

// Iterations a share has at least: below it, joining a tile's pieces costs more than another pair
// saves (421 rows over 8 groups, 520 x 1000, all three products with every tile cut: 75.5, 71.9, 63.6, 63.2
// and 73.9 us with 1, 2, 4, 8 and 16).
constexpr int kMinBlocks = 4;

// K blocks of the deepest tile there can be.
template <GroupMode MODE>
int64_t deepest_tile(const GroupedProblem& p) {
  return MODE == GroupMode::kWeightGrad ? cdiv(p.rows, 64) : p.k_blocks;
}

// K blocks a pair may idle before tiles are cut (GroupShares), from both sides measured (us):
//   forward, 256 wide   1300 x 2560 x 4096, 28 blocks: 30.7 whole, 32.9 cut; 1300 x 4096 x 4096, 45: 43.2 and 43.0
//   forward, 32 wide    16 x 1536 x 4096, 19: 11.4 and 13.5; 16 x 2560 x 4096, 31: 15.1 and 13.9
//   weight gradient     2048 rows, 520 x 1000, 27: 21.3 and 26.4; 4096 rows, 54: 34.7 and 28.7
//   scaled              512 x 4096 x 4096, 18: 22.8 and 28.4; 2048 x 4096 x 9728, 28: 92.3 and 92.7; 257 x 8192 x 12800,
//                       42: 70.9 and 60.7
//   scaled, few rows    1 x 2176 x 12800, 6: 11.6 and 14.8; 128 x 4096 x 2816 over 32 groups, 8: 84.6 and 76.6
// What is cut is written and read as FP32, so that narrow tiles cost less to cut.
template <GroupMode MODE>
int idle_limit(const GroupedProblem& p) {
  if (MODE == GroupMode::kForward) return 24 + 3 * p.width_cap / 32;
  if (MODE == GroupMode::kWeightGrad) return 40;
  return MODE == GroupMode::kScaled ? 24 : 7;
}

// Whether the shares end at tiles whatever the ends are: no tile can be deeper than the limit, or than
// 16 blocks (at 17, few rows in 8 bits: 1 x 2176 x 12800 11.6 us whole and 14.8 cut, 16 x 2176 x 4096 11.5 and 13.5).
constexpr int kWholeBlocks = 16;
template <GroupMode MODE>
bool whole_tiles(const GroupedProblem& p) {
  return deepest_tile<MODE>(p) <= std::max(kWholeBlocks, idle_limit<MODE>(p));
}

template <GroupMode MODE>
int plan_pairs(const GroupedProblem& p, int sms) {
  int64_t most = max_iterations<MODE>(p) / kMinBlocks;
  if (whole_tiles<MODE>(p)) {
    const int64_t cols = cdiv(p.cols, 256);
    most = MODE == GroupMode::kWeightGrad ? cols * cdiv(p.lrows, 256) * std::min<int64_t>(p.groups, p.rows)
                                          : max_iterations<MODE>(p) / std::max<int64_t>(1, p.k_blocks);
  }
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / 2, most)));
}

// Bytes of the pieces, at the start of the workspace; packed operands follow.
template <GroupMode MODE>
size_t piece_bytes(const GroupedProblem& p, int sms) {
  if (whole_tiles<MODE>(p)) return 0;
  return static_cast<size_t>(plan_pairs<MODE>(p, sms)) * 4 * 128 * p.width_cap * sizeof(float);
}

int width_cap(int64_t rows, int most) { return static_cast<int>(std::min<int64_t>(most, round_up(std::max<int64_t>(rows, 1), 32))); }

// The launches of one product. `maps` and the operand fields of `args` are set by the caller.
template <GroupMode MODE, bool L_MN, typename T>
int launch_grouped(const GroupedProblem& p, const GroupedMaps& maps, GroupedArgs args, int r_bytes, const DeviceState* dev,
                   void* workspace, cudaStream_t stream) {
  using S = GroupedShape<MODE>;
  // The schedule counts iterations, and tiles times pairs, in 32 bits.
  if (max_iterations<MODE>(p) * (MODE == GroupMode::kWeightGrad ? 1 : cdiv(dev->sm_count / 2, p.k_blocks)) > INT32_MAX)
    return fail(HST_ERR_UNSUPPORTED, "the grouped product has too many tiles");
  args.groups = p.groups;
  args.rows = static_cast<int>(p.rows);
  args.cols = static_cast<int>(p.cols);
  args.lrows = static_cast<int>(p.lrows);
  args.k_blocks = static_cast<int>(p.k_blocks);
  args.width_cap = p.width_cap;
  args.r_bytes = r_bytes;
  args.pairs = plan_pairs<MODE>(p, dev->sm_count);
  args.min_blocks = kMinBlocks;
  args.idle_limit = idle_limit<MODE>(p);
  args.whole = whole_tiles<MODE>(p);
  if (args.ends == nullptr && MODE != GroupMode::kWeightGrad && args.whole == 0) {  // one group: its tiles are known
    const int tiles = group_row_tiles<MODE>(args, args.rows) * ceil_div(args.cols, 256);
    args.whole = GroupShares(args, tiles, tiles * args.k_blocks, args.k_blocks).whole;
  }
  args.vec = 32;
  while (args.vec > 2 && (p.cols * 2 % args.vec != 0 || reinterpret_cast<uintptr_t>(args.out) % args.vec != 0)) args.vec /= 2;
  args.status = dev->status;
  args.partials = static_cast<float*>(workspace);
  args.piece_floats = 128 * p.width_cap;
  int stages = kMaxStages;
  while (stages > 2 && S::smem_bytes(stages, r_bytes, p.groups, args.pairs) > kMaxDynamicSmem) --stages;
  args.stages = stages;
  {
    static std::atomic<uint64_t> smem_done{0};
    HST_TRY(allow_smem(grouped_gemm_kernel<MODE, L_MN, T>, smem_done));
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(static_cast<unsigned>(2 * args.pairs));
    lc.blockDim = dim3(group_threads(MODE));
    lc.dynamicSmemBytes = S::smem_bytes(stages, r_bytes, p.groups, args.pairs);
    lc.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    HST_CUDA(cudaLaunchKernelEx(&lc, grouped_gemm_kernel<MODE, L_MN, T>, maps, args));
  }
  if (args.whole) return HST_OK;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>(std::max(1, args.pairs - 1)), 2,
                    static_cast<unsigned>(cdiv(args.piece_floats / 128, finish_cols<MODE>())));
  lc.blockDim = dim3(kFinishThreads);
  lc.dynamicSmemBytes = static_cast<size_t>(group_table_ints(p.groups, args.pairs)) * 4;
  lc.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  HST_CUDA(cudaLaunchKernelEx(&lc, grouped_finish_kernel<MODE, T>, args));
  return HST_OK;
}

// A row matrix in boxes of 128 bytes x `box_rows`.
int encode_rows(CUtensorMap* map, CUtensorMapDataType type, const Stack& s, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(s.cols), static_cast<uint64_t>(s.rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(s.s_row * s.elem)};
  const uint32_t box[2] = {static_cast<uint32_t>(128 / s.elem), static_cast<uint32_t>(box_rows)};
  return encode_tiled(map, type, 2, s.ptr, dims, strides, box);
}

// A stack of weights, in boxes within one of them.
int encode_weights(CUtensorMap* map, CUtensorMapDataType type, const Stack& s, int box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(s.cols), static_cast<uint64_t>(s.rows), static_cast<uint64_t>(s.groups)};
  const uint64_t strides[2] = {static_cast<uint64_t>(s.s_row * s.elem), static_cast<uint64_t>(s.s_group * s.elem)};
  const uint32_t box[3] = {static_cast<uint32_t>(128 / s.elem), static_cast<uint32_t>(box_rows), 1};
  return encode_tiled(map, type, 3, s.ptr, dims, strides, box);
}

// Checks the workspace for `pieces` bytes and two operands, and copies those that need it behind the
// pieces.
int place_operands(size_t pieces, Stack* first, const int32_t* first_ends, Stack* second, const int32_t* second_ends,
                   int64_t total_rows, void* workspace, size_t workspace_size, cudaStream_t stream) {
  pieces = static_cast<size_t>(round_up(static_cast<int64_t>(pieces), 256));
  const size_t first_bytes = pack_bytes(*first), need = pieces + first_bytes + pack_bytes(*second);
  if (need > 0 && (workspace_size < need || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
    return fail(HST_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, needed; got %zu", need, workspace_size);
  uint8_t* at = static_cast<uint8_t*>(workspace) + pieces;
  if (!first->readable()) HST_TRY(pack(first, at, first_ends, total_rows, stream));
  if (!second->readable()) HST_TRY(pack(second, at + first_bytes, second_ends, total_rows, stream));
  return HST_OK;
}

// Weights W [groups, k, n] as stored: [k, n] or [n, k] matrices, whichever a tensor map can describe; of
// neither, the one whose rows are contiguous.
Stack stored_weights(const void* w, int64_t groups, int64_t k, int64_t n, int64_t w_group, int64_t w_k, int64_t w_n, bool* kn) {
  const Stack by_k = make_stack(w, 2, groups, k, n, w_group, w_k, w_n);
  const Stack by_n = make_stack(w, 2, groups, n, k, w_group, w_n, w_k);
  *kn = by_k.readable() || (!by_n.readable() && (w_n == 1 || w_k != 1));
  return *kn ? by_k : by_n;
}

int total_bytes(size_t pieces, const Stack& a, const Stack& b, size_t* bytes) {
  *bytes = static_cast<size_t>(round_up(static_cast<int64_t>(pieces), 256)) + pack_bytes(a) + pack_bytes(b);
  return HST_OK;
}

int device_sms(int device, int* sms) {
  HST_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
  return HST_OK;
}

CUtensorMapDataType map_type(int32_t dtype) {
  return dtype == HST_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

int box_rows_of(int index) { return 128 >> index; }

int zero_output(void* out, int64_t values, cudaStream_t stream) {
  if (values > 0) HST_CUDA(cudaMemsetAsync(out, 0, static_cast<size_t>(values) * 2, stream));
  return HST_OK;
}

GroupedProblem forward_problem(int64_t rows, int groups, int64_t n, int64_t k) {
  return GroupedProblem{rows, groups, n, 0, cdiv(k, 64), width_cap(rows, 256)};
}
GroupedProblem grad_problem(int64_t rows, int groups, int64_t lcols, int64_t rcols) {
  return GroupedProblem{rows, groups, rcols, lcols, 0, 256};
}
// Few rows go on the R side (kScaledFew): up to 64 (K = 4096, N = 12800: 64 rows 25.4 us there and 28.9 on the L
// side, 96 rows 35.0 and 30.9), or up to 8 a group on average. How they are spread is known to the GPU alone, and
// a group of many costs 64 rows a tile there, each reading its weight. 4096 x 4096, us there / on the L side:
//   rows a group, groups   even      in a quarter of the groups   in one
//   8 x 32                 135/143   55/57                        31/34
//   8 x 128                418/498   156/152                      82/37
//   16 x 32                141/143   62/57                        49/33
//   64 x 32                160/156   139/64                       137/53
bool scaled_few(int64_t rows, int groups) { return rows <= std::max<int64_t>(64, int64_t(8) * groups); }
GroupedProblem scaled_problem(int64_t rows, int groups, int64_t n, int64_t k) {
  return GroupedProblem{rows, groups, n, 0, cdiv(k, 128), scaled_few(rows, groups) ? width_cap(rows, 64) : 256};
}

size_t scaled_piece_bytes(const GroupedProblem& p, int sms) {
  return scaled_few(p.rows, p.groups) ? piece_bytes<GroupMode::kScaledFew>(p, sms) : piece_bytes<GroupMode::kScaled>(p, sms);
}

}  // namespace
}  // namespace hst

using namespace hst;

extern "C" {

int hst_grouped_matmul_workspace(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_group, int64_t w_k,
                                 int64_t w_n, int32_t groups, int64_t rows, int64_t n, int64_t k, int device,
                                 size_t* bytes) {
  if (bytes == nullptr) return fail(HST_ERR_INVALID, "bytes is null");
  *bytes = 0;
  HST_TRY(check_groups("the grouped matmul", rows, groups, bytes));
  HST_TRY(check_extents("the grouped matmul", n, k));
  if (rows == 0 || n == 0 || k == 0) return HST_OK;
  bool kn = false;
  const Stack xs = make_stack(x, 2, 1, rows, k, 0, x_row, x_col);
  const Stack ws = stored_weights(w, groups, k, n, w_group, w_k, w_n, &kn);
  HST_TRY(check_copies("the grouped matmul", xs, ws));
  int sms = 0;
  HST_TRY(device_sms(device, &sms));
  return total_bytes(piece_bytes<GroupMode::kForward>(forward_problem(rows, groups, n, k), sms), xs, ws, bytes);
}

int hst_grouped_matmul(int32_t dtype, const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_group,
                       int64_t w_k, int64_t w_n, const int32_t* ends, int32_t groups, void* y, int64_t rows, int64_t n,
                       int64_t k, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != HST_F16 && dtype != HST_BF16) return fail(HST_ERR_INVALID, "unknown data type %d", dtype);
  HST_TRY(check_groups("the grouped matmul", rows, groups, ends));
  HST_TRY(check_extents("the grouped matmul", n, k));
  if (rows == 0 || n == 0) return HST_OK;
  if (y == nullptr) return fail(HST_ERR_INVALID, "y is null");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (k == 0) return zero_output(y, rows * n, s);
  if (x == nullptr || w == nullptr) return fail(HST_ERR_INVALID, "x or w is null");
  HST_TRY(check_aligned("x", x, 2));
  HST_TRY(check_aligned("w", w, 2));
  HST_TRY(check_aligned("ends", ends, 4));
  HST_TRY(check_aligned("y", y, 2));
  bool kn = false;
  Stack xs = make_stack(x, 2, 1, rows, k, 0, x_row, x_col);
  Stack ws = stored_weights(w, groups, k, n, w_group, w_k, w_n, &kn);
  HST_TRY(check_copies("the grouped matmul", xs, ws));
  DeviceState* dev = nullptr;
  HST_TRY(device_state(&dev));
  const GroupedProblem p = forward_problem(rows, groups, n, k);
  HST_TRY(place_operands(piece_bytes<GroupMode::kForward>(p, dev->sm_count), &xs, nullptr, &ws, ends, rows, workspace,
                         workspace_bytes, s));
  GroupedMaps maps = {};
  HST_TRY(encode_weights(&maps.l[0], map_type(dtype), ws, kn ? 64 : 128));
  for (int i = 0; i < 4; ++i) HST_TRY(encode_rows(&maps.r[i], map_type(dtype), xs, box_rows_of(i)));
  GroupedArgs args = {};
  args.ends = ends;
  args.out = y;
  const int r_bytes = box_rows_of(group_box(p.width_cap / 2)) * 128;
#define HST_GROUPED_CASE(KN_, DT_, T_) \
  if (kn == KN_ && dtype == DT_) return launch_grouped<GroupMode::kForward, KN_, T_>(p, maps, args, r_bytes, dev, workspace, s);
  HST_GROUPED_CASE(true, HST_F16, __half)
  HST_GROUPED_CASE(false, HST_F16, __half)
  HST_GROUPED_CASE(true, HST_BF16, __nv_bfloat16)
  HST_GROUPED_CASE(false, HST_BF16, __nv_bfloat16)
#undef HST_GROUPED_CASE
  return HST_ERR_UNSUPPORTED;
}

int hst_grouped_weight_grad_workspace(const void* left, int64_t l_row, int64_t l_col, const void* right, int64_t r_row,
                                      int64_t r_col, int32_t groups, int64_t rows, int64_t lcols, int64_t rcols, int device,
                                      size_t* bytes) {
  if (bytes == nullptr) return fail(HST_ERR_INVALID, "bytes is null");
  *bytes = 0;
  HST_TRY(check_groups("the grouped weight gradient", rows, groups, bytes));
  HST_TRY(check_extents("the grouped weight gradient", lcols, rcols));
  if (rows == 0 || lcols == 0 || rcols == 0) return HST_OK;
  const Stack ls = make_stack(left, 2, 1, rows, lcols, 0, l_row, l_col), rs = make_stack(right, 2, 1, rows, rcols, 0, r_row, r_col);
  HST_TRY(check_copies("the grouped weight gradient", ls, rs));
  int sms = 0;
  HST_TRY(device_sms(device, &sms));
  return total_bytes(piece_bytes<GroupMode::kWeightGrad>(grad_problem(rows, groups, lcols, rcols), sms), ls, rs, bytes);
}

int hst_grouped_weight_grad(int32_t dtype, const void* left, int64_t l_row, int64_t l_col, const void* right, int64_t r_row,
                            int64_t r_col, const int32_t* ends, int32_t groups, void* out, int64_t rows, int64_t lcols,
                            int64_t rcols, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != HST_F16 && dtype != HST_BF16) return fail(HST_ERR_INVALID, "unknown data type %d", dtype);
  HST_TRY(check_groups("the grouped weight gradient", rows, groups, ends));
  HST_TRY(check_extents("the grouped weight gradient", lcols, rcols));
  if (lcols == 0 || rcols == 0) return HST_OK;
  if (out == nullptr) return fail(HST_ERR_INVALID, "out is null");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) return zero_output(out, lcols * rcols * groups, s);
  if (left == nullptr || right == nullptr) return fail(HST_ERR_INVALID, "left or right is null");
  HST_TRY(check_aligned("left", left, 2));
  HST_TRY(check_aligned("right", right, 2));
  HST_TRY(check_aligned("ends", ends, 4));
  HST_TRY(check_aligned("out", out, 2));
  Stack ls = make_stack(left, 2, 1, rows, lcols, 0, l_row, l_col), rs = make_stack(right, 2, 1, rows, rcols, 0, r_row, r_col);
  HST_TRY(check_copies("the grouped weight gradient", ls, rs));
  DeviceState* dev = nullptr;
  HST_TRY(device_state(&dev));
  const GroupedProblem p = grad_problem(rows, groups, lcols, rcols);
  HST_TRY(place_operands(piece_bytes<GroupMode::kWeightGrad>(p, dev->sm_count), &ls, nullptr, &rs, nullptr, rows, workspace,
                         workspace_bytes, s));
  GroupedMaps maps = {};
  HST_TRY(encode_rows(&maps.l[0], map_type(dtype), ls, 64));
  HST_TRY(encode_rows(&maps.r[0], map_type(dtype), rs, 64));
  GroupedArgs args = {};
  args.ends = ends;
  args.out = out;
  if (dtype == HST_F16) return launch_grouped<GroupMode::kWeightGrad, true, __half>(p, maps, args, 16384, dev, workspace, s);
  return launch_grouped<GroupMode::kWeightGrad, true, __nv_bfloat16>(p, maps, args, 16384, dev, workspace, s);
}

int hst_matmul_blockscaled_workspace(const void* a, int64_t a_row, int64_t a_col, const void* b, int64_t b_group,
                                     int64_t b_row, int64_t b_col, int32_t groups, int64_t rows, int64_t n, int64_t k,
                                     int device, size_t* bytes) {
  if (bytes == nullptr) return fail(HST_ERR_INVALID, "bytes is null");
  *bytes = 0;
  HST_TRY(check_groups("the block-scaled matmul", rows, groups, bytes));
  HST_TRY(check_extents("the block-scaled matmul", n, k));
  if (rows == 0 || n == 0 || k == 0) return HST_OK;
  const Stack as = make_stack(a, 1, 1, rows, k, 0, a_row, a_col), bs = make_stack(b, 1, groups, n, k, b_group, b_row, b_col);
  HST_TRY(check_copies("the block-scaled matmul", as, bs));
  int sms = 0;
  HST_TRY(device_sms(device, &sms));
  return total_bytes(scaled_piece_bytes(scaled_problem(rows, groups, n, k), sms), as, bs, bytes);
}

int hst_matmul_blockscaled(int32_t out_dtype, const void* a, int64_t a_row, int64_t a_col, const float* a_scales,
                           int64_t sa_row, int64_t sa_block, const void* b, int64_t b_group, int64_t b_row, int64_t b_col,
                           const float* b_scales, int64_t sb_group, int64_t sb_row, int64_t sb_block, const int32_t* ends,
                           int32_t groups, void* y, int64_t rows, int64_t n, int64_t k, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (out_dtype != HST_F16 && out_dtype != HST_BF16) return fail(HST_ERR_INVALID, "unknown data type %d", out_dtype);
  HST_TRY(check_groups("the block-scaled matmul", rows, groups, ends));
  HST_TRY(check_extents("the block-scaled matmul", n, k));
  if (rows == 0 || n == 0) return HST_OK;
  if (y == nullptr) return fail(HST_ERR_INVALID, "y is null");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (k == 0) return zero_output(y, rows * n, s);
  if (a == nullptr || b == nullptr) return fail(HST_ERR_INVALID, "a or b is null");
  if (a_scales == nullptr || b_scales == nullptr) return fail(HST_ERR_INVALID, "scales are null");
  HST_TRY(check_aligned("a_scales", a_scales, 4));
  HST_TRY(check_aligned("b_scales", b_scales, 4));
  HST_TRY(check_aligned("ends", ends, 4));
  HST_TRY(check_aligned("y", y, 2));
  Stack as = make_stack(a, 1, 1, rows, k, 0, a_row, a_col), bs = make_stack(b, 1, groups, n, k, b_group, b_row, b_col);
  HST_TRY(check_copies("the block-scaled matmul", as, bs));
  DeviceState* dev = nullptr;
  HST_TRY(device_state(&dev));
  const GroupedProblem p = scaled_problem(rows, groups, n, k);
  HST_TRY(place_operands(scaled_piece_bytes(p, dev->sm_count), &as, nullptr, &bs, ends, rows, workspace, workspace_bytes, s));
  const CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  GroupedMaps maps = {};
  const bool few = scaled_few(rows, groups);
  for (int i = 0; i < 4; ++i) HST_TRY(encode_rows(few ? &maps.r[i] : &maps.l[i], type, as, box_rows_of(i)));
  HST_TRY(encode_weights(few ? &maps.l[0] : &maps.r[0], type, bs, 128));
  if (!few) HST_TRY(encode_weights(&maps.r[1], type, bs, 64));
  GroupedArgs args = {};
  args.ends = ends;
  args.out = y;
  args.row_scales = a_scales;
  args.rs_row = sa_row;
  args.rs_k = sa_block;
  args.tile_scales = b_scales;
  args.ts_group = sb_group;
  args.ts_n = sb_row;
  args.ts_k = sb_block;
  const int r_bytes = few ? box_rows_of(group_box(p.width_cap / 2)) * 128 : 16384;
#define HST_SCALED_CASE(FEW_, MODE_, DT_, T_) \
  if (few == FEW_ && out_dtype == DT_)        \
    return launch_grouped<GroupMode::MODE_, false, T_>(p, maps, args, r_bytes, dev, workspace, s);
  HST_SCALED_CASE(true, kScaledFew, HST_F16, __half)
  HST_SCALED_CASE(true, kScaledFew, HST_BF16, __nv_bfloat16)
  HST_SCALED_CASE(false, kScaled, HST_F16, __half)
  HST_SCALED_CASE(false, kScaled, HST_BF16, __nv_bfloat16)
#undef HST_SCALED_CASE
  return HST_ERR_UNSUPPORTED;
}

int hst_quantize_e4m3(int32_t dtype, int32_t tiles, const void* x, int64_t x_batch, int64_t x_row, int64_t x_col,
                      void* q, int64_t q_batch, int64_t q_row, float* scales, int64_t s_batch, int64_t s_row,
                      int64_t s_col, int64_t batch, int64_t rows, int64_t cols, void* stream) {
  if (dtype != HST_F16 && dtype != HST_BF16) return fail(HST_ERR_INVALID, "unknown data type %d", dtype);
  HST_TRY(check_extents("the quantiser", rows, cols));
  if (batch < 0 || batch > 65535) return fail(HST_ERR_INVALID, "the quantiser serves at most 65535 matrices");
  if (!tiles && batch > 1) return fail(HST_ERR_INVALID, "row scales are for one matrix");
  if (rows == 0 || cols == 0 || batch == 0) return HST_OK;
  if (x == nullptr || q == nullptr || scales == nullptr) return fail(HST_ERR_INVALID, "null pointer");
  HST_TRY(check_aligned("x", x, 2));
  HST_TRY(check_aligned("scales", scales, 4));
  if (q_row < cols) return fail(HST_ERR_INVALID, "q's rows are shorter than its columns");
  const int64_t col_blocks = cdiv(cols, 128), row_blocks = cdiv(rows, 128);
  if (rows * col_blocks > INT32_MAX || (tiles && row_blocks > 65535))
    return fail(HST_ERR_UNSUPPORTED, "the quantiser's matrix is too large");
  QuantizeArgs a = {x, x_batch, x_row, x_col, static_cast<uint8_t*>(q), q_batch, q_row, scales, s_batch, s_row, s_col,
                    static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(col_blocks)};
  const bool vec = (x_col == 1 || cols == 1) && cols % 8 == 0 && x_row % 8 == 0 && x_batch % 8 == 0 && q_row % 8 == 0 &&
                   q_batch % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tiles) {
    const dim3 grid(static_cast<unsigned>(col_blocks), static_cast<unsigned>(row_blocks), static_cast<unsigned>(batch));
    if (vec && dtype == HST_F16) quantize_tiles_kernel<__half><<<grid, kQuantThreads, 0, st>>>(a);
    else if (vec) quantize_tiles_kernel<__nv_bfloat16><<<grid, kQuantThreads, 0, st>>>(a);
    else if (dtype == HST_F16) quantize_tiles_any_kernel<__half><<<grid, kQuantThreads, 0, st>>>(a);
    else quantize_tiles_any_kernel<__nv_bfloat16><<<grid, kQuantThreads, 0, st>>>(a);
  } else {
    const int64_t units = rows * col_blocks;
    const unsigned vec_grid = static_cast<unsigned>(cdiv(rows, kQuantRows) * cdiv(col_blocks, kQuantBlocks));
    const unsigned any_grid = static_cast<unsigned>(cdiv(units, kQuantThreads / 32));
    if (vec && dtype == HST_F16) quantize_rows_kernel<__half><<<vec_grid, kQuantThreads, 0, st>>>(a);
    else if (vec) quantize_rows_kernel<__nv_bfloat16><<<vec_grid, kQuantThreads, 0, st>>>(a);
    else if (dtype == HST_F16) quantize_rows_any_kernel<__half><<<any_grid, kQuantThreads, 0, st>>>(a);
    else quantize_rows_any_kernel<__nv_bfloat16><<<any_grid, kQuantThreads, 0, st>>>(a);
  }
  HST_CUDA(cudaGetLastError());
  return HST_OK;
}

}  // extern "C"
