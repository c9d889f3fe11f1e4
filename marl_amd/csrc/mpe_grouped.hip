// C ABI of the grouped products (include/mpe_hip.h); kernels in mpe_grouped_kernel.h.
#include <initializer_list>

#include "../../include/mpe_hip.h"
#include "mpe_grouped_kernel.h"

using namespace mpe;
#ifndef MKC
#define MKC 4
#define MST 4
#endif
#ifndef SKC
#define SKC 8
#define SST 2
#endif
#ifndef MASKSH
#define MASKSH 18
#endif
#ifndef LBN
#define LBN 256
#define LWM 2
#define LWN 4
#define LKC 4
#define LST 4
#endif
#ifndef LARGE_MEAN
#define LARGE_MEAN 384
#endif

namespace {

constexpr int kMaxGroups = 1024;
constexpr int64_t kMaxGrid = 0x7fffffff;

int dtype_size(int dtype) { return dtype == MPE_F32 ? 4 : 2; }
bool bad_align(const void *p, int size) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }

int grouped_check(const mpe_grouped_desc *d) {
  if (!d || !d->ends) return MPE_ERR_NULL;
  if (d->dtype != MPE_F32 && d->dtype != MPE_BF16 && d->dtype != MPE_F16) return MPE_ERR_UNSUPPORTED;
  if (d->groups < 1 || d->groups > kMaxGroups || d->n < 1 || d->k < 1 || d->rows < 0 || d->rows > INT32_MAX) return MPE_ERR_ARG;
  if ((int64_t)d->n * d->k > INT32_MAX) return MPE_ERR_ARG;
  if (d->ends64 != 0 && d->ends64 != 1) return MPE_ERR_ARG;
  if (bad_align(d->ends, d->ends64 ? 8 : 4)) return MPE_ERR_ALIGN;
  return MPE_OK;
}

// Tiles (rows x columns of the output, wavefronts): small 64 x 64 (2 x 2), middle 128 x 128 (2 x 2), large 256 x 256 (2 x 4).
enum Tile { SMALL = 0, MIDDLE = 1, LARGE = 2 };
constexpr int kTile[3] = {64, 128, 256}, kTileJ[3] = {64, 128, LBN};

// A 16-bit product is bound by what the tile reads from LDS per matrix instruction: the largest tile that still leaves every
// CU a workgroup and does not mostly overhang its group's rows.  f32 matrix instructions are 16 times slower: small tiles.
Tile pick_tile(int dtype, bool fast, int64_t mean_rows, int64_t cols, int64_t groups_rows, int64_t others) {
  if (dtype == MPE_F32) return SMALL;
  const auto tiles = [&](int64_t t) { return (groups_rows + t - 1) / t * ((cols + t - 1) / t) * others; };
  if (fast && mean_rows >= LARGE_MEAN && cols >= 256 && tiles(256) >= 256) return LARGE;
  if (mean_rows >= 96 && cols >= 96 && tiles(128) >= 256) return MIDDLE;
  return SMALL;
}

// dweight: rows and columns of the output are n and k, the contraction runs over the group's rows.
Tile dw_tile(const mpe_grouped_desc *d, bool fast) { return pick_tile(d->dtype, fast, d->n, d->k, d->n, d->groups); }
int64_t dw_tiles(const mpe_grouped_desc *d, Tile t) {
  return (int64_t)((d->n + kTile[t] - 1) / kTile[t]) * ((d->k + kTileJ[t] - 1) / kTileJ[t]);
}
// Where the outputs are too few tiles to fill the chip, each group's rows are split; goes by sizes alone (the workspace is
// made before the call).  Enough tiles for the large one are enough not to split.
int dw_splits(const mpe_grouped_desc *d) {
  const int64_t tiles = dw_tiles(d, dw_tile(d, false)) * d->groups, mean = d->rows / d->groups;
  int s = 1;
  while (s < 64 && tiles * s < 512 && mean / (s * 2) >= 64) s *= 2;
  return s;
}

GroupedArgs base_args(const mpe_grouped_desc *d) {
  GroupedArgs a{};
  a.ends = d->ends;
  a.ends64 = d->ends64;
  a.rows = d->rows;
  a.groups = d->groups;
  a.n = d->n;
  a.k = d->k;
  a.splits = 1;
  return a;
}

template <typename T, int MODE, int BM, int BN, int WM, int WN, int PATH, int KC, int STAGES>
int launch_tile(const GroupedArgs &a, int64_t grid, hipStream_t s) {
  if (grid > kMaxGrid) return MPE_ERR_ARG;
  hipLaunchKernelGGL((grouped_kernel<T, MODE, BM, BN, WM, WN, PATH, KC, STAGES>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, s, a);
  return (int)hipGetLastError();
}

template <typename T, int MODE, int PATH>
int launch_as(const GroupedArgs &a, Tile tile, int64_t grid, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (PATH == GROUPED_FAST)
      if (tile == LARGE) return launch_tile<T, MODE, 256, LBN, LWM, LWN, PATH, LKC, LST>(a, grid, s);
    if (tile != SMALL) return launch_tile<T, MODE, 128, 128, 2, 2, PATH, PATH == GROUPED_FAST ? MKC : 8, PATH == GROUPED_FAST ? MST : 2>(a, grid, s);
  }
  return launch_tile<T, MODE, 64, 64, 2, 2, PATH, PATH == GROUPED_FAST ? SKC : 8, PATH == GROUPED_FAST ? SST : 2>(a, grid, s);
}

template <typename T, int MODE>
int launch(const GroupedArgs &a, bool fast, Tile tile, int64_t grid, hipStream_t s) {
  if (!fast) return launch_as<T, MODE, GROUPED_ANY>(a, tile, grid, s);
  if constexpr (MODE != GROUPED_FWD)
    if (a.mask) return launch_as<T, MODE, GROUPED_FAST_MASK>(a, tile, grid, s);
  return launch_as<T, MODE, GROUPED_FAST>(a, tile, grid, s);
}

template <typename T, int MODE>
int launch_rows(GroupedArgs a, bool fast, int dtype, int cols, hipStream_t s) {
  const Tile tile = pick_tile(dtype, fast && !a.mask, a.rows / a.groups, cols, a.rows, 1);
  a.tiles_j = (cols + kTileJ[tile] - 1) / kTileJ[tile];
  const int64_t most = a.groups + 1 < a.rows ? a.groups + 1 : a.rows;  // groups (and the tail) with rows: each may add a partial tile
  return launch<T, MODE>(a, fast, tile, (a.rows / kTile[tile] + most) * a.tiles_j, s);
}

template <typename T>
int launch_dw(GroupedArgs a, const mpe_grouped_desc *d, bool fast, hipStream_t s) {
  const Tile tile = dw_tile(d, fast && !a.mask);
  a.tiles_i = (d->n + kTile[tile] - 1) / kTile[tile];
  a.tiles_j = (d->k + kTileJ[tile] - 1) / kTileJ[tile];
  a.splits = dw_splits(d);
  const int rc = launch<T, GROUPED_DW>(a, fast, tile, dw_tiles(d, tile) * a.splits * a.groups, s);
  if (rc || a.splits == 1) return rc;
  const int64_t cw = (int64_t)a.groups * a.n * a.k, cb = a.dbias ? (int64_t)a.groups * a.n : 0;
  hipLaunchKernelGGL(grouped_join_kernel<T>, dim3((unsigned)((cw + 1023) / 1024 + (cb + 1023) / 1024)), dim3(256), 0, s, a.part,
                     (T *)a.out, cw, a.part_bias, (T *)a.dbias, cb, a.splits);
  return (int)hipGetLastError();
}

// An array that tiles may be copied from: dwords stay dwords from row to row, a tile (256 lines) spans less than kGroupedSpan
bool copyable(const void *p, int64_t ld, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 3) == 0 && ld * size % 4 == 0 && ld < (int64_t)kGroupedSpan / (256 * size) - 16;
}

template <int MODE>
int launch_type(const GroupedArgs &a, int dtype, bool fast, int cols, hipStream_t s) {
  return dtype == MPE_F32    ? launch_rows<float, MODE>(a, fast, dtype, cols, s)
         : dtype == MPE_BF16 ? launch_rows<__bf16, MODE>(a, fast, dtype, cols, s)
                             : launch_rows<_Float16, MODE>(a, fast, dtype, cols, s);
}

}  // namespace

extern "C" int mpe_grouped_linear(const mpe_grouped_desc *d, const void *x, int64_t ld_x, const void *weight, const void *bias,
                                  void *y, int64_t ld_y, int relu, int zero_tail, void *stream) {
  if (const int rc = grouped_check(d)) return rc;
  if (relu != 0 && relu != 1) return MPE_ERR_ARG;
  if (zero_tail != 0 && zero_tail != 1) return MPE_ERR_ARG;
  if (d->rows == 0) return MPE_OK;
  if (!x || !weight || !y) return MPE_ERR_NULL;
  if (ld_x < d->k || ld_y < d->n) return MPE_ERR_ARG;
  const int size = dtype_size(d->dtype);
  if (bad_align(x, size) || bad_align(weight, size) || bad_align(bias, size) || bad_align(y, size)) return MPE_ERR_ALIGN;
  GroupedArgs a = base_args(d);
  a.a = x;
  a.ld_a = ld_x;
  a.b = weight;
  a.ld_b = d->k;
  a.bias = bias;
  a.out = y;
  a.ld_out = ld_y;
  a.relu = relu;
  a.zero_tail = zero_tail;
  const bool fast = copyable(x, ld_x, size) && copyable(weight, d->k, size);
  return launch_type<GROUPED_FWD>(a, d->dtype, fast, d->n, (hipStream_t)stream);
}

namespace {

// A masked gradient is written once (in rows of whole chunks) and read by plain copies where there is enough of it; otherwise
// each product masks what it loads.
bool mask_first(const mpe_grouped_desc *d) { return d->rows * d->n >= (int64_t)1 << MASKSH; }
int64_t masked_ld(const mpe_grouped_desc *d) {
  const int chunk = 16 / dtype_size(d->dtype);
  return (d->n + chunk - 1) / chunk * chunk;
}

// Scratch of a backward pass: the masked gradient, the partial sums of dweight and of dbias.
struct Scratch { int64_t masked, part, part_bias, total; };
Scratch scratch_of(const mpe_grouped_desc *d, bool masked, bool want_dw) {
  const int splits = dw_splits(d);
  const auto up = [](int64_t b) { return (b + 15) / 16 * 16; };
  Scratch s{};
  s.part = masked ? up(d->rows * masked_ld(d) * dtype_size(d->dtype)) : 0;
  const int64_t one = want_dw && splits > 1 ? (int64_t)splits * d->groups * d->n * 4 : 0;
  s.part_bias = s.part + up(one * d->k);
  s.total = s.part_bias + up(one);
  return s;
}

template <typename T>
int launch_mask(const void *dy, int64_t ld_dy, const void *y, int64_t ld_y, void *out, int64_t rows, int n, hipStream_t s) {
  constexpr int chunk = 16 / (int)sizeof(T);
  const int64_t grid = (rows * ((n + chunk - 1) / chunk) + 255) / 256;
  if (grid > kMaxGrid) return MPE_ERR_ARG;
  hipLaunchKernelGGL(grouped_mask_kernel<T>, dim3((unsigned)grid), dim3(256), 0, s, (const T *)dy, ld_dy, (const T *)y, ld_y, (T *)out, rows, n);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int64_t mpe_grouped_backward_workspace(const mpe_grouped_desc *d, int with_y, int with_dweight) {
  if (const int rc = grouped_check(d)) return rc;
  if (with_y < 0 || with_y > 1 || with_dweight < 0 || with_dweight > 1) return MPE_ERR_ARG;
  return scratch_of(d, with_y && mask_first(d), with_dweight).total;
}

extern "C" int mpe_grouped_linear_backward(const mpe_grouped_desc *d, const void *dy, int64_t ld_dy, const void *y, int64_t ld_y,
                                           const void *x, int64_t ld_x, const void *weight, void *dx, int64_t ld_dx, int zero_tail,
                                           void *dweight, void *dbias, void *workspace, int64_t workspace_bytes, void *stream) {
  if (const int rc = grouped_check(d)) return rc;
  if (zero_tail != 0 && zero_tail != 1) return MPE_ERR_ARG;
  if (dbias && !dweight) return MPE_ERR_NULL;
  if (d->rows > 0 && (!dy || (dx && !weight) || (dweight && !x))) return MPE_ERR_NULL;
  if (d->rows > 0 && (ld_dy < d->n || (y && ld_y < d->n) || (dx && ld_dx < d->k) || (dweight && ld_x < d->k))) return MPE_ERR_ARG;
  const int size = dtype_size(d->dtype);
  for (const void *p : {dy, y, x, weight, (const void *)dx, (const void *)dweight, (const void *)dbias})
    if (bad_align(p, size)) return MPE_ERR_ALIGN;
  if (bad_align(workspace, 16)) return MPE_ERR_ALIGN;
  const bool masked = y && mask_first(d);
  const Scratch w = scratch_of(d, masked, dweight != nullptr);
  if (w.total > 0 && !workspace) return MPE_ERR_NULL;
  if (workspace_bytes < w.total) return MPE_ERR_SCRATCH;
  hipStream_t s = (hipStream_t)stream;
  if (masked) {
    const int rc = d->dtype == MPE_F32    ? launch_mask<float>(dy, ld_dy, y, ld_y, workspace, d->rows, d->n, s)
                   : d->dtype == MPE_BF16 ? launch_mask<__bf16>(dy, ld_dy, y, ld_y, workspace, d->rows, d->n, s)
                                          : launch_mask<_Float16>(dy, ld_dy, y, ld_y, workspace, d->rows, d->n, s);
    if (rc) return rc;
    dy = workspace;
    ld_dy = masked_ld(d);
    y = nullptr;
  }
  const bool fast_d = d->rows > 0 && copyable(dy, ld_dy, size);
  GroupedArgs a = base_args(d);
  a.a = dy;
  a.ld_a = ld_dy;
  a.mask = y;
  a.ld_mask = ld_y;
  if (dx && d->rows > 0) {
    GroupedArgs b = a;
    b.b = weight;
    b.ld_b = d->k;
    b.out = dx;
    b.ld_out = ld_dx;
    b.zero_tail = zero_tail;
    if (const int rc = launch_type<GROUPED_DX>(b, d->dtype, fast_d && copyable(weight, d->k, size), d->k, s)) return rc;
  }
  if (!dweight) return MPE_OK;
  a.b = x;
  a.ld_b = ld_x;
  a.out = dweight;
  a.dbias = dbias;
  a.part = (float *)((char *)workspace + w.part);
  a.part_bias = (float *)((char *)workspace + w.part_bias);
  return d->dtype == MPE_F32    ? launch_dw<float>(a, d, fast_d && copyable(x, ld_x, size), s)
         : d->dtype == MPE_BF16 ? launch_dw<__bf16>(a, d, fast_d && copyable(x, ld_x, size), s)
                                : launch_dw<_Float16>(a, d, fast_d && copyable(x, ld_x, size), s);
}
