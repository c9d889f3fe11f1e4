// C ABI of the grouped products (include/mpe_hip.h); kernels in mpe_grouped_kernel.h.
#include <initializer_list>

#include "../../include/mpe_hip.h"
#include "mpe_grouped_kernel.h"

using namespace mpe;

namespace {

constexpr int kMaxGroups = 1024, kMaxWidth = 1 << 20;
constexpr int64_t kMaxGrid = (1 << 23) - 1;  // workgroups: a launch has less than 2^32 threads, a workgroup up to 512
// rows this far apart (elements of `size` bytes): a tile of 256 of them spans less than a copy may reach
constexpr bool copyable(int64_t ld, int size) { return ld < (int64_t)kGroupedSpan / (256 * size) - 16; }
static_assert(copyable(kMaxWidth, 4) && copyable(kMaxWidth, 2), "packed rows and weights always are");

int dtype_size(int dtype) { return dtype == MPE_F32 ? 4 : 2; }
bool bad_align(const void *p, int size) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }

int grouped_check(const mpe_grouped_desc *d) {
  if (!d || !d->ends) return MPE_ERR_NULL;
  if (d->dtype != MPE_F32 && d->dtype != MPE_BF16 && d->dtype != MPE_F16) return MPE_ERR_UNSUPPORTED;
  if (d->groups < 1 || d->groups > kMaxGroups || d->n < 1 || d->k < 1 || d->rows < 0 || d->rows > INT32_MAX) return MPE_ERR_ARG;
  if (d->n > kMaxWidth || d->k > kMaxWidth || (int64_t)d->n * d->k > INT32_MAX) return MPE_ERR_ARG;
  if (d->ends64 != 0 && d->ends64 != 1) return MPE_ERR_ARG;
  if (bad_align(d->ends, d->ends64 ? 8 : 4)) return MPE_ERR_ALIGN;
  return MPE_OK;
}

// ---- what the tiles are copied from --------------------------------------------------------------------------------------
// A matrix of the call, and whether it is packed into the workspace first: a tile (256 lines) of it would span too much, or it
// is masked and its readers do not apply the mask.  The larger tiles have no room for it; the small ones load and apply it once
// per 64 columns of x, which pays while those are few (rows x k x n in groups, us, mask in the tiles / masked first):
// f32 4 096 x 64 x 64 in 4 9.6 / 11.4, 32 768 x 64 x 64 in 8 17.9 / 24.2, 4 096 x 256 x 256 in 8 23.2 / 27.1, 1 024 x 512 x 512 in 4
// 27.5 / 26.9, 16 384 x 512 x 512 in 16 180 / 163; fp16 5 003 x 333 x 517 in 7 33 / 27.
constexpr int kMaskCols = 256;
struct Matrix {
  const void *p, *mask;
  int64_t ld, ld_mask, lines, at;  // at: offset in the workspace, or -1
  int cols;
};

struct Workspace {
  int size;  // of an element
  int64_t total = 0;
  GroupedPacks packs{};
  int jobs = 0;
  int64_t blocks = 0;

  int chunk() const { return 16 / size; }
  int64_t packed_ld(const Matrix &m) const { return (m.cols + chunk() - 1) / chunk() * chunk(); }
  int64_t take(int64_t bytes) {
    const int64_t at = total;
    total += (bytes + 15) / 16 * 16;
    return at;
  }
  // masks: the kernel that reads m applies its mask
  void plan(Matrix &m, bool masks = false) {
    const bool as_it_is = copyable(m.ld, size) && (!m.mask || (masks && copyable(m.ld_mask, size)));
    m.at = m.lines > 0 && !as_it_is ? take(m.lines * packed_ld(m) * size) : -1;
  }
  // after the plan: the matrix as the kernels read it
  void place(Matrix &m, void *base) {
    if (m.at < 0) return;
    GroupedPack &j = packs.job[jobs++];
    const int64_t chunks = packed_ld(m) / chunk();  // of a line; workgroups as grouped_pack_kernel counts them
    const int64_t many = chunks <= 256 ? (m.lines + 256 / chunks - 1) / (256 / chunks) : m.lines * ((chunks + 255) / 256);
    j = GroupedPack{m.p, m.mask, (char *)base + m.at, m.ld, m.ld_mask, m.lines, m.cols, (int)(many < kMaxGrid ? many : kMaxGrid)};
    blocks += many;
    m.p = j.dst;
    m.ld = packed_ld(m);
    m.mask = nullptr;
  }
  int run(int dtype, hipStream_t s) {
    if (jobs == 0) return MPE_OK;
    if (blocks > kMaxGrid) return MPE_ERR_ARG;
    const dim3 grid((unsigned)blocks), block(256);
    if (dtype == MPE_F32) hipLaunchKernelGGL(grouped_pack_kernel<float>, grid, block, 0, s, packs);
    else if (dtype == MPE_BF16) hipLaunchKernelGGL(grouped_pack_kernel<__bf16>, grid, block, 0, s, packs);
    else hipLaunchKernelGGL(grouped_pack_kernel<_Float16>, grid, block, 0, s, packs);
    return (int)hipGetLastError();
  }
};

// ---- tiles ---------------------------------------------------------------------------------------------------------------
// Tiles (rows x columns of the output, wavefronts): small 64 x 64 (2 x 2), middle 128 x 128 (2 x 2), large 256 x 256 (2 x 4).
enum Tile { SMALL = 0, MIDDLE = 1, LARGE = 2 };
constexpr int kTile[3] = {64, 128, 256};

// A 16-bit product is bound by what the tiles read per matrix instruction: the largest tile that still leaves every CU a
// workgroup and does not mostly overhang its group's rows.  f32 matrix instructions are 16 times slower: small tiles.
// mean_rows: of a group; rows: of all; others: independent products.  The host knows the mean only (`ends` is on the device); forward
// and dx count their tiles on the device and hold their speed where one group has all rows (32 768 x 512 x 512 bf16 in 64: 30 us even,
// 40 with half of the rows in one group, 30 with all of them).
// bf16 forward, us (small / middle / large, rows x k x n in groups): 4 096 x 512 x 512 in 16 8.6 / 11.1 / 22, 8 192 x 1 024 x 1 024 in
// 16 37 / 28 / 36, 16 384 x 512 x 512 in 16 22 / 18 / 26, 32 768 x 512 x 512 in 32 41 / 32 / 28; dweight: 8 192 x 1 024 x 1 024 in 16
// 43 / 33 / 30, 32 768 x 512 x 512 in 32 34 / 27 / 42.  The large tile has no registers for n or k that end inside a chunk.
Tile pick_tile(const mpe_grouped_desc *d, int64_t mean_rows, int64_t cols, int64_t rows, int64_t others) {
  if (d->dtype == MPE_F32) return SMALL;
  const auto tiles = [&](int64_t t) { return (rows + t - 1) / t * ((cols + t - 1) / t) * others; };
  if (mean_rows >= 384 && cols >= 256 && tiles(256) >= 256 && d->n % 8 == 0 && d->k % 8 == 0) return LARGE;
  if (mean_rows >= 96 && cols >= 96 && tiles(128) >= 256) return MIDDLE;
  return SMALL;
}

// dweight: rows and columns of the output are n and k, the contraction runs over the group's rows.
Tile dw_tile(const mpe_grouped_desc *d) { return pick_tile(d, d->n, d->k, d->n, d->groups); }
int64_t dw_tiles(const mpe_grouped_desc *d) {
  const int t = kTile[dw_tile(d)];
  return (int64_t)((d->n + t - 1) / t) * ((d->k + t - 1) / t) * d->groups;
}
// Where the outputs are few tiles that each run over many rows, a group's rows are split over workgroups and the partial sums
// joined.  The join is a launch (4 us) and 8 bytes a partial sum: the split with the least sum of both, from the rows a tile gets
// through per us.  f32 65 536 x 64 x 64 in 64 groups 28 us as one, 15 in eight parts; bf16 4 096 x 256 x 256 in 8 7.2 as one, 12 in
// four, 8 192 x 512 x 512 in 4 17 as one, 19 in two.  Large tiles are enough by pick_tile's rule.
// Its limit: the split is for groups of the mean size.  A group of most of the rows runs through them in the same few parts while the
// chip idles (dweight, us, even groups / half of the rows in one / all: f32 65 536 x 64 x 64 in 64 16 / 104 / 195, in 1 024 16 / 747 /
// 1 486; bf16 65 536 x 256 x 256 in 64 23 / 443 / 889, 16 384 x 1 024 x 1 024 in 16 48 / 224 / 436).
int dw_splits(const mpe_grouped_desc *d) {
  const Tile tile = dw_tile(d);
  if (tile == LARGE) return 1;
  const int64_t tiles = dw_tiles(d), mean = d->rows / d->groups;
  const double rate = d->dtype == MPE_F32 ? 44.0 : tile == SMALL ? 142.0 : 64.0;
  const double sums = (double)d->groups * d->n * d->k;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && (s == 1 || mean / s >= 64); s *= 2) {
    const int64_t rounds = (tiles * s + 511) / 512;  // two workgroups a CU at a time
    const double us = (double)mean / s / rate * (double)rounds + (s > 1 ? 4.0 + s * sums * 8 / 4e6 : 0.0);
    if (s == 1 || us < least) {
      least = us;
      best = s;
    }
  }
  return best;
}

// ---- launches ------------------------------------------------------------------------------------------------------------
template <typename T, int MODE>
int launch(const GroupedArgs &a, Tile tile, int64_t grid, hipStream_t s) {
  if (grid > kMaxGrid) return MPE_ERR_ARG;
  const dim3 blocks((unsigned)grid);
  if (sizeof(T) == 2 && tile == LARGE) {
    if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((grouped_kernel<T, MODE, 256, 256, 2, 4, 4, 4>), blocks, dim3(512), 0, s, a);
  } else if (sizeof(T) == 2 && tile == MIDDLE) {
    if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((grouped_kernel<T, MODE, 128, 128, 2, 2, 4, 4>), blocks, dim3(256), 0, s, a);
  } else if constexpr (sizeof(T) == 2 || MODE == GROUPED_FWD) {  // an f32 backward is grouped_both_kernel's
    hipLaunchKernelGGL((grouped_kernel<T, MODE, 64, 64, 2, 2, 8, 2>), blocks, dim3(256), 0, s, a);
  }
  return (int)hipGetLastError();
}

// tiles over a.rows (forward, dx): groups (and the tail) with rows may each add a partial tile
int64_t rows_grid(GroupedArgs &a, Tile tile, int64_t cols) {
  a.tiles_j = (int)((cols + kTile[tile] - 1) / kTile[tile]);
  const int64_t most = a.groups + 1 < a.rows ? a.groups + 1 : a.rows;
  return (a.rows / kTile[tile] + most) * a.tiles_j;
}
Tile rows_tile(const mpe_grouped_desc *d, int64_t cols) { return pick_tile(d, d->rows / d->groups, cols, d->rows, 1); }

template <typename T, int MODE>
int launch_rows(GroupedArgs a, const mpe_grouped_desc *d, hipStream_t s) {
  const int64_t cols = MODE == GROUPED_FWD ? d->n : d->k;
  const Tile tile = rows_tile(d, cols);
  const int64_t grid = rows_grid(a, tile, cols);
  return launch<T, MODE>(a, tile, grid, s);
}

template <typename T>
int launch_join(const GroupedArgs &a, hipStream_t s) {
  if (a.splits == 1) return MPE_OK;
  const int64_t cw = (int64_t)a.groups * a.n * a.k, cb = a.dbias ? (int64_t)a.groups * a.n : 0;
  hipLaunchKernelGGL(grouped_join_kernel<T>, dim3((unsigned)((cw + 1023) / 1024 + (cb + 1023) / 1024)), dim3(256), 0, s, a.part,
                     (T *)a.out, cw, a.part_bias, (T *)a.dbias, cb, a.splits);
  return (int)hipGetLastError();
}

// dx and dw: w.tiles_* and w.splits are set
template <typename T>
int launch_backward(GroupedArgs x, const GroupedArgs &w, const mpe_grouped_desc *d, hipStream_t s) {
  const Tile tx = rows_tile(d, d->k), tw = dw_tile(d);
  const int64_t nx = x.out ? rows_grid(x, tx, d->k) : 0, nw = w.out ? dw_tiles(d) * w.splits : 0;
  if (nx + nw + 7 > kMaxGrid) return MPE_ERR_ARG;
  int rc = MPE_OK;
  if (tx == tw || nx == 0 || nw == 0) {
    if (nx + nw > 0) {
      const dim3 grid((unsigned)(nx + (nw + 7) / 8 * 8));
      const Tile tile = nw ? tw : tx;
      if (sizeof(T) == 2 && tile == LARGE) {
        if constexpr (sizeof(T) == 2)
          hipLaunchKernelGGL((grouped_both_kernel<T, 256, 256, 2, 4, 4, 4, false>), grid, dim3(512), 0, s, x, w, (int)nw);
      } else if (sizeof(T) == 2 && tile == MIDDLE) {
        if constexpr (sizeof(T) == 2)
          hipLaunchKernelGGL((grouped_both_kernel<T, 128, 128, 2, 2, 4, 4, false>), grid, dim3(256), 0, s, x, w, (int)nw);
      } else if (x.mask) {
        hipLaunchKernelGGL((grouped_both_kernel<T, 64, 64, 2, 2, 8, 2, true>), grid, dim3(256), 0, s, x, w, (int)nw);
      } else {
        hipLaunchKernelGGL((grouped_both_kernel<T, 64, 64, 2, 2, 8, 2, false>), grid, dim3(256), 0, s, x, w, (int)nw);
      }
      rc = (int)hipGetLastError();
    }
  } else {
    rc = launch<T, GROUPED_DW>(w, tw, nw, s);
    if (!rc) rc = launch<T, GROUPED_DX>(x, tx, nx, s);
  }
  return rc || !w.out ? rc : launch_join<T>(w, s);
}

#define GROUPED_BY_TYPE(dtype, F, ...) \
  ((dtype) == MPE_F32 ? F<float __VA_ARGS__ : (dtype) == MPE_BF16 ? F<__bf16 __VA_ARGS__ : F<_Float16 __VA_ARGS__)

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

Matrix rows_of(const mpe_grouped_desc *d, const void *p, int64_t ld, int cols) { return Matrix{p, nullptr, ld, 0, d->rows, -1, cols}; }

struct Forward {
  Matrix x;
  Workspace ws;
  Forward(const mpe_grouped_desc *d, const void *px, int64_t ld_x) : x(rows_of(d, px, ld_x, d->k)), ws{dtype_size(d->dtype)} { ws.plan(x); }
};

// The gradient of the result, the operands that are wanted, and the partial sums of dweight and dbias.
struct Backward {
  Matrix d_, x;
  Workspace ws;
  bool small;  // all tiles: one launch, which applies the mask itself
  int64_t part = 0, part_bias = 0;
  Backward(const mpe_grouped_desc *d, const void *dy, int64_t ld_dy, const void *y, int64_t ld_y, const void *px, int64_t ld_x, bool dx,
           bool dw)
      : d_(rows_of(d, dy, ld_dy, d->n)), x(rows_of(d, px, ld_x, d->k)), ws{dtype_size(d->dtype)},
        small((!dx || rows_tile(d, d->k) == SMALL) && (!dw || dw_tile(d) == SMALL)) {
    d_.mask = y;
    d_.ld_mask = ld_y;
    if (dx || dw) ws.plan(d_, small && d->k <= kMaskCols);
    if (dw) ws.plan(x);
    const int splits = dw_splits(d);
    if (dw && splits > 1) {
      const int64_t one = (int64_t)splits * d->groups * d->n * 4;
      part = ws.take(one * d->k);
      part_bias = ws.take(one);
    }
  }
};

}  // namespace

extern "C" int64_t mpe_grouped_linear_workspace(const mpe_grouped_desc *d, const void *x, int64_t ld_x, const void * /*weight*/) {
  if (const int rc = grouped_check(d)) return rc;
  return Forward(d, x, ld_x).ws.total;
}

extern "C" int mpe_grouped_linear(const mpe_grouped_desc *d, const void *x, int64_t ld_x, const void *weight, const void *bias,
                                  void *y, int64_t ld_y, int relu, int zero_tail, void *workspace, int64_t workspace_bytes,
                                  void *stream) {
  if (const int rc = grouped_check(d)) return rc;
  if (relu != 0 && relu != 1) return MPE_ERR_ARG;
  if (zero_tail != 0 && zero_tail != 1) return MPE_ERR_ARG;
  if (d->rows == 0) return MPE_OK;
  if (!x || !weight || !y) return MPE_ERR_NULL;
  if (ld_x < d->k || ld_y < d->n) return MPE_ERR_ARG;
  const int size = dtype_size(d->dtype);
  for (const void *p : {x, weight, bias, (const void *)y})
    if (bad_align(p, size)) return MPE_ERR_ALIGN;
  if (bad_align(workspace, 16)) return MPE_ERR_ALIGN;
  Forward f(d, x, ld_x);
  if (f.ws.total > 0 && !workspace) return MPE_ERR_NULL;
  if (workspace_bytes < f.ws.total) return MPE_ERR_SCRATCH;
  hipStream_t s = (hipStream_t)stream;
  f.ws.place(f.x, workspace);
  if (const int rc = f.ws.run(d->dtype, s)) return rc;
  GroupedArgs a = base_args(d);
  a.a = f.x.p;
  a.ld_a = f.x.ld;
  a.b = weight;
  a.ld_b = d->k;
  a.bias = bias;
  a.out = y;
  a.ld_out = ld_y;
  a.relu = relu;
  a.zero_tail = zero_tail;
  return GROUPED_BY_TYPE(d->dtype, launch_rows, , GROUPED_FWD>(a, d, s));
}

extern "C" int64_t mpe_grouped_backward_workspace(const mpe_grouped_desc *d, const void *dy, int64_t ld_dy, const void *y, int64_t ld_y,
                                                  const void *x, int64_t ld_x, const void * /*weight*/, int with_dx, int with_dweight) {
  if (const int rc = grouped_check(d)) return rc;
  if (with_dx < 0 || with_dx > 1 || with_dweight < 0 || with_dweight > 1) return MPE_ERR_ARG;
  return Backward(d, dy, ld_dy, y, ld_y, x, ld_x, with_dx, with_dweight).ws.total;
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
  Backward b(d, dy, ld_dy, y, ld_y, x, ld_x, dx != nullptr, dweight != nullptr);
  if (b.ws.total > 0 && !workspace) return MPE_ERR_NULL;
  if (workspace_bytes < b.ws.total) return MPE_ERR_SCRATCH;
  hipStream_t s = (hipStream_t)stream;
  b.ws.place(b.d_, workspace);
  b.ws.place(b.x, workspace);
  if (const int rc = b.ws.run(d->dtype, s)) return rc;
  GroupedArgs a = base_args(d);
  a.a = b.d_.p;
  a.ld_a = b.d_.ld;
  a.mask = b.d_.mask;
  a.ld_mask = b.d_.ld_mask;
  GroupedArgs gx = a, gw = a;
  if (dx && d->rows > 0) {
    gx.b = weight;
    gx.ld_b = d->k;
    gx.out = dx;
    gx.ld_out = ld_dx;
    gx.zero_tail = zero_tail;
  }
  if (dweight) {
    gw.b = b.x.p;
    gw.ld_b = b.x.ld;
    gw.out = dweight;
    gw.dbias = dbias;
    gw.part = (float *)((char *)workspace + b.part);
    gw.part_bias = (float *)((char *)workspace + b.part_bias);
    const int t = kTile[dw_tile(d)];
    gw.tiles_i = (d->n + t - 1) / t;
    gw.tiles_j = (d->k + t - 1) / t;
    gw.splits = dw_splits(d);
  }
  return GROUPED_BY_TYPE(d->dtype, launch_backward, >(gx, gw, d, s));
}
