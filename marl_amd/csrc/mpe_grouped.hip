// C ABI of the grouped products (include/mpe_hip.h); kernels in mpe_grouped_kernel.h.
#include "../../include/mpe_hip.h"
#include "mpe_grouped_kernel.h"

using namespace mpe;

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

struct DwPlan { int tiles_i, tiles_j, splits; };

constexpr int kBM = 64, kBN = 64;

DwPlan dw_plan(const mpe_grouped_desc *d) {
  DwPlan p{(d->n + kBM - 1) / kBM, (d->k + kBN - 1) / kBN, 1};
  const int64_t tiles = (int64_t)p.tiles_i * p.tiles_j * d->groups;
  const int64_t mean = d->rows / d->groups;
  while (p.splits < 64 && tiles * p.splits < 512 && mean / (p.splits * 2) >= 64) p.splits *= 2;
  return p;
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

template <typename T, int MODE>
int launch_rows(GroupedArgs a, int cols, hipStream_t s) {
  a.tiles_j = (cols + kBN - 1) / kBN;
  const int64_t most = a.groups + 1 < a.rows ? a.groups + 1 : a.rows;  // groups (and the tail) with rows: each may add a partial tile
  const int64_t grid = (a.rows / kBM + most) * a.tiles_j;
  if (grid > kMaxGrid) return MPE_ERR_ARG;
  hipLaunchKernelGGL((grouped_kernel<T, MODE, kBM, kBN, 2, 2>), dim3((unsigned)grid), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <typename T>
int launch_dw(GroupedArgs a, const DwPlan &p, hipStream_t s) {
  a.tiles_i = p.tiles_i;
  a.tiles_j = p.tiles_j;
  a.splits = p.splits;
  const int64_t grid = (int64_t)p.tiles_i * p.tiles_j * p.splits * a.groups;
  if (grid > kMaxGrid) return MPE_ERR_ARG;
  hipLaunchKernelGGL((grouped_kernel<T, GROUPED_DW, kBM, kBN, 2, 2>), dim3((unsigned)grid), dim3(256), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return (int)e;
  const int64_t cw = (int64_t)a.groups * a.n * a.k, cb = (int64_t)a.groups * a.n;
  hipLaunchKernelGGL(grouped_join_kernel<T>, dim3((unsigned)((cw + 1023) / 1024)), dim3(256), 0, s, a.part, (T *)a.out, cw, p.splits);
  if (a.dbias)
    hipLaunchKernelGGL(grouped_join_kernel<T>, dim3((unsigned)((cb + 1023) / 1024)), dim3(256), 0, s, a.part_bias, (T *)a.dbias, cb, p.splits);
  return (int)hipGetLastError();
}

#define BY_TYPE(dtype, call)                        \
  ((dtype) == MPE_F32 ? call<float> : (dtype) == MPE_BF16 ? call<__bf16> : call<_Float16>)

template <typename T> int fwd(const GroupedArgs &a, hipStream_t s) { return launch_rows<T, GROUPED_FWD>(a, a.n, s); }
template <typename T> int dx(const GroupedArgs &a, hipStream_t s) { return launch_rows<T, GROUPED_DX>(a, a.k, s); }
template <typename T> int dw(const GroupedArgs &a, const DwPlan &p, hipStream_t s) { return launch_dw<T>(a, p, s); }

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
  return BY_TYPE(d->dtype, fwd)(a, (hipStream_t)stream);
}

extern "C" int mpe_grouped_linear_dx(const mpe_grouped_desc *d, const void *dy, int64_t ld_dy, const void *y, int64_t ld_y,
                                     const void *weight, void *dx_, int64_t ld_dx, int zero_tail, void *stream) {
  if (const int rc = grouped_check(d)) return rc;
  if (zero_tail != 0 && zero_tail != 1) return MPE_ERR_ARG;
  if (d->rows == 0) return MPE_OK;
  if (!dy || !weight || !dx_) return MPE_ERR_NULL;
  if (ld_dy < d->n || (y && ld_y < d->n) || ld_dx < d->k) return MPE_ERR_ARG;
  const int size = dtype_size(d->dtype);
  if (bad_align(dy, size) || bad_align(y, size) || bad_align(weight, size) || bad_align(dx_, size)) return MPE_ERR_ALIGN;
  GroupedArgs a = base_args(d);
  a.a = dy;
  a.ld_a = ld_dy;
  a.mask = y;
  a.ld_mask = ld_y;
  a.b = weight;
  a.ld_b = d->k;
  a.out = dx_;
  a.ld_out = ld_dx;
  a.zero_tail = zero_tail;
  return BY_TYPE(d->dtype, dx)(a, (hipStream_t)stream);
}

extern "C" int64_t mpe_grouped_dw_workspace(const mpe_grouped_desc *d) {
  if (const int rc = grouped_check(d)) return rc;
  const DwPlan p = dw_plan(d);
  return p.splits == 1 ? 0 : (int64_t)p.splits * d->groups * d->n * ((int64_t)d->k + 1) * 4;
}

extern "C" int mpe_grouped_linear_dw(const mpe_grouped_desc *d, const void *dy, int64_t ld_dy, const void *y, int64_t ld_y,
                                     const void *x, int64_t ld_x, void *dweight, void *dbias, void *workspace,
                                     int64_t workspace_bytes, void *stream) {
  if (const int rc = grouped_check(d)) return rc;
  if (!dweight || (d->rows > 0 && (!dy || !x))) return MPE_ERR_NULL;
  if (d->rows > 0 && (ld_dy < d->n || (y && ld_y < d->n) || ld_x < d->k)) return MPE_ERR_ARG;
  const int size = dtype_size(d->dtype);
  if (bad_align(dy, size) || bad_align(y, size) || bad_align(x, size) || bad_align(dweight, size) || bad_align(dbias, size) ||
      bad_align(workspace, 16))
    return MPE_ERR_ALIGN;
  const DwPlan p = dw_plan(d);
  const int64_t need = mpe_grouped_dw_workspace(d);
  if (need > 0 && !workspace) return MPE_ERR_NULL;
  if (workspace_bytes < need) return MPE_ERR_SCRATCH;
  GroupedArgs a = base_args(d);
  a.a = dy;
  a.ld_a = ld_dy;
  a.mask = y;
  a.ld_mask = ld_y;
  a.b = x;
  a.ld_b = ld_x;
  a.out = dweight;
  a.dbias = dbias;
  a.part = (float *)workspace;
  a.part_bias = a.part + (need > 0 ? (int64_t)p.splits * d->groups * d->n * d->k : 0);
  return BY_TYPE(d->dtype, dw)(a, p, (hipStream_t)stream);
}
