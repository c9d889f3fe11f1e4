// C ABI of the AdamW step over many tensors (include/mpe_hip.h); kernels in mpe_adamw_kernel.h.
#include <cfloat>
#include <cmath>
#include <cstring>

#include "../../include/mpe_hip.h"
#include "mpe_adamw_kernel.h"

using namespace mpe;

namespace {

bool bad_align(const void *p, int size) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }
int64_t items_of(int64_t count) { return (count + kAdamItem - 1) / kAdamItem; }

int tensors_check(int n, const mpe_adamw_tensor *t, int dtype, int state_bits, int64_t *items) {
  if (!t) return MPE_ERR_NULL;
  if (dtype != MPE_F32 && dtype != MPE_BF16 && dtype != MPE_F16) return MPE_ERR_UNSUPPORTED;
  if (state_bits != 8 && state_bits != 32) return MPE_ERR_UNSUPPORTED;
  if (n < 1 || n > (1 << 24)) return MPE_ERR_ARG;
  const int size = dtype == MPE_F32 ? 4 : 2;
  *items = 0;
  for (int i = 0; i < n; ++i) {
    if (t[i].count < 0) return MPE_ERR_ARG;
    if (t[i].count == 0) continue;
    if (!t[i].param || !t[i].exp_avg || !t[i].exp_avg_sq) return MPE_ERR_NULL;
    if (state_bits == 8 && (!t[i].exp_avg_base || !t[i].exp_avg_sq_base)) return MPE_ERR_NULL;
    if (bad_align(t[i].param, size) || bad_align(t[i].target, size) || bad_align(t[i].exp_avg, 16) ||
        bad_align(t[i].exp_avg_sq, 16) || bad_align(t[i].exp_avg_base, 2) || bad_align(t[i].exp_avg_sq_base, 2))
      return MPE_ERR_ALIGN;
    *items += items_of(t[i].count);
    if (*items > 0xffffff) return MPE_ERR_ARG;  // a launch has less than 2^32 threads
  }
  return MPE_OK;
}

// plan in device memory: AdamTensor[n], AdamItem[items], partial norms double[items]
int64_t plan_items_at(int n) { return (int64_t)n * (int64_t)sizeof(AdamTensor); }
int64_t plan_norms_at(int n, int64_t items) { return plan_items_at(n) + items * (int64_t)sizeof(AdamItem); }

template <typename T, bool EIGHT, bool FAST>
int launch(const AdamArgs &a, unsigned items, bool clip, bool norms, hipStream_t s) {
  if (clip) {
    if (norms) hipLaunchKernelGGL(adamw_norm_kernel<T>, dim3(items), dim3(kAdamThreads), 0, s, a);
    hipLaunchKernelGGL((adamw_kernel<T, EIGHT, true, FAST>), dim3(items), dim3(kAdamThreads), 0, s, a);
  } else {
    hipLaunchKernelGGL((adamw_kernel<T, EIGHT, false, FAST>), dim3(items), dim3(kAdamThreads), 0, s, a);
  }
  return (int)hipGetLastError();
}

template <typename T>
int launch_bits(const AdamArgs &a, int bits, bool fast, unsigned items, bool clip, bool norms, hipStream_t s) {
  if (bits != 8) return launch<T, false, false>(a, items, clip, norms, s);
  if constexpr (sizeof(T) == 2) {
    if (fast) return launch<T, true, true>(a, items, clip, norms, s);
  }
  return launch<T, true, false>(a, items, clip, norms, s);
}

}  // namespace

extern "C" int64_t mpe_adamw_plan(int n, const mpe_adamw_tensor *tensors, int dtype, int state_bits, void *blob,
                                  int64_t blob_bytes) {
  int64_t items = 0;
  if (const int rc = tensors_check(n, tensors, dtype, state_bits, &items)) return rc;
  const int64_t need = plan_norms_at(n, items) + items * (int64_t)sizeof(double);
  if (!blob) return need;
  if (blob_bytes < need) return MPE_ERR_SCRATCH;
  if (bad_align(blob, 8)) return MPE_ERR_ALIGN;
  char *at = static_cast<char *>(blob);
  AdamTensor *out = reinterpret_cast<AdamTensor *>(at);
  AdamItem *item = reinterpret_cast<AdamItem *>(at + plan_items_at(n));
  uint32_t next = 0;
  for (int i = 0; i < n; ++i) {
    const mpe_adamw_tensor &t = tensors[i];
    const uint32_t many = (uint32_t)items_of(t.count);
    out[i] = AdamTensor{t.param, t.target, t.exp_avg, t.exp_avg_base, t.exp_avg_sq, t.exp_avg_sq_base, t.count, next, many};
    for (uint32_t j = 0; j < many; ++j) item[next + j] = AdamItem{(uint32_t)i, j};
    next += many;
  }
  std::memset(at + plan_norms_at(n, items), 0, (size_t)items * sizeof(double));
  return need;
}

extern "C" int mpe_adamw_step(const mpe_adamw_args *h, int n, const mpe_adamw_tensor *tensors, const void *plan,
                              const void *const *grads, void *stream) {
  if (!h || !plan || !grads) return MPE_ERR_NULL;
  int64_t items = 0;
  if (const int rc = tensors_check(n, tensors, h->dtype, h->state_bits, &items)) return rc;
  const int size = h->dtype == MPE_F32 ? 4 : 2;
  for (int i = 0; i < n; ++i)
    if (bad_align(grads[i], size)) return MPE_ERR_ALIGN;
  if (bad_align(plan, 8) || bad_align(h->clock, 8)) return MPE_ERR_ALIGN;
  if (!(h->lr >= 0) || !(h->beta1 >= 0 && h->beta1 < 1) || !(h->beta2 >= 0 && h->beta2 < 1) || !(h->eps >= 0) ||
      !(h->weight_decay >= 0) || !(h->polyak >= 0 && h->polyak <= 1) || !(h->max_norm >= 0) || std::isinf(h->lr) ||
      (h->max_norm > 0 && !((float)h->max_norm >= FLT_MIN && (float)h->max_norm <= FLT_MAX)) || (!h->clock && h->step < 1))
    return MPE_ERR_ARG;
  AdamArgs a{};
  const char *at = static_cast<const char *>(plan);
  a.tensors = reinterpret_cast<const AdamTensor *>(at);
  a.items = reinterpret_cast<const AdamItem *>(at + plan_items_at(n));
  a.norms = reinterpret_cast<double *>(const_cast<char *>(at) + plan_norms_at(n, items));
  a.beta1 = (float)h->beta1;
  a.beta1c = (float)(1.0 - h->beta1);
  a.beta2 = (float)h->beta2;
  a.beta2c = (float)(1.0 - h->beta2);
  a.eps = (float)h->eps;
  a.max_norm = (float)h->max_norm;
  a.polyak = (float)h->polyak;
  a.polyakc = (float)(1.0 - h->polyak);
  hipStream_t s = (hipStream_t)stream;
  if (h->clock) {
    hipLaunchKernelGGL(adamw_clock_kernel, dim3(1), dim3(1), 0, s, static_cast<AdamClock *>(h->clock), h->lr, h->beta1, h->beta2,
                       h->weight_decay, h->seed);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    a.clock = static_cast<const AdamClock *>(h->clock);
  } else {
    a.s.step_size = (float)(h->lr / (1.0 - std::pow(h->beta1, (double)h->step)));
    a.s.root = (float)(1.0 / std::sqrt(1.0 - std::pow(h->beta2, (double)h->step)));
    a.s.decay = (float)(1.0 - h->lr * h->weight_decay);
    a.s.key = adam_step_key(h->seed, h->step);
  }
  // a root that reads v < 2^-126 as zero is off by 2^-63 / sqrt(1 - b2^t) at most: no more than half a step of eps
  const bool fast = h->eps * std::sqrt(1.0 - h->beta2) >= 0x1p-39;
  uint32_t first = 0;
  for (int i0 = 0; i0 < n; i0 += kAdamMaxGrads) {
    const int many = n - i0 < kAdamMaxGrads ? n - i0 : kAdamMaxGrads;
    uint32_t batch = 0;
    bool norms = false;
    for (int i = 0; i < many; ++i) {
      a.grads[i] = grads[i0 + i];
      const int64_t it = items_of(tensors[i0 + i].count);
      batch += (uint32_t)it;
      norms = norms || it > 1;
    }
    a.first_tensor = (uint32_t)i0;
    a.first_item = first;
    a.index0 = h->index0 + (uint32_t)i0;
    first += batch;
    if (batch == 0) continue;
    const bool clip = h->max_norm > 0;
    const int rc = h->dtype == MPE_F32    ? launch_bits<float>(a, h->state_bits, fast, batch, clip, norms, s)
                   : h->dtype == MPE_BF16 ? launch_bits<__bf16>(a, h->state_bits, fast, batch, clip, norms, s)
                                          : launch_bits<_Float16>(a, h->state_bits, fast, batch, clip, norms, s);
    if (rc) return rc;
  }
  return MPE_OK;
}

extern "C" int mpe_adamw_moments(const void *exp_avg, const void *exp_avg_base, const void *exp_avg_sq, const void *exp_avg_sq_base,
                                 void *out, void *out_sq, int64_t count, int dtype, void *stream) {
  if (count < 0 || count % kAdamBlock != 0) return MPE_ERR_ARG;
  if (dtype != MPE_F32 && dtype != MPE_BF16) return MPE_ERR_UNSUPPORTED;
  if (count == 0) return MPE_OK;
  if ((!out && !out_sq) || (out && (!exp_avg || !exp_avg_base)) || (out_sq && (!exp_avg_sq || !exp_avg_sq_base))) return MPE_ERR_NULL;
  const int size = dtype == MPE_F32 ? 4 : 2;
  if (bad_align(exp_avg, 8) || bad_align(exp_avg_sq, 8) || bad_align(exp_avg_base, 2) || bad_align(exp_avg_sq_base, 2) ||
      bad_align(out, size) || bad_align(out_sq, size))
    return MPE_ERR_ALIGN;
  const int64_t grid = (count / 8 + 255) / 256;
  if (grid > 0xffffff) return MPE_ERR_ARG;
  const AdamMoments a = {{out ? (const uint8_t *)exp_avg : nullptr, out_sq ? (const uint8_t *)exp_avg_sq : nullptr},
                         {(const int16_t *)exp_avg_base, (const int16_t *)exp_avg_sq_base},
                         {out, out_sq}};
  if (dtype == MPE_F32)
    hipLaunchKernelGGL(adamw_moments_kernel<float>, dim3((unsigned)grid, out_sq ? 2 : 1), dim3(256), 0, (hipStream_t)stream, a, count);
  else
    hipLaunchKernelGGL(adamw_moments_kernel<__bf16>, dim3((unsigned)grid, out_sq ? 2 : 1), dim3(256), 0, (hipStream_t)stream, a, count);
  return (int)hipGetLastError();
}
