// Products grouped by agent (expert) with ragged row counts: the dense layers of many networks in one launch.
//
// Rows 0 .. T-1 of x belong to G groups in order: group g owns rows [end(g-1), end(g)), end(-1) = 0, and has its own
// weight W_g [N][K] (torch.nn.Linear's layout) and bias b_g [N].  With d = dy, or dy where y > 0 and 0 elsewhere (relu):
//     forward   y[r][n]    = act(sum_k x[r][k] W_g[n][k] + b_g[n])
//     dx        dx[r][k]   = sum_n d[r][n] W_g[n][k]
//     dw        dW_g[n][k] = sum_{r in g} d[r][n] x[r][k],   db_g[n] = sum_{r in g} d[r][n]
// All three are C[i][j] = sum_c A(i, c) B(j, c) with f32 accumulators; they differ in which index of an operand is
// contiguous in memory:
//     forward   A = x   (c = k contiguous)   B = W (c = k contiguous)
//     dx        A = d   (c = n contiguous)   B = W (j = k contiguous)
//     dw        A = d   (i = n contiguous)   B = x (j = k contiguous)
// `ends` lives on the device (a captured launch follows it): it is read as its running maximum clamped to [0, T], so
// whatever it holds, no row belongs to two groups and no access leaves the arrays.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mpe {

enum GroupedMode { GROUPED_FWD = 0, GROUPED_DX = 1, GROUPED_DW = 2 };

struct GroupedArgs {
  const void *a, *b;        // forward: x, weight; dx: dy, weight; dw: dy, x
  const void *mask;         // dx, dw: y (same layout as dy up to ld_mask), or NULL
  const void *bias;         // forward: [G][N] or NULL
  void *out;                // forward: y; dx: dx; dw: dweight
  void *dbias;              // dw: [G][N] or NULL
  float *part, *part_bias;  // dw over splits: [S][G][N][K] and [S][G][N] partial sums
  const void *ends;
  int64_t rows, ld_a, ld_b, ld_mask, ld_out;
  int32_t groups, n, k, ends64, relu, zero_tail;
  int32_t tiles_i, tiles_j, splits;  // dw: tiles over n, over k, over rows; forward / dx: tiles_j only
};

typedef float f4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 hf8v __attribute__((ext_vector_type(8)));

// 16 bytes with the alignment of one element (gfx950 loads and stores multi-dword data at any byte address)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Chunk16 { T v[16 / sizeof(T)]; };
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Quad { T v[4]; };

template <typename T> struct GroupedType;
template <> struct GroupedType<float> {
  static constexpr int kSteps = 4;  // matrix instructions per 16-byte chunk: 16x16x4 takes one f32 a lane
  static __device__ __forceinline__ f4v mma(const uint4 &p, const uint4 &q, f4v c) {
    const float *a = reinterpret_cast<const float *>(&p), *b = reinterpret_cast<const float *>(&q);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};
template <> struct GroupedType<__bf16> {
  static __device__ __forceinline__ f4v mma(const uint4 &p, const uint4 &q, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, p), __builtin_bit_cast(bf8v, q), c, 0, 0, 0);
  }
};
template <> struct GroupedType<_Float16> {
  static __device__ __forceinline__ f4v mma(const uint4 &p, const uint4 &q, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8v, p), __builtin_bit_cast(hf8v, q), c, 0, 0, 0);
  }
};

__device__ __forceinline__ int64_t grouped_end(const GroupedArgs &a, int g) {
  return a.ends64 ? static_cast<const int64_t *>(a.ends)[g] : (int64_t)static_cast<const int32_t *>(a.ends)[g];
}

// Rows [r0, r1) of group g (dw).  Every wavefront computes it for itself.
__device__ __forceinline__ void grouped_rows_of(const GroupedArgs &a, int g, int64_t &r0, int64_t &r1) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = 0;  // running maximum before g, and through g
  for (int i = lane; i <= g; i += 64) {
    const int64_t e = grouped_end(a, i);
    if (i < g && e > lo) lo = e;
    if (e > hi) hi = e;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const int64_t l2 = __shfl_xor(lo, d), h2 = __shfl_xor(hi, d);
    lo = l2 > lo ? l2 : lo;
    hi = h2 > hi ? h2 : hi;
  }
  r0 = lo < a.rows ? lo : a.rows;
  r1 = hi < a.rows ? hi : a.rows;
}

// The group of row tile `tile` (tiles of BM rows, counted group by group) and its rows [r0, r1); behind the last group's
// tiles come those of the rows that belong to none (g == groups).  false: no such tile.
template <int BM>
__device__ __forceinline__ bool grouped_tile(const GroupedArgs &a, int tile, int &g, int64_t &r0, int64_t &r1) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;   // running maximum of the ends before this batch of 64 groups
  int tiles_before = 0;
  for (int base = 0; base <= a.groups; base += 64) {
    const int i = base + lane;
    int64_t e = i < a.groups ? grouped_end(a, i) : a.rows;  // the last, pseudo, group ends with the rows
    e = e < 0 ? 0 : (e < a.rows ? e : a.rows);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(e, d);
      if (lane >= d && o > e) e = o;
    }
    e = e > before ? e : before;
    int64_t s = __shfl_up(e, 1);
    if (lane == 0) s = before;
    int sum = (int)((e - s + BM - 1) / BM);
    const int mine = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    sum += tiles_before;
    const uint64_t hit = __ballot(tile < sum);
    if (hit != 0) {
      const int w = __ffsll((unsigned long long)hit) - 1;
      const int64_t first = __shfl(s, w), last = __shfl(e, w);
      g = base + w;
      r0 = first + (int64_t)(tile - __shfl(sum - mine, w)) * BM;
      r1 = last < r0 + BM ? last : r0 + BM;
      return true;
    }
    before = __shfl(e, 63);
    tiles_before = __shfl(sum, 63);
  }
  return false;
}

// One operand's tile: ROWS of i (or j) by 128 bytes of c, staged from memory through registers to LDS.
//   CONTIG (c contiguous in memory): LDS holds [row][8 chunks of 16 bytes], chunk q of row i at place q ^ (i & 7), so that
//   eight rows' chunks of one column lie in different banks; a fragment is one 16-byte read.
//   otherwise (row index contiguous): LDS holds [c][ROWS].
template <typename T, int ROWS, int NT, bool CONTIG>
struct GroupedOperand {
  static constexpr int CE = 16 / sizeof(T), KE = 128 / sizeof(T), N = ROWS * 8 / NT;
  static_assert(ROWS * 8 % NT == 0, "whole chunks per thread");
  uint4 r[N];

  static __device__ __forceinline__ uint4 load(const T *p, int64_t off, int valid) {
    if (valid >= CE) return __builtin_bit_cast(uint4, *reinterpret_cast<const Chunk16<T> *>(p + off));
    Chunk16<T> c;
#pragma unroll
    for (int e = 0; e < CE; ++e) c.v[e] = e < valid ? p[off + e] : T(0);
    return __builtin_bit_cast(uint4, c);
  }
  // keeps the elements of v whose saved output is > 0 or NaN (as relu's derivative: zero where y <= 0)
  static __device__ __forceinline__ uint4 keep(uint4 v, uint4 y) {
    Chunk16<T> c = __builtin_bit_cast(Chunk16<T>, v), m = __builtin_bit_cast(Chunk16<T>, y);
#pragma unroll
    for (int e = 0; e < CE; ++e) c.v[e] = (float)m.v[e] <= 0.0f ? T(0) : c.v[e];
    return __builtin_bit_cast(uint4, c);
  }
  // p: element (row 0, c 0) of the tile column; rows / cs: how many of them from there exist
  __device__ __forceinline__ void fetch(const T *p, int64_t ld, const T *mask, int64_t ld_mask, int64_t rows, int64_t cs) {
    const int t = threadIdx.x;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = t + u * NT;
      int64_t line, valid;
      int pos;
      if (CONTIG) {
        line = id >> 3;
        pos = (id & 7) * CE;
        valid = line < rows ? cs - pos : 0;
      } else {
        line = id / (ROWS / CE);
        pos = (id % (ROWS / CE)) * CE;
        valid = line < cs ? rows - pos : 0;
      }
      const int v = valid < 0 ? 0 : (valid < CE ? (int)valid : CE);
      r[u] = v > 0 ? load(p, line * ld + pos, v) : uint4{0, 0, 0, 0};
      if (mask != nullptr && v > 0) r[u] = keep(r[u], load(mask, line * ld_mask + pos, v));
    }
  }
  __device__ __forceinline__ void put(uint4 *lds) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = t + u * NT;
      if (CONTIG) lds[(id >> 3) * 8 + ((id & 7) ^ ((id >> 3) & 7))] = r[u];
      else lds[id] = r[u];
    }
  }
  // lane l's share of k-step kk: row i0 + l % 16, c = kk * 4 CE + (l / 16) * CE .. + CE
  static __device__ __forceinline__ uint4 frag(const uint4 *lds, int i0, int kk) {
    const int lane = threadIdx.x & 63, i = i0 + (lane & 15), q = kk * 4 + (lane >> 4);
    if (CONTIG) return lds[i * 8 + (q ^ (i & 7))];
    const T *s = reinterpret_cast<const T *>(lds);
    Chunk16<T> c;
#pragma unroll
    for (int e = 0; e < CE; ++e) c.v[e] = s[(q * CE + e) * ROWS + i];
    return __builtin_bit_cast(uint4, c);
  }
};

template <typename T>
__device__ __forceinline__ void grouped_store4(T *p, f4v v, int valid) {
  if (valid >= 4) {
    Quad<T> q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = (T)v[e];
    *reinterpret_cast<Quad<T> *>(p) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) p[e] = (T)v[e];
  }
}

template <typename T, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void grouped_kernel(GroupedArgs a) {
  constexpr int NT = 64 * WM * WN, KE = 128 / (int)sizeof(T);
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  using OpA = GroupedOperand<T, BM, NT, MODE != GROUPED_DW>;
  using OpB = GroupedOperand<T, BN, NT, MODE == GROUPED_FWD>;
  __shared__ uint4 la[BM * 8], lb[BN * 8];
  const T *pa = static_cast<const T *>(a.a), *pb = static_cast<const T *>(a.b), *pm = static_cast<const T *>(a.mask);

  // ---- which tile ------------------------------------------------------------------------------------------------------
  int g, tj = 0, split = 0;
  int64_t i0, i_end, j0, j_end, c0, c_end;  // output rows, output columns, contraction
  if (MODE == GROUPED_DW) {
    int id = blockIdx.x;
    tj = id % a.tiles_j;
    id /= a.tiles_j;
    const int ti = id % a.tiles_i;
    id /= a.tiles_i;
    split = id % a.splits;
    g = id / a.splits;
    int64_t r0, r1;
    grouped_rows_of(a, g, r0, r1);
    const int64_t per = ((r1 - r0 + a.splits - 1) / a.splits + KE - 1) / KE * KE;  // rows of a split: whole k-steps
    c0 = r0 + split * per;
    c_end = c0 + per < r1 ? c0 + per : r1;
    i0 = (int64_t)ti * BM;
    i_end = a.n;
    j0 = (int64_t)tj * BN;
    j_end = a.k;
  } else {
    tj = blockIdx.x % a.tiles_j;
    if (!grouped_tile<BM>(a, blockIdx.x / a.tiles_j, g, i0, i_end)) return;
    j0 = (int64_t)tj * BN;
    j_end = MODE == GROUPED_FWD ? a.n : a.k;
    c0 = 0;
    c_end = MODE == GROUPED_FWD ? a.k : a.n;
    if (g == a.groups) {  // rows of no group
      if (!a.zero_tail) return;
      c_end = 0;
      g = 0;
    }
  }
  const bool tail = MODE != GROUPED_DW && c_end == 0;
  if (MODE != GROUPED_DW) pb += (int64_t)g * a.n * a.k;

  // ---- the product -----------------------------------------------------------------------------------------------------
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
  f4v acc[MI][NJ] = {}, accb[MI] = {};
  OpA oa;
  OpB ob;
  auto fetch = [&](int64_t c) {
    if (MODE == GROUPED_DW) {
      oa.fetch(pa + c * a.ld_a + i0, a.ld_a, pm ? pm + c * a.ld_mask + i0 : nullptr, a.ld_mask, i_end - i0, c_end - c);
      ob.fetch(pb + c * a.ld_b + j0, a.ld_b, nullptr, 0, j_end - j0, c_end - c);
    } else {
      oa.fetch(pa + i0 * a.ld_a + c, a.ld_a, pm ? pm + i0 * a.ld_mask + c : nullptr, a.ld_mask, i_end - i0, c_end - c);
      if (MODE == GROUPED_FWD) ob.fetch(pb + j0 * a.ld_b + c, a.ld_b, nullptr, 0, j_end - j0, c_end - c);
      else ob.fetch(pb + c * a.ld_b + j0, a.ld_b, nullptr, 0, j_end - j0, c_end - c);
    }
  };
  uint4 ones;
  {
    Chunk16<T> o;
#pragma unroll
    for (int e = 0; e < OpA::CE; ++e) o.v[e] = T(1);
    ones = __builtin_bit_cast(uint4, o);
  }
  const bool with_bias = MODE == GROUPED_DW && a.dbias != nullptr && tj == 0 && wj == 0;
  if (c0 < c_end) fetch(c0);
  for (int64_t c = c0; c < c_end; c += KE) {
    oa.put(la);
    ob.put(lb);
    __syncthreads();
    if (c + KE < c_end) fetch(c + KE);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 fa[MI], fb[NJ];
#pragma unroll
      for (int m = 0; m < MI; ++m) fa[m] = OpA::frag(la, wi + m * 16, kk);
#pragma unroll
      for (int n = 0; n < NJ; ++n) fb[n] = OpB::frag(lb, wj + n * 16, kk);
      // operands swapped: the result's rows are j, so a lane holds four neighbours of one output row
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = GroupedType<T>::mma(fb[n], fa[m], acc[m][n]);
      if (with_bias)
#pragma unroll
        for (int m = 0; m < MI; ++m) accb[m] = GroupedType<T>::mma(ones, fa[m], accb[m]);
    }
    __syncthreads();
  }

  // ---- epilogue: lane holds output row i0 + wi + 16 m + lane % 16, columns j0 + wj + 16 n + 4 (lane / 16) .. + 4 ----------
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int64_t i = i0 + wi + m * 16 + (lane & 15);
    if (i >= i_end) continue;
    if (with_bias && lane < 16) {
      if (a.splits > 1) a.part_bias[((int64_t)split * a.groups + g) * a.n + i] = accb[m][0];
      else static_cast<T *>(a.dbias)[(int64_t)g * a.n + i] = (T)accb[m][0];
    }
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int64_t j = j0 + wj + n * 16 + 4 * (lane >> 4);
      const int valid = j_end - j >= 4 ? 4 : (int)(j_end - j);
      if (valid <= 0) continue;
      f4v v = acc[m][n];
      if (MODE == GROUPED_DW) {
        if (a.splits > 1) grouped_store4(a.part + (((int64_t)split * a.groups + g) * a.n + i) * a.k + j, v, valid);
        else grouped_store4(static_cast<T *>(a.out) + ((int64_t)g * a.n + i) * a.k + j, v, valid);
      } else {
        if (MODE == GROUPED_FWD && !tail) {
          if (a.bias) {
            const T *b = static_cast<const T *>(a.bias) + (int64_t)g * a.n + j;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < valid) v[e] += (float)b[e];
          }
          if (a.relu)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.0f ? 0.0f : v[e];  // NaN stays
        }
        grouped_store4(static_cast<T *>(a.out) + i * a.ld_out + j, v, valid);
      }
    }
  }
}

// dw over splits: the partial sums in split order, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void grouped_join_kernel(const float *part, T *out, int64_t count, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  const int valid = count - i >= 4 ? 4 : (int)(count - i);
  f4v sum = {};
  for (int s = 0; s < splits; ++s) {
    const float *p = part + (int64_t)s * count + i;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) sum[e] += p[e];
  }
  grouped_store4(out + i, sum, valid);
}

}  // namespace mpe
