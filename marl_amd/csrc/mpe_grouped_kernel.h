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
//
// What bounds it (one MI355X; a copy of 4 GiB moves 4.76 TB/s, one library product of 8 192^3 1 274 TFLOP/s bf16, 154 f32):
//     small calls        launch and one trip to memory: 4 096 x 16 x 64 f32 6 us, 5 003 x 333 x 517 f16 in 7 groups 12 (six
//                        stages of 64 elements of c, two buffers: each waits for most of a trip to memory)
//     few rows           the weights: 13 rows over 16 of 1 024 x 2 048 bf16, 55 MB, 13 us = 4.2 TB/s
//     f32                the matrix units: 65 536 x 14 752 x 64 in 64 groups 1 100 us, 3.7 TB/s, matrix units busy 78 % of the time
//     16-bit, many rows  32 768 x 2 048 x 2 048 bf16 in 32 unlike groups 333 us = 825 TFLOP/s (even groups 288, one group 256), matrix
//                        units busy 38 %.  No faster: a second set of fragments read ahead (70 us a round of tiles instead of
//                        65), 128 elements of c a stage (whole cache lines) with two stages (70); a wavefront on 128 x 128 spills
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace mpe {

enum GroupedMode { GROUPED_FWD = 0, GROUPED_DX = 1, GROUPED_DW = 2 };

struct GroupedArgs {
  const void *a, *b;        // forward: x, weight; dx: d, weight; dw: d, x
  const void *mask;         // dx, dw of the small tile: y, where d is dy times relu's mask (else NULL)
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

template <typename T> struct GroupedType;
template <> struct GroupedType<float> {
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

// A value that all lanes hold alike, in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
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
  r0 = uniform(lo < a.rows ? lo : a.rows);
  r1 = uniform(hi < a.rows ? hi : a.rows);
}

// Lane l's rows [s, e) of group base + l; `before`: the running maximum of the ends before this batch, updated.
__device__ __forceinline__ void grouped_batch(const GroupedArgs &a, int base, int64_t &before, int64_t &s, int64_t &e) {
  const int lane = threadIdx.x & 63, i = base + lane;
  e = i < a.groups ? grouped_end(a, i) : a.rows;  // the last, pseudo, group ends with the rows
  e = e < 0 ? 0 : (e < a.rows ? e : a.rows);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(e, d);
    if (lane >= d && o > e) e = o;
  }
  e = e > before ? e : before;
  s = __shfl_up(e, 1);
  if (lane == 0) s = before;
  before = __shfl(e, 63);
}

// The group of row tile `tile` (tiles of BM rows, counted group by group) and its rows [r0, r1); behind the last group's
// tiles come those of the rows that belong to none (g == groups).  false: no such tile.
// Large tiles are counted in three turns: those with all their rows, those with more than half, the others.  The last ones take
// half as long and fill the chip's last round (dx of 16 384 x 1 024 x 1 024 bf16 in 16 unlike groups: 64 us in order, 55).
template <int BM>
__device__ __forceinline__ bool grouped_tile(const GroupedArgs &a, int tile, int &g, int64_t &r0, int64_t &r1) {
  constexpr bool kWholeFirst = BM == 256;
  const int lane = threadIdx.x & 63;
  int64_t before = 0, s, e;
  int tiles_before = 0, more = 0, less = 0;
  for (int base = 0; base <= a.groups; base += 64) {
    grouped_batch(a, base, before, s, e);
    const int mine = (int)((e - s + (kWholeFirst ? 0 : BM - 1)) / BM);
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    sum += tiles_before;
    const uint64_t hit = __ballot(tile < sum);
    if (hit != 0) {
      const int w = __ffsll((unsigned long long)hit) - 1;
      const int64_t first = uniform(__shfl(s, w)), last = uniform(__shfl(e, w));
      g = base + w;
      r0 = first + (int64_t)(tile - uniform(__shfl(sum - mine, w))) * BM;
      r1 = last < r0 + BM ? last : r0 + BM;
      return true;
    }
    tiles_before = __shfl(sum, 63);
    if (kWholeFirst) {
      const int rest = (int)((e - s) % BM);
      more += __popcll(__ballot(rest > BM / 2));
      less += __popcll(__ballot(rest > 0 && rest <= BM / 2));
    }
  }
  if (!kWholeFirst) return false;
  int at = uniform(tile - tiles_before);
  const bool half = at >= more;
  if (half) at -= more;
  if (half && at >= less) return false;
  before = 0;
  for (int base = 0; base <= a.groups; base += 64) {
    grouped_batch(a, base, before, s, e);
    const int rest = (int)((e - s) % BM);
    const uint64_t any = __ballot(half ? rest > 0 && rest <= BM / 2 : rest > BM / 2);
    const int below = __popcll(any & ((1ull << lane) - 1)), count = __popcll(any);
    if (at < count) {
      const int w = __ffsll((unsigned long long)__ballot((any >> lane & 1) && below == at)) - 1;
      g = base + w;
      r1 = uniform(__shfl(e, w));
      r0 = r1 - uniform(__shfl(rest, w));
      return true;
    }
    at -= count;
  }
  return false;
}

constexpr uint32_t kGroupedSpan = 0x7ffffff0u;  // bytes a tile's copies may reach (the host checks it); an offset outside

// One operand's tile: ROWS of i (or j) by KC 16-byte chunks of c (KC = 4 or 8), copied from memory straight to LDS.
//   CONTIG (c contiguous in memory): [row][KC chunks], chunk q of row i at place q ^ swizzle(i); a fragment is one 16-byte read.
//   otherwise (row index contiguous): [c][ROWS elements], in units of 16 elements, unit u of line c at place u ^ swizzle(c); a
//   fragment is two transposing reads (16 bits) or four 4-byte reads (f32).
// The swizzles spread what one read touches over the LDS banks.
// The copies are buffer loads: the buffer ends where the array does (checked dword by dword, reads as zeros), rows and columns
// outside the tile's are given an offset outside every buffer.
template <typename T, int ROWS, int KC, int NT, bool CONTIG>
struct GroupedOperand {
  static constexpr int CE = 16 / sizeof(T), N = ROWS * KC / NT;
  static constexpr int kLine = CONTIG ? KC : ROWS / CE;  // chunks of a line (a row, or a c)
  static constexpr int kUnit = 16 / CE;                 // chunks of 16 elements
  static_assert(ROWS * KC % NT == 0, "whole chunks per thread");

  static __device__ __forceinline__ int swizzle(int line) {  // on chunks for CONTIG, on units otherwise
    if (CONTIG) return KC == 8 ? line & 7 : (line >> 1) & 3;            // 8 lanes' chunks in one pass of 128 bytes: 8 places
    if (sizeof(T) == 4) return (line >> 2) & 3;                         // 32 lanes on two c's four apart
    if (ROWS == 64) return ((line >> 1) & 1) | ((line >> 3) & 1) << 1;  // 32 lanes on eight c's: 256 bytes
    return (line & 3) | ((line >> 3) & 1) << 2;
  }
  static __device__ __forceinline__ int place(int line, int pos) {  // of chunk pos of a line; its own inverse in pos
    return CONTIG ? pos ^ swizzle(line) : (((pos / kUnit) ^ swizzle(line)) * kUnit + pos % kUnit);
  }
  // A wavefront's 64 chunks land side by side in LDS, so each lane fetches what belongs at its place.
  // at: the chunks' byte offsets in the tile; left: how many c's exist from there on (none for a chunk outside the rows).
  uint32_t at[N];
  int left[N];
  __device__ __forceinline__ void aim(int64_t ld, int64_t rows, int64_t cs) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = threadIdx.x + u * NT, line = id / kLine, pos = place(line, id % kLine) * CE;
      at[u] = ((uint32_t)line * (uint32_t)ld + pos) * sizeof(T);
      left[u] = (CONTIG ? line : pos) < rows ? (int)cs - (CONTIG ? pos : line) : 0;
    }
  }
  // p: the tile at its next c; bytes: from there to the array's end
  __device__ __forceinline__ void copy(uint4 *lds, const T *p, int64_t bytes) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass does not know buffer resources
    const int records = (int)(bytes < 0 ? 0 : (bytes < (int64_t)kGroupedSpan ? bytes : (int64_t)kGroupedSpan));
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(p), 0, records, 0x00027000);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(lds + u * NT + uniform((int)threadIdx.x & ~63)),
                                               16, left[u] > 0 ? at[u] : kGroupedSpan, 0, 0, 0);
      left[u] -= KC * CE;
    }
#endif
  }
  // The last k-step of a c that ends inside a chunk: what the copies brought from behind it becomes zero (times the other
  // operand's zeros it would still be NaN where it is not finite).  ago: copies since this stage's, itself included.
  __device__ __forceinline__ void trim(uint4 *lds, int ago) {
    if (!CONTIG) return;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int have = left[u] + ago * KC * CE;
      if (have > 0 && have < CE) {
        T *c = reinterpret_cast<T *>(lds + u * NT + threadIdx.x);
#pragma unroll
        for (int e = 1; e < CE; ++e)
          if (e >= have) c[e] = T(0);
      }
    }
  }
  // the place in LDS, in elements, of column `pos` of line `line`, or -1 where another thread copies it
  static __device__ __forceinline__ int mine(int line, int pos) {
    const int id = line * kLine + place(line, pos / CE);
    return (int)threadIdx.x == id % NT ? id * CE + pos % CE : -1;
  }
  // lane l's share of the fragment of rows i0 .. i0 + 15 (i0: a multiple of 16), k-step kk: row l % 16, c = kk * 4 CE +
  // (l / 16) * CE .. + CE
  static __device__ __forceinline__ uint4 frag(const uint4 *lds, int i0, int kk) {
    const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    if (CONTIG) return lds[(i0 + t) * KC + ((kk * 4 + q) ^ swizzle(t))];
    if constexpr (sizeof(T) == 4) {
      const float *s = reinterpret_cast<const float *>(lds);
      float4 out;
      float *v = reinterpret_cast<float *>(&out);
      const int at = q * 4 * ROWS + ((i0 / 16) ^ swizzle(q * 4)) * 16 + t;  // swizzle: the same for every kk and e
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = s[(kk * 16 + e) * ROWS + at];
      return __builtin_bit_cast(uint4, out);
    } else {
      // 16 lanes read 4 c's of 16 elements, 8 bytes a lane; each lane gets its element of the four
      typedef short s4 __attribute__((ext_vector_type(4)));
      const short *s = reinterpret_cast<const short *>(lds);
      uint4 out;
      s4 *o = reinterpret_cast<s4 *>(&out);
      const int c = q * 8 + (t >> 2), at = c * ROWS + ((i0 / 16) ^ swizzle(c)) * 16 + (t & 3) * 4;  // swizzle: the same for every kk and h
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4 *)const_cast<short *>(s + (kk * 32 + h * 4) * ROWS + at));
      return out;
    }
  }
};

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Quad { T v[4]; };
// four neighbours of an output row, valid of them inside it
template <typename T>
__device__ __forceinline__ void grouped_store4(T *p, f4v v, int valid) {
  if (valid >= 4) {
    Quad<T> q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = (T)v[e];
    *reinterpret_cast<Quad<T> *>(p) = q;
    asm volatile("");  // or the compiler shares the last element's store with the other branch: three stores for one
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) p[e] = (T)v[e];
  }
}

// Workgroups are handed to the eight dies in turn: runs of 32 consecutive tiles (which share a weight or its rows) go to one
// die's L2.  Not longer runs: the grid has a few tiles too many at its end, which must not all fall to one die.
// b: the workgroup's number among n, whose first one's number is a multiple of 8.
__device__ __forceinline__ int grouped_block(int b, int n) {
  constexpr int kRun = 32;
  if (b >= n / (8 * kRun) * (8 * kRun)) return b;
  const int at = b / 8;
  return at / kRun * (8 * kRun) + b % 8 * kRun + at % kRun;
}

// keeps the elements of v whose saved output is > 0 or NaN (relu's derivative: zero where y <= 0)
template <typename T>
__device__ __forceinline__ Chunk16<T> grouped_keep(Chunk16<T> v, const Chunk16<T> &y) {
#pragma unroll
  for (int e = 0; e < 16 / (int)sizeof(T); ++e) v.v[e] = (float)y.v[e] <= 0.0f ? T(0) : v.v[e];
  return v;
}
// The tile kernel's LDS: STAGES buffers of KC chunks a row; while one is multiplied, STAGES - 1 are on their way.  Separate
// arrays: the compiler then knows that a read of one does not wait for copies into another.
#define GROUPED_STAGES(chunks, STAGES) \
  __shared__ uint4 s0[chunks], s1[chunks], s2[(STAGES) == 4 ? (chunks) : 1], s3[(STAGES) == 4 ? (chunks) : 1]

// One output tile: number `block` of a.tiles_* (and splits).  MASK: A times relu's mask, on its fragments.
template <typename T, int MODE, int BM, int BN, int WM, int WN, int KC, int STAGES, bool MASK>
__device__ __forceinline__ void grouped_body(const GroupedArgs &a, int block, uint4 *s0, uint4 *s1, uint4 *s2, uint4 *s3) {
  constexpr int NT = 64 * WM * WN, KE = KC * 16 / (int)sizeof(T);
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  constexpr bool EDGES = BM < 256;  // the large tile, short of registers, takes whole chunks only (n and k multiples of 8)
  using OpA = GroupedOperand<T, BM, KC, NT, MODE != GROUPED_DW>;
  using OpB = GroupedOperand<T, BN, KC, NT, MODE == GROUPED_FWD>;
  static_assert(STAGES == 2 || STAGES == 4, "the loop below");
  const T *pa = static_cast<const T *>(a.a), *pb = static_cast<const T *>(a.b), *pm = static_cast<const T *>(a.mask);

  // ---- which tile ------------------------------------------------------------------------------------------------------
  int g, tj = 0, split = 0;
  int64_t i0, i_end, j0, j_end, c0, c_end;  // output rows, output columns, contraction
  if (MODE == GROUPED_DW) {
    int id = block;
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
    tj = block % a.tiles_j;
    if (!grouped_tile<BM>(a, block / a.tiles_j, g, i0, i_end)) return;
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
  // the arrays: lines, columns, elements to their ends
  const int64_t lines_b = MODE == GROUPED_DW ? a.rows : (int64_t)a.groups * a.n;
  const int cols_a = MODE == GROUPED_FWD ? a.k : a.n, cols_b = a.k;
  const int64_t end_a = (a.rows - 1) * a.ld_a + cols_a, end_b = (lines_b - 1) * a.ld_b + cols_b;
  const int64_t b0 = MODE == GROUPED_DW ? 0 : (int64_t)g * a.n * a.ld_b;

  // ---- the product: one barrier a stage; the next stages are on their way while this one is multiplied ---------------------
  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
  f4v acc[MI][NJ] = {};
  // dbias: this lane's share of its rows' (n's) sums; the wavefronts of the same rows take kSums of their MI tiles of 16 rows each
  constexpr int kSums = MI / WN;
  static_assert(MI % WN == 0, "");
  float sum[kSums] = {};
  const int wn = wave % WN;
  OpA oa, om;
  OpB ob;
  oa.aim(a.ld_a, i_end - i0, c_end - c0);
  ob.aim(a.ld_b, j_end - j0, c_end - c0);
  if constexpr (MASK) om.aim(a.ld_mask, i_end - i0, c_end - c0);
  auto fetch = [&](int64_t c, uint4 *la) {
    const int64_t at = MODE == GROUPED_DW ? c * a.ld_a + i0 : i0 * a.ld_a + c;
    const int64_t bt = b0 + (MODE == GROUPED_FWD ? j0 * a.ld_b + c : c * a.ld_b + j0);
    oa.copy(la, pa + at, (end_a - at) * (int64_t)sizeof(T));
    ob.copy(la + BM * KC, pb + bt, (end_b - bt) * (int64_t)sizeof(T));
    if constexpr (MASK) {
      const int64_t mt = MODE == GROUPED_DW ? c * a.ld_mask + i0 : i0 * a.ld_mask + c;
      om.copy(la + (BM + BN) * KC, pm + mt, ((a.rows - 1) * a.ld_mask + cols_a - mt) * (int64_t)sizeof(T));
    }
  };
  // 2-byte elements in lines of odd width: an array's last element is half of a dword that the buffer's bounds cut off, and its copy
  // brings zero.  The thread of that copy puts it in place before its stage is multiplied (adding its product afterwards would not
  // undo a zero times an infinity).  fill_*: how far from c0 the element is multiplied, or -1; put_*: its place in the stage.
  const bool cuts = EDGES && sizeof(T) == 2 && ((cols_a | cols_b) & 1);
  int fill_a = -1, fill_b = -1, put_a = 0, put_b = 0;
  if (cuts) {
    const int64_t last_b = lines_b - 1 - (MODE == GROUPED_DW ? 0 : (int64_t)g * a.n);  // B's last line: a c, or forward a j
    const int64_t ia = MODE == GROUPED_DW ? cols_a - 1 : a.rows - 1, ca = MODE == GROUPED_DW ? a.rows - 1 : cols_a - 1;
    const int64_t jb = MODE == GROUPED_FWD ? last_b : cols_b - 1, cb = MODE == GROUPED_FWD ? cols_b - 1 : last_b;
    if ((cols_a & 1) && ia >= i0 && ia < i0 + BM && ia < i_end && ca >= c0 && ca < c_end) {
      const int i = (int)(ia - i0), c = (int)(ca - c0);
      put_a = MODE == GROUPED_DW ? OpA::mine(c % KE, i) : OpA::mine(i, c % KE);
      fill_a = put_a < 0 ? -1 : c;
    }
    if ((cols_b & 1) && jb >= j0 && jb < j0 + BN && jb < j_end && cb >= c0 && cb < c_end) {
      const int j = (int)(jb - j0), c = (int)(cb - c0);
      put_b = MODE == GROUPED_FWD ? OpB::mine(j, c % KE) : OpB::mine(c % KE, j);
      fill_b = put_b < 0 ? -1 : c;
    }
  }
  const bool with_bias = MODE == GROUPED_DW && a.dbias != nullptr && tj == 0;
  constexpr int kAhead = (STAGES - 2) * ((MASK ? 2 : 1) * OpA::N + OpB::N);  // copies of later stages that may still be under way
  // this wavefront's copies of this stage have landed, its reads of LDS are done; then so are everybody's
  auto landed = [&](int64_t c, uint4 *la) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAhead) : "memory");
    if (EDGES && MODE != GROUPED_DW && c_end - c < KE && (c_end - c) % OpA::CE != 0) {
      oa.trim(la, STAGES - 1);
      ob.trim(la + BM * KC, STAGES - 1);
    }
    if (cuts) {
      const int past = (int)(c - c0);
      if ((uint32_t)(fill_a - past) < (uint32_t)KE) {
        reinterpret_cast<T *>(la)[put_a] = pa[end_a - 1];
        if constexpr (MASK) reinterpret_cast<T *>(la + (BM + BN) * KC)[put_a] = pm[(a.rows - 1) * a.ld_mask + cols_a - 1];
      }
      if ((uint32_t)(fill_b - past) < (uint32_t)KE) reinterpret_cast<T *>(la + BM * KC)[put_b] = pb[end_b - 1];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto read = [&](uint4 *la, int kk, uint4 (&fa)[MI], uint4 (&fb)[NJ]) {
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      fa[m] = OpA::frag(la, wi + m * 16, kk);
      if constexpr (MASK)
        fa[m] = __builtin_bit_cast(uint4, grouped_keep(__builtin_bit_cast(Chunk16<T>, fa[m]),
                                                       __builtin_bit_cast(Chunk16<T>, OpA::frag(la + (BM + BN) * KC, wi + m * 16, kk))));
    }
#pragma unroll
    for (int n = 0; n < NJ; ++n) fb[n] = OpB::frag(la + BM * KC, wj + n * 16, kk);
  };
  auto multiply = [&](const uint4 (&fa)[MI], const uint4 (&fb)[NJ]) {
    // operands swapped: the result's rows are j, so a lane holds four neighbours of one output row
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NJ; ++n) acc[m][n] = GroupedType<T>::mma(fb[n], fa[m], acc[m][n]);
    if (with_bias) {
#pragma unroll
      for (int m = 0; m < kSums; ++m) {
        uint4 f = fa[m];
#pragma unroll
        for (int w = 1; w < WN; ++w) {  // selects: an index that is not constant would put the fragments into memory
          const uint4 o = fa[w * kSums + m];
          f = uint4{wn == w ? o.x : f.x, wn == w ? o.y : f.y, wn == w ? o.z : f.z, wn == w ? o.w : f.w};
        }
        const Chunk16<T> c = __builtin_bit_cast(Chunk16<T>, f);
#pragma unroll
        for (int e = 0; e < OpA::CE; ++e) sum[m] += (float)c.v[e];
      }
    }
  };
  // Two halves of the wavefronts, one of each on every matrix unit, half a step apart: while one half reads its fragments the other
  // multiplies.  32 768 x 2 048 x 2 048 bf16 in 32 unlike groups: 327 us, all in step 338; dx 278 / 275, dweight 331 / 308 of
  // 32 768 x 2 048 x 2 048 in 8 (their transposing reads need more registers): there in step.
  constexpr bool HALVES = BM == 256 && MODE == GROUPED_FWD;
  // stages past the end are zeros: fetched and multiplied like the others
  auto steps = [&](auto works) {
    auto step = [&](int64_t c, uint4 *la, uint4 *next) {
      landed(c, la);
      fetch(c + (STAGES - 1) * KE, next);
      if constexpr (decltype(works)::value) {
#pragma unroll
        for (int kk = 0; kk < KC / 4; ++kk) {
          uint4 fa[MI], fb[NJ];
          read(la, kk, fa, fb);
          multiply(fa, fb);
        }
      }
    };
    if constexpr (HALVES) {
      static_assert(!HALVES || (STAGES == 4 && KC == 4 && WM * WN == 8), "one fragment a stage, two wavefronts a matrix unit");
      const bool late = wave >= 4;
      auto turn = [&](int64_t c, uint4 *la, uint4 *free) {
        uint4 fa[MI], fb[NJ];
        fetch(c + 3 * KE, free);  // its last reads ended before the last barrier
        if constexpr (decltype(works)::value) read(la, 0, fa, fb);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kAhead) : "memory");  // the next stage has landed; the reads are done
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(works)::value) {
          __builtin_amdgcn_s_setprio(1);
          multiply(fa, fb);
          __builtin_amdgcn_s_setprio(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      };
      landed(c0, s0);
      if (late) __builtin_amdgcn_s_barrier();
      for (int64_t c = c0; c < c_end; c += 4 * KE) {
        turn(c, s0, s3);
        turn(c + KE, s1, s0);
        turn(c + 2 * KE, s2, s1);
        turn(c + 3 * KE, s3, s2);
      }
      if (!late) __builtin_amdgcn_s_barrier();
    } else {
      for (int64_t c = c0; c < c_end; c += STAGES * KE) {
        if constexpr (STAGES == 2) {
          step(c, s0, s1);
          step(c + KE, s1, s0);
        } else {
          step(c, s0, s3);
          step(c + KE, s1, s0);
          step(c + 2 * KE, s2, s1);
          step(c + 3 * KE, s3, s2);
        }
      }
    }
  };
  if (c0 < c_end) {
    fetch(c0, s0);
    if constexpr (STAGES == 4) fetch(c0 + KE, s1), fetch(c0 + 2 * KE, s2);
    // a wavefront of a large tile whose rows or columns do not exist only copies: its neighbour on the matrix unit goes on alone
    // (dweight's first column tile is whole, large tiles have 256 columns at least: every share of dbias is summed)
    if (BM < 256 || (i0 + wi < i_end && j0 + wj < j_end)) steps(std::true_type());
    else steps(std::false_type());
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the tile
  }

  // ---- epilogue: lane holds output row i0 + wi + 16 m + lane % 16, columns j0 + wj + 16 n + 4 (lane / 16) .. + 4 ----------
  const int64_t j_lane = j0 + wj + 4 * (lane >> 4);
  const bool whole = j0 + BN <= j_end;  // all columns exist
  const auto valid_of = [&](int n) { return j_end - j_lane - n * 16 >= 4 ? 4 : (int)(j_end - j_lane - n * 16); };
  if constexpr (MODE == GROUPED_FWD) {
    if (a.bias != nullptr && !tail) {  // all of it first: one wait
      const T *b = static_cast<const T *>(a.bias) + (int64_t)g * a.n + j_lane;
      f4v bias[NJ];
#pragma unroll
      for (int n = 0; n < NJ; ++n) {
        const int valid = valid_of(n);
        if (whole || !EDGES) {
          Quad<T> q{};
          if (whole || valid == 4) q = *reinterpret_cast<const Quad<T> *>(b + n * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) bias[n][e] = (float)q.v[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) bias[n][e] = e < valid ? (float)b[n * 16 + e] : 0.0f;
        }
      }
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] += bias[n];
    }
    if (a.relu) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][n][e] = acc[m][n][e] < 0.0f ? 0.0f : acc[m][n][e];  // NaN stays
    }
  }
  const auto store = [&](auto *out, int64_t ld) {  // out: the array's row 0
    auto *at = out + (i0 + wi + (lane & 15)) * ld + j_lane;
    if (whole && i0 + BM <= i_end) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n) grouped_store4(at + m * 16 * ld + n * 16, acc[m][n], 4);
      return;
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      if (i0 + wi + m * 16 + (lane & 15) >= i_end) continue;
#pragma unroll
      for (int n = 0; n < NJ; ++n) {
        if (EDGES) grouped_store4(at + m * 16 * ld + n * 16, acc[m][n], valid_of(n));
        else if (valid_of(n) == 4) grouped_store4(at + m * 16 * ld + n * 16, acc[m][n], 4);
      }
    }
  };
  if constexpr (MODE == GROUPED_DW) {
    const int64_t part = ((int64_t)split * a.groups + g) * a.n;
    if (with_bias) {
#pragma unroll
      for (int m = 0; m < kSums; ++m) {
        float v = sum[m] + __shfl_xor(sum[m], 16);  // lanes l, l + 16, .. hold the same row's other c's
        v += __shfl_xor(v, 32);
        const int64_t i = i0 + wi + (wn * kSums + m) * 16 + lane;
        if (lane >= 16 || i >= i_end) continue;
        if (EDGES && a.splits > 1) a.part_bias[part + i] = v;
        else static_cast<T *>(a.dbias)[(int64_t)g * a.n + i] = (T)v;
      }
    }
    if (EDGES && a.splits > 1) store(a.part + part * a.k, a.k);  // the large tile's sums are never split
    else store(static_cast<T *>(a.out) + (int64_t)g * a.n * a.k, a.k);
  } else {
    store(static_cast<T *>(a.out), a.ld_out);
  }
}

template <typename T, int MODE, int BM, int BN, int WM, int WN, int KC, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, WM * WN <= 4 ? 2 : 1) void grouped_kernel(GroupedArgs a) {
  GROUPED_STAGES((BM + BN) * KC, STAGES);
  grouped_body<T, MODE, BM, BN, WM, WN, KC, STAGES, false>(a, grouped_block(blockIdx.x, gridDim.x), s0, s1, s2, s3);
}

// A backward pass in one launch: the first dw_tiles workgroups make dw's tiles, those behind them dx's; with MASK both mask what
// they load.  One launch also fills the chip where the first product's last tiles leave it empty, and dw's, which run longest,
// come first: 65 536 x 226 x 64 f32 in 64 groups, masked: two products in two launches 85 us, dx first 92, dw first 70;
// 4 096 x 64 x 64 in 4 groups: mask, dx, dw and join as four launches 16.7 us, this and the join 9.6;
// 16 384 x 1 024 x 1 024 bf16 in 16 unlike groups, without the mask: 116 us as two launches, 101 as one.
template <typename T, int BM, int BN, int WM, int WN, int KC, int STAGES, bool MASK>
__global__ __launch_bounds__(64 * WM * WN, WM * WN <= 4 ? 2 : 1) void grouped_both_kernel(GroupedArgs dx, GroupedArgs dw, int dw_tiles) {
  GROUPED_STAGES((BM + BN + (MASK ? BM : 0)) * KC, STAGES);
  const int b = (int)blockIdx.x, first = (dw_tiles + 7) & ~7;
  if (b >= first) {
    grouped_body<T, GROUPED_DX, BM, BN, WM, WN, KC, STAGES, MASK>(dx, grouped_block(b - first, (int)gridDim.x - first), s0, s1, s2, s3);
  } else if (b < dw_tiles) {
    grouped_body<T, GROUPED_DW, BM, BN, WM, WN, KC, STAGES, MASK>(dw, grouped_block(b, dw_tiles), s0, s1, s2, s3);
  }
}

// Copies matrices into rows of whole chunks where their stride is too large for a tile's copies, and applies relu's mask to dy
// on the way: d = dy where y is not <= 0, zero elsewhere.
struct GroupedPack { const void *src, *mask; void *dst; int64_t ld, ld_mask, lines; int32_t cols, blocks; };
struct GroupedPacks { GroupedPack job[2]; };  // x, dy

// the chunk at element off, valid of it kept; end: elements of the whole matrix (a chunk may reach into the next line)
template <typename T>
__device__ __forceinline__ Chunk16<T> grouped_chunk(const T *p, int64_t off, int valid, int64_t end) {
  constexpr int CE = 16 / sizeof(T);
  Chunk16<T> c;
  if (valid > 0 && off + CE <= end) {
    c = *reinterpret_cast<const Chunk16<T> *>(p + off);
#pragma unroll
    for (int e = 1; e < CE; ++e) c.v[e] = e < valid ? c.v[e] : T(0);
  } else {
#pragma unroll
    for (int e = 0; e < CE; ++e) c.v[e] = e < valid ? p[off + e] : T(0);
  }
  return c;
}
template <typename T>
__global__ __launch_bounds__(256) void grouped_pack_kernel(GroupedPacks a) {
  constexpr int CE = 16 / sizeof(T);
  uint32_t b = blockIdx.x, k = 0;
  if (b >= (uint32_t)a.job[0].blocks) b -= a.job[k++].blocks;
  const GroupedPack &j = a.job[k];
  // a workgroup: some whole lines of up to 256 chunks, or up to 256 chunks of one line; one chunk a thread
  const uint32_t chunks = (uint32_t)((j.cols + CE - 1) / CE), t = threadIdx.x;
  int64_t line;
  uint32_t at;
  if (chunks <= 256) {
    const uint32_t lines = 256 / chunks, sub = t / chunks;
    line = (int64_t)b * lines + sub;
    at = t - sub * chunks;
    if (sub >= lines) return;
  } else {
    const uint32_t per = (chunks + 255) / 256, q = b / per;
    line = q;
    at = (b - q * per) * 256 + t;
    if (at >= chunks) return;
  }
  if (line >= j.lines) return;
  const int col = (int)at * CE, valid = j.cols - col < CE ? j.cols - col : CE;
  Chunk16<T> c = grouped_chunk(static_cast<const T *>(j.src), line * j.ld + col, valid, (j.lines - 1) * j.ld + j.cols);
  if (j.mask)
    c = grouped_keep(c, grouped_chunk(static_cast<const T *>(j.mask), line * j.ld_mask + col, valid, (j.lines - 1) * j.ld_mask + j.cols));
  *reinterpret_cast<uint4 *>(static_cast<T *>(j.dst) + (line * chunks + at) * CE) = __builtin_bit_cast(uint4, c);
}

// dw over splits: the partial sums of dweight (cw values) and dbias (cb) in split order, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void grouped_join_kernel(const float *part, T *out, int64_t cw, const float *part_bias, T *dbias,
                                                           int64_t cb, int splits) {
  const int64_t blocks = (cw + 1023) / 1024;
  const bool bias = blockIdx.x >= blocks;
  const int64_t count = bias ? cb : cw, i = (((int64_t)blockIdx.x - (bias ? blocks : 0)) * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  const int valid = count - i >= 4 ? 4 : (int)(count - i);
  const float *p = (bias ? part_bias : part) + i;
  f4v sum = {};
  for (int s0 = 0; s0 < splits; s0 += 8) {
    f4v v[8] = {};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (s0 + s >= splits) continue;
      const float *q = p + (int64_t)(s0 + s) * count;
      if (valid == 4) v[s] = __builtin_bit_cast(f4v, *reinterpret_cast<const Quad<float> *>(q));
      else
        for (int e = 0; e < valid; ++e) v[s][e] = q[e];
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) sum += v[s];
  }
  grouped_store4((bias ? dbias : out) + i, sum, valid);
}

}  // namespace mpe
