// products.hip — the experts' matrix products outside the fused layer, for MI355X (gfx950):
// grouped by expert in bf16 and fp16 with the weights' gradient, in int8 with a scale for each
// token and channel, and the quantization of rows that feeds the latter (megamoe_products.h).
//
// Every product is out[j][i] = sum_c A[i][c] * B[j][c] with i along the output's contiguous
// dimension:
//   y  = x w^T   A = w[e]  [n][k], c contiguous      B = x  [row][k], c contiguous, j ragged
//   y  = x w     A = w[e]  [k][n], i contiguous      B = x  [row][k], c contiguous, j ragged
//   dw = dy^T x  A = x  [row][k], i contiguous       B = dy [row][n], j contiguous, c ragged
// A is the MFMA's first operand, so a lane's four results of a 16x16 tile are neighbours in the
// output's rows. bf16 and fp16 multiply 32 values of c per 16x16 MFMA, int8 64: 16 bytes a lane
// of each operand in all three, so one kernel body serves the types.

#include <hip/hip_runtime.h>
#include <atomic>
#include <stddef.h>
#include <stdint.h>

#include "megamoe.h"
#include "megamoe_products.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxGroups = 1024;

// What an element type of the operands brings: its accumulator and its 16x16 MFMA, whose lane l
// holds row l % 16 and the 16 bytes at 16 * (l / 16) of both operands' c, and of the result rows
// 4 * (l / 16) .. +3 (of A) in column l % 16 (of B).
struct Bf16 {
  using Elem = __bf16;
  using Acc = f32x4;
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
struct Fp16 {
  using Elem = _Float16;
  using Acc = f32x4;
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
};
struct Int8 {
  using Elem = int8_t;
  using Acc = i32x4;
  static constexpr int kBytes = 1;
  static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};

// One call. For the int8 product sx and sw are the scales; `out` has rows of ldo elements.
struct Args {
  const uint8_t* x;       // x; for the weights' gradient as well
  const uint8_t* w;       // w, or dy for the weights' gradient
  uint8_t* out;
  const int64_t* counts;  // NULL: one group of all the rows
  const float* sx;
  const float* sw;
  int rows, groups, n, k;
  int64_t ldx, ldy;       // row strides of x and of y (dy), in elements
  int fill_rest;
  int tiles_j, tiles_i;   // the grid's tiles: along the rows (an upper bound) and the columns
};

// ---------------------------------------------------------------------------------------
// Groups
// ---------------------------------------------------------------------------------------

constexpr int kNoTile = -1, kRest = -2, kBad = -3;

// The rows [first, last) of one tile and whose they are: a group, kRest (rows of no group),
// kBad (the counts do not fit the rows: the tile's share of all rows, to be NaN) or kNoTile.
struct Tile {
  int group, first, last;
};

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Inclusive scan over the wavefront, saturating (sums of counts that are too large stay too large).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)v, d, 64);
    if (lane >= d) v = add_sat(v, u);
  }
  return v;
}

__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// Tile `tile` of the groups' rows cut into tiles of `height`, in order; after the last group's
// the rows of no group. Every wavefront walks the counts itself (64 at a time), so no barrier
// is needed; the result is uniform.
__device__ Tile locate(const int64_t* counts, int groups, int rows, int height, int tile) {
  if (!counts) {
    const int64_t first = (int64_t)tile * height;
    if (first >= rows) return Tile{kNoTile, 0, 0};
    return Tile{0, (int)first, (int)min(first + height, (int64_t)rows)};
  }
  const int lane = threadIdx.x & 63;
  uint32_t row0 = 0, tile0 = 0;
  bool bad = false;
  Tile found{kNoTile, 0, 0};
  for (int g0 = 0; g0 < groups; g0 += 64) {
    int64_t c = g0 + lane < groups ? counts[g0 + lane] : 0;
    const bool wrong = c < 0 || c > rows;
    bad |= __ballot(wrong) != 0;
    const uint32_t n = wrong ? 0 : (uint32_t)c, t = (n + (uint32_t)height - 1) / (uint32_t)height;
    const uint32_t rows_to = add_sat(row0, wave_scan(n)), tiles_to = add_sat(tile0, wave_scan(t));
    const uint64_t mask = __ballot((uint32_t)tile < tiles_to && (uint32_t)tile >= tiles_to - t);
    if (mask) {
      const int l = __builtin_ctzll(mask);
      const int start = (int)(lane_value(rows_to, l) - lane_value(n, l));
      const int within = tile - (int)(lane_value(tiles_to, l) - lane_value(t, l));
      found.group = g0 + l;
      found.first = start + within * height;
      found.last = min(found.first + height, (int)lane_value(rows_to, l));
    }
    row0 = lane_value(rows_to, 63);
    tile0 = lane_value(tiles_to, 63);
  }
  if (bad || row0 > (uint32_t)rows) {
    const int64_t first = (int64_t)tile * height;
    if (first >= rows) return Tile{kNoTile, 0, 0};
    return Tile{kBad, (int)first, (int)min(first + height, (int64_t)rows)};
  }
  if (found.group == kNoTile) {
    const int64_t first = row0 + ((int64_t)tile - tile0) * height;
    if (first < rows) return Tile{kRest, (int)first, (int)min(first + height, (int64_t)rows)};
  }
  return found;
}

// All the rows of group `group`, or kBad.
__device__ Tile rows_of(const int64_t* counts, int groups, int rows, int group) {
  const int lane = threadIdx.x & 63;
  uint32_t row0 = 0;
  bool bad = false;
  Tile found{kNoTile, 0, 0};
  for (int g0 = 0; g0 < groups; g0 += 64) {
    int64_t c = g0 + lane < groups ? counts[g0 + lane] : 0;
    const bool wrong = c < 0 || c > rows;
    bad |= __ballot(wrong) != 0;
    const uint32_t n = wrong ? 0 : (uint32_t)c;
    const uint32_t rows_to = add_sat(row0, wave_scan(n));
    if (group >= g0 && group < g0 + 64) {
      found.group = group;
      found.last = (int)lane_value(rows_to, group - g0);
      found.first = found.last - (int)lane_value(n, group - g0);
    }
    row0 = lane_value(rows_to, 63);
  }
  if (bad || row0 > (uint32_t)rows) found.group = kBad;
  return found;
}

// ---------------------------------------------------------------------------------------
// The product of any alignment
//
// A workgroup of four wavefronts computes 64x64 outputs, 64 bytes of c at a time: each thread
// loads its elements of the next step one by one (any stride and alignment) into registers
// while the MFMAs of this step read theirs from LDS, where both operands lie with c contiguous
// (rows of 80 bytes: 16 consecutive rows' 16-byte chunks start in different banks). It is bound
// by its element loads; operands whose rows are 16-byte aligned take the kernels below.
// ---------------------------------------------------------------------------------------

constexpr int kAnyTile = 64, kAnyStep = 64, kAnyPitch = 80;

// One operand: element (r, c) at p[r * sr + c * sc], zero outside the limits.
template <class Elem>
struct Operand {
  const Elem* p;
  int64_t sr, sc;
  int nr;
};

template <class Elem, int COUNT>
__device__ __forceinline__ void any_load(Elem (&v)[COUNT], const Operand<Elem>& o, int c0, int nc, bool c_fast) {
  constexpr int kC = kAnyStep / (int)sizeof(Elem);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const int at = i * 256 + (int)threadIdx.x;
    const int r = c_fast ? at / kC : at % kAnyTile, c = c0 + (c_fast ? at % kC : at / kAnyTile);
    v[i] = r < o.nr && c < nc ? o.p[r * o.sr + c * o.sc] : Elem(0);
  }
}

template <class Elem, int COUNT>
__device__ __forceinline__ void any_store(uint8_t* lds, const Elem (&v)[COUNT], bool c_fast) {
  constexpr int kC = kAnyStep / (int)sizeof(Elem);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const int at = i * 256 + (int)threadIdx.x;
    const int r = c_fast ? at / kC : at % kAnyTile, c = c_fast ? at % kC : at / kAnyTile;
    reinterpret_cast<Elem*>(lds + r * kAnyPitch)[c] = v[i];
  }
}

// out[j][i] of one tile, i < ni and j < nj: f(j, i, acc value).
template <class Ty, class F>
__device__ __forceinline__ void any_tile(uint8_t* lds, const Operand<typename Ty::Elem>& a, bool a_fast,
                                         const Operand<typename Ty::Elem>& b, bool b_fast, int nc, F&& f) {
  using Elem = typename Ty::Elem;
  constexpr int kC = kAnyStep / (int)sizeof(Elem), kCount = kAnyTile * kC / 256;
  uint8_t* const la = lds;
  uint8_t* const lb = lds + kAnyTile * kAnyPitch;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave & 1) * 32, wj = (wave >> 1) * 32;
  typename Ty::Acc acc[2][2] = {};
  Elem va[kCount], vb[kCount];
  any_load(va, a, 0, nc, a_fast);
  any_load(vb, b, 0, nc, b_fast);
  for (int c0 = 0; c0 < nc; c0 += kC) {
    __syncthreads();
    any_store(la, va, a_fast);
    any_store(lb, vb, b_fast);
    __syncthreads();
    any_load(va, a, c0 + kC, nc, a_fast);
    any_load(vb, b, c0 + kC, nc, b_fast);
    i32x4 fa[2], fb[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      fa[t] = *reinterpret_cast<const i32x4*>(la + (wi + 16 * t + (lane & 15)) * kAnyPitch + (lane >> 4) * 16);
      fb[t] = *reinterpret_cast<const i32x4*>(lb + (wj + 16 * t + (lane & 15)) * kAnyPitch + (lane >> 4) * 16);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) acc[s][t] = Ty::mfma(fa[s], fb[t], acc[s][t]);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int i = wi + 16 * s + 4 * (lane >> 4) + v, j = wj + 16 * t + (lane & 15);
        if (i < a.nr && j < b.nr) f(j, i, acc[s][t][v]);
      }
}

// A dequantized sum: each step rounds to fp32 (the barrier keeps the last product from being
// rounded to the result's type in the same instruction).
__device__ __forceinline__ float scaled(int sum, float sx, float sw) {
  float f = (float)sum * sx * sw;
  asm("" : "+v"(f));
  return f;
}

// `value` into rows [first, last) and columns [c0, c1) of out.
template <class Out>
__device__ __forceinline__ void fill_rows(Out* out, int64_t ld, int first, int last, int c0, int c1, float value) {
  const int width = c1 - c0;
  for (int64_t at = threadIdx.x; at < (int64_t)(last - first) * width; at += blockDim.x)
    out[(first + at / width) * ld + c0 + at % width] = (Out)value;
}

template <class Ty, class Out, bool TRANS>
__global__ __launch_bounds__(256) void k_product_any(Args p) {
  using Elem = typename Ty::Elem;
  __shared__ __align__(16) uint8_t lds[2 * kAnyTile * kAnyPitch];
  Out* const out = reinterpret_cast<Out*>(p.out);
  const int64_t total = (int64_t)p.tiles_j * p.tiles_i;
  for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
    const int i0 = (int)(at % p.tiles_i) * kAnyTile, i1 = min(i0 + kAnyTile, p.n);
    const Tile t = locate(p.counts, p.groups, p.rows, kAnyTile, (int)(at / p.tiles_i));
    if (t.group == kNoTile) continue;
    if (t.group < 0) {
      if (t.group == kBad || p.fill_rest)
        fill_rows(out, p.ldy, t.first, t.last, i0, i1, t.group == kBad ? __builtin_nanf("") : 0.f);
      continue;
    }
    const Elem* w = reinterpret_cast<const Elem*>(p.w) + (size_t)t.group * p.n * p.k;
    const Operand<Elem> a{TRANS ? w + i0 : w + (size_t)i0 * p.k, TRANS ? 1 : p.k, TRANS ? p.n : 1, i1 - i0};
    const Operand<Elem> b{reinterpret_cast<const Elem*>(p.x) + (int64_t)t.first * p.ldx, p.ldx, 1, t.last - t.first};
    any_tile<Ty>(lds, a, !TRANS, b, true, p.k, [&](int j, int i, auto v) {
      float f;
      if constexpr (Ty::kBytes == 1)
        f = scaled(v, p.sx[t.first + j], p.sw[(size_t)t.group * p.n + i0 + i]);
      else
        f = v;
      out[(int64_t)(t.first + j) * p.ldy + i0 + i] = (Out)f;
    });
  }
}

template <class Ty>
__global__ __launch_bounds__(256) void k_wgrad_any(Args p) {
  using Elem = typename Ty::Elem;
  __shared__ __align__(16) uint8_t lds[2 * kAnyTile * kAnyPitch];
  const int64_t each = (int64_t)p.tiles_j * p.tiles_i, total = each * p.groups;
  for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
    const int group = (int)(at / each), i0 = (int)(at % p.tiles_i) * kAnyTile, i1 = min(i0 + kAnyTile, p.k);
    const int j0 = (int)(at % each / p.tiles_i) * kAnyTile, j1 = min(j0 + kAnyTile, p.n);
    Elem* const out = reinterpret_cast<Elem*>(p.out) + (size_t)group * p.n * p.k;
    const Tile t = rows_of(p.counts, p.groups, p.rows, group);
    if (t.group == kBad) {
      fill_rows(out, p.k, j0, j1, i0, i1, __builtin_nanf(""));
      continue;
    }
    const Operand<Elem> a{reinterpret_cast<const Elem*>(p.x) + (int64_t)t.first * p.ldx + i0, 1, p.ldx, i1 - i0};
    const Operand<Elem> b{reinterpret_cast<const Elem*>(p.w) + (int64_t)t.first * p.ldy + j0, 1, p.ldy, j1 - j0};
    any_tile<Ty>(lds, a, false, b, false, t.last - t.first,
                 [&](int j, int i, auto v) { out[(size_t)(j0 + j) * p.k + i0 + i] = (Elem)v; });
  }
}

// ---------------------------------------------------------------------------------------
// The tiled product (16-byte aligned operands)
//
// A persistent workgroup of eight wavefronts per CU computes tiles of 256 (i) by TJ (j) outputs,
// stage by stage of 128 bytes of c. Each stage's operands are cut into four regions, the halves
// A0, A1 (128 i each) and B0, B1 (TJ/2 j each), and a stage into four phases of one quadrant:
//
//   phase         0         1         2         3
//   reads         A0        B1        A1        B0 of the next stage   (LDS -> registers)
//   multiplies    A0 B0     A0 B1     A1 B1     A1 B0
//   loads         B0        A0        B1        A1, of the stage after next, into the regions
//                                               that the phase before freed
//
// A wavefront's share of a quadrant takes rows of both operands' halves, so that a region is
// read by all wavefronts in one phase and free in the next. Every region is loaded seven phases
// before it is read (about 100 KB in flight per CU, no registers), straight into LDS; the wait
// in a phase lets the last six regions' loads stay pending. Wavefronts 4-7 run half a phase
// behind 0-3 (one barrier more at the start), so on every SIMD one wavefront multiplies while the
// other reads LDS and issues loads.
//
// The stages of consecutive tiles follow each other without a gap: loads run two stages ahead,
// over the tile's end, so a tile's first stage is in LDS when the last tile's results are
// stored. (A tile has at least two stages; a short c is padded with zeros.)
//
// LDS layout. An operand with c contiguous: rows of 128 bytes, 16-byte chunk p of row r at
// position p ^ (r % 8): one load instruction fills eight whole rows from full 128-byte lines,
// and the MFMA's reads (16 rows of one chunk) fall into different banks. An operand with c
// across: 64 rows (c) of 256 bytes (128 i or j), chunk p of row c at p ^ 2 f(c), f = c % 4 +
// 4 (c / 8 % 2): the transposing reads (ds_read_b64_tr_b16: four c of 16 neighbours, for c = 8g ..
// of the lane group g) fall into different banks as well.
//
// Everything outside a tensor reads as zero: rows past the tile's are past the end of the buffer
// resource, chunks past the operand's width get an offset past it.
// ---------------------------------------------------------------------------------------

enum Form { kNT, kNN, kTN };  // y = x w^T, y = x w, dw = dy^T x

constexpr int kThreads = 512, kTileI = 256, kStage = 128;
constexpr int kRegionA = 128 * kStage;

typedef int i32x2 __attribute__((ext_vector_type(2)));

template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N <= 63, "vmcnt holds 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | (((N >> 4) & 3) << 14));
  asm volatile("" ::: "memory");
}

// A phase boundary: nothing moves across it.
__device__ __forceinline__ void boundary() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// LDS reads in inline asm with their wait: the compiler would take an LDS read as depending on
// every load into LDS in flight and wait for all of them.
template <int OFF>
__device__ __forceinline__ void read_rows(i32x4 (&f)[4][2], const uint32_t (&at)[2]) {
  asm volatile(
      "ds_read_b128 %0, %8 offset:%c10\n\tds_read_b128 %1, %9 offset:%c10\n\t"
      "ds_read_b128 %2, %8 offset:%c11\n\tds_read_b128 %3, %9 offset:%c11\n\t"
      "ds_read_b128 %4, %8 offset:%c12\n\tds_read_b128 %5, %9 offset:%c12\n\t"
      "ds_read_b128 %6, %8 offset:%c13\n\tds_read_b128 %7, %9 offset:%c13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1]), "=&v"(f[2][0]), "=&v"(f[2][1]),
        "=&v"(f[3][0]), "=&v"(f[3][1])
      : "v"(at[0]), "v"(at[1]), "i"(OFF), "i"(OFF + 2048), "i"(OFF + 4096), "i"(OFF + 6144)
      : "memory");
}
template <int OFF>
__device__ __forceinline__ void read_rows(i32x4 (&f)[2][2], const uint32_t (&at)[2]) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%c6\n\tds_read_b128 %1, %5 offset:%c6\n\t"
      "ds_read_b128 %2, %4 offset:%c7\n\tds_read_b128 %3, %5 offset:%c7\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1])
      : "v"(at[0]), "v"(at[1]), "i"(OFF), "i"(OFF + 2048)
      : "memory");
}
// The transposing reads: per fragment and half stage (32 c) two, of c +0..3 and +4..7 of a lane.
template <int OFF>
__device__ __forceinline__ void read_cols2(i32x4 (&f)[2], i32x4 (&g)[2], uint32_t at_f, uint32_t at_g) {
  i32x2 r[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%c10\n\tds_read_b64_tr_b16 %1, %8 offset:%c11\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%c12\n\tds_read_b64_tr_b16 %3, %8 offset:%c13\n\t"
      "ds_read_b64_tr_b16 %4, %9 offset:%c10\n\tds_read_b64_tr_b16 %5, %9 offset:%c11\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%c12\n\tds_read_b64_tr_b16 %7, %9 offset:%c13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
      : "v"(at_f), "v"(at_g), "i"(OFF), "i"(OFF + 1024), "i"(OFF + 8192), "i"(OFF + 9216)
      : "memory");
  f[0] = __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3);
  f[1] = __builtin_shufflevector(r[2], r[3], 0, 1, 2, 3);
  g[0] = __builtin_shufflevector(r[4], r[5], 0, 1, 2, 3);
  g[1] = __builtin_shufflevector(r[6], r[7], 0, 1, 2, 3);
}
template <int OFF, int F>
__device__ __forceinline__ void read_cols(i32x4 (&f)[F][2], const uint32_t (&at)[F]) {
#pragma unroll
  for (int i = 0; i < F; i += 2) read_cols2<OFF>(f[i], f[i + 1], at[i], at[i + 1]);
}

// One operand as this wavefront loads and reads it. COL: c across (else contiguous). F: the
// 16-row fragments of a wavefront in one half. L: load instructions of a wavefront per region.
template <bool COL, int F, int L>
struct Side {
  uint32_t load[L];       // byte offset of the lane's 16 bytes from the half's first row, per instruction
  uint32_t chunk;         // of them, the bytes along the contiguous dimension
  uint32_t at[COL ? F : 2];  // LDS addresses of the lane's fragments in half 0, buffer `buf`

  // `first`: the wavefront's first row in a half; `base`: LDS address of half 0 of buffer 0.
  __device__ __forceinline__ void init(uint32_t ld, int wave, int first, uint32_t base) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    if constexpr (COL) {
      chunk = ((lane & 15) ^ (2 * ((lane >> 4) | ((uint32_t)(wave & 1) << 2)))) * 16;
#pragma unroll
      for (int i = 0; i < L; ++i) load[i] = (4 * (L * wave + i) + (lane >> 4)) * ld + chunk;
      const uint32_t f2 = 2 * (((lane >> 2) & 3) | ((g & 1) << 2));
#pragma unroll
      for (int f = 0; f < F; ++f)
        at[f] = base + (8 * g + ((lane & 15) >> 2)) * 256 +
                ((((uint32_t)(first >> 3) + 2 * f + ((lane & 3) >> 1)) ^ f2) << 4) + (lane & 1) * 8;
    } else {
      chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
      for (int i = 0; i < L; ++i) load[i] = (8 * (L * wave + i) + (lane >> 3)) * ld + chunk;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        at[s] = base + ((uint32_t)first + (lane & 15)) * 128 + (((4 * s + g) ^ (lane & 7)) << 4);
    }
  }
  // The reads to the other buffer, `by` bytes on (or back).
  __device__ __forceinline__ void move(uint32_t by) {
#pragma unroll
    for (uint32_t& a : at) a += by;
  }
  template <int OFF>
  __device__ __forceinline__ void read(i32x4 (&f)[F][2]) const {
    if constexpr (COL)
      read_cols<OFF>(f, at);
    else
      read_rows<OFF>(f, at);
  }
};

constexpr uint32_t kOutside = 0xC0000000u;  // an offset past every buffer resource

template <class T>
__device__ __forceinline__ T uniform(T v) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t u = (uint64_t)v;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return (T)(((uint64_t)hi << 32) | lo);
  } else {
    return (T)__builtin_amdgcn_readfirstlane((int)v);
  }
}

// 16 bytes a lane into LDS (1024 consecutive ones from `lds`), from `base` + at + along; zero from
// `bytes` on.
__device__ __forceinline__ void load_lds(uint8_t* lds, const uint8_t* base, uint32_t bytes, uint32_t at, uint32_t along) {
#ifdef __HIP_DEVICE_COMPILE__
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)uniform(base), 0, uniform(bytes), 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, at, along, 0, 0);
#endif
}

// One region's loads: `live` tells the lanes whose bytes exist, `bytes` the length of the rows that do.
template <int L>
__device__ __forceinline__ void load_region(uint8_t* lds, int wave, const uint8_t* base, uint32_t bytes,
                                            const uint32_t (&at)[L], bool live, uint32_t along) {
#pragma unroll
  for (int i = 0; i < L; ++i) load_lds(lds + (L * wave + i) * 1024, base, bytes, live ? at[i] : kOutside, along);
}

// The groups' tables in LDS: rows and row tiles before each group (entry g), to the end of the
// last (entry `groups` and on).
struct Table {
  uint32_t rows[kMaxGroups + 16], tiles[kMaxGroups + 16];
};

// Fills the table; false if the counts do not fit the rows. Every thread of the workgroup calls it.
__device__ bool make_table(Table& t, const Args& p, int height) {
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x; g < p.groups; g += kThreads) {
    const int64_t v = p.counts ? p.counts[g] : p.rows;
    t.rows[g] = v < 0 || v > p.rows ? 0xffffffffu : (uint32_t)v;  // sums saturate at a value past the rows
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t row0 = 0, tile0 = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
      const uint32_t c = g0 + lane < p.groups ? t.rows[g0 + lane] : 0u;
      const uint32_t n = (uint32_t)(((uint64_t)c + height - 1) / (uint32_t)height);
      const uint32_t rows_to = add_sat(row0, wave_scan(c)), tiles_to = add_sat(tile0, wave_scan(n));
      t.rows[g0 + lane] = rows_to - c;  // exact wherever the sums are
      t.tiles[g0 + lane] = tiles_to - n;
      row0 = lane_value(rows_to, 63);
      tile0 = lane_value(tiles_to, 63);
    }
    for (int g = (p.groups + 63) / 64 * 64 + lane; g < kMaxGroups + 16; g += 64) {
      t.rows[g] = row0;
      t.tiles[g] = tile0;
    }
  }
  __syncthreads();
  return t.rows[kMaxGroups] <= (uint32_t)p.rows;
}

__device__ __forceinline__ uint32_t lds_word(const uint32_t* p) {
  uint32_t v;
  asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(v)
               : "v"((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint32_t*)p)
               : "memory");
  return v;
}

// Row tile `tile` (below the table's total): its group and rows.
__device__ __forceinline__ Tile table_tile(const Table& t, int tile, int height) {
  const int lane = threadIdx.x & 63;
  const uint32_t coarse = lds_word(&t.tiles[16 * lane + 16]);
  const int block = __builtin_popcountll(__ballot(coarse <= (uint32_t)tile));
  const uint32_t fine = lds_word(&t.tiles[16 * block + 1 + (lane & 15)]);
  const int group = 16 * block + __builtin_popcountll(__ballot(fine <= (uint32_t)tile) & 0xffff);
  const uint32_t v = lds_word(lane == 0 ? &t.tiles[group] : &t.rows[group + (lane & 1 ? 0 : 1)]);
  const int first = (int)lane_value(v, 1) + (tile - (int)lane_value(v, 0)) * height;
  return Tile{group, first, min(first + height, (int)lane_value(v, 2))};
}

// Workgroups of a grid go to the eight XCDs in turn, each with an L2 of its own: step s of the
// persistent grid is `grid` consecutive tiles, of which each XCD takes a consecutive eighth. -1:
// none for this workgroup.
__device__ __forceinline__ int xcd_tile(int step, int total) {
  const int grid = (int)gridDim.x, first = step * grid, left = min(total - first, grid);
  if (left <= 0) return -1;
  const int each = (left + 7) / 8, at = ((int)blockIdx.x & 7) * each + ((int)blockIdx.x >> 3);
  return ((int)blockIdx.x >> 3) < each && at < left ? first + at : -1;
}

constexpr int kBand = 4;  // row tiles that are walked together, column by column

// What the loads need of a tile, and the results.
struct Work {
  const uint8_t* a;  // first row of A's half 0
  const uint8_t* b;
  int group, first, last;  // rows of y (the products), of the group (the weights' gradient)
  int i0, j0;              // first column and row of the output tile (j0: within rows first..last)
  int stages;
};

template <class Ty, class Out, Form FORM, int TJ>
__global__ __launch_bounds__(kThreads, 2) void k_tiles(Args p) {
  constexpr bool kAcol = FORM != kNT, kBcol = FORM == kTN;
  constexpr int WI = TJ == 256 ? 2 : 4, WJ = 8 / WI;     // wavefronts along i and j
  constexpr int FA = 128 / WI / 16, FB = TJ / 2 / WJ / 16;  // fragments of a wavefront in a half
  constexpr int LA = 2, LB = TJ / 128;                    // loads of a wavefront per region
  constexpr int kRegionB = TJ / 2 * kStage;
  constexpr int kPending = 3 * (LA + LB);
  constexpr int kC = kStage / Ty::kBytes;  // c of one stage
  __shared__ __align__(1024) uint8_t lds[4 * kRegionA + 4 * kRegionB];
  __shared__ Table table;

  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wi = wave % WI, wj = wave / WI;
  Out* const out = reinterpret_cast<Out*>(p.out);
  const int ni = FORM == kTN ? p.k : p.n;
  const int64_t ldo = FORM == kTN ? p.k : p.ldy;
  const int tiles_i = (ni + kTileI - 1) / kTileI;

  const bool fits = uniform((int)make_table(table, p, TJ)) != 0;
  if (!fits) {  // NaN everywhere
    const int64_t rows = FORM == kTN ? (int64_t)p.groups * p.n : p.rows;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
      for (int i = threadIdx.x; i < ni; i += kThreads) out[r * ldo + i] = (Out)__builtin_nanf("");
    return;
  }
  const int used = uniform((int)table.rows[kMaxGroups]);
  const int row_tiles = FORM == kTN ? p.groups * ((p.n + TJ - 1) / TJ) : uniform((int)table.tiles[kMaxGroups]);
  const int total = row_tiles * tiles_i;
  if (FORM != kTN && p.fill_rest)
    for (int64_t r = used + blockIdx.x; r < p.rows; r += gridDim.x)
      for (int i = threadIdx.x; i < ni; i += kThreads) out[r * ldo + i] = (Out)0.f;

  const int64_t lda = (int64_t)Ty::kBytes * (FORM == kNT ? p.k : FORM == kNN ? p.n : p.ldx);
  const int64_t ldb = (int64_t)Ty::kBytes * (FORM == kTN ? p.ldy : p.ldx);
  auto locate_work = [&](int tile) {
    const int width = kBand * tiles_i, band = tile / width, in = tile % width;
    const int high = min(kBand, row_tiles - band * kBand);
    const int rt = band * kBand + in % high, it = in / high;
    Work w;
    w.i0 = it * kTileI;
    if constexpr (FORM == kTN) {
      const int tiles_j = (p.n + TJ - 1) / TJ;
      w.group = rt / tiles_j;
      w.j0 = rt % tiles_j * TJ;
      const uint32_t v = lds_word(&table.rows[w.group + (lane & 1)]);
      w.first = (int)lane_value(v, 0);
      w.last = (int)lane_value(v, 1);
      w.a = p.x + (int64_t)w.first * lda + (int64_t)w.i0 * Ty::kBytes;
      w.b = p.w + (int64_t)w.first * ldb + (int64_t)w.j0 * Ty::kBytes;
      w.stages = max(2, (w.last - w.first + kC - 1) / kC);
    } else {
      const Tile t = table_tile(table, rt, TJ);
      w.group = t.group;
      w.first = t.first;
      w.last = t.last;
      w.j0 = 0;
      w.a = p.w + (size_t)w.group * p.n * p.k * Ty::kBytes +
            (FORM == kNT ? (int64_t)w.i0 * lda : (int64_t)w.i0 * Ty::kBytes);
      w.b = p.x + (int64_t)w.first * ldb;
      w.stages = max(2, (p.k + kC - 1) / kC);
    }
    return w;
  };

  int step = 0;
  int tile = xcd_tile(step, total);
  if (tile < 0) return;
  Work ahead = locate_work(tile);  // the tile that is being loaded
  Work now = ahead;                // the tile that is being multiplied
  int stage = 0;                   // of `ahead`
  bool more = true;

  Side<kAcol, FA, LA> sa;
  Side<kBcol, FB, LB> sb;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  sa.init((uint32_t)lda, wave, wi * (128 / WI), lds0);
  sb.init((uint32_t)ldb, wave, wj * (TJ / 2 / WJ), lds0 + 4 * kRegionA);

  // Loads of half `h` of A (or B) at the load cursor into buffer `buf`.
  auto load_a = [&](int h, int buf) {
    uint8_t* const to = lds + (2 * buf + h) * kRegionA;
    if constexpr (kAcol) {
      const int rows = (FORM == kTN ? ahead.last - ahead.first : p.k) - stage * kC;
      const bool live = sa.chunk + 256u * h < (uint32_t)(ni - ahead.i0) * Ty::kBytes;
      load_region(to, wave, ahead.a + (int64_t)stage * kC * lda + 256 * h,
                  more ? (uint32_t)min(max(rows, 0), kC) * (uint32_t)lda : 0u, sa.load, live, 0u);
    } else {
      const int rows = min(max(p.n - ahead.i0 - 128 * h, 0), 128);
      load_region(to, wave, ahead.a + (int64_t)128 * h * lda, more ? (uint32_t)rows * (uint32_t)lda : 0u, sa.load,
                  (uint32_t)stage * kStage + sa.chunk < (uint32_t)p.k * Ty::kBytes, (uint32_t)stage * kStage);
    }
  };
  auto load_b = [&](int h, int buf) {
    uint8_t* const to = lds + 4 * kRegionA + (2 * buf + h) * kRegionB;
    if constexpr (kBcol) {
      const int rows = ahead.last - ahead.first - stage * kC;
      const bool live = sb.chunk + 256u * h < (uint32_t)(p.n - ahead.j0) * Ty::kBytes;
      load_region(to, wave, ahead.b + (int64_t)stage * kC * ldb + 256 * h,
                  more ? (uint32_t)min(max(rows, 0), kC) * (uint32_t)ldb : 0u, sb.load, live, 0u);
    } else {
      const int rows = min(max(ahead.last - ahead.first - TJ / 2 * h, 0), TJ / 2);
      load_region(to, wave, ahead.b + (int64_t)(TJ / 2) * h * ldb, more ? (uint32_t)rows * (uint32_t)ldb : 0u, sb.load,
                  (uint32_t)stage * kStage + sb.chunk < (uint32_t)p.k * Ty::kBytes, (uint32_t)stage * kStage);
    }
  };
  // The load cursor to the next stage, over the tile's end.
  auto advance = [&]() {
    if (++stage < ahead.stages || !more) return;
    stage = 0;
    tile = xcd_tile(++step, total);
    more = tile >= 0;
    if (more) ahead = locate_work(tile);
  };

  typename Ty::Acc acc[2][2][FA][FB];
  i32x4 a[FA][2], b0[FB][2], b1[FB][2], bn[FB][2];
  auto clear = [&]() {
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int f = 0; f < FA; ++f)
#pragma unroll
        for (int t = 0; t < FB; ++t) acc[h >> 1][h & 1][f][t] = typename Ty::Acc{0, 0, 0, 0};
  };
  auto multiply = [&](typename Ty::Acc(&c)[FA][FB], const i32x4(&b)[FB][2]) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int f = 0; f < FA; ++f)
#pragma unroll
        for (int t = 0; t < FB; ++t) c[f][t] = Ty::mfma(a[f][s], b[t][s], c[f][t]);
    __builtin_amdgcn_s_setprio(0);
  };
  // Results: lane l has i = 4 (l / 16) .. +3 of a fragment at j = l % 16.
  auto store = [&]() {
    const bool wide = ldo % 4 == 0 && (uintptr_t)p.out % (4 * sizeof(Out)) == 0;
    const int nj = FORM == kTN ? p.n : now.last - now.first;
    Out* const base = FORM == kTN ? out + (size_t)now.group * p.n * p.k : out + (int64_t)now.first * ldo;
#pragma unroll
    for (int hb = 0; hb < 2; ++hb)
#pragma unroll
      for (int t = 0; t < FB; ++t) {
        const int j = now.j0 + TJ / 2 * hb + wj * (TJ / 2 / WJ) + 16 * t + (lane & 15);
        if (j >= nj) continue;
        Out* const row = base + (int64_t)j * ldo;
        float sx = 0.f;
        if constexpr (Ty::kBytes == 1) sx = p.sx[now.first + j];
#pragma unroll
        for (int ha = 0; ha < 2; ++ha)
#pragma unroll
          for (int f = 0; f < FA; ++f) {
            const int i = now.i0 + 128 * ha + wi * (128 / WI) + 16 * f + 4 * (lane >> 4);
            typedef Out Out4 __attribute__((ext_vector_type(4)));
            Out4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (Ty::kBytes == 1)
                v[e] = (Out)scaled(acc[ha][hb][f][t][e], sx,
                                   i + e < ni ? p.sw[(size_t)now.group * p.n + i + e] : 0.f);
              else
                v[e] = (Out)acc[ha][hb][f][t][e];
            }
            if (wide && i + 3 < ni) {
              *reinterpret_cast<Out4*>(row + i) = v;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (i + e < ni) row[i + e] = v[e];
            }
          }
      }
  };

  load_b(0, 0);
  load_a(0, 0);
  load_b(1, 0);
  load_a(1, 0);
  advance();
  load_b(0, 1);
  load_a(0, 1);
  load_b(1, 1);
  load_a(1, 1);
  advance();
  wait_loads<kPending>();
  boundary();
  sb.template read<0>(b0);
  boundary();
  if (wave >= 4) boundary();
  clear();
  int left = now.stages, buf = 0;
  for (;;) {
    load_b(0, buf);
    sa.template read<0>(a);
    wait_loads<kPending>();
    boundary();
    multiply(acc[0][0], b0);
    boundary();

    load_a(0, buf);
    sb.template read<kRegionB>(b1);
    wait_loads<kPending>();
    boundary();
    multiply(acc[0][1], b1);
    boundary();

    load_b(1, buf);
    sa.template read<kRegionA>(a);
    wait_loads<kPending>();
    boundary();
    multiply(acc[1][1], b1);
    boundary();

    load_a(1, buf);
    sa.move(buf ? -2 * kRegionA : 2 * kRegionA);
    sb.move(buf ? -2 * kRegionB : 2 * kRegionB);
    sb.template read<0>(bn);
    wait_loads<kPending>();
    boundary();
    multiply(acc[1][0], b0);
    boundary();
#pragma unroll
    for (int t = 0; t < FB; ++t) {
      b0[t][0] = bn[t][0];
      b0[t][1] = bn[t][1];
    }
    buf ^= 1;
    if (--left == 0) {
      store();
      if (!more) break;  // (the loads are two stages ahead: past the last tile only now)
      now = ahead;
      left = now.stages;
      clear();
    }
    advance();
  }
  if (wave < 4) boundary();
  wait_loads<0>();  // loads into LDS may not outlive the workgroup
}

// ---------------------------------------------------------------------------------------
// Rows to int8
// ---------------------------------------------------------------------------------------

template <class In>
__global__ __launch_bounds__(256) void k_quantize_int8(int64_t rows, int cols, int64_t ldx, const In* x, int8_t* q,
                                                       float* scale) {
  __shared__ float part[4];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const In* const row = x + r * ldx;
    float a = 0.f;
    bool odd = false;
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float v = __builtin_fabsf((float)row[c]);
      odd |= !(v < __builtin_inff());
      a = fmaxf(a, v);
    }
    if (odd) a = __builtin_inff();
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) a = fmaxf(a, __shfl_xor(a, d, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
    __syncthreads();
    a = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    __syncthreads();
    const bool finite = a < __builtin_inff();
    a = fmaxf(a, 0x1p-100f);
    const float inv = 127.0f / a;
    if (threadIdx.x == 0) scale[r] = finite ? a / 127.0f : __builtin_nanf("");
    for (int c = threadIdx.x; c < cols; c += 256)
      q[r * cols + c] = finite ? (int8_t)(int)__builtin_rintf((float)row[c] * inv) : (int8_t)0;
  }
}

// ---------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------

constexpr int64_t kMaxStrideBytes = 8 << 20, kMaxBlocks = 1 << 20;

int launched() { return hipGetLastError() == hipSuccess ? MEGAMOE_OK : MEGAMOE_ERR_HIP; }

int check(const megamoe_product* p, int elem, bool wide_out) {
  if (!p) return MEGAMOE_ERR_INVALID_ARGUMENT;
  if (p->rows < 0 || p->groups < 1 || p->n < 0 || p->k < 0 || p->ldx < p->k || p->ldy < p->n) return MEGAMOE_ERR_SHAPE;
  if (p->dtype < MEGAMOE_BF16 || p->dtype > (wide_out ? MEGAMOE_FP32 : MEGAMOE_FP16)) return MEGAMOE_ERR_SHAPE;
  if (p->groups > kMaxGroups || p->rows > INT32_MAX) return MEGAMOE_ERR_UNSUPPORTED;
  if (p->ldx > kMaxStrideBytes / elem || p->ldy > kMaxStrideBytes / 4) return MEGAMOE_ERR_UNSUPPORTED;
  return MEGAMOE_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles of `height` that the groups' rows and the rows of no group can take at most: each group
// (and the rest) adds at most one that is not full.
int64_t row_tiles(int64_t rows, int groups, int height, bool grouped) {
  return grouped ? rows / height + (groups + 1 < rows ? groups + 1 : rows) : ceil_div(rows, height);
}

template <class Ty, class Out, bool TRANS>
int launch_any(Args a, hipStream_t stream) {
  const int64_t tj = row_tiles(a.rows, a.groups, kAnyTile, a.counts != nullptr);
  if (tj > INT32_MAX) return MEGAMOE_ERR_UNSUPPORTED;
  a.tiles_j = (int)tj;
  a.tiles_i = (int)ceil_div(a.n, kAnyTile);
  const int64_t blocks = tj * a.tiles_i < kMaxBlocks ? tj * a.tiles_i : kMaxBlocks;
  hipLaunchKernelGGL((k_product_any<Ty, Out, TRANS>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return launched();
}

template <class Ty>
int launch_wgrad_any(Args a, hipStream_t stream) {
  a.tiles_j = (int)ceil_div(a.n, kAnyTile);
  a.tiles_i = (int)ceil_div(a.k, kAnyTile);
  const int64_t total = (int64_t)a.tiles_j * a.tiles_i * a.groups;
  hipLaunchKernelGGL((k_wgrad_any<Ty>), dim3((unsigned)(total < kMaxBlocks ? total : kMaxBlocks)), dim3(256), 0,
                     stream, a);
  return launched();
}

// Compute units of the current device.
int compute_units() {
  static std::atomic<int> known[64];
  int device = 0, n = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return 0;
  n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return 0;
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <class Ty, class Out, Form FORM, int TJ>
int launch_tiles(Args a, hipStream_t stream) {
  const int cus = compute_units();
  if (cus <= 0) return MEGAMOE_ERR_HIP;
  const int64_t rows = FORM == kTN ? a.groups * ceil_div(a.n, TJ) : row_tiles(a.rows, a.groups, TJ, a.counts != nullptr);
  const int64_t total = rows * ceil_div(FORM == kTN ? a.k : a.n, kTileI);
  if (total > INT32_MAX) return MEGAMOE_ERR_UNSUPPORTED;
  const int64_t grid = ceil_div(total < cus ? total : cus, 8) * 8;
  hipLaunchKernelGGL((k_tiles<Ty, Out, FORM, TJ>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  return launched();
}

Args make_args(const megamoe_product* p, const void* x, const void* w, const int64_t* counts, void* out) {
  Args a{};
  a.x = (const uint8_t*)x;
  a.w = (const uint8_t*)w;
  a.out = (uint8_t*)out;
  a.counts = counts;
  a.rows = (int)p->rows;
  a.groups = p->groups;
  a.n = p->n;
  a.k = p->k;
  a.ldx = p->ldx;
  a.ldy = p->ldy;
  a.fill_rest = p->fill_rest;
  return a;
}

bool aligned(const void* p, unsigned to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Whether the tiled kernels can load an operand: whole 16-byte chunks at 16-byte places.
bool chunks(const void* p, int64_t ld, int64_t width, int elem) {
  return aligned(p, 16) && ld * elem % 16 == 0 && width * elem % 16 == 0;
}

template <class Ty, class Out, Form FORM>
int launch_rows(const Args& a, hipStream_t s) {
  return a.rows >= (int64_t)192 * a.groups ? launch_tiles<Ty, Out, FORM, 256>(a, s)
                                           : launch_tiles<Ty, Out, FORM, 128>(a, s);
}

template <class Ty>
int product16(const megamoe_product* p, const Args& a, hipStream_t s) {
  using Out = typename Ty::Elem;
  if (p->k > 0 && chunks(a.x, a.ldx, a.k, 2) && chunks(a.w, 0, p->transposed ? a.n : a.k, 2))
    return p->transposed ? launch_rows<Ty, Out, kNN>(a, s) : launch_rows<Ty, Out, kNT>(a, s);
  return p->transposed ? launch_any<Ty, Out, true>(a, s) : launch_any<Ty, Out, false>(a, s);
}

template <class Ty>
int wgrad16(const Args& a, hipStream_t s) {
  if (a.rows > 0 && chunks(a.x, a.ldx, a.k, 2) && chunks(a.w, a.ldy, a.n, 2))
    return launch_tiles<Ty, typename Ty::Elem, kTN, 256>(a, s);
  return launch_wgrad_any<Ty>(a, s);
}

template <class Out>
int product8(const Args& a, hipStream_t s) {
  if (a.k > 0 && chunks(a.x, a.ldx, a.k, 1) && chunks(a.w, 0, a.k, 1)) return launch_rows<Int8, Out, kNT>(a, s);
  return launch_any<Int8, Out, false>(a, s);
}

}  // namespace

extern "C" {

int megamoe_products_version(void) { return 1; }

int megamoe_grouped_mm(const megamoe_product* p, const void* x, const void* w, const int64_t* counts, void* y,
                       void* stream) {
  const int rc = check(p, 2, false);
  if (rc) return rc;
  if (p->rows == 0 || p->n == 0) return MEGAMOE_OK;
  if (!counts || !y || (p->k && (!x || !w))) return MEGAMOE_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 2) || !aligned(w, 2) || !aligned(y, 2) || !aligned(counts, 8)) return MEGAMOE_ERR_INVALID_ARGUMENT;
  const Args a = make_args(p, x, w, counts, y);
  return p->dtype == MEGAMOE_BF16 ? product16<Bf16>(p, a, (hipStream_t)stream)
                                  : product16<Fp16>(p, a, (hipStream_t)stream);
}

int megamoe_grouped_mm_wgrad(const megamoe_product* p, const void* dy, const void* x, const int64_t* counts, void* dw,
                             void* stream) {
  const int rc = check(p, 2, false);
  if (rc) return rc;
  if (p->n == 0 || p->k == 0) return MEGAMOE_OK;
  if (!counts || !dw || (p->rows && (!x || !dy))) return MEGAMOE_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 2) || !aligned(dy, 2) || !aligned(dw, 2) || !aligned(counts, 8)) return MEGAMOE_ERR_INVALID_ARGUMENT;
  const Args a = make_args(p, x, dy, counts, dw);
  return p->dtype == MEGAMOE_BF16 ? wgrad16<Bf16>(a, (hipStream_t)stream)
                                  : wgrad16<Fp16>(a, (hipStream_t)stream);
}

int megamoe_int8_mm(const megamoe_product* p, const int8_t* x, const float* x_scale, const int8_t* w,
                    const float* w_scale, const int64_t* counts, void* y, void* stream) {
  const int rc = check(p, 1, true);
  if (rc) return rc;
  if (p->transposed || (!counts && p->groups != 1)) return MEGAMOE_ERR_SHAPE;
  if (p->k > 131071) return MEGAMOE_ERR_UNSUPPORTED;
  if (p->rows == 0 || p->n == 0) return MEGAMOE_OK;
  if (!y || !x_scale || !w_scale || (p->k && (!x || !w))) return MEGAMOE_ERR_INVALID_ARGUMENT;
  if (!aligned(x_scale, 4) || !aligned(w_scale, 4) || !aligned(y, p->dtype == MEGAMOE_FP32 ? 4 : 2) ||
      !aligned(counts, 8))
    return MEGAMOE_ERR_INVALID_ARGUMENT;
  Args a = make_args(p, x, w, counts, y);
  a.sx = x_scale;
  a.sw = w_scale;
  hipStream_t s = (hipStream_t)stream;
  if (p->dtype == MEGAMOE_BF16) return product8<__bf16>(a, s);
  if (p->dtype == MEGAMOE_FP16) return product8<_Float16>(a, s);
  return product8<float>(a, s);
}

int megamoe_quantize_rows_int8(int64_t rows, int32_t cols, int64_t ldx, int32_t dtype, const void* x, int8_t* q,
                               float* scale, void* stream) {
  if (rows < 0 || cols < 0 || ldx < cols || dtype < MEGAMOE_BF16 || dtype > MEGAMOE_FP32) return MEGAMOE_ERR_SHAPE;
  if (rows == 0) return MEGAMOE_OK;
  if (!scale || (cols && (!x || !q))) return MEGAMOE_ERR_INVALID_ARGUMENT;
  if (!aligned(x, dtype == MEGAMOE_FP32 ? 4 : 2) || !aligned(scale, 4)) return MEGAMOE_ERR_INVALID_ARGUMENT;
  const dim3 grid((unsigned)(rows < kMaxBlocks ? rows : kMaxBlocks));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MEGAMOE_BF16)
    hipLaunchKernelGGL(k_quantize_int8<__bf16>, grid, dim3(256), 0, s, rows, cols, ldx, (const __bf16*)x, q, scale);
  else if (dtype == MEGAMOE_FP16)
    hipLaunchKernelGGL(k_quantize_int8<_Float16>, grid, dim3(256), 0, s, rows, cols, ldx, (const _Float16*)x, q, scale);
  else
    hipLaunchKernelGGL(k_quantize_int8<float>, grid, dim3(256), 0, s, rows, cols, ldx, (const float*)x, q, scale);
  return launched();
}

}  // extern "C"
