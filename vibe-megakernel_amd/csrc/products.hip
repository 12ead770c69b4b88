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
#include <math.h>
#include <type_traits>
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

// One fragment of A by four of B, accumulated in place: left to itself, the compiler moves the
// accumulators of a long loop between registers and spills. The wait states in front are those
// between a VALU result and an MFMA that reads it, which it cannot see in here. (The results of
// the last MFMAs may be read only after mfma_done().)
#define MEGAMOE_MFMA4(name, c, a, b)                                                                             \
  asm("s_nop 1\n\t" name " %0, %4, %5, %0\n\t" name " %1, %4, %6, %1\n\t" name " %2, %4, %7, %2\n\t" name        \
      " %3, %4, %8, %3"                                                                                          \
      : "+v"(c[0]), "+v"(c[1]), "+v"(c[2]), "+v"(c[3])                                                           \
      : "v"(a), "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]))

// One MFMA with the accumulator in AGPRs, for a wavefront that has a SIMD for itself; FIRST starts it
// at zero. The operands come from LDS reads, so no wait states are needed; mfma_start() has those
// behind what the compiler may copy between two steps.
#define MEGAMOE_MFMA_ACC(name, c, a, b)                                     \
  if constexpr (FIRST)                                                      \
    asm(name " %0, %1, %2, 0" : "=a"(c) : "v"(a), "v"(b));                  \
  else                                                                      \
    asm(name " %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b))

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
  static __device__ __forceinline__ void mfma4(Acc (&c)[4], i32x4 a, const i32x4 (&b)[4]) {
    MEGAMOE_MFMA4("v_mfma_f32_16x16x32_bf16", c, a, b);
  }
  template <bool FIRST>
  static __device__ __forceinline__ void mfma_acc(Acc& c, i32x4 a, i32x4 b) {
    MEGAMOE_MFMA_ACC("v_mfma_f32_16x16x32_bf16", c, a, b);
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
  static __device__ __forceinline__ void mfma4(Acc (&c)[4], i32x4 a, const i32x4 (&b)[4]) {
    MEGAMOE_MFMA4("v_mfma_f32_16x16x32_f16", c, a, b);
  }
  template <bool FIRST>
  static __device__ __forceinline__ void mfma_acc(Acc& c, i32x4 a, i32x4 b) {
    MEGAMOE_MFMA_ACC("v_mfma_f32_16x16x32_f16", c, a, b);
  }
};
struct Int8 {
  using Elem = int8_t;
  using Acc = i32x4;
  static constexpr int kBytes = 1;
  static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ void mfma4(Acc (&c)[4], i32x4 a, const i32x4 (&b)[4]) {
    MEGAMOE_MFMA4("v_mfma_i32_16x16x64_i8", c, a, b);
  }
  template <bool FIRST>
  static __device__ __forceinline__ void mfma_acc(Acc& c, i32x4 a, i32x4 b) {
    MEGAMOE_MFMA_ACC("v_mfma_i32_16x16x64_i8", c, a, b);
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
  for (int g0 = 0; g0 < groups; g0 += 256) {
    int64_t c[4];  // four loads in flight
#pragma unroll
    for (int q = 0; q < 4; ++q) c[q] = g0 + 64 * q + lane < groups ? counts[g0 + 64 * q + lane] : 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (g0 + 64 * q >= groups) break;
      const bool wrong = c[q] < 0 || c[q] > rows;
      bad |= __ballot(wrong) != 0;
      const uint32_t n = wrong ? 0 : (uint32_t)c[q], t = (n + (uint32_t)height - 1) / (uint32_t)height;
      const uint32_t rows_to = add_sat(row0, wave_scan(n)), tiles_to = add_sat(tile0, wave_scan(t));
      const uint64_t mask = __ballot((uint32_t)tile < tiles_to && (uint32_t)tile >= tiles_to - t);
      if (mask) {
        const int l = __builtin_ctzll(mask);
        const int start = (int)(lane_value(rows_to, l) - lane_value(n, l));
        const int within = tile - (int)(lane_value(tiles_to, l) - lane_value(t, l));
        found.group = g0 + 64 * q + l;
        found.first = start + within * height;
        found.last = min(found.first + height, (int)lane_value(rows_to, l));
      }
      row0 = lane_value(rows_to, 63);
      tile0 = lane_value(tiles_to, 63);
    }
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
// A persistent workgroup per CU computes tiles of TI (i) by TJ (j) outputs, stage by stage of c. The
// loads of a stage go straight into LDS (no registers), BUFFERS stages ahead, 64 KB or more in flight
// per CU; its fragments come to registers in halves of 64 bytes of c, one half ahead of the MFMAs.
//
// 256x256: four wavefronts of 128x128 outputs each, one to a SIMD, with the accumulators in AGPRs.
// They read a third less from LDS than eight of 128x64 (128 KB a stage of 128 bytes instead of 192,
// at 128 bytes a clock against 2048 clocks of MFMAs, and 64 KB of loads written besides). A
// wavefront alone has to issue everything between its own MFMAs: in the 16 clocks that one of them
// takes three or four other instructions go, so reads and loads are dealt out singly between them.
// (8192 cubed in bf16: 816 us with eight wavefronts, 800 with four and the reads and loads in bursts,
// 755 so. The MFMAs alone are 457 us at 2.4 GHz, which the card does not hold under them: 1.8 to 2.0.)
// A stage is 128 bytes of c where both operands have c contiguous (whole cache lines: half of them at a
// time took 867 us instead of 755, and 173 instead of 135 for 128 experts of 256 rows, 2048 by 768),
// and its loads go out in its second half, whose fragments are then in registers. It is 64 bytes in
// four buffers instead of two where one has c across, and its loads go out in all of it (y = x w,
// 8192 cubed: 910 us with eight wavefronts, 968 in stages of 128 bytes, 868 so).
//
// 256x128 and 128x128: eight wavefronts, two to a SIMD, that fill each other's pauses; a stage is 128
// bytes. One operand's fragments come to registers of their own, the other's in two parts of which the
// second takes the registers of fragments that are done with.
//
// Either way there is one barrier a stage, behind which the buffer read last is free for loads, and the
// stages of consecutive tiles follow each other without a gap: loads run over the tile's end, so a
// tile's first stages are in LDS when the last tile's results are stored. (A tile has more than
// BUFFERS stages; a short c is padded with zeros.)
//
// LDS layout. An operand with c contiguous: rows of the stage's 128 (64) bytes, 16-byte chunk p of
// row r at position p ^ (r % 8) (p ^ (r / 2 % 4)): one load instruction fills eight (sixteen) whole
// rows, and the MFMA's reads (16 rows of one chunk) fall into different banks. An operand with c
// across: 64 (32) rows (c) of all the tile's i or j, chunk p of row c at p ^ 2 f(c), f = c % 4 +
// 4 (c / 8 % 2): the transposing reads (ds_read_b64_tr_b16: four c of 16 neighbours, for c = 8g ..
// of the lane group g) fall into different banks as well.
//
// Everything outside a tensor reads as zero: rows past the tile's are past the end of the buffer
// resource, chunks past the operand's width get an offset past it.
// ---------------------------------------------------------------------------------------

enum Form { kNT, kNN, kTN };  // y = x w^T, y = x w, dw = dy^T x

constexpr int kThreads = 512, kStage = 128;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Until this wavefront's LDS reads have arrived and at most N of its loads into LDS are pending;
// then the workgroup's wavefronts meet. Nothing moves across it.
template <int N>
__device__ __forceinline__ void meet() {
  static_assert(N >= 0 && N <= 63, "vmcnt holds 6 bits");
  __builtin_amdgcn_sched_barrier(0);
  // gfx9 s_waitcnt immediate: vmcnt[3:0] | expcnt[6:4] | lgkmcnt[11:8] | vmcnt[5:4] << 14
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (((N >> 4) & 3) << 14));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Wait states until the results of every MFMA issued so far can be read.
__device__ __forceinline__ void mfma_done() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Wait states between a VALU result and an MFMA that reads it.
__device__ __forceinline__ void mfma_start() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 1");
  __builtin_amdgcn_sched_barrier(0);
}

// The value of an accumulator in an AGPR, read where it is used.
template <class T>
__device__ __forceinline__ T from_acc(T v) {
  T r;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(r) : "a"(v));
  return r;
}

// LDS at a byte address. The loads into LDS are inline asm without results (load_lds), so the
// compiler counts the LDS reads alone and schedules them under the MFMAs by itself; the waits
// for the loads are the phases' own.
template <class T>
__device__ __forceinline__ T lds_at(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)at;
}
__device__ __forceinline__ i32x2 lds_transposed(uint32_t at) {
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)at));
}

// One operand as this wavefront loads and reads it. COL: c across (else contiguous). L: the load
// instructions of a wavefront per stage; load i fills the 1024 bytes wave + 8 i of the operand.
// STEP: fragments between two of this wavefront.
template <bool COL, int STAGE, int WAVES, int L, int STEP>
struct Side {
  static constexpr uint32_t kRow = COL ? 2048 * WAVES * L / STAGE : STAGE;  // bytes of a row in LDS (COL: all of i or j)
  // Loads in turn that differ in their chunk, where eight c are between two of them.
  static constexpr int kKinds = COL && WAVES * 1024 / kRow % 16 ? 2 : 1;
  uint32_t load[kKinds];   // byte offset of the lane's 16 bytes of the first load from the tile's first row
  uint32_t next;           // from one load of the wavefront to the next
  uint32_t chunk[kKinds];  // of `load`, the bytes along the contiguous dimension
  uint32_t at[COL ? 1 : STAGE / 64];  // LDS addresses of the lane's part of fragment 0

  // `first`: the wavefront's first row; `base`: LDS address of the operand in buffer 0.
  __device__ __forceinline__ void init(uint32_t ld, int wave, int first, uint32_t base) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    if constexpr (COL) {
      constexpr uint32_t kRows = 1024 / kRow, kLanes = 64 / kRows;  // of one load, of one row
      const uint32_t c = kRows * wave + lane / kLanes;
#pragma unroll
      for (uint32_t q = 0; q < kKinds; ++q) {
        chunk[q] = ((lane % kLanes) ^ (2 * ((c & 3) | (((c >> 1) ^ (4 * q)) & 4)))) * 16;
        load[q] = c * ld + chunk[q];
      }
      next = WAVES * kRows * ld;
      at[0] = base + (8 * g + ((lane & 15) >> 2)) * kRow +
              ((((uint32_t)(first >> 3) + ((lane & 3) >> 1)) ^ (2 * (((lane >> 2) & 3) | ((g & 1) << 2)))) << 4) +
              (lane & 1) * 8;
    } else {
      // A load fills 1024 / STAGE rows; chunk p of row r is at p ^ swizzle(r).
      constexpr uint32_t kChunks = STAGE / 16, kRows = 64 / kChunks;
      const uint32_t row = lane / kChunks, r = lane & 15;
      auto swizzle = [](uint32_t row) { return STAGE == 128 ? row & 7 : (row >> 1) & 3; };
      chunk[0] = ((lane % kChunks) ^ swizzle(row)) * 16;
      load[0] = (kRows * wave + row) * ld + chunk[0];
      next = kRows * WAVES * ld;
#pragma unroll
      for (int s = 0; s < STAGE / 64; ++s) at[s] = base + ((uint32_t)first + r) * STAGE + (((4 * s + g) ^ swizzle(r)) << 4);
    }
  }
  // The reads to another buffer, `by` bytes on (or back).
  __device__ __forceinline__ void move(uint32_t by) {
#pragma unroll
    for (uint32_t& a : at) a += by;
  }
  // Fragments BEGIN .. BEGIN + N - 1 (16 rows each) of the stage's half s.
  template <int BEGIN, int N>
  __device__ __forceinline__ void read(i32x4 (&f)[N], int s) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (COL) {
        const uint32_t p = (at[0] ^ (32u * STEP * (BEGIN + i))) + 32 * kRow * s;
        const i32x2 lo = lds_transposed(p), hi = lds_transposed(p + 4 * kRow);
        f[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
      } else {
        f[i] = lds_at<i32x4>(at[s] + 16 * STAGE * STEP * (BEGIN + i));
      }
    }
  }
  template <int I>
  __device__ __forceinline__ void read_one(i32x4& f, int s) const {
    i32x4 one[1];
    read<I>(one, s);
    f = one[0];
  }
};

// An offset past every buffer resource (256 rows of kMaxStrideBytes), also with the loads' largest
// second offset (192 rows and a row) added.
constexpr uint32_t kOutside = 0x80000000u;

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

// The buffer resource of the `bytes` bytes from `base`.
__device__ __forceinline__ i32x4 resource(const void* base, uint32_t bytes) {
  const uint64_t b = (uint64_t)uniform((const uint8_t*)base);
  return i32x4{(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), (int)uniform(bytes), 0x00020000};
}

// 16 bytes a lane into LDS (1024 consecutive ones from byte address `to`), from `base` + at +
// along; zero from `bytes` on. ONCE: past the caches. (Five wait states have to be between a
// v_readfirstlane and a load that reads its SGPR; in here the compiler does not put them in.)
template <bool ONCE>
__device__ __forceinline__ void load_lds(uint32_t to, const uint8_t* base, uint32_t bytes, uint32_t at, uint32_t along) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                 :
                 : "s"(uniform(to)), "v"(at), "s"(resource(base, bytes)), "s"(uniform(along))
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(uniform(to)), "v"(at), "s"(resource(base, bytes)), "s"(uniform(along))
                 : "memory", "m0");
#endif
}

// The same with 4 bytes a lane: `count` floats (up to 64, zero behind them).
__device__ __forceinline__ void load_floats(uint32_t to, const float* base, int count) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(uniform(to)), "v"((threadIdx.x & 63) * 4), "s"(resource(base, (uint32_t)max(count, 0) * 4))
               : "memory", "m0");
#endif
}

// Load I of one operand's stage: `live` tells the lanes whose bytes exist, `bytes` the length of
// the rows that do (the range check takes the sum of both offsets).
template <int I, bool ONCE = false, bool COL, int STAGE, int WAVES, int L, int STEP>
__device__ __forceinline__ void load_one(uint32_t to, int wave, const uint8_t* base, uint32_t bytes,
                                         const Side<COL, STAGE, WAVES, L, STEP>& side, bool live, uint32_t along) {
  load_lds<ONCE>(to + (uint32_t)(wave + WAVES * I) * 1024, base, bytes,
                 live ? side.load[I % side.kKinds] : kOutside, along + I * side.next);
}

// The same load of a row of them, 4096 bytes of LDS and `next` of the operand apart: I of them, with
// `along` starting one `next` in front. The resource, `to` and `along` come from settled().
template <int I, bool ONCE>
__device__ __forceinline__ void load_next(uint32_t to, i32x4 from, uint32_t at, uint32_t& along, uint32_t next) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (ONCE)
    asm volatile("s_add_u32 m0, %1, %5\n\ts_add_u32 %0, %0, %4\n\tbuffer_load_dwordx4 %2, %3, %0 offen nt lds"
                 : "+s"(along)
                 : "s"(to), "v"(at), "s"(from), "s"(next), "i"(4096 * I)
                 : "memory", "m0", "scc");
  else
    asm volatile("s_add_u32 m0, %1, %5\n\ts_add_u32 %0, %0, %4\n\tbuffer_load_dwordx4 %2, %3, %0 offen lds"
                 : "+s"(along)
                 : "s"(to), "v"(at), "s"(from), "s"(next), "i"(4096 * I)
                 : "memory", "m0", "scc");
#endif
}
// What load_next() takes, with the wait states between a v_readfirstlane and a load behind it.
__device__ __forceinline__ void settled(i32x4& from, uint32_t& to, uint32_t& along, uint32_t& next) {
#ifdef __HIP_DEVICE_COMPILE__
  int f0 = uniform(from[0]), f1 = uniform(from[1]), f2 = uniform(from[2]), f3 = uniform(from[3]);
  to = uniform(to), along = uniform(along), next = uniform(next);
  asm volatile("s_nop 4" : "+s"(f0), "+s"(f1), "+s"(f2), "+s"(f3), "+s"(to), "+s"(along), "+s"(next));
  from = i32x4{f0, f1, f2, f3};
#endif
}

// Calls f(std::integral_constant<int, I>{}) for I = B .. E-1.
template <int B, int E, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (B < E) {
    f(std::integral_constant<int, B>{});
    static_for<B + 1, E>(f);
  }
}

// The lane index, opaque to the compiler: what is derived from it is not kept in registers across
// the loop that it is used behind.
__device__ __forceinline__ int opaque_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// The groups' tables in LDS: before each group (entry g), and to the end of the last (entry `groups`
// and on), its rows, its tiles of more than half the height (all but its last, perhaps) and its
// smaller ones (its last, perhaps).
struct Table {
  uint32_t rows[kMaxGroups + 16], tiles[kMaxGroups + 16], small[kMaxGroups + 16];
};

// Fills the table; false if the counts do not fit the rows. Every thread of the workgroup calls it.
__device__ bool make_table(Table& t, const Args& p, int height) {
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x; g < p.groups; g += blockDim.x) {
    const int64_t v = p.counts ? p.counts[g] : p.rows;
    t.rows[g] = v < 0 || v > p.rows ? 0xffffffffu : (uint32_t)v;  // sums saturate at a value past the rows
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t row0 = 0, tile0 = 0, small0 = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
      const uint32_t c = g0 + lane < p.groups ? t.rows[g0 + lane] : 0u, rest = c % (uint32_t)height;
      const uint32_t half = (uint32_t)height / 2, n = c / (uint32_t)height + (rest > half), s = rest > 0 && rest <= half;
      const uint32_t rows_to = add_sat(row0, wave_scan(c)), tiles_to = add_sat(tile0, wave_scan(n));
      const uint32_t small_to = small0 + wave_scan(s);
      t.rows[g0 + lane] = rows_to - c;  // exact wherever the sums are
      t.tiles[g0 + lane] = tiles_to - n;
      t.small[g0 + lane] = small_to - s;
      row0 = lane_value(rows_to, 63);
      tile0 = lane_value(tiles_to, 63);
      small0 = lane_value(small_to, 63);
    }
    for (int g = (p.groups + 63) / 64 * 64 + lane; g < kMaxGroups + 16; g += 64) {
      t.rows[g] = row0;
      t.tiles[g] = tile0;
      t.small[g] = small0;
    }
  }
  __syncthreads();
  return t.rows[kMaxGroups] <= (uint32_t)p.rows;
}

// Row tile `tile` (below the table's total): its group and rows. The tiles of more than half the
// height come first, so that the last ones of a launch are the short ones.
__device__ __forceinline__ Tile table_tile(const Table& t, int tile, int height) {
  const int lane = threadIdx.x & 63;
  const int big = uniform((int)t.tiles[kMaxGroups]);
  const bool small = tile >= big;
  const uint32_t* const before = small ? t.small : t.tiles;
  const uint32_t at = (uint32_t)(small ? tile - big : tile);
  const int block = __builtin_popcountll(__ballot(before[16 * lane + 16] <= at));
  const int group = 16 * block + __builtin_popcountll(__ballot(before[16 * block + 1 + (lane & 15)] <= at) & 0xffff);
  const uint32_t v = lane < 2 ? t.tiles[group + lane] : t.rows[group + (lane & 1)];
  const int within = small ? (int)(lane_value(v, 1) - lane_value(v, 0)) : (int)(at - lane_value(v, 0));
  const int first = (int)lane_value(v, 2) + within * height;
  return Tile{group, first, min(first + height, (int)lane_value(v, 3))};
}

// Workgroups of a grid go to the eight XCDs in turn, each with an L2 of its own: step s of the
// persistent grid is `grid` consecutive tiles, of which each XCD takes a consecutive eighth. The
// last tiles of several steps go to the workgroups whose step before was the shortest, the last
// ones. -1: none for this workgroup.
__device__ __forceinline__ int xcd_tile(int step, int total) {
  const int grid = (int)gridDim.x, first = step * grid, left = min(total - first, grid);
  if (left <= 0) return -1;
  const int xcd = (int)blockIdx.x & 7, in = (int)blockIdx.x >> 3;
  if (step > 0 && left < grid) {
    const int at = xcd * (grid / 8) + in - (grid - left);
    return at >= 0 ? first + at : -1;
  }
  const int each = (left + 7) / 8, at = xcd * each + in;
  return in < each && at < left ? first + at : -1;
}

// Groups start at different places of c: rows whose pitch is a large power of two (4 KB and on) would
// otherwise have all workgroups at addresses of few memory channels (256 experts of 2 rows, 4096 by
// 2048: 655 us without, 607 with it; pitches of no such power are indifferent to it).
constexpr uint32_t kTurn = 3;

constexpr int kBand = 4;  // row tiles that are walked together, column by column

// What the loads need of a tile, and the results.
struct Work {
  const uint8_t* a;  // first rows of the operands
  const uint8_t* b;
  int group, first, last;  // rows of y (the products), of the group (the weights' gradient)
  int i0, j0;              // first column and row of the output tile (j0: within rows first..last)
  int stages;
  int place;               // of its scales
  int turn;                // the stage that comes first (c is walked in a circle)
  uint32_t rows_a, rows_b;  // bytes of the rows that exist (c contiguous)
};

// Workgroups of a CU: two where tiles are mostly their start and their end, the small ones of the
// weights' gradient, so that one of them multiplies while the other stores (13 experts, 1736 by 1000,
// 1235 rows: 41.9 us with one that loads further ahead, 29.2 with two; 8 experts, 1024 by 512, 64 rows:
// 10.8 and 9.1). The products want the loads further ahead (4096 by 4096, 512 rows: 36.8 us against
// 46.0).
template <Form FORM, int TI>
constexpr int kPerCu = FORM == kTN && TI == 128 ? 2 : 1;

// Wavefronts of a workgroup.
template <int TI, int TJ>
constexpr int kWaves = TI == 256 && TJ == 256 ? 4 : 8;

template <class Ty, class Out, Form FORM, int TI, int TJ, bool ONCE>
__global__ __launch_bounds__((64 * kWaves<TI, TJ>), (kWaves<TI, TJ> / 4 * kPerCu<FORM, TI>)) void k_tiles(Args p) {
  constexpr bool kAcol = FORM != kNT, kBcol = FORM == kTN;
  constexpr int WAVES = kWaves<TI, TJ>, THREADS = 64 * WAVES;
  constexpr bool FOUR = WAVES == 4;
  constexpr int WJ = FOUR ? 2 : TJ / 64, WI = WAVES / WJ;           // wavefronts along i and j
  constexpr int FA = TI / WI / 16, FB = TJ / WJ / 16, FH = FA / 2;  // fragments of a wavefront
  static_assert(FB == (FOUR ? 8 : 4), "mfma4");
  // Four wavefronts take the fragments of j in turn, so that a tile of at most half the height has
  // half of the fragments of each.
  constexpr int STEP = FOUR ? WJ : 1;
  constexpr int STAGE = FOUR && (kAcol || kBcol) ? 64 : kStage;     // bytes of c
  constexpr int HALVES = STAGE / 64;
  constexpr int LA = TI * STAGE / 1024 / WAVES, LB = TJ * STAGE / 1024 / WAVES;  // loads of a wavefront per stage
  constexpr int kBytesA = TI * STAGE, kBytes = kBytesA + TJ * STAGE;
  constexpr int BUFFERS = 147456 / kPerCu<FORM, TI> / kBytes;
  constexpr int kPending = (BUFFERS - 2) * (LA + LB);
  constexpr int kC = STAGE / Ty::kBytes;  // c of one stage
  __shared__ __align__(1024) uint8_t lds[BUFFERS * kBytes];
  __shared__ Table table;
  // The int8 product's scales of two tiles' i and j, loaded with the tile's first stage.
  __shared__ __align__(16) float scales[2][Ty::kBytes == 1 ? TI + TJ : 1];

  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wi = wave % WI, wj = wave / WI;
  Out* const out = reinterpret_cast<Out*>(p.out);
  const int ni = FORM == kTN ? p.k : p.n;
  const int64_t ldo = FORM == kTN ? p.k : p.ldy;
  const int tiles_i = (ni + TI - 1) / TI;

  const bool fits = uniform((int)make_table(table, p, TJ)) != 0;
  if (!fits) {  // NaN everywhere
    const int64_t rows = FORM == kTN ? (int64_t)p.groups * p.n : p.rows;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
      for (int i = threadIdx.x; i < ni; i += THREADS) out[r * ldo + i] = (Out)__builtin_nanf("");
    return;
  }
  const int used = uniform((int)table.rows[kMaxGroups]);
  const int row_tiles = FORM == kTN ? p.groups * ((p.n + TJ - 1) / TJ)
                                    : uniform((int)(table.tiles[kMaxGroups] + table.small[kMaxGroups]));
  const int total = row_tiles * tiles_i;
  if (FORM != kTN && p.fill_rest)  // the last workgroups first: the ones that may have no tile
    for (int64_t r = used + (gridDim.x - 1 - blockIdx.x); r < p.rows; r += gridDim.x)
      for (int i = threadIdx.x; i < ni; i += THREADS) out[r * ldo + i] = (Out)0.f;

  const int64_t lda = (int64_t)Ty::kBytes * (FORM == kNT ? p.k : FORM == kNN ? p.n : p.ldx);
  const int64_t ldb = (int64_t)Ty::kBytes * (FORM == kTN ? p.ldy : p.ldx);
  // A tile's stages: more than the buffers, and with four wavefronts, which take two in turn, even.
  auto whole = [](int stages) { return FOUR && HALVES == 1 ? max(BUFFERS + 2, (stages + 1) / 2 * 2) : max(BUFFERS + 1, stages); };
  auto locate_work = [&](int tile) __attribute__((always_inline)) {
    const int width = kBand * tiles_i, band = tile / width, in = tile % width;
    const int high = min(kBand, row_tiles - band * kBand);
    const int rt = band * kBand + in % high, it = in / high;
    Work w;
    w.i0 = it * TI;
    if constexpr (FORM == kTN) {
      const int tiles_j = (p.n + TJ - 1) / TJ;
      w.group = rt / tiles_j;
      w.j0 = rt % tiles_j * TJ;
      const uint32_t v = table.rows[w.group + (lane & 1)];
      w.first = (int)lane_value(v, 0);
      w.last = (int)lane_value(v, 1);
      w.a = p.x + (int64_t)w.first * lda + (int64_t)w.i0 * Ty::kBytes;
      w.b = p.w + (int64_t)w.first * ldb + (int64_t)w.j0 * Ty::kBytes;
      w.stages = whole((w.last - w.first + kC - 1) / kC);
    } else {
      const Tile t = table_tile(table, rt, TJ);
      w.group = t.group;
      w.first = t.first;
      w.last = t.last;
      w.j0 = 0;
      w.a = p.w + (size_t)w.group * p.n * p.k * Ty::kBytes +
            (FORM == kNT ? (int64_t)w.i0 * lda : (int64_t)w.i0 * Ty::kBytes);
      w.b = p.x + (int64_t)w.first * ldb;
      w.stages = whole((p.k + kC - 1) / kC);
    }
    w.turn = FORM == kTN ? 0 : uniform((int)((uint32_t)w.group * (kTurn * kStage / STAGE) % (uint32_t)w.stages));
    w.rows_a = uniform((uint32_t)min(p.n - w.i0, TI) * (uint32_t)lda);
    w.rows_b = uniform((uint32_t)(w.last - w.first) * (uint32_t)ldb);
    return w;
  };

  int step = 0;
  int tile = xcd_tile(step, total);
  if (tile < 0) return;
  Work ahead = locate_work(tile);  // the tile that is being loaded
  ahead.place = 0;
  Work now = ahead;                // the tile that is being multiplied
  int stage = 0;                   // of `ahead`
  bool more = true;

  Side<kAcol, STAGE, WAVES, LA, 1> sa;
  Side<kBcol, STAGE, WAVES, LB, STEP> sb;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  sa.init((uint32_t)lda, wave, wi * (TI / WI), lds0);
  const int wave_j = FOUR ? 16 * wj : wj * (TJ / WJ);  // the wavefront's first j
  sb.init((uint32_t)ldb, wave, wave_j, lds0 + kBytesA);

  uint32_t row_bytes = (uint32_t)p.k * Ty::kBytes;  // (kept in a register, not loaded again in the loop)
  asm("" : "+s"(row_bytes));
  // Load `i` of A's (or B's) loads at the load cursor, into buffer `buf`.
  auto at_stage = [&]() {
    const int s = stage + ahead.turn;
    return s >= ahead.stages && more ? s - ahead.stages : s;
  };
  auto load_scales = [&]() __attribute__((always_inline)) {
    if (stage == 0 && more) {
      const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float*)scales[ahead.place];
      if (wave < TI / 64)
        load_floats(at + 256 * wave, p.sw + (size_t)ahead.group * p.n + ahead.i0 + 64 * wave,
                    min(p.n - ahead.i0 - 64 * wave, 64));
      const int part = wave - (WAVES - TJ / 64);
      if (part >= 0)
        load_floats(at + 4 * TI + 256 * part, p.sx + ahead.first + 64 * part, min(ahead.last - ahead.first - 64 * part, 64));
    }
  };
  auto load_a = [&](auto i, int buf) {
    if constexpr (Ty::kBytes == 1 && i.value == 0) load_scales();
    const int stage = at_stage();
    const uint32_t to = lds0 + buf * kBytes;
    if constexpr (kAcol) {
      const int rows = (FORM == kTN ? ahead.last - ahead.first : p.k) - stage * kC;
      load_one<i.value, ONCE>(to, wave, ahead.a + (int64_t)stage * kC * lda,
                       more ? (uint32_t)min(max(rows, 0), kC) * (uint32_t)lda : 0u, sa,
                       sa.chunk[i.value % sa.kKinds] < (uint32_t)(ni - ahead.i0) * Ty::kBytes, 0u);
    } else {
      load_one<i.value, ONCE>(to, wave, ahead.a, ahead.rows_a, sa,
                       (uint32_t)stage * STAGE + sa.chunk[0] < row_bytes, (uint32_t)stage * STAGE);
    }
  };
  auto load_b = [&](auto i, int buf) {
    const int stage = at_stage();
    const uint32_t to = lds0 + buf * kBytes + kBytesA;
    if constexpr (kBcol) {
      const int rows = ahead.last - ahead.first - stage * kC;
      load_one<i.value>(to, wave, ahead.b + (int64_t)stage * kC * ldb,
                       more ? (uint32_t)min(max(rows, 0), kC) * (uint32_t)ldb : 0u, sb,
                       sb.chunk[i.value % sb.kKinds] < (uint32_t)(p.n - ahead.j0) * Ty::kBytes, 0u);
    } else {
      load_one<i.value>(to, wave, ahead.b, ahead.rows_b, sb,
                       (uint32_t)stage * STAGE + sb.chunk[0] < row_bytes, (uint32_t)stage * STAGE);
    }
  };
  // The load cursor to the next stage, over the tile's end.
  auto advance = [&]() __attribute__((always_inline)) {
    if (++stage < ahead.stages || !more) return;
    stage = 0;
    tile = xcd_tile(++step, total);
    more = tile >= 0;
    const int place = ahead.place ^ 1;
    if (more)
      ahead = locate_work(tile);
    else
      ahead.rows_a = ahead.rows_b = 0;
    ahead.place = place;
  };

  typename Ty::Acc acc[FA][FB];
  // Results: lane l has i = 4 (l / 16) .. +3 of a fragment at j = l % 16.
  auto store = [&]() {
    mfma_done();
    const int lane = opaque_lane();
    constexpr int kWide = 16 / (int)sizeof(Out);  // outputs of one store
    typedef Out OutN __attribute__((ext_vector_type(kWide)));
    const bool wide = ldo % kWide == 0 && ni % kWide == 0 && (uintptr_t)p.out % 16 == 0;
    const int nj = (FORM == kTN ? p.n : now.last - now.first) - now.j0;
    // (Stores past the buffer, to kOutside, are dropped: no branches.)
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(
        uniform(out + (FORM == kTN ? (size_t)now.group * p.n * p.k + (int64_t)now.j0 * ldo : (int64_t)now.first * ldo) + now.i0),
        0, kOutside - 1, 0x00020000);
    f32x4 sw[FA];
    if constexpr (Ty::kBytes == 1) {
#pragma unroll
      for (int f = 0; f < FA; ++f)
        sw[f] = *reinterpret_cast<const f32x4*>(&scales[now.place][wi * (TI / WI) + 16 * f + 4 * (lane >> 4)]);
    }
    auto all = [&](auto wide) {
#pragma unroll
      for (int t = 0; t < FB; ++t) {
        const int j = wave_j + 16 * STEP * t + (lane & 15);
        float sx = 0.f;
        if constexpr (Ty::kBytes == 1) sx = scales[now.place][TI + wave_j + 16 * STEP * t + (lane & 15)];
        auto value = [&](int f, int e) {
          const auto v = FOUR ? from_acc(acc[f][t][e]) : acc[f][t][e];
          if constexpr (Ty::kBytes == 1)
            return scaled(v, sx, sw[f][e]);
          else
            return v;
        };
        auto put = [&](int i, OutN v) {
          const uint32_t at = ((uint32_t)j * (uint32_t)ldo + (uint32_t)i) * (uint32_t)sizeof(Out);
          if constexpr (wide.value) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, j < nj && now.i0 + i < ni ? at : kOutside, 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < kWide; ++e) {
              const Out element = v[e];  // (__builtin_bit_cast of v[e] itself takes v[0])
              const uint32_t one = j < nj && now.i0 + i + e < ni ? at + e * (uint32_t)sizeof(Out) : kOutside;
              if constexpr (sizeof(Out) == 2)
                __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, element), to, one, 0, 0);
              else
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, element), to, one, 0, 0);
            }
          }
        };
#pragma unroll
        for (int f = 0; f < FA; f += kWide / 4) {
          const int i = wi * (TI / WI) + 16 * f;
          if constexpr (kWide == 4) {
            put(i + 4 * (lane >> 4), OutN{(Out)value(f, 0), (Out)value(f, 1), (Out)value(f, 2), (Out)value(f, 3)});
          } else {
            // Two fragments' halves change places between neighbouring groups of 16 lanes, so that a
            // lane has eight neighbours of one of them.
            typedef Out Out2 __attribute__((ext_vector_type(2)));
            uint32_t u[2][2];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                u[q][h] = __builtin_bit_cast(uint32_t, Out2{(Out)value(f + q, 2 * h), (Out)value(f + q, 2 * h + 1)});
            const auto lo = __builtin_amdgcn_permlane16_swap(u[0][0], u[1][0], false, false);
            const auto hi = __builtin_amdgcn_permlane16_swap(u[0][1], u[1][1], false, false);
            const i32x4 all = {(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
            put(i + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5), __builtin_bit_cast(OutN, all));
          }
        }
      }
    };
    if (wide) all(std::true_type{});
    else all(std::false_type{});
  };

  for (int i = 0; i < BUFFERS; ++i) {
    static_for<0, LA>([&](auto l) { load_a(l, i); });
    static_for<0, LB>([&](auto l) { load_b(l, i); });
    advance();
  }
  meet<(FOUR && HALVES == 1 ? BUFFERS - 2 : BUFFERS - 1) * (LA + LB)>();
  int buf = 0, last = 0;  // the buffer that is read, and the one before it
  auto next_buffer = [&]() {
    last = buf;
    buf = buf + 1 == BUFFERS ? 0 : buf + 1;
    sa.move(buf == 0 ? -(BUFFERS - 1) * kBytes : kBytes);
    sb.move(buf == 0 ? -(BUFFERS - 1) * kBytes : kBytes);
  };
  if constexpr (FOUR) {
    // What is loaded of one operand at the load cursor.
    struct Loads {
      i32x4 from;
      uint32_t to, along, next, at[2];
    };
    auto loads_a = [&](int buf) __attribute__((always_inline)) {
      const int stage = at_stage();
      Loads l;
      if constexpr (kAcol) {
        const int rows = (FORM == kTN ? ahead.last - ahead.first : p.k) - stage * kC;
        l.from = resource(ahead.a + (int64_t)stage * kC * lda, more ? (uint32_t)min(max(rows, 0), kC) * (uint32_t)lda : 0u);
        l.along = 0u - sa.next;
#pragma unroll
        for (int q = 0; q < sa.kKinds; ++q)
          l.at[q] = sa.chunk[q] < (uint32_t)(ni - ahead.i0) * Ty::kBytes ? sa.load[q] : kOutside;
      } else {
        l.from = resource(ahead.a, ahead.rows_a);
        l.along = (uint32_t)stage * STAGE - sa.next;
        l.at[0] = (uint32_t)stage * STAGE + sa.chunk[0] < row_bytes ? sa.load[0] : kOutside;
      }
      l.to = lds0 + buf * kBytes + wave * 1024;
      l.next = sa.next;
      settled(l.from, l.to, l.along, l.next);
      return l;
    };
    auto loads_b = [&](int buf) __attribute__((always_inline)) {
      const int stage = at_stage();
      Loads l;
      if constexpr (kBcol) {
        const int rows = ahead.last - ahead.first - stage * kC;
        l.from = resource(ahead.b + (int64_t)stage * kC * ldb, more ? (uint32_t)min(max(rows, 0), kC) * (uint32_t)ldb : 0u);
        l.along = 0u - sb.next;
#pragma unroll
        for (int q = 0; q < sb.kKinds; ++q)
          l.at[q] = sb.chunk[q] < (uint32_t)(p.n - ahead.j0) * Ty::kBytes ? sb.load[q] : kOutside;
      } else {
        l.from = resource(ahead.b, ahead.rows_b);
        l.along = (uint32_t)stage * STAGE - sb.next;
        l.at[0] = (uint32_t)stage * STAGE + sb.chunk[0] < row_bytes ? sb.load[0] : kOutside;
      }
      l.to = lds0 + buf * kBytes + kBytesA + wave * 1024;
      l.next = sb.next;
      settled(l.from, l.to, l.along, l.next);
      return l;
    };
    // Read I of a stage's fragments, in the order of their use.
    auto read = [&](auto i, auto wide, i32x4(&a)[FA], i32x4(&b)[FB], int s) __attribute__((always_inline)) {
      constexpr int I = i.value;
      if constexpr (I < 4) sb.template read_one<I>(b[I], s);
      else if constexpr (I == 4) sa.template read_one<0>(a[0], s);
      else if constexpr (!wide.value) sa.template read_one<I - 4>(a[I - 4], s);
      else if constexpr (I < 9) sb.template read_one<I - 1>(b[I - 1], s);
      else sa.template read_one<I - 8>(a[I - 8], s);
    };
    // One stage: a by b, while the next one's fragments arrive in an and bn (all of them for the
    // `last` of a narrow tile, as the next tile may be a wide one), and the loads of the stage
    // BUFFERS on are issued into this one's buffer: after every MFMA at most a few instructions, or
    // the matrix pipe would run dry.
    auto step_of = [&](auto half, auto first, auto wide, auto last_one, const i32x4(&a)[FA], const i32x4(&b)[FB], i32x4(&an)[FA],
                        i32x4(&bn)[FB]) __attribute__((always_inline)) {
      constexpr int NB = wide.value ? FB : FB / 2, MFMAS = FA * NB;
      constexpr bool kAll = wide.value || last_one.value;
      constexpr int READS = kAll ? FA + FB : FA + FB / 2;
      // Of a stage of two halves, the first one's step reads on in its buffer, the other one's loads.
      constexpr bool kReadOn = HALVES == 2 && half.value == 0, kMeet = HALVES == 1 || kReadOn;
      Loads la, lb;
      const int from = buf;
      if constexpr (!kReadOn) next_buffer();
      mfma_start();
      static_for<0, MFMAS>([&](auto m) __attribute__((always_inline)) {
        constexpr int M = m.value;
        if constexpr (!kReadOn && M == 0) la = loads_a(from);
        if constexpr (!kReadOn && M == MFMAS / 2) lb = loads_b(from);
        if constexpr (!kReadOn && Ty::kBytes == 1 && M == 1) load_scales();
        // Reads over the first half, loads over all of it.
        static_for<(M < MFMAS / 2 ? READS * M / (MFMAS / 2) : READS), (M < MFMAS / 2 ? READS * (M + 1) / (MFMAS / 2) : READS)>(
            [&](auto i) { read(i, std::bool_constant<kAll>{}, an, bn, kReadOn ? 1 : 0); });
        constexpr int kEach = MFMAS / (LA + LB), L = M / kEach;
        if constexpr (!kReadOn && M % kEach == kEach - 2) {
          if constexpr (L < LA) load_next<L, ONCE>(la.to, la.from, la.at[L % sa.kKinds], la.along, la.next);
          else load_next<L - LA, false>(lb.to, lb.from, lb.at[(L - LA) % sb.kKinds], lb.along, lb.next);
        }
        __builtin_amdgcn_sched_barrier(0);
        Ty::template mfma_acc<first.value>(acc[M / NB][M % NB], a[M / NB], b[M % NB]);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (!kReadOn) advance();
      if constexpr (kMeet) meet<kPending>();
    };
    i32x4 a0[FA], b0[FB], a1[FA], b1[FB];  // fragments of two stages
    auto tile = [&](auto wide) __attribute__((always_inline)) {
      constexpr std::false_type no;
      constexpr std::true_type yes;
      constexpr std::integral_constant<int, 0> lower;
      constexpr std::integral_constant<int, HALVES - 1> upper;
      step_of(lower, yes, wide, no, a0, b0, a1, b1);
      step_of(upper, no, wide, no, a1, b1, a0, b0);
      for (int left = now.stages * HALVES - 4; left > 0; left -= 2) {
        step_of(lower, no, wide, no, a0, b0, a1, b1);
        step_of(upper, no, wide, no, a1, b1, a0, b0);
      }
      step_of(lower, no, wide, no, a0, b0, a1, b1);
      step_of(upper, no, wide, yes, a1, b1, a0, b0);
    };
    static_for<0, FA + FB>([&](auto i) { read(i, std::true_type{}, a0, b0, 0); });
    if constexpr (HALVES == 1) meet<kPending>();
    for (;;) {
      const int nj = FORM == kTN ? p.n - now.j0 : now.last - now.first;
      if (nj > TJ / 2) {
        tile(std::true_type{});
      } else {
        tile(std::false_type{});
        // The others' results are not stored: they need not outlive the loop.
#pragma unroll
        for (int f = 0; f < FA; ++f)
#pragma unroll
          for (int t = FB / 2; t < FB; ++t) asm("" : "=a"(acc[f][t]));
      }
      store();
      if (!more) break;  // (the loads are BUFFERS stages ahead, within the next tile)
      now = ahead;
    }
  } else {
    // A's fragments of the lower and upper rows, one set more, and B's of two halves.
    i32x4 x[FH], y[FH], z[FH], b0[FB], b1[FB];
    auto clear = [&]() {
#pragma unroll
      for (int f = 0; f < FA; ++f)
#pragma unroll
        for (int t = 0; t < FB; ++t) acc[f][t] = typename Ty::Acc{0, 0, 0, 0};
    };
    // Fragments at .. at + n - 1 of a[], which are f0 .. of the tile, by b; the scheduler keeps it in
    // one piece.
    auto multiply = [&](const i32x4(&a)[FH], int f0, const i32x4(&b)[FB], int at, int n) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = at; f < at + n; ++f) Ty::mfma4(acc[f0 + f], a[f], b);
      __builtin_amdgcn_sched_barrier(0);
    };

    sb.template read<0>(b0, 0);
    sa.template read<0>(x, 0);
    sa.template read<FH>(y, 0);
    for (;;) {
      clear();
      const int nj = FORM == kTN ? p.n - now.j0 : now.last - now.first;
      if (wj * (TJ / WJ) < nj) {
        for (int left = now.stages; left > 0; --left) {
          // First half of the stage: x, y and b0. The second half's fragments arrive in z, x and b1.
          sb.template read<0>(b1, 1);
          sa.template read<0>(z, 1);
          multiply(x, 0, b0, 0, FH);
          sa.template read<FH>(x, 1);
          multiply(y, FH, b0, 0, FH);
          meet<kPending>();
          // Second half: z, x and b1. The next stage's first half arrives in x, y and b0.
          next_buffer();
          sb.template read<0>(b0, 0);
          static_for<0, LA>([&](auto l) { load_a(l, last); });
          sa.template read<FH>(y, 0);
          multiply(x, FH, b1, 0, FH / 2);
          static_for<0, LB>([&](auto l) { load_b(l, last); });
          multiply(x, FH, b1, FH / 2, FH - FH / 2);
          sa.template read<0>(x, 0);
          multiply(z, 0, b1, 0, FH);
          advance();
        }
      } else {
        // No rows for this wavefront: it loads, and leaves the MFMAs to the one beside it (of a tile
        // of at most half the height, every SIMD has one of either kind).
        for (int left = now.stages; left > 0; --left) {
          meet<kPending>();
          next_buffer();
          static_for<0, LA>([&](auto l) { load_a(l, last); });
          static_for<0, LB>([&](auto l) { load_b(l, last); });
          advance();
        }
        sb.template read<0>(b0, 0);
        sa.template read<0>(x, 0);
        sa.template read<FH>(y, 0);
      }
      store();
      if (!more) break;  // (the loads are BUFFERS + 1 stages ahead, within the next tile)
      now = ahead;
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // loads into LDS may not outlive the workgroup
}

// ---------------------------------------------------------------------------------------
// The product by strips (16-byte aligned operands, c contiguous): calls with too few tiles to
// occupy the GPU
//
// A workgroup of eight wavefronts computes 16 MI by 16 MJ outputs, the wavefronts taking the
// 128-byte steps of c in turn; their sums are added through LDS in wavefront order. A step's
// fragments are loaded straight into registers: lane l has the 32 bytes at 32 * (l / 16) of row
// l % 16, so four lanes cover a whole 128-byte line (the MFMAs see c in another order, the same
// for both operands). kDeep steps are in flight per wavefront, 16 wavefronts on a CU.
// ---------------------------------------------------------------------------------------

constexpr int kDeep = 4;

// 16 bytes a lane from `base` + at + along; zero from `bytes` on.
__device__ __forceinline__ i32x4 load_16(const uint8_t* base, uint32_t bytes, uint32_t at, uint32_t along) {
#ifdef __HIP_DEVICE_COMPILE__
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)uniform(base), 0, uniform(bytes), 0x00020000);
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, along, 0));
#else
  return i32x4{};
#endif
}

template <class Ty, class Out, int MI, int MJ>
__global__ __launch_bounds__(kThreads, 4) void k_strips(Args p) {
  __shared__ typename Ty::Acc part[8][MI * MJ][64];
  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t kbytes = (uint32_t)p.k * Ty::kBytes;
  const uint32_t lda = kbytes, ldb = (uint32_t)(p.ldx * Ty::kBytes);
  const int steps = (int)((kbytes + 127) / 128);
  Out* const out = reinterpret_cast<Out*>(p.out);
  const int64_t total = (int64_t)p.tiles_j * p.tiles_i;
  for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
    const int i0 = (int)(at % p.tiles_i) * 16 * MI, i1 = min(i0 + 16 * MI, p.n);
    const Tile t = locate(p.counts, p.groups, p.rows, 16 * MJ, (int)(at / p.tiles_i));
    if (t.group == kNoTile) continue;
    if (t.group < 0) {
      if (t.group == kBad || p.fill_rest)
        fill_rows(out, p.ldy, t.first, t.last, i0, i1, t.group == kBad ? __builtin_nanf("") : 0.f);
      continue;
    }
    const uint8_t* const a = p.w + ((size_t)t.group * p.n + i0) * kbytes;
    const uint8_t* const b = p.x + (int64_t)t.first * p.ldx * Ty::kBytes;
    const uint32_t rows_a = (uint32_t)(i1 - i0) * lda, rows_b = (uint32_t)(t.last - t.first) * ldb;
    const uint32_t part_c = (uint32_t)(lane >> 4) * 32;
    typename Ty::Acc acc[MI][MJ] = {};
    for (int s0 = wave; s0 < steps; s0 += 8 * kDeep) {
      i32x4 fa[kDeep][MI][2], fb[kDeep][MJ][2];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const uint32_t along = (uint32_t)(s0 + 8 * d) * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t c = part_c + 16 * h;
          const bool live = along + c < kbytes;
#pragma unroll
          for (int m = 0; m < MI; ++m)
            fa[d][m][h] = load_16(a, rows_a, live ? (16 * m + (lane & 15)) * lda + c : kOutside, along);
#pragma unroll
          for (int m = 0; m < MJ; ++m)
            fb[d][m][h] = load_16(b, rows_b, live ? (16 * m + (lane & 15)) * ldb + c : kOutside, along);
        }
      }
#pragma unroll
      for (int d = 0; d < kDeep; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int m = 0; m < MI; ++m)
#pragma unroll
            for (int n = 0; n < MJ; ++n) acc[m][n] = Ty::mfma(fa[d][m][h], fb[d][n][h], acc[m][n]);
    }
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < MJ; ++n) part[wave][m * MJ + n][lane] = acc[m][n];
    __syncthreads();
    for (int o = threadIdx.x; o < 256 * MI * MJ; o += kThreads) {
      const int j = o / (16 * MI), i = o % (16 * MI);
      if (i0 + i < i1 && t.first + j < t.last) {
        const int f = i / 16 * MJ + j / 16, l = (i % 16 / 4) * 16 + j % 16;
        auto sum = part[0][f][l][i % 4];
#pragma unroll
        for (int w = 1; w < 8; ++w) sum += part[w][f][l][i % 4];
        float v;
        if constexpr (Ty::kBytes == 1)
          v = scaled(sum, p.sx[t.first + j], p.sw[(size_t)t.group * p.n + i0 + i]);
        else
          v = sum;
        out[(int64_t)(t.first + j) * p.ldy + i0 + i] = (Out)v;
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// Rows to int8
//
// One pass over the row: it is held in registers (CHUNKS 16-byte chunks a thread) between the
// search for the largest magnitude and the rounding, so each byte is read once. The search runs
// on the magnitudes' bits, where NaN and infinity are the largest. Rows of other alignments, and
// longer ones, are read twice, element by element.
// ---------------------------------------------------------------------------------------

// The row's scale (thread 0 writes it) and 127 / a from the largest magnitude's bits; 0 for a row
// that holds NaN or an infinity.
__device__ __forceinline__ float int8_factor(uint32_t largest, float* scale, bool write) {
  const bool finite = largest < 0x7f800000u;
  const float a = fmaxf(__uint_as_float(largest), 0x1p-100f);
  if (write) *scale = finite ? a / 127.0f : __builtin_nanf("");
  return finite ? 127.0f / a : 0.f;
}

// x * factor rounded to nearest even; 0 for factor 0 (whatever x is).
__device__ __forceinline__ int to_int8(float x, float factor) {
  return factor == 0.f ? 0 : (int)__builtin_rintf(x * factor);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest of the workgroup's (or, ROW_WAVE, of the wavefront's) values.
template <bool ROW_WAVE>
__device__ __forceinline__ uint32_t largest_of(uint32_t v, uint32_t* part) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d, 64));
  if constexpr (!ROW_WAVE) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  return v;
}

// A row for each wavefront (ROW_WAVE) or for each workgroup of 256 threads; rows of 16-byte
// chunks, at most CHUNKS a thread.
template <class In, int CHUNKS, bool ROW_WAVE>
__global__ __launch_bounds__(256) void k_quantize_int8(int64_t rows, int cols, int64_t ldx, const In* x, int8_t* q,
                                                       float* scale) {
  constexpr int kPer = 16 / (int)sizeof(In), kWidth = ROW_WAVE ? 64 : 256;
  typedef In Chunk __attribute__((ext_vector_type(kPer)));
  __shared__ uint32_t part[4];
  const int64_t row = ROW_WAVE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= rows) return;
  const int t = ROW_WAVE ? threadIdx.x & 63 : threadIdx.x;
  const Chunk* const from = reinterpret_cast<const Chunk*>(x + row * ldx);
  const int chunks = cols / kPer;
  Chunk v[CHUNKS];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) v[i] = t + i * kWidth < chunks ? from[t + i * kWidth] : Chunk{};
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
    for (int e = 0; e < kPer; ++e) largest = max(largest, magnitude((float)v[i][e]));
  largest = largest_of<ROW_WAVE>(largest, part);
  const float factor = int8_factor(largest, scale + row, t == 0);
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    if (t + i * kWidth >= chunks) break;
    typedef int8_t Bytes __attribute__((ext_vector_type(kPer)));
    Bytes b;
#pragma unroll
    for (int e = 0; e < kPer; ++e) b[e] = (int8_t)to_int8((float)v[i][e], factor);
    reinterpret_cast<Bytes*>(q + row * cols)[t + i * kWidth] = b;
  }
}

template <class In>
__global__ __launch_bounds__(256) void k_quantize_int8_any(int64_t rows, int cols, int64_t ldx, const In* x, int8_t* q,
                                                           float* scale) {
  __shared__ uint32_t part[4];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const In* const row = x + r * ldx;
    uint32_t largest = 0;
    for (int c = threadIdx.x; c < cols; c += 256) largest = max(largest, magnitude((float)row[c]));
    largest = largest_of<false>(largest, part);
    const float factor = int8_factor(largest, scale + r, threadIdx.x == 0);
    for (int c = threadIdx.x; c < cols; c += 256) q[r * cols + c] = (int8_t)to_int8((float)row[c], factor);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------

constexpr int64_t kMaxRows = 1 << 30, kMaxStrideBytes = 4 << 20, kMaxBlocks = 1 << 20, kMaxRowBlocks = 1 << 23;  // (a grid holds fewer than 2^32 threads)

int launched() { return hipGetLastError() == hipSuccess ? MEGAMOE_OK : MEGAMOE_ERR_HIP; }

int check(const megamoe_product* p, int elem, bool wide_out) {
  if (!p) return MEGAMOE_ERR_INVALID_ARGUMENT;
  if (p->rows < 0 || p->groups < 1 || p->n < 0 || p->k < 0 || p->ldx < p->k || p->ldy < p->n) return MEGAMOE_ERR_SHAPE;
  if (p->dtype < MEGAMOE_BF16 || p->dtype > (wide_out ? MEGAMOE_FP32 : MEGAMOE_FP16)) return MEGAMOE_ERR_SHAPE;
  if (p->groups > kMaxGroups || p->rows > kMaxRows) return MEGAMOE_ERR_UNSUPPORTED;
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

template <class Ty, class Out, int MI, int MJ>
int launch_strips(Args a, hipStream_t stream) {
  a.tiles_j = (int)row_tiles(a.rows, a.groups, 16 * MJ, a.counts != nullptr);
  a.tiles_i = (int)ceil_div(a.n, 16 * MI);
  const int64_t total = (int64_t)a.tiles_j * a.tiles_i;
  hipLaunchKernelGGL((k_strips<Ty, Out, MI, MJ>), dim3((unsigned)(total < kMaxBlocks ? total : kMaxBlocks)),
                     dim3(kThreads), 0, stream, a);
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

template <class Ty, class Out, Form FORM, int TI, int TJ, bool ONCE>
int launch_tiles(Args a, hipStream_t stream) {
  const int most = compute_units() * kPerCu<FORM, TI>;
  if (most <= 0) return MEGAMOE_ERR_HIP;
  const int64_t rows = FORM == kTN ? a.groups * ceil_div(a.n, TJ) : row_tiles(a.rows, a.groups, TJ, a.counts != nullptr);
  const int64_t total = rows * ceil_div(FORM == kTN ? a.k : a.n, TI);
  if (total > INT32_MAX) return MEGAMOE_ERR_UNSUPPORTED;
  const int64_t grid = ceil_div(total < most ? total : most, 8) * 8;
  hipLaunchKernelGGL((k_tiles<Ty, Out, FORM, TI, TJ, ONCE>), dim3((unsigned)grid), dim3(64 * kWaves<TI, TJ>), 0, stream, a);
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

// What is known of a call before it runs: the groups that have rows, and rows of one of those.
// Groups' counts are on the device, so as many as uniform routing would hit.
struct Load {
  double groups, rows;
};

Load expected(const Args& a) {
  if (!a.counts) return Load{1.0, (double)a.rows};
  const double mean = (double)a.rows / a.groups, hit = a.groups * (1.0 - exp(-mean));
  return Load{hit, a.rows / hit};
}

// Row tiles of `height` to expect where groups' rows are spread like a geometric distribution: one
// of a small group, half a tile more than full ones of a large one.
double expected_tiles(const Args& a, const Load& l, int height) {
  if (!a.counts) return (double)ceil_div(a.rows, height);
  return l.groups / (1.0 - exp(-height / l.rows));
}

double clamp01(double v) { return v < 0 ? 0 : v > 1 ? 1 : v; }

// The tiled kernel for a product. Each size's time is its rounds of the GPU (not a whole number of
// them costs about a third of one, just more than the first 0.6) times a tile's: its stages, and what
// its start and end cost in stages. A stage of 256x128 takes 0.63 of one of 256x256 where the MFMAs
// decide (8192 cubed in bf16: 189 us a round against 120) and 0.78 where the weights stream from memory
// (rows of a group up to 128); one of 128x128 0.585 and 0.5 of 256x128's (7168 by 2048, 2 rows a group:
// 131 us a round against 66). Over 100 calls of 8 to 128 experts, 8 to 1024 uneven rows each, the size
// that this takes is 0.6% slower than the fastest of the three in the geometric mean, 12% at most.
//
// ONCE loads the weights past the caches: they are not read again where a group's rows make up to
// two tiles (225 of 256 experts hit, 7168 by 2048 in bf16: 1078 us without, 955 with it; 1024 rows a
// group and more lose up to 7% by it).
template <class Ty, class Out, Form FORM>
int launch_rows(const Args& a, hipStream_t s) {
  const int cus = compute_units();
  if (cus <= 0) return MEGAMOE_ERR_HIP;
  const Load l = expected(a);
  const double kbytes = (double)a.k * Ty::kBytes, stages = ceil(kbytes / kStage);
  auto rounds = [&](int ti, int tj) {
    const double r = expected_tiles(a, l, tj) * ceil_div(a.n, ti) / cus;
    return r <= 1 ? 1 : fmax(r + 0.3, 1.6);
  };
  const double unit_128 = 0.78 - 0.15 * clamp01((l.rows - 128) / 256);
  const double unit_64 = unit_128 * (0.5 + 0.085 * clamp01(l.rows / 128));
  const double large = rounds(256, 256) * (stages + 3), middle = rounds(256, 128) * unit_128 * (stages + 4.2);
  const double small = rounds(128, 128) * unit_64 * (stages + 5.4);
  if constexpr (FORM == kNT) {
    // Strips, where not even the small tiles occupy the GPU. Nanoseconds: a strip moves 30 bytes a ns
    // into its CU, all of them 9200, weights from memory 6000; a small tile takes 300 to 430 a stage.
    if (expected_tiles(a, l, 128) * ceil_div(a.n, 128) <= cus) {
      auto strips = [&](int t) {
        const double per = (t + (l.rows < t ? l.rows : t)) * kbytes;
        const double all = expected_tiles(a, l, t) * ceil_div(a.n, t) * per, weights = l.groups * a.n * kbytes;
        return 3500 + fmax(fmax(all / 9200, per / 30), weights / 6000);
      };
      const double one = strips(16), two = strips(32), tile = 9000 + stages * (300 + fmin(l.rows, 128));
      if (fmin(one, two) < tile)
        return one <= two ? launch_strips<Ty, Out, 1, 1>(a, s) : launch_strips<Ty, Out, 2, 2>(a, s);
    }
  }
  if (large <= middle && large <= small)
    return l.rows <= 512 ? launch_tiles<Ty, Out, FORM, 256, 256, true>(a, s)
                         : launch_tiles<Ty, Out, FORM, 256, 256, false>(a, s);
  if (middle <= small)
    return l.rows <= 256 ? launch_tiles<Ty, Out, FORM, 256, 128, true>(a, s)
                         : launch_tiles<Ty, Out, FORM, 256, 128, false>(a, s);
  return l.rows <= 256 ? launch_tiles<Ty, Out, FORM, 128, 128, true>(a, s)
                       : launch_tiles<Ty, Out, FORM, 128, 128, false>(a, s);
}

template <class In, int CHUNKS, bool ROW_WAVE>
int launch_quantize_rows(int64_t rows, int cols, int64_t ldx, const In* x, int8_t* q, float* scale, hipStream_t s) {
  const dim3 grid((unsigned)(ROW_WAVE ? ceil_div(rows, 4) : rows));
  hipLaunchKernelGGL((k_quantize_int8<In, CHUNKS, ROW_WAVE>), grid, dim3(256), 0, s, rows, cols, ldx, x, q, scale);
  return launched();
}

// Short rows go to a wavefront each (no barrier), longer ones to a workgroup each; CHUNKS is what
// holds the row.
template <class In>
int launch_quantize(int64_t rows, int cols, int64_t ldx, const In* x, int8_t* q, float* scale, hipStream_t s) {
  constexpr int kPer = 16 / (int)sizeof(In);
  const int64_t count = cols / kPer, blocks = rows < kMaxBlocks ? rows : kMaxBlocks;
  if (cols > 0 && chunks(x, ldx, cols, (int)sizeof(In)) && aligned(q, kPer) && count <= 8 * 256 && rows <= kMaxRowBlocks) {
    if (count <= 64) return launch_quantize_rows<In, 1, true>(rows, cols, ldx, x, q, scale, s);
    if (count <= 2 * 64) return launch_quantize_rows<In, 2, true>(rows, cols, ldx, x, q, scale, s);
    if (count <= 256) return launch_quantize_rows<In, 1, false>(rows, cols, ldx, x, q, scale, s);
    if (count <= 2 * 256) return launch_quantize_rows<In, 2, false>(rows, cols, ldx, x, q, scale, s);
    if (count <= 4 * 256) return launch_quantize_rows<In, 4, false>(rows, cols, ldx, x, q, scale, s);
    return launch_quantize_rows<In, 8, false>(rows, cols, ldx, x, q, scale, s);
  }
  hipLaunchKernelGGL((k_quantize_int8_any<In>), dim3((unsigned)blocks), dim3(256), 0, s, rows, cols, ldx, x, q, scale);
  return launched();
}

template <class Ty>
int product16(const megamoe_product* p, const Args& a, hipStream_t s) {
  using Out = typename Ty::Elem;
  if (p->k > 0 && chunks(a.x, a.ldx, a.k, 2) && chunks(a.w, 0, p->transposed ? a.n : a.k, 2))
    return p->transposed ? launch_rows<Ty, Out, kNN>(a, s) : launch_rows<Ty, Out, kNT>(a, s);
  return p->transposed ? launch_any<Ty, Out, true>(a, s) : launch_any<Ty, Out, false>(a, s);
}

// The large tiles wherever they occupy the GPU: four small ones write as much and read twice as much
// (128 experts, 2048 by 768, 32768 uneven rows: 213 us against 258). Fewer leave CUs idle (8 experts,
// 1024 by 512, 144 rows, 64 large tiles: 14.8 us against 9.3 with small ones; 2048 by 2048, 4096 rows, also
// 64: 110 against 66).
template <class Ty>
int wgrad16(const Args& a, hipStream_t s) {
  if (!chunks(a.x, a.ldx, a.k, 2) || !chunks(a.w, a.ldy, a.n, 2)) return launch_wgrad_any<Ty>(a, s);
  if (a.groups * ceil_div(a.n, 256) * ceil_div(a.k, 256) >= compute_units())
    return launch_tiles<Ty, typename Ty::Elem, kTN, 256, 256, false>(a, s);
  return launch_tiles<Ty, typename Ty::Elem, kTN, 128, 128, false>(a, s);
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
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MEGAMOE_BF16) return launch_quantize(rows, cols, ldx, (const __bf16*)x, q, scale, s);
  if (dtype == MEGAMOE_FP16) return launch_quantize(rows, cols, ldx, (const _Float16*)x, q, scale, s);
  return launch_quantize(rows, cols, ldx, (const float*)x, q, scale, s);
}

}  // extern "C"
