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

template <class Ty>
int product16(const megamoe_product* p, const Args& a, hipStream_t s) {
  return p->transposed ? launch_any<Ty, typename Ty::Elem, true>(a, s) : launch_any<Ty, typename Ty::Elem, false>(a, s);
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
  return p->dtype == MEGAMOE_BF16 ? launch_wgrad_any<Bf16>(a, (hipStream_t)stream)
                                  : launch_wgrad_any<Fp16>(a, (hipStream_t)stream);
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
  if (p->dtype == MEGAMOE_BF16) return launch_any<Int8, __bf16, false>(a, s);
  if (p->dtype == MEGAMOE_FP16) return launch_any<Int8, _Float16, false>(a, s);
  return launch_any<Int8, float, false>(a, s);
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
