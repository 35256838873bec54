// gqe_xent.h — softmax cross entropy of queries against every row of a table, logits never kept (include/gqe_ops.h).
//
// With x_v the table rows and y_b the queries (z_bv = scale q_b . t_v in base 2: s_bv = z_bv log2 e) everything that is needed is
//   lse_b = log2 sum_v 2^s_bv           dq_b = g_b scale (sum_v p_bv t_v - t_target)           dt_v = scale sum_b g_b (p_bv - [v = target_b]) q_b
// and both gradients have ONE form: for a stationary row y and streamed rows x,   out_y = sum_x 2^(s_xy + lambda_x) sign_x x,
//   dq: y = query,     x = table row,   lambda = 0 (the sum of the 2^s beside it gives lse)
//   dt: y = table row, x = query,       lambda_b = log2 |g_b| - lse_b,  sign_b = sign of g_b
// so one kernel does both: a wave keeps 32 stationary rows as matrix-core operands in registers, tiles of 32 streamed rows go
// through LDS, S^T = X Y^T puts a stationary row in a LANE (lane & 31; the streamed rows are the accumulator's registers), so the
// running maximum of s + lambda and the sum are per-lane scalars, and the exponentials are, register for register, the second
// operand of out^T += X^T P (v_mfma 32x32x16: k = 8 (lane >> 5) + j; the k order of X^T is chosen to match and read transposed out
// of the same LDS tile by ds_read_b64_tr_b16).  Nothing is shuffled between the two products.
//
// float32 operands: each row is scaled by a power of two (its largest element to [2^14, 2^15)) and split into two fp16 values,
// x = hi + lo to 22 bits of the row's largest element; a product is hi hi + hi lo + lo hi on the fp16 matrix cores with float32
// accumulation (the dropped lo lo is below 2^-22), three times the work of one fp16 product where the float32 matrix
// instructions take sixteen times.  Scales are exact: they re-enter through the factors cs / cy of s and through lambda.  The
// exponentials are relative to their running maximum, times 2^11 to 2^15, so that the split keeps 22 bits of those that matter.
// bfloat16 operands: one plane, as they are; the exponentials are rounded to bfloat16 (relative error 2^-9, as the output's own).
//
// The target's own term is never part of the sums: dq needs p_target - 1, which cancels when the query is answered well, so the
// sum over the OTHER rows (share r = 1 - p_target) is kept and dq = g scale (sum_others p t - r t_target), and in dt the entry of
// a target is - g_b r_b.  loss = log(1 + 2^(lse_others - s_target)) likewise loses nothing.
//
// What it reaches, 8 B V d operations counted (the products of the first pass are computed again in the second: keeping them would write
// and read B V numbers, 512 x 500000: 2 GB, which takes as long): float32, 512 x 500000 x 256: 174 us to prepare the operands (5.9 TB/s),
// 700 us and 1000 us for the passes = 930 TFLOP/s of fp16 products, where a library product of 8192^3 reaches 1110; the matrix units
// are busy 52 % (first pass) and 35 % (second: 16 tiles to a workgroup, so a third of its time is reading 128 rows and writing 128 gradients).
// bfloat16, 4608 x 131071 x 256: 830 + 940 us = 700 TFLOP/s; one wave per SIMD holds 330 registers, so vector work (7 instructions and an
// exponential a number), the tile's loads (18 %) and the first product's chain (21 %) add up instead of hiding behind other waves;
// d <= 192, two waves per SIMD, gains 40 %.  64 stationary rows a wave (half the LDS traffic) were no faster at d = 128 and do not fit at
// 256.  Few queries (6 x 427109 x 206: 153 + 199 us): memory, at 2.3 TB/s in the first pass, where three waves of four only convert, and 3.5
// in the second, where a workgroup is 1 us of starting, 3 of reading, 4 of products for one tile, 3 of the length's gradient and 3 of writing.
#ifndef GQE_XENT_H
#define GQE_XENT_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gqe_common.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

#define XENT_BM 128            // stationary rows of a workgroup: 32 for each of its four waves
#define XENT_TR 32             // streamed rows of an LDS tile
// closes a step of n matrix instructions: LDS reads first, then matrix instructions with vector work between them (4 to 7 instructions
// after each: within 1 %)
#define XENT_V 5
#define XENT_GROUP(mask, n) __builtin_amdgcn_sched_group_barrier(mask, n, 0)
#define XENT_MIX(n)                                      \
  do {                                                   \
    XENT_GROUP(0x100, 4);                                \
    XENT_GROUP(0x008, 1);                                \
    XENT_GROUP(0x002, XENT_V);                           \
    if ((n) > 1) {                                       \
      XENT_GROUP(0x008, 1);                              \
      XENT_GROUP(0x002, XENT_V);                         \
    }                                                    \
    if ((n) > 2) {                                       \
      XENT_GROUP(0x008, 1);                              \
      XENT_GROUP(0x002, XENT_V);                         \
    }                                                    \
    __builtin_amdgcn_sched_barrier(0);                   \
  } while (0)
// two waves in a SIMD's 512 registers, where the operands and sums of 32 stationary rows leave room
#define XENT_TWO (DK <= 128 || (BF16 && DMA && DK <= 192))
#define XENT_NONE (-1.0e30f)   // running maximum before the first term (finite: its difference from -inf is -inf)

enum { XENT_MODE_LSE = 0, XENT_MODE_DQ = 1, XENT_MODE_DT = 2 };

struct XentPass {
  const void* y;               // stationary rows: queries (LSE, DQ), table rows (DT)
  const void* x;               // streamed rows:   table rows (LSE, DQ), queries (DT)
  int64_t y_stride, x_stride;
  int32_t ny, nx, d;
  const char *y_image, *x_image;      // DMA: prepared tiles, or bfloat16 rows (then the strides are not 0)
  const float2* y_fac;         // DMA: factors of the stationary rows
  const struct XentRec* x_rec; // DMA: the streamed rows' part
  int32_t unit;                // DMA, DT: table rows count divided by their length
  float scale2;                // scale * log2(e): multiplies s
  float scale;                 // DT: multiplies the result
  int32_t n_tiles, tiles_per_split, n_split, n_yblk;
  const int32_t* target;       // [queries]
  const float* weight;         // DT: [queries] or NULL
  const float* stat;           // DT: [queries][2]
  float* part_m;               // [n_split][ny] running maximum (its unit of the sums)
  float* part_l;               // [n_split][ny] LSE / DQ: sum over the other rows in units of 2^part_m
  float* part_o;               // [n_split][ny][pitch] (DQ; DT when split)
  float* st;                   // [queries] LSE / DQ: s of the target
  void* out;                   // DT, n_split == 1: dtable
  int64_t out_stride;
  int32_t pitch, accumulate;   // pitch: d up to whole 16 bytes
};

__device__ __forceinline__ float xent_pow2(int k) { return __int_as_float((k + 127) << 23); }   // -126 <= k <= 127
// the power of two that takes a row whose largest magnitude is m to [2^14, 2^15)
__device__ __forceinline__ int xent_row_scale(float m) {
  const int e = ((__float_as_int(m) >> 23) & 255) - 127;
  int k = 14 - e;
  k = k > 126 ? 126 : k;
  return m > 0.f ? k : 0;
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t xent_pack_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2)); }
__device__ __forceinline__ uint32_t xent_pack_f16(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2)); }
// x = hi + lo in fp16, two values at a time.  hi has to be ONE number for both uses: left alone, the compiler fuses the product that
// made x into the conversion on one side only (a single rounding there, two here), and once in some thousand values lo is then the
// remainder of another hi.  The empty asm makes the values opaque; the remainders are mixed-precision multiply-adds, x - 1 * hi.
__device__ __forceinline__ void xent_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  asm("" : "+v"(a), "+v"(b));
  hi = xent_pack_f16(a, b);
  float ra, rb;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
  lo = xent_pack_f16(ra, rb);
}
// 1 / sqrt(ss) to an ulp; a row of zeros has length "infinity", a row that is not finite stays so
__device__ __forceinline__ float xent_rsqrt(float ss) {
  const float y = __builtin_amdgcn_rsqf(ss);
  const float z = y * fmaf(-0.5f * ss * y, y, 1.5f);
  return ss > 0.f ? z : (ss == 0.f ? 0.f : ss);
}

union XentFrag {
  uint32_t u[4];
  f16x8 h;
  bf16x8 b;
  s16x8 s;
  s16x4 q[2];
};

template <bool BF16>
__device__ __forceinline__ f32x16 xent_mfma(const XentFrag& a, const XentFrag& b, f32x16 c) {
  if (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.b, b.b, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
}

// Rows of a matrix in global memory, and 16 bytes of them at an element's alignment.
struct XentRows {
  const void* p;
  int64_t stride;
  int32_t n, d;
  __device__ __forceinline__ const char* row(int i, int size) const { return (const char*)p + (i < n ? i : n - 1) * stride * size; }
};
struct __attribute__((packed, aligned(2))) XentU4 {
  uint32_t v[4];
};
struct __attribute__((packed, aligned(4))) XentF4 {
  float v[4];
};
struct __attribute__((packed, aligned(2))) XentU2 {
  uint32_t v[2];
};

// Tile of operands, in LDS and (where it is prepared once) in memory alike: each plane is sub-tiles of 32 rows x 128 columns (8 KB) and,
// where DK is 64 or 192, a last one of 32 rows x 64 (4 KB).  A row's 16-byte pieces are permuted so that 16 rows at one piece (the
// first product's operand) and 4 rows at 4 neighbouring pieces (the transposed reads of the second) both touch all 64 banks once:
//   full sub-tile: row r, piece c at 256 r + 16 (c ^ f(r)),  f(r) = 4 (r & 3) + (r >> 2 & 3)
//   half sub-tile: two rows share 256 bytes:  256 (r >> 1) + 16 (8 (r & 1) + (c ^ g(r >> 1))),  g(s) = 4 (s & 1) + (s >> 1 & 3)
// Neighbouring column groups are an exclusive or away (bits 5 .. 7), further sub-tiles and rows + 16 a constant, rows + 8 a constant
// and an exclusive or with 32.
__device__ __forceinline__ int xent_full(int row, int piece) { return 256 * row + 16 * (piece ^ ((row & 3) << 2 | (row >> 2 & 3))); }
__device__ __forceinline__ int xent_half(int row, int piece) {
  const int s = row >> 1;
  return 256 * s + 16 * (8 * (row & 1) + (piece ^ ((s & 1) << 2 | (s >> 1 & 3))));
}
template <int DK>
struct XentTile {
  static constexpr int FULL = DK / 128;                    // full sub-tiles
  static constexpr bool HALF = DK % 128 != 0;
  static constexpr int PLANE = XENT_TR * DK * 2;
  int full, half;                                          // a thread's place in a full / half sub-tile
  // chunk: which 64 columns; x: the exclusive or that selects 16 / 32 columns inside them or, in a full sub-tile, the other 64
  __device__ __forceinline__ int at(int chunk, int x) const {
    return (chunk >> 1) * 8192 + (chunk >> 1 < FULL ? full ^ (x | (chunk & 1) << 7) : half ^ x);
  }
  // the same place of another tile.  (The exclusive ors come after the addition, so that they are not kept in registers for all of
  // the loop; the addition is of whole kilobytes and leaves their bits alone.)
  __device__ __forceinline__ XentTile plus(int off) const { return XentTile{full + off, half + off}; }
};

// What a streamed row adds to its exponents, per tile of 32 rows: [0] factor of s, [1] lambda, [2] LSE / DQ: 2^-lambda; DT: exponent of a
// target's entry, [3] DT: the target's row (low 31 bits; 0x7fffffff: none) and the sign of the weight (bit 31).
struct XentRec {
  float v[4][XENT_TR];
};
struct XentRecs {              // DT: from the queries' factors, statistics and weights
  XentRec* rec;
  const float2* fac;
  const int32_t* target;
  const float* weight;
  const float* stat;
  float scale2;
  int32_t n, n_rows, bf16;
};
__device__ __forceinline__ void xent_rec_dt(XentRec& r, int i, bool ok, float c, float lam, int tg, float g, float lse2, float lr, int n_rows, float scale2) {
  const bool counts = ok && tg >= 0 && tg < n_rows;
  const float lg = counts ? __builtin_amdgcn_logf(fabsf(g)) : -INFINITY;      // log2; 0 and what is below float32's normal range: no share
  r.v[0][i] = c * scale2;
  r.v[1][i] = ok ? lam + (lg - lse2) : -INFINITY;
  r.v[2][i] = lam + (lg + lr);
  r.v[3][i] = __uint_as_float((counts ? (uint32_t)tg : 0x7fffffffu) | (__float_as_uint(g) & 0x80000000u));
}
__device__ __forceinline__ float xent_exponent(float c) { return (float)((__float_as_int(c) >> 23) - 127); }      // log2 of a power of two

template <bool BF16, int DK, int MODE, bool DMA>
struct XentLds {
  static constexpr int PLANES = BF16 ? 1 : 2;
  static constexpr int PLANE = XentTile<DK>::PLANE;
  static constexpr int TILE = PLANES * PLANE;
  static constexpr int DIST = 2;                                      // tile t + DIST is asked for while tile t is summed (3: no faster)
  static constexpr int TILES = (MODE == XENT_MODE_LSE ? 0 : 1) + DIST;
  static constexpr int RECS = DIST + 1;
  static constexpr int OUT_ROW = 68;                                  // floats of a row of the outputs' turn (64 columns at a time)
  static constexpr int OUT = MODE == XENT_MODE_LSE ? (DMA ? 0 : 4 * PLANES * 4096) : 4 * 32 * OUT_ROW * 4;      // (LSE: the stationary rows' way in)
  char tile[TILES * TILE > OUT ? TILES * TILE : OUT];
  XentRec rec[RECS];
  float rn[XENT_BM];         // DT: 1 / length of the stationary rows, for the end
};

// Eight elements of a row, as they are: 16 bytes at a time wherever rows begin (the memory takes any alignment).  Rows behind the last one
// are the last one (their exponents are -inf, their results are not written).  CUT: d may cut the piece; its 16 bytes are then the row's
// last ones, and xent_cut8 brings them, once they are there, to their places, with zeros behind column d: no branches, for those would
// keep vector work out of the shadow of matrix instructions (element by element d = 211 cost a third of the whole pass, and code).
template <bool BF16, bool CUT>
__device__ __forceinline__ void xent_load8(const char* row, int d, int col, uint32_t* raw) {
  constexpr int SIZE = BF16 ? 2 : 4, N = BF16 ? 8 : 4;
  if (CUT && d < N) {                            // (the same for all: a row of less than 16 bytes)
#pragma unroll
    for (int i = 0; i < (BF16 ? 4 : 8); ++i) raw[i] = 0;
    if (col) return;
    if (BF16) {
      const uint16_t* q = (const uint16_t*)row;
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < d) raw[i >> 1] |= (uint32_t)q[i] << (16 * (i & 1));
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < d) raw[i] = ((const uint32_t*)row)[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i += N) {
    const int at = CUT ? min(col + i, d - N) : col + i;
    const XentU4 u = *(const XentU4*)(row + SIZE * at);
#pragma unroll
    for (int k = 0; k < 4; ++k) raw[i + k] = u.v[k];
  }
}
template <bool BF16>
__device__ __forceinline__ void xent_cut8(int d, int col, uint32_t* raw) {
  constexpr int N = BF16 ? 8 : 4;
  if (d < N) return;
  if (BF16) {
    const int left = d - col, shift = 16 * (8 - left);
    const uint64_t lo = raw[0] | (uint64_t)raw[1] << 32, hi = raw[2] | (uint64_t)raw[3] << 32;
    const uint64_t a = shift < 64 ? lo >> (shift & 63) | hi << (64 - shift & 63) : hi >> (shift & 63), b = shift < 64 ? hi >> (shift & 63) : 0;
    const bool whole = left >= 8, none = left <= 0;
    raw[0] = whole ? raw[0] : none ? 0 : (uint32_t)a;
    raw[1] = whole ? raw[1] : none ? 0 : (uint32_t)(a >> 32);
    raw[2] = whole ? raw[2] : none ? 0 : (uint32_t)b;
    raw[3] = whole ? raw[3] : none ? 0 : (uint32_t)(b >> 32);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const int left = d - col - i;
      const float a = __uint_as_float(raw[i]), b = __uint_as_float(raw[i + 1]), e = __uint_as_float(raw[i + 2]), f = __uint_as_float(raw[i + 3]);
      const auto pick = [](bool yes, float x, float y) { return yes ? x : y; };
      raw[i] = __float_as_uint(pick(left >= 4, a, pick(left == 3, b, pick(left == 2, e, pick(left == 1, f, 0.f)))));
      raw[i + 1] = __float_as_uint(pick(left >= 4, b, pick(left == 3, e, pick(left == 2, f, 0.f))));
      raw[i + 2] = __float_as_uint(pick(left >= 4, e, pick(left == 3, f, 0.f)));
      raw[i + 3] = __float_as_uint(pick(left >= 4, f, 0.f));
    }
  }
}

// One thread's share of 32 rows between their global loads and their LDS stores: 8 threads per row, DK / 8 elements each.
template <bool BF16, int DK, bool UNIT>
struct XentStage {
  static constexpr int PLANE = XentTile<DK>::PLANE;
  static constexpr int NCH = DK / 64;          // pieces of 8 elements: piece c of thread t holds columns 64 c + 8 t ..
  uint32_t raw[NCH][BF16 ? 4 : 8];

  __device__ __forceinline__ void load(const XentRows& r, int row, int t8) {      // (d is more than DK - 64)
    const char* from = r.row(row, BF16 ? 2 : 4);
#pragma unroll
    for (int c = 0; c < NCH - 1; ++c) xent_load8<BF16, false>(from, r.d, 64 * c + 8 * t8, raw[c]);
    xent_load8<BF16, true>(from, r.d, 64 * (NCH - 1) + 8 * t8, raw[NCH - 1]);
  }

  // Operands into the tile (w: this thread's place), in STEPS pieces of work that a caller may put between matrix instructions:
  // largest element, length, then the split and its stores.  Afterwards: operand times cs is the row (the unit row if UNIT); k its
  // power of two, where that is all there is (float32); rn: 1 / length.
  static constexpr int STEPS = DK / 16, HEAD = NCH + 2, PER = (STEPS + STEPS - HEAD - 1) / (STEPS - HEAD);
  float cs, rn, f, sum;
  int k;
  uint32_t hi[4], lo[4];

  __device__ __forceinline__ void largest(int d, int t8) {
    xent_cut8<BF16>(d, 64 * (NCH - 1) + 8 * t8, raw[NCH - 1]);
    k = 0;
    cs = rn = 1.f;
    sum = 0.f;
    if (BF16 && !UNIT) return;
    float mx = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int i = 0; i < (BF16 ? 4 : 8); ++i) {
        if (BF16) mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(raw[c][i])), fabsf(bf16_hi(raw[c][i]))));
        else mx = fmaxf(mx, fabsf(__uint_as_float(raw[c][i])));
      }
    mx = fmaxf(mx, dpp_get<0xB1, 0xF>(mx));        // the row's 8 threads: swaps in fours, then halves mirrored
    mx = fmaxf(mx, dpp_get<0x4E, 0xF>(mx));
    mx = fmaxf(mx, dpp_get<0x141, 0xF>(mx));
    k = xent_row_scale(mx);
    f = xent_pow2(k);
  }
  __device__ __forceinline__ void squares(int c) {
#pragma unroll
    for (int i = 0; i < (BF16 ? 4 : 8); ++i) {
      if (BF16) {
        const float a = bf16_lo(raw[c][i]) * f, b = bf16_hi(raw[c][i]) * f;
        sum = fmaf(a, a, sum);
        sum = fmaf(b, b, sum);
      } else {
        const float a = __uint_as_float(raw[c][i]) * f;
        raw[c][i] = __float_as_uint(a);
        sum = fmaf(a, a, sum);
      }
    }
  }
  __device__ __forceinline__ void length() {
    sum += dpp_get<0xB1, 0xF>(sum);
    sum += dpp_get<0x4E, 0xF>(sum);
    sum += dpp_get<0x141, 0xF>(sum);
    const float g = xent_rsqrt(sum);
    rn = g * f;
    cs = rn;
    k = 14;
    f = g * 16384.f;
  }
  // all of that at once, and then piece c
  __device__ __forceinline__ void scale(int d, int t8) {
    largest(d, t8);
    if (UNIT) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) squares(c);
      length();
    }
    if (!BF16) cs = xent_pow2(-k);
  }
  __device__ __forceinline__ void piece(int c, uint4& a, uint4& b) const {
    if (BF16) {
      a = make_uint4(raw[c][0], raw[c][1], raw[c][2], raw[c][3]);
      return;
    }
    uint32_t x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xent_split(__uint_as_float(raw[c][2 * i]) * f, __uint_as_float(raw[c][2 * i + 1]) * f, x[i], y[i]);
    a = make_uint4(x[0], x[1], x[2], x[3]);
    b = make_uint4(y[0], y[1], y[2], y[3]);
  }

  __device__ __forceinline__ void step(int j, char* tile, const XentTile<DK>& w, int d, int t8) {
    if (j == 0) {
      largest(d, t8);
      if (BF16) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) *(uint4*)(tile + w.at(c, 0)) = make_uint4(raw[c][0], raw[c][1], raw[c][2], raw[c][3]);
      }
    } else if (UNIT && j <= NCH) {
      squares(j - 1);
    } else if (UNIT && j == NCH + 1) {
      length();
    } else if (!BF16 && j >= HEAD) {
#pragma unroll
      for (int q = (j - HEAD) * PER; q < (j - HEAD + 1) * PER && q < STEPS; ++q) {
        const int c = q >> 2, i = q & 3;
        xent_split(__uint_as_float(raw[c][2 * i]) * f, __uint_as_float(raw[c][2 * i + 1]) * f, hi[i], lo[i]);
        if (i == 3) {
          char* to = tile + w.at(c, 0);
          *(uint4*)to = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *(uint4*)(to + PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
    }
    if (!BF16 && j == STEPS - 1) cs = xent_pow2(-k);
  }
  __device__ __forceinline__ void store(char* tile, const XentTile<DK>& w, int d, int t8) {
#pragma unroll
    for (int j = 0; j < STEPS; ++j) step(j, tile, w, d, t8);
  }
};

// Operands prepared once: tiles of both matrices in the layout of LDS, and each row's factors {operand -> row, 1 / length}.  IMAGE =
// false: only the factors (bfloat16 rows are operands as they are).  One workgroup per 32 rows: memory's rate.
struct XentPrep {
  XentRows r[2];               // queries, table
  char* image[2];
  float2* fac[2];
  int32_t tiles[2];
  XentRec* rec;                // of the table as streamed rows
};
template <bool BF16, int DK, bool UNIT>
__device__ __forceinline__ void xent_prep(const XentPrep& p, int which, int tile, char* turn) {
  constexpr int TILE = (BF16 ? 1 : 2) * XentTile<DK>::PLANE;
  const int row = threadIdx.x >> 3, t8 = threadIdx.x & 7;
  XentStage<BF16, DK, UNIT> st;
  st.load(p.r[which], tile * XENT_TR + row, t8);
  st.store(turn, XentTile<DK>{xent_full(row, t8), xent_half(row, t8)}, p.r[which].d, t8);
  if (t8 == 0) {
    const bool ok = tile * XENT_TR + row < p.r[which].n;
    if (ok) p.fac[which][tile * XENT_TR + row] = make_float2(st.cs, st.rn);
    if (which == 1 && p.rec) {
      // float32: the operand's power of two; bfloat16 unit rows: 1 / length
      const float lam = !BF16 ? xent_exponent(st.cs) : UNIT && st.cs > 0.f ? __builtin_amdgcn_logf(st.cs) : 0.f;
      XentRec& r = p.rec[tile];
      r.v[0][row] = st.cs;
      r.v[1][row] = ok ? lam : -INFINITY;
      r.v[2][row] = BF16 ? __builtin_amdgcn_exp2f(-lam) : xent_pow2((int)-lam);
      r.v[3][row] = 0.f;
    }
  }
  if (!p.image[which]) return;
  __syncthreads();             // through LDS: the image is written in order
  uint4* out = (uint4*)(p.image[which] + (int64_t)tile * TILE);
#pragma unroll
  for (int i = 0; i < TILE / 4096; ++i) out[i * 256 + threadIdx.x] = ((const uint4*)turn)[i * 256 + threadIdx.x];
}
template <bool BF16, int DK, bool UNIT>
__global__ __launch_bounds__(256) void gqe_xent_prep_kernel(XentPrep p) {
  __shared__ __align__(16) char turn[(BF16 ? 1 : 2) * XentTile<DK>::PLANE];
  const int b = blockIdx.x;
  if (b < p.tiles[0]) xent_prep<BF16, DK, false>(p, 0, b, turn);
  else xent_prep<BF16, DK, UNIT>(p, 1, b - p.tiles[0], turn);
}

// 64 pieces of 16 (4) bytes from base + off(lane) into LDS at `to`, in order of lanes.  Written out: through the builtin the compiler has
// every LDS read wait for every such load that is under way, wherever it goes.  Nobody but the caller waits for these (vmcnt, in order).
__device__ __forceinline__ void xent_dma16(const char* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void xent_dma4(const char* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ uint32_t xent_lds_addr(const void* p) {      // wave-uniform
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}

template <int>
__global__ __launch_bounds__(256) void gqe_xent_recs_kernel(XentRecs p) {
  const int x = blockIdx.x * 256 + threadIdx.x;
  if (x >= (p.n + XENT_TR - 1) / XENT_TR * XENT_TR) return;
  const bool ok = x < p.n;
  const float c = ok ? p.fac[x].x : 1.f;
  xent_rec_dt(p.rec[x / XENT_TR], x % XENT_TR, ok, c, p.bf16 ? 0.f : xent_exponent(c), ok ? p.target[x] : -1, !ok ? 0.f : p.weight ? p.weight[x] : 1.f,
              ok ? p.stat[2 * (int64_t)x] : 0.f, ok ? p.stat[2 * (int64_t)x + 1] : 0.f, p.n_rows, p.scale2);
}

// Tiles by direct loads into LDS: a wave takes every fourth KB.  Out of an image in order; out of bfloat16 rows (16-byte aligned, d =
// DK) each lane picks the row and piece that belong at its place, rows behind the last one again (their exponents are -inf).
template <bool BF16, int DK>
struct XentDma {
  static constexpr int TILE = (BF16 ? 1 : 2) * XentTile<DK>::PLANE, N = TILE / 4096;
  const char* base;
  int64_t step;                // bytes from tile to tile
  int64_t stride;              // bytes of a row, 0: image
  int rows;

  // piece i of N of this wave's share of a tile
  __device__ __forceinline__ void piece(int i, int tile, char* lds, int wave, int lane) const {
    const char* from = base + (int64_t)tile * step;
    const uint32_t to = xent_lds_addr(lds + 1024 * wave) + 4096 * i;
    if (BF16 && stride) {
      const int o = 4096 * i + 1024 * wave + 16 * lane, sub = o >> 13, in = o & 8191;
      int row, piece;
      if (sub < XentTile<DK>::FULL) {
        row = in >> 8;
        piece = 16 * sub + ((in >> 4 & 15) ^ ((row & 3) << 2 | (row >> 2 & 3)));
      } else {
        const int s = in >> 8;
        row = 2 * s + (in >> 7 & 1);
        piece = 16 * sub + ((in >> 4 & 7) ^ ((s & 1) << 2 | (s >> 1 & 3)));
      }
      const int last = rows - 1 - tile * XENT_TR;
      xent_dma16(from, (uint32_t)(row < last ? row : last) * (uint32_t)stride + 16 * piece, to);
    } else {
      xent_dma16(from + 4096 * i, 1024 * wave + 16 * lane, to);
    }
  }
  __device__ __forceinline__ void load(int tile, char* lds, int wave, int lane) const {
#pragma unroll
    for (int i = 0; i < N; ++i) piece(i, tile, lds, wave, lane);
  }
};

// UNIT: table rows count divided by their length (the streamed rows of LSE / DQ, the stationary ones of DT).  DMA: operands were prepared
// (gqe_xent_prep_kernel); else rows are converted here, in the shadow of the second product - right where few queries share a table
// that would otherwise be read, written and read again.
template <bool BF16, int DK, int MODE, bool UNIT, bool DMA>
__global__ __launch_bounds__(256, XENT_TWO ? 2 : 1) void gqe_xent_kernel(XentPass p) {
  typedef XentLds<BF16, DK, MODE, DMA> L;
  typedef XentStage<BF16, DK, UNIT && MODE != XENT_MODE_DT> Stage;
  typedef XentStage<BF16, DK, UNIT && MODE == XENT_MODE_DT> Own;
  typedef XentTile<DK> Tile;
  extern __shared__ __align__(16) char smem[];
  L& lds = *(L*)smem;
  constexpr int PL = BF16 ? 1 : 2, KS = DK / 16, DT = DK / 32;
  constexpr bool OUT = MODE != XENT_MODE_LSE, IS_DT = MODE == XENT_MODE_DT;
  // The running maximum follows only when it has fallen behind by 2^SLACK (new maxima are frequent, large steps are not): exponentials
  // reach 2^(TOP + SLACK), which is fp16's range where they are split in two of it, and far from float32's where they are bfloat16.
  constexpr float TOP = BF16 ? 0.f : 11.f, SLACK = BF16 ? 24.f : 4.f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5;
  const int srow = tid >> 3, t8 = tid & 7;       // staging: 8 threads per row
  const int split = blockIdx.x % p.n_split, yblk = blockIdx.x / p.n_split;
  const int y0 = yblk * XENT_BM + wave * 32, y = y0 + n;
  const bool active = y0 < p.ny, y_ok = y < p.ny;
  const int tile0 = split * p.tiles_per_split;
  const int tile1 = min(tile0 + p.tiles_per_split, p.n_tiles);
  const XentRows xr = {p.x, p.x_stride, p.nx, p.d}, yr = {p.y, p.y_stride, p.ny, p.d};

  // this thread's places in a tile
  const Tile wr = {xent_full(srow, t8), xent_half(srow, t8)};                            // stage stores
  const Tile rs = {xent_full(n, h), xent_half(n, h)};                                    // first product: row n, half h of 16 columns
  const int orow = 4 * h + ((lane & 15) >> 2), opiece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const Tile ro = {xent_full(orow, opiece) + 8 * (lane & 1), xent_half(orow, opiece) + 8 * (lane & 1)};      // second product, 32 columns

  // Streamed rows.  DMA: tile t + 2 is under way while tile t + 1 is multiplied and tile t summed; the vector unit has nothing to do with
  // it.  Otherwise: loads of tile t + 3 are under way while tile t + 2 is converted and stored.
  struct Feed {
    Stage st;
    float g, lse2, lr;        // DT: weight and statistics of this thread's query
    int target;
  } feed;
  const XentDma<BF16, DK> dx = {p.x_image, p.x_stride ? 64 * p.x_stride : (int64_t)L::TILE, 2 * p.x_stride, p.nx};
  constexpr int IN_FLIGHT = XentDma<BF16, DK>::N + 1;      // direct loads of a tile, per wave
  // DMA: piece i of IN_FLIGHT of tile t; the last one is the rows' part: 512 bytes, each half by two waves (all have as many under way)
  const auto load_piece = [&](int i, int t, int tb, int ab) {
    if (i < IN_FLIGHT - 1) dx.piece(i, t, lds.tile + tb * L::TILE, wave, lane);
    else xent_dma4((const char*)(p.x_rec + t), 256 * (wave & 1) + 4 * lane, xent_lds_addr((char*)&lds.rec[ab] + 256 * (wave & 1)));
  };
  const auto load = [&](int t, int tb, int ab) {
#pragma unroll
    for (int i = 0; i < IN_FLIGHT; ++i) load_piece(i, t, tb, ab);
  };
  const auto load_rows = [&](Feed& f, int t) {
    const int x = t * XENT_TR + srow;
    f.st.load(xr, x, t8);
    if (IS_DT) {
      f.g = f.lse2 = f.lr = 0.f;
      f.target = -1;
      if (x < p.nx) {
        f.target = p.target[x];
        f.g = p.weight ? p.weight[x] : 1.f;
        f.lse2 = p.stat[2 * (int64_t)x];
        f.lr = p.stat[2 * (int64_t)x + 1];
      }
    }
  };

  // stationary rows -> operand registers.  Everything that can be is asked for at once, the first two streamed tiles too: small problems are
  // a chain of latencies.
  XentFrag yf[PL][KS];
  float cy = 1.f, ry = 0.f;
  int tgt = -1;
  if (!IS_DT && y_ok) tgt = p.target[y];
  Feed second;
  if (DMA) {
#pragma unroll
    for (int i = 0; i < L::DIST; ++i)
      if (tile0 + i < tile1) load(tile0 + i, i, i);
  } else {
    if (tile0 < tile1) load_rows(feed, tile0);
    if (tile0 + 1 < tile1) load_rows(second, tile0 + 1);
  }
  const auto take = [&](const char* tile) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int q = 0; q < PL; ++q) *(uint4*)yf[q][ks].u = *(const uint4*)(tile + rs.at(ks >> 2, 32 * (ks & 3)) + q * L::PLANE);
  };
  if (DMA) {                                     // straight out of memory: every 128 bytes are used, by four loads in a row
    if (active) {
      if (BF16 && p.y_stride) {                  // (a row behind the last one: the last one again, it is not written)
        const char* from = p.y_image + 2 * (int64_t)(y_ok ? y : p.ny - 1) * p.y_stride + 16 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) *(uint4*)yf[0][ks].u = *(const uint4*)(from + 32 * ks);
      } else {
        take(p.y_image + (int64_t)(y0 / 32) * L::TILE);
      }
    }
    if (y_ok) {
      const float2 f = p.y_fac[y];
      cy = f.x;
      ry = f.y;
    }
    if (IS_DT && h == 0) lds.rn[32 * wave + n] = ry;
  } else if (active) {
    // Each wave its own 32 rows, eight threads a row (whole cache lines), four rows a thread; converted, and turned into operands by way of
    // 4 KB of LDS a plane that no other wave touches: no barriers.  (Read in the operands' own order, 32 bytes of 32 rows at a time,
    // 128 rows of 1 KB took 6 us instead of 3.)
    char* mine = lds.tile + wave * PL * 4096;
    const int r8 = lane >> 3;
    Own own[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) own[g].load(yr, y0 + 8 * g + r8, t8);
#pragma unroll
    for (int g = 0; g < 4; ++g) own[g].scale(p.d, t8);
#pragma unroll
    for (int c = 0; c < DK / 64; ++c) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint4 hi, lo = make_uint4(0, 0, 0, 0);
        own[g].piece(c, hi, lo);
        char* to = mine + xent_half(8 * g + r8, t8);
        *(uint4*)to = hi;
        if (!BF16) *(uint4*)(to + 4096) = lo;
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int q = 0; q < PL; ++q) *(uint4*)yf[q][4 * c + ks].u = *(const uint4*)(mine + q * 4096 + (rs.half ^ (32 * ks)));
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {                // each row's factors to the lanes that now hold it
      const float c = __shfl(own[g].cs, 8 * (n & 7)), r = __shfl(own[g].rn, 8 * (n & 7));
      if (n >> 3 == g) {
        cy = c;
        ry = r;
      }
    }
    if (IS_DT && h == 0) lds.rn[32 * wave + n] = ry;
  }
  if (!IS_DT) cy *= p.scale2;

  // DMA: what this wave asked for has arrived (everyone's: behind the barrier that follows)
  const auto arrived = [&]() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
  const auto factors = [&](const Feed& f, int t, int ab) {       // (not DMA) behind the tile's operands: its rows' part
    const float c = f.st.cs;
    const bool ok = t * XENT_TR + srow < p.nx;
    XentRec& r = lds.rec[ab];
    float lam = BF16 ? 0.f : (float)-f.st.k;
    if (IS_DT) {
      xent_rec_dt(r, srow, ok, c, lam, f.target, f.g, f.lse2, f.lr, p.ny, p.scale2);
    } else {
      if (BF16 && UNIT) lam = c > 0.f ? __builtin_amdgcn_logf(c) : 0.f;
      r.v[0][srow] = c;
      r.v[1][srow] = ok ? lam : -INFINITY;
      r.v[2][srow] = BF16 ? __builtin_amdgcn_exp2f(-lam) : xent_pow2((int)-lam);
    }
  };

  float m = XENT_NONE, l = 0.f;
  f32x16 o[OUT ? DT : 1];
#pragma unroll
  for (int i = 0; i < (OUT ? DT : 1); ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;

  // First product of one tile, S^T = X Y^T, a k step at a time; operands are read AHEAD steps before they are used, and `between` is
  // work for the vector unit in the shadow of each step's matrix instructions (XENT_MIX lays it out).  The small products have a sum of
  // their own, or go before the large ones: every addition rounds at the sum's size, and theirs is 2^-11 of the large one's.  (d <= 128
  // runs two waves in 512 registers: there one sum, and the high halves are read twice.)
  constexpr bool APART = !BF16 && DK > 128;
  constexpr int AHEAD = BF16 ? (DK == 192 ? 3 : KS < 6 ? KS : 6) : APART ? 3 : 2;
  f32x16 s;
  XentFrag fa[AHEAD + 1], fl[AHEAD + 1];
  const auto fetch = [&](const Tile& rt, int ks, bool low) {
    const char* q = lds.tile + rt.at(ks >> 2, 32 * (ks & 3));
    *(uint4*)fa[ks % (AHEAD + 1)].u = *(const uint4*)q;
    if (low) *(uint4*)fl[ks % (AHEAD + 1)].u = *(const uint4*)(q + L::PLANE);
  };
  const auto product = [&](int tb, auto&& between) {
    const Tile rt = rs.plus(tb * L::TILE);
    f32x16 acc, small;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = small[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < AHEAD; ++ks) fetch(rt, ks, !BF16);
    __builtin_amdgcn_sched_barrier(0);
    if (!BF16 && !APART) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + AHEAD < KS) fetch(rt, ks + AHEAD, true);
        acc = xent_mfma<BF16>(fa[ks % (AHEAD + 1)], yf[PL - 1][ks], acc);
        acc = xent_mfma<BF16>(fl[ks % (AHEAD + 1)], yf[0][ks], acc);
        between(ks);
        XENT_MIX(2);
      }
      asm volatile("" ::: "memory");             // (the high halves are read again, not kept)
#pragma unroll
      for (int ks = 0; ks < AHEAD; ++ks) fetch(rt, ks, false);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + AHEAD < KS) fetch(rt, ks + AHEAD, APART);
      if (APART) small = xent_mfma<BF16>(fa[ks % (AHEAD + 1)], yf[PL - 1][ks], small);
      acc = xent_mfma<BF16>(fa[ks % (AHEAD + 1)], yf[0][ks], acc);
      if (APART) small = xent_mfma<BF16>(fl[ks % (AHEAD + 1)], yf[0][ks], small);
      if (BF16 || APART) between(ks);
      XENT_MIX(APART ? 3 : 1);
    }
    s = APART ? acc + small : acc;
  };
  // exponents of a tile whose s is complete, and their largest; register r holds streamed row 8 (r >> 2) + 4 h + (r & 3)
  float e[16], top = 0.f;
  const auto exponents = [&](int q, int ab) {
    const float4 cs = *(const float4*)&lds.rec[ab].v[0][8 * q + 4 * h];
    const float4 la = *(const float4*)&lds.rec[ab].v[1][8 * q + 4 * h];
    e[4 * q] = fmaf(s[4 * q], cs.x * cy, la.x);
    e[4 * q + 1] = fmaf(s[4 * q + 1], cs.y * cy, la.y);
    e[4 * q + 2] = fmaf(s[4 * q + 2], cs.z * cy, la.z);
    e[4 * q + 3] = fmaf(s[4 * q + 3], cs.w * cy, la.w);
    const float t4 = fmaxf(fmaxf(e[4 * q], e[4 * q + 1]), fmaxf(e[4 * q + 2], e[4 * q + 3]));
    top = q ? fmaxf(top, t4) : t4;
  };

  if (tile0 < tile1) {
    if (DMA) {
      arrived();
    } else {
      __syncthreads();                           // the stationary rows have passed
      feed.st.store(lds.tile, wr, p.d, t8);
      factors(feed, tile0, 0);
      if (tile0 + 2 < tile1) load_rows(feed, tile0 + 2);
      if (tile0 + 1 < tile1) {
        second.st.store(lds.tile + L::TILE, wr, p.d, t8);
        factors(second, tile0 + 1, 1);
      }
    }
    __syncthreads();
    if (active) {
      product(0, [](int) {});
#pragma unroll
      for (int q = 0; q < 4; ++q) exponents(q, 0);
    }
    if (!OUT) __syncthreads();                   // two places: the first one is taken next, when everyone has read it
  }
  int mark = 0x7fffffff;                         // DT: target and sign of the next tile's row n
  if (IS_DT && tile0 < tile1) mark = __float_as_int(lds.rec[0].v[3][n]);
  int tb = 0, ab = 0;                            // places of tile t: tile modulo TILES, its rows' part modulo RECS
  for (int t = tile0; t < tile1; ++t) {
    const int tb1 = tb + 1 == L::TILES ? 0 : tb + 1, tb2 = tb1 + 1 == L::TILES ? 0 : tb1 + 1;
    const int ab1 = ab + 1 == L::RECS ? 0 : ab + 1, ab2 = ab1 + 1 == L::RECS ? 0 : ab1 + 1;
    unsigned neg = 0;                            // DT: registers whose entry is subtracted: a negative weight, a target's own (or neither: both)
    const bool more = t + 1 < tile1;
    // DMA: tile t + DIST goes into the place before tile t's, last read by the step before this one (LSE: into tile t's own, its product
    // is done).  Asked for in one go: spread over the steps of the first product it took 4 % longer.
    if (DMA && t + L::DIST < tile1) load(t + L::DIST, OUT ? (tb == 0 ? L::TILES - 1 : tb - 1) : tb, ab == 0 ? L::RECS - 1 : ab - 1);
    if (active) {
      bool found;                                // a target in this tile: its entry is changed, the largest is taken again
      if (!IS_DT) {
        const unsigned at = (unsigned)(tgt - t * XENT_TR);
        found = __any(at < XENT_TR);
        if (found) {
          float own = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool hit = (int)at == 8 * (r >> 2) + 4 * h + (r & 3);
            own = hit ? s[r] : own;
            e[r] = hit ? -INFINITY : e[r];
          }
          if (at < XENT_TR && (int)(at >> 2 & 1) == h) p.st[y] = own * (lds.rec[ab].v[0][at] * cy);
        }
      } else {
        const unsigned below = (unsigned)__ballot(mark < 0) >> 4 * h;      // bit 8 q + i: register 4 q + i
        if (below) neg = (below & 15) | (below >> 4 & 0xf0) | (below >> 8 & 0xf00) | (below >> 12 & 0xf000);
        found = __any((unsigned)((mark & 0x7fffffff) - y0) < 32u);
        if (found) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 own = *(const float4*)&lds.rec[ab].v[2][8 * q + 4 * h], who = *(const float4*)&lds.rec[ab].v[3][8 * q + 4 * h];
            const float o4[4] = {own.x, own.y, own.z, own.w}, w4[4] = {who.x, who.y, who.z, who.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const bool hit = (__float_as_int(w4[k]) & 0x7fffffff) == y;
              e[4 * q + k] = hit ? o4[k] : e[4 * q + k];
              neg ^= hit ? 1u << (4 * q + k) : 0u;
            }
          }
        }
      }
      if (found) {
        top = e[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, e[r]);
      }
      {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) - TOP;
      }
      // (a tile with a target: at once, so that a row's largest entry, its own target's, is 1 and rounds to itself)
      if (__any(top > m + (IS_DT && found ? 0.f : SLACK))) {
        const float now = fmaxf(top, m), alpha = exp2f(m - now);
        m = now;
        l *= alpha;
        if (OUT) {
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
        }
      }
      // the next tile's first product with this tile's exponentials in its shadow
      XentFrag pf[PL][2];
      float4 iv[IS_DT ? 1 : 4];
      if (!IS_DT) {
#pragma unroll
        for (int q = 0; q < 4; ++q) iv[q] = *(const float4*)&lds.rec[ab].v[2][8 * q + 4 * h];
      }
      const auto exponential = [&](int r) {
        e[r] = __builtin_amdgcn_exp2f(e[r] - m);
        if (IS_DT) {
          e[r] = __uint_as_float(__float_as_uint(e[r]) ^ ((neg << (31 - r)) & 0x80000000u));
        } else {
          const float inv = (r & 3) == 0 ? iv[r >> 2].x : (r & 3) == 1 ? iv[r >> 2].y : (r & 3) == 2 ? iv[r >> 2].z : iv[r >> 2].w;
          l = fmaf(e[r], inv, l);
        }
        if (OUT && (r & 1)) {
          if (BF16) pf[0][r >> 3].u[(r & 7) >> 1] = xent_pack_bf16(e[r - 1], e[r]);
          else xent_split(e[r - 1], e[r], pf[0][r >> 3].u[(r & 7) >> 1], pf[PL - 1][r >> 3].u[(r & 7) >> 1]);
        }
      };
      typedef __attribute__((address_space(3))) s16x4* lp;
      const Tile rt2 = ro.plus(tb * L::TILE);
      constexpr int NS = 2 * DT, AH = BF16 ? (DK == 192 ? 3 : NS < 4 ? NS : 4) : 2;
      XentFrag oa[OUT ? AH + 1 : 1], ol[OUT ? AH + 1 : 1];
      const auto fetch2 = [&](int j) {
        const int sk = j / DT, i = j % DT, chunk = i >> 1, rows = (chunk >> 1 < Tile::FULL ? 256 : 128);
        const int x = 64 * (i & 1) | (rows == 256 ? (chunk & 1) << 7 : 0), from = 8192 * (chunk >> 1) + 16 * sk * rows;
        const int r0 = rows == 256 ? rt2.full : rt2.half;
        const char *q0 = lds.tile + (r0 ^ x) + from, *q1 = lds.tile + ((r0 + 8 * rows) ^ (x | 32)) + from;
        oa[j % (AH + 1)].q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q0);
        oa[j % (AH + 1)].q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q1);
        if (!BF16) {
          ol[j % (AH + 1)].q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q0 + L::PLANE));
          ol[j % (AH + 1)].q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q1 + L::PLANE));
        }
      };
      if (more) {
        product(tb1, [&](int ks) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (r * KS / 16 == ks) exponential(r);
        });
      } else {
        // (opaque: else the compiler moves what both branches compute, the exponentials, to before the matrix instructions)
#pragma unroll
        for (int r = 0; r < 16; ++r) asm volatile("" : "+v"(e[r]));
#pragma unroll
        for (int r = 0; r < 16; ++r) exponential(r);
      }
      if (OUT) {
#pragma unroll
        for (int j = 0; j < AH; ++j) fetch2(j);
        __builtin_amdgcn_sched_barrier(0);
      }
      // second product, out^T += X^T P, with the conversion of the tile after next (behind the last tiles: of nothing, into a place
      // that nobody reads) and the next tile's exponents in its shadow
      if (OUT) {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int sk = j / DT, i = j % DT;
          if (j + AH < NS) fetch2(j + AH);
          o[i] = xent_mfma<BF16>(oa[j % (AH + 1)], pf[0][sk], o[i]);
          if (!BF16) {
            o[i] = xent_mfma<BF16>(oa[j % (AH + 1)], pf[PL - 1][sk], o[i]);
            o[i] = xent_mfma<BF16>(ol[j % (AH + 1)], pf[0][sk], o[i]);
          }
          if (!DMA) feed.st.step(j, lds.tile + tb2 * L::TILE, wr, p.d, t8);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q * NS / 4 == j) exponents(q, ab1);
          if (IS_DT && j == NS - 1) mark = __float_as_int(lds.rec[ab1].v[3][n]);
          XENT_MIX(BF16 ? 1 : 3);
        }
      }
    }
    if (!DMA && (!OUT || !active)) feed.st.store(lds.tile + tb2 * L::TILE, wr, p.d, t8);
    if (!OUT && active) {
#pragma unroll
      for (int q = 0; q < 4; ++q) exponents(q, ab1);
    }
    if (!DMA) {
      factors(feed, t + 2, ab2);
      if (t + 3 < tile1) load_rows(feed, t + 3);
    } else {
      arrived();
    }
    __syncthreads();
    tb = tb1;
    ab = ab1;
  }
  if (!active) return;
  if (!IS_DT) l += __shfl_xor(l, 32);
  const int64_t at = (int64_t)split * p.ny + y;
  const int here = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));      // the lane again: not kept through the loop
  if (here < 32 && y_ok && (!IS_DT || p.n_split > 1)) {
    p.part_m[at] = m;
    if (!IS_DT) p.part_l[at] = l;
  }
  if (!OUT) return;
  const bool last = IS_DT && p.n_split == 1;
  if (last) {
    // every query seen: the gradient of the table's row.  Through t = w / |w|: (g - t (t . g)) / |w|; t is in the operand
    // registers, whose halves stand in the other half's order: one exchange between the halves each
    const float half = exp2f(0.5f * m), f = p.scale * half;     // 2^m in two factors: the sums carry the operands' 2^30, 2^m alone may vanish
    if (DMA ? p.unit != 0 : UNIT) {
      const float rn = lds.rn[32 * wave + n];
      float along = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int q = 0; q < PL; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const auto sw = __builtin_amdgcn_permlane32_swap(yf[q][ks].u[i], yf[q][ks].u[2 + i], false, false);
            yf[q][ks].u[i] = sw[0];
            yf[q][ks].u[2 + i] = sw[1];
          }
      // element j of the exchanged operands; t = cy times it (float32: the sum of its two halves, each a mixed-precision multiply-add)
      const auto with = [&](int ks, int j, float x, float y) {
        if (BF16) return fmaf(j & 1 ? bf16_hi(yf[0][ks].u[j >> 1]) : bf16_lo(yf[0][ks].u[j >> 1]), x, y);
        return fmaf((float)yf[PL - 1][ks].h[j], x, fmaf((float)yf[0][ks].h[j], x, y));
      };
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 8; ++j) along = with(ks, j, o[ks >> 1][8 * (ks & 1) + j], along);
      along += __shfl_xor(along, 32);
      const float back = -along * cy * cy;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = with(ks, j, back, o[ks >> 1][8 * (ks & 1) + j]);
          o[ks >> 1][8 * (ks & 1) + j] = v * half * f * rn;
        }
    } else {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= half * f;
    }
  }
  // 64 columns at a time through LDS, so that whole pieces of rows are written.  Partial sums have rows of whole 16 bytes, zero behind d.
  float* turn = (float*)lds.tile + wave * 32 * L::OUT_ROW;
  const int trow = here >> 4, tcol = 4 * (here & 15);
  const bool half = BF16 && last;                // bfloat16 results
  const int size = half ? 2 : 4;
  const int64_t stride = (last ? p.out_stride : (int64_t)p.pitch) * size;
  const int width = last ? p.d : p.pitch, rows = p.ny - y0 - trow;       // rows 4 k + trow, while 4 k is less
  char* to[8];
  to[0] = (last ? (char*)p.out : (char*)(p.part_o + (int64_t)split * p.ny * p.pitch)) + (y0 + trow) * stride + tcol * size;
#pragma unroll
  for (int k = 1; k < 8; ++k) to[k] = to[k - 1] + 4 * stride;
#pragma unroll
  for (int c = 0; c < DK / 64; ++c) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(float4*)(turn + n * L::OUT_ROW + 32 * i + 8 * q + 4 * h) =
            make_float4(o[2 * c + i][4 * q], o[2 * c + i][4 * q + 1], o[2 * c + i][4 * q + 2], o[2 * c + i][4 * q + 3]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int left = width - 64 * c - tcol;      // columns from here on
    const bool some = c < DK / 64 - 1 || left > 0, whole = c < DK / 64 - 1 || left >= 4;
    const auto write = [&](auto&& one) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 v = *(const float4*)(turn + (4 * k + trow) * L::OUT_ROW + tcol);
        if (some && 4 * k < rows) one(to[k] + 64 * c * size, v);
      }
    };
    if (half) {
      write([&](char* at, const float4& v) {
        const uint32_t a = xent_pack_bf16(v.x, v.y), b = xent_pack_bf16(v.z, v.w);
        if (whole) {
          *(XentU2*)at = XentU2{{a, b}};
        } else {
          uint16_t* po = (uint16_t*)at;
          po[0] = (uint16_t)a;
          if (left > 1) po[1] = (uint16_t)(a >> 16);
          if (left > 2) po[2] = (uint16_t)b;
        }
      });
    } else if (last && p.accumulate) {
      write([&](char* at, const float4& v) {
        float* po = (float*)at;
        if (whole) {
          const XentF4 w = *(const XentF4*)po;
          *(XentF4*)po = XentF4{{w.v[0] + v.x, w.v[1] + v.y, w.v[2] + v.z, w.v[3] + v.w}};
        } else {
          po[0] += v.x;
          if (left > 1) po[1] += v.y;
          if (left > 2) po[2] += v.z;
        }
      });
    } else {
      write([&](char* at, const float4& v) {
        if (whole) {
          *(XentF4*)at = XentF4{{v.x, v.y, v.z, v.w}};
        } else {
          float* po = (float*)at;
          po[0] = v.x;
          if (left > 1) po[1] = v.y;
          if (left > 2) po[2] = v.z;
        }
      });
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

#endif
