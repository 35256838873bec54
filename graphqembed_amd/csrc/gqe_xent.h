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
// exponentials are relative to their running maximum, times 2^15, so that the split keeps 22 bits of those that matter.
// bfloat16 operands: one plane, as they are; the exponentials are rounded to bfloat16 (relative error 2^-9, as the output's own).
//
// The target's own term is never part of the sums: dq needs p_target - 1, which cancels when the query is answered well, so the
// sum over the OTHER rows (share r = 1 - p_target) is kept and dq = g scale (sum_others p t - r t_target), and in dt the entry of
// a target is - g_b r_b.  loss = log(1 + 2^(lse_others - s_target)) likewise loses nothing.
#ifndef GQE_XENT_H
#define GQE_XENT_H

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

#define XENT_BM 128            // stationary rows of a workgroup: 32 for each of its four waves
#define XENT_TR 32             // streamed rows of an LDS tile
#ifndef XENT_GROUP
#define XENT_GROUP 4
#endif
#define XENT_NONE (-1.0e30f)   // running maximum before the first term (finite: its difference from -inf is -inf)

enum { XENT_MODE_LSE = 0, XENT_MODE_DQ = 1, XENT_MODE_DT = 2 };

struct XentPass {
  const void* y;               // stationary rows: queries (LSE, DQ), table rows (DT)
  const void* x;               // streamed rows:   table rows (LSE, DQ), queries (DT)
  int64_t y_stride, x_stride;
  int32_t ny, nx, d;
  int32_t y_vec, x_vec;        // rows are 16-byte aligned and d is whole vectors
  int32_t y_unit, x_unit;      // divide these rows by their length
  float scale2;                // scale * log2(e): multiplies s
  float scale;                 // DT: multiplies the result
  int32_t n_tiles, tiles_per_split, n_split, n_yblk;
  const int32_t* target;       // [queries]
  const float* weight;         // DT: [queries] or NULL
  const float* stat;           // DT: [queries][2]
  float* part_m;               // [n_split][ny] running maximum (its unit of the sums)
  float* part_l;               // [n_split][ny] LSE / DQ: sum over the other rows in units of 2^part_m
  float* part_o;               // [n_split][ny][d] (DQ; DT when split)
  float* st;                   // [queries] LSE / DQ: s of the target
  void* out;                   // DT, n_split == 1: dtable
  int64_t out_stride;
  int32_t out_vec, accumulate;
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
__device__ __forceinline__ uint32_t xent_pack_bf16(float a, float b) {
  union { __bf16 h[2]; uint32_t u; } r;
  r.h[0] = (__bf16)a;
  r.h[1] = (__bf16)b;
  return r.u;
}
__device__ __forceinline__ uint32_t xent_pack_f16(float a, float b) {
  union { _Float16 h[2]; uint32_t u; } r;
  r.h[0] = (_Float16)a;
  r.h[1] = (_Float16)b;
  return r.u;
}
// x = hi + lo in fp16, two values at a time.  hi has to be ONE number for both uses: left alone, the compiler fuses the product that
// made x into the conversion on one side only (a single rounding there, two here), and once in some thousand values lo is then the
// remainder of another hi.  The empty asm makes the values opaque.
__device__ __forceinline__ void xent_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  asm("" : "+v"(a), "+v"(b));
  union { _Float16 h[2]; uint32_t u; } r;
  r.u = xent_pack_f16(a, b);
  asm("" : "+v"(r.u));
  hi = r.u;
  lo = xent_pack_f16(a - (float)r.h[0], b - (float)r.h[1]);
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

// n consecutive elements of a row as float, guarded by the row's end (scalar) or whole (vec)
template <bool BF16, int N>
__device__ __forceinline__ void xent_load(const void* base, int64_t row_off, int col, int d, bool row_ok, bool vec, float* v) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  if (!row_ok || col >= d) return;
  if (BF16) {
    const uint16_t* p = (const uint16_t*)base + row_off + col;
    if (vec) {
      static_assert(N == 8 || N == 4, "");
      uint32_t u[N / 2];
      if (N == 8) {
        const uint4 t = *(const uint4*)p;
        u[0] = t.x; u[1] = t.y; u[N / 2 - 2] = t.z; u[N / 2 - 1] = t.w;
      } else {
        const uint2 t = *(const uint2*)p;
        u[0] = t.x; u[1] = t.y;
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) { v[2 * i] = bf16_lo(u[i]); v[2 * i + 1] = bf16_hi(u[i]); }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col + i < d) v[i] = __uint_as_float((uint32_t)p[i] << 16);
    }
  } else {
    const float* p = (const float*)base + row_off + col;
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 t = *(const float4*)(p + i);
        v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col + i < d) v[i] = p[i];
    }
  }
}

template <bool BF16, int DK, int MODE>
struct XentLds {
  static constexpr int PLANES = BF16 ? 1 : 2;
  static constexpr int ROW = 2 * DK + 16;               // bytes of a row of one plane
  static constexpr int PLANE = XENT_TR * ROW;
  static constexpr int TILE = PLANES * PLANE;
  char tile[2][TILE];
  float cs[2][XENT_TR];      // factor of s
  float lam[2][XENT_TR];     // added to s
  float inv[2][XENT_TR];     // LSE / DQ: 2^-lambda
  float sgn[2][XENT_TR];     // DT
  float lamt[2][XENT_TR];    // DT: exponent of a target's entry
  int tgt[2][XENT_TR];       // DT
};

// One thread's share of a streamed tile between its global loads and its LDS stores: 8 threads per row, DK / 8 elements each.
template <bool BF16, int DK, int MODE>
struct XentStage {
  static constexpr int NCH = DK / 64;          // chunks of 8 elements: chunk c of thread t holds columns 64 c + 8 t ..
  uint32_t raw[NCH][BF16 ? 4 : 8];
  float g, lse2, lr;
  int tg;

  __device__ __forceinline__ void load(const XentPass& p, int tile, int tid) {
    const int x = tile * XENT_TR + (tid >> 3), t8 = tid & 7;
    const bool ok = x < p.nx;
    const int64_t off = (int64_t)x * p.x_stride;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = 64 * c + 8 * t8;
      if (BF16) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (ok && col < p.d) {
          const uint16_t* q = (const uint16_t*)p.x + off + col;
          if (p.x_vec) u = *(const uint4*)q;
          else {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = col + i < p.d ? q[i] : 0;
            u = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
          }
        }
        raw[c][0] = u.x; raw[c][1] = u.y; raw[c][2] = u.z; raw[c][3] = u.w;
      } else {
        float v[8];
        xent_load<false, 8>(p.x, off, col, p.d, ok, p.x_vec != 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[c][i] = __float_as_uint(v[i]);
      }
    }
    if (MODE == XENT_MODE_DT) {
      g = 0.f; lse2 = 0.f; lr = 0.f; tg = -1;
      if (ok) {
        tg = p.target[x];
        g = p.weight ? p.weight[x] : 1.f;
        lse2 = p.stat[2 * (int64_t)x];
        lr = p.stat[2 * (int64_t)x + 1];
        if (tg < 0 || tg >= p.ny) { g = 0.f; tg = -1; }
      }
    }
  }

  __device__ __forceinline__ void store(const XentPass& p, XentLds<BF16, DK, MODE>& lds, int buf, int tile, int tid) {
    typedef XentLds<BF16, DK, MODE> L;
    const int row = tid >> 3, t8 = tid & 7;
    const bool ok = tile * XENT_TR + row < p.nx;
    char* base = lds.tile[buf] + row * L::ROW;
    float cs = 1.f, lam = 0.f;
    if (BF16) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) *(uint4*)(base + 2 * (64 * c + 8 * t8)) = make_uint4(raw[c][0], raw[c][1], raw[c][2], raw[c][3]);
      if (p.x_unit) {
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(raw[c][i])), fabsf(bf16_hi(raw[c][i]))));
        mx = fmaxf(mx, __shfl_xor(mx, 1)); mx = fmaxf(mx, __shfl_xor(mx, 2)); mx = fmaxf(mx, __shfl_xor(mx, 4));
        const float f = xent_pow2(xent_row_scale(mx));
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) { const float a = bf16_lo(raw[c][i]) * f, b = bf16_hi(raw[c][i]) * f; ss += a * a + b * b; }
        ss += __shfl_xor(ss, 1); ss += __shfl_xor(ss, 2); ss += __shfl_xor(ss, 4);
        cs = ss > 0.f ? f / sqrtf(ss) : (ss == 0.f ? 0.f : ss);
        if (MODE == XENT_MODE_DQ) lam = cs > 0.f ? log2f(cs) : 0.f;
      }
    } else {
      float mx = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(__uint_as_float(raw[c][i])));
      mx = fmaxf(mx, __shfl_xor(mx, 1)); mx = fmaxf(mx, __shfl_xor(mx, 2)); mx = fmaxf(mx, __shfl_xor(mx, 4));
      int k = xent_row_scale(mx);
      float f = xent_pow2(k);
      if (p.x_unit) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) { const float a = __uint_as_float(raw[c][i]) * f; raw[c][i] = __float_as_uint(a); ss += a * a; }
        ss += __shfl_xor(ss, 1); ss += __shfl_xor(ss, 2); ss += __shfl_xor(ss, 4);
        k = 14;
        f = ss > 0.f ? 16384.f / sqrtf(ss) : (ss == 0.f ? 0.f : ss);
      }
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xent_split(__uint_as_float(raw[c][2 * i]) * f, __uint_as_float(raw[c][2 * i + 1]) * f, hi[i], lo[i]);
        char* q = base + 2 * (64 * c + 8 * t8);
        *(uint4*)q = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *(uint4*)(q + L::PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      cs = xent_pow2(-k);
      if (MODE != XENT_MODE_LSE) lam = (float)-k;
    }
    if (t8 == 0) {
      if (MODE == XENT_MODE_DT) {
        const float lg = g != 0.f ? log2f(fabsf(g)) : -INFINITY;
        lds.cs[buf][row] = cs * p.scale2;
        lds.lam[buf][row] = ok ? lam + (lg - lse2) : -INFINITY;
        lds.lamt[buf][row] = lam + (lg + lr);
        lds.sgn[buf][row] = copysignf(1.f, g);
        lds.tgt[buf][row] = tg;
      } else {
        lds.cs[buf][row] = cs;
        lds.lam[buf][row] = ok ? lam : -INFINITY;
        lds.inv[buf][row] = BF16 ? exp2f(-lam) : xent_pow2((int)-lam);
      }
    }
  }
};

template <bool BF16, int DK, int MODE>
__global__ __launch_bounds__(256, DK <= 128 ? 2 : 1) void gqe_xent_kernel(XentPass p) {
  typedef XentLds<BF16, DK, MODE> L;
  extern __shared__ char smem[];
  L& lds = *(L*)smem;
  constexpr int PL = BF16 ? 1 : 2, KS = DK / 16, DT = DK / 32;
  constexpr bool OUT = MODE != XENT_MODE_LSE;
  constexpr float TOP = BF16 ? 0.f : 15.f;       // exponentials reach 2^TOP
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5;
  const int split = blockIdx.x % p.n_split, yblk = blockIdx.x / p.n_split;
  const int y0 = yblk * XENT_BM + wave * 32, y = y0 + n;
  const bool active = y0 < p.ny, y_ok = y < p.ny;
  const int tile0 = split * p.tiles_per_split;
  const int tile1 = min(tile0 + p.tiles_per_split, p.n_tiles);

  // stationary rows -> operand registers
  XentFrag yf[PL][KS];
  float cy = 1.f;
  {
    const int64_t off = (int64_t)y * p.y_stride;
    if (BF16) {
      float ss = 0.f, mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float v[8];
        xent_load<true, 8>(p.y, off, 16 * ks + 8 * h, p.d, y_ok, p.y_vec != 0, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          yf[0][ks].u[i] = __float_as_uint(v[2 * i]) >> 16 | (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
          mx = fmaxf(mx, fmaxf(fabsf(v[2 * i]), fabsf(v[2 * i + 1])));
        }
      }
      if (MODE == XENT_MODE_DT && p.y_unit) {
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float f = xent_pow2(xent_row_scale(mx));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) { const float a = bf16_lo(yf[0][ks].u[i]) * f, b = bf16_hi(yf[0][ks].u[i]) * f; ss += a * a + b * b; }
        ss += __shfl_xor(ss, 32);
        cy = ss > 0.f ? f / sqrtf(ss) : (ss == 0.f ? 0.f : ss);
      }
    } else {
      // the row is read twice (it comes out of the cache the second time): its largest element and length first, then the split,
      // so that the whole row never sits in registers next to its operands
      float mx = 0.f, ss = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float v[8];
        xent_load<false, 8>(p.y, off, 16 * ks + 8 * h, p.d, y_ok, p.y_vec != 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(v[i]));
      }
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      int k = xent_row_scale(mx);
      const float f = xent_pow2(k);
      float f2 = 1.f;
      if (MODE == XENT_MODE_DT && p.y_unit) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          float v[8];
          xent_load<false, 8>(p.y, off, 16 * ks + 8 * h, p.d, y_ok, p.y_vec != 0, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) { const float a = v[i] * f; ss += a * a; }
        }
        ss += __shfl_xor(ss, 32);
        k = 14;
        f2 = ss > 0.f ? 16384.f / sqrtf(ss) : (ss == 0.f ? 0.f : ss);
      }
      asm volatile("" ::: "memory");
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float v[8];
        xent_load<false, 8>(p.y, off, 16 * ks + 8 * h, p.d, y_ok, p.y_vec != 0, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) xent_split(v[2 * i] * f * f2, v[2 * i + 1] * f * f2, yf[0][ks].u[i], yf[PL - 1][ks].u[i]);
        if (ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      cy = xent_pow2(-k);
    }
    if (MODE != XENT_MODE_DT) cy *= p.scale2;
  }
  int tgt = -1;
  if (MODE != XENT_MODE_DT && y_ok) tgt = p.target[y];

  float m = XENT_NONE, l = 0.f;
  f32x16 o[OUT ? DT : 1];
#pragma unroll
  for (int i = 0; i < (OUT ? DT : 1); ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;

  __builtin_amdgcn_sched_barrier(0);
  XentStage<BF16, DK, MODE> stage;
  if (tile0 < tile1) {
    stage.load(p, tile0, tid);
    stage.store(p, lds, 0, tile0, tid);
  }
  __syncthreads();
  for (int t = tile0; t < tile1; ++t) {
    const int buf = (t - tile0) & 1;
    const bool more = t + 1 < tile1;
    if (more) stage.load(p, t + 1, tid);
    __builtin_amdgcn_sched_barrier(0);
    if (active) {
      const char* xt = lds.tile[buf];
      // the small products in a sum of their own: every addition rounds at the sum's size, and theirs is 2^-11 of the large one's
      f32x16 s, sx;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = sx[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        XentFrag a, al;
        const char* q = xt + n * L::ROW + 2 * (16 * ks + 8 * h);
        *(uint4*)a.u = *(const uint4*)q;
        s = xent_mfma<BF16>(a, yf[0][ks], s);
        if (!BF16) {
          *(uint4*)al.u = *(const uint4*)(q + L::PLANE);
          sx = xent_mfma<BF16>(a, yf[PL - 1][ks], sx);
          sx = xent_mfma<BF16>(al, yf[0][ks], sx);
        }
        if (ks % XENT_GROUP == XENT_GROUP - 1) __builtin_amdgcn_sched_barrier(0);
      }
      if (!BF16) s += sx;
      __builtin_amdgcn_sched_barrier(0);
      // exponents; register r holds streamed row 8 (r >> 2) + 4 h + (r & 3)
      float e[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 cs = *(const float4*)&lds.cs[buf][8 * q + 4 * h];
        const float4 la = *(const float4*)&lds.lam[buf][8 * q + 4 * h];
        e[4 * q] = fmaf(s[4 * q], cs.x * cy, la.x);
        e[4 * q + 1] = fmaf(s[4 * q + 1], cs.y * cy, la.y);
        e[4 * q + 2] = fmaf(s[4 * q + 2], cs.z * cy, la.z);
        e[4 * q + 3] = fmaf(s[4 * q + 3], cs.w * cy, la.w);
      }
      unsigned hit = 0;          // DT: registers that hold a target's own entry (subtracted)
      if (MODE != XENT_MODE_DT) {
        const unsigned at = (unsigned)(tgt - t * XENT_TR);
        if (__any(at < XENT_TR)) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = 8 * (r >> 2) + 4 * h + (r & 3);
            if ((int)at == row) {
              p.st[y] = s[r] * (lds.cs[buf][row] * cy);
              e[r] = -INFINITY;
            }
          }
        }
      } else {
        const unsigned at = (unsigned)(lds.tgt[buf][n] - y0);
        if (__any(at < 32)) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = 8 * (r >> 2) + 4 * h + (r & 3);
            if (lds.tgt[buf][row] == y) {
              e[r] = lds.lamt[buf][row];
              hit |= 1u << r;
            }
          }
        }
      }
      float top = e[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, e[r]);
      top = fmaxf(top, __shfl_xor(top, 32)) - TOP;
      if (__any(top > m)) {
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
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 iv = *(const float4*)(MODE == XENT_MODE_DT ? &lds.sgn[buf][8 * q + 4 * h] : &lds.inv[buf][8 * q + 4 * h]);
        const float inv[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * q + i;
          e[r] = __builtin_amdgcn_exp2f(e[r] - m);
          if (MODE == XENT_MODE_DT) e[r] *= inv[i];
          else l = fmaf(e[r], inv[i], l);
        }
      }
      if (MODE == XENT_MODE_DT && __any(hit != 0)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = hit >> r & 1 ? -e[r] : e[r];
      }
      if (OUT) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int sk = 0; sk < 2; ++sk) {
          XentFrag pf[PL];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (BF16) pf[0].u[i] = xent_pack_bf16(e[8 * sk + 2 * i], e[8 * sk + 2 * i + 1]);
            else xent_split(e[8 * sk + 2 * i], e[8 * sk + 2 * i + 1], pf[0].u[i], pf[PL - 1].u[i]);
          }
          // X^T operand: lane's 16-lane group reads 4 rows x 16 columns, transposed
          const int row = 16 * sk + 4 * h + ((lane & 15) >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
          const char* q = xt + row * L::ROW + 2 * col;
          typedef __attribute__((address_space(3))) s16x4* lp;
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            XentFrag a, al;
            a.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 64 * i));
            a.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 64 * i + 8 * L::ROW));
            o[i] = xent_mfma<BF16>(a, pf[0], o[i]);
            if (!BF16) {
              al.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + L::PLANE + 64 * i));
              al.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + L::PLANE + 64 * i + 8 * L::ROW));
              o[i] = xent_mfma<BF16>(a, pf[PL - 1], o[i]);
              o[i] = xent_mfma<BF16>(al, pf[0], o[i]);
            }
            if (i % XENT_GROUP == XENT_GROUP - 1) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) stage.store(p, lds, buf ^ 1, t + 1, tid);
    __syncthreads();
  }
  if (!active) return;
  if (MODE != XENT_MODE_DT) l += __shfl_xor(l, 32);
  if (!y_ok) return;
  if (MODE != XENT_MODE_DT || p.n_split > 1) {
    const int64_t at = (int64_t)split * p.ny + y;
    if (h == 0) {
      p.part_m[at] = m;
      if (MODE != XENT_MODE_DT) p.part_l[at] = l;
    }
    if (OUT) {
      float* po = p.part_o + at * p.d;
      const bool v4 = (p.d & 3) == 0;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * i + 8 * q + 4 * h;
          if (v4) {
            if (c < p.d) *(float4*)(po + c) = make_float4(o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < p.d) po[c + j] = o[i][4 * q + j];
          }
        }
    }
    return;
  }
  // DT, every query seen: the gradient of the table's row
  if (MODE == XENT_MODE_DT) {
    const float half = exp2f(0.5f * m), f = p.scale * half;     // 2^m in two factors: the sums carry the operands' 2^30, 2^m alone may vanish
    const int64_t off = (int64_t)y * p.y_stride;
    float along = 0.f, rn2 = 0.f, rn = 1.f;
    if (p.y_unit) {        // through t = w / |w|: (g - t (t . g)) / |w|
      // f32: cy undoes the operand's scale 2^14 only, the length is taken from the row again
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float w[4];
          xent_load<BF16, 4>(p.y, off, 32 * i + 8 * q + 4 * h, p.d, true, p.y_vec != 0, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) { along = fmaf(w[j], o[i][4 * q + j], along); ss = fmaf(w[j], w[j], ss); }
        }
      along += __shfl_xor(along, 32);
      ss += __shfl_xor(ss, 32);
      rn = ss > 0.f ? 1.f / sqrtf(ss) : (ss == 0.f ? 0.f : ss);
      rn2 = along * rn * rn;
    }
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * i + 8 * q + 4 * h;
        float v[4];
        if (p.y_unit) {
          float w[4];
          xent_load<BF16, 4>(p.y, off, c, p.d, true, p.y_vec != 0, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = (o[i][4 * q + j] - w[j] * rn2) * half * f * rn;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = o[i][4 * q + j] * half * f;
        }
        if (BF16) {
          uint16_t* po = (uint16_t*)p.out + (int64_t)y * p.out_stride + c;
          const uint32_t a = xent_pack_bf16(v[0], v[1]), b = xent_pack_bf16(v[2], v[3]);
          if (p.out_vec) {
            if (c < p.d) *(uint2*)po = make_uint2(a, b);
          } else {
            const uint16_t e4[4] = {(uint16_t)a, (uint16_t)(a >> 16), (uint16_t)b, (uint16_t)(b >> 16)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < p.d) po[j] = e4[j];
          }
        } else {
          float* po = (float*)p.out + (int64_t)y * p.out_stride + c;
          if (p.out_vec) {
            if (c < p.d) {
              if (p.accumulate) { const float4 w = *(const float4*)po; v[0] += w.x; v[1] += w.y; v[2] += w.z; v[3] += w.w; }
              *(float4*)po = make_float4(v[0], v[1], v[2], v[3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < p.d) po[j] = p.accumulate ? po[j] + v[j] : v[j];
          }
        }
      }
  }
}

#endif
