// gqe_ops.hip — the operators of include/gqe_ops.h: entry points, the joins of the softmax cross entropy's splits, gradient norm and
// clipping, layer normalisation.  The softmax cross entropy's two passes are gqe_xent.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/gqe_ops.h"
#include "gqe_common.h"
#include "gqe_ops_dev.h"
#include "gqe_xent.h"

namespace {

thread_local std::string g_ops_error;

int refuse(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  try {
    g_ops_error = buf;
  } catch (...) {
  }
  return code;
}

// the launches of a call go to `device`, whatever device the caller has current
struct OnDevice {
  int before = -1;
  hipError_t status;
  explicit OnDevice(int device) {
    status = hipGetDevice(&before);
    if (status == hipSuccess && before != device) status = hipSetDevice(device);
    else if (status == hipSuccess) before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

int hip_refuse(hipError_t e, const char* what) { return refuse(GQE_ERR_HIP, "%s: %s", what, hipGetErrorString(e)); }

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// ------------------------------------------------------------------------------------------------------------------------------
// softmax cross entropy: join of the splits
// ------------------------------------------------------------------------------------------------------------------------------
#define XENT_MAX_SPLIT 1024
#define XENT_JOIN_BATCH 8

struct XentJoin {
  const float *part_m, *part_l, *part_o, *st;
  int32_t n_split, ny, d, n_rows;
  const int32_t* target;
  const float* weight;
  const void* table;       // DQ: the target's row; DT: the row itself
  int64_t table_stride;
  int32_t unit, out_f32, accumulate, lanes, pitch;
  float scale;
  float *loss, *lse, *stat;
  XentRec* rec;            // LSE / DQ: the queries as streamed rows of the table's gradient, which this call goes on to
  const float2* fac;
  float scale2;
  void* out;
  int64_t out_stride;
};

template <bool BF16>
__device__ __forceinline__ float row_elem(const void* p, int64_t i) {
  if (BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  return ((const float*)p)[i];
}
template <bool BF16>
__device__ __forceinline__ void put_elem(void* p, int64_t i, float v, bool accumulate) {
  if (BF16) {
    ((uint16_t*)p)[i] = (uint16_t)xent_pack_bf16(v, v);
  } else {
    float* q = (float*)p + i;
    *q = accumulate ? *q + v : v;
  }
}

// f(x of this lane, x of lane ^ O), f commutative, as the arithmetic unit itself moves lanes: a shuffle goes through LDS, 60 cycles and more
// that nothing hides where a row's sums follow one another.  O = 4: lanes 8 apart hold the same x already (rows of 16 are turned by 4).
template <int O>
__device__ __forceinline__ void lane_pair(uint32_t x, uint32_t& a, uint32_t& b) {
  if (O == 32 || O == 16) {
    const auto r = O == 32 ? __builtin_amdgcn_permlane32_swap(x, x, false, false) : __builtin_amdgcn_permlane16_swap(x, x, false, false);
    a = r[0];
    b = r[1];
  } else {
    constexpr int how = O == 8 ? 0x128 : O == 4 ? 0x124 : O == 2 ? 0x4e : 0xb1;      // row_ror:8, row_ror:4, quad_perm [2,3,0,1], [1,0,3,2]
    a = x;
    b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, how, 0xf, 0xf, true);
  }
}
template <int O>
__device__ __forceinline__ float lane_sum(float x) {
  uint32_t a, b;
  lane_pair<O>(__float_as_uint(x), a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}
template <int O>
__device__ __forceinline__ float lane_max(float x) {
  uint32_t a, b;
  lane_pair<O>(__float_as_uint(x), a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
template <int O>
__device__ __forceinline__ double lane_sum(double x) {
  uint32_t a[2], b[2];
  lane_pair<O>((uint32_t)__double2loint(x), a[0], b[0]);
  lane_pair<O>((uint32_t)__double2hiint(x), a[1], b[1]);
  return __hiloint2double((int)a[1], (int)a[0]) + __hiloint2double((int)b[1], (int)b[0]);
}
// over all 64 lanes, the same bits in each
template <typename T>
__device__ __forceinline__ T wave_total(T x) {
  return lane_sum<1>(lane_sum<2>(lane_sum<4>(lane_sum<8>(lane_sum<16>(lane_sum<32>(x))))));
}
__device__ __forceinline__ float wave_max(float x) {
  return lane_max<1>(lane_max<2>(lane_max<4>(lane_max<8>(lane_max<16>(lane_max<32>(x))))));
}
// 2^x and log2 x of a 64-bit number to float32's relative (absolute, below 1) precision: whole powers apart, the rest in float32
__device__ __forceinline__ float exp2_of(double x) {
  const double n = floor(fmax(x, -1000.0));
  return ldexpf(exp2f((float)(x - n)), (int)n);
}
__device__ __forceinline__ double log2_of(double x) {
  int e;
  const double f = frexp(x, &e);
  return x > 0.0 ? (double)(e - 1) + (double)log2f((float)(f + f)) : x == 0.0 ? -INFINITY : x;
}

// four elements of a row, wherever it begins (those behind column d: zero)
template <bool BF16>
__device__ __forceinline__ void row_four(const void* p, int64_t at, int left, float* t) {
  if (left >= 4) {
    if (BF16) {
      const XentU2 u = *(const XentU2*)((const uint16_t*)p + at);
      t[0] = bf16_lo(u.v[0]); t[1] = bf16_hi(u.v[0]); t[2] = bf16_lo(u.v[1]); t[3] = bf16_hi(u.v[1]);
    } else {
      const XentF4 u = *(const XentF4*)((const float*)p + at);
      t[0] = u.v[0]; t[1] = u.v[1]; t[2] = u.v[2]; t[3] = u.v[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = i < left ? row_elem<BF16>(p, at + i) : 0.f;
  }
}
template <bool BF16>
__device__ __forceinline__ void put_four(void* p, int64_t at, int left, const float* v, bool accumulate) {
  if (left >= 4) {
    if (BF16) {
      *(XentU2*)((uint16_t*)p + at) = XentU2{{xent_pack_bf16(v[0], v[1]), xent_pack_bf16(v[2], v[3])}};
    } else {
      XentF4* q = (XentF4*)((float*)p + at);
      const XentF4 w = accumulate ? *q : XentF4{{0.f, 0.f, 0.f, 0.f}};
      *q = XentF4{{accumulate ? w.v[0] + v[0] : v[0], accumulate ? w.v[1] + v[1] : v[1], accumulate ? w.v[2] + v[2] : v[2], accumulate ? w.v[3] + v[3] : v[3]}};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) put_elem<BF16>(p, at + i, v[i], accumulate);
  }
}

// The splits' sums of a stationary row, each with its own unit 2^part_m, added in a fixed order.  Bound by latency: a lane takes 16 bytes of
// a split, `lanes` of them a row, so that a wave has 64 / lanes splits at once and eight times as many under way, and nothing waits for
// the largest unit: each lane's sums follow a running one of their own and are brought together at the end.  WAVES = 1: a wave per row,
// four rows a workgroup (few splits, or many rows); more: a workgroup per row.
template <bool BF16, int MODE, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void gqe_xent_join_kernel(XentJoin p) {
  constexpr bool LSE = MODE == XENT_MODE_LSE, DT = MODE == XENT_MODE_DT;
  constexpr int BATCH = XENT_JOIN_BATCH;
  __shared__ float redm[WAVES];
  __shared__ double redl[WAVES];
  __shared__ __align__(16) float acc[WAVES == 1 || LSE ? 1 : WAVES][256];
  const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6;
  const int64_t y = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (WAVES == 1 && y >= p.ny) return;
  const int lanes = LSE ? 1 : p.lanes, c = 4 * (lane & (lanes - 1)), left = p.d - c;
  const int at_once = 64 / lanes * WAVES, first = wave * (64 / lanes) + lane / lanes;
  // what the end needs is asked for first: behind the sums it would be latencies in a row
  int tg = -1;
  float st = 0.f, g = 1.f, factor = 1.f;
  if (!DT) {
    tg = p.target[y];
    st = p.st[y];
    if (p.weight) g = p.weight[y];
    if (p.rec) factor = p.fac[y].x;
  }
  float t[4] = {0.f, 0.f, 0.f, 0.f};             // the target's row (DQ), the row itself (DT), once the splits' are under way

  float m = XENT_NONE, v[4] = {0.f, 0.f, 0.f, 0.f};
  double l = 0.0;
  for (int s0 = first; s0 < p.n_split; s0 += BATCH * at_once) {
    float pm[BATCH], pl[BATCH];
    float4 u[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int64_t at = (int64_t)(s0 + i * at_once) * p.ny + y;
      const bool in = s0 + i * at_once < p.n_split;
      pm[i] = in ? p.part_m[at] : XENT_NONE;
      pl[i] = !DT && in && c == 0 ? p.part_l[at] : 0.f;
      u[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!LSE && in && left > 0) u[i] = *(const float4*)(p.part_o + at * p.pitch + c);
    }
    if (!LSE && s0 == 0) {                       // (the first lanes of the first wave: those that write the row)
      const int64_t row = DT ? y : tg >= 0 && tg < p.n_rows ? tg : -1;
      if (row >= 0 && (!DT || p.unit) && left > 0) row_four<BF16>(p.table, row * p.table_stride + c, left, t);
    }
    float now = m;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) now = fmaxf(now, pm[i]);
    const float w0 = __builtin_amdgcn_exp2f(m - now);
    m = now;
    l *= (double)w0;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= w0;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float w = __builtin_amdgcn_exp2f(pm[i] - m);
      l += (double)pl[i] * (double)w;
      v[0] = fmaf(w, u[i].x, v[0]); v[1] = fmaf(w, u[i].y, v[1]); v[2] = fmaf(w, u[i].z, v[2]); v[3] = fmaf(w, u[i].w, v[3]);
    }
  }
  {
    const float top = wave_max(m), w = __builtin_amdgcn_exp2f(m - top);
    m = top;
    if (!DT) l = wave_total(l * (double)w);
    if (!LSE) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= w;
      for (int k = 0; k < 4; ++k) {      // lanes that hold the same columns
        if (lanes <= 32) v[k] = lane_sum<32>(v[k]);
        if (lanes <= 16) v[k] = lane_sum<16>(v[k]);
        if (lanes <= 8) v[k] = lane_sum<8>(v[k]);
        if (lanes <= 4) v[k] = lane_sum<4>(v[k]);
        if (lanes <= 2) v[k] = lane_sum<2>(v[k]);
        if (lanes <= 1) v[k] = lane_sum<1>(v[k]);
      }
    }
  }
  if (WAVES > 1) {
    if (lane == 0) { redm[wave] = m; redl[wave] = l; }
    if (!LSE && lane < lanes) *(float4*)&acc[wave][c] = make_float4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, redm[w]);
    l = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(redm[w] - m);
      l += redl[w] * (double)f;
      if (!LSE) {
        const float4 u = *(const float4*)&acc[w][c];
        v[0] = fmaf(f, u.x, v[0]); v[1] = fmaf(f, u.y, v[1]); v[2] = fmaf(f, u.z, v[2]); v[3] = fmaf(f, u.w, v[3]);
      }
    }
  }
  float lse2, lr, above;
  float half, f, share = 0.f;               // half * f: the unit's power in two factors, the sums carry the operands' 2^30
  if (!DT) {
    // In base 2 and 64 bits: the other rows' sum, -inf where the target is the only row; diff: its log2 over the target's term.  (In 32 bits
    // 0.2 us less at 100 x 1000 x 128, and the loss twice as far off: 8.5e-7 for 4.4e-7.)
    const bool has = tg >= 0 && tg < p.n_rows;
    const double others = (double)m + log2_of(l), diff = others - (double)st;
    const double soft = has ? (double)log1pf(exp2_of(-fabs(diff))) * 1.4426950408889634 : 0.0;
    const double big = has ? fmax(others, (double)st) + soft : others;
    const bool nan = has && diff != diff;
    const float loss = nan ? (float)diff : has ? (float)((fmax(diff, 0.0) + soft) * 0.6931471805599453) : tg >= p.n_rows ? NAN : 0.f;
    const float lse = nan ? loss : (float)(big * 0.6931471805599453);
    lse2 = nan ? loss : (float)big;
    lr = nan ? loss : (float)(fmin(diff, 0.0) - soft);
    above = nan ? loss : (float)((double)m - big);
    if (!has) g = 0.f;
    if (lane == 0) {
      if (p.loss) p.loss[y] = loss;
      if (p.lse) p.lse[y] = lse;
      p.stat[2 * y] = lse2;
      p.stat[2 * y + 1] = lr;
    }
    if (p.rec && lane < XENT_TR) {      // (the last row: also what fills its tile)
      const int i = (int)(y % XENT_TR), last = y == p.ny - 1 ? XENT_TR - 1 : i;
      if (lane >= i && lane <= last) {
        const bool ok = lane == i;
        const float k = ok ? factor : 1.f;
        xent_rec_dt(p.rec[y / XENT_TR], lane, ok, k, BF16 ? 0.f : xent_exponent(k), ok ? tg : -1, ok ? g : 0.f, lse2, lr, p.n_rows, p.scale2);
      }
    }
    if (LSE) return;
    share = exp2f(lr);
    half = f = exp2f(0.5f * above);
  } else {
    half = exp2f(0.5f * m);
    f = p.scale * half;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = v[k] * half * f;
  const bool mine = lane < lanes && left > 0;     // (behind the sums every group of `lanes` holds the row)
  float rn = 1.f;
  if (p.unit) {                                  // (no target: zeros stay zeros)
    const float k = xent_pow2(xent_row_scale(wave_max(fmaxf(fmaxf(fabsf(t[0]), fabsf(t[1])), fmaxf(fabsf(t[2]), fabsf(t[3]))))));
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = fmaf(t[i] * k, t[i] * k, ss);
    rn = xent_rsqrt(wave_total(lane < lanes ? ss : 0.f)) * k;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] *= rn;
  }
  if (!DT) {
    const float gs = g * p.scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = g != 0.f ? gs * fmaf(-share, t[i], v[i]) : 0.f;
  } else if (p.unit) {
    float along = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) along = fmaf(t[i], v[i], along);
    along = wave_total(lane < lanes ? along : 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (v[i] - t[i] * along) * rn;
  }
  if (!mine) return;
  if (p.out_f32) put_four<false>(p.out, y * p.out_stride + c, left, v, p.accumulate != 0);
  else put_four<BF16>(p.out, y * p.out_stride + c, left, v, p.accumulate != 0);
}

struct XentPlan {
  int dk, n_tiles, n_yblk, n_split, per;
};

// Splits of the streamed axis: enough workgroups to fill the 256 CUs (`slots` of them at once), `least` tiles in each at least.
XentPlan xent_plan(int64_t ny, int64_t nx, int dim, int slots, int least) {
  XentPlan r;
  r.dk = dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
  r.n_tiles = (int)((nx + XENT_TR - 1) / XENT_TR);
  r.n_yblk = (int)((ny + XENT_BM - 1) / XENT_BM);
  int64_t s = std::min<int64_t>(slots / std::max(r.n_yblk, 1), XENT_MAX_SPLIT);
  s = std::max<int64_t>(1, std::min<int64_t>(s, r.n_tiles / least));
  r.per = (int)std::max<int64_t>(1, (r.n_tiles + s - 1) / s);
  r.n_split = std::max(1, (r.n_tiles + r.per - 1) / r.per);
  return r;
}

// Operands are prepared (one more pass over the table: read, written, and read again instead of it) where more than one block of
// queries would convert the same rows again; up to XENT_BM queries the passes are bound by memory and convert as they go.
bool xent_prepares(const gqe_xent_args* a) { return a->n_queries > XENT_BM; }
// workgroups at once: two a CU where the kernels' registers allow it (XENT_TWO)
int xent_slots(const gqe_xent_args* a) { return a->dim <= 128 || (a->dtype == GQE_BF16 && a->dim <= 192 && xent_prepares(a)) ? 512 : 256; }
XentPlan xent_plan_queries(const gqe_xent_args* a) { return xent_plan(a->n_queries, a->n_rows, a->dim, xent_slots(a), 1); }
// The table's gradient takes four tiles of queries at least: below that the join costs more than a split saves (136 queries, 14575 rows of
// d = 200, 5 tiles: 20 us, and a join of 11 us as 4 + 1).  Where float32 rows of d > 64 are converted on the way a tile takes 3 to 8 us, and
// with three or four of them and few rows to join each goes by itself (100 queries, 1000 rows of d = 128: 20 us, apart 12 + 4; d = 64: 13
// us, apart 10 + 5).  Where tiles are cheap (0.5 to 1.1 us: bfloat16, or d <= 64) and rows to join are many, a workgroup takes up to 19 itself (11
// tiles, 11988 bfloat16 rows of d = 175: 22 us against 17 + 10 in two splits; 19 tiles, 20000 float32 rows of d = 64: 30 us against 23 + 13 in
// three; with 8000 rows or d = 128 the two are even, and 32 tiles of d = 64, 12000 rows, are 23 + 10 us in four splits, 27 + 9 in three).
XentPlan xent_plan_table(const gqe_xent_args* a) {
  const int64_t blocks = (a->n_rows + XENT_BM - 1) / XENT_BM, tiles = (a->n_queries + XENT_TR - 1) / XENT_TR;
  const bool apart = a->dtype == GQE_F32 && a->dim > 64 && !xent_prepares(a) && tiles >= 3 && blocks * tiles <= 128;
  const bool cheap = (a->dtype == GQE_BF16 || a->dim <= 64) && blocks >= 80 && tiles < 20;
  return xent_plan(a->n_rows, a->n_queries, a->dim, xent_slots(a), apart ? 1 : cheap ? 20 : 4);
}
// bfloat16 rows that are operands as they lie: whole tiles wide, 16-byte pieces
bool xent_as_is(bool bf16, int dk, int dim, const void* ptr, int64_t stride) { return bf16 && dk == dim && aligned(ptr, 16) && stride % 8 == 0 && stride < (1 << 25); }

struct XentSpace {
  int64_t part_m, part_l, st, stat, part_o, image[2], fac[2], rec, total;
};
XentSpace xent_space(const gqe_xent_args* a, const XentPlan& q, const XentPlan& t) {
  XentSpace s;
  const bool dq = a->phase & GQE_XENT_DQ, dt = (a->phase & GQE_XENT_DTABLE) && t.n_split > 1;
  const bool first = a->phase & (GQE_XENT_LOSS | GQE_XENT_DQ);
  const int64_t pq = first ? (int64_t)q.n_split * a->n_queries : 0, pt = dt ? (int64_t)t.n_split * a->n_rows : 0;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at = up(at + bytes, 256); return o; };
  s.part_m = take(4 * std::max(pq, pt));
  s.part_l = take(4 * pq);
  s.st = take(first ? 4 * a->n_queries : 0);
  s.stat = take(a->stat ? 0 : 8 * a->n_queries);
  s.part_o = take(4 * up(a->dim, 4) * std::max(dq ? pq : 0, pt));
  const int64_t n[2] = {a->n_queries, a->n_rows};
  for (int i = 0; i < 2; ++i) {      // (sizes alone decide: room for the image also where the rows turn out to be usable as they lie)
    s.image[i] = take(xent_prepares(a) ? up(n[i], XENT_TR) * q.dk * (a->dtype == GQE_BF16 ? 2 : 4) : 0);
    s.fac[i] = take(xent_prepares(a) ? 8 * n[i] : 0);
  }
  s.rec = take(xent_prepares(a) ? up(std::max(n[0], n[1]), XENT_TR) / XENT_TR * (int64_t)sizeof(XentRec) : 0);
  s.total = at;
  return s;
}

hipError_t xent_launch(bool bf16, int dk, int mode, bool unit, bool dma, const XentPass& p, hipStream_t s) {
  switch (dk) {
    case 64: return bf16 ? gqe_xent_launch_1_64(mode, unit, dma, p, s) : gqe_xent_launch_0_64(mode, unit, dma, p, s);
    case 128: return bf16 ? gqe_xent_launch_1_128(mode, unit, dma, p, s) : gqe_xent_launch_0_128(mode, unit, dma, p, s);
    case 192: return bf16 ? gqe_xent_launch_1_192(mode, unit, dma, p, s) : gqe_xent_launch_0_192(mode, unit, dma, p, s);
    default: return bf16 ? gqe_xent_launch_1_256(mode, unit, dma, p, s) : gqe_xent_launch_0_256(mode, unit, dma, p, s);
  }
}

hipError_t xent_prep(bool bf16, int dk, bool unit, const XentPrep& p, hipStream_t s) {
  switch (dk) {
    case 64: return bf16 ? gqe_xent_prep_1_64(unit, p, s) : gqe_xent_prep_0_64(unit, p, s);
    case 128: return bf16 ? gqe_xent_prep_1_128(unit, p, s) : gqe_xent_prep_0_128(unit, p, s);
    case 192: return bf16 ? gqe_xent_prep_1_192(unit, p, s) : gqe_xent_prep_0_192(unit, p, s);
    default: return bf16 ? gqe_xent_prep_1_256(unit, p, s) : gqe_xent_prep_0_256(unit, p, s);
  }
}

template <int MODE, int WAVES>
void join_launch(bool bf16, const XentJoin& j, hipStream_t s) {
  const dim3 grid((unsigned)(WAVES == 1 ? (j.ny + 3) / 4 : j.ny)), block(WAVES == 1 ? 256 : 64 * WAVES);
  if (bf16) gqe_xent_join_kernel<true, MODE, WAVES><<<grid, block, 0, s>>>(j);
  else gqe_xent_join_kernel<false, MODE, WAVES><<<grid, block, 0, s>>>(j);
}
// Waves a row by `loads`, 16 bytes each, that a row takes (64 a wave at once, XENT_JOIN_BATCH of those under way).  One wave for up to 64, and
// for up to 512 where rows alone fill the CUs (2000 rows of 10 splits of d = 128: 8 us, with four waves 10); four take up to 2048 (100 rows of
// 16 splits of d = 128: 5.4 us against 7.7 with one; 1203 rows of 25 splits of d = 217: 10 us against 15 with eight, fewer rows at once); else
// 8, or 16 where there are not rows for every CU (229 splits of d = 208: 58 rows 12 us against 18; 512 rows of 64 splits 16 us against
// 11).  One wave anyway where rows are many (4608 rows of 14 splits of d = 192: eight waves 42 us).
template <int MODE>
void join_launch(bool bf16, XentJoin j, hipStream_t s) {
  j.lanes = 1;
  while (MODE != XENT_MODE_LSE && 4 * j.lanes < j.d) j.lanes *= 2;
  const int64_t loads = (int64_t)j.n_split * j.lanes, wave = 64 * XENT_JOIN_BATCH;
  if (loads <= 64 || j.ny > 2048 || (loads <= wave && j.ny > 1024)) join_launch<MODE, 1>(bf16, j, s);
  else if (loads <= 4 * wave) join_launch<MODE, 4>(bf16, j, s);
  else if (j.ny > 256) join_launch<MODE, 8>(bf16, j, s);
  else join_launch<MODE, 16>(bf16, j, s);
}

// sizes alone: what the workspace depends on
int xent_check_sizes(const gqe_xent_args* a) {
  if (!a) return refuse(GQE_ERR_ARG, "softmax_xent: args is NULL");
  if (a->phase < 1 || a->phase > 7) return refuse(GQE_ERR_ARG, "softmax_xent: phase %d", a->phase);
  if (a->dtype != GQE_F32 && a->dtype != GQE_BF16) return refuse(GQE_ERR_ARG, "softmax_xent: dtype %d is neither float32 nor bfloat16", a->dtype);
  if (a->dim < 1 || a->dim > GQE_MAX_DIM) return refuse(GQE_ERR_ARG, "softmax_xent: dim %d is not in 1 .. %d", a->dim, GQE_MAX_DIM);
  if (a->n_rows < 1 || a->n_rows > 0x7fffff00LL) return refuse(GQE_ERR_ARG, "softmax_xent: a table of %lld rows", (long long)a->n_rows);
  if (a->n_queries < 0 || a->n_queries > 0x7fffff00LL) return refuse(GQE_ERR_ARG, "softmax_xent: %lld queries", (long long)a->n_queries);
  return GQE_OK;
}

}  // namespace

extern "C" {

const char* gqe_ops_last_error(void) { return g_ops_error.c_str(); }

int64_t gqe_softmax_xent_workspace(const gqe_xent_args* a) {
  const int rc = xent_check_sizes(a);
  if (rc) return rc;
  const XentPlan q = xent_plan_queries(a), t = xent_plan_table(a);
  return std::max<int64_t>(256, xent_space(a, q, t).total);
}

int gqe_softmax_xent(const gqe_xent_args* a) {
  int rc = xent_check_sizes(a);
  if (rc) return rc;
  const bool first = a->phase & (GQE_XENT_LOSS | GQE_XENT_DQ), dq = a->phase & GQE_XENT_DQ, dt = a->phase & GQE_XENT_DTABLE;
  const bool bf16 = a->dtype == GQE_BF16;
  const int64_t B = a->n_queries, V = a->n_rows;
  const size_t esize = bf16 ? 2 : 4;
  if (!a->table || (B && (!a->q || !a->target))) return refuse(GQE_ERR_ARG, "softmax_xent: q, table or target is NULL");
  if (dq && B && !a->dq) return refuse(GQE_ERR_ARG, "softmax_xent: dq is NULL");
  if (dt && !a->dtable) return refuse(GQE_ERR_ARG, "softmax_xent: dtable is NULL");
  if (dt && !first && B && !a->stat) return refuse(GQE_ERR_ARG, "softmax_xent: the table's gradient alone needs stat of an earlier call");
  if (a->accumulate && bf16) return refuse(GQE_ERR_ARG, "softmax_xent: accumulate needs a float32 table");
  if (!isfinite(a->scale)) return refuse(GQE_ERR_ARG, "softmax_xent: scale is not finite");
  if (a->table_stride < a->dim || (B > 1 && a->q_stride < a->dim) || (dt && a->dtable_stride < a->dim) || (dq && B > 1 && a->dq_stride < a->dim))
    return refuse(GQE_ERR_ARG, "softmax_xent: a row stride is smaller than dim %d", a->dim);
  if (!aligned(a->q, esize) || !aligned(a->table, esize) || !aligned(a->dq, a->dq_f32 ? 4 : esize) || !aligned(a->dtable, esize))
    return refuse(GQE_ERR_ARG, "softmax_xent: a pointer is not aligned to its element");
  const XentPlan pq = xent_plan_queries(a), pt = xent_plan_table(a);
  const XentSpace sp = xent_space(a, pq, pt);
  if (a->workspace_bytes < sp.total || (sp.total && (!a->workspace || !aligned(a->workspace, 256))))
    return refuse(GQE_ERR_WORKSPACE, "softmax_xent: needs %lld workspace bytes, 256-byte aligned; got %lld", (long long)sp.total, (long long)a->workspace_bytes);
  if ((dq && B && (a->dq == a->q || a->dq == a->table)) || (dt && (a->dtable == a->table || a->dtable == a->q)))
    return refuse(GQE_ERR_ARG, "softmax_xent: a gradient shares memory with q or table");      // later launches still read both
  OnDevice dev(a->device);
  if (dev.status != hipSuccess) return hip_refuse(dev.status, "softmax_xent");
  hipStream_t stream = (hipStream_t)a->stream;
  char* w = (char*)a->workspace;

  XentPass p = {};
  p.d = a->dim;
  p.pitch = (int32_t)up(a->dim, 4);
  p.scale2 = (float)((double)a->scale * 1.4426950408889634);
  p.scale = a->scale;
  p.target = a->target;
  p.part_m = (float*)(w + sp.part_m);
  p.part_l = (float*)(w + sp.part_l);
  p.part_o = (float*)(w + sp.part_o);
  p.st = (float*)(w + sp.st);
  float* stat = a->stat ? a->stat : (float*)(w + sp.stat);
  p.stat = stat;
  XentJoin j = {};
  j.part_m = p.part_m; j.part_l = p.part_l; j.part_o = p.part_o; j.st = p.st;
  j.d = a->dim; j.pitch = p.pitch; j.n_rows = (int32_t)V; j.target = a->target; j.weight = a->weight;
  j.table = a->table; j.table_stride = a->table_stride; j.unit = a->normalize ? 1 : 0; j.scale = a->scale;
  const bool unit = a->normalize != 0, dma = xent_prepares(a);
  const char* image[2] = {};
  const float2* fac[2] = {};
  int64_t stride[2] = {};
  p.unit = unit;
  if (dma) {
    XentPrep r = {};
    const void* rows[2] = {a->q, a->table};
    const int64_t n[2] = {B, V}, st[2] = {a->q_stride, a->table_stride};
    for (int i = 0; i < 2; ++i) {
      r.r[i] = XentRows{rows[i], st[i], (int32_t)n[i], a->dim};
      r.fac[i] = (float2*)(w + sp.fac[i]);
      r.tiles[i] = (int32_t)((n[i] + XENT_TR - 1) / XENT_TR);
      fac[i] = r.fac[i];
      if (xent_as_is(bf16, pq.dk, a->dim, rows[i], st[i])) {
        image[i] = (const char*)rows[i];
        stride[i] = st[i];
      } else {
        image[i] = r.image[i] = w + sp.image[i];
      }
    }
    r.rec = first ? (XentRec*)(w + sp.rec) : nullptr;
    const hipError_t e = xent_prep(bf16, pq.dk, unit, r, stream);
    if (e != hipSuccess) return hip_refuse(e, "softmax_xent");
  }
  if (first && B) {
    p.y = a->q; p.y_stride = a->q_stride; p.ny = (int32_t)B;
    p.x = a->table; p.x_stride = a->table_stride; p.nx = (int32_t)V;
    p.n_tiles = pq.n_tiles; p.tiles_per_split = pq.per; p.n_split = pq.n_split; p.n_yblk = pq.n_yblk;
    if (dma) {
      p.y_image = image[0]; p.y_fac = fac[0]; p.y_stride = stride[0];
      p.x_image = image[1]; p.x_rec = (const XentRec*)(w + sp.rec); p.x_stride = stride[1];
    }
    hipError_t e = xent_launch(bf16, pq.dk, dq ? XENT_MODE_DQ : XENT_MODE_LSE, unit, dma, p, stream);
    if (e != hipSuccess) return hip_refuse(e, "softmax_xent");
    j.n_split = pq.n_split; j.ny = (int32_t)B;
    j.loss = a->loss; j.lse = a->lse; j.stat = stat;
    j.out = a->dq; j.out_stride = a->dq_stride; j.out_f32 = a->dq_f32 || !bf16;
    if (dma && dt) {
      j.rec = (XentRec*)(w + sp.rec); j.fac = fac[0]; j.scale2 = p.scale2;
    }
    if (dq) join_launch<XENT_MODE_DQ>(bf16, j, stream);
    else join_launch<XENT_MODE_LSE>(bf16, j, stream);
    if ((e = hipGetLastError()) != hipSuccess) return hip_refuse(e, "softmax_xent");
  }
  if (dt) {
    p.y = a->table; p.y_stride = a->table_stride; p.ny = (int32_t)V;
    p.x = a->q; p.x_stride = a->q_stride; p.nx = (int32_t)B;
    p.weight = a->weight;
    p.n_tiles = pt.n_tiles; p.tiles_per_split = pt.per; p.n_split = pt.n_split; p.n_yblk = pt.n_yblk;
    p.out = a->dtable; p.out_stride = a->dtable_stride; p.accumulate = a->accumulate;
    if (dma) {
      p.y_image = image[1]; p.y_fac = fac[1]; p.y_stride = stride[1];
      p.x_image = image[0]; p.x_rec = (const XentRec*)(w + sp.rec); p.x_stride = stride[0];
      if (!first) {
        XentRecs r = {(XentRec*)(w + sp.rec), fac[0], a->target, a->weight, stat, p.scale2, (int32_t)B, (int32_t)V, bf16};
        const hipError_t e = gqe_xent_recs(r, stream);
        if (e != hipSuccess) return hip_refuse(e, "softmax_xent");
      }
    }
    hipError_t e = xent_launch(bf16, pt.dk, XENT_MODE_DT, unit, dma, p, stream);
    if (e != hipSuccess) return hip_refuse(e, "softmax_xent");
    if (pt.n_split > 1) {
      j.n_split = pt.n_split; j.ny = (int32_t)V;
      j.out = a->dtable; j.out_stride = a->dtable_stride; j.out_f32 = !bf16; j.accumulate = a->accumulate;
      join_launch<XENT_MODE_DT>(bf16, j, stream);
      if ((e = hipGetLastError()) != hipSuccess) return hip_refuse(e, "softmax_xent");
    }
  }
  return GQE_OK;
}

}  // extern "C"

#include "gqe_clip.h"
#include "gqe_layer_norm.h"
#include "gqe_chain.h"
