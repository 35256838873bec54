// gqe_layer_norm.h — layer normalisation, forward and backward (include/gqe_ops.h).
//
// Bound by memory: x is read and y written once; backward reads x and dy and writes dx once.  A row stays in the registers of G
// threads (a part of a wave, a wave, or a workgroup), EPL elements each in 16-byte pieces, so mean and variance are two passes
// over registers (no cancellation) and nothing is read twice.  The weight's and bias's gradients are column sums: each thread
// keeps its columns' sums over the rows its group takes, a workgroup adds its groups and writes one row of partial sums, a second
// launch adds the workgroups' rows in order (no atomics: the same bits every time).  500000 x 256 float32: forward 225 us (4.6 TB/s; with the
// next row under way while one is summed, 2048 workgroups: the same), backward 290 us (5.3 TB/s) + 5 us of column sums, where a copy of
// that size reaches 4.8 TB/s; 512 x 128: 3.0 + 3.5 us, launches.
#ifndef GQE_LAYER_NORM_H
#define GQE_LAYER_NORM_H

#define LN_MAX_DIM 16384
#define LN_BLOCKS 1024         // workgroups of the backward launch, = rows of partial sums
#define LN_STREAM (64LL << 20)    // bytes of an output from which it is written past the caches: 154 MB forward 76 -> 60 us, backward 89 -> 69; 512 MB 247 -> 240 and
                               // 299 -> 275; 55 MB the same (and there whoever reads it next finds it)
#define LN_FEW 2048            // rows up to which weight's and bias's gradients need no launch of their own (2048 x 128: 6.4 us against 3.9 + 3.0, and
                               // 4 us less of the host's time; 4609 x 257: 20 us against 9 + 5)

struct LnPass {
  const void *x, *dy;
  void *y, *dx;
  int64_t x_stride, y_stride, dy_stride, dx_stride, n;
  const float *weight, *bias;
  float *mean, *rstd;
  float* partial;              // [blocks][2][d]
  float *dweight, *dbias;      // few rows: written by the backward launch itself
  float eps;
  int32_t d, row_blocks, accumulate, stream;
};

// N = 16 bytes of elements at any element's alignment (the memory path takes unaligned vectors), the row's end guarded
template <bool BF16, int N>
__device__ __forceinline__ void ln_load(const void* row, int col, int d, float* v) {
  if (BF16) {
    const uint16_t* p = (const uint16_t*)row + col;
    if (col + N <= d) {
      uint32_t u[N / 2];
      __builtin_memcpy(u, p, 2 * N);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) { v[2 * i] = bf16_lo(u[i]); v[2 * i + 1] = bf16_hi(u[i]); }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = col + i < d ? __uint_as_float((uint32_t)p[i] << 16) : 0.f;
    }
  } else {
    const float* p = (const float*)row + col;
    if (col + N <= d) {
      __builtin_memcpy(v, p, 4 * N);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = col + i < d ? p[i] : 0.f;
    }
  }
}
// STREAM: past the caches (LnPass::stream)
typedef uint32_t ln_u4 __attribute__((ext_vector_type(4), aligned(2)));
template <bool BF16, int N, bool STREAM = false>
__device__ __forceinline__ void ln_store(void* row, int col, int d, const float* v) {
  if (BF16) {
    uint16_t* p = (uint16_t*)row + col;
    uint32_t u[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) u[i] = xent_pack_bf16(v[2 * i], v[2 * i + 1]);
    if (STREAM && col + N <= d) {
      __builtin_nontemporal_store((ln_u4){u[0], u[1], u[2], u[3]}, (ln_u4*)p);
    } else if (col + N <= d) {
      __builtin_memcpy(p, u, 2 * N);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col + i < d) p[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
  } else {
    float* p = (float*)row + col;
    if (STREAM && col + N <= d) {
      __builtin_nontemporal_store((ln_u4){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}, (ln_u4*)p);
    } else if (col + N <= d) {
      __builtin_memcpy(p, v, 4 * N);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col + i < d) p[i] = v[i];
    }
  }
}

// sums of a and b over the G threads of a row
template <int G>
__device__ __forceinline__ void ln_sum2(float& a, float& b, float (*lds)[2]) {
  if (G >= 64) { a = lane_sum<32>(a); b = lane_sum<32>(b); }
  if (G >= 32) { a = lane_sum<16>(a); b = lane_sum<16>(b); }
  if (G >= 16) { a = lane_sum<8>(a); b = lane_sum<8>(b); }
  if (G >= 16) { a = lane_sum<4>(a); b = lane_sum<4>(b); }
  else { a += __shfl_xor(a, 4); b += __shfl_xor(b, 4); }      // lanes 8 apart are another row's
  a = lane_sum<1>(lane_sum<2>(a));
  b = lane_sum<1>(lane_sum<2>(b));
  if (G > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();                       // the sums before these have been read
    if ((threadIdx.x & 63) == 0) { lds[wave][0] = a; lds[wave][1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) { a += lds[w][0]; b += lds[w][1]; }
  }
}

#define LN_THREADS(G) ((G) > 256 ? (G) : 256)

template <bool BF16, int EPL, int G>
__global__ __launch_bounds__(LN_THREADS(G)) void gqe_layer_norm_fwd_kernel(LnPass p) {
  constexpr int N = BF16 ? 8 : 4, C = EPL / N, GROUPS = LN_THREADS(G) / G;
  __shared__ float lds[G > 64 ? G / 64 : 1][2];
  const int g = threadIdx.x / G, t = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * GROUPS + g;
  if (row >= p.n) return;
  float x[C][N];
  const char* xr = (const char*)p.x + row * p.x_stride * (BF16 ? 2 : 4);
#pragma unroll
  for (int c = 0; c < C; ++c) ln_load<BF16, N>(xr, (c * G + t) * N, p.d, x[c]);
  float s = 0.f, z = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) s += x[c][i];
  ln_sum2<G>(s, z, lds);
  const float mean = s / (float)p.d;
  float v = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[c][i] = (c * G + t) * N + i < p.d ? x[c][i] - mean : 0.f;
      v = fmaf(x[c][i], x[c][i], v);
    }
  ln_sum2<G>(v, z, lds);
  const float rstd = 1.f / sqrtf(v / (float)p.d + p.eps);
  if (t == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  char* yr = (char*)p.y + row * p.y_stride * (BF16 ? 2 : 4);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * G + t) * N;
    float w[N], b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { w[i] = 1.f; b[i] = 0.f; }
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if (p.weight) ln_load<false, 4>(p.weight, col + i, p.d, w + i);
      if (p.bias) ln_load<false, 4>(p.bias, col + i, p.d, b + i);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[c][i] = fmaf(x[c][i] * rstd, w[i], b[i]);
    if (p.stream) ln_store<BF16, N, true>(yr, col, p.d, x[c]);
    else ln_store<BF16, N>(yr, col, p.d, x[c]);
  }
}

// Few rows: the gradients of weight and bias in the same launch, by workgroups of their own behind the rows' (8 columns of all rows each,
// a share of the rows a thread, shares added in order).
template <bool BF16, int THREADS>
__device__ __forceinline__ void ln_columns(const LnPass& p, int block) {
  constexpr int SHARES = THREADS / 8;
  __shared__ float lds[2][SHARES][9];
  const int j = threadIdx.x & 7, k = threadIdx.x >> 3, col = block * 8 + j;
  float dw = 0.f, db = 0.f;
  if (col < p.d) {
#pragma unroll 16
    for (int row = k; row < (int)p.n; row += SHARES) {
      const float x = row_elem<BF16>(p.x, row * p.x_stride + col), dy = row_elem<BF16>(p.dy, row * p.dy_stride + col);
      dw = fmaf(dy, (x - p.mean[row]) * p.rstd[row], dw);
      db += dy;
    }
  }
  lds[0][k][j] = dw;
  lds[1][k][j] = db;
  __syncthreads();
  if (k > 1 || col >= p.d) return;
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < SHARES; ++i) s += lds[k][i][j];
  float* out = k ? p.dbias : p.dweight;
  if (out) out[col] = p.accumulate ? out[col] + s : s;
}

template <bool BF16, int EPL, int G>
__global__ __launch_bounds__(LN_THREADS(G)) void gqe_layer_norm_bwd_kernel(LnPass p) {
  constexpr int N = BF16 ? 8 : 4, C = EPL / N, THREADS = LN_THREADS(G), GROUPS = THREADS / G;
  if ((int)blockIdx.x >= p.row_blocks) return ln_columns<BF16, THREADS>(p, (int)blockIdx.x - p.row_blocks);
  __shared__ float lds[G > 64 ? G / 64 : 1][2];
  __shared__ float cols[GROUPS > 1 ? THREADS * EPL : 1];
  const int g = threadIdx.x / G, t = threadIdx.x % G;
  float w[C][N], dw[C][N], db[C][N];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) { w[c][i] = 1.f; dw[c][i] = 0.f; db[c][i] = 0.f; }
  if (p.weight) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; i += 4) ln_load<false, 4>(p.weight, (c * G + t) * N + i, p.d, w[c] + i);
  }
  const float over = 1.f / (float)p.d;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + g; row < p.n; row += (int64_t)p.row_blocks * GROUPS) {
    float x[C][N], dy[C][N];
    const char* xr = (const char*)p.x + row * p.x_stride * (BF16 ? 2 : 4);
    const char* gr = (const char*)p.dy + row * p.dy_stride * (BF16 ? 2 : 4);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      ln_load<BF16, N>(xr, (c * G + t) * N, p.d, x[c]);
      ln_load<BF16, N>(gr, (c * G + t) * N, p.d, dy[c]);
    }
    const float mean = p.mean[row], rstd = p.rstd[row];
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[c][i] = (c * G + t) * N + i < p.d ? (x[c][i] - mean) * rstd : 0.f;      // xhat; past the end it could overflow and meet dy = 0
        dw[c][i] = fmaf(dy[c][i], x[c][i], dw[c][i]);
        db[c][i] += dy[c][i];
        dy[c][i] *= w[c][i];
        a += dy[c][i];
        b = fmaf(dy[c][i], x[c][i], b);
      }
    if (p.dx) {
      ln_sum2<G>(a, b, lds);
      a *= over;
      b *= over;
      char* out = (char*)p.dx + row * p.dx_stride * (BF16 ? 2 : 4);
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < N; ++i) dy[c][i] = rstd * (dy[c][i] - a - x[c][i] * b);
        if (p.stream) ln_store<BF16, N, true>(out, (c * G + t) * N, p.d, dy[c]);
        else ln_store<BF16, N>(out, (c * G + t) * N, p.d, dy[c]);
      }
    }
  }
  if (!p.partial) return;
  float* out = p.partial + (int64_t)blockIdx.x * 2 * p.d;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) cols[g * (G * EPL) + (c * G + t) * N + i] = which ? db[c][i] : dw[c][i];
      __syncthreads();
      for (int j = threadIdx.x; j < p.d; j += THREADS) {
        float s = 0.f;
#pragma unroll 4
        for (int k = 0; k < GROUPS; ++k) s += cols[k * (G * EPL) + j];
        out[which * p.d + j] = s;
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) ln_store<false, 4>(out + which * p.d, (c * G + t) * N, p.d, which ? db[c] : dw[c]);
      if (N == 8) {
#pragma unroll
        for (int c = 0; c < C; ++c) ln_store<false, 4>(out + which * p.d, (c * G + t) * N + 4, p.d, (which ? db[c] : dw[c]) + 4);
      }
    }
  }
}

// Column sums of the workgroups' rows: 8 columns x 32 row shares per workgroup, every share's rows in order, then the shares in order.
__global__ __launch_bounds__(256) void gqe_layer_norm_cols_kernel(const float* partial, int blocks, int d, float* dweight, float* dbias, int accumulate) {
  __shared__ float lds[32][9];
  const int j = threadIdx.x & 7, k = threadIdx.x >> 3;
  const int col = blockIdx.x * 8 + j;
  float s = 0.f;
  if (col < 2 * d) {
#pragma unroll 8
    for (int b = k; b < blocks; b += 32) s += partial[(int64_t)b * 2 * d + col];
  }
  lds[k][j] = s;
  __syncthreads();
  if (k == 0 && col < 2 * d) {
    s = 0.f;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) s += lds[i][j];
    float* out = col < d ? dweight : dbias;
    if (out) {
      out += col < d ? col : col - d;
      *out = accumulate ? *out + s : s;
    }
  }
}

namespace {

int ln_check(const gqe_layer_norm_args* a, bool backward) {
  const char* who = backward ? "layer_norm backward" : "layer_norm";
  if (!a) return refuse(GQE_ERR_ARG, "%s: args is NULL", who);
  if (a->dtype != GQE_F32 && a->dtype != GQE_BF16) return refuse(GQE_ERR_ARG, "%s: dtype %d is neither float32 nor bfloat16", who, a->dtype);
  if (a->dim < 1 || a->dim > LN_MAX_DIM) return refuse(GQE_ERR_ARG, "%s: dim %d is not in 1 .. %d", who, a->dim, LN_MAX_DIM);
  if (a->n_rows < 0 || a->n_rows > 0x7fffff00LL) return refuse(GQE_ERR_ARG, "%s: %lld rows", who, (long long)a->n_rows);
  if (a->n_rows == 0) return GQE_OK;
  const size_t e = a->dtype == GQE_BF16 ? 2 : 4;
  if (!a->x || !a->mean || !a->rstd) return refuse(GQE_ERR_ARG, "%s: x, mean or rstd is NULL", who);
  if (backward ? !a->dy : !a->y) return refuse(GQE_ERR_ARG, "%s: %s is NULL", who, backward ? "dy" : "y");
  if (!aligned(a->x, e) || !aligned(a->y, e) || !aligned(a->dy, e) || !aligned(a->dx, e)) return refuse(GQE_ERR_ARG, "%s: a pointer is not aligned to its element", who);
  if (a->n_rows > 1 && (a->x_stride < a->dim || (backward ? a->dy_stride < a->dim || (a->dx && a->dx_stride < a->dim) : a->y_stride < a->dim)))
    return refuse(GQE_ERR_ARG, "%s: a row stride is smaller than dim %d", who, a->dim);
  if (!backward && !(a->eps >= 0.f)) return refuse(GQE_ERR_ARG, "layer_norm: eps is negative or NaN");
  return GQE_OK;
}

struct LnShape {
  int epl, g, groups;
};
LnShape ln_shape(bool bf16, int d) {
  const int n = bf16 ? 8 : 4;
  LnShape s;
  if (d <= 64 * n) {
    s.epl = n;
    s.g = 8;
    while (s.g * n < d) s.g *= 2;
  } else {
    s.g = d <= 1024 ? 64 : d <= 4096 ? 256 : 1024;
    s.epl = !bf16 && d <= 512 ? 8 : 16;
  }
  s.groups = LN_THREADS(s.g) / s.g;
  return s;
}
int ln_blocks(const LnShape& s, int64_t n) { return (int)std::min<int64_t>(std::max<int64_t>((n + s.groups - 1) / s.groups, 1), LN_BLOCKS); }

template <bool BF16, int EPL, int G>
void ln_launch(const LnPass& p, bool backward, int blocks, hipStream_t s) {
  if (backward) gqe_layer_norm_bwd_kernel<BF16, EPL, G><<<dim3(blocks), dim3(LN_THREADS(G)), 0, s>>>(p);
  else gqe_layer_norm_fwd_kernel<BF16, EPL, G><<<dim3(blocks), dim3(LN_THREADS(G)), 0, s>>>(p);
}
void ln_dispatch(bool bf16, const LnShape& q, const LnPass& p, bool backward, int blocks, hipStream_t s) {
  if (bf16) {
    if (q.epl == 8 && q.g == 8) return ln_launch<true, 8, 8>(p, backward, blocks, s);
    if (q.epl == 8 && q.g == 16) return ln_launch<true, 8, 16>(p, backward, blocks, s);
    if (q.epl == 8 && q.g == 32) return ln_launch<true, 8, 32>(p, backward, blocks, s);
    if (q.epl == 8) return ln_launch<true, 8, 64>(p, backward, blocks, s);
    if (q.g == 64) return ln_launch<true, 16, 64>(p, backward, blocks, s);
    if (q.g == 256) return ln_launch<true, 16, 256>(p, backward, blocks, s);
    return ln_launch<true, 16, 1024>(p, backward, blocks, s);
  }
  if (q.epl == 4 && q.g == 8) return ln_launch<false, 4, 8>(p, backward, blocks, s);
  if (q.epl == 4 && q.g == 16) return ln_launch<false, 4, 16>(p, backward, blocks, s);
  if (q.epl == 4 && q.g == 32) return ln_launch<false, 4, 32>(p, backward, blocks, s);
  if (q.epl == 4) return ln_launch<false, 4, 64>(p, backward, blocks, s);
  if (q.epl == 8) return ln_launch<false, 8, 64>(p, backward, blocks, s);
  if (q.g == 64) return ln_launch<false, 16, 64>(p, backward, blocks, s);
  if (q.g == 256) return ln_launch<false, 16, 256>(p, backward, blocks, s);
  return ln_launch<false, 16, 1024>(p, backward, blocks, s);
}

LnPass ln_pass(const gqe_layer_norm_args* a) {
  LnPass p = {};
  p.x = a->x; p.dy = a->dy; p.y = a->y; p.dx = a->dx;
  p.x_stride = a->x_stride; p.y_stride = a->y_stride; p.dy_stride = a->dy_stride; p.dx_stride = a->dx_stride;
  p.n = a->n_rows; p.weight = a->weight; p.bias = a->bias; p.mean = a->mean; p.rstd = a->rstd; p.eps = a->eps; p.d = a->dim;
  p.stream = a->n_rows * a->dim * (a->dtype == GQE_BF16 ? 2 : 4) > LN_STREAM;
  p.dweight = a->dweight; p.dbias = a->dbias; p.accumulate = a->accumulate;
  return p;
}

}  // namespace

extern "C" {

int64_t gqe_layer_norm_workspace(const gqe_layer_norm_args* a) {
  if (!a) return refuse(GQE_ERR_ARG, "layer_norm: args is NULL");
  if ((a->dtype != GQE_F32 && a->dtype != GQE_BF16) || a->dim < 1 || a->dim > LN_MAX_DIM || a->n_rows < 0)
    return refuse(GQE_ERR_ARG, "layer_norm: dtype %d, dim %d, %lld rows", a->dtype, a->dim, (long long)a->n_rows);
  return a->n_rows <= LN_FEW ? 0 : (int64_t)ln_blocks(ln_shape(a->dtype == GQE_BF16, a->dim), a->n_rows) * 2 * a->dim * 4;
}

int gqe_layer_norm_forward(const gqe_layer_norm_args* a) {
  const int rc = ln_check(a, false);
  if (rc || a->n_rows == 0) return rc;
  OnDevice dev(a->device);
  if (dev.status != hipSuccess) return hip_refuse(dev.status, "layer_norm");
  const LnShape s = ln_shape(a->dtype == GQE_BF16, a->dim);
  ln_dispatch(a->dtype == GQE_BF16, s, ln_pass(a), false, (int)((a->n_rows + s.groups - 1) / s.groups), (hipStream_t)a->stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GQE_OK : hip_refuse(e, "layer_norm");
}

int gqe_layer_norm_backward(const gqe_layer_norm_args* a) {
  const int rc = ln_check(a, true);
  if (rc) return rc;
  const bool cols = a->dweight || a->dbias;
  if (!a->dx && !cols) return GQE_OK;
  const LnShape s = ln_shape(a->dtype == GQE_BF16, a->dim);
  const int blocks = ln_blocks(s, a->n_rows);
  const int64_t need = cols ? gqe_layer_norm_workspace(a) : 0;
  if (need && (a->workspace_bytes < need || !a->workspace || !aligned(a->workspace, 16)))
    return refuse(GQE_ERR_WORKSPACE, "layer_norm backward: needs %lld workspace bytes, 16-byte aligned; got %lld", (long long)need,
                  (long long)a->workspace_bytes);
  if (a->dx && (a->dx == a->x || a->dx == a->dy)) return refuse(GQE_ERR_ARG, "layer_norm backward: dx shares memory with x or dy");
  OnDevice dev(a->device);
  if (dev.status != hipSuccess) return hip_refuse(dev.status, "layer_norm backward");
  LnPass p = ln_pass(a);
  p.row_blocks = a->dx || need ? blocks : 0;
  p.partial = need ? (float*)a->workspace : nullptr;
  const int extra = cols && !need ? (a->dim + 7) / 8 : 0;
  ln_dispatch(a->dtype == GQE_BF16, s, p, true, p.row_blocks + extra, (hipStream_t)a->stream);
  if (need) gqe_layer_norm_cols_kernel<<<dim3((2 * a->dim + 7) / 8), dim3(256), 0, (hipStream_t)a->stream>>>(p.partial, blocks, a->dim, a->dweight, a->dbias, a->accumulate);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GQE_OK : hip_refuse(e, "layer_norm backward");
}

}  // extern "C"

#endif
