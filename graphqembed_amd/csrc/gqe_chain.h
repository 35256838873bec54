// gqe_chain.h — the query side of a bilinear-diag relation chain, forward and backward (include/gqe_ops.h).
//
// q_b = a_b r_1 .. r_k element by element, a_b = the anchor's table row over its length.  One wave per query, one pass over its row.
// Backward: da = dq r_1 .. r_k through the length into the anchor's row, (da - a (a . da)) / |w|; the relations are the batch's, so their
// gradients need one column sum, S = sum_b dq_b a_b, and dr_j = S times the other relations.  Anchors repeat: the first query of a row
// adds up all of that row's gradients in order (a scan over the batch's rows; no atomics, the same bits every time).
// 512 queries of d = 128: four launches of 4 to 5 us; 4608 of d = 256: 5 us forward, 8 + 20 + 10 us backward; the scan is quadratic (65536
// queries: 1.9 ms), nothing next to the products with a whole table that follow.
#ifndef GQE_CHAIN_H
#define GQE_CHAIN_H

#define CHAIN_MAX 65536        // queries of a call: the scan for equal rows is quadratic

struct ChainPass {
  const float *table, *rel[3], *dq;
  const int32_t* rows;
  float *q, *dtable, *drel[3], *da, *c;      // da, c: [n][d] of the workspace
  int64_t table_stride, q_stride, dq_stride, dtable_stride, n_rows;
  int32_t n, d, n_rels;
};

__device__ __forceinline__ void chain_row(const ChainPass& p, int64_t row, int lane, float* a, float& rn) {
  float mx = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    a[c] = lane + 64 * c < p.d ? p.table[row * p.table_stride + lane + 64 * c] : 0.f;
    mx = fmaxf(mx, fabsf(a[c]));
  }
  const float k = xent_pow2(xent_row_scale(wave_max(mx)));
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    a[c] *= k;             // a power of two: no square over- or underflows
    ss = fmaf(a[c], a[c], ss);
  }
  const float g = xent_rsqrt(wave_total(ss));
  rn = fminf(g * k, 3.0e38f);
#pragma unroll
  for (int c = 0; c < 4; ++c) a[c] *= g;
}

__global__ __launch_bounds__(256) void gqe_chain_fwd_kernel(ChainPass p) {
  const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= p.n) return;
  const int row = p.rows[b];
  const bool ok = row >= 0 && row < p.n_rows;
  float a[4] = {NAN, NAN, NAN, NAN}, rn;
  if (ok) chain_row(p, row, lane, a, rn);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int i = lane + 64 * c;
    if (i >= p.d) continue;
    for (int j = 0; j < p.n_rels; ++j) a[c] *= p.rel[j][i];
    p.q[b * p.q_stride + i] = a[c];
  }
}

__global__ __launch_bounds__(256) void gqe_chain_bwd_kernel(ChainPass p) {
  const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= p.n) return;
  const int row = p.rows[b];
  const bool ok = row >= 0 && row < p.n_rows;
  float a[4] = {0.f, 0.f, 0.f, 0.f}, da[4] = {0.f, 0.f, 0.f, 0.f}, rn = 0.f, along = 0.f;
  if (ok) {
    chain_row(p, row, lane, a, rn);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = lane + 64 * c;
      if (i >= p.d) continue;
      const float g = p.dq[b * p.dq_stride + i];
      da[c] = g;
      for (int j = 0; j < p.n_rels; ++j) da[c] *= p.rel[j][i];
      along = fmaf(da[c], a[c], along);
      p.c[(int64_t)b * p.d + i] = g * a[c];
    }
  }
  along = wave_total(along);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int i = lane + 64 * c;
    if (i >= p.d) continue;
    if (!ok) p.c[(int64_t)b * p.d + i] = 0.f;
    p.da[(int64_t)b * p.d + i] = fmaf(-along, a[c], da[c]) * rn;
  }
}

__global__ __launch_bounds__(256) void gqe_chain_rows_kernel(ChainPass p) {
  const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= p.n) return;
  const int row = p.rows[b];
  if (row < 0 || row >= p.n_rows) return;
  for (int k = 0; k < b; k += 64)              // an earlier query has this row: it adds for both
    if (__any(k + lane < b && p.rows[k + lane] == row)) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = b & ~63; k < p.n; k += 64) {
    unsigned long long same = __ballot(k + lane >= b && k + lane < p.n && p.rows[min(k + lane, p.n - 1)] == row);
    while (same) {
      const int64_t o = (int64_t)(k + __builtin_ctzll(same)) * p.d + lane;
      same &= same - 1;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < p.d) s[c] += p.da[o + 64 * c];
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < p.d) p.dtable[row * p.dtable_stride + lane + 64 * c] += s[c];
}

// 32 columns x 32 shares of the batch; shares added in order
__global__ __launch_bounds__(1024) void gqe_chain_rels_kernel(ChainPass p) {
  __shared__ float lds[32][33];
  const int j = threadIdx.x & 31, k = threadIdx.x >> 5, col = blockIdx.x * 32 + j;
  float s = 0.f;
  if (col < p.d) {
#pragma unroll 8
    for (int b = k; b < p.n; b += 32) s += p.c[(int64_t)b * p.d + col];
  }
  lds[k][j] = s;
  __syncthreads();
  if (k || col >= p.d) return;
  s = 0.f;
#pragma unroll 8
  for (int i = 0; i < 32; ++i) s += lds[i][j];
  float r[3];
  for (int i = 0; i < 3; ++i) r[i] = i < p.n_rels ? p.rel[i][col] : 1.f;
  for (int i = 0; i < p.n_rels; ++i) p.drel[i][col] += s * (i == 0 ? r[1] * r[2] : i == 1 ? r[0] * r[2] : r[0] * r[1]);      // the same relation twice: one after the other
}

namespace {

int chain_check(const gqe_chain_args* a, bool backward) {
  const char* who = backward ? "chain_rows backward" : "chain_rows";
  if (!a) return refuse(GQE_ERR_ARG, "%s: args is NULL", who);
  if (a->dim < 1 || a->dim > GQE_MAX_DIM) return refuse(GQE_ERR_ARG, "%s: dim %d is not in 1 .. %d", who, a->dim, GQE_MAX_DIM);
  if (a->n < 0 || a->n > CHAIN_MAX) return refuse(GQE_ERR_ARG, "%s: %lld queries are not in 0 .. %d", who, (long long)a->n, CHAIN_MAX);
  if (a->n_rows < 1 || a->n_rows > 0x7fffff00LL) return refuse(GQE_ERR_ARG, "%s: a table of %lld rows", who, (long long)a->n_rows);
  if (a->n_rels < 0 || a->n_rels > 3) return refuse(GQE_ERR_ARG, "%s: %d relations are not in 0 .. 3", who, a->n_rels);
  for (int j = 0; j < a->n_rels; ++j)
    if (!a->rel[j] || (backward && !a->drel[j])) return refuse(GQE_ERR_ARG, "%s: relation %d is NULL", who, j);
  if (!a->table || (backward && !a->dtable) || (a->n && (!a->rows || (backward ? !a->dq : !a->q)))) return refuse(GQE_ERR_ARG, "%s: a pointer is NULL", who);
  if (a->table_stride < a->dim || (backward && a->dtable_stride < a->dim) || (a->n > 1 && (backward ? a->dq_stride : a->q_stride) < a->dim))
    return refuse(GQE_ERR_ARG, "%s: a row stride is smaller than dim %d", who, a->dim);
  if (backward && a->n && (a->workspace_bytes < 8 * a->n * a->dim || !a->workspace || !aligned(a->workspace, 4)))
    return refuse(GQE_ERR_WORKSPACE, "%s: needs %lld workspace bytes; got %lld", who, (long long)(8 * a->n * a->dim), (long long)a->workspace_bytes);
  if (a->n && (backward ? a->dtable == a->table : a->q == a->table)) return refuse(GQE_ERR_ARG, "%s: the result shares memory with the table", who);
  for (int j = 0; backward && j < a->n_rels; ++j)
    for (int i = 0; i < a->n_rels; ++i)
      if (a->drel[j] == a->rel[i]) return refuse(GQE_ERR_ARG, "%s: gradient %d shares memory with relation %d", who, j, i);
  return GQE_OK;
}

ChainPass chain_pass(const gqe_chain_args* a) {
  ChainPass p = {};
  p.table = a->table; p.table_stride = a->table_stride; p.n_rows = a->n_rows; p.rows = a->rows;
  p.q = a->q; p.q_stride = a->q_stride; p.dq = a->dq; p.dq_stride = a->dq_stride; p.dtable = a->dtable; p.dtable_stride = a->dtable_stride;
  for (int j = 0; j < 3; ++j) { p.rel[j] = a->rel[j]; p.drel[j] = a->drel[j]; }
  p.n = (int32_t)a->n; p.d = a->dim; p.n_rels = a->n_rels;
  p.da = (float*)a->workspace;
  p.c = p.da + a->n * a->dim;
  return p;
}

}  // namespace

extern "C" {

int gqe_chain_rows_forward(const gqe_chain_args* a) {
  const int rc = chain_check(a, false);
  if (rc || a->n == 0) return rc;
  OnDevice dev(a->device);
  if (dev.status != hipSuccess) return hip_refuse(dev.status, "chain_rows");
  const ChainPass p = chain_pass(a);
  gqe_chain_fwd_kernel<<<dim3((p.n + 3) / 4), dim3(256), 0, (hipStream_t)a->stream>>>(p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GQE_OK : hip_refuse(e, "chain_rows");
}

int gqe_chain_rows_backward(const gqe_chain_args* a) {
  const int rc = chain_check(a, true);
  if (rc || a->n == 0) return rc;
  OnDevice dev(a->device);
  if (dev.status != hipSuccess) return hip_refuse(dev.status, "chain_rows backward");
  const ChainPass p = chain_pass(a);
  const hipStream_t s = (hipStream_t)a->stream;
  gqe_chain_bwd_kernel<<<dim3((p.n + 3) / 4), dim3(256), 0, s>>>(p);
  gqe_chain_rows_kernel<<<dim3((p.n + 3) / 4), dim3(256), 0, s>>>(p);
  if (p.n_rels) gqe_chain_rels_kernel<<<dim3((p.d + 31) / 32), dim3(1024), 0, s>>>(p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GQE_OK : hip_refuse(e, "chain_rows backward");
}

}  // extern "C"

#endif
