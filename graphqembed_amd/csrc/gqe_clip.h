// gqe_clip.h — global gradient norm over many tensors, and clipping (include/gqe_ops.h).
//
// Two launches: every workgroup writes the 64-bit sum of squares of its share; every workgroup of the second adds those (at most
// CLIP_BLOCKS for each CLIP_TENSORS tensors) in the same order, has the norm without another launch, and scales its share.  The
// tensors' descriptors travel in the kernel arguments: no upload, nothing to keep.  Squares are summed in 64 bits: a float32
// gradient's square neither overflows nor vanishes there, and the 64-bit multiply-adds stay far below the rate memory delivers at.
// Bound by memory: 462 MB of bfloat16 are read in 97 us (4.8 TB/s) and scaled in 141 us (6.5 TB/s, part of them still cached: the second launch
// goes backwards through the chunks); 50 MB of float32 in 29 us for both, the caches' rate.
#ifndef GQE_CLIP_H
#define GQE_CLIP_H

#define CLIP_TENSORS 96
#define CLIP_BLOCKS 1024
#define CLIP_THREADS 256
#define CLIP_CHUNK 32768       // bytes of a tensor that a workgroup takes at a time: 8 vectors a thread

struct ClipGroup {
  void* data[CLIP_TENSORS];
  int64_t numel[CLIP_TENSORS];
  int32_t chunk0[CLIP_TENSORS + 1];    // first chunk of each tensor
  uint8_t bf16[CLIP_TENSORS];
  int32_t n;
  double* partial;             // this group's CLIP_BLOCKS sums
};

struct ClipScale {
  const double* partial;       // all groups' sums
  int32_t n_partial;
  float max_norm;
  float* norm;
};

// the tensor that chunk c belongs to
__device__ __forceinline__ int clip_find(const ClipGroup& g, int c) {
  int lo = 0, hi = g.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (g.chunk0[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double clip_block_sum(double x, double* lds) {
  x = wave_total(x);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[wave] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_THREADS / 64; ++w) s += lds[w];
  return s;
}

// Chunk c of a tensor: bytes [c CLIP_CHUNK, (c + 1) CLIP_CHUNK) counted from the 16-byte boundary below its first element, so that
// vectors are aligned wherever the tensor starts; elements in front of it or behind it are left out of the first / last vector.
template <bool BF16, typename F>
__device__ __forceinline__ void clip_chunk(void* data, int64_t numel, int64_t c, F&& each) {
  constexpr int E = BF16 ? 2 : 4, N = 16 / E;
  const uintptr_t a = (uintptr_t)data & ~(uintptr_t)15;
  const int64_t skip = ((uintptr_t)data - a) / E, end = skip + numel;
  const int64_t v0 = c * (CLIP_CHUNK / 16);
  uint4* base = (uint4*)a;
  uint4 u[CLIP_CHUNK / 16 / CLIP_THREADS];
  const bool whole = v0 * N >= skip && (v0 + CLIP_CHUNK / 16) * N <= end;
  if (whole) {
#pragma unroll
    for (int k = 0; k < CLIP_CHUNK / 16 / CLIP_THREADS; ++k) u[k] = base[v0 + k * CLIP_THREADS + threadIdx.x];
#pragma unroll
    for (int k = 0; k < CLIP_CHUNK / 16 / CLIP_THREADS; ++k) each(u[k], base + v0 + k * CLIP_THREADS + threadIdx.x);
    return;
  }
  for (int k = 0; k < CLIP_CHUNK / 16 / CLIP_THREADS; ++k) {
    const int64_t v = v0 + k * CLIP_THREADS + threadIdx.x;
    if (v * N >= skip && (v + 1) * N <= end) {
      each(base[v], base + v);
    } else if ((v + 1) * N > skip && v * N < end) {
      for (int64_t i = v * N < skip ? skip : v * N; i < (v + 1) * N && i < end; ++i) each.one((char*)a + i * E);
    }
  }
}

template <bool BF16>
struct ClipSquares {
  double s0 = 0.0, s1 = 0.0;
  __device__ __forceinline__ void add(float a, float b) {
    s0 = fma((double)a, (double)a, s0);
    s1 = fma((double)b, (double)b, s1);
  }
  __device__ __forceinline__ void operator()(const uint4& u, uint4*) {
    if (BF16) {
      add(bf16_lo(u.x), bf16_hi(u.x)); add(bf16_lo(u.y), bf16_hi(u.y)); add(bf16_lo(u.z), bf16_hi(u.z)); add(bf16_lo(u.w), bf16_hi(u.w));
    } else {
      add(__uint_as_float(u.x), __uint_as_float(u.y)); add(__uint_as_float(u.z), __uint_as_float(u.w));
    }
  }
  __device__ __forceinline__ void one(const void* p) { add(BF16 ? __uint_as_float((uint32_t) * (const uint16_t*)p << 16) : *(const float*)p, 0.f); }
};

template <bool BF16>
struct ClipTimes {
  float c;
  __device__ __forceinline__ uint32_t two(uint32_t u) const { return xent_pack_bf16(bf16_lo(u) * c, bf16_hi(u) * c); }
  __device__ __forceinline__ void operator()(const uint4& u, uint4* p) {
    if (BF16) {
      *p = make_uint4(two(u.x), two(u.y), two(u.z), two(u.w));
    } else {
      *p = make_uint4(__float_as_uint(__uint_as_float(u.x) * c), __float_as_uint(__uint_as_float(u.y) * c), __float_as_uint(__uint_as_float(u.z) * c),
                      __float_as_uint(__uint_as_float(u.w) * c));
    }
  }
  __device__ __forceinline__ void one(void* p) {
    if (BF16) *(uint16_t*)p = (uint16_t)two(*(const uint16_t*)p);
    else *(float*)p *= c;
  }
};

__global__ __launch_bounds__(CLIP_THREADS) void gqe_clip_squares_kernel(ClipGroup g) {
  __shared__ double lds[CLIP_THREADS / 64];
  ClipSquares<false> f;
  ClipSquares<true> b;
  for (int c = blockIdx.x; c < g.chunk0[g.n]; c += gridDim.x) {
    const int t = clip_find(g, c);
    if (g.bf16[t]) clip_chunk<true>(g.data[t], g.numel[t], c - g.chunk0[t], b);
    else clip_chunk<false>(g.data[t], g.numel[t], c - g.chunk0[t], f);
  }
  const double s = clip_block_sum((f.s0 + f.s1) + (b.s0 + b.s1), lds);
  if (threadIdx.x == 0) g.partial[blockIdx.x] = s;
}

__device__ __forceinline__ double clip_norm(const ClipScale& q, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < q.n_partial; i += CLIP_THREADS) s += q.partial[i];
  return sqrt(clip_block_sum(s, lds));
}

__global__ __launch_bounds__(CLIP_THREADS) void gqe_clip_norm_kernel(ClipScale q) {
  __shared__ double lds[CLIP_THREADS / 64];
  const double n = clip_norm(q, lds);
  if (threadIdx.x == 0) *q.norm = (float)n;
}

__global__ __launch_bounds__(CLIP_THREADS) void gqe_clip_scale_kernel(ClipGroup g, ClipScale q) {
  __shared__ double lds[CLIP_THREADS / 64];
  const double n = clip_norm(q, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0) *q.norm = (float)n;
  const double r = (double)q.max_norm / (n + 1e-6);
  if (r >= 1.0) return;
  ClipTimes<false> f;
  ClipTimes<true> b;
  f.c = b.c = (float)r;
  for (int c = g.chunk0[g.n] - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {      // the squares' launch ended here: what it read last may still be cached
    const int t = clip_find(g, c);
    if (g.bf16[t]) clip_chunk<true>(g.data[t], g.numel[t], c - g.chunk0[t], b);
    else clip_chunk<false>(g.data[t], g.numel[t], c - g.chunk0[t], f);
  }
}

// Little to clip: one workgroup does it all.  Whole 16-byte vectors of all tensors in one row (chunk0: first of each tensor), eight a thread, kept
// in registers between the sum and the product; what lies in front of a tensor's first whole vector and behind its last is a thread's each.
// 14 vectors of 63 and two matrices of 63 x 63: 6 us in one launch against 5 + 5 in two, and 3 us less of the host's time.
#define CLIP_FEW 8192          // whole vectors (128 KB)
#define CLIP_FEW_THREADS 1024
struct ClipEnds {              // a tensor's first whole vector, and how many elements are in front of it; whole vectors; elements behind them
  char* first;
  int64_t head, whole, tail;
};
__host__ __device__ __forceinline__ ClipEnds clip_ends(void* data, int64_t numel, bool bf16) {
  const int64_t e = bf16 ? 2 : 4, per = 16 / e;
  ClipEnds r;
  const int64_t gap = (int64_t)((16 - ((uintptr_t)data & 15)) & 15) / e;
  r.head = gap < numel ? gap : numel;
  r.first = (char*)data + r.head * e;
  r.whole = (numel - r.head) / per;
  r.tail = numel - r.head - r.whole * per;
  return r;
}
template <typename T, typename B>
__device__ __forceinline__ void clip_ragged(const ClipGroup& g, T&& each32, B&& each16) {
  for (int i = threadIdx.x; i < 2 * g.n; i += CLIP_FEW_THREADS) {
    const int t = i >> 1;
    const ClipEnds r = clip_ends(g.data[t], g.numel[t], g.bf16[t]);
    const int e = g.bf16[t] ? 2 : 4;
    char* p = i & 1 ? r.first + 16 * r.whole : (char*)g.data[t];
    for (int64_t k = 0, n = i & 1 ? r.tail : r.head; k < n; ++k) {
      if (g.bf16[t]) each16.one(p + e * k);
      else each32.one(p + e * k);
    }
  }
}
__global__ __launch_bounds__(CLIP_FEW_THREADS) void gqe_clip_few_kernel(ClipGroup g, float max_norm, float* norm) {
  constexpr int K = CLIP_FEW / CLIP_FEW_THREADS;
  __shared__ int first[CLIP_TENSORS + 1];
  __shared__ double lds[CLIP_FEW_THREADS / 64];
  if (threadIdx.x <= g.n) first[threadIdx.x] = g.chunk0[threadIdx.x];
  __syncthreads();
  ClipSquares<false> f;
  ClipSquares<true> b;
  uint4 u[K];
  uint4* at[K];
  bool half[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int v = k * CLIP_FEW_THREADS + threadIdx.x;
    at[k] = nullptr;
    if (v >= first[g.n]) continue;
    int lo = 0, hi = g.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= v) lo = mid;
      else hi = mid - 1;
    }
    half[k] = g.bf16[lo];
    at[k] = (uint4*)clip_ends(g.data[lo], g.numel[lo], half[k]).first + (v - first[lo]);
    u[k] = *at[k];
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (at[k]) {
      if (half[k]) b(u[k], at[k]);
      else f(u[k], at[k]);
    }
  clip_ragged(g, f, b);
  const double s = wave_total((f.s0 + f.s1) + (b.s0 + b.s1));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  double n = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_FEW_THREADS / 64; ++w) n += lds[w];
  n = sqrt(n);
  if (threadIdx.x == 0) *norm = (float)n;
  const double r = (double)max_norm / (n + 1e-6);
  if (max_norm < 0.f || r >= 1.0) return;
  ClipTimes<false> tf;
  ClipTimes<true> tb;
  tf.c = tb.c = (float)r;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (at[k]) {
      if (half[k]) tb(u[k], at[k]);
      else tf(u[k], at[k]);
    }
  clip_ragged(g, tf, tb);
}

namespace {

int64_t clip_chunks(const gqe_tensor& t) {
  const int64_t e = t.dtype == GQE_BF16 ? 2 : 4;
  if (t.numel == 0) return 0;
  return (t.numel * e + (int64_t)((uintptr_t)t.data & 15) + CLIP_CHUNK - 1) / CLIP_CHUNK;
}

int clip_check(const gqe_tensor* t, int32_t n) {
  if (n < 0 || (n && !t)) return refuse(GQE_ERR_ARG, "clip_grads: %d tensors", n);
  int64_t chunks = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (t[i].dtype != GQE_F32 && t[i].dtype != GQE_BF16) return refuse(GQE_ERR_ARG, "clip_grads: tensor %d: dtype %d is neither float32 nor bfloat16", i, t[i].dtype);
    if (t[i].numel < 0 || (t[i].numel && !t[i].data)) return refuse(GQE_ERR_ARG, "clip_grads: tensor %d has no data", i);
    if (!aligned(t[i].data, t[i].dtype == GQE_BF16 ? 2 : 4)) return refuse(GQE_ERR_ARG, "clip_grads: tensor %d is not aligned to its element", i);
    if (t[i].numel <= (int64_t)1 << 45) chunks += clip_chunks(t[i]);
    if (t[i].numel > (int64_t)1 << 45 || chunks > 0x3fffffff) return refuse(GQE_ERR_ARG, "clip_grads: too many elements");
  }
  return GQE_OK;
}

// two tensors on the same memory would be counted and scaled twice, at once
int clip_apart(const gqe_tensor* t, int32_t n) {
  struct Span { uintptr_t a, b; int32_t i; };
  std::vector<Span> s;
  s.reserve(n);
  for (int32_t i = 0; i < n; ++i)
    if (t[i].numel) s.push_back({(uintptr_t)t[i].data, (uintptr_t)t[i].data + (uintptr_t)t[i].numel * (t[i].dtype == GQE_BF16 ? 2 : 4), i});
  std::sort(s.begin(), s.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  for (size_t i = 1; i < s.size(); ++i)
    if (s[i].a < s[i - 1].b) return refuse(GQE_ERR_ARG, "clip_grads: tensors %d and %d share memory", s[i - 1].i, s[i].i);
  return GQE_OK;
}

}  // namespace

extern "C" {

int64_t gqe_clip_grads_workspace(const gqe_tensor* tensors, int32_t n) {
  if (n < 0 || (n && !tensors)) return refuse(GQE_ERR_ARG, "clip_grads: %d tensors", n);
  return (int64_t)((std::max(n, 1) + CLIP_TENSORS - 1) / CLIP_TENSORS) * CLIP_BLOCKS * 8;
}

int gqe_clip_grads(int32_t device, const gqe_tensor* tensors, int32_t n, float max_norm, float* norm, void* workspace, int64_t workspace_bytes,
                   void* stream_) {
  int rc = clip_check(tensors, n);
  if (rc) return rc;
  if (!norm || !aligned(norm, 4)) return refuse(GQE_ERR_ARG, "clip_grads: norm is NULL");
  if (max_norm != max_norm) return refuse(GQE_ERR_ARG, "clip_grads: max_norm is NaN");
  const int64_t need = gqe_clip_grads_workspace(tensors, n);
  if (workspace_bytes < need || !workspace || !aligned(workspace, 8))
    return refuse(GQE_ERR_WORKSPACE, "clip_grads: needs %lld workspace bytes, 8-byte aligned; got %lld", (long long)need, (long long)workspace_bytes);
  try {
    if (max_norm >= 0.f && (rc = clip_apart(tensors, n))) return rc;
  } catch (...) {
    return refuse(GQE_ERR_STATE, "clip_grads: out of host memory");
  }
  OnDevice dev(device);
  if (dev.status != hipSuccess) return hip_refuse(dev.status, "clip_grads");
  hipStream_t stream = (hipStream_t)stream_;
  if (n > 0 && n <= CLIP_TENSORS) {
    ClipGroup g;
    int64_t whole = 0;
    g.n = 0;
    for (int32_t i = 0; i < n && whole <= CLIP_FEW; ++i) {
      if (!tensors[i].numel) continue;
      g.data[g.n] = tensors[i].data;
      g.numel[g.n] = tensors[i].numel;
      g.bf16[g.n] = tensors[i].dtype == GQE_BF16;
      g.chunk0[g.n] = (int32_t)whole;
      whole += clip_ends(g.data[g.n], g.numel[g.n], g.bf16[g.n]).whole;
      ++g.n;
    }
    if (whole <= CLIP_FEW && g.n) {
      g.chunk0[g.n] = (int32_t)whole;
      g.partial = nullptr;
      gqe_clip_few_kernel<<<dim3(1), dim3(CLIP_FEW_THREADS), 0, stream>>>(g, max_norm, norm);
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? GQE_OK : hip_refuse(e, "clip_grads");
    }
  }
  ClipScale q = {(const double*)workspace, 0, max_norm, norm};
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1 && (max_norm < 0.f || q.n_partial == 0)) break;
    int32_t i = 0;
    while (i < n) {
      ClipGroup g;
      int32_t k = 0, chunks = 0;
      for (; i < n && k < CLIP_TENSORS; ++i) {
        if (!tensors[i].numel) continue;
        g.data[k] = tensors[i].data;
        g.numel[k] = tensors[i].numel;
        g.bf16[k] = tensors[i].dtype == GQE_BF16;
        g.chunk0[k++] = chunks;
        chunks += (int32_t)clip_chunks(tensors[i]);
      }
      if (!k) break;
      g.chunk0[k] = chunks;
      g.n = k;
      const int blocks = std::min(chunks, CLIP_BLOCKS);
      if (pass == 0) {
        g.partial = (double*)workspace + q.n_partial;
        q.n_partial += blocks;
        gqe_clip_squares_kernel<<<dim3(blocks), dim3(CLIP_THREADS), 0, stream>>>(g);
      } else {
        g.partial = nullptr;
        gqe_clip_scale_kernel<<<dim3(blocks), dim3(CLIP_THREADS), 0, stream>>>(g, q);
      }
    }
  }
  if (max_norm < 0.f || q.n_partial == 0) gqe_clip_norm_kernel<<<dim3(1), dim3(CLIP_THREADS), 0, stream>>>(q);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GQE_OK : hip_refuse(e, "clip_grads");
}

}  // extern "C"

#endif
