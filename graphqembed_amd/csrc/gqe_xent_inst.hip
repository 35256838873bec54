// One (type, padded dim) of the softmax cross entropy's kernels per translation unit: -DGQE_XENT_BF16=0|1 -DGQE_XENT_DK=64|128|192|256.
#include <atomic>

#include "gqe_xent.h"
#include "gqe_ops_dev.h"

#define XENT_CAT3(a, b, c, d) a##b##_##c##d
#define XENT_NAME(b, dk) XENT_CAT3(gqe_xent_launch_, b, dk, )

template <int MODE, bool UNIT, bool DMA>
static hipError_t launch(const XentPass& p, hipStream_t stream) {
  typedef XentLds<GQE_XENT_BF16 != 0, GQE_XENT_DK, MODE, DMA> L;
  const void* f = (const void*)gqe_xent_kernel<GQE_XENT_BF16 != 0, GQE_XENT_DK, MODE, UNIT, DMA>;
  if (sizeof(L) > 65536) {            // once per device
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev > 63 || !(done.load() >> dev & 1)) {
      if ((e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(L))) != hipSuccess) return e;
      if (dev <= 63) done.fetch_or((uint64_t)1 << dev);
    }
  }
  gqe_xent_kernel<GQE_XENT_BF16 != 0, GQE_XENT_DK, MODE, UNIT, DMA><<<dim3((unsigned)(p.n_split * p.n_yblk)), dim3(256), sizeof(L), stream>>>(p);
  return hipGetLastError();
}

hipError_t XENT_NAME(GQE_XENT_BF16, GQE_XENT_DK)(int mode, bool unit, bool dma, const XentPass& p, hipStream_t stream) {
  if (dma) {
    if (mode == XENT_MODE_LSE) return launch<XENT_MODE_LSE, false, true>(p, stream);
    if (mode == XENT_MODE_DQ) return launch<XENT_MODE_DQ, false, true>(p, stream);
    return launch<XENT_MODE_DT, false, true>(p, stream);
  }
  if (mode == XENT_MODE_LSE) return unit ? launch<XENT_MODE_LSE, true, false>(p, stream) : launch<XENT_MODE_LSE, false, false>(p, stream);
  if (mode == XENT_MODE_DQ) return unit ? launch<XENT_MODE_DQ, true, false>(p, stream) : launch<XENT_MODE_DQ, false, false>(p, stream);
  return unit ? launch<XENT_MODE_DT, true, false>(p, stream) : launch<XENT_MODE_DT, false, false>(p, stream);
}

#define XENT_PREP_CAT(a, b, c) a##b##_##c
#define XENT_PREP_NAME(b, dk) XENT_PREP_CAT(gqe_xent_prep_, b, dk)
hipError_t XENT_PREP_NAME(GQE_XENT_BF16, GQE_XENT_DK)(bool unit, const XentPrep& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.tiles[0] + p.tiles[1]));
  if (unit) gqe_xent_prep_kernel<GQE_XENT_BF16 != 0, GQE_XENT_DK, true><<<grid, dim3(256), 0, stream>>>(p);
  else gqe_xent_prep_kernel<GQE_XENT_BF16 != 0, GQE_XENT_DK, false><<<grid, dim3(256), 0, stream>>>(p);
  return hipGetLastError();
}

#if GQE_XENT_BF16 == 0 && GQE_XENT_DK == 64
hipError_t gqe_xent_recs(const XentRecs& p, hipStream_t stream) {
  gqe_xent_recs_kernel<0><<<dim3((unsigned)((p.n + 255) / 256)), dim3(256), 0, stream>>>(p);
  return hipGetLastError();
}
#endif
