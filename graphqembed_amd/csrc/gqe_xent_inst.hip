// One (type, padded dim) of the softmax cross entropy's kernels per translation unit: -DGQE_XENT_BF16=0|1 -DGQE_XENT_DK=64|128|192|256.
#include "gqe_xent.h"
#include "gqe_ops_dev.h"

#define XENT_CAT3(a, b, c, d) a##b##_##c##d
#define XENT_NAME(b, dk) XENT_CAT3(gqe_xent_launch_, b, dk, )

template <int MODE, bool UNIT>
static hipError_t launch(const XentPass& p, hipStream_t stream) {
  typedef XentLds<GQE_XENT_BF16 != 0, GQE_XENT_DK, MODE> L;
  const void* f = (const void*)gqe_xent_kernel<GQE_XENT_BF16 != 0, GQE_XENT_DK, MODE, UNIT>;
  if (sizeof(L) > 65536) {
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(L));
    if (e != hipSuccess) return e;
  }
  gqe_xent_kernel<GQE_XENT_BF16 != 0, GQE_XENT_DK, MODE, UNIT><<<dim3((unsigned)(p.n_split * p.n_yblk)), dim3(256), sizeof(L), stream>>>(p);
  return hipGetLastError();
}

hipError_t XENT_NAME(GQE_XENT_BF16, GQE_XENT_DK)(int mode, bool unit, const XentPass& p, hipStream_t stream) {
  if (mode == XENT_MODE_LSE) return unit ? launch<XENT_MODE_LSE, true>(p, stream) : launch<XENT_MODE_LSE, false>(p, stream);
  if (mode == XENT_MODE_DQ) return unit ? launch<XENT_MODE_DQ, true>(p, stream) : launch<XENT_MODE_DQ, false>(p, stream);
  return unit ? launch<XENT_MODE_DT, true>(p, stream) : launch<XENT_MODE_DT, false>(p, stream);
}
