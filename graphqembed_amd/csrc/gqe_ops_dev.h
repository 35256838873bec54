// gqe_ops_dev.h — launchers that the operators' translation units share.
#ifndef GQE_OPS_DEV_H
#define GQE_OPS_DEV_H

#include <hip/hip_runtime.h>

struct XentPass;
struct XentPrep;
struct XentRecs;
hipError_t gqe_xent_recs(const XentRecs& p, hipStream_t stream);
#define GQE_XENT_DECL(b, dk) \
  hipError_t gqe_xent_launch_##b##_##dk(int mode, bool unit, bool dma, const XentPass& p, hipStream_t stream); \
  hipError_t gqe_xent_prep_##b##_##dk(bool unit, const XentPrep& p, hipStream_t stream);
GQE_XENT_DECL(0, 64) GQE_XENT_DECL(0, 128) GQE_XENT_DECL(0, 192) GQE_XENT_DECL(0, 256)
GQE_XENT_DECL(1, 64) GQE_XENT_DECL(1, 128) GQE_XENT_DECL(1, 192) GQE_XENT_DECL(1, 256)
#undef GQE_XENT_DECL

#endif
