// Cross attention, fp32 elements (kernels in cross_kernels.h and cross_bwd.h).
#include "cross_bwd.h"

int pf_xa_fwd_fp32(const XaParams& p, hipStream_t st) { return fwd_type<float>(p, st); }
int pf_xa_delta_fp32(const XaParams& p, float* amax, hipStream_t st) { return delta_type<float>(p, amax, st); }
int pf_xa_dq_fp32(const XaParams& p, hipStream_t st) { return dq_type<float>(p, st); }
int pf_xa_dkv_fp32(const XaParams& p, hipStream_t st) { return dkv_type<float>(p, st); }
