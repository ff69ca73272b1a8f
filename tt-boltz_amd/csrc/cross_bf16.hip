// Cross attention, bf16 elements (kernels in cross_kernels.h and cross_bwd.h).
#include "cross_bwd.h"

int pf_xa_fwd_bf16(const XaParams& p, hipStream_t st) { return fwd_type<bhalf_t>(p, st); }
int pf_xa_delta_bf16(const XaParams& p, float* amax, hipStream_t st) { return delta_type<bhalf_t>(p, amax, st); }
int pf_xa_dq_bf16(const XaParams& p, hipStream_t st) { return dq_type<bhalf_t>(p, st); }
int pf_xa_dkv_bf16(const XaParams& p, hipStream_t st) { return dkv_type<bhalf_t>(p, st); }
