// Cross attention, fp16 elements (kernels in cross_kernels.h and cross_bwd.h).
#include "cross_bwd.h"

int pf_xa_fwd_fp16(const XaParams& p, hipStream_t st) { return fwd_type<half_t>(p, st); }
int pf_xa_delta_fp16(const XaParams& p, float* amax, hipStream_t st) { return delta_type<half_t>(p, amax, st); }
int pf_xa_dq_fp16(const XaParams& p, hipStream_t st) { return dq_type<half_t>(p, st); }
int pf_xa_dkv_fp16(const XaParams& p, hipStream_t st) { return dkv_type<half_t>(p, st); }
