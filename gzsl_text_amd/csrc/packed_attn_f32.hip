// fp32 instantiation of the packed label attention.
#include "packed_attn_kernels.h"

int pa_run_f32(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) { return pa_go<float, 4>(a, p, backward, st); }
