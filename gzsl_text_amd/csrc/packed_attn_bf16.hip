// bf16 instantiation of the packed label attention.
#include "packed_attn_kernels.h"

int pa_run_bf16(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    return p.waves == 8 && !backward ? pa_go<bf16, 8>(a, p, false, st) : pa_go<bf16, 4>(a, p, backward, st);
}
