// fp32 tensors of a key width above 112: exact fp32 matrix instructions.
#include "packed_attn_kernels.h"

int pa_run_f32(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    typedef PaGeo<PaF32, 13, 13> G;
    if (backward) return pa_go_bwd<PaF32, G, 8, 1>(a, p, st);
    return p.waves == 8 ? pa_go_fwd<PaF32, G, 8, 2>(a, st) : pa_go_fwd<PaF32, G, 4, 3>(a, st);
}
