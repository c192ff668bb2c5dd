// bf16 tensors.
#include "packed_attn_kernels.h"

int pa_run_bf16(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    typedef PaGeo<PaBF, 7, 13> A;
    typedef PaGeo<PaBF, 13, 13> B;
    if (backward) {
        if (p.waves == 8) return p.kind ? pa_go_bwd<PaBF, B, 8, 1>(a, p, st) : pa_go_bwd<PaBF, A, 8, 1>(a, p, st);
        return p.kind ? pa_go_bwd<PaBF, B, 4, 2>(a, p, st) : pa_go_bwd<PaBF, A, 4, 2>(a, p, st);
    }
    if (p.waves == 8) return p.kind ? pa_go_fwd<PaBF, B, 8, 4>(a, st) : pa_go_fwd<PaBF, A, 8, 4>(a, st);
    return p.kind ? pa_go_fwd<PaBF, B, 4, 3>(a, st) : pa_go_fwd<PaBF, A, 4, 3>(a, st);
}
