// fp32 tensors of a key width up to 112: products of three bf16 pieces.
#include "packed_attn_kernels.h"

int pa_run_x3(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    typedef PaGeo<PaX3, 7, 13> G;
    return backward ? pa_go_bwd<PaX3, G, 8, 1>(a, p, st) : pa_go_fwd<PaX3, G, 8, 2>(a, st);
}
