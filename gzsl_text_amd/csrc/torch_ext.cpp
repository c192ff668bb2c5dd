// TORCH_LIBRARY form of the hot path's operators: a thin C++ extension over the C ABI (include/gzsl_hip.h).
//
// SURVEY 8b / north_star name "a thin C++ extension" as the boundary; the ctypes host mirror (gzsl_text_amd/modules) is
// one binding of libgzsl_hip.so, this file is the other.  It registers differentiable torch operators that a maintainer
// of the reference can call from the UNCHANGED modules:
//   gzsl::label_attention  replaces modules/icd_modules.py:137-142 (scores, softmax over tokens, attn dropout, pooling)
//                          and its autograd; the B x L x T' score tensor is never formed
//   gzsl::label_logits     replaces modules/icd_modules.py:177-182 (relu, multiply by the label embedding, sum)
//   gzsl::ldam_bce         replaces modules/icd_modules.py:162-172 + BCEWithLogitsLoss(sum) / B (common_module.py:29-30)
// and, beyond the reference, for notes of unequal length and for training with clipped gradients:
//   gzsl::packed_label_attention, gzsl::gated_scan (differentiable), gzsl::gated_scan_step_, gzsl::clip_grad_norm_,
//   gzsl::adamw_clip_step_
// Tensors are allocated here with ATen (the C ABI itself never allocates); launches go to the CURRENT HIP stream of the
// tensors' device.  Built with g++ (no device code): __graft_entry__.build() -> gzsl_text_amd/lib/libgzsl_torch.so.
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <vector>

#include "../../include/gzsl_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_f32_cuda(const Tensor& t, const char* name, int64_t dims) {
    TORCH_CHECK(t.is_cuda(), "gzsl: ", name, " must be a GPU tensor (there is no CPU path)");
    TORCH_CHECK(t.scalar_type() == at::kFloat, "gzsl: ", name, " must be float32");
    TORCH_CHECK(t.dim() == dims, "gzsl: ", name, " must have ", dims, " dimensions");
}
void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, "gzsl: ", what, " failed with code ", rc); }
// (ROCm builds of torch present the GPU as device type "cuda": the stream getter is the masquerading one)
void* cur_stream() { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
const float* cptr(const Tensor& t) { return t.data_ptr<float>(); }

// (threshold, keep scale) of the counter RNG for drop probability p -- ops_hip.drop_params / oracle/rng.py
void drop_params(double p, uint32_t& thresh, float& scale) {
    if (p <= 0.0) {
        thresh = 0, scale = 1.f;
        return;
    }
    const double t = p * 4294967296.0;
    thresh = t >= 4294967295.0 ? 0xFFFFFFFFu : (uint32_t)t;
    scale = (float)(1.0 / (1.0 - p));
}

// label splits of the backward launch: enough workgroups for 256 CUs (the rule of ops_hip.HipOps.attn_bwd)
int bwd_nsplit(int64_t B, int64_t Tp, int64_t E, int64_t L) {
    const int64_t tok = E <= 100 ? 128 : 64, wgs = B * ((Tp + tok - 1) / tok);
    int ns = 1;
    while (wgs * ns < 1024 && (int64_t)ns * 2 * 16 <= L) ns *= 2;
    return ns;
}

struct LabelAttention : public torch::autograd::Function<LabelAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& keys, const Tensor& values, const Tensor& queries,
                                 double p_drop, int64_t seed, int64_t l_offset, int64_t L_total) {
        check_f32_cuda(keys, "keys", 3);
        check_f32_cuda(values, "values", 3);
        check_f32_cuda(queries, "queries", 2);
        TORCH_CHECK(keys.size(0) == values.size(0) && keys.size(1) == values.size(1), "gzsl: keys / values disagree");
        TORCH_CHECK(keys.size(2) == queries.size(1), "gzsl: keys / queries disagree on the embedding width");
        TORCH_CHECK(keys.device() == values.device() && keys.device() == queries.device(), "gzsl: tensors on one device");
        const c10::DeviceGuard guard(keys.device());
        const Tensor PX = keys.contiguous(), X = values.contiguous(), Q = queries.contiguous();
        const int64_t B = PX.size(0), Tp = PX.size(1), E = PX.size(2), F = X.size(2), L = Q.size(0);
        if (L_total <= 0) L_total = L;
        Tensor O = at::empty({B, L, F}, PX.options()), lse = at::empty({B, L}, PX.options());
        uint32_t th;
        float sc;
        drop_params(p_drop, th, sc);
        check_rc(gzsl_label_attn_fwd(cptr(PX), cptr(X), cptr(Q), O.data_ptr<float>(), lse.data_ptr<float>(), (int)B, (int)Tp,
                                     (int)E, (int)F, (int)L, (int)l_offset, (int)L_total, (uint32_t)seed, th, sc, cur_stream()),
                 "gzsl_label_attn_fwd");
        ctx->save_for_backward({PX, X, Q, O, lse});
        ctx->saved_data["p"] = p_drop;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["l_offset"] = l_offset;
        ctx->saved_data["L_total"] = L_total;
        ctx->mark_non_differentiable({lse});
        return {O, lse};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &PX = saved[0], &X = saved[1], &Q = saved[2], &O = saved[3], &lse = saved[4];
        const c10::DeviceGuard guard(PX.device());
        const Tensor dO = grads[0].contiguous();
        const int64_t B = PX.size(0), Tp = PX.size(1), E = PX.size(2), F = X.size(2), L = Q.size(0);
        Tensor delta = at::empty({B, L}, PX.options());
        Tensor dPX = at::zeros_like(PX), dX = at::zeros_like(X), dQ = at::zeros_like(Q);
        uint32_t th;
        float sc;
        drop_params(ctx->saved_data["p"].toDouble(), th, sc);
        void* st = cur_stream();
        check_rc(gzsl_attn_delta(cptr(dO), cptr(O), delta.data_ptr<float>(), B * L, (int)F, st), "gzsl_attn_delta");
        check_rc(gzsl_label_attn_bwd(cptr(dO), cptr(PX), cptr(X), cptr(Q), cptr(lse), cptr(delta), dPX.data_ptr<float>(),
                                     dX.data_ptr<float>(), dQ.data_ptr<float>(), (int)B, (int)Tp, (int)E, (int)F, (int)L,
                                     (int)ctx->saved_data["l_offset"].toInt(), (int)ctx->saved_data["L_total"].toInt(),
                                     bwd_nsplit(B, Tp, E, L), (uint32_t)ctx->saved_data["seed"].toInt(), th, sc, st),
                 "gzsl_label_attn_bwd");
        return {dPX, dX, dQ, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> label_attention(const Tensor& keys, const Tensor& values, const Tensor& queries, double p_drop,
                                           int64_t seed, int64_t l_offset, int64_t L_total) {
    auto out = LabelAttention::apply(keys, values, queries, p_drop, seed, l_offset, L_total);
    return {out[0], out[1]};
}

struct LabelLogits : public torch::autograd::Function<LabelLogits> {
    static Tensor forward(AutogradContext* ctx, const Tensor& direct, const Tensor& clf) {
        check_f32_cuda(direct, "direct", 3);
        check_f32_cuda(clf, "label_emb", 2);
        TORCH_CHECK(direct.size(1) == clf.size(0) && direct.size(2) == clf.size(1), "gzsl: direct [B,L,D] vs label_emb [L,D]");
        const c10::DeviceGuard guard(direct.device());
        const Tensor d = direct.contiguous(), c = clf.contiguous();
        Tensor logits = at::empty({d.size(0), d.size(1)}, d.options());
        check_rc(gzsl_logits_fwd(cptr(d), cptr(c), logits.data_ptr<float>(), (int)d.size(0), (int)d.size(1), (int)d.size(2),
                                 cur_stream()),
                 "gzsl_logits_fwd");
        ctx->save_for_backward({d, c});
        return logits;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &d = saved[0], &c = saved[1];
        const c10::DeviceGuard guard(d.device());
        const Tensor dl = grads[0].contiguous();
        Tensor dd = at::empty_like(d), dc = at::empty_like(c);
        check_rc(gzsl_logits_bwd(cptr(d), cptr(c), cptr(dl), dd.data_ptr<float>(), dc.data_ptr<float>(), (int)d.size(0),
                                 (int)d.size(1), (int)d.size(2), 0, cur_stream()),
                 "gzsl_logits_bwd");
        return {dd, dc};
    }
};
Tensor label_logits(const Tensor& direct, const Tensor& clf) { return LabelLogits::apply(direct, clf); }

struct LdamBce : public torch::autograd::Function<LdamBce> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& y, const c10::optional<Tensor>& margin,
                          double C) {
        check_f32_cuda(logits, "logits", 2);
        check_f32_cuda(y, "y", 2);
        TORCH_CHECK(logits.sizes() == y.sizes(), "gzsl: logits / y shapes differ");
        const c10::DeviceGuard guard(logits.device());
        const Tensor z = logits.contiguous(), yy = y.contiguous();
        Tensor m;
        if (margin.has_value() && margin->defined() && C > 0.0) {
            check_f32_cuda(*margin, "class_margin", 1);
            TORCH_CHECK(margin->size(0) == z.size(1), "gzsl: class_margin has one entry per label");
            m = margin->contiguous();
        }
        Tensor loss = at::zeros({}, z.options()), dlogits = at::empty_like(z);
        check_rc(gzsl_ldam_bce(cptr(z), cptr(yy), m.defined() ? cptr(m) : nullptr, (float)C, 1.f / (float)z.size(0),
                               loss.data_ptr<float>(), dlogits.data_ptr<float>(), nullptr, (int)z.size(0), (int)z.size(1),
                               cur_stream()),
                 "gzsl_ldam_bce");
        ctx->save_for_backward({dlogits});
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor dlogits = ctx->get_saved_variables()[0];
        return {dlogits * grads[0], Tensor(), Tensor(), Tensor()};
    }
};
Tensor ldam_bce(const Tensor& logits, const Tensor& y, const c10::optional<Tensor>& margin, double C) {
    return LdamBce::apply(logits, y, margin, C);
}

// ---- packed notes (gzsl_packed_attn_*, gzsl_gated_scan_*)
int type_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "gzsl: ", name, " must be a GPU tensor (there is no CPU path)");
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, "gzsl: ", name, " must be float32 or bfloat16");
    return t.scalar_type() == at::kFloat ? GZSL_F32 : GZSL_BF16;
}
// [rows, width] with contiguous rows, any row pitch
Tensor rows_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() == 2, "gzsl: ", name, " must have 2 dimensions");
    const bool ok = (t.stride(1) == 1 || t.size(1) <= 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return ok ? t : t.contiguous();
}
long long pitch_of(const Tensor& t) { return t.size(0) > 1 ? std::max<int64_t>(t.stride(0), t.size(1)) : t.size(1); }
void check_spans(const Tensor& spans, int64_t max_len, const Tensor& ref) {
    TORCH_CHECK(spans.is_cuda() && spans.scalar_type() == at::kLong && spans.dim() == 2 && spans.size(1) == 2 && spans.is_contiguous(),
                "gzsl: spans must be a contiguous int64 [B, 2] GPU tensor");
    TORCH_CHECK(spans.device() == ref.device(), "gzsl: tensors on one device");
    TORCH_CHECK(max_len >= 0 && max_len < (1LL << 31), "gzsl: max_len out of range");
    TORCH_CHECK(spans.size(0) < (1LL << 31) && ref.size(0) < (1LL << 40), "gzsl: too many notes");
}
Tensor scratch(long long bytes, const Tensor& ref, const char* what) {
    TORCH_CHECK(bytes >= 0, "gzsl: ", what, ": unsupported arguments");
    return at::empty({std::max<long long>(bytes, 16)}, ref.options().dtype(at::kByte));
}

// written in place by a kernel: autograd has to see it (a saved copy of the old value must not be used silently)
void touched(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The gradients come from kernels that autograd does not see through: a graph of them would miss every term.
void check_once(const char* what) { TORCH_CHECK(!at::GradMode::is_enabled(), "gzsl: ", what, " is differentiable once (backward with create_graph)"); }

struct PackedLabelAttention : public torch::autograd::Function<PackedLabelAttention> {
    static GzslPackedAttn describe(const Tensor& k, const Tensor& v, const Tensor& q, const Tensor& spans, int64_t max_len, double cap, double p,
                                   int64_t seed, int64_t l_offset, int64_t L_total) {
        GzslPackedAttn d{};
        d.keys = k.data_ptr(), d.values = v.data_ptr(), d.queries = q.data_ptr(), d.spans = spans.data_ptr<int64_t>();
        d.rows = k.size(0), d.ldk = pitch_of(k), d.ldv = pitch_of(v), d.ldq = pitch_of(q);
        d.B = (int)spans.size(0), d.max_len = (int)max_len, d.L = (int)q.size(0), d.E = (int)k.size(1), d.F = (int)v.size(1);
        d.dtype = type_of(k, "keys"), d.cap = (float)cap;
        d.l_offset = (int)l_offset, d.L_total = (int)L_total, d.seed = (uint32_t)seed;
        drop_params(p, d.drop_thresh, d.drop_scale);
        return d;
    }
    static variable_list forward(AutogradContext* ctx, const Tensor& keys, const Tensor& values, const Tensor& queries, const Tensor& spans,
                                 int64_t max_len, double cap, double p_drop, int64_t seed, int64_t l_offset, int64_t L_total, bool grad) {
        const int t = type_of(keys, "keys");
        TORCH_CHECK(type_of(values, "values") == t && type_of(queries, "queries") == t, "gzsl: keys, values and queries must have one type");
        const Tensor k = rows_of(keys, "keys"), v = rows_of(values, "values"), q = rows_of(queries, "queries");
        TORCH_CHECK(k.size(0) == v.size(0), "gzsl: keys / values disagree");
        TORCH_CHECK(k.size(1) == q.size(1), "gzsl: keys / queries disagree on the embedding width");
        TORCH_CHECK(k.device() == v.device() && k.device() == q.device(), "gzsl: tensors on one device");
        TORCH_CHECK(k.size(1) <= 208 && v.size(1) <= 208 && k.size(1) > 0 && v.size(1) > 0, "gzsl: widths from 1 to 208");
        TORCH_CHECK(cap == 0.0 || (cap >= 1e-30 && cap <= 1e30), "gzsl: cap must be 0 (none) or from 1e-30 to 1e30");
        TORCH_CHECK(p_drop >= 0.0 && p_drop < 1.0, "gzsl: drop probability in [0, 1)");
        check_spans(spans, max_len, k);
        if (L_total <= 0) L_total = q.size(0);
        TORCH_CHECK(l_offset >= 0 && L_total < (1LL << 31) && l_offset <= L_total - q.size(0), "gzsl: labels outside of L_total");
        const c10::DeviceGuard guard(k.device());
        const GzslPackedAttn d = describe(k, v, q, spans, max_len, cap, p_drop, seed, l_offset, L_total);
        Tensor O = at::empty({d.B, d.L, d.F}, v.options()), lse = at::empty({d.B, d.L}, v.options().dtype(at::kFloat));
        const Tensor work = scratch(gzsl_packed_attn_work_bytes(&d, 0), k, "packed_label_attention");
        Tensor rest;
        if (grad) rest = scratch(gzsl_packed_attn_rest_bytes(&d), k, "packed_label_attention");
        check_rc(gzsl_packed_attn_fwd(&d, O.data_ptr(), lse.data_ptr<float>(), grad ? rest.data_ptr() : nullptr, work.data_ptr(), work.numel(), cur_stream()),
                 "gzsl_packed_attn_fwd");
        ctx->mark_non_differentiable({lse});
        if (!grad) return {O, lse};
        ctx->save_for_backward({k, v, q, spans, O, lse, rest});
        ctx->saved_data["max_len"] = max_len;
        ctx->saved_data["cap"] = cap;
        ctx->saved_data["p"] = p_drop;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["l_offset"] = l_offset;
        ctx->saved_data["L_total"] = L_total;
        return {O, lse};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_once("packed_label_attention");
        const auto saved = ctx->get_saved_variables();
        const Tensor &k = saved[0], &v = saved[1], &q = saved[2], &spans = saved[3], &O = saved[4], &lse = saved[5], &rest = saved[6];
        const c10::DeviceGuard guard(k.device());
        const GzslPackedAttn d = describe(k, v, q, spans, ctx->saved_data["max_len"].toInt(), ctx->saved_data["cap"].toDouble(), ctx->saved_data["p"].toDouble(),
                                          ctx->saved_data["seed"].toInt(), ctx->saved_data["l_offset"].toInt(), ctx->saved_data["L_total"].toInt());
        Tensor dK = at::empty(k.sizes(), k.options()), dV = at::empty(v.sizes(), v.options()), dQ = at::empty(q.sizes(), q.options());
        if (d.B == 0 || d.L == 0) {
            dK.zero_(), dV.zero_(), dQ.zero_();
        } else {
            const Tensor dO = grads[0].contiguous();
            const Tensor work = scratch(gzsl_packed_attn_work_bytes(&d, 1), k, "packed_label_attention");
            check_rc(gzsl_packed_attn_bwd(&d, O.data_ptr(), lse.data_ptr<float>(), rest.data_ptr(), dO.data_ptr(), dK.data_ptr(), dV.data_ptr(), dQ.data_ptr(), work.data_ptr(),
                                          work.numel(), cur_stream()),
                     "gzsl_packed_attn_bwd");
        }
        return {dK, dV, dQ, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
std::tuple<Tensor, Tensor> packed_label_attention(const Tensor& keys, const Tensor& values, const Tensor& queries, const Tensor& spans, int64_t max_len,
                                                  double cap, double p_drop, int64_t seed, int64_t l_offset, int64_t L_total) {
    const bool grad = at::GradMode::is_enabled() && (keys.requires_grad() || values.requires_grad() || queries.requires_grad());
    auto out = PackedLabelAttention::apply(keys, values, queries, spans, max_len, cap, p_drop, seed, l_offset, L_total, grad);
    return {out[0], out[1]};
}

struct GatedScan : public torch::autograd::Function<GatedScan> {
    static GzslGatedScan describe(const Tensor& g, const Tensor& c, const Tensor& spans, int64_t max_len, const Tensor& h0, bool reverse, const Tensor& rest) {
        GzslGatedScan d{};
        d.gates = g.data_ptr(), d.cands = c.data_ptr(), d.spans = spans.data_ptr<int64_t>(), d.h0 = h0.defined() ? h0.data_ptr<float>() : nullptr;
        d.rows = g.size(0), d.ldg = pitch_of(g), d.ldc = pitch_of(c);
        d.B = (int)spans.size(0), d.max_len = (int)max_len, d.H = (int)g.size(1), d.reverse = reverse, d.dtype = type_of(g, "gates");
        d.rest = rest.defined() ? rest.data_ptr() : nullptr;
        return d;
    }
    static variable_list forward(AutogradContext* ctx, const Tensor& gates, const Tensor& cands, const Tensor& spans, int64_t max_len,
                                 const c10::optional<Tensor>& h0_, bool reverse, bool grad) {
        TORCH_CHECK(type_of(gates, "gates") == type_of(cands, "cands"), "gzsl: gates and cands must have one type");
        const Tensor g = rows_of(gates, "gates"), c = rows_of(cands, "cands");
        TORCH_CHECK(g.sizes() == c.sizes(), "gzsl: gates / cands shapes differ");
        TORCH_CHECK(g.device() == c.device(), "gzsl: tensors on one device");
        TORCH_CHECK(g.size(1) > 0 && g.size(1) < (1LL << 31), "gzsl: at least one channel");
        check_spans(spans, max_len, g);
        const c10::DeviceGuard guard(g.device());
        Tensor h0;
        if (h0_.has_value() && h0_->defined()) {
            check_f32_cuda(*h0_, "h0", 2);
            TORCH_CHECK(h0_->size(0) == spans.size(0) && h0_->size(1) == g.size(1) && h0_->device() == g.device(), "gzsl: h0 is [B, H] on the same device");
            h0 = h0_->contiguous();
        }
        Tensor rest;  // (what a backward needs of 16-bit states)
        if (grad && g.scalar_type() == at::kBFloat16) rest = at::empty(g.sizes(), g.options());
        const GzslGatedScan d = describe(g, c, spans, max_len, h0, reverse, rest);
        Tensor h = at::empty(g.sizes(), g.options()), last = at::empty({d.B, d.H}, g.options().dtype(at::kFloat));
        if (d.B == 0) {
            h.zero_();
        } else {
            const Tensor work = scratch(gzsl_gated_scan_work_bytes(&d, 0), g, "gated_scan");
            check_rc(gzsl_gated_scan_fwd(&d, h.data_ptr(), last.data_ptr<float>(), work.data_ptr(), work.numel(), cur_stream()), "gzsl_gated_scan_fwd");
        }
        if (!grad) return {h, last};
        ctx->save_for_backward({g, c, spans, h, h0, rest});
        ctx->saved_data["max_len"] = max_len;
        ctx->saved_data["reverse"] = reverse;
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_once("gated_scan");
        const auto saved = ctx->get_saved_variables();
        const Tensor &g = saved[0], &c = saved[1], &spans = saved[2], &h = saved[3], &h0 = saved[4], &rest = saved[5];
        const c10::DeviceGuard guard(g.device());
        const GzslGatedScan d = describe(g, c, spans, ctx->saved_data["max_len"].toInt(), h0, ctx->saved_data["reverse"].toBool(), rest);
        Tensor dg = at::empty(g.sizes(), g.options()), dc = at::empty(g.sizes(), g.options()), dh0;
        if (h0.defined()) dh0 = at::empty_like(h0);
        if (d.B == 0) {
            dg.zero_(), dc.zero_();
        } else {
            const Tensor dh = grads[0].defined() ? grads[0].contiguous() : Tensor(), dl = grads[1].defined() ? grads[1].contiguous() : Tensor();
            const Tensor work = scratch(gzsl_gated_scan_work_bytes(&d, 1), g, "gated_scan");
            check_rc(gzsl_gated_scan_bwd(&d, h.data_ptr(), dh.defined() ? dh.data_ptr() : nullptr, dl.defined() ? dl.data_ptr<float>() : nullptr, dg.data_ptr(),
                                         dc.data_ptr(), h0.defined() ? dh0.data_ptr<float>() : nullptr, work.data_ptr(), work.numel(), cur_stream()),
                     "gzsl_gated_scan_bwd");
        }
        return {dg, dc, Tensor(), Tensor(), dh0, Tensor(), Tensor()};
    }
};
std::tuple<Tensor, Tensor> gated_scan(const Tensor& gates, const Tensor& cands, const Tensor& spans, int64_t max_len, const c10::optional<Tensor>& h0,
                                      bool reverse) {
    const bool grad = at::GradMode::is_enabled() && (gates.requires_grad() || cands.requires_grad() || (h0.has_value() && h0->requires_grad()));
    auto out = GatedScan::apply(gates, cands, spans, max_len, h0, reverse, grad);
    return {out[0], out[1]};
}

void gated_scan_step_(const Tensor& gates, const Tensor& cands, const Tensor& state, const c10::optional<Tensor>& active) {
    // autograd would take the state behind the step for the one in front of it, and miss the gates and candidates
    TORCH_CHECK(!at::GradMode::is_enabled() || !(gates.requires_grad() || cands.requires_grad() || state.requires_grad()),
                "gzsl: gated_scan_step_ is not differentiable: call gated_scan, or the step under no_grad or on detached tensors");
    const int t = type_of(gates, "gates");
    TORCH_CHECK(type_of(cands, "cands") == t, "gzsl: gates and cands must have one type");
    check_f32_cuda(state, "state", 2);
    const Tensor g = rows_of(gates, "gates"), c = rows_of(cands, "cands");
    TORCH_CHECK(g.sizes() == c.sizes() && g.sizes() == state.sizes(), "gzsl: gates, cands and state have one shape");
    TORCH_CHECK(state.is_contiguous(), "gzsl: state must be contiguous");
    TORCH_CHECK(g.device() == c.device() && g.device() == state.device(), "gzsl: tensors on one device");
    const uint8_t* on = nullptr;
    if (active.has_value() && active->defined()) {
        TORCH_CHECK(active->scalar_type() == at::kBool && active->dim() == 1 && active->size(0) == state.size(0) && active->is_contiguous() &&
                        active->device() == state.device(),
                    "gzsl: active must be a contiguous bool [B] tensor on the same device");
        on = (const uint8_t*)active->data_ptr();
    }
    if (state.numel() == 0) return;
    const c10::DeviceGuard guard(state.device());
    check_rc(gzsl_gated_scan_step(g.data_ptr(), c.data_ptr(), state.data_ptr<float>(), on, (int)state.size(0), (int)state.size(1), pitch_of(g), pitch_of(c),
                                  t, cur_stream()),
             "gzsl_gated_scan_step");
    touched(state);
}

// ---- gradient clipping (gzsl_clip_grad_norm, gzsl_adamw_clip_step)
// Addresses of contiguous tensors on one device.
std::vector<void*> pointers(at::TensorList ts, const c10::Device& dev, const char* name, bool f32_only) {
    std::vector<void*> out;
    out.reserve(ts.size());
    for (const Tensor& t : ts) {
        TORCH_CHECK(t.is_cuda() && t.device() == dev, "gzsl: ", name, ": GPU tensors on one device");
        TORCH_CHECK(t.scalar_type() == at::kFloat || (!f32_only && t.scalar_type() == at::kBFloat16), "gzsl: ", name, ": float32", f32_only ? "" : " or bfloat16");
        TORCH_CHECK(t.is_contiguous(), "gzsl: ", name, ": contiguous tensors");
        out.push_back(t.data_ptr());
    }
    return out;
}
// Written tensors may share memory with nothing else of the call: it would be updated twice at once, or read in between.
struct Extent {
    const char *at, *end;
    bool written;
};
void extents(std::vector<Extent>& all, at::TensorList ts, bool written) {
    all.reserve(all.size() + ts.size());
    for (const Tensor& t : ts)
        if (t.numel() > 0) all.push_back({(const char*)t.data_ptr(), (const char*)t.data_ptr() + t.nbytes(), written});
}
void check_apart(std::vector<Extent>& all) {
    std::sort(all.begin(), all.end(), [](const Extent& a, const Extent& b) { return a.at < b.at; });
    const char *end = nullptr, *written = nullptr;  // of the extents so far: furthest end, and that of a written one
    for (const Extent& e : all) {
        TORCH_CHECK(e.at >= (e.written ? end : written), "gzsl: the same tensor appears twice in the list, or two of them overlap");
        end = std::max(end, e.end);
        if (e.written) written = std::max(written, e.end);
    }
}
c10::Device device_of(at::TensorList ts) { return ts.empty() ? c10::Device(c10::kCUDA, c10::hip::current_device()) : ts[0].device(); }

Tensor clip_grad_norm_(at::TensorList grads, double max_norm) {
    TORCH_CHECK(max_norm > 0.0, "gzsl: max_norm must be positive");
    const c10::Device dev = device_of(grads);
    const auto g = pointers(grads, dev, "grads", false);
    std::vector<Extent> held;
    extents(held, grads, true);
    check_apart(held);
    std::vector<long long> n;
    std::vector<int> t;
    for (const Tensor& x : grads) n.push_back(x.numel()), t.push_back(x.scalar_type() == at::kFloat ? GZSL_F32 : GZSL_BF16);
    const c10::DeviceGuard guard(dev);
    const auto opt = at::TensorOptions().device(dev).dtype(at::kFloat);
    Tensor norm = at::empty({}, opt);
    const Tensor work = scratch(gzsl_clip_work_bytes(n.data(), (int)n.size()), norm, "clip_grad_norm_");
    check_rc(gzsl_clip_grad_norm(g.data(), n.data(), t.data(), (int)n.size(), (float)max_norm, norm.data_ptr<float>(), work.data_ptr(), work.numel(), cur_stream()),
             "gzsl_clip_grad_norm");
    for (const Tensor& x : grads) touched(x);
    return norm;
}

Tensor adamw_clip_step_(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList v, double max_norm, double lr, double beta1, double beta2,
                        double eps, double wd) {
    TORCH_CHECK(max_norm > 0.0, "gzsl: max_norm must be positive");
    TORCH_CHECK(params.size() == grads.size() && params.size() == m.size() && params.size() == v.size(), "gzsl: params, grads and moments do not fit");
    const c10::Device dev = device_of(params);
    const auto p = pointers(params, dev, "params", true), g = pointers(grads, dev, "grads", true), mm = pointers(m, dev, "m", true), vv = pointers(v, dev, "v", true);
    std::vector<Extent> held;
    extents(held, params, true), extents(held, m, true), extents(held, v, true), extents(held, grads, false);
    check_apart(held);
    std::vector<long long> n;
    for (size_t i = 0; i < params.size(); ++i) {
        TORCH_CHECK(grads[i].sizes() == params[i].sizes() && m[i].sizes() == params[i].sizes() && v[i].sizes() == params[i].sizes(),
                    "gzsl: params, grads and moments do not fit");
        n.push_back(params[i].numel());
    }
    const c10::DeviceGuard guard(dev);
    const auto opt = at::TensorOptions().device(dev).dtype(at::kFloat);
    Tensor norm = at::empty({}, opt);
    const Tensor work = scratch(gzsl_clip_work_bytes(n.data(), (int)n.size()), norm, "adamw_clip_step_");
    check_rc(gzsl_adamw_clip_step((float* const*)p.data(), (const float* const*)g.data(), (float* const*)mm.data(), (float* const*)vv.data(), n.data(),
                                  (int)n.size(), (float)max_norm, lr, beta1, beta2, eps, wd, norm.data_ptr<float>(),
                                  work.data_ptr(), work.numel(), cur_stream()),
             "gzsl_adamw_clip_step");
    for (const at::TensorList ts : {params, m, v})
        for (const Tensor& x : ts) touched(x);
    return norm;
}

}  // namespace

TORCH_LIBRARY(gzsl, m) {
    m.def("label_attention(Tensor keys, Tensor values, Tensor queries, float p_drop=0.0, int seed=0, int l_offset=0, "
          "int L_total=0) -> (Tensor, Tensor)");
    m.def("label_logits(Tensor direct, Tensor label_emb) -> Tensor");
    m.def("ldam_bce(Tensor logits, Tensor y, Tensor? class_margin=None, float C=0.0) -> Tensor");
    m.def("packed_label_attention(Tensor keys, Tensor values, Tensor queries, Tensor spans, int max_len, float cap=0.0, "
          "float p_drop=0.0, int seed=0, int l_offset=0, int L_total=0) -> (Tensor, Tensor)");
    m.def("gated_scan(Tensor gates, Tensor cands, Tensor spans, int max_len, Tensor? h0=None, bool reverse=False) -> (Tensor, Tensor)");
    m.def("gated_scan_step_(Tensor gates, Tensor cands, Tensor(a!) state, Tensor? active=None) -> ()");
    m.def("clip_grad_norm_(Tensor(a!)[] grads, float max_norm) -> Tensor");
    m.def("adamw_clip_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] m, Tensor(c!)[] v, float max_norm, float lr, float beta1, "
          "float beta2, float eps, float weight_decay) -> Tensor");
}

// The autograd::Function::apply wrappers record the graph themselves; they are registered for the Autograd key so that
// tensors that require grad reach them, and for the backend key for calls under no_grad.
TORCH_LIBRARY_IMPL(gzsl, Autograd, m) {
    m.impl("label_attention", label_attention);
    m.impl("label_logits", label_logits);
    m.impl("ldam_bce", ldam_bce);
    m.impl("packed_label_attention", packed_label_attention);
    m.impl("gated_scan", gated_scan);
    m.impl("gated_scan_step_", gated_scan_step_);  // (in place and not differentiable: refused where a gradient would be missed)
    m.impl("clip_grad_norm_", clip_grad_norm_);
    m.impl("adamw_clip_step_", adamw_clip_step_);
}
TORCH_LIBRARY_IMPL(gzsl, CUDA, m) {
    m.impl("label_attention", label_attention);
    m.impl("label_logits", label_logits);
    m.impl("ldam_bce", ldam_bce);
    m.impl("packed_label_attention", packed_label_attention);
    m.impl("gated_scan", gated_scan);
    m.impl("gated_scan_step_", gated_scan_step_);
}
// (an empty list names no backend: these two are reached without one, and check their tensors themselves)
TORCH_LIBRARY_IMPL(gzsl, CompositeExplicitAutograd, m) {
    m.impl("clip_grad_norm_", clip_grad_norm_);
    m.impl("adamw_clip_step_", adamw_clip_step_);
}
