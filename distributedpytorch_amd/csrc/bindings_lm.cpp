// Bindings for the language-model kernels: attention with score modifiers, head norms with rotation, the scaled token
// embedding and the distillation loss, each as an autograd node of its own.  The Python side (ops/attend.py, ops/heads.py,
// ops/embed.py, ops/distill.py) states what a call may be; the checks here are what the kernels' addressing relies on.
//
// The nodes are C++ and not Python functions because the smallest calls are all host time: the engine runs a backward on a
// thread of its own, and a Python node has to win the interpreter lock there first.
#include <torch/extension.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "kernels.h"

namespace {
using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
inline hipStream_t cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

#define CHECK_ON(t, like) TORCH_CHECK((t).is_cuda() && (t).device() == (like).device(), #t " must be on " #like "'s GPU")
#define CHECK_FLAT(t, like, type) do { CHECK_ON(t, like); TORCH_CHECK((t).is_contiguous(), #t " must be contiguous"); \
                                       TORCH_CHECK((t).scalar_type() == (type), #t ": wrong type"); } while (0)
inline bool on16(const Tensor& t) { return ((uintptr_t)t.data_ptr()) % 16 == 0; }
#define CHECK_FLAT16(t, like, type) do { CHECK_FLAT(t, like, type); TORCH_CHECK(on16(t), #t " must be 16-byte aligned"); } while (0)

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The kernels form first derivatives only.
void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "this operator's gradient cannot be differentiated again"); }

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor bare(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

Tensor flat16(const Tensor& t) { return t.is_contiguous() && on16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
// last axis contiguous, every row on 16 bytes, 64 tokens within 32-bit offsets
Tensor rows16(const Tensor& t) {
    bool ok = on16(t) && (t.size(-1) <= 1 || t.stride(-1) == 1);
    for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && (i != 1 || t.stride(i) < (1 << 23))));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ---------------------------------------------------------------- attention
// element stride of axis i (0 where the axis has one entry), in whole 16-byte steps
long row_stride(const Tensor& t, int i) {
    if (t.size(i) <= 1) return 0;
    TORCH_CHECK(t.stride(i) % 8 == 0 && t.stride(i) >= 0, "attend: rows must be 16-byte aligned");
    return (long)t.stride(i);
}

dpa::AttendArgs attend_args(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale, double softcap, const OptTensor& slopes,
                            const OptTensor& documents, const OptTensor& prefix) {
    for (const Tensor* t : {&q, &k, &v}) {
        TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->dim() == 4 && t->scalar_type() == at::kBFloat16, "attend: q, k, v must be bf16 [B,T,H,D] on one GPU");
        TORCH_CHECK(t->size(3) == 1 || t->stride(3) == 1, "attend: the last axis must be contiguous");
        TORCH_CHECK(on16(*t), "attend: 16-byte alignment");
    }
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(2);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(1) == T && k.size(3) == D, "attend: shapes");
    TORCH_CHECK(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && D >= 8 && D % 8 == 0 && D <= 128, "attend: heads");
    TORCH_CHECK(B <= 65535 && T <= (1 << 22) && Hq <= 65535 && (int64_t)Hq * D < (1 << 23), "attend: oversized problem");
    for (const Tensor* t : {&q, &k, &v}) TORCH_CHECK(T <= 1 || t->stride(1) < (1 << 23), "attend: token stride");
    TORCH_CHECK(scale > 1e-12 && scale < 1e12 && (softcap == 0.0 || (softcap > 1e-12 && softcap < 1e12)), "attend: scale, softcap");
    dpa::AttendArgs a{};
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
    a.qb = row_stride(q, 0); a.qt = row_stride(q, 1); a.qh = row_stride(q, 2);
    a.kb = row_stride(k, 0); a.kt = row_stride(k, 1); a.kh = row_stride(k, 2);
    a.vb = row_stride(v, 0); a.vt = row_stride(v, 1); a.vh = row_stride(v, 2);
    if (slopes.has_value()) {
        CHECK_FLAT((*slopes), q, at::kFloat);
        TORCH_CHECK(slopes->numel() == Hq, "attend: slopes");
        a.slopes = slopes->data_ptr<float>();
    }
    if (documents.has_value()) {
        CHECK_FLAT((*documents), q, at::kInt);
        TORCH_CHECK(documents->numel() == B * T, "attend: documents");
        a.docs = documents->data_ptr<int>();
    }
    if (prefix.has_value()) {
        CHECK_FLAT((*prefix), q, at::kInt);
        TORCH_CHECK(prefix->numel() == B, "attend: prefix");
        a.prefix = prefix->data_ptr<int>();
    }
    a.B = (int)B; a.T = (int)T; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = (int)D; a.causal = causal;
    a.scale = (float)scale; a.softcap = (float)softcap;
    return a;
}

// -> out [B,T,Hq,D], lse2 [B,Hq,T], ranges (undefined without documents), rest (what rounding took from out; for backward)
std::vector<Tensor> attend_fwd(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale, double softcap, const OptTensor& slopes,
                               const OptTensor& documents, const OptTensor& prefix, bool for_backward) {
    dpa::AttendArgs a = attend_args(q, k, v, causal, scale, softcap, slopes, documents, prefix);
    Guard guard(q.device());
    Tensor out = torch::empty(q.sizes(), q.options()), rest;
    Tensor lse2 = torch::empty({a.B, a.Hq, a.T}, q.options().dtype(at::kFloat));
    Tensor ranges;
    if (for_backward) rest = torch::empty(q.sizes(), q.options());
    if (out.numel() == 0) return {out, lse2, ranges, rest};
    if (a.docs != nullptr) {
        ranges = torch::empty({a.B, (a.T + 63) / 64, 4}, q.options().dtype(at::kInt));
        dpa::attend_doc_ranges(a.docs, ranges.data_ptr(), a.B, a.T, cur_stream());
        a.ranges = (const int4*)ranges.data_ptr();
    }
    dpa::attend_fwd(a, out.data_ptr(), for_backward ? rest.data_ptr() : nullptr, lse2.data_ptr<float>(), cur_stream());
    return {out, lse2, ranges, rest};
}

// -> dq, dk, dv, contiguous
std::vector<Tensor> attend_bwd(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale, double softcap, const OptTensor& slopes,
                               const OptTensor& documents, const OptTensor& prefix, const OptTensor& ranges, const Tensor& out, const Tensor& rest,
                               const Tensor& dout, const Tensor& lse2) {
    dpa::AttendArgs a = attend_args(q, k, v, causal, scale, softcap, slopes, documents, prefix);
    CHECK_FLAT16(out, q, at::kBFloat16); CHECK_FLAT16(rest, q, at::kBFloat16); CHECK_FLAT16(dout, q, at::kBFloat16); CHECK_FLAT(lse2, q, at::kFloat);
    TORCH_CHECK(out.sizes() == q.sizes() && rest.sizes() == q.sizes() && dout.sizes() == q.sizes() && lse2.numel() == (int64_t)a.B * a.Hq * a.T, "attend_bwd: shapes");
    Guard guard(q.device());
    Tensor dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), q.options()), dv = torch::empty(k.sizes(), q.options());
    if (out.numel() == 0) return {dq, dk, dv};
    if (a.docs != nullptr) {
        TORCH_CHECK(ranges.has_value() && ranges->numel() == (int64_t)a.B * ((a.T + 63) / 64) * 4, "attend_bwd: ranges");
        CHECK_FLAT16((*ranges), q, at::kInt);
        a.ranges = (const int4*)ranges->data_ptr();
    }
    Tensor stats = torch::empty({a.B, a.Hq, a.T, 2}, lse2.options());
    const int parts = dpa::attend_kv_parts(a);
    Tensor part;
    if (parts > 1) part = torch::empty({parts, 2, dk.numel()}, lse2.options());
    dpa::attend_bwd(a, out.data_ptr(), rest.data_ptr(), dout.data_ptr(), lse2.data_ptr<float>(), stats.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                    parts > 1 ? part.data_ptr<float>() : nullptr, cur_stream());
    return {dq, dk, dv};
}

struct AttendNode : public torch::autograd::Function<AttendNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, bool causal, double scale, double softcap,
                          const OptTensor& slopes, const OptTensor& documents, const OptTensor& prefix, bool for_backward) {
        const Tensor q = rows16(q_), k = rows16(k_), v = rows16(v_);
        auto r = attend_fwd(q, k, v, causal, scale, softcap, slopes, documents, prefix, for_backward);
        if (for_backward) {
            ctx->save_for_backward({q, k, v, bare(slopes), bare(documents), bare(prefix), r[2], r[0], r[3], r[1]});
            ctx->saved_data["causal"] = causal; ctx->saved_data["scale"] = scale; ctx->saved_data["softcap"] = softcap;
        }
        return r[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        auto d = attend_bwd(s[0], s[1], s[2], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), ctx->saved_data["softcap"].toDouble(),
                            opt(s[3]), opt(s[4]), opt(s[5]), opt(s[6]), s[7], s[8], flat16(g[0]), s[9]);
        return {d[0], d[1], d[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
Tensor attention_ex(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale, double softcap, const OptTensor& slopes,
                    const OptTensor& documents, const OptTensor& prefix) {
    const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    return AttendNode::apply(q, k, v, causal, scale, softcap, slopes, documents, prefix, grad);
}

// ---------------------------------------------------------------- head norms and rotation
dpa::HeadsArgs heads_args(const Tensor& qkv, int64_t Hq, int64_t Hkv, const OptTensor& qw, const OptTensor& kw, const OptTensor& inv_freq,
                          const OptTensor& positions, double eps, bool interleaved) {
    CHECK_FLAT16(qkv, qkv, at::kBFloat16);
    TORCH_CHECK(qkv.dim() == 3 && Hq >= 1 && Hkv >= 1 && qkv.size(2) % (Hq + 2 * Hkv) == 0, "heads: qkv must be [B,T,(Hq + 2 Hkv) D]");
    const int64_t D = qkv.size(2) / (Hq + 2 * Hkv);
    TORCH_CHECK(D >= 8 && D % 8 == 0 && D <= 256 && Hq + 2 * Hkv < (1 << 20), "heads: D must be a multiple of 8, <= 256");
    dpa::HeadsArgs a{};
    a.qkv = qkv.data_ptr();
    TORCH_CHECK(qw.has_value() == kw.has_value(), "heads: both gains or none");
    if (qw.has_value()) {
        CHECK_FLAT((*qw), qkv, at::kFloat); CHECK_FLAT((*kw), qkv, at::kFloat);
        TORCH_CHECK(qw->numel() == D && kw->numel() == D, "heads: gains");
        a.qw = qw->data_ptr<float>(); a.kw = kw->data_ptr<float>();
    }
    a.tokens = qkv.size(0) * qkv.size(1);
    if (inv_freq.has_value()) {
        CHECK_FLAT((*inv_freq), qkv, at::kDouble);
        a.R = (int)(2 * inv_freq->numel());
        TORCH_CHECK(a.R >= 16 && a.R % 16 == 0 && a.R <= D, "heads: rotated channels");
        a.inv_freq = inv_freq->data_ptr<double>();
        if (positions.has_value()) {
            CHECK_FLAT((*positions), qkv, at::kLong);
            TORCH_CHECK(positions->numel() == a.tokens, "heads: positions");
            a.positions = positions->data_ptr<int64_t>();
        }
    }
    TORCH_CHECK(qkv.size(1) < (1ll << 31), "heads: oversized problem");
    a.T = (int)qkv.size(1); a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = (int)D; a.interleaved = interleaved; a.eps = (float)eps;
    return a;
}

std::vector<Tensor> heads_fwd(const Tensor& qkv, int64_t Hq, int64_t Hkv, const OptTensor& qw, const OptTensor& kw, const OptTensor& inv_freq,
                              const OptTensor& positions, double eps, bool interleaved) {
    const dpa::HeadsArgs a = heads_args(qkv, Hq, Hkv, qw, kw, inv_freq, positions, eps, interleaved);
    Guard guard(qkv.device());
    Tensor q = torch::empty({qkv.size(0), qkv.size(1), Hq, a.D}, qkv.options()), k = torch::empty({qkv.size(0), qkv.size(1), Hkv, a.D}, qkv.options());
    if (a.tokens > 0) dpa::heads_fwd(a, q.data_ptr(), k.data_ptr(), cur_stream());
    return {q, k};
}

// -> dqkv, dqw, dkw (the last two undefined without gains)
std::vector<Tensor> heads_bwd(const Tensor& qkv, int64_t Hq, int64_t Hkv, const OptTensor& qw, const OptTensor& kw, const OptTensor& inv_freq,
                              const OptTensor& positions, double eps, bool interleaved, const Tensor& dq, const Tensor& dk, const Tensor& dv) {
    const dpa::HeadsArgs a = heads_args(qkv, Hq, Hkv, qw, kw, inv_freq, positions, eps, interleaved);
    CHECK_FLAT16(dq, qkv, at::kBFloat16); CHECK_FLAT16(dk, qkv, at::kBFloat16); CHECK_FLAT16(dv, qkv, at::kBFloat16);
    TORCH_CHECK(dq.numel() == a.tokens * Hq * a.D && dk.numel() == a.tokens * Hkv * a.D && dv.numel() == dk.numel(), "heads_bwd: shapes");
    Guard guard(qkv.device());
    Tensor dqkv = torch::empty_like(qkv), partial, dw;
    const auto fopt = qkv.options().dtype(at::kFloat);
    if (a.qw != nullptr) {
        if (a.tokens == 0) dw = torch::zeros({2, a.D}, fopt);
        else { dw = torch::empty({2, a.D}, fopt); partial = torch::empty({2, dpa::heads_partial_rows(a.tokens), a.D}, fopt); }
    }
    if (a.tokens > 0)
        dpa::heads_bwd(a, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dqkv.data_ptr(), a.qw != nullptr ? partial.data_ptr<float>() : nullptr,
                       a.qw != nullptr ? dw.data_ptr<float>() : nullptr, a.qw != nullptr ? dw.data_ptr<float>() + a.D : nullptr, cur_stream());
    if (a.qw == nullptr) return {dqkv, Tensor(), Tensor()};
    return {dqkv, dw[0], dw[1]};
}

struct HeadsNode : public torch::autograd::Function<HeadsNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const OptTensor& qw, const OptTensor& kw, const OptTensor& inv_freq,
                                 const OptTensor& positions, int64_t Hq, int64_t Hkv, double eps, bool interleaved) {
        const Tensor x = flat16(qkv);
        auto r = heads_fwd(x, Hq, Hkv, qw, kw, inv_freq, positions, eps, interleaved);
        ctx->save_for_backward({x, bare(qw), bare(kw), bare(inv_freq), bare(positions)});
        ctx->saved_data["Hq"] = Hq; ctx->saved_data["Hkv"] = Hkv; ctx->saved_data["eps"] = eps; ctx->saved_data["interleaved"] = interleaved;
        const int64_t n = Hq + 2 * Hkv;
        return {r[0], r[1], qkv.view({qkv.size(0), qkv.size(1), n, qkv.size(2) / n}).narrow(2, Hq + Hkv, Hkv)};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        auto d = heads_bwd(s[0], ctx->saved_data["Hq"].toInt(), ctx->saved_data["Hkv"].toInt(), opt(s[1]), opt(s[2]), opt(s[3]), opt(s[4]),
                           ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(), flat16(g[0]), flat16(g[1]), flat16(g[2]));
        return {d[0], d[1], d[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
variable_list qk_norm_rotary(const Tensor& qkv, const OptTensor& qw, const OptTensor& kw, const OptTensor& inv_freq, const OptTensor& positions, int64_t Hq,
                             int64_t Hkv, double eps, bool interleaved) {
    return HeadsNode::apply(qkv, qw, kw, inv_freq, positions, Hq, Hkv, eps, interleaved);
}

// ---------------------------------------------------------------- token embedding
bool tok64(const Tensor& tok) {
    TORCH_CHECK(tok.scalar_type() == at::kLong || tok.scalar_type() == at::kInt, "token_embedding: tokens must be int64 or int32");
    return tok.scalar_type() == at::kLong;
}

Tensor token_embedding_fwd(const Tensor& tok, const Tensor& w_, double scale) {
    const Tensor w = flat16(w_);
    CHECK_FLAT16(w, w, at::kBFloat16);
    CHECK_ON(tok, w); TORCH_CHECK(tok.is_contiguous(), "token_embedding: tokens must be contiguous");
    TORCH_CHECK(w.dim() == 2 && w.size(1) >= 8 && w.size(1) % 8 == 0 && w.size(1) < (1 << 24) && w.size(0) >= 1, "token_embedding: table [V, C], C % 8 == 0");
    const bool t64 = tok64(tok);
    Guard guard(w.device());
    auto shape = tok.sizes().vec();
    shape.push_back(w.size(1));
    Tensor y = torch::empty(shape, w.options());
    dpa::token_embedding_fwd(tok.data_ptr(), t64, w.data_ptr(), y.data_ptr(), tok.numel(), (int)w.size(1), w.size(0), (float)scale, cur_stream());
    return y;
}

// dw given: the named rows are added to it; else a whole gradient [V, C] is returned
Tensor token_embedding_bwd(const Tensor& tok, const Tensor& dy_, int64_t V, double scale, const OptTensor& acc) {
    const Tensor dy = flat16(dy_);
    CHECK_FLAT16(dy, dy, at::kBFloat16);
    CHECK_ON(tok, dy); TORCH_CHECK(tok.is_contiguous(), "token_embedding: tokens must be contiguous");
    const int64_t C = dy.size(-1), n = tok.numel();
    TORCH_CHECK(dy.numel() == n * C && C >= 8 && C % 8 == 0 && C < (1 << 24) && V >= 1 && V < (1ll << 30) && n <= (1ll << 27), "token_embedding_bwd: shapes");
    const bool t64 = tok64(tok), add = acc.has_value();
    Guard guard(dy.device());
    const auto fopt = dy.options().dtype(at::kFloat), iopt = dy.options().dtype(at::kInt);
    Tensor dw;
    if (add) {
        dw = *acc;
        CHECK_FLAT(dw, dy, at::kFloat);
        TORCH_CHECK(dw.numel() == V * C, "token_embedding_bwd: accumulator");
    } else {
        dw = torch::empty({V, C}, fopt);
    }
    Tensor scratch = torch::empty({2 * (V + 1) + 2 * n}, iopt), partial;
    const long partials = dpa::token_embedding_partials(n);
    if (partials > 0) partial = torch::empty({partials, C}, fopt);
    int* span = scratch.data_ptr<int>();
    dpa::token_embedding_bwd(tok.data_ptr(), t64, dy.data_ptr(), dw.data_ptr<float>(), add, n, (int)C, V, (float)scale, span, span + 2 * (V + 1), span + 2 * (V + 1) + n,
                             partials > 0 ? partial.data_ptr<float>() : nullptr, cur_stream());
    return dw;
}

struct EmbedNode : public torch::autograd::Function<EmbedNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& tok, const Tensor& w, const Tensor& w_lp, double scale) {
        ctx->save_for_backward({tok});
        ctx->saved_data["scale"] = scale; ctx->saved_data["V"] = w.size(0);
        return token_embedding_fwd(tok, w_lp, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        return {Tensor(), token_embedding_bwd(s[0], g[0], ctx->saved_data["V"].toInt(), ctx->saved_data["scale"].toDouble(), c10::nullopt), Tensor(), Tensor()};
    }
};
Tensor token_embedding(const Tensor& tok, const Tensor& w, const Tensor& w_lp, double scale) { return EmbedNode::apply(tok, w, w_lp, scale); }

// ---------------------------------------------------------------- distillation
// ids and teacher's entries per row, the classes and the temperature as the kernel takes them; logits contiguous, on 16 bytes
dpa::DistillArgs distill_args(const Tensor& logits, const Tensor& ids, const Tensor& teacher, int64_t V, double tau) {
    TORCH_CHECK(logits.dim() == 2, "distill: logits [N, ld]");
    const bool bf = logits.scalar_type() == at::kBFloat16;
    TORCH_CHECK(bf || logits.scalar_type() == at::kFloat, "distill: logits must be bf16 or fp32");
    CHECK_FLAT16(logits, logits, logits.scalar_type());
    CHECK_ON(ids, logits); TORCH_CHECK(ids.is_contiguous() && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt), "distill: ids int64 or int32");
    CHECK_FLAT(teacher, logits, at::kFloat);
    const int64_t N = logits.size(0), ld = logits.size(1);
    TORCH_CHECK(ids.dim() == 2 && ids.sizes() == teacher.sizes() && ids.size(0) == N, "distill: ids and teacher [N, K]");
    const int64_t K = ids.size(1);
    TORCH_CHECK(K >= 1 && K <= dpa::distill_max_entries() && V >= 1 && V <= ld && ld < (1 << 30) && N < (1ll << 31), "distill: sizes");
    TORCH_CHECK(tau > 0.0, "distill: temperature");
    dpa::DistillArgs a{};
    a.logits = logits.data_ptr(); a.ids = ids.data_ptr(); a.teacher = teacher.data_ptr<float>();
    a.N = N; a.ld = ld; a.V = (int)V; a.K = (int)K; a.ids64 = ids.scalar_type() == at::kLong;
    a.inv_tau = (float)(1.0 / tau);
    a.grad_scale = (float)(tau / (N > 0 ? (double)N : 1.0));
    return a;
}

// -> loss [1], and the logits' gradient for an upstream gradient of 1 (undefined unless asked for)
std::vector<Tensor> distill(const Tensor& logits, const Tensor& ids, const Tensor& teacher, int64_t V, double tau, bool want_grad) {
    dpa::DistillArgs a = distill_args(logits, ids, teacher, V, tau);
    const bool bf = logits.scalar_type() == at::kBFloat16;
    Guard guard(logits.device());
    const auto fopt = logits.options().dtype(at::kFloat);
    Tensor loss = torch::empty({1}, fopt), rows = torch::empty({dpa::distill_blocks(bf, a.N, a.ld)}, fopt), d;
    if (want_grad) d = torch::empty_like(logits);
    a.dlogits = want_grad ? d.data_ptr() : nullptr;
    a.row_loss = rows.data_ptr<float>();
    const double n = a.N > 0 ? (double)a.N : 1.0;
    dpa::distill(a, bf, (float)(tau * tau / n), loss.data_ptr<float>(), cur_stream());
    return {loss, d};
}

// the gradient for an upstream gradient of `g`; `d`, if defined, holds the one for 1 and is written only where g is not
Tensor distill_grad(const Tensor& logits, const Tensor& ids, const Tensor& teacher, int64_t V, double tau, const Tensor& g, Tensor d) {
    dpa::DistillArgs a = distill_args(logits, ids, teacher, V, tau);
    CHECK_FLAT(g, logits, at::kFloat);
    TORCH_CHECK(g.numel() == 1, "distill: upstream gradient");
    Guard guard(logits.device());
    a.unless_one = d.defined();
    if (!d.defined()) d = torch::empty_like(logits);
    CHECK_FLAT16(d, logits, logits.scalar_type());
    TORCH_CHECK(d.sizes() == logits.sizes(), "distill: gradient");
    a.dlogits = d.data_ptr();
    a.upstream = g.data_ptr<float>();
    dpa::distill(a, logits.scalar_type() == at::kBFloat16, 0.f, nullptr, cur_stream());
    return d;
}
// A saved tensor apart from the node's others, so that backward can let go of it while the node lives on.  Saved-tensor hooks
// (offloading, checkpointing) see it as they see those.
struct Kept : public torch::CustomClassHolder {
    torch::autograd::SavedVariable t;
    explicit Kept(const Tensor& x) : t(x, false) {}
};

// When a gradient will be asked for the forward kernel writes it beside the loss, for an upstream gradient of 1; backward
// forms it again only when the real one is not 1 (tested on the device), and so does a second backward through the node.
struct DistillNode : public torch::autograd::Function<DistillNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits_, const Tensor& ids, const Tensor& teacher, int64_t V, double tau, bool for_backward) {
        const Tensor logits = flat16(logits_);                                 // rows lie on 16 bytes as those of the gradient do
        auto r = distill(logits, ids, teacher, V, tau, for_backward);
        if (for_backward) {
            ctx->save_for_backward({logits, ids, teacher});
            ctx->saved_data["V"] = V; ctx->saved_data["tau"] = tau; ctx->saved_data["d"] = at::IValue::make_capsule(c10::make_intrusive<Kept>(r[1]));
        }
        return r[0].view(at::IntArrayRef());
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        Tensor d;
        const auto at = ctx->saved_data.find("d");
        if (at != ctx->saved_data.end()) {
            d = c10::static_intrusive_pointer_cast<Kept>(at->second.toCapsule())->t.unpack();
            ctx->saved_data.erase(at);
            // a hook kept it, or made something else of it
            if (d.use_count() > 1 || d.storage().use_count() > 1 || !d.is_contiguous() || !on16(d)) d = Tensor();
        }
        return {distill_grad(s[0], s[1], s[2], ctx->saved_data["V"].toInt(), ctx->saved_data["tau"].toDouble(), g[0].reshape({1}), d),
                Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
Tensor distillation_loss(const Tensor& logits, const Tensor& ids, const Tensor& teacher, int64_t V, double tau) {
    return DistillNode::apply(logits, ids, teacher, V, tau, at::GradMode::is_enabled() && logits.requires_grad());
}
}  // namespace

void bind_lm(pybind11::module_& m) {
    m.def("attention_ex", &attention_ex);
    m.def("qk_norm_rotary", &qk_norm_rotary);
    m.def("token_embedding", &token_embedding);
    m.def("token_embedding_fwd", &token_embedding_fwd);
    m.def("token_embedding_bwd", &token_embedding_bwd);
    m.def("distillation_loss", &distillation_loss);
}
