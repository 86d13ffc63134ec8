// Bindings of the operators of packed language-model training: attention over packed sequences.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "bindings_decl.h"
#include "mt_host.h"
#include "packed_attn.h"

namespace sgb {
namespace py = pybind11;
namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// A gradient pass that is to be differentiated again would lose terms without a word.
void refuse_second_order(const char* what) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated (create_graph=True)");
}

bool head_rows_ok(const Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1; }

sg::PackedAttn packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, bool causal, double scale) {
    TORCH_CHECK(q.is_cuda() && q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(2) == k.size(2),
                "attention_packed: q [rows, heads, head_dim], k and v [rows, kv_heads, head_dim]");
    TORCH_CHECK(k.device() == q.device() && v.device() == q.device() && cu.device() == q.device(), "attention_packed: all tensors on one device");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "attention_packed: q, k and v of one dtype");
    TORCH_CHECK(q.size(0) < ((int64_t)1 << 30) && cu.numel() < ((int64_t)1 << 30), "attention_packed: fewer than 2^30 rows");
    TORCH_CHECK(k.size(1) > 0 && q.size(1) % k.size(1) == 0 && q.size(1) <= 65535, "attention_packed: heads must be a multiple of kv_heads, 65,535 at most");
    TORCH_CHECK(q.size(2) >= 1 && q.size(2) <= 128, "attention_packed: head_dim 1 to 128");
    TORCH_CHECK(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.is_contiguous() && cu.numel() >= 1, "attention_packed: cu_seqlens [sequences + 1]");
    TORCH_CHECK(head_rows_ok(q) && head_rows_ok(k) && head_rows_ok(v), "attention_packed: the last index must be contiguous");
    sg::PackedAttn p{};
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr();
    p.q_ld = q.stride(0); p.k_ld = k.stride(0); p.v_ld = v.stride(0);
    p.q_hs = q.stride(1); p.k_hs = k.stride(1); p.v_hs = v.stride(1);
    p.seqs = {cu.data_ptr<int>(), (int)cu.numel() - 1, (int)q.size(0)};
    p.heads = (int)q.size(1); p.group = (int)(q.size(1) / k.size(1)); p.hd = (int)q.size(2);
    p.causal = causal; p.scale = (float)scale;
    return p;
}

// returns (out, what the rounding took from it, lse [heads, rows]); without `train` the last two are empty
std::vector<Tensor> packed_attn_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, bool causal, double scale, bool train) {
    sg::PackedAttn p = packed_args(q, k, v, cu, causal, scale);
    c10::cuda::CUDAGuard guard(q.device());
    const auto dense = q.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor out = at::empty(q.sizes(), dense);
    Tensor lo = train && q.scalar_type() != at::kFloat ? at::empty(q.sizes(), dense) : at::empty({0}, dense);
    Tensor lse = at::empty({train ? q.size(1) : 0, q.size(0)}, q.options().dtype(at::kFloat));
    if (q.numel() == 0) return {out, lo, lse};
    p.out = out.data_ptr();
    p.out_lo = lo.numel() ? lo.data_ptr() : nullptr;
    p.lse = train ? lse.data_ptr<float>() : nullptr;
    const int rc = sg::packed_attn_fwd(dtype_code(q), p, at::cuda::getCurrentCUDAStream());
    TORCH_CHECK(rc == 0, "attention_packed: launch failed (code ", rc, ")");
    return {out, lo, lse};
}

// gradients of packed_attn_fwd: (dq, dk, dv), dense
std::vector<Tensor> packed_attn_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, const Tensor& out, const Tensor& lo, const Tensor& lse,
                                    const Tensor& dout_, bool causal, double scale) {
    sg::PackedAttn p = packed_args(q, k, v, cu, causal, scale);
    c10::cuda::CUDAGuard guard(q.device());
    Tensor dout = dout_.contiguous();
    TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() && dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() &&
                out.scalar_type() == q.scalar_type() && dout.device() == q.device(), "attention_packed: out and its gradient like q");
    TORCH_CHECK(lo.numel() == (q.scalar_type() == at::kFloat ? 0 : q.numel()) && lo.is_contiguous() && lo.scalar_type() == q.scalar_type(), "attention_packed: rest of out");
    TORCH_CHECK(lse.is_contiguous() && lse.scalar_type() == at::kFloat && lse.numel() == q.size(0) * q.size(1), "attention_packed: lse fp32 [heads, rows]");
    Tensor dq = at::empty(q.sizes(), out.options()), dk = at::empty(k.sizes(), out.options()), dv = at::empty(v.sizes(), out.options());
    if (q.numel() == 0) return {dq, dk, dv};
    Tensor delta = at::empty_like(lse);
    p.out = out.data_ptr(); p.out_lo = lo.numel() ? lo.data_ptr() : nullptr;
    p.lse = lse.data_ptr<float>(); p.dout = dout.data_ptr(); p.delta = delta.data_ptr<float>();
    p.dq = dq.data_ptr(); p.dk = dk.data_ptr(); p.dv = dv.data_ptr();
    const int rc = sg::packed_attn_bwd(dtype_code(q), p, at::cuda::getCurrentCUDAStream());
    TORCH_CHECK(rc == 0, "attention_packed: launch of the backward pass failed (code ", rc, ")");
    return {dq, dk, dv};
}

struct PackedAttnNode : Function<PackedAttnNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, bool causal, double scale, bool train) {
        auto r = packed_attn_fwd(q, k, v, cu, causal, scale, train);
        if (!train) return r[0];
        ctx->save_for_backward({q, k, v, cu, r[0], r[1], r[2]});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        return r[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        refuse_second_order("attention_packed");
        const auto s = ctx->get_saved_variables();
        auto r = packed_attn_bwd(s[0], s[1], s[2], s[3], s[4], s[5], s[6], dy[0], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
        return {r[0], r[1], r[2], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
}  // namespace

void register_packed(pybind11::module_& m) {
    m.def("packed_attn_fwd", &packed_attn_fwd);
    m.def("packed_attn_bwd", &packed_attn_bwd);
    m.def("packed_attn_node", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, bool causal, double scale, bool train) {
        return PackedAttnNode::apply(q, k, v, cu, causal, scale, train);
    });
}
}  // namespace sgb
