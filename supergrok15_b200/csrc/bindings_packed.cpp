// Bindings of the operators of packed language-model training: attention over packed sequences, cross-entropy of a linear head.
#include <cmath>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "bindings_decl.h"
#include "mt_host.h"
#include "linear_ce.h"
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

// A 16-bit view whose base or pitches the tensor-core kernels cannot load from is copied once: they then take it (a few per cent of their time
// for short sequences, less for long ones; the CUDA cores take over a hundred times longer).  Other views are used where they are.
Tensor loadable(const Tensor& t) {
    if (t.dim() != 3 || t.element_size() != 2 || t.size(2) % 8 != 0 || t.numel() == 0) return t;
    if (sg::packed_tma_view(t.data_ptr(), t.stride(0), t.stride(1), t.size(0), t.size(1))) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

sg::PackedAttn packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, bool causal, double scale) {
    TORCH_CHECK_VALUE(q.is_cuda() && q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(2) == k.size(2),
                      "attention_packed: q [rows, heads, hd] and k, v [rows, kv_heads, hd] expected, got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
    TORCH_CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "attention_packed: ", q.size(1), " query heads are not a multiple of ", k.size(1), " key heads");
    TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 1 && cu.scalar_type() == at::kInt, "attention_packed: cu_seqlens must be a vector of sequences + 1 int32 or int64 offsets");
    TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() && v.device() == q.device() &&
                      cu.device() == q.device(), "attention_packed: q, k and v need one dtype, and all tensors one device");
    TORCH_CHECK_VALUE((q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat) && q.size(2) >= 1 && q.size(2) <= 128,
                      "attention_packed: bf16, fp16 or fp32 with head sizes up to 128 on CUDA, got ", q.scalar_type(), " with ", q.size(2));
    TORCH_CHECK_VALUE(q.size(0) < ((int64_t)1 << 30) && cu.numel() < ((int64_t)1 << 30) && q.size(1) <= 65535, "attention_packed: fewer than 2^30 rows, 65,535 heads at most");
    TORCH_CHECK(cu.is_contiguous() && head_rows_ok(q) && head_rows_ok(k) && head_rows_ok(v), "attention_packed: the last index must be contiguous");
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
std::vector<Tensor> packed_attn_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu, bool causal, double scale, bool train, Tensor err) {
    const Tensor q = loadable(q_), k = loadable(k_), v = loadable(v_);
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
    const int dt = dtype_code(q);
    auto st = at::cuda::getCurrentCUDAStream();
    const int rc = sg::packed_attn_sm100_takes(dt, p) ? sg::packed_attn_sm100_fwd(dt, p, err.data_ptr<int>(), st) : sg::packed_attn_fwd(dt, p, st);
    TORCH_CHECK(rc == 0, "attention_packed: launch failed (code ", rc, ")");
    return {out, lo, lse};
}

// gradients of packed_attn_fwd: (dq, dk, dv), dense
std::vector<Tensor> packed_attn_bwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu, const Tensor& out, const Tensor& lo, const Tensor& lse,
                                    const Tensor& dout_, bool causal, double scale, Tensor err) {
    const Tensor q = loadable(q_), k = loadable(k_), v = loadable(v_);
    sg::PackedAttn p = packed_args(q, k, v, cu, causal, scale);
    c10::cuda::CUDAGuard guard(q.device());
    Tensor dout = loadable(dout_.contiguous());
    TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() && dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() &&
                out.scalar_type() == q.scalar_type() && dout.device() == q.device(), "attention_packed: out and its gradient like q");
    TORCH_CHECK(lo.numel() == (q.scalar_type() == at::kFloat ? 0 : q.numel()) && lo.is_contiguous() && lo.scalar_type() == q.scalar_type(), "attention_packed: rest of out");
    TORCH_CHECK(lse.is_contiguous() && lse.scalar_type() == at::kFloat && lse.numel() == q.size(0) * q.size(1), "attention_packed: lse fp32 [heads, rows]");
    Tensor dq = at::empty(q.sizes(), out.options()), dk = at::empty(k.sizes(), out.options()), dv = at::empty(v.sizes(), out.options());
    if (q.numel() == 0) return {dq, dk.zero_(), dv.zero_()};               // no rows, or no query heads
    Tensor delta = at::empty_like(lse);
    p.out = out.data_ptr(); p.out_lo = lo.numel() ? lo.data_ptr() : nullptr;
    p.lse = lse.data_ptr<float>(); p.dout = dout.data_ptr(); p.delta = delta.data_ptr<float>();
    p.dq = dq.data_ptr(); p.dk = dk.data_ptr(); p.dv = dv.data_ptr();
    const int dt = dtype_code(q);
    auto st = at::cuda::getCurrentCUDAStream();
    Tensor parts, units;
    if (sg::packed_attn_sm100_takes(dt, p)) {
        const int split = sg::packed_attn_sm100_split(p);
        if (split > 1) { parts = at::empty({2 * split * k.numel()}, lse.options()); p.kv_parts = parts.data_ptr<float>(); }
        const int64_t n = sg::packed_attn_sm100_units(dt, p);
        if (n > 0) { units = at::empty({n}, lse.options()); p.units = units.data_ptr<float>(); }
    }
    const int rc = sg::packed_attn_sm100_takes(dt, p) ? sg::packed_attn_sm100_bwd(dt, p, err.data_ptr<int>(), st) : sg::packed_attn_bwd(dt, p, st);
    TORCH_CHECK(rc == 0, "attention_packed: launch of the backward pass failed (code ", rc, ")");
    return {dq, dk, dv};
}

struct PackedAttnNode : Function<PackedAttnNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu, bool causal, double scale, bool train, const Tensor& err) {
        const Tensor q = loadable(q_), k = loadable(k_), v = loadable(v_);   // the copy, where there is one, is what the backward pass reads
        auto r = packed_attn_fwd(q, k, v, cu, causal, scale, train, err);
        if (!train) return r[0];
        ctx->save_for_backward({q, k, v, cu, r[0], r[1], r[2]});
        ctx->saved_data["err"] = err;                                     // the process's time-out flag itself, not a saved tensor
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        return r[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        refuse_second_order("attention_packed");
        const auto s = ctx->get_saved_variables();
        auto r = packed_attn_bwd(s[0], s[1], s[2], s[3], s[4], s[5], s[6], dy[0], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
                                 ctx->saved_data["err"].toTensor());
        return {r[0], r[1], r[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ---- cross-entropy of a linear head
// Rows of a piece: u (rows x vocabulary, the type of x) takes 256 MB at most, but at least 256 rows go together, so that w is not read for
// less work than that.  A pass without gradients keeps two floats per row and tile of columns only, to the same bound.  65,536 rows at most:
// tile rows are the second dimension of a grid, which has 65,535, and dw is one chain of fp32 additions over a piece, in which terms below half a
// step of the sum are lost (8,400,000 rows of 5 columns in two pieces: dw 0.2 % off).
int64_t lce_piece_rows(int64_t rows, int64_t ldu, int64_t elem, bool train) {
    const int64_t each = train ? ldu * elem : (ldu + sg::LCE_COLUMNS - 1) / sg::LCE_COLUMNS * (int64_t)sizeof(float2), top = 65536;
    int64_t most = ((int64_t)256 << 20) / each;
    if (most > top) most = top;
    most = most / 256 * 256;
    if (most < 256) most = 256;
    if (rows <= most) return rows;
    const int64_t pieces = (rows + most - 1) / most;
    return ((rows + pieces - 1) / pieces + 255) / 256 * 256;
}

// 16-bit rows that the tensor-core kernels cannot load (base or pitch not on 16 bytes) are copied once
Tensor loadable_rows(const Tensor& t) {
    if (t.dim() != 2 || t.element_size() != 2 || t.size(1) % 8 != 0 || t.numel() == 0) return t;
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(1) == 1 && t.stride(0) > 0 && t.stride(0) % 8 == 0) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

struct LceShape {
    sg::LceArgs a{};
    int dtype = 0;
    int64_t rows = 0, piece = 0, elem = 0;
    // the piece of the counted rows from r0 on (sized as if all rows were counted)
    sg::LceArgs at(int64_t r0) const {
        sg::LceArgs p = a;
        p.first = (int)r0;
        p.rows = (int)(rows - r0 < piece ? rows - r0 : piece);
        p.x = (const char*)a.x + r0 * a.ldx * elem;
        p.target = a.target ? a.target + r0 : nullptr;
        p.loss = a.loss ? a.loss + r0 : nullptr;
        return p;                                                         // u, stats, z_target and row_scale are those of any piece
    }
    int64_t last() const { return rows == 0 ? 0 : (rows - 1) / piece * piece; }      // first row of the last piece
};

LceShape lce_shape(int64_t rows, const Tensor& w, bool train) {
    LceShape s;
    s.dtype = dtype_code(w);
    s.elem = w.element_size();
    s.rows = rows;
    s.a.w = w.data_ptr(); s.a.ldw = w.stride(0);
    s.a.V = (int)w.size(0); s.a.D = (int)w.size(1);
    s.a.ldx = sg::lce_pitch(w.size(1), s.elem);
    s.a.ldu = sg::lce_pitch(w.size(0), s.elem);
    s.piece = lce_piece_rows(s.rows, s.a.ldu, s.elem, train);
    return s;
}

// What a training pass keeps from forward to backward: the counted rows xc (scaled where lce_scales_rows says so), where they came from (keep:
// [rows] places, then the count, the counter of the row pass, 1 / count as a float and the last piece's row scales as floats), u or d of the
// last piece, and with several pieces fp32 dx and dw of the others.
enum { KEEP_COUNT = 0, KEEP_DONE = 1, KEEP_INV = 2, KEEP_MORE = 4 };

// Returns (loss, xc, keep, d, dx of earlier pieces, dw of earlier pieces).  The gradient products of the last piece are left to the backward
// pass, which writes them in the final type; of the pieces before it the products are taken here, because their d makes room for the next one's.
std::vector<Tensor> lce_fwd(const Tensor& x, const Tensor& w_, const Tensor& t, int64_t ignore_index, bool need_x, bool need_w, Tensor err) {
    TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && w_.dim() == 2 && t.dim() == 1 && x.size(1) == w_.size(1) && t.size(0) == x.size(0),
                      "linear_cross_entropy: x [..., D], weight [vocabulary, D] and target [...] expected, got ", x.sizes(), ", ", w_.sizes(), ", ", t.sizes());
    TORCH_CHECK_VALUE(w_.scalar_type() == x.scalar_type() && t.scalar_type() == at::kLong && w_.device() == x.device() && t.device() == x.device(),
                      "linear_cross_entropy: x and weight need one dtype, target int64, and all tensors one device");
    TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat,
                      "linear_cross_entropy: bf16, fp16 or fp32 on CUDA, got ", x.scalar_type());
    TORCH_CHECK_VALUE(w_.size(0) >= 1 && w_.size(0) < (1 << 22) && x.size(1) >= 1 && x.size(1) < (1 << 22) && x.size(0) < ((int64_t)1 << 30),
                      "linear_cross_entropy: vocabulary and width from 1 to below 2^22, fewer than 2^30 rows");
    TORCH_CHECK(t.is_contiguous() && (x.stride(1) == 1 || x.size(1) == 1) && (w_.stride(1) == 1 || w_.size(1) == 1),
                "linear_cross_entropy: the last index must be contiguous");
    const bool train = need_x || need_w;
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor w = loadable_rows(w_);
    LceShape s = lce_shape(x.size(0), w, train);
    auto st = at::cuda::getCurrentCUDAStream();
    const auto fo = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
    const auto xo = x.options().memory_format(at::MemoryFormat::Contiguous);
    const Tensor none = at::empty({0}, fo);
    if (s.rows == 0) return {at::zeros({}, fo), none, none, none, none, none};
    Tensor loss = at::empty({}, fo), xc = at::empty({s.rows, s.a.ldx}, xo), keep = at::empty({s.rows + KEEP_MORE + (train ? s.piece : 0)}, fo.dtype(at::kInt));
    Tensor u = train ? at::empty({s.piece, s.a.ldu}, xo) : none, dx = none, dw = none;
    s.a.x = xc.data_ptr();
    const int64_t tiles = (s.a.V + sg::LCE_COLUMNS - 1) / sg::LCE_COLUMNS, blocks = sg::lce_gather_blocks((int)s.rows);
    // scratch of this pass: targets [rows] (8 bytes each), statistics [piece][tiles] (8), target logits [piece], losses [rows], block counts
    Tensor scratch = at::empty({2 * s.rows + 2 * s.piece * tiles + s.piece + s.rows + blocks}, fo);
    float* f = scratch.data_ptr<float>();
    int64_t* tc = reinterpret_cast<int64_t*>(f);
    s.a.stats = reinterpret_cast<float2*>(f + 2 * s.rows);
    s.a.z_target = f + 2 * s.rows + 2 * s.piece * tiles;
    s.a.loss = s.a.z_target + s.piece;
    int* kept = keep.data_ptr<int>() + s.rows;
    s.a.target = tc;
    s.a.count = kept + KEEP_COUNT;
    s.a.u = train ? u.data_ptr() : nullptr;
    s.a.loss_all = s.a.loss;
    s.a.out_loss = loss.data_ptr<float>();
    s.a.inv_count = reinterpret_cast<float*>(kept + KEEP_INV);
    s.a.done = reinterpret_cast<unsigned*>(kept + KEEP_DONE);
    s.a.row_scale = train && sg::lce_scales_rows(s.dtype, s.a) ? reinterpret_cast<float*>(kept + KEEP_MORE) : nullptr;
    int rc = sg::lce_gather(s.dtype, x.data_ptr(), x.stride(0), t.data_ptr<int64_t>(), ignore_index, (int)s.rows, s.a.V, s.a.D, keep.data_ptr<int>(), xc.data_ptr(), tc,
                            kept + KEEP_COUNT, s.a.done, reinterpret_cast<int*>(s.a.loss + s.rows), st);
    const int64_t last = s.last();
    if (train && last > 0 && need_x) dx = at::empty({last, x.size(1)}, fo);
    if (train && last > 0 && need_w) dw = at::empty(w.sizes(), fo);
    for (int64_t r0 = 0; r0 < s.rows && rc == 0; r0 += s.piece) {
        const sg::LceArgs a = s.at(r0);
        rc = sg::lce_logits(s.dtype, a, err.data_ptr<int>(), st);
        if (rc == 0) rc = sg::lce_rows(s.dtype, a, r0 == last, st);
        if (rc == 0 && train && r0 < last) {
            sg::LceGrads g{};
            Tensor part;
            if (need_x) {
                g.parts = sg::lce_dx_parts(s.dtype, a, need_w, &g.row_pitch);
                part = g.parts == 1 && g.row_pitch == a.rows ? dx.narrow(0, r0, a.rows) : at::empty({g.parts * g.row_pitch, x.size(1)}, fo);
                g.dx_part = part.data_ptr<float>();
            }
            g.dw = need_w ? dw.data_ptr() : nullptr;
            g.dw_prev = need_w && r0 > 0 ? dw.data_ptr<float>() : nullptr;
            g.f32_dw = true;
            rc = sg::lce_grads(s.dtype, a, g, err.data_ptr<int>(), st);
            if (rc == 0 && need_x && part.size(0) != a.rows)
                rc = sg::lce_add_parts(g.dx_part, g.parts, g.row_pitch * x.size(1), a.rows * x.size(1), dx.data_ptr<float>() + r0 * x.size(1), st);
        }
    }
    TORCH_CHECK(rc == 0, "linear_cross_entropy: launch failed (code ", rc, ")");
    return {loss, xc, keep, u, dx, dw};
}

std::vector<Tensor> lce_bwd(const Tensor& w_, const Tensor& xc, const Tensor& keep, const Tensor& u, const Tensor& dx32, const Tensor& dw32, const Tensor& gout_,
                            at::IntArrayRef x_size, bool need_x, bool need_w, Tensor err) {
    c10::cuda::CUDAGuard guard(w_.device());
    auto st = at::cuda::getCurrentCUDAStream();
    Tensor dx, dw;
    const auto xo = w_.options().memory_format(at::MemoryFormat::Contiguous);
    const int64_t rows = x_size[0], D = w_.size(1);
    if (rows == 0) return {need_x ? at::zeros(x_size, xo) : dx, need_w ? at::zeros(w_.sizes(), xo) : dw};
    const Tensor w = loadable_rows(w_);
    LceShape s = lce_shape(rows, w, true);
    Tensor gout = gout_.to(at::kFloat).reshape({1}).contiguous();
    if (need_x) dx = at::empty(x_size, xo);
    if (need_w) dw = at::empty(w.sizes(), xo);
    const int64_t last = s.last();
    TORCH_CHECK(xc.is_contiguous() && xc.size(0) == rows && xc.size(1) == s.a.ldx && u.is_contiguous() && u.dim() == 2 && u.size(0) == s.piece && u.size(1) == s.a.ldu &&
                u.scalar_type() == w.scalar_type() && keep.numel() == rows + KEEP_MORE + s.piece && (!need_x || dx32.numel() == last * D) &&
                (!need_w || dw32.numel() == (last > 0 ? w.numel() : 0)), "linear_cross_entropy: not what the forward pass left");
    int* kept = keep.data_ptr<int>() + rows;
    s.a.x = xc.data_ptr();
    s.a.u = u.data_ptr();
    s.a.count = kept + KEEP_COUNT;
    s.a.row_scale = sg::lce_scales_rows(s.dtype, s.a) ? reinterpret_cast<float*>(kept + KEEP_MORE) : nullptr;
    const sg::LceArgs a = s.at(last);
    sg::LceGrads g{};
    Tensor part;
    if (need_x) {
        g.parts = sg::lce_dx_parts(s.dtype, a, need_w, &g.row_pitch);
        part = at::empty({g.parts * g.row_pitch, D}, gout.options());
        g.dx_part = part.data_ptr<float>();
    }
    g.dw = need_w ? dw.data_ptr() : nullptr;
    g.dw_prev = need_w && last > 0 ? dw32.data_ptr<float>() : nullptr;
    g.gout = gout.data_ptr<float>();
    g.inv_count = reinterpret_cast<const float*>(kept + KEEP_INV);
    int rc = sg::lce_grads(s.dtype, a, g, err.data_ptr<int>(), st);
    if (rc == 0 && need_x)
        rc = sg::lce_scatter(s.dtype, keep.data_ptr<int>(), (int)rows, (int)D, (int)last, last > 0 ? dx32.data_ptr<float>() : nullptr, g.dx_part, g.parts, g.row_pitch,
                             g.gout, g.inv_count, dx.data_ptr(), st);
    TORCH_CHECK(rc == 0, "linear_cross_entropy: launch of the backward pass failed (code ", rc, ")");
    return {dx, dw};
}

struct LceNode : Function<LceNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& t, int64_t ignore_index, bool need_x, bool need_w, const Tensor& err) {
        auto r = lce_fwd(x, w, t, ignore_index, need_x, need_w, err);
        if (need_x || need_w) {
            ctx->save_for_backward({w, r[1], r[2], r[3], r[4], r[5]});
            ctx->saved_data["err"] = err;                                 // the process's time-out flag itself, not a saved tensor
            ctx->saved_data["x"] = x.sizes();
            ctx->saved_data["need_x"] = need_x;
            ctx->saved_data["need_w"] = need_w;
        }
        return r[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        refuse_second_order("linear_cross_entropy");
        const auto s = ctx->get_saved_variables();
        auto r = lce_bwd(s[0], s[1], s[2], s[3], s[4], s[5], dy[0], ctx->saved_data["x"].toIntVector(), ctx->saved_data["need_x"].toBool(),
                         ctx->saved_data["need_w"].toBool(), ctx->saved_data["err"].toTensor());
        return {r[0], r[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
}  // namespace

void register_packed(pybind11::module_& m) {
    m.def("lce_fwd", &lce_fwd);
    m.def("lce_bwd", [](const Tensor& w, const Tensor& xc, const Tensor& keep, const Tensor& u, const Tensor& dx, const Tensor& dw, const Tensor& gout,
                        std::vector<int64_t> x_size, bool need_x, bool need_w, Tensor err) { return lce_bwd(w, xc, keep, u, dx, dw, gout, x_size, need_x, need_w, err); });
    m.def("lce_piece_rows", &lce_piece_rows);
    // x [..., D] and target [...] of any strides
    m.def("lce_node", [](const Tensor& x_, const Tensor& w_, const Tensor& t_, int64_t ignore_index, const Tensor& err) {
        TORCH_CHECK_VALUE(x_.dim() >= 1 && w_.dim() == 2 && t_.sizes() == x_.sizes().slice(0, x_.dim() - 1),
                          "linear_cross_entropy: x [..., D], weight [vocabulary, D] and target [...] expected, got ", x_.sizes(), ", ", w_.sizes(), ", ", t_.sizes());
        const bool grad = at::GradMode::is_enabled();
        Tensor x = x_.dim() == 2 ? x_ : x_.reshape({t_.numel(), x_.size(-1)}), w = w_, t = t_.dim() == 1 ? t_ : t_.reshape({-1});
        if (x.stride(1) != 1) x = x.contiguous();
        if (w.stride(1) != 1) w = w.contiguous();
        if (!t.is_contiguous()) t = t.contiguous();
        return LceNode::apply(x, w, t, ignore_index, grad && x.requires_grad(), grad && w.requires_grad(), err);
    });
    m.def("packed_attn_fwd", &packed_attn_fwd);
    m.def("packed_attn_bwd", &packed_attn_bwd);
    m.def("packed_attn_node", [](const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu_, bool causal, c10::optional<double> scale, const Tensor& err) {
        const auto rows = [](const Tensor& t) { return t.dim() != 3 || t.stride(2) == 1 ? t : t.contiguous(); };
        const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
        Tensor cu = cu_.scalar_type() == at::kLong ? cu_.to(at::kInt) : cu_;
        if (!cu.is_contiguous()) cu = cu.contiguous();
        const bool train = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
        return PackedAttnNode::apply(q, k, v, cu, causal, scale.has_value() ? *scale : (q.dim() == 3 && q.size(2) > 0 ? 1.0 / std::sqrt((double)q.size(2)) : 1.0), train, err);
    });
}
}  // namespace sgb
