// ROTARY and ATTENTION (additive): a transformer block's position rotation and
// its masked softmax attention. Both compute in float32 and round once to their
// result's type; their adjoints are ops of their own (a rotation back, and
// ATTENTION_GRAD), which have no adjoint in turn.
#include <cmath>
#include <stdexcept>
#include <string>
#include "core/ops/api.h"
#include "core/shape.h"
#include "core/adjoint.h"
#include "core/registry.h"

namespace ormi {
    using ops::OpEnum;
    using NodeVec = std::vector<std::shared_ptr<Node>>;

    static bool is_float(DType d) { return d == DType::Float32 || d == DType::BFloat16 || d == DType::Float16; }

    static void require(bool ok, const char* op, const char* what) {
        if (!ok) throw std::runtime_error(std::string(op) + " " + what);
    }

    static void check_constant(const std::shared_ptr<Node>& n, const std::shared_ptr<Node>& x, DType dtype, const char* op, const char* what) {
        const std::string name(what);
        require(n->device.type == x->device.type, op, ("got " + name + " on another device.").c_str());
        require(n->dtype == dtype, op, ("takes " + name + " as " + dtype_name(dtype) + ".").c_str());
        require(!n->requires_grad, op, ("has no gradient for " + name + ".").c_str());
    }

    namespace ops {
        NodePtr rotary(NodePtr x, NodePtr cos, NodePtr sin, NodePtr positions, int offset, bool interleaved, DType dtype) {
            require(x && cos && sin, "ROTARY", "got a null operand.");
            const auto& xs = x->view.shape;
            require(xs.size() == 4, "ROTARY", "takes (batch, length, heads, features).");
            require(is_float(x->dtype) && is_float(dtype), "ROTARY", "takes and gives float32, bfloat16 or float16.");
            check_constant(cos, x, DType::Float32, "ROTARY", "its tables");
            check_constant(sin, x, DType::Float32, "ROTARY", "its tables");
            require(cos->view.shape.size() == 2 && cos->view.shape == sin->view.shape, "ROTARY", "takes tables of one shape (positions, pairs).");
            require(2ll * cos->view.shape[1] <= xs[3], "ROTARY", "tables hold more pairs than the features.");
            RotaryAttrs a;
            a.part = 2 * cos->view.shape[1];
            a.interleaved = interleaved;
            a.offset = offset;
            a.dtype = dtype;
            NodeVec parents{x, cos, sin};
            if (positions) {
                check_constant(positions, x, DType::Int32, "ROTARY", "positions");
                const auto& ps = positions->view.shape;
                const bool one = ps.size() == 1 && ps[0] == xs[1];
                const bool each = ps.size() == 2 && (ps[0] == xs[0] || ps[0] == 1) && ps[1] == xs[1];
                require(one || each, "ROTARY", "takes positions (length) or (batch, length).");
                a.positions = true;
                parents.push_back(positions);
            } else {
                // Positions on the device are checked by the kernel (NaN), these here.
                require(offset >= 0 && (a.part == 0 || (long long)offset + xs[1] <= cos->view.shape[0]), "ROTARY", "positions lie outside the tables.");
            }
            return std::make_shared<Node>(OpEnum::ROTARY, parents, x->device, a);
        }

        NodePtr attention(NodePtr q, NodePtr k, NodePtr v, float scale, float cap, bool causal, NodePtr slopes, NodePtr documents,
                          NodePtr prefix, NodePtr lengths) {
            const char* op = "ATTENTION";
            require(q && k && v, op, "got a null operand.");
            require(q->device.type == k->device.type && q->device.type == v->device.type, op, "got operands on different devices.");
            const auto& qs = q->view.shape;
            const auto& ks = k->view.shape;
            require(qs.size() == 4 && ks.size() == 4, op, "takes (batch, length, heads, features).");
            require(ks == v->view.shape, op, "takes k and v of one shape.");
            require(is_float(q->dtype) && q->dtype == k->dtype && q->dtype == v->dtype, op, "takes q, k and v of one type: float32, bfloat16 or float16.");
            require(qs[0] == ks[0] && qs[3] == ks[3], op, "takes q and k of one batch and as many features.");
            require(ks[2] > 0 && qs[2] > 0 && qs[2] % ks[2] == 0, op, "takes query heads in multiples of the key heads.");
            require(qs[3] >= 1 && qs[3] <= 256, op, "takes 1 to 256 features per head.");
            require(std::isfinite(scale), op, "takes a finite scale.");
            require(std::isfinite(cap) && cap >= 0.0f, op, "takes a cap of zero (none) or more.");
            require(causal || !prefix, op, "takes a prefix with causal only.");
            AttentionAttrs a;
            a.scale = scale;
            a.cap = cap;
            a.causal = causal;
            NodeVec parents{q, k, v};
            auto rule = [&](const NodePtr& n, DType dtype, std::vector<int> shape, const char* what, bool& flag) {
                if (!n) return;
                check_constant(n, q, dtype, op, what);
                require(n->view.shape == shape, op, (std::string("got ") + what + " of another shape.").c_str());
                flag = true;
                parents.push_back(n);
            };
            rule(slopes, DType::Float32, {qs[2]}, "slopes (heads)", a.slopes);
            rule(documents, DType::Int32, {ks[0], ks[1]}, "documents (batch, keys)", a.documents);
            rule(prefix, DType::Int32, {ks[0]}, "prefix (batch)", a.prefix);
            rule(lengths, DType::Int32, {ks[0]}, "lengths (batch)", a.lengths);
            a.saved = std::make_shared<AttentionAttrs::Saved>();
            return std::make_shared<Node>(OpEnum::ATTENTION, parents, q->device, a);
        }
    }

    static std::vector<int> first_shape(const NodeVec& parents, const OpAttributes&) { return parents[0]->view.shape; }
    static std::vector<int> grad_shape(const NodeVec& parents, const OpAttributes& attrs) {
        return parents[2 + std::get<AttentionAttrs>(attrs).which]->view.shape;
    }

    // g of the dtype that an op's gradient kernel reads; a gradient that is one
    // already, or a backward pass's seed times one, is read as it is.
    static std::shared_ptr<Node> as_dtype(const std::shared_ptr<Node>& g, DType dtype) {
        return g->dtype == dtype ? g : std::make_shared<Node>(OpEnum::CAST, NodeVec{g}, g->device, CastAttrs{dtype});
    }

    // The rotation is orthogonal (times the tables' magnitude): its adjoint turns back.
    static void adjoint_rotary(std::shared_ptr<Node> n) {
        auto x = n->parents[0];
        if (!x->requires_grad) return;
        auto a = std::get<RotaryAttrs>(n->attrs);
        require(!a.inverse, "ROTARY", "has no second gradient.");
        a.inverse = true;
        a.upstream = n->dtype;
        a.dtype = x->dtype;
        NodeVec parents{n->grad};
        parents.insert(parents.end(), n->parents.begin() + 1, n->parents.end());
        accumulate_grad(x, std::make_shared<Node>(OpEnum::ROTARY, parents, n->device, a), n->device);
    }

    static void adjoint_attention(std::shared_ptr<Node> n) {
        auto a = std::get<AttentionAttrs>(n->attrs);
        a.grads = std::make_shared<AttentionAttrs::Grads>();
        NodeVec parents{n, as_dtype(n->grad, n->dtype)};
        parents.insert(parents.end(), n->parents.begin(), n->parents.end());
        for (int w = 0; w < 3; ++w) {
            const auto& x = n->parents[w];
            if (!x->requires_grad) continue;
            a.grads->want[w] = true;
            a.which = w;
            accumulate_grad(x, std::make_shared<Node>(OpEnum::ATTENTION_GRAD, parents, n->device, a), n->device);
        }
    }

    static RegisterShape rs_rotary(OpEnum::ROTARY, first_shape);
    static RegisterShape rs_attention(OpEnum::ATTENTION, first_shape);
    static RegisterShape rs_attention_grad(OpEnum::ATTENTION_GRAD, grad_shape);
    static RegisterAdjoint ra_rotary(OpEnum::ROTARY, adjoint_rotary);
    static RegisterAdjoint ra_attention(OpEnum::ATTENTION, adjoint_attention);
}
