// RECURRENCE and CONV (additive): a recurrent block's gated linear recurrence and
// its short causal convolution; SEQUENCE_OUT and LAST_STATE: what either gives, and
// the state that it leaves for the tokens after it. The adjoints are ops of their own (RECURRENCE_GRAD,
// CONV_GRAD), which have no adjoint in turn.
#include <stdexcept>
#include <string>
#include "core/ops/api.h"
#include "core/shape.h"
#include "core/adjoint.h"
#include "core/registry.h"

namespace ormi {
    using ops::OpEnum;
    using NodeVec = std::vector<std::shared_ptr<Node>>;
    using NodePtr = std::shared_ptr<Node>;

    constexpr int kMostTokens = 1 << 30;
    constexpr int kMostWidth = 8;

    static bool is_float(DType d) { return d == DType::Float32 || d == DType::BFloat16 || d == DType::Float16; }

    static void require(bool ok, const char* op, const std::string& what) {
        if (!ok) throw std::runtime_error(std::string(op) + " " + what);
    }

    // An operand beside the first, of one shape and type.
    static void check_operand(const NodePtr& n, const NodePtr& x, DType dtype, const std::vector<int>& shape, const char* op, const std::string& what) {
        require(n->device.type == x->device.type, op, "got " + what + " on another device.");
        require(n->dtype == dtype, op, "takes " + what + " as " + dtype_name(dtype) + ".");
        require(n->view.shape == shape, op, "got " + what + " of another shape.");
    }

    // The masks, which end a node's parents.
    static void add_masks(const NodePtr& x, const NodePtr& documents, const NodePtr& lengths, const char* op, SequenceAttrs& a, NodeVec& parents) {
        const auto& xs = x->view.shape;
        auto mask = [&](const NodePtr& n, const std::vector<int>& shape, const char* what, bool& flag) {
            if (!n) return;
            check_operand(n, x, DType::Int32, shape, op, what);
            require(!n->requires_grad, op, std::string("has no gradient for ") + what + ".");
            flag = true;
            parents.push_back(n);
        };
        mask(documents, {xs[0], xs[1]}, "documents (batch, length)", a.documents);
        mask(lengths, {xs[0]}, "lengths (batch)", a.lengths);
        a.shape = xs;
        a.saved = std::make_shared<SequenceAttrs::Saved>();
    }

    static void check_x(const NodePtr& x, const char* op) {
        require(x->view.shape.size() == 3, op, "takes (batch, length, channels).");
        require(is_float(x->dtype), op, "takes and gives float32, bfloat16 or float16.");
        require(x->view.shape[1] <= kMostTokens, op, "takes at most 2^30 tokens.");
    }

    namespace ops {
        NodePtr recurrence(NodePtr gates, NodePtr x, NodePtr initial, NodePtr documents, NodePtr lengths, bool logits) {
            const char* op = "RECURRENCE";
            require(gates && x, op, "got a null operand.");
            check_x(x, op);
            require(gates->device.type == x->device.type, op, "got gates on another device.");
            require(gates->dtype == x->dtype || gates->dtype == DType::Float32, op, "takes gates of x's type or float32.");
            require(gates->view.shape == x->view.shape, op, "got gates of another shape.");
            SequenceAttrs a;
            a.logits = logits;
            NodeVec parents{gates, x};
            if (initial) {
                check_operand(initial, x, DType::Float32, {x->view.shape[0], x->view.shape[2]}, op, "initial (batch, channels)");
                a.initial = true;
                parents.push_back(initial);
            }
            add_masks(x, documents, lengths, op, a, parents);
            return std::make_shared<Node>(OpEnum::RECURRENCE, parents, x->device, a);
        }

        NodePtr conv(NodePtr x, NodePtr weight, NodePtr bias, NodePtr initial, NodePtr documents, NodePtr lengths, bool silu) {
            const char* op = "CONV";
            require(x && weight, op, "got a null operand.");
            check_x(x, op);
            const auto& xs = x->view.shape;
            require(weight->view.shape.size() == 2, op, "takes weights (channels, width).");
            const int width = weight->view.shape[1];
            require(width >= 1 && width <= kMostWidth, op, "takes widths from 1 to 8.");
            check_operand(weight, x, DType::Float32, {xs[2], width}, op, "weights (channels, width)");
            SequenceAttrs a;
            a.width = width;
            a.silu = silu;
            NodeVec parents{x, weight};
            if (bias) {
                check_operand(bias, x, DType::Float32, {xs[2]}, op, "a bias (channels)");
                a.bias = true;
                parents.push_back(bias);
            }
            if (initial) {
                check_operand(initial, x, x->dtype, {xs[0], width - 1, xs[2]}, op, "initial (batch, width - 1, channels)");
                a.initial = true;
                parents.push_back(initial);
            }
            add_masks(x, documents, lengths, op, a, parents);
            return std::make_shared<Node>(OpEnum::CONV, parents, x->device, a);
        }

        NodePtr sequence_out(NodePtr n) {
            require(n && (n->op == OpEnum::RECURRENCE || n->op == OpEnum::CONV), "SEQUENCE_OUT", "takes a recurrence or a convolution.");
            return std::make_shared<Node>(OpEnum::SEQUENCE_OUT, NodeVec{n}, n->device);
        }

        NodePtr last_state(NodePtr n) {
            require(n && (n->op == OpEnum::RECURRENCE || n->op == OpEnum::CONV), "LAST_STATE", "takes a recurrence or a convolution.");
            return std::make_shared<Node>(OpEnum::LAST_STATE, NodeVec{n}, n->device, n->attrs);
        }
    }

    static std::vector<int> shape_of_result(const NodeVec&, const OpAttributes& attrs) { return std::get<SequenceAttrs>(attrs).shape; }
    static std::vector<int> shape_of_state(const NodeVec&, const OpAttributes& attrs) {
        const auto& a = std::get<SequenceAttrs>(attrs);
        if (!a.width) return {a.shape[0], a.shape[2]};
        return {a.shape[0], a.width - 1, a.shape[2]};
    }
    static std::vector<int> shape_of_gradient(const NodeVec& parents, const OpAttributes& attrs) {
        const auto& a = std::get<SequenceAttrs>(attrs);
        return parents[a.first() + a.which]->view.shape;
    }

    static void adjoint_out(std::shared_ptr<Node> n) {
        if (n->parents[0]->requires_grad) accumulate_grad(n->parents[0], n->grad, n->device);
    }
    static void adjoint_last_state(std::shared_ptr<Node> n) {
        const auto& of = n->parents[0];
        if (!of->requires_grad) return;
        SequenceAttrs a = std::get<SequenceAttrs>(n->attrs);
        a.saved = nullptr;
        accumulate_grad(of, std::make_shared<Node>(OpEnum::LAST_STATE_GRAD, NodeVec{n->grad}, n->device, a), n->device);
    }

    // A sequence's gradient is a sum of what its two readers passed on, each added
    // on the right: the last state's parts go to `last`, the rest is returned (null
    // where there is none).
    static NodePtr without_last(NodePtr g, NodePtr& last) {
        const auto shape = g->view.shape;
        auto is_last = [](const NodePtr& n) { return n->op == OpEnum::LAST_STATE_GRAD; };
        std::vector<NodePtr> sums;  // from the outermost in
        size_t deepest = 0;         // sums beyond this many add none of them
        while (g->op == OpEnum::ADD && !g->is_realized() && g->parents[0]->view.shape == shape && g->parents[1]->view.shape == shape) {
            sums.push_back(g);
            if (is_last(g->parents[1])) deepest = sums.size();
            g = g->parents[0];
        }
        if (is_last(g)) deepest = sums.size();
        NodePtr rest = deepest < sums.size() ? sums[deepest] : g;
        auto take = [&](const NodePtr& part) {
            const NodePtr& x = part->parents[0];
            last = last ? std::make_shared<Node>(OpEnum::ADD, NodeVec{last, x}, x->device) : x;
        };
        if (is_last(rest)) {
            take(rest);
            rest = nullptr;
        }
        for (size_t i = deepest; i-- > 0;) {
            const NodePtr& part = sums[i]->parents[1];
            if (is_last(part)) take(part);
            else rest = rest ? std::make_shared<Node>(OpEnum::ADD, NodeVec{rest, part}, part->device) : part;
        }
        return rest;
    }

    static void adjoint_sequence(std::shared_ptr<Node> n) {
        auto a = std::get<SequenceAttrs>(n->attrs);
        a.grads = std::make_shared<SequenceAttrs::Grads>();
        NodePtr last;
        const NodePtr dout = without_last(n->grad, last);
        NodeVec parents{n};
        if (dout) parents.push_back(dout);
        if (last) parents.push_back(last);
        a.dout = dout != nullptr;
        a.dlast = last != nullptr;
        parents.insert(parents.end(), n->parents.begin(), n->parents.end());
        const OpEnum op = n->op == OpEnum::CONV ? OpEnum::CONV_GRAD : OpEnum::RECURRENCE_GRAD;
        // The learned parents come first, the masks behind them.
        const int learned = 2 + a.bias + a.initial;
        for (int w = 0; w < learned; ++w) {
            const auto& x = n->parents[w];
            if (!x->requires_grad) continue;
            a.grads->want[w] = true;
            a.which = w;
            accumulate_grad(x, std::make_shared<Node>(op, parents, n->device, a), n->device);
        }
    }

    static RegisterShape rs_recurrence(OpEnum::RECURRENCE, shape_of_result);
    static RegisterShape rs_conv(OpEnum::CONV, shape_of_result);
    static RegisterShape rs_out(OpEnum::SEQUENCE_OUT, infer_unary_shape);
    static RegisterViewOp rv_out(OpEnum::SEQUENCE_OUT);
    static RegisterShape rs_last(OpEnum::LAST_STATE, shape_of_state);
    static RegisterShape rs_last_grad(OpEnum::LAST_STATE_GRAD, shape_of_result);
    static RegisterShape rs_recurrence_grad(OpEnum::RECURRENCE_GRAD, shape_of_gradient);
    static RegisterShape rs_conv_grad(OpEnum::CONV_GRAD, shape_of_gradient);
    static RegisterAdjoint ra_recurrence(OpEnum::RECURRENCE, adjoint_sequence);
    static RegisterAdjoint ra_conv(OpEnum::CONV, adjoint_sequence);
    static RegisterAdjoint ra_out(OpEnum::SEQUENCE_OUT, adjoint_out);
    static RegisterAdjoint ra_last(OpEnum::LAST_STATE, adjoint_last_state);
}
