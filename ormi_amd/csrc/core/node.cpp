#include <stdexcept>
#include "core/node.h"
#include "core/registry.h"
#include "runtime/runtime.h"

namespace ormi {
    // Leaf constructor (reference: csrc/core/node.cpp:8-13).
    Node::Node(std::shared_ptr<Buffer> mem, bool req_grad, Device dev)
        : op(ops::OpEnum::LEAF), data(std::move(mem)), requires_grad(req_grad), device(dev) {
        if (!data) throw std::runtime_error("Leaf node requires a buffer.");
        view.shape = data->shape;
        view.strides = calc_contiguous_strides(data->shape);
        dtype = data->dtype;
    }

    static DType result_dtype(ops::OpEnum op, const std::vector<std::shared_ptr<Node>>& parents, const OpAttributes& attrs) {
        switch (op) {
            case ops::OpEnum::TRANSPOSE: case ops::OpEnum::RESHAPE: case ops::OpEnum::EXPAND: case ops::OpEnum::SEQUENCE_OUT:
                return parents.empty() ? DType::Float32 : parents[0]->dtype;
            case ops::OpEnum::CAST: return std::get<CastAttrs>(attrs).dtype;
            case ops::OpEnum::ROTARY: return std::get<RotaryAttrs>(attrs).dtype;
            case ops::OpEnum::ATTENTION: return parents[0]->dtype;
            case ops::OpEnum::ATTENTION_GRAD: return parents[2 + std::get<AttentionAttrs>(attrs).which]->dtype;
            case ops::OpEnum::RECURRENCE: return parents[1]->dtype;
            case ops::OpEnum::CONV: return parents[0]->dtype;
            case ops::OpEnum::RECURRENCE_GRAD: case ops::OpEnum::CONV_GRAD: {
                const auto& a = std::get<SequenceAttrs>(attrs);
                return parents[a.first() + a.which]->dtype;
            }
            // The states of a recurrence are float32, those of a convolution its inputs.
            case ops::OpEnum::LAST_STATE: return std::get<SequenceAttrs>(attrs).width ? parents[0]->dtype : DType::Float32;
            case ops::OpEnum::ARGMAX: return DType::Int64;
            default: return DType::Float32;
        }
    }

    // Internal constructor (reference: csrc/core/node.cpp:16-32).
    Node::Node(ops::OpEnum operation, std::vector<std::shared_ptr<Node>> parent_nodes, Device dev, OpAttributes attributes)
        : op(operation), parents(std::move(parent_nodes)), requires_grad(false), device(dev), attrs(std::move(attributes)) {
        for (const auto& p : parents) {
            if (!p) throw std::runtime_error("Node parent is null.");
            if (p->requires_grad) requires_grad = true;
        }
        // Piecewise-constant and integer-valued results carry no gradient.
        if (op == ops::OpEnum::ARGMAX || op == ops::OpEnum::STEP || op == ops::OpEnum::EQ) requires_grad = false;

        view.shape = infer_shape(op, parents, attrs);
        const StrideInferFunc* stride_func = Registry<StrideInferFunc>::find(op);
        view.strides = stride_func ? (*stride_func)(parents, attrs, view.shape) : calc_contiguous_strides(view.shape);
        dtype = result_dtype(op, parents, attrs);
    }

    // Nodes to let go of, while some node's destructor on this thread is at it.
    static thread_local std::vector<std::shared_ptr<Node>>* t_releasing = nullptr;

    Node::~Node() {
        auto leave = [](std::shared_ptr<Node>& n) {
            if (n.use_count() == 1) t_releasing->push_back(std::move(n));
            else n.reset();  // perhaps the last of two references of its child: that one comes here with t_releasing set
        };
        auto leave_all = [&] {
            for (auto& p : parents) leave(p);
            if (grad) leave(grad);
        };
        if (t_releasing) {
            leave_all();
            return;
        }
        if (parents.empty() && !grad) return;
        std::vector<std::shared_ptr<Node>> list;
        t_releasing = &list;
        leave_all();
        while (!list.empty()) {
            const auto n = std::move(list.back());
            list.pop_back();
        }
        t_releasing = nullptr;
    }

    bool Node::is_realized() const { return data != nullptr; }

    void Node::realize() {
        if (!is_realized()) execute_graph(shared_from_this());
    }
}
