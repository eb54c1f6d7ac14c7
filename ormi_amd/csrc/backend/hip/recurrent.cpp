// HIP device: RECURRENCE, CONV, their gradients and last states as graph breakers
// over the C ABI.
#include <stdexcept>
#include <string>
#include <vector>

#include "backend/hip/operands.h"
#include "core/shape.h"
#include "ormi_hip.h"
#include "runtime/graph_breakers.h"

namespace ormi::hip {
    using ops::OpEnum;

    namespace {
        // n (batch, length, channels) as the entries read it: neighbouring channels, and
        // tokens at most 2^20 elements apart.
        NodePtr rows(const NodePtr& n) {
            realize(n);
            const auto& v = n->view;
            return (v.shape[2] <= 1 || v.strides[2] == 1) && (v.shape[1] <= 1 || v.strides[1] <= 1 << 20) ? n : contiguous(n);
        }
        void strides2(const Node& n, int64_t (&out)[2]) {
            out[0] = n.view.strides[0];
            out[1] = n.view.strides[1];
        }

        // Reads a node's parents in order, keeping copies alive.
        struct Operands {
            const NodePtr* at;
            std::vector<NodePtr> hold;
            Node& rows_of() {
                hold.push_back(rows(*at++));
                return *hold.back();
            }
            const void* packed(bool on) {
                if (!on) return nullptr;
                hold.push_back(contiguous(*at++));
                return hold.back()->data->ptr;
            }
        };

        ormi_recurrence_desc recurrence_desc(const SequenceAttrs& a, Operands& in) {
            ormi_recurrence_desc d{};
            const Node& g = in.rows_of();
            const Node& x = in.rows_of();
            d.dtype = abi_dtype(x.data->dtype);
            d.gate_dtype = abi_dtype(g.data->dtype);
            d.batch = a.shape[0];
            d.length = a.shape[1];
            d.channels = a.shape[2];
            d.logits = a.logits;
            d.gates = g.data->ptr;
            strides2(g, d.gate_strides);
            d.x = x.data->ptr;
            strides2(x, d.x_strides);
            d.initial = (const float*)in.packed(a.initial);
            d.documents = (const int32_t*)in.packed(a.documents);
            d.documents_batch_stride = d.length;
            d.lengths = (const int32_t*)in.packed(a.lengths);
            return d;
        }

        ormi_conv_desc conv_desc(const SequenceAttrs& a, Operands& in) {
            ormi_conv_desc d{};
            const Node& x = in.rows_of();
            d.dtype = abi_dtype(x.data->dtype);
            d.batch = a.shape[0];
            d.length = a.shape[1];
            d.channels = a.shape[2];
            d.width = a.width;
            d.silu = a.silu;
            d.x = x.data->ptr;
            strides2(x, d.x_strides);
            d.weight = (const float*)in.packed(true);
            d.bias = (const float*)in.packed(a.bias);
            d.initial = in.packed(a.initial);
            d.documents = (const int32_t*)in.packed(a.documents);
            d.documents_batch_stride = d.length;
            d.lengths = (const int32_t*)in.packed(a.lengths);
            return d;
        }

        void finish(const NodePtr& n, const std::shared_ptr<Buffer>& out) {
            n->data = out;
            n->view.strides = calc_contiguous_strides(n->view.shape);
        }

        void recurrence_handler(const NodePtr& n) {
            const auto& a = std::get<SequenceAttrs>(n->attrs);
            Operands in{n->parents.data(), {}};
            ormi_recurrence_desc d = recurrence_desc(a, in);
            const auto out = empty(n->view.shape, DeviceEnum::HIP, n->dtype);
            const auto last = empty({d.batch, d.channels}, DeviceEnum::HIP);
            std::shared_ptr<Buffer> states;
            if (n->requires_grad) states = empty({d.batch, (d.length + ORMI_RECURRENCE_TILE - 1) / ORMI_RECURRENCE_TILE, d.channels}, DeviceEnum::HIP);
            d.out = out->ptr;
            d.last = (float*)last->ptr;
            d.states = states ? (float*)states->ptr : nullptr;
            size_t bytes = 0;
            ORMI_HIP_CHECK(ormi_hip_recurrence_workspace_size(&d, &bytes));
            const auto ws = workspace(bytes);
            if (ws) d.workspace = ws->ptr, d.workspace_bytes = ws->bytes;
            ORMI_HIP_CHECK(ormi_hip_recurrence(&d));
            a.saved->last = last;
            a.saved->states = states;
            finish(n, out);
        }

        void conv_handler(const NodePtr& n) {
            const auto& a = std::get<SequenceAttrs>(n->attrs);
            Operands in{n->parents.data(), {}};
            ormi_conv_desc d = conv_desc(a, in);
            const auto out = empty(n->view.shape, DeviceEnum::HIP, n->dtype);
            const auto last = empty({d.batch, d.width - 1, d.channels}, DeviceEnum::HIP, n->dtype);
            d.out = out->ptr;
            d.last = last->ptr;
            ORMI_HIP_CHECK(ormi_hip_conv(&d));
            a.saved->last = last;
            finish(n, out);
        }

        // A state that no gradient goes back through lets go of the call that left it:
        // passed from call to call it would hold on to all of them.
        void last_state_handler(const NodePtr& n) {
            auto& a = std::get<SequenceAttrs>(n->attrs);
            if (!a.saved->last) throw std::runtime_error("LAST_STATE: its sequence kept none.");
            finish(n, a.saved->last);
            if (n->requires_grad) return;
            a.saved = nullptr;
            n->parents.clear();
        }

        // The upstream gradients of node n: that of the result as it comes, of x's type
        // or float32, and that of the last state as contiguous float32.
        struct Upstream {
            NodePtr dout, dlast;
        };
        Upstream upstream(const Node& n, const SequenceAttrs& a) {
            Upstream u;
            int at = 1;
            if (a.dout) {
                const DType want = gradient_dtype(n);
                NodePtr g = gradient_operand(n.parents[at++], want);
                realize(g);
                if (g->data->dtype != want && g->data->dtype != DType::Float32)
                    g = std::make_shared<Node>(OpEnum::CAST, std::vector<NodePtr>{g}, g->device, CastAttrs{DType::Float32});
                u.dout = rows(g);
            }
            if (a.dlast) {
                NodePtr g = n.parents[at];
                if (g->dtype != DType::Float32)
                    g = std::make_shared<Node>(OpEnum::CAST, std::vector<NodePtr>{g}, g->device, CastAttrs{DType::Float32});
                u.dlast = contiguous(g);
            }
            return u;
        }

        // A wanted gradient's buffer, or null.
        void* wanted(FilledTogether<4>& filled, const Node& n, const SequenceAttrs& a, int w) {
            return a.grads->want[w] ? filled.add(w, *n.parents[a.first() + w]) : nullptr;
        }
        void take_made(const NodePtr& n, const SequenceAttrs& a) {
            finish(n, a.grads->made[a.which]);
            a.grads->made[a.which] = nullptr;  // the node's own from here on
        }

        void recurrence_grad_handler(const NodePtr& n) {
            const auto& a = std::get<SequenceAttrs>(n->attrs);
            if (!a.grads->made[a.which]) {
                const Upstream u = upstream(*n, a);
                Operands in{n->parents.data() + a.first(), {}};
                ormi_recurrence_grad_desc d{};
                d.forward = recurrence_desc(a, in);
                if (!a.saved->states) throw std::runtime_error("RECURRENCE_GRAD: its recurrence kept no states.");
                d.forward.states = (float*)a.saved->states->ptr;
                if (u.dout) {
                    d.dout = u.dout->data->ptr;
                    d.dout_dtype = abi_dtype(u.dout->data->dtype);
                    strides2(*u.dout, d.dout_strides);
                }
                if (u.dlast) d.dlast = (const float*)u.dlast->data->ptr;
                FilledTogether<4> filled;
                d.dgates = wanted(filled, *n, a, 0);
                d.dx = wanted(filled, *n, a, 1);
                if (a.initial) d.dinitial = (float*)wanted(filled, *n, a, 2);
                size_t bytes = 0;
                ORMI_HIP_CHECK(ormi_hip_recurrence_workspace_size(&d.forward, &bytes));
                const auto ws = workspace(bytes);
                if (ws) d.forward.workspace = ws->ptr, d.forward.workspace_bytes = ws->bytes;
                ORMI_HIP_CHECK(ormi_hip_recurrence_grad(&d));
                filled.leave(a.grads->made);
            }
            take_made(n, a);
        }

        void conv_grad_handler(const NodePtr& n) {
            const auto& a = std::get<SequenceAttrs>(n->attrs);
            if (!a.grads->made[a.which]) {
                const Upstream u = upstream(*n, a);
                Operands in{n->parents.data() + a.first(), {}};
                ormi_conv_grad_desc d{};
                d.forward = conv_desc(a, in);
                if (u.dout) {
                    d.dout = u.dout->data->ptr;
                    d.dout_dtype = abi_dtype(u.dout->data->dtype);
                    strides2(*u.dout, d.dout_strides);
                }
                if (u.dlast) d.dlast = (const float*)u.dlast->data->ptr;
                int w = 2;
                FilledTogether<4> filled;
                d.dx = wanted(filled, *n, a, 0);
                d.dweight = (float*)wanted(filled, *n, a, 1);
                if (a.bias) d.dbias = (float*)wanted(filled, *n, a, w++);
                if (a.initial) d.dinitial = wanted(filled, *n, a, w);
                size_t bytes = 0;
                ORMI_HIP_CHECK(ormi_hip_conv_grad_workspace_size(&d, &bytes));
                const auto ws = workspace(bytes);
                if (ws) d.workspace = ws->ptr, d.workspace_bytes = ws->bytes;
                ORMI_HIP_CHECK(ormi_hip_conv_grad(&d));
                filled.leave(a.grads->made);
            }
            take_made(n, a);
        }

        RegisterGraphBreaker reg_recurrence(DeviceEnum::HIP, OpEnum::RECURRENCE, recurrence_handler);
        RegisterGraphBreaker reg_recurrence_grad(DeviceEnum::HIP, OpEnum::RECURRENCE_GRAD, recurrence_grad_handler);
        RegisterGraphBreaker reg_conv(DeviceEnum::HIP, OpEnum::CONV, conv_handler);
        RegisterGraphBreaker reg_conv_grad(DeviceEnum::HIP, OpEnum::CONV_GRAD, conv_grad_handler);
        RegisterGraphBreaker reg_last(DeviceEnum::HIP, OpEnum::LAST_STATE, last_state_handler);
    }
}
