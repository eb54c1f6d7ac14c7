// HIP device: ROTARY, ATTENTION and ATTENTION_GRAD as graph breakers over the
// C ABI, and the AdamW step.
#include <algorithm>
#include <stdexcept>
#include <string>
#include <vector>

#include "backend/hip/hip_backend.h"
#include "core/memory.h"
#include "core/shape.h"
#include "ormi_hip.h"
#include "runtime/graph_breakers.h"

namespace ormi::hip {
    using ops::OpEnum;

    static int abi_dtype(DType d) {
        switch (d) {
            case DType::Float32: return ORMI_DTYPE_F32;
            case DType::BFloat16: return ORMI_DTYPE_BF16;
            case DType::Float16: return ORMI_DTYPE_F16;
            default: throw std::runtime_error("Unsupported DType.");
        }
    }

    static void strides4(const Node& n, int64_t (&out)[4]) {
        for (int i = 0; i < 4; ++i) out[i] = n.view.strides[i];
    }

    static bool is_integer(DType d) { return d == DType::Int32 || d == DType::Int64 || d == DType::Bool; }

    // n's values in a contiguous buffer: n's own, or a copy, by the map kernel where
    // its float32 holds them and bit for bit where they are integers.
    static NodePtr contiguous(const NodePtr& n) {
        realize(n);
        const auto& shape = n->view.shape;
        if (n->view.strides == calc_contiguous_strides(shape) && (long long)n->data->numel() == shape_numel(shape)) return n;
        if (is_integer(n->dtype)) {
            auto c = std::make_shared<Node>(empty(shape, DeviceEnum::HIP, n->dtype), false, n->device);
            const std::vector<int64_t> strides(n->view.strides.begin(), n->view.strides.end());
            ORMI_HIP_CHECK(ormi_hip_copy_view(c->data->ptr, n->data->ptr, dtype_size(n->dtype), (int)shape.size(), shape.data(), strides.data()));
            return c;
        }
        auto c = std::make_shared<Node>(OpEnum::CAST, std::vector<NodePtr>{n}, n->device, CastAttrs{n->dtype});
        realize(c);
        return c;
    }

    // In rows of 256 bytes, what the entries' sizes are multiples of: packed operands
    // alone can pass the 2^31 elements of one extent.
    static std::shared_ptr<Buffer> workspace(size_t bytes) {
        return bytes ? empty({checked_extent((long long)((bytes + 255) / 256), "attention: workspace"), 64}, DeviceEnum::HIP) : nullptr;
    }

    // ----------------------------------------------------------- gradients --
    int gradient_parent(const Node& n) {
        if (n.op == OpEnum::ATTENTION_GRAD) return 1;
        return n.op == OpEnum::ROTARY && std::get<RotaryAttrs>(n.attrs).inverse ? 0 : -1;
    }
    DType gradient_dtype(const Node& n) {
        // A rotation back reads the gradient as it comes; where that is a product
        // with the seed, as what the product holds.
        return n.op == OpEnum::ATTENTION_GRAD ? n.parents[0]->dtype : std::get<RotaryAttrs>(n.attrs).upstream;
    }

    // -------------------------------------------------------------- rotary --
    static void rotary_handler(const NodePtr& n) {
        const auto& a = std::get<RotaryAttrs>(n->attrs);
        const NodePtr& x = a.inverse ? gradient_operand(n->parents[0], gradient_dtype(*n)) : n->parents[0];
        realize(x);
        const NodePtr cos = contiguous(n->parents[1]), sin = contiguous(n->parents[2]);
        const auto& s = n->view.shape;
        auto out = empty(s, DeviceEnum::HIP, a.dtype);
        ormi_rotary_desc d{};
        d.dtype = abi_dtype(x->data->dtype);
        d.out_dtype = abi_dtype(a.dtype);
        d.batch = s[0];
        d.length = s[1];
        d.heads = s[2];
        d.dim = s[3];
        d.part = a.part;
        d.interleaved = a.interleaved;
        d.inverse = a.inverse;
        d.x = x->data->ptr;
        strides4(*x, d.x_strides);
        d.out = out->ptr;
        d.cos = (const float*)cos->data->ptr;
        d.sin = (const float*)sin->data->ptr;
        d.table_rows = cos->view.shape[0];
        d.offset = a.offset;
        if (a.positions) {
            const NodePtr& p = n->parents[3];
            const auto& v = p->view;
            d.positions = (const int32_t*)p->data->ptr;
            d.positions_strides[0] = v.shape.size() == 2 && v.shape[0] > 1 ? v.strides[0] : 0;
            d.positions_strides[1] = v.strides.back();
        }
        ORMI_HIP_CHECK(ormi_hip_rotary(&d));
        n->data = out;
        n->view.strides = calc_contiguous_strides(s);
    }

    // ----------------------------------------------------------- attention --
    // The call that node `n` (an ATTENTION, or the parents of its gradient)
    // describes; operand(i) is its i-th parent, `hold` keeps copies alive.
    static ormi_attention_desc attention_desc(const AttentionAttrs& a, const NodePtr* parents, std::vector<NodePtr>& hold) {
        const Node &q = *parents[0], &k = *parents[1], &v = *parents[2];
        ormi_attention_desc d{};
        d.dtype = abi_dtype(q.data->dtype);
        d.batch = q.view.shape[0];
        d.queries = q.view.shape[1];
        d.keys = k.view.shape[1];
        d.heads = q.view.shape[2];
        d.kv_heads = k.view.shape[2];
        d.dim = q.view.shape[3];
        d.q = q.data->ptr;
        d.k = k.data->ptr;
        d.v = v.data->ptr;
        strides4(q, d.q_strides);
        strides4(k, d.k_strides);
        strides4(v, d.v_strides);
        d.scale = a.scale;
        d.cap = a.cap;
        d.causal = a.causal;
        int at = 3;
        auto rule = [&](bool on) -> const void* {
            if (!on) return nullptr;
            hold.push_back(contiguous(parents[at++]));
            return hold.back()->data->ptr;
        };
        d.slopes = (const float*)rule(a.slopes);
        d.documents = (const int32_t*)rule(a.documents);
        d.documents_batch_stride = d.keys;
        d.prefix = (const int32_t*)rule(a.prefix);
        d.lengths = (const int32_t*)rule(a.lengths);
        return d;
    }

    static void attention_handler(const NodePtr& n) {
        const auto& a = std::get<AttentionAttrs>(n->attrs);
        std::vector<NodePtr> hold;
        ormi_attention_desc d = attention_desc(a, n->parents.data(), hold);
        auto out = empty(n->view.shape, DeviceEnum::HIP, n->dtype);
        std::shared_ptr<Buffer> lse, rest;
        if (n->requires_grad && n->dtype != DType::Float32) rest = empty(n->view.shape, DeviceEnum::HIP, n->dtype);
        if (n->requires_grad) lse = empty({d.batch, d.kv_heads, d.queries, d.heads / d.kv_heads}, DeviceEnum::HIP);
        d.out = out->ptr;
        d.rest = rest ? rest->ptr : nullptr;
        d.lse = lse ? (float*)lse->ptr : nullptr;
        size_t bytes = 0;
        ORMI_HIP_CHECK(ormi_hip_attention_workspace_size(&d, &bytes));
        const auto ws = workspace(bytes);
        if (ws) d.workspace = ws->ptr, d.workspace_bytes = ws->bytes;
        ORMI_HIP_CHECK(ormi_hip_attention(&d));
        a.saved->lse = lse;
        a.saved->rest = rest;
        n->data = out;
        n->view.strides = calc_contiguous_strides(n->view.shape);
    }

    static void attention_grad_handler(const NodePtr& n) {
        const auto& a = std::get<AttentionAttrs>(n->attrs);
        auto& made = a.grads->made;
        if (!made[a.which]) {
            const NodePtr& out = n->parents[0];
            const NodePtr& g = gradient_operand(n->parents[1], gradient_dtype(*n));
            realize(g);
            if (!a.saved->lse) throw std::runtime_error("ATTENTION_GRAD: its attention kept no sums.");
            std::vector<NodePtr> hold;
            ormi_attention_grad_desc d{};
            d.forward = attention_desc(a, n->parents.data() + 2, hold);
            d.forward.out = out->data->ptr;
            d.forward.rest = a.saved->rest ? a.saved->rest->ptr : nullptr;
            d.forward.lse = (float*)a.saved->lse->ptr;
            d.dout = g->data->ptr;
            strides4(*g, d.dout_strides);
            void** outs[3] = {&d.dq, &d.dk, &d.dv};
            for (int w = 0; w < 3; ++w) {
                if (!a.grads->want[w]) continue;
                made[w] = empty(n->parents[2 + w]->view.shape, DeviceEnum::HIP, n->parents[2 + w]->dtype);
                *outs[w] = made[w]->ptr;
            }
            size_t bytes = 0;
            ORMI_HIP_CHECK(ormi_hip_attention_grad_workspace_size(&d, &bytes));
            const auto ws = workspace(bytes);
            if (ws) d.forward.workspace = ws->ptr, d.forward.workspace_bytes = ws->bytes;
            ORMI_HIP_CHECK(ormi_hip_attention_grad(&d));
        }
        n->data = made[a.which];
        made[a.which] = nullptr;  // the node's own from here on
        n->view.strides = calc_contiguous_strides(n->view.shape);
    }

    // --------------------------------------------------------------- AdamW --
    static void require(bool ok, const char* what) {
        if (!ok) throw std::runtime_error(std::string("adamw: ") + what);
    }

    static NodePtr state_leaf(std::vector<int> shape, DType dtype, const Device& dev) {
        return std::make_shared<Node>(empty(std::move(shape), DeviceEnum::HIP, dtype), false, dev);
    }

    static std::vector<int> words_shape(long long count) {
        return {checked_extent((count + ORMI_ADAMW_BLOCK - 1) / ORMI_ADAMW_BLOCK * (ORMI_ADAMW_BLOCK / 4), "adamw: code words")};
    }
    static std::vector<int> scales_shape(long long count) { return {(int)((count + ORMI_ADAMW_BLOCK - 1) / ORMI_ADAMW_BLOCK)}; }

    static void check_state(const std::vector<NodePtr>& s, const std::vector<int>& shape, int bits, const Device& dev) {
        const long long n = shape_numel(shape);
        require(s.size() == (bits == 32 ? 2u : 4u), "a state of another kind.");
        for (size_t i = 0; i < s.size(); ++i) {
            require(s[i] && s[i]->device.type == dev.type, "a state on another device.");
            const bool codes = bits == 8 && i % 2 == 0;
            require(s[i]->dtype == (codes ? DType::Int32 : DType::Float32), "a state of another type.");
            require(s[i]->view.shape == (bits == 32 ? shape : codes ? words_shape(n) : scales_shape(n)), "a state of another shape.");
        }
    }

    void adamw(const std::vector<NodePtr>& params, const std::vector<NodePtr>& grads, const std::vector<std::vector<NodePtr>>& states,
               const AdamWOptions& o, std::vector<NodePtr>* new_params, std::vector<std::vector<NodePtr>>* new_states) {
        require(params.size() == grads.size() && params.size() == states.size(), "as many gradients and states as parameters, please.");
        require(o.bits == 32 || o.bits == 8, "states have 32 or 8 bits.");
        for (size_t i = 0; i < params.size(); ++i) {
            const NodePtr &p = params[i], &g = grads[i];
            require(p && g, "a null tensor.");
            require(p->device.type == DeviceEnum::HIP && g->device.type == DeviceEnum::HIP, "parameters and gradients live on the hip device.");
            require(p->view.shape == g->view.shape, "a gradient of another shape than its parameter.");
            abi_dtype(p->dtype);
            abi_dtype(g->dtype);
            check_state(states[i], p->view.shape, o.bits, p->device);
        }
        realize_group(grads);
        std::vector<NodePtr> hold;
        std::vector<ormi_adamw_tensor> list;
        new_params->clear();
        new_states->clear();
        auto in = [&](const NodePtr& n) -> const void* {
            hold.push_back(contiguous(n));
            return hold.back()->data->ptr;
        };
        for (size_t i = 0; i < params.size(); ++i) {
            const auto& s = states[i];
            ormi_adamw_tensor t{};
            t.count = shape_numel(params[i]->view.shape);
            t.p = in(params[i]);
            t.p_dtype = abi_dtype(params[i]->dtype);
            t.g = in(grads[i]);
            t.g_dtype = abi_dtype(grads[i]->dtype);
            auto np = std::make_shared<Node>(empty(params[i]->view.shape, DeviceEnum::HIP, params[i]->dtype), params[i]->requires_grad, params[i]->device);
            t.out = np->data->ptr;
            std::vector<NodePtr> ns;
            for (const auto& x : s) ns.push_back(state_leaf(x->view.shape, x->dtype, x->device));
            const int v = o.bits == 32 ? 1 : 2;
            t.m = in(s[0]);
            t.v = in(s[v]);
            t.m_out = ns[0]->data->ptr;
            t.v_out = ns[v]->data->ptr;
            if (o.bits == 8) {
                t.m_scale = (const float*)in(s[1]);
                t.v_scale = (const float*)in(s[3]);
                t.m_scale_out = (float*)ns[1]->data->ptr;
                t.v_scale_out = (float*)ns[3]->data->ptr;
            }
            list.push_back(t);
            new_params->push_back(np);
            new_states->push_back(ns);
        }
        ormi_adamw_desc d{};
        d.num_tensors = (int)list.size();
        d.tensors = list.data();
        d.state_bits = o.bits;
        d.step = o.step;
        d.lr = o.lr;
        d.beta1 = o.beta1;
        d.beta2 = o.beta2;
        d.eps = o.eps;
        d.weight_decay = o.weight_decay;
        ORMI_HIP_CHECK(ormi_hip_adamw(&d));
    }

    std::pair<NodePtr, NodePtr> adamw_values(const std::vector<NodePtr>& state, const std::vector<int>& shape) {
        require(!state.empty() && state[0], "a null state.");
        check_state(state, shape, 8, state[0]->device);
        auto m = state_leaf(shape, DType::Float32, state[0]->device), v = state_leaf(shape, DType::Float32, state[0]->device);
        std::vector<NodePtr> s;
        for (const auto& x : state) s.push_back(contiguous(x));
        ORMI_HIP_CHECK(ormi_hip_adamw_values((float*)m->data->ptr, (float*)v->data->ptr, s[0]->data->ptr, (const float*)s[1]->data->ptr,
                                             s[2]->data->ptr, (const float*)s[3]->data->ptr, shape_numel(shape)));
        return {m, v};
    }

    static RegisterGraphBreaker reg_rotary(DeviceEnum::HIP, OpEnum::ROTARY, rotary_handler);
    static RegisterGraphBreaker reg_attention(DeviceEnum::HIP, OpEnum::ATTENTION, attention_handler);
    static RegisterGraphBreaker reg_attention_grad(DeviceEnum::HIP, OpEnum::ATTENTION_GRAD, attention_grad_handler);
}
