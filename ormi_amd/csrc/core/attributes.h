#pragma once
#include <memory>
#include <vector>
#include <variant>
#include "core/dtype.h"

namespace ormi {
    struct NoAttrs {};

    struct ReduceAttrs {
        std::vector<int> axes;     // empty = reduce every axis
        bool keepdims = false;
    };

    struct PermuteAttrs { std::vector<int> axes; };
    struct ReshapeAttrs { std::vector<int> shape; };
    struct ExpandAttrs  { std::vector<int> shape; };
    struct CastAttrs    { DType dtype = DType::Float32; };

    struct Buffer;

    // ROTARY: parents x, cos, sin and, when positions is set, the positions.
    struct RotaryAttrs {
        int part = 0;              // features turned
        bool interleaved = false;  // pairs (2p, 2p + 1) instead of (p, p + part / 2)
        bool inverse = false;      // turned back: the adjoint
        int offset = 0;            // position of token 0 without positions
        bool positions = false;
        DType dtype = DType::Float32;
        DType upstream = DType::Float32;  // inverse: the type of the rotated result
    };

    // ATTENTION: parents q, k, v, then those of slopes, documents, prefix and
    // lengths that are set. ATTENTION_GRAD: parents the ATTENTION node, its
    // gradient, and the ATTENTION node's parents.
    struct AttentionAttrs {
        float scale = 1.0f, cap = 0.0f;
        bool causal = false;
        bool slopes = false, documents = false, prefix = false, lengths = false;
        // What realizing the node leaves for its gradient: each row's log-sum, and
        // what rounding a 16-bit result left.
        struct Saved { std::shared_ptr<Buffer> lse, rest; };
        std::shared_ptr<Saved> saved;
        // The gradients of one backward pass are computed together by the first
        // of them that is realized; the others take theirs from here.
        struct Grads {
            bool want[3] = {false, false, false};
            std::shared_ptr<Buffer> made[3];
        };
        std::shared_ptr<Grads> grads;
        int which = 0;             // ATTENTION_GRAD: 0 q, 1 k, 2 v
    };

    // RECURRENCE: parents gates, x, then those of initial, documents and lengths
    // that are set. CONV: parents x, weight, then those of bias, initial, documents
    // and lengths that are set. A graph reads either through SEQUENCE_OUT, a view of
    // its result, and LAST_STATE, the state it leaves, so that each has a gradient of
    // its own; LAST_STATE_GRAD is the latter's, of the result's shape only to be
    // added to the former's. The gradients: the node,
    // its result's gradient and its last state's (those that are set), and the
    // node's parents.
    struct SequenceAttrs {
        int width = 0;             // of a convolution; 0: a recurrence
        bool logits = false;       // recurrence: gates are logits
        bool silu = false;         // convolution
        bool bias = false, initial = false, documents = false, lengths = false;
        std::vector<int> shape;    // of the result
        // What realizing the node leaves: the state after the last token, and for a
        // recurrence's gradient those before its tiles. A realized LAST_STATE without a
        // gradient has no parents and no `saved` any more.
        struct Saved { std::shared_ptr<Buffer> last, states; };
        std::shared_ptr<Saved> saved;
        // As of an attention's gradients.
        struct Grads {
            bool want[4] = {false, false, false, false};
            std::shared_ptr<Buffer> made[4];
        };
        std::shared_ptr<Grads> grads;
        int which = 0;             // gradients: the node's parent that it belongs to
        bool dout = false, dlast = false;
        int first() const { return 1 + dout + dlast; }  // where a gradient's parents hold the node's
    };

    using OpAttributes = std::variant<NoAttrs, ReduceAttrs, PermuteAttrs, ReshapeAttrs, ExpandAttrs, CastAttrs, RotaryAttrs, AttentionAttrs, SequenceAttrs>;
}
