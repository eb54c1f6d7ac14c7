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

    using OpAttributes = std::variant<NoAttrs, ReduceAttrs, PermuteAttrs, ReshapeAttrs, ExpandAttrs, CastAttrs, RotaryAttrs, AttentionAttrs>;
}
