// What the handlers of ops that call C entries of their own share.
#pragma once
#include <memory>

#include "backend/hip/hip_backend.h"
#include "core/memory.h"

namespace ormi::hip {
    // The C ABI's code of a float type; throws for the others.
    int abi_dtype(DType d);
    // n's values in a contiguous buffer: n's own, or a copy, by the map kernel where
    // its float32 holds them and bit for bit where they are integers.
    NodePtr contiguous(const NodePtr& n);
    // Device memory of at least `bytes`, null for 0.
    std::shared_ptr<Buffer> workspace(size_t bytes);

    // Buffers of gradients that one call fills, with the first of them that is
    // realized. The others find theirs only once the call is made: where it is refused,
    // or memory runs out, each tries again.
    template <size_t N>
    struct FilledTogether {
        std::shared_ptr<Buffer> buffers[N];
        void* add(size_t w, const Node& like) {
            buffers[w] = empty(like.view.shape, DeviceEnum::HIP, like.dtype);
            return buffers[w]->ptr;
        }
        void leave(std::shared_ptr<Buffer> (&made)[N]) {
            for (size_t w = 0; w < N; ++w) made[w] = std::move(buffers[w]);
        }
    };
}
