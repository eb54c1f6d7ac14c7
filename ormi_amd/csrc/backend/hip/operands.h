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
}
