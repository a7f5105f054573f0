// The size that a library workspace grows to (host code only, without HIP, so
// that it is tested without a GPU).
#pragma once

#include <algorithm>
#include <cstddef>

// Room for any prefill call (at most one 128-row record a CU, 17 MB) and any
// one-stream decode call, so that those never grow it (a growth waits for the
// device and fails inside a capture).
constexpr size_t kWorkspaceLeast = (size_t) 20 << 20;

// A workspace of `bytes` at least beside one of `held` bytes, which is kept for
// the graphs that use it: twice that, so that all that are kept take less than
// the one in use, or, where that much is not to be had, what the call needs.
// allocate(n) gives success (true) or not. The size that was allocated, 0: none.
template <typename Allocate>
size_t grow_workspace(const size_t bytes, const size_t held, Allocate && allocate) {
    const size_t want = std::max({bytes, 2 * held, kWorkspaceLeast});
    if (allocate(want)) return want;
    return bytes < want && allocate(bytes) ? bytes : 0;
}
