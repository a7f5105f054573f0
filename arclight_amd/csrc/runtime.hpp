// Host-side helpers shared by the C ABI translation units.
#pragma once

#include <hip/hip_runtime.h>

// Record a failure message for al_last_error() and return `code`.
int al_fail(int code, const char * fmt, ...) __attribute__((format(printf, 2, 3)));
int al_hip_fail(hipError_t e, const char * what);
void al_clear_error();

// Per-device state, created on first use with the device current.
int al_device_cu_count(int * n_cu);
int al_device_lds_per_block(int * bytes);
int al_device_error_flag(int ** flag);   // its words: device_errors.hpp

// Records of a call with no workspace of its own: `bytes` of the library's
// workspace of (current device, stream), behind its counters. No initial
// value; calls on one stream share it.
int al_library_workspace(size_t bytes, void * stream, void ** ptr);

// The quantized activations of the Q4_0 projection: memory of (current device,
// stream) apart from its workspace, kOperandBytes whatever `bytes` (64 tokens
// of K = 16384 take 1.1 MB). Allocated on first use, inside a capture too.
constexpr size_t kOperandBytes = (size_t) 2 << 20;
int al_library_operands(size_t bytes, void * stream, void ** ptr);
