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

// Where a call's `bytes` of records lie: in the caller's workspace, or (NULL) in
// the library's of (current device, stream). No initial value; calls on one
// stream share it. They lie behind the counters that every workspace begins
// with, which al_fattn_f16 carries from call to call, so that any calls may
// share one. what: the caller's name.
size_t al_workspace_bytes(size_t records);      // of a workspace with so many of records
int al_workspace_records(const char * what, size_t bytes, void * workspace, uint64_t workspace_bytes, void * stream, void ** ptr);

// The quantized activations of the Q4_0 projection: memory of (current device,
// stream) apart from its workspace, kOperandBytes whatever `bytes` (64 tokens
// of K = 16384 take 1.1 MB). Allocated on first use, inside a capture too.
constexpr size_t kOperandBytes = (size_t) 2 << 20;
int al_library_operands(size_t bytes, void * stream, void ** ptr);
