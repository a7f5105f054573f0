// The Q4_0 projection as a part of other calls (matmul_q4.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/arclight_matmul.h"

// The checks of al_mul_mat_q4_0_f32; *scratch_bytes: the device scratch that
// the call needs (0: none).
int mul_mat_q4_0_check(const al_tensor * w, const al_tensor * x, const al_tensor * y, size_t * scratch_bytes);

// The call, with scratch of that size (checked arguments).
int mul_mat_q4_0_run(const al_tensor * w, const al_tensor * x, const al_tensor * y, void * scratch, hipStream_t stream);
