// The Q4_0 projection as a part of other calls (matmul_q4.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/arclight_matmul.h"
#include "lora.hpp"

// The checks of al_mul_mat_q4_0_f32; *scratch_bytes: the device scratch that
// the call needs (0: none).
int mul_mat_q4_0_check(const al_tensor * w, const al_tensor * x, const al_tensor * y, size_t * scratch_bytes);

// The call, with scratch of that size (checked arguments). p: the adapters'
// products added (NULL: none), where mul_mat_q4_0_takes_lora; their first one
// is part of it for the sizes that mul_mat_q4_0_shrinks says, and has
// to be there before it otherwise.
int mul_mat_q4_0_run(const al_tensor * w, const al_tensor * x, const al_tensor * y, const lora::LoraParams * p, void * scratch,
                     hipStream_t stream);
bool mul_mat_q4_0_takes_lora(const al_tensor * w, int T, int R);
bool mul_mat_q4_0_shrinks(const al_tensor * w, int T, int R);
