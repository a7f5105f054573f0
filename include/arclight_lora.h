/*
 * arclight_lora.h - C ABI of low-rank adapters of many requests at once,
 * beside a projection that the requests share.
 *
 * The reference's build_lora_mm (nnml/src/cgraph.cpp:497-500) adds to a
 * projection W x the product of the one adapter that its context has loaded.
 * Here every row of activations names its own adapter, as the rows of a
 * server's batch do:
 *     y[t] = base[t] + s_a B_a (A_a x[t]),   a = ids[t]   (a < 0: base[t])
 * with the adapters resident in slots of one size, their ranks their own.
 * Both products are those of f32 arithmetic for finite operands: a row whose x
 * is not finite, or whose adapter's weights in use are not, may be NaN where
 * f32 arithmetic gives an infinity.
 *
 * All data pointers are device pointers of the current device; no pointer is
 * kept after a call returns. Error convention as arclight_fattn.h. Calls
 * enqueue on `stream` without synchronizing.
 */
#ifndef ARCLIGHT_LORA_H
#define ARCLIGHT_LORA_H

#include <stdint.h>

#include "arclight_fattn.h"
#include "arclight_matmul.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 *   a       f16 ne = [K, R, n_adapters], nb0 = 2: A_a, a row for each rank
 *   b       f16 ne = [R, N, n_adapters], nb0 = 2: B_a, R values for each
 *           output. Rows of a and b 16-byte aligned (data and strides).
 *   ranks   i32 [n_adapters], device: each adapter's rank, 0 to R (data NULL:
 *           R). What a slot holds beyond it is not used and may be anything.
 *   scales  f32 [n_adapters], device (data NULL: 1)
 *   ids     i32 [T], device: the adapter of each row, negative: none
 *   x       f32 ne = [K, T], nb0 = 4, rows 16-byte aligned
 *   base    f32 ne = [N, T], nb0 = 4, or data NULL: y's own content (y +=).
 *           May be y itself, or columns beside y's of a wider matrix, and may
 *           not overlap it otherwise.
 *           (al_mul_mat_q4_0_lora_f32: not used)
 *   y       f32 ne = [N, T], nb0 = 4. May not overlap x.
 *   w       Q4_0 ne = [K, N] (al_mul_mat_q4_0_lora_f32 only)
 * K and R are multiples of 8, R at most 128, K at most 65536, T at most 2^19,
 * n_adapters at most 2^20; an adapter's A and its B span less than 4 GB each
 * (AL_ERR_UNSUPPORTED otherwise). The rows of ids, x and y may name the
 * adapters in any order. An id of
 * n_adapters or more, or a rank outside 0 to R, is not followed: the row is
 * NaN, and al_device_errors() returns AL_ERR_INVALID after the stream
 * completes.
 * workspace: device scratch (al_lora_workspace_bytes), NULL: the library's
 * own for (current device, stream), as al_fattn_f16: then one eager call of
 * the same shapes has to come before a capture. Calls and replays that share
 * a workspace must be ordered on one stream. It needs no initial value; its
 * first 256 KiB are not touched, so that it may also be al_fattn_f16's.
 */
typedef struct al_lora_args {
    al_tensor a;
    al_tensor b;
    al_tensor ranks;
    al_tensor scales;
    al_tensor ids;
    al_tensor x;
    al_tensor base;
    al_tensor y;
    al_tensor w;
    void *    stream;
    void *    workspace;
    uint64_t  workspace_bytes;
} al_lora_args;

/* y = base + the adapters' products, beside any projection (w is not used). */
int al_lora_f32(const al_lora_args * args);

/* y = W x, as al_mul_mat_q4_0_f32 computes it and with its limits on K, N and
 * T, + the adapters' products of x (of its f32 values, not of the 8-bit
 * blocks that the projection rounds them to). */
int al_mul_mat_q4_0_lora_f32(const al_lora_args * args);

/* Bytes of a caller's workspace that al_mul_mat_q4_0_lora_f32 needs for these
 * arguments, or without w al_lora_f32; 0 for refused ones. */
uint64_t al_lora_workspace_bytes(const al_lora_args * args);

#ifdef __cplusplus
}
#endif

#endif /* ARCLIGHT_LORA_H */
