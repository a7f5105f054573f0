// Cells of a paged KV cache (include/arclight_paged.h), as its kernels
// address them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/arclight_paged.h"
#include "device_errors.hpp"

// Pools of f16 [128, P, Hkv, n_pages] and the sequences' page tables. Strides
// in bytes, the table's in entries.
struct PagedPools {
    char * k;  int64_t k_nb1, k_nb2, k_nb3;    // cell, head, page
    char * v;  int64_t v_nb1, v_nb2, v_nb3;
    const int32_t * table;  int64_t t_nb1;
    int32_t n_seq, n_pages, max_pages, page_size;
    int32_t groups;                            // page_size / 8: pages in groups of 8 cells
    uint32_t magic;                            // ceil(2^32 / groups) (0 for 1)
    int * err;                                 // device error words (device_errors.hpp)
};

__device__ __forceinline__ void paged_error(const PagedPools & p, const int what, const int value) {
    if (atomicCAS(p.err + kErrPaged, 0, 1) == 0) {
        p.err[kErrPaged + 1] = what;
        p.err[kErrPaged + 2] = value;
    }
}

// Page (index into the sequence's table) of an 8-cell group, exact while
// group * groups < 2^32, which the host checks for the table's last one.
__device__ __forceinline__ uint32_t page_of_group(const PagedPools & p, const uint32_t group) {
    return p.groups == 1 ? group : __umulhi(group, p.magic);
}

// Checks the pools and the table and fills p. what: the caller's name.
int paged_pools(const char * what, const al_tensor * k, const al_tensor * v, const al_tensor * table, PagedPools * p);
