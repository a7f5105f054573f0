// Low-rank adapters of many requests beside a shared projection
// (include/arclight_lora.h), for gfx950.
//
// Mathematics: v[t] = s_a A_a x[t], y[t] = base[t] + B_a v[t] for a = ids[t],
// to the accuracy of f32: the f16 weights are exact, and x and v are carried
// as pairs of f16, hi + lo to 2^-22, after a power of two for each row (and
// run of columns) that brings the largest to [2^11, 2^12), so that values of
// any size keep their bits. Two f16 products of 16 x 16 x 32 take an eighth of
// the matrix cores' time that f32 products (16 x 16 x 4) do.
//
// The products take 16 rows at a time, of one adapter: out of 64 or 256 rows at
// a time those of each adapter are picked, in any order (rows that lie next to
// one another, as a prompt's, come out as they are), so that A and B are read
// once for 16 of them. The first launch leaves the groups for the second.
//
// Two launches: the first product into the workspace, K split over workgroups
// where there are few rows, then the second, which sums the parts, for a slice
// of the outputs. (Beside the Q4_0 projection: parts of its launches.) 300 rows
// of 2560 -> 4096 in the order of their requests, ranks to 64: 13.4 us; shuffled
// over 12 adapters 21.2, as a group of rows then is of 5 on average.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/arclight_lora.h"
#include "device_common.hpp"
#include "kernel_args.hpp"
#include "lora.hpp"
#include "matmul_q4.hpp"
#include "runtime.hpp"

namespace {

using namespace lora;

constexpr int kWaves = 4;
constexpr int kCols = 256;                      // outputs of a workgroup

// Parts of v for at most kFew rows: (row, part of K) for each workgroup.
template <int RT>
__global__ __launch_bounds__(64 * shrink_waves<RT>(), RT == 8 ? 2 : 4) void lora_shrink_few_kernel(const LoraParams p) {
    __shared__ __attribute__((aligned(16))) float lds[shrink_waves<RT>() * shrink_lds<RT, shrink_unroll<RT>()>()];
    prefetch_params(p);
    shrink_few<RT, shrink_waves<RT>()>(p, blockIdx.x, blockIdx.y, lds);
}

__device__ __forceinline__ int32_t * record(const LoraParams & p, const int window, const int k) {
    return p.groups + (int64_t) (window * (p.window + p.slots) + k) * kRecord;
}

// Parts of v for more: every p.slots-th group of 64 W rows for a workgroup,
// which leaves its groups, and the end of them, for the second launch.
// Bound by x. Measured at 8000 rows of 4096, rank 16: 32 us, 4.1 TB/s.
template <int RT, int W>
__global__ __launch_bounds__(64 * shrink_waves<RT>(), RT == 8 ? 2 : 4) void lora_shrink_kernel(const LoraParams p) {
    constexpr int WAVES = shrink_waves<RT>();
    __shared__ __attribute__((aligned(16))) float lds[WAVES * shrink_lds<RT, shrink_unroll<RT>()>()];
    prefetch_params(p);
    const int lane = threadIdx.x & 63;
    for (int k = blockIdx.x;; k += p.slots) {
        Group<W> rows(p, blockIdx.y * 64 * W, lane);                   // anew, to leave the registers to the products
        const bool more = rows.at(p, k, p.copy, lane);
        if (!more) rows.count = 0;
        if (blockIdx.z == 0 && threadIdx.x < 64) put_rows(record(p, blockIdx.y, k), rows, lane);
        if (!more) break;
        if (rows.a < 0) continue;
        shrink_group<RT, WAVES>(p, rows, blockIdx.z, blockIdx.y * p.slots + blockIdx.x, lds);
        __syncthreads();                                               // the sums are read before the next group's
    }
}

// A slice of 256 outputs of a group's rows (with base that is not y, rows
// without an adapter are groups too, and copied). FEW: at most kFew rows, row
// blockIdx.y's group; else every p.slots-th group of p.window rows for a workgroup.
// The rows are the product's rows, the outputs its columns, output 4 n + u of a
// wave's 64 in column n of product u: lane 16 g + n holds outputs 4 n .. 4 n + 3
// of rows 4 g .. 4 g + 3, and a load or store covers 256 bytes of each of 4
// rows. The slices of a row come next to one another in the grid, so that
// workgroups that run together use all memory channels (the groups next to one
// another: 70 us instead of 55, then, for 8000 rows of 4096 outputs; several slices to
// a workgroup gained nothing). VEC: rows of y and base in whole 16 bytes;
// SPLIT: v in parts.
// Measured there, rank 16: 51.7 us, 5.1 TB/s (a plain copy: 5.5 at the best).
template <int RT, bool VEC, bool SPLIT>
__device__ __forceinline__ void expand_group(const LoraParams & p, const Rows & rows, float (*v)[RT * 16 + 4]) {
    constexpr int kPiece = RT == 1 ? 16 : 32;                          // ranks of a lane's load of B: 4 or 8 in each quarter
    constexpr int kSteps = kPiece / 4;
    constexpr int kPieces = RT * 16 / kPiece;
    typedef _Float16 piece __attribute__((ext_vector_type(kSteps)));
    typedef short bits __attribute__((ext_vector_type(kSteps)));
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = blockIdx.x * kCols + 64 * wave + 4 * n;            // the lane's outputs
    const int rank = rows.a >= 0 ? __builtin_amdgcn_readfirstlane(rank_of(p, rows.a)) : 0;
    // the lane's rows 4 g + i
    int at[4];
    float acc[4][4];                                               // [row][output]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        at[i] = __shfl(rows.row, 4 * g + i);
        const bool own = 4 * g + i < rows.count;
        const float * br = (const float *) (p.base + (int64_t) at[i] * p.base_nb1) + c0;
        if constexpr (VEC) {
            float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (own && c0 < p.N) x = *(const float4 *) br;
            acc[i][0] = x.x; acc[i][1] = x.y; acc[i][2] = x.z; acc[i][3] = x.w;
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[i][u] = own && c0 + u < p.N ? br[u] : 0.0f;
        }
    }
    // v, zeros beyond the ranks
    for (int i = threadIdx.x; i < kTile * RT * 4; i += 64 * kWaves) {
        const int tok = i / (RT * 4), j = 4 * (i - tok * (RT * 4));
        const int src = __shfl(rows.row, tok);
        float4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (j < rank && tok < rows.count) {
            if constexpr (SPLIT) s = sum_parts(p, src, j);
            else s = *(const float4 *) (p.v + (int64_t) src * p.R + j);
            if (j + 1 >= rank) s.y = 0.0f;
            if (j + 2 >= rank) s.z = 0.0f;
            if (j + 3 >= rank) s.w = 0.0f;
        }
        *(float4 *) &v[tok][j] = s;
    }
    __syncthreads();
    // this lane's ranks of row n, as the products' operands
    piece hi[kPieces], lo[kPieces];
    float up, down, top = 0.0f;
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) top = fmaxf(top, fabsf(v[n][q * kPiece + kSteps * g + s]));
    row_scale(colmax4(top), up, down);
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const float z = v[n][q * kPiece + kSteps * g + s] * up;
            hi[q][s] = (_Float16) z;
            lo[q][s] = (_Float16) (z - (float) hi[q][s]);
        }
    float downs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) downs[i] = __shfl(down, 4 * g + i);

    if (rows.a >= 0) {
        piece w[kPieces][4];
        const char * b = p.b + (int64_t) rows.a * p.b_nb2;
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
            if (q * kPiece >= rank) break;
            const int j0 = q * kPiece + kSteps * g;            // this lane's ranks
#pragma unroll
            for (int u = 0; u < 4; ++u)
                w[q][u] = *(const piece *) (b + ((uint32_t) min(c0 + u, p.N - 1) * (uint32_t) p.b_nb1 + 2u * (uint32_t) min(j0, p.R - kSteps)));
            if (q * kPiece + kPiece > rank) {                     // what lies behind the rank may be NaN
                bits in;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) in[s] = j0 + s < rank ? -1 : 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) w[q][u] = __builtin_bit_cast(piece, __builtin_bit_cast(bits, w[q][u]) & in);
            }
        }
        floatx4 sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
            if (q * kPiece >= rank) break;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (kSteps == 4) {
                    sum[u] = __builtin_amdgcn_mfma_f32_16x16x16f16(lo[q], w[q][u], sum[u], 0, 0, 0);
                    sum[u] = __builtin_amdgcn_mfma_f32_16x16x16f16(hi[q], w[q][u], sum[u], 0, 0, 0);
                } else {
                    sum[u] = mfma_16x16x32(hi[q], w[q][u], mfma_16x16x32(lo[q], w[q][u], sum[u]));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[i][u] = rank < 0 ? __builtin_nanf("") : acc[i][u] + sum[u][i] * downs[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (4 * g + i >= rows.count) continue;
        float * yr = (float *) (p.y + (int64_t) at[i] * p.y_nb1) + c0;
        if constexpr (VEC) {
            if (c0 < p.N) *(float4 *) yr = float4{acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (c0 + u < p.N) yr[u] = acc[i][u];
        }
    }
}

template <int RT, bool VEC, bool SPLIT, bool FEW>
__global__ __launch_bounds__(64 * kWaves) void lora_expand_kernel(const LoraParams p) {
    __shared__ __attribute__((aligned(16))) float v[kTile][RT * 16 + 4];
    prefetch_params(p);
    const int lane = threadIdx.x & 63;
    if constexpr (FEW) {
        Group<1> rows(p, 0, lane);
        if (rows.from_row(blockIdx.y, lane) && (rows.a >= 0 || p.copy)) expand_group<RT, VEC, SPLIT>(p, rows, v);
    } else {
        for (int k = blockIdx.y;; k += p.slots) {
            const Rows rows = get_rows(record(p, blockIdx.z, k), lane);
            if (rows.count == 0) break;
            if (k != (int) blockIdx.y) __syncthreads();                // the last group's v is read
            expand_group<RT, VEC, SPLIT>(p, rows, v);
        }
    }
}

struct Plan {
    LoraParams p;
    bool empty = false;
    size_t v_bytes = 0, g_bytes = 0, q_bytes = 0;       // v, then the groups or the projection's scratch
};

int make_plan(const al_lora_args * g, bool project, int n_cu, Plan * out) {
    if (!g) return al_fail(AL_ERR_INVALID, "lora: null arguments");
    const al_tensor &a = g->a, &b = g->b, &x = g->x, &y = g->y;
    if (!a.data || !b.data || !x.data || !y.data || !g->ids.data)
        return al_fail(AL_ERR_INVALID, "lora: a, b, x, ids and y are required");
    if (a.type != AL_TYPE_F16 || b.type != AL_TYPE_F16)
        return al_fail(AL_ERR_UNSUPPORTED, "lora: adapter types %d / %d (f16 only)", a.type, b.type);
    if (x.type != AL_TYPE_F32 || y.type != AL_TYPE_F32)
        return al_fail(AL_ERR_UNSUPPORTED, "lora: x / y types %d / %d (f32 only)", x.type, y.type);
    const int64_t K = a.ne[0], R = a.ne[1], A = a.ne[2], N = b.ne[1], T = x.ne[1];
    if (b.ne[0] != R || b.ne[2] != A || a.ne[3] != 1 || b.ne[3] != 1 || x.ne[0] != K || x.ne[2] != 1 || x.ne[3] != 1 ||
        y.ne[0] != N || y.ne[1] != T || y.ne[2] != 1 || y.ne[3] != 1)
        return al_fail(AL_ERR_INVALID, "lora: shapes a [K, R, n], b [R, N, n], x [K, T], y [N, T] do not fit: K %lld / %lld, R %lld / %lld",
                       (long long) K, (long long) x.ne[0], (long long) R, (long long) b.ne[0]);
    if (K < 8 || K % 8 || K > 65536 || R < 8 || R % 8 || R > kMaxR)
        return al_fail(AL_ERR_UNSUPPORTED, "lora: K %lld, R %lld (multiples of 8, at most 65536 and %d)", (long long) K, (long long) R, kMaxR);
    if (A < 1 || A > (1 << 20) || N < 1 || N > (1 << 22) || T < 0 || T > (1 << 19))
        return al_fail(AL_ERR_UNSUPPORTED, "lora: sizes out of range");
    auto al = [](const al_tensor & t, uint64_t by) { return !(((uintptr_t) t.data | t.nb[1] | t.nb[2]) & (by - 1)); };
    if (a.nb[0] != 2 || b.nb[0] != 2 || !al(a, 16) || !al(b, 16))
        return al_fail(AL_ERR_INVALID, "lora: rows of a and b must be contiguous and 16-byte aligned");
    if ((uint64_t) R * a.nb[1] >= (1ull << 32) || (uint64_t) N * b.nb[1] >= (1ull << 32))
        return al_fail(AL_ERR_UNSUPPORTED, "lora: an adapter spans more than 4 GB");
    if (x.nb[0] != 4 || ((uintptr_t) x.data & 15u) || x.nb[1] % 16 || y.nb[0] != 4 || ((uintptr_t) y.data & 3u) || y.nb[1] % 4 ||
        (T > 1 && y.nb[1] < (uint64_t) N * 4))
        return al_fail(AL_ERR_INVALID, "lora: rows of x must be 16-byte aligned, those of y contiguous and apart");
    if (g->ids.type != AL_TYPE_I32 || g->ids.ne[0] != T || g->ids.nb[0] != 4 || ((uintptr_t) g->ids.data & 3u))
        return al_fail(AL_ERR_INVALID, "lora: ids must be i32 [T]");
    if (g->ranks.data && (g->ranks.type != AL_TYPE_I32 || g->ranks.ne[0] != A || g->ranks.nb[0] != 4))
        return al_fail(AL_ERR_INVALID, "lora: ranks must be i32 [n_adapters]");
    if (g->scales.data && (g->scales.type != AL_TYPE_F32 || g->scales.ne[0] != A || g->scales.nb[0] != 4))
        return al_fail(AL_ERR_INVALID, "lora: scales must be f32 [n_adapters]");
    const al_tensor & base = g->base.data && !project ? g->base : y;
    if (base.type != AL_TYPE_F32 || base.ne[0] != N || base.ne[1] != T || base.ne[2] != 1 || base.ne[3] != 1 || base.nb[0] != 4 ||
        ((uintptr_t) base.data & 3u) || base.nb[1] % 4)
        return al_fail(AL_ERR_INVALID, "lora: base must be f32 [N, T]");
    if (T > 0 && (base.data != y.data || (T > 1 && base.nb[1] != y.nb[1]))) {
        const uintptr_t b0 = (uintptr_t) base.data, b1 = b0 + (uint64_t) (T - 1) * base.nb[1] + (uint64_t) N * 4;
        const uintptr_t y0 = (uintptr_t) y.data, y1 = y0 + (uint64_t) (T - 1) * y.nb[1] + (uint64_t) N * 4;
        // rows side by side, as columns of one wider matrix, are apart too
        const uint64_t s = y.nb[1], d = s ? (b0 - y0 + (b0 < y0 ? (y0 - b0 + s - 1) / s * s : 0)) % s : 0, row = (uint64_t) N * 4;
        const bool apart = base.nb[1] == s && d >= row && s - d >= row;
        if (b0 < y1 && y0 < b1 && !apart) return al_fail(AL_ERR_INVALID, "lora: base overlaps y and is not y");
    }
    Plan pl;
    LoraParams & p = pl.p;
    memset(&p, 0, sizeof(p));
    pl.empty = T == 0;
    p.a = (const char *) a.data; p.a_nb1 = a.nb[1]; p.a_nb2 = a.nb[2];
    p.b = (const char *) b.data; p.b_nb1 = b.nb[1]; p.b_nb2 = b.nb[2];
    p.ranks = (const int32_t *) g->ranks.data;
    p.scales = (const float *) g->scales.data;
    p.ids = (const int32_t *) g->ids.data;
    p.x = (const char *) x.data; p.x_nb1 = x.nb[1];
    p.base = (const char *) base.data; p.base_nb1 = base.nb[1];
    p.y = (char *) y.data; p.y_nb1 = y.nb[1];
    p.K = (int32_t) K; p.N = (int32_t) N; p.R = (int32_t) R; p.T = (int32_t) T; p.n_adapters = (int32_t) A;
    p.y_vec = N % 4 == 0 && !(((uintptr_t) y.data | y.nb[1] | (uintptr_t) base.data | base.nb[1]) & 15u);
    const int64_t tiles = (T + kTile - 1) / kTile;
    // Up to kFew rows take a workgroup for each row, of which those of an
    // adapter's first, 17th ... row work. Of more, groups are picked out of 64
    // rows at a time or of 256, which costs more for a small batch in the order
    // of its requests and saves half the groups of a shuffled one (us, ordered
    // and shuffled over 12 adapters of ranks 8 to 64, 2560 -> 4096: 300 rows
    // 13.5, 21.2 with 64, 18.9, 20.6 with 256; 500 16.8, 26.4 and 17.1, 22.2;
    // 2000 37, 68 and 38, 47).
    // They have at least 4 or 16 groups, which p.slots workgroups share, an odd
    // number, as workgroups go to the 8 XCDs in turn and the last slots have
    // little to do (8000 rows with 4, 5, 8 for 64 rows: 93, 86, 97). Many
    // adapters make many groups (us with 9 and 17: 122 rows shuffled over 29
    // adapters 36.2, 28.0, 300 rows over 9 13.7, 17.0).
    p.window = T <= 384 ? 64 : 256;
    p.slots = p.window == 256 ? 21 : A < 16 ? 9 : 17;
    p.copy = base.data != y.data;
    // K in parts of at least 512 columns while the CUs are not full.
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({kParts, (K + 511) / 512, T <= kFew ? n_cu / 16 : 2 * n_cu / tiles}));
    p.k_step = (int32_t) (((K + parts - 1) / parts + 31) / 32 * 32);
    p.ks = (int32_t) ((K + p.k_step - 1) / p.k_step);
    pl.v_bytes = ((size_t) p.ks * T * R * 4 + 255) / 256 * 256;
    if (!project && T > kFew) pl.g_bytes = (size_t) ((T + p.window - 1) / p.window) * (p.window + p.slots) * kRecord * 4;
    if (project) {
        const int rc = mul_mat_q4_0_check(&g->w, &x, &y, &pl.q_bytes);
        if (rc != AL_OK) return rc;
    }
    *out = pl;
    return AL_OK;
}

template <int RT, bool FEW>
hipError_t launch_expand(const LoraParams & p, const dim3 grid, hipStream_t st) {
    if (p.y_vec && p.ks > 1) hipLaunchKernelGGL((lora_expand_kernel<RT, true, true, FEW>), grid, dim3(64 * kWaves), 0, st, p);
    else if (p.y_vec)        hipLaunchKernelGGL((lora_expand_kernel<RT, true, false, FEW>), grid, dim3(64 * kWaves), 0, st, p);
    else                     hipLaunchKernelGGL((lora_expand_kernel<RT, false, true, FEW>), grid, dim3(64 * kWaves), 0, st, p);
    return hipGetLastError();
}

template <int RT>
hipError_t launch_shrink(const LoraParams & p, hipStream_t st) {
    constexpr int kThreads = 64 * shrink_waves<RT>();
    const unsigned windows = (unsigned) ((p.T + p.window - 1) / p.window);
    if (p.T <= kFew) hipLaunchKernelGGL(lora_shrink_few_kernel<RT>, dim3((unsigned) p.T, (unsigned) p.ks), dim3(kThreads), 0, st, p);
    else if (p.window == 64) hipLaunchKernelGGL((lora_shrink_kernel<RT, 1>), dim3((unsigned) p.slots, windows, (unsigned) p.ks), dim3(kThreads), 0, st, p);
    else hipLaunchKernelGGL((lora_shrink_kernel<RT, 4>), dim3((unsigned) p.slots, windows, (unsigned) p.ks), dim3(kThreads), 0, st, p);
    return hipGetLastError();
}

template <int RT>
hipError_t launch_expand(const LoraParams & p, hipStream_t st) {
    const unsigned windows = (unsigned) ((p.T + p.window - 1) / p.window), slices = (unsigned) ((p.N + kCols - 1) / kCols);
    return p.T <= kFew ? launch_expand<RT, true>(p, dim3(slices, (unsigned) p.T), st)
                       : launch_expand<RT, false>(p, dim3(slices, (unsigned) p.slots, windows), st);
}

int run(const al_lora_args * g, bool project) {
    Plan pl;
    int rc = make_plan(g, project, 1, &pl);                            // refusals need no device
    if (rc != AL_OK || pl.empty) return rc;
    int n_cu = 0;
    rc = al_device_cu_count(&n_cu);
    if (rc == AL_OK) rc = make_plan(g, project, n_cu, &pl);
    if (rc == AL_OK) rc = al_device_error_flag(&pl.p.err);
    if (rc != AL_OK) return rc;
    void * ws = nullptr;
    rc = al_workspace_records("lora", pl.v_bytes + pl.g_bytes + pl.q_bytes, g->workspace, g->workspace_bytes, g->stream, &ws);
    if (rc != AL_OK) return rc;
    pl.p.v = (float *) ws;
    pl.p.groups = (int32_t *) ((char *) ws + pl.v_bytes);
    const hipStream_t st = (hipStream_t) g->stream;
    const LoraParams & p = pl.p;
    const bool fused = project && mul_mat_q4_0_takes_lora(&g->w, p.T, p.R);
    hipError_t e = hipSuccess;
    if (!(fused && mul_mat_q4_0_shrinks(&g->w, p.T, p.R)))
        e = p.R <= 16 ? launch_shrink<1>(p, st) : p.R <= 32 ? launch_shrink<2>(p, st) : p.R <= 64 ? launch_shrink<4>(p, st) : launch_shrink<8>(p, st);
    if (e != hipSuccess) return al_hip_fail(e, "lora: launch");
    if (project) {
        rc = mul_mat_q4_0_run(&g->w, &g->x, &g->y, fused ? &p : nullptr, (char *) ws + pl.v_bytes, st);
        if (rc != AL_OK || fused) return rc;
    }
    e = p.R <= 16 ? launch_expand<1>(p, st) : p.R <= 32 ? launch_expand<2>(p, st) : p.R <= 64 ? launch_expand<4>(p, st) : launch_expand<8>(p, st);
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "lora: launch");
}

}  // namespace

extern "C" int al_lora_f32(const al_lora_args * args) { return run(args, false); }

extern "C" int al_mul_mat_q4_0_lora_f32(const al_lora_args * args) { return run(args, true); }

extern "C" uint64_t al_lora_workspace_bytes(const al_lora_args * args) {
    int n_cu = 0;
    Plan pl;
    if (al_device_cu_count(&n_cu) != AL_OK || make_plan(args, args && args->w.data != nullptr, n_cu, &pl) != AL_OK) return 0;
    return pl.empty ? 0 : al_workspace_bytes(pl.v_bytes + pl.g_bytes + pl.q_bytes);
}
