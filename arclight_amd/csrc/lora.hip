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
// Rows are taken in tiles of 16. A tile's columns (its rows of x) are
// independent in both products, so a tile of several adapters is computed
// once for each of them and every column kept from its own adapter's: right
// for any order of the ids, and done once where, as in a prompt, the rows of
// a tile share one.
//
// Two launches: lora_shrink_kernel (v, K split over workgroups, partial sums
// into the workspace) and lora_expand_kernel (sums the parts, then a slice of
// the outputs).

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

// The rows of a tile whose adapter no earlier row of it has, of a wave whose
// lanes hold row lane % 16's id (negative: none): one bit each.
__device__ __forceinline__ uint32_t leaders(const int id) {
    uint32_t left = (uint32_t) __ballot(id >= 0) & 0xffffu, out = 0;
    while (left) {
        const int i = __builtin_ctz(left);
        out |= 1u << i;
        left &= ~(uint32_t) __ballot(id == __builtin_amdgcn_readlane(id, i));
    }
    return out;
}

// The adapter of a workgroup: the slot-th (and every p.slots-th after it) of
// those that the tile's rows have, in the order of their first rows.
struct Turn {
    uint32_t todo;
    __device__ __forceinline__ void skip(const int n) {
        for (int i = 0; i < n && todo; ++i) todo &= todo - 1;
    }
};

// Parts of v for at most 64 rows: (row, part of K) for each workgroup.
template <int RT>
__global__ __launch_bounds__(64 * shrink_waves<RT>(), RT == 8 ? 2 : 4) void lora_shrink_few_kernel(const LoraParams p) {
    __shared__ float part[shrink_waves<RT>()][RT * 16][kTile + 1];
    prefetch_params(p);
    shrink_few<RT, shrink_waves<RT>()>(p, blockIdx.x, blockIdx.y, part);
}

// Parts of v for more: the columns of one part of K, of a tile's rows with the
// workgroup's adapters. RT: tiles of 16 ranks at most. The first round's
// activations, which need no id, are loaded before the ids are known.
template <int RT>
__global__ __launch_bounds__(64 * shrink_waves<RT>(), RT == 8 ? 2 : 4) void lora_shrink_kernel(const LoraParams p) {
    constexpr int WAVES = shrink_waves<RT>();
    constexpr int U = RT <= 2 ? 2 : 1;
    __shared__ float part[WAVES][RT * 16][kTile + 1];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kTile + n;
    const int id = t < p.T ? p.ids[t] : -1;
    const Columns c = Columns::of<U>(p, blockIdx.z, blockIdx.x, wave, WAVES);
    const char * xr = p.x + (int64_t) min(t, p.T - 1) * p.x_nb1;
    float4 x[U][2];
    load_x<U>(xr, c.column<U>(), c.k1, g, x);
    asm volatile("" ::: "memory");
    const int row_rank = id >= 0 ? rank_of(p, id) : 0;                 // every row's at once, not adapter by adapter
    const float row_scale = p.scales && row_rank > 0 ? p.scales[id] : 1.0f;
    Turn turn{leaders(id)};
    turn.skip(blockIdx.y);
    for (bool again = false; turn.todo; turn.skip(p.slots), again = true) {
        const int lead = __builtin_ctz(turn.todo);
        const int a = __builtin_amdgcn_readlane(id, lead), rank = __builtin_amdgcn_readlane(row_rank, lead);
        if (rank < 0) {
            if (threadIdx.x == 0) lora_error(p, a);
            continue;
        }
        if (rank == 0) continue;
        if (again && c.rounds != 1) load_x<U>(xr, c.column<U>(), c.k1, g, x);   // one round: x is still there
        const char * ar = p.a + (int64_t) a * p.a_nb2;
        if (RT >= 8 && rank > 64)      shrink<min_c(RT, 8), U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        else if (RT >= 4 && rank > 32) shrink<min_c(RT, 4), U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        else if (RT >= 2 && rank > 16) shrink<min_c(RT, 2), U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        else                           shrink<1, U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        __syncthreads();
        const float scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(row_scale), lead));
        const uint32_t rows = (uint32_t) __ballot(id == a) & 0xffffu;
        for (int i = threadIdx.x; i < kTile * RT * 16; i += 64 * WAVES) {
            const int tok = i / (RT * 16), j = i % (RT * 16);
            if (j >= rank || !(rows >> tok & 1)) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v += part[w][j][tok];
            p.v[((int64_t) blockIdx.z * p.T + blockIdx.x * kTile + tok) * p.R + j] = v * scale;
        }
        __syncthreads();
    }
}

// A slice of 256 outputs of rows that share a workgroup: with at most 64 rows
// (FEW) those of row `blockIdx.y`'s adapter, if it is their first; with more
// those of a tile that have one of the workgroup's adapters. Rows without an
// adapter are copied where base is not y: by their own workgroup, or by the
// tile's slot 0. Lane 16 g + n holds outputs 4 g .. 4 g + 3 of each 16, of row
// n. The slices of a row come next to one another in the grid, so that
// workgroups that run together use all memory channels. VEC: rows of y and
// base in whole 16 bytes; SPLIT: v in parts.
// Measured at 8000 rows of 4096 outputs, rank 16: 55 us, 4.8 TB/s, what a copy
// reaches; with 1024 or more outputs to a workgroup 63 to 72.
template <int RT, bool VEC, bool SPLIT, bool FEW>
__global__ __launch_bounds__(64 * kWaves) void lora_expand_kernel(const LoraParams p) {
    constexpr int kRow = RT * 16 + 4;
    constexpr int kPiece = RT == 1 ? 16 : 32;                          // ranks of a lane's load of B: 4 or 8 in each quarter
    constexpr int kSteps = kPiece / 4;
    constexpr int kPieces = RT * 16 / kPiece;
    typedef _Float16 piece __attribute__((ext_vector_type(kSteps)));
    typedef short bits __attribute__((ext_vector_type(kSteps)));
    __shared__ __attribute__((aligned(16))) float v[kTile][kRow];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = blockIdx.x * kCols + 64 * wave;
    // the columns' rows: which (row), whether they are this workgroup's
    // (mine), their adapters and ranks, and the first column of each adapter
    int row, id, rank;
    uint32_t mine, turns;
    uint64_t left = 0;
    if constexpr (FEW) {
        const int lead = blockIdx.y;
        id = lane < p.T ? p.ids[lane] : -1;
        const int a = __builtin_amdgcn_readlane(id, lead);
        left = a >= 0 ? __ballot(id == a) : p.copy ? 1ull << lead : 0;
        if (left == 0 || __builtin_ctzll(left) != lead) return;
        id = a;
        rank = a >= 0 ? rank_of(p, a) : 0;
        turns = a >= 0 ? 1 : 0;
    } else {
        row = blockIdx.y * kTile + n;
        id = row < p.T ? p.ids[row] : -1;
        rank = id >= 0 ? rank_of(p, id) : 0;
        Turn turn{leaders(id)};
        turn.skip(blockIdx.z);
        mine = turns = 0;
        for (; turn.todo; turn.skip(p.slots)) {
            const int l = __builtin_ctz(turn.todo);
            turns |= 1u << l;
            mine |= (uint32_t) __ballot(id == __builtin_amdgcn_readlane(id, l));
        }
        if (blockIdx.z == 0 && p.copy) mine |= (uint32_t) __ballot(id < 0 && row < p.T);
        mine &= 0xffffu;
        if (!mine) return;
        row = min(row, p.T - 1);
    }
    do {
        if constexpr (FEW) {
            row = nth_row(left, n);
            mine = (1u << min(__builtin_popcountll(left), kTile)) - 1;
            left = without_16(left);
        }
        const bool own = mine >> n & 1;
        const char * br = p.base + (int64_t) row * p.base_nb1 + 16 * g;
        char * yr = p.y + (int64_t) row * p.y_nb1 + 16 * g;
        floatx4 acc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            acc[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            const int c = c0 + 16 * u + 4 * g;
            if constexpr (VEC) {
                if (own && c < p.N) acc[u] = *(const floatx4 *) (br + (int64_t) (c0 + 16 * u) * 4);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (own && c + i < p.N) acc[u][i] = *(const float *) (br + (int64_t) (c0 + 16 * u + i) * 4);
            }
        }
        // v, zeros beyond the ranks
        for (int i = threadIdx.x; i < kTile * RT * 4; i += 64 * kWaves) {
            const int tok = i / (RT * 4), j = 4 * (i - tok * (RT * 4));
            const int r = __shfl(rank, tok), at = __shfl(row, tok);
            float4 s = {0.0f, 0.0f, 0.0f, 0.0f};
            if (j < r && (mine >> tok & 1)) {
                if constexpr (SPLIT) s = sum_parts(p, at, j);
                else s = *(const float4 *) (p.v + (int64_t) at * p.R + j);
                if (j + 1 >= r) s.y = 0.0f;
                if (j + 2 >= r) s.z = 0.0f;
                if (j + 3 >= r) s.w = 0.0f;
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
        row_scale(top, up, down);
#pragma unroll
        for (int q = 0; q < kPieces; ++q)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const float z = v[n][q * kPiece + kSteps * g + s] * up;
                hi[q][s] = (_Float16) z;
                lo[q][s] = (_Float16) (z - (float) hi[q][s]);
            }

        for (uint32_t todo = turns; todo; todo &= todo - 1) {
            const int l = __builtin_ctz(todo);
            const int a = __builtin_amdgcn_readlane(id, l), r = __builtin_amdgcn_readlane(rank, l);
            const char * b = p.b + (int64_t) a * p.b_nb2;
            floatx4 sum[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < kPieces; ++q) {
                if (q * kPiece >= r) break;
                const int j0 = q * kPiece + kSteps * g;                // this lane's ranks
                piece w[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    w[u] = *(const piece *) (b + (int64_t) min(c0 + 16 * u + n, p.N - 1) * p.b_nb1 + 2 * min(j0, p.R - kSteps));
                if (q * kPiece + kPiece > r) {                         // what lies behind the rank may be NaN
                    bits in;
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) in[s] = j0 + s < r ? -1 : 0;
#pragma unroll
                    for (int u = 0; u < 4; ++u) w[u] = __builtin_bit_cast(piece, __builtin_bit_cast(bits, w[u]) & in);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if constexpr (kSteps == 4) {
                        sum[u] = __builtin_amdgcn_mfma_f32_16x16x16f16(w[u], lo[q], sum[u], 0, 0, 0);
                        sum[u] = __builtin_amdgcn_mfma_f32_16x16x16f16(w[u], hi[q], sum[u], 0, 0, 0);
                    } else {
                        sum[u] = mfma_16x16x32(w[u], hi[q], mfma_16x16x32(w[u], lo[q], sum[u]));
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] = acc[u] + sum[u] * down;
            if (r < 0)
#pragma unroll
                for (int u = 0; u < 4; ++u) sum[u] = floatx4{1.0f, 1.0f, 1.0f, 1.0f} * __builtin_nanf("");
            if (id == a)
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[u] = sum[u];
        }
        if (own)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = c0 + 16 * u + 4 * g;
                if constexpr (VEC) {
                    if (c < p.N) *(floatx4 *) (yr + (int64_t) (c0 + 16 * u) * 4) = acc[u];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c + i < p.N) *(float *) (yr + (int64_t) (c0 + 16 * u + i) * 4) = acc[u][i];
                }
            }
        if constexpr (FEW) __syncthreads();                                // v is read before the next rows' is written
    } while (FEW && left);
}

struct Plan {
    LoraParams p;
    bool empty = false;
    size_t v_bytes = 0, q_bytes = 0;            // v, then the projection's scratch
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
    if (T > 0 && (base.data != y.data || base.nb[1] != y.nb[1])) {
        const uintptr_t b0 = (uintptr_t) base.data, b1 = b0 + (uint64_t) (T - 1) * base.nb[1] + (uint64_t) N * 4;
        const uintptr_t y0 = (uintptr_t) y.data, y1 = y0 + (uint64_t) (T - 1) * y.nb[1] + (uint64_t) N * 4;
        if (b0 < y1 && y0 < b1) return al_fail(AL_ERR_INVALID, "lora: base overlaps y and is not y");
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
    // Up to 64 rows take a workgroup for each row, of which those of an
    // adapter's first row work; more take tiles, whose adapters share 4
    // workgroups up to 64 tiles, 1 beyond. K in parts of at least 512 columns
    // while there are CUs for them.
    p.slots = tiles <= 64 ? 4 : 1;
    p.copy = base.data != y.data;
    const int64_t groups = T <= kFew ? 16 : 2 * tiles;
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({kParts, (K + 511) / 512, n_cu / std::max<int64_t>(1, groups)}));
    p.k_step = (int32_t) (((K + parts - 1) / parts + 31) / 32 * 32);
    p.ks = (int32_t) ((K + p.k_step - 1) / p.k_step);
    pl.v_bytes = ((size_t) p.ks * T * R * 4 + 255) / 256 * 256;
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
    const unsigned tiles = (unsigned) ((p.T + kTile - 1) / kTile);
    if (p.T <= kFew) hipLaunchKernelGGL(lora_shrink_few_kernel<RT>, dim3((unsigned) p.T, (unsigned) p.ks), dim3(kThreads), 0, st, p);
    else             hipLaunchKernelGGL(lora_shrink_kernel<RT>, dim3(tiles, (unsigned) p.slots, (unsigned) p.ks), dim3(kThreads), 0, st, p);
    return hipGetLastError();
}

template <int RT>
hipError_t launch_expand(const LoraParams & p, hipStream_t st) {
    const unsigned tiles = (unsigned) ((p.T + kTile - 1) / kTile), slices = (unsigned) ((p.N + kCols - 1) / kCols);
    return p.T <= kFew ? launch_expand<RT, true>(p, dim3(slices, (unsigned) p.T), st)
                       : launch_expand<RT, false>(p, dim3(slices, tiles, (unsigned) p.slots), st);
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
    const size_t need = pl.v_bytes + pl.q_bytes;
    void * ws = g->workspace;
    if (ws) {
        if (g->workspace_bytes < need || ((uintptr_t) ws & 15u))
            return al_fail(AL_ERR_WORKSPACE, "lora: workspace %llu bytes (16-byte aligned) < %zu needed",
                           (unsigned long long) g->workspace_bytes, need);
    } else {
        rc = al_library_workspace(need, g->stream, &ws);
        if (rc != AL_OK) return rc;
    }
    pl.p.v = (float *) ws;
    const hipStream_t st = (hipStream_t) g->stream;
    const LoraParams & p = pl.p;
    const bool fused = project && mul_mat_q4_0_takes_lora(&g->w, p.T, p.R);
    hipError_t e = hipSuccess;
    if (!(fused && mul_mat_q4_0_shrinks(p.T)))
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
    return pl.empty ? 0 : pl.v_bytes + pl.q_bytes;
}
