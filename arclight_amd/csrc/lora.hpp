// Low-rank adapters of many requests: the parts that the adapters' own kernels
// (lora.hip) and the Q4_0 projection's (matmul_q4.hip) share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/arclight_lora.h"
#include "device_common.hpp"

namespace lora {

constexpr int kTile = 16;                       // rows of x of a matrix product
constexpr int kMaxR = 128;
constexpr int kParts = 8;                       // parts of K at most
constexpr int kFew = 64;                        // rows that one wave's lanes hold the ids of

struct LoraParams {
    const char * a;  int64_t a_nb1, a_nb2;      // rank row, adapter
    const char * b;  int64_t b_nb1, b_nb2;      // output, adapter
    const int32_t * ranks;                      // or null
    const float * scales;                       // or null
    const int32_t * ids;
    const char * x;     int64_t x_nb1;
    const char * base;  int64_t base_nb1;
    char * y;           int64_t y_nb1;
    float * v;                                  // [ks][T][R]
    int32_t K, N, R, T, n_adapters;
    int32_t ks, k_step;                         // parts of K, columns of one (a multiple of 32)
    int32_t slots;                              // workgroups that share a tile's adapters (more than kFew rows)
    int32_t copy;                               // base is not y: rows without an adapter are copied
    int32_t y_vec;                              // y and base rows 16-byte aligned, N a multiple of 4
    int * err;
};

constexpr int min_c(int a, int b) { return a < b ? a : b; }

// Power of two that brings a row's largest value to [2^11, 2^12), and its
// inverse. top: the largest size of this lane's values, the row in the 4 lanes
// {n, n + 16, n + 32, n + 48}.
__device__ __forceinline__ void row_scale(float top, float & up, float & down) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_int(top), __float_as_int(top), false, false);
    top = fmaxf(__int_as_float((int) a[0]), __int_as_float((int) a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_int(top), __float_as_int(top), false, false);
    top = fmaxf(__int_as_float((int) b[0]), __int_as_float((int) b[1]));
    const int ex = min(max((int) (__float_as_uint(top) >> 23), 12), 253) - 127;
    up = __uint_as_float((uint32_t) (11 - ex + 127) << 23);
    down = __uint_as_float((uint32_t) (ex - 11 + 127) << 23);
}

// Rank of adapter a, -1 for one that is not to be used.
__device__ __forceinline__ int rank_of(const LoraParams & p, const int a) {
    if (a >= p.n_adapters) return -1;
    const int r = p.ranks ? p.ranks[a] : p.R;
    return r < 0 || r > p.R ? -1 : r;
}

__device__ __forceinline__ void lora_error(const LoraParams & p, const int a) {
    if (atomicCAS(p.err + 8, 0, 1) == 0) p.err[9] = a;
}

// Rows that share an adapter, out of at most 64 whose ids the wave's lanes
// hold: lane n's row is the n-th bit of `rows`, the first one beyond the last.
__device__ __forceinline__ int nth_row(uint64_t rows, const int n) {
    int row = __builtin_ctzll(rows);
    for (int i = 0; i < kTile && rows; ++i, rows &= rows - 1)
        if (n == i) row = __builtin_ctzll(rows);
    return row;
}
__device__ __forceinline__ uint64_t without_16(uint64_t rows) {
    for (int i = 0; i < kTile && rows; ++i) rows &= rows - 1;
    return rows;
}

// The columns of a wave: rounds of 32 U from k0 to k1, beginning with another
// round in every tile. Rows of x are often a power of two apart, and so the
// same columns of all rows in the same few memory channels: waves that take
// ranges apart from one another, and tiles that begin apart, use them all.
struct Columns {
    int k0, k1, rounds, at;
    template <int U> __device__ __forceinline__ static Columns of(const LoraParams & p, const int part, const int tile, const int wave,
                                                                  const int waves) {
        const int a = part * p.k_step, b = min(a + p.k_step, p.K), own = (p.k_step / 32 + waves - 1) / waves * 32;
        Columns c;
        c.k0 = min(a + wave * own, b);
        c.k1 = min(c.k0 + own, b);
        c.rounds = (c.k1 - c.k0 + 32 * U - 1) / (32 * U);
        c.at = c.rounds > 1 ? tile % c.rounds : 0;
        return c;
    }
    template <int U> __device__ __forceinline__ int column() const { return k0 + at * 32 * U; }
    __device__ __forceinline__ void next() { at = at + 1 == rounds ? 0 : at + 1; }
};

// This lane's columns of U runs of 32 from k on; column 0 for those
// beyond k1, which shrink() zeroes.
template <int U>
__device__ __forceinline__ void load_x(const char * xr, const int k, const int k1, const int g, float4 (&x)[U][2]) {
#pragma unroll
    for (int b = 0; b < U; ++b) {
        const int kl = k + 32 * b + 8 * g;                             // K is a multiple of 8
        const float4 * at = (const float4 *) (xr + (int64_t) (kl < k1 ? kl : 0) * 4);
        x[b][0] = at[0];
        x[b][1] = at[1];
    }
}

// Sum of A's rows with the tile's rows over a wave's columns, RT tiles of 16
// ranks. Lane 16 g + n loads 8 columns of rank row n and of row n of x (8 g ..
// 8 g + 7 of each 32). x holds the first round's activations. The next round's loads go out before this round's
// products (the asm statements keep the compiler from sinking them to their
// uses): without that all waves of a launch load and compute in step.
template <int RT, int U>
__device__ __forceinline__ void shrink(const LoraParams & p, const char * ar, const int rank, const char * xr, float4 (&x)[U][2],
                                       Columns c, const int n, const int g, float (*part)[kTile + 1]) {
    floatx4 acc[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) acc[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const char * rows[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) rows[u] = ar + (int64_t) min(16 * u + n, rank - 1) * p.a_nb1;
    auto load_w = [&](const int k, half8 (&w)[U][RT]) {
#pragma unroll
        for (int b = 0; b < U; ++b) {
            const int kl = k + 32 * b + 8 * g;
#pragma unroll
            for (int u = 0; u < RT; ++u) w[b][u] = *(const half8 *) (rows[u] + (int64_t) (kl < c.k1 ? kl : 0) * 2);
        }
        asm volatile("" ::: "memory");
    };
    auto multiply = [&](const int k, float4 (&y)[U][2], half8 (&w)[U][RT]) {
        if (k + 32 * U > c.k1) {
#pragma unroll
            for (int b = 0; b < U; ++b)
                if (k + 32 * b + 8 * g >= c.k1) {
                    y[b][0] = y[b][1] = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int u = 0; u < RT; ++u) w[b][u] = half8{};
                }
        }
        float top = 0.0f, up, down;
#pragma unroll
        for (int b = 0; b < U; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                top = fmaxf(fmaxf(fmaxf(top, fabsf(y[b][h].x)), fmaxf(fabsf(y[b][h].y), fabsf(y[b][h].z))), fabsf(y[b][h].w));
        row_scale(top, up, down);
        floatx4 sum[RT];
#pragma unroll
        for (int u = 0; u < RT; ++u) sum[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < U; ++b) {
            const float xs[8] = {y[b][0].x, y[b][0].y, y[b][0].z, y[b][0].w, y[b][1].x, y[b][1].y, y[b][1].z, y[b][1].w};
            half8 hi, lo;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const float z = xs[s] * up;
                hi[s] = (_Float16) z;
                lo[s] = (_Float16) (z - (float) hi[s]);
            }
#pragma unroll
            for (int u = 0; u < RT; ++u) sum[u] = mfma_16x16x32(w[b][u], hi, mfma_16x16x32(w[b][u], lo, sum[u]));
        }
#pragma unroll
        for (int u = 0; u < RT; ++u) acc[u] += sum[u] * down;
    };
    if (c.rounds > 0) {
        int k = c.column<U>();
        half8 w[U][RT];
        load_w(k, w);
        for (int i = 1; i < c.rounds; ++i) {
            c.next();
            const int kn = c.column<U>();
            float4 xn[U][2];
            half8 wn[U][RT];
            load_x<U>(xr, kn, c.k1, g, xn);
            load_w(kn, wn);
            multiply(k, x, w);
            k = kn;
#pragma unroll
            for (int b = 0; b < U; ++b) {
                x[b][0] = xn[b][0];
                x[b][1] = xn[b][1];
#pragma unroll
                for (int u = 0; u < RT; ++u) w[b][u] = wn[b][u];
            }
        }
        multiply(k, x, w);
    }
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[16 * u + 4 * g + i][n] = acc[u][i];
}

// A workgroup's part of v with few rows: those of row `lead`'s adapter, if it
// is the first of them (else another workgroup's), as the product's columns,
// so that A is read once whatever the order of the rows. part: WAVES x RT * 16
// x 17 floats.
template <int RT, int WAVES>
__device__ __forceinline__ void shrink_few(const LoraParams & p, const int lead, const int part_k, float (*part)[RT * 16][kTile + 1]) {
    constexpr int U = RT <= 2 ? 2 : 1;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = lane < p.T ? p.ids[lane] : -1;
    const int a = __builtin_amdgcn_readlane(id, lead);
    if (a < 0) return;
    uint64_t rows = __ballot(id == a);
    if (__builtin_ctzll(rows) != lead) return;
    const int rank = __builtin_amdgcn_readfirstlane(rank_of(p, a));
    const float scale = p.scales && rank > 0 ? p.scales[a] : 1.0f;
    if (rank < 0 && threadIdx.x == 0) lora_error(p, a);
    if (rank <= 0) return;
    const Columns c = Columns::of<U>(p, part_k, 0, wave, WAVES);
    const char * ar = p.a + (int64_t) a * p.a_nb2;
    for (; rows; rows = without_16(rows)) {
        const int row = nth_row(rows, n);
        const int count = min(__builtin_popcountll(rows), kTile);
        const char * xr = p.x + (int64_t) row * p.x_nb1;
        float4 x[U][2];
        load_x<U>(xr, c.column<U>(), c.k1, g, x);
        if (RT >= 8 && rank > 64)      shrink<min_c(RT, 8), U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        else if (RT >= 4 && rank > 32) shrink<min_c(RT, 4), U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        else if (RT >= 2 && rank > 16) shrink<min_c(RT, 2), U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        else                           shrink<1, U>(p, ar, rank, xr, x, c, n, g, part[wave]);
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * RT * 16; i += 64 * WAVES) {
            const int tok = i / (RT * 16), j = i % (RT * 16);
            const int r = __shfl(row, tok);
            if (j >= rank || tok >= count) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v += part[w][j][tok];
            p.v[((int64_t) part_k * p.T + r) * p.R + j] = v * scale;
        }
        __syncthreads();
    }
}

// Waves of a workgroup that computes parts of v (RT 8: its LDS).
template <int RT> constexpr int shrink_waves() { return RT == 8 ? 4 : 8; }

// v of ranks j .. j + 3 of a row: its parts, and their sum in order. Ranks that
// the row's adapter does not have were never written and are anything.
__device__ __forceinline__ void load_parts(const LoraParams & p, const int row, const int j, float4 (&x)[kParts]) {
    const float * src = p.v + (int64_t) row * p.R + j;
    const int64_t part = (int64_t) p.T * p.R;
#pragma unroll
    for (int k = 0; k < kParts; ++k) x[k] = *(const float4 *) (src + min(k, p.ks - 1) * part);
}
__device__ __forceinline__ float4 sum_of(const LoraParams & p, const float4 (&x)[kParts]) {
    float4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kParts; ++k)
        if (k < p.ks) {
            s.x += x[k].x; s.y += x[k].y; s.z += x[k].z; s.w += x[k].w;
        }
    return s;
}
__device__ __forceinline__ float4 sum_parts(const LoraParams & p, const int row, const int j) {
    float4 x[kParts];
    load_parts(p, row, j, x);
    asm volatile("" ::: "memory");
    return sum_of(p, x);
}

// 8 ranks' share of an output: b . v over those below the rank.
__device__ __forceinline__ float dot8(const half8 b, const float * v, const int ranks) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(e < ranks ? (float) b[e] : 0.0f, e < ranks ? v[e] : 0.0f, s);
    return s;
}

}  // namespace lora
