// Low-rank adapters of many requests: the parts that the adapters' own kernels
// (lora.hip) and the Q4_0 projection's (matmul_q4.hip) share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/arclight_lora.h"
#include "device_common.hpp"
#include "device_errors.hpp"

namespace lora {

constexpr int kTile = 16;                       // rows of x of a matrix product
constexpr int kMaxR = 128;
constexpr int kParts = 8;                       // parts of K at most
constexpr int kFew = 64;                        // rows whose ids a wave's lanes hold, one each

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
    int32_t * groups;                           // [T / window][window + slots] records (more than kFew rows)
    int32_t K, N, R, T, n_adapters;
    int32_t ks, k_step;                         // parts of K, columns of one (a multiple of 32)
    int32_t window, slots;                      // rows that groups are picked from, workgroups that share those (more than kFew rows)
    int32_t copy;                               // base is not y: rows without an adapter are copied
    int32_t y_vec;                              // y and base rows 16-byte aligned, N a multiple of 4
    int * err;
};

constexpr int min_c(int a, int b) { return a < b ? a : b; }

// Power of two that brings a row's largest value, of size top, to [2^11,
// 2^12), and its inverse.
__device__ __forceinline__ void row_scale(const float top, float & up, float & down) {
    const int ex = min(max((int) (__float_as_uint(top) >> 23), 12), 253) - 127;
    up = __uint_as_float((uint32_t) (11 - ex + 127) << 23);
    down = __uint_as_float((uint32_t) (ex - 11 + 127) << 23);
}
// The value of another lane of the quad.
template <int CTRL>
__device__ __forceinline__ float quad_perm(const float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}

// Rank of adapter a, -1 for one that is not to be used.
__device__ __forceinline__ int rank_of(const LoraParams & p, const int a) {
    if (a >= p.n_adapters) return -1;
    const int r = p.ranks ? p.ranks[a] : p.R;
    return r < 0 || r > p.R ? -1 : r;
}

__device__ __forceinline__ void lora_error(const LoraParams & p, const int a) {
    if (atomicCAS(p.err + kErrLora, 0, 1) == 0) p.err[kErrLora + 1] = a;
}

// Up to 16 rows that share an adapter (a < 0: have none). Lane n < 16 has the
// n-th in `row` (the first one beyond the last).
struct Rows {
    int a, count, row;
};
// As the first launch leaves them for the second.
constexpr int kRecord = 20;                     // rows, a, count
__device__ __forceinline__ void put_rows(int32_t * at, const Rows r, const int lane) {
    if (lane < 18) at[lane] = lane == 17 ? +r.count : lane == 16 ? +r.a : +r.row;
}
__device__ __forceinline__ Rows get_rows(const int32_t * at, const int lane) {
    const int x = at[min(lane, 17)];
    return {__builtin_amdgcn_readlane(x, 16), __builtin_amdgcn_readlane(x, 17), x};
}

// Picks them out of the 64 W rows from `first` on, whose ids the lanes of a
// wave hold.
template <int W>
struct Group : Rows {
    int id[W], first;                           // the ids of rows first + 64 w + lane
    __device__ __forceinline__ Group(const LoraParams & p, const int first, const int lane) : first(first) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int r = first + 64 * w + lane;
            id[w] = r < p.T ? p.ids[r] : -1;
        }
    }
    // The `all` rows of `same` from its 16 chunk-th on: each sends its number to
    // the lane of its place (the others' go to lane 63, which nothing reads;
    // lanes that nothing is sent to get 0).
    __device__ __forceinline__ void take(const uint64_t (&same)[W], const int all, const int chunk, const int lane) {
        int before = -chunk * kTile;
        row = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int place = __builtin_amdgcn_mbcnt_hi((uint32_t) (same[w] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) same[w], before));
            const bool mine = (same[w] >> lane & 1) && place >= 0 && place < kTile;
            row |= __builtin_amdgcn_ds_permute(4 * (mine ? place : 63), 64 * w + lane);
            before += __builtin_popcountll(same[w]);
        }
        row += first;
        count = min(all - chunk * kTile, kTile);
        if (lane >= count) row = __builtin_amdgcn_readfirstlane(row);
    }
    // Those of row `lead` on that share its adapter, if it is the first of
    // them, or the 17th, the 33rd ...; false if another row is. (W = 1)
    __device__ __forceinline__ bool from_row(const int lead, const int lane) {
        a = __builtin_amdgcn_readlane(id[0], lead);
        const uint64_t same[1] = {a < 0 ? 1ull << lead : __ballot(id[0] == a)};
        const int before = __builtin_popcountll(same[0] & ((1ull << lead) - 1));
        if (before % kTile) return false;
        take(same, __builtin_popcountll(same[0]), before / kTile, lane);
        return true;
    }
    // The k-th group, adapters in the order of their first rows, then, if
    // `none` is set, the rows without one; false beyond the last.
    __device__ __forceinline__ bool at(const LoraParams & p, int k, const bool none, const int lane) {
        uint64_t left[W], same[W];
        int all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            left[w] = __ballot(id[w] >= 0);
            same[w] = 0;
        }
#pragma unroll
        for (int v = 0; v < W; ++v) {
            while (left[v]) {
                a = __builtin_amdgcn_readlane(id[v], __builtin_ctzll(left[v]));
                all = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    same[w] = w < v ? 0 : __ballot(id[w] == a);
                    left[w] &= ~same[w];
                    all += __builtin_popcountll(same[w]);
                }
                const int chunks = (all + kTile - 1) / kTile;
                if (k < chunks) {
                    take(same, all, k, lane);
                    return true;
                }
                k -= chunks;
            }
        }
        a = -1;
        all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            same[w] = none ? __ballot(id[w] < 0 && first + 64 * w + lane < p.T) : 0;
            all += __builtin_popcountll(same[w]);
        }
        if (k * kTile >= all) return false;
        take(same, all, k, lane);
        return true;
    }
};

// The columns of a wave: rounds of 32 U from k0 to k1, beginning with another
// round in every workgroup. Rows of x are often a power of two apart, and so the
// same columns of all rows in the same few memory channels: waves that take
// ranges apart from one another, and workgroups that begin apart, use them all.
struct Columns {
    int k0, k1, rounds, at;
    template <int U> __device__ __forceinline__ static Columns of(const LoraParams & p, const int part, const int turn, const int wave,
                                                                  const int waves) {
        const int a = part * p.k_step, b = min(a + p.k_step, p.K), own = (p.k_step / 32 + waves - 1) / waves * 32;
        Columns c;
        c.k0 = min(a + wave * own, b);
        c.k1 = min(c.k0 + own, b);
        c.rounds = (c.k1 - c.k0 + 32 * U - 1) / (32 * U);
        c.at = c.rounds > 1 ? turn % c.rounds : 0;
        return c;
    }
    template <int U> __device__ __forceinline__ int column() const { return k0 + at * 32 * U; }
    __device__ __forceinline__ void next() { at = at + 1 == rounds ? 0 : at + 1; }
};

// Loads and products hold a tile differently. A load's consecutive lanes take
// consecutive 16 bytes, four lanes a row's run (row l / 4, piece l % 4): lanes
// that lie in different rows cost a cycle each, 64 instead of 16 for a load.
// The product's operands have row n and piece g in lane 16 g + n. A wave turns
// one into the other through 1 KB of LDS of its own; the xor keeps both sides
// free of bank conflicts.
__device__ __forceinline__ int slot(const int row, const int piece) { return 4 * row + (piece ^ (row >> 2)); }

// This lane's 8 columns of its row in U runs of 32 from k on; column 0 for
// those beyond k1, which shrink() zeroes.
template <int U>
__device__ __forceinline__ void load_x(const char * xr, const int k, const int k1, const int piece, float4 (&x)[U][2]) {
#pragma unroll
    for (int b = 0; b < U; ++b) {
        const int kl = k + 32 * b + 8 * piece;                         // K is a multiple of 8
        const float4 * at = (const float4 *) (xr + (int64_t) (kl < k1 ? kl : 0) * 4);
        x[b][0] = at[0];
        x[b][1] = at[1];
    }
}

// Waves of a workgroup that computes parts of v, and runs of 32 columns that a
// wave loads before it uses them (RT 8: its LDS and registers).
template <int RT> constexpr int shrink_waves() { return RT == 8 ? 4 : 8; }
template <int RT> constexpr int shrink_unroll() { return RT <= 2 ? 2 : 1; }

// Floats of LDS that shrink() needs for a wave: the tile's turning, then the
// wave's sums.
template <int RT, int U> constexpr int shrink_lds() {
    return (2 * U + U * RT) * 256 > RT * 16 * (kTile + 1) ? (2 * U + U * RT) * 256 : RT * 16 * (kTile + 1);
}

// Sum of A's rows with the group's rows over a wave's columns, RT tiles of 16
// ranks, into part[rank][row]. xr: the row of x that this lane loads of, x: its
// first round's activations. The next round's loads go out before this round's
// products (the asm statement keeps the compiler from sinking them to their
// uses): without that all waves of a launch load and compute in step.
template <int RT, int U>
__device__ __forceinline__ void shrink(const LoraParams & p, const char * ar, const int rank, const char * xr, float4 (&x)[U][2],
                                       Columns c, const int lane, float * lds) {
    const int n = lane & 15, g = lane >> 4, lrow = lane >> 2, piece = lane & 3;
    floatx4 acc[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) acc[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t rows[RT];                                                 // (an adapter's A is below 4 GB)
#pragma unroll
    for (int u = 0; u < RT; ++u) rows[u] = (uint32_t) min(16 * u + lrow, rank - 1) * (uint32_t) p.a_nb1;
    auto load_w = [&](const int k, half8 (&w)[U][RT]) {
#pragma unroll
        for (int b = 0; b < U; ++b) {
            const int kl = k + 32 * b + 8 * piece;
#pragma unroll
            for (int u = 0; u < RT; ++u) w[b][u] = *(const half8 *) (ar + (rows[u] + 2u * (uint32_t) (kl < c.k1 ? kl : 0)));
        }
        asm volatile("" ::: "memory");
    };
    u32x4 * turn = (u32x4 *) lds;
    auto multiply = [&](const int k, float4 (&y)[U][2], half8 (&w)[U][RT]) {
        if (k + 32 * U > c.k1) {
#pragma unroll
            for (int b = 0; b < U; ++b)
                if (k + 32 * b + 8 * piece >= c.k1) {
                    y[b][0] = y[b][1] = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int u = 0; u < RT; ++u) w[b][u] = half8{};
                }
        }
        // the row, in 4 neighbouring lanes: its scale, and its two f16 parts
        float top = 0.0f, up, down;
#pragma unroll
        for (int b = 0; b < U; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                top = fmaxf(fmaxf(fmaxf(top, fabsf(y[b][h].x)), fmaxf(fabsf(y[b][h].y), fabsf(y[b][h].z))), fabsf(y[b][h].w));
        top = fmaxf(top, quad_perm<0xb1>(top));
        top = fmaxf(top, quad_perm<0x4e>(top));
        row_scale(top, up, down);
        down = __shfl(down, 4 * n);                                    // row n's
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
            turn[2 * b * 64 + slot(lrow, piece)] = __builtin_bit_cast(u32x4, hi);
            turn[(2 * b + 1) * 64 + slot(lrow, piece)] = __builtin_bit_cast(u32x4, lo);
#pragma unroll
            for (int u = 0; u < RT; ++u) turn[(2 * U + b * RT + u) * 64 + slot(lrow, piece)] = __builtin_bit_cast(u32x4, w[b][u]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        floatx4 sum[RT];
#pragma unroll
        for (int u = 0; u < RT; ++u) sum[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < U; ++b) {
            const half8 hi = as_half8(turn[2 * b * 64 + slot(n, g)]), lo = as_half8(turn[(2 * b + 1) * 64 + slot(n, g)]);
#pragma unroll
            for (int u = 0; u < RT; ++u) {
                const half8 a = as_half8(turn[(2 * U + b * RT + u) * 64 + slot(n, g)]);
                sum[u] = mfma_16x16x32(a, hi, mfma_16x16x32(a, lo, sum[u]));
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
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
            load_x<U>(xr, kn, c.k1, piece, xn);
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
        for (int i = 0; i < 4; ++i) lds[(16 * u + 4 * g + i) * (kTile + 1) + n] = acc[u][i];
}

// A workgroup's part of v for the rows of a group, as the product's columns, so
// that A is read once for 16 rows of an adapter. lds: shrink_lds floats for
// each wave. turn: what tells workgroups that run side by side apart.
template <int RT, int WAVES>
__device__ __forceinline__ void shrink_group(const LoraParams & p, const Rows rows, const int part_k, const int turn, float * lds) {
    constexpr int U = shrink_unroll<RT>(), kLds = shrink_lds<RT, U>();
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rank = __builtin_amdgcn_readfirstlane(rank_of(p, rows.a));
    const float scale = p.scales && rank > 0 ? p.scales[rows.a] : 1.0f;
    if (rank < 0 && threadIdx.x == 0) lora_error(p, rows.a);
    if (rank <= 0) return;
    const Columns c = Columns::of<U>(p, part_k, turn, wave, WAVES);
    const char * ar = p.a + (int64_t) rows.a * p.a_nb2;
    const char * xr = p.x + (int64_t) __shfl(rows.row, lane >> 2) * p.x_nb1;
    float * own = lds + wave * kLds;
    float4 x[U][2];
    load_x<U>(xr, c.column<U>(), c.k1, lane & 3, x);
    if (RT >= 8 && rank > 64)      shrink<min_c(RT, 8), U>(p, ar, rank, xr, x, c, lane, own);
    else if (RT >= 4 && rank > 32) shrink<min_c(RT, 4), U>(p, ar, rank, xr, x, c, lane, own);
    else if (RT >= 2 && rank > 16) shrink<min_c(RT, 2), U>(p, ar, rank, xr, x, c, lane, own);
    else                           shrink<1, U>(p, ar, rank, xr, x, c, lane, own);
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * RT * 16; i += 64 * WAVES) {
        const int tok = i / (RT * 16), j = i % (RT * 16);
        const int r = __shfl(rows.row, tok);
        if (j >= rank || tok >= rows.count) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += lds[w * kLds + j * (kTile + 1) + tok];
        p.v[((int64_t) part_k * p.T + r) * p.R + j] = v * scale;
    }
}

// The same with at most kFew rows: row `lead`'s group, if it is its first.
template <int RT, int WAVES>
__device__ __forceinline__ void shrink_few(const LoraParams & p, const int lead, const int part_k, float * lds) {
    Group<1> rows(p, 0, threadIdx.x & 63);
    if (rows.from_row(lead, threadIdx.x & 63) && rows.a >= 0) shrink_group<RT, WAVES>(p, rows, part_k, 0, lds);
}

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
    if (ranks >= 8) {
        const float4 x = ((const float4 *) v)[0], y = ((const float4 *) v)[1];
        const float z[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float) b[e], z[e], s);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(e < ranks ? (float) b[e] : 0.0f, e < ranks ? v[e] : 0.0f, s);
    }
    return s;
}

}  // namespace lora
