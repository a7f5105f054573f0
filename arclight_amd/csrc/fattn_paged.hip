// Attention of a batch's new tokens over a paged KV cache
// (include/arclight_paged.h), for gfx950.
//
// Mathematics. For a query row q and the cells c that it sees,
//   s_c = scale q . k_c,  m = max s_c,  p_c = e^(s_c - m),
//   o = sum p_c v_c / sum p_c,
// in one pass over the cells with a running m and sum (rows rescaled when m
// grows), and, where the cells of a sequence are split over workgroups, the
// parts (m, l, o) joined by the same rule: o = sum e^(m_i - M) o_i / sum
// e^(m_i - M) l_i.
//
// A wave takes 32 cells at a time, all in registers, no LDS. The scores are
// S^T = K Q^T and the output O^T = V^T P^T by mfma 16x16x32 with the query
// rows as columns, so that a row's maximum, sum and rescaling belong to the
// lanes of its column (lane 16 g + n: column n). The K rows of an MFMA are
// taken in the order 8 (i / 4) + i % 4 (+ 4 in the second), which leaves lane
// 16 g + n with the scores of cells 8 g .. 8 g + 7: the operand layout of the
// second product, so that P needs no exchange between lanes. For V^T lane
// 16 g + n loads dims 8 n .. 8 n + 7 of cells 8 g .. 8 g + 7 (256 contiguous
// bytes of a cell to a load's 16 lanes) and transposes the 8 x 8 block with 32
// byte permutes; the MFMA of dims 8 n + j then takes dword column j.
//
// Queries (scaled by a power of two to use the range) and probabilities
// (times 2^14) are each split into two f16, x = hi + lo to 2^-22, and both
// products run twice: the results are those of f32, and the matrix cores,
// idle most of the time in a kernel bound by the cells' bytes, have room for
// it.
//
// Work. The cells that a batch's sequences hold differ and are known on the
// device only. Every workgroup reads the lengths, cuts every sequence into
// chunks of at most C tiles with C such that the chunks of a (KV head, row
// group) are about as many as the workgroups that fit, and finds its own.
// Sequences of one chunk are written at once, the parts of the others are
// joined by a second launch.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/arclight_paged.h"
#include "device_common.hpp"
#include "kernel_args.hpp"
#include "paged.hpp"
#include "runtime.hpp"

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;                       // cells of a wave's step
constexpr int kMinTiles = 4;                    // least tiles of a chunk: one for each wave
constexpr float kPScale = 16384.0f;             // probabilities: 2^14 p stays normal in f16 down to p = 2^-28

struct PagedFattnParams {
    PagedPools c;
    const char * q;  int64_t q_nb1, q_nb2, q_nb3;       // token, head, sequence
    char * dst;      int64_t d_nb1, d_nb2, d_nb3;       // head, token, sequence
    const int32_t * lens;
    const int32_t * counts;                             // or null
    const float * sinks;                                // or null
    float * part;                                       // records: rows x 128 sums, then rows x {m, l}
    int32_t T, G, Hkv, R, row_groups;
    uint32_t g_magic;                                   // ceil(2^32 / G) (0 for 1)
    int32_t target;                                     // chunks aimed at for a (head, row group)
    int32_t max_chunks;                                 // grid size: chunks there can be
    float scale, softcap;
};

__device__ __forceinline__ int wave_sum_int(int x) {
#pragma unroll
    for (int o = 32; o >= 1; o /= 2) x += __shfl_xor(x, o);
    return x;
}

// What a row group of a sequence has to do.
struct SeqWork {
    int len, count, limit;                      // cells (within the table), new tokens, cells its last row sees
    bool bad;
};

__device__ __forceinline__ SeqWork seq_work(const PagedFattnParams & p, const int s, const int t0, const int t1) {
    SeqWork w;
    const int cap = p.c.max_pages * p.c.page_size;
    const int len = p.lens[s], count = p.counts ? p.counts[s] : p.T;
    w.len = min(max(len, 0), cap);
    w.count = min(max(count, 0), p.T);
    w.bad = len != w.len || count != w.count;
    w.limit = w.count > t0 ? min(max(w.len - w.count + 1 + min(t1, w.count - 1), 0), w.len) : -1;
    return w;
}

__device__ __forceinline__ int tiles_of(const SeqWork & w) { return w.limit > 0 ? (w.limit + kTile - 1) / kTile : 0; }
__device__ __forceinline__ int chunks_of(const SeqWork & w, const int C) {
    return w.limit < 0 ? 0 : max(1, (tiles_of(w) + C - 1) / C);
}

// Tiles of a chunk at most, the same in every wave of the launch's row group.
__device__ __forceinline__ int chunk_tiles(const PagedFattnParams & p, const int lane, const int t0, const int t1) {
    int sum = 0;
    for (int s = lane; s < p.c.n_seq; s += 64) sum += tiles_of(seq_work(p, s, t0, t1));
    sum = wave_sum_int(sum);
    const int c = (sum + p.target - 1) / p.target;
    return max(kMinTiles, (c + kWaves - 1) / kWaves * kWaves);
}

// The tokens of a row group.
__device__ __forceinline__ void group_tokens(const PagedFattnParams & p, const int r0, const int rows, int & t0, int & t1) {
    t0 = p.G == 1 ? r0 : (int) __umulhi((uint32_t) r0, p.g_magic);
    const int last = min(r0 + rows, p.R) - 1;
    t1 = p.G == 1 ? last : (int) __umulhi((uint32_t) last, p.g_magic);
}

__device__ __forceinline__ const char * record(const PagedFattnParams & p, const int unit, const int chunk, const int rows) {
    return (const char *) p.part + ((int64_t) unit * p.max_chunks + chunk) * rows * 130 * 4;
}

// NR: row tiles of 16 query rows. CAP: logits soft-capped.
template <int NR, bool CAP>
__global__ __launch_bounds__(64 * kWaves, NR == 1 ? 2 : 1) void paged_fattn_kernel(const PagedFattnParams p) {
    __shared__ __attribute__((aligned(16))) float o_lds[kWaves][16][132];
    __shared__ float ml_lds[NR][kWaves][16][2];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.y, h = unit % p.Hkv, r0 = unit / p.Hkv * (16 * NR);
    int t0, t1;
    group_tokens(p, r0, 16 * NR, t0, t1);

    // this workgroup's chunk
    const int C = chunk_tiles(p, lane, t0, t1);
    int seq = -1, chunk = 0, n_chunks = 0, before = 0;
    for (int s0 = 0; s0 < p.c.n_seq && seq < 0; s0 += 64) {
        const int s = s0 + lane;
        const int mine = s < p.c.n_seq ? chunks_of(seq_work(p, s, t0, t1), C) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int x = __shfl_up(upto, o);
            if (lane >= o) upto += x;
        }
        const int x = (int) blockIdx.x - before;
        const uint64_t hit = __ballot(x < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            seq = s0 + l;
            n_chunks = __builtin_amdgcn_readlane(mine, l);
            chunk = x - (__builtin_amdgcn_readlane(upto, l) - n_chunks);
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (seq < 0) return;
    seq = __builtin_amdgcn_readfirstlane(seq);
    const SeqWork w = seq_work(p, seq, t0, t1);
    bool bad = w.bad;
    if (bad && threadIdx.x == 0)
        paged_error(p.c, p.lens[seq] != w.len ? kPagedBadLength : kPagedBadCount, p.lens[seq] != w.len ? p.lens[seq] : p.counts[seq]);
    const int tiles = tiles_of(w);
    const int first = (int) ((int64_t) tiles * chunk / n_chunks), end = (int) ((int64_t) tiles * (chunk + 1) / n_chunks);

    // the query rows of this lane's columns: their limits, and their operands
    // times a power of two that brings the largest value to [2^11, 2^12)
    int limit[NR];
    float fac[NR], m[NR], l[NR];
    half8 q_hi[NR][4], q_lo[NR][4];
    floatx4 acc[NR][8];
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        const int r = r0 + 16 * u + n;
        const int t = p.G == 1 ? r : (int) __umulhi((uint32_t) r, p.g_magic);
        const bool valid = r < p.R && t < w.count;
        limit[u] = valid ? w.len - w.count + 1 + t : w.limit;
        float4 x[4][2];
        const char * qr = p.q + (int64_t) seq * p.q_nb3 + (int64_t) (valid ? t : 0) * p.q_nb1 +
                          (int64_t) (h * p.G + (valid ? r - t * p.G : 0)) * p.q_nb2 + 32 * g;
        float top = 0.0f;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                x[kk][e] = *(const float4 *) (qr + 128 * kk + 16 * e);
                if (!valid) x[kk][e] = float4{0.0f, 0.0f, 0.0f, 0.0f};
                top = fmaxf(fmaxf(fmaxf(top, fabsf(x[kk][e].x)), fmaxf(fabsf(x[kk][e].y), fabsf(x[kk][e].z))), fabsf(x[kk][e].w));
            }
        top = colmax4(top);
        // 2^(11 - exponent of top), within the normal range
        const int ex = min(max((int) (__float_as_uint(top) >> 23), 12), 253) - 127;
        const float up = __uint_as_float((uint32_t) (11 - ex + 127) << 23), down = __uint_as_float((uint32_t) (ex - 11 + 127) << 23);
        fac[u] = p.scale * down;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const float y[8] = {x[kk][0].x, x[kk][0].y, x[kk][0].z, x[kk][0].w, x[kk][1].x, x[kk][1].y, x[kk][1].z, x[kk][1].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float z = y[e] * up;
                const _Float16 hi = (_Float16) z;
                q_hi[u][kk][e] = hi;
                q_lo[u][kk][e] = (_Float16) (z - (float) hi);
            }
        }
        m[u] = -AL_INF;
        l[u] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[u][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int least = max(w.len - w.count + 1 + t0, 0);         // cells that every row of the group sees

    // Pages of a tile's cells: K by lanes n (group n / 4), V by lanes g. Cells
    // past the last group that anyone sees are taken from that group.
    struct Where {
        int k_page, v_page;
        int k_cell, v_cell;                                      // in the page
    };
    const int32_t * table = p.c.table + (int64_t) seq * p.c.t_nb1;
    const uint32_t last_group = (uint32_t) max(w.limit - 1, 0) / 8;
    auto look_up = [&](const int tile) {
        Where a;
        const uint32_t kg = min((uint32_t) tile * 4 + (n >> 2), last_group), vg = min((uint32_t) tile * 4 + g, last_group);
        const uint32_t kp = page_of_group(p.c, kg), vp = page_of_group(p.c, vg);
        a.k_page = table[kp];
        a.v_page = table[vp];
        a.k_cell = (int) (kg - kp * p.c.groups) * 8 + (n & 3);
        a.v_cell = (int) (vg - vp * p.c.groups) * 8;
        return a;
    };
    auto page = [&](const int x) {
        const bool ok = (uint32_t) x < (uint32_t) p.c.n_pages;
        bad |= !ok;
        return ok ? x : 0;
    };
    const char * k_head = p.c.k + (int64_t) h * p.c.k_nb2 + 16 * g;
    const char * v_head = p.c.v + (int64_t) h * p.c.v_nb2 + 16 * n;
    half8 k[2][4];
    u32x4 v[8];
    auto load_k = [&](const Where & a) {
        const char * b = k_head + page(a.k_page) * p.c.k_nb3 + a.k_cell * p.c.k_nb1;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) k[e][kk] = *(const half8 *) (b + 4 * e * p.c.k_nb1 + 64 * kk);
    };
    auto load_v = [&](const Where & a) {
        const char * b = v_head + page(a.v_page) * p.c.v_nb3 + a.v_cell * p.c.v_nb1;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *(const u32x4 *) (b + i * p.c.v_nb1);
    };
    // V^T operand of dims 8 n + j: this lane's 8 cells of dim j
    auto v_operand = [&](const int j) {
        u32x4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            a[i] = __builtin_amdgcn_perm(v[2 * i + 1][j / 2], v[2 * i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
        return as_half8(a);
    };

    floatx4 s[NR][2];
    auto scores = [&]() {
#pragma unroll
        for (int u = 0; u < NR; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[u][e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) s[u][e] = mfma_16x16x32(k[e][kk], q_lo[u][kk], s[u][e]);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) s[u][e] = mfma_16x16x32(k[e][kk], q_hi[u][kk], s[u][e]);
            }
    };
    half8 p_hi[NR], p_lo[NR];
    // Probabilities of the tile against the rows' running maxima.
    auto softmax = [&](const int tile) {
        const int c0 = tile * kTile + 8 * g;
        const bool masked = (tile + 1) * kTile > least;          // some row does not see all of it
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            float x[8];
            float top = -AL_INF;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = s[u][i / 4][i % 4] * fac[u];
                if constexpr (CAP) x[i] = p.softcap * tanhf(x[i] / p.softcap);
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 + i >= limit[u]) x[i] = -AL_INF;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
            if (__any(top > m[u])) {
                top = fmaxf(m[u], colmax4(top));
                const float r = top > m[u] ? exp_fast(m[u] - top) : 1.0f;
                m[u] = top;
                l[u] *= r;
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[u][j] *= r;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float e = exp_fast(x[i] - m[u]) * kPScale;
                if (masked && c0 + i >= limit[u]) e = 0.0f;
                l[u] += e;
                const _Float16 hi = (_Float16) e;
                p_hi[u][i] = hi;
                p_lo[u][i] = (_Float16) (e - (float) hi);
            }
        }
    };
    // o += P V of the tile. Cells past the sequence's last are stale memory:
    // zeroed, as 0 times NaN is not 0. So are, row by row, the cells that only
    // later tokens of the group see, where they hold no finite value.
    auto product = [&](const int tile) {
        if ((tile + 1) * kTile > least) {
            const int c0 = tile * kTile + 8 * g;
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c0 + i >= w.limit) v[i] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    odd |= c0 + i >= least && ((v[i][d] & 0x7c00u) == 0x7c00u || (v[i][d] & 0x7c000000u) == 0x7c000000u);
            }
            if (__any(odd)) {
                for (int t = t0; t <= t1; ++t) {
                    const int lim = w.len - w.count + 1 + t;
                    u32x4 keep[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        keep[i] = v[i];
                        if (c0 + i >= lim) v[i] = u32x4{0, 0, 0, 0};
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const half8 a = v_operand(j);
#pragma unroll
                        for (int u = 0; u < NR; ++u) {
                            const floatx4 x = mfma_16x16x32(a, p_hi[u], mfma_16x16x32(a, p_lo[u], acc[u][j]));
                            if (limit[u] == lim) acc[u][j] = x;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = keep[i];
                }
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const half8 a = v_operand(j);
#pragma unroll
            for (int u = 0; u < NR; ++u) acc[u][j] = mfma_16x16x32(a, p_hi[u], mfma_16x16x32(a, p_lo[u], acc[u][j]));
        }
    };

    // The wave's tiles, every kWaves-th of the chunk. The next tile's K is
    // loaded once this one's scores are done, its V once this one's product
    // is; pages are looked up a tile earlier. The last tile is a copy of its
    // own, so that no branch around the loads makes the compiler wait for all
    // of them.
    if (first + wave < end) {
        int tile = first + wave;
        Where next = look_up(tile);
        load_k(next);
        load_v(next);
        next = look_up(tile + kWaves);
        for (; tile + kWaves < end; tile += kWaves) {
            const Where after = look_up(tile + 2 * kWaves);
            scores();
            load_k(next);
            softmax(tile);
            product(tile);
            load_v(next);
            next = after;
        }
        scores();
        softmax(tile);
        product(tile);
    }

    // join the waves: maxima and sums, then the rescaled outputs through LDS
    const bool any_bad = __any(bad);
    if (any_bad && lane == 0 && !w.bad) paged_error(p.c, kPagedBadPage, seq);
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        l[u] = colsum4(l[u]);
        if (any_bad) l[u] = __builtin_nanf("");
        if (g == 0) {
            ml_lds[u][wave][n][0] = m[u];
            ml_lds[u][wave][n][1] = l[u];
        }
    }
    __syncthreads();
    const int row = threadIdx.x >> 4, dim = (threadIdx.x & 15) * 8;
    char * rec = const_cast<char *>(record(p, unit, blockIdx.x, 16 * NR));
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        float M = ml_lds[u][0][n][0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) M = fmaxf(M, ml_lds[u][i][n][0]);
        const float f = m[u] == M ? 1.0f : exp_fast(m[u] - M);
        if (u) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4 a = {acc[u][0][i] * f, acc[u][1][i] * f, acc[u][2][i] * f, acc[u][3][i] * f};
            float4 b = {acc[u][4][i] * f, acc[u][5][i] * f, acc[u][6][i] * f, acc[u][7][i] * f};
            *(float4 *) &o_lds[wave][n][8 * (4 * g + i)] = a;
            *(float4 *) &o_lds[wave][n][8 * (4 * g + i) + 4] = b;
        }
        __syncthreads();
        float Mr = ml_lds[u][0][row][0], L = 0.0f;
#pragma unroll
        for (int i = 1; i < kWaves; ++i) Mr = fmaxf(Mr, ml_lds[u][i][row][0]);
        float o[8] = {};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float mi = ml_lds[u][i][row][0];
            L += ml_lds[u][i][row][1] * (mi == Mr ? 1.0f : exp_fast(mi - Mr));
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d] += o_lds[i][row][dim + d];
        }
        const int r = r0 + 16 * u + row;
        const int t = p.G == 1 ? r : (int) __umulhi((uint32_t) r, p.g_magic);
        if (r >= p.R || t >= w.count) continue;
        if (n_chunks > 1) {
            float * d = (float *) rec + (16 * u + row) * 128 + dim;
            *(float4 *) d = float4{o[0], o[1], o[2], o[3]};
            *(float4 *) (d + 4) = float4{o[4], o[5], o[6], o[7]};
            if (dim == 0) *(float2 *) ((float *) rec + 16 * NR * 128 + (16 * u + row) * 2) = float2{Mr, L};
            continue;
        }
        const int head = h * p.G + r - t * p.G;
        // the sink as one more logit, without a value
        L *= 1.0f / kPScale;
        float up = 1.0f / kPScale;
        if (p.sinks) {
            const float sink = p.sinks[head], top = fmaxf(Mr, sink);
            const float e = Mr == top ? 1.0f : exp_fast(Mr - top);
            up *= e;
            L = L * e + (sink == top ? 1.0f : exp_fast(sink - top));
        }
        const float inv = L == 0.0f ? 0.0f : up / L;
        float * d = (float *) (p.dst + (int64_t) seq * p.d_nb3 + (int64_t) t * p.d_nb2 + (int64_t) head * p.d_nb1) + dim;
        *(float4 *) d = float4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        *(float4 *) (d + 4) = float4{o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv};
    }
}

// Joins the chunks' parts: a workgroup per sequence and unit, a wave per row,
// two dims to a lane.
template <int NR>
__global__ __launch_bounds__(64 * kWaves) void paged_join_kernel(const PagedFattnParams p) {
    prefetch_params(p);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int seq = blockIdx.x, unit = blockIdx.y, h = unit % p.Hkv, r0 = unit / p.Hkv * (16 * NR);
    int t0, t1;
    group_tokens(p, r0, 16 * NR, t0, t1);
    const int C = chunk_tiles(p, lane, t0, t1);
    const SeqWork w = seq_work(p, seq, t0, t1);
    const int n_chunks = chunks_of(w, C);
    if (n_chunks < 2) return;
    int before = 0;
    for (int s = lane; s < seq; s += 64) before += chunks_of(seq_work(p, s, t0, t1), C);
    before = wave_sum_int(before);
    for (int row = wave; row < 16 * NR; row += kWaves) {
        const int r = r0 + row;
        const int t = p.G == 1 ? r : (int) __umulhi((uint32_t) r, p.g_magic);
        if (r >= p.R || t >= w.count) break;
        const char * rec = record(p, unit, before, 16 * NR);
        const int64_t step = 16 * NR * 130 * 4;
        float M = -AL_INF;
        for (int i = lane; i < n_chunks; i += 64) M = fmaxf(M, *(const float *) (rec + i * step + (16 * NR * 128 + row * 2) * 4));
#pragma unroll
        for (int o = 32; o >= 1; o /= 2) M = fmaxf(M, __shfl_xor(M, o));
        float L = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll 8
        for (int i = 0; i < n_chunks; ++i) {
            const float2 ml = *(const float2 *) (rec + i * step + (16 * NR * 128 + row * 2) * 4);
            const float2 o = *(const float2 *) (rec + i * step + (row * 128 + 2 * lane) * 4);
            const float e = ml.x == M ? 1.0f : exp_fast(ml.x - M);
            L += ml.y * e;
            x += o.x * e;
            y += o.y * e;
        }
        const int head = h * p.G + r - t * p.G;
        L *= 1.0f / kPScale;
        float up = 1.0f / kPScale;
        if (p.sinks) {
            const float sink = p.sinks[head], top = fmaxf(M, sink);
            const float e = M == top ? 1.0f : exp_fast(M - top);
            up *= e;
            L = L * e + (sink == top ? 1.0f : exp_fast(sink - top));
        }
        const float inv = L == 0.0f ? 0.0f : up / L;
        *(float2 *) ((float *) (p.dst + (int64_t) seq * p.d_nb3 + (int64_t) t * p.d_nb2 + (int64_t) head * p.d_nb1) + 2 * lane) =
            float2{x * inv, y * inv};
    }
}

struct Plan {
    PagedFattnParams p;
    int nr = 1;
    bool empty = false;
    size_t bytes = 0;                                   // records
};

bool aligned16(const al_tensor & t, int from) {
    for (int i = from; i < 4; ++i)
        if (t.ne[i] > 1 && t.nb[i] % 16) return false;
    return ((uintptr_t) t.data & 15u) == 0;
}

int make_plan(const al_paged_fattn_args * a, int n_cu, Plan * out) {
    if (!a) return al_fail(AL_ERR_INVALID, "paged_fattn: null arguments");
    const al_tensor &q = a->q, &d = a->dst;
    if (!q.data || !d.data || !a->lens.data) return al_fail(AL_ERR_INVALID, "paged_fattn: q, dst and lens are required");
    if (q.type != AL_TYPE_F32 || d.type != AL_TYPE_F32)
        return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: q / dst types %d / %d (f32 only)", q.type, d.type);
    const int64_t T = q.ne[1], Hq = q.ne[2], n_seq = q.ne[3];
    if (q.ne[0] != 128) return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: head dim %lld (128 only)", (long long) q.ne[0]);
    if (T < 0 || Hq < 1 || n_seq < 0 || d.ne[0] != 128 || d.ne[1] != Hq || d.ne[2] != T || d.ne[3] != n_seq)
        return al_fail(AL_ERR_INVALID, "paged_fattn: dst must be [128, Hq, T, n_seq] for q [128, T, Hq, n_seq]");
    if (q.nb[0] != 4 || d.nb[0] != 4 || !aligned16(q, 1) || !aligned16(d, 1))
        return al_fail(AL_ERR_INVALID, "paged_fattn: q and dst rows must be contiguous and 16-byte aligned");
    Plan pl;
    PagedFattnParams & p = pl.p;
    memset(&p, 0, sizeof(p));
    int rc = paged_pools("paged_fattn", &a->k_pool, &a->v_pool, &a->table, &p.c);
    if (rc != AL_OK) return rc;
    const int64_t Hkv = a->k_pool.ne[2];
    if (Hq % Hkv != 0) return al_fail(AL_ERR_INVALID, "paged_fattn: %lld query heads over %lld KV heads", (long long) Hq, (long long) Hkv);
    if (p.c.n_seq != n_seq) return al_fail(AL_ERR_INVALID, "paged_fattn: the table has %d sequences, q %lld", p.c.n_seq, (long long) n_seq);
    auto index = [&](const al_tensor & t) { return t.type == AL_TYPE_I32 && t.ne[0] == n_seq && t.nb[0] == 4 && ((uintptr_t) t.data & 3u) == 0; };
    if (!index(a->lens) || (a->counts.data && !index(a->counts)))
        return al_fail(AL_ERR_INVALID, "paged_fattn: lens and counts must be i32 [n_seq]");
    if (a->sinks.data && (a->sinks.type != AL_TYPE_F32 || a->sinks.ne[0] != Hq || a->sinks.nb[0] != 4))
        return al_fail(AL_ERR_INVALID, "paged_fattn: sinks must be f32 [Hq]");
    if (!(a->logit_softcap >= 0.0f)) return al_fail(AL_ERR_INVALID, "paged_fattn: softcap %g", (double) a->logit_softcap);
    if (T > (1 << 16) || Hq > (1 << 12) || T * Hq > (1 << 22) || n_seq > (1 << 16))
        return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: sizes out of range");
    pl.empty = T == 0 || n_seq == 0;
    p.q = (const char *) q.data; p.q_nb1 = q.nb[1]; p.q_nb2 = q.nb[2]; p.q_nb3 = q.nb[3];
    p.dst = (char *) d.data; p.d_nb1 = d.nb[1]; p.d_nb2 = d.nb[2]; p.d_nb3 = d.nb[3];
    p.lens = (const int32_t *) a->lens.data;
    p.counts = (const int32_t *) a->counts.data;
    p.sinks = (const float *) a->sinks.data;
    p.T = (int32_t) T; p.G = (int32_t) (Hq / Hkv); p.Hkv = (int32_t) Hkv;
    p.R = p.T * p.G;
    p.g_magic = p.G > 1 ? (uint32_t) (((1ull << 32) + (uint64_t) p.G - 1) / (uint64_t) p.G) : 0u;
    pl.nr = p.R <= 16 ? 1 : 2;
    const int rows = 16 * pl.nr;
    p.row_groups = (p.R + rows - 1) / rows;
    const int64_t units = (int64_t) p.row_groups * Hkv;
    if (units > 65535) return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: sizes out of range");
    p.target = (int32_t) std::max<int64_t>(1, (pl.nr == 1 ? 2 : 1) * (int64_t) n_cu / std::max<int64_t>(1, units));
    const int64_t most = ((int64_t) p.c.max_pages * p.c.page_size + kTile * kMinTiles - 1) / (kTile * kMinTiles);   // chunks of a sequence
    p.max_chunks = (int32_t) std::min<int64_t>(p.target + n_seq, n_seq * std::max<int64_t>(1, most));
    p.scale = a->scale;
    p.softcap = a->logit_softcap;
    pl.bytes = (size_t) units * p.max_chunks * rows * 130 * 4;
    *out = pl;
    return AL_OK;
}

template <int NR>
hipError_t launch(const PagedFattnParams & p, hipStream_t st) {
    const dim3 grid((unsigned) p.max_chunks, (unsigned) (p.row_groups * p.Hkv));
    if (p.softcap != 0.0f) hipLaunchKernelGGL((paged_fattn_kernel<NR, true>), grid, dim3(64 * kWaves), 0, st, p);
    else                   hipLaunchKernelGGL((paged_fattn_kernel<NR, false>), grid, dim3(64 * kWaves), 0, st, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_join_kernel<NR>), dim3((unsigned) p.c.n_seq, (unsigned) (p.row_groups * p.Hkv)), dim3(64 * kWaves), 0, st, p);
    return hipGetLastError();
}

}  // namespace

int paged_pools(const char * what, const al_tensor * k, const al_tensor * v, const al_tensor * table, PagedPools * out) {
    if (!k->data || !v->data || !table->data) return al_fail(AL_ERR_INVALID, "%s: the pools and the table are required", what);
    if (k->type != AL_TYPE_F16 || v->type != AL_TYPE_F16)
        return al_fail(AL_ERR_UNSUPPORTED, "%s: pool types %d / %d (f16 only)", what, k->type, v->type);
    if (k->ne[0] != 128 || v->ne[0] != 128) return al_fail(AL_ERR_UNSUPPORTED, "%s: head dim %lld / %lld (128 only)", what, (long long) k->ne[0], (long long) v->ne[0]);
    for (int i = 1; i < 4; ++i)
        if (k->ne[i] != v->ne[i] || k->ne[i] < 1) return al_fail(AL_ERR_INVALID, "%s: k and v pools must both be [128, P, Hkv, n_pages]", what);
    if (k->nb[0] != 2 || v->nb[0] != 2 || !aligned16(*k, 1) || !aligned16(*v, 1))
        return al_fail(AL_ERR_INVALID, "%s: pool rows must be contiguous and 16-byte aligned", what);
    if (table->type != AL_TYPE_I32 || table->nb[0] != 4 || table->nb[1] % 4 || ((uintptr_t) table->data & 3u) ||
        table->ne[0] < 1 || table->ne[1] < 0 || table->ne[2] != 1 || table->ne[3] != 1)
        return al_fail(AL_ERR_INVALID, "%s: the table must be i32 [max_pages, n_seq]", what);
    const int64_t P = k->ne[1];
    if (P % 8) return al_fail(AL_ERR_UNSUPPORTED, "%s: pages of %lld cells (multiples of 8)", what, (long long) P);
    if (k->ne[3] > INT32_MAX || table->ne[0] > (1 << 26) || table->ne[1] > (1 << 24) || P > (1 << 20) || k->ne[2] > (1 << 12) ||
        table->ne[0] * P > (1 << 30) || (double) table->ne[0] * (double) P * (double) P >= 64.0 * 4294967296.0)
        return al_fail(AL_ERR_UNSUPPORTED, "%s: sizes out of range", what);
    PagedPools p;
    p.k = (char *) k->data; p.k_nb1 = k->nb[1]; p.k_nb2 = k->nb[2]; p.k_nb3 = k->nb[3];
    p.v = (char *) v->data; p.v_nb1 = v->nb[1]; p.v_nb2 = v->nb[2]; p.v_nb3 = v->nb[3];
    p.table = (const int32_t *) table->data; p.t_nb1 = (int64_t) (table->nb[1] / 4);
    p.n_seq = (int32_t) table->ne[1]; p.n_pages = (int32_t) k->ne[3]; p.max_pages = (int32_t) table->ne[0];
    p.page_size = (int32_t) P;
    p.groups = (int32_t) (P / 8);
    p.magic = p.groups > 1 ? (uint32_t) (((1ull << 32) + (uint64_t) p.groups - 1) / (uint64_t) p.groups) : 0u;
    p.err = nullptr;
    *out = p;
    return AL_OK;
}

extern "C" uint64_t al_paged_fattn_workspace_bytes(const al_paged_fattn_args * a) {
    int n_cu = 0;
    Plan pl;
    if (al_device_cu_count(&n_cu) != AL_OK || make_plan(a, n_cu, &pl) != AL_OK) return 0;
    return pl.empty ? 0 : pl.bytes;
}

extern "C" int al_paged_fattn_f16(const al_paged_fattn_args * a) {
    // the arguments first: refusals need no device
    Plan pl;
    int rc = make_plan(a, 1, &pl);
    if (rc != AL_OK || pl.empty) return rc;
    int n_cu = 0;
    rc = al_device_cu_count(&n_cu);
    if (rc == AL_OK) rc = make_plan(a, n_cu, &pl);
    if (rc == AL_OK) rc = al_device_error_flag(&pl.p.c.err);
    if (rc != AL_OK) return rc;
    if (a->workspace) {
        if (a->workspace_bytes < pl.bytes || ((uintptr_t) a->workspace & 15u))
            return al_fail(AL_ERR_WORKSPACE, "paged_fattn: workspace %llu bytes (16-byte aligned) < %zu needed",
                           (unsigned long long) a->workspace_bytes, pl.bytes);
        pl.p.part = (float *) a->workspace;
    } else {
        rc = al_library_workspace(pl.bytes, a->stream, (void **) &pl.p.part);
        if (rc != AL_OK) return rc;
    }
    const hipError_t e = pl.nr == 1 ? launch<1>(pl.p, (hipStream_t) a->stream) : launch<2>(pl.p, (hipStream_t) a->stream);
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "paged_fattn: launch");
}
