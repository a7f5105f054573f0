// Attention over a paged KV cache of many query rows that see a window or a
// tree (include/arclight_paged.h), for gfx950: prompts in layers with a window,
// trees of dozens of drafted tokens.
//
// Mathematics, sharing out of the work and records as fattn_paged.hip, which
// takes fewer rows. There every wave loads a tile's cells itself; here the tile
// is in LDS, and a workgroup's four waves take 32 query rows each over it, so
// that a byte of it feeds 128 rows.
//
// Per wave and tile of 64 cells, by mfma 32x32x16:
//   S^T [64 cells x 32 rows]  = K Q^T     2 x 16 products
//   O^T [128 dims x 32 rows] += V^T P^T   2 x 16 products
// Each twice, as queries and probabilities are pairs of f16, x = hi + lo, which
// gives the results of f32. A score register of lane 32 h + n holds row n and cell
// v % 4 + 8 (v / 4) + 4 h of a block of 32 (v: the register): with the k slots of
// a product taken in that order the probabilities are the operand of the second
// product in place, and V's operand of that order comes from LDS by transposing
// reads (ds_read_b64_tr_b16).
//
// Softmax in log2 units: p = 2^(s f - m) by one fma and one exponential, m a
// reference 8 below the row's maximum when it was last moved, which it is when
// a score is 14 above it: then 2^14 is the largest p, and what lies 2^33 below the
// maximum is still carried.
//
// Tiles go from memory into LDS directly (buffer_load ... lds), one tile ahead,
// each wave a quarter, its pages looked up another tile ahead by scalar loads.
// A tile is [cell][128] with 16-byte pieces permuted within a cell so that the
// operand reads are free of bank conflicts: piece j of K's cell c at j ^ (c &
// 15), of V's at j ^ 4 (c & 3). Two workgroups to a CU: while one waits for its
// scores' exponentials the other has the matrix cores.
//
// Tiles that some row does not see all of are masked value by value; V of cells
// that no row sees is cleared there (0 times NaN is not 0), and so are single
// values that are not finite: the rows that do see them get NaN in their dim,
// found by a product of ones.

#include <hip/hip_runtime.h>

#include "fattn_paged.hpp"
#include "fattn_prefill_common.hpp"

namespace paged_fattn {

namespace {

using fattn::dma16;
using fattn::half4;
using fattn::int4v;
using fattn::lds_addr;
using fattn::lds_read_tr16;
using fattn_prefill::floatx16;
using fattn_prefill::mfma32;
using fattn_prefill::pair_max;
using fattn_prefill::pair_sum;
using fattn_prefill::wait_vm;

constexpr int kTileBytes = PagedRowsParams::kTile * 256;
constexpr float kBelow = 8.0f, kOutgrown = 14.0f;        // log2: the reference below the maximum, a score that moves it

// The first k of 64 cells, a bit each.
__device__ __forceinline__ uint64_t upto64(const int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; }
// span8 and nodes8 of 64 cells
__device__ __forceinline__ uint64_t span64(const int c0, const int limit, const int low, const int first) {
    return upto64(limit - c0) & (~upto64(low - c0) | upto64(first - c0));
}
__device__ __forceinline__ uint64_t nodes64(const PagedSeesParams & p, const int32_t * words, const int32_t * pos, const int u0, const int count,
                                            const int low) {
    if (u0 <= -64 || u0 >= count) return 0;
    const int u = max(u0, 0), i = u >> 5, last = (count - 1) >> 5, sh = u & 31;
    const uint64_t two = (uint32_t) words[i] | (uint64_t) (uint32_t) words[min(i + 1, last)] << 32;
    const uint64_t third = (uint32_t) words[min(i + 2, last)];
    uint64_t m = (sh ? two >> sh | third << (64 - sh) : two) << (u - u0) & upto64(count - u0);
    // (positions of nodes are within a window that is as long as the tree)
    if (p.window && p.window < count)
        for (uint64_t rest = m; rest; rest &= rest - 1) {
            const int at = pos[u0 + __builtin_ctzll(rest)];
            if (at < low && at >= p.first) m &= ~(rest & -rest);
        }
    return m;
}

// A descriptor of `bytes` from memory that the wave addresses alike in every lane.
__device__ __forceinline__ int4v uniform_desc(const char * base, const uint32_t bytes) {
    const uint64_t a = (uint64_t) base;
    return int4v{__builtin_amdgcn_readfirstlane((int) (uint32_t) a), __builtin_amdgcn_readfirstlane((int) (uint32_t) (a >> 32)),
                 __builtin_amdgcn_readfirstlane((int) bytes), 0x00020000};
}

// CAP: logits soft-capped.
template <bool CAP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_rows_kernel(const PagedRowsParams p) {
    using P = PagedRowsParams;
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];  // K and V of two tiles
    __shared__ uint64_t odd[128];                   // of each dim, the tile's cells whose value is not finite
    __shared__ int any_odd, any_bad;
    prefetch_params(p);
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, lr = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the heads of the same cells next to one another in the grid
    const int units = p.row_groups * p.Hkv, unit = blockIdx.x % units, wg = blockIdx.x / units;
    const int head = unit % p.Hkv, group0 = unit / p.Hkv * P::kRows;
    // tokens of the group, and of the wave's rows (none past the last row)
    const int t0 = token_of(p, group0), t1 = token_of(p, min(group0 + P::kRows, p.R) - 1);
    const int r0 = group0 + 32 * wave;
    const int wt0 = token_of(p, min(r0, p.R - 1)), wt1 = token_of(p, min(r0 + 32, p.R) - 1);

    const int n_blocks = (p.c.n_seq + 63) / 64;
    Block b;
    MyPart part;
    if (!find_part(p, wg, lane, t0, t1, blockIdx.x == 0 && wave == 0, b, part)) return;
    int at = part.at, block = 0, before = 0;
    const int stop = part.stop;
    if (tid < 128) odd[tid] = 0;
    if (tid == 0) any_odd = any_bad = 0;

    const uint32_t k_nb1 = (uint32_t) p.c.k_nb1, v_nb1 = (uint32_t) p.c.v_nb1, lds0 = lds_addr(lds);
    // this lane's offset within 4 cells of K (their place among 16 cells) and of V
    uint32_t k_lane[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) k_lane[q] = (uint32_t) (lane >> 4) * k_nb1 + (uint32_t) (((lane & 15) ^ (4 * q + (lane >> 4))) * 16);
    const uint32_t v_lane = (uint32_t) (lane >> 4) * v_nb1 + (uint32_t) (((lane & 15) ^ (4 * (lane >> 4))) * 16);
    const char * k_head = p.c.k + (int64_t) head * p.c.k_nb2;
    const char * v_head = p.c.v + (int64_t) head * p.c.v_nb2;
    // operand reads: K of cell lr, V as 4 x 16 pieces
    const int k_at = lr * 256 + ((h ^ (lr & 15)) << 4);
    const int s16 = lane & 15, v_sw = s16 >> 2;
    const int v_at = (4 * h + v_sw) * 256 + ((2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1)) << 4) + (s16 & 1) * 8;

    while (at < stop) {
        // the sequence that holds tile `at`
        while (at >= before + b.total()) {
            before += b.total();
            if (++block >= n_blocks) return;                         // (lengths that change meanwhile: not without an end)
            b.load(p, block, lane, t0, t1);
        }
        const int l64 = __builtin_ctzll(__ballot(at < before + b.upto));
        const int seq = 64 * block + l64;
        const int tiles = __builtin_amdgcn_readlane(b.tiles, l64);
        const int base = before + __builtin_amdgcn_readlane(b.upto, l64) - tiles;
        const int raw_len = __builtin_amdgcn_readlane(b.len, l64), raw_count = __builtin_amdgcn_readlane(b.count, l64);
        const SeqWork w = seq_work(p, raw_len, raw_count);
        const int first = at - base, end = min(tiles, stop - base);
        at = base + end;
        const bool whole = first == 0 && end == tiles;
        if (tid == 0) {
            if (first == 0) p.info[(int64_t) unit * p.c.n_seq + seq] = int2{wg, whole ? 1 : part.parts.of(base + tiles - 1) - wg + 1};
            if (w.bad) paged_error(p.c, raw_len != w.len ? kPagedBadLength : kPagedBadCount, raw_len != w.len ? raw_len : raw_count);
        }
        const int begin = w.len - w.count;
        // what the group sees, what the wave sees, what all of the group's or the wave's rows see
        const Span group = span_of(p, w, t0, t1), mine = span_of(p, w, wt0, wt1);
        const int gap = group.gap(p), gap_at = group.gap_at(p);
        auto tile_at = [&](const int i) { return i >= gap_at ? i + gap : i; };
        auto least_of = [&](const int first_token) { return p.bits ? max(begin, 0) : max(begin + 1 + first_token, 0); };
        auto low_of = [&](const int last_token) {
            return p.window ? (p.bits ? w.len : begin + 1 + min(last_token, w.count - 1)) - p.window : 0;
        };
        auto partly = [&](const int tile, const int least, const int low) {
            return (tile + 1) * P::kTile > least || (tile * P::kTile < low && (tile + 1) * P::kTile > p.first);
        };
        const int least = least_of(t0), low_last = low_of(t1), my_least = least_of(wt0), my_low_last = low_of(wt1);
        const int tiles_end = group.limit > 0 ? end : first;             // (nothing is seen: no tile)

        // Pages of this wave's 16 cells of a tile, two groups of 8, those past
        // the last that the group sees taken from that one, those before the
        // first window from its.
        struct Where {
            int page[2], cell[2];
        };
        const int32_t * table = p.c.table + (int64_t) seq * p.c.t_nb1;
        const int last_group = max(group.limit - 1, 0) / 8, from = (p.first + 7) >> 3, low_group = group.low >> 3;
        bool bad = false;
        auto look_up = [&](const int i) {
            Where a;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                int g = min(tile_at(i) * 8 + 2 * wave + e, last_group);
                if (g >= from) g = max(g, low_group);
                const int pg = (int) page_of_group(p.c, (uint32_t) g);
                a.page[e] = ld_uniform(table + pg);
                a.cell[e] = (g - pg * p.c.groups) * 8;
            }
            return a;
        };
        auto load = [&](const Where & a, const int buf) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool ok = (uint32_t) a.page[e] < (uint32_t) p.c.n_pages;
                bad |= !ok;
                const int pg = ok ? a.page[e] : 0;
                const char * k = k_head + pg * p.c.k_nb3 + a.cell[e] * p.c.k_nb1;
                const char * v = v_head + pg * p.c.v_nb3 + a.cell[e] * p.c.v_nb1;
                const uint32_t to = lds0 + (uint32_t) (buf * 2 * kTileBytes + (16 * wave + 8 * e) * 256);
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    dma16(uniform_desc(k + 4 * f * p.c.k_nb1, 3 * k_nb1 + 256), k_lane[2 * e + f], to + 1024 * f);
                    dma16(uniform_desc(v + 4 * f * p.c.v_nb1, 3 * v_nb1 + 256), v_lane, to + kTileBytes + 1024 * f);
                }
            }
        };
        Where next;
        if (first < tiles_end) {
            load(look_up(first), 0);
            next = look_up(min(first + 1, tiles_end - 1));
        }

        // This lane's query row: its operands times a power of two that brings
        // the largest value to [2^11, 2^12), the scores' factor, what it sees
        const int r = r0 + lr, t = token_of(p, min(r, p.R - 1));
        const bool valid = r < p.R && t < w.count;
        half8 q_hi[8], q_lo[8];
        float fac;
        {
            const float * qr = (const float *) (p.q + (int64_t) seq * p.q_nb3 + (int64_t) (valid ? t : 0) * p.q_nb1 +
                                                (int64_t) (head * p.G + (valid ? r - t * p.G : 0)) * p.q_nb2) + 8 * h;
            float4 x[8][2];
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[ks][e] = *(const float4 *) (qr + 16 * ks + 4 * e);
            float top = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (!valid) x[ks][e] = float4{0.0f, 0.0f, 0.0f, 0.0f};
                    top = fmaxf(fmaxf(fmaxf(top, fabsf(x[ks][e].x)), fmaxf(fabsf(x[ks][e].y), fabsf(x[ks][e].z))), fabsf(x[ks][e].w));
                }
            top = pair_max(top);
            // 2^(11 - exponent of top), within the normal range; the scale's
            // sign goes with the queries, so that the factor is positive
            const int ex = min(max((int) (__float_as_uint(top) >> 23), 12), 253) - 127;
            float up = __uint_as_float((uint32_t) (11 - ex + 127) << 23);
            const float down = __uint_as_float((uint32_t) (ex - 11 + 127) << 23);
            if (p.scale < 0.0f) up = -up;
            fac = fabsf(p.scale) * down;
            fac = CAP ? fac / p.softcap : fac * kLog2e;
            // (a factor of 0 would make NaN of the -inf of hidden cells)
            if (!CAP) fac = fmaxf(fac, 1.17549435e-38f);
            if (p.scale == 0.0f) up = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const float y[8] = {x[ks][0].x, x[ks][0].y, x[ks][0].z, x[ks][0].w, x[ks][1].x, x[ks][1].y, x[ks][1].z, x[ks][1].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = y[e] * up;
                    const _Float16 hi = (_Float16) z;
                    q_hi[ks][e] = hi;
                    q_lo[ks][e] = (_Float16) (z - (float) hi);
                }
            }
        }
        const int limit = valid ? begin + 1 + t : group.limit;
        int low = 0;
        const int32_t * words = nullptr;
        const int32_t * node_pos = nullptr;
        bool bad_row = false;
        {
            int place = begin + t;
            if (p.bits) {
                words = p.bits + (int64_t) seq * p.b_nb2 + (int64_t) (valid ? t : 0) * p.b_nb1;
                node_pos = p.pos + (int64_t) seq * p.p_nb1;
                if (p.window && valid) {
                    place = node_pos[t];
                    bad_row = place < begin || place >= w.len;
                    if (bad_row && h == 0) paged_error(p.c, kPagedBadPos, place);
                }
            }
            if (p.window && valid && !bad_row) low = place + 1 - p.window;
        }
        // Of the 64 cells from c0 on: those that this lane's row sees.
        auto sees64 = [&](const int c0) {
            if (p.bits) return span64(c0, begin, low, p.first) | nodes64(p, words, node_pos, c0 - begin, w.count, low);
            return span64(c0, limit, low, p.first);
        };

        floatx16 o[4];
#pragma unroll
        for (int db = 0; db < 4; ++db) o[db] = floatx16{};
        float m = -AL_INF, l = 0.0f;
        const bool has_rows = r0 < p.R && wt0 < w.count;
        for (int i = first; i < tiles_end; ++i) {
            const int buf = (i - first) & 1, tile = tile_at(i), c0 = tile * P::kTile;
            wait_vm<0>();
            __syncthreads();                                             // the tile is there, the other buffer free
            if (i + 1 < tiles_end) {
                load(next, buf ^ 1);
                next = look_up(min(i + 2, tiles_end - 1));
            }
            const char * k_tile = lds + buf * 2 * kTileBytes;
            char * v_tile = lds + buf * 2 * kTileBytes + kTileBytes;
            const bool edge = partly(tile, least, low_last);             // some row of the group does not see all of it
            if (edge) {
                const uint64_t some = span64(c0, group.limit, group.low, p.first), all = span64(c0, least, low_last, p.first);
                const int c = tid >> 2;
                if (!(all >> c & 1)) {
                    const bool none = !(some >> c & 1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int slot = (tid & 3) * 4 + e, j = slot ^ (4 * (c & 3));
                        u32x4 * x = (u32x4 *) (v_tile + c * 256 + slot * 16);
                        u32x4 y = *x;
                        bool change = none;
                        if (none) y = u32x4{0, 0, 0, 0};
                        else
#pragma unroll
                            for (int d = 0; d < 4; ++d)
#pragma unroll
                                for (int half = 0; half < 2; ++half)
                                    if ((y[d] >> (16 * half) & 0x7c00u) == 0x7c00u) {
                                        y[d] &= half ? 0xffffu : 0xffff0000u;
                                        atomicOr((unsigned long long *) &odd[8 * j + 2 * d + half], 1ull << c);
                                        any_odd = 1;
                                        change = true;
                                    }
                        if (change) *x = y;
                    }
                }
                __syncthreads();
            }
            const bool work = has_rows && c0 < mine.limit && !(c0 >= p.first && c0 + P::kTile <= mine.low);
            if (work) {
                floatx16 s[2] = {floatx16{}, floatx16{}};
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    half8 k[2];
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) k[cb] = as_half8(*(const u32x4 *) (k_tile + 32 * 256 * cb + (k_at ^ (ks << 5))));
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) s[cb] = mfma32(k[cb], q_lo[ks], s[cb]);
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) s[cb] = mfma32(k[cb], q_hi[ks], s[cb]);
                }
                float f = fac;
                if constexpr (CAP) {
                    f = p.softcap * kLog2e;
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                        for (int v = 0; v < 16; ++v) s[cb][v] = tanhf(s[cb][v] * fac);
                }
                if (partly(tile, my_least, my_low_last)) {
                    uint64_t sees = valid ? sees64(c0) : ~0ull;
                    sees >>= 4 * h;
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (!((uint32_t) (sees >> (32 * cb)) >> (8 * (v >> 2) + (v & 3)) & 1)) s[cb][v] = -AL_INF;
                }
                float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
                for (int v = 1; v < 16; ++v) top = fmaxf(fmaxf(top, s[0][v]), s[1][v]);
                if (__any(top * f > m + kOutgrown)) {
                    top = pair_max(top) * f;
                    const float to = top > m + kOutgrown ? top - kBelow : m;
                    const float g = grow<P>(m, to);
                    m = to;
                    l *= g;
#pragma unroll
                    for (int db = 0; db < 4; ++db) o[db] *= g;
                }
                const float ref = m == -AL_INF ? 0.0f : m;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    half8 p_hi, p_lo;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][8 * (kk & 1) + e], f, -ref));
                        sum[e & 3] += x;
                        const _Float16 hi = (_Float16) x;
                        p_hi[e] = hi;
                        p_lo[e] = (_Float16) (x - (float) hi);
                    }
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
                        const char * x = v_tile + ((v_at ^ (64 * v_sw)) ^ (64 * db)) + 16 * 256 * kk;
                        const half4 a = lds_read_tr16(x), c = lds_read_tr16(x + 8 * 256);
                        const half8 v = {a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
                        o[db] = mfma32(v, p_lo, o[db]);
                        o[db] = mfma32(v, p_hi, o[db]);
                    }
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            if (edge && any_odd) {                                       // (written before the barrier above)
                if (work) {
                    const uint64_t sees = (valid ? sees64(c0) : 0ull) >> (4 * h);
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
                        const uint64_t mask = odd[32 * db + lr] >> (4 * h);
                        floatx16 x = {};
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            half8 a, c;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int bit = 16 * kk + (e & 3) + 8 * (e >> 2);
                                a[e] = mask >> bit & 1 ? (_Float16) 1.0f : (_Float16) 0.0f;
                                c[e] = sees >> bit & 1 ? (_Float16) 1.0f : (_Float16) 0.0f;
                            }
                            x = mfma32(a, c, x);
                        }
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (x[v] > 0.0f) o[db][v] = __builtin_nanf("");
                    }
                }
                __syncthreads();
                if (tid < 128) odd[tid] = 0;
                if (tid == 0) any_odd = 0;                               // (used next behind the next tile's barrier)
            }
        }

        if (bad && lane == 0) {
            any_bad = 1;
            if (!w.bad) paged_error(p.c, kPagedBadPage, seq);
        }
        __syncthreads();
        l = pair_sum(l);
        if (any_bad || w.bad || bad_row) l = __builtin_nanf("");
        if (valid) {
            float f = 1.0f;
            float * d;
            if (whole) {
                const int hq = head * p.G + r - t * p.G;
                f = row_factor(p, p, w, seq, t, m, l, hq);
                d = (float *) (p.dst + (int64_t) seq * p.d_nb3 + (int64_t) t * p.d_nb2 + (int64_t) hq * p.d_nb1);
            } else {
                float * rec = (float *) record(p, unit, wg, first == 0 ? 1 : 0);
                d = rec + (r - group0) * 128;
                if (h == 0) *(float2 *) (rec + P::kRows * 128 + (r - group0) * 2) = float2{m, l};
            }
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int bq = 0; bq < 4; ++bq)
                    *(float4 *) (d + 32 * db + 8 * bq + 4 * h) = float4{o[db][4 * bq] * f, o[db][4 * bq + 1] * f, o[db][4 * bq + 2] * f, o[db][4 * bq + 3] * f};
        }
        if (at < stop) {
            __syncthreads();                                             // the LDS is free for the next piece
            if (tid == 0) any_bad = 0;
        }
    }
}

}  // namespace

hipError_t launch_rows(const PagedRowsParams & p, hipStream_t st) {
    const dim3 grid((unsigned) (p.target * p.row_groups * p.Hkv));
    if (p.softcap != 0.0f) hipLaunchKernelGGL(paged_rows_kernel<true>, grid, dim3(64 * kWaves), 0, st, p);
    else                   hipLaunchKernelGGL(paged_rows_kernel<false>, grid, dim3(64 * kWaves), 0, st, p);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_join(p, st) : e;
}

}  // namespace paged_fattn
