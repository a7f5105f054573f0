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
// device only. For each (KV head, row group) the tiles of all sequences are
// thought of as one row, cut into equal parts for the workgroups that fit the
// card (between sequences, where all are short); every workgroup reads the
// lengths and finds the sequences, or pieces of them, of its own part. A
// sequence within one workgroup is written at once; the pieces of the others
// go to records (at most two of a workgroup's pieces are such), which a second
// launch joins. (Joined by the workgroup that ends last instead: 100000 cells 88
// us instead of 83, as the records then have to pass through memory that all
// XCDs see.)
//
// More than 16 query rows (T tokens of G heads) are taken by the workgroup's
// waves side by side, 16 rows each, over the same cells: the second wave that
// reads a line finds it in the L1. (Two row tiles in one wave need 500
// registers, one wave for each SIMD: 54.9 us instead of 51.1 for 10 sequences of
// up to 6 drafts over 2100 to 6000 cells.)
//
// What bounds it: the cells' bytes, and for small calls the chain lengths ->
// page numbers -> keys -> scores -> values, then the join. Measured, 8 KV heads
// of 4 query heads each: one sequence of 700 cells 9.4 us, 24 of 1400 to 4000
// 51.1 us, 100000 cells (64 query heads) 79 us, 5.2 TB/s. Prompts are bound
// elsewhere: every wave reads its 16 KB of a tile through the L1 and turns V
// itself (4 prompts of 2048 tokens, 32 heads over 8: 749 us, 184 TFLOP/s).

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
constexpr int kMinTiles = 4;                    // least tiles of a part: one for each wave
constexpr int kWhole = 16;                      // sequences of up to so many tiles are not cut
constexpr float kPScale = 16384.0f;             // probabilities: 2^14 p stays normal in f16 down to p = 2^-28

struct PagedFattnParams {
    PagedPools c;
    const char * q;  int64_t q_nb1, q_nb2, q_nb3;       // token, head, sequence
    char * dst;      int64_t d_nb1, d_nb2, d_nb3;       // head, token, sequence
    const int32_t * lens;
    const int32_t * counts;                             // or null
    const float * sinks;                                // or null
    int2 * info;                                        // [unit][n_seq]: first workgroup of the sequence, pieces
    float * part;                                       // records [unit][workgroup][2]: rows x 128 sums, rows x {m, l}
    int32_t T, G, Hkv, R, row_groups, row_tiles;        // row tiles of 16 in a group
    uint32_t g_magic;                                   // ceil(2^32 / G) (0 for 1)
    int32_t target, long_target;                        // workgroups of a unit (head, row group), those that long sequences use
    int32_t row_waves;                                  // join: waves of a row
    float scale, softcap;
};

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_add(const int x) {
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xf, false);
}
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_max(const int x) {                 // (of values that are not negative)
    return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xf, false));
}
// Sum of the lanes up to and with this one (DPP: within rows of 16, then the
// rows' last lanes into those after them).
__device__ __forceinline__ int wave_scan(int x) {
    x = dpp_add<0x111, 0xf>(x);
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);
    x = dpp_add<0x143, 0xc>(x);
    return x;
}

template <typename P>
__device__ __forceinline__ int token_of(const P & p, const int r) {
    return p.G == 1 ? r : (int) __umulhi((uint32_t) r, p.g_magic);
}

// What a row group has to do for a sequence, t0 and t1 its first and last token.
struct SeqWork {
    int len, count;                             // cells (within the table), new tokens
    bool bad;
    // cells that the group's last row sees, -1 if it has no row
    __device__ __forceinline__ int limit(const int t0, const int t1) const {
        return count > t0 ? min(max(len - count + 1 + min(t1, count - 1), 0), len) : -1;
    }
};

__device__ __forceinline__ SeqWork seq_work(const PagedFattnParams & p, const int len, const int count) {
    SeqWork w;
    w.len = min(max(len, 0), p.c.max_pages * p.c.page_size);
    w.count = min(max(count, 0), p.T);
    w.bad = len != w.len || count != w.count;
    return w;
}

// Tiles of a sequence in the row of all tiles: one at least, so that rows that
// see nothing are written too.
__device__ __forceinline__ int tiles_of(const int limit) {
    return limit < 0 ? 0 : max(1, (limit + kTile - 1) / kTile);
}

// S tiles cut into W parts, the first S % W of them one tile longer: the first
// tile of a part, and the part that holds a tile.
struct Parts {
    int each, longer;
    __device__ __forceinline__ Parts(const int S, const int W) : each(S / W), longer(S - S / W * W) {}
    __device__ __forceinline__ int begin(const int w) const { return w * each + min(w, longer); }
    __device__ __forceinline__ int of(const int x) const {
        const int y = x - longer * (each + 1);
        return y < 0 ? x / (each + 1) : longer + y / each;
    }
};

// Sequences 64 b .. 64 b + 63, one to a lane.
struct Block {
    int len, count, tiles, upto;                // as read; tiles, and those of all sequences up to this one
    __device__ __forceinline__ void load(const PagedFattnParams & p, const int b, const int lane, const int t0, const int t1) {
        const int s = 64 * b + lane;
        const bool in = s < p.c.n_seq;
        len = in ? p.lens[s] : 0;
        count = !in ? 0 : p.counts ? p.counts[s] : p.T;
        tiles = in ? tiles_of(seq_work(p, len, count).limit(t0, t1)) : 0;
        upto = wave_scan(tiles);
    }
    // A negative count makes an empty slot, which no workgroup comes to.
    __device__ __forceinline__ void report(const PagedFattnParams & p) const {
        if (count < 0) paged_error(p.c, kPagedBadCount, count);
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(upto, 63); }
    __device__ __forceinline__ int active() const { return __builtin_popcountll(__ballot(tiles > 0)); }
    __device__ __forceinline__ int longest() const {
        int x = tiles;
        x = dpp_max<0x111, 0xf>(x);
        x = dpp_max<0x112, 0xf>(x);
        x = dpp_max<0x114, 0xf>(x);
        x = dpp_max<0x118, 0xf>(x);
        x = dpp_max<0x142, 0xa>(x);
        x = dpp_max<0x143, 0xc>(x);
        return __builtin_amdgcn_readlane(x, 63);
    }
};

template <typename P>
__device__ __forceinline__ char * record(const P & p, const int unit, const int wg, const int slot) {
    return (char *) p.part + (((int64_t) unit * p.target + wg) * 2 + slot) * (16 * p.row_tiles) * 130 * 4;
}

// e^(a - b) for running maxima a <= b, 1 where they are equal (both -inf too).
__device__ __forceinline__ float grow(const float a, const float b) { return a == b ? 1.0f : exp_fast(a - b); }

// Factor of a row's sums, with the sink as one more logit without a value: 0
// for a row that sees nothing, NaN where all logits are -inf.
template <typename P>
__device__ __forceinline__ float row_factor(const P & p, const float M, float L, const int head, const bool sees) {
    L *= 1.0f / kPScale;
    float up = 1.0f / kPScale;
    if (p.sinks) {
        const float sink = p.sinks[head], top = fmaxf(M, sink);
        const float e = grow(M, top);
        up *= e;
        L = L * e + (sink == -AL_INF ? 0.0f : grow(sink, top));
    }
    return L == 0.0f ? sees ? __builtin_nanf("") : 0.0f : up / L;
}

// The kernel's arguments as memory, to be loaded where they are used: held in
// scalar registers from the start, those that only a piece's beginning and end
// use displace what the loop over the cells needs.
__device__ __forceinline__ const __attribute__((address_space(4))) PagedFattnParams & arguments() {
    auto a = (const __attribute__((address_space(4))) PagedFattnParams *) __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return *a;
}

// ROWT: row tiles of 16 query rows that the waves take side by side (1, 2 or
// 4); the tiles of cells go round the waves of a row tile. CAP: logits
// soft-capped.
template <int ROWT, bool CAP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_fattn_kernel(const PagedFattnParams p) {
    constexpr int kCellWaves = kWaves / ROWT;
    __shared__ __attribute__((aligned(16))) float o_lds[kWaves][16][132];
    __shared__ float ml_lds[kWaves][16][2];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rt = wave / kCellWaves, cw = wave % kCellWaves;
    // the heads of the same cells next to one another in the grid
    const int units = p.row_groups * p.Hkv, unit = blockIdx.x % units, wg = blockIdx.x / units;
    const int h = unit % p.Hkv, group0 = unit / p.Hkv * (16 * ROWT);
    // tokens of the group, and of the wave's row tile (empty past the last row)
    const int t0 = token_of(p, group0), t1 = token_of(p, min(group0 + 16 * ROWT, p.R) - 1);
    const int r0 = group0 + 16 * rt;
    const int wt0 = token_of(p, min(r0, p.R - 1)), wt1 = token_of(p, min(r0 + 16, p.R) - 1);

    // this workgroup's part of all tiles
    const int n_blocks = (p.c.n_seq + 63) / 64;
    Block b;
    b.load(p, 0, lane, t0, t1);
    const bool first_wave = blockIdx.x == 0 && wave == 0;
    if (first_wave) b.report(p);
    int S = b.total(), active = b.active(), longest = b.longest(), block = 0, before = 0;
    for (int i = 1; i < n_blocks; ++i) {
        Block x;
        x.load(p, i, lane, t0, t1);
        if (first_wave) x.report(p);
        S += x.total();
        active += x.active();
        longest = max(longest, x.longest());
    }
    // Several sequences of up to kWhole tiles each are left whole, one or some to
    // a workgroup: equal parts cut them at places of their own, and a second
    // piece costs a workgroup more than the rounds that the cut saves (us, cut
    // and whole: 4 sequences of up to 200 cells 13.4, 10.1, 64 of 100 16.4, 11.5,
    // 10 of 500 14.1, 12.3; whole up to 32 tiles: 128 of 700 56.4, 60.2). Else
    // kMinTiles a workgroup at least, or a sequence; p.target workgroups for
    // sequences of up to 16 tiles on average, p.long_target for longer ones.
    const bool cut = longest > kWhole || active == 1;
    const int W = cut ? min(S > 16 * active ? p.long_target : p.target, max((S + kMinTiles - 1) / kMinTiles, active)) : min(p.target, active);
    if (wg >= W) return;
    const Parts parts(S, W);
    int at = parts.begin(wg), stop = parts.begin(wg + 1);
    if (!cut) {
        const Parts seqs(active, W);
        auto tile_of = [&](int i) {                                    // first tile of the i-th sequence that has any
            Block x = b;
            for (int k = 0, tiles = 0;;) {
                const uint64_t mask = __ballot(x.tiles > 0);
                const int have = __builtin_popcountll(mask);
                if (i < have) {
                    const int nth = __builtin_amdgcn_mbcnt_hi((uint32_t) (mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) mask, 0));
                    const int l = __builtin_ctzll(__ballot(x.tiles > 0 && nth == i));
                    return tiles + __builtin_amdgcn_readlane(x.upto, l) - __builtin_amdgcn_readlane(x.tiles, l);
                }
                i -= have;
                tiles += x.total();
                if (++k == n_blocks) return tiles;
                x.load(p, k, lane, t0, t1);
            }
        };
        at = tile_of(seqs.begin(wg));
        stop = tile_of(seqs.begin(wg + 1));
    }

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
        const auto & ap = arguments();
        if (threadIdx.x == 0) {
            if (first == 0)
                ap.info[(int64_t) unit * ap.c.n_seq + seq] =
                    int2{wg, whole ? 1 : parts.of(base + tiles - 1) - wg + 1};
            if (w.bad) paged_error(p.c, raw_len != w.len ? kPagedBadLength : kPagedBadCount, raw_len != w.len ? raw_len : raw_count);
        }
        bool bad = w.bad;
        const int seen = w.limit(wt0, wt1);                        // cells that the wave's last row sees
        const int least = max(w.len - w.count + 1 + wt0, 0);       // cells that all its rows see

        // Pages of a tile's cells: K by lanes n (group n / 4), V by lanes g.
        // Cells past the last group that the wave sees are taken from that one.
        struct Where {
            int k_page, v_page;
            int k_cell, v_cell;                                      // in the page
        };
        const int32_t * table = p.c.table + (int64_t) seq * p.c.t_nb1;
        const uint32_t last_group = (uint32_t) max(seen - 1, 0) / 8;
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
        auto page = [&](const int x, const bool used) {
            const bool ok = (uint32_t) x < (uint32_t) p.c.n_pages;
            bad |= !ok && used;
            return ok ? x : 0;
        };
        const char * k_head = p.c.k + (int64_t) h * p.c.k_nb2 + 16 * g;
        const char * v_head = p.c.v + (int64_t) h * p.c.v_nb2 + 16 * n;
        half8 k[2][4];
        u32x4 v[8];
        auto load_k = [&](const Where & a, const bool used) {
            const char * x = k_head + page(a.k_page, used) * p.c.k_nb3 + a.k_cell * p.c.k_nb1;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) k[e][kk] = *(const half8 *) (x + 4 * e * p.c.k_nb1 + 64 * kk);
        };
        auto load_v = [&](const Where & a, const bool used) {
            const char * x = v_head + page(a.v_page, used) * p.c.v_nb3 + a.v_cell * p.c.v_nb1;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = *(const u32x4 *) (x + i * p.c.v_nb1);
        };
        // The query row of this lane's column: its limit, and its operands
        // times a power of two that brings the largest value to [2^11, 2^12)
        const int r = r0 + n, t = token_of(p, min(r, p.R - 1));
        const bool valid = r < p.R && t < w.count;
        const int limit = valid ? w.len - w.count + 1 + t : seen;
        half8 q_hi[4], q_lo[4];
        float fac, m = -AL_INF, l = 0.0f;
        floatx4 acc[8];
        // Everything that the first tile needs goes out before anything is
        // computed: pages, query rows, then K and V (a wave without a tile
        // loads another wave's and uses none of it).
        const int wave_end = min(end, seen > 0 ? (seen + kTile - 1) / kTile : 0);
        const bool has = first + cw < wave_end;
        int tile = has ? first + cw : max(wave_end - 1, 0);
        const Where here = look_up(tile);
        Where next = look_up(tile + kCellWaves);
        asm volatile("" ::: "memory");
        float4 x[4][2];
        {
            const char * qr = ap.q + (int64_t) seq * ap.q_nb3 + (int64_t) (valid ? t : 0) * ap.q_nb1 +
                              (int64_t) (h * ap.G + (valid ? r - t * ap.G : 0)) * ap.q_nb2 + 32 * g;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[kk][e] = *(const float4 *) (qr + 128 * kk + 16 * e);
        }
        asm volatile("" ::: "memory");
        load_k(here, has);
        load_v(here, has);
        asm volatile("" ::: "memory");
        {
            float top = 0.0f;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (!valid) x[kk][e] = float4{0.0f, 0.0f, 0.0f, 0.0f};
                    top = fmaxf(fmaxf(fmaxf(top, fabsf(x[kk][e].x)), fmaxf(fabsf(x[kk][e].y), fabsf(x[kk][e].z))), fabsf(x[kk][e].w));
                }
            top = colmax4(top);
            // 2^(11 - exponent of top), within the normal range
            const int ex = min(max((int) (__float_as_uint(top) >> 23), 12), 253) - 127;
            const float up = __uint_as_float((uint32_t) (11 - ex + 127) << 23), down = __uint_as_float((uint32_t) (ex - 11 + 127) << 23);
            fac = p.scale * down;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                const float y[8] = {x[kk][0].x, x[kk][0].y, x[kk][0].z, x[kk][0].w, x[kk][1].x, x[kk][1].y, x[kk][1].z, x[kk][1].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = y[e] * up;
                    const _Float16 hi = (_Float16) z;
                    q_hi[kk][e] = hi;
                    q_lo[kk][e] = (_Float16) (z - (float) hi);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // V^T operand of dims 8 n + j: this lane's 8 cells of dim j
        auto v_operand = [&](const int j) {
            u32x4 a;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a[i] = __builtin_amdgcn_perm(v[2 * i + 1][j / 2], v[2 * i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
            return as_half8(a);
        };
        floatx4 s[2];
        auto scores = [&]() {
#pragma unroll
            for (int e = 0; e < 2; ++e) s[e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e) s[e] = mfma_16x16x32(k[e][kk], q_lo[kk], s[e]);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e) s[e] = mfma_16x16x32(k[e][kk], q_hi[kk], s[e]);
        };
        half8 p_hi, p_lo;
        // Probabilities of the tile against the rows' running maxima.
        auto softmax = [&](const int tile) {
            const int c0 = tile * kTile + 8 * g;
            const bool masked = (tile + 1) * kTile > least;          // some row does not see all of it
            float x[8];
            float top = -AL_INF;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = s[i / 4][i % 4] * fac;
                if constexpr (CAP) x[i] = p.softcap * tanhf(x[i] / p.softcap);
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 + i >= limit) x[i] = -AL_INF;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
            if (__any(top > m)) {
                top = fmaxf(m, colmax4(top));
                const float f = top > m ? exp_fast(m - top) : 1.0f;
                m = top;
                l *= f;
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] *= f;
            }
            // (a row that has met no logit but -inf, as products that overflow
            // give it, has m = -inf still: their weights are 0, not e^(-inf + inf))
            const float from = m == -AL_INF ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float e = exp_fast(x[i] - from) * kPScale;
                if (masked && c0 + i >= limit) e = 0.0f;
                l += e;
                const _Float16 hi = (_Float16) e;
                p_hi[i] = hi;
                p_lo[i] = (_Float16) (e - (float) hi);
            }
        };
        // o += P V of the tile. Cells past the wave's last are stale memory:
        // zeroed, as 0 times NaN is not 0. So are, one by one, the values that
        // are not finite of cells that some row does not see; the rows that do
        // see one get NaN in its dim, found by a product of ones.
        auto product = [&](const int tile) {
            const int c0 = tile * kTile + 8 * g;
            if ((tile + 1) * kTile > seen) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 + i >= seen) v[i] = u32x4{0, 0, 0, 0};
            }
            if (least < seen && (tile + 1) * kTile > least) {        // (one token: never)
                uint32_t odd[2] = {0, 0};                            // bit 8 (i % 4) + j of word i / 4: cell i, dim j
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (c0 + i >= least)
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            if ((v[i][d] & 0x7c00u) == 0x7c00u) odd[i / 4] |= 1u << (8 * (i % 4) + 2 * d), v[i][d] &= 0xffff0000u;
                            if ((v[i][d] & 0x7c000000u) == 0x7c000000u) odd[i / 4] |= 2u << (8 * (i % 4) + 2 * d), v[i][d] &= 0xffffu;
                        }
                }
                if (__any((odd[0] | odd[1]) != 0)) {
                    half8 sees;
#pragma unroll
                    for (int i = 0; i < 8; ++i) sees[i] = c0 + i < limit ? (_Float16) 1.0f : (_Float16) 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        half8 a;
#pragma unroll
                        for (int i = 0; i < 8; ++i) a[i] = odd[i / 4] >> (8 * (i % 4) + j) & 1 ? (_Float16) 1.0f : (_Float16) 0.0f;
                        const floatx4 x = mfma_16x16x32(a, sees, floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (x[e] > 0.0f) acc[j][e] = __builtin_nanf("");
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const half8 a = v_operand(j);
                acc[j] = mfma_16x16x32(a, p_hi, mfma_16x16x32(a, p_lo, acc[j]));
            }
        };

        // The wave's tiles. The next tile's K is loaded once this one's scores
        // are done, its V once this one's product is; pages are looked up a
        // tile earlier (the first two before any K: a page that is waited for
        // waits for all that was loaded before it). The last tile is a copy of
        // its own, so that no branch around the loads makes the compiler wait
        // for all of them.
        if (has) {
            for (; tile + kCellWaves < wave_end; tile += kCellWaves) {
                const Where after = look_up(tile + 2 * kCellWaves);
                scores();
                load_k(next, true);
                softmax(tile);
                product(tile);
                load_v(next, true);
                next = after;
            }
            scores();
            softmax(tile);
            product(tile);
        }

        // join the row tile's waves: maxima and sums, then the rescaled outputs
        // through LDS
        const bool any_bad = __any(bad);
        if (any_bad && lane == 0 && !w.bad) paged_error(p.c, kPagedBadPage, seq);
        l = colsum4(l);
        if (any_bad) l = __builtin_nanf("");
        if (g == 0) {
            ml_lds[wave][n][0] = m;
            ml_lds[wave][n][1] = l;
        }
        __syncthreads();
        {
            float M = m;
#pragma unroll
            for (int i = 0; i < kCellWaves; ++i) M = fmaxf(M, ml_lds[rt * kCellWaves + i][n][0]);
            const float f = grow(m, M);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *(float4 *) &o_lds[wave][n][8 * (4 * g + i)] = float4{acc[0][i] * f, acc[1][i] * f, acc[2][i] * f, acc[3][i] * f};
                *(float4 *) &o_lds[wave][n][8 * (4 * g + i) + 4] = float4{acc[4][i] * f, acc[5][i] * f, acc[6][i] * f, acc[7][i] * f};
            }
        }
        __syncthreads();
        const auto & ep = arguments();
        char * rec = record(ep, unit, wg, first == 0 ? 1 : 0);
        for (int item = threadIdx.x; item < 16 * ROWT * 16; item += 64 * kWaves) {
            const int row = item >> 4, dim = (item & 15) * 8;        // of the group
            const int w0 = row / 16 * kCellWaves, rr = row % 16;
            const int gr = group0 + row, tok = token_of(ep, min(gr, ep.R - 1));
            if (gr >= ep.R || tok >= w.count) continue;
            float M = ml_lds[w0][rr][0], L = 0.0f, o[8] = {};
#pragma unroll
            for (int i = 1; i < kCellWaves; ++i) M = fmaxf(M, ml_lds[w0 + i][rr][0]);
#pragma unroll
            for (int i = 0; i < kCellWaves; ++i) {
                L += ml_lds[w0 + i][rr][1] * grow(ml_lds[w0 + i][rr][0], M);
#pragma unroll
                for (int d = 0; d < 8; ++d) o[d] += o_lds[w0 + i][rr][dim + d];
            }
            float * d;
            float f = 1.0f;
            if (whole) {
                const int head = h * ep.G + gr - tok * ep.G;
                f = row_factor(ep, M, L, head, w.len - w.count + 1 + tok > 0);
                d = (float *) (ep.dst + (int64_t) seq * ep.d_nb3 + (int64_t) tok * ep.d_nb2 + (int64_t) head * ep.d_nb1) + dim;
            } else {
                d = (float *) rec + row * 128 + dim;
                if (dim == 0) *(float2 *) ((float *) rec + 16 * ROWT * 128 + row * 2) = float2{M, L};
            }
            *(float4 *) d = float4{o[0] * f, o[1] * f, o[2] * f, o[3] * f};
            *(float4 *) (d + 4) = float4{o[4] * f, o[5] * f, o[6] * f, o[7] * f};
        }
        if (at < stop) __syncthreads();                              // the LDS is free for the next piece
    }
}

// A row of the group, joined from the pieces of a sequence that has several.
// p.row_waves waves (1 or kWaves) take it, the halves of a wave every second
// piece, 4 dims to a lane; all loads of 8 of a half's pieces are in flight
// together.
__device__ __forceinline__ void join_row(const PagedFattnParams & p, const int2 info, const int unit, const int seq, const int count,
                                         const int row, float (*o_lds)[132]) {
    const int lane = threadIdx.x & 63, half = lane >> 5, d4 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows = 16 * p.row_tiles, row_waves = p.row_waves;
    const int h = unit % p.Hkv, gr = unit / p.Hkv * rows + row, t = token_of(p, min(gr, p.R - 1));
    const bool mine = gr < p.R && t < min(count, p.T);
    float M = -AL_INF, L = 0.0f;
    float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine) {
        for (int i0 = row_waves == 1 ? 0 : 16 * wave; i0 < info.y; i0 += 16 * row_waves) {
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = min(i0 + 2 * i + half, info.y - 1);
                const char * rec = record(p, unit, info.x + c, c == 0 ? 1 : 0);
                ml[i] = *(const float2 *) ((const float *) rec + rows * 128 + row * 2);
                x[i] = *(const float4 *) ((const float *) rec + row * 128 + 4 * d4);
            }
            asm volatile("" ::: "memory");
            float top = M;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i0 + 2 * i + half < info.y) top = fmaxf(top, ml[i].x);
            const float f = grow(M, top);
            L *= f; o.x *= f; o.y *= f; o.z *= f; o.w *= f;
            M = top;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i0 + 2 * i + half < info.y) {
                    const float e = grow(ml[i].x, M);
                    L += ml[i].y * e;
                    o.x += x[i].x * e; o.y += x[i].y * e; o.z += x[i].z * e; o.w += x[i].w * e;
                }
        }
    }
    // the wave's halves, then the row's waves
    {
        const float M2 = __shfl_xor(M, 32), L2 = __shfl_xor(L, 32);
        const float4 o2 = {__shfl_xor(o.x, 32), __shfl_xor(o.y, 32), __shfl_xor(o.z, 32), __shfl_xor(o.w, 32)};
        const float top = fmaxf(M, M2), f = grow(M, top), f2 = grow(M2, top);
        M = top;
        L = half ? L2 * f2 + L * f : L * f + L2 * f2;
        o = half ? float4{o2.x * f2 + o.x * f, o2.y * f2 + o.y * f, o2.z * f2 + o.z * f, o2.w * f2 + o.w * f}
                 : float4{o.x * f + o2.x * f2, o.y * f + o2.y * f2, o.z * f + o2.z * f2, o.w * f + o2.w * f2};
    }
    if (row_waves > 1) {
        if (half == 0) {
            *(float4 *) &o_lds[wave][4 * d4] = o;
            if (d4 == 0) o_lds[wave][128] = M, o_lds[wave][129] = L;
        }
        __syncthreads();
        if (wave) return;
        float top = M;
#pragma unroll
        for (int i = 1; i < kWaves; ++i) top = fmaxf(top, o_lds[i][128]);
        L = 0.0f;
        o = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float f = grow(o_lds[i][128], top);
            const float4 x = *(const float4 *) &o_lds[i][4 * d4];
            L += o_lds[i][129] * f;
            o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
        }
        M = top;
    }
    if (!mine || half) return;
    const int head = h * p.G + gr - t * p.G;
    const SeqWork w = seq_work(p, p.lens[seq], count);
    const float f = row_factor(p, M, L, head, w.len - w.count + 1 + t > 0);
    *(float4 *) ((float *) (p.dst + (int64_t) seq * p.d_nb3 + (int64_t) t * p.d_nb2 + (int64_t) head * p.d_nb1) + 4 * d4) =
        float4{o.x * f, o.y * f, o.z * f, o.w * f};
}

// Workgroups (rows, sequence, unit); few of them where most have nothing to join.
__global__ __launch_bounds__(64 * kWaves) void paged_join_kernel(const PagedFattnParams p) {
    __shared__ __attribute__((aligned(16))) float o_lds[kWaves][132];
    prefetch_params(p);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows = min(16 * p.row_tiles, p.R), seq = blockIdx.y, unit = blockIdx.z;
    const int2 info = p.info[(int64_t) unit * p.c.n_seq + seq];
    const int count = p.counts ? p.counts[seq] : p.T;
    // (no row of the group: nothing was written to info)
    if (min(count, p.T) <= token_of(p, unit / p.Hkv * (16 * p.row_tiles)) || info.y < 2) return;
    if (p.row_waves > 1) join_row(p, info, unit, seq, count, blockIdx.x, o_lds);
    else
        for (int row = blockIdx.x * kWaves + wave; row < rows; row += gridDim.x * kWaves) join_row(p, info, unit, seq, count, row, o_lds);
}

struct Plan {
    PagedFattnParams p;
    bool empty = false;
    size_t info_bytes = 0, bytes = 0;                   // of the info, of it and the records
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
    // (a row's token is found exactly while rows times heads of a group stay below 2^32)
    if (T > (1 << 16) || Hq > (1 << 12) || T * Hq > (1 << 22) || n_seq > 65535 || T * (Hq / Hkv) * (Hq / Hkv) >= (1ll << 32))
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
    p.row_tiles = p.R <= 16 ? 1 : p.R <= 32 ? 2 : 4;
    const int rows = 16 * p.row_tiles;
    p.row_groups = (p.R + rows - 1) / rows;
    const int64_t units = (int64_t) p.row_groups * Hkv;
    if (units > 65535) return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: sizes out of range");
    const int64_t most = n_seq * std::max<int64_t>(1, ((int64_t) p.c.max_pages * p.c.page_size + kTile - 1) / kTile);   // tiles there can be
    if (most > INT32_MAX) return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: sizes out of range");
    // One workgroup a CU, 48 to 64 KB of its waves' loads in flight: more only
    // lengthen the queues (us with one / two / four: 24 sequences to 4000 cells
    // 51.3 / 52.6 / 54.6, 100000 cells of 64 heads 79.4 / 81.7 / 85.7, 8000 cells
    // 13.2 / 14.2 / 13.9). Two where row tiles share the loads (verify of 10
    // sequences 48.5 / 47.1 / 50.0), and for many short sequences, whose ends
    // are not hidden (96 to 300 cells 30.8 / 24.9, 128 to 700 57.2 / 57.2).
    const int64_t per_cu = n_cu / std::max<int64_t>(1, units);
    const int64_t useful = std::max(n_seq, (most + kMinTiles - 1) / kMinTiles);
    p.target = (int32_t) std::max<int64_t>(1, std::min<int64_t>(2 * n_cu / std::max<int64_t>(1, units), useful));
    p.long_target = p.row_tiles == 1 ? (int32_t) std::max<int64_t>(1, std::min<int64_t>(per_cu, p.target)) : p.target;
    // few sequences have many pieces each
    p.row_waves = p.long_target > 16 * n_seq ? kWaves : 1;
    p.scale = a->scale;
    p.softcap = a->logit_softcap;
    pl.info_bytes = ((size_t) units * n_seq * sizeof(int2) + 255) / 256 * 256;
    pl.bytes = pl.info_bytes + (p.target > 1 ? (size_t) units * p.target * 2 * rows * 130 * 4 : 0);     // one workgroup a unit: no pieces
    *out = pl;
    return AL_OK;
}

template <int ROWT>
void launch(const PagedFattnParams & p, hipStream_t st) {
    const dim3 grid((unsigned) (p.target * p.row_groups * p.Hkv));
    if (p.softcap != 0.0f) hipLaunchKernelGGL((paged_fattn_kernel<ROWT, true>), grid, dim3(64 * kWaves), 0, st, p);
    else                   hipLaunchKernelGGL((paged_fattn_kernel<ROWT, false>), grid, dim3(64 * kWaves), 0, st, p);
}

hipError_t launch(const PagedFattnParams & p, hipStream_t st) {
    switch (p.row_tiles) {
        case 1: launch<1>(p, st); break;
        case 2: launch<2>(p, st); break;
        default: launch<4>(p, st); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.target == 1) return e;                    // one workgroup a unit: no pieces
    const int rows = std::min(16 * p.row_tiles, p.R);
    // (all rows side by side: 98 sequences of one tile, 56 rows, 24.6 us in all instead of 20.7)
    const int64_t pairs = (int64_t) p.c.n_seq * p.row_groups * p.Hkv;
    const int side = (int) std::max<int64_t>(1, std::min<int64_t>((rows + kWaves - 1) / kWaves, 2048 / pairs));
    const dim3 grid((unsigned) (p.row_waves == 1 ? side : rows), (unsigned) p.c.n_seq, (unsigned) (p.row_groups * p.Hkv));
    hipLaunchKernelGGL(paged_join_kernel, grid, dim3(64 * kWaves), 0, st, p);
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
    return pl.empty ? 0 : al_workspace_bytes(pl.bytes);
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
    rc = al_workspace_records("paged_fattn", pl.bytes, a->workspace, a->workspace_bytes, a->stream, (void **) &pl.p.info);
    if (rc != AL_OK) return rc;
    pl.p.part = (float *) ((char *) pl.p.info + pl.info_bytes);
    const hipError_t e = launch(pl.p, (hipStream_t) a->stream);
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "paged_fattn: launch");
}
