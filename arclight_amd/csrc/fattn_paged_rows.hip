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
// each wave a quarter: one of its 8 instructions beside every second pair of the
// first products (8 in a row took 0.6 us of a tile's 3), by page numbers that a
// vector load finds for 32 tiles at once. A tile is [cell][128] with 16-byte
// pieces permuted within a cell so that the operand reads are free of bank
// conflicts: piece j of K's cell c at j ^ (c & 15), of V's at j ^ 4 (c & 3). The
// probabilities of 16 cells are made beside the products of the 16 before. Two
// workgroups to a CU, each wave with half of a SIMD's registers.
//
// Tiles that some row does not see all of are masked value by value; V of cells
// that no row sees is cleared there (0 times NaN is not 0), and so are single
// values that are not finite: the rows that do see them get NaN in their dim,
// found by a product of ones.
//
// What bounds it: the matrix cores, each product taken twice, which are busy half
// of the time over a launch and run at 1.9 GHz under this load; what else there
// is are a tile's barrier (0.24 us of 3), the query rows' way into registers (3 us
// a sequence and workgroup) and parts of tiles that are hidden. Measured, 32 heads
// over 8: two prompts of 4000 over windows of 1000 270 to 292 us on several cards,
// 450 to 485 TFLOP/s by the cells that are seen, twice that as executed (a plain
// f16 product of 8192^3 runs at 1250 to 1300, products from registers alone at
// 1400 to 1550), one of 4096 over windows of 8192 558; 11 trees of 31 to 61 nodes
// over 2000 to 6000 cells, 64 heads, 160 to 172 us. (The next tile's scores beside
// this one's probabilities, tiles of 32 cells in a ring of four: 330 us instead of
// 294, for twice the barriers; of 64 cells it does not fit the registers. Rows
// stored through LDS, waves' priorities raised for the products: no gain.)

#include <hip/hip_runtime.h>

#include "fattn_paged.hpp"
#include "fattn_prefill_common.hpp"

namespace paged_fattn {

namespace {

using fattn::half4;
using fattn::int4v;
using fattn::lds_addr;
using fattn_prefill::float2v;
using fattn_prefill::floatx16;
using fattn_prefill::half2v;
using fattn_prefill::mfma32;
using fattn_prefill::pair_max;
using fattn_prefill::pair_sum;
using fattn_prefill::wait_vm;

// LDS by address.
template <typename T>
__device__ __forceinline__ T lds_at(const uint32_t at) { return *(const __attribute__((address_space(3))) T *) (uintptr_t) at; }
__device__ __forceinline__ half4 read_tr16(const uint32_t at) {
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((fattn::lds_short4v *) (uintptr_t) at));
}
// x - (a half of) hi. hi is made of x in an instruction between, so x, an
// exponential, is never read here by the instruction right after it.
__device__ __forceinline__ float rest(const half2v hi, const int half, const float x) {
    float y;
    if (half) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(hi), "v"(x));
    else      asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(y) : "v"(hi), "v"(x));
    return y;
}

constexpr int kTileBytes = PagedRowsParams::kTile * 256;
constexpr float kBelow = 8.0f, kOutgrown = 14.0f;        // log2: the reference below the maximum, a score that moves it

// The first k of 64 cells, a bit each.
__device__ __forceinline__ uint64_t upto64(const int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; }
// span8 and nodes8 of 64 cells
__device__ __forceinline__ uint64_t span64(const int c0, const int limit, const int low, const int first) {
    return upto64(limit - c0) & (~upto64(low - c0) | upto64(first - c0));
}
template <typename A>
__device__ __forceinline__ uint64_t nodes64(const A & p, const int32_t * words, const int32_t * pos, const int u0, const int count,
                                            const int low) {
    if (u0 <= -64 || u0 >= count) return 0;
    const int u = max(u0, 0), i = u >> 5, last = (count - 1) >> 5, sh = u & 31;
    const uint64_t two = (uint32_t) words[i] | (uint64_t) (uint32_t) words[min(i + 1, last)] << 32;
    const uint64_t third = (uint32_t) words[min(i + 2, last)];
    uint64_t m = (sh ? two >> sh | third << (64 - sh) : two) << (u - u0) & upto64(count - u0);
    // (positions of nodes are within a window that is as long as the tree)
    if (pos && p.window < count)
        for (uint64_t rest = m; rest; rest &= rest - 1) {
            const int at = pos[u0 + __builtin_ctzll(rest)];
            if (at < low && at >= p.first) m &= ~(rest & -rest);
        }
    return m;
}

// 16 bytes a lane from page + at + lane_at into LDS at `to` + 16 * lane, without
// passing registers. page, at and to are the wave's. (M0 carries the LDS address;
// nothing else in this kernel uses it.) A scalar register that a vector
// instruction wrote, as readlane writes `at` or brings back a spilled one, may be
// read by a vector memory instruction 5 wait states later, which the compiler does
// not see to within an asm statement: the move to M0 and four of s_nop.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds(const int4v page, const uint32_t at, const uint32_t lane_at, const uint32_t to) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(lane_at), "s"(page), "s"(at), "s"(to)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ int4v page_desc(const char * head, const uint32_t page, const uint32_t nb3) {
    const uint64_t a = (uint64_t) head + (uint64_t) page * nb3;
    return int4v{(int) (uint32_t) a, (int) (uint32_t) (a >> 32), -1, 0x00020000};
}

// Of a KV head's workgroups each row group gets a share by its tiles, one at
// least, where sequences differ in their groups: those of few rows are not in
// the last ones (us, equal shares and so: 4 prompts of 1 to 200 tokens over
// windows of 1024 33.4, 24.1, 8 trees of 30 to 60 nodes over 4000 cells 67.9, 62.5,
// 11 of 31 to 61 over up to 6000, 64 heads, 165.5, 162.6). Changes this
// workgroup's unit, its number within it, the unit's workgroups, and what brings
// the number to its record among the head's.
template <typename P>
__device__ __forceinline__ void share(const P & p, const int lane, int & unit, int & wg, int & target, int & records) {
    const int n_blocks = (p.c.n_seq + 63) / 64, last = token_of(p, (p.row_groups - 1) * P::kRows);
    bool fewer = false;
    for (int k = 0; k < n_blocks; ++k) {
        const int s = 64 * k + lane, count = s < p.c.n_seq ? p.counts[s] : 0;
        fewer |= count > 0 && count <= last;
    }
    if (!__any(fewer)) return;
    const int head = blockIdx.x % p.Hkv, places = p.row_groups * p.target, place = blockIdx.x / p.Hkv;
    int tiles = 0;                                                       // lane g: tiles of group g
    float total = 0.0f;
    for (int k = 0; k < n_blocks; ++k)
        for (int g = 0; g < p.row_groups; ++g) {
            const int r = g * P::kRows;
            Block x;
            x.load(p, k, lane, token_of(p, r), token_of(p, min(r + P::kRows, p.R) - 1));
            const int S = x.total();
            if (lane == g) tiles += S;
            total += (float) S;
        }
    const float each = (float) places / fmaxf(total, 1.0f);
    float upto = 0.0f;
    int start = 0, stop = 0, g = 0;
    for (;; ++g) {
        upto += (float) __builtin_amdgcn_readlane(tiles, g);
        const int after = p.row_groups - 1 - g;
        stop = min(max(__builtin_amdgcn_readfirstlane((int) (upto * each + 0.5f)), start + 1), places - after);
        if (after == 0) stop = places;
        if (place < stop || after == 0) break;
        start = stop;
    }
    unit = g * p.Hkv + head;
    wg = place - start;
    target = stop - start;
    records = head * places + start - unit * p.target;
}

// CAP: logits soft-capped. P: PagedRowsParams, or with a window or bits alone.
template <bool CAP, typename P>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_rows_kernel(const P p) {
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];  // K and V of two tiles
    __shared__ uint64_t odd[128];                   // of each dim, the tile's cells whose value is not finite
    __shared__ int any_odd, any_bad;
    prefetch_params(p);
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, lr = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The heads of the same cells next to one another in the grid, and the last
    // row groups first: those of a prompt's beginning see the fewest cells and end
    // the launch (us, first groups first: two prompts of 4000 over windows of 1000
    // 301, 294).
    const int units = p.row_groups * p.Hkv;
    int unit = units - 1 - (int) (blockIdx.x % units), wg = blockIdx.x / units, target = p.target, records = 0;
    if (__builtin_expect(p.shared, 0)) share(p, lane, unit, wg, target, records);
    const int head = unit % p.Hkv, group0 = unit / p.Hkv * P::kRows;
    // tokens of the group, and of the wave's rows (none past the last row)
    const int t0 = token_of(p, group0), t1 = token_of(p, min(group0 + P::kRows, p.R) - 1);
    const int r0 = group0 + 32 * wave;
    const int wt0 = token_of(p, min(r0, p.R - 1)), wt1 = token_of(p, min(r0 + 32, p.R) - 1);

    const int n_blocks = (p.c.n_seq + 63) / 64;
    Block b;
    MyPart part;
    if (!find_part(p, wg, target, target, lane, t0, t1, blockIdx.x == 0 && wave == 0, b, part)) return;
    int at = part.at, block = 0, before = 0;
    const int stop = part.stop;
    if (tid < 128) odd[tid] = 0;
    if (tid == 0) any_odd = any_bad = 0;

    const uint32_t k_nb1 = (uint32_t) p.c.k_nb1, k_nb3 = (uint32_t) p.c.k_nb3, v_nb1 = (uint32_t) p.c.v_nb1, v_nb3 = (uint32_t) p.c.v_nb3, lds0 = lds_addr(lds);
    // this lane's offset within 4 cells of K (their place among 16 cells) and of V
    uint32_t k_lane[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) k_lane[q] = (uint32_t) (lane >> 4) * k_nb1 + (uint32_t) (((lane & 15) ^ (4 * q + (lane >> 4))) * 16);
    const uint32_t v_lane = (uint32_t) (lane >> 4) * v_nb1 + (uint32_t) (((lane & 15) ^ (4 * (lane >> 4))) * 16);
    const char * k_head = p.c.k + (int64_t) head * p.c.k_nb2;
    const char * v_head = p.c.v + (int64_t) head * p.c.v_nb2;
    // operand reads: K of cell lr, V as 4 x 16 pieces
    // (the permutation's bits are flipped in the address: a tile begins at a
    // multiple of its size)
    const int s16 = lane & 15, v_sw = s16 >> 2;
    const uint32_t k_at = lds0 + lr * 256 + ((h ^ (lr & 15)) << 4);
    const uint32_t v_at = lds0 + kTileBytes + (((4 * h + v_sw) * 256 + ((2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1)) << 4) + (s16 & 1) * 8) ^ (64 * v_sw));

    while (at < stop) {
        // the sequence that holds tile `at`
        while (__builtin_expect(at >= before + b.total(), 0)) {
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
        const auto & ap = arguments<P>();
        if (tid == 0) {
            if (first == 0) ap.info[(int64_t) unit * ap.c.n_seq + seq] = int2{wg + records, whole ? 1 : part.pieces(base, tiles, wg, l64)};
            if (__builtin_expect(w.bad, 0)) paged_error(p.c, raw_len != w.len ? kPagedBadLength : kPagedBadCount, raw_len != w.len ? raw_len : raw_count);
        }
        const int begin = w.len - w.count;
        // what the group sees, what the wave sees, what all of the group's or the wave's rows see
        const Span group = span_of(p, w, t0, t1), mine = span_of(p, w, wt0, wt1);
        const int gap = group.gap(p), gap_at = group.gap_at(p);
        auto tile_at = [&](const int i) { return P::kWindow && i >= gap_at ? i + gap : i; };
        // Tiles that some row does not see all of: from `from` on, and from `a` to `b`.
        struct Edges {
            int from, a, b;
            __device__ __forceinline__ bool has(const int tile) const { return tile >= from || (P::kWindow && tile >= a && tile < b); }
        };
        auto edges_of = [&](const int least, const int low) {
            return Edges{least / P::kTile, p.first / P::kTile, (max(low, 0) + P::kTile - 1) / P::kTile};
        };
        // cells that all rows from a token on see, and the last window's beginning
        auto least_of = [&](const int first_token) { return has_bits(p) ? max(begin, 0) : max(begin + 1 + first_token, 0); };
        auto low_of = [&](const int last_token) {
            return P::kWindow ? (has_bits(p) ? w.len : begin + 1 + min(last_token, w.count - 1)) - p.window : 0;
        };
        const Edges edges = edges_of(least_of(t0), low_of(t1)), my_edges = edges_of(least_of(wt0), low_of(wt1));
        const int tiles_end = group.limit > 0 ? end : first;             // (nothing is seen: no tile)

        // Where this wave's 16 cells of 32 tiles lie, two groups of 8 to a tile:
        // lane 2 (i % 32) + e that of group e of tile i. Groups past the last
        // that the group of rows sees are taken from that one, those before the
        // first window from its.
        struct Where {
            uint32_t page, k, v;                                         // bytes in the page
        };
        bool bad = false;
        auto look_up = [&](const int i) {                                // of tiles i / 32 * 32 on
            const int last_group = max(group.limit - 1, 0) / 8, from = (ap.first + 7) >> 3;
            const int of = min(i / 32 * 32 + (lane >> 1), tiles_end - 1);
            int g = min(tile_at(of) * 8 + 2 * wave + (lane & 1), last_group);
            if (P::kWindow && g >= from) g = max(g, group.low >> 3);
            const int pg = (int) page_of_group(p.c, (uint32_t) g);
            const uint32_t cell = (uint32_t) (g - pg * p.c.groups) * 8;
            return Where{(uint32_t) ap.c.table[(int64_t) seq * ap.c.t_nb1 + pg], cell * k_nb1, cell * v_nb1};
        };
        auto check = [&](Where & a, const int i) {                       // (apart, as it waits for the table)
            const bool ok = a.page < (uint32_t) ap.c.n_pages;
            bad |= !ok && min(i / 32 * 32 + (lane >> 1), tiles_end - 1) >= first;
            if (!ok) a.page = 0;
        };
        // One of the 8 instructions that load tile i: cells 8 e + 4 f on of this
        // wave's, K or V.
        int4v desc[2];
        auto load = [&](const Where & a, const int i, const int buf, const int q) {
            const int e = q >> 2, v = q >> 1 & 1, f = q & 1, from = 2 * (i & 31) + e;
            if ((q & 3) == 0) {
                const uint32_t pg = (uint32_t) __builtin_amdgcn_readlane((int) a.page, from);
                desc[0] = page_desc(k_head, pg, k_nb3);
                desc[1] = page_desc(v_head, pg, v_nb3);
            }
            load_lds(desc[v], (uint32_t) __builtin_amdgcn_readlane((int) (v ? a.v : a.k), from) + 4 * f * (v ? v_nb1 : k_nb1),
                     v ? v_lane : k_lane[2 * e + f], lds0 + (uint32_t) (buf * 2 * kTileBytes + v * kTileBytes + (16 * wave + 8 * e + 4 * f) * 256));
        };

        // This lane's query row, loaded while the first pages are looked up
        const int r = r0 + lr, t = token_of(p, min(r, p.R - 1));
        const bool valid = r < p.R && t < w.count;
        Where where = {0, 0, 0};
        if (first < tiles_end) where = look_up(first);
        float4 x[8][2];
        {
            const float * qr = (const float *) (ap.q + (int64_t) seq * ap.q_nb3 + (int64_t) (valid ? t : 0) * ap.q_nb1 +
                                                (int64_t) (head * ap.G + (valid ? r - t * ap.G : 0)) * ap.q_nb2) + 8 * h;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[ks][e] = *(const float4 *) (qr + 16 * ks + 4 * e);
        }
        asm volatile("" ::: "memory");
        if (first < tiles_end) {
            check(where, first);
#pragma unroll
            for (int q = 0; q < 8; ++q) load(where, first, 0, q);
        }
        // its operands times a power of two that brings the largest value to
        // [2^11, 2^12), and the scores' factor
        half8 q_hi[8], q_lo[8];
        float fac;
        {
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
            if (!CAP && fac < 1.17549435e-38f) fac = 1.17549435e-38f;
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
        // what it sees
        const int limit = valid ? begin + 1 + t : group.limit;
        int low = 0;
        const int32_t * words = nullptr;
        const int32_t * node_pos = nullptr;
        bool bad_row = false;
        {
            int place = begin + t;
            if (P::kBits && ap.bits) {
                words = ap.bits + (int64_t) seq * ap.b_nb2 + (int64_t) (valid ? t : 0) * ap.b_nb1;
                if (P::kWindow && ap.pos) node_pos = ap.pos + (int64_t) seq * ap.p_nb1;
                if (node_pos && valid) {
                    place = node_pos[t];
                    bad_row = place < begin || place >= w.len;
                    if (__builtin_expect(bad_row && h == 0, 0)) paged_error(p.c, kPagedBadPos, place);
                }
            }
            if (P::kWindow && valid && !bad_row) low = place + 1 - ap.window;
        }
        // Of the 64 cells from c0 on: those that this lane's row sees.
        auto sees64 = [&](const int c0) {
            const auto & sp = arguments<P>();
            if constexpr (!P::kWindow) return upto64(begin - c0) | nodes64(sp, words, nullptr, c0 - begin, w.count, 0);
            if (P::kBits && sp.bits) return span64(c0, begin, low, sp.first) | nodes64(sp, words, node_pos, c0 - begin, w.count, low);
            return span64(c0, limit, low, sp.first);
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
            const bool more = i + 1 < tiles_end;                         // (loaded beside the scores)
            if (more && ((i + 1) & 31) == 0) {
                where = look_up(i + 1);
                check(where, i + 1);
            }
            char * v_tile = lds + buf * 2 * kTileBytes + kTileBytes;
            const bool edge = edges.has(tile);                           // some row of the group does not see all of it
            if (edge) {
                const uint64_t some = P::kWindow ? span64(c0, group.limit, group.low, ap.first) : upto64(group.limit - c0);
                const uint64_t all = P::kWindow ? span64(c0, least_of(t0), low_of(t1), ap.first) : upto64(least_of(t0) - c0);
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
            const bool work = has_rows && c0 < mine.limit && !(P::kWindow && c0 >= p.first && c0 + P::kTile <= mine.low);
            if (!work && more)
#pragma unroll
                for (int q = 0; q < 8; ++q) load(where, i + 1, buf ^ 1, q);
            if (work) {
                // scores: K's operands read one step ahead, an instruction of
                // the next tile's loads a step
                floatx16 s[2] = {floatx16{}, floatx16{}};
                half8 k[2][2];
                const uint32_t kx = k_at + buf * 2 * kTileBytes;
                auto k_read = [&](const int ks) {
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) k[ks & 1][cb] = as_half8(lds_at<u32x4>((kx ^ (ks << 5)) + 32 * 256 * cb));
                };
                k_read(0);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    if (ks + 1 < 8) k_read(ks + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) s[cb] = mfma32(k[ks & 1][cb], q_lo[ks], s[cb]);
                    if (more) load(where, i + 1, buf ^ 1, ks);
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) s[cb] = mfma32(k[ks & 1][cb], q_hi[ks], s[cb]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                float f = fac;
                if constexpr (CAP) {
                    f = p.softcap * kLog2e;
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                        for (int v = 0; v < 16; ++v) s[cb][v] = tanhf(s[cb][v] * fac);
                }
                if (my_edges.has(tile)) {
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
                // probabilities and products, 16 cells (kk) and 32 dims (db) a
                // step: a step's V is read one step ahead, and beside its two
                // products a quarter of the next 16 cells' probabilities is made
                const float ref = m == -AL_INF ? 0.0f : m;
                float sum[2] = {0.0f, 0.0f};
                half8 p_hi[2], p_lo[2], v[2];
                const uint32_t vx = v_at + buf * 2 * kTileBytes;
                auto v_read = [&](const int step) {
                    const uint32_t x = (vx ^ (64 * (step & 3))) + 16 * 256 * (step >> 2);
                    const half4 a = read_tr16(x), c = read_tr16(x + 8 * 256);
                    v[step & 1] = half8{a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
                };
                auto probabilities = [&](const int kk, const int e) {    // of slots e and e + 1
                    float x[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        x[u] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][8 * (kk & 1) + e + u], f, -ref));
                        sum[u] += x[u];
                    }
                    half2v hi = __builtin_convertvector(float2v{x[0], x[1]}, half2v);
                    asm volatile("" : "+v"(hi));                         // (kept in this step)
                    half2v lo = __builtin_convertvector(float2v{rest(hi, 0, x[0]), rest(hi, 1, x[1])}, half2v);
                    asm volatile("" : "+v"(lo));
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        p_hi[kk & 1][e + u] = hi[u];
                        p_lo[kk & 1][e + u] = lo[u];
                    }
                };
                v_read(0);
#pragma unroll
                for (int e = 0; e < 8; e += 2) probabilities(0, e);
#pragma unroll
                for (int step = 0; step < 16; ++step) {
                    const int kk = step >> 2, db = step & 3;
                    if (step + 1 < 16) v_read(step + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    o[db] = mfma32(v[step & 1], p_lo[kk & 1], o[db]);
                    if (kk < 3) probabilities(kk + 1, 2 * db);
                    o[db] = mfma32(v[step & 1], p_hi[kk & 1], o[db]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                l += sum[0] + sum[1];
            }
            if (__builtin_expect(edge && any_odd, 0)) {                                       // (written before the barrier above)
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

        if (__builtin_expect(__any(bad) && lane == 0, 0)) {
            any_bad = 1;
            if (!w.bad) paged_error(p.c, kPagedBadPage, seq);
        }
        __syncthreads();
        l = pair_sum(l);
        if (any_bad || w.bad || bad_row) l = __builtin_nanf("");
        if (valid) {
            const auto & ep = arguments<P>();
            float factor = 1.0f;
            float * d;
            if (whole) {
                const int hq = head * ep.G + r - t * ep.G;
                factor = row_factor<P>(ep, w, seq, t, m, l, hq);
                d = (float *) (ep.dst + (int64_t) seq * ep.d_nb3 + (int64_t) t * ep.d_nb2 + (int64_t) hq * ep.d_nb1);
            } else {
                float * rec = (float *) record(ep, unit, wg + records, first == 0 ? 1 : 0);
                d = rec + (r - group0) * 128;
                if (h == 0) *(float2 *) (rec + P::kRows * 128 + (r - group0) * 2) = float2{m, l};
            }
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int bq = 0; bq < 4; ++bq)
                    *(float4 *) (d + 32 * db + 8 * bq + 4 * h) =
                        float4{o[db][4 * bq] * factor, o[db][4 * bq + 1] * factor, o[db][4 * bq + 2] * factor, o[db][4 * bq + 3] * factor};
        }
        if (at < stop) {
            __syncthreads();                                             // the LDS is free for the next piece
            if (tid == 0) any_bad = 0;
        }
    }
}

// The join of sequences with few pieces each: half a wave to a row, 4 dims to a
// lane, the loads of 4 pieces in flight together. Workgroups (rows, sequence,
// unit). (A wave to a row, its halves every second piece, as the join of few
// rows has it: 28 us instead of 12 for 11 trees of up to 488 rows. 12 pieces in
// flight where there are more than 4: one tree of 26 nodes over 2000 cells 0.3 us
// less, a prompt of 300 tokens 1.8 more.)
__global__ __launch_bounds__(64 * kWaves) void paged_join_rows_kernel(const PagedRowsParams p) {
    using P = PagedRowsParams;
    prefetch_params(p);
    const int seq = blockIdx.y, unit = blockIdx.z, d4 = threadIdx.x & 31;
    const int2 info = p.info[(int64_t) unit * p.c.n_seq + seq];
    const int count = min(p.counts ? p.counts[seq] : p.T, p.T), len = p.lens[seq];
    const int head = unit % p.Hkv, group0 = unit / p.Hkv * P::kRows;
    // (no row of the group: nothing was written to info)
    if (count <= token_of(p, group0) || info.y < 2) return;
    const SeqWork w = seq_work(p, len, count);
    const int end = min(P::kRows, min(p.R, count * p.G) - group0);
    for (int row = blockIdx.x * (2 * kWaves) + (threadIdx.x >> 5); row < end; row += gridDim.x * (2 * kWaves)) {
        float M = -AL_INF, L = 0.0f;
        float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = 0; i0 < info.y; i0 += 4) {
            float2 ml[4];
            float4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = min(i0 + i, info.y - 1);
                const float * rec = (const float *) record(p, unit, info.x + c, c == 0 ? 1 : 0);
                ml[i] = *(const float2 *) (rec + P::kRows * 128 + row * 2);
                x[i] = *(const float4 *) (rec + row * 128 + 4 * d4);
            }
            asm volatile("" ::: "memory");
            float top = M;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i0 + i < info.y) top = fmaxf(top, ml[i].x);
            const float f = grow<P>(M, top);
            L *= f; o.x *= f; o.y *= f; o.z *= f; o.w *= f;
            M = top;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i0 + i < info.y) {
                    const float e = grow<P>(ml[i].x, M);
                    L += ml[i].y * e;
                    o.x += x[i].x * e; o.y += x[i].y * e; o.z += x[i].z * e; o.w += x[i].w * e;
                }
        }
        const int gr = group0 + row, t = token_of(p, gr), hq = head * p.G + gr - t * p.G;
        const float f = row_factor<P>(p, w, seq, t, M, L, hq);
        *(float4 *) ((float *) (p.dst + (int64_t) seq * p.d_nb3 + (int64_t) t * p.d_nb2 + (int64_t) hq * p.d_nb1) + 4 * d4) =
            float4{o.x * f, o.y * f, o.z * f, o.w * f};
    }
}

}  // namespace

template <typename P>
void launch(const PagedRowsParams & all, hipStream_t st) {
    P p;
    static_cast<PagedRowsParams &>(p) = all;
    const dim3 grid((unsigned) (p.target * p.row_groups * p.Hkv));
    if (p.softcap != 0.0f) hipLaunchKernelGGL((paged_rows_kernel<true, P>), grid, dim3(64 * kWaves), 0, st, p);
    else                   hipLaunchKernelGGL((paged_rows_kernel<false, P>), grid, dim3(64 * kWaves), 0, st, p);
}

hipError_t launch_rows(const PagedRowsParams & p, hipStream_t st) {
    if (!p.bits) launch<PagedRowsWindowParams>(p, st);
    else if (!p.pos) launch<PagedRowsTreeParams>(p, st);
    else launch<PagedRowsParams>(p, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.target == 1 || p.whole) return e;           // no pieces
    if (p.row_waves > 1) return launch_join(p, st);
    const int64_t pairs = (int64_t) p.c.n_seq * p.row_groups * p.Hkv;
    const int side = (int) std::max<int64_t>(1, std::min<int64_t>(PagedRowsParams::kRows / (2 * kWaves), 4096 / pairs));
    hipLaunchKernelGGL(paged_join_rows_kernel, dim3((unsigned) side, (unsigned) p.c.n_seq, (unsigned) (p.row_groups * p.Hkv)), dim3(64 * kWaves), 0, st, p);
    return hipGetLastError();
}

}  // namespace paged_fattn
