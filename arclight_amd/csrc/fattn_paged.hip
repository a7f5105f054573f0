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
//
// Calls with a rule (al_paged_sees: windows with first cells, trees) take the
// same code with PagedSeesParams, or its parts for windows or trees alone: tiles
// that no row of the group sees are left out of the row of tiles, those that some
// row does not see all of are masked by a bit for each of a lane's 8 cells, and
// pages outside of what is seen are not looked up. With little to do every 16 rows
// are a group of their own (few_row_cells), and many query rows go to the kernel of
// fattn_paged_rows.hip. Measured, 32 heads over 8: one token over a window of 1024
// 9.9 us, 30 over windows of 4096 90.1 us (5.6 TB/s), 64 of 1024 55.2, a tree of 26
// nodes over 2000 cells 16.1.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "fattn_paged.hpp"
#include "runtime.hpp"

namespace {

using namespace paged_fattn;

// ROWT: row tiles of 16 query rows that the waves take side by side (1, 2 or
// 4); the tiles of cells go round the waves of a row tile. CAP: logits
// soft-capped. P: PagedFattnParams, or PagedSeesParams for tokens that see
// other cells than all before them.
template <int ROWT, bool CAP, typename P>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_fattn_kernel(const P p) {
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
    MyPart part;
    if (!find_part(p, wg, p.target, p.long_target, lane, t0, t1, blockIdx.x == 0 && wave == 0, b, part)) return;
    int at = part.at, block = 0, before = 0;
    const int stop = part.stop;

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
        if (threadIdx.x == 0) {
            if (first == 0)
                ap.info[(int64_t) unit * ap.c.n_seq + seq] =
                    int2{wg, whole ? 1 : part.pieces(base, tiles, wg, l64)};
            if (__builtin_expect(w.bad, 0)) paged_error(p.c, raw_len != w.len ? kPagedBadLength : kPagedBadCount, raw_len != w.len ? raw_len : raw_count);
        }
        bool bad = w.bad;
        const Span wave_span = span_of(p, w, wt0, wt1);
        const int seen = wave_span.limit;                          // cells that the wave's last row sees
        int least = max(w.len - w.count + 1 + wt0, 0);             // cells that all its rows see
        // Of a rule: the tiles that the group leaves out, and where the last of
        // the rows' windows begins.
        int gap = 0, gap_at = 0, low_last = 0, first_cells = 0;
        const int begin = w.len - w.count;
        if constexpr (P::kSees) {
            const Span all = span_of(p, w, t0, t1);
            first_cells = p.first;
            gap = all.gap(p);
            gap_at = all.gap_at(p);
            if (has_bits(p)) least = max(begin, 0);
            if constexpr (P::kWindow) low_last = (has_bits(p) ? w.len : begin + 1 + min(wt1, w.count - 1)) - p.window;
        }
        auto tile_at = [&](const int i) { return P::kWindow && i >= gap_at ? i + gap : i; };

        // Pages of a tile's cells: K by lanes n (group n / 4), V by lanes g.
        // Cells past the last group that the wave sees are taken from that one.
        struct Where {
            int k_page, v_page;
            int k_cell, v_cell;                                      // in the page
        };
        const int32_t * table = p.c.table + (int64_t) seq * p.c.t_nb1;
        const uint32_t last_group = (uint32_t) max(seen - 1, 0) / 8;
        auto look_up = [&](const int i) {
            Where a;
            const int tile = tile_at(i);
            uint32_t kg = min((uint32_t) tile * 4 + (n >> 2), last_group), vg = min((uint32_t) tile * 4 + g, last_group);
            if constexpr (P::kWindow) {                                // and those that no window has from the first that one has
                const int low = wave_span.low, from = (p.first + 7) >> 3;
                if ((int) kg >= from) kg = max((int) kg, low >> 3);
                if ((int) vg >= from) vg = max((int) vg, low >> 3);
            }
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
        // its window's beginning, the words of the nodes that it sees
        int low = 0;
        const int32_t * words = nullptr;
        const int32_t * node_pos = nullptr;
        bool bad_row = false;
        if constexpr (P::kSees) {
            int at = begin + t;
            if (has_bits(p)) {
                words = p.bits + (int64_t) seq * p.b_nb2 + (int64_t) (valid ? t : 0) * p.b_nb1;
                if (P::kWindow && p.pos) node_pos = p.pos + (int64_t) seq * p.p_nb1;
                if (node_pos && valid) {
                    at = node_pos[t];
                    bad_row = at < begin || at >= w.len;
                    if (__builtin_expect(bad_row && g == 0, 0)) paged_error(p.c, kPagedBadPos, at);
                }
            }
            if (P::kWindow && valid && !bad_row) low = at + 1 - p.window;
        }
        // Of cells c0 to c0 + 7: those that this lane's row sees.
        auto sees8 = [&](const int c0) {
            if constexpr (!P::kWindow && P::kBits) return upto8(begin - c0) | nodes8(p, words, nullptr, c0 - begin, w.count, 0);
            else if constexpr (P::kSees) {
                if (has_bits(p)) return span8(c0, begin, low, p.first) | nodes8(p, words, node_pos, c0 - begin, w.count, low);
                return span8(c0, limit, low, p.first);
            } else return upto8(limit - c0);
        };
        half8 q_hi[4], q_lo[4];
        float fac, m = -AL_INF, l = 0.0f;
        floatx4 acc[8];
        // Everything that the first tile needs goes out before anything is
        // computed: pages, query rows, then K and V (a wave without a tile
        // loads another wave's and uses none of it).
        const int wave_end = min(end, seen > 0 ? (seen + P::kTile - 1) / P::kTile - gap : 0);
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
        // Whether some row does not see all of a tile.
        auto partly = [&](const int tile) {
            return (tile + 1) * P::kTile > least || (P::kWindow && tile * P::kTile < low_last && (tile + 1) * P::kTile > first_cells);
        };
        // Probabilities of the tile against the rows' running maxima.
        auto softmax = [&](const int tile) {
            const int c0 = tile * P::kTile + 8 * g;
            const bool masked = partly(tile);
            uint32_t sees = 0xffu;
            if constexpr (P::kSees) {
                if (masked) sees = sees8(c0);
            }
            auto hidden = [&](const int i) { return P::kSees ? !(sees >> i & 1) : c0 + i >= limit; };
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
                    if (hidden(i)) x[i] = -AL_INF;
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
                if (masked && hidden(i)) e = 0.0f;
                l += e;
                const _Float16 hi = (_Float16) e;
                p_hi[i] = hi;
                p_lo[i] = (_Float16) (e - (float) hi);
            }
        };
        // (the wave's rows see the same cells)
        const bool one_token = !(has_bits(p)) && wt0 >= min(wt1, w.count - 1);
        // o += P V of the tile. Cells past the wave's last are stale memory:
        // zeroed, as 0 times NaN is not 0. So are, one by one, the values that
        // are not finite of cells that some row does not see; the rows that do
        // see one get NaN in its dim, found by a product of ones.
        auto product = [&](const int tile) {
            const int c0 = tile * P::kTile + 8 * g;
            bool differ = least < seen && (tile + 1) * P::kTile > least;   // (one token: never)
            uint32_t some = 0xffu, all = upto8(least - c0);          // cells that some, that all rows see
            if constexpr (P::kSees) {
                if (partly(tile)) {
                    some = P::kWindow ? span8(c0, seen, wave_span.low, p.first) : upto8(seen - c0);
                    all = P::kWindow ? span8(c0, least, low_last, p.first) : upto8(least - c0);
                    differ = !one_token;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!(some >> i & 1)) v[i] = u32x4{0, 0, 0, 0};
                }
            } else if ((tile + 1) * P::kTile > seen) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 + i >= seen) v[i] = u32x4{0, 0, 0, 0};
            }
            if (__builtin_expect(differ, P::kBits)) {
                uint32_t odd[2] = {0, 0};                            // bit 8 (i % 4) + j of word i / 4: cell i, dim j
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (P::kSees ? (some & ~all) >> i & 1 : c0 + i >= least)
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            if ((v[i][d] & 0x7c00u) == 0x7c00u) odd[i / 4] |= 1u << (8 * (i % 4) + 2 * d), v[i][d] &= 0xffff0000u;
                            if ((v[i][d] & 0x7c000000u) == 0x7c000000u) odd[i / 4] |= 2u << (8 * (i % 4) + 2 * d), v[i][d] &= 0xffffu;
                        }
                }
                if (__any((odd[0] | odd[1]) != 0)) {
                    const uint32_t mine = P::kSees ? sees8(c0) : 0;
                    half8 sees;
#pragma unroll
                    for (int i = 0; i < 8; ++i) sees[i] = (P::kSees ? mine >> i & 1 : c0 + i < limit) ? (_Float16) 1.0f : (_Float16) 0.0f;
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
                softmax(tile_at(tile));
                product(tile_at(tile));
                load_v(next, true);
                next = after;
            }
            scores();
            softmax(tile_at(tile));
            product(tile_at(tile));
        }

        // join the row tile's waves: maxima and sums, then the rescaled outputs
        // through LDS
        const bool any_bad = __any(bad);
        if (__builtin_expect(any_bad && lane == 0 && !w.bad, 0)) paged_error(p.c, kPagedBadPage, seq);
        l = colsum4(l);
        if (any_bad || bad_row) l = __builtin_nanf("");
        if (g == 0) {
            ml_lds[wave][n][0] = m;
            ml_lds[wave][n][1] = l;
        }
        __syncthreads();
        {
            float M = m;
#pragma unroll
            for (int i = 0; i < kCellWaves; ++i) M = fmaxf(M, ml_lds[rt * kCellWaves + i][n][0]);
            const float f = grow<P>(m, M);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *(float4 *) &o_lds[wave][n][8 * (4 * g + i)] = float4{acc[0][i] * f, acc[1][i] * f, acc[2][i] * f, acc[3][i] * f};
                *(float4 *) &o_lds[wave][n][8 * (4 * g + i) + 4] = float4{acc[4][i] * f, acc[5][i] * f, acc[6][i] * f, acc[7][i] * f};
            }
        }
        __syncthreads();
        const auto & ep = arguments<P>();
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
                L += ml_lds[w0 + i][rr][1] * grow<P>(ml_lds[w0 + i][rr][0], M);
#pragma unroll
                for (int d = 0; d < 8; ++d) o[d] += o_lds[w0 + i][rr][dim + d];
            }
            float * d;
            float f = 1.0f;
            if (whole) {
                const int head = h * ep.G + gr - tok * ep.G;
                f = row_factor<P>(ep, w, seq, tok, M, L, head);
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

struct Plan {
    PagedSeesParams p;                                  // (without a rule: its PagedFattnParams)
    bool empty = false;
    bool many = false;                                  // by the kernel of many query rows
    size_t info_bytes = 0, bytes = 0;                   // of the info, of it and the records
};

bool aligned16(const al_tensor & t, int from) {
    for (int i = from; i < 4; ++i)
        if (t.ne[i] > 1 && t.nb[i] % 16) return false;
    return ((uintptr_t) t.data & 15u) == 0;
}

// The rule's operands, checked, in p; *tiles: at most so many of a sequence's
// tiles are seen.
int make_rule(const al_paged_sees * r, PagedSeesParams * p, int64_t T, int64_t n_seq, int64_t tile, int64_t * tiles) {
    if (r->window < 0 || r->first < 0)
        return al_fail(AL_ERR_INVALID, "paged_fattn: a window of %d cells and %d first ones", r->window, r->first);
    // (positions are below 2^30: a longer window is all of them)
    p->window = r->window ? std::min(r->window, 1 << 30) : 1 << 30;
    p->first = r->window ? std::min(r->first, 1 << 30) : 0;
    if (r->bits.data) {
        const al_tensor & b = r->bits;
        if (b.type != AL_TYPE_I32 || b.ne[0] < (T + 31) / 32 || b.ne[1] != T || b.ne[2] != n_seq || b.ne[3] != 1 || b.nb[0] != 4 || b.nb[1] % 4 ||
            b.nb[2] % 4 || ((uintptr_t) b.data & 3u))
            return al_fail(AL_ERR_INVALID, "paged_fattn: bits must be i32 [words, T, n_seq], 32 tokens to a word");
        p->bits = (const int32_t *) b.data; p->b_nb1 = (int64_t) (b.nb[1] / 4); p->b_nb2 = (int64_t) (b.nb[2] / 4);
    }
    if (r->pos.data) {
        const al_tensor & t = r->pos;
        if (!r->bits.data) return al_fail(AL_ERR_INVALID, "paged_fattn: positions without bits");
        if (t.type != AL_TYPE_I32 || t.ne[0] != T || t.ne[1] != n_seq || t.ne[2] != 1 || t.ne[3] != 1 || t.nb[0] != 4 || t.nb[1] % 4 ||
            ((uintptr_t) t.data & 3u))
            return al_fail(AL_ERR_INVALID, "paged_fattn: positions must be i32 [T, n_seq]");
        if (r->window) p->pos = (const int32_t *) t.data, p->p_nb1 = (int64_t) (t.nb[1] / 4);
    } else if (r->bits.data && r->window) {
        return al_fail(AL_ERR_INVALID, "paged_fattn: bits and a window need positions");
    }
    if (r->window)
        *tiles = std::min(*tiles, ((int64_t) p->first + tile - 1) / tile + ((int64_t) p->window + T + tile - 1) / tile + 1);
    return AL_OK;
}

// Whether a call with a rule goes to the kernel of many query rows: for more
// than 64 of a KV head, and for more than 32 of several sequences (us, this
// kernel and that one, trees over 3000 cells of 8 heads: 40 rows of one sequence
// 18.5, 20.0, of 8 37.2, 34.3, 64 rows of one 21.0, 23.1, of 8 42.7, 35.5, of 30
// 113, 81.6, 100 rows of one over 6000 cells 33, 27).
bool many_rows(const PagedFattnParams & p) {
    // (it counts bytes within a page, and from page to page, in 32 bits)
    constexpr int64_t kMost = 0xffffffffll;
    return p.R > (p.c.n_seq > 1 ? 32 : 64) && p.c.page_size * p.c.k_nb1 <= kMost && p.c.page_size * p.c.v_nb1 <= kMost && p.c.k_nb3 <= kMost &&
           p.c.v_nb3 <= kMost;
}

// Whether a call with a rule has so little to do that each row tile of 16 is a
// group of its own, its workgroups' waves side by side over cells: few rounds and
// small records, though the groups load the same cells. By the rows times the
// cells that there can be (the table's, or the window's) for each CU, and by the
// pairs of a group and a sequence, which are one workgroup's at least.
// us, the other choice and so, 32 heads over 8 but where they are of all kinds: for
// the kernel of many rows a tree of 26 nodes over 300 cells 18.9, 12.8, 2000 19.5,
// 16.7, 8000 (26 K a CU) 29.9, 30.6, 4 of 12 over 1500 23.8, 20.5, 40 tokens over a
// window of 1024 23.2, 14.2, 128 (18 K) 28.2, 20.3, 200 (30 K) 34.4, 28.0, a tree of 100
// over 2000 (26 K) 32.8, 29.2, of 50 over 5000 (31 K) 30.4, 34.5, 15 trees of 52 rows over 384 (480 pairs) 22.0, 18.9, 4 of
// 368 over 144 (736) 21.4, 23.3, 14 of 364 over 96 (2576) 26.5, 58; for two and four row
// tiles a tree of 16 over 20000 (39 K) 39.6, 35.6, 10 of 28 rows over 512 17.4, 13.8, 9
// of 21 over 4000 (23 K) 33.7, 37.3, 46 of 32 over 48 (368) 12.5, 14.1.
bool few_row_cells(const PagedFattnParams & p, const al_paged_sees & r, const int n_cu) {
    double cells = (double) p.c.max_pages * p.c.page_size;
    if (r.window > 0) cells = std::min(cells, (double) r.window + std::max(r.first, 0) + p.T);
    const bool many = many_rows(p);
    const double pairs = (double) ((p.R + 15) / 16) * p.Hkv * p.c.n_seq;
    const double most = many ? (p.c.n_seq > 1 ? 16.0 : r.bits.data ? 28.0 : 32.0) : p.c.n_seq > 1 ? 8.0 : 48.0;
    return pairs <= (many ? 2 : 1) * n_cu && cells * p.R * p.Hkv * p.c.n_seq <= most * 1024 * n_cu;
}

int make_plan(const al_paged_fattn_args * a, const al_paged_sees * rule, int n_cu, Plan * out) {
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
    PagedSeesParams & p = pl.p;
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
    const bool few = rule && few_row_cells(p, *rule, n_cu);
    pl.many = rule && !few && many_rows(p);
    p.row_tiles = pl.many ? PagedRowsParams::kRows / 16 : p.R <= 16 || few ? 1 : p.R <= 32 ? 2 : 4;
    const int rows = 16 * p.row_tiles;
    p.row_groups = (p.R + rows - 1) / rows;
    const int64_t units = (int64_t) p.row_groups * Hkv;
    if (units > 65535) return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: sizes out of range");
    const int tile = pl.many ? PagedRowsParams::kTile : PagedFattnParams::kTile;
    const int min_tiles = pl.many ? PagedRowsParams::kMinTiles : PagedFattnParams::kMinTiles;
    int64_t tiles = std::max<int64_t>(1, ((int64_t) p.c.max_pages * p.c.page_size + tile - 1) / tile);
    if (rule) rc = make_rule(rule, &p, T, n_seq, tile, &tiles);
    if (rc != AL_OK) return rc;
    const int64_t most = n_seq * tiles;                                                                                 // tiles there can be
    if (most > INT32_MAX) return al_fail(AL_ERR_UNSUPPORTED, "paged_fattn: sizes out of range");
    // One workgroup a CU, 48 to 64 KB of its waves' loads in flight: more only
    // lengthen the queues (us with one / two / four: 24 sequences to 4000 cells
    // 51.3 / 52.6 / 54.6, 100000 cells of 64 heads 79.4 / 81.7 / 85.7, 8000 cells
    // 13.2 / 14.2 / 13.9). Two where row tiles share the loads (verify of 10
    // sequences 48.5 / 47.1 / 50.0), and for many short sequences, whose ends
    // are not hidden (96 to 300 cells 30.8 / 24.9, 128 to 700 57.2 / 57.2). Row
    // tiles that are groups have one (a tree of 26 nodes over 2000 cells 16.8 / 19.0).
    const int64_t per_cu = n_cu / std::max<int64_t>(1, units);
    const int64_t useful = std::max(n_seq, (most + min_tiles - 1) / min_tiles);
    p.target = (int32_t) std::max<int64_t>(1, std::min<int64_t>(2 * n_cu / std::max<int64_t>(1, units), useful));
    // Where the row groups alone fill the card twice over, a workgroup takes whole
    // sequences, one or some: nothing to join, and many short workgroups rather
    // than a round of long ones and a part of another (us, all of a unit's
    // sequences by one workgroup, and so: two prompts of 1000 over windows of 1024
    // 62.9, 60.1, of 4000 280.0, 279.1).
    p.whole = pl.many && 2 * n_cu <= 2 * units;
    if (p.whole) p.target = (int32_t) std::min<int64_t>(n_seq, std::max<int64_t>(1, 8192 / units));
    p.long_target = p.row_tiles == 1 ? (int32_t) std::max<int64_t>(1, std::min<int64_t>(per_cu, p.target)) : p.target;
    // few sequences have many pieces each
    p.row_waves = p.long_target > 16 * n_seq ? kWaves : 1;
    p.scale = a->scale;
    p.softcap = a->logit_softcap;
    pl.info_bytes = ((size_t) units * n_seq * sizeof(int2) + 255) / 256 * 256;
    pl.bytes = pl.info_bytes + (p.target > 1 && !p.whole ? (size_t) units * p.target * 2 * rows * 130 * 4 : 0);     // one workgroup a unit: no pieces
    *out = pl;
    return AL_OK;
}

template <int ROWT, typename P>
void launch(const P & p, hipStream_t st) {
    const dim3 grid((unsigned) (p.target * p.row_groups * p.Hkv));
    if (p.softcap != 0.0f) hipLaunchKernelGGL((paged_fattn_kernel<ROWT, true, P>), grid, dim3(64 * kWaves), 0, st, p);
    else                   hipLaunchKernelGGL((paged_fattn_kernel<ROWT, false, P>), grid, dim3(64 * kWaves), 0, st, p);
}

template <typename P>
hipError_t launch(const P & p, hipStream_t st) {
    switch (p.row_tiles) {
        case 1: launch<1>(p, st); break;
        case 2: launch<2>(p, st); break;
        default: launch<4>(p, st); break;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_join(p, st) : e;
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

namespace {

bool leaves_nothing_out(const al_paged_sees & r) { return r.window == 0 && r.first >= 0 && !r.bits.data && !r.pos.data; }

uint64_t workspace_bytes(const al_paged_fattn_args * a, const al_paged_sees * rule) {
    if (rule && leaves_nothing_out(*rule)) rule = nullptr;
    int n_cu = 0;
    Plan pl;
    if (al_device_cu_count(&n_cu) != AL_OK || make_plan(a, rule, n_cu, &pl) != AL_OK) return 0;
    return pl.empty ? 0 : al_workspace_bytes(pl.bytes);
}

int attend(const al_paged_fattn_args * a, const al_paged_sees * rule) {
    if (rule && leaves_nothing_out(*rule)) rule = nullptr;
    // the arguments first: refusals need no device
    Plan pl;
    int rc = make_plan(a, rule, 1, &pl);
    if (rc != AL_OK || pl.empty) return rc;
    int n_cu = 0;
    rc = al_device_cu_count(&n_cu);
    if (rc == AL_OK) rc = make_plan(a, rule, n_cu, &pl);
    if (rc == AL_OK) rc = al_device_error_flag(&pl.p.c.err);
    if (rc != AL_OK) return rc;
    rc = al_workspace_records("paged_fattn", pl.bytes, a->workspace, a->workspace_bytes, a->stream, (void **) &pl.p.info);
    if (rc != AL_OK) return rc;
    pl.p.part = (float *) ((char *) pl.p.info + pl.info_bytes);
    const hipStream_t st = (hipStream_t) a->stream;
    hipError_t e;
    if (pl.many) {
        PagedRowsParams p;
        static_cast<PagedSeesParams &>(p) = pl.p;
        p.shared = p.counts && !p.whole && p.target > 1 && p.row_groups > 1 && p.row_groups * ((p.c.n_seq + 63) / 64) <= PagedRowsParams::kShared;
        e = launch_rows(p, st);
    } else if (rule && (!pl.p.bits || !pl.p.pos)) {
        PagedWindowParams w;
        PagedTreeParams t;
        static_cast<PagedSeesParams &>(w) = static_cast<PagedSeesParams &>(t) = pl.p;
        e = pl.p.bits ? launch(t, st) : launch(w, st);
    } else {
        e = rule ? launch(pl.p, st) : launch<PagedFattnParams>(pl.p, st);
    }
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "paged_fattn: launch");
}

}  // namespace

extern "C" uint64_t al_paged_fattn_workspace_bytes(const al_paged_fattn_args * a) { return workspace_bytes(a, nullptr); }

extern "C" int al_paged_fattn_f16(const al_paged_fattn_args * a) { return attend(a, nullptr); }

extern "C" uint64_t al_paged_fattn_sees_workspace_bytes(const al_paged_fattn_args * a, const al_paged_sees * sees) {
    return sees ? workspace_bytes(a, sees) : 0;
}

extern "C" int al_paged_fattn_sees_f16(const al_paged_fattn_args * a, const al_paged_sees * sees) {
    return sees ? attend(a, sees) : al_fail(AL_ERR_INVALID, "paged_fattn: null rule");
}
