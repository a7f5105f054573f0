// Device code shared by the kernels of attention over a paged cache
// (fattn_paged.hip, fattn_paged_rows.hip): what a token sees, how the tiles of
// all sequences are shared out, and the join of a sequence's pieces.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/arclight_paged.h"
#include "device_common.hpp"
#include "kernel_args.hpp"
#include "paged.hpp"

namespace paged_fattn {

constexpr int kWaves = 4;
constexpr float kLog2e = 1.44269504088896341f;
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

    static constexpr bool kSees = false;                // a rule beside the lengths
    static constexpr bool kBits = false;                // it may have bits,
    static constexpr bool kWindow = false;              // or a window
    static constexpr bool kLog2 = false;                // maxima in log2 units, weights unscaled
    static constexpr int kTile = 32;                    // cells of a tile, the units that work is shared out in
    static constexpr int kMinTiles = 4;                 // least tiles of a part: one for each wave
    static constexpr int kWhole = 16;                   // sequences of up to so many tiles are not cut
};

// The same with a rule for what a token sees (al_paged_sees).
struct PagedSeesParams : PagedFattnParams {
    int32_t window, first;                              // no window: 2^30, which no cell lies before
    const int32_t * bits;  int64_t b_nb1, b_nb2;        // or null; token, sequence, in words
    const int32_t * pos;   int64_t p_nb1;               // or null; sequence (with bits and a window)
    int32_t whole;                                      // sequences are not cut, however long
    static constexpr int kPiece = 16;                   // tiles that a workgroup could do instead of beginning a second piece
    static constexpr bool kSees = true;
    static constexpr bool kBits = true;
    static constexpr bool kWindow = true;
};

// Windows alone, and trees alone: a launch begins with an empty instruction
// cache, and code that a call steps over costs it too (us with the code of both,
// with one's own: one token over a window of 1024 11.5, 10.1, 10 sequences of 6
// 25.9, 24.7, a tree of 26 nodes over 2000 cells 20.1, 19.5, of 10 over 3000 18.9,
// 17.9).
struct PagedWindowParams : PagedSeesParams {
    static constexpr bool kBits = false;
};
struct PagedTreeParams : PagedSeesParams {
    static constexpr bool kWindow = false;
};

// The same for the kernel of many query rows (fattn_paged_rows.hip).
struct PagedRowsParams : PagedSeesParams {
    static constexpr bool kLog2 = true;
    static constexpr int kTile = 64;
    // (us with parts of 1, 2, 3, 4 tiles at least: a tree of 26 nodes over 2000
    // cells 23.1, 21.9, 20.4, 22.0, 2 prompts of 40 over windows of 1024 29.1,
    // 27.8, 24.8, 32.4, one of 500 30.6, 29.6, 29.1, 26.6)
    static constexpr int kMinTiles = 3;
    static constexpr int kWhole = 8;
    static constexpr int kPiece = 8;
    static constexpr int kRows = 128;                   // of a group
    static constexpr int kShared = 8;                   // row groups times blocks of 64 sequences whose tiles are counted
    int32_t shared;                                     // a head's workgroups go to its row groups by their tiles
};
struct PagedRowsWindowParams : PagedRowsParams {
    static constexpr bool kBits = false;
};
struct PagedRowsTreeParams : PagedRowsParams {
    static constexpr bool kWindow = false;
};
hipError_t launch_rows(const PagedRowsParams & p, hipStream_t stream);

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

template <typename A>
__device__ __forceinline__ int token_of(const A & p, const int r) {
    return p.G == 1 ? r : (int) __umulhi((uint32_t) r, p.g_magic);
}

// Whether the call's rule has bits (a constant for kernels without).
template <typename P>
__device__ __forceinline__ bool has_bits(const P & p) {
    if constexpr (P::kBits) return p.bits != nullptr;
    else return false;
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

template <typename P>
__device__ __forceinline__ SeqWork seq_work(const P & p, const int len, const int count) {
    SeqWork w;
    w.len = min(max(len, 0), p.c.max_pages * p.c.page_size);
    w.count = min(max(count, 0), p.T);
    w.bad = len != w.len || count != w.count;
    return w;
}

// The cells that tokens t0 to t1 of a sequence see, as a whole: those before
// `limit` (-1: there are no such tokens), but none from p.first to `low`.
struct Span {
    int limit, low;
    // Tiles without such a cell, and the first of them.
    template <typename P>
    __device__ __forceinline__ int gap_at(const P & p) const { return (min(p.first, low) + P::kTile - 1) / P::kTile; }
    template <typename P>
    __device__ __forceinline__ int gap(const P & p) const { return P::kWindow ? max(low / P::kTile - gap_at(p), 0) : 0; }
};

template <typename P>
__device__ __forceinline__ Span span_of(const P & p, const SeqWork & w, const int t0, const int t1) {
    Span a = {w.limit(t0, t1), 0};
    if constexpr (P::kSees) {
        const bool bits = has_bits(p);
        if (bits && a.limit >= 0) a.limit = w.len;                     // of nodes each may see any
        if constexpr (P::kWindow) a.low = min(max(w.len - w.count + (bits ? 0 : t0) + 1 - p.window, 0), max(a.limit - 1, 0));
    }
    return a;
}

// Tiles of a sequence in the row of all tiles: one at least, so that rows that
// see nothing are written too.
template <typename P>
__device__ __forceinline__ int tiles_of(const P & p, const Span a) {
    int gap = 0;
    if constexpr (P::kSees) gap = a.gap(p);
    return a.limit < 0 ? 0 : max(1, (a.limit + P::kTile - 1) / P::kTile - gap);
}

// The first k of 8 cells, a bit each.
__device__ __forceinline__ uint32_t upto8(const int k) { return (1u << min(max(k, 0), 8)) - 1; }
// Of cells c0 to c0 + 7: those before `limit` that are not from `first` to `low`.
__device__ __forceinline__ uint32_t span8(const int c0, const int limit, const int low, const int first) {
    return upto8(limit - c0) & (~upto8(low - c0) | upto8(first - c0));
}

// Of nodes u0 to u0 + 7 (u0 may be negative) those that a token sees, whose
// words are `words`, among the sequence's first `count`.
__device__ __forceinline__ uint32_t nodes8(const int32_t * words, const int u0, const int count) {
    if (u0 <= -8 || u0 >= count) return 0;
    const int u = max(u0, 0), i = u >> 5, last = (count - 1) >> 5;
    const uint64_t two = (uint32_t) words[i] | (uint64_t) (uint32_t) words[min(i + 1, last)] << 32;
    return (uint32_t) (two >> (u & 31)) << (u - u0) & upto8(count - u0);
}

// The same, without those that lie before the token's window and are not among
// the first cells either; pos: the nodes' positions.
template <typename A>
__device__ __forceinline__ uint32_t nodes8(const A & p, const int32_t * words, const int32_t * pos, const int u0, const int count,
                                           const int low) {
    uint32_t m = nodes8(words, u0, count);
    if (pos)
        for (uint32_t rest = m; rest; rest &= rest - 1) {
            const int at = pos[u0 + __builtin_ctz(rest)];
            if (at < low && at >= p.first) m &= ~(rest & -rest);
        }
    return m;
}

// Whether token t of sequence s sees a cell at all.
template <typename P, typename A>
__device__ __forceinline__ bool sees_any(const A & p, const SeqWork & w, const int s, const int t) {
    const int begin = w.len - w.count;
    if constexpr (P::kBits) {
        if (p.bits) {
            const int32_t * words = p.bits + (int64_t) s * p.b_nb2 + (int64_t) t * p.b_nb1;
            const int32_t * pos = P::kWindow && p.pos ? p.pos + (int64_t) s * p.p_nb1 : nullptr;
            const int low = pos ? pos[t] + 1 - p.window : 0;
            if (begin > 0 && (begin > low || p.first > 0)) return true;
            for (int u = max(-begin, 0); u < w.count; u += 8)
                if (nodes8(p, words, pos, u, w.count, low)) return true;
            return false;
        }
    }
    return begin + 1 + t > 0;
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
    template <typename P>
    __device__ __forceinline__ void load(const P & p, const int b, const int lane, const int t0, const int t1) {
        const int s = 64 * b + lane;
        const bool in = s < p.c.n_seq;
        len = in ? p.lens[s] : 0;
        count = !in ? 0 : p.counts ? p.counts[s] : p.T;
        tiles = in ? tiles_of(p, span_of(p, seq_work(p, len, count), t0, t1)) : 0;
        upto = wave_scan(tiles);
    }
    // A negative count makes an empty slot, which no workgroup comes to.
    __device__ __forceinline__ void report(const PagedFattnParams & p) const {
        if (__builtin_expect(count < 0, 0)) paged_error(p.c, kPagedBadCount, count);
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

template <typename A>
__device__ __forceinline__ char * record(const A & p, const int unit, const int wg, const int slot) {
    return (char *) p.part + (((int64_t) unit * p.target + wg) * 2 + slot) * (16 * p.row_tiles) * 130 * 4;
}

// e^(a - b) for running maxima a <= b, 1 where they are equal (both -inf too).
template <typename P>
__device__ __forceinline__ float grow(const float a, const float b) {
    return a == b ? 1.0f : P::kLog2 ? __builtin_amdgcn_exp2f(a - b) : exp_fast(a - b);
}

// Factor of a row's sums, with the sink as one more logit without a value: 0
// for a row that sees nothing, NaN where all logits are -inf.
// a: the arguments, of type P.
template <typename P, typename A>
__device__ __forceinline__ float row_factor(const A & a, const SeqWork & w, const int s, const int t, const float M, float L,
                                            const int head) {
    float up = P::kLog2 ? 1.0f : 1.0f / kPScale;
    L *= up;
    if (a.sinks) {
        const float sink = P::kLog2 ? a.sinks[head] * kLog2e : a.sinks[head], top = fmaxf(M, sink);
        const float e = grow<P>(M, top);
        up *= e;
        L = L * e + (sink == -AL_INF ? 0.0f : grow<P>(sink, top));
    }
    return L == 0.0f ? sees_any<P>(a, w, s, t) ? __builtin_nanf("") : 0.0f : up / L;
}

// The kernel's arguments as memory, to be loaded where they are used: held in
// scalar registers from the start, those that only a piece's beginning and end
// use displace what the loop over the cells needs.
template <typename P>
__device__ __forceinline__ const __attribute__((address_space(4))) P & arguments() {
    auto a = (const __attribute__((address_space(4))) P *) __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return *a;
}

// A workgroup's part of all tiles of a unit: the tiles from `at` to `stop`.
struct MyPart {
    Parts parts{0, 1};
    int at, stop;
    bool apart = false;                         // each sequence has workgroups of its own
    int each = 0;                               // then: those of this lane's
    // Pieces of a sequence of `tiles` tiles from `base` on, lane l's, that is not
    // whole and whose first one is workgroup wg's.
    __device__ __forceinline__ int pieces(const int base, const int tiles, const int wg, const int l) const {
        return apart ? min(tiles, __builtin_amdgcn_readlane(each, l)) : parts.of(base + tiles - 1) - wg + 1;
    }
};

// Finds it, false if there is none; b: sequences 0 to 63. report: record counts
// that are wrong. t0, t1: the group's first and last token; target, long_target:
// the unit's workgroups, and those that long sequences use.
template <typename P>
__device__ __forceinline__ bool find_part(const P & p, const int wg, const int target, const int long_target, const int lane, const int t0, const int t1,
                                          const bool report, Block & b, MyPart & m) {
    const int n_blocks = (p.c.n_seq + 63) / 64;
    b.load(p, 0, lane, t0, t1);
    if (report) b.report(p);
    int S = b.total(), active = b.active(), longest = b.longest();
    // (said to be unlikely, this loop leaves the kernels 20 bytes of private memory)
    for (int i = 1; i < n_blocks; ++i) {
        Block x;
        x.load(p, i, lane, t0, t1);
        if (report) x.report(p);
        S += x.total();
        active += x.active();
        longest = max(longest, x.longest());
    }
    // Several sequences of up to kWhole tiles each are left whole, one or some to
    // a workgroup: equal parts cut them at places of their own, and a second
    // piece costs a workgroup more than the rounds that the cut saves (us, cut
    // and whole: 4 sequences of up to 200 cells 13.4, 10.1, 64 of 100 16.4, 11.5,
    // 10 of 500 14.1, 12.3; whole up to 32 tiles: 128 of 700 56.4, 60.2). Else
    // kMinTiles a workgroup at least, or a sequence; `target` workgroups for
    // sequences of up to 16 tiles on average, `long_target` for longer ones.
    bool cut = longest > P::kWhole || active == 1;
    if constexpr (P::kSees) {
        // Nor are sequences cut that are about as long as one another, as those
        // are that a window is shorter than, where one each is what the card
        // holds (us, cut and whole: 30 windows of 4096 94.8, 90.3, 64 of 1024
        // 63.6, 55.2, 29 of 1000 33.0, 29.3; where it holds more, 40 of 2048 71.9,
        // 81.6, 33 of 4096 104, 135).
        auto fills = [&](const int places) { return active <= places && 10 * active >= 9 * places; };
        const bool even = (int64_t) longest * active * 8 <= (int64_t) S * 9;
        cut &= !p.whole && !(even && (fills(long_target) || fills(target)));
    }
    const int W = cut ? min(S > 16 * active ? long_target : target, max((S + P::kMinTiles - 1) / P::kMinTiles, active)) : min(target, active);
    if constexpr (P::kSees) {
        // Else each sequence has workgroups of its own, by its tiles, where equal
        // parts of them all are not shorter by more than what a second piece costs
        // (us, equal parts of all and so: 8 windows of 1024 16.3, 14.3, 5 of 600
        // 14.2, 11.8, 20 of 1024 22.4, 21.5, 10 of 6 tokens 22.9, 20.4, 4 of 6 17.8,
        // 14.1, 8 trees of 8 nodes over up to 3000 cells 29.6, 25.7, 3 of 12 over 1000
        // 19.0, 14.6, 12 of 30 over 2000 45.5, 41.5; 12 windows of 2048 25.1, 25.7).
        if (cut && active > 1 && n_blocks == 1) {
            m.each = b.tiles > 0 ? max((int) ((float) b.tiles * (float) W / (float) S), 1) : 0;
            const int upto = wave_scan(m.each);
            if (__builtin_amdgcn_readlane(upto, 63) <= W && !__any(b.tiles > m.each * (S / W + P::kPiece))) {
                m.apart = true;
                const uint64_t mask = __ballot(wg < upto);
                if (!mask) return false;
                const int l = __builtin_ctzll(mask), n = __builtin_amdgcn_readlane(b.tiles, l), k = __builtin_amdgcn_readlane(m.each, l);
                const int base = __builtin_amdgcn_readlane(b.upto, l) - n, j = wg - (__builtin_amdgcn_readlane(upto, l) - k);
                const Parts own(n, k);
                m.at = base + own.begin(j);
                m.stop = base + own.begin(j + 1);
                return m.at < m.stop;
            }
        }
    }
    if (wg >= W) return false;
    m.parts = Parts(S, W);
    m.at = m.parts.begin(wg);
    m.stop = m.parts.begin(wg + 1);
    if (__builtin_expect(!cut, 0)) {
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
        m.at = tile_of(seqs.begin(wg));
        m.stop = tile_of(seqs.begin(wg + 1));
    }
    return true;
}

// A row of the group, joined from the pieces of a sequence that has several.
// p.row_waves waves (1 or kWaves) take it, the halves of a wave every second
// piece, 4 dims to a lane; all loads of 8 of a half's pieces are in flight
// together.
template <typename P>
__device__ __forceinline__ void join_row(const P & p, const int2 info, const int unit, const int seq, const int count,
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
            const float f = grow<P>(M, top);
            L *= f; o.x *= f; o.y *= f; o.z *= f; o.w *= f;
            M = top;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i0 + 2 * i + half < info.y) {
                    const float e = grow<P>(ml[i].x, M);
                    L += ml[i].y * e;
                    o.x += x[i].x * e; o.y += x[i].y * e; o.z += x[i].z * e; o.w += x[i].w * e;
                }
        }
    }
    // the wave's halves, then the row's waves
    {
        const float M2 = __shfl_xor(M, 32), L2 = __shfl_xor(L, 32);
        const float4 o2 = {__shfl_xor(o.x, 32), __shfl_xor(o.y, 32), __shfl_xor(o.z, 32), __shfl_xor(o.w, 32)};
        const float top = fmaxf(M, M2), f = grow<P>(M, top), f2 = grow<P>(M2, top);
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
            const float f = grow<P>(o_lds[i][128], top);
            const float4 x = *(const float4 *) &o_lds[i][4 * d4];
            L += o_lds[i][129] * f;
            o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
        }
        M = top;
    }
    if (!mine || half) return;
    const int head = h * p.G + gr - t * p.G;
    const SeqWork w = seq_work(p, p.lens[seq], count);
    const float f = row_factor<P>(p, w, seq, t, M, L, head);
    *(float4 *) ((float *) (p.dst + (int64_t) seq * p.d_nb3 + (int64_t) t * p.d_nb2 + (int64_t) head * p.d_nb1) + 4 * d4) =
        float4{o.x * f, o.y * f, o.z * f, o.w * f};
}

// Workgroups (rows, sequence, unit); few of them where most have nothing to join.
template <typename P>
__global__ __launch_bounds__(64 * kWaves) void paged_join_kernel(const P p) {
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

// Enqueues the join of what a launch of p.target workgroups a unit left.
template <typename P>
hipError_t launch_join(const P & p, hipStream_t st) {
    if (p.target == 1) return hipSuccess;                              // one workgroup a unit: no pieces
    const int rows = std::min(16 * p.row_tiles, p.R);
    // (all rows side by side: 98 sequences of one tile, 56 rows, 24.6 us in all instead of 20.7)
    const int64_t pairs = (int64_t) p.c.n_seq * p.row_groups * p.Hkv;
    const int side = (int) std::max<int64_t>(1, std::min<int64_t>((rows + kWaves - 1) / kWaves, 2048 / pairs));
    const dim3 grid((unsigned) (p.row_waves == 1 ? side : rows), (unsigned) p.c.n_seq, (unsigned) (p.row_groups * p.Hkv));
    hipLaunchKernelGGL((paged_join_kernel<P>), grid, dim3(64 * kWaves), 0, st, p);
    return hipGetLastError();
}

}  // namespace paged_fattn
