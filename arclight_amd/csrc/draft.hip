// Trees of drafted tokens (include/arclight_draft.h), for gfx950: positions,
// cells and the bits of what each node sees from the parents, and verification
// against the target's probabilities.
//
// Tree. A wave takes 64 nodes of a tree, a lane each, which goes up its parents
// in LDS: the steps are its depth, and as a parent's number is smaller the words
// of its bits come one after another from the last to the first.
//
// Verification. Accept and reject take a few numbers of each node (its
// parent's p and q at its token), gathered by a workgroup into LDS; the walk down
// the tree is then ballots over the nodes. The token that follows is drawn from
// one row of V: the row's weights are summed in 64 bits by waves, kChunk tokens
// each, and a last workgroup for each sequence finds the chunk in which the sum
// passes sample times the whole, and the token in it. Every sum is taken in one
// fixed order, so that equal inputs give equal tokens.
//
// Where several children of a node were drawn from a draft's row, what is left
// after each rejection has to be normalised before the next child is tried: a
// sum over the row within the walk, which a workgroup for each sequence then
// does in a launch of its own. It keeps what is left of the row in memory from one
// rejection to the next, as a node's rejections cost their square if each begins
// from the row again.
//
// What bounds them: chains of loads. The tables of one tree of 26 nodes or of 50
// of up to 200 take 3.7 us, a launch and two loads in series. Verification is two
// launches, count and nodes -> their p -> the row -> its sums, and sums -> the
// chunk: one tree of 26 nodes over 32003 tokens 9.5 us, 30 chains with a draft's
// rows of 128000 (31 MB) 13.9, 20 trees of 40 nodes over 152000 (12 MB) 14.0. Trees
// with a draft's rows are bound by the slowest sequence's rejections one after another,
// 34 us and more each at 128000 tokens: 8 trees of 40 nodes 105 us, 30 of 26 251.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/arclight_draft.h"
#include "device_errors.hpp"
#include "kernel_args.hpp"
#include "overlap.hpp"
#include "runtime.hpp"

namespace {

constexpr int kMaxNodes = 1024;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 8;                        // a lane's tokens of a chunk
constexpr int kChunk = 64 * kEach;              // tokens that a wave sums

typedef double pair64 __attribute__((ext_vector_type(2)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void draft_error(int * err, const int what, const int value) {
    if (atomicCAS(err + kErrDraft, 0, 1) == 0) {
        err[kErrDraft + 1] = what;
        err[kErrDraft + 2] = value;
    }
}

struct TreeParams {
    const int32_t * parents;  int64_t par_nb1;  // sequence, in entries
    const int32_t * lens;
    const int32_t * counts;                     // or null
    int32_t * pos;    int64_t pos_nb1;          // each or null
    int32_t * cells;  int64_t cells_nb1;
    int32_t * seq;    int64_t seq_nb1;
    int32_t * bits;   int64_t b_nb1, b_nb2;
    int32_t T, words;
    int * err;
};

// Grid: 64 nodes, sequences.
__global__ __launch_bounds__(64) void draft_tree_kernel(const TreeParams p) {
    __shared__ int32_t par[kMaxNodes];
    prefetch_params(p);
    const int s = blockIdx.y, lane = threadIdx.x, t = blockIdx.x * 64 + lane;
    const int len = p.lens[s], raw = p.counts ? p.counts[s] : p.T;
    const bool ok = raw >= 0 && raw <= p.T && raw <= len;
    const int count = ok ? raw : 0;
    if (!ok && t == 0) draft_error(p.err, kDraftBadCount, raw);
    const int last = min((int) blockIdx.x * 64 + 63, count - 1);         // no lane comes past it
    for (int u = lane; u <= last; u += 64) {
        int x = p.parents[(int64_t) s * p.par_nb1 + u];
        if (x >= u) {
            if (u == t) draft_error(p.err, kDraftBadParent, x);
            x = -1;
        }
        par[u] = x;
    }
    __syncthreads();
    if (t >= p.T) return;
    int depth = -1;
    int32_t * words = p.bits + (int64_t) s * p.b_nb2 + (int64_t) t * p.b_nb1;
    int w = p.words - 1;
    uint32_t word = 0;
    if (t < count)
        for (int u = t; u >= 0; u = par[u], ++depth) {
            if (p.bits)
                for (; w > u >> 5; --w, word = 0) words[w] = (int32_t) word;
            word |= 1u << (u & 31);
        }
    if (p.bits)
        for (; w >= 0; --w, word = 0) words[w] = (int32_t) word;
    if (p.pos) p.pos[(int64_t) s * p.pos_nb1 + t] = t < count ? len - count + depth : 0;
    if (p.cells) p.cells[(int64_t) s * p.cells_nb1 + t] = t < count ? len - count + t : 0;
    if (p.seq) p.seq[(int64_t) s * p.seq_nb1 + t] = t < count ? s : -1;
}

struct VerifyParams {
    const char * target;  int64_t t_nb1, t_nb2; // node, sequence, in bytes
    const char * draft;   int64_t d_nb1, d_nb2; // or null
    const int32_t * tokens;   int64_t tok_nb1;  // sequence, in entries
    const int32_t * parents;  int64_t par_nb1;  // or null
    const int32_t * counts;                     // or null
    const float * accept;     int64_t acc_nb1;
    const float * sample;
    int32_t * path;           int64_t path_nb1;
    int32_t * kept;
    int32_t * next;
    int2 * state;                               // [sequence]: the last accepted node (-1: none), its rejected children
    double * rest;                              // [sequence][V]: of three siblings of a draft and more, what all rejections but the last left
    double * norm;                              // [sequence]: of two and more, its sum
    pair64 * sums;                             // [sequence][chunk]: of what is left, of the row itself
    int32_t T, V, chunks, walked;               // walked: state, rest and norm are there
    int * err;
};

__device__ __forceinline__ float weight(const float x) { return x > 0.0f ? x : 0.0f; }

// Sums of the workgroup's lanes, in a fixed order; every thread gets them.
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i);
    return x;
}
__device__ __forceinline__ double block_sum(double x, double * lds) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) x += lds[i];
    return x;
}

// What is left of a token's p, q in the draft's row, by two rejections of children
// drawn from it. norm: the sum of what the first left of all.
__device__ __forceinline__ double left_by_one(const double p, const double q) { return fmax(p - q, 0.0); }
__device__ __forceinline__ double left_by_two(const double p, const double q, const double norm) { return fmax(left_by_one(p, q) / norm - q, 0.0); }

// Rejection m of a child of node v drawn from its row q, by a workgroup: the sum of
// what it leaves of p, which every thread gets, and from the second on that itself,
// before it is normalised, to p.rest. norm: the sum of what rejection m - 1 left. M:
// 1, 2, or 3 for all behind. A thread's tokens are its own in all rejections; others
// read them behind block_sum's barriers.
template <int M>
__device__ __forceinline__ double reject(const VerifyParams & p, const int s, const int v, const double norm, double * lds) {
    constexpr int kHeld = 8;                                             // a thread's loads in flight, of each row
    const float * pr = (const float *) (p.target + (int64_t) s * p.t_nb2 + (int64_t) v * p.t_nb1);
    const float * qr = (const float *) (p.draft + (int64_t) s * p.d_nb2 + (int64_t) v * p.d_nb1);
    double * rest = p.rest + (int64_t) s * p.V;
    double sum = 0.0;
    for (int y0 = threadIdx.x; y0 < p.V; y0 += kThreads * kHeld) {
        double f[kHeld];
        float q[kHeld];
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int y = min(y0 + j * kThreads, p.V - 1);
            f[j] = M < 3 ? (double) weight(pr[y]) : rest[y];
            q[j] = weight(qr[y]);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (y0 + j * kThreads < p.V) {
                const double left = M == 1 ? left_by_one(f[j], q[j]) : M == 2 ? left_by_two(f[j], q[j], norm) : fmax(f[j] / norm - q[j], 0.0);
                if (M > 1) rest[y0 + j * kThreads] = left;
                sum += left;
            }
    }
    return block_sum(sum, lds);
}

struct WalkLds {
    int32_t par[kMaxNodes];                     // -1: nobody's child
    int32_t tok[kMaxNodes];
    float p[kMaxNodes], q[kMaxNodes], r[kMaxNodes];
    int32_t path[kMaxNodes];
    double red[kWaves];
};

struct Walked {
    int v, m;                                   // as VerifyParams::state
    int kept;
};

__device__ __forceinline__ int nodes_of(const VerifyParams & p, const int s, const bool report) {
    const int raw = p.counts ? p.counts[s] : p.T;
    const bool ok = raw >= 0 && raw <= p.T;
    if (!ok && report) draft_error(p.err, kDraftBadCount, raw);
    return ok ? raw : 0;
}

// The parent of node u, -1 where it is nobody's child; up: as it was given.
__device__ __forceinline__ int valid_parent(const VerifyParams & p, const int u, const int up, const int token) {
    return up < u && (uint32_t) token < (uint32_t) p.V ? max(up, -1) : -1;
}
__device__ __forceinline__ int parent_of(const VerifyParams & p, const int s, const int u, const int token) {
    return valid_parent(p, u, p.parents ? p.parents[(int64_t) s * p.par_nb1 + u] : u - 1, token);
}

// The walk down the tree, by every wave of a workgroup alike. NORMS: with a
// draft whose nodes can have several children.
template <bool NORMS>
__device__ __forceinline__ Walked walk(const VerifyParams & p, const int s, const int count, const bool report, WalkLds & x) {
    const int tid = threadIdx.x, lane = tid & 63;
    const char * target = p.target + (int64_t) s * p.t_nb2;
    const char * draft = p.draft ? p.draft + (int64_t) s * p.d_nb2 : nullptr;
    // (all T places are read, so that nothing waits for the count)
    for (int u = tid; u < p.T; u += kThreads) {
        const float r = p.accept[(int64_t) s * p.acc_nb1 + u];
        const int tok = u ? p.tokens[(int64_t) s * p.tok_nb1 + u] : 0;
        const int up = p.parents ? p.parents[(int64_t) s * p.par_nb1 + u] : u - 1;
        const int par = valid_parent(p, u, up, tok);
        float pu = 0.0f, qu = 1.0f;
        if (par >= 0) {
            pu = *(const float *) (target + (int64_t) par * p.t_nb1 + (int64_t) tok * 4);
            if (draft) qu = *(const float *) (draft + (int64_t) par * p.d_nb1 + (int64_t) tok * 4);
        }
        if (report && u < count && up >= 0 && par < 0) draft_error(p.err, up >= u ? kDraftBadParent : kDraftBadToken, up >= u ? up : tok);
        x.par[u] = par;
        x.tok[u] = tok;
        x.r[u] = r;
        x.p[u] = weight(pu);
        x.q[u] = weight(qu);
    }
    __syncthreads();
    Walked at = {count > 0 ? 0 : -1, 0, count > 0};
    if (tid == 0) x.path[0] = 0;
    double norm = 1.0;                                                   // of the last row that was left
    while (at.v >= 0) {
        // the children of v in their order
        double mass = 1.0;
        bool nothing = false;
        int m = 0, found = -1, first = -1;
        for (int base = (at.v + 1) & ~63; base < count && found < 0; base += 64) {
            const int u = base + lane;
            uint64_t todo = __ballot(u > at.v && u < count && x.par[min(u, count - 1)] == at.v);
            for (; todo && found < 0; todo &= todo - 1) {
                const int c = base + __builtin_ctzll(todo), tok = x.tok[c];
                if (first < 0) first = c;
                bool pass;
                if (!p.draft) {
                    // a token that was rejected already has nothing left
                    bool twice = false;
                    for (int b = first & ~63; m > 0 && b < c; b += 64) {
                        const int e = b + lane;
                        twice |= __any(e >= first && e < c && x.par[min(e, count - 1)] == at.v && x.tok[min(e, count - 1)] == tok);
                    }
                    const double pc = x.p[c];
                    pass = !twice && pc > 0.0 && (double) x.r[c] * mass < pc;
                    if (!pass && !twice) mass -= pc;
                } else {
                    double pc = x.p[c];
                    const double qc = x.q[c];
                    if (NORMS && m > 0) {
                        // what the last rejection left, and its sum
                        if (!nothing) {
                            norm = m == 1 ? reject<1>(p, s, at.v, norm, x.red) : m == 2 ? reject<2>(p, s, at.v, norm, x.red) : reject<3>(p, s, at.v, norm, x.red);
                            nothing = !(norm > 0.0 && norm < __builtin_inf());
                        }
                        pc = nothing ? 0.0 : (m == 1 ? left_by_one(pc, qc) : p.rest[(int64_t) s * p.V + tok]) / norm;
                        __syncthreads();                                 // (all have read it: the next rejection writes there)
                    }
                    pass = pc > 0.0 && (double) x.r[c] * qc < pc;
                }
                if (pass) found = c;
                else ++m;
            }
        }
        if (found < 0) {
            at.m = nothing ? 0 : m;
            if (NORMS && tid == 0) p.norm[s] = norm;
            break;
        }
        at.v = found;
        if (tid == 0) x.path[at.kept] = found;
        ++at.kept;
    }
    __syncthreads();
    return at;
}

__device__ __forceinline__ void write_path(const VerifyParams & p, const int s, const Walked & at, const WalkLds & x) {
    for (int i = threadIdx.x; i < p.T; i += kThreads) p.path[(int64_t) s * p.path_nb1 + i] = i < at.kept ? x.path[i] : -1;
    if (threadIdx.x == 0) {
        p.kept[s] = at.kept;
        p.state[s] = int2{at.v, at.m};
    }
}

__global__ __launch_bounds__(kThreads) void verify_walk_kernel(const VerifyParams p) {
    __shared__ WalkLds x;
    const int s = blockIdx.x;
    const int count = nodes_of(p, s, threadIdx.x == 0);
    const Walked at = walk<true>(p, s, count, true, x);
    write_path(p, s, at, x);
}

// A thread's tokens of the last accepted node's rows, as they are: 0 past the
// last one.
struct Row {
    float p[kEach], q[kEach];
};
__device__ __forceinline__ Row load_row(const VerifyParams & p, const int s, const Walked & at, const int first) {
    Row x;
    const bool drafted = p.draft && at.m > 0;
    const char * pr = p.target + (int64_t) s * p.t_nb2 + (int64_t) at.v * p.t_nb1 + (int64_t) first * 4;
    const char * qr = p.draft + (int64_t) s * p.d_nb2 + (int64_t) at.v * p.d_nb1 + (int64_t) first * 4;
#pragma unroll
    for (int j = 0; j < kEach; ++j) x.p[j] = x.q[j] = 0.0f;
    if (first + kEach <= p.V) {
#pragma unroll
        for (int j = 0; j < kEach; j += 4) {
            const float4u y = *(const float4u *) (pr + 4 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) x.p[j + e] = y[e];
        }
        if (drafted) {
#pragma unroll
            for (int j = 0; j < kEach; j += 4) {
                const float4u y = *(const float4u *) (qr + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.q[j + e] = y[e];
            }
        }
    } else if (first < p.V) {
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (first + j < p.V) {
                x.p[j] = *(const float *) (pr + 4 * j);
                if (drafted) x.q[j] = *(const float *) (qr + 4 * j);
            }
    }
    return x;
}

// What is left of them, and they themselves. first: the first of them; gone: the
// tokens of the chunk that were rejected, a bit each.
__device__ __forceinline__ void row_weights(const VerifyParams & p, const int s, const Walked & at, const Row & x, const int first, const uint32_t * gone,
                                            double (&left)[kEach], double (&own)[kEach]) {
    const bool drafted = p.draft && at.m > 0;
    const int lane = threadIdx.x & 63;
    const uint32_t out = p.draft ? 0u : gone[lane * kEach / 32] >> (lane * kEach % 32);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        own[j] = weight(x.p[j]);
        left[j] = drafted ? left_by_one(own[j], weight(x.q[j])) : out >> j & 1 ? 0.0 : own[j];
    }
    if (drafted && at.m > 1) {
        const double * rest = p.rest + (int64_t) s * p.V, norm = p.norm[s];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const double q = weight(x.q[j]);
            left[j] = at.m == 2 ? left_by_two(own[j], q, norm) : first + j < p.V ? fmax(rest[first + j] / norm - q, 0.0) : 0.0;
        }
    }
}

// Waits for this wave's LDS accesses, and keeps those after it behind them.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The tokens of a chunk that the last accepted node's children had, without a
// draft, by one wave.
__device__ __forceinline__ void rejected(const WalkLds & x, const Walked & at, const int count, const int chunk, uint32_t * gone) {
    const int lane = threadIdx.x & 63;
    wave_lds();
    if (lane < kChunk / 32) gone[lane] = 0;
    wave_lds();
    for (int u = at.v + 1 + lane; u < count; u += 64)
        if (x.par[u] == at.v && x.tok[u] / kChunk == chunk) atomicOr(gone + x.tok[u] % kChunk / 32, 1u << (x.tok[u] % 32));
    wave_lds();
}

// Grid: workgroups of a sequence, sequences. A wave takes the chunks that follow
// its number in steps of all of the sequence's waves, each loaded while the one
// before is summed.
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyParams p) {
    __shared__ WalkLds x;
    __shared__ uint32_t gone[kWaves][kChunk / 32];
    prefetch_params(p);
    const int s = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool first = blockIdx.x == 0;
    Walked at;
    int count = 0;
    if (p.walked) {
        const int2 st = p.state[s];
        at = {st.x, st.y, 0};
    } else {
        count = nodes_of(p, s, first && threadIdx.x == 0);
        at = walk<false>(p, s, count, first, x);
        if (first) write_path(p, s, at, x);
    }
    if (at.v < 0) return;
    const int step = gridDim.x * kWaves;
    int chunk = blockIdx.x * kWaves + wave;
    Row row = load_row(p, s, at, chunk * kChunk + lane * kEach);
    for (; chunk < p.chunks; chunk += step) {
        const Row next = load_row(p, s, at, (chunk + step) * kChunk + lane * kEach);
        if (!p.draft) rejected(x, at, count, chunk, gone[wave]);         // (the walk was this workgroup's own)
        double left[kEach], own[kEach], a = 0.0, b = 0.0;
        row_weights(p, s, at, row, chunk * kChunk + lane * kEach, gone[wave], left, own);
#pragma unroll
        for (int j = 0; j < kEach; ++j) a += left[j], b += own[j];
        a = wave_sum(a);
        b = wave_sum(b);
        if (lane == 0) p.sums[(int64_t) s * p.chunks + chunk] = pair64{a, b};
        row = next;
    }
}

// Sums of the workgroup's pairs before this thread's, and of all.
__device__ __forceinline__ pair64 block_before(const pair64 v, pair64 & all, pair64 * lds) {
    double a = v.x, b = v.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const double oa = __shfl_up(a, i), ob = __shfl_up(b, i);
        if (lane >= i) a += oa, b += ob;
    }
    pair64 before = {__shfl_up(a, 1), __shfl_up(b, 1)};
    if (lane == 0) before = pair64{0.0, 0.0};
    __syncthreads();
    if (lane == 63) lds[wave] = pair64{a, b};
    __syncthreads();
    pair64 from = {0.0, 0.0};
    all = pair64{0.0, 0.0};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) from = all;
        all.x += lds[i].x;
        all.y += lds[i].y;
    }
    return pair64{from.x + before.x, from.y + before.y};
}

// Grid: sequences. What does not depend on the state is loaded with it; one
// load, of the chunk, follows. (Nothing is gathered by atomics on one word: 256
// of them took 4.4 us.)
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(const VerifyParams p) {
    __shared__ pair64 lds[kWaves];
    __shared__ uint32_t gone[kChunk / 32];
    __shared__ int s_hit[kWaves], s_last[kWaves];
    __shared__ double s_hit_before[kWaves], s_last_before[kWaves];
    prefetch_params(p);
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the chunks: each thread some that follow one another, the first kHeld of
    // them at once
    constexpr int kHeld = 4;
    const pair64 * sums = p.sums + (int64_t) s * p.chunks;
    const int each = (p.chunks + kThreads - 1) / kThreads, c0 = min(tid * each, p.chunks), c1 = min(c0 + each, p.chunks);
    pair64 held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = sums[min(c0 + i, p.chunks - 1)];
    const float u = p.sample[s];
    const int2 st = p.state[s];
    // the node of this thread (of trees of up to kThreads)
    const bool node = !p.draft && tid < p.T && tid > 0;
    const int tok = node ? p.tokens[(int64_t) s * p.tok_nb1 + tid] : 0;
    const int par = node ? parent_of(p, s, tid, tok) : -1;
    const int count = nodes_of(p, s, false);
    if (tid < kChunk / 32) gone[tid] = 0;
    const Walked at = {st.x, st.y, 0};
    if (at.v < 0) {
        if (tid == 0) p.next[s] = -1;
        return;
    }
    auto sum_of = [&](const int c) {
        const int i = c - c0;
        return i == 0 ? held[0] : i == 1 ? held[1] : i == 2 ? held[2] : i == 3 ? held[3] : sums[c];
    };
    pair64 part = {0.0, 0.0}, whole;
    for (int c = c0; c < c1; ++c) part += sum_of(c);
    const pair64 ahead = block_before(part, whole, lds);
    // where nothing is left the row itself
    const bool own = !(whole.x > 0.0);
    const double total = own ? whole.y : whole.x;
    double before = own ? ahead.y : ahead.x;
    if (!(total > 0.0 && total < __builtin_inf())) {
        if (tid == 0) {
            draft_error(p.err, kDraftBadRow, s);
            p.next[s] = -1;
        }
        return;
    }
    const double goal = (double) u * total;
    // the first chunk that goes past the goal; else the last that holds any
    {
        int hit = -1, last = -1;
        double hit_before = 0.0, last_before = 0.0;
        for (int c = c0; c < c1; ++c) {
            const pair64 x = sum_of(c);
            const double w = own ? x.y : x.x;
            if (w > 0.0) {
                last = c;
                last_before = before;
                if (hit < 0 && before + w > goal) hit = c, hit_before = before;
            }
            before += w;
        }
        const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
        if (hits ? lane == __builtin_ctzll(hits) : lane == 0) s_hit[wave] = hit, s_hit_before[wave] = hit_before;
        if (lasts ? lane == 63 - __builtin_clzll(lasts) : lane == 0) s_last[wave] = last, s_last_before[wave] = last_before;
    }
    __syncthreads();
    int chunk = -1, last_chunk = -1;
    double from = 0.0, last_from = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (chunk < 0 && s_hit[i] >= 0) chunk = s_hit[i], from = s_hit_before[i];
        if (s_last[i] >= 0) last_chunk = s_last[i], last_from = s_last_before[i];
    }
    if (chunk < 0) chunk = last_chunk, from = last_from;
    // the token in it: by the first wave, once the rejected ones are known
    Row row;
    const int first = chunk * kChunk + lane * kEach;
    if (wave == 0) row = load_row(p, s, at, first);
    if (tid < count && par == at.v && tok / kChunk == chunk) atomicOr(gone + tok % kChunk / 32, 1u << (tok % 32));
    if (!p.draft)
        for (int v = kThreads + tid; v < count; v += kThreads) {
            const int x = p.tokens[(int64_t) s * p.tok_nb1 + v];
            if (parent_of(p, s, v, x) == at.v && x / kChunk == chunk) atomicOr(gone + x % kChunk / 32, 1u << (x % 32));
        }
    __syncthreads();
    if (wave) return;
    double left[kEach], weights[kEach], sum = 0.0;
    row_weights(p, s, at, row, first, gone, left, weights);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        if (own) left[j] = weights[j];
        sum += left[j];
    }
    double upto = sum;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const double o = __shfl_up(upto, i);
        if (lane >= i) upto += o;
    }
    double run = __shfl_up(upto, 1);
    run = from + (lane == 0 ? 0.0 : run);
    int hit = -1, last = -1;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        run += left[j];
        if (left[j] > 0.0) {
            last = first + j;
            if (hit < 0 && run > goal) hit = first + j;
        }
    }
    const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
    if (hits) {
        if (lane == __builtin_ctzll(hits)) p.next[s] = hit;
    } else if (lasts && lane == 63 - __builtin_clzll(lasts)) {
        p.next[s] = last;
    }
}

bool index(const al_tensor & t, const int64_t n) {
    return t.data && t.type == AL_TYPE_I32 && t.ne[0] == n && t.ne[1] == 1 && t.ne[2] == 1 && t.ne[3] == 1 && t.nb[0] == 4 &&
           ((uintptr_t) t.data & 3u) == 0;
}

// [T, n_seq] of 32-bit values
bool nodes(const al_tensor & t, const int type, const int64_t T, const int64_t n) {
    return t.data && t.type == type && t.ne[0] == T && t.ne[1] == n && t.ne[2] == 1 && t.ne[3] == 1 && t.nb[0] == 4 && t.nb[1] % 4 == 0 &&
           ((uintptr_t) t.data & 3u) == 0;
}

int64_t entries(const uint64_t bytes) { return (int64_t) (bytes / 4); }

struct VerifyPlan {
    VerifyParams p;
    int64_t n_seq = 0;
    size_t norm_at = 0, rest_at = 0, sums_at = 0, bytes = 0;
};

int make_plan(const al_draft_verify_args * a, VerifyPlan * out) {
    if (!a) return al_fail(AL_ERR_INVALID, "draft_verify: null arguments");
    const al_tensor & t = a->target;
    if (!t.data) return al_fail(AL_ERR_INVALID, "draft_verify: target is required");
    const int64_t V = t.ne[0], T = t.ne[1], n = t.ne[2];
    auto rows = [&](const al_tensor & x) {
        return x.type == AL_TYPE_F32 && x.ne[0] == V && x.ne[1] == T && x.ne[2] == n && x.ne[3] == 1 && x.nb[0] == 4 && x.nb[1] % 4 == 0 &&
               x.nb[2] % 4 == 0 && ((uintptr_t) x.data & 3u) == 0;
    };
    if (V < 1 || T < 0 || n < 0 || !rows(t) || (a->draft.data && !rows(a->draft)))
        return al_fail(AL_ERR_INVALID, "draft_verify: target and draft must be f32 [V, T, n_seq]");
    if (!nodes(a->tokens, AL_TYPE_I32, T, n) || !nodes(a->path, AL_TYPE_I32, T, n) || !nodes(a->accept, AL_TYPE_F32, T, n) ||
        (a->parents.data && !nodes(a->parents, AL_TYPE_I32, T, n)))
        return al_fail(AL_ERR_INVALID, "draft_verify: tokens, parents and path must be i32 [T, n_seq], accept f32 [T, n_seq]");
    al_tensor u = a->sample;
    if (u.type != AL_TYPE_F32) return al_fail(AL_ERR_INVALID, "draft_verify: sample must be f32 [n_seq]");
    u.type = AL_TYPE_I32;
    if (!index(u, n) || !index(a->kept, n) || !index(a->next, n) || (a->counts.data && !index(a->counts, n)))
        return al_fail(AL_ERR_INVALID, "draft_verify: sample, counts, kept and next must be [n_seq], i32 but for sample");
    if (V > (1 << 24) || T > kMaxNodes || n > 65535) return al_fail(AL_ERR_UNSUPPORTED, "draft_verify: sizes out of range");
    if (outputs_overlap({&a->path, &a->kept, &a->next, &a->target, &a->draft, &a->tokens, &a->parents, &a->counts, &a->accept, &a->sample}, 3))
        return al_fail(AL_ERR_INVALID, "draft_verify: path, kept and next may not be another operand's memory");
    VerifyPlan pl;
    VerifyParams & p = pl.p;
    memset(&p, 0, sizeof(p));
    p.target = (const char *) t.data; p.t_nb1 = (int64_t) t.nb[1]; p.t_nb2 = (int64_t) t.nb[2];
    p.draft = (const char *) a->draft.data; p.d_nb1 = (int64_t) a->draft.nb[1]; p.d_nb2 = (int64_t) a->draft.nb[2];
    p.tokens = (const int32_t *) a->tokens.data; p.tok_nb1 = entries(a->tokens.nb[1]);
    p.parents = (const int32_t *) a->parents.data; p.par_nb1 = entries(a->parents.nb[1]);
    p.counts = (const int32_t *) a->counts.data;
    p.accept = (const float *) a->accept.data; p.acc_nb1 = entries(a->accept.nb[1]);
    p.sample = (const float *) a->sample.data;
    p.path = (int32_t *) a->path.data; p.path_nb1 = entries(a->path.nb[1]);
    p.kept = (int32_t *) a->kept.data;
    p.next = (int32_t *) a->next.data;
    p.T = (int32_t) T; p.V = (int32_t) V;
    p.chunks = (int32_t) ((V + kChunk - 1) / kChunk);
    // only siblings of a draft's tokens need sums within the walk
    p.walked = p.draft && p.parents && T > 2;
    pl.n_seq = n;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    pl.norm_at = up((size_t) n * sizeof(int2));
    pl.rest_at = pl.norm_at + (p.walked ? up((size_t) n * sizeof(double)) : 0);
    pl.sums_at = pl.rest_at + (p.walked ? up((size_t) n * V * sizeof(double)) : 0);
    pl.bytes = pl.sums_at + (size_t) n * p.chunks * sizeof(pair64);
    *out = pl;
    return AL_OK;
}

}  // namespace

extern "C" int al_draft_tree_i32(const al_draft_tree_args * a) {
    if (!a) return al_fail(AL_ERR_INVALID, "draft_tree: null arguments");
    const int64_t T = a->parents.ne[0], n = a->parents.ne[1];
    if (T < 0 || n < 0 || !nodes(a->parents, AL_TYPE_I32, T, n)) return al_fail(AL_ERR_INVALID, "draft_tree: parents must be i32 [T, n_seq]");
    if (!index(a->lens, n) || (a->counts.data && !index(a->counts, n)))
        return al_fail(AL_ERR_INVALID, "draft_tree: lens and counts must be i32 [n_seq]");
    for (const al_tensor * t : {&a->pos, &a->cells, &a->seq})
        if (t->data && !nodes(*t, AL_TYPE_I32, T, n)) return al_fail(AL_ERR_INVALID, "draft_tree: pos, cells and seq must be i32 [T, n_seq]");
    const al_tensor & b = a->bits;
    if (b.data && (b.type != AL_TYPE_I32 || b.ne[0] < (T + 31) / 32 || b.ne[1] != T || b.ne[2] != n || b.ne[3] != 1 || b.nb[0] != 4 || b.nb[1] % 4 ||
                   b.nb[2] % 4 || ((uintptr_t) b.data & 3u)))
        return al_fail(AL_ERR_INVALID, "draft_tree: bits must be i32 [words, T, n_seq], 32 nodes to a word");
    if (T > kMaxNodes || n > 65535 || (b.data && b.ne[0] > (1 << 16))) return al_fail(AL_ERR_UNSUPPORTED, "draft_tree: sizes out of range");
    if (outputs_overlap({&a->pos, &a->cells, &a->seq, &a->bits, &a->parents, &a->lens, &a->counts}, 4))
        return al_fail(AL_ERR_INVALID, "draft_tree: pos, cells, seq and bits may not be another operand's memory");
    if (T == 0 || n == 0) return AL_OK;
    TreeParams p;
    memset(&p, 0, sizeof(p));
    p.parents = (const int32_t *) a->parents.data; p.par_nb1 = entries(a->parents.nb[1]);
    p.lens = (const int32_t *) a->lens.data;
    p.counts = (const int32_t *) a->counts.data;
    p.pos = (int32_t *) a->pos.data; p.pos_nb1 = entries(a->pos.nb[1]);
    p.cells = (int32_t *) a->cells.data; p.cells_nb1 = entries(a->cells.nb[1]);
    p.seq = (int32_t *) a->seq.data; p.seq_nb1 = entries(a->seq.nb[1]);
    p.bits = (int32_t *) b.data; p.b_nb1 = entries(b.nb[1]); p.b_nb2 = entries(b.nb[2]);
    p.T = (int32_t) T;
    p.words = b.data ? (int32_t) b.ne[0] : 0;
    const int rc = al_device_error_flag(&p.err);
    if (rc != AL_OK) return rc;
    const dim3 grid((unsigned) ((T + 63) / 64), (unsigned) n);
    hipLaunchKernelGGL(draft_tree_kernel, grid, dim3(64), 0, (hipStream_t) a->stream, p);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "draft_tree: launch");
}

extern "C" uint64_t al_draft_verify_workspace_bytes(const al_draft_verify_args * a) {
    VerifyPlan pl;
    return make_plan(a, &pl) != AL_OK || pl.n_seq == 0 ? 0 : al_workspace_bytes(pl.bytes);
}

extern "C" int al_draft_verify_f32(const al_draft_verify_args * a) {
    VerifyPlan pl;
    int rc = make_plan(a, &pl);
    if (rc != AL_OK || pl.n_seq == 0) return rc;
    VerifyParams & p = pl.p;
    int n_cu = 0;
    rc = al_device_cu_count(&n_cu);
    if (rc == AL_OK) rc = al_device_error_flag(&p.err);
    if (rc != AL_OK) return rc;
    char * at = nullptr;
    rc = al_workspace_records("draft_verify", pl.bytes, a->workspace, a->workspace_bytes, a->stream, (void **) &at);
    if (rc != AL_OK) return rc;
    p.state = (int2 *) at;
    p.norm = (double *) (at + pl.norm_at);
    p.rest = (double *) (at + pl.rest_at);
    p.sums = (pair64 *) (at + pl.sums_at);
    const hipStream_t st = (hipStream_t) a->stream;
    const unsigned n = (unsigned) pl.n_seq;
    hipError_t e = hipSuccess;
    if (p.walked) {
        hipLaunchKernelGGL(verify_walk_kernel, dim3(n), dim3(kThreads), 0, st, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess) {
        // four workgroups a CU walk the tree, and take the chunks between them
        const unsigned side = (unsigned) std::max<int64_t>(1, std::min<int64_t>((p.chunks + kWaves - 1) / kWaves, 4ll * n_cu / n));
        hipLaunchKernelGGL(verify_sums_kernel, dim3(side, n), dim3(kThreads), 0, st, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess) {
        hipLaunchKernelGGL(verify_pick_kernel, dim3(n), dim3(kThreads), 0, st, p);
        e = hipGetLastError();
    }
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "draft_verify: launch");
}
