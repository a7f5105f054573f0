// Cells of a paged KV cache moved in all layers at once
// (include/arclight_paged.h), for gfx950: those of an accepted path to the
// places behind the sequence's cells, and pages, or their first cells, into
// other pages.
//
// A cell of a layer is Hkv rows of 256 bytes in the K and in the V pool; a
// thread moves 16 bytes of a row at a time, several of them in flight before the
// first is stored. Copied pages are not read again by the launch, so that their
// stores do not stay in the cache (us with ordinary stores, with these: 64 parts
// of pages of 16 cells in 36 layers 38, 29.8, 30 of pages of 64 in 64 layers 109.5,
// 106, 20 of them 76.6, 77.5).
//
// A path's cells move down, path[i] >= i, and may overlap: cell b + i can be the
// source of an earlier entry (path[j] = i, j < i) but of no later one. A thread
// keeps its 16 bytes of the row through all of the path, loads the entries in
// their order and stores a batch of them after its loads, so that an entry's
// place is not written before the entry that comes from there is read.
//
// What bounds them: the moved cells, read once and written once (4.1 TB/s for 20
// parts of pages in 64 layers, 320 MB; 5.4 for 160 MB in 36), and for few the
// chain lengths -> path -> pages -> cells: 40 paths in 36 layers, 25 MB, 7.3 us,
// one 4.9.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/arclight_paged.h"
#include "device_common.hpp"
#include "paged.hpp"
#include "runtime.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8;                       // 16-byte pieces of a path that a thread has in flight
constexpr int kCopyBatch = 4;                   // and of a page
constexpr int kCopyGroups = 4096;               // workgroups that copy pages, if there are so many pieces
constexpr int kPath = 64;                       // entries of a path looked up together
constexpr int kLayers = 64;                     // layers of a launch: pointers among its arguments

struct LayerPools {
    char * k[kLayers];
    char * v[kLayers];
};

struct KeepParams {
    PagedPools c;                               // (of a layer: without k and v)
    const int32_t * lens;
    const int32_t * counts;                     // or null
    const int32_t * path;  int64_t p_nb1;       // sequence, in entries
    const int32_t * kept;
    int32_t * lens_out;                         // or null
    int32_t T, Hkv;
    LayerPools layers;
};

struct CopyParams {
    PagedPools c;
    const int32_t * src;
    const int32_t * dst;
    const int32_t * cells;                      // or null
    int32_t Hkv, blocks;                        // workgroups of a page in one pool, which take its pieces in turn
    int32_t heads_first;                        // a head's cells lie closer than a cell's heads
    LayerPools layers;
};

// A layer's pool, by a scalar load from the arguments.
template <typename P>
__device__ __forceinline__ char * layer_pool(const int layer, const bool v) {
    auto a = (const __attribute__((address_space(4))) P *) __builtin_amdgcn_kernarg_segment_ptr();
    return v ? a->layers.v[layer] : a->layers.k[layer];
}

// Grid: pieces of a cell (those of K, then those of V), layers, sequences.
__global__ __launch_bounds__(kThreads) void paged_keep_kernel(const KeepParams p) {
    __shared__ int2 s_src[kPath], s_dst[kPath];                          // page, cell in it; page -1: nothing to move
    const int s = blockIdx.z, tid = threadIdx.x;
    const int len = p.lens[s], count = p.counts ? p.counts[s] : p.T, kept = p.kept[s];
    const bool len_ok = len >= 0 && len <= p.c.max_pages * p.c.page_size;
    const bool count_ok = count >= 0 && count <= p.T && count <= len, kept_ok = kept >= 0 && kept <= count;
    const bool first = blockIdx.x == 0 && blockIdx.y == 0;
    if (first && tid == 0) {
        if (!len_ok || !count_ok || !kept_ok)
            paged_error(p.c, !len_ok ? kPagedBadLength : !count_ok ? kPagedBadCount : kPagedBadKept, !len_ok ? len : !count_ok ? count : kept);
        if (p.lens_out) p.lens_out[s] = len_ok && count_ok && kept_ok ? len - count + kept : len;
    }
    if (!len_ok || !count_ok || !kept_ok) return;
    const int begin = len - count, units = p.Hkv * 16;
    const int unit = blockIdx.x * kThreads + tid;
    const bool v = unit >= units, mine = unit < 2 * units;
    const int head = (v ? unit - units : unit) >> 4;
    const int64_t nb1 = v ? p.c.v_nb1 : p.c.k_nb1, nb3 = v ? p.c.v_nb3 : p.c.k_nb3;
    const int layer = blockIdx.y;
    char * k_pool = layer_pool<KeepParams>(layer, false);
    char * v_pool = layer_pool<KeepParams>(layer, true);
    char * base = (v ? v_pool : k_pool) + head * (v ? p.c.v_nb2 : p.c.k_nb2) + (unit & 15) * 16;
    for (int i0 = 0; i0 < kept; i0 += kPath) {
        if (i0) __syncthreads();
        const int n = min(kPath, kept - i0);
        if (tid < kPath) {
            const int i = i0 + tid;
            int2 from = {-1, 0}, to = {-1, 0};
            if (tid < n) {
                const int at = p.path[(int64_t) s * p.p_nb1 + i];
                const bool ok = at >= i && at < count;
                if (!ok && first) paged_error(p.c, kPagedBadPath, at);
                if (ok && at != i) {
                    const int32_t * table = p.c.table + (int64_t) s * p.c.t_nb1;
                    const int a = begin + at, b = begin + i;
                    const int pa = (int) page_of_group(p.c, (uint32_t) a / 8), pb = (int) page_of_group(p.c, (uint32_t) b / 8);
                    from = {table[pa], a - pa * p.c.page_size};
                    to = {table[pb], b - pb * p.c.page_size};
                    if ((uint32_t) from.x >= (uint32_t) p.c.n_pages || (uint32_t) to.x >= (uint32_t) p.c.n_pages) {
                        if (first) paged_error(p.c, kPagedBadPage, s);
                        from = {-1, 0};
                    }
                }
            }
            s_src[tid] = from;
            s_dst[tid] = to;
        }
        __syncthreads();
        if (!mine) continue;
        for (int i = 0; i < n; i += kBatch) {
            u32x4 x[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {                           // (entries behind the path: page -1 too)
                const int2 a = s_src[i + j];
                x[j] = *(const u32x4 *) (base + max(a.x, 0) * nb3 + a.y * nb1);
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int2 b = s_dst[i + j];
                if (s_src[i + j].x >= 0) *(u32x4 *) (base + b.x * nb3 + b.y * nb1) = x[j];
            }
        }
    }
}

// Grid: workgroups of a page (those of K, then those of V), layers, pairs.
__global__ __launch_bounds__(kThreads) void paged_copy_kernel(const CopyParams p) {
    const int i = blockIdx.z, tid = threadIdx.x;
    const int src = p.src[i], dst = p.dst[i], cells = p.cells ? p.cells[i] : p.c.page_size;
    if (src < 0 || dst < 0) return;
    const bool pages_ok = src < p.c.n_pages && dst < p.c.n_pages, cells_ok = cells >= 0 && cells <= p.c.page_size;
    if (!pages_ok || !cells_ok) {
        if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0)
            paged_error(p.c, !pages_ok ? kPagedBadCopy : kPagedBadCells, !pages_ok ? max(src, dst) : cells);
        return;
    }
    const bool v = (int) blockIdx.x >= p.blocks;
    const int units = cells * p.Hkv * 16;
    if (src == dst) return;
    const int64_t nb1 = v ? p.c.v_nb1 : p.c.k_nb1, nb2 = v ? p.c.v_nb2 : p.c.k_nb2, nb3 = v ? p.c.v_nb3 : p.c.k_nb3;
    char * pool = layer_pool<CopyParams>(blockIdx.y, v);
    const char * from = pool + src * nb3;
    char * to = pool + dst * nb3;
    const uint32_t inner = p.heads_first ? cells : p.Hkv;
    constexpr int kStep = kThreads * kCopyBatch;
    for (int at = ((int) blockIdx.x - (v ? p.blocks : 0)) * kStep + tid; at < units; at += p.blocks * kStep) {
        u32x4 x[kCopyBatch];
        int64_t off[kCopyBatch];
#pragma unroll
        for (int j = 0; j < kCopyBatch; ++j) {
            const uint32_t u = min(at + j * kThreads, units - 1), row = u >> 4, o = row / inner, in = row - o * inner;
            off[j] = (p.heads_first ? in : o) * nb1 + (p.heads_first ? o : in) * nb2 + (u & 15) * 16;
            x[j] = *(const u32x4 *) (from + off[j]);
        }
#pragma unroll
        for (int j = 0; j < kCopyBatch; ++j)
            if (at + j * kThreads < units) __builtin_nontemporal_store(x[j], (u32x4 *) (to + off[j]));
    }
}

bool index(const al_tensor & t, const int64_t n) {
    return t.data && t.type == AL_TYPE_I32 && t.ne[0] == n && t.ne[1] == 1 && t.ne[2] == 1 && t.ne[3] == 1 && t.nb[0] == 4 &&
           ((uintptr_t) t.data & 3u) == 0;
}

// The pools' shape, by a table that only stands for one.
int layer_pools(const char * what, const al_paged_layers & l, const al_tensor * table, PagedPools * out) {
    if (l.n_layers < 1 || l.n_layers > 65535 || !l.k || !l.v) return al_fail(AL_ERR_INVALID, "%s: %d layers", what, l.n_layers);
    for (int i = 0; i < l.n_layers; ++i)
        if (!l.k[i] || !l.v[i] || (((uintptr_t) l.k[i] | (uintptr_t) l.v[i]) & 15u))
            return al_fail(AL_ERR_INVALID, "%s: the pools of layer %d must be 16-byte aligned", what, i);
    al_tensor k = l.k_pool, v = l.v_pool, none;
    k.data = l.k[0];
    v.data = l.v[0];
    if (!table) {
        memset(&none, 0, sizeof(none));
        none.data = k.data;
        none.type = AL_TYPE_I32;
        none.ne[0] = none.ne[2] = none.ne[3] = 1;
        none.nb[0] = none.nb[1] = 4;
        table = &none;
    }
    return paged_pools(what, &k, &v, table, out);
}

// The launches of `enqueue`, of up to kLayers layers each.
template <typename P, typename F>
int for_layers(const char * what, const al_paged_layers & l, P & p, F && enqueue) {
    for (int l0 = 0; l0 < l.n_layers; l0 += kLayers) {
        const int n = std::min(kLayers, l.n_layers - l0);
        for (int i = 0; i < n; ++i) {
            p.layers.k[i] = (char *) l.k[l0 + i];
            p.layers.v[i] = (char *) l.v[l0 + i];
        }
        enqueue(n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return al_hip_fail(e, what);
    }
    return AL_OK;
}

bool overlap(const void * a, size_t a_bytes, const void * b, size_t b_bytes) {
    return (const char *) a < (const char *) b + b_bytes && (const char *) b < (const char *) a + a_bytes;
}

}  // namespace

extern "C" int al_paged_keep_f16(const al_paged_keep_args * a) {
    if (!a) return al_fail(AL_ERR_INVALID, "paged_keep: null arguments");
    KeepParams p;
    memset(&p, 0, sizeof(p));
    int rc = layer_pools("paged_keep", a->layers, &a->table, &p.c);
    if (rc != AL_OK) return rc;
    const int64_t n_seq = p.c.n_seq, T = a->path.ne[0];
    const al_tensor & t = a->path;
    if (!t.data || t.type != AL_TYPE_I32 || T < 0 || t.ne[1] != n_seq || t.ne[2] != 1 || t.ne[3] != 1 || t.nb[0] != 4 || t.nb[1] % 4 ||
        ((uintptr_t) t.data & 3u))
        return al_fail(AL_ERR_INVALID, "paged_keep: the path must be i32 [T, n_seq] of the table's %d sequences", p.c.n_seq);
    if (!index(a->lens, n_seq) || !index(a->kept, n_seq) || (a->counts.data && !index(a->counts, n_seq)) ||
        (a->lens_out.data && !index(a->lens_out, n_seq)))
        return al_fail(AL_ERR_INVALID, "paged_keep: lens, counts, kept and lens_out must be i32 [n_seq]");
    if (T > (1 << 16) || n_seq > 65535) return al_fail(AL_ERR_UNSUPPORTED, "paged_keep: sizes out of range");
    const size_t bytes = (size_t) n_seq * 4;
    if (n_seq == 0) return AL_OK;
    if (a->lens_out.data) {
        bool bad = false;
        for (const al_tensor * x : {&a->lens, &a->kept, &a->counts}) bad |= x->data && overlap(a->lens_out.data, bytes, x->data, bytes);
        for (const al_tensor * x : {&a->path, &a->table})
            bad |= overlap(a->lens_out.data, bytes, x->data, (size_t) (n_seq - 1) * x->nb[1] + (size_t) x->ne[0] * 4);
        if (bad) return al_fail(AL_ERR_INVALID, "paged_keep: lens_out overlaps an operand");
    }
    p.lens = (const int32_t *) a->lens.data;
    p.counts = (const int32_t *) a->counts.data;
    p.path = (const int32_t *) t.data; p.p_nb1 = (int64_t) (t.nb[1] / 4);
    p.kept = (const int32_t *) a->kept.data;
    p.lens_out = (int32_t *) a->lens_out.data;
    p.T = (int32_t) T; p.Hkv = (int32_t) a->layers.k_pool.ne[2];
    rc = al_device_error_flag(&p.c.err);
    if (rc != AL_OK) return rc;
    return for_layers("paged_keep: launch", a->layers, p, [&](const int n) {
        const dim3 grid((unsigned) ((2 * p.Hkv * 16 + kThreads - 1) / kThreads), (unsigned) n, (unsigned) n_seq);
        hipLaunchKernelGGL(paged_keep_kernel, grid, dim3(kThreads), 0, (hipStream_t) a->stream, p);
        p.lens_out = nullptr;                                            // once
    });
}

extern "C" int al_paged_copy_f16(const al_paged_copy_args * a) {
    if (!a) return al_fail(AL_ERR_INVALID, "paged_copy: null arguments");
    CopyParams p;
    memset(&p, 0, sizeof(p));
    int rc = layer_pools("paged_copy", a->layers, nullptr, &p.c);
    if (rc != AL_OK) return rc;
    const int64_t n = a->src.ne[0];
    if (n < 0 || !index(a->src, n) || !index(a->dst, n) || (a->cells.data && !index(a->cells, n)))
        return al_fail(AL_ERR_INVALID, "paged_copy: src, dst and cells must be i32 [n]");
    p.Hkv = (int32_t) a->layers.k_pool.ne[2];
    const int64_t units = (int64_t) p.c.page_size * p.Hkv * 16;
    if (n > 65535 || units > (1 << 30)) return al_fail(AL_ERR_UNSUPPORTED, "paged_copy: sizes out of range");
    if (n == 0) return AL_OK;
    p.src = (const int32_t *) a->src.data;
    p.dst = (const int32_t *) a->dst.data;
    p.cells = (const int32_t *) a->cells.data;
    const int64_t most = (units + kThreads * kCopyBatch - 1) / (kThreads * kCopyBatch), launched = 2 * n * std::min(kLayers, a->layers.n_layers);
    p.blocks = (int32_t) std::max<int64_t>(1, std::min(most, (kCopyGroups + launched - 1) / launched));
    p.heads_first = p.c.k_nb1 < p.c.k_nb2;
    rc = al_device_error_flag(&p.c.err);
    if (rc != AL_OK) return rc;
    return for_layers("paged_copy: launch", a->layers, p, [&](const int layers) {
        const dim3 grid((unsigned) (2 * p.blocks), (unsigned) layers, (unsigned) n);
        hipLaunchKernelGGL(paged_copy_kernel, grid, dim3(kThreads), 0, (hipStream_t) a->stream, p);
    });
}
