// Appending a batch's keys and values to a paged KV cache, queries alongside
// (include/arclight_paged.h), for gfx950.
//
// Mathematics: per row of 128, optionally x / sqrt(mean x^2 + eps) * w, then
// pair i rotated by the angle pos * base^(-2 i / 128) (taken as i float
// products), by the code of the ring's producers, so that a cache can be
// filled by either; keys and values rounded to f16 (to nearest even).
//
// One wavefront takes 8 heads of one token, 8 lanes to a row, as those
// producers do: lane j of 8 holds dims 4j .. 4j + 3 of each 32, so that the
// wave's loads and stores cover whole 128-byte lines, and the rotation's 64
// (cos, sin) pairs are computed once for the 8 rows. The page of the token's
// cell is looked up while its row is loaded.
//
// What bounds it: for many tokens memory (everything is read and written
// once), for few the chain position -> angle (63 products in series) -> sine
// -> rows. Measured with norms: 40 tokens of 32 + 8 heads 4.2 us, 8192 of 64 + 8
// 118 us, 5.4 TB/s.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/arclight_paged.h"
#include "kernel_args.hpp"
#include "norm_rope.hpp"
#include "paged.hpp"
#include "runtime.hpp"

namespace {

constexpr int kRows = 8;                         // rows of a wave: heads of one token
constexpr int kWaves = 4;                        // waves of a workgroup: tokens

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

struct AppendParams {
    PagedPools c;
    const char * q;  int64_t q_nb1, q_nb2;       // head, token
    const char * k;  int64_t k_nb1, k_nb2;
    const char * v;  int64_t v_nb1, v_nb2;
    const float * q_w;
    const float * k_w;
    char * q_out;    int64_t o_nb1, o_nb2;
    const int32_t * pos;
    const int32_t * seq;
    const int32_t * cells;                       // or null: pos
    int32_t T, Hq, Hkv, norm;
    int32_t yq, yk;                              // blocks of 8 heads of q, of k (and v)
    float eps;
    RopeConsts rope;
};

// Cell of token t, or -1 when it has none that can be written.
__device__ __forceinline__ int64_t cell_of(const PagedPools & c, const int s, const int pos, const bool report, const bool own_cell, int & page) {
    const bool seq_ok = s < c.n_seq;
    const bool pos_ok = pos >= 0 && pos < c.max_pages * c.page_size;
    int pg = -1, at = 0;
    if (seq_ok && pos_ok) {
        const uint32_t i = page_of_group(c, (uint32_t) pos / 8);
        at = pos - (int) i * c.page_size;
        pg = c.table[(int64_t) s * c.t_nb1 + i];
    }
    const bool ok = (uint32_t) pg < (uint32_t) c.n_pages;
    if (!ok && report) paged_error(c, !seq_ok ? kPagedBadSeq : !pos_ok ? (own_cell ? kPagedBadCell : kPagedBadPos) : kPagedBadPage, !seq_ok ? s : !pos_ok ? pos : s);
    page = pg;
    return ok ? at : -1;
}

// blockIdx.y < yq: 8 query heads, then yk blocks of 8 key heads, then as many
// of values.
template <int MODE>
__global__ __launch_bounds__(64 * kWaves) void paged_append_kernel(const AppendParams p) {
    __shared__ __attribute__((aligned(16))) float2 rot[kWaves][64];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, l8 = lane & 7;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kWaves + wave;
    if (t >= p.T) return;
    const int by = blockIdx.y;
    const int kind = by < p.yq ? 0 : by < p.yq + p.yk ? 1 : 2;          // q, k, v
    const int H = kind == 0 ? p.Hq : p.Hkv;
    const int h = (by - (kind == 0 ? 0 : kind == 1 ? p.yq : p.yq + p.yk)) * kRows + (lane >> 3);
    const char * src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const int64_t nb1 = kind == 0 ? p.q_nb1 : kind == 1 ? p.k_nb1 : p.v_nb1;
    const int64_t nb2 = kind == 0 ? p.q_nb2 : kind == 1 ? p.k_nb2 : p.v_nb2;
    const float * xr = (const float *) (src + (int64_t) min(h, H - 1) * nb1 + (int64_t) t * nb2);
    float4u x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = *(const float4u *) (xr + 32 * j + 4 * l8);
    const int s = p.seq[t], pos = p.pos[t];
    if (s < 0) return;                                                   // wave-uniform: a row of no sequence
    int page = 0;
    int64_t cell = 0;
    if (kind != 0) cell = cell_of(p.c, s, p.cells ? p.cells[t] : pos, lane == 0 && h == 0, p.cells != nullptr, page);

    if (kind != 2) {
        float lo[8], hi[8], wl[8], wh[8];
        float2 cs[8];
        const float * w = kind == 0 ? p.q_w : p.k_w;
        float4u ww[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ww[j] = w ? *(const float4u *) (w + 32 * j + 4 * l8) : float4u{1.0f, 1.0f, 1.0f, 1.0f};
        // pair k of the lane: in place (k % 4) of piece k / 4 and of the piece
        // 64 dims on, or (MODE 1) values 2 (k % 2), 2 (k % 2) + 1 of piece k / 2
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int j = MODE == 1 ? k / 2 : k / 4, e = MODE == 1 ? 2 * (k % 2) : k % 4;
            lo[k] = x[j][e];
            hi[k] = MODE == 1 ? x[j][e + 1] : x[j + 2][e];
            wl[k] = ww[j][e];
            wh[k] = MODE == 1 ? ww[j][e + 1] : ww[j + 2][e];
        }
        if constexpr (MODE != 0) {
            float c, n;
            rope_cos_sin<MODE>(p.rope, pos, lane, c, n);
            rot[wave][lane] = float2{c, n};
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const int first = MODE == 1 ? 16 * (k / 2) + 2 * l8 : 32 * (k / 4) + 4 * l8 + k % 4;   // its pair
                const float4 r = *(const float4 *) (rot[wave] + first);
                cs[k] = float2{r.x, r.y};
                cs[k + 1] = float2{r.z, r.w};
            }
        }
        float yl[8], yh[8];
        if (p.norm) norm_rope_group8<MODE>(lo, hi, wl, wh, p.eps, cs, yl, yh);
        else        rope_group8<MODE>(lo, hi, cs, yl, yh);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int j = MODE == 1 ? k / 2 : k / 4, e = MODE == 1 ? 2 * (k % 2) : k % 4;
            x[j][e] = yl[k];
            if constexpr (MODE == 1) x[j][e + 1] = yh[k];
            else x[j + 2][e] = yh[k];
        }
    }
    if (h >= H) return;
    if (kind == 0) {
        float * d = (float *) (p.q_out + (int64_t) h * p.o_nb1 + (int64_t) t * p.o_nb2);
#pragma unroll
        for (int j = 0; j < 4; ++j) *(float4u *) (d + 32 * j + 4 * l8) = x[j];
    } else if (cell >= 0) {
        const PagedPools & c = p.c;
        _Float16 * d = (_Float16 *) (kind == 1 ? c.k + page * c.k_nb3 + cell * c.k_nb1 + h * c.k_nb2
                                               : c.v + page * c.v_nb3 + cell * c.v_nb1 + h * c.v_nb2);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(half4 *) (d + 32 * j + 4 * l8) = half4{(_Float16) x[j][0], (_Float16) x[j][1], (_Float16) x[j][2], (_Float16) x[j][3]};
    }
}

int make_params(const al_paged_append_args * a, const al_tensor * cells, AppendParams * out, int * mode, bool * empty) {
    if (!a) return al_fail(AL_ERR_INVALID, "paged_append: null arguments");
    AppendParams p;
    memset(&p, 0, sizeof(p));
    int rc = paged_pools("paged_append", &a->k_pool, &a->v_pool, &a->table, &p.c);
    if (rc != AL_OK) return rc;
    const int64_t T = a->k.ne[2], Hkv = a->k_pool.ne[2], Hq = a->q.data ? a->q.ne[1] : 0;
    auto rows = [](const al_tensor & t, int64_t H, int64_t n) {
        return t.data && t.type == AL_TYPE_F32 && t.ne[0] == 128 && t.ne[1] == H && t.ne[2] == n && t.ne[3] == 1 && t.nb[0] == 4 &&
               t.nb[1] % 4 == 0 && t.nb[2] % 4 == 0 && ((uintptr_t) t.data & 3u) == 0;
    };
    if (T < 0 || T > (1 << 24) || !rows(a->k, Hkv, T) || !rows(a->v, Hkv, T))
        return al_fail(AL_ERR_INVALID, "paged_append: k and v must be f32 [128, Hkv, T] with the pools' %lld heads", (long long) Hkv);
    if (a->q.data && (Hq < 1 || Hq > (1 << 12) || !rows(a->q, Hq, T) || !rows(a->q_out, Hq, T)))
        return al_fail(AL_ERR_INVALID, "paged_append: q and q_out must be f32 [128, Hq, T]");
    auto index = [&](const al_tensor & t) { return t.data && t.type == AL_TYPE_I32 && t.ne[0] == T && t.nb[0] == 4 && ((uintptr_t) t.data & 3u) == 0; };
    if (!index(a->pos) || !index(a->seq)) return al_fail(AL_ERR_INVALID, "paged_append: pos and seq must be i32 [T]");
    if (cells && !index(*cells)) return al_fail(AL_ERR_INVALID, "paged_append: cells must be i32 [T]");
    auto weight = [](const al_tensor & t) { return !t.data || (t.type == AL_TYPE_F32 && t.ne[0] >= 128 && t.nb[0] == 4 && ((uintptr_t) t.data & 3u) == 0); };
    if (!weight(a->q_w) || !weight(a->k_w)) return al_fail(AL_ERR_INVALID, "paged_append: q_w and k_w must be f32 [128]");
    if (!a->norm && (a->q_w.data || a->k_w.data)) return al_fail(AL_ERR_INVALID, "paged_append: norm weights without the norm");
    if (a->norm && !(a->eps >= 0.0f)) return al_fail(AL_ERR_INVALID, "paged_append: eps %g < 0", (double) a->eps);
    rc = rope_consts("paged_append", a->rope, &p.rope, mode);
    if (rc != AL_OK) return rc;
    p.q = (const char *) a->q.data; p.q_nb1 = a->q.nb[1]; p.q_nb2 = a->q.nb[2];
    p.k = (const char *) a->k.data; p.k_nb1 = a->k.nb[1]; p.k_nb2 = a->k.nb[2];
    p.v = (const char *) a->v.data; p.v_nb1 = a->v.nb[1]; p.v_nb2 = a->v.nb[2];
    p.q_w = (const float *) a->q_w.data;
    p.k_w = (const float *) a->k_w.data;
    p.q_out = (char *) a->q_out.data; p.o_nb1 = a->q_out.nb[1]; p.o_nb2 = a->q_out.nb[2];
    p.pos = (const int32_t *) a->pos.data;
    p.seq = (const int32_t *) a->seq.data;
    p.cells = cells ? (const int32_t *) cells->data : nullptr;
    p.T = (int32_t) T; p.Hq = (int32_t) Hq; p.Hkv = (int32_t) Hkv; p.norm = a->norm != 0;
    p.yq = (int32_t) ((Hq + kRows - 1) / kRows);
    p.yk = (int32_t) ((Hkv + kRows - 1) / kRows);
    p.eps = a->eps;
    *empty = T == 0;
    *out = p;
    return AL_OK;
}

int append(const al_paged_append_args * a, const al_tensor * cells) {
    AppendParams p;
    int mode = 0;
    bool empty = false;
    int rc = make_params(a, cells, &p, &mode, &empty);
    if (rc != AL_OK || empty) return rc;
    rc = al_device_error_flag(&p.c.err);
    if (rc != AL_OK) return rc;
    const dim3 grid((unsigned) ((p.T + kWaves - 1) / kWaves), (unsigned) (p.yq + 2 * p.yk));
    hipStream_t s = (hipStream_t) a->stream;
    switch (mode) {
        case 2: hipLaunchKernelGGL(paged_append_kernel<2>, grid, dim3(64 * kWaves), 0, s, p); break;
        case 1: hipLaunchKernelGGL(paged_append_kernel<1>, grid, dim3(64 * kWaves), 0, s, p); break;
        default: hipLaunchKernelGGL(paged_append_kernel<0>, grid, dim3(64 * kWaves), 0, s, p); break;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "paged_append: launch");
}

}  // namespace

extern "C" int al_paged_append_f32(const al_paged_append_args * a) { return append(a, nullptr); }

extern "C" int al_paged_append_cells_f32(const al_paged_append_args * a, const al_tensor * cells) {
    return cells ? append(a, cells) : al_fail(AL_ERR_INVALID, "paged_append: null cells");
}
