// Low-rank adapters of many requests beside a shared projection
// (include/arclight_lora.h), for gfx950.
//
// Mathematics: v[t] = s_a A_a x[t], y[t] = base[t] + B_a v[t] for a = ids[t],
// both in f32: the f16 weights are exact in f32, and the products run on the
// f32 matrix instruction (16 x 16 x 4), so that activations of any size need
// no scaling. Its rate is a sixteenth of f16's, and enough: at rank 16 the
// products of 8000 tokens take 7 us of the matrix cores, the activations'
// bytes 80.
//
// Rows are taken in tiles of 16. A tile's columns (its rows of x) are
// independent in both products, so a tile of several adapters is computed
// once for each of them and every column kept from its own adapter's: right
// for any order of the ids, and done once where, as in a prompt, the rows of
// a tile share one.
//
// Two launches: lora_shrink_kernel (v, K split over workgroups, partial sums
// into the workspace) and lora_expand_kernel (sums the parts, then a slice of
// the outputs).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/arclight_lora.h"
#include "device_common.hpp"
#include "kernel_args.hpp"
#include "matmul_q4.hpp"
#include "runtime.hpp"

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 16;                       // rows of x
constexpr int kMaxR = 128;
constexpr int kSlots = 4;                       // workgroups that share a tile's adapters
constexpr int kCols = 256;                      // outputs of a workgroup

typedef _Float16 half4 __attribute__((ext_vector_type(4)));

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
    int32_t K, N, R, T, n_adapters;
    int32_t ks, k_step;                         // parts of K, columns of one (a multiple of 128)
    int32_t y_vec;                              // y and base rows 16-byte aligned, N a multiple of 4
    int * err;
};

__device__ __forceinline__ floatx4 mfma_f32(const float a, const float b, const floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Rank of adapter a, -1 for one that is not to be used.
__device__ __forceinline__ int rank_of(const LoraParams & p, const int a) {
    if (a >= p.n_adapters) return -1;
    const int r = p.ranks ? p.ranks[a] : p.R;
    return r < 0 || r > p.R ? -1 : r;
}

__device__ __forceinline__ void lora_error(const LoraParams & p, const int a) {
    if (atomicCAS(p.err + 8, 0, 1) == 0) p.err[9] = a;
}

// The rows of a tile whose adapter no earlier row of it has, of a wave whose
// lanes hold row lane % 16's id (negative: none): one bit each.
__device__ __forceinline__ uint32_t leaders(const int id) {
    uint32_t left = (uint32_t) __ballot(id >= 0) & 0xffffu, out = 0;
    while (left) {
        const int i = __builtin_ctz(left);
        out |= 1u << i;
        left &= ~(uint32_t) __ballot(id == __builtin_amdgcn_readlane(id, i));
    }
    return out;
}

// Parts of v: columns k0 .. k0 + k_step - 1 of K, of a tile's rows. RT: tiles
// of 16 ranks. Lane 16 g + n loads 8 columns of rank row n and of row n of x
// (8 g .. 8 g + 7 of each 32); matrix step s takes column s of them.
template <int RT>
__global__ __launch_bounds__(64 * kWaves) void lora_shrink_kernel(const LoraParams p) {
    __shared__ float part[kWaves][RT * 16][kTile + 1];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kTile + n;
    const int id = t < p.T ? p.ids[t] : -1;
    uint32_t todo = leaders(id);
    for (int i = 0; i < (int) blockIdx.y && todo; ++i) todo &= todo - 1;
    const int k0 = blockIdx.z * p.k_step, k1 = min(k0 + p.k_step, p.K);
    const char * xr = p.x + (int64_t) min(t, p.T - 1) * p.x_nb1;
    while (todo) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
        for (int i = 0; i < kSlots && todo; ++i) todo &= todo - 1;
        const int rank = rank_of(p, a);
        if (rank < 0) {
            if (threadIdx.x == 0) lora_error(p, a);
            continue;
        }
        if (rank == 0) continue;
        const char * ar = p.a + (int64_t) a * p.a_nb2;
        floatx4 acc[RT];
#pragma unroll
        for (int u = 0; u < RT; ++u) acc[u] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = k0 + 32 * wave; k < k1; k += 32 * kWaves) {
            const int kl = k + 8 * g;
            const bool in = kl < p.K;                                  // K is a multiple of 8
            const int kc = in ? kl : 0;
            float4 x0 = *(const float4 *) (xr + (int64_t) kc * 4), x1 = *(const float4 *) (xr + (int64_t) kc * 4 + 16);
            if (!in) x0 = x1 = float4{0.0f, 0.0f, 0.0f, 0.0f};
            const float xs[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
            for (int u = 0; u < RT; ++u) {
                if (16 * u >= rank) break;
                half8 w = *(const half8 *) (ar + (int64_t) min(16 * u + n, rank - 1) * p.a_nb1 + (int64_t) kc * 2);
                if (!in) w = half8{};
#pragma unroll
                for (int s = 0; s < 8; ++s) acc[u] = mfma_f32((float) w[s], xs[s], acc[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][16 * u + 4 * g + i][n] = acc[u][i];
        __syncthreads();
        const float scale = p.scales ? p.scales[a] : 1.0f;
        for (int i = threadIdx.x; i < kTile * p.R; i += 64 * kWaves) {
            const int tok = i / p.R, j = i - tok * p.R;
            const int row = blockIdx.x * kTile + tok;
            if (row >= p.T || p.ids[row] != a) continue;
            float v = 0.0f;
            if (j < rank) {
#pragma unroll
                for (int w = 0; w < kWaves; ++w) v += part[w][j][tok];
                v *= scale;
            }
            p.v[((int64_t) blockIdx.z * p.T + row) * p.R + j] = v;
        }
        __syncthreads();
    }
}

// Outputs n0 .. n0 + 255 of a tile's rows. Lane 16 g + n holds outputs 4 g ..
// 4 g + 3 of each 16, of row n.
template <int RT>
__global__ __launch_bounds__(64 * kWaves) void lora_expand_kernel(const LoraParams p) {
    constexpr int kRow = RT * 16 + 4;
    __shared__ __attribute__((aligned(16))) float v[kTile][kRow];
    prefetch_params(p);
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x * kTile + n;
    const int id = row < p.T ? p.ids[row] : -1;
    const int n0 = blockIdx.y * kCols + 64 * wave;

    floatx4 acc[4];
    const char * br = p.base + (int64_t) min(row, p.T - 1) * p.base_nb1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int c = n0 + 16 * u + 4 * g;
        if (p.y_vec) {
            acc[u] = *(const floatx4 *) (br + (int64_t) min(c, p.N - 4) * 4);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[u][i] = *(const float *) (br + (int64_t) min(c + i, p.N - 1) * 4);
        }
    }
    // v, its parts summed in order; zeros for rows without an adapter
    for (int i = threadIdx.x; i < kTile * RT * 16; i += 64 * kWaves) {
        const int tok = i / (RT * 16), j = i - tok * (RT * 16);
        const int r = blockIdx.x * kTile + tok;
        float s = 0.0f;
        const int a = r < p.T ? p.ids[r] : -1;
        const int rank = a >= 0 ? rank_of(p, a) : 0;
        if (j < rank)
            for (int k = 0; k < p.ks; ++k) s += p.v[((int64_t) k * p.T + r) * p.R + j];
        v[tok][j] = s;
    }
    __syncthreads();

    uint32_t todo = leaders(id);
    while (todo) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
        todo &= todo - 1;
        const int rank = rank_of(p, a);
        const bool mine = id == a;
        if (rank < 0) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (mine) acc[u] = floatx4{1.0f, 1.0f, 1.0f, 1.0f} * __builtin_nanf("");
            continue;
        }
        const char * b = p.b + (int64_t) a * p.b_nb2 + 8 * g;
        floatx4 sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[u] = acc[u];
#pragma unroll
        for (int q = 0; q < RT; ++q) {
            if (16 * q >= rank) break;
            const float4 x = *(const float4 *) &v[n][16 * q + 4 * g];
            const float xs[4] = {x.x, x.y, x.z, x.w};
            const int j0 = 16 * q + 4 * g;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = min(n0 + 16 * u + n, p.N - 1);
                half4 w = j0 < p.R ? *(const half4 *) (b + (int64_t) c * p.b_nb1 + 32 * q) : half4{};
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    sum[u] = mfma_f32(j0 + s < rank ? (float) w[s] : 0.0f, xs[s], sum[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (mine) acc[u] = sum[u];
    }
    if (row >= p.T) return;
    char * yr = p.y + (int64_t) row * p.y_nb1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int c = n0 + 16 * u + 4 * g;
        if (p.y_vec) {
            if (c < p.N) *(floatx4 *) (yr + (int64_t) c * 4) = acc[u];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < p.N) *(float *) (yr + (int64_t) (c + i) * 4) = acc[u][i];
        }
    }
}

struct Plan {
    LoraParams p;
    bool empty = false;
    size_t v_bytes = 0, q_bytes = 0;            // v, then the projection's scratch
};

int make_plan(const al_lora_args * g, bool project, int n_cu, Plan * out) {
    if (!g) return al_fail(AL_ERR_INVALID, "lora: null arguments");
    const al_tensor &a = g->a, &b = g->b, &x = g->x, &y = g->y;
    if (!a.data || !b.data || !x.data || !y.data || !g->ids.data)
        return al_fail(AL_ERR_INVALID, "lora: a, b, x, ids and y are required");
    if (a.type != AL_TYPE_F16 || b.type != AL_TYPE_F16)
        return al_fail(AL_ERR_UNSUPPORTED, "lora: adapter types %d / %d (f16 only)", a.type, b.type);
    if (x.type != AL_TYPE_F32 || y.type != AL_TYPE_F32)
        return al_fail(AL_ERR_UNSUPPORTED, "lora: x / y types %d / %d (f32 only)", x.type, y.type);
    const int64_t K = a.ne[0], R = a.ne[1], A = a.ne[2], N = b.ne[1], T = x.ne[1];
    if (b.ne[0] != R || b.ne[2] != A || a.ne[3] != 1 || b.ne[3] != 1 || x.ne[0] != K || x.ne[2] != 1 || x.ne[3] != 1 ||
        y.ne[0] != N || y.ne[1] != T || y.ne[2] != 1 || y.ne[3] != 1)
        return al_fail(AL_ERR_INVALID, "lora: shapes a [K, R, n], b [R, N, n], x [K, T], y [N, T] do not fit: K %lld / %lld, R %lld / %lld",
                       (long long) K, (long long) x.ne[0], (long long) R, (long long) b.ne[0]);
    if (K < 8 || K % 8 || K > 65536 || R < 8 || R % 8 || R > kMaxR)
        return al_fail(AL_ERR_UNSUPPORTED, "lora: K %lld, R %lld (multiples of 8, at most 65536 and %d)", (long long) K, (long long) R, kMaxR);
    if (A < 1 || A > (1 << 20) || N < 1 || N > (1 << 22) || T < 0 || T > (1 << 20))
        return al_fail(AL_ERR_UNSUPPORTED, "lora: sizes out of range");
    auto al = [](const al_tensor & t, uint64_t by) { return !(((uintptr_t) t.data | t.nb[1] | t.nb[2]) & (by - 1)); };
    if (a.nb[0] != 2 || b.nb[0] != 2 || !al(a, 16) || !al(b, 16))
        return al_fail(AL_ERR_INVALID, "lora: rows of a and b must be contiguous and 16-byte aligned");
    if (x.nb[0] != 4 || ((uintptr_t) x.data & 15u) || x.nb[1] % 16 || y.nb[0] != 4 || ((uintptr_t) y.data & 3u) || y.nb[1] % 4 ||
        (T > 1 && y.nb[1] < (uint64_t) N * 4))
        return al_fail(AL_ERR_INVALID, "lora: rows of x must be 16-byte aligned, those of y contiguous and apart");
    if (g->ids.type != AL_TYPE_I32 || g->ids.ne[0] != T || g->ids.nb[0] != 4 || ((uintptr_t) g->ids.data & 3u))
        return al_fail(AL_ERR_INVALID, "lora: ids must be i32 [T]");
    if (g->ranks.data && (g->ranks.type != AL_TYPE_I32 || g->ranks.ne[0] != A || g->ranks.nb[0] != 4))
        return al_fail(AL_ERR_INVALID, "lora: ranks must be i32 [n_adapters]");
    if (g->scales.data && (g->scales.type != AL_TYPE_F32 || g->scales.ne[0] != A || g->scales.nb[0] != 4))
        return al_fail(AL_ERR_INVALID, "lora: scales must be f32 [n_adapters]");
    const al_tensor & base = g->base.data && !project ? g->base : y;
    if (base.type != AL_TYPE_F32 || base.ne[0] != N || base.ne[1] != T || base.ne[2] != 1 || base.ne[3] != 1 || base.nb[0] != 4 ||
        ((uintptr_t) base.data & 3u) || base.nb[1] % 4)
        return al_fail(AL_ERR_INVALID, "lora: base must be f32 [N, T]");
    if (T > 0 && (base.data != y.data || base.nb[1] != y.nb[1])) {
        const uintptr_t b0 = (uintptr_t) base.data, b1 = b0 + (uint64_t) (T - 1) * base.nb[1] + (uint64_t) N * 4;
        const uintptr_t y0 = (uintptr_t) y.data, y1 = y0 + (uint64_t) (T - 1) * y.nb[1] + (uint64_t) N * 4;
        if (b0 < y1 && y0 < b1) return al_fail(AL_ERR_INVALID, "lora: base overlaps y and is not y");
    }
    Plan pl;
    LoraParams & p = pl.p;
    memset(&p, 0, sizeof(p));
    pl.empty = T == 0;
    p.a = (const char *) a.data; p.a_nb1 = a.nb[1]; p.a_nb2 = a.nb[2];
    p.b = (const char *) b.data; p.b_nb1 = b.nb[1]; p.b_nb2 = b.nb[2];
    p.ranks = (const int32_t *) g->ranks.data;
    p.scales = (const float *) g->scales.data;
    p.ids = (const int32_t *) g->ids.data;
    p.x = (const char *) x.data; p.x_nb1 = x.nb[1];
    p.base = (const char *) base.data; p.base_nb1 = base.nb[1];
    p.y = (char *) y.data; p.y_nb1 = y.nb[1];
    p.K = (int32_t) K; p.N = (int32_t) N; p.R = (int32_t) R; p.T = (int32_t) T; p.n_adapters = (int32_t) A;
    p.y_vec = N % 4 == 0 && !(((uintptr_t) y.data | y.nb[1] | (uintptr_t) base.data | base.nb[1]) & 15u);
    const int64_t tiles = (T + kTile - 1) / kTile;
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({16, (K + 255) / 256, n_cu / std::max<int64_t>(1, tiles)}));
    p.k_step = (int32_t) (((K + parts - 1) / parts + 127) / 128 * 128);
    p.ks = (int32_t) ((K + p.k_step - 1) / p.k_step);
    pl.v_bytes = ((size_t) p.ks * T * R * 4 + 255) / 256 * 256;
    if (project) {
        const int rc = mul_mat_q4_0_check(&g->w, &x, &y, &pl.q_bytes);
        if (rc != AL_OK) return rc;
    }
    *out = pl;
    return AL_OK;
}

template <int RT>
hipError_t launch(const LoraParams & p, hipStream_t st) {
    const unsigned tiles = (unsigned) ((p.T + kTile - 1) / kTile);
    hipLaunchKernelGGL(lora_shrink_kernel<RT>, dim3(tiles, kSlots, (unsigned) p.ks), dim3(64 * kWaves), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(lora_expand_kernel<RT>, dim3(tiles, (unsigned) ((p.N + kCols - 1) / kCols)), dim3(64 * kWaves), 0, st, p);
    return hipGetLastError();
}

int run(const al_lora_args * g, bool project) {
    Plan pl;
    int rc = make_plan(g, project, 1, &pl);                            // refusals need no device
    if (rc != AL_OK || pl.empty) return rc;
    int n_cu = 0;
    rc = al_device_cu_count(&n_cu);
    if (rc == AL_OK) rc = make_plan(g, project, n_cu, &pl);
    if (rc == AL_OK) rc = al_device_error_flag(&pl.p.err);
    if (rc != AL_OK) return rc;
    const size_t need = pl.v_bytes + pl.q_bytes;
    void * ws = g->workspace;
    if (ws) {
        if (g->workspace_bytes < need || ((uintptr_t) ws & 15u))
            return al_fail(AL_ERR_WORKSPACE, "lora: workspace %llu bytes (16-byte aligned) < %zu needed",
                           (unsigned long long) g->workspace_bytes, need);
    } else {
        rc = al_library_workspace(need, g->stream, &ws);
        if (rc != AL_OK) return rc;
    }
    pl.p.v = (float *) ws;
    if (project) {
        rc = mul_mat_q4_0_run(&g->w, &g->x, &g->y, (char *) ws + pl.v_bytes, (hipStream_t) g->stream);
        if (rc != AL_OK) return rc;
    }
    hipError_t e;
    const hipStream_t st = (hipStream_t) g->stream;
    if (pl.p.R <= 16) e = launch<1>(pl.p, st);
    else if (pl.p.R <= 32) e = launch<2>(pl.p, st);
    else if (pl.p.R <= 64) e = launch<4>(pl.p, st);
    else e = launch<8>(pl.p, st);
    return e == hipSuccess ? AL_OK : al_hip_fail(e, "lora: launch");
}

}  // namespace

extern "C" int al_lora_f32(const al_lora_args * args) { return run(args, false); }

extern "C" int al_mul_mat_q4_0_lora_f32(const al_lora_args * args) { return run(args, true); }

extern "C" uint64_t al_lora_workspace_bytes(const al_lora_args * args) {
    int n_cu = 0;
    Plan pl;
    if (al_device_cu_count(&n_cu) != AL_OK || make_plan(args, args && args->w.data != nullptr, n_cu, &pl) != AL_OK) return 0;
    return pl.empty ? 0 : pl.v_bytes + pl.q_bytes;
}
