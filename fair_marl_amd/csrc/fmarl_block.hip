// The end of a residual block and the start of the next one in one pass on gfx950: with n(a) = a / sqrt(mean a^2 + eps) (rms) or
// (a - mean a) / sqrt(var a + eps) (layer),
//     u = n_groups(branch) * post_weight + post_bias      r = u * act(gate)      y = x + scale * r      h = n(y) * pre_weight + pre_bias.
// Backwards, with the norm's transpose N^T(d) = (d - n mean(d n) [- mean d]) / sqrt(..):
//     dy' = dy + N^T(dh pre_weight) = dx      dr = dy' scale      du = dr act(gate)      dgate = dr u act'(gate)
//     dbranch = N_groups^T(du post_weight)    and the weights' gradients are sums over the rows of dy' r, du n, du, dh n, dh.
// Nothing is kept from the forward pass: the backward one reads x, branch and gate again and forms y unrounded.  All of it is bytes: forward five
// rows, backward eight; the arithmetic is float32.  655 360 rows of 64 float32: 165 us forwards (5.1 TB/s), 270 + 5 us backwards (5.0 TB/s); 16 383 rows of 1 000 bfloat16 in groups of
// 125: 44 us (3.7 TB/s) and 94 + 9 us (2.8 TB/s): there the sums between the waves of a row bound it, two for each group norm through LDS.
#include "fmarl_policy_dev.h"

namespace fmarl {
namespace policy {

struct Block {
    int64_t rows;
    int dim, groups, group_mode, layer, silu, post_norm, pre_norm, vec;
    float eps;
    const char *x, *branch, *gate; int64_t xs, bs, gs;      // row strides in elements
    const float *scale, *post_w, *post_b, *pre_w, *pre_b;   // (dim), NULL: 1, 1, 0, 1, 0
    char *y, *h;                                            // forward outputs, contiguous; NULL: not wanted
    const char *dy, *dh; int64_t dys, dhs;                  // backward; NULL: zeros
    char *dx, *dbranch, *dgate;
    float *partial;                                         // (workgroups, 5, dim): the weights' gradients of each workgroup's rows
};

// floats of a team's row in LDS: the row, then its groups' means
__host__ __device__ inline int block_row_floats(int dim, int groups) { return ((dim + 3) & ~3) + ((groups + 3) & ~3); }

enum { kGroupRow = 0, kGroupLanes = 1, kGroupLds = 2 };     // how a group's elements lie over the team: all of it, 2^k neighbouring lanes, anyhow

// A row belongs to a team of TL threads, TL * 4 * NV >= dim: thread l holds the four columns from (n TL + l) 4 on, n < NV, so that a team's loads are
// consecutive.  Teams of 16 lanes up to dim 64, 32, 64, then of a workgroup of 128 ... 1 024: four columns a thread (eight beyond 2 048), so that the weights and the sums of
// their gradients fit the registers four waves a SIMD deep.  (A wave per row of 1 024, sixteen columns a lane, held 256 + 96 registers: one wave a SIMD, 226 us for
// 16 383 bf16 rows backwards.)  The next row's loads are in flight while a row is computed.  What a team of several waves exchanges lies in one of two places in turn: a
// barrier before the reads is enough, the next but one write comes behind another.
struct Exchange { float *red, *row; int row_floats, flip; };

template <int TL>
__device__ __forceinline__ void team_sum2(float &v, float &w, Exchange &x) {
    v = lanes_sum<1>(v, TL < 64 ? TL : 64); w = lanes_sum<1>(w, TL < 64 ? TL : 64);
    if (TL > 64) {
        float *red = x.red + x.flip * 32;
        x.flip ^= 1;
        if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = v; red[16 + (threadIdx.x >> 6)] = w; }
        __syncthreads();
        v = w = 0.f;
#pragma unroll
        for (int k = 0; k < TL / 64; ++k) { v += red[k]; w += red[16 + k]; }
    }
}

template <int TL> __device__ __forceinline__ float team_sum(float v, Exchange &x) { float w = 0.f; team_sum2<TL>(v, w, x); return v; }

template <int TL> __device__ __forceinline__ void team_sync() { if (TL > 64) __syncthreads(); else wave_sync(); }

// v <- the mean over the group of each element; columns beyond dim hold 0 before and anything behind
template <int TL, int NV>
__device__ __forceinline__ void group_means(const Block &a, float (&v)[NV][4], int l, Exchange &x) {
    if (a.group_mode == kGroupRow) {
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n) s += (v[n][0] + v[n][1]) + (v[n][2] + v[n][3]);
        s = team_sum<TL>(s, x) * (1.f / a.dim);
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[n][r] = s;
    } else if (a.group_mode == kGroupLanes) {
        const int lanes = a.dim / a.groups / 4;
        const float inv = 1.f / (4 * lanes);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            float s = (v[n][0] + v[n][1]) + (v[n][2] + v[n][3]);
            s = lanes_sum<1>(s, lanes);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[n][r] = s * inv;
        }
    } else {
        const int size = a.dim / a.groups;
        const float inv = 1.f / size;
        float *row = x.row + x.flip * x.row_floats, *sums = row + ((a.dim + 3) & ~3);
        x.flip ^= 1;
        if (TL <= 64) team_sync<TL>();
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int col = (n * TL + l) * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r) if (col + r < a.dim) row[col + r] = v[n][r];
        }
        team_sync<TL>();
        int per = 1;   // lanes on one group: as many as there are, up to a wave
        while (per < 64 && per * 2 * a.groups <= TL) per <<= 1;
        for (int g0 = 0; g0 < a.groups; g0 += TL / per) {
            const int g = g0 + l / per;
            float s = 0.f;
            if (g < a.groups) for (int e = l % per; e < size; e += per) s += row[g * size + e];
            s = lanes_sum<1>(s, per);
            if (l % per == 0 && g < a.groups) sums[g] = s * inv;
        }
        team_sync<TL>();
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int col = (n * TL + l) * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[n][r] = col + r < a.dim ? sums[min(a.groups - 1, (int)((col + r + 0.5f) * inv))] : 0.f;
        }
    }
}

template <int TL, int NV>
__device__ __forceinline__ void row_means(const Block &a, float (&v)[NV][4], float &mean, Exchange &x) {
    float s = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) s += (v[n][0] + v[n][1]) + (v[n][2] + v[n][3]);
    mean = team_sum<TL>(s, x) * (1.f / a.dim);
}

#define FMARL_EACH(body)                                                \
    _Pragma("unroll") for (int n = 0; n < NV; ++n) {                    \
        const int col = (n * TL + l) * 4; (void)col;                    \
        _Pragma("unroll") for (int r = 0; r < 4; ++r) { const bool in = col + r < a.dim; (void)in; body; } }

// n (in place) and 1 / sqrt(..) of the groups of o; two passes over the registers where the mean is taken off first
template <int TL, int NV>
__device__ __forceinline__ void norm_groups(const Block &a, float eps, float (&o)[NV][4], float (&inv)[NV][4], int l, Exchange &x) {
    if (a.layer) {
        FMARL_EACH(inv[n][r] = o[n][r])
        group_means<TL, NV>(a, inv, l, x);
        FMARL_EACH(o[n][r] = in ? o[n][r] - inv[n][r] : 0.f)
    }
    FMARL_EACH(inv[n][r] = o[n][r] * o[n][r])
    group_means<TL, NV>(a, inv, l, x);
    FMARL_EACH(inv[n][r] = rsqrtf(inv[n][r] + eps); o[n][r] *= inv[n][r])
}

template <int TL, int NV>
__device__ __forceinline__ float norm_row(const Block &a, float eps, float (&y)[NV][4], int l, Exchange &x) {
    float mean;
    if (a.layer) {
        row_means<TL, NV>(a, y, mean, x);
        FMARL_EACH(y[n][r] = in ? y[n][r] - mean : 0.f)
    }
    float s = 0.f;
    FMARL_EACH(s += y[n][r] * y[n][r])
    const float inv = rsqrtf(team_sum<TL>(s, x) * (1.f / a.dim) + eps);
    FMARL_EACH(y[n][r] *= inv)
    return inv;
}

template <typename T, int TL, int NV, bool VEC>
__device__ __forceinline__ void fetch_row(const Block &a, typename Vec4<T>::type (&v)[NV], const char *base, int64_t stride, int64_t row, int l) {
    if (!base) return;   // (what is not given stays zero)
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int col = (n * TL + l) * 4, left = row < a.rows ? a.dim - col : 0;
        const T *p = (const T *)base + row * stride + col;
        // (100 000 rows of 350 bfloat16: 577 us backwards element by element, 523 with one access of four where they are there, 406 so)
        // a row's last elements come with those before them, in one load like every other thread's, and are moved to their places when they are used (widen_row)
        if (VEC || a.dim < 4) v[n] = load4<T>(p, left, VEC);
        else if (left > 0) v[n] = *(const typename Loose4<T>::type *)(p + min(0, left - 4));
        else v[n] = typename Vec4<T>::type{};
    }
}

template <int TL, bool VEC, typename V, int NV> __device__ __forceinline__ void widen_row(const Block &a, float (&v)[NV][4], const V (&raw)[NV], int l) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        f32x4 w = widen(raw[n]);
        if (!VEC && a.dim >= 4) {
            const int left = a.dim - (n * TL + l) * 4, by = left >= 4 ? 0 : left > 0 ? 4 - left : 4;   // places
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = by & 1 ? (r < 3 ? w[r < 3 ? r + 1 : 3] : 0.f) : w[r];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = by & 2 ? (r < 2 ? w[r < 2 ? r + 2 : 3] : 0.f) : w[r];
            if (by == 4) w = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[n][r] = w[r];
    }
}

template <typename T, int TL, int NV, bool VEC>
__device__ __forceinline__ void store_row(const Block &a, const float (&v)[NV][4], char *base, int64_t row, int l) {
    if (!base || row >= a.rows) return;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int col = (n * TL + l) * 4;
        store4<T>((T *)base + row * a.dim + col, f32x4{v[n][0], v[n][1], v[n][2], v[n][3]}, a.dim - col, VEC);
    }
}

template <int TL, int NV>
__device__ __forceinline__ void load_weights(const Block &a, float (&v)[NV][4], const float *w, float none, int l) {
    FMARL_EACH(v[n][r] = in ? (w ? w[col + r] : none) : 0.f)
}

__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-1.44269504f * x)); }

template <typename TX, typename TB, int TL, int NV, int THREADS, bool VEC>
__global__ __launch_bounds__(THREADS) void block_norm_kernel(Block a) {
    extern __shared__ __align__(16) float lds[];
    const int l = threadIdx.x % TL, team = threadIdx.x / TL;
    constexpr int kTeams = THREADS / TL;
    Exchange ex = {lds, lds + 64 + team * 2 * block_row_floats(a.dim, a.groups), block_row_floats(a.dim, a.groups), 0};
    float sc[NV][4], pw[NV][4], pb[NV][4], rw[NV][4], rb[NV][4];
    load_weights<TL, NV>(a, sc, a.scale, 1.f, l);
    load_weights<TL, NV>(a, pw, a.post_w, 1.f, l);
    load_weights<TL, NV>(a, pb, a.post_b, 0.f, l);
    load_weights<TL, NV>(a, rw, a.pre_w, 1.f, l);
    load_weights<TL, NV>(a, rb, a.pre_b, 0.f, l);
    typename Vec4<TX>::type nx[NV] = {};
    typename Vec4<TB>::type no[NV] = {}, ng[NV] = {};
    const int64_t step = (int64_t)gridDim.x * kTeams;
    auto fetch = [&](int64_t row) {
        fetch_row<TX, TL, NV, VEC>(a, nx, a.x, a.xs, row, l);
        fetch_row<TB, TL, NV, VEC>(a, no, a.branch, a.bs, row, l);
        fetch_row<TB, TL, NV, VEC>(a, ng, a.gate, a.gs, row, l);
    };
    fetch((int64_t)blockIdx.x * kTeams + team);
    // every thread of the workgroup makes the same trips: rows beyond the last one are zeros and not stored
    for (int64_t row0 = (int64_t)blockIdx.x * kTeams; row0 < a.rows; row0 += step) {
        const int64_t row = row0 + team;
        float y[NV][4], o[NV][4], g[NV][4];
        widen_row<TL, VEC>(a, y, nx, l); widen_row<TL, VEC>(a, o, no, l); widen_row<TL, VEC>(a, g, ng, l);
        fetch(row + step);
        if (a.branch) {
            if (a.post_norm) {
                float inv[NV][4];
                norm_groups<TL, NV>(a, a.eps, o, inv, l, ex);
                FMARL_EACH(o[n][r] = o[n][r] * pw[n][r] + pb[n][r])
            }
            if (a.gate) FMARL_EACH(const float s = sigmoid(g[n][r]); o[n][r] *= a.silu ? g[n][r] * s : s)
            FMARL_EACH(y[n][r] = in ? y[n][r] + sc[n][r] * o[n][r] : 0.f)
            store_row<TX, TL, NV, VEC>(a, y, a.y, row, l);
        }
        if (a.h) {
            norm_row<TL, NV>(a, a.eps, y, l, ex);
            FMARL_EACH(y[n][r] = y[n][r] * rw[n][r] + rb[n][r])
            store_row<TB, TL, NV, VEC>(a, y, a.h, row, l);
        }
    }
}

template <typename TX, typename TB, int TL, int NV, int THREADS, bool VEC>
__global__ __launch_bounds__(THREADS, NV == 1 && sizeof(TX) == 2 ? 4 : 1) void block_norm_backward_kernel(Block a) {
    extern __shared__ __align__(16) float lds[];
    const int l = threadIdx.x % TL, team = threadIdx.x / TL;
    constexpr int kTeams = THREADS / TL;
    Exchange ex = {lds, lds + 64 + team * 2 * block_row_floats(a.dim, a.groups), block_row_floats(a.dim, a.groups), 0};
    float sc[NV][4], pw[NV][4], pb[NV][4], rw[NV][4];
    load_weights<TL, NV>(a, sc, a.scale, 1.f, l);
    load_weights<TL, NV>(a, pw, a.post_w, 1.f, l);
    load_weights<TL, NV>(a, pb, a.post_b, 0.f, l);
    load_weights<TL, NV>(a, rw, a.pre_w, 1.f, l);
    float acc[5][NV][4];
#pragma unroll
    for (int k = 0; k < 5; ++k) FMARL_EACH(acc[k][n][r] = 0.f)
    typename Vec4<TX>::type nx[NV] = {}, nd[NV] = {};
    typename Vec4<TB>::type no[NV] = {}, ng[NV] = {}, nh[NV] = {};
    const int64_t step = (int64_t)gridDim.x * kTeams;
    auto fetch = [&](int64_t row) {
        fetch_row<TX, TL, NV, VEC>(a, nx, a.x, a.xs, row, l);
        fetch_row<TB, TL, NV, VEC>(a, no, a.branch, a.bs, row, l);
        fetch_row<TB, TL, NV, VEC>(a, ng, a.gate, a.gs, row, l);
        fetch_row<TX, TL, NV, VEC>(a, nd, a.dy, a.dys, row, l);
        fetch_row<TB, TL, NV, VEC>(a, nh, a.dh, a.dhs, row, l);
    };
    fetch((int64_t)blockIdx.x * kTeams + team);
    for (int64_t row0 = (int64_t)blockIdx.x * kTeams; row0 < a.rows; row0 += step) {
        const int64_t row = row0 + team;
        const float eps = row < a.rows ? a.eps : 1.f;   // a row of zeros beyond the last one adds nothing to the sums, nor where eps is 0 (1 / sqrt(0) times 0 would be NaN)
        float y[NV][4], u[NV][4], g[NV][4], inv[NV][4], d[NV][4], dh[NV][4];
        widen_row<TL, VEC>(a, y, nx, l); widen_row<TL, VEC>(a, u, no, l); widen_row<TL, VEC>(a, g, ng, l); widen_row<TL, VEC>(a, d, nd, l); widen_row<TL, VEC>(a, dh, nh, l);
        fetch(row + step);
        // forward again: u = n(branch) from here on, y unrounded
        if (a.branch) {
            if (a.post_norm) norm_groups<TL, NV>(a, eps, u, inv, l, ex);
            FMARL_EACH(const float s = a.gate ? sigmoid(g[n][r]) : 1.f;
                       const float f = a.gate && a.silu ? g[n][r] * s : s;
                       y[n][r] = in ? y[n][r] + sc[n][r] * (u[n][r] * pw[n][r] + pb[n][r]) * f : 0.f)
        }
        if (a.pre_norm && a.dh) {
            const float yi = norm_row<TL, NV>(a, eps, y, l, ex);   // y: its norm from here on
            float m1 = 0.f, m2 = 0.f;
            FMARL_EACH(acc[3][n][r] += dh[n][r] * y[n][r]; acc[4][n][r] += dh[n][r]; dh[n][r] *= rw[n][r];
                       m1 += dh[n][r]; m2 += dh[n][r] * y[n][r])
            team_sum2<TL>(m1, m2, ex);
            m2 *= 1.f / a.dim;
            m1 = a.layer ? m1 * (1.f / a.dim) : 0.f;
            FMARL_EACH(d[n][r] += yi * (dh[n][r] - y[n][r] * m2 - m1))
        }
        store_row<TX, TL, NV, VEC>(a, d, a.dx, row, l);
        if (a.branch) {
            FMARL_EACH(const float s = a.gate ? sigmoid(g[n][r]) : 1.f;
                       const float f = a.gate && a.silu ? g[n][r] * s : s;
                       const float slope = a.silu ? s + f * (1.f - s) : s * (1.f - s);
                       const float w = u[n][r] * pw[n][r] + pb[n][r];
                       acc[0][n][r] += in ? d[n][r] * w * f : 0.f;
                       d[n][r] = in ? d[n][r] * sc[n][r] : 0.f;
                       g[n][r] = d[n][r] * w * slope;
                       d[n][r] *= f;
                       acc[1][n][r] += d[n][r] * u[n][r]; acc[2][n][r] += d[n][r];
                       d[n][r] *= pw[n][r])
            if (a.gate) store_row<TB, TL, NV, VEC>(a, g, a.dgate, row, l);
            if (a.post_norm) {
                float m[NV][4];
                FMARL_EACH(m[n][r] = d[n][r] * u[n][r])
                group_means<TL, NV>(a, m, l, ex);
                FMARL_EACH(u[n][r] = d[n][r] - u[n][r] * m[n][r])
                if (a.layer) {
                    FMARL_EACH(m[n][r] = d[n][r])
                    group_means<TL, NV>(a, m, l, ex);
                    FMARL_EACH(u[n][r] -= m[n][r])
                }
                FMARL_EACH(d[n][r] = in ? u[n][r] * inv[n][r] : 0.f)
            }
            store_row<TB, TL, NV, VEC>(a, d, a.dbranch, row, l);
        }
    }
    // the workgroup's sums, teams in a fixed order
    float *mine = a.partial + (int64_t)blockIdx.x * 5 * a.dim;
    for (int k = 0; k < 5; ++k) {
        if (kTeams == 1) {
            FMARL_EACH(if (in) mine[k * a.dim + col + r] = acc[k][n][r])
        } else {
            __syncthreads();
            FMARL_EACH(if (in) lds[team * a.dim + col + r] = acc[k][n][r])
            __syncthreads();
            for (int c = threadIdx.x; c < a.dim; c += THREADS) {
                float s = 0.f;
                for (int t = 0; t < kTeams; ++t) s += lds[t * a.dim + c];
                mine[k * a.dim + c] = s;
            }
        }
    }
}
#undef FMARL_EACH

struct BlockSums { float *out[5]; const float *partial; int dim, parts; };

// 8 columns a workgroup, 32 threads a column: each adds every 32nd workgroup's partial in float64, then the 32 are added in order
__global__ __launch_bounds__(256) void block_sums_kernel(BlockSums a) {
    __shared__ double red[32][9];
    const int c = threadIdx.x & 7, s = threadIdx.x >> 3, n = 5 * a.dim, i = blockIdx.x * 8 + c;
    double sum = 0.0;
    if (i < n && a.out[i / a.dim]) {
#pragma unroll 8
        for (int p = s; p < a.parts; p += 32) sum += (double)a.partial[(int64_t)p * n + i];
    }
    red[s][c] = sum;
    __syncthreads();
    if (s == 0 && i < n && a.out[i / a.dim]) {
        for (int k = 1; k < 32; ++k) sum += red[k][c];
        a.out[i / a.dim][i % a.dim] = (float)sum;
    }
}

}  // namespace policy
}  // namespace fmarl

using namespace fmarl;
using namespace fmarl::policy;

namespace {

const int kMaxBlockDim = 8192;

int block_check(const FmarlBlock *b, const char *who) {
    if (!b) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    if (b->rows < 0 || b->rows > (1ll << 40)) return policy_fail(FMARL_EINVAL, "%s: bad number of rows", who);
    if (b->dim < 1 || b->dim > kMaxBlockDim) return policy_fail(FMARL_EINVAL, "%s: dim must lie in 1..8192", who);
    if (b->groups < 1 || b->groups > 256 || b->dim % b->groups) return policy_fail(FMARL_EINVAL, "%s: groups must lie in 1..256 and divide dim", who);
    if (b->dtype < FMARL_T_F32 || b->dtype > FMARL_T_F16 || (b->x_dtype != b->dtype && b->x_dtype != FMARL_T_F32))
        return policy_fail(FMARL_EINVAL, "%s: x must have the branch's type, or float32", who);
    if (b->kind < 0 || b->kind > 1 || b->gate_act < 0 || b->gate_act > 1) return policy_fail(FMARL_EINVAL, "%s: unknown kind or gate_act", who);
    if (!(b->eps >= 0.f)) return policy_fail(FMARL_EINVAL, "%s: eps must not be negative", who);
    if (b->rows > 0 && !b->x) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    if (b->rows > 0 && !b->branch && (b->gate || b->scale || b->post_weight || b->post_bias)) return policy_fail(FMARL_EINVAL, "%s: gate, scale and post weights need a branch", who);
    if (!b->post_norm && (b->post_weight || b->post_bias)) return policy_fail(FMARL_EINVAL, "%s: post weights need post_norm", who);
    return FMARL_OK;
}

Block block_args(const FmarlBlock *b) {
    Block a = {};
    a.rows = b->rows; a.dim = b->dim; a.groups = b->groups; a.layer = b->kind == 1; a.silu = b->gate_act == 1; a.post_norm = b->post_norm != 0; a.pre_norm = b->pre_norm != 0;
    a.eps = b->eps;
    a.x = (const char *)b->x; a.branch = (const char *)b->branch; a.gate = (const char *)b->gate; a.xs = b->x_stride; a.bs = b->branch_stride; a.gs = b->gate_stride;
    a.scale = b->scale; a.post_w = b->post_weight; a.post_b = b->post_bias; a.pre_w = b->pre_weight; a.pre_b = b->pre_bias;
    const int lanes = b->dim / b->groups / 4;
    const int team = b->dim <= 64 ? 16 : b->dim <= 128 ? 32 : 64;   // lanes that can exchange without LDS
    a.group_mode = b->groups == 1 ? kGroupRow : b->dim / b->groups % 4 == 0 && (lanes & (lanes - 1)) == 0 && lanes <= team ? kGroupLanes : kGroupLds;
    return a;
}

bool row_aligned(const void *p, int64_t stride, int bytes) { return ((uintptr_t)p & (4 * bytes - 1)) == 0 && (stride & 3) == 0; }

int block_threads(int dim) { return dim <= 256 ? 256 : dim <= 512 ? 128 : dim <= 1024 ? 256 : dim <= 4096 ? 512 : 1024; }

// Workgroups: each loops over its share of the rows.  Forwards five waves a SIMD, backwards three, one more of half precision rows and of long ones, whose bytes in flight or
// barriers ask for it (us for training, three | four: 655 360 x 64 float32 443 | 473, bfloat16 276 | 265; 20 000 x 2 048 float32 476 | 436, bfloat16 324 | 275); backwards few beside the
// rows, so that their partial sums of the weights' gradients (5 dim floats each) stay below a sixteenth of the bytes of the rows
int block_workgroups(const FmarlBlock *b, bool backward) {
    const int threads = block_threads(b->dim), teams = b->dim <= 64 ? 16 : b->dim <= 128 ? 8 : b->dim <= 256 ? 4 : 1;
    const int64_t want = backward ? (b->rows + 15) / 16 : (b->rows + teams - 1) / teams, deep = b->dtype != FMARL_T_F32 || b->dim > 1024, most = ((backward ? 3 : 5) + deep) * 65536 / threads;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename TX, typename TB, int TL, int NV, int THREADS>
int launch_block_as(const Block &a, bool backward, int blocks, hipStream_t st) {
    const size_t teams = THREADS / TL;
    size_t lds = 64 + (a.group_mode == kGroupLds ? teams * 2 * block_row_floats(a.dim, a.groups) : 0);
    if (backward && teams > 1 && lds < teams * a.dim) lds = teams * a.dim;
    lds *= 4;
    auto kernel = backward ? a.vec ? block_norm_backward_kernel<TX, TB, TL, NV, THREADS, true> : block_norm_backward_kernel<TX, TB, TL, NV, THREADS, false>
                           : a.vec ? block_norm_kernel<TX, TB, TL, NV, THREADS, true> : block_norm_kernel<TX, TB, TL, NV, THREADS, false>;
    if (lds > 64 * 1024) HIP_OK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(THREADS), lds, st, a);
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

template <typename TX, typename TB>
int launch_block_t(const Block &a, bool backward, int blocks, hipStream_t st) {
    if (a.dim <= 64) return launch_block_as<TX, TB, 16, 1, 256>(a, backward, blocks, st);
    if (a.dim <= 128) return launch_block_as<TX, TB, 32, 1, 256>(a, backward, blocks, st);
    if (a.dim <= 256) return launch_block_as<TX, TB, 64, 1, 256>(a, backward, blocks, st);
    if (a.dim <= 512) return launch_block_as<TX, TB, 128, 1, 128>(a, backward, blocks, st);
    if (a.dim <= 1024) return launch_block_as<TX, TB, 256, 1, 256>(a, backward, blocks, st);
    if (a.dim <= 2048) return launch_block_as<TX, TB, 512, 1, 512>(a, backward, blocks, st);
    if (a.dim <= 4096) return launch_block_as<TX, TB, 512, 2, 512>(a, backward, blocks, st);
    return launch_block_as<TX, TB, 1024, 2, 1024>(a, backward, blocks, st);
}

int launch_block(const FmarlBlock *b, const Block &a, bool backward, int blocks, hipStream_t st) {
    if (b->dtype == FMARL_T_F32) return launch_block_t<float, float>(a, backward, blocks, st);
    if (b->x_dtype == FMARL_T_F32)
        return b->dtype == FMARL_T_BF16 ? launch_block_t<float, __bf16>(a, backward, blocks, st) : launch_block_t<float, _Float16>(a, backward, blocks, st);
    return b->dtype == FMARL_T_BF16 ? launch_block_t<__bf16, __bf16>(a, backward, blocks, st) : launch_block_t<_Float16, _Float16>(a, backward, blocks, st);
}

}  // namespace

extern "C" {

int fmarl_block_norm(const FmarlBlock *b, void *y, void *h, void *stream) {
    if (int rc = block_check(b, "fmarl_block_norm")) return rc;
    if (b->rows == 0) return FMARL_OK;
    if ((b->branch && !y) || (b->pre_norm && !h) || (!b->branch && !b->pre_norm)) return policy_fail(FMARL_EINVAL, "fmarl_block_norm: null argument");
    Block a = block_args(b);
    const int xb = elem_bytes(b->x_dtype), tb = elem_bytes(b->dtype);
    a.y = b->branch ? (char *)y : nullptr; a.h = b->pre_norm ? (char *)h : nullptr;
    a.vec = (b->dim & 3) == 0 && row_aligned(a.x, a.xs, xb) && row_aligned(a.branch, a.bs, tb) && row_aligned(a.gate, a.gs, tb) && row_aligned(a.y, 0, xb) && row_aligned(a.h, 0, tb);
    return launch_block(b, a, false, block_workgroups(b, false), (hipStream_t)stream);
}

size_t fmarl_block_norm_workspace(const FmarlBlock *b) {
    if (block_check(b, "fmarl_block_norm_workspace")) return 0;
    return (size_t)block_workgroups(b, true) * 5 * b->dim * 4;
}

int fmarl_block_norm_backward(const FmarlBlock *b, const void *d_y, int64_t d_y_stride, const void *d_h, int64_t d_h_stride, void *d_x, void *d_branch,
                              void *d_gate, float *const *d_weights, void *workspace, void *stream) {
    if (int rc = block_check(b, "fmarl_block_norm_backward")) return rc;
    if (!workspace || !d_weights) return policy_fail(FMARL_EINVAL, "fmarl_block_norm_backward: null argument");
    if (b->rows > 0 && (!d_x || (b->branch && !d_branch) || (b->gate && !d_gate))) return policy_fail(FMARL_EINVAL, "fmarl_block_norm_backward: null argument");
    if (d_h && !b->pre_norm) return policy_fail(FMARL_EINVAL, "fmarl_block_norm_backward: d_h without pre_norm");
    Block a = block_args(b);
    const int xb = elem_bytes(b->x_dtype), tb = elem_bytes(b->dtype);
    a.dy = (const char *)d_y; a.dys = d_y_stride; a.dh = (const char *)d_h; a.dhs = d_h_stride;
    a.dx = (char *)d_x; a.dbranch = (char *)d_branch; a.dgate = (char *)d_gate; a.partial = (float *)workspace;
    a.vec = (b->dim & 3) == 0 && row_aligned(a.x, a.xs, xb) && row_aligned(a.branch, a.bs, tb) && row_aligned(a.gate, a.gs, tb) && row_aligned(a.dy, a.dys, xb) &&
            row_aligned(a.dh, a.dhs, tb) && row_aligned(a.dx, 0, xb) && row_aligned(a.dbranch, 0, tb) && row_aligned(a.dgate, 0, tb);
    const int blocks = block_workgroups(b, true);
    if (int rc = launch_block(b, a, true, blocks, (hipStream_t)stream)) return rc;
    BlockSums s = {};
    bool any = false;
    for (int k = 0; k < 5; ++k) { s.out[k] = d_weights[k]; any = any || d_weights[k]; }
    if (any) {
        s.partial = (const float *)workspace; s.dim = b->dim; s.parts = blocks;
        hipLaunchKernelGGL(block_sums_kernel, dim3((5 * b->dim + 7) / 8), dim3(256), 0, (hipStream_t)stream, s);
        HIP_OK(hipGetLastError());
    }
    return FMARL_OK;
}

}  // extern "C"
