// Log-probability and entropy of discrete actions from the policy's features on gfx950, without keeping the logits:
//     z = x W^T + bias, -inf where an action is not available;   log_prob = z_a - lse,  entropy = lse - sum_v p_v z_v,  p = e^{z - lse}
//     dz_v = dlog_prob (1[v = a] - p_v) - dentropy p_v (log p_v + entropy);   dx = dz W,  dW = dz^T x,  dbias = sum dz.
// Rows that take no part (a negative action: padding; nothing available) give 0, 0 and no gradient.  The logits are formed again for the
// gradient.  Two ways to do it:
//   * few actions (five per agent: the env's own): one pass over x per direction, W in LDS, bound by HBM -- actions_few_kernel;
//   * many (the joint actions of several agents): matrix products on the matrix units whose epilogues hold the softmax's running maximum and
//     sums (forwards) or write dz for a piece of the actions at a time (backwards) -- actions_wide_kernel, and actions_gemm_kernel for float32.
#include "fmarl_policy_dev.h"

namespace fmarl {
namespace policy {

constexpr float kLog2e = 1.44269504f;

struct Actions {
    int64_t rows;
    int K, V, act_type, avail_u8, xvec, dxvec;
    const char *x; int64_t xs;
    const char *w; int64_t ws;
    const float *bias;
    const void *act;
    const void *avail; int64_t as;
    float *logp, *ent, *lse;                          // forward outputs; backward: ent and lse are read
    const float *dlogp, *dent;                        // NULL: zeros
    char *dx;
    float *partial;                                   // (workgroups, V * K + V)
};

// negative: the row takes no part; V and beyond (a NaN too): no such action
__device__ __forceinline__ int action_of(const Actions &a, int64_t row) {
    if (a.act_type == 0) {
        const int64_t v = ((const int64_t *)a.act)[row];
        return v < 0 ? -1 : v > 0x7fffffff ? 0x7fffffff : (int)v;
    }
    if (a.act_type == 1) return ((const int32_t *)a.act)[row];
    const float f = ((const float *)a.act)[row];
    return f < 0.f ? -1 : f < 2147483000.f ? (int)f : 0x7fffffff;
}

// which of the actions v .. v + 3 exist and are available to a row, as bits.  Loads at clamped places and selects, no branch per action: the four loads leave
// together.  (A branch per action around `z = -inf` was dropped by the compiler, ROCm 7.2: the condition was formed and the assignment left out.)
__device__ __forceinline__ uint32_t available4(const Actions &a, int64_t row, int v) {
    const bool real = row < a.rows;
    uint32_t bits = 0;
    if (a.avail) {
        const int64_t at = (real ? row : a.rows - 1) * a.as;
        if (a.avail_u8) {
#pragma unroll
            for (int r = 0; r < 4; ++r) bits |= ((const uint8_t *)a.avail)[at + min(v + r, a.V - 1)] != 0 ? 1u << r : 0u;
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) bits |= ((const float *)a.avail)[at + min(v + r, a.V - 1)] != 0.f ? 1u << r : 0u;
        }
    } else bits = 15u;
    const int left = real ? a.V - v : 0;
    return bits & (left >= 4 ? 15u : left > 0 ? (1u << left) - 1 : 0u);
}

__device__ __forceinline__ float exp_of(float x) { return exp2_fast(x * kLog2e); }

// what the tiles' (max, sum e^{z - max}, sum (z - max) e^{z - max}) say of a row, logits in units of `unit`; top == -inf and !some: nothing available
__device__ __forceinline__ void row_result(const Actions &a, int64_t row, int act, float top, float s, float t, bool some, float za, float unit) {
    float lp = 0.f, en = 0.f, ls = __builtin_inff();
    if (act >= 0 && some) {
        const float l = logf(s);
        lp = (za - top) * unit - l; en = l - t * unit / s; ls = top * unit + l;   // (the difference first: 0 where the action is the largest, however far out)
        if (act >= a.V) { lp = en = __builtin_nanf(""); ls = __builtin_inff(); }   // no such action: seen in the result, without a gradient
    }
    a.logp[row] = lp; a.ent[row] = en; a.lse[row] = ls;
}

// dz of one logit; `in`: the row takes part
__device__ __forceinline__ float dlogit(float z, bool hot, bool in, float lse, float ent, float dl, float de) {
    const float lp = z - lse, p = exp_of(lp), d = dl * ((hot ? 1.f : 0.f) - p) - de * (p * (lp + ent));
    return in && z != -__builtin_inff() ? d : 0.f;
}

// ---- few actions ------------------------------------------------------------------------------------------------------------
// 16 rows a wave at a time, logits as z^T = W x^T in the accumulator layout of mfma_f32_16x16x4f32 (row 4 * (lane / 16) + r: action, column lane % 16: row of
// x), so a row's softmax is over a lane's registers and two lane exchanges, and dx^T = W^T dz^T takes dz^T as it lies.  VT * 16 >= V, KT * 16 >= K.  x is loaded
// once, in float4s; float32 products for every type.  The gradient of W is summed over a wave's tiles in registers, over the workgroup in LDS and
// over the workgroups by actions_sums_kernel, always in the same order.  2 097 152 rows of 64 float32, five actions: 131 us forwards back to back (4.4 TB/s; 152 between other passes), 227 + 5 us backwards (4.9 TB/s).
template <typename T, int VT, int KT, bool BACK, bool VEC>
__global__ __launch_bounds__(256) void actions_few_kernel(Actions a) {
    constexpr int PK = 16 * KT + 4;
    __shared__ __align__(16) float lw[16 * VT * PK], lb[16 * VT];
    __shared__ __align__(16) float lx[BACK ? 4 * 16 * PK : 4], lt[BACK ? 4 * 16 * 20 : 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g4 = (lane >> 4) * 4;
    for (int i = threadIdx.x; i < 16 * VT * PK; i += 256) {
        const int v = i / PK, k = i % PK;
        lw[i] = v < a.V && k < a.K ? (float)((const T *)a.w)[v * a.ws + k] : 0.f;
    }
    for (int v = threadIdx.x; v < 16 * VT; v += 256) lb[v] = a.bias && v < a.V ? a.bias[v] : 0.f;
    __syncthreads();
    float *wx = lx + (BACK ? wave * 16 * PK : 0), *wt = lt + (BACK ? wave * 16 * 20 : 0);
    f32x4 accw[BACK ? VT : 1][BACK ? KT : 1], accb[BACK ? VT : 1];
    if (BACK)
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            accb[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KT; ++k) accw[j][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    const int64_t tiles = (a.rows + 15) / 16, step = (int64_t)gridDim.x * 4;
    typedef typename Vec4<T>::type V4;
    V4 next[KT];
    int next_act = -1;
    float next_lse = 0.f, next_ent = 0.f, next_dl = 0.f, next_de = 0.f;
    auto fetch = [&](int64_t tile) {   // in flight while the tile before is computed
        const int64_t row = tile * 16 + c, at = min(row, a.rows - 1);
        next_act = action_of(a, at);
        if (BACK) { next_lse = a.lse[at]; next_ent = a.ent[at]; if (a.dlogp) next_dl = a.dlogp[at]; if (a.dent) next_de = a.dent[at]; }
#pragma unroll
        for (int k = 0; k < KT; ++k) next[k] = load4<T>((const T *)a.x + row * a.xs + 16 * k + g4, row < a.rows ? a.K - 16 * k - g4 : 0, VEC);
    };
    int64_t tile = (int64_t)blockIdx.x * 4 + wave;
    if (tile < tiles) fetch(tile);
    for (; tile < tiles; tile += step) {
        const int64_t row = tile * 16 + c;
        const bool real = row < a.rows;
        f32x4 x[KT], z[VT];
#pragma unroll
        for (int k = 0; k < KT; ++k) x[k] = widen(next[k]);
        const int act = real ? next_act : -1;
        const float lse = next_lse, ent = next_ent, dl = next_dl, de = next_de;
        if (tile + step < tiles) fetch(tile + step);
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            z[j] = *(const f32x4 *)(lb + 16 * j + g4);
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const f32x4 w = *(const f32x4 *)(lw + (16 * j + c) * PK + 16 * k + g4);
#pragma unroll
                for (int r = 0; r < 4; ++r) z[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], x[k][r], z[j], 0, 0, 0);
            }
            const uint32_t ok = available4(a, row, 16 * j + g4);
#pragma unroll
            for (int r = 0; r < 4; ++r) z[j][r] = (ok >> r) & 1 ? z[j][r] : -__builtin_inff();
        }
        if (!BACK) {
            float top = -__builtin_inff(), s = 0.f, t = 0.f, za = 0.f;
            bool some = false;
#pragma unroll
            for (int j = 0; j < VT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) { top = fmaxf(top, z[j][r]); some |= !(z[j][r] == -__builtin_inff()); }
            top = lanes_max<16>(top, 64);
#pragma unroll
            for (int j = 0; j < VT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool none = z[j][r] == -__builtin_inff();
                    const float d = none ? 0.f : z[j][r] - top, e = none ? 0.f : exp_of(d);
                    s += e; t += d * e;
                    za = 16 * j + g4 + r == act ? z[j][r] : za;
                }
            s = lanes_sum<16>(s, 64); t = lanes_sum<16>(t, 64); za = lanes_sum<16>(za, 64);
            const float any = lanes_max<16>(some ? 1.f : 0.f, 64);
            if (lane < 16 && real) row_result(a, row, act, top, s, t, any != 0.f, za, 1.f);
        } else {
            const bool in = real && lse != __builtin_inff();
#pragma unroll
            for (int j = 0; j < VT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) z[j][r] = dlogit(z[j][r], 16 * j + g4 + r == act, in, lse, ent, dl, de);
            wave_sync();
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                *(f32x4 *)(wx + c * PK + 16 * k + g4) = in ? x[k] : f32x4{0.f, 0.f, 0.f, 0.f};   // what a padded row holds (NaN too) does not reach dW
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < VT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o = __builtin_amdgcn_mfma_f32_16x16x4f32(lw[(16 * j + g4 + r) * PK + 16 * k + c], z[j][r], o, 0, 0, 0);
                if (real) store4<T>((T *)a.dx + row * a.K + 16 * k + g4, o, a.K - 16 * k - g4, VEC);
            }
#pragma unroll
            for (int j = 0; j < VT; ++j) {
                accb[j] += z[j];
                *(f32x4 *)(wt + c * 20 + g4) = z[j];
                wave_sync();
                float d[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) d[r] = wt[(g4 + r) * 20 + c];
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) accw[j][k] = __builtin_amdgcn_mfma_f32_16x16x4f32(d[r], wx[(g4 + r) * PK + 16 * k + c], accw[j][k], 0, 0, 0);
                wave_sync();
            }
        }
    }
    if (BACK) {
        // the four waves' sums one after the other, through W's place in LDS
        float *mine = a.partial + (int64_t)blockIdx.x * ((int64_t)a.V * a.K + a.V);
        __syncthreads();
        for (int w = 0; w < 4; ++w) {
            if (wave == w) {
#pragma unroll
                for (int j = 0; j < VT; ++j) {
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float *p = lw + (16 * j + g4 + r) * PK + 16 * k + c;
                            *p = w ? *p + accw[j][k][r] : accw[j][k][r];
                        }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float s = accb[j][r];
                        s = lanes_sum<1>(s, 16);
                        if (c == 0) lb[16 * j + g4 + r] = w ? lb[16 * j + g4 + r] + s : s;
                    }
                }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < a.V * a.K; i += 256) mine[i] = lw[(i / a.K) * PK + i % a.K];
        for (int v = threadIdx.x; v < a.V; v += 256) mine[(int64_t)a.V * a.K + v] = lb[v];
    }
}

// sums over the workgroups: 16 entries a workgroup, 16 threads an entry, float64, a fixed order
template <typename T>
__global__ __launch_bounds__(256) void actions_sums_kernel(const float *partial, int parts, int64_t n, int64_t nw, T *dw, float *db) {
    __shared__ double red[16][17];
    const int c = threadIdx.x & 15, s = threadIdx.x >> 4;
    const int64_t i = (int64_t)blockIdx.x * 16 + c;
    double sum = 0.0;
    if (i < n)
#pragma unroll 16
        for (int p = s; p < parts; p += 16) sum += (double)partial[p * n + i];
    red[s][c] = sum;
    __syncthreads();
    if (s == 0 && i < n) {
        for (int k = 1; k < 16; ++k) sum += red[k][c];
        if (i < nw) dw[i] = (T)(float)sum;
        else if (db) db[i - nw] = (float)sum;
    }
}

// ---- many actions -----------------------------------------------------------------------------------------------------------
// dst (rows_pad, cols_pad) <- src (rows, cols; row stride), zeros around, and trans <- its transpose where wanted; with `lse` without the rows that take no
// part (what they hold, NaN too, does not reach dW).  64 x 64 tiles; up to two matrices of the same columns in a launch, the first one's `blocks` tiles of rows first.
struct PackJob { const char *src; int64_t stride, rows, rows_pad; char *dst, *trans; const float *lse; };

template <typename T>
__global__ __launch_bounds__(256) void actions_pack_kernel(PackJob j0, PackJob j1, int blocks, int cols, int cols_pad) {
    __shared__ T tile[64][66];
    const bool second = (int)blockIdx.x >= blocks;
    const T *src = (const T *)(second ? j1.src : j0.src);
    T *dst = (T *)(second ? j1.dst : j0.dst), *trans = (T *)(second ? j1.trans : j0.trans);
    const float *lse = second ? j1.lse : j0.lse;
    const int64_t stride = second ? j1.stride : j0.stride, rows = second ? j1.rows : j0.rows, rows_pad = second ? j1.rows_pad : j0.rows_pad;
    const int64_t r0 = (int64_t)(second ? blockIdx.x - blocks : blockIdx.x) * 64;
    const int c0 = blockIdx.y * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6, at = min(c0 + tx, cols - 1);
    T v[16];
    float l[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {   // every load is made, from a row and a column that are there, so that all are in flight
        const int64_t r = min(r0 + ty + 4 * i, rows - 1);
        v[i] = src[r * stride + at];
        l[i] = lse ? lse[r] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = r0 + ty + 4 * i;
        const T w = r < rows && c0 + tx < cols && l[i] != __builtin_inff() ? v[i] : (T)0.f;
        dst[r * cols_pad + c0 + tx] = w;
        if (trans) tile[ty + 4 * i][tx] = w;
    }
    if (trans) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) trans[(int64_t)(c0 + ty + 4 * i) * rows_pad + r0 + tx] = tile[tx][ty + 4 * i];
    }
}

enum { kStore = 0, kStats = 1, kDlogits = 2 };

struct Gemm {
    const char *A, *B;             // rows of lda / ldb elements, 128-byte steps of the contraction contiguous; both padded to whole tiles
    int64_t lda, ldb;
    int ta, tb, splits, steps;     // 128-row tiles of A and B, parts of the contraction, 128-byte steps in all
    float *out; int64_t ldo, split_out;     // kStore: out[split][row of B][row of A]
    Actions act;                   // kStats, kDlogits: A = W (actions), B = x (rows); row0 / v0: where the tiles begin in them
    int64_t row0; int v0;
    float *stats; int64_t stat_stride;      // kStats: (slots of 64 actions, 3, stat_stride)
    float *za;                     // kStats: the taken action's logit, by row of the chunk
    char *dz, *dzt; int64_t ldz, ldzt;      // kDlogits: dz (rows, ldz) and its transpose
    float *db; int64_t ldb_part;   // kDlogits: (tiles of 64 rows, ldb_part) sums over the rows
};

template <typename T> struct Frag;
template <> struct Frag<float> {   // four steps of four: the order of the contraction is free as long as both sides share it
    typedef f32x4 type;
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
#pragma unroll
        for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
        return c;
    }
};

// Tiles of 128 x 128, four waves of 64 x 64, steps of 128 bytes along the contraction.  A step's rows go from memory straight to LDS (16 bytes a
// lane, 64 lanes side by side), the next step's while this one is multiplied.  The LDS image is linear -- the hardware writes lane after lane --
// so the 16-byte pieces of a row are permuted on the way in by the addresses the lanes load from (piece p of row r lies in place p ^ (r & 7)): the 16 rows that
// a fragment read touches then spread over the banks.  12 345 x 100 x 625 float32: 27 us a product, 36 us with the softmax's sums, 48 us with dz and its transpose
// written (64 MB): the four steps of a tile (K = 100) do not hide what stands before and behind them.
template <typename T, int EPI>
__global__ __launch_bounds__(256) void actions_gemm_kernel(Gemm q) {
    constexpr int kTile = 128 * 128;                                           // bytes of one operand's step
    constexpr int PZ = 128 + 16 / (int)sizeof(T);                              // kDlogits: row of the transposing buffer, elements
    constexpr int kLds = EPI == kDlogits && 128 * PZ * (int)sizeof(T) > 4 * kTile ? 128 * PZ * (int)sizeof(T) : 4 * kTile;
    __shared__ __align__(128) char lds[kLds];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4, g4 = g * 4;
    // workgroups go round the eight XCDs in turn: each XCD takes a run of neighbouring tiles, whose operands its L2 then holds
    const int n = q.ta * q.tb * q.splits, per = n / 8, extra = n % 8, xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
    int id = xcd * per + min(xcd, extra) + nth;
    const int ia = id % q.ta; id /= q.ta;
    const int ib = id % q.tb, split = id / q.tb;
    const int s0 = (int)((int64_t)q.steps * split / q.splits), s1 = (int)((int64_t)q.steps * (split + 1) / q.splits);
    const char *pa = q.A + (int64_t)ia * 128 * q.lda * sizeof(T), *pb = q.B + (int64_t)ib * 128 * q.ldb * sizeof(T);
    const int lr = lane >> 3, lp = (lane & 7) ^ lr;                            // row and piece this lane loads of each eight rows
    auto load = [&](int s, int buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (wave * 4 + i) * 8;
            const char *ga = pa + ((int64_t)(r + lr) * q.lda) * sizeof(T) + (int64_t)s * 128 + lp * 16;
            const char *gb = pb + ((int64_t)(r + lr) * q.ldb) * sizeof(T) + (int64_t)s * 128 + lp * 16;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)ga, (__attribute__((address_space(3))) void *)(lds + buf * 2 * kTile + r * 128), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)gb, (__attribute__((address_space(3))) void *)(lds + buf * 2 * kTile + kTile + r * 128), 16, 0, 0);
        }
    };
    const int ra = (wave & 1) * 64, rb = (wave >> 1) * 64;
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s0 < s1) load(s0, 0);
    for (int s = s0; s < s1; ++s) {
        const int buf = (s - s0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's share of the step is in LDS
        __syncthreads();                                   // everybody's is, and nobody reads the other buffer any more
        if (s + 1 < s1) load(s + 1, buf ^ 1);
        const char *la = lds + buf * 2 * kTile, *lb = la + kTile;
        typedef typename Frag<T>::type F;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            F fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fa[i] = *(const F *)(la + (ra + 16 * i + c) * 128 + (((kk * 4 + g) ^ (c & 7)) * 16));
                fb[i] = *(const F *)(lb + (rb + 16 * i + c) * 128 + (((kk * 4 + g) ^ (c & 7)) * 16));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = Frag<T>::mma(fa[i], fb[j], acc[i][j]);
        }
    }
    if (EPI == kStore) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float *o = q.out + split * q.split_out + ((int64_t)ib * 128 + rb + 16 * j + c) * q.ldo + (int64_t)ia * 128 + ra + g4;
#pragma unroll
            for (int i = 0; i < 4; ++i) *(f32x4 *)(o + 16 * i) = acc[i][j];
        }
        return;
    }
    const Actions &a = q.act;
    const int vbase = q.v0 + ia * 128 + ra + g4;
    float bias[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) { const int v = vbase + 16 * i + r; bias[i][r] = a.bias && v < a.V ? a.bias[v] : 0.f; }
    if (EPI == kDlogits) __syncthreads();   // the operands' LDS is dead from here on
    float dbs[4][4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t m = (int64_t)ib * 128 + rb + 16 * j + c, row = q.row0 + m;   // row of the chunk, row of x
        const bool real = row < a.rows;
        const int act = real ? action_of(a, row) : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t ok = available4(a, row, vbase + 16 * i);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = (ok >> r) & 1 ? acc[i][j][r] + bias[i][r] : -__builtin_inff();
        }
        if (EPI == kStats) {
            float top = -__builtin_inff(), s = 0.f, t = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float z = acc[i][j][r];
                    top = fmaxf(top, z != z ? __builtin_inff() : z);      // a NaN is not passed over: it makes the sums NaN
                    if (vbase + 16 * i + r == act) q.za[m] = z;
                }
            top = lanes_max<16>(top, 64);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool none = acc[i][j][r] == -__builtin_inff();
                    const float d = none ? 0.f : acc[i][j][r] - top, e = none ? 0.f : exp_of(d);
                    s += e; t += d * e;
                }
            s = lanes_sum<16>(s, 64); t = lanes_sum<16>(t, 64);
            if (g == 0 && real) {
                float *o = q.stats + (int64_t)(ia * 2 + (wave & 1)) * 3 * q.stat_stride + m;
                o[0] = top; o[q.stat_stride] = s; o[2 * q.stat_stride] = t;
            }
        } else {
            float lse = 0.f, ent = 0.f, dl = 0.f, de = 0.f;
            if (real) { lse = a.lse[row]; ent = a.ent[row]; dl = a.dlogp ? a.dlogp[row] : 0.f; de = a.dent ? a.dent[row] : 0.f; }
            const bool in = real && lse != __builtin_inff();
            T *zrow = (T *)lds + (rb + 16 * j + c) * PZ + ra + g4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 d;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    d[r] = dlogit(acc[i][j][r], vbase + 16 * i + r == act, in, lse, ent, dl, de);
                    dbs[i][r] += d[r];
                }
                store4<T>(zrow + 16 * i, d, 4, true);
            }
        }
    }
    if (EPI == kDlogits) {
        // sums over this wave's 64 rows, from the unrounded values
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float s = dbs[i][r];
                s = lanes_sum<1>(s, 16);
                if (c == 0) q.db[(int64_t)(ib * 2 + (wave >> 1)) * q.ldb_part + ia * 128 + ra + 16 * i + g4 + r] = s;
            }
        __syncthreads();
        constexpr int W = 16 / sizeof(T), kPer = 128 / W;   // elements per 16-byte piece, pieces per row
        typedef typename Frag<T>::type P;
        const T *zl = (const T *)lds;
        for (int i = threadIdx.x; i < 128 * kPer; i += 256) {
            const int r = i / kPer, p = i % kPer;
            *(P *)((T *)q.dz + ((int64_t)ib * 128 + r) * q.ldz + ia * 128 + p * W) = *(const P *)(zl + r * PZ + p * W);
        }
        for (int i = threadIdx.x; i < 128 * kPer; i += 256) {
            const int v = i % 128, p = i / 128;   // neighbouring lanes: neighbouring columns of the buffer
            P o;
#pragma unroll
            for (int e = 0; e < W; ++e) o[e] = zl[(p * W + e) * PZ + v];
            *(P *)((T *)q.dzt + ((int64_t)ia * 128 + v) * q.ldzt + (int64_t)ib * 128 + p * W) = o;
        }
    }
}

// ---- many actions, half precision -------------------------------------------------------------------------------------------
// Tiles of 256 x 256 by eight waves of 128 x 64 (a wave's fragments are then read 0.75 times as fast as LDS can give them while its matrix instructions run), steps of
// 32 along the contraction, 32 KB each; four of them have room in LDS, so three are on their way -- over the end of a tile into the next one's -- while one is multiplied.
// They go from memory straight to LDS (16 bytes a lane, 64 lanes side by side).  The compiler waits for every such load before the next LDS read of any kind (it
// took the loads of the next step for possible writers of this step's: 107 us for dx at 8 192 x 256 x 15 625 with two steps of 64), so they are issued in
// assembly -- they have no result registers -- and waited for by count before the barrier: loads come back in order, and of those behind a step's at most eight are open.
// The LDS image is linear -- the hardware writes lane after lane -- so its 16-byte pieces are permuted by the addresses that the lanes load from, such that what a
// fragment read touches spreads over the banks.
//   an operand whose contraction is contiguous: 256 rows of 64 bytes, piece p of row r in place p ^ ((r >> 2) & 3), a fragment is one 16-byte read;
//   an operand whose rows are the contraction (T): 32 rows of 512 bytes, piece p of row r in place p ^ f(r), f(r) = 2 ((r & 3) + 4 (r >> 3)); a fragment is two
//   transposing reads (ds_read_b64_tr_b16: 16 lanes point at four rows of 16 and get a column each).  So dz, x and W serve both of their products as they lie.
// What an epilogue needs per action and per row comes the same way, with the first step of its tile: a load of its own would be waited for behind all steps on
// their way.  Logits are formed in base 2: v_exp_f32 is a power of two, and z log2(e) - max one multiply-add.
// 8 192 x 256 x 15 625 bfloat16, 65.5 GFLOP a product: dx 87 us, dW 75 us (753, 873 TFLOP/s; a large product by the library 1 085), with the softmax's sums 113 us, with dz
// written 152 us: their epilogues (an exponential per logit; 256 MB of dz) are not hidden behind the matrix instructions.
struct Wide {
    const char *A, *B; int64_t lda, ldb;     // elements; whole tiles can be read
    int ta, tb, steps, splits;               // tiles of A and of B, steps of the contraction; kStore: parts of the contraction, else parts of the outer tile's run
    float *out; int64_t ldo, split_out;      // kStore: out[split][row of B][row of A]
    Actions act; int64_t row0; int v0;       // kStats, kDlogits: A = W (actions from v0 on), B = x (rows from row0 on)
    const float *bias2;                      // bias log2(e) of the padded actions from v0 on, -inf beyond the last one
    const int *taken;                        // the rows' actions of the chunk, -1: takes no part; padded to whole tiles
    const f32x4 *rows;                       // kDlogits: what the rows' gradients are made of (actions_rows_kernel), padded to whole tiles
    float *stats; int64_t stat_stride;       // kStats: (2 splits, 3, stat_stride)
    float *za;                               // kStats: the taken action's logit in base 2, by row of the chunk
    char *dz; int64_t ldz;                   // kDlogits: (rows, ldz)
    float *db; int64_t ldb_part;             // kDlogits: (tiles of 64 rows, ldb_part) sums over the rows
    const float *dz_scale;                   // kDlogits: NULL or the power of two that dz is stored times
};

template <typename T> struct Half;
template <> struct Half<__bf16> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Half<_Float16> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kWideOperand = 16384, kWideStep = 2 * kWideOperand, kWideExtra = 6144;   // bytes of an operand's step, of a step, of what a tile's epilogue needs: bias 1 KB, actions 1 KB, rows 4 KB
constexpr int kWideLds = 4 * (kWideStep + kWideExtra);                                  // 152 KB of the CU's 160

// 16 bytes a lane from memory to LDS, lane after lane from byte `at` on (the same in every lane)
__device__ __forceinline__ void load_lds(const char *p, uint32_t at) {
    uint32_t m0;   // put back as it was: the compiler does not expect it to change
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0" : "=&s"(m0) : "s"(at), "v"(p) : "memory");
}

// What a row's gradient is made of: (lse log2(e), A, B, dlog_prob), dz = p (log2(p) A + B) + dlog_prob [v = a], A = -de ln 2, B = -(dlog_prob + de H), times the power of
// two of `scale`; and its action.  Rows that take no part: 3e38, 0, 0, 0 and -1.
__global__ __launch_bounds__(256) void actions_rows_kernel(Actions a, int64_t row0, int64_t padded, f32x4 *rows, int *taken, const float *scale) {
    const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x, row = row0 + m;
    if (m >= padded) return;
    f32x4 v = {3e38f, 0.f, 0.f, 0.f};
    int act = -1;
    if (row < a.rows) {
        act = action_of(a, row);
        if (rows) {
            const float lse = a.lse[row], s = scale ? *scale : 1.f;
            if (lse != __builtin_inff()) {
                const float de = a.dent ? a.dent[row] * s : 0.f, dl = a.dlogp ? a.dlogp[row] * s : 0.f;
                // a row of lowest biases only: exactly where actions_bias2_kernel leaves its logits, so that their difference is 0
                const float lse2 = lse <= -2.3e38f ? -3.4028234e38f : lse * kLog2e;
                v = f32x4{lse2, de * -0.693147181f, lse != lse ? lse : -(dl + de * a.ent[row]), dl};   // logits that hold a NaN: a gradient of NaN
            } else act = -1;
        }
    }
    taken[m] = act;
    if (rows) rows[m] = v;
}

template <typename T, int EPI, bool TA, bool TB, bool AVAIL>
__global__ __launch_bounds__(512) void actions_wide_kernel(Wide q) {
    extern __shared__ __align__(128) char lds[];
    typedef typename Half<T>::frag F;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4, g4 = g * 4;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uint64_t)(__attribute__((address_space(3))) char *)lds);
    // workgroups go round the eight XCDs in turn: each XCD takes a run of neighbouring work, whose operands its L2 then holds
    const int n = gridDim.x, per = n / 8, extra = n % 8, xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
    const int id = xcd * per + min(xcd, extra) + nth;
    // kStore: one tile and a part of the contraction.  kStats: one tile of rows (B) and a run of the actions' tiles (A); kDlogits: one tile of actions and a run of the
    // rows' tiles -- what is summed over the run stays in registers.
    int ia, ib, split, tiles = 1, s0 = 0, s1 = q.steps;
    if (EPI == kStore) {
        ia = id % q.ta; ib = id / q.ta % q.tb; split = id / (q.ta * q.tb);
        s0 = (int)((int64_t)q.steps * split / q.splits); s1 = (int)((int64_t)q.steps * (split + 1) / q.splits);
    } else if (EPI == kStats) {
        ib = id % q.tb; split = id / q.tb;
        ia = (int)((int64_t)q.ta * split / q.splits); tiles = (int)((int64_t)q.ta * (split + 1) / q.splits) - ia;
    } else {
        ia = id % q.ta; split = id / q.ta;
        ib = (int)((int64_t)q.tb * split / q.splits); tiles = (int)((int64_t)q.tb * (split + 1) / q.splits) - ib;
    }
    const int steps = s1 - s0, total = steps * tiles;
    // this lane's addresses of a step, from the tile's start: two pieces of each operand per wave
    int64_t fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rn = (wave * 2 + i) * 16 + (lane >> 2), pn = (lane & 3) ^ ((lane >> 4) & 3);                          // contiguous contraction: row and piece
        const int rt = (wave * 2 + i) * 2 + (lane >> 5), pt = (lane & 31) ^ (2 * ((rt & 3) + 4 * (rt >> 3)));            // T
        fa[i] = TA ? (int64_t)rt * q.lda * 2 + pt * 16 : (int64_t)rn * q.lda * 2 + pn * 16;
        fb[i] = TB ? (int64_t)rt * q.ldb * 2 + pt * 16 : (int64_t)rn * q.ldb * 2 + pn * 16;
    }
    const int64_t step_a = TA ? 32 * q.lda * 2 : 64, step_b = TB ? 32 * q.ldb * 2 : 64, tile_a = TA ? 512 : 256 * q.lda * 2, tile_b = TB ? 512 : 256 * q.ldb * 2;
    const char *pa0 = q.A + ia * tile_a + s0 * step_a, *pb0 = q.B + ib * tile_b + s0 * step_b;
    int lk = 0, ls = 0, lt = 0;   // the next step to load: of the run, of its tile, its tile of the run
    auto load = [&]() {
        const char *pa = pa0 + (EPI == kStats ? lt * tile_a : 0) + ls * step_a, *pb = pb0 + (EPI == kDlogits ? lt * tile_b : 0) + ls * step_b;
        const uint32_t at = lds0 + (lk & 3) * kWideStep + wave * 2048;
        if (EPI != kStore && ls == 0) {   // what the tile's epilogue needs: 256 biases (wave 0), 256 actions (wave 1), 256 rows (waves 2 .. 5)
            const uint32_t to = lds0 + 4 * kWideStep + (lt & 3) * kWideExtra;
            const int64_t v = (int64_t)(EPI == kStats ? ia + lt : ia) * 256, m = (int64_t)(EPI == kDlogits ? ib + lt : ib) * 256;
            if (wave == 0) load_lds((const char *)(q.bias2 + v) + lane * 16, to);
            else if (wave == 1) load_lds((const char *)(q.taken + m) + lane * 16, to + 1024);
            else if (EPI == kDlogits && wave < 6) load_lds((const char *)(q.rows + m) + (wave - 2) * 1024 + lane * 16, to + wave * 1024);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            load_lds(pa + fa[i], at + i * 1024);
            load_lds(pb + fb[i], at + kWideOperand + i * 1024);
        }
        ++lk;
        if (++ls == steps) { ls = 0; ++lt; }
    };
    const int ra = (wave & 1) * 128, rb = (wave >> 1) * 64;
    auto fragment = [&](const char *at, bool t, int row) -> F {   // rows (T: columns) row .. row + 15 of a step
        if (!t) return *(const F *)(at + (row + c) * 64 + ((g ^ ((c >> 2) & 3)) * 16));
        const int f = 2 * ((c >> 2) + 4 * g);
        const char *p = at + (8 * g + (c >> 2)) * 512 + ((((row >> 3) ^ f) | ((c >> 1) & 1)) * 16) + (c & 1) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p + 4 * 512));
        return __builtin_bit_cast(F, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    const Actions &a = q.act;
    // kStats: this lane's running maximum and sums of its four rows
    float top[4], sum[4], tsum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { top[j] = -__builtin_inff(); sum[j] = tsum[j] = 0.f; }
    const float inv_scale = EPI == kDlogits && q.dz_scale ? 1.f / *q.dz_scale : 1.f;
    f32x4 acc[8][4];
    for (int i = 0; i < 3 && lk < total; ++i) load();
    int k = 0;
    for (int tile = 0; tile < tiles; ++tile) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < steps; ++s, ++k) {
            // this wave's share of step k is in LDS once at most the four loads of each step behind it are open; behind the barrier everybody's is, and nobody reads step
            // k - 1 any more, whose place the next load takes
            if (k + 2 < total) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
            else if (k + 1 < total) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (lk < total) load();
            const char *la = lds + (k & 3) * kWideStep, *lb = la + kWideOperand;
            F fb_[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) fb_[j] = fragment(lb, TB, rb + 16 * j);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const F fa_ = fragment(la, TA, ra + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = Half<T>::mma(fa_, fb_[j], acc[i][j]);
            }
        }
        if (EPI == kStore) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float *o = q.out + split * q.split_out + ((int64_t)ib * 256 + rb + 16 * j + c) * q.ldo + (int64_t)ia * 256 + ra + g4;
#pragma unroll
                for (int i = 0; i < 8; ++i) *(f32x4 *)(o + 16 * i) = acc[i][j];
            }
            continue;
        }
        const char *more = lds + 4 * kWideStep + (tile & 3) * kWideExtra;
        const int va = (EPI == kStats ? ia + tile : ia) * 256 + ra + g4;   // this lane's actions of the chunk: va + 16 i + r
        const int64_t m0 = (int64_t)(EPI == kDlogits ? ib + tile : ib) * 256 + rb + c;   // its rows of the chunk: m0 + 16 j
        int want[4];   // the taken action among this lane's: want = 16 i + r
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = ((const int *)(more + 1024))[rb + 16 * j + c];
            want[j] = t < 0 ? -1 : t - q.v0 - va;
        }
        // z log2(e) + bias, -inf beyond the last action and where not available
        auto logits = [&](int i, int j, f32x4 bv) {
            f32x4 z;
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] = __builtin_fmaf(acc[i][j][r], kLog2e, bv[r]);
            if (AVAIL) {
                const uint32_t ok = available4(a, q.row0 + m0 + 16 * j, q.v0 + va + 16 * i);
#pragma unroll
                for (int r = 0; r < 4; ++r) z[r] = (ok >> r) & 1 ? z[r] : -__builtin_inff();
            }
            return z;
        };
        auto bias = [&](int i) { return *(const f32x4 *)(more + (ra + 16 * i + g4) * 4); };
        if (EPI == kStats) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x4 bv = bias(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] = logits(i, j, bv);
                    if ((unsigned)(want[j] - 16 * i) < 4u) {
                        const int r = want[j] - 16 * i;
                        q.za[m0 + 16 * j] = r == 0 ? acc[i][j][0] : r == 1 ? acc[i][j][1] : r == 2 ? acc[i][j][2] : acc[i][j][3];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float most = top[j];
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(fmaxf(most, fmaxf(acc[i][j][0], acc[i][j][1])), fmaxf(acc[i][j][2], acc[i][j][3]));
                const float ref = most == -__builtin_inff() ? 0.f : most;   // nothing yet: no infinity minus infinity
                const float old = top[j] == -__builtin_inff() ? 0.f : exp2_fast(top[j] - ref);
                float s = sum[j] * old, t = old == 0.f ? 0.f : old * (tsum[j] + (top[j] - ref) * sum[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float d = acc[i][j][r] - ref, e = exp2_fast(d);
                        s += e;
                        t += fmaxf(d, -1e4f) * e;   // (-inf times 0)
                    }
                top[j] = most; sum[j] = s; tsum[j] = t;
            }
        } else {
            f32x4 rc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) rc[j] = ((const f32x4 *)(more + 2048))[rb + 16 * j + c];
            T *zrow = (T *)q.dz + m0 * q.ldz + va;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x4 bv = bias(i);
                f32x4 all = {0.f, 0.f, 0.f, 0.f};   // over this wave's 64 rows, unrounded
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 z = logits(i, j, bv);
                    f32x4 d;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = fmaxf(z[r] - rc[j][0], -1e4f);   // log2 p; -1e4: p is 0, and what it is multiplied with is finite
                        d[r] = exp2_fast(x) * __builtin_fmaf(x, rc[j][1], rc[j][2]);
                    }
                    if ((unsigned)(want[j] - 16 * i) < 4u) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) d[r] += want[j] - 16 * i == r && z[r] != -__builtin_inff() ? rc[j][3] : 0.f;
                    }
                    all += d;
                    // rounded to the operands' type: what the two products read.  The gradients' error is then 1.4 times that of their own rounding (8 192 x 256 x 15 625 bfloat16: 0.0023
                    // of their norm, 0.0017 with dz in float32, as here with dz in two pieces, whose second writing and products made the training pass 781 us instead of 475)
                    store4<T>(zrow + 16 * j * q.ldz + 16 * i, d, 4, true);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) all[r] = lanes_sum<1>(all[r], 16);
                if (c == 0) *(f32x4 *)(q.db + (int64_t)((ib + tile) * 4 + (wave >> 1)) * q.ldb_part + va + 16 * i) = all * inv_scale;
            }
        }
    }
    if (EPI == kStats) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // the four lanes of a row, then one slot per wave
            const float m = lanes_max<16>(top[j], 64);
            const float ref = m == -__builtin_inff() ? 0.f : m, f = top[j] == -__builtin_inff() ? (sum[j] == 0.f ? 0.f : 1.f) : exp2_fast(top[j] - ref);
            float s = sum[j] * f, t = f == 0.f ? 0.f : f * (tsum[j] + (top[j] == -__builtin_inff() ? 0.f : top[j] - ref) * sum[j]);
            s = lanes_sum<16>(s, 64); t = lanes_sum<16>(t, 64);
            if (g == 0) {
                float *o = q.stats + (int64_t)(split * 2 + (wave & 1)) * 3 * q.stat_stride + (int64_t)ib * 256 + rb + 16 * j + c;
                o[0] = m; o[q.stat_stride] = s; o[2 * q.stat_stride] = t;
            }
        }
    }
}

__global__ __launch_bounds__(256) void actions_bias2_kernel(const float *bias, int V, float *out, int n) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= n) return;
    const float b = v >= V ? -__builtin_inff() : bias ? bias[v] : 0.f;
    out[v] = b == -__builtin_inff() ? b : fmaxf(b * kLog2e, -3.4028234e38f);   // a bias of the type's lowest value stays a number: its action is there
}

// the row's result from its slots' maxima and sums: 16 rows a workgroup, 16 threads a row.  `two`: maxima, sums and the taken logit are in base 2
__global__ __launch_bounds__(256) void actions_join_kernel(Actions a, const float *stats, int64_t stride, int slots, const float *za, int64_t row0, int64_t count, int two) {
    __shared__ float red[3][16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t m = (int64_t)blockIdx.x * 16 + c;
    float top = -__builtin_inff(), s = 0.f, t = 0.f;
    auto power = [&](float x) { return two ? exp2_fast(x) : exp_of(x); };
    auto add = [&](float t1, float s1, float d1) {
        if (s1 == 0.f) return;              // nothing there (a NaN is not 0)
        if (!(t1 <= top)) {
            const float f = top == -__builtin_inff() ? (s == 0.f ? 0.f : 1.f) : power(top - t1);
            t = f == 0.f ? 0.f : f * (t + (top == -__builtin_inff() ? 0.f : top - t1) * s);
            s *= f; top = t1;
            s += s1; t += d1;
        } else {
            const float f = t1 == -__builtin_inff() ? 1.f : power(t1 - top);
            s += f * s1; t += f == 0.f ? 0.f : f * (d1 + (t1 == -__builtin_inff() ? 0.f : t1 - top) * s1);
        }
    };
    if (m < count)
        for (int i = k; i < slots; i += 16) {
            const float *p = stats + (int64_t)i * 3 * stride + m;
            add(p[0], p[stride], p[2 * stride]);
        }
    red[0][k][c] = top; red[1][k][c] = s; red[2][k][c] = t;
    __syncthreads();
    if (k == 0 && m < count) {
        for (int i = 1; i < 16; ++i) add(red[0][i][c], red[1][i][c], red[2][i][c]);
        const int act = action_of(a, row0 + m);
        const float z = act >= 0 && act < a.V ? za[m] : 0.f;
        row_result(a, row0 + m, act, two && top == -__builtin_inff() ? 0.f : top, s, t, s != 0.f, z, two ? 0.693147181f : 1.f);
    }
}

// out[row][col] = scale * sum of the parts (+ what `sum` holds); `sum` takes it while more is to come
template <typename T>
__global__ __launch_bounds__(256) void actions_reduce_kernel(const float *part, int64_t split_stride, int splits, int64_t ld, float *sum, int first, int last, T *out,
                                                             int64_t rows, int cols, const float *inv_scale) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, at = r * ld + (i - r * cols);
        float s = first ? 0.f : sum[at];
#pragma unroll 8
        for (int k = 0; k < splits; ++k) s += part[k * split_stride + at];
        if (last) out[i] = (T)(inv_scale ? s / *inv_scale : s);
        else sum[at] = s;
    }
}

__global__ __launch_bounds__(256) void actions_bias_kernel(const float *part, int64_t ld, int parts, float *db, int n, int add) {
    __shared__ double red[16][17];
    const int c = threadIdx.x & 15, s = threadIdx.x >> 4, v = blockIdx.x * 16 + c;
    double sum = 0.0;
    if (v < n)
#pragma unroll 16
        for (int p = s; p < parts; p += 16) sum += (double)part[p * ld + v];
    red[s][c] = sum;
    __syncthreads();
    if (s == 0 && v < n) {
        for (int k = 1; k < 16; ++k) sum += red[k][c];
        db[v] = (float)(add ? (double)db[v] + sum : sum);
    }
}

// float16 operands: dz is stored times the power of two that brings the largest |dlog_prob| + |dentropy| (1 + log V) to 2^12, so that small upstream gradients
// (a mean over a million rows) do not fall below float16's smallest numbers; the products are divided by it again.  Maxima of up to 256 workgroups' rows first.
const int kMaxima = 256;
__global__ __launch_bounds__(256) void actions_maxima_kernel(Actions a, float *maxima) {
    __shared__ float red[4];
    const float lv = 1.f + logf((float)a.V);
    float m = 0.f;
#pragma unroll 4
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * 256) {
        const float v = (a.dlogp ? fabsf(a.dlogp[r]) : 0.f) + (a.dent ? fabsf(a.dent[r]) : 0.f) * lv;
        if (a.lse[r] != __builtin_inff() && v < __builtin_inff()) m = fmaxf(m, v);
    }
    m = lanes_max<1>(m, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) maxima[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

__global__ __launch_bounds__(64) void actions_scale_kernel(const float *maxima, int parts, float *scale) {
    float m = 0.f;
    for (int i = threadIdx.x; i < parts; i += 64) m = fmaxf(m, maxima[i]);
    m = lanes_max<1>(m, 64);
    if (threadIdx.x == 0) {
        int e = 0;
        if (m > 0.f) (void)frexpf(m, &e);
        *scale = ldexpf(1.f, min(120, max(-120, 12 - e)));
    }
}

}  // namespace policy
}  // namespace fmarl

using namespace fmarl;
using namespace fmarl::policy;

namespace {

int actions_check(const FmarlActions *a, const char *who) {
    if (!a) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    if (a->rows < 0 || a->rows > (1ll << 36)) return policy_fail(FMARL_EINVAL, "%s: bad number of rows", who);
    if (a->features < 1 || a->features > 16384) return policy_fail(FMARL_EINVAL, "%s: features must lie in 1..16384", who);
    if (a->actions < 1 || a->actions > (1 << 20)) return policy_fail(FMARL_EINVAL, "%s: actions must lie in 1..1048576", who);
    if (a->dtype < FMARL_T_F32 || a->dtype > FMARL_T_F16) return policy_fail(FMARL_EINVAL, "%s: unknown dtype", who);
    if (a->action_type < 0 || a->action_type > 2 || a->available_type < 0 || a->available_type > 1) return policy_fail(FMARL_EINVAL, "%s: unknown action_type or available_type", who);
    if (a->rows > 0 && (!a->x || !a->weight || !a->action)) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    return FMARL_OK;
}

Actions actions_args(const FmarlActions *a) {
    Actions s = {};
    const int e = elem_bytes(a->dtype);
    s.rows = a->rows; s.K = a->features; s.V = a->actions; s.act_type = a->action_type; s.avail_u8 = a->available_type;
    s.x = (const char *)a->x; s.xs = a->x_stride; s.w = (const char *)a->weight; s.ws = a->weight_stride; s.bias = a->bias;
    s.act = a->action; s.avail = a->available; s.as = a->available_stride;
    s.xvec = (a->features & 3) == 0 && (a->x_stride & 3) == 0 && ((uintptr_t)a->x & (4 * e - 1)) == 0;
    return s;
}

// Few actions: the tiles of W's gradient (16 x 16, four registers a lane each) have to stay in registers beside the operands, and padding V to 16 must not cost
// more than the products of the other way
bool actions_few(const FmarlActions *a) {
    const int vt = (a->actions + 15) / 16, kt = (a->features + 15) / 16;
    return vt <= 4 && kt <= 16 && (vt <= 1 ? 1 : vt <= 2 ? 2 : 4) * (kt <= 2 ? 2 : kt <= 4 ? 4 : kt <= 8 ? 8 : 16) <= 16;
}

int few_workgroups(const FmarlActions *a) {   // four waves of 16 rows each; 1 024 of them fill the chip, and their partial sums stay small
    const int64_t n = (a->rows + 63) / 64;
    return (int)(n < 1 ? 1 : n < 1024 ? n : 1024);
}

template <typename T, bool BACK>
int launch_few(const Actions &s, int blocks, hipStream_t st) {
    const int vt = (s.V + 15) / 16, kt = (s.K + 15) / 16;
    const bool vec = s.xvec && (!BACK || s.dxvec);   // known at compile time: as an argument it costs the loads in flight (2 097 152 x 64 x 5 training: 438 us, 368)
#define FMARL_FEW(VT, KT) do { if (vec) hipLaunchKernelGGL((actions_few_kernel<T, VT, KT, BACK, true>), dim3(blocks), dim3(256), 0, st, s); \
                               else hipLaunchKernelGGL((actions_few_kernel<T, VT, KT, BACK, false>), dim3(blocks), dim3(256), 0, st, s); } while (0)
    if (vt <= 1) { if (kt <= 2) FMARL_FEW(1, 2); else if (kt <= 4) FMARL_FEW(1, 4); else if (kt <= 8) FMARL_FEW(1, 8); else FMARL_FEW(1, 16); }
    else if (vt <= 2) { if (kt <= 2) FMARL_FEW(2, 2); else if (kt <= 4) FMARL_FEW(2, 4); else FMARL_FEW(2, 8); }
    else { if (kt <= 2) FMARL_FEW(4, 2); else FMARL_FEW(4, 4); }
#undef FMARL_FEW
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

template <bool BACK>
int launch_few_t(int dtype, const Actions &s, int blocks, hipStream_t st) {
    return dtype == FMARL_T_F32 ? launch_few<float, BACK>(s, blocks, st) : dtype == FMARL_T_BF16 ? launch_few<__bf16, BACK>(s, blocks, st) : launch_few<_Float16, BACK>(s, blocks, st);
}

int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// The sizes of the way for many actions.  Rows go in chunks and (backwards) actions in pieces, so that what is kept of a chunk -- dz (float32: and its transpose),
// three floats per row and 64 actions -- stays within 256 MB, the size of the last-level cache.
struct Plan {
    int tile;                     // rows and columns of a tile: 128 (float32), 256
    int64_t Kp, Vp, Mc, P;        // padded features and actions, rows of a chunk, actions of a piece
    int split_x, split_w;         // parts of the contraction of dx and dW
    int split_z;                  // half precision: parts of a run of tiles (kStats: of the actions, kDlogits: of the rows)
    size_t xp, wp, bias2, taken, rows, stats, za, xt, wt, dz, dzt, out, sumx, sumw, db, scale, total;
};

// parts of a contraction of `steps` for `tiles` tiles: enough that the chip is full (`fill` workgroups), none with fewer than four steps
int parts_of(int64_t tiles, int64_t steps, int fill, int most) {
    int64_t n = fill / tiles;
    if (n > steps / 4) n = steps / 4;
    return (int)(n < 1 ? 1 : n > most ? most : n);
}

Plan actions_plan(const FmarlActions *a, bool backward) {
    Plan p = {};
    const bool half = a->dtype != FMARL_T_F32;
    const int64_t e = elem_bytes(a->dtype), budget = 256ll << 20;
    p.tile = half ? 256 : 128;
    const int64_t M = up(a->rows, p.tile), tile = p.tile, per = 128 / e;
    p.Kp = up(a->features, tile); p.Vp = up(a->actions, tile);
    int64_t keep = half ? 2 * p.Kp : backward ? 2 * e * 128 : 12 * (p.Vp / 64);   // bytes per row that a chunk cannot do without
    int64_t mc = budget / keep / tile * tile;
    if (mc > 65536) mc = 65536;
    if (mc < 1024) mc = 1024;
    p.Mc = M < mc ? M : mc;
    p.P = budget / ((half ? 1 : 2) * e * p.Mc) / tile * tile;
    if (p.P < tile) p.P = tile;
    if (p.P > p.Vp) p.P = p.Vp;
    const int64_t tm = p.Mc / tile, tk = p.Kp / tile, tv = p.P / tile;
    // a workgroup per CU: half precision by its LDS (128 KB); float32 could hold two, whose shorter parts and longer sums cost more (12 345 x 625: 45 us a product, 32 us)
    p.split_x = parts_of(tm * tk, p.P / per, 256, half ? 16 : 64);
    p.split_w = parts_of(tv * tk, p.Mc / per, 256, half ? 16 : 64);
    const int64_t run = backward ? tm : p.Vp / tile, rest = backward ? tv : tm;
    p.split_z = (int)(256 / rest < 1 ? 1 : 256 / rest > run ? run : 256 / rest);
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += up256(bytes); return at; };
    p.xp = take(e * p.Mc * p.Kp); p.wp = take(e * p.Vp * p.Kp);
    if (half) { p.bias2 = take(4 * p.Vp); p.taken = take(4 * p.Mc); p.rows = take(backward ? 16 * p.Mc : 0); }
    if (!backward) { p.stats = take(12 * (half ? 2 * p.split_z : p.Vp / 64) * p.Mc); p.za = take(4 * p.Mc); }
    else {
        if (!half) { p.xt = take(e * p.Mc * p.Kp); p.wt = take(e * p.Vp * p.Kp); p.dzt = take(e * p.Mc * p.P); }
        p.dz = take(e * p.Mc * p.P);
        const int64_t ox = p.split_x * p.Mc * p.Kp, ow = p.split_w * p.P * p.Kp;
        p.out = take(4 * (ox > ow ? ox : ow));
        p.sumx = take(p.P < p.Vp ? 4 * p.Mc * p.Kp : 0);
        p.sumw = take(p.Mc < M ? 4 * p.Vp * p.Kp : 0);
        p.db = take(4 * (p.Mc / 64) * p.P);
        p.scale = take(4 * (1 + kMaxima));
    }
    p.total = off;
    return p;
}

// dst and (float32, backwards) its transpose
// the rows from r0 on, and with the first of them the weights
template <typename T>
void pack(const Actions &s, const Plan &p, int64_t r0, int64_t m, int64_t mp, T *xp, T *xt, T *wp, T *wt, const float *lse, hipStream_t st) {
    const PackJob x = {(const char *)((const T *)s.x + r0 * s.xs), s.xs, m, mp, (char *)xp, (char *)xt, lse}, w = {(const char *)s.w, s.ws, s.V, p.Vp, (char *)wp, (char *)wt, nullptr};
    const int64_t blocks = mp / 64 + (r0 == 0 ? p.Vp / 64 : 0);
    hipLaunchKernelGGL((actions_pack_kernel<T>), dim3((unsigned)blocks, (unsigned)(p.Kp / 64)), dim3(256), 0, st, x, w, (int)(mp / 64), (int)s.K, (int)p.Kp);
}

template <int EPI>
void gemm(const Gemm &q, hipStream_t st) {
    hipLaunchKernelGGL((actions_gemm_kernel<float, EPI>), dim3((unsigned)(q.ta * q.tb * q.splits)), dim3(256), 0, st, q);
}

template <typename T, int EPI, bool TA, bool TB, bool AVAIL>
int wide_as(const Wide &q, int64_t blocks, hipStream_t st) {
    HIP_OK(hipFuncSetAttribute((const void *)actions_wide_kernel<T, EPI, TA, TB, AVAIL>, hipFuncAttributeMaxDynamicSharedMemorySize, kWideLds));
    hipLaunchKernelGGL((actions_wide_kernel<T, EPI, TA, TB, AVAIL>), dim3((unsigned)blocks), dim3(512), kWideLds, st, q);
    return FMARL_OK;
}

template <typename T, int EPI, bool TA, bool TB>
int wide(const Wide &q, int64_t blocks, hipStream_t st) {
    if constexpr (EPI != kStore)
        if (q.act.avail) return wide_as<T, EPI, TA, TB, true>(q, blocks, st);
    return wide_as<T, EPI, TA, TB, false>(q, blocks, st);
}

int many_forward_f32(const Actions &s, const Plan &p, char *base, hipStream_t st) {
    float *xp = (float *)(base + p.xp), *wp = (float *)(base + p.wp);
    for (int64_t r0 = 0; r0 < s.rows; r0 += p.Mc) {
        const int64_t m = s.rows - r0 < p.Mc ? s.rows - r0 : p.Mc, mp = up(m, 128);
        pack<float>(s, p, r0, m, mp, xp, nullptr, wp, nullptr, nullptr, st);
        Gemm q = {};
        q.A = (const char *)wp; q.B = (const char *)xp; q.lda = q.ldb = p.Kp; q.ta = (int)(p.Vp / 128); q.tb = (int)(mp / 128); q.splits = 1; q.steps = (int)(up(s.K, 32) / 32);
        q.act = s; q.row0 = r0; q.stats = (float *)(base + p.stats); q.stat_stride = p.Mc; q.za = (float *)(base + p.za);
        gemm<kStats>(q, st);
        hipLaunchKernelGGL(actions_join_kernel, dim3((unsigned)((m + 15) / 16)), dim3(256), 0, st, s, (const float *)q.stats, p.Mc, (int)(p.Vp / 64), (const float *)q.za, r0, m, 0);
        HIP_OK(hipGetLastError());
    }
    return FMARL_OK;
}

template <typename T>
void reduce(const float *part, int64_t split_stride, int splits, int64_t ld, float *sum, bool first, bool last, T *out, int64_t rows, int cols, const float *scale, hipStream_t st) {
    const int64_t blocks = (rows * cols + 255) / 256, most = 1 << 22;   // a launch holds fewer than 2^32 threads, the weights may be 2^34
    hipLaunchKernelGGL((actions_reduce_kernel<T>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, part, split_stride, splits, ld, sum, (int)first, (int)last, out, rows,
                       cols, scale);
}

int many_backward_f32(const Actions &s, const Plan &p, float *dx, float *dw, float *db, char *base, hipStream_t st) {
    float *xp = (float *)(base + p.xp), *wp = (float *)(base + p.wp), *xt = (float *)(base + p.xt), *wt = (float *)(base + p.wt), *dz = (float *)(base + p.dz), *dzt = (float *)(base + p.dzt);
    float *out = (float *)(base + p.out), *sumx = (float *)(base + p.sumx), *sumw = (float *)(base + p.sumw), *dbp = (float *)(base + p.db);
    for (int64_t r0 = 0; r0 < s.rows; r0 += p.Mc) {
        const int64_t m = s.rows - r0 < p.Mc ? s.rows - r0 : p.Mc, mp = up(m, 128);
        pack<float>(s, p, r0, m, mp, xp, xt, wp, wt, s.lse + r0, st);
        for (int64_t v0 = 0; v0 < p.Vp; v0 += p.P) {
            const int64_t n = p.Vp - v0 < p.P ? p.Vp - v0 : p.P, nv = s.V - v0 < n ? s.V - v0 : n;   // of this piece: padded and real actions
            Gemm q = {};
            q.A = (const char *)(wp + v0 * p.Kp); q.B = (const char *)xp; q.lda = q.ldb = p.Kp; q.ta = (int)(n / 128); q.tb = (int)(mp / 128); q.splits = 1; q.steps = (int)(up(s.K, 32) / 32);
            q.act = s; q.row0 = r0; q.v0 = (int)v0; q.dz = (char *)dz; q.dzt = (char *)dzt; q.ldz = p.P; q.ldzt = p.Mc; q.db = dbp; q.ldb_part = p.P;
            gemm<kDlogits>(q, st);
            if (db) hipLaunchKernelGGL(actions_bias_kernel, dim3((unsigned)((nv + 15) / 16)), dim3(256), 0, st, (const float *)dbp, p.P, (int)(mp / 64), db + v0, (int)nv, (int)(r0 > 0));
            q = Gemm{};   // dx += dz W: rows of W^T (features) against rows of dz
            q.A = (const char *)(wt + v0); q.lda = p.Vp; q.B = (const char *)dz; q.ldb = p.P; q.ta = (int)(p.Kp / 128); q.tb = (int)(mp / 128); q.steps = (int)(n / 32);
            q.splits = p.split_x < q.steps ? p.split_x : q.steps; q.out = out; q.ldo = p.Kp; q.split_out = p.Mc * p.Kp;
            gemm<kStore>(q, st);
            reduce<float>(out, q.split_out, q.splits, p.Kp, sumx, v0 == 0, v0 + n >= p.Vp, dx + r0 * s.K, m, s.K, nullptr, st);
            q.A = (const char *)xt; q.lda = mp; q.B = (const char *)dzt; q.ldb = p.Mc; q.tb = (int)(n / 128); q.steps = (int)(mp / 32);   // dW: rows of x^T against rows of dz^T
            q.splits = p.split_w < q.steps ? p.split_w : q.steps; q.split_out = p.P * p.Kp;
            gemm<kStore>(q, st);
            reduce<float>(out, q.split_out, q.splits, p.Kp, sumw + v0 * p.Kp, r0 == 0, r0 + m >= s.rows, dw + v0 * s.K, nv, s.K, nullptr, st);
            HIP_OK(hipGetLastError());
        }
    }
    return FMARL_OK;
}

template <typename T>
int many_forward(const Actions &s, const Plan &p, char *base, hipStream_t st) {
    T *xp = (T *)(base + p.xp), *wp = (T *)(base + p.wp);
    float *bias2 = (float *)(base + p.bias2);
    hipLaunchKernelGGL(actions_bias2_kernel, dim3((unsigned)(p.Vp / 256)), dim3(256), 0, st, s.bias, s.V, bias2, (int)p.Vp);
    for (int64_t r0 = 0; r0 < s.rows; r0 += p.Mc) {
        const int64_t m = s.rows - r0 < p.Mc ? s.rows - r0 : p.Mc, mp = up(m, 256);
        pack<T>(s, p, r0, m, mp, xp, nullptr, wp, nullptr, nullptr, st);
        Wide q = {};
        q.A = (const char *)wp; q.B = (const char *)xp; q.lda = q.ldb = p.Kp; q.ta = (int)(p.Vp / 256); q.tb = (int)(mp / 256); q.steps = (int)(up(s.K, 32) / 32); q.splits = p.split_z;
        q.act = s; q.row0 = r0; q.bias2 = bias2; q.taken = (const int *)(base + p.taken); q.stats = (float *)(base + p.stats); q.stat_stride = p.Mc; q.za = (float *)(base + p.za);
        hipLaunchKernelGGL(actions_rows_kernel, dim3((unsigned)(mp / 256)), dim3(256), 0, st, s, r0, mp, (f32x4 *)nullptr, (int *)(base + p.taken), (const float *)nullptr);
        if (int rc = wide<T, kStats, false, false>(q, (int64_t)q.tb * q.splits, st)) return rc;
        hipLaunchKernelGGL(actions_join_kernel, dim3((unsigned)((m + 15) / 16)), dim3(256), 0, st, s, (const float *)q.stats, p.Mc, 2 * q.splits, (const float *)q.za, r0, m, 1);
        HIP_OK(hipGetLastError());
    }
    return FMARL_OK;
}

template <typename T>
int many_backward(const Actions &s, const Plan &p, T *dx, T *dw, float *db, char *base, hipStream_t st) {
    T *xp = (T *)(base + p.xp), *wp = (T *)(base + p.wp), *dz = (T *)(base + p.dz);
    float *bias2 = (float *)(base + p.bias2), *out = (float *)(base + p.out), *sumx = (float *)(base + p.sumx), *sumw = (float *)(base + p.sumw), *dbp = (float *)(base + p.db);
    const float *scale = nullptr;
    if ((float)(T)1e-30f == 0.f) {   // float16
        scale = (const float *)(base + p.scale);
        const int parts = (int)(s.rows < 256 * kMaxima ? (s.rows + 255) / 256 : kMaxima);
        hipLaunchKernelGGL(actions_maxima_kernel, dim3(parts), dim3(256), 0, st, s, (float *)(base + p.scale) + 1);
        hipLaunchKernelGGL(actions_scale_kernel, dim3(1), dim3(64), 0, st, (const float *)(base + p.scale) + 1, parts, (float *)(base + p.scale));
    }
    hipLaunchKernelGGL(actions_bias2_kernel, dim3((unsigned)(p.Vp / 256)), dim3(256), 0, st, s.bias, s.V, bias2, (int)p.Vp);
    for (int64_t r0 = 0; r0 < s.rows; r0 += p.Mc) {
        const int64_t m = s.rows - r0 < p.Mc ? s.rows - r0 : p.Mc, mp = up(m, 256);
        pack<T>(s, p, r0, m, mp, xp, nullptr, wp, nullptr, s.lse + r0, st);
        hipLaunchKernelGGL(actions_rows_kernel, dim3((unsigned)(mp / 256)), dim3(256), 0, st, s, r0, mp, (f32x4 *)(base + p.rows), (int *)(base + p.taken), scale);
        for (int64_t v0 = 0; v0 < p.Vp; v0 += p.P) {
            const int64_t n = p.Vp - v0 < p.P ? p.Vp - v0 : p.P, nv = s.V - v0 < n ? s.V - v0 : n;   // of this piece: padded and real actions
            Wide q = {};
            q.A = (const char *)(wp + v0 * p.Kp); q.B = (const char *)xp; q.lda = q.ldb = p.Kp; q.ta = (int)(n / 256); q.tb = (int)(mp / 256); q.steps = (int)(up(s.K, 32) / 32);
            q.splits = p.split_z < q.tb ? p.split_z : q.tb;
            q.act = s; q.row0 = r0; q.v0 = (int)v0; q.bias2 = bias2 + v0; q.taken = (const int *)(base + p.taken); q.rows = (const f32x4 *)(base + p.rows);
            q.dz = (char *)dz; q.ldz = p.P; q.db = dbp; q.ldb_part = p.P; q.dz_scale = scale;
            if (int rc = wide<T, kDlogits, false, false>(q, (int64_t)q.ta * q.splits, st)) return rc;
            if (db) hipLaunchKernelGGL(actions_bias_kernel, dim3((unsigned)((nv + 15) / 16)), dim3(256), 0, st, (const float *)dbp, p.P, (int)(mp / 64), db + v0, (int)nv, (int)(r0 > 0));
            q = Wide{};   // dx += dz W: columns of W (features) against rows of dz
            q.A = (const char *)(wp + v0 * p.Kp); q.lda = p.Kp; q.B = (const char *)dz; q.ldb = p.P; q.ta = (int)(p.Kp / 256); q.tb = (int)(mp / 256); q.steps = (int)(n / 32);
            q.splits = p.split_x < q.steps ? p.split_x : q.steps; q.out = out; q.ldo = p.Kp; q.split_out = p.Mc * p.Kp;
            if (int rc = wide<T, kStore, true, false>(q, (int64_t)q.ta * q.tb * q.splits, st)) return rc;
            reduce<T>(out, q.split_out, q.splits, p.Kp, sumx, v0 == 0, v0 + n >= p.Vp, dx + r0 * s.K, m, s.K, scale, st);
            q.A = (const char *)xp; q.B = (const char *)dz; q.tb = (int)(n / 256); q.steps = (int)(mp / 32);   // dW: columns of x against columns of dz
            q.splits = p.split_w < q.steps ? p.split_w : q.steps; q.split_out = p.P * p.Kp;
            if (int rc = wide<T, kStore, true, true>(q, (int64_t)q.ta * q.tb * q.splits, st)) return rc;
            reduce<T>(out, q.split_out, q.splits, p.Kp, sumw + v0 * p.Kp, r0 == 0, r0 + m >= s.rows, dw + v0 * s.K, nv, s.K, scale, st);
            HIP_OK(hipGetLastError());
        }
    }
    return FMARL_OK;
}

}  // namespace

extern "C" {

size_t fmarl_action_log_probs_workspace(const FmarlActions *a, int backward) {
    if (actions_check(a, "fmarl_action_log_probs_workspace")) return 0;
    if (a->rows == 0) return 256;   // (nothing runs; a plan divides by the rows)
    if (actions_few(a)) return backward ? up256((size_t)few_workgroups(a) * ((size_t)a->actions * a->features + a->actions) * 4) : 256;
    return actions_plan(a, backward != 0).total;
}

int fmarl_action_log_probs(const FmarlActions *a, float *log_probs, float *entropy, float *lse, void *workspace, void *stream) {
    if (int rc = actions_check(a, "fmarl_action_log_probs")) return rc;
    if (a->rows == 0) return FMARL_OK;
    if (!log_probs || !entropy || !lse || !workspace) return policy_fail(FMARL_EINVAL, "fmarl_action_log_probs: null argument");
    hipStream_t st = (hipStream_t)stream;
    Actions s = actions_args(a);
    s.logp = log_probs; s.ent = entropy; s.lse = lse;
    if (actions_few(a)) {
        const int64_t n = (a->rows + 63) / 64;
        return launch_few_t<false>(a->dtype, s, (int)(n < 2048 ? n : 2048), st);
    }
    const Plan p = actions_plan(a, false);
    return a->dtype == FMARL_T_F32 ? many_forward_f32(s, p, (char *)workspace, st)
         : a->dtype == FMARL_T_BF16 ? many_forward<__bf16>(s, p, (char *)workspace, st) : many_forward<_Float16>(s, p, (char *)workspace, st);
}

int fmarl_action_log_probs_backward(const FmarlActions *a, const float *entropy, const float *lse, const float *d_log_probs, const float *d_entropy,
                                    void *d_x, void *d_weight, float *d_bias, void *workspace, void *stream) {
    if (int rc = actions_check(a, "fmarl_action_log_probs_backward")) return rc;
    if (a->rows < 1) return policy_fail(FMARL_EINVAL, "fmarl_action_log_probs_backward: rows must be positive");
    if (!entropy || !lse || !d_x || !d_weight || !workspace) return policy_fail(FMARL_EINVAL, "fmarl_action_log_probs_backward: null argument");
    hipStream_t st = (hipStream_t)stream;
    Actions s = actions_args(a);
    s.ent = (float *)entropy; s.lse = (float *)lse; s.dlogp = d_log_probs; s.dent = d_entropy; s.dx = (char *)d_x; s.partial = (float *)workspace;
    s.dxvec = (a->features & 3) == 0 && ((uintptr_t)d_x & (4 * elem_bytes(a->dtype) - 1)) == 0;
    if (actions_few(a)) {
        const int parts = few_workgroups(a);
        if (int rc = launch_few_t<true>(a->dtype, s, parts, st)) return rc;
        const int64_t nw = (int64_t)a->actions * a->features, n = nw + a->actions;
        const dim3 grid((unsigned)((n + 15) / 16));
        if (a->dtype == FMARL_T_F32) hipLaunchKernelGGL((actions_sums_kernel<float>), grid, dim3(256), 0, st, (const float *)workspace, parts, n, nw, (float *)d_weight, d_bias);
        else if (a->dtype == FMARL_T_BF16) hipLaunchKernelGGL((actions_sums_kernel<__bf16>), grid, dim3(256), 0, st, (const float *)workspace, parts, n, nw, (__bf16 *)d_weight, d_bias);
        else hipLaunchKernelGGL((actions_sums_kernel<_Float16>), grid, dim3(256), 0, st, (const float *)workspace, parts, n, nw, (_Float16 *)d_weight, d_bias);
        HIP_OK(hipGetLastError());
        return FMARL_OK;
    }
    const Plan p = actions_plan(a, true);
    char *ws = (char *)workspace;
    return a->dtype == FMARL_T_F32 ? many_backward_f32(s, p, (float *)d_x, (float *)d_weight, d_bias, ws, st)
         : a->dtype == FMARL_T_BF16 ? many_backward<__bf16>(s, p, (__bf16 *)d_x, (__bf16 *)d_weight, d_bias, ws, st)
                                    : many_backward<_Float16>(s, p, (_Float16 *)d_x, (_Float16 *)d_weight, d_bias, ws, st);
}

}  // extern "C"
