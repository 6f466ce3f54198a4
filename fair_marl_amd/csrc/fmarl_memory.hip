// The memory of a recurrent policy on gfx950: linear attention with a decay per head.  With r_t = 0 where an episode starts at t
// (masks_t == 0; also where the decay is exactly zero) and 1 elsewhere,
//     S_t = r_t e^{g_t} S_{t-1} + k_t^T v_t          o_t = scale * q_t S_t
// and backwards, with G_t the gradient of S_t,
//     G_t = scale * q_t^T do_t + r_{t+1} e^{g_{t+1}} G_{t+1}      dq_t = scale * do_t S_t^T     dk_t = v_t G_t^T     dv_t = k_t G_t
//     dS_0 = r_1 e^{g_1} G_1                                      dg_t = r_t e^{g_t} <S_{t-1}, G_t>.
// o, dq, dk and dv are the same walk over the tokens, forwards or backwards, with the operands in other roles:
//     out_t = sum_{s before or at t} w(t, s) (x_t . y_s) z_s + (what the walk carries):
//     o: x, y, z = q, k, v forwards;  dq: do, v, k forwards (state S^T);  dk: v, do, q backwards (state G^T);  dv: k, q, do backwards.
// memory_walk_kernel is that walk.
#pragma once
#include "fmarl_policy_dev.h"

namespace fmarl {
namespace policy {

struct WalkRows {            // a (L, B, H, d) tensor whose last axis is contiguous
    char *p;
    int64_t sl, sb, sh;      // strides in elements
    int vec;                 // rows start on multiples of four elements and hold a multiple of four
};

struct Walk {
    WalkRows x, y, z, w, out;          // w: NULL, or what out is dotted with for the decay's gradient
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    const float *state;                // initial state, NULL: zeros; element (y, z) of (b, h) at (b * H + h) * state_elems + y * s_y + z * s_z
    float *state_out;                  // NULL: not wanted
    int64_t s_y, s_z, o_y, o_z;        // the strides of the two
    int64_t seg_state_in, seg_state_out;   // elements from one segment's states to the next one's (0: the same for all)
    float *seg_decay;                  // state_only: the segment's whole decay, (nseg, B * H)
    float *dot;                        // (slices, L, B, H) sums of out * w without the token's own term
    int64_t L, B;
    int H, dy, dz, nseg, seg_len, slices;
    int reverse, state_only;
    float y_scale, out_scale;
};

// One wave walks one (batch, head, segment of the tokens, slice of at most 16 NZ columns of z) in chunks of 16 tokens; the state (16 NY x 16 NZ)
// stays in registers in the accumulator layout of mfma_f32_16x16x4f32 (row 4 * (lane / 16) + r, column lane % 16).  That layout is also a valid
// B operand that contracts over the rows in the order k = 4 * (lane / 16) + r, and the A operand of its transpose, so neither the weights
// (kept as P^T: rows s, columns t) nor the state ever moves between lanes:
//     P^T = y x^T;  out^T = z^T P^T + S^T x^T;  S = e^C S + (u y)^T z.
// Float32 products and sums throughout (the inputs' bf16 / f16 values are exact in it); the decays' prefix sums are float64, so a weight
// e^{C_t - C_s} is right to float32 however fast the tokens before forgot.  A weight is selected, not multiplied to zero: what an episode left
// behind (infinities too) does not reach the next one; a chunk that holds a value that is not finite is walked token by token, so that
// it reaches later tokens only.
template <typename T, int NY, int NZ>
__global__ __launch_bounds__(256) void memory_walk_kernel(Walk a) {
    constexpr int PY = 16 * NY + 4, PZ = 16 * NZ + 4;   // 4 rows apart = 16 banks apart: column reads of four row groups do not meet
    constexpr int kWave = 16 * (2 * PY + 2 * PZ) + 32 + 16;
    __shared__ __align__(16) float lds[4 * kWave];
    typedef typename Vec4<T>::type V;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g4 = (lane >> 4) * 4;
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
    const int64_t heads = a.B * a.H;
    if (unit >= heads * a.nseg * a.slices) return;
    // neighbouring waves take neighbouring heads of one batch entry: their rows share cache lines
    const int64_t bh = unit % heads;
    const int64_t rest = unit / heads;
    const int slice = (int)(rest % a.slices), seg = (int)(rest / a.slices);
    const int64_t b = bh / a.H;
    const int h = (int)(bh - b * a.H);
    const int z0 = slice * 16 * NZ, dz = min(a.dz - z0, 16 * NZ), dy = a.dy;
    const int64_t t_begin = (int64_t)seg * a.seg_len, t_end = min(a.L, t_begin + a.seg_len);

    float *lx = lds + wave * kWave, *ly = lx + 16 * PY, *lz = ly + 16 * PY, *lw = lz + 16 * PZ;
    double *lc = (double *)(lw + 16 * PZ);      // prefix sums of the chunk's log decays
    const T *px = (const T *)a.x.p + b * a.x.sb + h * a.x.sh, *py = (const T *)a.y.p + b * a.y.sb + h * a.y.sh;
    const T *pz = (const T *)a.z.p + b * a.z.sb + h * a.z.sh + z0, *pw = a.w.p ? (const T *)a.w.p + b * a.w.sb + h * a.w.sh + z0 : nullptr;
    T *po = a.state_only ? nullptr : (T *)a.out.p + b * a.out.sb + h * a.out.sh + z0;

    f32x4 S[NY][NZ];
#pragma unroll
    for (int i = 0; i < NY; ++i)
#pragma unroll
        for (int j = 0; j < NZ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int y = 16 * i + g4 + r, z = 16 * j + c;
                S[i][j][r] = a.state && y < dy && z < dz
                    ? a.state[seg * a.seg_state_in + bh * (int64_t)a.dy * a.dz + y * a.s_y + (z0 + z) * a.s_z] : 0.f;
            }
    float whole = 1.f;   // state_only: the decay over the whole segment

    const int64_t chunks = (t_end - t_begin + 15) / 16;
    V rx[NY], ry[NY], rz[NZ], rw[NZ];
    float rg = 0.f, rm = 1.f;
    auto fetch = [&](int64_t t0) {
#pragma unroll
        for (int n = 0; n < NY; ++n) {
            const int idx = lane + 64 * n, tok = idx / (4 * NY), col = (idx % (4 * NY)) * 4;
            const int64_t t = t0 + tok;
            const int left = t < t_end ? dy - col : 0;
            if (!a.state_only) rx[n] = load4<T>(px + t * a.x.sl + col, left, a.x.vec);
            ry[n] = load4<T>(py + t * a.y.sl + col, left, a.y.vec);
        }
#pragma unroll
        for (int n = 0; n < NZ; ++n) {
            const int idx = lane + 64 * n, tok = idx / (4 * NZ), col = (idx % (4 * NZ)) * 4;
            const int64_t t = t0 + tok;
            const int left = t < t_end ? dz - col : 0;
            rz[n] = load4<T>(pz + t * a.z.sl + col, left, a.z.vec);
            if (pw) rw[n] = load4<T>(pw + t * a.w.sl + col, left, a.w.vec);
        }
        const int64_t t = t0 + c;
        rg = t < t_end ? a.g[t * a.gl + b * a.gb + h * a.gh] : 0.f;
        rm = t < t_end && a.masks ? a.masks[t * a.ml + b * a.mb] : 1.f;
    };
    auto chunk_at = [&](int64_t n) { return t_begin + 16 * (a.reverse ? chunks - 1 - n : n); };
    fetch(chunk_at(0));
    for (int64_t n = 0; n < chunks; ++n) {
        const int64_t t0 = chunk_at(n);
        float bad = 0.f;   // not zero (NaN) where a value of y or z is not finite
        float ndt = 0.f;   // this lane's token's own weight (x . y), for the diagonal
        const float gt = rg, mt = rm;
        V sy[NY], sz[NZ];
#pragma unroll
        for (int k = 0; k < NY; ++k) { sy[k] = ry[k]; const f32x4 f = widen(ry[k]); bad += f[0] * 0.f + f[1] * 0.f + f[2] * 0.f + f[3] * 0.f; }
#pragma unroll
        for (int k = 0; k < NZ; ++k) { sz[k] = rz[k]; const f32x4 f = widen(rz[k]); bad += f[0] * 0.f + f[1] * 0.f + f[2] * 0.f + f[3] * 0.f; }
        const bool careful = __ballot(!(bad == 0.f)) != 0;
        wave_sync();
        if (!a.state_only)
#pragma unroll
            for (int k = 0; k < NY; ++k) { const int idx = lane + 64 * k; *(f32x4 *)(lx + (idx / (4 * NY)) * PY + (idx % (4 * NY)) * 4) = widen(rx[k]); }
        if (pw)
#pragma unroll
            for (int k = 0; k < NZ; ++k) { const int idx = lane + 64 * k; *(f32x4 *)(lw + (idx / (4 * NZ)) * PZ + (idx % (4 * NZ)) * 4) = widen(rw[k]); }
        if (n + 1 < chunks) fetch(chunk_at(n + 1));   // in flight while this chunk is computed

        const int subs = careful ? 16 : 1;
        for (int sub = 0; sub < subs; ++sub) {
            const int only = a.reverse ? 15 - sub : sub;
            const bool live = !careful || c == only;      // this lane's token takes part in this pass
            wave_sync();
#pragma unroll
            for (int k = 0; k < NY; ++k) {
                const int idx = lane + 64 * k, tok = idx / (4 * NY);
                *(f32x4 *)(ly + tok * PY + (idx % (4 * NY)) * 4) = !careful || tok == only ? widen(sy[k]) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int k = 0; k < NZ; ++k) {
                const int idx = lane + 64 * k, tok = idx / (4 * NZ);
                *(f32x4 *)(lz + tok * PZ + (idx % (4 * NZ)) * 4) = !careful || tok == only ? widen(sz[k]) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
            // prefix sums of the log decays (base 2), tokens that start afresh as bits
            const bool fresh = live && (mt == 0.f || gt == -__builtin_inff());
            const uint32_t fr = (uint32_t)(__ballot(fresh) & 0xffff);
            double C = live && !fresh ? (double)gt * 1.4426950408889634074 : 0.0;
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) { const double o = __shfl_up(C, off, 16); if (c >= off) C += o; }
            if (lane < 16) lc[lane] = C;
            wave_sync();
            const double C15 = lc[15];
            // `head`: decay from before the chunk up to and with token c; `tail`: from behind token c to the chunk's end
            const bool head_ok = (fr & ((2u << c) - 1)) == 0, tail_ok = (fr >> (c + 1)) == 0;
            const float head = head_ok ? exp2_fast((float)C) : 0.f, tail = tail_ok ? exp2_fast((float)(C15 - C)) : 0.f;
            const bool all_ok = fr == 0;
            const float all = all_ok ? exp2_fast((float)C15) : 0.f;
            const bool in_ok = a.reverse ? tail_ok : head_ok;      // the carried state reaches this lane's token
            const float win = a.reverse ? tail : head, wout = (a.reverse ? head : tail) * a.y_scale;

            if (!a.state_only) {
                f32x4 P = {0.f, 0.f, 0.f, 0.f};
                f32x4 xr[NY];
#pragma unroll
                for (int i = 0; i < NY; ++i) {
                    xr[i] = *(const f32x4 *)(lx + c * PY + 16 * i + g4);
                    const f32x4 yr = *(const f32x4 *)(ly + c * PY + 16 * i + g4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) P = __builtin_amdgcn_mfma_f32_16x16x4f32(yr[r], xr[i][r], P, 0, 0, 0);
                }
                float own = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int s = g4 + r;
                    const double Cs = lc[s];
                    const int lo = min(s, c), hi = max(s, c);
                    const bool order = a.reverse ? s >= c : s <= c;
                    const bool ok = order && ((fr >> (lo + 1)) & ((1u << (hi - lo)) - 1)) == 0;
                    const float wt = exp2_fast((float)(a.reverse ? Cs - C : C - Cs)) * a.y_scale;
                    P[r] = ok ? P[r] * wt : 0.f;
                    if (s == c) { own = P[r]; if (pw) P[r] = 0.f; }
                }
                if (pw) { own += __shfl_xor(own, 16); own += __shfl_xor(own, 32); ndt = own; }
                float dot = 0.f;
#pragma unroll
                for (int j = 0; j < NZ; ++j) {
                    f32x4 o = {0.f, 0.f, 0.f, 0.f}, in = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int r = 0; r < 4; ++r) o = __builtin_amdgcn_mfma_f32_16x16x4f32(lz[(g4 + r) * PZ + 16 * j + c], P[r], o, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < NY; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) in = __builtin_amdgcn_mfma_f32_16x16x4f32(S[i][j][r], xr[i][r], in, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = (in_ok ? o[r] + win * in[r] : o[r]) * a.out_scale;
                    const int z = 16 * j + g4;
                    if (pw) {
                        const f32x4 wv = *(const f32x4 *)(lw + c * PZ + z), zv = *(const f32x4 *)(lz + c * PZ + z);
                        dot += o[0] * wv[0] + o[1] * wv[1] + o[2] * wv[2] + o[3] * wv[3];
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[r] += ndt * a.out_scale * zv[r];
                    }
                    const int64_t t = t0 + c;
                    if (t < t_end && live) store4<T>(po + t * a.out.sl + z, o, dz - z, a.out.vec);
                }
                if (pw) {
                    dot += __shfl_xor(dot, 16); dot += __shfl_xor(dot, 32);
                    const int64_t t = t0 + c;
                    if (lane < 16 && t < t_end && live) a.dot[((slice * a.L + t) * a.B + b) * a.H + h] = dot;
                }
            }
            // S = all * S + sum_s wout_s y_s z_s
            float u[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) u[r] = __shfl(wout, g4 + r);
#pragma unroll
            for (int i = 0; i < NY; ++i) {
                float yv[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) yv[r] = ly[(g4 + r) * PY + 16 * i + c] * u[r];
#pragma unroll
                for (int j = 0; j < NZ; ++j) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[i][j][r] = all_ok ? S[i][j][r] * all : 0.f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(yv[r], lz[(g4 + r) * PZ + 16 * j + c], S[i][j], 0, 0, 0);
                }
            }
            whole *= all;
        }
    }
    if (a.state_out) {
#pragma unroll
        for (int i = 0; i < NY; ++i)
#pragma unroll
            for (int j = 0; j < NZ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int y = 16 * i + g4 + r, z = 16 * j + c;
                    if (y < dy && z < dz)
                        a.state_out[seg * a.seg_state_out + bh * (int64_t)a.dy * a.dz + y * a.o_y + (z0 + z) * a.o_z] = S[i][j][r];
                }
    }
    if (a.seg_decay && slice == 0 && lane == 0) a.seg_decay[seg * heads + bh] = whole;
}

// The states at the segments' starts (backwards: behind their ends) from what each segment adds to an empty state: in place, one thread per element.
__global__ __launch_bounds__(256) void memory_join_kernel(float *seg_states, const float *seg_decay, const float *init, float *last,
                                                          int64_t heads, int elems, int nseg, int reverse) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = heads * elems;
    if (i >= total) return;
    const int64_t bh = i / elems;
    float S = init ? init[i] : 0.f;
    for (int n = 0; n < nseg; ++n) {
        const int seg = reverse ? nseg - 1 - n : n;
        const float d = seg_decay[seg * heads + bh], u = seg_states[seg * total + i];
        seg_states[seg * total + i] = S;
        S = (d == 0.f ? 0.f : d * S) + u;
    }
    if (last) last[i] = S;
}

// dg_1 = <S_0, dS_0>, dg_{t+1} = dg_t - (q_t . dq_t - k_t . dk_t), 0 where an episode starts: the gradient of the log decays from the sums that the dq and
// dk walks left, each without the token's own term (which is in both and cancels).  float64: the running difference outlives many tokens.
// One workgroup of `blockDim` threads per (batch, head); every thread takes a run of tokens, the runs are joined by a scan.
// THREADS = 1 workgroup of 256 serves 256 (batch, head) pairs, one per thread: short sequences.
struct DecayGrad {
    const float *dot_q, *dot_k;      // (slices_q | slices_k, L, B, H)
    const float *state, *d_state;    // (B, H, elems); state may be NULL
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    float *dg;                       // (L, B, H) or NULL
    double *partial;                 // (B, H): sums over the tokens, or NULL
    int64_t L, B;
    int H, elems, slices_q, slices_k;
};

__device__ __forceinline__ double decay_step(const DecayGrad &a, int64_t t, int64_t bh) {
    const int64_t n = a.L * a.B * a.H, i = t * a.B * a.H + bh;
    double d = 0.0;
    for (int s = 0; s < a.slices_q; ++s) d += a.dot_q[s * n + i];
    for (int s = 0; s < a.slices_k; ++s) d -= a.dot_k[s * n + i];
    return d;
}

__device__ __forceinline__ bool decay_fresh(const DecayGrad &a, int64_t t, int64_t b, int h) {
    return (a.masks && a.masks[t * a.ml + b * a.mb] == 0.f) || a.g[t * a.gl + b * a.gb + h * a.gh] == -__builtin_inff();
}

__global__ __launch_bounds__(256) void decay_grad_short_kernel(DecayGrad a) {
    const int64_t bh = (int64_t)blockIdx.x * 256 + threadIdx.x, heads = a.B * a.H;
    // <S_0, dS_0> of the workgroup's pairs first: a wave per pair, coalesced
    __shared__ double first[256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int p = wave; p < 256; p += 4) {
        const int64_t q = (int64_t)blockIdx.x * 256 + p;
        double d = 0.0;
        if (a.state && q < heads)
            for (int e = lane; e < a.elems; e += 64) d += (double)a.state[q * a.elems + e] * (double)a.d_state[q * a.elems + e];
        for (int off = 32; off; off >>= 1) d += __shfl_down(d, off);
        if (lane == 0) first[p] = d;
    }
    __syncthreads();
    if (bh >= heads) return;
    const int64_t b = bh / a.H;
    const int h = (int)(bh - b * a.H);
    double run = first[threadIdx.x], sum = 0.0;
    for (int64_t t = 0; t < a.L; ++t) {
        if (decay_fresh(a, t, b, h)) run = 0.0;
        if (a.dg) a.dg[t * heads + bh] = (float)run;
        sum += run;
        run -= decay_step(a, t, bh);
    }
    if (a.partial) a.partial[bh] = sum;
}

__global__ __launch_bounds__(1024) void decay_grad_long_kernel(DecayGrad a) {
    __shared__ double part[1024], sums[16];
    __shared__ int cut[1024];
    const int64_t bh = blockIdx.x, heads = a.B * a.H, b = bh / a.H;
    const int h = (int)(bh - b * a.H), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double first = 0.0;
    if (a.state)
        for (int e = tid; e < a.elems; e += 1024) first += (double)a.state[bh * a.elems + e] * (double)a.d_state[bh * a.elems + e];
    for (int off = 32; off; off >>= 1) first += __shfl_down(first, off);
    if (lane == 0) sums[wave] = first;
    __syncthreads();
    first = 0.0;
    for (int w = 0; w < 16; ++w) first += sums[w];
    // this thread's run of tokens: what it adds behind its last start of an episode, and whether it holds one
    const int64_t per = (a.L + 1023) / 1024, t0 = min(a.L, tid * per), t1 = min(a.L, t0 + per);
    double add = 0.0;
    int any = 0;
    for (int64_t t = t0; t < t1; ++t) {
        if (decay_fresh(a, t, b, h)) { add = 0.0; any = 1; }
        add -= decay_step(a, t, bh);
    }
    part[tid] = add; cut[tid] = any;
    __syncthreads();
    for (int off = 1; off < 1024; off <<= 1) {   // inclusive scan of (add, cut): the later one wins where it holds a start
        double p = part[tid]; int q = cut[tid];
        if (tid >= off && !q) { p += part[tid - off]; q = cut[tid - off]; }
        __syncthreads();
        part[tid] = p; cut[tid] = q;
        __syncthreads();
    }
    double run = tid ? part[tid - 1] + (cut[tid - 1] ? 0.0 : first) : first, sum = 0.0;
    for (int64_t t = t0; t < t1; ++t) {
        if (decay_fresh(a, t, b, h)) run = 0.0;
        if (a.dg) a.dg[t * heads + bh] = (float)run;
        sum += run;
        run -= decay_step(a, t, bh);
    }
    __syncthreads();
    for (int off = 32; off; off >>= 1) sum += __shfl_down(sum, off);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0 && a.partial) {
        double s = 0.0;
        for (int w = 0; w < 16; ++w) s += sums[w];
        a.partial[bh] = s;
    }
}

// the sums over the batch of a decay that all tokens of a head share: one workgroup per head, a fixed order
__global__ __launch_bounds__(256) void decay_sum_kernel(const double *partial, float *dg, int64_t B, int H) {
    __shared__ double red[4];
    double s = 0.0;
    for (int64_t b = threadIdx.x; b < B; b += 256) s += partial[b * H + blockIdx.x];
    for (int off = 32; off; off >>= 1) s += __shfl_down(s, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) dg[blockIdx.x] = (float)(red[0] + red[1] + red[2] + red[3]);
}

// One token per sequence (a rollout's env step): S' = r e^g S + k^T v, o = scale q S'.  The state is read and written once, 8 dk dv bytes per head, and
// nothing else weighs: HBM.  A wave takes 64 / LZ rows of the state at a time, lane = (row group, four columns); o is summed over the row groups.
struct Step {
    WalkRows q, k, v, out;
    const float *g; int64_t gb, gh;
    const float *masks; int64_t mb;
    const float *state; float *state_out;
    int64_t B; int H, dk, dv;
    int vec;                     // state rows are float4-aligned: dv % 4 == 0 and both bases on 16 bytes
    float scale;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void memory_step_kernel(Step a) {
    const int lane = threadIdx.x & 63;
    const int64_t bh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bh >= a.B * a.H) return;
    const int64_t b = bh / a.H;
    const int h = (int)(bh - b * a.H);
    const T *q = (const T *)a.q.p + b * a.q.sb + h * a.q.sh, *k = (const T *)a.k.p + b * a.k.sb + h * a.k.sh, *v = (const T *)a.v.p + b * a.v.sb + h * a.v.sh;
    T *out = (T *)a.out.p + b * a.out.sb + h * a.out.sh;
    const float *S = a.state ? a.state + bh * (int64_t)a.dk * a.dv : nullptr;
    float *So = a.state_out + bh * (int64_t)a.dk * a.dv;
    const float g = a.g[b * a.gb + h * a.gh];
    const bool carry = S && !(a.masks && a.masks[b * a.mb] == 0.f) && g != -__builtin_inff();
    const float decay = carry ? exp2_fast((float)((double)g * 1.4426950408889634074)) : 0.f;
    constexpr int W = VEC ? 4 : 1;
    // lanes along a row: the smallest power of two that covers it, so that few lanes idle and several rows share a wave
    int lz = 1;
    while (lz < 64 && lz * W < a.dv) lz <<= 1;
    const int rows = 64 / lz, row = lane / lz, cl = lane % lz;
    for (int z0 = 0; z0 < a.dv; z0 += lz * W) {
        const int z = z0 + cl * W;
        float vv[W], o[W];
#pragma unroll
        for (int r = 0; r < W; ++r) { vv[r] = z + r < a.dv ? (float)v[z + r] : 0.f; o[r] = 0.f; }
        for (int y = row; y < a.dk; y += rows) {
            const float kv = (float)k[y], qv = (float)q[y];
            if (z < a.dv) {
                const int64_t at = (int64_t)y * a.dv + z;
                if (VEC) {
                    f32x4 s = {0.f, 0.f, 0.f, 0.f};
                    if (carry) s = *(const f32x4 *)(S + at) * decay;
#pragma unroll
                    for (int r = 0; r < W; ++r) { s[r] += kv * vv[r]; o[r] += qv * s[r]; }
                    *(f32x4 *)(So + at) = s;
                } else {
                    const float s = (carry ? S[at] * decay : 0.f) + kv * vv[0];
                    o[0] += qv * s;
                    So[at] = s;
                }
            }
        }
        for (int off = lz; off < 64; off <<= 1)
#pragma unroll
            for (int r = 0; r < W; ++r) o[r] += __shfl_xor(o[r], off);
        if (row == 0)
#pragma unroll
            for (int r = 0; r < W; ++r) if (z + r < a.dv) out[z + r] = (T)(o[r] * a.scale);
    }
}

}  // namespace policy
}  // namespace fmarl
