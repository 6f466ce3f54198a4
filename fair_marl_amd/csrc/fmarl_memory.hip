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
#include <type_traits>

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

// ---- small heads ------------------------------------------------------------------------------------------------------------
// dy <= 32: the recurrence itself, token by token, on the vector units.  16 lanes (a DPP row) hold one head: lane c column c of its slice of the state, 16 NY
// values of y each; y and x are broadcast from the lane that holds them by the multiply's own operand (row_newbcast), so a token costs three
// instructions per 64 state entries and no LDS.  Four neighbouring heads share a wave: 256 bytes of a token's row side by side.  Against the matrix walk at
// heads of 16 x 16, where half of every 16-token tile is above the diagonal and chunks of ten tokens waste the rest: 239 -> 156 us for 30 720 x 4 heads of ten
// tokens (float32, 566 MB: 111 us at the copy rate of 5.1 TB/s).
template <int M> __device__ __forceinline__ float row_lane(float v) {   // lane M of each row of 16, in every lane of the row
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + M, 0xf, 0xf, true));
}

template <int M, int N, typename F> __device__ __forceinline__ void unroll(F f) {
    if constexpr (M < N) { f(std::integral_constant<int, M>()); unroll<M + 1, N>(f); }
}

template <int CTRL> __device__ __forceinline__ float row_turn(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

__device__ __forceinline__ float row_sum(float v) {   // over the 16 lanes of a row, in every lane: rotations by 8, 4, 2, 1
    v += row_turn<0x128>(v); v += row_turn<0x124>(v); v += row_turn<0x122>(v); v += row_turn<0x121>(v);
    return v;
}

// sum_m x_m S[m], x_m in lane m of the row; four partial sums, so that no add waits for the one before.  In assembly because the compiler does not put the lane
// selection into a multiply-add (it emits a move for each: twice the instructions); s_nop 1: the two wait states between a vector write of x and its
// use by another lane.
__device__ __forceinline__ float row_dot16(float x, const float *S) {
    float a, b, c, d;
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %4, %5 row_newbcast:0 row_mask:0xf bank_mask:0xf\n\t"
        "v_mul_f32_dpp %1, %4, %6 row_newbcast:1 row_mask:0xf bank_mask:0xf\n\t"
        "v_mul_f32_dpp %2, %4, %7 row_newbcast:2 row_mask:0xf bank_mask:0xf\n\t"
        "v_mul_f32_dpp %3, %4, %8 row_newbcast:3 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %4, %9 row_newbcast:4 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %4, %10 row_newbcast:5 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %4, %11 row_newbcast:6 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %4, %12 row_newbcast:7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %4, %13 row_newbcast:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %4, %14 row_newbcast:9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %4, %15 row_newbcast:10 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %4, %16 row_newbcast:11 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %4, %17 row_newbcast:12 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %4, %18 row_newbcast:13 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %4, %19 row_newbcast:14 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %4, %20 row_newbcast:15 row_mask:0xf bank_mask:0xf"
        : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
        : "v"(x), "v"(S[0]), "v"(S[1]), "v"(S[2]), "v"(S[3]), "v"(S[4]), "v"(S[5]), "v"(S[6]), "v"(S[7]), "v"(S[8]), "v"(S[9]), "v"(S[10]), "v"(S[11]), "v"(S[12]),
          "v"(S[13]), "v"(S[14]), "v"(S[15]));
    return (a + b) + (c + d);
}

template <int NY> __device__ __forceinline__ float row_dot(const float (&x)[NY], const float (&S)[16 * NY]) {
    float o = row_dot16(x[0], S);
    if constexpr (NY == 2) o += row_dot16(x[1], S + 16);
    return o;
}

// S <- keep ? a S + y z : y z, y_m in lane m of the row: one multiply that selects the lane, one multiply-add.  Selected, not multiplied by zero, where the state
// is not kept: whatever it held is gone.
template <int NY> __device__ __forceinline__ void row_update(float (&S)[16 * NY], float a, bool fresh, const float (&y)[NY], float z) {
    if (__ballot(fresh))
#pragma unroll
        for (int m = 0; m < 16 * NY; ++m) S[m] = fresh ? 0.f : S[m];
    unroll<0, 16 * NY>([&](auto m) { S[m] = __builtin_fmaf(S[m], a, row_lane<m % 16>(y[m / 16]) * z); });
}

// S[m] <- element (m, z) of a state; `run`: its y axis is contiguous and float4s line up
template <int N> __device__ __forceinline__ void row_state(float (&S)[N], const float *p, int64_t s_y, int dy, bool real, bool run) {
    if (run) {
#pragma unroll
        for (int m = 0; m < N; m += 4) {
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (real && m < dy) v = *(const f32x4 *)(p + m);
#pragma unroll
            for (int r = 0; r < 4; ++r) S[m + r] = v[r];
        }
    } else {
#pragma unroll
        for (int m = 0; m < N; ++m) S[m] = real && m < dy ? p[m * s_y] : 0.f;
    }
}

template <typename T, int NY, bool DOT>
__global__ __launch_bounds__(256) void memory_rows_kernel(Walk a) {
    constexpr int TB = NY == 1 ? 8 : 4;   // tokens whose rows are in flight while as many are computed
    const int lane = threadIdx.x & 63, c = lane & 15;
    const int64_t heads = a.B * a.H, groups = (heads + 3) / 4;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= groups * a.nseg * a.slices) return;
    const int64_t mine = unit % groups * 4 + (lane >> 4), rest = unit / groups;
    const bool have = mine < heads;
    const int64_t bh = have ? mine : heads - 1;
    const int slice = (int)(rest % a.slices), seg = (int)(rest / a.slices);
    const int64_t b = bh / a.H;
    const int h = (int)(bh - b * a.H);
    const int z = slice * 16 + c, dy = a.dy;
    const bool zin = z < a.dz;
    const int64_t t_begin = (int64_t)seg * a.seg_len, t_end = min(a.L, t_begin + a.seg_len), count = t_end - t_begin;
    const T *px = a.state_only ? nullptr : (const T *)a.x.p + b * a.x.sb + h * a.x.sh + c, *py = (const T *)a.y.p + b * a.y.sb + h * a.y.sh + c;
    const T *pz = (const T *)a.z.p + b * a.z.sb + h * a.z.sh + z, *pw = DOT ? (const T *)a.w.p + b * a.w.sb + h * a.w.sh + z : nullptr;
    T *po = a.state_only ? nullptr : (T *)a.out.p + b * a.out.sb + h * a.out.sh + z;
    const float *pg = a.g + b * a.gb + h * a.gh, *pm = a.masks ? a.masks + b * a.mb : nullptr;

    float S[16 * NY];
    if (a.state) {
        const float *ps = a.state + seg * a.seg_state_in + bh * (int64_t)a.dy * a.dz + (int64_t)z * a.s_z;
        row_state(S, ps, a.s_y, dy, zin, a.s_y == 1 && (dy & 3) == 0 && ((uintptr_t)a.state & 15) == 0);
    } else {
#pragma unroll
        for (int m = 0; m < 16 * NY; ++m) S[m] = 0.f;
    }
    float whole = 1.f;
    float nx[TB][NY], ny[TB][NY], nz[TB], nw[TB], ng = 0.f, nm = 1.f;
    // step i of the walk is token i of the segment, or token i from its end
    auto token = [&](int64_t i) { return a.reverse ? t_end - 1 - i : t_begin + i; };
    auto fetch = [&](int64_t i0) {
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const bool in = i0 + i < count;
            const int64_t t = in ? token(i0 + i) : t_begin;
#pragma unroll
            for (int n = 0; n < NY; ++n) {
                const bool yin = in && 16 * n + c < dy;
                nx[i][n] = px && yin ? (float)px[t * a.x.sl + 16 * n] : 0.f;
                ny[i][n] = yin ? (float)py[t * a.y.sl + 16 * n] : 0.f;
            }
            nz[i] = in && zin ? (float)pz[t * a.z.sl] : 0.f;
            if (DOT) nw[i] = in && zin ? (float)pw[t * a.w.sl] : 0.f;
        }
        const bool in = c < TB && i0 + c < count;   // lane c: the decay of step i0 + c
        const int64_t t = in ? token(i0 + c) : t_begin;
        ng = in ? pg[t * a.gl] : 0.f;
        nm = in && pm ? pm[t * a.ml] : 1.f;
    };
    fetch(0);
    for (int64_t i0 = 0; i0 < count; i0 += TB) {
        float x[TB][NY], y[TB][NY], zz[TB], ww[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
#pragma unroll
            for (int n = 0; n < NY; ++n) { x[i][n] = nx[i][n]; y[i][n] = ny[i][n] * a.y_scale; }
            zz[i] = nz[i]; ww[i] = DOT ? nw[i] : 0.f;
        }
        const float fresh_l = nm == 0.f || ng == -__builtin_inff() ? 1.f : 0.f;
        const float decay_l = fresh_l != 0.f ? 0.f : exp2_fast((float)((double)ng * 1.4426950408889634074));
        if (i0 + TB < count) fetch(i0 + TB);
        unroll<0, TB>([&](auto ii) {
            constexpr int i = ii;
            if (i0 + i < count) {
                const float d = row_lane<i>(decay_l);
                const bool fresh = row_lane<i>(fresh_l) != 0.f;
                if (a.state_only) whole *= fresh ? 0.f : d;
                else {
                    float nd = row_dot<NY>(x[i], S);       // from the tokens before (backwards: behind); forwards the token's decay lies between
                    if (!a.reverse) nd = fresh ? 0.f : nd * d;
                    float xy = 0.f;
#pragma unroll
                    for (int n = 0; n < NY; ++n) xy += x[i][n] * y[i][n];
                    xy = row_sum(xy);
                    const int64_t t = token(i0 + i);
                    if (have && zin) po[t * a.out.sl] = (T)((nd + xy * zz[i]) * a.out_scale);
                    if (DOT) {
                        const float dot = row_sum(nd * a.out_scale * ww[i]);
                        if (have && c == 0) a.dot[((slice * a.L + t) * a.B + b) * a.H + h] = dot;
                    }
                }
                if (!a.reverse) row_update<NY>(S, d, fresh, y[i], zz[i]);
                else {
                    row_update<NY>(S, d, false, y[i], zz[i] * d);
                    if (__ballot(fresh))
#pragma unroll
                        for (int m = 0; m < 16 * NY; ++m) S[m] = fresh ? 0.f : S[m];
                }
            }
        });
    }
    if (a.state_out && have && zin) {
        float *ps = a.state_out + seg * a.seg_state_out + bh * (int64_t)a.dy * a.dz + (int64_t)z * a.o_z;
#pragma unroll
        for (int m = 0; m < 16 * NY; ++m) if (m < dy) ps[m * a.o_y] = S[m];
    }
    if (a.seg_decay && slice == 0 && c == 0 && have) a.seg_decay[seg * heads + bh] = whole;
}

// All gradients of up to 16 tokens of heads up to 16 x 16 in one pass (the update's chunks): q, k, v and dout stay in registers -- 16 lanes a head, as above --, the state is walked
// forwards for dq, its gradient backwards for dk (lane = row) and dv (lane = column).  dg_t = <S_L, dS_L> + sum_{i >= t} (q_i . dq_i - k_i . dk_i), each
// without the token's own term, 0 where an episode starts.  Reads and writes everything once: 928 MB for 30 720 x 4 heads of ten tokens, 182 us at the copy
// rate; it takes 221 us, three walks and the decay's kernel took 872 us.
struct ShortGrad {
    WalkRows q, k, v, o, dq, dk, dv;
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    const float *state, *d_state;
    float *d_state0, *dg;            // NULL: not wanted
    double *partial;                 // (B, H) sums of dg, or NULL
    int64_t B;
    int L, H, dk_dim, dv_dim, wide;  // wide: states are read and written in float4s
    float scale;
};

template <typename T>
__global__ __launch_bounds__(256) void memory_short_backward_kernel(ShortGrad a) {
    const int lane = threadIdx.x & 63, c = lane & 15;
    const int64_t heads = a.B * a.H;
    const int64_t mine = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 + (lane >> 4);
    if ((mine & ~(int64_t)3) >= heads) return;
    const bool have = mine < heads;
    const int64_t bh = have ? mine : heads - 1;
    const int64_t b = bh / a.H;
    const int h = (int)(bh - b * a.H), K = a.dk_dim, V = a.dv_dim, L = a.L;
    const bool kin = c < K, vin = c < V;
    float q[16], k[16], v[16], o[16], xs[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const bool in = t < L;
        q[t] = in && kin ? (float)((const T *)a.q.p)[t * a.q.sl + b * a.q.sb + h * a.q.sh + c] : 0.f;
        k[t] = in && kin ? (float)((const T *)a.k.p)[t * a.k.sl + b * a.k.sb + h * a.k.sh + c] : 0.f;
        v[t] = in && vin ? (float)((const T *)a.v.p)[t * a.v.sl + b * a.v.sb + h * a.v.sh + c] : 0.f;
        o[t] = in && vin ? (float)((const T *)a.o.p)[t * a.o.sl + b * a.o.sb + h * a.o.sh + c] : 0.f;
    }
    const float gl = c < L ? a.g[c * a.gl + b * a.gb + h * a.gh] : 0.f, ml = c < L && a.masks ? a.masks[c * a.ml + b * a.mb] : 1.f;
    const int64_t at = bh * (int64_t)K * V;
    float S[16], G[16], C[16];        // S, G: row c of the state and of its gradient; C: column c of the gradient
    if (a.state) row_state(S, a.state + at + c * V, 1, V, kin, a.wide);
    else {
#pragma unroll
        for (int m = 0; m < 16; ++m) S[m] = 0.f;
    }
    const float fresh_l = ml == 0.f || gl == -__builtin_inff() ? 1.f : 0.f;
    const float decay_l = fresh_l != 0.f ? 0.f : exp2_fast((float)((double)gl * 1.4426950408889634074));
    unroll<0, 16>([&](auto tt) {
        constexpr int t = tt;
        if (t < L) {
            const bool fresh = row_lane<t>(fresh_l) != 0.f;
            const float d = row_lane<t>(decay_l), x1[1] = {o[t]}, nd = fresh ? 0.f : row_dot<1>(x1, S) * d, vo = row_sum(v[t] * o[t]);
            if (have && kin) ((T *)a.dq.p)[t * a.dq.sl + b * a.dq.sb + h * a.dq.sh + c] = (T)((nd + k[t] * vo) * a.scale);
            xs[t] = row_sum(q[t] * nd) * a.scale;
            const float y1[1] = {v[t]};
            row_update<1>(S, d, fresh, y1, k[t]);
            q[t] *= a.scale;           // from here on only in G's and dk's, dv's own terms
        }
    });
    float run = 0.f;
    if (a.d_state) {
        row_state(G, a.d_state + at + c * V, 1, V, kin, a.wide);
        row_state(C, a.d_state + at + c, V, K, vin, false);
#pragma unroll
        for (int m = 0; m < 16; ++m) run += S[m] * G[m];
        run = row_sum(run);
    } else {
#pragma unroll
        for (int m = 0; m < 16; ++m) G[m] = C[m] = 0.f;
    }
    double sum = 0.0;
    unroll<0, 16>([&](auto tt) {
        constexpr int t = 15 - tt;
        if (t < L) {
            const float v1[1] = {v[t]}, k1[1] = {k[t]}, q1[1] = {q[t]}, o1[1] = {o[t]};
            const float nk = row_dot<1>(v1, G), nv = row_dot<1>(k1, C), vo = row_sum(v[t] * o[t]), qk = row_sum(q[t] * k[t]);
            if (have && kin) ((T *)a.dk.p)[t * a.dk.sl + b * a.dk.sb + h * a.dk.sh + c] = (T)(nk + q[t] * vo);
            if (have && vin) ((T *)a.dv.p)[t * a.dv.sl + b * a.dv.sb + h * a.dv.sh + c] = (T)(nv + o[t] * qk);
            run += xs[t] - row_sum(k[t] * nk);
            const bool fresh = row_lane<t>(fresh_l) != 0.f;
            const float dg = fresh ? 0.f : run, d = row_lane<t>(decay_l);
            if (fresh) run = 0.f;
            sum += dg;
            if (a.dg && have && c == 0) a.dg[t * heads + bh] = dg;
            row_update<1>(G, d, false, o1, q[t] * d);
            row_update<1>(C, d, false, q1, o[t] * d);
            if (__ballot(fresh))
#pragma unroll
                for (int m = 0; m < 16; ++m) { G[m] = fresh ? 0.f : G[m]; C[m] = fresh ? 0.f : C[m]; }
        }
    });
    if (a.d_state0 && have && kin) {
        float *p = a.d_state0 + at + c * V;
        if (a.wide) {
#pragma unroll
            for (int m = 0; m < 16; m += 4) if (m < V) *(f32x4 *)(p + m) = f32x4{G[m], G[m + 1], G[m + 2], G[m + 3]};
        } else {
#pragma unroll
            for (int m = 0; m < 16; ++m) if (m < V) p[m] = G[m];
        }
    }
    if (a.partial && have && c == 0) a.partial[bh] = sum;
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

using namespace fmarl;
using namespace fmarl::policy;

namespace {

// rows start on multiples of four elements and hold a multiple of four: one load takes four
int rows_vec(const FmarlRows &r, int d, int dtype) {
    return (d & 3) == 0 && (r.stride_l & 3) == 0 && (r.stride_b & 3) == 0 && (r.stride_h & 3) == 0 &&
           ((uintptr_t)r.data & (4 * elem_bytes(dtype) - 1)) == 0;
}

WalkRows walk_rows(const FmarlRows &r, int d, int dtype) { return WalkRows{(char *)r.data, r.stride_l, r.stride_b, r.stride_h, rows_vec(r, d, dtype)}; }

const int kMaxMemoryDim = 128;

int memory_check(const FmarlMemory *m, const char *who) {
    if (!m) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    if (m->L < 0 || m->B < 0 || m->H < 1) return policy_fail(FMARL_EINVAL, "%s: L and B must not be negative, H must be positive", who);
    if (m->dk < 1 || m->dk > kMaxMemoryDim || m->dv < 1 || m->dv > kMaxMemoryDim) return policy_fail(FMARL_EINVAL, "%s: dk and dv must lie in 1..128", who);
    if (m->dtype < FMARL_T_F32 || m->dtype > FMARL_T_F16) return policy_fail(FMARL_EINVAL, "%s: unknown dtype", who);
    if (m->shared_decay < 0 || m->shared_decay > 1 || (m->shared_decay && (m->decay_stride_l || m->decay_stride_b)))
        return policy_fail(FMARL_EINVAL, "%s: shared_decay must be 0, or 1 with strides of 0 over tokens and sequences", who);
    // a wave per head and slice: a launch holds fewer than 2^32 threads
    if (m->B >= (1ll << 26) / m->H || m->L > (1ll << 40)) return policy_fail(FMARL_EINVAL, "%s: too many sequences (B H must stay below 2^26) or tokens", who);
    if (m->L > 0 && m->B > 0 && (!m->q.data || !m->k.data || !m->v.data || !m->log_decay)) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    return FMARL_OK;
}

// Waves that walk at once: a batch with fewer heads than 2 048 (8 waves per CU) has its tokens cut into segments that are walked side by side, at least 64 tokens
// each (a segment costs a second read of k and v and a state in the workspace, which shorter ones would not repay).
struct Segments { int nseg, len; };
Segments memory_segments(const FmarlMemory *m) {
    const int64_t heads = m->B * m->H;
    int64_t n = (2048 + heads - 1) / heads, most = m->L / 64;
    if (n > most) n = most;
    if (n < 2) return {1, (int)(m->L > 0x40000000 ? 0x40000000 : m->L)};
    const int64_t len = ((m->L + n - 1) / n + 15) / 16 * 16;
    return {(int)((m->L + len - 1) / len), (int)len};
}

// The recurrence on the vector units for y up to 32 wide, the matrix walk beyond: at 16 x 16 the former takes half the latter's time, at 64 x 64
// its three instructions per 64 state entries would cost twice the matrix units' time
bool small_heads(int dy) { return dy <= 32; }

int tiles(int d) { return d <= 16 ? 1 : d <= 32 ? 2 : d <= 64 ? 4 : 8; }
// columns of z that one wave takes, in tiles of 16: the state's dy x dz accumulators have to fit its registers beside the operands
int slice_tiles(int dy, int dz) { const int t = tiles(dz), most = tiles(dy) == 8 ? 2 : 4; return t > most ? most : t; }
int slices_of(int dy, int dz) { const int w = small_heads(dy) ? 16 : 16 * slice_tiles(dy, dz); return (dz + w - 1) / w; }

// up to 16 tokens of heads up to 16 x 16: every gradient in one kernel, whose registers hold all of it
bool short_backward(const FmarlMemory *m) { return m->L <= 16 && m->dk <= 16 && m->dv <= 16; }

struct Workspace {
    size_t seg_s, seg_g, decay, dot_q, dot_k, partial, d_state, total;
};
Workspace memory_layout(const FmarlMemory *m, int backward) {
    const Segments s = memory_segments(m);
    const size_t heads = (size_t)(m->B * m->H), elems = (size_t)m->dk * m->dv;
    Workspace w = {};
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += up256(bytes); return at; };
    if (s.nseg > 1) {
        w.seg_s = take(4 * s.nseg * heads * elems);
        if (backward) w.seg_g = take(4 * s.nseg * heads * elems);
        w.decay = take(4 * s.nseg * heads);
    }
    if (backward && short_backward(m)) w.partial = take(8 * heads);
    else if (backward) {
        w.dot_q = take(4 * (size_t)slices_of(m->dv, m->dk) * m->L * heads);
        w.dot_k = take(4 * (size_t)slices_of(m->dv, m->dk) * m->L * heads);
        w.partial = take(8 * heads);
        w.d_state = take(4 * heads * elems);
    }
    w.total = off;
    return w;
}

template <typename T, int NY>
void launch_walk_nz(const Walk &w, unsigned blocks, hipStream_t st) {
    switch (slice_tiles(w.dy, w.dz)) {
    case 1: hipLaunchKernelGGL((memory_walk_kernel<T, NY, 1>), dim3(blocks), dim3(256), 0, st, w); break;
    case 2: hipLaunchKernelGGL((memory_walk_kernel<T, NY, 2>), dim3(blocks), dim3(256), 0, st, w); break;
    default:
        if constexpr (NY < 8) hipLaunchKernelGGL((memory_walk_kernel<T, NY, 4>), dim3(blocks), dim3(256), 0, st, w);
    }
}

template <typename T>
void launch_walk_t(const Walk &w, unsigned blocks, hipStream_t st) {
    if (w.dy <= 16 && w.w.p) hipLaunchKernelGGL((memory_rows_kernel<T, 1, true>), dim3(blocks), dim3(256), 0, st, w);
    else if (w.dy <= 16) hipLaunchKernelGGL((memory_rows_kernel<T, 1, false>), dim3(blocks), dim3(256), 0, st, w);
    else if (w.dy <= 32 && w.w.p) hipLaunchKernelGGL((memory_rows_kernel<T, 2, true>), dim3(blocks), dim3(256), 0, st, w);
    else if (w.dy <= 32) hipLaunchKernelGGL((memory_rows_kernel<T, 2, false>), dim3(blocks), dim3(256), 0, st, w);
    else if (w.dy <= 64) launch_walk_nz<T, 4>(w, blocks, st);
    else launch_walk_nz<T, 8>(w, blocks, st);
}

int launch_walk(Walk w, int dtype, hipStream_t st) {
    w.slices = slices_of(w.dy, w.dz);
    const int64_t heads = w.B * w.H, units = small_heads(w.dy) ? (heads + 3) / 4 : heads;   // waves per segment and slice
    const int64_t blocks = (units * w.nseg * w.slices + 3) / 4;
    if (blocks > 0xffffff) return policy_fail(FMARL_EINVAL, "memory: too many sequences");
    if (dtype == FMARL_T_F32) launch_walk_t<float>(w, (unsigned)blocks, st);
    else if (dtype == FMARL_T_BF16) launch_walk_t<__bf16>(w, (unsigned)blocks, st);
    else launch_walk_t<_Float16>(w, (unsigned)blocks, st);
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

Walk walk_base(const FmarlMemory *m) {
    Walk w = {};
    const Segments s = memory_segments(m);
    w.g = m->log_decay; w.gl = m->decay_stride_l; w.gb = m->decay_stride_b; w.gh = m->decay_stride_h;
    w.masks = m->masks; w.ml = m->mask_stride_l; w.mb = m->mask_stride_b;
    w.L = m->L; w.B = m->B; w.H = m->H; w.nseg = s.nseg; w.seg_len = s.len;
    w.y_scale = w.out_scale = 1.f;
    return w;
}

// the states at the segments' starts (reverse: the gradients of the states behind their ends) into seg_states; the last one of the walk into `last`
int segment_states(const FmarlMemory *m, const FmarlRows &y, const FmarlRows &z, bool reverse, const float *init, float *last, float *seg_states,
                   float *seg_decay, hipStream_t st) {
    Walk w = walk_base(m);
    const int64_t heads = m->B * m->H, elems = (int64_t)m->dk * m->dv;
    w.y = walk_rows(y, m->dk, m->dtype); w.z = walk_rows(z, m->dv, m->dtype);
    w.dy = m->dk; w.dz = m->dv; w.state_only = 1; w.reverse = reverse;
    if (reverse) w.y_scale = m->scale;
    w.state_out = seg_states; w.o_y = m->dv; w.o_z = 1; w.seg_state_out = heads * elems; w.seg_decay = seg_decay;
    if (int rc = launch_walk(w, m->dtype, st)) return rc;
    const int64_t blocks = (heads * elems + 255) / 256;
    hipLaunchKernelGGL(memory_join_kernel, dim3((unsigned)blocks), dim3(256), 0, st, seg_states, (const float *)seg_decay, init, last, heads, (int)elems, w.nseg, (int)reverse);
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

}  // namespace

extern "C" {

int fmarl_memory_step(const FmarlMemory *m, const FmarlRows *out, float *state_out, void *stream) {
    if (int rc = memory_check(m, "fmarl_memory_step")) return rc;
    if (m->L != 1) return policy_fail(FMARL_EINVAL, "fmarl_memory_step: L must be 1");
    if (m->B == 0) return FMARL_OK;
    if (!out || !out->data || !state_out) return policy_fail(FMARL_EINVAL, "fmarl_memory_step: null argument");
    Step s = {};
    s.q = walk_rows(m->q, m->dk, m->dtype); s.k = walk_rows(m->k, m->dk, m->dtype); s.v = walk_rows(m->v, m->dv, m->dtype);
    s.out = walk_rows(*out, m->dv, m->dtype);
    s.g = m->log_decay; s.gb = m->decay_stride_b; s.gh = m->decay_stride_h; s.masks = m->masks; s.mb = m->mask_stride_b;
    s.state = m->state; s.state_out = state_out; s.B = m->B; s.H = m->H; s.dk = m->dk; s.dv = m->dv; s.scale = m->scale;
    const bool vec = (m->dv & 3) == 0 && (((uintptr_t)m->state | (uintptr_t)state_out) & 15) == 0;
    const int64_t blocks = (m->B * m->H + 3) / 4;
    hipStream_t st = (hipStream_t)stream;
#define FMARL_STEP(T) do { if (vec) hipLaunchKernelGGL((memory_step_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, s); \
                           else hipLaunchKernelGGL((memory_step_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, s); } while (0)
    if (m->dtype == FMARL_T_F32) FMARL_STEP(float);
    else if (m->dtype == FMARL_T_BF16) FMARL_STEP(__bf16);
    else FMARL_STEP(_Float16);
#undef FMARL_STEP
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

size_t fmarl_memory_workspace(const FmarlMemory *m, int backward) {
    if (memory_check(m, "fmarl_memory_workspace")) return 0;
    if (m->L == 0 || m->B == 0) return 256;
    const size_t n = memory_layout(m, backward).total;
    return n ? n : 256;
}

int fmarl_memory_chunk(const FmarlMemory *m, const FmarlRows *out, float *state_out, void *workspace, void *stream) {
    if (int rc = memory_check(m, "fmarl_memory_chunk")) return rc;
    if (m->B == 0) return FMARL_OK;
    if (m->L < 1) return policy_fail(FMARL_EINVAL, "fmarl_memory_chunk: L must be positive");
    if (!out || !out->data || !state_out || !workspace) return policy_fail(FMARL_EINVAL, "fmarl_memory_chunk: null argument");
    hipStream_t st = (hipStream_t)stream;
    const Workspace ws = memory_layout(m, 0);
    char *base = (char *)workspace;
    Walk w = walk_base(m);
    if (w.nseg > 1)
        if (int rc = segment_states(m, m->k, m->v, false, m->state, state_out, (float *)(base + ws.seg_s), (float *)(base + ws.decay), st)) return rc;
    w.x = walk_rows(m->q, m->dk, m->dtype); w.y = walk_rows(m->k, m->dk, m->dtype); w.z = walk_rows(m->v, m->dv, m->dtype);
    w.out = walk_rows(*out, m->dv, m->dtype);
    w.dy = m->dk; w.dz = m->dv; w.out_scale = m->scale;
    w.s_y = w.o_y = m->dv; w.s_z = w.o_z = 1;
    if (w.nseg > 1) { w.state = (const float *)(base + ws.seg_s); w.seg_state_in = m->B * m->H * (int64_t)m->dk * m->dv; }
    else { w.state = m->state; w.state_out = state_out; }
    return launch_walk(w, m->dtype, st);
}

int fmarl_memory_chunk_backward(const FmarlMemory *m, const FmarlRows *d_out, const float *d_state, const FmarlRows *d_q, const FmarlRows *d_k,
                                const FmarlRows *d_v, float *d_log_decay, float *d_state0, void *workspace, void *stream) {
    if (int rc = memory_check(m, "fmarl_memory_chunk_backward")) return rc;
    if (m->B == 0) return FMARL_OK;
    if (m->L < 1) return policy_fail(FMARL_EINVAL, "fmarl_memory_chunk_backward: L must be positive");
    if (!d_out || !d_out->data || !d_q || !d_q->data || !d_k || !d_k->data || !d_v || !d_v->data || !workspace)
        return policy_fail(FMARL_EINVAL, "fmarl_memory_chunk_backward: null argument");
    hipStream_t st = (hipStream_t)stream;
    const Workspace ws = memory_layout(m, 1);
    char *base = (char *)workspace;
    const Walk w0 = walk_base(m);
    const int64_t heads = m->B * m->H;
    if (short_backward(m)) {
        ShortGrad g = {};
        const int dt = m->dtype;
        g.q = walk_rows(m->q, m->dk, dt); g.k = walk_rows(m->k, m->dk, dt); g.v = walk_rows(m->v, m->dv, dt); g.o = walk_rows(*d_out, m->dv, dt);
        g.dq = walk_rows(*d_q, m->dk, dt); g.dk = walk_rows(*d_k, m->dk, dt); g.dv = walk_rows(*d_v, m->dv, dt);
        g.g = w0.g; g.gl = w0.gl; g.gb = w0.gb; g.gh = w0.gh; g.masks = w0.masks; g.ml = w0.ml; g.mb = w0.mb;
        g.state = m->state; g.d_state = d_state; g.d_state0 = d_state0; g.dg = m->shared_decay ? nullptr : d_log_decay;
        g.partial = m->shared_decay && d_log_decay ? (double *)(base + ws.partial) : nullptr;
        g.B = m->B; g.L = (int)m->L; g.H = m->H; g.dk_dim = m->dk; g.dv_dim = m->dv; g.scale = m->scale;
        g.wide = (m->dv & 3) == 0 && (((uintptr_t)m->state | (uintptr_t)d_state | (uintptr_t)d_state0) & 15) == 0;
        const dim3 grid((unsigned)((heads + 15) / 16));
        if (dt == FMARL_T_F32) hipLaunchKernelGGL(memory_short_backward_kernel<float>, grid, dim3(256), 0, st, g);
        else if (dt == FMARL_T_BF16) hipLaunchKernelGGL(memory_short_backward_kernel<__bf16>, grid, dim3(256), 0, st, g);
        else hipLaunchKernelGGL(memory_short_backward_kernel<_Float16>, grid, dim3(256), 0, st, g);
        if (g.partial) hipLaunchKernelGGL(decay_sum_kernel, dim3((unsigned)m->H), dim3(256), 0, st, (const double *)g.partial, d_log_decay, m->B, m->H);
        HIP_OK(hipGetLastError());
        return FMARL_OK;
    }
    const int elems = m->dk * m->dv;
    float *seg_s = (float *)(base + ws.seg_s), *seg_g = (float *)(base + ws.seg_g), *decay = (float *)(base + ws.decay);
    float *ds0 = d_state0 ? d_state0 : (float *)(base + ws.d_state);
    if (w0.nseg > 1) {
        if (int rc = segment_states(m, m->k, m->v, false, m->state, nullptr, seg_s, decay, st)) return rc;
        if (int rc = segment_states(m, m->q, *d_out, true, d_state, ds0, seg_g, decay, st)) return rc;
    }
    const int64_t seg_elems = w0.nseg > 1 ? heads * elems : 0;
    const int dt = m->dtype;
    const WalkRows q = walk_rows(m->q, m->dk, dt), k = walk_rows(m->k, m->dk, dt), v = walk_rows(m->v, m->dv, dt), o = walk_rows(*d_out, m->dv, dt);
    Walk w = w0;   // dq: forwards, the state seen as its transpose
    w.x = o; w.y = v; w.z = k; w.w = q; w.out = walk_rows(*d_q, m->dk, dt); w.dot = (float *)(base + ws.dot_q);
    w.dy = m->dv; w.dz = m->dk; w.out_scale = m->scale; w.s_y = 1; w.s_z = m->dv;
    w.state = w0.nseg > 1 ? seg_s : m->state; w.seg_state_in = seg_elems;
    if (int rc = launch_walk(w, dt, st)) return rc;
    w = w0;        // dk: backwards
    w.x = v; w.y = o; w.z = q; w.w = k; w.out = walk_rows(*d_k, m->dk, dt); w.dot = (float *)(base + ws.dot_k);
    w.dy = m->dv; w.dz = m->dk; w.y_scale = m->scale; w.s_y = 1; w.s_z = m->dv; w.reverse = 1;
    w.state = w0.nseg > 1 ? seg_g : d_state; w.seg_state_in = seg_elems;
    if (int rc = launch_walk(w, dt, st)) return rc;
    w = w0;        // dv, and the gradient of the initial state
    w.x = k; w.y = q; w.z = o; w.out = walk_rows(*d_v, m->dv, dt);
    w.dy = m->dk; w.dz = m->dv; w.y_scale = m->scale; w.s_y = w.o_y = m->dv; w.s_z = w.o_z = 1; w.reverse = 1;
    w.state = w0.nseg > 1 ? seg_g : d_state; w.seg_state_in = seg_elems;
    if (w0.nseg == 1) w.state_out = ds0;
    if (int rc = launch_walk(w, dt, st)) return rc;
    if (d_log_decay) {
        DecayGrad g = {};
        const bool shared = m->shared_decay != 0;
        g.dot_q = (const float *)(base + ws.dot_q); g.dot_k = (const float *)(base + ws.dot_k);
        g.state = m->state; g.d_state = ds0; g.g = w0.g; g.gl = w0.gl; g.gb = w0.gb; g.gh = w0.gh; g.masks = w0.masks; g.ml = w0.ml; g.mb = w0.mb;
        g.dg = shared ? nullptr : d_log_decay; g.partial = shared ? (double *)(base + ws.partial) : nullptr;
        g.L = m->L; g.B = m->B; g.H = m->H; g.elems = elems; g.slices_q = g.slices_k = slices_of(m->dv, m->dk);
        // a thread per (batch, head) while its tokens are few; otherwise a workgroup per (batch, head), whose threads share the tokens
        if (m->L <= 64) hipLaunchKernelGGL(decay_grad_short_kernel, dim3((unsigned)((heads + 255) / 256)), dim3(256), 0, st, g);
        else hipLaunchKernelGGL(decay_grad_long_kernel, dim3((unsigned)heads), dim3(1024), 0, st, g);
        if (shared) hipLaunchKernelGGL(decay_sum_kernel, dim3((unsigned)m->H), dim3(256), 0, st, (const double *)(base + ws.partial), d_log_decay, m->B, m->H);
        HIP_OK(hipGetLastError());
    }
    return FMARL_OK;
}

}  // extern "C"
