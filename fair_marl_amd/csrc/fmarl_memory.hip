// The memory of a recurrent policy on gfx950: linear attention with a decay per head.  With r_t = 0 where an episode starts at t
// (masks_t == 0; also where e^{g_t} is below float32's smallest number) and 1 elsewhere,
//     S_t = r_t e^{g_t} S_{t-1} + k_t^T v_t          o_t = scale * q_t S_t
// and backwards, with G_t the gradient of S_t,
//     G_t = scale * q_t^T do_t + r_{t+1} e^{g_{t+1}} G_{t+1}      dq_t = scale * do_t S_t^T     dk_t = v_t G_t^T     dv_t = k_t G_t
//     dS_0 = r_1 e^{g_1} G_1                                      dg_t = r_t e^{g_t} <S_{t-1}, G_t>.
// o, dq, dk and dv are the same walk over the tokens, forwards or backwards, with the operands in other roles:
//     out_t = sum_{s before or at t} w(t, s) (x_t . y_s) z_s + (what the walk carries):
//     o: x, y, z = q, k, v forwards;  dq: do, v, k forwards (state S^T);  dk: v, do, q backwards (state G^T);  dv: k, q, do backwards.
// memory_tiles_kernel (large heads, the matrix units) and memory_rows_kernel (small ones) are that walk.
#include <type_traits>

#include "fmarl_policy_dev.h"

namespace fmarl {
namespace policy {

struct WalkRows {            // a (L, B, H, d) tensor whose last axis is contiguous
    char *p;
    int64_t sl, sb, sh;      // strides in elements
    int vec;                 // rows start on multiples of four elements and hold a multiple of four
};

// A walk goes through its tokens in memory order; the host turns the arrays round for a backwards one (the last token first, negative strides).  Forwards a token's decay lies
// before it, backwards behind it: with `shift` the state is decayed by the token before's, and by the last one's at the end.
struct Walk {
    WalkRows x, y, z, w, out;          // w: what out is dotted with for the decay's gradient, or NULL
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    const float *state;                // initial state, NULL: zeros; element (y, z) of (b, h) at (b * H + h) * dy * dz + y * s_y + z * s_z
    float *state_out;                  // NULL: not wanted
    int64_t s_y, s_z, o_y, o_z;        // the strides of the two
    int64_t seg_state_in, seg_state_out;   // elements from one segment's states to the next one's (0: the same for all)
    float *seg_decay;                  // state_only: the segment's whole decay, (nseg, B * H)
    float *dot; int64_t dot_sl, dot_sh, dot_slice;   // sums of out * w without the token's own term: strides of token, (b, h) and slice
    int64_t L, B;
    int H, dy, dz, nseg, seg_len, slices;
    int shift, state_only;
    float y_scale, out_scale;
};

// nothing from before reaches a token: an episode starts at it, or its decay's factor is below float32's smallest number (-inf, or a type's lowest value in its place, whose sum
// with the other tokens' decays would lose theirs)
__device__ __forceinline__ bool forgets(float g, float mask) { return mask == 0.f || g < -128.f; }

// ---- large heads ------------------------------------------------------------------------------------------------------------
// A workgroup walks one (batch, head, segment) in chunks of 32 tokens; wave w holds columns 16 w .. 16 w + 15 of the state (float32, in the accumulator layout of
// mfma_f32_16x16x32_bf16: row 4 * (lane / 16) + r, column lane % 16), so a chunk is read once for all of it:
//     P^T = y x^T, weighted (three 16 x 16 tiles, shared out over the waves);  out^T = z^T P^T + S^T x^T;  S = e^C S + y^T (u z).
// All products are bfloat16 ones of exact pieces: a bfloat16 value is one piece, a float16 value two, a float32 value three (8 + 8 + 8 bits), and what is
// formed in float32 (P, S, u z) is cut into three, whatever the output's type: terms that cancel leave what their last bits hold.  Products whose place is below 2^-24 of the result
// are left out.  Per product of 16 x 16 x 32 that is 1 to 6 instructions of 16 cycles against eight of 32 cycles of mfma_f32_16x16x4f32.
// The accumulator layout serves as either operand's layout if the contraction runs in the order 8 * (lane / 16) + 4 * tile + r for the index 16 * tile + 4 * (lane / 16) + r
// (two tiles to a contraction of 32): rows in LDS are stored in that order, so every operand is one 16-byte read.
// The decays' prefix sums are float64, so a weight e^{C_t - C_s} is right to float32 however fast the tokens before forgot.  A weight is selected, not multiplied to
// zero: what an episode left behind (infinities too) does not reach the next one; a chunk that holds a value that is not finite is walked token by token, so
// that it reaches later tokens only.
// 64 heads of 4 096 tokens, 64 x 64, bfloat16 (segments of 256 tokens, four workgroups a CU): 33 us for the states alone, 53 us for out, 77 us for out with its sums against w, where the
// bytes take 13 to 27 us and the matrix instructions 4 us: a chunk is three barriers and some 400 vector instructions a wave (pieces, weights, prefix sums), and those bound it.
// pieces of an input, and the highest order (sum of the pieces' numbers) kept in x y; P, the state as an operand and u z have three pieces, kept to order 2
template <typename T> struct Pieces;
template <> struct Pieces<__bf16> { static constexpr int in = 1, in_order = 0; };
template <> struct Pieces<_Float16> { static constexpr int in = 2, in_order = 2; };
template <> struct Pieces<float> { static constexpr int in = 3, in_order = 2; };

// the pieces of four inputs, piece by piece; a bfloat16 value is its own.  What float32 holds beyond bfloat16's largest number (3.39e38) leaves a remainder, not an infinity: a type's
// lowest value may stand where nothing is read
template <typename T, int N> __device__ __forceinline__ void cut4(typename Vec4<T>::type v, bf16x4 (&p)[N]) {
    f32x4 f = widen(v);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            p[i][r] = (__bf16)(N == 3 && i == 0 ? __builtin_amdgcn_fmed3f(f[r], -0x1.fep127f, 0x1.fep127f) : f[r]);
            f[r] -= (float)p[i][r];
        }
}
template <> __device__ __forceinline__ void cut4<__bf16, 1>(bf16x4 v, bf16x4 (&p)[1]) { p[0] = v; }

// whether one of the four is not finite: its exponent's bits are all set
__device__ __forceinline__ bool not_finite(f32x4 v) { return !(v[0] - v[0] == 0.f && v[1] - v[1] == 0.f && v[2] - v[2] == 0.f && v[3] - v[3] == 0.f); }
__device__ __forceinline__ bool not_finite(bf16x4 v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 u = __builtin_bit_cast(u32x2, v);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) bad |= (u[i] & 0x7f80u) == 0x7f80u || (u[i] & 0x7f800000u) == 0x7f800000u;
    return bad;
}
__device__ __forceinline__ bool not_finite(f16x4 v) { return not_finite(widen(v)); }

template <int NA, int NB, int ORDER>
__device__ __forceinline__ f32x4 mma_pieces(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 c) {
#pragma unroll
    for (int i = NA - 1; i >= 0; --i)
#pragma unroll
        for (int j = NB - 1; j >= 0; --j)
            if (i + j <= ORDER) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], c, 0, 0, 0);
    return c;
}

// prefix sum over lanes 0 .. 31 (lanes 32 .. 63 repeat it): rows of 16 by lane shifts, the second row plus the first one's total
template <int CTRL> __device__ __forceinline__ double row_shift(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ double scan32(double v, int lane) {
    v += row_shift<0x111>(v); v += row_shift<0x112>(v); v += row_shift<0x114>(v); v += row_shift<0x118>(v);   // (lanes without a source add 0)
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t l0 = __builtin_amdgcn_readlane((int)(uint32_t)u, 15), h0 = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 15);
    return lane & 16 ? v + __builtin_bit_cast(double, ((uint64_t)h0 << 32) | l0) : v;
}

// LDS of a workgroup, in bytes: x, y (32 tokens), y^T, z^T (rows of 32 tokens), P^T, per-token floats
template <typename T> __host__ __device__ constexpr int tiles_lds(int nk, int nz) {
    return Pieces<T>::in * 2 * (2 * 32 * (32 * nk + 8) + (32 * nk + 16 * nz) * 40) + 3 * 2 * 32 * 40 + 32 * 8 + 4 * 32 * 4 + 8 * 32 * 4;
}

enum { kOut = 0, kOutDot = 1, kState = 2 };   // what a walk leaves: out; out and its dots with w; the state alone

template <typename T, int NK, int MODE, bool VEC>
__global__ __launch_bounds__(512, NK == 2 && sizeof(T) == 2 ? 4 : 2) void memory_tiles_kernel(Walk arg) {
    constexpr bool DOT = MODE == kOutDot, OUT = MODE != kState;
    constexpr int NP = Pieces<T>::in, PP = 3, XS = 32 * NK + 8;
    typedef typename Vec4<T>::type V;
    extern __shared__ __align__(16) char smem[];
    // the arguments are read where they are used, through a pointer the compiler cannot see through: all at once they do not fit the scalar registers (a hundred
    // were spilled into vector lanes, 400 v_readlane in the loop: 55 us instead of 33 us at 8 x 8 heads of 4 096 tokens)
    typedef const Walk __attribute__((address_space(4))) *WalkArg;
    uint64_t at_args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at_args));
    const Walk &a = *(const Walk *)(WalkArg)at_args;
    (void)arg;
    const int dy = a.dy, dz = a.dz, nz = (dz + 15) / 16, threads = blockDim.x;
    __bf16 *lx = (__bf16 *)smem, *ly = lx + NP * 32 * XS, *lyt = ly + NP * 32 * XS, *lzt = lyt + NP * 32 * NK * 40, *lp = lzt + NP * 16 * nz * 40;
    double *lc = (double *)(lp + PP * 32 * 40);
    float *lwin = (float *)(lc + 32), *lwout = lwin + 32, *lown = lwout + 32, *ldot = lown + 64, *lall = lown + 32;   // ldot: (waves, 32)
    uint32_t *lfr = (uint32_t *)(lown + 40);   // [0] tokens that start afresh; [1], [2]: a value is not finite, by the chunk's parity (cleared in the chunk between)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4, g4 = g * 4;
    const int heads = (int)(a.B * a.H), bh = blockIdx.x % heads, seg = blockIdx.x / heads;
    const int64_t b = bh / a.H, h = bh - b * a.H;
    const int64_t t_begin = (int64_t)seg * a.seg_len;
    const int length = (int)min(a.L - t_begin, (int64_t)a.seg_len), chunks = (length + 31) / 32;
    const int zc = 16 * wave;                  // this wave's columns of z; waves beyond nz only load and help with P
    const bool holds = wave < nz;

    f32x4 S[2 * NK];
    if (a.state) {
        const float *ps = a.state + seg * a.seg_state_in + bh * (int64_t)(dy * dz) + (zc + c) * a.s_z;
        const int64_t s_y = a.s_y;
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) { const int y = 16 * i + g4 + r; S[i][r] = y < dy && zc + c < dz ? ps[y * s_y] : 0.f; }
    } else {
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i) S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (tid < 3) lfr[tid] = 0;
    if (OUT) for (int i = tid; i < PP * 32 * 40; i += threads) lp[i] = (__bf16)0.f;   // the tile beyond the diagonal stays zero
    float whole = 1.f;

    // a thread's share of a chunk: NK pieces of four of x and of y each, two at most of z.  Where they lie is worked out once; from chunk to chunk the
    // pointers move on by 32 tokens
    auto slot = [](int s) { return 8 * ((s >> 2) & 3) + 4 * (s >> 4) + (s & 3); };   // place of index s of 32 in a stored row
    V rx[OUT ? NK : 1], ry[NK], rz[2];
    const T *qx[OUT ? NK : 1], *qy[NK], *qz[2];
    int xtok[NK], ztok[2];   // the piece's token; beyond every chunk if it lies outside the row
    int xat[NK], yat[NK], zat[2];
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        const int idx = tid + threads * n, col = (idx % (8 * NK)) * 4, tok = idx / (8 * NK);
        xtok[n] = tok < 32 ? tok : 1 << 20;
        xat[n] = tok * XS + (col & ~31) + slot(col & 31);
        yat[n] = col * 40 + slot(tok & 31);
        if (OUT) qx[n] = (const T *)a.x.p + b * a.x.sb + h * a.x.sh + (t_begin + tok) * a.x.sl + col;
        qy[n] = (const T *)a.y.p + b * a.y.sb + h * a.y.sh + (t_begin + tok) * a.y.sl + col;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int idx = tid + threads * n, tok = idx / (4 * nz), col = (idx - tok * 4 * nz) * 4;
        ztok[n] = tok < 32 ? tok : 1 << 20;
        zat[n] = col * 40 + slot(tok & 31);
        qz[n] = (const T *)a.z.p + b * a.z.sb + h * a.z.sh + (t_begin + tok) * a.z.sl + col;
    }
    const int shift = a.shift, tl = lane & 31;
    const float *qg = a.g + b * a.gb + h * a.gh + (t_begin + tl - shift) * a.gl, *qm = a.masks ? a.masks + b * a.mb + (t_begin + tl - shift) * a.ml : nullptr;
    const int64_t sx = 32 * a.x.sl, sy = 32 * a.y.sl, sz = 32 * a.z.sl, sg = 32 * a.gl, sm = 32 * a.ml;
    float rg = 0.f, rm = 1.f;
    auto fetch = [&](int t0) {   // the chunk from token t0 of the segment on
        const int count = length - t0;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const int left = xtok[n] < count ? dy - ((tid + threads * n) % (8 * NK)) * 4 : 0;
            if (OUT) { rx[n] = load4<T>(qx[n], left, VEC); qx[n] += sx; }
            ry[n] = load4<T>(qy[n], left, VEC); qy[n] += sy;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            rz[n] = load4<T>(qz[n], ztok[n] < count ? dz - (zat[n] / 160) * 4 : 0, VEC);   // (zat / 40 is the column)
            qz[n] += sz;
        }
        if (wave == 0) {
            const bool in = tl < count && (!shift || t0 + tl > 0);
            rg = in ? *qg : 0.f;
            rm = in && qm ? *qm : 1.f;
            qg += sg;
            if (qm) qm += sm;
        }
    };
    // where this lane's part of out goes, of w and z (its own token's) comes from: token c of the chunk's first half
    T *qo = OUT ? (T *)a.out.p + b * a.out.sb + h * a.out.sh + (t_begin + c) * a.out.sl + zc + g4 : nullptr;
    const T *qw = DOT ? (const T *)a.w.p + b * a.w.sb + h * a.w.sh + (t_begin + c) * a.w.sl + zc + g4 : nullptr;
    const T *qv = DOT ? (const T *)a.z.p + b * a.z.sb + h * a.z.sh + (t_begin + c) * a.z.sl + zc + g4 : nullptr;
    const int64_t so = OUT ? 16 * a.out.sl : 0, sw = DOT ? 16 * a.w.sl : 0;
    const float y_scale = a.y_scale, out_scale = a.out_scale;
    const int zleft = dz - zc - g4;
    fetch(0);
    for (int n = 0; n < chunks; ++n) {
        const int flag = 1 + (n & 1), count = length - 32 * n;
        int subs = 1;
        for (int sub = 0; sub < subs; ++sub) {
            const int only = subs == 1 ? -1 : sub;   // token by token: the others are zeros
            __syncthreads();                         // the chunk before is done with the LDS
            bool bad = false;
            const V zero = {(T)0.f, (T)0.f, (T)0.f, (T)0.f};
#pragma unroll
            for (int k = 0; k < NK; ++k)
                if (xtok[k] < 32) {
                    bf16x4 cx[NP], cy[NP];
                    cut4<T, NP>(only < 0 || xtok[k] == only ? ry[k] : zero, cy);
                    bad |= not_finite(ry[k]);
                    if (OUT) {
                        cut4<T, NP>(rx[k], cx);
#pragma unroll
                        for (int i = 0; i < NP; ++i) { *(bf16x4 *)(lx + i * 32 * XS + xat[k]) = cx[i]; *(bf16x4 *)(ly + i * 32 * XS + xat[k]) = cy[i]; }
                    }
#pragma unroll
                    for (int i = 0; i < NP; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) lyt[(i * 32 * NK + r) * 40 + yat[k]] = cy[i][r];
                }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (ztok[k] < 32) {
                    bf16x4 cz[NP];
                    cut4<T, NP>(only < 0 || ztok[k] == only ? rz[k] : zero, cz);
                    bad |= not_finite(rz[k]);
#pragma unroll
                    for (int i = 0; i < NP; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) lzt[(i * 16 * nz + r) * 40 + zat[k]] = cz[i][r];
                }
            if (wave == 0) bad |= rm != 0.f && !(rg < 89.f);   // nor is a decay's factor in float32: its sums would reach the tokens behind a start
            if (subs == 1 && __ballot(bad) && lane == 0) lfr[flag] = 1;
            if (tid == 0) lfr[3 - flag] = 0;
            if (wave == 0) {
                // prefix sums of the log decays (base 2), tokens that start afresh as bits; `head`: decay from before the chunk up to and with the token, `tail`: from behind it on
                const bool live = only < 0 || tl == only;
                const bool fresh = live && forgets(rg, rm);
                const uint32_t fr = (uint32_t)__ballot(fresh);
                const double C = scan32(live && !fresh ? (double)rg * 1.4426950408889634074 : 0.0, lane);
                const uint64_t u = __builtin_bit_cast(uint64_t, C);
                const double last = __builtin_bit_cast(double, ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 31) << 32) |
                                                                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 31));
                const bool head_ok = (fr & (0xffffffffu >> (31 - tl))) == 0, tail_ok = tl == 31 || (fr >> (tl + 1)) == 0;
                if (lane < 32) {
                    lc[tl] = C;
                    lwin[tl] = head_ok ? exp2_fast((float)C) : -1.f;   // -1: nothing carried reaches the token
                    lwout[tl] = tail_ok ? exp2_fast((float)(last - C)) * y_scale : 0.f;
                }
                if (lane == 0) lfr[0] = fr;
                if (lane == 31) lall[0] = fr == 0 ? exp2_fast((float)C) : -1.f;
            }
            __syncthreads();
            if (subs == 1 && lfr[flag]) {   // a value that is not finite: again, token by token
                subs = 32;
                sub = -1;
                continue;
            }
            if (subs == 1 && n + 1 < chunks) fetch(32 * (n + 1));   // in flight while this chunk is computed
            const float all = lall[0];
            if (OUT) {
                // P^T: (s tile, t tile) = (0, 0), (1, 1), (0, 1): one wave each
                if (wave < 3) {
                    const uint32_t fr = lfr[0];
                    const int ts = wave == 1, tt = wave != 0;
                    f32x4 P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < NK; ++kk) {
                        bf16x8 fy[NP], fx[NP];
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            fy[i] = *(const bf16x8 *)(ly + (i * 32 + 16 * ts + c) * XS + 32 * kk + 8 * g);
                            fx[i] = *(const bf16x8 *)(lx + (i * 32 + 16 * tt + c) * XS + 32 * kk + 8 * g);
                        }
                        P = mma_pieces<NP, NP, Pieces<T>::in_order>(fy, fx, P);
                    }
                    const int t = 16 * tt + c;
                    const double Ct = lc[t];
                    bf16x4 cp[PP];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int s = 16 * ts + g4 + r;
                        // no token afresh in (s, t]: bits s + 1 .. t
                        const uint32_t between = (0xfffffffeu << s) & (0xffffffffu >> (31 - t));
                        const float wt = exp2_fast((float)(Ct - lc[s])) * y_scale;
                        float p = s <= t && (fr & between) == 0 ? P[r] * wt : 0.f;
                        if (DOT && s == t) { lown[t] = p; p = 0.f; }   // the token's own term: apart
#pragma unroll
                        for (int i = 0; i < PP; ++i) { cp[i][r] = (__bf16)p; p -= (float)cp[i][r]; }
                    }
#pragma unroll
                    for (int i = 0; i < PP; ++i) *(bf16x4 *)(lp + (i * 32 + t) * 40 + 8 * g + 4 * ts) = cp[i];
                }
                __syncthreads();
            }
            if (holds) {
                bf16x8 zt[NP];
#pragma unroll
                for (int i = 0; i < NP; ++i) zt[i] = *(const bf16x8 *)(lzt + (i * 16 * nz + zc + c) * 40 + 8 * g);
                if (OUT) {
                    f32x4 in[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                    for (int kk = 0; kk < NK; ++kk) {
                        bf16x8 st[PP];
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            float v = S[2 * kk + r / 4][r % 4];
#pragma unroll
                            for (int i = 0; i < PP; ++i) { st[i][r] = (__bf16)v; v -= (float)st[i][r]; }
                        }
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt) {
                            bf16x8 fx[NP];
#pragma unroll
                            for (int i = 0; i < NP; ++i) fx[i] = *(const bf16x8 *)(lx + (i * 32 + 16 * tt + c) * XS + 32 * kk + 8 * g);
                            in[tt] = mma_pieces<PP, NP, 2>(st, fx, in[tt]);
                        }
                    }
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
                        const int t = 16 * tt + c;
                        const bool store = t < count && (only < 0 || t == only);
                        V wv, zv;
                        if (DOT) {
                            wv = load4<T>(qw + tt * sw, store ? zleft : 0, VEC);
                            zv = load4<T>(qv + tt * (sz >> 1), store ? zleft : 0, VEC);
                        }
                        f32x4 o = {0.f, 0.f, 0.f, 0.f};
                        bf16x8 fp[PP];
#pragma unroll
                        for (int i = 0; i < PP; ++i) fp[i] = *(const bf16x8 *)(lp + (i * 32 + t) * 40 + 8 * g);
                        o = mma_pieces<NP, PP, 2>(zt, fp, o);
                        const float win = lwin[t];
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[r] = (win != -1.f ? o[r] + win * in[tt][r] : o[r]) * out_scale;
                        if (DOT) {
                            const f32x4 wf = widen(wv), zf = widen(zv);
                            float dot = o[0] * wf[0] + o[1] * wf[1] + o[2] * wf[2] + o[3] * wf[3];
                            dot = lanes_sum<16>(dot, 64);
                            if (g == 0) ldot[wave * 32 + t] = dot;
                            const float own = lown[t] * out_scale;
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[r] += own * zf[r];
                        }
                        if (store) store4<T>(qo + tt * so, o, zleft, VEC);
                    }
                }
                // S = all * S + y^T (u z): u z in the place of z's column, exact to float32
                bf16x8 uz[3];
                const f32x4 u0 = *(const f32x4 *)(lwout + g4), u1 = *(const f32x4 *)(lwout + 16 + g4);
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float v = (float)zt[NP - 1][r];   // (the small ones first: exact, and no infinity on the way)
#pragma unroll
                    for (int i = NP - 2; i >= 0; --i) v += (float)zt[i][r];
                    v *= r < 4 ? u0[r & 3] : u1[r & 3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) { uz[i][r] = (__bf16)v; v -= (float)uz[i][r]; }
                }
                if (all == -1.f) {
#pragma unroll
                    for (int i = 0; i < 2 * NK; ++i) S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) {
                    S[i] *= all;
                    bf16x8 yt[NP];
#pragma unroll
                    for (int k = 0; k < NP; ++k) yt[k] = *(const bf16x8 *)(lyt + (k * 32 * NK + 16 * i + c) * 40 + 8 * g);
                    S[i] = mma_pieces<NP, 3, 2>(yt, uz, S[i]);
                }
            }
            whole = all != -1.f ? whole * all : 0.f;   // (selected: a factor that is not finite ends at a start too)
            if (DOT) {
                __syncthreads();
                if (wave == 0 && lane < 32 && lane < count && (only < 0 || lane == only)) {
                    float d = 0.f;
                    for (int w = 0; w < nz; ++w) d += ldot[w * 32 + lane];
                    a.dot[(t_begin + 32 * n + lane) * a.dot_sl + bh * a.dot_sh] = d;
                }
            }
        }
        if (subs > 1 && n + 1 < chunks) fetch(32 * (n + 1));
        if (OUT) qo += 2 * so;
        if (DOT) { qw += 2 * sw; qv += sz; }
    }
    asm volatile("" : "+s"(at_args));
    const Walk &e = *(const Walk *)(WalkArg)at_args;
    float behind = 1.f;   // the last token's own decay, where it lies behind it; -1: nothing is carried on
    if (shift) {
        const int64_t t = t_begin + length - 1;
        const float gt = e.g[t * e.gl + b * e.gb + h * e.gh], mt = e.masks ? e.masks[t * e.ml + b * e.mb] : 1.f;
        behind = forgets(gt, mt) ? -1.f : exp2_fast((float)((double)gt * 1.4426950408889634074));
    }
    if (e.state_out && holds) {
        float *ps = e.state_out + seg * e.seg_state_out + bh * (int64_t)(dy * dz) + (zc + c) * e.o_z;
        const int64_t o_y = e.o_y;
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int y = 16 * i + g4 + r;
                if (y < dy && zc + c < dz) ps[y * o_y] = behind != -1.f ? S[i][r] * behind : 0.f;
            }
    }
    if (MODE == kState && e.seg_decay && tid == 0) e.seg_decay[(int64_t)seg * heads + bh] = behind != -1.f ? whole * behind : 0.f;
}

// ---- small heads ------------------------------------------------------------------------------------------------------------
// dy <= 32, or few tokens: the recurrence itself, token by token, on the vector units.  16 lanes (a DPP row) hold one head, or R rows its y in shares of 32: lane c column c of
// its slice of the state, 16 NY values of y each; y and x are broadcast from the lane that holds them by the multiply's own operand (row_newbcast), so a token costs three
// instructions per 64 state entries and no LDS.  Four neighbouring heads share a wave: 256 bytes of a token's row side by side.  Against a walk on the
// matrix units, where half of every 16-token tile is above the diagonal and chunks of ten tokens waste the rest: 239 -> 133 us for 30 720 x 4 heads of ten
// tokens (float32, 566 MB: 111 us at the copy rate of 5.1 TB/s; 118 since the sums over lanes leave the LDS pipe).  Long sequences of small heads are bound by its
// instructions: 2 000 heads of 16 x 16 and 3 193 tokens take 690 us, their bytes 330 us.
template <int M> __device__ __forceinline__ float row_lane(float v) {   // lane M of each row of 16, in every lane of the row
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + M, 0xf, 0xf, true));
}

template <int M, int N, typename F> __device__ __forceinline__ void unroll(F f) {
    if constexpr (M < N) { f(std::integral_constant<int, M>()); unroll<M + 1, N>(f); }
}

__device__ __forceinline__ float row_sum(float v) { return lanes_sum<1>(v, 16); }

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
#pragma unroll
    for (int n = 1; n < NY; ++n) o += row_dot16(x[n], S + 16 * n);
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

template <typename T, int NY, int R, bool DOT>
__global__ __launch_bounds__(256) void memory_rows_kernel(Walk a) {
    constexpr int TB = NY == 1 ? 8 : NY == 2 ? 4 : 2;   // tokens whose rows are in flight while as many are computed
    const int lane = threadIdx.x & 63, c = lane & 15;
    const int64_t heads = a.B * a.H, groups = (heads + 4 / R - 1) / (4 / R);
    const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // (the same in the wave: what follows from it is scalar)
    if (unit >= groups * a.nseg * a.slices) return;
    const int64_t mine = unit % groups * (4 / R) + (lane >> 4) / R, rest = unit / groups;
    const bool have = mine < heads;
    const int64_t bh = have ? mine : heads - 1;
    const int slice = (int)(rest % a.slices), seg = (int)(rest / a.slices);
    const int64_t b = bh / a.H;
    const int h = (int)(bh - b * a.H);
    const int part = (lane >> 4) % R, y0 = 16 * NY * part, dy = a.dy - y0;   // this row's share of y (none left: dy <= 0)
    const int z = slice * 16 + c;
    const bool zin = z < a.dz;
    const int64_t t_begin = (int64_t)seg * a.seg_len, t_end = min(a.L, t_begin + a.seg_len), count = t_end - t_begin;
    // every load is made, from a place inside the row where the lane's own lies beyond it (a conditional load would have to arrive before its value's conversion, one after
    // another), and kept as it lies until its token is computed
    const int zs = zin ? z : 0;
    const T *px = a.state_only ? nullptr : (const T *)a.x.p + b * a.x.sb + h * a.x.sh, *py = (const T *)a.y.p + b * a.y.sb + h * a.y.sh;
    const T *pz = (const T *)a.z.p + b * a.z.sb + h * a.z.sh + zs, *pw = DOT ? (const T *)a.w.p + b * a.w.sb + h * a.w.sh + zs : nullptr;
    T *po = a.state_only ? nullptr : (T *)a.out.p + b * a.out.sb + h * a.out.sh + z;
    const float *pg = a.g + b * a.gb + h * a.gh, *pm = a.masks ? a.masks + b * a.mb : nullptr;

    float S[16 * NY];
    if (a.state) {
        const float *ps = a.state + seg * a.seg_state_in + bh * (int64_t)a.dy * a.dz + (int64_t)z * a.s_z + y0 * a.s_y;
        row_state(S, ps, a.s_y, dy, zin, a.s_y == 1 && (a.dy & 3) == 0 && ((uintptr_t)a.state & 15) == 0);
    } else {
#pragma unroll
        for (int m = 0; m < 16 * NY; ++m) S[m] = 0.f;
    }
    float whole = 1.f;
    T nx[TB][NY], ny[TB][NY], nz[TB], nw[TB];
    float ng = 0.f, nm = 1.f;
    auto decayed = [&](int64_t i0) { return c < TB && i0 + c < count && (!a.shift || i0 + c > 0); };   // lane c: the decay before token i0 + c
    auto fetch = [&](int64_t i0) {
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int64_t t = t_begin + min(i0 + i, count - 1);
#pragma unroll
            for (int n = 0; n < NY; ++n) {
                const int at = min(y0 + 16 * n + c, a.dy - 1);
                if (!a.state_only) nx[i][n] = px[t * a.x.sl + at];
                ny[i][n] = py[t * a.y.sl + at];
            }
            nz[i] = pz[t * a.z.sl];
            if (DOT) nw[i] = pw[t * a.w.sl];
        }
        const int64_t t = t_begin + (decayed(i0) ? i0 + c - a.shift : 0);
        ng = pg[t * a.gl];
        if (pm) nm = pm[t * a.ml];
    };
    fetch(0);
    for (int64_t i0 = 0; i0 < count; i0 += TB) {
        float x[TB][NY], y[TB][NY], zz[TB], ww[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
#pragma unroll
            for (int n = 0; n < NY; ++n) {
                const bool yin = 16 * n + c < dy;
                x[i][n] = yin && !a.state_only ? (float)nx[i][n] : 0.f;
                y[i][n] = yin ? (float)ny[i][n] * a.y_scale : 0.f;
            }
            zz[i] = zin ? (float)nz[i] : 0.f;
            ww[i] = DOT && zin ? (float)nw[i] : 0.f;
        }
        const bool real_decay = decayed(i0);
        const float fresh_l = real_decay && forgets(ng, nm) ? 1.f : 0.f;
        const float decay_l = !real_decay ? 1.f : fresh_l != 0.f ? 0.f : exp2_fast((float)((double)ng * 1.4426950408889634074));
        if (i0 + TB < count) fetch(i0 + TB);
        unroll<0, TB>([&](auto ii) {
            constexpr int i = ii;
            if (i0 + i < count) {
                const float d = row_lane<i>(decay_l);
                const bool fresh = row_lane<i>(fresh_l) != 0.f;
                if (a.state_only) whole = fresh ? 0.f : whole * d;
                else {
                    float nd = row_dot<NY>(x[i], S);       // from the tokens before
                    nd = fresh ? 0.f : lanes_sum<16>(nd, 16 * R) * d;
                    float xy = 0.f;
#pragma unroll
                    for (int n = 0; n < NY; ++n) xy += x[i][n] * y[i][n];
                    xy = lanes_sum<1>(xy, 16 * R);
                    const int64_t t = t_begin + i0 + i;
                    if (have && zin && part == 0) po[t * a.out.sl] = (T)((nd + xy * zz[i]) * a.out_scale);
                    if (DOT) {
                        const float dot = lanes_sum<1>(zin ? nd * a.out_scale * ww[i] : 0.f, 16);
                        if (have && c == 0 && part == 0) a.dot[slice * a.dot_slice + t * a.dot_sl + bh * a.dot_sh] = dot;
                    }
                }
                row_update<NY>(S, d, fresh, y[i], zz[i]);
            }
        });
    }
    if (a.shift) {   // the last token's own decay lies behind it
        const float gt = pg[(t_end - 1) * a.gl], mt = pm ? pm[(t_end - 1) * a.ml] : 1.f;
        const bool fresh = forgets(gt, mt);
        const float d = exp2_fast((float)((double)gt * 1.4426950408889634074));
#pragma unroll
        for (int m = 0; m < 16 * NY; ++m) S[m] = fresh ? 0.f : S[m] * d;
        whole = fresh ? 0.f : whole * d;
    }
    if (a.state_out && have && zin) {
        float *ps = a.state_out + seg * a.seg_state_out + bh * (int64_t)a.dy * a.dz + (int64_t)z * a.o_z + y0 * a.o_y;
#pragma unroll
        for (int m = 0; m < 16 * NY; ++m) if (m < dy) ps[m * a.o_y] = S[m];
    }
    if (a.seg_decay && slice == 0 && part == 0 && c == 0 && have) a.seg_decay[seg * heads + bh] = whole;
}

// All gradients of up to 16 tokens of heads up to 16 x 16 in one pass (the update's chunks): q, k, v and dout stay in registers -- 16 lanes a head, as above --, the state is walked
// forwards for dq, its gradient backwards for dk (lane = row) and dv (lane = column).  dg_t = <S_L, dS_L> + sum_{i >= t} (q_i . dq_i - k_i . dk_i), each
// without the token's own term, 0 where an episode starts: its error is 2^-24 of the terms from the token to the end.  Reads and writes everything once: 928 MB for 30 720 x 4 heads of ten tokens, 182 us at the copy
// rate; it takes 229 us, three walks and the decay's kernel took 872 us.
struct ShortGrad {
    WalkRows q, k, v, o, dq, dk, dv;
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    const float *state, *d_state;
    float *d_state0, *dg;            // NULL: not wanted
    double *partial;                 // (B, H) sums of dg; NULL: dg is not wanted
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
    {
        T rq[16], rk[16], rv[16], ro[16];   // as in memory_rows_kernel: every load is made, from a token and a column that are there
        const int ck = min(c, K - 1), cv = min(c, V - 1);
        const T *pq = (const T *)a.q.p + b * a.q.sb + h * a.q.sh + ck, *pk = (const T *)a.k.p + b * a.k.sb + h * a.k.sh + ck;
        const T *pv = (const T *)a.v.p + b * a.v.sb + h * a.v.sh + cv, *po = (const T *)a.o.p + b * a.o.sb + h * a.o.sh + cv;
#pragma unroll
        for (int t = 0; t < 16; ++t)
            if (t < L) { rq[t] = pq[t * a.q.sl]; rk[t] = pk[t * a.k.sl]; rv[t] = pv[t * a.v.sl]; ro[t] = po[t * a.o.sl]; }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const bool in = t < L;
            q[t] = in && kin ? (float)rq[t] : 0.f;
            k[t] = in && kin ? (float)rk[t] : 0.f;
            v[t] = in && vin ? (float)rv[t] : 0.f;
            o[t] = in && vin ? (float)ro[t] : 0.f;
        }
    }
    const float gl = c < L ? a.g[c * a.gl + b * a.gb + h * a.gh] : 0.f, ml = c < L && a.masks ? a.masks[c * a.ml + b * a.mb] : 1.f;
    const int64_t at = bh * (int64_t)K * V;
    float S[16], G[16], C[16];        // S, G: row c of the state and of its gradient; C: column c of the gradient
    if (a.state) row_state(S, a.state + at + c * V, 1, V, kin, a.wide);
    else {
#pragma unroll
        for (int m = 0; m < 16; ++m) S[m] = 0.f;
    }
    const float fresh_l = forgets(gl, ml) ? 1.f : 0.f;
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
    double run = 0.0;   // (its terms are float32, their sum on the way may need more)
    if (a.d_state) {
        row_state(G, a.d_state + at + c * V, 1, V, kin, a.wide);
        row_state(C, a.d_state + at + c, V, K, vin, false);
        float last = 0.f;
#pragma unroll
        for (int m = 0; m < 16; ++m) last += S[m] * G[m];
        run = row_sum(last);
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
            run += (double)xs[t] - row_sum(k[t] * nk);
            const bool fresh = row_lane<t>(fresh_l) != 0.f;
            if (fresh) run = 0.0;
            const float d = row_lane<t>(decay_l);
            sum += run;
            if (a.dg && have && c == 0) a.dg[t * heads + bh] = (float)run;
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

// The states at the segments' starts from what each segment adds to an empty state: in place, one thread per element.
__global__ __launch_bounds__(256) void memory_join_kernel(float *seg_states, const float *seg_decay, const float *init, float *last,
                                                          int64_t heads, int elems, int nseg) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = heads * elems;
    if (i >= total) return;
    const int64_t bh = i / elems;
    float S = init ? init[i] : 0.f;
    for (int seg0 = 0; seg0 < nseg; seg0 += 8) {   // eight loads in flight
        float d[8], u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int seg = min(seg0 + k, nseg - 1);
            d[k] = seg_decay[seg * heads + bh];
            u[k] = seg_states[seg * total + i];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (seg0 + k < nseg) {
                seg_states[(seg0 + k) * total + i] = S;
                S = (d[k] == 0.f ? 0.f : d[k] * S) + u[k];
            }
    }
    if (last) last[i] = S;
}

// dg_1 = <S_0, dS_0>, dg_{t+1} = dg_t - (q_t . dq_t - k_t . dk_t), 0 where an episode starts: the gradient of the log decays from the sums that the dq and
// dk walks left, each without the token's own term (which is in both and cancels).  float64: the running difference outlives many tokens.
// One workgroup per (batch, head); every thread takes four tokens at a time, what they add is joined by a scan (64 heads of 4 096 tokens: 19 us).
// Up to 64 tokens (decay_grad_short_kernel): `team` lanes per pair share its <S_0, dS_0>, one of them walks the tokens, eight of them loaded at a time.  (A
// wave of 64 pairs after another: 1 650 us for 192 heads of 91 x 82.)
struct DecayGrad {
    const float *dot_q, *dot_k;      // (slices), L and (B, H) by these strides
    int64_t dot_sl, dot_sh;
    const float *state, *d_state;    // (B, H, elems); state may be NULL
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    float *dg;                       // (L, B, H) or NULL
    double *partial;                 // (B, H): sums over the tokens
    int64_t L, B;
    int H, elems, slices, team, vec;   // vec: both states on 16 bytes, elems a multiple of four
};

__device__ __forceinline__ bool decay_fresh(const DecayGrad &a, int64_t t, int64_t b, int h) {
    return forgets(a.g[t * a.gl + b * a.gb + h * a.gh], a.masks ? a.masks[t * a.ml + b * a.mb] : 1.f);
}

__global__ __launch_bounds__(256) void decay_grad_short_kernel(DecayGrad a) {
    const int64_t bh = ((int64_t)blockIdx.x * 256 + threadIdx.x) / a.team, heads = a.B * a.H;
    const int j = threadIdx.x & (a.team - 1);
    double run = 0.0;
    if (a.state && bh < heads) {
        const float *p = a.state + bh * a.elems, *q = a.d_state + bh * a.elems;
        if (a.vec)
            for (int e = 4 * j; e < a.elems; e += 4 * a.team) {
                const f32x4 u = *(const f32x4 *)(p + e), v = *(const f32x4 *)(q + e);
                run += ((double)u[0] * v[0] + (double)u[1] * v[1]) + ((double)u[2] * v[2] + (double)u[3] * v[3]);
            }
        else
#pragma unroll 4
            for (int e = j; e < a.elems; e += a.team) run += (double)p[e] * (double)q[e];
    }
    for (int off = a.team >> 1; off; off >>= 1) run += __shfl_xor(run, off);
    if (bh >= heads || j) return;
    const int64_t b = bh / a.H, n = a.L * heads;
    const int h = (int)(bh - b * a.H);
    const float *pq = a.dot_q + bh * a.dot_sh, *pk = a.dot_k + bh * a.dot_sh;
    double sum = 0.0;
    for (int64_t t0 = 0; t0 < a.L; t0 += 8) {
        double step[8];
        bool fresh[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t t = min(t0 + i, a.L - 1);
            fresh[i] = decay_fresh(a, t, b, h);
            step[i] = 0.0;
        }
        for (int s = 0; s < a.slices; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) step[i] += (double)pq[s * n + min(t0 + i, a.L - 1) * a.dot_sl] - (double)pk[s * n + min(t0 + i, a.L - 1) * a.dot_sl];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (t0 + i < a.L) {
                if (fresh[i]) run = 0.0;
                if (a.dg) a.dg[(t0 + i) * heads + bh] = (float)run;
                sum += run;
                run -= step[i];
            }
    }
    a.partial[bh] = sum;
}

__global__ __launch_bounds__(1024) void decay_grad_long_kernel(DecayGrad a) {
    __shared__ double sums[16];
    __shared__ int cuts[16];
    const int64_t bh = blockIdx.x, heads = a.B * a.H, b = bh / a.H, n = a.L * heads;
    const int h = (int)(bh - b * a.H), tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
    double first = 0.0;
    if (a.state)
#pragma unroll 4
        for (int e = tid; e < a.elems; e += threads) first += (double)a.state[bh * a.elems + e] * (double)a.d_state[bh * a.elems + e];
    for (int off = 32; off; off >>= 1) first += __shfl_down(first, off);
    if (lane == 0) sums[wave] = first;
    __syncthreads();
    double carry = 0.0, sum = 0.0;   // carry: the gradient at the tokens' start
    for (int w = 0; w < waves; ++w) carry += sums[w];
    const float *pq = a.dot_q + bh * a.dot_sh, *pk = a.dot_k + bh * a.dot_sh;
    for (int64_t tile = 0; tile < a.L; tile += 4 * threads) {
        const int64_t t0 = tile + 4 * tid;
        double step[4] = {0.0, 0.0, 0.0, 0.0};
        bool fresh[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fresh[i] = decay_fresh(a, min(t0 + i, a.L - 1), b, h) && t0 + i < a.L;
        for (int s = 0; s < a.slices; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = s * n + min(t0 + i, a.L - 1) * a.dot_sl;
                step[i] += (double)pq[at] - (double)pk[at];
            }
        // what this thread's tokens add behind their last start of an episode, and whether they hold one; both scanned over the workgroup: the later one wins where
        // it holds a start
        double add = 0.0;
        int cut = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (fresh[i]) { add = 0.0; cut = 1; }
            add -= t0 + i < a.L ? step[i] : 0.0;
        }
        for (int off = 1; off < 64; off <<= 1) {
            const double p = __shfl_up(add, off);
            const int q = __shfl_up(cut, off);
            if (lane >= off && !cut) { add += p; cut = q; }
        }
        __syncthreads();   // the sums before are read
        if (lane == 63) { sums[wave] = add; cuts[wave] = cut; }
        __syncthreads();
        double run = carry;
        for (int w = 0; w < waves; ++w) {
            if (w == wave) run = carry;
            carry = cuts[w] ? sums[w] : carry + sums[w];
        }
        const double p = __shfl_up(add, 1);
        const int q = __shfl_up(cut, 1);
        if (lane > 0) run = q ? p : run + p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (t0 + i < a.L) {
                if (fresh[i]) run = 0.0;
                if (a.dg) a.dg[(t0 + i) * heads + bh] = (float)run;
                sum += run;
                run -= step[i];
            }
    }
    __syncthreads();
    for (int off = 32; off; off >>= 1) sum += __shfl_down(sum, off);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        double s = 0.0;
        for (int w = 0; w < waves; ++w) s += sums[w];
        a.partial[bh] = s;
    }
}

// The running difference does not come back from an infinity or a NaN: one in q or d_out reaches the gradients behind it, one in k or v (in the short kernel, which runs backwards)
// those before it, where the definition has numbers.  A head whose sum is not finite is formed again from the definition, an episode at a time: backwards the gradient of the
// state, G, down to the token whose G_t is not finite (all before it are not either); at the token behind that one -- or at the episode's start --
// dg_t = r_t e^{g_t} <S_{t-1}, G_t> itself, with the state walked there forwards, and the running difference on from it up to the first S_t that is not finite.  The tokens outside have
// no finite gradient.  A workgroup takes its share of the heads and passes over those with finite sums: 5 us of a backward pass where all are (chunks of ten tokens 320 -> 326 us, 4 096
// tokens 332 -> 337).  States in LDS: in registers they spilled, and the launch alone cost 17 to 36 us.
struct DecayAgain {
    WalkRows q, k, v, o;
    const float *g; int64_t gl, gb, gh;
    const float *masks; int64_t ml, mb;
    const float *state, *d_state;           // NULL: zeros
    float *dg;                              // (L, B, H) or NULL
    double *partial;                        // (B, H)
    float *behind; int64_t b_sl, b_sh;      // room for L floats of each (b, h); NULL: up to 16 tokens
    int64_t L, B;
    int H, dk, dv;
    float scale;
};

__device__ __forceinline__ bool not_finite(float v) { return !(v - v == 0.f); }

template <typename T>
__global__ __launch_bounds__(1024) void decay_again_kernel(DecayAgain a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ double sums[2][16];
    __shared__ float few[16];
    __shared__ int flags[1024], start;
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, elems = a.dk * a.dv;
    float *G = (float *)smem, *S = G + elems;   // (a thread reads and writes its own entries only)
    const int64_t heads = a.B * a.H, first = heads * blockIdx.x / gridDim.x, end = heads * (blockIdx.x + 1) / gridDim.x;
    int flip = 0;
    auto total = [&](double v) {                // over the workgroup; two places in turn: one barrier
        for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
        flip ^= 1;
        if (lane == 0) sums[flip][wave] = v;
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < threads >> 6; ++w) v += sums[flip][w];
        return v;
    };
    for (int64_t base = first; base < end; base += threads) {
        const int count = (int)min((int64_t)threads, end - base);
        const double s = tid < count ? a.partial[base + tid] : 0.0;
        flags[tid] = !(s - s == 0.0);
        if (!__syncthreads_or(flags[tid])) continue;
        for (int j = 0; j < count; ++j) {
            if (!flags[j]) continue;
            const int64_t bh = base + j, b = bh / a.H;
            const int h = (int)(bh - b * a.H);
            const float *pg = a.g + b * a.gb + h * a.gh, *pm = a.masks ? a.masks + b * a.mb : nullptr;
            const T *pq = (const T *)a.q.p + b * a.q.sb + h * a.q.sh, *pk = (const T *)a.k.p + b * a.k.sb + h * a.k.sh;
            const T *pv = (const T *)a.v.p + b * a.v.sb + h * a.v.sh, *po = (const T *)a.o.p + b * a.o.sb + h * a.o.sh;
            float *behind = a.behind ? a.behind + bh * a.b_sh : few;
            const int64_t b_sl = a.behind ? a.b_sl : 1;
            auto fresh = [&](int64_t t) { return forgets(pg[t * a.gl], pm ? pm[t * a.ml] : 1.f); };
            auto decay = [&](int64_t t) { return exp2_fast((float)((double)pg[t * a.gl] * 1.4426950408889634074)); };
            double sum = 0.0;                   // (thread 0)
            for (int64_t e1 = a.L, e0; e1 > 0; e1 = e0) {
                int bad = 0;
                for (int e = tid; e < elems; e += threads) {
                    G[e] = e1 == a.L && a.d_state ? a.d_state[bh * elems + e] : 0.f;
                    bad |= not_finite(G[e]);
                }
                int64_t from = e1;              // the first token whose G_t is finite, as far as they are walked
                e0 = e1 - 1;
                bool dead = __syncthreads_or(bad);
                for (; !dead; --e0) {
                    const T *q = pq + e0 * a.q.sl, *k = pk + e0 * a.k.sl, *v = pv + e0 * a.v.sl, *o = po + e0 * a.o.sl;
                    double x = 0.0;
                    bad = 0;
                    for (int e = tid; e < elems; e += threads) {
                        const int y = e / a.dv, z = e - y * a.dv;
                        x += (double)((float)k[y] * (float)v[z]) * G[e];
                        bad |= not_finite(G[e] + a.scale * (float)q[y] * (float)o[z]);
                    }
                    x = total(x);
                    if (tid == 0) behind[e0 * b_sl] = (float)x;
                    dead = __syncthreads_or(bad);
                    if (dead) break;            // G: what the token behind passes on
                    from = e0;
                    const bool starts = fresh(e0);
                    const float d = starts ? 0.f : decay(e0);
                    for (int e = tid; e < elems; e += threads) {
                        const int y = e / a.dv, z = e - y * a.dv;
                        G[e] = starts ? 0.f : (G[e] + a.scale * (float)q[y] * (float)o[z]) * d;
                    }
                    if (starts || e0 == 0) break;
                }
                if (dead) {                     // the episode's start, as many tokens at a time as there are threads
                    for (;; e0 -= threads) {
                        if (tid == 0) start = -1;
                        __syncthreads();
                        const int64_t t = e0 - tid;
                        if (t >= 0 && (t == 0 || fresh(t))) atomicMax(&start, threads - 1 - tid);
                        __syncthreads();
                        const int found = start;
                        __syncthreads();
                        if (found >= 0) { e0 -= threads - 1 - found; break; }
                    }
                }
                const bool starts = fresh(e0);
                if (from == e1) {               // no finite gradient in it but a start's
                    const float nan = __builtin_nanf("");
                    if (a.dg) for (int64_t t = e0 + tid; t < e1; t += threads) a.dg[t * heads + bh] = t == e0 && starts ? 0.f : nan;
                    if (!starts || e1 - e0 > 1) sum += nan;
                    continue;
                }
                bad = 0;
                for (int e = tid; e < elems; e += threads) {
                    S[e] = !starts && a.state ? a.state[bh * elems + e] : 0.f;
                    bad |= not_finite(S[e]);
                }
                bool lost = __syncthreads_or(bad);
                double run = 0.0;
                for (int64_t t = e0; t < e1; ++t) {
                    const bool afresh = starts && t == e0, there = t >= from && !lost;
                    if (there && t == from && !afresh) {
                        double x = 0.0;
                        for (int e = tid; e < elems; e += threads) x += (double)S[e] * G[e];
                        run = total(x);
                    }
                    const double dg = afresh ? 0.0 : there ? run : (double)__builtin_nanf("");
                    if (tid == 0) {
                        if (a.dg) a.dg[t * heads + bh] = (float)dg;
                        sum += dg;
                    }
                    if (lost) continue;
                    const T *q = pq + t * a.q.sl, *k = pk + t * a.k.sl, *v = pv + t * a.v.sl, *o = po + t * a.o.sl;
                    const float d = afresh ? 0.f : decay(t);
                    double x = 0.0;
                    bad = 0;
                    for (int e = tid; e < elems; e += threads) {
                        const int y = e / a.dv, z = e - y * a.dv;
                        const float c = S[e] * d;
                        if (there && !afresh) x += (double)(a.scale * (float)q[y] * (float)o[z]) * c;
                        S[e] = c + (float)k[y] * (float)v[z];
                        bad |= not_finite(S[e]);
                    }
                    if (there) {
                        x = total(x);
                        if (tid == 0) run -= x - (double)behind[t * b_sl];
                    }
                    lost = __syncthreads_or(bad);
                }
            }
            if (tid == 0) a.partial[bh] = sum;
        }
        __syncthreads();
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
// nothing else weighs: HBM.  A head has a team of lanes that covers its state in float4s, up to a wave, lane = (row group, four columns); o is summed over the row groups.  Float4s
// go past the caches, which no byte of them finds again.  16 x 16 float32, 2 621 440 heads (6.0 GB): 1 286 us, 4.7 TB/s; 64 x 64, 160 000 heads: 930 us, 5.8 TB/s; 4 x 4, 4 million heads: 130 us
// (a wave each 1 480 us).  A loop over the heads in as many workgroups as are resident is slower (1 377 us at best): too few loads are in flight.
struct Step {
    WalkRows q, k, v, out;
    const float *g; int64_t gb, gh;
    const float *masks; int64_t mb;
    const float *state; float *state_out;
    int64_t B; int H, dk, dv;
    int lz, team;                // lanes along a row of the state, lanes of a head: powers of two
    float scale;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void memory_step_kernel(Step a) {
    constexpr int W = VEC ? 4 : 1;
    const int lz = 1 << a.lz, team = 1 << a.team, rows = team >> a.lz, j = threadIdx.x & (team - 1), row = j >> a.lz, cl = j & (lz - 1);
    const uint32_t bh = (blockIdx.x * 256 + threadIdx.x) >> a.team;   // (fewer than 2^32 threads)
    if (bh >= a.B * a.H) return;
    const uint32_t b = bh / (uint32_t)a.H, h = bh - b * (uint32_t)a.H;
    const T *q = (const T *)a.q.p + b * a.q.sb + h * a.q.sh, *k = (const T *)a.k.p + b * a.k.sb + h * a.k.sh, *v = (const T *)a.v.p + b * a.v.sb + h * a.v.sh;
    T *out = (T *)a.out.p + b * a.out.sb + h * a.out.sh;
    const float *S = a.state ? a.state + bh * (int64_t)(a.dk * a.dv) : nullptr;
    float *So = a.state_out + bh * (int64_t)(a.dk * a.dv);
    const float g = a.g[b * a.gb + h * a.gh], mask = a.masks ? a.masks[b * a.mb] : 1.f;
    const bool carry = S && !forgets(g, mask);
    const float decay = carry ? exp2_fast((float)((double)g * 1.4426950408889634074)) : 0.f;
    for (int z0 = 0; z0 < a.dv; z0 += lz * W) {
        const int z = z0 + cl * W, zs = min(z, a.dv - W);
        T vr[W];   // kept as it lies until the state has arrived: a conversion here would be one more wait before it
        float o[W];
#pragma unroll
        for (int r = 0; r < W; ++r) { vr[r] = v[zs + r]; o[r] = 0.f; }
        for (int y = row; y < a.dk; y += rows) {
            const T kr = k[y], qr = q[y];
            if (z < a.dv) {
                const int at = y * a.dv + z;
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
                if (carry) {
                    if (VEC) s = __builtin_nontemporal_load((const f32x4 *)(S + at)) * decay;
                    else s[0] = S[at] * decay;
                }
#pragma unroll
                for (int r = 0; r < W; ++r) { s[r] += (float)kr * (float)vr[r]; o[r] += (float)qr * s[r]; }
                if (VEC) __builtin_nontemporal_store(s, (f32x4 *)(So + at));
                else So[at] = s[0];
            }
        }
        for (int off = lz; off < team; off <<= 1)
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
    if (m->B >= (1ll << 26) / m->H || m->L > (1ll << 30)) return policy_fail(FMARL_EINVAL, "%s: too many sequences (B H must stay below 2^26) or tokens (2^30)", who);
    if (m->L > 0 && m->B > 0 && (!m->q.data || !m->k.data || !m->v.data || !m->log_decay)) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    return FMARL_OK;
}

// The recurrence on the vector units for y up to 32 wide and for few tokens, the matrix units beyond.  At 16 x 16 the former takes two thirds of the latter's time.  Wider,
// its three instructions per 64 state entries and token cost more than a chunk of 32 tokens on the matrix units from about ten tokens on, or 32 where z has one
// tile only (4 096 heads forwards, us, vector | matrix units: 64 x 64 bfloat16 1 token 37 | 53, 10 tokens 54 | 51, 16 tokens 64 | 51; 128 x 128 float32 1 token 160 | 265, 10
// tokens 217 | 262, 32 tokens 440 | 286; 128 x 16 bfloat16 16 tokens 38 | 88, 32 tokens 62 | 89, 64 tokens 112 | 120).  Beyond 64 with one tile of z a workgroup on the matrix
// units has one wave that holds a state and three that only load, so many tokens are faster on the vector units too (106 x 7, 266 heads of 1 500 tokens: bfloat16 280 | 448, float32
// 279 | 800; 72 heads of 412 tokens 81 | 57, 79 | 81).
bool small_heads(int dy, int dz, int64_t L, int64_t heads) {
    return dy <= 32 || L <= (dz <= 16 ? 32 : 10) || (dy > 64 && dz <= 16 && heads * L >= 65536);
}
bool small_heads(const FmarlMemory *m, int dy, int dz) { return small_heads(dy, dz, m->L, m->B * m->H); }

// heads that share a wave of memory_rows_kernel
int heads_of_wave(int dy) { return dy <= 32 ? 4 : dy <= 64 ? 2 : 1; }

// workgroups of memory_tiles_kernel that a CU holds at a time: by registers (launch bounds) and LDS
int tiles_resident(const FmarlMemory *m) {
    const int nk = m->dk <= 64 ? 2 : 4, nz = (m->dv + 15) / 16, waves = nz < 4 ? 4 : nz;
    const int regs = (nk == 4 ? 2 : m->dtype == FMARL_T_F32 ? 3 : 4) * 4 / waves;
    const int lds = m->dtype == FMARL_T_F32 ? tiles_lds<float>(nk, nz) : m->dtype == FMARL_T_BF16 ? tiles_lds<__bf16>(nk, nz) : tiles_lds<_Float16>(nk, nz);
    const int n = 160 * 1024 / lds < regs ? 160 * 1024 / lds : regs;
    return n < 1 ? 1 : n;
}

// A batch with few heads has its tokens cut into segments that are walked side by side, at the price of a walk that leaves their states (a second read of k and v) and a
// join, if that makes the walk shorter.  Small heads: with n waves on a SIMD, four at most, a token takes about 25 + 11 n units of time; segments of 32 tokens at least (24 heads of
// 16 x 16 and 500 tokens: 71 us with 64, 50 with 32; 1 000 heads of 8 x 100 and 64 tokens: 67 us in two segments, 38 in one).  Large heads: with n workgroups on its CU a chunk
// takes about 3 + 2 n units (64 x 64 bfloat16, 64 heads of 4 096 tokens, training: n = 2 420 us, n = 3 372 us, n = 4 336 us; 40 x 72 float16, 72 heads of 1 023 tokens: n = 2
// 60 us, n = 3 70 us, whose segments are of 96 tokens and end unevenly); more segments where the gradient's walks are those of small heads and would
// leave most of the chip idle (48 x 16 bfloat16, 266 heads of 412 tokens, backwards: 445 us in one segment, 167 in six).
struct Segments { int nseg, len; };
Segments memory_segments(const FmarlMemory *m) {
    const int64_t heads = m->B * m->H;
    Segments best = {1, (int)(m->L > 0x40000000 ? 0x40000000 : m->L)};
    auto cut = [&](int64_t n, int least) {   // into n segments of `least` tokens at least
        if (n > m->L / least) n = m->L / least;
        if (n < 2) return Segments{1, best.len};
        const int64_t len = ((m->L + n - 1) / n + 31) / 32 * 32;
        return Segments{(int)((m->L + len - 1) / len), (int)len};
    };
    const auto waves = [&](int dy, int dz) { return (heads + heads_of_wave(dy) - 1) / heads_of_wave(dy) * ((dz + 15) / 16); };   // of an uncut walk of small heads
    if (small_heads(m, m->dk, m->dv)) {
        const int64_t uncut = waves(m->dk, m->dv);
        const auto cost = [&](const Segments &s) {
            const int64_t on_simd = (uncut * s.nseg + 1023) / 1024, rounds = (on_simd + 3) / 4;
            return (s.nseg > 1 ? 16 : 10) * (int64_t)s.len * rounds * (25 + 11 * (on_simd < 4 ? on_simd : 4));
        };
        for (int k = 1; k <= 4; ++k) {
            const Segments s = cut(1024 * k / uncut, 32);
            if (cost(s) < cost(best)) best = s;
        }
        return best;
    }
    const int resident = tiles_resident(m);
    const auto cost = [&](const Segments &s) {
        const int64_t blocks = heads * s.nseg, on_cu = (blocks + 255) / 256, rounds = (on_cu + resident - 1) / resident;
        return (s.nseg > 1 ? 17 : 10) * ((s.len + 31ll) / 32) * rounds * (3 + 2 * (on_cu < resident ? on_cu : resident));
    };
    for (int k = 1; k <= resident; ++k) {
        const Segments s = cut(256 * k / heads, 64);
        if (cost(s) < cost(best)) best = s;
    }
    if (small_heads(m, m->dv, m->dk) && waves(m->dv, m->dk) < 512) {   // the gradient's walks of dq and dk would leave most of the chip idle
        const Segments s = cut(2048 / waves(m->dv, m->dk), 64);
        if (s.nseg > best.nseg) best = s;
    }
    return best;
}

template <typename T>
int launch_again(const DecayAgain &a, hipStream_t st) {
    const int64_t heads = a.B * a.H;
    const int elems = a.dk * a.dv, threads = elems > 960 ? 1024 : (elems + 63) / 64 * 64, lds = 8 * elems;   // a state entry a thread, up to 1 024
    if (lds > 48 * 1024) HIP_OK(hipFuncSetAttribute((const void *)decay_again_kernel<T>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL(decay_again_kernel<T>, dim3((unsigned)(heads < 512 ? heads : 512)), dim3(threads), lds, st, a);
    return FMARL_OK;
}

// the decay's gradient again for heads that hold what is not finite, and its sums over the batch
int finish_decay(const FmarlMemory *m, const FmarlRows &d_out, const float *d_state, float *d_log_decay, double *partial, float *behind, int64_t b_sl, int64_t b_sh, hipStream_t st) {
    DecayAgain a = {};
    const int dt = m->dtype;
    a.q = walk_rows(m->q, m->dk, dt); a.k = walk_rows(m->k, m->dk, dt); a.v = walk_rows(m->v, m->dv, dt); a.o = walk_rows(d_out, m->dv, dt);
    a.g = m->log_decay; a.gl = m->decay_stride_l; a.gb = m->decay_stride_b; a.gh = m->decay_stride_h; a.masks = m->masks; a.ml = m->mask_stride_l; a.mb = m->mask_stride_b;
    a.state = m->state; a.d_state = d_state; a.dg = m->shared_decay ? nullptr : d_log_decay; a.partial = partial; a.behind = behind; a.b_sl = b_sl; a.b_sh = b_sh;
    a.L = m->L; a.B = m->B; a.H = m->H; a.dk = m->dk; a.dv = m->dv; a.scale = m->scale;
    const int rc = dt == FMARL_T_F32 ? launch_again<float>(a, st) : dt == FMARL_T_BF16 ? launch_again<__bf16>(a, st) : launch_again<_Float16>(a, st);
    if (rc) return rc;
    if (m->shared_decay) hipLaunchKernelGGL(decay_sum_kernel, dim3((unsigned)m->H), dim3(256), 0, st, (const double *)partial, d_log_decay, m->B, m->H);
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

// columns of z that a wave of the small heads' kernel takes: 16; the large heads' workgroup takes them all
int slices_of(const FmarlMemory *m, int dy, int dz) { return small_heads(m, dy, dz) ? (dz + 15) / 16 : 1; }

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
        w.dot_q = take(4 * (size_t)slices_of(m, m->dv, m->dk) * m->L * heads);
        w.dot_k = take(4 * (size_t)slices_of(m, m->dv, m->dk) * m->L * heads);
        w.partial = take(8 * heads);
        w.d_state = take(4 * heads * elems);
    }
    w.total = off;
    return w;
}

template <typename T, int NK, int MODE, bool VEC>
int launch_tiles(const Walk &w, int64_t blocks, hipStream_t st) {
    const int nz = (w.dz + 15) / 16, lds = tiles_lds<T>(NK, nz);
    if (lds > 64 * 1024) HIP_OK(hipFuncSetAttribute((const void *)memory_tiles_kernel<T, NK, MODE, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL((memory_tiles_kernel<T, NK, MODE, VEC>), dim3((unsigned)blocks), dim3(64 * (nz < 4 ? 4 : nz)), lds, st, w);
    return FMARL_OK;
}

template <typename T, int NK>
int launch_tiles_as(const Walk &w, int64_t blocks, hipStream_t st) {
    const bool vec = (w.state_only || (w.x.vec && w.out.vec)) && w.y.vec && w.z.vec && (!w.w.p || w.w.vec);
    if (w.state_only) return vec ? launch_tiles<T, NK, kState, true>(w, blocks, st) : launch_tiles<T, NK, kState, false>(w, blocks, st);
    if (w.w.p) return vec ? launch_tiles<T, NK, kOutDot, true>(w, blocks, st) : launch_tiles<T, NK, kOutDot, false>(w, blocks, st);
    return vec ? launch_tiles<T, NK, kOut, true>(w, blocks, st) : launch_tiles<T, NK, kOut, false>(w, blocks, st);
}

template <typename T>
int launch_walk_t(const Walk &w, hipStream_t st) {
    const int64_t heads = w.B * w.H;
    if (small_heads(w.dy, w.dz, w.L, heads)) {
        const int per = heads_of_wave(w.dy);
        const int64_t blocks = ((heads + per - 1) / per * w.nseg * w.slices + 3) / 4;
        if (blocks > 0xffffff) return policy_fail(FMARL_EINVAL, "memory: too many sequences");
        const dim3 grid((unsigned)blocks);
#define FMARL_ROWS(NY, R) do { if (w.w.p) hipLaunchKernelGGL((memory_rows_kernel<T, NY, R, true>), grid, dim3(256), 0, st, w); \
                               else hipLaunchKernelGGL((memory_rows_kernel<T, NY, R, false>), grid, dim3(256), 0, st, w); } while (0)
        if (w.dy <= 16) FMARL_ROWS(1, 1);
        else if (w.dy <= 32) FMARL_ROWS(2, 1);
        else if (w.dy <= 64) FMARL_ROWS(2, 2);
        else FMARL_ROWS(2, 4);
#undef FMARL_ROWS
        return FMARL_OK;
    }
    const int64_t blocks = heads * w.nseg;
    if (blocks > 0x7fffff) return policy_fail(FMARL_EINVAL, "memory: too many sequences for heads of this size");
    return w.dy <= 64 ? launch_tiles_as<T, 2>(w, blocks, st) : launch_tiles_as<T, 4>(w, blocks, st);
}

int launch_walk(Walk w, int dtype, hipStream_t st) {
    w.slices = small_heads(w.dy, w.dz, w.L, w.B * w.H) ? (w.dz + 15) / 16 : 1;
    const int rc = dtype == FMARL_T_F32 ? launch_walk_t<float>(w, st) : dtype == FMARL_T_BF16 ? launch_walk_t<__bf16>(w, st) : launch_walk_t<_Float16>(w, st);
    if (rc) return rc;
    HIP_OK(hipGetLastError());
    return FMARL_OK;
}

// the decay's gradient by a thread per (batch, head) while its tokens are few; otherwise by a workgroup per (batch, head), whose threads share the tokens
bool few_tokens(int64_t L) { return L <= 64; }

Walk walk_base(const FmarlMemory *m) {
    Walk w = {};
    const Segments s = memory_segments(m);
    w.g = m->log_decay; w.gl = m->decay_stride_l; w.gb = m->decay_stride_b; w.gh = m->decay_stride_h;
    w.masks = m->masks; w.ml = m->mask_stride_l; w.mb = m->mask_stride_b;
    w.L = m->L; w.B = m->B; w.H = m->H; w.nseg = s.nseg; w.seg_len = s.len;
    w.y_scale = w.out_scale = 1.f;
    // as the decay's kernel reads them: a thread per head (heads side by side), or a workgroup per head (tokens side by side)
    const bool few = few_tokens(m->L);
    w.dot_sl = few ? m->B * m->H : 1; w.dot_sh = few ? 1 : m->L; w.dot_slice = m->L * m->B * m->H;
    return w;
}

void turn(WalkRows &r, int64_t L, int dtype) {   // the last token first
    if (!r.p) return;
    r.p += (L - 1) * r.sl * elem_bytes(dtype);
    r.sl = -r.sl;
}

// a backwards walk: every array the last token first, decays behind their tokens
void turn_round(Walk &w, int dtype) {
    turn(w.x, w.L, dtype); turn(w.y, w.L, dtype); turn(w.z, w.L, dtype); turn(w.w, w.L, dtype); turn(w.out, w.L, dtype);
    w.g += (w.L - 1) * w.gl; w.gl = -w.gl;
    if (w.masks) { w.masks += (w.L - 1) * w.ml; w.ml = -w.ml; }
    if (w.dot) { w.dot += (w.L - 1) * w.dot_sl; w.dot_sl = -w.dot_sl; }
    w.shift = 1;
}

// the states at the segments' starts (of the backwards walk: the gradients of the states behind the tokens) into seg_states; the walk's last one into `last`
int segment_states(const FmarlMemory *m, const FmarlRows &y, const FmarlRows &z, bool reverse, const float *init, float *last, float *seg_states,
                   float *seg_decay, hipStream_t st) {
    Walk w = walk_base(m);
    const int64_t heads = m->B * m->H, elems = (int64_t)m->dk * m->dv;
    w.y = walk_rows(y, m->dk, m->dtype); w.z = walk_rows(z, m->dv, m->dtype);
    w.dy = m->dk; w.dz = m->dv; w.state_only = 1;
    if (reverse) { w.y_scale = m->scale; turn_round(w, m->dtype); }
    w.state_out = seg_states; w.o_y = m->dv; w.o_z = 1; w.seg_state_out = heads * elems; w.seg_decay = seg_decay;
    if (int rc = launch_walk(w, m->dtype, st)) return rc;
    const int64_t blocks = (heads * elems + 255) / 256;
    hipLaunchKernelGGL(memory_join_kernel, dim3((unsigned)blocks), dim3(256), 0, st, seg_states, (const float *)seg_decay, init, last, heads, (int)elems, w.nseg);
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
    // lanes along a row: the smallest power of two that covers it, so that few lanes idle; a head has a team of lanes that covers its rows too, up to a wave
    while (s.lz < 6 && (vec ? 4 : 1) << s.lz < m->dv) ++s.lz;
    for (s.team = s.lz; s.team < 6 && 1 << s.team < m->dk << s.lz;) ++s.team;
    const int64_t blocks = ((m->B * m->H << s.team) + 255) / 256;
    if (blocks > 0xffffff) return policy_fail(FMARL_EINVAL, "fmarl_memory_step: too many sequences for heads of this size (a launch holds fewer than 2^32 threads)");
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
                                const FmarlRows *d_v, float *d_log_decay, float *d_state0, const void *forward_workspace, void *workspace,
                                void *stream) {
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
        g.partial = d_log_decay ? (double *)(base + ws.partial) : nullptr;
        g.B = m->B; g.L = (int)m->L; g.H = m->H; g.dk_dim = m->dk; g.dv_dim = m->dv; g.scale = m->scale;
        g.wide = (m->dv & 3) == 0 && (((uintptr_t)m->state | (uintptr_t)d_state | (uintptr_t)d_state0) & 15) == 0;
        const dim3 grid((unsigned)((heads + 15) / 16));
        if (dt == FMARL_T_F32) hipLaunchKernelGGL(memory_short_backward_kernel<float>, grid, dim3(256), 0, st, g);
        else if (dt == FMARL_T_BF16) hipLaunchKernelGGL(memory_short_backward_kernel<__bf16>, grid, dim3(256), 0, st, g);
        else hipLaunchKernelGGL(memory_short_backward_kernel<_Float16>, grid, dim3(256), 0, st, g);
        HIP_OK(hipGetLastError());
        return d_log_decay ? finish_decay(m, *d_out, d_state, d_log_decay, g.partial, nullptr, 0, 0, st) : FMARL_OK;
    }
    const int elems = m->dk * m->dv;
    float *seg_s = (float *)(base + ws.seg_s), *seg_g = (float *)(base + ws.seg_g), *decay = (float *)(base + ws.decay);
    float *ds0 = d_state0 ? d_state0 : (float *)(base + ws.d_state);
    if (w0.nseg > 1) {
        if (forward_workspace) seg_s = (float *)((char *)forward_workspace + memory_layout(m, 0).seg_s);   // (only read)
        else if (int rc = segment_states(m, m->k, m->v, false, m->state, nullptr, seg_s, decay, st)) return rc;
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
    w.dy = m->dv; w.dz = m->dk; w.y_scale = m->scale; w.s_y = 1; w.s_z = m->dv;
    turn_round(w, dt);
    w.state = w0.nseg > 1 ? seg_g : d_state; w.seg_state_in = seg_elems;
    if (int rc = launch_walk(w, dt, st)) return rc;
    w = w0;        // dv, and the gradient of the initial state
    w.x = k; w.y = q; w.z = o; w.out = walk_rows(*d_v, m->dv, dt);
    w.dy = m->dk; w.dz = m->dv; w.y_scale = m->scale; w.s_y = w.o_y = m->dv; w.s_z = w.o_z = 1;
    turn_round(w, dt);
    w.state = w0.nseg > 1 ? seg_g : d_state; w.seg_state_in = seg_elems;
    if (w0.nseg == 1) w.state_out = ds0;
    if (int rc = launch_walk(w, dt, st)) return rc;
    if (d_log_decay) {
        DecayGrad g = {};
        g.dot_q = (const float *)(base + ws.dot_q); g.dot_k = (const float *)(base + ws.dot_k);
        g.state = m->state; g.d_state = ds0; g.g = w0.g; g.gl = w0.gl; g.gb = w0.gb; g.gh = w0.gh; g.masks = w0.masks; g.ml = w0.ml; g.mb = w0.mb;
        g.dg = m->shared_decay ? nullptr : d_log_decay; g.partial = (double *)(base + ws.partial);
        g.L = m->L; g.B = m->B; g.H = m->H; g.elems = elems; g.slices = slices_of(m, m->dv, m->dk);
        g.dot_sl = w0.dot_sl; g.dot_sh = w0.dot_sh;
        g.vec = (elems & 3) == 0 && (((uintptr_t)g.state | (uintptr_t)g.d_state) & 15) == 0;
        for (g.team = 1; g.state && g.team < 64 && g.team * 16 < elems;) g.team *= 2;   // 16 entries a lane at least
        if (few_tokens(m->L)) hipLaunchKernelGGL(decay_grad_short_kernel, dim3((unsigned)((heads * g.team + 255) / 256)), dim3(256), 0, st, g);
        else {
            const int64_t most = m->L / 4 > elems / 16 ? m->L / 4 : elems / 16;   // four tokens and 16 state entries a thread, up to 1 024 threads
            hipLaunchKernelGGL(decay_grad_long_kernel, dim3((unsigned)heads), dim3(most > 1024 ? 1024 : (int)(most + 63) / 64 * 64), 0, st, g);
        }
        HIP_OK(hipGetLastError());
        return finish_decay(m, *d_out, d_state, d_log_decay, g.partial, (float *)(base + ws.dot_k), w0.dot_sl, w0.dot_sh, st);   // (the sums of dk are read by then)
    }
    return FMARL_OK;
}

}  // extern "C"
