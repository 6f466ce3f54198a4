// C-ABI of the policy operators (include/fmarl.h, "the policy's operators"): a translation unit of its own, linked into libfmarl.so.
#include <stdint.h>

#include "fmarl_memory.hip"

using namespace fmarl;
using namespace fmarl::policy;

#define HIP_OK(call)                                                                                        \
    do {                                                                                                    \
        hipError_t e_ = (call);                                                                             \
        if (e_ != hipSuccess) return policy_fail(FMARL_EHIP, #call ": %s", hipGetErrorString(e_));          \
    } while (0)

namespace {

int elem_bytes(int dtype) { return dtype == FMARL_T_F32 ? 4 : 2; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// rows start on multiples of four elements and hold a multiple of four: one load takes four
int rows_vec(const FmarlRows &r, int d, int dtype) {
    return (d & 3) == 0 && (r.stride_l & 3) == 0 && (r.stride_b & 3) == 0 && (r.stride_h & 3) == 0 &&
           ((uintptr_t)r.data & (4 * elem_bytes(dtype) - 1)) == 0;
}

WalkRows walk_rows(const FmarlRows &r, int d, int dtype) { return WalkRows{(char *)r.data, r.stride_l, r.stride_b, r.stride_h, rows_vec(r, d, dtype)}; }

// ---- memory -------------------------------------------------------------------------------------------------------------
const int kMaxMemoryDim = 128;

int memory_check(const FmarlMemory *m, const char *who) {
    if (!m) return policy_fail(FMARL_EINVAL, "%s: null argument", who);
    if (m->L < 0 || m->B < 0 || m->H < 1) return policy_fail(FMARL_EINVAL, "%s: L and B must not be negative, H must be positive", who);
    if (m->dk < 1 || m->dk > kMaxMemoryDim || m->dv < 1 || m->dv > kMaxMemoryDim) return policy_fail(FMARL_EINVAL, "%s: dk and dv must lie in 1..128", who);
    if (m->dtype < FMARL_T_F32 || m->dtype > FMARL_T_F16) return policy_fail(FMARL_EINVAL, "%s: unknown dtype", who);
    if (m->shared_decay < 0 || m->shared_decay > 1 || (m->shared_decay && (m->decay_stride_l || m->decay_stride_b)))
        return policy_fail(FMARL_EINVAL, "%s: shared_decay must be 0, or 1 with strides of 0 over tokens and sequences", who);
    if (m->B > (1ll << 31) / m->H || m->L > (1ll << 40)) return policy_fail(FMARL_EINVAL, "%s: too many sequences or tokens", who);
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

int tiles(int d) { return d <= 16 ? 1 : d <= 32 ? 2 : d <= 64 ? 4 : 8; }
// columns of z that one wave takes, in tiles of 16: the state's dy x dz accumulators have to fit its registers beside the operands
int slice_tiles(int dy, int dz) { const int t = tiles(dz), most = tiles(dy) == 8 ? 2 : 4; return t > most ? most : t; }
int slices_of(int dy, int dz) { const int w = 16 * slice_tiles(dy, dz); return (dz + w - 1) / w; }

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
    if (backward) {
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
    switch (tiles(w.dy)) {
    case 1: launch_walk_nz<T, 1>(w, blocks, st); break;
    case 2: launch_walk_nz<T, 2>(w, blocks, st); break;
    case 4: launch_walk_nz<T, 4>(w, blocks, st); break;
    default: launch_walk_nz<T, 8>(w, blocks, st); break;
    }
}

int launch_walk(Walk w, int dtype, hipStream_t st) {
    w.slices = slices_of(w.dy, w.dz);
    const int64_t blocks = (w.B * w.H * w.nseg * w.slices + 3) / 4;
    if (blocks > 0x7fffffff) return policy_fail(FMARL_EINVAL, "memory: too many sequences");
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
    if (blocks > 0x7fffffff) return policy_fail(FMARL_EINVAL, "memory: too many sequences");
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
    if (blocks > 0x7fffffff) return policy_fail(FMARL_EINVAL, "fmarl_memory_step: too many sequences");
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
