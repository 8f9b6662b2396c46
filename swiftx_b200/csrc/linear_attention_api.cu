// C entry points of linear attention: argument checks, the segment plan, workspaces; and the
// single-token step, a stream over the state.
#include <algorithm>
#include <cstdint>

#include "linear_attention.cuh"
#include "launch_util.cuh"

namespace swx {

// ------------------------------------------------------------------ one token
// S = exp(g) S + k v^T in place, out = scale S^T q.  Reads and writes 8 bytes per state value and
// little else, so it is bound by HBM: one CTA per (row, head), thread = VEC columns of every
// R-th row of the state with four loads in flight, column sums joined through shared memory.
// 256 rows x 32 heads of 64 x 64: 41 to 45 us, 272 MB, 92 to 100 % of the copy rate; 1 x 8: 4 us, a launch.
struct LaStep {
    int H, Hk, dk, dv;
    float scale;
    const void *q, *k, *v;
    int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, g_sb, g_sh;
    const float* g;
    float* s;
    void* out;
};

constexpr int LS_THREADS = 256;

template <typename T, int VEC>
__global__ void __launch_bounds__(LS_THREADS) la_step_kernel(const LaStep p) {
    __shared__ float qs[128], ks[128];
    __shared__ float sum[LS_THREADS * VEC];
    const int h = (int)(blockIdx.x % p.H), hk = h / (p.H / p.Hk);
    const int64_t b = blockIdx.x / p.H;
    const int per = (p.dv + VEC - 1) / VEC, R = LS_THREADS / per;       // threads along a row; rows at once
    const int r = threadIdx.x / per, c = threadIdx.x % per * VEC;
    float* S = p.s + ((int64_t)blockIdx.x * p.dk) * p.dv + c;
    const bool on = r < R;
    float x[4][VEC], acc[VEC] = {};
    auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i0 + i * R;
            if (on && row < p.dk) {
                if (VEC == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(S + (int64_t)row * p.dv);
                else x[i][0] = S[(int64_t)row * p.dv];
            }
        }
    };
    load(r);                                                             // on their way while q, k, v arrive
    for (int i = threadIdx.x; i < p.dk; i += LS_THREADS) {
        qs[i] = Elem<T>::to_f(static_cast<const T*>(p.q)[b * p.q_sb + hk * p.q_sh + i]) * p.scale;
        ks[i] = Elem<T>::to_f(static_cast<const T*>(p.k)[b * p.k_sb + hk * p.k_sh + i]);
    }
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = on ? Elem<T>::to_f(static_cast<const T*>(p.v)[b * p.v_sb + h * p.v_sh + c + j]) : 0.f;
    const float a = expf(p.g[b * p.g_sb + h * p.g_sh]);
    __syncthreads();
    for (int i0 = r; i0 < p.dk; i0 += 4 * R) {
        if (i0 != r) load(i0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i0 + i * R;
            if (!on || row >= p.dk) continue;
            const float kr = ks[row], qr = qs[row];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                x[i][j] = fmaf(a, x[i][j], kr * v[j]);
                acc[j] = fmaf(qr, x[i][j], acc[j]);
            }
            if (VEC == 4) *reinterpret_cast<float4*>(S + (int64_t)row * p.dv) = *reinterpret_cast<const float4*>(x[i]);
            else S[(int64_t)row * p.dv] = x[i][0];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[threadIdx.x * VEC + j] = acc[j];
    __syncthreads();
    for (int i = threadIdx.x; i < p.dv; i += LS_THREADS) {
        float o = 0.f;
        for (int k = 0; k < min(R, p.dk); ++k) o += sum[k * per * VEC + i];
        static_cast<T*>(p.out)[(int64_t)blockIdx.x * p.dv + i] = Elem<T>::from_f(o);
    }
}

// ------------------------------------------------------------------ plans
// Segments of one direction: `nseg` of `segc` chunks of 64 tokens (an even number).
struct LaCut { int nseg, segc; };
struct LaPlan { int nsl, nc; bool tc; LaCut fwd, bwd; };

static LaCut la_cut(int nc, int64_t n) {
    n = std::max<int64_t>(1, std::min<int64_t>(n, nc / 2));
    LaCut c;
    c.segc = (int)((nc + n - 1) / n + 1) / 2 * 2;
    c.nseg = (nc + c.segc - 1) / std::max(1, c.segc);
    return c;
}

// One CTA walks a segment of one head's sequence.  Where the heads leave SMs idle the sequence is
// cut, so that the CTAs fill, and do not exceed, one round on 148 SMs; the states at the segments'
// starts cost one more reading of k and v, and two launches.
//
// The pipelined kernels (linear_attention_tc.cu, one CTA per SM, chunks of 128 tokens) take bf16 heads of up to 64
// from 65 tokens on, and from 129 on where the heads alone take several rounds.  us, theirs / the other
// kernels', forward, heads of 64: 8 heads x 64 tokens 8.5 / 8.5, x 100 8.6 / 10.6, x 512 14.5 / 18.6; 128 heads x 256
// 12.7 / 26.8, x 4096 83 / 187; 149 heads x 128 14.8 / 12.8, x 256 18.6 / 31.1, x 384 23.1 / 44.6; 512 heads x 128
// 30.9 / 22.7, x 256 39.1 / 40.3, x 384 49 / 62, x 4096 310 / 586.
// An uncut walk takes them 6 us and 2 for each chunk; a cut one 14 and 3 for each chunk of a segment, with the states
// and their chain; more than 64 segments make the chain longer than what they save (1 head x 16384
// tokens: 128 segments 28.7 us, 64 26.6, 32 30.3; 8 heads x 1024: uncut 24.8, segments of 4 chunks 27.4, of 2
// 22.5, of 1 18.6; x 512: uncut 16.6, cut 18.6; 64 heads x 2048: uncut 43.8, cut 47.3).
//
// The other kernels have three CTAs on an SM (bf16, two with dk > 64; two of the fp32 backward up to dk 64); the backward
// runs two walks at once, in two rounds rather than one (8 x 2048 x 8 heads of 64: 6 segments 115 us, 3 128, 2 141).
// The fp32 forward, and the fp32 backward above dk 64, fill an SM with one CTA and take two rounds of segments, of a
// third of the walk or less: with two segments the two rounds would be as long as one of whole walks, and the
// states come on top (4096 tokens, heads of 64, forward: 148 heads 734 us whole, 873 as two; 100 heads 699 and 793;
// 74 heads 697 whole, 476 as four, 505 as two in one round; dk 128, 100 heads, forward and backward: 5.78 ms with the backward
// whole, 6.29 as two; 40 heads 2.09 as seven, 2.40 as three in one round).  Where the backward's
// last segment would be less than half of the others, all are made shorter by two chunks (forward and
// backward, 64 heads x 2048 tokens 194 -> 191 us, x 1664 166 -> 153, 80 x 2100 238 -> 218).
static LaPlan la_plan(const swx_linattn_args* a) {
    LaPlan q{};
    q.nsl = (int)((a->dv + LA_DV - 1) / LA_DV);
    q.nc = (int)((a->seqlen + LA_C - 1) / LA_C);
    const int64_t heads = a->batch * a->heads * q.nsl, chunks = (q.nc + 1) / 2;
    q.tc = a->dtype == SWX_DTYPE_BF16 && a->dk <= 64 && q.nc >= (heads > 148 ? 3 : 2);
    const bool f32 = a->dtype == SWX_DTYPE_F32;
    const int64_t parts = 148 * (a->dk > 64 || f32 ? 2 : 3) / heads;
    auto one_to_an_sm = [parts](bool yes) { return yes && parts == 2 ? 1 : parts; };
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>(148 / heads, 64)), segment = (chunks + n - 1) / n;
    q.fwd = la_cut(q.nc, !q.tc ? one_to_an_sm(f32) : 2 * chunks > 3 * segment + 8 ? n : 1);
    q.bwd = la_cut(q.nc, one_to_an_sm(f32 && a->dk > 64));
    if (q.bwd.nseg > 1 && 2 * (q.nc - (q.bwd.nseg - 1) * q.bwd.segc) < q.bwd.segc) {       // a short last segment
        q.bwd.segc -= 2;
        q.bwd.nseg = (q.nc + q.bwd.segc - 1) / q.bwd.segc;
    }
    return q;
}

static int la_check(const swx_linattn_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->heads < 1 || a->qk_heads < 1 || a->dk < 1 || a->dv < 1) return SWX_ERR_INVALID_ARG;
    if (a->heads % a->qk_heads) return SWX_ERR_INVALID_ARG;
    if (a->dk > 128 || a->dv > 128) return SWX_ERR_UNSUPPORTED;
    if (a->dtype != SWX_DTYPE_F32 && a->dtype != SWX_DTYPE_BF16) return SWX_ERR_UNSUPPORTED;
    if (a->batch > (1 << 24) || a->heads > (1 << 16) || a->seqlen > (1 << 28)) return SWX_ERR_UNSUPPORTED;
    if (a->batch * a->heads * 2 > (int64_t(1) << 22)) return SWX_ERR_UNSUPPORTED;      // CTAs per launch
    return SWX_OK;
}

// The buffers that the caller makes for the states and the scratch start on 16 bytes.
static bool la_aligned(const swx_linattn_args* a) {
    return ((reinterpret_cast<uintptr_t>(a->final_state) | reinterpret_cast<uintptr_t>(a->seg_states) | reinterpret_cast<uintptr_t>(a->workspace)) & 15) == 0;
}

struct LaWs { int64_t dec, seg, rin, net, yseg, dg, dq, dk, total; };

static int64_t up(int64_t v) { return (v + 255) / 256 * 256; }

static bool la_shared(const swx_linattn_args* a, const LaPlan& q) { return a->heads != a->qk_heads || q.nsl > 1; }

// The backward's scratch: `seg` holds the gradient of the state at each segment's end.
static LaWs la_ws(const swx_linattn_args* a, const LaPlan& q) {
    LaWs w{};
    const int64_t bh = a->batch * a->heads, bv = bh * q.nsl;
    int64_t o = 0;
    auto take = [&](int64_t floats) { const int64_t at = o; o += up(floats * 4); return at; };
    w.dec = take(bh * q.bwd.nseg);
    w.seg = take(q.bwd.nseg > 1 ? bh * q.bwd.nseg * a->dk * a->dv : 0);
    w.rin = take(bv * a->seqlen);
    w.net = take(bv * a->seqlen);
    w.yseg = take(bv * (q.bwd.nseg + 1));
    w.dg = take(a->decay_per_head ? 2 * bh * q.bwd.nseg : 0);
    w.dq = take(la_shared(a, q) ? bv * a->seqlen * a->dk : 0);
    w.dk = take(la_shared(a, q) ? bv * a->seqlen * a->dk : 0);
    w.total = o;
    return w;
}

static LaTensor la_tensor(const void* p, int64_t sb, int64_t sl, int64_t sh, int64_t nb, int64_t nl, int64_t nh, int es) {
    LaTensor t{p, nb > 1 ? sb : 0, nl > 1 ? sl : 0, nh > 1 ? sh : 0, false};
    t.vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (t.sb * es) % 16 == 0 && (t.sl * es) % 16 == 0 && (t.sh * es) % 16 == 0;
    return t;
}

static LaDev la_pack(const swx_linattn_args* a, const LaPlan& q, const LaCut& c) {
    LaDev p{};
    const int es = a->dtype == SWX_DTYPE_F32 ? 4 : 2;
    p.b = (int)a->batch; p.L = (int)a->seqlen; p.H = (int)a->heads; p.Hk = (int)a->qk_heads; p.dk = (int)a->dk; p.dv = (int)a->dv;
    p.polls = a->wait_polls == 0 ? LT_POLLS : (uint32_t)std::max(0, a->wait_polls);
    p.nsl = q.nsl; p.tc = q.tc; p.nc = q.nc; p.nseg = c.nseg; p.segc = c.segc;
    p.q = la_tensor(a->q, a->q_sb, a->q_sl, a->q_sh, a->batch, a->seqlen, a->qk_heads, es);
    p.k = la_tensor(a->k, a->k_sb, a->k_sl, a->k_sh, a->batch, a->seqlen, a->qk_heads, es);
    p.v = la_tensor(a->v, a->v_sb, a->v_sl, a->v_sh, a->batch, a->seqlen, a->heads, es);
    p.dout = la_tensor(a->dout, a->do_sb, a->do_sl, a->do_sh, a->batch, a->seqlen, a->heads, es);
    p.g = a->log_decay; p.g_sb = a->g_sb; p.g_sl = a->g_sl; p.g_sh = a->g_sh;
    p.lengths = a->lengths; p.scale = a->scale; p.s0 = a->initial_state; p.out = a->out; p.s_last = a->final_state;
    p.ds = a->dfinal_state; p.ds0 = a->dinitial_state;
    auto whole = [es](const void* o, int64_t d) { return (reinterpret_cast<uintptr_t>(o) & 15) == 0 && (d * es) % 16 == 0; };
    p.vec_o = whole(a->out, a->dv) && whole(a->dv_out, a->dv);
    p.vec_qk = whole(a->dq, a->dk) && whole(a->dk_out, a->dk);
    return p;
}

}  // namespace swx

using namespace swx;

extern "C" {

int64_t swx_linattn_args_size(void) { return (int64_t)sizeof(swx_linattn_args); }

int swx_linattn_segments(const swx_linattn_args* a) {
    const int c = la_check(a);
    if (c != SWX_OK) return -c;
    return a->batch * a->seqlen == 0 ? 1 : la_plan(a).bwd.nseg;
}

int64_t swx_linattn_fwd_workspace_bytes(const swx_linattn_args* a) {
    const int c = la_check(a);
    if (c != SWX_OK) return -c;
    if (a->batch * a->seqlen == 0) return 0;
    const int64_t n = la_plan(a).fwd.nseg;
    return n > 1 ? up(a->batch * a->heads * n * 4) + up(a->batch * a->heads * n * a->dk * a->dv * 4) : 0;
}

int64_t swx_linattn_bwd_workspace_bytes(const swx_linattn_args* a) {
    const int c = la_check(a);
    if (c != SWX_OK) return -c;
    return a->batch * a->seqlen == 0 ? 0 : la_ws(a, la_plan(a)).total;
}

int swx_linattn_fwd(const swx_linattn_args* a, void* stream) {
    const int c = la_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->batch == 0) return SWX_OK;
    if (a->seqlen == 0) {
        if (!a->final_state) return SWX_OK;
        const size_t n = (size_t)(a->batch * a->heads * a->dk * a->dv) * 4;
        const cudaError_t e = a->initial_state ? cudaMemcpyAsync(a->final_state, a->initial_state, n, cudaMemcpyDeviceToDevice, st)
                                               : cudaMemsetAsync(a->final_state, 0, n, st);
        return e == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
    }
    if (!a->q || !a->k || !a->v || !a->log_decay || !a->out) return SWX_ERR_INVALID_ARG;
    if (!la_aligned(a)) return SWX_ERR_INVALID_ARG;
    const LaPlan q = la_plan(a);
    if (q.fwd.nseg > 1 && (!a->workspace || a->workspace_bytes < swx_linattn_fwd_workspace_bytes(a))) return SWX_ERR_INVALID_ARG;
    LaDev p = la_pack(a, q, q.fwd);
    p.dec = static_cast<float*>(a->workspace);
    p.seg = p.dec + up(a->batch * a->heads * q.fwd.nseg * 4) / 4;
    p.save = q.bwd.nseg > 1 ? a->seg_states : nullptr;
    p.save_n = q.bwd.nseg;
    p.save_c = q.bwd.segc;
    if (q.fwd.nseg > 1 && la_launch_state(p, a->dtype, false, st) != cudaSuccess) return SWX_ERR_CUDA;
    return la_launch_fwd(p, a->dtype, st) == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
}

int swx_linattn_bwd(const swx_linattn_args* a, void* stream) {
    const int c = la_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t state = (size_t)(a->batch * a->heads * a->dk * a->dv) * 4;
    if (a->batch * a->seqlen == 0) {
        cudaError_t e = cudaSuccess;
        if (a->decay_per_head && a->dlog_decay) e = cudaMemsetAsync(a->dlog_decay, 0, (size_t)a->heads * 4, st);
        if (e == cudaSuccess && a->dinitial_state && state)
            e = a->dfinal_state ? cudaMemcpyAsync(a->dinitial_state, a->dfinal_state, state, cudaMemcpyDeviceToDevice, st)
                                : cudaMemsetAsync(a->dinitial_state, 0, state, st);
        return e == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
    }
    if (!a->q || !a->k || !a->v || !a->log_decay || !a->dout || !a->dq || !a->dk_out || !a->dv_out || !a->dlog_decay || !a->workspace)
        return SWX_ERR_INVALID_ARG;
    const LaPlan q = la_plan(a);
    const LaWs w = la_ws(a, q);
    if (!la_aligned(a)) return SWX_ERR_INVALID_ARG;
    if (a->workspace_bytes < w.total || (q.bwd.nseg > 1 && !a->seg_states)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    auto at = [ws](int64_t o) { return reinterpret_cast<float*>(ws + o); };
    LaDev p = la_pack(a, q, q.bwd);
    // the reverse states: 64 heads of 8192 tokens (22 chunks a segment) 619 us with the pipelined kernel, 625 with
    // the other one; 64 x 2048 (6 chunks) 199 and 198
    p.tc = p.tc && q.bwd.segc >= 16;
    p.seg = a->seg_states;
    p.dec = at(w.dec); p.rseg = at(w.seg); p.rin = at(w.rin); p.yseg = at(w.yseg);
    p.shared_qk = la_shared(a, q);
    p.dq = p.shared_qk ? at(w.dq) : a->dq;
    p.dk_out = p.shared_qk ? at(w.dk) : a->dk_out;
    p.dv_out = a->dv_out;
    p.net = at(w.net);
    p.dg = a->decay_per_head ? nullptr : a->dlog_decay;
    p.dg_part = reinterpret_cast<double*>(ws + w.dg);
    auto whole = [a](const void* o, int64_t d) {
        return (reinterpret_cast<uintptr_t>(o) & 15) == 0 && (d * (a->dtype == SWX_DTYPE_F32 ? 4 : 2)) % 16 == 0;
    };
    p.vec_o = whole(a->dv_out, a->dv);
    if (q.bwd.nseg > 1 && la_launch_state(p, a->dtype, true, st) != cudaSuccess) return SWX_ERR_CUDA;
    if (la_launch_bwd(p, a->dtype, st) != cudaSuccess) return SWX_ERR_CUDA;
    if (a->decay_per_head && la_launch_dg_head(p.dg_part, a->dlog_decay, p.H, p.b * p.nseg, st) != cudaSuccess) return SWX_ERR_CUDA;
    if (p.shared_qk) {
        const int per = (int)(a->heads / a->qk_heads) * q.nsl;
        if (la_launch_group_sum(static_cast<float*>(p.dq), static_cast<float*>(p.dk_out), a->dq, a->dk_out, a->dtype, a->batch * a->seqlen, p.Hk,
                                per, p.dk, st) != cudaSuccess)
            return SWX_ERR_CUDA;
    }
    return SWX_OK;
}

int swx_linattn_step(const swx_linattn_args* a, void* stream) {
    const int c = la_check(a);
    if (c != SWX_OK) return c;
    if (a->batch == 0) return SWX_OK;
    if (!a->q || !a->k || !a->v || !a->log_decay || !a->out || !a->final_state) return SWX_ERR_INVALID_ARG;
    LaStep p{};
    p.H = (int)a->heads; p.Hk = (int)a->qk_heads; p.dk = (int)a->dk; p.dv = (int)a->dv; p.scale = a->scale;
    p.q = a->q; p.q_sb = a->q_sb; p.q_sh = a->q_sh;
    p.k = a->k; p.k_sb = a->k_sb; p.k_sh = a->k_sh;
    p.v = a->v; p.v_sb = a->v_sb; p.v_sh = a->v_sh;
    p.g = a->log_decay; p.g_sb = a->g_sb; p.g_sh = a->g_sh;
    p.s = a->final_state; p.out = a->out;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)(a->batch * a->heads);
    const bool vec = a->dv % 4 == 0 && (reinterpret_cast<uintptr_t>(a->final_state) & 15) == 0;
    const bool f32 = a->dtype == SWX_DTYPE_F32;
    if (f32 && vec) la_step_kernel<float, 4><<<grid, LS_THREADS, 0, st>>>(p);
    else if (f32) la_step_kernel<float, 1><<<grid, LS_THREADS, 0, st>>>(p);
    else if (vec) la_step_kernel<__nv_bfloat16, 4><<<grid, LS_THREADS, 0, st>>>(p);
    else la_step_kernel<__nv_bfloat16, 1><<<grid, LS_THREADS, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
}

}  // extern "C"
