// Linear attention with a decay for each head, chunked: forward kernel, segment states.
#include "linear_attention.cuh"
#include "launch_util.cuh"

#include <algorithm>

namespace swx {

// ------------------------------------------------------------------ one segment's state
// From zero: forward, S = sum of the segment's decayed k_s v_s^T; reverse (the state's
// gradient, walked from the segment's end), sum of exp(G_t) scale q_t do_t^T.  The segment's
// decay comes with it.
template <typename T, int DK, bool REV>
__global__ void __launch_bounds__(LA_THREADS) la_state_kernel(const LaDev p) {
    using Sh = LaShape<T, DK>;
    extern __shared__ __align__(16) uint8_t smem[];
    T* xs = reinterpret_cast<T*>(smem);
    T* ys = xs + 2 * Sh::QK;
    __shared__ LaGates gates[LA_RING];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rw = warp;
    // the last segment's state (reverse: the first one's) is not needed
    const int nrun = p.nseg - 1;
    const int seg = (int)(blockIdx.x % nrun) + (REV ? 1 : 0);
    const int64_t vh = blockIdx.x / nrun;
    const int sl = (int)(vh % p.nsl), h = (int)(vh / p.nsl % p.H), b = (int)(vh / p.nsl / p.H);
    const int hk = h / (p.H / p.Hk), c0 = sl * LA_DV, cols = min(LA_DV, p.dv - c0), len = la_len(p, b);
    const int first = seg * p.segc, last = min(min(first + p.segc, p.nc), (len + LA_C - 1) / LA_C);   // chunks with tokens
    const int n = max(0, last - first);

    float S[Sh::MI][Sh::NI][4] = {};
    auto chunk = [&](int i) { return REV ? last - 1 - i : first + i; };
    auto load = [&](int i) {
        const int t0 = chunk(i) * LA_C, rows = min(LA_C, len - t0);
        la_load<T, DK, Sh::LDK>(xs + (i & 1) * Sh::QK, REV ? p.q : p.k, b, t0, hk, 0, rows, p.dk);
        la_load<T, LA_DV, Sh::LDV>(ys + (i & 1) * Sh::V, REV ? p.dout : p.v, b, t0, h, c0, rows, cols);
        cp_async_commit();
    };
    if (n > 0) load(0);
    LaGateRing ring;
    ring.start(gates, p, b, h, len, n, chunk, warp, lane);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        cp_async_wait<0>();
        __syncthreads();
        if (i + 1 < n) load(i + 1);
        const LaGates& gt = ring.take(p, b, h, len, n, i, chunk, warp, lane);
        la_state_update<T, DK, REV>(S, xs + (i & 1) * Sh::QK, ys + (i & 1) * Sh::V, gt, p.scale, rw, lane);
        ring.make(n, i, warp, lane);
    }
    __shared__ double sums[4];
    if (lane == 0) sums[warp] = ring.total;
    __syncthreads();
    float* dst = (REV ? p.rseg : p.seg) + (((int64_t)b * p.H + h) * p.nseg + seg) * p.dk * p.dv;
    la_state_write<T, DK>(S, dst, p, c0, rw, lane);
    if (threadIdx.x == 0 && sl == 0) p.dec[((int64_t)b * p.H + h) * p.nseg + seg] =
            ex2((float)((sums[0] + sums[1]) + (sums[2] + sums[3])));
}

// Segment sums -> the state at each segment's start (reverse: its gradient at each segment's
// end), in place; thread = one value of one head's state.
__global__ void __launch_bounds__(256) la_chain_kernel(const LaDev p, bool rev) {
    const int64_t n = (int64_t)p.dk * p.dv, per = (n + 255) / 256;
    const int64_t bh = blockIdx.x / per, e = (blockIdx.x % per) * 256 + threadIdx.x;
    if (e >= n) return;
    const float* start = rev ? p.ds : p.s0;
    float run = start ? start[bh * n + e] : 0.f;
    float* s = (rev ? p.rseg : p.seg) + bh * p.nseg * n + e;
    const float* d = p.dec + bh * p.nseg;
    for (int i0 = 0; i0 < p.nseg; i0 += 8) {           // eight loads in flight before the first store
        float u[8], dec[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = rev ? p.nseg - 1 - i0 - i : i0 + i;
            const bool in = i0 + i + 1 < p.nseg;
            u[i] = in ? s[k * n] : 0.f;
            dec[i] = in ? d[k] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i >= p.nseg) break;
            s[(rev ? p.nseg - 1 - i0 - i : i0 + i) * n] = run;
            run = dec[i] * run + u[i];
        }
    }
}

// ------------------------------------------------------------------ forward
// Warp = 16 tokens of the chunk (and a quarter of the state).  Per chunk: the state's part of
// the output, exp(G_t) S^T q; the decayed scores of the 16 tokens with the tokens up to them; their product with v; then the
// state's update.  The scores, and the state where it is read out, are rounded to the inputs' type once as their products'
// operands: each term of a bf16 output has one factor rounded, and so a size of error like the output's own
// rounding (2.35e-3 together, 1.66e-3 by itself), where three pieces would be three products for one.  The state that
// is carried is fp32.  Tiles arrive by cp.async one chunk ahead.  Bound by the latency of its own steps, three warps to
// an SM quarter (two at dk 128): 16 x 512 x 16 heads, dk 128, dv 64, bf16 55 us; 2 x 777 x 6 heads, 40 and 56, fp32 47 us.
template <typename T, int DK> struct LaFwd {
    using Sh = LaShape<T, DK>;
    static constexpr int SMEM = (int)sizeof(T) * (4 * Sh::QK + 2 * Sh::V + Sh::S);
};

template <typename T, int DK>
__global__ void __launch_bounds__(LA_THREADS, sizeof(T) == 4 ? 1 : DK == 128 ? 2 : 3) la_fwd_kernel(const LaDev p) {
    using Sh = LaShape<T, DK>;
    extern __shared__ __align__(16) uint8_t smem[];
    T* qs = reinterpret_cast<T*>(smem);
    T* ks = qs + 2 * Sh::QK;
    T* vs = ks + 2 * Sh::QK;
    T* ss = vs + 2 * Sh::V;
    __shared__ LaGates gates[LA_RING];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rw = (warp + blockIdx.x) & 3;           // later tokens have more scores: spread them over the SM's quarters
    const int seg = (int)(blockIdx.x % p.nseg);
    const int64_t vh = blockIdx.x / p.nseg;
    const int sl = (int)(vh % p.nsl), h = (int)(vh / p.nsl % p.H), b = (int)(vh / p.nsl / p.H);
    const int hk = h / (p.H / p.Hk), c0 = sl * LA_DV, cols = min(LA_DV, p.dv - c0), len = la_len(p, b);
    const int first = seg * p.segc, last = min(first + p.segc, p.nc);
    const int live = max(first, min(last, (len + LA_C - 1) / LA_C));          // chunks from here on hold no token
    const int64_t bh = (int64_t)b * p.H + h, ssz = (int64_t)p.dk * p.dv;

    float S[Sh::MI][Sh::NI][4];
    la_state_read<T, DK>(S, p.nseg > 1 ? p.seg + (bh * p.nseg + seg) * ssz : (p.s0 ? p.s0 + bh * ssz : nullptr), p, c0, rw, lane);
    la_state_share<T, DK, 1>(S, ss, rw, lane);
    auto load = [&](int i) {
        const int t0 = (first + i) * LA_C, rows = min(LA_C, len - t0), u = i & 1;
        la_load<T, DK, Sh::LDK>(qs + u * Sh::QK, p.q, b, t0, hk, 0, rows, p.dk);
        la_load<T, DK, Sh::LDK>(ks + u * Sh::QK, p.k, b, t0, hk, 0, rows, p.dk);
        la_load<T, LA_DV, Sh::LDV>(vs + u * Sh::V, p.v, b, t0, h, c0, rows, cols);
        cp_async_commit();
    };
    const int n = live - first;
    auto chunk = [&](int i) { return first + i; };
    if (n > 0) load(0);
    LaGateRing ring;
    ring.start(gates, p, b, h, len, n, chunk, warp, lane);
    T* out = static_cast<T*>(p.out);
    const int64_t o_sl = (int64_t)p.H * p.dv;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int u = i & 1, t0 = (first + i) * LA_C;
        la_state_save<T, DK>(S, p, bh, first + i, c0, rw, lane);
        cp_async_wait<0>();
        __syncthreads();
        if (i + 1 < n) load(i + 1);
        const LaGates& gt = ring.take(p, b, h, len, n, i, chunk, warp, lane);
        T* q = qs + u * Sh::QK;
        const T* k = ks + u * Sh::QK;
        const T* v = vs + u * Sh::V;
        const T* s = ss;
        float o[8][4] = {}, sc[8][4] = {};
#pragma unroll
        for (int k0 = 0; k0 < DK; k0 += 16) {
            FragA<T> a;
            load_a(a, q, Sh::LDK, 16 * rw, k0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                FragB<T> f[2];
                load_b2_t(f, s, Sh::LDV, 16 * j, k0, lane);
                mma(o[2 * j], a, f[0]);
                mma(o[2 * j + 1], a, f[1]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j <= rw) {
                    FragB<T> f[2];
                    load_b2(f, k, Sh::LDK, 16 * j, k0, lane);
                    mma(sc[2 * j], a, f[0]);
                    mma(sc[2 * j + 1], a, f[1]);
                }
        }
        const int r0 = 16 * rw + (lane >> 2);
        const float e0 = gt.pre(r0) * p.scale, e1 = gt.pre(r0 + 8) * p.scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) { o[j][0] *= e0; o[j][1] *= e0; o[j][2] *= e1; o[j][3] *= e1; }
        const float2 G0 = gt.G[r0], G1 = gt.G[r0 + 8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j <= rw) {
                la_mask_rows(sc[2 * j], sc[2 * j + 1], gt, j, rw, r0, G0, G1, p.scale, lane);
                FragA<T> a;
                frag_from(a, sc[2 * j], sc[2 * j + 1]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    FragB<T> f[2];
                    load_b2_t(f, v, Sh::LDV, 16 * c, 16 * j, lane);
                    mma(o[2 * c], a, f[0]);
                    mma(o[2 * c + 1], a, f[1]);
                }
            }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) store_tile<1>(q, Sh::LDK, 0, 16 * rw, 8 * j, o[j], lane);   // this warp's own rows of q
        const int tr = t0 + 16 * rw;
        la_store<T, LA_DV, Sh::LDK>(q + 16 * rw * Sh::LDK, out + ((int64_t)b * p.L + tr) * o_sl + (int64_t)h * p.dv + c0, o_sl,
                                    len - tr, p.L - tr, cols, p.vec_o, lane);
        la_state_update<T, DK, false>(S, k, v, gt, 1.f, rw, lane);
        __syncthreads();                                  // all have read the state that this replaces
        la_state_share<T, DK, 1>(S, ss, rw, lane);
        ring.make(n, i, warp, lane);
    }
    // rows behind the row's last token
    for (int c = live; c < last; ++c) la_state_save<T, DK>(S, p, bh, c, c0, rw, lane);
    la_zero_rows<T>(p, b, h, c0, cols, live * LA_C, min(last * LA_C, p.L), threadIdx.x, LA_THREADS);
    if (p.s_last && seg == p.nseg - 1) la_state_write<T, DK>(S, p.s_last + bh * ssz, p, c0, rw, lane);
}

// ------------------------------------------------------------------ launches
template <typename T, int DK>
static cudaError_t fwd(const LaDev& p, cudaStream_t st) {
    auto k = la_fwd_kernel<T, DK>;
    constexpr int smem = LaFwd<T, DK>::SMEM;
    cudaError_t e = allow_smem(k, smem);
    if (e != cudaSuccess) return e;
    k<<<(unsigned)((int64_t)p.b * p.H * p.nsl * p.nseg), LA_THREADS, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int DK, bool REV>
static cudaError_t state(const LaDev& p, cudaStream_t st) {
    auto k = la_state_kernel<T, DK, REV>;
    constexpr int smem = (int)sizeof(T) * 2 * (LaShape<T, DK>::QK + LaShape<T, DK>::V);
    cudaError_t e = allow_smem(k, smem);
    if (e != cudaSuccess) return e;
    k<<<(unsigned)((int64_t)p.b * p.H * p.nsl * (p.nseg - 1)), LA_THREADS, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t fwd_dk(const LaDev& p, cudaStream_t st) {
    return p.dk <= 32 ? fwd<T, 32>(p, st) : p.dk <= 64 ? fwd<T, 64>(p, st) : fwd<T, 128>(p, st);
}
template <typename T, bool REV>
static cudaError_t state_dk(const LaDev& p, cudaStream_t st) {
    return p.dk <= 32 ? state<T, 32, REV>(p, st) : p.dk <= 64 ? state<T, 64, REV>(p, st) : state<T, 128, REV>(p, st);
}

cudaError_t la_launch_fwd(const LaDev& p, int dtype, cudaStream_t st) {
    if (dtype == SWX_DTYPE_F32) return fwd_dk<float>(p, st);
    bool taken = false;
    const cudaError_t e = lt_launch_fwd(p, &taken, st);
    return taken ? e : fwd_dk<__nv_bfloat16>(p, st);
}
cudaError_t la_launch_state(const LaDev& p, int dtype, bool reverse, cudaStream_t st) {
    cudaError_t e;
    bool taken = false;
    if (dtype == SWX_DTYPE_F32) e = reverse ? state_dk<float, true>(p, st) : state_dk<float, false>(p, st);
    else if ((e = lt_launch_state(p, reverse, &taken, st)), !taken)
        e = reverse ? state_dk<__nv_bfloat16, true>(p, st) : state_dk<__nv_bfloat16, false>(p, st);
    if (e != cudaSuccess) return e;
    const int64_t per = ((int64_t)p.dk * p.dv + 255) / 256;
    la_chain_kernel<<<(unsigned)((int64_t)p.b * p.H * per), 256, 0, st>>>(p, reverse);
    return cudaGetLastError();
}

}  // namespace swx
