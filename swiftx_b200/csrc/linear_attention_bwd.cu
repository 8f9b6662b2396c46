// Linear attention with a decay for each head, chunked: gradients.
//
// With P_ts = scale M_ts q_t . k_s and A_ts = scale M_ts do_t . v_s (s <= t), S_prev the state at
// the chunk's start and D the gradient of the state at its end:
//   dq_t = sum_s A_ts k_s + scale exp(G_t) S_prev do_t
//   dk_s = sum_t A_ts q_t + exp(G_64 - G_s) D v_s
//   dv_s = sum_t P_ts do_t + exp(G_64 - G_s) D^T k_s
//   D_prev = exp(G_64) D + sum_t scale exp(G_t) q_t do_t^T
// A forward walk carries S and gives dq; a reverse walk carries D and gives dk, dv.  The decay's
// gradient dg_t is the sum of all terms of the result that cross from before t to t or later, so
// dg_t = dg_{t+1} + q_t . dq_t - k_t . dk_t, from <S, D> at the segment's end.  The dot
// products are taken from unrounded sums: sum_s A_ts (q_t . k_s) from the two score tiles, and the
// states' parts with the state kept to 24 bits (three bf16 pieces), so that dg, fp32, has fp32
// accuracy although dq and dk are rounded to the inputs' type.  A and P are rounded to the inputs' type once as the
// operands of their products with k, q and dout, and D for dv: one rounded factor in each term.
#include "linear_attention.cuh"
#include "launch_util.cuh"

namespace swx {

template <typename T> struct Planes { static constexpr int N = sizeof(T) == 4 ? 1 : 3; };

// acc[DK / 8] += rows 16 rw of x (16 x 64) times S^T, S in shared memory in full precision.
// The small pieces of S come first: the tensor core cuts the low bits of each addition off, and with 12 additions at the
// sum's full size instead of 4 the decay's gradient is up to twice as far off (16 x 512 x 16 heads, dk 128, a decay for each:
// 2.7e-6 and 1.4e-6; the walks 1 % slower for the operand's repeated reads).
template <typename T, int DK>
__device__ __forceinline__ void la_times_state_t(float (&acc)[DK / 8][4], const T* x, const T* s, int rw, int lane) {
    using Sh = LaShape<T, DK>;
#pragma unroll 1
    for (int pl = Planes<T>::N - 1; pl >= 0; --pl)
#pragma unroll LA_UNROLL<T>
        for (int k0 = 0; k0 < LA_DV; k0 += 16) {
            FragA<T> a;
            load_a(a, x, Sh::LDV, 16 * rw, k0, lane);
#pragma unroll
            for (int j = 0; j < DK / 16; ++j) {
                FragB<T> f[2];
                load_b2(f, s + pl * Sh::S, Sh::LDV, 16 * j, k0, lane);
                mma(acc[2 * j], a, f[0]);
                mma(acc[2 * j + 1], a, f[1]);
            }
        }
}

// Row dot products of an accumulator (16 x DK) with this warp's rows of a tile in shared memory:
// {row g, row g + 8}, complete in every lane of the quad.
template <typename T, int DK>
__device__ __forceinline__ float2 la_row_dot(const float (&acc)[DK / 8][4], const T* x, int ld, int rw, int lane) {
    float2 r = make_float2(0.f, 0.f);
    const T* p = x + (16 * rw + (lane >> 2)) * ld + 2 * (lane & 3);
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) {
        r.x += acc[j][0] * Elem<T>::to_f(p[8 * j]) + acc[j][1] * Elem<T>::to_f(p[8 * j + 1]);
        r.y += acc[j][2] * Elem<T>::to_f(p[8 * ld + 8 * j]) + acc[j][3] * Elem<T>::to_f(p[8 * ld + 8 * j + 1]);
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
        r.x += __shfl_xor_sync(0xffffffffu, r.x, o);
        r.y += __shfl_xor_sync(0xffffffffu, r.y, o);
    }
    return r;
}

// A warp's 16 rows of dq or dk: rounded, through this warp's own rows of `tile`, or the fp32
// part of this head where several heads share the gradient.
template <typename T, int DK>
__device__ __forceinline__ void la_store_qk(const float (&acc)[DK / 8][4], T* tile, void* dst, const LaDev& p, int b, int hk,
                                            int64_t vhead, int tr, int len, int rw, int lane) {
    using Sh = LaShape<T, DK>;
    if (p.shared_qk) {
        const int64_t sl = (int64_t)p.H * p.nsl * p.dk;
        float* o = static_cast<float*>(dst) + ((int64_t)b * p.L + tr) * sl + vhead * p.dk;
#pragma unroll
        for (int j = 0; j < DK / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = (lane >> 2) + 8 * (e >> 1), c = 8 * j + 2 * (lane & 3) + (e & 1);
                if (c < p.dk && tr + r < p.L) o[(int64_t)r * sl + c] = tr + r < len ? acc[j][e] : 0.f;
            }
        return;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) store_tile<1>(tile, Sh::LDK, 0, 16 * rw, 8 * j, acc[j], lane);
    const int64_t sl = (int64_t)p.Hk * p.dk;
    la_store<T, DK, Sh::LDK>(tile + 16 * rw * Sh::LDK, static_cast<T*>(dst) + ((int64_t)b * p.L + tr) * sl + (int64_t)hk * p.dk, sl,
                             len - tr, p.L - tr, p.dk, p.vec_qk, lane);
}

// <a state in registers, one in memory (null: zero)> to `dst`, by the whole CTA; red: 4 floats that no one uses now.
template <typename T, int DK>
__device__ __forceinline__ void la_state_dot(const float (&S)[LaShape<T, DK>::MI][LaShape<T, DK>::NI][4], const float* other, float* dst,
                                             const LaDev& p, int c0, int rw, int lane, float* red) {
    using Sh = LaShape<T, DK>;
    float y = 0.f;
    if (other) {
        float R[Sh::MI][Sh::NI][4];
        la_state_read<T, DK>(R, other, p, c0, rw, lane);
#pragma unroll
        for (int i = 0; i < Sh::MI; ++i)
#pragma unroll
            for (int j = 0; j < Sh::NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) y += S[i][j][e] * R[i][j][e];
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (lane == 0) red[rw] = y;
    __syncthreads();
    if (threadIdx.x == 0) *dst = (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T, int DK> struct LaBwd {
    using Sh = LaShape<T, DK>;
    static constexpr int SMEM = (int)sizeof(T) * (2 * Sh::QK + 2 * Sh::V + Planes<T>::N * Sh::S);
};

// ------------------------------------------------------------------ dq: forward walk
// Warp = 16 tokens t of the chunk and a quarter of the state.
template <typename T, int DK>
__device__ __forceinline__ void la_dq_walk(const LaDev& p, int64_t block, uint8_t* smem, LaGates* gates, float* red) {
    using Sh = LaShape<T, DK>;
    T* q = reinterpret_cast<T*>(smem);
    T* k = q + Sh::QK;
    T* v = k + Sh::QK;
    T* dout = v + Sh::V;
    T* ss = dout + Sh::V;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rw = (int)(warp + block) & 3;
    const int seg = (int)(block % p.nseg);
    const int64_t vh = block / p.nseg;
    const int sl = (int)(vh % p.nsl), h = (int)(vh / p.nsl % p.H), b = (int)(vh / p.nsl / p.H);
    const int hk = h / (p.H / p.Hk), c0 = sl * LA_DV, cols = min(LA_DV, p.dv - c0), len = la_len(p, b);
    const int first = seg * p.segc, last = min(first + p.segc, p.nc);
    const int64_t bh = (int64_t)b * p.H + h, ssz = (int64_t)p.dk * p.dv, vhead = (int64_t)h * p.nsl + sl;

    float S[Sh::MI][Sh::NI][4];
    la_state_read<T, DK>(S, p.nseg > 1 ? p.seg + (bh * p.nseg + seg) * ssz : (p.s0 ? p.s0 + bh * ssz : nullptr), p, c0, rw, lane);
    const int n = last - first;
    auto chunk = [&](int i) { return first + i; };
    LaGateRing ring;
    ring.start(gates, p, b, h, len, n, chunk, warp, lane);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int t0 = chunk(i) * LA_C, rows = min(LA_C, len - t0);
        __syncthreads();                                     // the last chunk's tiles are done with
        la_load<T, DK, Sh::LDK>(q, p.q, b, t0, hk, 0, rows, p.dk);
        la_load<T, DK, Sh::LDK>(k, p.k, b, t0, hk, 0, rows, p.dk);
        la_load<T, LA_DV, Sh::LDV>(v, p.v, b, t0, h, c0, rows, cols);
        la_load<T, LA_DV, Sh::LDV>(dout, p.dout, b, t0, h, c0, rows, cols);
        cp_async_commit();
        la_state_share<T, DK, Planes<T>::N>(S, ss, rw, lane);
        cp_async_wait<0>();
        __syncthreads();
        const LaGates& gt = ring.take(p, b, h, len, n, i, chunk, warp, lane);
        const int r0 = 16 * rw + (lane >> 2), tr = t0 + 16 * rw;
        float dq[DK / 8][4] = {};
        la_times_state_t<T, DK>(dq, dout, ss, rw, lane);
        const float e0 = gt.pre(r0) * p.scale, e1 = gt.pre(r0 + 8) * p.scale;
#pragma unroll
        for (int j = 0; j < DK / 8; ++j) { dq[j][0] *= e0; dq[j][1] *= e0; dq[j][2] *= e1; dq[j][3] *= e1; }
        const float2 rd = la_row_dot<T, DK>(dq, q, Sh::LDK, rw, lane);
        if ((lane & 3) == 0) {
            float* rin = p.rin + (((int64_t)b * p.H * p.nsl) + vhead) * p.L;
            const int t = t0 + r0;
            if (t < p.L) rin[t] = rd.x;
            if (t + 8 < p.L) rin[t + 8] = rd.y;
        }
        float sc[8][4] = {};
#pragma unroll LA_UNROLL<T>
        for (int k0 = 0; k0 < LA_DV; k0 += 16) {
            FragA<T> a;
            load_a(a, dout, Sh::LDV, 16 * rw, k0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j <= rw) {
                    FragB<T> f[2];
                    load_b2(f, v, Sh::LDV, 16 * j, k0, lane);
                    mma(sc[2 * j], a, f[0]);
                    mma(sc[2 * j + 1], a, f[1]);
                }
        }
        const float2 G0 = gt.G[r0], G1 = gt.G[r0 + 8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j <= rw) {
                la_mask_rows(sc[2 * j], sc[2 * j + 1], gt, j, rw, r0, G0, G1, p.scale, lane);
                FragA<T> a;
                frag_from(a, sc[2 * j], sc[2 * j + 1]);
#pragma unroll
                for (int c = 0; c < DK / 16; ++c) {
                    FragB<T> f[2];
                    load_b2_t(f, k, Sh::LDK, 16 * c, 16 * j, lane);
                    mma(dq[2 * c], a, f[0]);
                    mma(dq[2 * c + 1], a, f[1]);
                }
            }
        la_store_qk<T, DK>(dq, q, p.dq, p, b, hk, vhead, tr, len, rw, lane);
        la_state_update<T, DK, false>(S, k, v, gt, 1.f, rw, lane);
        ring.make(n, i, warp, lane);
    }
    // <state, its gradient> at the segment's end
    la_state_dot<T, DK>(S, p.nseg > 1 ? p.rseg + (bh * p.nseg + seg) * ssz : (p.ds ? p.ds + bh * ssz : nullptr),
                        p.yseg + ((int64_t)b * p.H * p.nsl + vhead) * (p.nseg + 1) + seg + 1, p, c0, rw, lane, red);
}

// ------------------------------------------------------------------ dk, dv, dg: reverse walk
// Warp = 16 tokens s of the chunk and a quarter of the state's gradient.
template <typename T, int DK>
__device__ __forceinline__ void la_dkv_walk(const LaDev& p, int64_t block, uint8_t* smem, LaGates* gates, float (&rowsum)[4][LA_C],
                                            float (&colsum)[LA_C]) {
    using Sh = LaShape<T, DK>;
    T* q = reinterpret_cast<T*>(smem);
    T* k = q + Sh::QK;
    T* v = k + Sh::QK;
    T* dout = v + Sh::V;
    T* ss = dout + Sh::V;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rw = (int)(warp + block) & 3;
    const int seg = (int)(block % p.nseg);
    const int64_t vh = block / p.nseg;
    const int sl = (int)(vh % p.nsl), h = (int)(vh / p.nsl % p.H), b = (int)(vh / p.nsl / p.H);
    const int hk = h / (p.H / p.Hk), c0 = sl * LA_DV, cols = min(LA_DV, p.dv - c0), len = la_len(p, b);
    const int first = seg * p.segc, last = min(first + p.segc, p.nc);
    const int64_t bh = (int64_t)b * p.H + h, ssz = (int64_t)p.dk * p.dv, vhead = (int64_t)h * p.nsl + sl;

    float D[Sh::MI][Sh::NI][4];
    la_state_read<T, DK>(D, p.nseg > 1 ? p.rseg + (bh * p.nseg + seg) * ssz : (p.ds ? p.ds + bh * ssz : nullptr), p, c0, rw, lane);
    float* net = p.net + ((int64_t)b * p.H * p.nsl + vhead) * p.L;
    const int n = last - first;
    auto chunk = [&](int i) { return last - 1 - i; };
    LaGateRing ring;
    ring.start(gates, p, b, h, len, n, chunk, warp, lane);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int t0 = chunk(i) * LA_C, rows = min(LA_C, len - t0);
        __syncthreads();
        la_load<T, DK, Sh::LDK>(q, p.q, b, t0, hk, 0, rows, p.dk);
        la_load<T, DK, Sh::LDK>(k, p.k, b, t0, hk, 0, rows, p.dk);
        la_load<T, LA_DV, Sh::LDV>(v, p.v, b, t0, h, c0, rows, cols);
        la_load<T, LA_DV, Sh::LDV>(dout, p.dout, b, t0, h, c0, rows, cols);
        cp_async_commit();
        la_state_share<T, DK, Planes<T>::N>(D, ss, rw, lane);
        cp_async_wait<0>();
        __syncthreads();
        const LaGates& gt = ring.take(p, b, h, len, n, i, chunk, warp, lane);
        const int r0 = 16 * rw + (lane >> 2), tr = t0 + 16 * rw;
        // the scores of this warp's tokens s (rows) with the tokens t >= s (columns)
        float ps[8][4] = {}, as[8][4] = {};
#pragma unroll LA_UNROLL<T>
        for (int k0 = 0; k0 < DK; k0 += 16) {
            FragA<T> a;
            load_a(a, k, Sh::LDK, 16 * rw, k0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j >= rw) {
                    FragB<T> f[2];
                    load_b2(f, q, Sh::LDK, 16 * j, k0, lane);
                    mma(ps[2 * j], a, f[0]);
                    mma(ps[2 * j + 1], a, f[1]);
                }
        }
#pragma unroll LA_UNROLL<T>
        for (int k0 = 0; k0 < LA_DV; k0 += 16) {
            FragA<T> a;
            load_a(a, v, Sh::LDV, 16 * rw, k0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j >= rw) {
                    FragB<T> f[2];
                    load_b2(f, dout, Sh::LDV, 16 * j, k0, lane);
                    mma(as[2 * j], a, f[0]);
                    mma(as[2 * j + 1], a, f[1]);
                }
        }
        const float2 G0 = gt.G[r0], G1 = gt.G[r0 + 8];
        const float2 Ge = gt.G[16 * rw + 15];
        const float f0 = p.scale * gt.in_block[r0], f1 = p.scale * gt.in_block[r0 + 8];
        float cs0 = 0.f, cs1 = 0.f;                          // sums over t of this lane's two tokens s
        FragA<T> pf[4], af[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j >= rw) {
                float rs[4];                                 // this lane's two tokens s, for tokens t = 2t', 2t'+1, +8, +9
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int tb = 8 * x + 2 * (lane & 3) + e, sb = lane >> 2;     // within the blocks
                        const float2 Gt = gt.G[16 * j + tb];
                        float m0, m1;                        // scale exp(G_t - G_s), split at the end of s's block
                        if (j > rw) {
                            const float d = la_decay(Gt, Ge);
                            m0 = f0 * d;
                            m1 = f1 * d;
                        } else {
                            m0 = tb >= sb ? p.scale * la_decay(Gt, G0) : 0.f;
                            m1 = tb >= sb + 8 ? p.scale * la_decay(Gt, G1) : 0.f;
                        }
                        float p0 = ps[2 * j + x][e], p1 = ps[2 * j + x][2 + e], a0 = as[2 * j + x][e], a1 = as[2 * j + x][2 + e];
                        if (j == rw) {                       // no value of a later token s comes in
                            if (tb < sb) p0 = a0 = 0.f;
                            if (tb < sb + 8) p1 = a1 = 0.f;
                        }
                        a0 *= m0;
                        a1 *= m1;
                        const float x0 = a0 * p0, x1 = a1 * p1;
                        cs0 += x0;
                        cs1 += x1;
                        rs[2 * x + e] = x0 + x1;
                        as[2 * j + x][e] = a0;
                        as[2 * j + x][2 + e] = a1;
                        ps[2 * j + x][e] = p0 * m0;
                        ps[2 * j + x][2 + e] = p1 * m1;
                    }
                // over the 8 lanes that hold the same tokens t: half of the values each time
                const bool up = lane & 16, mid = lane & 8;
                float u0 = up ? rs[2] : rs[0], u1 = up ? rs[3] : rs[1];
                u0 += __shfl_xor_sync(0xffffffffu, up ? rs[0] : rs[2], 16);
                u1 += __shfl_xor_sync(0xffffffffu, up ? rs[1] : rs[3], 16);
                float w = mid ? u1 : u0;
                w += __shfl_xor_sync(0xffffffffu, mid ? u0 : u1, 8);
                w += __shfl_xor_sync(0xffffffffu, w, 4);
                if (!(lane & 4)) rowsum[rw][16 * j + (up ? 8 : 0) + 2 * (lane & 3) + (mid ? 1 : 0)] = w;
            } else if (lane < 16) {
                rowsum[rw][16 * j + lane] = 0.f;
            }
            frag_from(pf[j], ps[2 * j], ps[2 * j + 1]);
            frag_from(af[j], as[2 * j], as[2 * j + 1]);
        }
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
            cs0 += __shfl_xor_sync(0xffffffffu, cs0, o);
            cs1 += __shfl_xor_sync(0xffffffffu, cs1, o);
        }
        const float w0 = gt.post[r0], w1 = gt.post[r0 + 8];
        {
            float dv[8][4] = {};
#pragma unroll LA_UNROLL<T>
            for (int k0 = 0; k0 < DK; k0 += 16) {            // D^T k, D rounded once for a result in T
                FragA<T> a;
                load_a(a, k, Sh::LDK, 16 * rw, k0, lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    FragB<T> f[2];
                    load_b2_t(f, ss, Sh::LDV, 16 * j, k0, lane);
                    mma(dv[2 * j], a, f[0]);
                    mma(dv[2 * j + 1], a, f[1]);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) { dv[j][0] *= w0; dv[j][1] *= w0; dv[j][2] *= w1; dv[j][3] *= w1; }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j >= rw) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        FragB<T> f[2];
                        load_b2_t(f, dout, Sh::LDV, 16 * c, 16 * j, lane);
                        mma(dv[2 * c], pf[j], f[0]);
                        mma(dv[2 * c + 1], pf[j], f[1]);
                    }
                }
            // dk's part from the state reads this warp's rows of v first
            float dk[DK / 8][4] = {};
            la_times_state_t<T, DK>(dk, v, ss, rw, lane);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) store_tile<1>(v, Sh::LDV, 0, 16 * rw, 8 * j, dv[j], lane);
            const int64_t o_sl = (int64_t)p.H * p.dv;
            la_store<T, LA_DV, Sh::LDV>(v + 16 * rw * Sh::LDV, static_cast<T*>(p.dv_out) + ((int64_t)b * p.L + tr) * o_sl + (int64_t)h * p.dv + c0,
                                        o_sl, len - tr, p.L - tr, cols, p.vec_o, lane);
#pragma unroll
            for (int j = 0; j < DK / 8; ++j) { dk[j][0] *= w0; dk[j][1] *= w0; dk[j][2] *= w1; dk[j][3] *= w1; }
            const float2 rd = la_row_dot<T, DK>(dk, k, Sh::LDK, rw, lane);
            if ((lane & 3) == 0) {
                colsum[r0] = cs0 + rd.x;
                colsum[r0 + 8] = cs1 + rd.y;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j >= rw) {
#pragma unroll
                    for (int c = 0; c < DK / 16; ++c) {
                        FragB<T> f[2];
                        load_b2_t(f, q, Sh::LDK, 16 * c, 16 * j, lane);
                        mma(dk[2 * c], af[j], f[0]);
                        mma(dk[2 * c + 1], af[j], f[1]);
                    }
                }
            la_store_qk<T, DK>(dk, k, p.dk_out, p, b, hk, vhead, tr, len, rw, lane);
        }
        la_state_update<T, DK, true>(D, q, dout, gt, p.scale, rw, lane);
        ring.make(n, i, warp, lane);
        __syncthreads();                                     // the token sums are complete
        const int t = threadIdx.x;
        if (t < LA_C && t0 + t < p.L)
            net[t0 + t] = ((rowsum[0][t] + rowsum[1][t]) + (rowsum[2][t] + rowsum[3][t])) - colsum[t];
    }
    if (seg == 0) {
        if (p.ds0) la_state_write<T, DK>(D, p.ds0 + bh * ssz, p, c0, rw, lane);
        __syncthreads();
        la_state_dot<T, DK>(D, p.s0 ? p.s0 + bh * ssz : nullptr, p.yseg + ((int64_t)b * p.H * p.nsl + vhead) * (p.nseg + 1), p, c0, rw, lane,
                            colsum);
    }
}

// ------------------------------------------------------------------ sums over heads that share
// dst[row][hk][c] = sum over the group's parts of src[row][part][c], in order, for dq and dk in one
// launch; thread = VEC values.  A stream over the parts: 16 x 512 tokens x 16 heads of 128 in 23 us, 134 MB, most of it
// still in L2.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) la_group_sum_kernel(const float* src_q, const float* src_k, T* dst_q, T* dst_k, int64_t rows, int Hk,
                                                           int per, int d) {
    const int64_t n = rows * Hk * (d / VEC);
    int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= 2 * n) return;
    const float* src = i < n ? src_q : src_k;
    T* dst = i < n ? dst_q : dst_k;
    i %= n;
    const int c = (int)(i % (d / VEC)) * VEC;
    const int64_t rh = i / (d / VEC);
    const float* s = src + rh * per * d + c;
    float x[VEC] = {};
#pragma unroll 8
    for (int k = 0; k < per; ++k) {
        if constexpr (VEC == 4) {
            const float4 q = *reinterpret_cast<const float4*>(s + (int64_t)k * d);
            x[0] += q.x; x[1] += q.y; x[2] += q.z; x[3] += q.w;
        } else {
            x[0] += s[(int64_t)k * d];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) dst[rh * d + c + j] = Elem<T>::from_f(x[j]);
}

// ------------------------------------------------------------------ dg
// One CTA per segment of one head, from the segment's end: dg_t = <S, D> at the end + the sum of
// q . dq - k . dk over the tokens from t on (fp64), v's slices added up; or, for a decay per
// head, the segment's sum of it.  At the segment's first token the sum has to arrive at <S, D> of its start.  What it
// is off by there, mostly the low bits that the tensor core cuts off, all the same way, is taken out over the
// segment in proportion to the terms' sizes (5 x 1009 x 2 heads, a decay for each head: 3.0e-6 -> 1.1e-6 off; 8 x 2048 x 8
// heads 6.2e-7 -> 4.4e-7; 4 us either way).
constexpr int LG_THREADS = 256;

__global__ void __launch_bounds__(LG_THREADS) la_dg_kernel(const LaDev p) {
    __shared__ double ws[LG_THREADS / 32], wm[LG_THREADS / 32];
    const int seg = blockIdx.x % p.nseg, h = blockIdx.x / p.nseg % p.H, b = blockIdx.x / p.nseg / p.H;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, len = la_len(p, b);
    const int lo = seg * p.segc * LA_C, hi = min(p.L, (seg + 1) * p.segc * LA_C);
    const int64_t v0 = ((int64_t)b * p.H + h) * p.nsl;
    double run = 0., all = 0., start = 0.;
    for (int s = 0; s < p.nsl; ++s) {
        start += (double)p.yseg[(v0 + s) * (p.nseg + 1) + seg];
        run += (double)p.yseg[(v0 + s) * (p.nseg + 1) + seg + 1];
    }
    const float* g = p.g + (int64_t)b * p.g_sb + (int64_t)h * p.g_sh;
    auto term = [&](int t, double& size) {                   // a token's q . dq - k . dk
        double x = 0.;
        size = 0.;
        if (t < lo || t >= len) return x;
        for (int s = 0; s < p.nsl; ++s) {
            const float a = p.rin[(v0 + s) * p.L + t], c = p.net[(v0 + s) * p.L + t];
            x += (double)a + (double)c;
            size += (double)fabsf(a) + (double)fabsf(c);
        }
        return x;
    };
    // what the sum is off by at the segment's start, for each unit of the terms' sizes
    double sum = 0., sizes = 0.;
    for (int t = hi - 1 - (int)threadIdx.x; t >= lo; t -= LG_THREADS) {
        double m;
        sum += term(t, m);
        sizes += m;
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        sizes += __shfl_xor_sync(0xffffffffu, sizes, o);
    }
    if (lane == 0) {
        ws[warp] = sum;
        wm[warp] = sizes;
    }
    __syncthreads();
    sum = sizes = 0.;
    for (int w = 0; w < LG_THREADS / 32; ++w) {
        sum += ws[w];
        sizes += wm[w];
    }
    double off = sizes > 0. ? (run + sum - start) / sizes : 0.;
    if (!(fabs(off) < 1e-3)) off = 0.;                       // not a matter of rounding (values that are not finite)
    for (int t0 = hi; t0 > lo; t0 -= LG_THREADS) {
        const int t = t0 - 1 - (int)threadIdx.x;             // thread 0: the last token
        double m, x = term(t, m);
        const float gt = t >= lo && t < len ? g[(int64_t)t * p.g_sl] : 0.f;
        x -= off * m;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double z = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += z;
        }
        __syncthreads();
        if (lane == 31) ws[warp] = x;
        __syncthreads();
        double before = run;
        for (int w = 0; w < LG_THREADS / 32; ++w) {
            if (w < warp) before += ws[w];
            run += ws[w];
        }
        if (t >= lo) {
            // nothing crosses a reset (a decay of 0): no rounding noise there either
            const float d = t < len && !(gt < -1000.f) ? (float)(before + x) : 0.f;
            if (p.dg) p.dg[((int64_t)b * p.L + t) * p.H + h] = d;
            all += (double)d;
        }
    }
    if (p.dg) return;
#pragma unroll
    for (int o = 16; o > 0; o /= 2) all += __shfl_xor_sync(0xffffffffu, all, o);
    __syncthreads();
    if (lane == 0) ws[warp] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < LG_THREADS / 32; ++w) all += ws[w];
        p.dg_part[((int64_t)h * p.b + b) * p.nseg + seg] = all;
    }
}
__global__ void __launch_bounds__(32) la_dg_head_kernel(const double* part, float* dst, int n) {
    const double* s = part + (int64_t)blockIdx.x * n;
    double x = 0.;
    for (int i = threadIdx.x; i < n; i += 32) x += s[i];
#pragma unroll
    for (int o = 16; o > 0; o /= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (threadIdx.x == 0) dst[blockIdx.x] = (float)x;
}

// Both walks in one launch, the longer ones (dk, dv) first.  Bound by latency and issue (8 x 2048 x 8 heads of 64, bf16:
// 120 us, a warp issues in 40 % of a quarter's cycles, mma.sync busy in 35 %, three warps to a quarter: 64 KB of
// shared memory and 168 registers a thread leave no fourth CTA); of 17 products of 64^3 a chunk, 8 are the second and
// third pieces that keep the states and the decay's gradient to fp32.
template <typename T, int DK>
__global__ void __launch_bounds__(LA_THREADS, sizeof(T) == 4 ? 1 : DK == 128 ? 2 : 3) la_bwd_kernel(const LaDev p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ LaGates gates[LA_RING];
    __shared__ float rowsum[4][LA_C], colsum[LA_C];
    const int64_t half = gridDim.x / 2;
    if (blockIdx.x < half) la_dkv_walk<T, DK>(p, blockIdx.x, smem, gates, rowsum, colsum);
    else la_dq_walk<T, DK>(p, blockIdx.x - half, smem, gates, colsum);
}

template <typename T, int DK>
static cudaError_t bwd(const LaDev& p, cudaStream_t st) {
    constexpr int smem = LaBwd<T, DK>::SMEM;
    auto k = la_bwd_kernel<T, DK>;
    cudaError_t e = allow_smem(k, smem);
    if (e != cudaSuccess) return e;
    k<<<(unsigned)((int64_t)p.b * p.H * p.nsl * p.nseg * 2), LA_THREADS, smem, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    la_dg_kernel<<<(unsigned)(p.b * p.H * p.nseg), LG_THREADS, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t bwd_dk(const LaDev& p, cudaStream_t st) {
    return p.dk <= 32 ? bwd<T, 32>(p, st) : p.dk <= 64 ? bwd<T, 64>(p, st) : bwd<T, 128>(p, st);
}

cudaError_t la_launch_bwd(const LaDev& p, int dtype, cudaStream_t st) {
    return dtype == SWX_DTYPE_F32 ? bwd_dk<float>(p, st) : bwd_dk<__nv_bfloat16>(p, st);
}

cudaError_t la_launch_dg_head(const double* part, float* dst, int H, int n, cudaStream_t st) {
    la_dg_head_kernel<<<(unsigned)H, 32, 0, st>>>(part, dst, n);
    return cudaGetLastError();
}

template <typename T>
static void group_sum(const float* sq, const float* sk, void* dq, void* dk, int64_t rows, int Hk, int per, int d, cudaStream_t st) {
    const int vec = d % 4 == 0 ? 4 : 1;                          // the parts are 256-byte aligned
    const unsigned grid = (unsigned)((2 * rows * Hk * (d / vec) + 255) / 256);
    if (vec == 4) la_group_sum_kernel<T, 4><<<grid, 256, 0, st>>>(sq, sk, static_cast<T*>(dq), static_cast<T*>(dk), rows, Hk, per, d);
    else la_group_sum_kernel<T, 1><<<grid, 256, 0, st>>>(sq, sk, static_cast<T*>(dq), static_cast<T*>(dk), rows, Hk, per, d);
}

cudaError_t la_launch_group_sum(const float* sq, const float* sk, void* dq, void* dk, int dtype, int64_t rows, int Hk, int per, int d,
                                cudaStream_t st) {
    if (dtype == SWX_DTYPE_F32) group_sum<float>(sq, sk, dq, dk, rows, Hk, per, d, st);
    else group_sum<__nv_bfloat16>(sq, sk, dq, dk, rows, Hk, per, d, st);
    return cudaGetLastError();
}

}  // namespace swx
