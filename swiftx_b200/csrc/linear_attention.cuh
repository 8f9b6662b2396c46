// Shared parts of the chunked linear-attention kernels (forward and backward).
//
// For one head, with a_t = exp(g_t) and states S_t (dk x dv):
//   S_t = a_t S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t.
// In a chunk of 64 tokens with G_t = g_1 + .. + g_t and M_ts = exp(G_t - G_s) for s <= t:
//   o_t = scale * (sum_s M_ts (q_t . k_s) v_s + exp(G_t) S_prev^T q_t)
//   S_next = exp(G_64) S_prev + sum_s exp(G_64 - G_s) k_s v_s^T
// The chunk's products run on the tensor cores (warp_mma.cuh); the state stays in fp32
// registers for a whole segment of chunks.  One CTA of four warps walks a segment of one head and
// 64 columns of v; a v of more than 64 columns is treated as several heads that share q, k and g.
#pragma once
#include <cuda_runtime.h>

#include "common.cuh"
#include "warp_mma.cuh"

namespace swx {

constexpr int LA_C = 64;                  // tokens per chunk
constexpr int LA_DV = 64;                 // columns of v per CTA
constexpr int LA_THREADS = 128;
constexpr uint32_t LT_POLLS = 1u << 16;   // tries of the pipelined kernels' waits, up to 20 us each
// How far the loops over a product's contraction are unrolled: whole loops made the two gradient walks larger than
// the instruction caches (fp32 133 -> 110 us at 2 x 777 x 6 heads; bf16, shorter, the same either way).
template <typename T> constexpr int LA_UNROLL = sizeof(T) == 4 ? 1 : 2;

struct LaTensor { const void* p; int64_t sb, sl, sh; bool vec; };

struct LaDev {
    int b, L, H, Hk, dk, dv, nsl;         // nsl: slices of 64 columns of v
    int nc, nseg, segc;                   // chunks; segments; chunks per segment (even)
    bool tc;                              // the pipelined kernels, where the tensors allow it
    uint32_t polls;                       // tries of each of their waits
    LaTensor q, k, v, dout;
    const float* g; int64_t g_sb, g_sl, g_sh;
    const int64_t* lengths;
    float scale;
    const float* s0;                      // (b, H, dk, dv) or null: zero
    void* out;                            // (b, L, H, dv)
    float* s_last;                        // (b, H, dk, dv) or null
    float* seg;                           // (b, H, nseg, dk, dv): the state at each segment's start
    float* save;                          // the forward for the backward: (b, H, save_n, dk, dv), the state at
    int save_n, save_c;                   // each save_c-th chunk's start, or null
    float* rseg;                          // the same for the reverse pass: its gradient at each segment's end
    float* dec;                           // (b, H, nseg): each segment's decay
    // backward
    const float* ds;                      // gradient of the last state, or null
    float* ds0;                           // gradient of the initial state, or null
    void* dq; void* dk_out; void* dv_out; // dq, dk: (b, L, Hk, dk) in T, or (b, L, H nsl, dk) fp32 when several share
    bool shared_qk;
    float* rin;                           // (b, H nsl, L): the states' part of q . dq
    float* net;                           // (b, H nsl, L): the scores' part of q . dq, less k . dk
    float* yseg;                          // (b, H nsl, nseg + 1): <state, its gradient> at the start and at each segment's end
    float* dg;                            // (b, L, H), or null:
    double* dg_part;                      // (H, b nseg): each segment's sum
    bool vec_o, vec_qk;                   // 16-byte pieces of v-shaped (q-shaped) results are aligned and whole
};

template <typename T, int DK>
struct LaShape {
    static constexpr int LDK = (DK < 64 ? 64 : DK) + 16 / (int)sizeof(T) * (sizeof(T) == 4 ? 2 : 1);   // rows of q, k
    static constexpr int LDV = LA_DV + 8;                                                              // rows of v, do, S
    static constexpr int QK = LA_C * LDK, V = LA_C * LDV, S = DK * LDV;                                // elements
    // how the four warps share a (dk x 64) state: WM row groups x WN column groups
    static constexpr int MT = DK / 16, WM = MT < 4 ? MT : 4, WN = 4 / WM, MI = MT / WM, NI = 8 / WN;
};

// Per-chunk decays.  Sums of g are in fp64 and kept as two floats (in units of log 2), so
// that differences of far sums keep their precision; g below -1000 (or -inf: a reset) is
// taken as -1000, whose exponential is 0 as well.
struct LaGates {
    float2 G[LA_C];                       // G_t, high and low part
    float post[LA_C];                     // exp(G_64 - G_t)
    float in_block[LA_C];                 // exp(G_e - G_t), e the last token of t's block of 16
    float all;                            // exp(G_64)
    float unused[3];
    __device__ __forceinline__ float pre(int t) const { return ex2(G[t].x); }      // exp(G_t)
};
// exp(G_a - G_b) from the two-float sums
__device__ __forceinline__ float la_decay(float2 a, float2 b) { return ex2((a.x - b.x) + (a.y - b.y)); }

// The gates of a walk of n chunks, made for four chunks at a time, one chunk by each warp: their
// scan is a chain of a thousand cycles that would otherwise hold all warps up in every chunk.  The
// next four are made in the last step of the present four, whose own gates are the ring's fifth.
// take() after the barrier that starts step i, make() before the barrier that starts step i + 1.
struct LaG { float g0, g1; };
constexpr int LA_RING = 5;

__device__ __forceinline__ LaG la_load_g(const LaDev& p, int b, int h, int t0, int len, int lane) {
    const float* g = p.g + (int64_t)b * p.g_sb + (int64_t)h * p.g_sh;
    const int t = t0 + 2 * lane;
    LaG r{0.f, 0.f};
    if (t < len) r.g0 = g[(int64_t)t * p.g_sl];
    if (t + 1 < len) r.g1 = g[(int64_t)(t + 1) * p.g_sl];
    return r;
}

// One warp; lane holds tokens 2 lane, 2 lane + 1.  Returns the chunk's sum (log 2 units).
static __device__ __noinline__ double la_gates(LaGates& s, LaG r, int lane) {
    const double L2E = 1.4426950408889634073599;
    const double d0 = (r.g0 < -1000.f ? -1000. : (double)r.g0) * L2E, d1 = (r.g1 < -1000.f ? -1000. : (double)r.g1) * L2E;
    double x = d0 + d1;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    const double all = __shfl_sync(0xffffffffu, x, 31), g1 = x, g0 = x - d1;
    const int t = 2 * lane;
    const double ge = __shfl_sync(0xffffffffu, x, lane | 7);
    s.G[t] = make_float2((float)g0, (float)(g0 - (double)(float)g0));
    s.G[t + 1] = make_float2((float)g1, (float)(g1 - (double)(float)g1));
    s.post[t] = ex2((float)(all - g0)); s.post[t + 1] = ex2((float)(all - g1));
    s.in_block[t] = ex2((float)(ge - g0)); s.in_block[t + 1] = ex2((float)(ge - g1));
    if (lane == 0) s.all = ex2((float)all);
    return all;
}

struct LaGateRing {
    LaGates* s;
    LaG g;
    double total;                         // this warp's chunks (log 2 units)
    template <typename F>
    __device__ __forceinline__ void start(LaGates* slots, const LaDev& p, int b, int h, int len, int n, F chunk, int warp, int lane) {
        s = slots;
        total = 0.;
        if (warp < n) total += la_gates(s[warp], la_load_g(p, b, h, chunk(warp) * LA_C, len, lane), lane);
    }
    template <typename F>
    __device__ __forceinline__ const LaGates& take(const LaDev& p, int b, int h, int len, int n, int i, F chunk, int warp, int lane) {
        if ((i & 3) == 3 && i + 1 + warp < n) g = la_load_g(p, b, h, chunk(i + 1 + warp) * LA_C, len, lane);
        return s[i % LA_RING];
    }
    __device__ __forceinline__ void make(int n, int i, int warp, int lane) {
        if ((i & 3) == 3 && i + 1 + warp < n) total += la_gates(s[(i + 1 + warp) % LA_RING], g, lane);
    }
};

// Scores of the rows r0, r0 + 8 of block rw (G0, G1 their sums) with the 16 tokens of block j:
// times scale exp(G_t - G_s), 0 for s > t.  Off the diagonal the exponential is split at the
// end of block j, exp(G_t - G_e) exp(G_e - G_s), both at most 1 for decays at most 1: two products
// a value instead of a difference and an exponential.
__device__ __forceinline__ void la_mask_rows(float (&c0)[4], float (&c1)[4], const LaGates& gt, int j, int rw, int r0, float2 G0,
                                             float2 G1, float scale, int lane) {
    const int s0 = 16 * j + 2 * (lane & 3);
    if (j < rw) {
        const float2 Ge = gt.G[16 * j + 15];
        const float f0 = scale * la_decay(G0, Ge), f1 = scale * la_decay(G1, Ge);
        const float2 x = *reinterpret_cast<const float2*>(gt.in_block + s0), y = *reinterpret_cast<const float2*>(gt.in_block + s0 + 8);
        c0[0] *= f0 * x.x; c0[1] *= f0 * x.y; c0[2] *= f1 * x.x; c0[3] *= f1 * x.y;
        c1[0] *= f0 * y.x; c1[1] *= f0 * y.y; c1[2] *= f1 * y.x; c1[3] *= f1 * y.y;
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 a = gt.G[s0 + e], b = gt.G[s0 + 8 + e];
            c0[e] = s0 + e <= r0 ? c0[e] * (scale * la_decay(G0, a)) : 0.f;
            c0[2 + e] *= scale * la_decay(G1, a);
            c1[e] = 0.f;
            c1[2 + e] = s0 + e <= r0 ? c1[2 + e] * (scale * la_decay(G1, b)) : 0.f;
        }
    }
}

// Paths that aligned tensors do not take stay out of line: the walks' code has to fit the instruction caches.
template <typename T>
__device__ __noinline__ void la_load_scalar(T* s, int ld, int width, const T* g, int64_t sl, int rows, int cols) {
    for (int i = threadIdx.x; i < LA_C * width; i += LA_THREADS) {
        const int r = i / width, c = i % width;
        s[r * ld + c] = r < rows && c < cols ? g[(int64_t)r * sl + c] : T(0.f);
    }
}
template <typename T>
__device__ __noinline__ void la_store_scalar(const T* s, int ld, T* g, int64_t sl, int rows, int all_rows, int cols, int lane) {
    const int n = 16 * cols;
    for (int i = lane; i < n; i += 32) {
        const int r = i / cols, c = i % cols;
        if (r < all_rows) g[(int64_t)r * sl + c] = r < rows ? s[r * ld + c] : T(0.f);
    }
}

// 64 token rows x W columns into s (row length LD), zero past rows / cols; asynchronous when vec.
template <typename T, int W, int LD>
__device__ __forceinline__ void la_load(T* s, const LaTensor& x, int b, int t0, int h, int c0, int rows, int cols) {
    const T* g = static_cast<const T*>(x.p) + (int64_t)b * x.sb + (int64_t)t0 * x.sl + (int64_t)h * x.sh + c0;
    if (x.vec) {
        // this thread's column and rows r, r + STEP, ..
        constexpr int E = 16 / sizeof(T), PER = W / E, STEP = LA_THREADS / PER;
        const int r = threadIdx.x / PER, c = (threadIdx.x % PER) * E;
        const int n = min(E, max(0, cols - c)) * (int)sizeof(T);
        const T* src = g + (int64_t)r * x.sl + c;
        const int64_t step = STEP * x.sl;
        T* dst = s + r * LD + c;
#pragma unroll
        for (int i = 0; i < LA_C / STEP; ++i) {
            const bool in = r + i * STEP < rows && n > 0;
            cp_async16(dst + i * STEP * LD, in ? src + i * step : static_cast<const T*>(x.p), in ? n : 0);
        }
    } else {
        la_load_scalar(s, LD, W, g, x.sl, rows, cols);
    }
}

// (dk x dv slice) fp32 matrices in memory <-> the accumulator tiles of a state.
template <typename T, int DK>
__device__ __forceinline__ void la_state_read(float (&S)[LaShape<T, DK>::MI][LaShape<T, DK>::NI][4], const float* src,
                                              const LaDev& p, int c0, int rw, int lane) {
    using Sh = LaShape<T, DK>;
    const int m0 = (rw % Sh::WM) * Sh::MI * 16, n0 = (rw / Sh::WM) * Sh::NI * 8;
#pragma unroll
    for (int i = 0; i < Sh::MI; ++i)
#pragma unroll
        for (int j = 0; j < Sh::NI; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = m0 + 16 * i + (lane >> 2) + 8 * (e >> 1), c = n0 + 8 * j + 2 * (lane & 3) + (e & 1);
                S[i][j][e] = src && r < p.dk && c0 + c < p.dv ? src[(int64_t)r * p.dv + c0 + c] : 0.f;
            }
}
template <typename T, int DK>
__device__ __forceinline__ void la_state_write(const float (&S)[LaShape<T, DK>::MI][LaShape<T, DK>::NI][4], float* dst,
                                               const LaDev& p, int c0, int rw, int lane) {
    using Sh = LaShape<T, DK>;
    const int m0 = (rw % Sh::WM) * Sh::MI * 16, n0 = (rw / Sh::WM) * Sh::NI * 8;
#pragma unroll
    for (int i = 0; i < Sh::MI; ++i)
#pragma unroll
        for (int j = 0; j < Sh::NI; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = m0 + 16 * i + (lane >> 2) + 8 * (e >> 1), c = n0 + 8 * j + 2 * (lane & 3) + (e & 1);
                if (r < p.dk && c0 + c < p.dv) dst[(int64_t)r * p.dv + c0 + c] = S[i][j][e];
            }
}

// S = exp(G_64) S + sum over the chunk's tokens of (w_s x_s) y_s^T, w_s = exp(G_64 - G_s) or (PRE)
// scale exp(G_s).  The weighted x is kept to 24
// bits, so that the state, which is carried through the whole sequence, keeps fp32 accuracy.
// The chunk's own sum (bf16: its small pieces apart) is added to the state in fp32.  The tensor core cuts the low
// bits of each addition off, all the same way; with the state itself as the accumulator its 12 additions a chunk left a
// decay gradient for each head 2.1e-6 off where it is 0.7e-6 now (16 x 512 x 16 heads, dk 128; 294 -> 304 us), and fp32's 8
// a state after 4096 tokens without decay 8.4e-5 off, 1.1e-6 now (200 heads; 2 x 777 x 6 heads forward and backward 150 -> 154 us).
template <typename T, int DK, bool PRE>
__device__ __forceinline__ void la_state_update(float (&S)[LaShape<T, DK>::MI][LaShape<T, DK>::NI][4], const T* xs, const T* ys,
                                                const LaGates& gt, float scale, int rw, int lane) {
    using Sh = LaShape<T, DK>;
    const int m0 = (rw % Sh::WM) * Sh::MI * 16, n0 = (rw / Sh::WM) * Sh::NI * 8;
    auto weights = [&](float (&w4)[4], int k0) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int s = k0 + 2 * (lane & 3) + (x & 1) + (x >> 1) * 8;
            w4[x] = PRE ? scale * gt.pre(s) : gt.post[s];
        }
    };
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < Sh::MI; ++i) {
            float u[Sh::NI][4] = {}, lo[Sh::NI][4] = {};
#pragma unroll LA_UNROLL<T>
            for (int k0 = 0; k0 < LA_C; k0 += 16) {
                float w4[4];
                weights(w4, k0);
                FragA<T> a;
                load_a_t(a, xs, Sh::LDK, m0 + 16 * i, k0, lane);
                ScaledA<T> s;
                scale_a(s, a, w4);
#pragma unroll
                for (int j = 0; j < Sh::NI / 2; ++j) {
                    FragB<T> y[2];
                    load_b2_t(y, ys, Sh::LDV, n0 + 16 * j, k0, lane);
#pragma unroll
                    for (int q = 2; q >= 0; --q)
#pragma unroll
                        for (int x = 0; x < 2; ++x) mma_bf16(q > 0 ? lo[2 * j + x] : u[2 * j + x], s.p[q].r, y[x].r);
                }
            }
#pragma unroll
            for (int j = 0; j < Sh::NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[i][j][e] = fmaf(gt.all, S[i][j][e], u[j][e] + lo[j][e]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < Sh::MI; ++i) {
            float u[Sh::NI][4] = {};
#pragma unroll LA_UNROLL<T>
            for (int k0 = 0; k0 < LA_C; k0 += 16) {
                float w4[4];
                weights(w4, k0);
                FragA<T> a;
                load_a_t(a, xs, Sh::LDK, m0 + 16 * i, k0, lane);
                ScaledA<T> s;
                scale_a(s, a, w4);
#pragma unroll
                for (int j = 0; j < Sh::NI / 2; ++j) {
                    FragB<T> y[2];
                    load_b2_t(y, ys, Sh::LDV, n0 + 16 * j, k0, lane);
                    mma(u[2 * j], s.p, y[0]);
                    mma(u[2 * j + 1], s.p, y[1]);
                }
            }
#pragma unroll
            for (int j = 0; j < Sh::NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[i][j][e] = fmaf(gt.all, S[i][j][e], u[j][e]);
        }
    }
}

// The state before chunk c, kept for the backward's segment that starts there.
template <typename T, int DK>
__device__ __forceinline__ void la_state_save(const float (&S)[LaShape<T, DK>::MI][LaShape<T, DK>::NI][4], const LaDev& p, int64_t bh, int c,
                                              int c0, int rw, int lane) {
    if (p.save && c % p.save_c == 0)
        la_state_write<T, DK>(S, p.save + (bh * p.save_n + c / p.save_c) * p.dk * p.dv, p, c0, rw, lane);
}

template <typename T, int DK, int PLANES>
__device__ __forceinline__ void la_state_share(const float (&S)[LaShape<T, DK>::MI][LaShape<T, DK>::NI][4], T* s, int rw, int lane) {
    using Sh = LaShape<T, DK>;
    const int m0 = (rw % Sh::WM) * Sh::MI * 16, n0 = (rw / Sh::WM) * Sh::NI * 8;
#pragma unroll
    for (int i = 0; i < Sh::MI; ++i)
#pragma unroll
        for (int j = 0; j < Sh::NI; ++j) store_tile<PLANES>(s, Sh::LDV, Sh::S, m0 + 16 * i, n0 + 8 * j, S[i][j], lane);
}

// A warp's 16 finished rows, gathered in its own rows of a tile, to memory: `rows` live ones (later
// rows up to `all_rows` get zeros), `cols` columns.
template <typename T, int W, int LD>
__device__ __forceinline__ void la_store(const T* s, T* g, int64_t sl, int rows, int all_rows, int cols, bool vec, int lane) {
    __syncwarp();
    if (vec) {
        constexpr int E = 16 / sizeof(T), PER = W / E;
#pragma unroll
        for (int i = lane; i < 16 * PER; i += 32) {
            const int r = i / PER, c = (i % PER) * E;
            if (r < all_rows && c < cols) {
                const uint4 z = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(g + (int64_t)r * sl + c) = r < rows ? *reinterpret_cast<const uint4*>(s + r * LD + c) : z;
            }
        }
    } else {
        la_store_scalar(s, LD, g, sl, rows, all_rows, cols, lane);
    }
    __syncwarp();
}

// Tokens t0 .. t1 - 1 of one head's output columns: zeros, by `threads` threads of which this is `tid`.
template <typename T>
__device__ __forceinline__ void la_zero_rows(const LaDev& p, int b, int h, int c0, int cols, int t0, int t1, int tid, int threads) {
    const int64_t sl = (int64_t)p.H * p.dv;
    T* out = static_cast<T*>(p.out) + ((int64_t)b * p.L + t0) * sl + (int64_t)h * p.dv + c0;
    if (p.vec_o) {
        constexpr int E = 16 / sizeof(T);
        const int per = cols / E;
        for (int i = tid; i < (t1 - t0) * per; i += threads)
            *reinterpret_cast<uint4*>(out + (int64_t)(i / per) * sl + i % per * E) = make_uint4(0, 0, 0, 0);
    } else {
        for (int i = tid; i < (t1 - t0) * cols; i += threads) out[(int64_t)(i / cols) * sl + i % cols] = T(0.f);
    }
}

__device__ __forceinline__ int la_len(const LaDev& p, int b) {
    if (!p.lengths) return p.L;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : (n < p.L ? (int)n : p.L);
}

// linear_attention_tc.cu, bf16: *taken says whether it ran
cudaError_t lt_launch_fwd(const LaDev& p, bool* taken, cudaStream_t st);
cudaError_t lt_launch_state(const LaDev& p, bool reverse, bool* taken, cudaStream_t st);
cudaError_t la_launch_fwd(const LaDev& p, int dtype, cudaStream_t st);
cudaError_t la_launch_bwd(const LaDev& p, int dtype, cudaStream_t st);
cudaError_t la_launch_state(const LaDev& p, int dtype, bool reverse, cudaStream_t st);
cudaError_t la_launch_dg_head(const double* part, float* dst, int H, int n, cudaStream_t st);
cudaError_t la_launch_group_sum(const float* sq, const float* sk, void* dq, void* dk, int dtype, int64_t rows, int Hk, int per, int d,
                                cudaStream_t st);

}  // namespace swx
