// Log probabilities of given tokens under a linear head, with the entropy and the top alternatives, without keeping
// the logits:  z = x W^T,  l_v = z_v / tau - log sum exp(z / tau),  p = e^l,
//   log_probs = l_y,  entropy = -sum p l,  top: the K largest z (the lowest word first among equals).
// Backward, for upstream gradients g of log_probs and h of the entropy H:
//   dz_v = (g [v == y] - p_v (g + h (l_v + H))) / tau,  dx = dz W,  dW = dz^T x.
//
// Forward: the head's product (head_gemm.cuh) with an epilogue that keeps three floats for each half of a 256-column tile: the
// maximum m, s = sum e and w = sum e u of e = 2^u, u = (z - m) log2(e) / tau; with alternatives also the three largest logits of every
// 32 columns (12 bytes), or, for a small vocabulary, the logits.  Then one kernel for the rows: the statistics joined, and
//   H = ln s - ln2 w / s.
// Alternatives: the K + 8 groups of 32 columns with the largest maxima hold the K + 8 largest logits; a group whose second value
// passes too gives two, one whose third does is taken whole.  The tensor core's sums are a few 2^-23 off and the records hold 18
// bits, enough to turn two close logits round, so the candidates' products are formed again from the operands: in
// fp32, with a bound of the error, and those that the bound does not tell apart from another exactly.
//
// Backward: as the loss's, with dz in the epilogue (rounded to bf16 once, the tensor core's operand; fp32 operands: three pieces).
#include "head_gemm.cuh"
#include "topk.cuh"

namespace swx {

constexpr int SC_EXTRA = 8;                   // candidates beyond K
constexpr int SC_THREADS = 256, SC_PER = 8;
constexpr float LN2 = 0.69314718055994531f;

struct ScoreRows {
    int64_t T, V, d;
    int np;                                   // statistics per row
    const float4* score; const float* hit; const int64_t* target; int64_t ignore;
    float k2, inv_temp;
    float* row_max; float* row_sum; float* log_probs; float* entropy;
    // alternatives
    int top, cand;                            // K, candidates kept of the records
    const float2* rec; const float* third; const float* all; int64_t groups;
    const void* x; int64_t x_sr; const void* w; int64_t w_sr; int vec;
    float* top_log_probs; int64_t* top_ids;
};

// A row's results from its statistics.
__device__ __forceinline__ void score_finish(const ScoreRows& p, int64_t row, const Score& a) {
    const int64_t y = p.target[row];
    const float ls = logf(a.s);
    if (p.row_max) { p.row_max[row] = a.m; p.row_sum[row] = a.s; }
    const bool live = y != p.ignore;
    p.log_probs[row] = !live ? 0.f : y >= 0 && y < p.V ? (p.hit[row] - a.m) * p.inv_temp - ls : __int_as_float(0x7fc00000);
    p.entropy[row] = live ? ls - LN2 * a.w / a.s : 0.f;
}

// Warp = one row.
__global__ void __launch_bounds__(SC_THREADS) score_rows_kernel(const ScoreRows p) {
    const int64_t row = (int64_t)blockIdx.x * (SC_THREADS / 32) + threadIdx.x / 32;
    if (row >= p.T) return;
    const int lane = threadIdx.x % 32;
    Score a{-INFINITY, 0.f, 0.f};
    for (int i = lane; i < p.np; i += 32) {
        const float4 q = p.score[row * p.np + i];
        score_join(a, Score{q.x, q.y, q.z}, p.k2, SCORE_FAR);
    }
    score_join_warp(a, p.k2, SCORE_FAR);
    if (lane == 0) score_finish(p, row, a);
}

__device__ __forceinline__ float2 bf16_pair(uint32_t q) { return f2(__uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u)); }

// A 16-byte load's values in pairs.
__device__ __forceinline__ void unpack(const float*, const uint4& q, float2 (&v)[2]) {
    v[0] = f2(__uint_as_float(q.x), __uint_as_float(q.y));
    v[1] = f2(__uint_as_float(q.z), __uint_as_float(q.w));
}
__device__ __forceinline__ void unpack(const __nv_bfloat16*, const uint4& q, float2 (&v)[4]) {
    v[0] = bf16_pair(q.x); v[1] = bf16_pair(q.y); v[2] = bf16_pair(q.z); v[3] = bf16_pair(q.w);
}

// Products of a row of x with two rows of the weight over a warp, in fp32: z, and a bound of each one's error.  A lane sums d / 64
// products in each of two chains, which are joined in six steps, 2^-24 of the magnitudes each; |x| |w| bounds those.
struct Product2 { float z[2], e[2]; };
template <typename T>
__device__ __forceinline__ Product2 product2(const T* x, const T* w0, const T* w1, int64_t d, bool vec, int lane) {
    constexpr int N = 16 / sizeof(T);
    float2 a[2] = {}, n[3] = {};
    int64_t tail = 0;
    if (vec) {
#pragma unroll 4
        for (int64_t k = lane * N; k + N <= d; k += 32 * N) {
            float2 xv[N / 2], v0[N / 2], v1[N / 2];
            unpack(x, *reinterpret_cast<const uint4*>(x + k), xv);
            unpack(x, *reinterpret_cast<const uint4*>(w0 + k), v0);
            unpack(x, *reinterpret_cast<const uint4*>(w1 + k), v1);
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                a[0] = fma2(xv[j], v0[j], a[0]);
                a[1] = fma2(xv[j], v1[j], a[1]);
                n[0] = fma2(v0[j], v0[j], n[0]);
                n[1] = fma2(v1[j], v1[j], n[1]);
                n[2] = fma2(xv[j], xv[j], n[2]);
            }
        }
        tail = d / N * N;
    }
    for (int64_t k = tail + lane; k < d; k += 32) {
        const float xv = Elem<T>::to_f(x[k]), v0 = Elem<T>::to_f(w0[k]), v1 = Elem<T>::to_f(w1[k]);
        a[0].x = fmaf(xv, v0, a[0].x);
        a[1].x = fmaf(xv, v1, a[1].x);
        n[0].x = fmaf(v0, v0, n[0].x);
        n[1].x = fmaf(v1, v1, n[1].x);
        n[2].x = fmaf(xv, xv, n[2].x);
    }
    float r[5] = {a[0].x + a[0].y, a[1].x + a[1].y, n[0].x + n[0].y, n[1].x + n[1].y, n[2].x + n[2].y};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < 5; ++j) r[j] += __shfl_xor_sync(0xffffffffu, r[j], o);
    const float f = ((vec ? d * (1.f / 64) : d * (1.f / 32)) + 16.f) * 0x1p-24f * 1.01f;
    const float xn = f * sqrtf(fmaxf(r[4], 0x1p-100f));       // (smaller squares may have underflowed)
    return Product2{{r[0], r[1]}, {xn * sqrtf(fmaxf(r[2], 0x1p-100f)), xn * sqrtf(fmaxf(r[3], 0x1p-100f))}};
}

// The same product of one row of the weight, exact but for fp64's rounding (2^-53).
template <typename T>
__device__ __forceinline__ double product_exact(const T* x, const T* w, int64_t d, int lane) {
    double a = 0.;
    for (int64_t k = lane; k < d; k += 32) a = fma((double)Elem<T>::to_f(x[k]), (double)Elem<T>::to_f(w[k]), a);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}

static int score_candidates(bool all, int cand) { return all ? cand : 32 * cand; }

static size_t score_top_smem(bool all, int cand) {
    return (size_t)topk_capacity(cand, SC_PER) * 8 + cand * 8 + (size_t)score_candidates(all, cand) * 12;
}

__device__ __forceinline__ float drop_column(float v) { return __uint_as_float(__float_as_uint(v) & ~31u); }

// CTA = one row: its statistics, the candidates from the records (ALL: from the logits), their products, their ranks.
// THREADS is at least the number of candidates.
template <typename T, bool ALL, int THREADS>
__global__ void __launch_bounds__(THREADS) score_top_kernel(const ScoreRows p) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ int count, ncand, owners[THREADS];
    __shared__ uint32_t scratch[THREADS + 1], error;                 // error: the largest of the candidates' bounds, its bits
    __shared__ Score part[THREADS / 32];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint64_t* buf = reinterpret_cast<uint64_t*>(raw);
    uint64_t* kept = buf + topk_capacity(p.cand, SC_PER);
    double* val = reinterpret_cast<double*>(kept + p.cand);          // candidates' products
    int* col = reinterpret_cast<int*>(val + (ALL ? p.cand : 32 * p.cand));

    // the largest of this thread's share of the values: logits (a NaN as -inf), or the records' first ones without their columns
    const int64_t n = ALL ? p.V : p.groups;
    const float2* rec = p.rec + row * p.groups;
    const float* all = p.all + row * p.V;
    auto value = [&](int64_t i) { const float z = ALL ? all[i] : drop_column(rec[i].x); return ALL && z != z ? -INFINITY : z; };
    float most = -INFINITY;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += THREADS) most = fmaxf(most, value(i));
    Score a{-INFINITY, 0.f, 0.f};
    for (int i = threadIdx.x; i < p.np; i += THREADS) {
        const float4 q = p.score[row * p.np + i];
        score_join(a, Score{q.x, q.y, q.z}, p.k2, SCORE_FAR);
    }
    score_join_warp(a, p.k2, SCORE_FAR);
    if (lane == 0) part[warp] = a;
    if (threadIdx.x == 0) { ncand = 0; error = 0; }
    __syncthreads();
    a = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) score_join(a, part[i], p.k2, SCORE_FAR);
    if (threadIdx.x == 0) score_finish(p, row, a);
    if (p.target[row] == p.ignore) {                                 // a token that does not count
        for (int i = threadIdx.x; i < p.top; i += THREADS) {
            p.top_log_probs[row * p.top + i] = 0.f;
            p.top_ids[row * p.top + i] = -1;
        }
        return;
    }

    TopK<THREADS, SC_PER> best{};
    best.start(buf, kept, &count, p.cand);
    auto item = [&](int t, int64_t j, auto f) {
        const int64_t i = t + j * THREADS;
        if (i < n) f(value(i), (uint32_t)i);
    };
    if (!best.gather(threadIdx.x < n ? order_key(most) : 0, scratch, owners, (n + THREADS - 1) / THREADS, item)) {
        best.clear();
        for (int64_t i0 = 0; i0 < n; i0 += THREADS * SC_PER) {
            uint64_t key[SC_PER];
#pragma unroll
            for (int j = 0; j < SC_PER; ++j) {
                const int64_t i = i0 + j * THREADS + threadIdx.x;
                key[j] = i < n ? index_key(order_key(value(i)), (uint32_t)i) : 0;
            }
            best.push(key);
        }
    }
    best.rank();
    // the columns of the candidates
    const int m = best.n;
    if (ALL) {
        for (int i = threadIdx.x; i < m; i += THREADS) col[i] = (int)key_index(buf[i]);
        if (threadIdx.x == 0) ncand = m;
    } else {
        const float least = order_value((uint32_t)(buf[m - 1] >> 32));
        for (int i = threadIdx.x; i < m; i += THREADS) {
            const int g = (int)key_index(buf[i]);
            const float2 r = rec[g];
            const bool two = drop_column(r.y) >= least;
            if (two && drop_column(p.third[row * p.groups + g]) >= least) {
                const int c = (int)min((int64_t)32, p.V - (int64_t)g * 32), at = atomicAdd(&ncand, c);
                for (int j = 0; j < c; ++j) col[at + j] = g * 32 + j;
            } else {
                const int at = atomicAdd(&ncand, two ? 2 : 1);
                col[at] = g * 32 + (int)(__float_as_uint(r.x) & 31u);
                if (two) col[at + 1] = g * 32 + (int)(__float_as_uint(r.y) & 31u);
            }
        }
    }
    __syncthreads();
    const int nc = ncand;
    const T* x = static_cast<const T*>(p.x) + row * p.x_sr;
    const T* w = static_cast<const T*>(p.w);
    for (int i = 2 * warp; i < nc; i += 2 * (THREADS / 32)) {
        const int i1 = min(i + 1, nc - 1);
        const Product2 z = product2<T>(x, w + col[i] * p.w_sr, w + col[i1] * p.w_sr, p.d, p.vec, lane);
        if (lane == 0) {
            val[i] = z.z[0];
            if (i1 > i) val[i1] = z.z[1];
            const float e = fmaxf(z.e[0], z.e[1]);
            atomicMax(&error, e == e && z.e[0] + z.e[1] == z.e[0] + z.e[1] ? __float_as_uint(e) : 0x7f800000u);
        }
    }
    __syncthreads();
    // candidates that the bound does not tell apart from another, marked by the sign of their column
    const double apart = 2. * __uint_as_float(error);
    for (int i = threadIdx.x; i < nc; i += THREADS) {
        bool close = false;
        for (int j = 0; j < nc; ++j) close |= j != i && !(fabs(val[j] - val[i]) > apart);
        if (close) col[i] = ~col[i];
    }
    __syncthreads();
    for (int i = warp; i < nc; i += THREADS / 32) {
        const int c = col[i];
        if (c >= 0) continue;
        const double z = product_exact<T>(x, w + (int64_t)~c * p.w_sr, p.d, lane);
        if (lane == 0) { val[i] = z; col[i] = ~c; }
    }
    __syncthreads();
    const double lse = (double)a.m * p.inv_temp + log((double)a.s);
    for (int i = threadIdx.x; i < nc; i += THREADS) {
        const double z = val[i];
        const uint64_t v = order_key(z);
        const int c = col[i];
        int r = 0;
        for (int j = 0; j < nc; ++j) {
            const uint64_t o = order_key(val[j]);
            r += o > v || (o == v && col[j] < c);
        }
        if (r < p.top) {
            p.top_log_probs[row * p.top + r] = (float)(z * p.inv_temp - lse);
            p.top_ids[row * p.top + r] = c;
        }
    }
}

// ------------------------------------------------------------------ host side
cudaError_t launch_score(const XentGemm& g, const CUtensorMap& x, const CUtensorMap& w, cudaStream_t st) {
    return launch_logits<XE_SCORE>(g, x, w, x, st);
}
cudaError_t launch_grad(const XentGemm& g, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& store, cudaStream_t st) {
    return launch_logits<XE_GRAD>(g, x, w, store, st);
}

struct ScorePlan {
    int cand; bool all; int64_t groups;
    int64_t off_score, off_hit, off_rec, off_third, total;
};

static ScorePlan score_plan(const HeadPlan& q, int64_t T, int64_t V, int top) {
    ScorePlan f{};
    f.off_score = q.base;
    f.off_hit = f.off_score + up256(2 * q.nt * T * 16);
    f.off_rec = f.off_hit + up256(T * 4);
    f.total = f.off_rec;
    if (top > 0) {
        f.cand = (int)std::min<int64_t>(V, top + SC_EXTRA);
        f.groups = (V + 31) / 32;
        // few groups for each candidate: most would be taken whole, or there are not enough of them
        f.all = V <= 2048 || f.groups < 2 * f.cand;
        f.off_third = f.off_rec + up256(f.all ? T * V * 4 : T * f.groups * 8);
        f.total = f.off_third + (f.all ? 0 : up256(T * f.groups * 4));
    }
    return f;
}

static HeadOps ops_of(const swx_logprob_args* a) {
    return HeadOps{a->tokens, a->vocab, a->dim, a->dtype, a->x, a->x_sr, a->weight, a->w_sr};
}

static int score_check(const swx_logprob_args* a) {
    if (!a) return SWX_ERR_INVALID_ARG;
    const int c = head_check(ops_of(a));
    if (c != SWX_OK) return c;
    if (a->x_sr < a->dim || a->w_sr < a->dim) return SWX_ERR_INVALID_ARG;
    if (a->top_k < 0 || a->top_k > a->vocab) return SWX_ERR_INVALID_ARG;
    if (a->top_k > SWX_MAX_TOP) return SWX_ERR_UNSUPPORTED;
    if (!(a->temperature > 0.f) || a->temperature > 1e15f || a->temperature < 1e-15f) return SWX_ERR_INVALID_ARG;
    return SWX_OK;
}

template <typename T, bool ALL, int THREADS>
static cudaError_t launch_top(const ScoreRows& p, cudaStream_t st) {
    const int smem = (int)score_top_smem(ALL, p.cand);
    const cudaError_t e = allow_smem(score_top_kernel<T, ALL, THREADS>, (int)score_top_smem(ALL, std::min(THREADS, SWX_MAX_TOP + SC_EXTRA)));
    if (e != cudaSuccess) return e;
    score_top_kernel<T, ALL, THREADS><<<(unsigned)p.T, THREADS, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_top(const ScoreRows& p, bool all, cudaStream_t st) {
    if (p.cand <= 128) return all ? launch_top<T, true, 128>(p, st) : launch_top<T, false, 128>(p, st);
    return all ? launch_top<T, true, 256>(p, st) : launch_top<T, false, 256>(p, st);
}

}  // namespace swx

using namespace swx;

extern "C" {

int64_t swx_logprob_args_size(void) { return (int64_t)sizeof(swx_logprob_args); }

int64_t swx_logprob_fwd_workspace_bytes(const swx_logprob_args* a) {
    const int c = score_check(a);
    return c != SWX_OK ? -c : score_plan(head_plan(ops_of(a)), a->tokens, a->vocab, a->top_k).total;
}

int64_t swx_logprob_bwd_workspace_bytes(const swx_logprob_args* a) {
    const int c = score_check(a);
    return c != SWX_OK ? -c : head_plan(ops_of(a)).bwd_total;
}

int swx_logprob_fwd(const swx_logprob_args* a, void* stream) {
    const int c = score_check(a);
    if (c != SWX_OK) return c;
    if (a->tokens == 0) return SWX_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!a->x || !a->weight || !a->targets || !a->log_probs || !a->entropy || !a->workspace || (a->row_max == nullptr) != (a->row_sum == nullptr) ||
        (a->top_k > 0 && (!a->top_log_probs || !a->top_ids)))
        return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    const ScorePlan f = score_plan(q, o.T, o.V, a->top_k);
    if (a->workspace_bytes < f.total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    head_operands(o, q, ws, x, w, st);
    CUtensorMap mx, mw;
    if (!x.k_major(&mx) || !w.k_major(&mw)) return SWX_ERR_CUDA;
    XentGemm g = logits_gemm(o, q, 0, o.V, status);
    g.target = a->targets; g.ignore = a->ignore_index;
    g.inv_temp = 1.f / a->temperature; g.k2 = LOG2E * g.inv_temp;
    g.score = reinterpret_cast<float4*>(ws + f.off_score);
    g.hit = reinterpret_cast<float*>(ws + f.off_hit);
    g.rec = reinterpret_cast<float2*>(ws + f.off_rec); g.third = reinterpret_cast<float*>(ws + f.off_third); g.groups = f.groups;
    g.all = reinterpret_cast<float*>(ws + f.off_rec);
    const cudaError_t e = a->top_k == 0 ? launch_score(g, mx, mw, st)
                          : f.all       ? launch_logits<XE_SCORE_ALL>(g, mx, mw, mx, st)
                                        : launch_logits<XE_SCORE_TOP>(g, mx, mw, mx, st);
    if (e != cudaSuccess) return SWX_ERR_CUDA;
    ScoreRows p{};
    p.T = o.T; p.V = o.V; p.d = o.d; p.np = (int)(2 * q.nt);
    p.score = g.score; p.hit = g.hit; p.target = a->targets; p.ignore = a->ignore_index;
    p.k2 = g.k2; p.inv_temp = g.inv_temp;
    p.row_max = a->row_max; p.row_sum = a->row_sum; p.log_probs = a->log_probs; p.entropy = a->entropy;
    if (a->top_k == 0) {
        score_rows_kernel<<<(unsigned)((o.T + SC_THREADS / 32 - 1) / (SC_THREADS / 32)), SC_THREADS, 0, st>>>(p);
        return cudaGetLastError() == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
    }
    p.top = a->top_k; p.cand = f.cand; p.rec = g.rec; p.third = g.third; p.all = g.all; p.groups = f.groups;
    p.top_log_probs = a->top_log_probs; p.top_ids = a->top_ids;
    // the operands in their own type: bf16 ones from their copies where those were made (their rows start on 16 bytes)
    const bool bf = o.dtype == SWX_DTYPE_BF16;
    p.x = bf ? x.p : o.x; p.x_sr = bf ? x.row : o.x_sr;
    p.w = bf ? w.p : o.w; p.w_sr = bf ? w.row : o.w_sr;
    p.vec = bf || (aligned16(o.x) && aligned16(o.w) && o.x_sr % 4 == 0 && o.w_sr % 4 == 0);
    const cudaError_t r = bf ? launch_top<__nv_bfloat16>(p, f.all, st) : launch_top<float>(p, f.all, st);
    return r == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
}

int swx_logprob_bwd(const swx_logprob_args* a, void* stream) {
    const int c = score_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dweight && a->dw_dtype != SWX_DTYPE_F32 && (a->dw_dtype != SWX_DTYPE_BF16 || a->dtype == SWX_DTYPE_F32)) return SWX_ERR_UNSUPPORTED;
    if (!a->dx && !a->dweight) return SWX_OK;
    if (a->tokens == 0) {
        if (!a->dweight) return SWX_OK;
        return cudaMemsetAsync(a->dweight, 0, (size_t)(a->vocab * a->dim) * (a->dw_dtype == SWX_DTYPE_F32 ? 4 : 2), st) == cudaSuccess
                   ? SWX_OK : SWX_ERR_CUDA;
    }
    if (!a->x || !a->weight || !a->targets || !a->row_max || !a->row_sum || !a->workspace || (a->d_entropy && !a->entropy))
        return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    if (a->workspace_bytes < q.bwd_total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    const HeadGrads gr{a->dx, a->dweight, a->dw_dtype == SWX_DTYPE_BF16, nullptr, nullptr};
    return head_backward(o, q, static_cast<uint8_t*>(a->workspace), gr, st, launch_grad, [a](XentGemm& g) {
        g.target = a->targets; g.ignore = a->ignore_index;
        g.inv_temp = 1.f / a->temperature; g.k2 = LOG2E * g.inv_temp;
        g.row_max = a->row_max; g.row_sum = a->row_sum; g.entropy = a->entropy;
        g.d_logp = a->d_log_probs; g.d_entropy = a->d_entropy;
    }, [](__nv_bfloat16*, int64_t, int64_t) { return (int)SWX_OK; });
}

}  // extern "C"
