// Log probabilities of given tokens under a linear head, with the entropy and the top alternatives, without keeping
// the logits:  z = x W^T,  l_v = z_v / tau - log sum exp(z / tau),  p = e^l,
//   log_probs = l_y,  entropy = -sum p l,  top: the K largest z (the lowest word first among equals).
// Backward, for upstream gradients g of log_probs and h of the entropy H:
//   dz_v = (g [v == y] - p_v (g + h (l_v + H))) / tau,  dx = dz W,  dW = dz^T x.
//
// Forward: the head's product (head_gemm.cuh) with an epilogue that keeps three floats for each half of a 256-column tile: the
// maximum m, s = sum e and w = sum e u of e = 2^u, u = (z - m) log2(e) / tau; with alternatives also the two largest logits of every
// 32 columns (8 bytes), or, for a small vocabulary, the logits.  Then one kernel for the rows: the statistics joined, and
//   H = ln s - ln2 w / s.
// Alternatives: the K + 8 groups of 32 columns with the largest maxima hold the K + 8 largest logits, but for groups whose second
// value passes too, and those are taken whole.  The tensor core's sums are a few 2^-23 off, enough to turn two close logits
// round, so the candidates' products are formed again in fp64 from the operands, and those give the order, the ties
// and the values.
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
    const float2* rec; const float* all; int64_t groups;
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

// Products of a row of x with two rows of the weight, summed over a warp in fp64 (products of fp32 or bf16 values are exact in it).
template <typename T>
__device__ __forceinline__ double2 dot2(const T* x, const T* w0, const T* w1, int64_t d, bool vec, int lane) {
    constexpr int N = 16 / sizeof(T);
    double a0 = 0., a1 = 0.;
    int64_t tail = 0;
    if (vec) {
        for (int64_t k = lane * N; k + N <= d; k += 32 * N) {
            const uint4 qx = *reinterpret_cast<const uint4*>(x + k), q0 = *reinterpret_cast<const uint4*>(w0 + k),
                        q1 = *reinterpret_cast<const uint4*>(w1 + k);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const double xv = Elem<T>::to_f(reinterpret_cast<const T*>(&qx)[j]);
                a0 = fma(xv, (double)Elem<T>::to_f(reinterpret_cast<const T*>(&q0)[j]), a0);
                a1 = fma(xv, (double)Elem<T>::to_f(reinterpret_cast<const T*>(&q1)[j]), a1);
            }
        }
        tail = d / N * N;
    }
    for (int64_t k = tail + lane; k < d; k += 32) {
        const double xv = Elem<T>::to_f(x[k]);
        a0 = fma(xv, (double)Elem<T>::to_f(w0[k]), a0);
        a1 = fma(xv, (double)Elem<T>::to_f(w1[k]), a1);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a0 += __shfl_xor_sync(0xffffffffu, a0, o);
        a1 += __shfl_xor_sync(0xffffffffu, a1, o);
    }
    return make_double2(a0, a1);
}

static int score_candidates(bool all, int cand) { return all ? cand : 32 * cand; }

static size_t score_top_smem(bool all, int cand) {
    return (size_t)topk_capacity(cand, SC_PER) * 8 + cand * 8 + (size_t)score_candidates(all, cand) * 12;
}

// CTA = one row: its statistics, the candidates from the records (ALL: from the logits), their products in fp64, their ranks.
template <typename T, bool ALL>
__global__ void __launch_bounds__(SC_THREADS) score_top_kernel(const ScoreRows p) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ int count, ncand;
    __shared__ Score part[SC_THREADS / 32];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint64_t* buf = reinterpret_cast<uint64_t*>(raw);
    uint64_t* kept = buf + topk_capacity(p.cand, SC_PER);
    uint64_t* val = kept + p.cand;                                   // candidates' products, order-preserving
    int* col = reinterpret_cast<int*>(val + (ALL ? p.cand : 32 * p.cand));

    Score a{-INFINITY, 0.f, 0.f};
    for (int i = threadIdx.x; i < p.np; i += SC_THREADS) {
        const float4 q = p.score[row * p.np + i];
        score_join(a, Score{q.x, q.y, q.z}, p.k2, SCORE_FAR);
    }
    score_join_warp(a, p.k2, SCORE_FAR);
    if (lane == 0) part[warp] = a;
    if (threadIdx.x == 0) ncand = 0;
    __syncthreads();
    a = part[0];
#pragma unroll
    for (int i = 1; i < SC_THREADS / 32; ++i) score_join(a, part[i], p.k2, SCORE_FAR);
    if (threadIdx.x == 0) score_finish(p, row, a);
    if (p.target[row] == p.ignore) {                                 // a token that does not count
        for (int i = threadIdx.x; i < p.top; i += SC_THREADS) {
            p.top_log_probs[row * p.top + i] = 0.f;
            p.top_ids[row * p.top + i] = -1;
        }
        return;
    }

    TopK<SC_THREADS, SC_PER> best;
    best.start(buf, kept, &count, p.cand);
    const int64_t n = ALL ? p.V : p.groups;
    const float2* rec = p.rec + row * p.groups;
    const float* all = p.all + row * p.V;
    for (int64_t i0 = 0; i0 < n; i0 += SC_THREADS * SC_PER) {
        uint64_t key[SC_PER];
#pragma unroll
        for (int j = 0; j < SC_PER; ++j) {
            const int64_t i = i0 + j * SC_THREADS + threadIdx.x;
            key[j] = 0;
            if (i < n) {
                const float z = ALL ? all[i] : __uint_as_float(__float_as_uint(rec[i].x) & ~31u);
                key[j] = index_key(order_key(z != z ? -INFINITY : z), (uint32_t)i);
            }
        }
        best.push(key);
    }
    best.rank();
    // the columns of the candidates
    const int m = best.n;
    if (ALL) {
        for (int i = threadIdx.x; i < m; i += SC_THREADS) col[i] = (int)key_index(buf[i]);
        if (threadIdx.x == 0) ncand = m;
    } else {
        const float least = order_value((uint32_t)(buf[m - 1] >> 32));
        for (int i = threadIdx.x; i < m; i += SC_THREADS) {
            const int g = (int)key_index(buf[i]);
            const float2 r = rec[g];
            if (__uint_as_float(__float_as_uint(r.y) & ~31u) >= least) {
                const int c = (int)min((int64_t)32, p.V - (int64_t)g * 32), at = atomicAdd(&ncand, c);
                for (int j = 0; j < c; ++j) col[at + j] = g * 32 + j;
            } else {
                col[atomicAdd(&ncand, 1)] = g * 32 + (int)(__float_as_uint(r.x) & 31u);
            }
        }
    }
    __syncthreads();
    const int nc = ncand;
    const T* x = static_cast<const T*>(p.x) + row * p.x_sr;
    const T* w = static_cast<const T*>(p.w);
    for (int i = 2 * warp; i < nc; i += 2 * (SC_THREADS / 32)) {
        const int i1 = min(i + 1, nc - 1);
        const double2 z = dot2<T>(x, w + col[i] * p.w_sr, w + col[i1] * p.w_sr, p.d, p.vec, lane);
        if (lane == 0) {
            val[i] = order_key(z.x);
            if (i1 > i) val[i1] = order_key(z.y);
        }
    }
    __syncthreads();
    const double lse = (double)a.m * p.inv_temp + log((double)a.s);
    for (int i = threadIdx.x; i < nc; i += SC_THREADS) {
        const uint64_t v = val[i];
        const int c = col[i];
        int r = 0;
        for (int j = 0; j < nc; ++j) r += val[j] > v || (val[j] == v && col[j] < c);
        if (r < p.top) {
            const double z = __longlong_as_double((long long)(v >> 63 ? v & ~(1ull << 63) : ~v));
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
    int64_t off_score, off_hit, off_rec, total;
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
        f.total += up256(f.all ? T * V * 4 : T * f.groups * 8);
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

template <typename T, bool ALL>
static cudaError_t launch_top(const ScoreRows& p, cudaStream_t st) {
    const int smem = (int)score_top_smem(ALL, p.cand);
    const cudaError_t e = allow_smem(score_top_kernel<T, ALL>, (int)score_top_smem(ALL, SWX_MAX_TOP + SC_EXTRA));
    if (e != cudaSuccess) return e;
    score_top_kernel<T, ALL><<<(unsigned)p.T, SC_THREADS, smem, st>>>(p);
    return cudaGetLastError();
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
    g.rec = reinterpret_cast<float2*>(ws + f.off_rec); g.groups = f.groups;
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
    p.top = a->top_k; p.cand = f.cand; p.rec = g.rec; p.all = g.all; p.groups = f.groups;
    p.top_log_probs = a->top_log_probs; p.top_ids = a->top_ids;
    // the operands in their own type: bf16 ones from their copies where those were made (their rows start on 16 bytes)
    const bool bf = o.dtype == SWX_DTYPE_BF16;
    p.x = bf ? x.p : o.x; p.x_sr = bf ? x.row : o.x_sr;
    p.w = bf ? w.p : o.w; p.w_sr = bf ? w.row : o.w_sr;
    p.vec = bf || (aligned16(o.x) && aligned16(o.w) && o.x_sr % 4 == 0 && o.w_sr % 4 == 0);
    const cudaError_t r = bf ? (f.all ? launch_top<__nv_bfloat16, true>(p, st) : launch_top<__nv_bfloat16, false>(p, st))
                             : (f.all ? launch_top<float, true>(p, st) : launch_top<float, false>(p, st));
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
