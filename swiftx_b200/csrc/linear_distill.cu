// Distillation of a linear head from a teacher's top logits, without keeping the student's logits:
//   q = softmax over a row's used entries of t / tau,  l_v = z_v / tau - log sum exp(z / tau),  z = x W^T,
//   loss = tau^2 sum_j q_j (log q_j - l_{id_j}),  dz_v = tau c (p_v - Q_v),
// with p = e^l, Q_v the sum of the q of the entries of word v and c the row's upstream gradient (over the number of rows
// that count for the mean).
//
// Forward: a kernel sorts each row's words (and counts those before each half tile) and takes the softmax of its entries;
// the head's product with the scoring epilogue of head_gemm.cuh, which also picks the logits at the words; a kernel joins
// the rows' statistics and losses.  Backward: as the loss's, with tau c p in the epilogue, and tau c (p - Q) in its place at the
// words before the tile leaves shared memory, each rounded once.
// (With the words' logits as dot products of their own, 32 rows of the weight for each token, and dlogit set at the words by a
// launch after each piece, 8192 x 50001 x 1024 took 104 and 52 us more.)
#include "head_gemm.cuh"

namespace swx {

constexpr int DI_WARPS = 4, DI_THREADS = 32 * DI_WARPS;
constexpr float DI_LN2 = 0.69314718055994531f;

// What the forward leaves for the backward: rows' statistics, and their words.
struct DistillSaved {
    float* row_max; float* row_sum; float* teacher;    // (T): the teacher's sum q log q
    int* ids; float* share; float* logit;              // (T, K), ids in rising order and INT32_MAX behind them
    uint8_t* before; int stride;                       // (T, stride): how many ids lie before each 128 columns
};

struct DistillRows {
    int64_t T, V;
    int64_t r0, rows_all;                              // the rows of one product, r0 to T, of all
    int K, np;
    const float4* score;
    float k2, inv_temp;
    const int64_t* ids; int64_t ids_sr; const void* logits; int64_t tl_sr; int tl_bf16;
    DistillSaved s;
    float* rows; double2* sums; float* loss; float* count; int reduction; int* counter;
};

// Warp = one row, NL entries a lane: the softmax of its used entries, and its different words in rising order with their shares.
// row_sum: 1 for a row that counts, -1 for one that does not, NaN for one with a bad entry (no words then).
template <int NL>
__global__ void __launch_bounds__(DI_THREADS) distill_prepare_kernel(const DistillRows p) {
    __shared__ int sorted[DI_WARPS][32 * NL + 1];
    const int64_t row = (int64_t)blockIdx.x * DI_WARPS + threadIdx.x / 32;
    if (row >= p.T) return;
    const int lane = threadIdx.x % 32;
    int* mine = sorted[threadIdx.x / 32];
    float q[NL], all[NL];
    int id[NL];
    bool first[NL], odd = false;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int j = lane + 32 * i;
        id[i] = -1;
        q[i] = -INFINITY;
        if (j < p.K) {
            const int64_t v = p.ids[row * p.ids_sr + j];
            const float t = p.tl_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[row * p.tl_sr + j])
                                      : static_cast<const float*>(p.logits)[row * p.tl_sr + j];
            if (v >= 0 && t != -INFINITY) {
                odd |= v >= p.V || t != t || t == INFINITY;
                id[i] = v < p.V ? (int)v : 0;
                q[i] = t;
            }
        }
        top = fmaxf(top, q[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool bad = __any_sync(0xffffffffu, odd);
    bool some = false;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        some |= id[i] >= 0;
        // (the difference first: a type's lowest value over a small temperature would be -inf)
        q[i] = id[i] < 0 ? 0.f : ex2((q[i] - top) * (LOG2E * p.inv_temp));
        sum += q[i];
    }
    const bool live = __any_sync(0xffffffffu, some);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float self = 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        q[i] = live && !bad ? q[i] / sum : 0.f;
        if (q[i] != 0.f) self += q[i] * logf(q[i]);
        if (bad) id[i] = -1;
        all[i] = 0.f;
        first[i] = id[i] >= 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) self += __shfl_xor_sync(0xffffffffu, self, o);
    // a word's place is the number of smaller ones; the shares of one that stands in several entries go to the first of them, and the
    // others count it once
    int rank[NL] = {}, n = 0;
#pragma unroll
    for (int h = 0; h < NL; ++h)
        for (int j = 0; j < min(32, p.K - 32 * h); ++j) {
            const float qj = __shfl_sync(0xffffffffu, q[h], j);
            const int idj = __shfl_sync(0xffffffffu, id[h], j);
            bool again = false;               // an earlier entry is of the same word
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const bool same = id[i] == idj;
                const int apart = lane + 32 * i - (j + 32 * h);
                all[i] += same ? qj : 0.f;
                first[i] = first[i] && !(same && apart > 0);
                again |= __any_sync(0xffffffffu, same && apart < 0);
            }
            if (idj < 0 || again) continue;
            ++n;
#pragma unroll
            for (int i = 0; i < NL; ++i) rank[i] += idj < id[i];
        }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int j = lane + 32 * i;
        if (first[i]) {
            mine[rank[i]] = p.s.ids[row * p.K + rank[i]] = id[i];
            p.s.share[row * p.K + rank[i]] = all[i];
        }
        if (j >= n && j < p.K) p.s.ids[row * p.K + j] = INT32_MAX;
    }
    if (lane == 0) mine[n] = INT32_MAX;
    __syncwarp();
    // 16 counts a lane: a search, then along the words
    for (int h = 16 * lane; h < p.s.stride; h += 512) {
        int at = 0;
        for (int hi = n; at < hi;) {
            const int mid = (at + hi) / 2;
            if (mine[mid] < 128 * (int64_t)h) at = mid + 1;
            else hi = mid;
        }
        uint32_t w[4] = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            while (mine[at] < 128 * ((int64_t)h + i) && at < n) ++at;
            w[i / 4] |= (uint32_t)at << (8 * (i % 4));
        }
        *reinterpret_cast<uint4*>(p.s.before + row * p.s.stride + h) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (lane == 0) {
        p.s.row_sum[row] = bad ? __int_as_float(0x7fc00000) : live ? 1.f : -1.f;
        p.s.teacher[row] = self;
    }
}

// Warp = one row: its statistics and loss.  Each CTA leaves the sum of its rows' losses and the count of its rows; the last CTA of the
// last product's rows to finish adds those of all up (fp64, a fixed order whichever CTA it is).
__global__ void __launch_bounds__(DI_THREADS) distill_rows_kernel(const DistillRows p) {
    __shared__ int is_last;
    __shared__ double red[DI_WARPS][2];
    wait_for_previous();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t row = p.r0 + (int64_t)blockIdx.x * DI_WARPS + warp;
    double sum = 0., n = 0.;
    if (row < p.T) {
        const Score a = score_join_parts(p.score + (row - p.r0) * p.np, p.np, p.k2, lane, 32);
        const float ls = logf(a.s), mark = p.s.row_sum[row];
        float loss = 0.f;
        for (int j = lane; j < p.K; j += 32) {
            const float share = mark > 0.f && p.s.ids[row * p.K + j] != INT32_MAX ? p.s.share[row * p.K + j] : 0.f;
            if (share != 0.f) loss += share * ((p.s.logit[row * p.K + j] - a.m) * p.k2 * DI_LN2 - ls);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
        loss = mark < 0.f ? 0.f : mark > 0.f ? (p.s.teacher[row] - loss) / (p.inv_temp * p.inv_temp) : mark;
        __syncwarp();
        if (lane == 0) {
            p.s.row_max[row] = a.m;
            if (mark > 0.f) p.s.row_sum[row] = a.s;
            if (p.rows) p.rows[row] = loss;
        }
        sum = loss;
        n = mark < 0.f ? 0. : 1.;
    }
    if (p.reduction == SWX_XENT_NONE) return;
    if (lane == 0) { red[warp][0] = sum; red[warp][1] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < DI_WARPS; ++i) { sum += red[i][0]; n += red[i][1]; }
        p.sums[p.r0 / DI_WARPS + blockIdx.x] = make_double2(sum, n);
        __threadfence();
        is_last = p.T == p.rows_all && atomicAdd(p.counter, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    sum = n = 0.;
#pragma unroll 4
    for (int i = threadIdx.x; i < (int)(p.r0 / DI_WARPS + gridDim.x); i += DI_THREADS) {
        const double2 s = __ldcg(p.sums + i);
        sum += s.x;
        n += s.y;
    }
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    if (lane == 0) { red[warp][0] = sum; red[warp][1] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < DI_WARPS; ++i) { sum += red[i][0]; n += red[i][1]; }
        *p.count = (float)n;
        *p.loss = (float)(p.reduction == SWX_XENT_MEAN ? sum / n : sum);
    }
}

// ------------------------------------------------------------------ host side
struct DistillPlan { int64_t off_score, off_sums, off_cnt, total; };

static DistillPlan distill_plan(const HeadPlan& q, int64_t T) {
    DistillPlan f{};
    f.off_score = q.base;
    f.off_sums = f.off_score + up256(2 * q.nt * std::min(T, SC_ROWS) * 16);
    f.off_cnt = f.off_sums + up256((T + DI_WARPS - 1) / DI_WARPS * 16);
    f.total = f.off_cnt + 256;
    return f;
}

// Counts for each half of the vocabulary's tiles and their end, whole 16-byte pieces.
static int64_t before_stride(int64_t V) { return ((V + XE_TILE - 1) / XE_TILE * 2 + 1 + 15) / 16 * 16; }
static int64_t saved_bytes(int64_t T, int64_t V, int64_t K) { return 3 * up256(T * 4) + 3 * up256(T * K * 4) + T * before_stride(V); }

static DistillSaved saved_of(uint8_t* b, int64_t T, int64_t V, int64_t K) {
    DistillSaved s{};
    s.row_max = reinterpret_cast<float*>(b); b += up256(T * 4);
    s.row_sum = reinterpret_cast<float*>(b); b += up256(T * 4);
    s.teacher = reinterpret_cast<float*>(b); b += up256(T * 4);
    s.ids = reinterpret_cast<int*>(b); b += up256(T * K * 4);
    s.share = reinterpret_cast<float*>(b); b += up256(T * K * 4);
    s.logit = reinterpret_cast<float*>(b); b += up256(T * K * 4);
    s.before = b;
    s.stride = (int)before_stride(V);
    return s;
}

static HeadOps ops_of(const swx_distill_args* a) {
    return HeadOps{a->tokens, a->vocab, a->dim, a->dtype, a->x, a->x_sr, a->weight, a->w_sr};
}

static int distill_check(const swx_distill_args* a) {
    if (!a) return SWX_ERR_INVALID_ARG;
    const int c = head_check(ops_of(a));
    if (c != SWX_OK) return c;
    if (a->x_sr < a->dim || a->w_sr < a->dim) return SWX_ERR_INVALID_ARG;
    if (a->reduction < SWX_XENT_NONE || a->reduction > SWX_XENT_SUM || a->entries < 1) return SWX_ERR_INVALID_ARG;
    if (a->teacher_dtype != SWX_DTYPE_F32 && a->teacher_dtype != SWX_DTYPE_BF16) return SWX_ERR_UNSUPPORTED;
    if (a->entries > SWX_MAX_TOP) return SWX_ERR_UNSUPPORTED;
    if (!(a->temperature > 0.f) || a->temperature > 1e15f || a->temperature < 1e-15f) return SWX_ERR_INVALID_ARG;
    return SWX_OK;
}

static void fill_words(XentGemm& g, const DistillSaved& s, const swx_distill_args* a) {
    set_score_sums(g, ops_of(a));
    g.inv_temp = 1.f / a->temperature; g.k2 = exponent_scale(a->temperature, mean_cut((double)logit_additions(ops_of(a))));
    g.ids = s.ids; g.id_logit = s.logit; g.id_share = s.share; g.nids = (int)a->entries;
    g.before = s.before; g.before_stride = s.stride;
}

}  // namespace swx

using namespace swx;

extern "C" {

int64_t swx_distill_args_size(void) { return (int64_t)sizeof(swx_distill_args); }

int64_t swx_distill_saved_bytes(const swx_distill_args* a) {
    const int c = distill_check(a);
    return c != SWX_OK ? -c : saved_bytes(a->tokens, a->vocab, a->entries);
}

int64_t swx_distill_fwd_workspace_bytes(const swx_distill_args* a) {
    const int c = distill_check(a);
    return c != SWX_OK ? -c : distill_plan(head_plan(ops_of(a)), a->tokens).total;
}

int64_t swx_distill_bwd_workspace_bytes(const swx_distill_args* a) {
    const int c = distill_check(a);
    return c != SWX_OK ? -c : head_plan(ops_of(a)).bwd_total;
}

int swx_distill_fwd(const swx_distill_args* a, void* stream) {
    const int c = distill_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool none = a->reduction == SWX_XENT_NONE;
    if (!none && (!a->loss || !a->count)) return SWX_ERR_INVALID_ARG;
    if (a->tokens == 0) {
        if (none) return SWX_OK;
        // no row: a sum of 0, a mean of 0 / 0
        if (cudaMemsetAsync(a->count, 0, 4, st) != cudaSuccess) return SWX_ERR_CUDA;
        return cudaMemsetAsync(a->loss, a->reduction == SWX_XENT_MEAN ? 0xff : 0, 4, st) == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
    }
    if (!a->x || !a->weight || !a->teacher_ids || !a->teacher_logits || !a->saved || !a->workspace || (none && !a->loss)) return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    const DistillPlan f = distill_plan(q, o.T);
    if (a->workspace_bytes < f.total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    if (a->saved_bytes < saved_bytes(o.T, o.V, a->entries) || !aligned16(a->saved)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    DistillRows p{};
    p.T = o.T; p.V = o.V; p.K = (int)a->entries; p.np = (int)(2 * q.nt);
    p.inv_temp = 1.f / a->temperature;
    p.ids = a->teacher_ids; p.ids_sr = a->ids_sr; p.logits = a->teacher_logits; p.tl_sr = a->tl_sr;
    p.tl_bf16 = a->teacher_dtype == SWX_DTYPE_BF16;
    p.s = saved_of(static_cast<uint8_t*>(a->saved), o.T, o.V, p.K);
    const unsigned rows = (unsigned)((o.T + DI_WARPS - 1) / DI_WARPS);
    if (p.K <= 32) distill_prepare_kernel<1><<<rows, DI_THREADS, 0, st>>>(p);
    else if (p.K <= 64) distill_prepare_kernel<2><<<rows, DI_THREADS, 0, st>>>(p);
    else distill_prepare_kernel<4><<<rows, DI_THREADS, 0, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return SWX_ERR_CUDA;
    Operand x, w;
    head_operands(o, q, ws, x, w, st);
    CUtensorMap mw;
    if (!w.k_major(&mw)) return SWX_ERR_CUDA;
    p.rows = none ? a->loss : nullptr; p.sums = reinterpret_cast<double2*>(ws + f.off_sums);
    p.loss = a->loss; p.count = a->count; p.reduction = a->reduction; p.rows_all = o.T;
    for (int64_t r0 = 0; r0 < o.T; r0 += SC_ROWS) {
        HeadOps oc = o;
        oc.T = std::min(SC_ROWS, o.T - r0);
        HeadPlan qc = q;
        qc.mt = (oc.T + XE_TILE - 1) / XE_TILE;
        CUtensorMap mx;
        if (!x.part(r0, oc.T).k_major(&mx)) return SWX_ERR_CUDA;
        XentGemm g = logits_gemm(oc, qc, 0, o.V, status);
        DistillSaved s = p.s;                  // these rows' words
        s.ids += r0 * p.K; s.share += r0 * p.K; s.logit += r0 * p.K; s.before += r0 * s.stride;
        fill_words(g, s, a);
        g.score = reinterpret_cast<float4*>(ws + f.off_score);
        g.counter = reinterpret_cast<int*>(ws + f.off_cnt);
        if (launch_logits<XE_SCORE_IDS>(g, mx, mw, mx, st) != cudaSuccess) return SWX_ERR_CUDA;
        p.T = r0 + oc.T; p.r0 = r0; p.k2 = g.k2; p.score = g.score; p.counter = g.counter;
        const unsigned ctas = (unsigned)((oc.T + DI_WARPS - 1) / DI_WARPS);
        if (launch_after(distill_rows_kernel, ctas, DI_THREADS, 0, st, p) != cudaSuccess) return SWX_ERR_CUDA;
    }
    return SWX_OK;
}

int swx_distill_bwd(const swx_distill_args* a, void* stream) {
    const int c = distill_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dweight && a->dw_dtype != SWX_DTYPE_F32 && (a->dw_dtype != SWX_DTYPE_BF16 || a->dtype == SWX_DTYPE_F32)) return SWX_ERR_UNSUPPORTED;
    if (!a->dx && !a->dweight) return SWX_OK;
    if (a->tokens == 0) {
        if (!a->dweight) return SWX_OK;
        return cudaMemsetAsync(a->dweight, 0, (size_t)(a->vocab * a->dim) * (a->dw_dtype == SWX_DTYPE_F32 ? 4 : 2), st) == cudaSuccess
                   ? SWX_OK : SWX_ERR_CUDA;
    }
    if (!a->x || !a->weight || !a->saved || !a->dloss || !a->workspace || (a->reduction == SWX_XENT_MEAN && !a->count)) return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    if (a->workspace_bytes < q.bwd_total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    if (a->saved_bytes < saved_bytes(o.T, o.V, a->entries) || !aligned16(a->saved)) return SWX_ERR_INVALID_ARG;
    const DistillSaved s = saved_of(static_cast<uint8_t*>(a->saved), o.T, o.V, a->entries);
    const HeadGrads gr{a->dx, a->dweight, a->dw_dtype == SWX_DTYPE_BF16, a->reduction == SWX_XENT_NONE ? nullptr : a->dloss,
                       a->reduction == SWX_XENT_MEAN ? a->count : nullptr};
    return head_backward(o, q, static_cast<uint8_t*>(a->workspace), gr, st, launch_logits<XE_GRAD_IDS>, [&s, a](XentGemm& g) {
        fill_words(g, s, a);
        g.row_max = s.row_max; g.row_sum = s.row_sum; g.dloss = a->dloss; g.reduction = a->reduction;
    });
}

}  // extern "C"
