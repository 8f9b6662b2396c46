// Distillation of a linear head from a teacher's top logits, without keeping the student's logits:
//   q = softmax over a row's used entries of t / tau,  l_v = z_v / tau - log sum exp(z / tau),  z = x W^T,
//   loss = tau^2 sum_j q_j (log q_j - l_{id_j}),  dz_v = tau c (p_v - sum_j q_j [v == id_j]),
// with p = e^l and c the row's upstream gradient (over the number of rows that count for the mean).
//
// Forward: the head's product with the statistics of head_gemm.cuh's scoring epilogue, then one CTA for each row: the
// student's logits at the teacher's words as dot products of their own (the entries are spread over the vocabulary, at most a few
// to a tile), the softmax of the entries and the row's loss; the last CTA adds the rows up.  Backward: as the
// loss's, with tau p in the epilogue, and the teacher's words set to tau (p_j - q_j) by a small kernel
// between a piece of the vocabulary's dlogit and its products, each rounded once.
#include "head_gemm.cuh"

namespace swx {

constexpr int DI_THREADS = 128, DI_WARPS = DI_THREADS / 32, DI_PATCH_WARPS = 4;
constexpr int DI_LANE = SWX_MAX_TOP / 32;     // entries of a lane

struct DistillRows {
    int64_t T, V, d;
    int K, np;
    const float4* score;
    float k2, inv_temp;
    const int64_t* ids; int64_t ids_sr; const void* logits; int64_t tl_sr; int tl_bf16;
    const void* x; int64_t x_sr; const void* w; int64_t w_sr; int vec;
    float* row_max; float* row_sum; float* z;
    float* rows; double2* sums; float* loss; float* count; int reduction; int* counter;
    // backward
    const float* dloss; __nv_bfloat16* dz; int64_t ld, plane; int planes; int64_t c0, cw;
};

// A warp's softmax over the entries of a row: q (0 where not used), ids, whether an entry is used, whether one is outside the vocabulary.
__device__ __forceinline__ void teacher_row(const DistillRows& p, int64_t row, int lane, float (&q)[DI_LANE], int64_t (&id)[DI_LANE], bool& live, bool& bad) {
    float top = -INFINITY;
    bad = false;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < DI_LANE; ++i) {
        const int j = lane + 32 * i;
        id[i] = -1;
        q[i] = -INFINITY;
        if (j < p.K) {
            id[i] = p.ids[row * p.ids_sr + j];
            const float t = p.tl_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[row * p.tl_sr + j])
                                      : static_cast<const float*>(p.logits)[row * p.tl_sr + j];
            if (id[i] >= 0) q[i] = t * p.inv_temp;
        }
        if (q[i] == -INFINITY) id[i] = -1;
        bad |= id[i] >= p.V;
        nan |= q[i] != q[i];
        top = fmaxf(top, q[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad = __any_sync(0xffffffffu, bad || nan || top == INFINITY);
    live = bad || top > -INFINITY;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < DI_LANE; ++i) {
        q[i] = id[i] < 0 ? 0.f : ex2((q[i] - top) * LOG2E);
        sum += q[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float r = live ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < DI_LANE; ++i) q[i] *= r;
}

template <typename T>
__device__ __forceinline__ float dot(const T* x, const T* w, int64_t d, bool vec, int lane) {
    constexpr int N = 16 / sizeof(T);
    float a[2] = {0.f, 0.f};
    int64_t tail = 0;
    if (vec) {
#pragma unroll 2
        for (int64_t k = lane * N; k + N <= d; k += 32 * N) {
            const uint4 qx = *reinterpret_cast<const uint4*>(x + k), qw = *reinterpret_cast<const uint4*>(w + k);
#pragma unroll
            for (int j = 0; j < N; ++j) a[j & 1] = fmaf(Elem<T>::to_f(reinterpret_cast<const T*>(&qx)[j]), Elem<T>::to_f(reinterpret_cast<const T*>(&qw)[j]), a[j & 1]);
        }
        tail = d / N * N;
    }
    for (int64_t k = tail + lane; k < d; k += 32) a[0] = fmaf(Elem<T>::to_f(x[k]), Elem<T>::to_f(w[k]), a[0]);
    float s = a[0] + a[1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// CTA = one row.
template <typename T>
__global__ void __launch_bounds__(DI_THREADS) distill_rows_kernel(const DistillRows p) {
    __shared__ int64_t sid[SWX_MAX_TOP];
    __shared__ float sz[SWX_MAX_TOP];
    __shared__ Score part[DI_WARPS];
    __shared__ int is_last;
    __shared__ double red[DI_WARPS][2];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Score a = score_join_row<DI_THREADS>(p.score + row * p.np, p.np, part);
    float q[DI_LANE];
    int64_t id[DI_LANE];
    bool live = false, bad = false;
    if (warp == 0) {
        teacher_row(p, row, lane, q, id, live, bad);
#pragma unroll
        for (int i = 0; i < DI_LANE; ++i)
            if (lane + 32 * i < p.K) sid[lane + 32 * i] = bad ? -1 : id[i];
    }
    __syncthreads();
    const T* x = static_cast<const T*>(p.x) + row * p.x_sr;
    for (int j = warp; j < p.K; j += DI_WARPS) {
        const int64_t v = sid[j];
        if (v < 0) continue;
        const float z = dot<T>(x, static_cast<const T*>(p.w) + v * p.w_sr, p.d, p.vec, lane);
        if (lane == 0) { sz[j] = z; p.z[row * p.K + j] = z; }
    }
    __syncthreads();
    double sum = 0., n = 0.;
    if (warp == 0) {
        const float ls = logf(a.s);
        float loss = 0.f;
#pragma unroll
        for (int i = 0; i < DI_LANE; ++i)
            if (lane + 32 * i < p.K && id[i] >= 0 && !bad && q[i] != 0.f) loss += q[i] * (logf(q[i]) - (fmaf(sz[lane + 32 * i], p.k2, -a.m) * 0.69314718055994531f - ls));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
        loss = bad ? __int_as_float(0x7fc00000) : loss / (p.inv_temp * p.inv_temp);
        if (!live) loss = 0.f;
        if (lane == 0) {
            p.row_max[row] = a.m;
            p.row_sum[row] = !live ? -1.f : bad ? __int_as_float(0x7fc00000) : a.s;
            if (p.rows) p.rows[row] = loss;
        }
        sum = loss;
        n = live ? 1. : 0.;
    }
    if (p.reduction == SWX_XENT_NONE) return;
    if (threadIdx.x == 0) {
        p.sums[row] = make_double2(sum, n);
        __threadfence();
        is_last = atomicAdd(p.counter, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    sum = n = 0.;
#pragma unroll 4
    for (int i = threadIdx.x; i < (int)gridDim.x; i += DI_THREADS) {
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

// Warp = one row: dlogit at the teacher's words inside the piece, tau c (p_j - q_j) in place of tau c p_j.
__global__ void __launch_bounds__(32 * DI_PATCH_WARPS) distill_patch_kernel(const DistillRows p) {
    const int64_t row = (int64_t)blockIdx.x * DI_PATCH_WARPS + threadIdx.x / 32;
    if (row >= p.T) return;
    const int lane = threadIdx.x % 32;
    const float s = p.row_sum[row], m = p.row_max[row];
    if (!(s > 0.f)) return;                   // a row that does not count is zero, one with a bad entry NaN throughout
    float q[DI_LANE], all[DI_LANE];
    int64_t id[DI_LANE];
    bool live, bad, first[DI_LANE];
    teacher_row(p, row, lane, q, id, live, bad);
#pragma unroll
    for (int i = 0; i < DI_LANE; ++i) { all[i] = 0.f; first[i] = true; }
    for (int j = 0; j < p.K; ++j) {           // the same word may stand in several entries; its first one writes
        float qj = 0.f;
        int64_t idj = -1;
#pragma unroll
        for (int i = 0; i < DI_LANE; ++i)
            if (j / 32 == i) { qj = __shfl_sync(0xffffffffu, q[i], j % 32); idj = __shfl_sync(0xffffffffu, id[i], j % 32); }
#pragma unroll
        for (int i = 0; i < DI_LANE; ++i)
            if (id[i] == idj) { all[i] += qj; first[i] = first[i] && j >= lane + 32 * i; }
    }
    const float c = (p.reduction == SWX_XENT_NONE ? p.dloss[row] : 1.f) / p.inv_temp;
#pragma unroll
    for (int i = 0; i < DI_LANE; ++i) {
        const int j = lane + 32 * i;
        if (j >= p.K || id[i] < p.c0 || id[i] >= p.c0 + p.cw || !first[i]) continue;
        float v = c * (ex2(fmaf(p.z[row * p.K + j], p.k2, -m)) / s - all[i]);
        __nv_bfloat16* o = p.dz + row * p.ld + (id[i] - p.c0);
        for (int k = 0; k < p.planes; ++k) {
            const __nv_bfloat16 b = __float2bfloat16_rn(v);
            o[k * p.plane] = b;
            v -= __bfloat162float(b);
        }
    }
}

// ------------------------------------------------------------------ host side
struct DistillPlan { int64_t off_score, off_sums, off_cnt, total; };

static DistillPlan distill_plan(const HeadPlan& q, int64_t T) {
    DistillPlan f{};
    f.off_score = q.base;
    f.off_sums = f.off_score + up256(2 * q.nt * T * 16);
    f.off_cnt = f.off_sums + up256(T * 16);
    f.total = f.off_cnt + 256;
    return f;
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

static DistillRows distill_rows(const swx_distill_args* a) {
    DistillRows p{};
    p.T = a->tokens; p.V = a->vocab; p.d = a->dim; p.K = (int)a->entries;
    p.inv_temp = 1.f / a->temperature; p.k2 = LOG2E / a->temperature;
    p.ids = a->teacher_ids; p.ids_sr = a->ids_sr; p.logits = a->teacher_logits; p.tl_sr = a->tl_sr;
    p.tl_bf16 = a->teacher_dtype == SWX_DTYPE_BF16;
    p.row_max = a->row_max; p.row_sum = a->row_sum; p.z = a->entry_logits; p.reduction = a->reduction;
    return p;
}

}  // namespace swx

using namespace swx;

extern "C" {

int64_t swx_distill_args_size(void) { return (int64_t)sizeof(swx_distill_args); }

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
    if (!a->x || !a->weight || !a->teacher_ids || !a->teacher_logits || !a->row_max || !a->row_sum || !a->entry_logits || !a->workspace ||
        (none && !a->loss))
        return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    const DistillPlan f = distill_plan(q, o.T);
    if (a->workspace_bytes < f.total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    head_operands(o, q, ws, x, w, st);
    CUtensorMap mx, mw;
    if (!x.k_major(&mx) || !w.k_major(&mw)) return SWX_ERR_CUDA;
    DistillRows p = distill_rows(a);
    XentGemm g = logits_gemm(o, q, 0, o.V, status);
    g.inv_temp = p.inv_temp; g.k2 = p.k2;
    g.score = reinterpret_cast<float4*>(ws + f.off_score);
    g.counter = reinterpret_cast<int*>(ws + f.off_cnt);
    if (launch_score(g, mx, mw, st) != cudaSuccess) return SWX_ERR_CUDA;
    p.np = (int)(2 * q.nt); p.score = g.score;
    // the operands in their own type: bf16 ones from their copies where those were made (their rows start on 16 bytes)
    const bool bf = o.dtype == SWX_DTYPE_BF16;
    p.x = bf ? x.p : o.x; p.x_sr = bf ? x.row : o.x_sr;
    p.w = bf ? w.p : o.w; p.w_sr = bf ? w.row : o.w_sr;
    p.vec = bf || (aligned16(o.x) && aligned16(o.w) && o.x_sr % 4 == 0 && o.w_sr % 4 == 0);
    p.rows = none ? a->loss : nullptr; p.sums = reinterpret_cast<double2*>(ws + f.off_sums);
    p.loss = a->loss; p.count = a->count; p.counter = g.counter;
    if (bf) distill_rows_kernel<__nv_bfloat16><<<(unsigned)o.T, DI_THREADS, 0, st>>>(p);
    else distill_rows_kernel<float><<<(unsigned)o.T, DI_THREADS, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
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
    if (!a->x || !a->weight || !a->teacher_ids || !a->teacher_logits || !a->row_max || !a->row_sum || !a->entry_logits || !a->dloss ||
        !a->workspace || (a->reduction == SWX_XENT_MEAN && !a->count))
        return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    if (a->workspace_bytes < q.bwd_total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    DistillRows p = distill_rows(a);
    p.dloss = a->dloss; p.ld = q.ldp; p.plane = o.T * q.ldp; p.planes = q.planes;
    const HeadGrads gr{a->dx, a->dweight, a->dw_dtype == SWX_DTYPE_BF16, a->reduction == SWX_XENT_NONE ? nullptr : a->dloss,
                       a->reduction == SWX_XENT_MEAN ? a->count : nullptr};
    return head_backward(o, q, static_cast<uint8_t*>(a->workspace), gr, st, launch_grad, [&p, a](XentGemm& g) {
        g.inv_temp = p.inv_temp; g.k2 = p.k2;
        g.row_max = a->row_max; g.row_sum = a->row_sum; g.dloss = a->dloss; g.reduction = a->reduction;
    }, [&p, st](__nv_bfloat16* dz, int64_t c0, int64_t cw) {
        p.dz = dz; p.c0 = c0; p.cw = cw;
        distill_patch_kernel<<<(unsigned)((p.T + DI_PATCH_WARPS - 1) / DI_PATCH_WARPS), 32 * DI_PATCH_WARPS, 0, st>>>(p);
        return (int)(cudaGetLastError() == cudaSuccess ? SWX_OK : SWX_ERR_CUDA);
    });
}

}  // extern "C"
