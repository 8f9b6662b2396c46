// Log probabilities, entropy and top alternatives of rows of logits (a step of generation):
// with m the largest z, u = (z - m) log2(e) / tau, s = sum 2^u and w = sum 2^u u over the row,
//   log_probs = ln2 u_y - ln s,  entropy = ln s - ln2 w / s.
//
// One pass over the logits, which bound it.  A row goes to a cluster of 1 to 8 CTAs (so that a few rows
// reach many SMs, without a second launch); each thread walks its share of the CTA's part with 16-byte loads, four at a
// time, with running statistics and nothing to wait for; the alternatives come out of the shares whose maxima are
// large (topk.cuh).  The first CTA of the cluster joins the parts through distributed shared memory.
#include "launch_util.cuh"
#include "tc5.cuh"
#include "topk.cuh"

namespace swx {

constexpr int TL_LOADS = 4, TL_PER = 8, TL_MAX_PARTS = 8;
constexpr float TL_LN2 = 0.69314718055994531f;

struct TokenRows {
    int64_t V, stride;
    int parts, top;
    const void* z; const int64_t* target; int64_t ignore;
    float k2, inv_temp;
    float* log_probs; float* entropy; float* top_log_probs; int64_t* top_ids;
};

__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// Piece i of the row, N logits from column i N - shift on: -inf outside it.
template <typename T, int N = 16 / sizeof(T)>
__device__ __forceinline__ void load_piece(const T* z, int64_t V, int shift, int64_t i, float (&v)[N]) {
    const int64_t c = i * N - shift;
    if (c >= 0 && c + N <= V) {
        const uint4 q = *reinterpret_cast<const uint4*>(z + c);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = Elem<T>::to_f(reinterpret_cast<const T*>(&q)[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = c + k >= 0 && c + k < V ? Elem<T>::to_f(z[c + k]) : -INFINITY;
    }
}

template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS) token_logprob_kernel(const TokenRows p) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ Score part[THREADS / 32];
    __shared__ Score whole;
    __shared__ int count[2], found, owners[THREADS];
    __shared__ uint32_t scratch[THREADS + 1];
    constexpr int N = 16 / sizeof(T);          // logits of a 16-byte load
    const int64_t row = blockIdx.x / p.parts;
    const int rank = blockIdx.x % p.parts, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const T* z = static_cast<const T*>(p.z) + row * p.stride;

    // The row in 16-byte pieces counted from the last boundary at or before its start; the first and the last may be cut
    const int shift = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    const int64_t pieces = (p.V + shift + N - 1) / N, per = (pieces + p.parts - 1) / p.parts;
    const int64_t begin = rank * per, end = min(pieces, begin + per);
    Score a{-INFINITY, 0.f, 0.f};
    float v[TL_LOADS][N];
    if (threadIdx.x == 0) count[0] = count[1] = 0;
    for (int64_t i0 = begin + threadIdx.x; i0 < end; i0 += TL_LOADS * THREADS) {
#pragma unroll
        for (int j = 0; j < TL_LOADS; ++j) {
            if (i0 + j * THREADS < end) load_piece<T>(z, p.V, shift, i0 + j * THREADS, v[j]);
            else {
#pragma unroll
                for (int k = 0; k < N; ++k) v[j][k] = -INFINITY;
            }
        }
        float nm = a.m;
#pragma unroll
        for (int j = 0; j < TL_LOADS; ++j)
#pragma unroll
            for (int k = 0; k < N; ++k) nm = fmaxf(nm, v[j][k]);
        const float base = nm == -INFINITY ? 0.f : nm;                   // nothing but -inf so far: the sums stay 0
        const float da = fmaxf((a.m - base) * p.k2, SCORE_FAR), ca = ex2(da);
        float2 s = make_float2(ca * a.s, 0.f), w = make_float2(ca * (a.w + a.s * da), 0.f);
        a.m = nm;
#pragma unroll
        for (int j = 0; j < TL_LOADS; ++j)
#pragma unroll
            for (int k = 0; k < N; k += 2) {
                const float2 u = mul2(add2(f2(v[j][k], v[j][k + 1]), bc2(-base)), bc2(p.k2)), e = ex2x2(u);
                s = add2(s, e);
                w = fma2(e, f2(fmaxf(u.x, SCORE_FAR), fmaxf(u.y, SCORE_FAR)), w);
            }
        a.s = s.x + s.y;
        a.w = w.x + w.y;
    }
    // the share's largest; a NaN or +inf in it asks for no threshold
    const uint32_t most = begin + threadIdx.x >= end ? 0 : a.s != a.s ? ~0u : order_key(a.m);
    score_join_warp(a, p.k2);
    if (lane == 0) part[warp] = a;
    uint64_t* buf = reinterpret_cast<uint64_t*>(raw);
    uint64_t* kept = buf + topk_capacity(p.top, TL_PER);
    TopK<THREADS, TL_PER> best(buf, kept, count, p.top);
    if constexpr (TOP) {
        struct Piece { float v[N]; int64_t c; };
        auto load = [&](int t, int64_t j, Piece& e) {
            const int64_t i = begin + t + j * THREADS;
            e.c = i < end ? i * N - shift : p.V;
            if (i < end) load_piece<T>(z, p.V, shift, i, e.v);
        };
        auto emit = [&](const Piece& e, auto f) {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (e.c + k >= 0 && e.c + k < p.V) f(e.v[k], (uint32_t)(e.c + k));
        };
        auto each = [&](auto f) {
#pragma unroll
            for (int j = 0; j < TL_LOADS; ++j) {
                const int64_t i = begin + threadIdx.x + j * THREADS, c = i * N - shift;
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if (i < end && c + k >= 0 && c + k < p.V) f(v[j][k], (uint32_t)(c + k));
            }
        };
        // (a part of one batch is still in registers)
        const bool ok = end - begin <= TL_LOADS * THREADS
                            ? best.gather_held(most, scratch, each)
                            : best.template gather<Piece>(most, scratch, owners, (per + THREADS - 1) / THREADS, load, emit);
        if (!ok) {
            best.clear();
            for (int64_t i0 = begin; i0 < end; i0 += THREADS * (TL_PER / N)) {
                uint64_t key[TL_PER];
#pragma unroll
                for (int j = 0; j < TL_PER / N; ++j) {
                    const int64_t i = i0 + j * THREADS + threadIdx.x, c = i * N - shift;
                    float u[N];
                    if (i < end) load_piece<T>(z, p.V, shift, i, u);
#pragma unroll
                    for (int k = 0; k < N; ++k)
                        key[j * N + k] = i < end && c + k >= 0 && c + k < p.V ? index_key(order_key(u[k]), (uint32_t)(c + k)) : 0;
                }
                best.push(key);
            }
        }
        best.order();
    } else {
        __syncthreads();
    }
    a = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) score_join(a, part[i], p.k2);
    if (p.parts > 1) {
        if (threadIdx.x == 0) { whole = a; found = best.n; }
        cluster_sync_all();
        if (rank == 0) {
            for (int r = 1; r < p.parts; ++r) {
                const uint32_t o = map_to_rank(&whole, r);
                score_join(a, Score{ld_cluster_f32(o), ld_cluster_f32(o + 4), ld_cluster_f32(o + 8)}, p.k2);
            }
            if (TOP) {
                // the parts' largest, into the buffer (it holds more than 8 k keys), and their order
                int n = 0;
                for (int r = 0; r < p.parts; ++r) {
                    const int m = __float_as_int(ld_cluster_f32(map_to_rank(&found, r)));
                    const uint32_t from = map_to_rank(kept, r);
                    for (int i = threadIdx.x; i < m; i += THREADS) buf[n + i] = ld_cluster_u64(from + 8 * i);
                    n += m;
                }
                best.n = n;
                __syncthreads();
                best.order();
            }
        }
        cluster_sync_all();                    // no CTA goes while the first still reads its shared memory
        if (rank != 0) return;
    }
    const float ls = logf(a.s);
    const int64_t y = p.target ? p.target[row] : 0;
    const bool live = !p.target || y != p.ignore;
    if (threadIdx.x == 0) {
        if (p.target)
            p.log_probs[row] = !live ? 0.f : y >= 0 && y < p.V ? (Elem<T>::to_f(z[y]) - a.m) * p.inv_temp - ls : __int_as_float(0x7fc00000);
        p.entropy[row] = live ? ls - TL_LN2 * a.w / a.s : 0.f;
    }
    if (TOP) {
        for (int i = threadIdx.x; i < p.top; i += THREADS) {
            const uint64_t k = kept[i];
            p.top_log_probs[row * p.top + i] = live ? (order_value((uint32_t)(k >> 32)) - a.m) * p.inv_temp - ls : 0.f;
            p.top_ids[row * p.top + i] = live ? (int64_t)key_index(k) : -1;
        }
    }
}

// CTAs for each row: enough to reach every SM twice, 4096 logits each or more.
static int token_parts(int64_t rows, int64_t V) {
    int parts = 1;
    while (parts < TL_MAX_PARTS && rows * parts < 296 && V / (2 * parts) >= 4096) parts *= 2;
    return parts;
}

template <typename T, bool TOP, int THREADS>
static cudaError_t launch_token(const TokenRows& p, int64_t rows, cudaStream_t st) {
    auto k = token_logprob_kernel<T, TOP, THREADS>;
    const size_t smem = TOP ? (size_t)(topk_capacity(p.top, TL_PER) + p.top) * 8 : 0;
    static_assert((topk_capacity(SWX_MAX_TOP, TL_PER) + SWX_MAX_TOP) * 8 <= 40 * 1024, "more shared memory than a launch has by itself");
    if (p.parts == 1) {
        k<<<(unsigned)rows, THREADS, smem, st>>>(p);
        return cudaGetLastError();
    }
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(rows * p.parts));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)p.parts;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, k, p);
}

// Short parts take small CTAs (more of them at a time): 4096 rows of 4096 fp32 logits, 20 alternatives, 128 threads 34.6 us, 256
// 45; 1024 x 32768 bf16 29.7 and 33.5; 64 x 50001 fp32 in parts of 50 KB 19.8 and 17.2.  A threshold takes twice as many threads as alternatives.
template <typename T, bool TOP>
static cudaError_t launch_token(const TokenRows& p, int64_t rows, cudaStream_t st) {
    const int64_t bytes = p.V * (int64_t)sizeof(T) / p.parts;
    if (bytes <= 8192 && p.top <= 32) return launch_token<T, TOP, 64>(p, rows, st);
    if (bytes <= 65536 && p.top <= 64 && rows * p.parts > 592) return launch_token<T, TOP, 128>(p, rows, st);
    return launch_token<T, TOP, 256>(p, rows, st);
}

}  // namespace swx

using namespace swx;

extern "C" int swx_token_logprob(const swx_logprob_args* a, void* stream) {
    if (!a || a->tokens < 0 || a->vocab < 1 || a->top_k < 0 || a->top_k > a->vocab) return SWX_ERR_INVALID_ARG;
    if (!(a->temperature > 0.f) || a->temperature > 1e15f || a->temperature < 1e-15f) return SWX_ERR_INVALID_ARG;
    if (a->dtype != SWX_DTYPE_F32 && a->dtype != SWX_DTYPE_BF16) return SWX_ERR_UNSUPPORTED;
    if (a->tokens > (1 << 27) || a->vocab > (1 << 28) || a->top_k > SWX_MAX_TOP) return SWX_ERR_UNSUPPORTED;
    if (a->tokens == 0) return SWX_OK;
    if (!a->x || !a->entropy || (a->targets && !a->log_probs) || (a->top_k > 0 && (!a->top_log_probs || !a->top_ids))) return SWX_ERR_INVALID_ARG;
    TokenRows p{};
    p.V = a->vocab; p.stride = a->x_sr; p.top = a->top_k; p.z = a->x; p.target = a->targets; p.ignore = a->ignore_index;
    p.inv_temp = 1.f / a->temperature; p.k2 = LOG2E / a->temperature;
    p.log_probs = a->log_probs; p.entropy = a->entropy; p.top_log_probs = a->top_log_probs; p.top_ids = a->top_ids;
    p.parts = token_parts(a->tokens, a->vocab);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf = a->dtype == SWX_DTYPE_BF16;
    const cudaError_t e = a->top_k > 0 ? (bf ? launch_token<__nv_bfloat16, true>(p, a->tokens, st) : launch_token<float, true>(p, a->tokens, st))
                                       : (bf ? launch_token<__nv_bfloat16, false>(p, a->tokens, st) : launch_token<float, false>(p, a->tokens, st));
    return e == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
}
