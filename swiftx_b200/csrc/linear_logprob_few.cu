// The scoring of a few tokens (linear_logprob.cu's products and records for up to 8 rows, bf16): the weight is read once from
// HBM, which bounds it, straight into the A operand of mma.sync; there is nothing for a tile of 256 rows to share.
//
// A CTA of four warps takes groups of 16 words in turn.  Its warps split the width: lane (g, c) reads 16 bytes of words g and
// g + 8 from 8 c on of each 32 steps (all loads of a group are in flight together, 32 KB at a width of 1024) and the tokens'
// values in the same order from shared memory (a sum does not see the order of its terms).  The warps' sums meet in shared
// memory; thread (token, word) then keeps running statistics of its logits, and each half warp writes the group's two
// largest.
#include "head_gemm.cuh"
#include "warp_mma.cuh"

namespace swx {

constexpr int SF_WARPS = 4, SF_THREADS = 32 * SF_WARPS, SF_DEPTH = 8;   // steps of 32 values whose loads a warp issues together
constexpr int SF_PER_SM = 4;

template <bool TOP>
__global__ void __launch_bounds__(SF_THREADS, SF_PER_SM) score_few_kernel(const XentGemm p, const __nv_bfloat16* x, int64_t x_sr, const __nv_bfloat16* w, int64_t w_sr,
                                                               int64_t d) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ float sums[2][SF_WARPS][8][17];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    const int steps = (int)((d + 31) / 32);
    const int t = threadIdx.x / 16, word = threadIdx.x % 16;    // this thread's token, and its word of each group
    const int64_t y = t < p.M ? p.target[t] : -1;
    Score a{-INFINITY, 0.f, 0.f};
    const int64_t groups = ((int64_t)p.N + 15) / 16;
    int buf = 0;
    // steps s0, s0 + 1, ... of a group's words (512 bytes of a row together); the next group's are on their way while this one's sums are joined
    uint4 v0[SF_DEPTH], v1[SF_DEPTH];
    auto fetch = [&](int64_t q, int s0) {
        const __nv_bfloat16* w0 = w + min(16 * q + g, (int64_t)p.N - 1) * w_sr;
        const __nv_bfloat16* w1 = w + min(16 * q + 8 + g, (int64_t)p.N - 1) * w_sr;
#pragma unroll
        for (int i = 0; i < SF_DEPTH; ++i) {
            const int s = s0 + i;
            const int64_t k = 32 * (int64_t)s + 8 * c;
            if (s < steps) {
                v0[i] = load8(w0, k, d);
                v1[i] = load8(w1, k, d);
            }
        }
    };
    fetch(blockIdx.x, SF_DEPTH * warp);
    // the tokens' values, rows of 64 bytes a step and 64 more, so that the 8 rows of a load lie in different banks
    uint4* sx = reinterpret_cast<uint4*>(raw);
    const int stride = 4 * steps + 4;
    for (int i = threadIdx.x; i < 8 * 4 * steps; i += SF_THREADS) {
        const int r = i / (4 * steps), k = i % (4 * steps);
        sx[r * stride + k] = r < p.M ? load8(x + r * x_sr, 8 * (int64_t)k, d) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    for (int64_t q = blockIdx.x; q < groups; q += gridDim.x, buf ^= 1) {
        float acc[4] = {};
        for (int s0 = SF_DEPTH * warp;;) {
#pragma unroll
            for (int i = 0; i < SF_DEPTH; ++i) {
                const int s = s0 + i;
                if (s >= steps) continue;
                const uint32_t a0[4] = {v0[i].x, v1[i].x, v0[i].y, v1[i].y}, a1[4] = {v0[i].z, v1[i].z, v0[i].w, v1[i].w};
                const uint4 b = sx[g * stride + 4 * s + c];
                const uint32_t b0[2] = {b.x, b.y}, b1[2] = {b.z, b.w};
                mma_bf16(acc, a0, b0);
                mma_bf16(acc, a1, b1);
            }
            s0 += SF_DEPTH * SF_WARPS;
            if (s0 >= steps) break;
            fetch(q, s0);
        }
        if (q + gridDim.x < groups) fetch(q + gridDim.x, SF_DEPTH * warp);
        sums[buf][warp][2 * c][g] = acc[0];
        sums[buf][warp][2 * c + 1][g] = acc[1];
        sums[buf][warp][2 * c][8 + g] = acc[2];
        sums[buf][warp][2 * c + 1][8 + g] = acc[3];
        __syncthreads();                       // (two buffers: the next group's sums go to the other one)
        float z = sums[buf][0][t][word];
#pragma unroll
        for (int j = 1; j < SF_WARPS; ++j) z += sums[buf][j][t][word];
        const int64_t v = 16 * q + word;
        const bool in = v < p.N;
        if (in && t < p.M && v == y) p.hit[t] = z;
        if (in) {
            const float m = fmaxf(a.m, z), base = m == -INFINITY ? 0.f : m;
            score_move(a, base, p.k2);
            const float u = (z - base) * p.k2, e = ex2(u);
            a.m = m;
            a.s += e;
            a.w += e * fmaxf(u, SCORE_FAR);
        }
        if (TOP) {
            // the half warp's largest and its lowest column, and the largest of the others
            const float f = in ? fmaxf(z, SCORE_FLOOR) : SCORE_FLOOR;
            float most = f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const uint32_t at = __ballot_sync(0xffffffffu, f == most) >> (lane & 16) & 0xffffu;
            const int col = __ffs(at) - 1;
            float second = word == col ? SCORE_FLOOR : f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) second = fmaxf(second, __shfl_xor_sync(0xffffffffu, second, o));
            if (word == 0 && t < p.M) {
                p.largest[(int64_t)t * 16 * p.nt + q] = most;
                p.runner_up[(int64_t)t * 16 * p.nt + q] = __uint_as_float((__float_as_uint(second) & ~15u) | (uint32_t)col);
            }
        }
    }
    // this CTA's statistics of each token
    float m = a.m;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    score_move(a, m, p.k2);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
    }
    if (word == 0 && t < p.M) p.score[(int64_t)t * gridDim.x + blockIdx.x] = make_float4(m, a.s, a.w, 0.f);
}

// A warp's sums are of 8 steps (two products each) of every 32: their numbers of additions, weighed by the terms that they hold.
double few_additions(int64_t d) {
    const int64_t steps = (d + 31) / 32;
    double n = 0.;
    for (int w = 0; w < SF_WARPS; ++w) {
        const int64_t rest = steps % (SF_DEPTH * SF_WARPS) - SF_DEPTH * w;
        const double s = (double)(steps / (SF_DEPTH * SF_WARPS) * SF_DEPTH + std::max<int64_t>(0, std::min<int64_t>(rest, SF_DEPTH)));
        n += 2. * s * s / (double)steps;
    }
    return n;
}

static int few_smem(int64_t d) { return 8 * (int)(4 * ((d + 31) / 32) + 4) * 16; }

// CTAs of the kernel for these sizes (each leaves one statistic of a token); 0: not taken.
// bf16 rows up to 8 tokens whose values fit in shared memory beside other CTAs': 1 and 8 tokens of 50001 x 1024 take 24 and 28 us without
// alternatives and 32 and 34 with 5 (both kernels in a graph, the weight not in the L2; called eagerly 3 more), 9 tokens on 256-row
// tiles 34 and 43.  A vocabulary of 2048 and less is a few tiles there.
int score_few_ctas(const HeadOps& o) {
    if (o.dtype != SWX_DTYPE_BF16 || o.T > 8 || o.V <= 2048 || few_smem(o.d) > 72 * 1024) return 0;
    const int per_sm = std::min(SF_PER_SM, (200 * 1024) / (few_smem(o.d) + 6 * 1024));
    return (int)std::min<int64_t>((o.V + 15) / 16, 148 * per_sm);
}

template <bool TOP>
static cudaError_t launch_few(const XentGemm& g, const HeadOps& o, const Operand& x, const Operand& w, int ctas, cudaStream_t st) {
    const cudaError_t e = allow_smem(score_few_kernel<TOP>, 72 * 1024);
    if (e != cudaSuccess) return e;
    score_few_kernel<TOP><<<ctas, SF_THREADS, few_smem(o.d), st>>>(g, static_cast<const __nv_bfloat16*>(x.p), x.row,
                                                                           static_cast<const __nv_bfloat16*>(w.p), w.row, o.d);
    return cudaGetLastError();
}

cudaError_t launch_score_few(const XentGemm& g, const HeadOps& o, const Operand& x, const Operand& w, bool top, int ctas, cudaStream_t st) {
    return top ? launch_few<true>(g, o, x, w, ctas, st) : launch_few<false>(g, o, x, w, ctas, st);
}

}  // namespace swx
