// The products of a linear head over a large vocabulary, for the operators that never keep its
// logits (linear_xent.cu, linear_logprob.cu, linear_distill.cu): one matrix product kernel whose
// epilogue turns a tile of logits into what the operator keeps, and the host side of it.
//
// A persistent grid of CTA pairs, 256 x 256 tiles, operands staged by TMA into a ring, tcgen05
// products issued by one thread per pair into two alternating accumulators in tensor memory, and eight
// warps per CTA that read an accumulator while the next tile is computed.  linear_xent.cu holds the
// figures and the kernels that every operator shares (gradient products, operand layout).
#pragma once
#include <algorithm>

#include "common.cuh"
#include "launch_util.cuh"
#include "tc5.cuh"
#include "tma_util.cuh"
#include "topk.cuh"

namespace swx {

constexpr int XE_TILE = 256;                  // rows and columns of a pair's tile
constexpr int XE_K = 64;                      // contraction steps per ring stage (128 bytes of bf16)
constexpr int XE_STAGES = 6;
constexpr int XE_OPERAND = 128 * XE_K * 2;    // bytes of one operand of one CTA in a stage
constexpr int XE_STAGE = 2 * XE_OPERAND;
constexpr int XE_EPI_WARPS = 8;
constexpr int XE_THREADS = 64 + 32 * XE_EPI_WARPS;
constexpr int XE_OUT = 32 * 128;              // staging bytes of one epilogue warp: 32 rows x 128 bytes
constexpr int XE_SMEM = 1024 + XE_STAGES * XE_STAGE + XE_EPI_WARPS * XE_OUT;
// fp32 operands: stages summed in tensor memory at a time.  The tensor core cuts the low bits
// of each addition off (toward zero), an error that grows with the number of additions (dx
// 4.9e-6 off after 5001 terms in one sum); sums of 256 terms are added up in fp32 instead.
constexpr int XE_KSUB = 4;
// The same for the logits, over the width of the operands, 512 terms at a time: up to that nothing is summed outside
// (3.9e-7 off at operands of one sign, a library's fp32 products 4.8e-7); in one sum 1024 terms were 1.3e-6 off, 4096 8.7e-6
// and 16384 6.6e-5, 4e-7 each now.  2048 x 8192 x 1024 forward 148 -> 163 us; 256 terms at a time 176, and 384 instead of 326 us
// at 4096 x 20000 x 512.
constexpr int XE_KSUB_LOGITS = 8;
constexpr uint32_t XE_POLLS = 1u << 24;       // about a second

// Epilogues: XE_LSE (loss) and XE_SCORE* (log probabilities: statistics of scaled logits, with the entropy's sum; for the top
// alternatives also the two largest logits of 16 columns, or the logits themselves; for distillation the logits at each row's
// words) read logits, XE_PROB and XE_GRAD* write the logits' gradient (XE_GRAD_IDS: with a row's words apart), XE_DX and XE_DW are
// the gradient products.
enum XentEpi { XE_LSE, XE_PROB, XE_DX, XE_DW, XE_SCORE, XE_SCORE_TOP, XE_SCORE_ALL, XE_SCORE_IDS, XE_GRAD, XE_GRAD_IDS };
constexpr bool is_score(int epi) { return epi == XE_SCORE || epi == XE_SCORE_TOP || epi == XE_SCORE_ALL || epi == XE_SCORE_IDS; }
constexpr bool is_grad(int epi) { return epi == XE_GRAD || epi == XE_GRAD_IDS; }
constexpr bool is_dlogit(int epi) { return epi == XE_PROB || is_grad(epi); }
constexpr bool has_ids(int epi) { return epi == XE_SCORE_IDS || epi == XE_GRAD_IDS; }
constexpr bool is_logits(int epi) { return epi == XE_LSE || is_score(epi) || is_dlogit(epi); }
constexpr float SCORE_FLOOR = -0x1.ffffep127f;   // the records' lowest value: finite with any column in its low 4 bits
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

struct XentGemm {
    int M, N;                                 // rows and columns of the result
    int mt, nt, group;                        // tiles; row tiles walked together (logits)
    int nk, npair;                            // ring stages of the contraction; pairs of pieces
    int ksub;                                 // stages summed in tensor memory before the sum moves on
    int ka0, kb0;                             // first contraction index of A and of B
    int a0, b0;                               // first row of A and of B (M / N coordinate)
    int* status;
    // logits
    const int64_t* target;
    int64_t ignore;
    int64_t vocab;
    int col0;                                 // vocabulary index of column 0
    float2* part;                             // (2 nt, M): max and sum of a tile half's exponentials
    float* hit;                               // (M): the target's logit
    int* counter;                             // zeroed by the forward epilogues (where given) for the kernel after them
    const float* row_max; const float* row_rsum;
    const float* dloss; int reduction;
    int planes;                               // bf16 pieces of the dlogit
    // XE_DX / XE_DW
    // spread: the steps of all tiles are dealt out evenly and a tile's parts are summed in
    // acc[part][M][N]; else whole tiles go round and the last piece writes the result
    int spread;
    float* acc; void* out; int out_bf16; int64_t ld; int first, last;
    const float* scale_num; const float* scale_den;   // the result's factor: num / den, either may be absent
    // XE_SCORE*, XE_GRAD: exponents are (logit - m) * k2, k2 = log2(e) / temperature, m the largest logit.  The difference comes first,
    // so that the largest term is 1 at any temperature (with m k2 rounded and one fused operation for each exponent, its residual, a 2^-24th of
    // |m| k2, went into the sums: 2^500 at a temperature of 1e-8)
    float k2, inv_temp;
    float4* score;                            // (M, 2 nt): a tile half's m, sum of exponentials e, sum of e times its exponent
    // XE_SCORE_TOP, (M, 16 nt): the largest logit of 16 columns, and the second with the largest one's column in place of its
    // low 4 bits; SCORE_FLOOR stands for -inf, NaN and columns from N on
    float* largest; float* runner_up;
    float* all;                               // XE_SCORE_ALL, (M, N)
    int beside;                               // the next kernel (the words' norms) may start beside this one
    // XE_SCORE_IDS, XE_GRAD_IDS: each row's words in rising order, their logits and shares, (M, nids), and how many of them lie before
    // each 128 columns of the vocabulary, (M, stride)
    const int* ids; float* id_logit; const float* id_share; const uint8_t* before; int nids, before_stride;
    // XE_GRAD: dlogit = 2^u (A + B u) + [column == target] hot, see grad_row
    const float* row_sum; const float* entropy; const float* d_logp; const float* d_entropy;
};

// Pieces of A and B multiplied in turn (index: plane of the 3-D tensor map), smallest
// products first, so that few additions happen at the sum's full magnitude.
__device__ __forceinline__ int2 piece_pair(int npair, int i) {
    if (npair == 1) return make_int2(0, 0);
    constexpr uint32_t A = 2u | 1u << 2 | 0u << 4 | 1u << 6 | 0u << 8 | 0u << 10;
    constexpr uint32_t B = 0u | 1u << 2 | 2u << 4 | 0u << 6 | 1u << 8 | 0u << 10;
    return make_int2((A >> (2 * i)) & 3, (B >> (2 * i)) & 3);
}

// The work of one CTA pair: runs of contraction steps [k0, k1) of a tile, each summed in one
// accumulator.  Whole tiles go round the pairs; spread, pair c takes the steps
// [c S / P, (c + 1) S / P) of the S steps of all tiles, so that a tile can have several parts
// (numbered from the pair that has the tile's first step).
struct XentRuns {
    int64_t cur, end, tile;
    int nk, ksub, P, k0, k1, part;
    bool spread, fresh;
    __device__ __forceinline__ XentRuns(const XentGemm& p, int64_t c, int64_t P_) : nk(p.nk), ksub(p.ksub), P((int)P_), part(0), spread(p.spread) {
        const int64_t tiles = (int64_t)p.mt * p.nt;
        cur = spread ? c * (tiles * nk) / P : c;
        end = spread ? (c + 1) * (tiles * nk) / P : tiles;
        k1 = nk;
        fresh = true;
        tile = -1;
    }
    __device__ __forceinline__ bool next(const XentGemm& p) {
        if (cur >= end) return false;
        if (spread) {
            const int64_t t = cur / nk;
            k0 = (int)(cur - t * nk);
            k1 = (int)min((int64_t)min(nk, k0 + ksub), k0 + (end - cur));
            fresh = t != tile;
            if (fresh) {
                const int64_t total = (int64_t)p.mt * p.nt * nk;
                const int64_t c = ((cur + 1) * P - 1) / total, lo = ((t * nk + 1) * P - 1) / total;
                part = (int)(c - lo);
            }
            tile = t;
            cur += k1 - k0;
        } else {
            tile = cur;
            k0 = k1 < nk ? k1 : 0;
            fresh = k0 == 0;
            k1 = min(k0 + ksub, nk);
            if (k1 == nk) cur += P;
        }
        return true;
    }
};

// Tile t -> (row tile, column tile).  Logits: `group` row tiles of x stay in L2
// while the weight's column tiles pass by; the gradients: a row tile's column tiles together.
template <int EPI>
__device__ __forceinline__ int2 tile_of(const XentGemm& p, int64_t t) {
    if (is_logits(EPI)) {
        const int64_t per = (int64_t)p.group * p.nt;
        const int g = (int)(t / per);
        const int rows = min(p.group, p.mt - g * p.group);
        const int64_t r = t - g * per;
        return make_int2(g * p.group + (int)(r % rows), (int)(r / rows));
    }
    return make_int2((int)(t / p.nt), (int)(t % p.nt));
}

// Factor of a row's dlogit.  A mean's or a sum's upstream gradient is one number for all
// rows; it multiplies the gradients at the end instead, so that the target's column, near -1,
// is rounded near a power of two (with the factor inside, every row's -1/n was rounded the
// same way and the gradients were 3.1e-3 off, 1.9e-3 now, 256 tokens).
__device__ __forceinline__ float row_scale(const XentGemm& p, int row) {
    const int64_t y = p.target[row];
    if (y == p.ignore) return 0.f;
    if (y < 0 || y >= p.vocab) return __int_as_float(0x7fc00000);
    return p.reduction == SWX_XENT_NONE ? p.dloss[row] : 1.f;
}

// A row's coefficients of XE_GRAD.  With u = (z - m) k2, e = 2^u, s the sum of e: p = e / s, the log probability
// l = u ln2 - ln s, and for upstream gradients g of the target's log probability and h of the entropy H
//   dz = (g [v == y] - p (g + h (l + H))) / temperature = e (A + B u) + [v == y] hot.
// Distillation (no targets): dz = (p - Q) c / temperature with c = temperature^2 times the row's upstream gradient and Q the
// word's share, if it is one of the teacher's.
struct GradRow { float A, B, hot; };
__device__ __forceinline__ GradRow grad_row(const XentGemm& p, int row) {
    const float s = p.row_sum[row];
    if (!p.target) {                          // (XE_GRAD_IDS: at a row's words, less their share of c temperature)
        const float c = p.reduction == SWX_XENT_NONE ? p.dloss[row] : 1.f;
        return GradRow{s > 0.f ? c / (p.inv_temp * s) : s < 0.f ? 0.f : __int_as_float(0x7fc00000), 0.f, 0.f};     // s < 0: a row that does not count
    }
    const int64_t y = p.target[row];
    if (y == p.ignore) return GradRow{0.f, 0.f, 0.f};
    if (y < 0 || y >= p.vocab) return GradRow{__int_as_float(0x7fc00000), 0.f, 0.f};
    const float g = p.d_logp ? p.d_logp[row] : 0.f, h = p.d_entropy ? p.d_entropy[row] : 0.f;
    const float f = p.inv_temp / s;
    return GradRow{-f * (g + h * (p.entropy[row] - logf(s))), -f * h * 0.69314718055994531f, p.inv_temp * g};
}

// 32 columns of a row of a gradient (from cc on), to the running sum in memory or, the last time, to the result.
__device__ __forceinline__ void xent_emit(const XentGemm& p, float (&v)[32], int part, int row, int cc, bool first, bool last, float factor) {
    const int n = min(32, p.N - cc);
    float* acc = p.acc + ((int64_t)part * p.M + row) * p.N + cc;
    const bool whole = n == 32 && (reinterpret_cast<uintptr_t>(acc) & 15) == 0;
    if (!first) {
        if (whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float4 q = reinterpret_cast<const float4*>(acc)[j];
                v[4 * j] += q.x; v[4 * j + 1] += q.y; v[4 * j + 2] += q.z; v[4 * j + 3] += q.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) if (j < n) v[j] += acc[j];
        }
    }
    if (last) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= factor;
    }
    if (!last) {
        if (whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                reinterpret_cast<float4*>(acc)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) if (j < n) acc[j] = v[j];
        }
    } else if (p.out_bf16) {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + (int64_t)row * p.ld + cc;
        if (n == 32 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[8 * j + 2 * k], v[8 * j + 2 * k + 1]);
                    w[k] = *reinterpret_cast<const uint32_t*>(&b2);
                }
                reinterpret_cast<uint4*>(o)[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) if (j < n) o[j] = __float2bfloat16_rn(v[j]);
        }
    } else {
        float* o = static_cast<float*>(p.out) + (int64_t)row * p.ld + cc;
        if (n == 32 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                reinterpret_cast<float4*>(o)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) if (j < n) o[j] = v[j];
        }
    }
}

// SUMS: the steps of a tile come in several accumulators (fp32 operands: the gradients, and logits of wide operands); their sum stays in registers until the tile (or
// this pair's part of it) is complete: through memory each time, 1003 tokens x 10007 x 200 took 232 us, 219 with the registers.
template <int EPI, bool A_MN, bool B_MN, bool SUMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(XE_THREADS, 1)
xent_gemm_kernel(const XentGemm p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[XE_STAGES], empty[XE_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base;
    uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023) & ~1023u) - smem_u32(smem_raw));
    uint8_t* stage_out = smem + XE_STAGES * XE_STAGE;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_rank();
    const int64_t cluster = blockIdx.x / 2, nclusters = gridDim.x / 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < XE_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(&acc_full[a], 1); mbar_init(&acc_empty[a], 2 * XE_EPI_WARPS); }
        mbar_fence_init();
        if ((EPI == XE_LSE || (is_score(EPI) && p.counter)) && blockIdx.x == 0) *p.counter = 0;
    }
    if (warp == 1) tmem_alloc_pair(&tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    if ((EPI == XE_SCORE_TOP || EPI == XE_SCORE_ALL) && p.beside) let_next_start();

    if (warp == 0) {
        if (lane == 0) {
            // ---- loads: this CTA's half of the rows of A and B, counted on the leader's barrier
            int s = 0;
            uint32_t ph = 0;
            int64_t issued = 0;
            bool ok = true;
            for (XentRuns r(p, cluster, nclusters); ok && r.next(p);) {
                const int2 rc = tile_of<EPI>(p, r.tile);
                const int am = p.a0 + rc.x * XE_TILE + (int)rank * 128, bn = p.b0 + rc.y * XE_TILE + (int)rank * 128;
                for (int i = 0; ok && i < p.npair; ++i) {
                    const int2 pl = piece_pair(p.npair, i);
                    for (int k = r.k0; k < r.k1; ++k) {
                        if (!mbar_wait_cluster(&empty[s], ph ^ 1, XE_POLLS)) { ok = false; break; }
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * XE_STAGE);
                        const uint32_t bar = map_to_rank(&full[s], 0);
                        uint8_t* sa = smem + s * XE_STAGE;
                        uint8_t* sb = sa + XE_OPERAND;
                        const int ka = p.ka0 + k * XE_K, kb = p.kb0 + k * XE_K;
                        if (A_MN) {
                            tma_load_3d_pair(sa, &map_a, am, ka, pl.x, bar);
                            tma_load_3d_pair(sa + XE_OPERAND / 2, &map_a, am + 64, ka, pl.x, bar);
                        } else {
                            tma_load_3d_pair(sa, &map_a, ka, am, pl.x, bar);
                        }
                        if (B_MN) {
                            tma_load_3d_pair(sb, &map_b, bn, kb, pl.y, bar);
                            tma_load_3d_pair(sb + XE_OPERAND / 2, &map_b, bn + 64, kb, pl.y, bar);
                        } else {
                            tma_load_3d_pair(sb, &map_b, kb, bn, pl.y, bar);
                        }
                        ++issued;
                        if (++s == XE_STAGES) { s = 0; ph ^= 1; }
                    }
                }
            }
            // every stage's copies have landed (both CTAs' bytes count on the leader's barrier)
            // and every product that reads this CTA's ring has finished before it goes
            for (int q = 0; q < XE_STAGES; ++q) {
                const int64_t uses = (issued + XE_STAGES - 1 - q) / XE_STAGES;
                if (uses == 0) continue;
                const uint32_t par = (uint32_t)((uses - 1) & 1);
                if (rank == 0) ok = mbar_wait_cluster(&full[q], par, XE_POLLS) && ok;
                ok = mbar_wait_cluster(&empty[q], par, XE_POLLS) && ok;
            }
            if (!ok && p.status) *p.status = SWX_ERR_TIMEOUT;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // ---- products, for both CTAs (the whole warp, one lane of it issuing)
            constexpr uint32_t idesc = mma_bf16_idesc(XE_TILE, XE_TILE, A_MN, B_MN);
            // 16 contraction steps further: 32 bytes along a K-major row, 16 rows of 128 bytes otherwise
            constexpr uint64_t da = (A_MN ? 2048 : 32) >> 4, db = (B_MN ? 2048 : 32) >> 4;
            int s = 0, a = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            for (XentRuns r(p, cluster, nclusters); ok && r.next(p);) {
                if (!mbar_wait_cluster(&acc_empty[a], aph ^ 1, XE_POLLS)) { ok = false; break; }
                tc_fence_after();
                const int steps = (r.k1 - r.k0) * p.npair;
                for (int i = 0; i < steps; ++i) {
                    if (!mbar_wait_cluster(&full[s], ph, XE_POLLS)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t ad = operand_desc(smem + s * XE_STAGE, XE_OPERAND / 2);
                    const uint64_t bd = operand_desc(smem + s * XE_STAGE + XE_OPERAND, XE_OPERAND / 2);
#pragma unroll
                    for (int q = 0; q < XE_K / 16; ++q)
                        mma_bf16_pair(tmem + a * XE_TILE, ad + q * da, bd + q * db, idesc, i > 0 || q > 0);
                    mma_commit_pair(&empty[s]);
                    if (++s == XE_STAGES) { s = 0; ph ^= 1; }
                }
                mma_commit_pair(&acc_full[a]);
                if ((a ^= 1) == 0) aph ^= 1;
            }
            if (!ok && p.status) *p.status = SWX_ERR_TIMEOUT;
        }
        __syncwarp();
    } else {
        // ---- epilogue: this lane's row of the accumulator, one 128-column half per warp
        const int sub = warp & 3, half = (warp - 2) / 4;
        uint8_t* so = stage_out + (warp - 2) * XE_OUT;
        int a = 0;
        uint32_t aph = 0;
        bool ok = true;
        int flip = 0;                         // which half of the staging memory the next store of three pieces takes
        float factor = 1.f;
        float tot[SUMS ? 4 : 1][32];
        if (EPI == XE_DX || EPI == XE_DW) {
            if (p.scale_num) factor = *p.scale_num;
            if (p.scale_den) factor = *p.scale_den > 0.f ? factor / *p.scale_den : 0.f;   // no token counts: no gradient
        }
        for (XentRuns r(p, cluster, nclusters); r.next(p);) {
            const bool last = p.last && !p.spread;
            const int2 rc = tile_of<EPI>(p, r.tile);
            const int row = rc.x * XE_TILE + (int)rank * 128 + sub * 32 + lane;
            const int c0 = rc.y * XE_TILE + half * 128;
            const bool live = row < p.M;
            // the row's target as a column of the result (anything outside it: no match)
            int64_t y = -1;
            float scale = 0.f, rmax = 0.f, rsum = 0.f;
            GradRow gr{0.f, 0.f, 0.f};
            if (is_logits(EPI) && live) {
                if (!(is_score(EPI) || is_grad(EPI)) || (!has_ids(EPI) && p.target)) y = p.target[row] - p.col0;
                if (is_grad(EPI)) {
                    gr = grad_row(p, row);
                    rmax = p.row_max[row];
                    if (EPI == XE_GRAD_IDS) rsum = p.row_sum[row];
                }
                if (EPI == XE_PROB) {
                    scale = row_scale(p, row);
                    rmax = p.row_max[row];
                    rsum = p.row_rsum[row] * scale;
                }
            }
            // the row's next word in this half of the tile: its entry, its column, its logit and share (while the products run; a search
            // among the words here instead of two counts made by then took 5 to 15 % of the product's time)
            int id = 0, id_end = 0, word = INT32_MAX;
            float word_z = 0.f, word_share = 0.f;
            const int64_t words = (int64_t)row * p.nids;
            auto fetch_word = [&] {
                word = INT32_MAX;
                if (id >= id_end) return;
                word = p.ids[words + id] - p.col0;
                if (is_grad(EPI)) {
                    word_z = p.id_logit[words + id];
                    word_share = p.id_share[words + id];
                }
            };
            if (has_ids(EPI) && live && c0 < p.N) {
                const uint8_t* b = p.before + (int64_t)row * p.before_stride + (p.col0 + c0) / 128;       // (a piece starts at a whole tile)
                id = b[0];
                id_end = b[1];
                fetch_word();
            }
            if (!mbar_wait_cluster(&acc_full[a], aph, XE_POLLS)) { ok = false; break; }
            tc_fence_after();
            const uint32_t at = tmem + ((uint32_t)(sub * 32) << 16) + a * XE_TILE + half * 128;
            // 32 columns of the row, from 32 c on
            float m = -INFINITY, sum = 0.f, esum = 0.f;
            float* groups = reinterpret_cast<float*>(so) + lane * 20;   // XE_SCORE_TOP: the 8 groups' largest and second logits
            // what the scoring keeps of this half of the tile (after the accumulator is given back: the stores need not be
            // waited for then)
            auto keep = [&] {
                if (!is_score(EPI) || !live) return;
                const int64_t at = (int64_t)row * 2 * p.nt + 2 * rc.y + half;
                p.score[at] = make_float4(m, sum, esum, 0.f);
                if (EPI == XE_SCORE_TOP) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        reinterpret_cast<float4*>(p.largest)[2 * at + i] = reinterpret_cast<const float4*>(groups)[i];
                        reinterpret_cast<float4*>(p.runner_up)[2 * at + i] = reinterpret_cast<const float4*>(groups)[2 + i];
                    }
                }
            };
            auto columns = [&](int c, float (&v)[32]) {
                const int cc = c0 + c * 32;                 // first of these 32 columns
                const int64_t yc = y - cc;
                if (EPI == XE_LSE) {
                    if (yc >= 0 && yc < 32) {
                        float h = 0.f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) h = yc == j ? v[j] : h;
                        if (y < p.N) p.hit[row] = h;
                    }
                    if (cc + 32 > p.N) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = cc + j < p.N ? v[j] : -INFINITY;
                    }
                    float top = v[0];
#pragma unroll
                    for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);
                    const float nm = fmaxf(m, top);
                    const float base = nm == -INFINITY ? 0.f : nm;      // nothing but -inf so far: sum stays 0
                    float add = 0.f;
#pragma unroll
                    for (int j = 0; j < 32; ++j) add += ex2((v[j] - base) * LOG2E);
                    sum = sum * ex2((m - base) * LOG2E) + add;
                    m = nm;
                } else if (is_score(EPI)) {
                    if (cc >= p.N) return;
                    if (yc >= 0 && yc < 32) {
                        float h = 0.f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) h = yc == j ? v[j] : h;
                        if (y < p.N) p.hit[row] = h;
                    }
                    if (EPI == XE_SCORE_IDS && __any_sync(0xffffffffu, word < cc + 32)) {
                        // the columns through shared memory (16-byte parts of a lane's row swapped about, against bank conflicts)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(so + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        while (word < cc + 32) {
                            const int j = word - cc;
                            p.id_logit[words + id] = *reinterpret_cast<const float*>(so + lane * 128 + (((j >> 2) ^ (lane & 7)) << 4) + (j & 3) * 4);
                            ++id;
                            fetch_word();
                        }
                        __syncwarp();
                    }
                    if (EPI == XE_SCORE_ALL && live) {
                        float* o = p.all + (int64_t)row * p.N + cc;
                        if (cc + 32 <= p.N && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) reinterpret_cast<float4*>(o)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) if (cc + j < p.N) o[j] = v[j];
                        }
                    }
                    if (cc + 32 > p.N) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = cc + j < p.N ? v[j] : -INFINITY;
                    }
                    float top = -INFINITY;
                    if constexpr (EPI == XE_SCORE_TOP) {
                        // the two largest of either half, with their columns in place of their low bits, and the largest as it
                        // is (-inf, which the column makes a NaN, and a NaN are no value's column; beside one the second may be as large as the
                        // largest, and the group is taken whole)
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            float t1 = SCORE_FLOOR, t2 = SCORE_FLOOR, most = -INFINITY;
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                const float x0 = v[16 * g + j], x1 = v[16 * g + j + 1];
                                const float p0 = __uint_as_float((__float_as_uint(x0) & ~15u) | j), p1 = __uint_as_float((__float_as_uint(x1) & ~15u) | (j + 1));
                                const float hi = fmaxf(p0, p1), lo = fminf(p0, p1);
                                t2 = max3(t2, fminf(t1, hi), lo);
                                t1 = fmaxf(t1, hi);
                                most = max3(most, x0, x1);
                            }
                            groups[2 * c + g] = fmaxf(most, SCORE_FLOOR);
                            groups[8 + 2 * c + g] = __uint_as_float((__float_as_uint(t2) & ~15u) | (__float_as_uint(t1) & 15u));
                            top = fmaxf(top, most);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) top = max3(top, v[j], v[j + 1]);
                    }
                    // sums relative to the larger maximum: e u becomes c e (u + shift)
                    const float nm = fmaxf(m, top), base = nm == -INFINITY ? 0.f : nm;      // nothing but -inf so far: the sums stay 0
                    const float shift = fmaxf((m - base) * p.k2, SCORE_FAR), c2 = ex2(shift);
                    const float s0 = sum * c2, w0 = c2 * (esum + sum * shift);
                    float2 s2 = make_float2(s0, 0.f), w2 = make_float2(w0, 0.f);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 u = mul2(add2(f2(v[j], v[j + 1]), bc2(-base)), bc2(p.k2)), e = ex2x2(u);
                        s2 = add2(s2, e);
                        w2 = fma2(e, u, w2);
                    }
                    sum = s2.x + s2.y;
                    esum = w2.x + w2.y;
                    if (esum != esum) {                     // 0 times -inf: those terms are 0
                        esum = w0;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float u = (v[j] - base) * p.k2;
                            esum += ex2(u) * fmaxf(u, SCORE_FAR);
                        }
                    }
                    m = nm;
                } else if (is_dlogit(EPI)) {
                    if (is_grad(EPI) && (SUMS || has_ids(EPI))) {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 u = mul2(add2(f2(v[j], v[j + 1]), bc2(-rmax)), bc2(p.k2)), e = ex2x2(u);
                            const float2 x = mul2(e, has_ids(EPI) ? bc2(gr.A) : fma2(f2(fmaxf(u.x, SCORE_FAR), fmaxf(u.y, SCORE_FAR)), bc2(gr.B), bc2(gr.A)));
                            v[j] = x.x;
                            v[j + 1] = x.y;
                        }
                    } else if (is_grad(EPI)) {
                        float2 any = make_float2(0.f, 0.f);
                        float2 x[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float2 u = mul2(add2(f2(v[2 * j], v[2 * j + 1]), bc2(-rmax)), bc2(p.k2));
                            x[j] = mul2(ex2x2(u), fma2(u, bc2(gr.B), bc2(gr.A)));
                            any = add2(any, x[j]);
                        }
                        if (any.x + any.y != any.x + any.y) {                       // 0 times -inf: those are 0
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float u0 = (v[2 * j] - rmax) * p.k2, u1 = (v[2 * j + 1] - rmax) * p.k2;
                                x[j] = f2(ex2(u0) * fmaf(fmaxf(u0, SCORE_FAR), gr.B, gr.A), ex2(u1) * fmaf(fmaxf(u1, SCORE_FAR), gr.B, gr.A));
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) { v[2 * j] = x[j].x; v[2 * j + 1] = x[j].y; }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = ex2((v[j] - rmax) * LOG2E) * rsum;
                    }
                    if (yc >= 0 && yc < 32) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = yc == j ? v[j] - (is_grad(EPI) ? -gr.hot : scale) : v[j];
                    }
                    if (is_grad(EPI) ? gr.A == 0.f && gr.B == 0.f && gr.hot == 0.f : scale == 0.f) {   // a token that does not count, whatever its logits
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0.f;
                    }
                    // one piece: 64 columns make one store of 32 rows x 128 bytes; three: 32 columns of each one of 64 bytes, two of which
                    // have room, so that a store need not have been read before the next is made
                    for (int pl = 0; pl < p.planes; ++pl) {
                        uint8_t* to = so + (p.planes > 1 ? flip * (XE_OUT / 2) : 0);
                        if ((c & 1) == 0 || p.planes > 1) {
                            if (lane == 0) {
                                if (p.planes > 1) bulk_wait_read_but_one();
                                else bulk_wait_read();
                            }
                            __syncwarp();
                        }
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                            w[j] = *reinterpret_cast<const uint32_t*>(&b2);
                            if (p.planes > 1) {
                                v[2 * j] -= __low2float(b2);
                                v[2 * j + 1] -= __high2float(b2);
                            }
                        }
                        // rows swizzled: 16-byte part j of row r of 128 bytes lands at j ^ (r % 8), of 64 bytes at j ^ (r / 2 % 4)
                        auto part = [&](int j) { return p.planes > 1 ? lane * 64 + ((j ^ (lane >> 1 & 3)) << 4) : lane * 128 + ((((c & 1) * 4 + j) ^ (lane & 7)) << 4); };
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            *reinterpret_cast<uint4*>(to + part(j)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                        }
                        if (EPI == XE_GRAD_IDS) {
                            // the row's words among these columns: their own values, in place of what was just written
                            const int id0 = id;
                            while (word < cc + 32) {
                                float r = gr.A * (ex2((word_z - rmax) * p.k2) - rsum * word_share);
                                for (int q = 0; q < pl; ++q) r -= __bfloat162float(__float2bfloat16_rn(r));
                                const int j = word - cc;
                                *reinterpret_cast<__nv_bfloat16*>(to + part(j >> 3) + (j & 7) * 2) = __float2bfloat16_rn(r);
                                ++id;
                                fetch_word();
                            }
                            if (pl + 1 < p.planes && id != id0) { id = id0; fetch_word(); }
                        }
                        if (p.planes > 1 || (c & 1)) {
                            fence_proxy_async_smem();
                            __syncwarp();
                            const int x = p.planes > 1 ? cc : cc - 32;
                            const int y0 = rc.x * XE_TILE + (int)rank * 128 + sub * 32;
                            if (x < p.N && y0 < p.M) {
                                if (lane == 0) {
                                    tma_store_3d(&map_p, to, x, y0, pl);
                                    bulk_commit();
                                }
                                flip ^= 1;
                            }
                        }
                    }
                } else if (live && cc < p.N) {
                    xent_emit(p, v, r.part, row, cc, p.first, last, factor);
                }
            };
            if constexpr (SUMS) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    float v[16];
                    tmem_ld16(at + c * 16, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) tot[c / 2][c % 2 * 16 + j] = r.fresh ? v[j] : tot[c / 2][c % 2 * 16 + j] + v[j];
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_to_rank(&acc_empty[a], 0));
                if ((a ^= 1) == 0) aph ^= 1;
                if (r.k1 != p.nk && r.cur < r.end) continue;             // more of the tile (or of this pair's part of it) to come
#pragma unroll
                for (int c = 0; c < 4; ++c) columns(c, tot[c]);
                if (EPI == XE_LSE && live) p.part[(int64_t)(2 * rc.y + half) * p.M + row] = make_float2(m, sum);
                keep();
                continue;
            }
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                float v[32];
                tmem_ld32(at + c * 32, v);
                tmem_ld_wait();
                columns(c, v);
            }
            if (EPI == XE_LSE && live) p.part[(int64_t)(2 * rc.y + half) * p.M + row] = make_float2(m, sum);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_rank(&acc_empty[a], 0));
            if ((a ^= 1) == 0) aph ^= 1;
            keep();
        }
        if (is_dlogit(EPI) && lane == 0) bulk_wait_all();
        if (!ok && lane == 0 && p.status) *p.status = SWX_ERR_TIMEOUT;
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                       // neither CTA goes while the other may still reach its barriers
    if (warp == 1) tmem_free_pair(tmem, 512);
}

// Eight values of a row from k on (a multiple of 8; rows start on 16 bytes), zeros from d on.
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, int64_t k, int64_t d) {
    if (k + 8 <= d) return *reinterpret_cast<const uint4*>(p + k);
    __align__(16) __nv_bfloat16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < d ? p[k + j] : __nv_bfloat16(0.f);
    return *reinterpret_cast<const uint4*>(v);
}

// ------------------------------------------------------------------ host side
// How a gradient product's tiles are dealt out to the CTA pairs (linear_xent.cu `deal`).
struct XentDeal { int spread, pairs, parts; };
constexpr int XE_PAIRS = 74, XE_MIN_SHARE = 4;

// A head's operands: x (T, d) and the weight (V, d), row strides in elements.
struct HeadOps { int64_t T, V, d; int dtype; const void* x; int64_t x_sr; const void* w; int64_t w_sr; };

// What the tensor core takes off a sum of n additions of bf16 products on average, relative: it cuts each addition's low bits
// off (toward zero).  Sums of terms of either sign came out 0.20 2^-24 n too small at n = 4, 0.225 at 64 and 0.26 at 512; of one sign 0.14,
// 0.45 and 1.07.  All logits together too small act like a higher temperature, which the entropy shows first (8192 rows x
// 50001 x 1024: 8e-7 off); the scale of the exponents makes up for the mean of either sign.  Sums that are exact (rows of a few values, small
// integers) lose nothing: their differences come out 0.23 2^-24 n too large instead (9e-7 of them at a width of 1024).
constexpr int64_t XE_CUT_ADDITIONS = 512;
inline double mean_cut(double additions) { return 0.23 * 0x1p-24 * additions; }
// Scoring and distillation sum the logits of bf16 operands 8192 terms at a time in tensor memory, in fp32 beyond, so that no more
// additions come together than were measured (65536 terms: 6.6e-5 too small in one sum, 7.9e-6 so and 9e-7 with the mean made up for).
constexpr int XE_KSUB_SCORES = XE_CUT_ADDITIONS * 16 / XE_K;
inline int score_ksub(const HeadOps& o) { return o.dtype == SWX_DTYPE_BF16 ? XE_KSUB_SCORES : XE_KSUB_LOGITS; }
inline void set_score_sums(XentGemm& g, const HeadOps& o) { g.ksub = std::min(g.nk, score_ksub(o)); }
// Additions of a logit's sum at its full size (fp32 operands' largest pieces come last).
inline int64_t logit_additions(const HeadOps& o) { return std::min<int64_t>((o.d + 15) / 16, score_ksub(o) * XE_K / 16); }
inline float exponent_scale(float temperature, double cut) { return (float)(1.4426950408889634 / temperature * (1. + cut)); }

// Sizes and the workspace: copies of the operands, then (forward) whatever the operator keeps from
// `base` on, or (backward) a piece of the logits' gradient and the sums of the gradient products.
struct HeadPlan {
    int es, planes;                           // bytes of an input value; bf16 pieces
    int64_t dp;                               // padded contraction length of packed operands
    bool pack_x, pack_w;
    int64_t mt, nt, piece;                    // tiles; vocabulary columns per piece of the backward
    int64_t off_x, off_w, base;
    int64_t off_p, off_acc, off_acc_w, ldp, bwd_total;
    XentDeal dx;
};
HeadPlan head_plan(const HeadOps& o);
int head_check(const HeadOps& o);

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Stages of the logits' contraction summed in tensor memory at a time: all of them for bf16 operands.
inline int logits_ksub(const HeadPlan& q, int nk) { return q.planes == 3 ? std::min(nk, XE_KSUB_LOGITS) : nk; }

// A (rows, inner) bf16 matrix with `planes` pieces as a 3-D tensor map, swizzled within the box's rows of 128 or 64 bytes.
inline bool encode_operand(CUtensorMap* m, const void* base, int64_t inner, int64_t rows, int64_t planes, int64_t row,
                           int64_t plane, uint32_t box_inner, uint32_t box_rows, int swizzle = 128) {
    const EncodeTiledFn f = encode_tiled();
    if (!f || !base || (reinterpret_cast<uintptr_t>(base) & 15)) return false;
    const int64_t rs = row * 2, ps = (planes > 1 ? plane : row * rows) * 2;
    if (rs % 16 || ps % 16 || rs <= 0 || ps <= 0 || rs >= (int64_t(1) << 40) || ps >= (int64_t(1) << 40)) return false;
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)planes};
    cuuint64_t strides[2] = {(cuuint64_t)rs, (cuuint64_t)ps};
    cuuint32_t box[3] = {box_inner, box_rows, 1};
    cuuint32_t unit[3] = {1, 1, 1};
    return f(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, unit,
             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of one product of scoring and distillation: what it keeps for the rows' kernel is bounded (8192 rows x 50001: 51 MB of statistics,
// 205 MB of records), and 32 row tiles keep a tile of the weight in use as long as more would.
constexpr int64_t SC_ROWS = 32 * XE_TILE;

struct Operand {
    const void* p; int64_t inner, rows, planes, row, plane;
    // rows of the contraction's other index, 64 contraction steps wide / the transposed use
    bool k_major(CUtensorMap* m) const { return encode_operand(m, p, inner, rows, planes, row, plane, 64, 128); }
    bool mn_major(CUtensorMap* m) const { return encode_operand(m, p, inner, rows, planes, row, plane, 64, 64); }
    // n rows from r0 on (pieces keep their distance)
    Operand part(int64_t r0, int64_t n) const { return Operand{static_cast<const uint8_t*>(p) + r0 * row * 2, inner, n, planes, row, plane}; }
};

// x and the weight as the products read them: themselves, or their copies in the workspace.
void head_operands(const HeadOps& o, const HeadPlan& q, uint8_t* ws, Operand& x, Operand& w, cudaStream_t st);

template <int EPI, bool A_MN, bool B_MN, bool SUMS = false>
static cudaError_t launch_gemm(const XentGemm& p, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mp,
                               int64_t pairs, cudaStream_t st) {
    auto k = xent_gemm_kernel<EPI, A_MN, B_MN, SUMS>;
    cudaError_t e = allow_smem(k, XE_SMEM);
    if (e != cudaSuccess) return e;
    if (!p.spread) pairs = std::min<int64_t>((int64_t)p.mt * p.nt, pairs);
    k<<<(unsigned)(2 * pairs), XE_THREADS, XE_SMEM, st>>>(p, ma, mb, mp);
    return cudaGetLastError();
}

// What a backward pass wants: either gradient may be absent; the results' factor is num / den.
struct HeadGrads { void* dx; void* dw; int dw_bf16; const float* num; const float* den; };

// dx and dW of the vocabulary's columns [c0, c0 + cw), whose dlogit is in the workspace.
int head_piece_products(const HeadOps& o, const HeadPlan& q, uint8_t* ws, const Operand& x, const Operand& w, const Operand& pr,
                        const HeadGrads& gr, int64_t c0, int64_t cw, int* status, cudaStream_t st);

// The logits' product, with the epilogue EPI, over all columns or a piece of them.
inline XentGemm logits_gemm(const HeadOps& o, const HeadPlan& q, int64_t c0, int64_t cw, int* status) {
    XentGemm g{};
    g.status = status; g.npair = q.planes == 3 ? 6 : 1; g.planes = q.planes;
    g.M = (int)o.T; g.N = (int)cw; g.mt = (int)q.mt; g.nt = (int)((cw + XE_TILE - 1) / XE_TILE); g.group = 32;
    g.nk = (int)((o.d + XE_K - 1) / XE_K); g.b0 = g.col0 = (int)c0; g.vocab = o.V;
    g.ksub = logits_ksub(q, g.nk);
    return g;
}

template <int EPI>
static cudaError_t launch_logits(const XentGemm& g, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& store, cudaStream_t st) {
    return g.ksub < g.nk ? launch_gemm<EPI, false, false, true>(g, x, w, store, XE_PAIRS, st)
                         : launch_gemm<EPI, false, false>(g, x, w, store, XE_PAIRS, st);
}

// The scoring of a few rows without tiles (linear_logprob_few.cu): its CTAs, 0 where it does not take them, and the launch.
int score_few_ctas(const HeadOps& o);
double few_additions(int64_t d);              // of a logit there
cudaError_t launch_score_few(const XentGemm& g, const HeadOps& o, const Operand& x, const Operand& w, bool top, int ctas, cudaStream_t st);

// The gradients, piece by piece of the vocabulary: the logits again and dlogit in the epilogue (`launch`, with the
// fields that `fill` sets), and the two products.  `before` may use the operands' maps for a step ahead of them.
struct NoStep { int operator()(const CUtensorMap&, const CUtensorMap&, int*) const { return SWX_OK; } };
template <class Launch, class Fill, class Before = NoStep>
static int head_backward(const HeadOps& o, const HeadPlan& q, uint8_t* ws, const HeadGrads& gr, cudaStream_t st, Launch launch, Fill fill, Before before = {}) {
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    head_operands(o, q, ws, x, w, st);
    CUtensorMap x_k, w_k;
    if (!x.k_major(&x_k) || !w.k_major(&w_k)) return SWX_ERR_CUDA;
    const int ready = before(x_k, w_k, status);
    if (ready != SWX_OK) return ready;
    for (int64_t c0 = 0; c0 < o.V; c0 += q.piece) {
        const int64_t cw = std::min(q.piece, o.V - c0);
        const Operand pr{ws + q.off_p, cw, o.T, q.planes, q.ldp, o.T * q.ldp};
        CUtensorMap p_st;
        // stores of 32 rows: 64 columns at once for one piece, 32 for each of three
        if (!encode_operand(&p_st, pr.p, cw, o.T, q.planes, q.ldp, o.T * q.ldp, q.planes == 3 ? 32 : 64, 32, q.planes == 3 ? 64 : 128)) return SWX_ERR_CUDA;
        XentGemm g = logits_gemm(o, q, c0, cw, status);
        fill(g);
        if (launch(g, x_k, w_k, p_st, st) != cudaSuccess) return SWX_ERR_CUDA;
        const int c = head_piece_products(o, q, ws, x, w, pr, gr, c0, cw, status, st);
        if (c != SWX_OK) return c;
    }
    return SWX_OK;
}

}  // namespace swx
