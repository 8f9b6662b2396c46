// Softmax cross entropy of a linear head over a large vocabulary, without keeping the
// logits:  loss_t = log sum_v exp(x_t . W_v) - x_t . W_{y_t}, and
//   dlogit_tv = (exp(logit_tv - lse_t) - [v == y_t]) c_t,  dx = dlogit W,  dW = dlogit^T x,
// with c_t the loss's upstream gradient (over the number of counted tokens for the mean).
//
// Forward: one matrix product whose epilogue keeps, for each row and each half of a
// 256-column tile, the maximum and the sum of exponentials (two floats per 128 logits) and
// the target's logit; a second kernel joins the pieces.  Backward: the vocabulary is
// walked in pieces; each piece's logits are formed again, turned into dlogit in the epilogue
// (bf16, the tensor core's operand: gradients 2.0e-3 off at a vocabulary of 256, 1.7e-3 from their own rounding), and
// multiplied with the weight (dx, summed over the pieces in fp32) and with x (dW, complete for the piece's rows).
//
// Every product runs on the same kernel: a persistent grid of CTA pairs, 256 x 256 tiles,
// operands staged by TMA into a ring, tcgen05 products issued by one thread per pair into
// two alternating accumulators in tensor memory, and eight warps per CTA that read an
// accumulator while the next tile is computed.  The tensor pipe bounds it: 4096 tokens x 32768 x 1024 bf16, cold,
// forward 178 us (88 % of the SM's active cycles on products, 1547 TFLOP/s), dlogit 199 us (79 %; it writes 268 MB), dx 190
// (93 %, on 64 of 74 pairs); 8192 x 50001 x 1024 0.51, 0.57, 0.58 and 0.60 ms, where a library
// product of the same size alone takes 0.56 to 0.61.  The logits' epilogue (an exponential for each) fits behind a
// tile's products from about 512 values of the contraction on; below that it bounds the forward.
//
// fp32 operands are split into three bf16 pieces (24 bits) and multiplied as the six
// products of pieces above 2^-24, smallest first, on the same kernel.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "launch_util.cuh"
#include "tc5.cuh"
#include "tma_util.cuh"

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

enum XentEpi { XE_LSE, XE_PROB, XE_DX, XE_DW };

struct XentGemm {
    int M, N;                                 // rows and columns of the result
    int mt, nt, group;                        // tiles; row tiles walked together (XE_LSE, XE_PROB)
    int nk, npair;                            // ring stages of the contraction; pairs of pieces
    int ksub;                                 // stages summed in tensor memory before the sum moves on
    int ka0, kb0;                             // first contraction index of A and of B
    int a0, b0;                               // first row of A and of B (M / N coordinate)
    int* status;
    // XE_LSE / XE_PROB
    const int64_t* target;
    int64_t ignore;
    int64_t vocab;
    int col0;                                 // vocabulary index of column 0
    float2* part;                             // (2 nt, M): max and sum of a tile half's exponentials
    float* hit;                               // (M): the target's logit
    int* counter;                             // zeroed by XE_LSE for the joining kernel
    const float* row_max; const float* row_rsum;
    const float* dloss; int reduction;
    int planes;                               // bf16 pieces of the dlogit
    // XE_DX / XE_DW
    // spread: the steps of all tiles are dealt out evenly and a tile's parts are summed in
    // acc[part][M][N]; else whole tiles go round and the last piece writes the result
    int spread;
    float* acc; void* out; int out_bf16; int64_t ld; int first, last;
    const float* scale_num; const float* scale_den;   // the result's factor: num / den, either may be absent
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

// Tile t -> (row tile, column tile).  XE_LSE, XE_PROB: `group` row tiles of x stay in L2
// while the weight's column tiles pass by; the gradients: a row tile's column tiles together.
template <int EPI>
__device__ __forceinline__ int2 tile_of(const XentGemm& p, int64_t t) {
    if (EPI == XE_LSE || EPI == XE_PROB) {
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
        if (EPI == XE_LSE && blockIdx.x == 0) *p.counter = 0;
    }
    if (warp == 1) tmem_alloc_pair(&tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_base;

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
            if ((EPI == XE_LSE || EPI == XE_PROB) && live) {
                y = p.target[row] - p.col0;
                if (EPI == XE_PROB) {
                    scale = row_scale(p, row);
                    rmax = p.row_max[row];
                    rsum = p.row_rsum[row] * scale;
                }
            }
            if (!mbar_wait_cluster(&acc_full[a], aph, XE_POLLS)) { ok = false; break; }
            tc_fence_after();
            const uint32_t at = tmem + ((uint32_t)(sub * 32) << 16) + a * XE_TILE + half * 128;
            // 32 columns of the row, from 32 c on
            float m = -INFINITY, sum = 0.f;
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
                } else if (EPI == XE_PROB) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = ex2((v[j] - rmax) * LOG2E) * rsum;
                    if (yc >= 0 && yc < 32) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = yc == j ? v[j] - scale : v[j];
                    }
                    if (scale == 0.f) {                     // a token that does not count, whatever its logits
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0.f;
                    }
                    // 64 columns of each piece make one 32-row x 128-byte store
                    for (int pl = 0; pl < p.planes; ++pl) {
                        if ((c & 1) == 0 || p.planes > 1) {
                            if (lane == 0) bulk_wait_read();
                            __syncwarp();
                        }
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                            w[j] = *reinterpret_cast<const uint32_t*>(&b2);
                            v[2 * j] -= __low2float(b2);
                            v[2 * j + 1] -= __high2float(b2);
                        }
                        // one piece: 128-byte rows, swizzled (16-byte part j of row r lands at
                        // j ^ (r % 8)); three: 64-byte rows, plain
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int at_b = p.planes > 1 ? lane * 64 + j * 16
                                                          : lane * 128 + ((((c & 1) * 4 + j) ^ (lane & 7)) << 4);
                            *reinterpret_cast<uint4*>(so + at_b) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                        }
                        if (p.planes > 1 || (c & 1)) {
                            fence_proxy_async_smem();
                            __syncwarp();
                            const int x = p.planes > 1 ? cc : cc - 32;
                            const int y0 = rc.x * XE_TILE + (int)rank * 128 + sub * 32;
                            if (lane == 0 && x < p.N && y0 < p.M) {
                                tma_store_3d(&map_p, so, x, y0, pl);
                                bulk_commit();
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
        }
        if (EPI == XE_PROB && lane == 0) bulk_wait_all();
        if (!ok && lane == 0 && p.status) *p.status = SWX_ERR_TIMEOUT;
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                       // neither CTA goes while the other may still reach its barriers
    if (warp == 1) tmem_free_pair(tmem, 512);
}

// ------------------------------------------------------------------ joining the pieces
struct XentJoin {
    int64_t T, V;
    int np;                                   // pieces per row
    const float2* part; const float* hit; const int64_t* target; int64_t ignore;
    float* row_max; float* row_rsum;
    float* rows;                              // SWX_XENT_NONE: the losses
    double2* sums;                            // otherwise: each CTA's sum and count
    float* loss; float* count; int reduction; int* counter;
};

constexpr int XJ_ROWS = 8, XJ_SLICES = 32, XJ_WARPS = XJ_ROWS * XJ_SLICES / 32;

__device__ __forceinline__ void join_pair(float& m, float& s, float2 q) {
    const float nm = fmaxf(m, q.x), base = nm == -INFINITY ? 0.f : nm;
    s = s * ex2((m - base) * LOG2E) + q.y * ex2((q.x - base) * LOG2E);
    m = nm;
}

// CTA = 8 rows x 32 slices of the pieces (few rows per CTA, so that a short call still has
// many CTAs): each thread joins its slice, four pieces at a time, then the slices are joined
// by shuffles and through shared memory, always in the same order.  A few microseconds whatever the size
// (512 tokens x 392 pieces 4.4 us, 8192 x 2 6.8), latency.  Each CTA leaves the sum of
// its rows' losses and the count of its tokens; the last CTA to finish adds those up (fp64, a
// fixed order whichever CTA it is).
__global__ void __launch_bounds__(XJ_ROWS * XJ_SLICES) xent_join_kernel(const XentJoin p) {
    __shared__ float2 sp[XJ_WARPS][XJ_ROWS];
    __shared__ int is_last;
    __shared__ double red[XJ_WARPS][2];
    const int r = threadIdx.x % XJ_ROWS, sl = threadIdx.x / XJ_ROWS, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t row = (int64_t)blockIdx.x * XJ_ROWS + r;
    float m = -INFINITY, s = 0.f;
    if (row < p.T) {
        for (int i = sl; i < p.np; i += 4 * XJ_SLICES) {
            float2 q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                q[j] = i + j * XJ_SLICES < p.np ? p.part[(int64_t)(i + j * XJ_SLICES) * p.T + row] : make_float2(-INFINITY, 0.f);
            const float nm = fmaxf(fmaxf(fmaxf(m, q[0].x), fmaxf(q[1].x, q[2].x)), q[3].x), base = nm == -INFINITY ? 0.f : nm;
            s *= ex2((m - base) * LOG2E);
#pragma unroll
            for (int j = 0; j < 4; ++j) s += q[j].y * ex2((q[j].x - base) * LOG2E);
            m = nm;
        }
    }
#pragma unroll
    for (int o = XJ_ROWS; o < 32; o *= 2) {
        const float2 q = make_float2(__shfl_down_sync(0xffffffffu, m, o), __shfl_down_sync(0xffffffffu, s, o));
        join_pair(m, s, q);
    }
    if (lane < XJ_ROWS) sp[warp][lane] = make_float2(m, s);
    __syncthreads();
    double sum = 0., n = 0.;
    if (warp == 0) {
        if (lane < XJ_ROWS && row < p.T) {
            m = sp[0][lane].x;
            s = sp[0][lane].y;
#pragma unroll
            for (int i = 1; i < XJ_WARPS; ++i) join_pair(m, s, sp[i][lane]);
            p.row_max[row] = m;
            p.row_rsum[row] = 1.f / s;
            const int64_t y = p.target[row];
            float loss = 0.f;
            if (y != p.ignore) {
                loss = y >= 0 && y < p.V ? logf(s) + (m - p.hit[row]) : __int_as_float(0x7fc00000);
                n = 1.;
            }
            if (p.rows) p.rows[row] = loss;
            sum = loss;
        }
        for (int o = XJ_ROWS / 2; o > 0; o >>= 1) {
            sum += __shfl_down_sync(0xffffffffu, sum, o);
            n += __shfl_down_sync(0xffffffffu, n, o);
        }
    }
    if (p.reduction == SWX_XENT_NONE) return;
    if (threadIdx.x == 0) {
        p.sums[blockIdx.x] = make_double2(sum, n);
        __threadfence();
        is_last = atomicAdd(p.counter, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    sum = n = 0.;
#pragma unroll 4
    for (int i = threadIdx.x; i < (int)gridDim.x; i += XJ_ROWS * XJ_SLICES) {
        const double2 q = __ldcg(p.sums + i);
        sum += q.x;
        n += q.y;
    }
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    if (lane == 0) { red[warp][0] = sum; red[warp][1] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < XJ_WARPS; ++i) { sum += red[i][0]; n += red[i][1]; }
        *p.count = (float)n;
        *p.loss = (float)(p.reduction == SWX_XENT_MEAN ? sum / n : sum);
    }
}

// ------------------------------------------------------------------ summing a tile's parts
// out = factor * (parts in order), for the spread gradients; thread = 4 columns of a row.  The parts
// come from L2 (1003 tokens x 10007 x 200 fp32, dx and dW: 15 us of 216).
__global__ void __launch_bounds__(256) xent_sum_kernel(const XentGemm p, int P) {
    const int per = (p.N + 3) / 4;
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.M * per) return;
    const int row = (int)(i / per), c = (int)(i % per) * 4;
    const int64_t tile = (int64_t)(row / XE_TILE) * p.nt + c / XE_TILE, total = (int64_t)p.mt * p.nt * p.nk;
    const int parts = (int)((((tile + 1) * p.nk) * P - 1) / total - ((tile * p.nk + 1) * P - 1) / total) + 1;
    float factor = 1.f;
    if (p.scale_num) factor = *p.scale_num;
    if (p.scale_den) factor = *p.scale_den > 0.f ? factor / *p.scale_den : 0.f;
    const int n = min(4, p.N - c);
    const float* a = p.acc + (int64_t)row * p.N + c;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const bool vec = p.N % 4 == 0;
#pragma unroll 4
    for (int k = 0; k < parts; ++k, a += (int64_t)p.M * p.N) {
        if (vec) {
            const float4 q = *reinterpret_cast<const float4*>(a);
            v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) if (j < n) v[j] += a[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j >= n) break;
        const float o = v[j] * factor;
        if (p.out_bf16) static_cast<__nv_bfloat16*>(p.out)[(int64_t)row * p.ld + c + j] = __float2bfloat16_rn(o);
        else static_cast<float*>(p.out)[(int64_t)row * p.ld + c + j] = o;
    }
}

// ------------------------------------------------------------------ operand layout
// (rows, d) with any row stride -> dense bf16 pieces (planes, rows, dp), dp a multiple of
// 8: fp32 values as three bf16 pieces (each the rounding of what the earlier ones leave),
// bf16 values as themselves.  Columns d..dp are zero.
// Two matrices in one launch (rows 0: none).
struct XentPack { const void* src; int64_t sr, rows; __nv_bfloat16* dst; };

template <typename T>
__global__ void __launch_bounds__(256) xent_pack_kernel(const XentPack x, const XentPack w, int d, int dp) {
    const int per = dp / 8;
    const int64_t n = (x.rows + w.rows) * per;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const bool second = i / per >= x.rows;
        const XentPack& m = second ? w : x;
        const int64_t r = i / per - (second ? x.rows : 0);
        const int c = (int)(i % per) * 8;
        const T* s = static_cast<const T*>(m.src) + r * m.sr + c;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < d ? Elem<T>::to_f(s[j]) : 0.f;
        constexpr int planes = sizeof(T) == 4 ? 3 : 1;
#pragma unroll
        for (int pl = 0; pl < planes; ++pl) {
            __align__(16) __nv_bfloat16 o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[j] = __float2bfloat16_rn(v[j]);
                v[j] -= __bfloat162float(o[j]);
            }
            *reinterpret_cast<uint4*>(m.dst + ((int64_t)pl * m.rows + r) * dp + c) = *reinterpret_cast<const uint4*>(o);
        }
    }
}

// ------------------------------------------------------------------ host side
// How a gradient product's tiles are dealt out to the CTA pairs of a 148-SM B200.  Whole
// tiles where they keep the pairs busy for seven tenths of their rounds or more; otherwise the steps
// are spread evenly, at least XE_MIN_SHARE per pair, and the parts of a tile (at most `parts`)
// are summed afterwards.
struct XentDeal { int spread, pairs, parts; };
constexpr int XE_PAIRS = 74, XE_MIN_SHARE = 4;

static XentDeal deal(int64_t tiles, int64_t nk) {
    const int64_t rounds = (tiles + XE_PAIRS - 1) / XE_PAIRS, total = tiles * nk;
    XentDeal d{0, (int)std::min<int64_t>(tiles, XE_PAIRS), 1};
    if (tiles * 10 >= rounds * XE_PAIRS * 7) return d;
    const int64_t P = std::min<int64_t>(XE_PAIRS, std::max<int64_t>(1, total / XE_MIN_SHARE));
    if (P <= tiles && tiles % P == 0) return XentDeal{0, (int)P, 1};
    d.spread = 1;
    d.pairs = (int)P;
    for (int64_t t = 0; t < tiles; ++t)
        d.parts = std::max<int>(d.parts, (int)(((t + 1) * nk * P - 1) / total - ((t * nk + 1) * P - 1) / total) + 1);
    return d;
}

struct XentPlan {
    int es, planes;                           // bytes of an input value; bf16 pieces
    int64_t dp;                               // padded contraction length of packed operands
    bool pack_x, pack_w;
    int64_t mt, nt, piece;                    // tiles; vocabulary columns per piece of the backward
    int64_t off_x, off_w, off_part, off_hit, off_rows, off_cnt, fwd_total;
    int64_t off_p, off_acc, off_acc_w, ldp, bwd_total;
    XentDeal dx;
};

static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool direct_ok(const void* p, int64_t sr, int dtype) {
    return dtype == SWX_DTYPE_BF16 && aligned16(p) && sr % 8 == 0;
}

// Vocabulary columns per piece of the backward: 416 MB of dlogit (tokens x columns, 2 bytes for each bf16 piece),
// but not below 4096 columns (more than 416 MB from 53000 tokens on, 17700 in fp32): narrower pieces would leave dW few tiles.  The piece need not stay in the L2: its one write and two reads
// hide behind the products, while fewer pieces mean fewer launches, fewer rounds that do not
// fill the GPU and fewer passes over dx's running sum (8192 tokens x 50001 x 1024, forward
// and backward: pieces of 72 MB 2.92 ms, 160 MB 2.83, 288 MB 2.67, 450 MB 2.61, one piece 2.56).
//
// Among the sizes near that, the one whose dW tiles take the fewest rounds of the CTA pairs over
// all pieces (196 x 4 tiles: pieces of 104 and 92 column tiles 11 rounds, two of 98 12).
static int64_t piece_columns(int64_t T, int64_t V, int64_t d, int planes) {
    const int64_t vt = (V + XE_TILE - 1) / XE_TILE, dt = (d + XE_TILE - 1) / XE_TILE;
    const int64_t most = std::max<int64_t>((int64_t(416) << 20) / (2 * planes * std::max<int64_t>(T, 1)), 4096) / XE_TILE;
    if (vt <= most) return vt * XE_TILE;
    auto rounds = [dt](int64_t tiles) { return (tiles * dt + XE_PAIRS - 1) / XE_PAIRS; };
    int64_t best = most, least = INT64_MAX;
    for (int64_t c = most; c >= most * 3 / 4 && c > 0; --c) {
        const int64_t n = vt / c * rounds(c) + rounds(vt % c);
        if (n < least) {
            least = n;
            best = c;
        }
    }
    return best * XE_TILE;
}

static XentPlan xent_plan(const swx_xent_args* a) {
    XentPlan q{};
    const int64_t T = a->tokens, V = a->vocab, d = a->dim;
    q.es = a->dtype == SWX_DTYPE_F32 ? 4 : 2;
    q.planes = a->dtype == SWX_DTYPE_F32 ? 3 : 1;
    q.dp = (d + 7) / 8 * 8;
    q.pack_x = !direct_ok(a->x, a->x_sr, a->dtype);
    q.pack_w = !direct_ok(a->weight, a->w_sr, a->dtype);
    q.mt = (T + XE_TILE - 1) / XE_TILE;
    q.nt = (V + XE_TILE - 1) / XE_TILE;
    q.off_x = 0;
    q.off_w = q.off_x + (q.pack_x ? up256(q.planes * T * q.dp * 2) : 0);
    const int64_t base = q.off_w + (q.pack_w ? up256(q.planes * V * q.dp * 2) : 0);
    q.off_part = base;
    q.off_hit = q.off_part + up256(2 * q.nt * T * 8);
    q.off_rows = q.off_hit + up256(T * 4);
    q.off_cnt = q.off_rows + up256((T + XJ_ROWS - 1) / XJ_ROWS * 16);
    q.fwd_total = q.off_cnt + 256;
    q.piece = piece_columns(T, V, d, q.planes);
    q.ldp = q.piece;
    q.off_p = base;
    q.off_acc = q.off_p + up256((int64_t)q.planes * T * q.ldp * 2);
    // the running sums of dx (bf16 result: in fp32; one for each part of a spread tile), then
    // the parts of dW, which live for one piece
    const int64_t dt = (d + XE_TILE - 1) / XE_TILE;
    const int64_t cl = V - (V - 1) / q.piece * q.piece;      // columns of the last piece
    q.dx = deal(q.mt * dt, (std::min(q.piece, V) + XE_K - 1) / XE_K);
    const bool own_acc = q.dx.spread || (a->dtype == SWX_DTYPE_BF16 && q.piece < V);
    q.off_acc_w = q.off_acc + (own_acc ? up256(q.dx.parts * T * d * 4) : 0);
    int64_t w = 0;
    for (const int64_t cw : {std::min<int64_t>(q.piece, V), cl}) {
        const XentDeal e = deal((cw + XE_TILE - 1) / XE_TILE * dt, (T + XE_K - 1) / XE_K);
        if (e.spread) w = std::max<int64_t>(w, up256(e.parts * cw * d * 4));
    }
    q.bwd_total = q.off_acc_w + w;
    return q;
}

// Stages of the logits' contraction summed in tensor memory at a time: all of them for bf16 operands.
static int logits_ksub(const XentPlan& q, int nk) { return q.planes == 3 ? std::min(nk, XE_KSUB_LOGITS) : nk; }

// A (rows, inner) bf16 matrix with `planes` pieces as a 3-D tensor map, 128-byte swizzled.
static bool encode_operand(CUtensorMap* m, const void* base, int64_t inner, int64_t rows, int64_t planes, int64_t row,
                           int64_t plane, uint32_t box_inner, uint32_t box_rows, bool swizzle = true) {
    const EncodeTiledFn f = encode_tiled();
    if (!f || !base || (reinterpret_cast<uintptr_t>(base) & 15)) return false;
    const int64_t rs = row * 2, ps = (planes > 1 ? plane : row * rows) * 2;
    if (rs % 16 || ps % 16 || rs <= 0 || ps <= 0 || rs >= (int64_t(1) << 40) || ps >= (int64_t(1) << 40)) return false;
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)planes};
    cuuint64_t strides[2] = {(cuuint64_t)rs, (cuuint64_t)ps};
    cuuint32_t box[3] = {box_inner, box_rows, 1};
    cuuint32_t unit[3] = {1, 1, 1};
    return f(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, unit,
             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operand {
    const void* p; int64_t inner, rows, planes, row, plane;
    // rows of the contraction's other index, 64 contraction steps wide / the transposed use
    bool k_major(CUtensorMap* m) const { return encode_operand(m, p, inner, rows, planes, row, plane, 64, 128); }
    bool mn_major(CUtensorMap* m) const { return encode_operand(m, p, inner, rows, planes, row, plane, 64, 64); }
};

// x and the weight as the products read them: themselves, or their copies in the workspace.
static void operands(const swx_xent_args* a, const XentPlan& q, uint8_t* ws, Operand& x, Operand& w, cudaStream_t st) {
    const int64_t T = a->tokens, V = a->vocab, d = a->dim;
    x = q.pack_x ? Operand{ws + q.off_x, d, T, q.planes, q.dp, T * q.dp} : Operand{a->x, d, T, 1, a->x_sr, 0};
    w = q.pack_w ? Operand{ws + q.off_w, d, V, q.planes, q.dp, V * q.dp} : Operand{a->weight, d, V, 1, a->w_sr, 0};
    const XentPack px{a->x, a->x_sr, q.pack_x ? T : 0, reinterpret_cast<__nv_bfloat16*>(ws + q.off_x)};
    const XentPack pw{a->weight, a->w_sr, q.pack_w ? V : 0, reinterpret_cast<__nv_bfloat16*>(ws + q.off_w)};
    const int64_t n = (px.rows + pw.rows) * (q.dp / 8);
    if (n == 0) return;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 16);
    if (a->dtype == SWX_DTYPE_F32) xent_pack_kernel<float><<<grid, 256, 0, st>>>(px, pw, (int)d, (int)q.dp);
    else xent_pack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(px, pw, (int)d, (int)q.dp);
}

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

static cudaError_t launch_sum(const XentGemm& p, int pairs, cudaStream_t st) {
    const int64_t n = (int64_t)p.M * ((p.N + 3) / 4);
    xent_sum_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p, pairs);
    return cudaGetLastError();
}

static int xent_check(const swx_xent_args* a) {
    if (!a || a->tokens < 0 || a->vocab < 1 || a->dim < 1) return SWX_ERR_INVALID_ARG;
    if (a->dtype != SWX_DTYPE_F32 && a->dtype != SWX_DTYPE_BF16) return SWX_ERR_UNSUPPORTED;
    if (a->tokens > (1 << 28) || a->vocab > (1 << 28) || a->dim > (1 << 16)) return SWX_ERR_UNSUPPORTED;
    if (a->reduction < SWX_XENT_NONE || a->reduction > SWX_XENT_SUM) return SWX_ERR_INVALID_ARG;
    if (a->x_sr < a->dim || a->w_sr < a->dim) return SWX_ERR_INVALID_ARG;
    return SWX_OK;
}

}  // namespace swx

using namespace swx;

extern "C" {

int64_t swx_xent_args_size(void) { return (int64_t)sizeof(swx_xent_args); }

int64_t swx_xent_fwd_workspace_bytes(const swx_xent_args* a) {
    const int c = xent_check(a);
    return c != SWX_OK ? -c : xent_plan(a).fwd_total;
}

int64_t swx_xent_bwd_workspace_bytes(const swx_xent_args* a) {
    const int c = xent_check(a);
    return c != SWX_OK ? -c : xent_plan(a).bwd_total;
}

int swx_xent_fwd(const swx_xent_args* a, void* stream) {
    const int c = xent_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool none = a->reduction == SWX_XENT_NONE;
    if (!none && (!a->loss || !a->count)) return SWX_ERR_INVALID_ARG;
    if (a->tokens > 0 && (!a->x || !a->weight || !a->targets || !a->row_max || !a->row_rsum || !a->workspace || (none && !a->loss)))
        return SWX_ERR_INVALID_ARG;
    const XentPlan q = xent_plan(a);
    if (a->tokens > 0 && (a->workspace_bytes < q.fwd_total || !aligned16(a->workspace))) return SWX_ERR_INVALID_ARG;
    if (a->tokens == 0) {
        if (none) return SWX_OK;
        // no token: a sum of 0, a mean of 0 / 0
        if (cudaMemsetAsync(a->count, 0, 4, st) != cudaSuccess) return SWX_ERR_CUDA;
        return cudaMemsetAsync(a->loss, a->reduction == SWX_XENT_MEAN ? 0xff : 0, 4, st) == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
    }
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    operands(a, q, ws, x, w, st);
    CUtensorMap mx, mw;
    if (!x.k_major(&mx) || !w.k_major(&mw)) return SWX_ERR_CUDA;
    XentGemm g{};
    g.M = (int)a->tokens; g.N = (int)a->vocab; g.mt = (int)q.mt; g.nt = (int)q.nt; g.group = 32;
    g.nk = (int)((a->dim + XE_K - 1) / XE_K); g.npair = q.planes == 3 ? 6 : 1;
    g.ksub = logits_ksub(q, g.nk);
    g.status = status;
    g.target = a->targets; g.ignore = a->ignore_index;
    g.part = reinterpret_cast<float2*>(ws + q.off_part);
    g.hit = reinterpret_cast<float*>(ws + q.off_hit);
    g.counter = reinterpret_cast<int*>(ws + q.off_cnt);
    if ((g.ksub < g.nk ? launch_gemm<XE_LSE, false, false, true>(g, mx, mw, mx, XE_PAIRS, st)
                       : launch_gemm<XE_LSE, false, false>(g, mx, mw, mx, XE_PAIRS, st)) != cudaSuccess)
        return SWX_ERR_CUDA;
    XentJoin j{};
    j.T = a->tokens; j.V = a->vocab; j.np = (int)(2 * q.nt); j.part = g.part; j.hit = g.hit; j.target = a->targets;
    j.ignore = a->ignore_index; j.row_max = a->row_max; j.row_rsum = a->row_rsum;
    j.rows = none ? a->loss : nullptr; j.sums = reinterpret_cast<double2*>(ws + q.off_rows);
    j.loss = a->loss; j.count = a->count; j.reduction = a->reduction; j.counter = g.counter;
    xent_join_kernel<<<(unsigned)((a->tokens + XJ_ROWS - 1) / XJ_ROWS), XJ_ROWS * XJ_SLICES, 0, st>>>(j);
    return cudaGetLastError() == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
}

int swx_xent_bwd(const swx_xent_args* a, void* stream) {
    const int c = xent_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dweight && a->dw_dtype != SWX_DTYPE_F32 && (a->dw_dtype != SWX_DTYPE_BF16 || a->dtype == SWX_DTYPE_F32)) return SWX_ERR_UNSUPPORTED;
    if (!a->dx && !a->dweight) return SWX_OK;
    const int64_t T = a->tokens, V = a->vocab, d = a->dim;
    if (T == 0) {
        if (!a->dweight) return SWX_OK;
        return cudaMemsetAsync(a->dweight, 0, (size_t)(V * d) * (a->dw_dtype == SWX_DTYPE_F32 ? 4 : 2), st) == cudaSuccess
                   ? SWX_OK : SWX_ERR_CUDA;
    }
    if (!a->x || !a->weight || !a->targets || !a->row_max || !a->row_rsum || !a->dloss || !a->workspace ||
        (a->reduction == SWX_XENT_MEAN && !a->count))
        return SWX_ERR_INVALID_ARG;
    const XentPlan q = xent_plan(a);
    if (a->workspace_bytes < q.bwd_total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    operands(a, q, ws, x, w, st);
    CUtensorMap x_k, w_k, x_mn, w_mn;
    if (!x.k_major(&x_k) || !w.k_major(&w_k) || !x.mn_major(&x_mn) || !w.mn_major(&w_mn)) return SWX_ERR_CUDA;
    const int npair = q.planes == 3 ? 6 : 1;
    const float* num = a->reduction == SWX_XENT_NONE ? nullptr : a->dloss;
    const float* den = a->reduction == SWX_XENT_MEAN ? a->count : nullptr;
    for (int64_t c0 = 0; c0 < V; c0 += q.piece) {
        const int64_t cw = std::min(q.piece, V - c0);
        const Operand pr{ws + q.off_p, cw, T, q.planes, q.ldp, T * q.ldp};
        CUtensorMap p_st, p_k, p_mn;
        // stores of 32 rows: 64 columns at once for one piece, 32 for each of three
        if (!encode_operand(&p_st, pr.p, cw, T, q.planes, q.ldp, T * q.ldp, q.planes == 3 ? 32 : 64, 32, q.planes == 1) ||
            !pr.k_major(&p_k) || !pr.mn_major(&p_mn))
            return SWX_ERR_CUDA;
        XentGemm g{};
        g.status = status; g.npair = npair; g.planes = q.planes;
        g.M = (int)T; g.N = (int)cw; g.mt = (int)q.mt; g.nt = (int)((cw + XE_TILE - 1) / XE_TILE); g.group = 32;
        g.nk = (int)((d + XE_K - 1) / XE_K); g.b0 = (int)c0;
        g.ksub = logits_ksub(q, g.nk);
        g.target = a->targets; g.ignore = a->ignore_index; g.col0 = (int)c0; g.vocab = V;
        g.row_max = a->row_max; g.row_rsum = a->row_rsum; g.dloss = a->dloss; g.reduction = a->reduction;
        if ((g.ksub < g.nk ? launch_gemm<XE_PROB, false, false, true>(g, x_k, w_k, p_st, XE_PAIRS, st)
                           : launch_gemm<XE_PROB, false, false>(g, x_k, w_k, p_st, XE_PAIRS, st)) != cudaSuccess)
            return SWX_ERR_CUDA;
        if (a->dx) {
            XentGemm h{};
            h.status = status; h.npair = npair;
            h.M = (int)T; h.N = (int)d; h.mt = (int)q.mt; h.nt = (int)((d + XE_TILE - 1) / XE_TILE);
            // spread: every piece the same number of steps (a short last one reads zeros), so that a
            // tile has the same parts in each
            h.nk = (int)(((q.dx.spread ? std::min(q.piece, V) : cw) + XE_K - 1) / XE_K); h.ksub = q.planes == 3 ? XE_KSUB : h.nk; h.kb0 = (int)c0;
            h.scale_num = num; h.scale_den = den;
            h.first = c0 == 0; h.last = c0 + cw == V; h.out = a->dx; h.ld = d;
            h.out_bf16 = a->dtype == SWX_DTYPE_BF16;
            h.spread = q.dx.spread;
            h.acc = h.out_bf16 || h.spread ? reinterpret_cast<float*>(ws + q.off_acc) : static_cast<float*>(a->dx);
            const cudaError_t e = q.planes == 3 ? launch_gemm<XE_DX, false, true, true>(h, p_k, w_mn, p_st, q.dx.pairs, st)
                                                : launch_gemm<XE_DX, false, true>(h, p_k, w_mn, p_st, q.dx.pairs, st);
            if (e != cudaSuccess) return SWX_ERR_CUDA;
            if (h.spread && h.last && launch_sum(h, q.dx.pairs, st) != cudaSuccess) return SWX_ERR_CUDA;
        }
        if (a->dweight) {
            XentGemm h{};
            h.status = status; h.npair = npair;
            h.M = (int)cw; h.N = (int)d; h.mt = (int)((cw + XE_TILE - 1) / XE_TILE); h.nt = (int)((d + XE_TILE - 1) / XE_TILE);
            h.nk = (int)((T + XE_K - 1) / XE_K); h.ksub = q.planes == 3 ? XE_KSUB : h.nk;
            h.scale_num = num; h.scale_den = den;
            h.first = h.last = 1; h.ld = d;
            h.out_bf16 = a->dw_dtype == SWX_DTYPE_BF16;
            h.out = static_cast<uint8_t*>(a->dweight) + c0 * d * (h.out_bf16 ? 2 : 4);
            const XentDeal e = deal((int64_t)h.mt * h.nt, h.nk);
            h.spread = e.spread;
            // whole tiles with fp32 operands sum up in the (fp32) result
            h.acc = e.spread ? reinterpret_cast<float*>(ws + q.off_acc_w) : static_cast<float*>(h.out);
            const cudaError_t r = q.planes == 3 ? launch_gemm<XE_DW, true, true, true>(h, p_mn, x_mn, p_st, e.pairs, st)
                                                : launch_gemm<XE_DW, true, true>(h, p_mn, x_mn, p_st, e.pairs, st);
            if (r != cudaSuccess) return SWX_ERR_CUDA;
            if (e.spread && launch_sum(h, e.pairs, st) != cudaSuccess) return SWX_ERR_CUDA;
        }
    }
    return SWX_OK;
}

}  // extern "C"
