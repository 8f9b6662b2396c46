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
// forward 178 us (88 % of the SM's active cycles on products, 1547 TFLOP/s), dlogit 184 us (it writes 268 MB), dx 190
// (93 %, on 64 of 74 pairs); 8192 x 50001 x 1024 0.51, 0.57, 0.58 and 0.60 ms, where a library
// product of the same size alone takes 0.56 to 0.61.  The logits' epilogue (an exponential for each) fits behind a
// tile's products from about 512 values of the contraction on; below that it bounds the forward.
//
// fp32 operands are split into three bf16 pieces (24 bits) and multiplied as the six
// products of pieces above 2^-24, smallest first, on the same kernel.
#include <algorithm>
#include <cmath>

#include "head_gemm.cuh"

namespace swx {

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

HeadPlan head_plan(const HeadOps& o) {
    HeadPlan q{};
    const int64_t T = o.T, V = o.V, d = o.d;
    q.es = o.dtype == SWX_DTYPE_F32 ? 4 : 2;
    q.planes = o.dtype == SWX_DTYPE_F32 ? 3 : 1;
    q.dp = (d + 7) / 8 * 8;
    q.pack_x = !direct_ok(o.x, o.x_sr, o.dtype);
    q.pack_w = !direct_ok(o.w, o.w_sr, o.dtype);
    q.mt = (T + XE_TILE - 1) / XE_TILE;
    q.nt = (V + XE_TILE - 1) / XE_TILE;
    q.off_x = 0;
    q.off_w = q.off_x + (q.pack_x ? up256(q.planes * T * q.dp * 2) : 0);
    q.base = q.off_w + (q.pack_w ? up256(q.planes * V * q.dp * 2) : 0);
    q.piece = piece_columns(T, V, d, q.planes);
    q.ldp = q.piece;
    q.off_p = q.base;
    q.off_acc = q.off_p + up256((int64_t)q.planes * T * q.ldp * 2);
    // the running sums of dx (bf16 result: in fp32; one for each part of a spread tile), then
    // the parts of dW, which live for one piece
    const int64_t dt = (d + XE_TILE - 1) / XE_TILE;
    const int64_t cl = V - (V - 1) / q.piece * q.piece;      // columns of the last piece
    q.dx = deal(q.mt * dt, (std::min(q.piece, V) + XE_K - 1) / XE_K);
    const bool own_acc = q.dx.spread || (o.dtype == SWX_DTYPE_BF16 && q.piece < V);
    q.off_acc_w = q.off_acc + (own_acc ? up256(q.dx.parts * T * d * 4) : 0);
    int64_t w = 0;
    for (const int64_t cw : {std::min<int64_t>(q.piece, V), cl}) {
        const XentDeal e = deal((cw + XE_TILE - 1) / XE_TILE * dt, (T + XE_K - 1) / XE_K);
        if (e.spread) w = std::max<int64_t>(w, up256(e.parts * cw * d * 4));
    }
    q.bwd_total = q.off_acc_w + w;
    return q;
}

int head_check(const HeadOps& o) {
    if (o.T < 0 || o.V < 1 || o.d < 1) return SWX_ERR_INVALID_ARG;
    if (o.dtype != SWX_DTYPE_F32 && o.dtype != SWX_DTYPE_BF16) return SWX_ERR_UNSUPPORTED;
    if (o.T > (1 << 28) || o.V > (1 << 28) || o.d > (1 << 16)) return SWX_ERR_UNSUPPORTED;
    return SWX_OK;
}

void head_operands(const HeadOps& o, const HeadPlan& q, uint8_t* ws, Operand& x, Operand& w, cudaStream_t st) {
    x = q.pack_x ? Operand{ws + q.off_x, o.d, o.T, q.planes, q.dp, o.T * q.dp} : Operand{o.x, o.d, o.T, 1, o.x_sr, 0};
    w = q.pack_w ? Operand{ws + q.off_w, o.d, o.V, q.planes, q.dp, o.V * q.dp} : Operand{o.w, o.d, o.V, 1, o.w_sr, 0};
    const XentPack px{o.x, o.x_sr, q.pack_x ? o.T : 0, reinterpret_cast<__nv_bfloat16*>(ws + q.off_x)};
    const XentPack pw{o.w, o.w_sr, q.pack_w ? o.V : 0, reinterpret_cast<__nv_bfloat16*>(ws + q.off_w)};
    const int64_t n = (px.rows + pw.rows) * (q.dp / 8);
    if (n == 0) return;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 16);
    if (o.dtype == SWX_DTYPE_F32) xent_pack_kernel<float><<<grid, 256, 0, st>>>(px, pw, (int)o.d, (int)q.dp);
    else xent_pack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(px, pw, (int)o.d, (int)q.dp);
}

static cudaError_t launch_sum(const XentGemm& p, int pairs, cudaStream_t st) {
    const int64_t n = (int64_t)p.M * ((p.N + 3) / 4);
    xent_sum_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p, pairs);
    return cudaGetLastError();
}

int head_piece_products(const HeadOps& o, const HeadPlan& q, uint8_t* ws, const Operand& x, const Operand& w, const Operand& pr,
                        const HeadGrads& gr, int64_t c0, int64_t cw, int* status, cudaStream_t st) {
    const int64_t T = o.T, V = o.V, d = o.d;
    const int npair = q.planes == 3 ? 6 : 1;
    CUtensorMap x_mn, w_mn, p_k, p_mn;
    if (!x.mn_major(&x_mn) || !w.mn_major(&w_mn) || !pr.k_major(&p_k) || !pr.mn_major(&p_mn)) return SWX_ERR_CUDA;
    if (gr.dx) {
        XentGemm h{};
        h.status = status; h.npair = npair;
        h.M = (int)T; h.N = (int)d; h.mt = (int)q.mt; h.nt = (int)((d + XE_TILE - 1) / XE_TILE);
        // spread: every piece the same number of steps (a short last one reads zeros), so that a
        // tile has the same parts in each
        h.nk = (int)(((q.dx.spread ? std::min(q.piece, V) : cw) + XE_K - 1) / XE_K); h.ksub = q.planes == 3 ? XE_KSUB : h.nk; h.kb0 = (int)c0;
        h.scale_num = gr.num; h.scale_den = gr.den;
        h.first = c0 == 0; h.last = c0 + cw == V; h.out = gr.dx; h.ld = d;
        h.out_bf16 = o.dtype == SWX_DTYPE_BF16;
        h.spread = q.dx.spread;
        h.acc = h.out_bf16 || h.spread ? reinterpret_cast<float*>(ws + q.off_acc) : static_cast<float*>(gr.dx);
        const cudaError_t e = q.planes == 3 ? launch_gemm<XE_DX, false, true, true>(h, p_k, w_mn, p_k, q.dx.pairs, st)
                                            : launch_gemm<XE_DX, false, true>(h, p_k, w_mn, p_k, q.dx.pairs, st);
        if (e != cudaSuccess) return SWX_ERR_CUDA;
        if (h.spread && h.last && launch_sum(h, q.dx.pairs, st) != cudaSuccess) return SWX_ERR_CUDA;
    }
    if (gr.dw) {
        XentGemm h{};
        h.status = status; h.npair = npair;
        h.M = (int)cw; h.N = (int)d; h.mt = (int)((cw + XE_TILE - 1) / XE_TILE); h.nt = (int)((d + XE_TILE - 1) / XE_TILE);
        h.nk = (int)((T + XE_K - 1) / XE_K); h.ksub = q.planes == 3 ? XE_KSUB : h.nk;
        h.scale_num = gr.num; h.scale_den = gr.den;
        h.first = h.last = 1; h.ld = d;
        h.out_bf16 = gr.dw_bf16;
        h.out = static_cast<uint8_t*>(gr.dw) + c0 * d * (h.out_bf16 ? 2 : 4);
        const XentDeal e = deal((int64_t)h.mt * h.nt, h.nk);
        h.spread = e.spread;
        // whole tiles with fp32 operands sum up in the (fp32) result
        h.acc = e.spread ? reinterpret_cast<float*>(ws + q.off_acc_w) : static_cast<float*>(h.out);
        const cudaError_t r = q.planes == 3 ? launch_gemm<XE_DW, true, true, true>(h, p_mn, x_mn, p_k, e.pairs, st)
                                            : launch_gemm<XE_DW, true, true>(h, p_mn, x_mn, p_k, e.pairs, st);
        if (r != cudaSuccess) return SWX_ERR_CUDA;
        if (e.spread && launch_sum(h, e.pairs, st) != cudaSuccess) return SWX_ERR_CUDA;
    }
    return SWX_OK;
}

// The forward's workspace: the operands' copies, then the pieces of each row's sum, the targets' logits, the joining
// CTAs' sums and their counter.
struct XentFwd { int64_t off_part, off_hit, off_rows, off_cnt, total; };

static XentFwd xent_fwd_plan(const HeadPlan& q, int64_t T) {
    XentFwd f{};
    f.off_part = q.base;
    f.off_hit = f.off_part + up256(2 * q.nt * T * 8);
    f.off_rows = f.off_hit + up256(T * 4);
    f.off_cnt = f.off_rows + up256((T + XJ_ROWS - 1) / XJ_ROWS * 16);
    f.total = f.off_cnt + 256;
    return f;
}

static HeadOps ops_of(const swx_xent_args* a) {
    return HeadOps{a->tokens, a->vocab, a->dim, a->dtype, a->x, a->x_sr, a->weight, a->w_sr};
}

static int xent_check(const swx_xent_args* a) {
    if (!a) return SWX_ERR_INVALID_ARG;
    const int c = head_check(ops_of(a));
    if (c != SWX_OK) return c;
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
    return c != SWX_OK ? -c : xent_fwd_plan(head_plan(ops_of(a)), a->tokens).total;
}

int64_t swx_xent_bwd_workspace_bytes(const swx_xent_args* a) {
    const int c = xent_check(a);
    return c != SWX_OK ? -c : head_plan(ops_of(a)).bwd_total;
}

int swx_xent_fwd(const swx_xent_args* a, void* stream) {
    const int c = xent_check(a);
    if (c != SWX_OK) return c;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool none = a->reduction == SWX_XENT_NONE;
    if (!none && (!a->loss || !a->count)) return SWX_ERR_INVALID_ARG;
    if (a->tokens > 0 && (!a->x || !a->weight || !a->targets || !a->row_max || !a->row_rsum || !a->workspace || (none && !a->loss)))
        return SWX_ERR_INVALID_ARG;
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    const XentFwd f = xent_fwd_plan(q, a->tokens);
    if (a->tokens > 0 && (a->workspace_bytes < f.total || !aligned16(a->workspace))) return SWX_ERR_INVALID_ARG;
    if (a->tokens == 0) {
        if (none) return SWX_OK;
        // no token: a sum of 0, a mean of 0 / 0
        if (cudaMemsetAsync(a->count, 0, 4, st) != cudaSuccess) return SWX_ERR_CUDA;
        return cudaMemsetAsync(a->loss, a->reduction == SWX_XENT_MEAN ? 0xff : 0, 4, st) == cudaSuccess ? SWX_OK : SWX_ERR_CUDA;
    }
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    head_operands(o, q, ws, x, w, st);
    CUtensorMap mx, mw;
    if (!x.k_major(&mx) || !w.k_major(&mw)) return SWX_ERR_CUDA;
    XentGemm g = logits_gemm(o, q, 0, o.V, status);
    g.target = a->targets; g.ignore = a->ignore_index;
    g.part = reinterpret_cast<float2*>(ws + f.off_part);
    g.hit = reinterpret_cast<float*>(ws + f.off_hit);
    g.counter = reinterpret_cast<int*>(ws + f.off_cnt);
    if (launch_logits<XE_LSE>(g, mx, mw, mx, st) != cudaSuccess) return SWX_ERR_CUDA;
    XentJoin j{};
    j.T = a->tokens; j.V = a->vocab; j.np = (int)(2 * q.nt); j.part = g.part; j.hit = g.hit; j.target = a->targets;
    j.ignore = a->ignore_index; j.row_max = a->row_max; j.row_rsum = a->row_rsum;
    j.rows = none ? a->loss : nullptr; j.sums = reinterpret_cast<double2*>(ws + f.off_rows);
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
    const HeadOps o = ops_of(a);
    const HeadPlan q = head_plan(o);
    if (a->workspace_bytes < q.bwd_total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    const HeadGrads gr{a->dx, a->dweight, a->dw_dtype == SWX_DTYPE_BF16, a->reduction == SWX_XENT_NONE ? nullptr : a->dloss,
                       a->reduction == SWX_XENT_MEAN ? a->count : nullptr};
    return head_backward(o, q, static_cast<uint8_t*>(a->workspace), gr, st, launch_logits<XE_PROB>, [a](XentGemm& g) {
        g.target = a->targets; g.ignore = a->ignore_index;
        g.row_max = a->row_max; g.row_rsum = a->row_rsum; g.dloss = a->dloss; g.reduction = a->reduction;
    });
}

}  // extern "C"
