// Log probabilities of given tokens under a linear head, with the entropy and the top alternatives, without keeping
// the logits:  z = x W^T,  l_v = z_v / tau - log sum exp(z / tau),  p = e^l,
//   log_probs = l_y,  entropy = -sum p l,  top: the K largest z (the lowest word first among equals).
// Backward, for upstream gradients g of log_probs and h of the entropy H:
//   dz_v = (g [v == y] - p_v (g + h (l_v + H))) / tau,  dx = dz W,  dW = dz^T x.
//
// Forward: the head's product (head_gemm.cuh) with an epilogue that keeps three floats for each half of a 256-column tile: the
// maximum m, s = sum e and w = sum e u of e = 2^u, u = (z - m) log2(e) / tau; with alternatives also the two largest logits of every
// 16 columns (8 bytes), or, for a small vocabulary, the logits.  Then one kernel for the rows: the statistics joined, and
//   H = ln s - ln2 w / s.
// Alternatives: the K + 4 groups of 16 columns with the largest maxima hold the K + 4 largest logits; a group whose second value
// passes too is taken whole.  The tensor core's sums are a few 2^-23 off, enough to turn two close logits round.  So where two
// candidates are closer than a bound of that error (from the norms of the row and of the longest word, or unknown where few rows do not
// pay for reading the words' norms), their products are formed again with a bound of their own, and those that are still
// too close exactly.  The bounds rest on measured sums: n additions of 16 products lost 0.6 n 2^-24 of the magnitudes at most at n = 32,
// 0.94 at 256 and 1.2 at 512 (terms of one sign, the worst), a warp's mma.sync 0.44 to 0.48; they allow 2 and 4.
//
// Backward: as the loss's, with dz in the epilogue (rounded to bf16 once, the tensor core's operand; fp32 operands: three pieces).
#include "head_gemm.cuh"
#include "warp_mma.cuh"

namespace swx {

constexpr int SC_EXTRA = 4;                   // candidates beyond K
constexpr int SC_THREADS = 256, SC_PER = 8;
constexpr int SC_NORM_THREADS = 128;
constexpr float LN2 = 0.69314718055994531f;

struct ScoreRows {
    int64_t T, V, d;
    int np;                                   // statistics per row
    const float4* score; const float* hit; const int64_t* target; int64_t ignore;
    // the statistics' exponents' scale (the products': (1 + cut) log2(e) / temperature); the products' mean cut, and log2(e) /
    // temperature for logits that carry it or do without
    float k2, cut, exact_k2;
    float* row_max; float* row_sum; float* log_probs; float* entropy;
    // alternatives
    int top, cand;                            // K, candidates kept of the records
    const float* largest; const float* runner_up; const float* all; int64_t groups, stride;
    const void* x; int64_t x_sr; const void* w; int64_t w_sr; int vec;
    const uint32_t* longest;                  // the largest squared norm of a word, its bits; or none
    float* top_log_probs; int64_t* top_ids;
};

// A row's results from its statistics: the target's logit as the sums saw it, so that no value is above 0.
__device__ __forceinline__ void score_finish(const ScoreRows& p, int64_t row, const Score& a) {
    const int64_t y = p.target[row];
    const float ls = logf(a.s);
    if (p.row_max) { p.row_max[row] = a.m; p.row_sum[row] = a.s; }
    const bool live = y != p.ignore;
    p.log_probs[row] = !live ? 0.f : y >= 0 && y < p.V ? (p.hit[row] - a.m) * p.k2 * LN2 - ls : __int_as_float(0x7fc00000);
    p.entropy[row] = live ? ls - LN2 * a.w / a.s : 0.f;
}

// Warp = one row.
__global__ void __launch_bounds__(SC_THREADS) score_rows_kernel(const ScoreRows p) {
    wait_for_previous();
    const int64_t row = (int64_t)blockIdx.x * (SC_THREADS / 32) + threadIdx.x / 32;
    if (row >= p.T) return;
    const int lane = threadIdx.x % 32;
    const Score a = score_join_parts(p.score + row * p.np, p.np, p.k2, lane, 32);
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

// Products of a row of x with R rows of the weight over a warp, in fp32: z, and a bound of each one's error.  A lane sums d / 64
// products in each of two chains, which are joined in six steps, 2^-24 of the magnitudes each; |x| |w| bounds those.
constexpr int SC_DOTS = 4;
struct Products { float z[SC_DOTS], e[SC_DOTS]; };
template <typename T>
__device__ __forceinline__ Products products(const T* x, const T* const (&w)[SC_DOTS], int64_t d, bool vec, int lane) {
    constexpr int N = 16 / sizeof(T);
    float2 a[SC_DOTS] = {}, n[SC_DOTS + 1] = {};
    int64_t tail = 0;
    if (vec) {
#pragma unroll 2
        for (int64_t k = lane * N; k + N <= d; k += 32 * N) {
            const uint4 qx = *reinterpret_cast<const uint4*>(x + k);
            uint4 q[SC_DOTS];
#pragma unroll
            for (int r = 0; r < SC_DOTS; ++r) q[r] = *reinterpret_cast<const uint4*>(w[r] + k);
            float2 xv[N / 2], v[N / 2];
            unpack(x, qx, xv);
#pragma unroll
            for (int j = 0; j < N / 2; ++j) n[SC_DOTS] = fma2(xv[j], xv[j], n[SC_DOTS]);
#pragma unroll
            for (int r = 0; r < SC_DOTS; ++r) {
                unpack(x, q[r], v);
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    a[r] = fma2(xv[j], v[j], a[r]);
                    n[r] = fma2(v[j], v[j], n[r]);
                }
            }
        }
        tail = d / N * N;
    }
    for (int64_t k = tail + lane; k < d; k += 32) {
        const float xv = Elem<T>::to_f(x[k]);
        n[SC_DOTS].x = fmaf(xv, xv, n[SC_DOTS].x);
#pragma unroll
        for (int r = 0; r < SC_DOTS; ++r) {
            const float v = Elem<T>::to_f(w[r][k]);
            a[r].x = fmaf(xv, v, a[r].x);
            n[r].x = fmaf(v, v, n[r].x);
        }
    }
    Products out;
    float s[2 * SC_DOTS + 1];
#pragma unroll
    for (int r = 0; r < SC_DOTS; ++r) { s[r] = a[r].x + a[r].y; s[SC_DOTS + r] = n[r].x + n[r].y; }
    s[2 * SC_DOTS] = n[SC_DOTS].x + n[SC_DOTS].y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < 2 * SC_DOTS + 1; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
    const float f = ((vec ? d * (1.f / 64) : d * (1.f / 32)) + 16.f) * 0x1p-24f * 1.01f;
    const float xn = f * sqrtf(fmaxf(s[2 * SC_DOTS], 0x1p-100f));       // (smaller squares may have underflowed)
#pragma unroll
    for (int r = 0; r < SC_DOTS; ++r) { out.z[r] = s[r]; out.e[r] = xn * sqrtf(fmaxf(s[SC_DOTS + r], 0x1p-100f)); }
    return out;
}

// Products of the candidates list[0 .. n) with the row, z and a bound of the error in out (the order of out is the
// candidates').  fp32 operands: a warp takes four candidates at a time.
template <int THREADS>
__device__ __forceinline__ void candidate_products(const float* x, const float* w, int64_t w_sr, int64_t d, bool vec, const int* col, const int* list,
                                                   int n, float2* out, float2*) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int i = SC_DOTS * warp; i < n; i += SC_DOTS * (THREADS / 32)) {
        const float* rows[SC_DOTS];
#pragma unroll
        for (int r = 0; r < SC_DOTS; ++r) rows[r] = w + col[list[min(i + r, n - 1)]] * w_sr;
        const Products q = products(x, rows, d, vec, lane);
        if (lane == 0) {
#pragma unroll
            for (int r = 0; r < SC_DOTS; ++r)
                if (i + r < n) out[list[i + r]] = make_float2(q.z[r], q.e[r]);
        }
    }
}

// bf16 operands: on mma.sync, 16 candidates by 16 steps of the width, straight from memory into the A operand (lane (g, c) takes the 8
// values from 8 c on of rows g and g + 8 of 32 steps, and the row of x in the same order into column 0 of B; a sum does not see the
// order).  A second product of the magnitudes into column 1 bounds the error: a warp's sum is cut 2^-22 at most of the magnitudes at
// each product, the warps' sums are added in fp32.  The warps split the width.  Two steps' loads at a time: for 16 candidates in the small
// CTAs that many rows take (their registers decide how many run), for 32 in the large ones.
constexpr int score_block(int threads) { return threads == 128 ? 16 : 32; }
template <int THREADS>
__device__ __forceinline__ void candidate_products(const __nv_bfloat16* x, const __nv_bfloat16* w, int64_t w_sr, int64_t d, bool, const int* col,
                                                   const int* list, int n, float2* out, float2* dots) {
    constexpr int W = THREADS / 32, B = score_block(THREADS), G = B / 16;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    const int steps = (int)((d + 31) / 32);
    const float cut = (2 * ((steps + W - 1) / W) + W + 4) * 0x1p-22f * 1.02f;
    for (int b = 0; b < n; b += B) {
        const __nv_bfloat16* rows[G][2];
        float acc[G][4] = {};
        const int groups = (min(B, n - b) + 15) / 16;
#pragma unroll
        for (int r = 0; r < G; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) rows[r][h] = w + col[list[min(b + 16 * r + 8 * h + g, n - 1)]] * w_sr;
        constexpr int D = 2;                   // steps whose loads are issued together
        for (int s0 = warp; s0 < steps; s0 += D * W) {
            uint4 q[D][G][2], xq[D];
#pragma unroll
            for (int i = 0; i < D; ++i) {
                const int s = s0 + i * W;
                const int64_t k = 32 * (int64_t)s + 8 * c;
                if (s >= steps) continue;
                xq[i] = load8(x, k, d);
#pragma unroll
                for (int r = 0; r < G; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (r < groups) q[i][r][h] = load8(rows[r][h], k, d);
            }
            const uint32_t sign = 0x7fff7fffu;
#pragma unroll
            for (int i = 0; i < D; ++i) {
                if (s0 + i * W >= steps) continue;
                const uint4 v = xq[i];
                const uint32_t bz[2][2] = {{g == 0 ? v.x : 0, g == 0 ? v.y : 0}, {g == 0 ? v.z : 0, g == 0 ? v.w : 0}};
                const uint32_t bm[2][2] = {{g == 1 ? v.x & sign : 0, g == 1 ? v.y & sign : 0}, {g == 1 ? v.z & sign : 0, g == 1 ? v.w & sign : 0}};
#pragma unroll
                for (int r = 0; r < G; ++r) {
                    if (r >= groups) continue;
                    const uint4 *u = q[i][r];
                    const uint32_t a0[4] = {u[0].x, u[1].x, u[0].y, u[1].y}, a1[4] = {u[0].z, u[1].z, u[0].w, u[1].w};
                    mma_bf16(acc[r], a0, bz[0]);
                    mma_bf16(acc[r], a1, bz[1]);
                    const uint32_t m0[4] = {a0[0] & sign, a0[1] & sign, a0[2] & sign, a0[3] & sign};
                    const uint32_t m1[4] = {a1[0] & sign, a1[1] & sign, a1[2] & sign, a1[3] & sign};
                    mma_bf16(acc[r], m0, bm[0]);
                    mma_bf16(acc[r], m1, bm[1]);
                }
            }
        }
        if (c == 0) {
#pragma unroll
            for (int r = 0; r < G; ++r) {
                dots[warp * B + 16 * r + g] = make_float2(acc[r][0], acc[r][1]);
                dots[warp * B + 16 * r + 8 + g] = make_float2(acc[r][2], acc[r][3]);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < min(B, n - b); i += THREADS) {
            float2 t = dots[i];
#pragma unroll
            for (int j = 1; j < W; ++j) {
                const float2 u = dots[j * B + i];
                t.x += u.x;
                t.y += u.y;
            }
            out[list[b + i]] = make_float2(t.x, t.y * cut);
        }
        __syncthreads();
    }
}

// The same product of one row of the weight, exact but for a last rounding.  fp32 operands: in fp64 (2^-53 of the magnitudes).
__device__ __forceinline__ double product_exact(const float* x, const float* w, int64_t d, bool vec, int lane) {
    double a = 0.;
    int64_t tail = 0;
    if (vec) {
#pragma unroll 4
        for (int64_t k = lane * 4; k + 4 <= d; k += 128) {
            const float4 xv = *reinterpret_cast<const float4*>(x + k), v = *reinterpret_cast<const float4*>(w + k);
            a = fma((double)xv.x, (double)v.x, fma((double)xv.y, (double)v.y, fma((double)xv.z, (double)v.z, fma((double)xv.w, (double)v.w, a))));
        }
        tail = d / 4 * 4;
    }
    for (int64_t k = tail + lane; k < d; k += 32) a = fma((double)x[k], (double)w[k], a);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}
// bf16 operands: the products (16 bits) are exact in fp32; a lane sums its own with what each addition rounds off kept in a second
// sum (Knuth's two-sum; hi + lo is good to about 2^-46 of the magnitudes), the lanes' sums are added in fp64.
struct TwoSum {
    float2 hi = {0.f, 0.f}, lo = {0.f, 0.f};
    __device__ __forceinline__ void add(float2 p) {
        const float2 s = add2(hi, p), b = add2(s, f2(-hi.x, -hi.y));
        const float2 r = add2(hi, f2(b.x - s.x, b.y - s.y)), q = add2(p, f2(-b.x, -b.y));
        lo = add2(lo, add2(r, q));
        hi = s;
    }
    static __device__ __forceinline__ double one(float h, float l) { return isinf(h) ? (double)h : (double)h + (double)l; }
    __device__ __forceinline__ double value() const { return one(hi.x, lo.x) + one(hi.y, lo.y); }
};
__device__ __forceinline__ double product_exact(const __nv_bfloat16* x, const __nv_bfloat16* w, int64_t d, bool, int lane) {
    TwoSum s[2];
#pragma unroll 1
    for (int64_t k = lane * 8; k < d; k += 256) {
        float2 xv[4], v[4];
        unpack(x, load8(x, k, d), xv);
        unpack(x, load8(w, k, d), v);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j & 1].add(mul2(xv[j], v[j]));
    }
    double a = s[0].value() + s[1].value();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}

// Columns that the candidates can come to: cand + cand / 2 values, or groups taken whole.
static __host__ __device__ int score_candidates(bool all, int cand) { return (all ? 1 : 16) * (cand + cand / 2); }

static size_t score_top_smem(bool all, int cand) {
    return (size_t)topk_capacity(cand, SC_PER) * 8 + cand * 8 + (size_t)score_candidates(all, cand) * 16;
}

__device__ __forceinline__ float drop_column(float v) { return __uint_as_float(__float_as_uint(v) & ~15u); }

// CTA = one row: its statistics, the candidates from the records (ALL: from the logits), their order.
// THREADS is at least the number of candidates.  Large CTAs: three on an SM (96 registers let two in; 2048 rows of 50001 x 1024 with
// 128 alternatives 566 us then, 491 now, with 64 366 and 308).
template <typename T, bool ALL, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 0) score_top_kernel(const ScoreRows p) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ int count[2], ncand, nlist, nexact, owners[THREADS];
    __shared__ uint32_t scratch[THREADS + 1];
    __shared__ Score part[THREADS / 32];
    __shared__ float norms[THREADS / 32], logsum;
    __shared__ float2 dots[sizeof(T) == 2 ? THREADS / 32 * score_block(THREADS) : 1];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint64_t* buf = reinterpret_cast<uint64_t*>(raw);
    uint64_t* kept = buf + topk_capacity(p.cand, SC_PER);
    uint64_t* val = kept + p.cand;                                   // candidates' logits: value and error, then order_key bits of fp64
    float2* ze = reinterpret_cast<float2*>(val);
    int* col = reinterpret_cast<int*>(val + score_candidates(ALL, p.cand));
    int* list = col + score_candidates(ALL, p.cand);
    const T* x = static_cast<const T*>(p.x) + row * p.x_sr;
    const T* w = static_cast<const T*>(p.w);
    wait_for_previous();

    // the largest of this thread's share of the values: logits (a NaN as -inf), or the records' largest ones
    const int64_t n = ALL ? p.V : p.groups;
    const float* from = ALL ? p.all + row * p.V : p.largest + row * p.stride;
    auto value = [&](int64_t i) { const float z = from[i]; return ALL && z != z ? -INFINITY : z; };
    float most = -INFINITY;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < n; i += THREADS) most = fmaxf(most, value(i));
    if (threadIdx.x == 0) count[0] = count[1] = ncand = nlist = 0;
    if (p.longest) {
        float xx = 0.f;
        for (int64_t k = threadIdx.x; k < p.d; k += THREADS) { const float v = Elem<T>::to_f(x[k]); xx = fmaf(v, v, xx); }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) xx += __shfl_xor_sync(0xffffffffu, xx, o);
        if (lane == 0) norms[warp] = xx;
    }
    const Score a = score_join_row<THREADS>(p.score + row * p.np, p.np, p.k2, part);
    if (threadIdx.x == 0) {
        score_finish(p, row, a);
        logsum = logf(a.s);
    }
    if (p.target[row] == p.ignore) {                                 // a token that does not count
        for (int i = threadIdx.x; i < p.top; i += THREADS) {
            p.top_log_probs[row * p.top + i] = 0.f;
            p.top_ids[row * p.top + i] = -1;
        }
        return;
    }

    TopK<THREADS, SC_PER> best(buf, kept, count, p.cand);
    struct Entry { float v; uint32_t i; };
    auto load = [&](int t, int64_t j, Entry& e) {
        const int64_t i = t + j * THREADS;
        e.i = (uint32_t)i;
        e.v = i < n ? value(i) : __int_as_float(0x7fc00000);
    };
    auto emit = [&](const Entry& e, auto f) { if (e.v == e.v) f(e.v, e.i); };
    if (!best.template gather<Entry>(threadIdx.x < n ? order_key(most) : 0, scratch, owners, (n + THREADS - 1) / THREADS, load, emit)) {
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
    // candidates: what passed the threshold, cut to the largest where that is far more than asked for; ze.y < 0: not known yet
    if (best.n > p.cand + p.cand / 2) best.rank();
    const int m = best.n;
    float off = INFINITY;                                            // bound of the error of the product's logits
    if (p.longest) {
        float xx = norms[0];
#pragma unroll
        for (int i = 1; i < THREADS / 32; ++i) xx += norms[i];
        // (d / 16 + 8) additions' cuts of 2^-23 of the magnitudes (see above), as much again for three pieces; norms of squares that
        // underflowed
        off = (p.d * (1.f / 16) + 8.f) * (sizeof(T) == 4 ? 0x1p-22f : 0x1p-23f) * 1.01f * sqrtf(fmaxf(xx, 0x1p-100f)) *
              sqrtf(fmaxf(__uint_as_float(*p.longest), 0x1p-100f));
    }
    const float least = ALL ? 0.f : order_value((uint32_t)(best.floor >> 32));
    for (int i = threadIdx.x; i < p.cand; i += THREADS) kept[i] = 0;  // from here on: the candidates by rank
    for (int i = threadIdx.x; i < m; i += THREADS) {
        const uint32_t g = key_index(buf[i]);
        const float z = order_value((uint32_t)(buf[i] >> 32));
        const float second = ALL ? 0.f : p.runner_up[row * p.stride + g];
        if (ALL) {
            const int at = atomicAdd(&ncand, 1);
            col[at] = (int)g;
            ze[at] = make_float2(fmaf(z, p.cut, z), off);
        } else if (drop_column(second) >= drop_column(least)) {
            const int c = (int)min((int64_t)16, p.V - (int64_t)g * 16), at = atomicAdd(&ncand, c);
            for (int j = 0; j < c; ++j) {
                col[at + j] = (int)g * 16 + j;
                ze[at + j] = make_float2(0.f, -1.f);
            }
        } else {
            const int at = atomicAdd(&ncand, 1);
            col[at] = (int)(g * 16 + (__float_as_uint(second) & 15u));
            ze[at] = make_float2(fmaf(z, p.cut, z), off);
        }
    }
    __syncthreads();
    const int nc = ncand;
    // those not known, or not told apart from a known one: their products again
    for (int i = threadIdx.x; i < nc; i += THREADS) {
        const float2 z = ze[i];
        bool close = z.y < 0.f || off == INFINITY;
        if (off < INFINITY) {
#pragma unroll 4
            for (int j = 0; j < nc; ++j) {
                const float2 o = ze[j];
                close |= (j != i) & (o.y >= 0.f) & !(fabsf(o.x - z.x) > 2.0001f * off);
            }
        }
        if (close) list[atomicAdd(&nlist, 1)] = i;
    }
    __syncthreads();
    candidate_products<THREADS>(x, w, p.w_sr, p.d, p.vec, col, list, nlist, ze, dots);
    if (threadIdx.x == 0) nexact = 0;
    __syncthreads();
    // their ranks (equal ones by their columns), and those still not told apart from another (the bounds' sum, and the difference's own rounding)
    auto put = [&](int rank, int i) { if (rank < p.top) kept[rank] = i; };
    for (int i = threadIdx.x; i < nc; i += THREADS) {
        const float2 z = ze[i];
        const int c = col[i];
        int r = 0;
        bool close = false;
#pragma unroll 4
        for (int j = 0; j < nc; ++j) {
            const float2 o = ze[j];
            r += (int)(o.x > z.x) + (int)((o.x == z.x) & (col[j] < c));
            close |= (j != i) & !(fabsf(o.x - z.x) > (o.y + z.y) * 1.0001f);
        }
        if (close) list[atomicAdd(&nexact, 1)] = i;
        else put(r, i);
    }
    __syncthreads();
    const int ne = nexact;
    // the first alternative has the statistics' maximum (its own sum, with other roundings, would put its probability above 1, by a part of
    // |z| / temperature), and the others their distance from the first
    const float ls = logsum;
    auto write = [&](auto z) {
        for (int i = threadIdx.x; i < p.top; i += THREADS) {
            p.top_log_probs[row * p.top + i] = (float)((z(kept[i]) - z(kept[0])) * p.exact_k2) * LN2 - ls;
            p.top_ids[row * p.top + i] = col[kept[i]];
        }
    };
    if (ne == 0) {
        write([&](uint64_t i) { return (double)ze[i].x; });
        return;
    }
    // exactly: a candidate that is told apart from all others keeps its rank, so the close ones are ranked anew
    for (int i = threadIdx.x; i < nc; i += THREADS) val[i] = order_key((double)ze[i].x);
    __syncthreads();
    for (int k = warp; k < ne; k += THREADS / 32) {
        const int i = list[k];
        const double z = product_exact(x, w + (int64_t)col[i] * p.w_sr, p.d, p.vec, lane);
        if (lane == 0) val[i] = order_key(z);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < ne; k += THREADS) {
        const int i = list[k], c = col[i];
        const uint64_t v = val[i];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < nc; ++j) {
            const uint64_t o = val[j];
            r += (int)(o > v) + (int)((o == v) & (col[j] < c));
        }
        put(r, i);
    }
    __syncthreads();
    write([&](uint64_t i) { const uint64_t v = val[i]; return __longlong_as_double((long long)(v >> 63 ? v & ~(1ull << 63) : ~v)); });
}

// The largest squared norm of a word, a warp for each (fp32 sums of squares: 2^-24 for each of d / 32 additions, far inside the
// bound's slack).  One read of the weight, beside the logits' product: that kernel's 10 warps of up to 160 registers leave
// each quarter of an SM one warp of 32 (4096 rows of 50001 x 1024 with 32 alternatives 431 us with this kernel behind the
// product, 410 so).  Where the product takes more registers (fp32 operands) this one fills the SMs after it.
template <typename T>
__global__ void __launch_bounds__(SC_NORM_THREADS, 2048 / SC_NORM_THREADS) longest_word_kernel(const T* w, int64_t w_sr, int64_t V, int64_t d, bool vec, uint32_t* longest) {
    constexpr int N = 16 / sizeof(T), W = SC_NORM_THREADS / 32;
    const int lane = threadIdx.x % 32;
    float top = 0.f;
    for (int64_t v = (int64_t)blockIdx.x * W + threadIdx.x / 32; v < V; v += (int64_t)gridDim.x * W) {
        const T* r = w + v * w_sr;
        float2 s = make_float2(0.f, 0.f);
        int64_t tail = 0;
        if (vec) {
#pragma unroll 4
            for (int64_t k = lane * N; k + N <= d; k += 32 * N) {
                float2 q[N / 2];
                unpack(r, *reinterpret_cast<const uint4*>(r + k), q);
#pragma unroll
                for (int j = 0; j < N / 2; ++j) s = fma2(q[j], q[j], s);
            }
            tail = d / N * N;
        }
        for (int64_t k = tail + lane; k < d; k += 32) { const float q = Elem<T>::to_f(r[k]); s.x = fmaf(q, q, s.x); }
        float t = s.x + s.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        top = t == t ? fmaxf(top, t) : INFINITY;
    }
    if (lane == 0) atomicMax(longest, __float_as_uint(top));
    if (blockIdx.x == 0) wait_for_previous(); // so that this kernel ends after the product's
}

// ------------------------------------------------------------------ host side
struct ScorePlan {
    int few, np;                              // CTAs of the few rows' kernel or 0; statistics of a row
    int cand; bool all; int64_t groups, stride;
    int64_t off_score, off_hit, off_rec, off_second, off_longest, total;
    bool longest;
};

static ScorePlan score_plan(const HeadOps& o, const HeadPlan& q, int top) {
    const int64_t T = std::min(o.T, SC_ROWS), V = o.V;
    ScorePlan f{};
    f.few = score_few_ctas(o);
    f.np = f.few ? f.few : (int)(2 * q.nt);
    f.off_score = q.base;
    f.off_hit = f.off_score + up256(f.np * T * 16);
    f.off_rec = f.off_hit + up256(T * 4);
    f.total = f.off_rec;
    if (top > 0) {
        f.cand = (int)std::min<int64_t>(V, top + SC_EXTRA);
        f.groups = (V + 15) / 16;
        f.stride = 16 * q.nt;
        // few groups for each candidate: most would be taken whole, or there are not enough of them
        f.all = V <= 2048 || V < 32 * f.cand;
        if (f.all) f.few = 0;
        f.np = f.few ? f.few : (int)(2 * q.nt);
        f.off_second = f.off_rec + up256(f.all ? T * V * 4 : T * f.stride * 4);
        f.off_longest = f.off_second + (f.all ? 0 : up256(T * f.stride * 4));
        f.total = f.off_longest + 256;
        // the words' norms are one read of the weight beside the product, and without them every candidate's word is read (64 MB of them, which
        // come from the L2 as a rule, take less time than a launch and its read)
        f.longest = !f.few && o.T * f.cand > V && o.T * f.cand * o.d * q.es > (int64_t(64) << 20);
    }
    return f;
}

// The backward's workspace.  Few rows' statistics come from other products than the backward's (mma.sync's sums differ from the tiles' by
// their roundings, which a small temperature makes large: a certain word's dlogit was 0.87 instead of 0 at 1e-3): it
// takes them again from its own (forward and backward of 1 and 8 tokens x 50001 x 1024: 175 -> 199 us, 167 -> 187).
struct ScoreBwd { bool again; int64_t off_score, off_hit, off_stats, total; };
static ScoreBwd score_bwd_plan(const HeadOps& o, const HeadPlan& q) {
    ScoreBwd f{};
    f.again = score_few_ctas(o) > 0;
    f.off_score = up256(q.bwd_total);
    f.off_hit = f.off_score + up256(2 * q.nt * o.T * 16);
    f.off_stats = f.off_hit + up256(o.T * 4);
    f.total = f.again ? f.off_stats + up256(4 * o.T * 4) : q.bwd_total;
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
    return launch_after(score_top_kernel<T, ALL, THREADS>, (unsigned)p.T, THREADS, smem, st, p);
}

// One CTA an SM, with the shared memory's split that the product needs (a kernel that wants another one has to wait for the SM).
template <typename T>
static cudaError_t launch_longest(const HeadOps& o, const void* w, int64_t w_sr, bool vec, uint32_t* out, cudaStream_t st) {
    auto k = longest_word_kernel<T>;
    cudaError_t e;
    if ((e = allow_smem(k, cudaSharedmemCarveoutMaxShared, cudaFuncAttributePreferredSharedMemoryCarveout)) != cudaSuccess) return e;
    const unsigned grid = (unsigned)std::min<int64_t>((o.V + SC_NORM_THREADS / 32 - 1) / (SC_NORM_THREADS / 32), 148 * (2048 / SC_NORM_THREADS));
    return launch_after(k, grid, SC_NORM_THREADS, 0, st, static_cast<const T*>(w), w_sr, o.V, o.d, vec, out);
}

template <typename T>
static cudaError_t launch_top(const ScoreRows& p, bool all, cudaStream_t st) {
    // many candidates (a threshold needs many more shares than those), or few rows (more warps for each): larger CTAs
    if (p.cand <= 64 && p.T > 148) return all ? launch_top<T, true, 128>(p, st) : launch_top<T, false, 128>(p, st);
    return all ? launch_top<T, true, 256>(p, st) : launch_top<T, false, 256>(p, st);
}

}  // namespace swx

using namespace swx;

extern "C" {

int64_t swx_logprob_args_size(void) { return (int64_t)sizeof(swx_logprob_args); }

int64_t swx_logprob_fwd_workspace_bytes(const swx_logprob_args* a) {
    const int c = score_check(a);
    return c != SWX_OK ? -c : score_plan(ops_of(a), head_plan(ops_of(a)), a->top_k).total;
}

int64_t swx_logprob_bwd_workspace_bytes(const swx_logprob_args* a) {
    const int c = score_check(a);
    return c != SWX_OK ? -c : score_bwd_plan(ops_of(a), head_plan(ops_of(a))).total;
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
    const ScorePlan f = score_plan(o, q, a->top_k);
    if (a->workspace_bytes < f.total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* status = wait_status_address();      // also makes a context current on this thread, which the tensor maps need
    Operand x, w;
    head_operands(o, q, ws, x, w, st);
    const bool bf = o.dtype == SWX_DTYPE_BF16;
    // the rows' operands in their own type: bf16 ones from their copies where those were made (their rows start on 16 bytes)
    const void* sw = bf ? w.p : o.w;
    const int64_t w_sr = bf ? w.row : o.w_sr;
    const bool vec = bf || (aligned16(o.x) && aligned16(o.w) && o.x_sr % 4 == 0 && o.w_sr % 4 == 0);
    uint32_t* norm = reinterpret_cast<uint32_t*>(ws + f.off_longest);
    bool longest = f.longest;                 // the words' norms are still to be read
    for (int64_t r0 = 0; r0 < o.T; r0 += SC_ROWS) {
        HeadOps oc = o;
        oc.T = std::min(SC_ROWS, o.T - r0);
        oc.x = static_cast<const uint8_t*>(o.x) + r0 * o.x_sr * q.es;
        HeadPlan qc = q;
        qc.mt = (oc.T + XE_TILE - 1) / XE_TILE;
        const Operand xc = x.part(r0, oc.T);
        CUtensorMap mx, mw;
        if (!xc.k_major(&mx) || !w.k_major(&mw)) return SWX_ERR_CUDA;
        XentGemm g = logits_gemm(oc, qc, 0, o.V, status);
        set_score_sums(g, o);
        g.target = a->targets + r0; g.ignore = a->ignore_index;
        const double cut = mean_cut(f.few ? few_additions(o.d) : (double)logit_additions(o));
        g.inv_temp = 1.f / a->temperature; g.k2 = exponent_scale(a->temperature, cut);
        g.score = reinterpret_cast<float4*>(ws + f.off_score);
        g.hit = reinterpret_cast<float*>(ws + f.off_hit);
        g.largest = reinterpret_cast<float*>(ws + f.off_rec); g.runner_up = reinterpret_cast<float*>(ws + f.off_second);
        g.all = reinterpret_cast<float*>(ws + f.off_rec);
        if (longest && cudaMemsetAsync(norm, 0, 4, st) != cudaSuccess) return SWX_ERR_CUDA;
        g.beside = longest;
        const cudaError_t e = f.few ? launch_score_few(g, oc, xc, w, a->top_k > 0, f.few, st)
                              : a->top_k == 0 ? launch_logits<XE_SCORE>(g, mx, mw, mx, st)
                              : f.all       ? launch_logits<XE_SCORE_ALL>(g, mx, mw, mx, st)
                                            : launch_logits<XE_SCORE_TOP>(g, mx, mw, mx, st);
        if (e != cudaSuccess) return SWX_ERR_CUDA;
        if (longest && (bf ? launch_longest<__nv_bfloat16>(o, sw, w_sr, vec, norm, st) : launch_longest<float>(o, sw, w_sr, vec, norm, st)) != cudaSuccess)
            return SWX_ERR_CUDA;
        longest = false;
        ScoreRows p{};
        p.T = oc.T; p.V = o.V; p.d = o.d; p.np = f.np;
        p.score = g.score; p.hit = g.hit; p.target = g.target; p.ignore = a->ignore_index;
        p.k2 = g.k2; p.cut = (float)cut; p.exact_k2 = exponent_scale(a->temperature, 0.);
        p.row_max = a->row_max ? a->row_max + r0 : nullptr; p.row_sum = a->row_sum ? a->row_sum + r0 : nullptr;
        p.log_probs = a->log_probs + r0; p.entropy = a->entropy + r0;
        if (a->top_k == 0) {
            const unsigned grid = (unsigned)((oc.T + SC_THREADS / 32 - 1) / (SC_THREADS / 32));
            if (launch_after(score_rows_kernel, grid, SC_THREADS, 0, st, p) != cudaSuccess) return SWX_ERR_CUDA;
            continue;
        }
        p.top = a->top_k; p.cand = f.cand; p.largest = g.largest; p.runner_up = g.runner_up; p.stride = f.stride; p.all = g.all; p.groups = f.groups;
        p.top_log_probs = a->top_log_probs + r0 * a->top_k; p.top_ids = a->top_ids + r0 * a->top_k;
        p.x = bf ? xc.p : oc.x; p.x_sr = bf ? x.row : o.x_sr;
        p.w = sw; p.w_sr = w_sr; p.vec = vec;
        if (f.longest) p.longest = norm;
        if ((bf ? launch_top<__nv_bfloat16>(p, f.all, st) : launch_top<float>(p, f.all, st)) != cudaSuccess) return SWX_ERR_CUDA;
    }
    return SWX_OK;
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
    const ScoreBwd f = score_bwd_plan(o, q);
    if (a->workspace_bytes < f.total || !aligned16(a->workspace)) return SWX_ERR_INVALID_ARG;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    float* stats = reinterpret_cast<float*>(ws + f.off_stats);
    const float* row_max = f.again ? stats : a->row_max;
    const float* row_sum = f.again ? stats + o.T : a->row_sum;
    const float* entropy = f.again ? stats + 2 * o.T : a->entropy;
    const float k2 = exponent_scale(a->temperature, mean_cut((double)logit_additions(o)));
    const HeadGrads gr{a->dx, a->dweight, a->dw_dtype == SWX_DTYPE_BF16, nullptr, nullptr};
    auto fill = [=](XentGemm& g) {
        set_score_sums(g, o);                 // the same sums as the forward's
        g.target = a->targets; g.ignore = a->ignore_index;
        g.inv_temp = 1.f / a->temperature; g.k2 = k2;
        g.row_max = row_max; g.row_sum = row_sum; g.entropy = entropy;
        g.d_logp = a->d_log_probs; g.d_entropy = a->d_entropy;
    };
    auto statistics = [=](const CUtensorMap& x, const CUtensorMap& w, int* status) -> int {
        if (!f.again) return SWX_OK;
        XentGemm g = logits_gemm(o, q, 0, o.V, status);
        set_score_sums(g, o);
        g.target = a->targets; g.ignore = a->ignore_index; g.k2 = k2;
        g.score = reinterpret_cast<float4*>(ws + f.off_score);
        g.hit = reinterpret_cast<float*>(ws + f.off_hit);
        if (launch_logits<XE_SCORE>(g, x, w, x, st) != cudaSuccess) return SWX_ERR_CUDA;
        ScoreRows p{};
        p.T = o.T; p.V = o.V; p.np = (int)(2 * q.nt);
        p.score = g.score; p.hit = g.hit; p.target = g.target; p.ignore = g.ignore; p.k2 = k2;
        p.row_max = stats; p.row_sum = stats + o.T; p.entropy = stats + 2 * o.T; p.log_probs = stats + 3 * o.T;
        return launch_after(score_rows_kernel, (unsigned)((o.T + SC_THREADS / 32 - 1) / (SC_THREADS / 32)), SC_THREADS, 0, st, p) == cudaSuccess
                   ? SWX_OK : SWX_ERR_CUDA;
    };
    return head_backward(o, q, ws, gr, st, launch_logits<XE_GRAD>, fill, statistics);
}

}  // extern "C"
