// Linear attention on the fifth-generation tensor cores: the forward pass and the segment
// states for bf16 inputs with dk <= 64 whose tensors TMA can describe.
//
// The products of a chunk (128 tokens here) are about 2000 cycles of tcgen05, and the work on
// values between them about 1300 issue slots of each quarter of the SM, so what matters is that the two
// and the loads overlap.  One CTA per SM, its warps in roles that run on different chunks at once:
//   loader    the tiles of q, k, v by TMA into a ring of three chunks, and the chunk's decays
//   issuer    all products
//   8 warps A k weighted by exp(G_end - G_s), as three bf16 pieces (24 bits), in the tile's own
//             (swizzled) layout; U = weighted k^T v; S = exp(G_end) S + U in fp32 registers, shared in bf16 for
//             q S alone (one factor of each term rounded, as with P; shared memory has no room for more pieces)
//   8 warps B P = masked, decayed scores (bf16), written over the scores in tensor memory, where the
//             product with v reads them; o = scale exp(G_t) q S + P v, to memory
// The weighted tile has one buffer in two halves of 64 tokens: one half is made while the other's
// products run.  The scores and U have two places each in tensor memory.
// Warp w of a role works on rows 32 (w % 4) .. and, of their columns, on half w / 4.
// What bounds it now is the chain through a chunk's roles rather than a pipe: 2.2 us a chunk, on an idle GPU and with
// 128 CTAs (4 x 8192 x 32 heads of 64: 154 us, products in 33 % of the cycles, a quarter issues in 48 %, shared memory 49 %,
// DRAM 3.5 TB/s); 4 x 65536 x 32 heads 1.15 ms, 0.66 at the copy rate; 8 x 1000 x 16 heads with dv 128, padded, 37 us.
// The loader's and the issuer's warps vote in each chunk whether to go on, which also keeps them converged: without
// the vote 200 us, 1.42 ms and 43 us.
// Separate rings for q, k and v and a second issuing warp were 20 to 30 % slower.
#include "linear_attention.cuh"
#include "launch_util.cuh"
#include "tc5.cuh"
#include "tma_util.cuh"

namespace swx {

constexpr int LT_C = 128;                     // tokens per chunk
constexpr int LT_BOX = LT_C * 128;            // bytes of 128 rows of 64 bf16 values
constexpr int LT_RING = 4;                    // gates: one being made, three in use (A is at most two chunks ahead of B)

// Decays of a chunk of 128 tokens, as LaGates.
struct __align__(16) LtGates {
    float2 G[LT_C];
    float in_block[LT_C];                     // exp(G_a - G_t), a the first token of t's block of 16
    float2 Gend;
    float all;
    int steep;                                // some block's decays span more than 2^60: in_block would overflow
};

struct LtG { float g[4]; };

__device__ __forceinline__ LtG lt_load_g(const LaDev& p, int b, int h, int t0, int len, int lane) {
    const float* g = p.g + (int64_t)b * p.g_sb + (int64_t)h * p.g_sh;
    LtG r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int t = t0 + 4 * lane + e;
        r.g[e] = t < len ? g[(int64_t)t * p.g_sl] : 0.f;
    }
    return r;
}
__device__ __forceinline__ float2 lt_split(double x) { return make_float2((float)x, (float)(x - (double)(float)x)); }

__device__ __forceinline__ double lt_gates(LtGates& s, LtG r, int lane) {
    const double L2E = 1.4426950408889634073599;
    double d[4], x = 0.;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x += (r.g[e] < -1000.f ? -1000. : (double)r.g[e]) * L2E;
        d[e] = x;
    }
    double sum = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
    }
    const double all = __shfl_sync(0xffffffffu, sum, 31), before = sum - x;
    const double ga = __shfl_sync(0xffffffffu, before + d[0], lane & ~3);        // the block's first token
    double lo = before + d[0], hi = lo;
#pragma unroll
    for (int e = 1; e < 4; ++e) {
        lo = fmin(lo, before + d[e]);
        hi = fmax(hi, before + d[e]);
    }
    const bool steep = !(ga - lo < 60. && hi - ga < 60.);
    const unsigned any = __ballot_sync(0xffffffffu, steep);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double G = before + d[e];
        s.G[4 * lane + e] = lt_split(G);
        s.in_block[4 * lane + e] = ex2((float)(ga - G));
    }
    if (lane == 0) {
        s.Gend = lt_split(all);
        s.all = ex2((float)all);
        s.steep = any != 0;
    }
    return all;
}

// A bounded wait that every thread makes.  After one that ran out a warp makes no further ones, and the status word
// says so.  The working warps run on to their end (on whatever is there: all their addresses are in bounds); the loader
// issues no more copies and the issuer no more products (lt_going), and both see what they have issued end
// before the CTA goes (lt_landed): its shared and tensor memory may be another CTA's then.
__device__ __forceinline__ void lt_wait(uint64_t* bar, uint32_t parity, bool& ok, uint32_t polls) {
    if (ok && !mbar_wait_suspended(bar, parity, polls)) ok = false;
}
__device__ __forceinline__ bool lt_going(bool& ok) { return ok = __all_sync(0xffffffffu, ok); }
__device__ __forceinline__ void lt_landed(uint64_t* bar, uint32_t parity, bool& ok) {
    if (!mbar_wait_suspended(bar, parity, LT_POLLS)) ok = false;
}

// 16-byte part j of row r of a swizzled 64-column tile.
__device__ __forceinline__ uint32_t lt_at(int r, int j) { return (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4)); }

// This thread's half row of x, times w, as three pieces (LT_BOX apart) in the tile's own layout; zero
// for a row without a token.
__device__ __forceinline__ void lt_weigh(const uint8_t* x, uint8_t* planes, int row, int half, float w, bool live) {
    const float2 w2 = bc2(w), neg = bc2(-1.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t at = lt_at(row, 4 * half + j);
        uint4 r = *reinterpret_cast<const uint4*>(x + at);
        if (!live) r = make_uint4(0, 0, 0, 0);
        const uint32_t in[4] = {r.x, r.y, r.z, r.w};
        uint32_t o[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 v = mul2(f2(bf16_lo(in[e]), bf16_hi(in[e])), w2);
            o[0][e] = pack_bf16(v.x, v.y);
            v = fma2(f2(bf16_lo(o[0][e]), bf16_hi(o[0][e])), neg, v);
            o[1][e] = pack_bf16(v.x, v.y);
            v = fma2(f2(bf16_lo(o[1][e]), bf16_hi(o[1][e])), neg, v);
            o[2][e] = pack_bf16(v.x, v.y);
        }
#pragma unroll
        for (int q = 0; q < 3; ++q)
            *reinterpret_cast<uint4*>(planes + q * LT_BOX + at) = make_uint4(o[q][0], o[q][1], o[q][2], o[q][3]);
    }
}

// U (64 x 64) = sum over the planes of plane^T y, over the contraction steps of 16 tokens K0 .. K1 - 1.
template <int K0, int K1>
__device__ __forceinline__ void lt_issue_u(uint32_t d, const uint8_t* planes, const uint8_t* y) {
    constexpr uint32_t id = mma_bf16_idesc(64, 64, true, true);
    const uint64_t yd = operand_desc(y, LT_BOX), a = operand_desc(planes, LT_BOX);
#pragma unroll
    for (int q = 2; q >= 0; --q)
#pragma unroll
        for (int k = K0; k < K1; ++k)
            mma_bf16_cta(d, a + q * (LT_BOX >> 4) + k * (2048 >> 4), yd + k * (2048 >> 4), id, q < 2 || k > 0);
}

// State values of a thread: row lt_state_row(), columns 32 half .. 32 half + 31.  A 64-row product fills
// the first 16 lanes of each warp's 32.
__device__ __forceinline__ int lt_state_row(int warp, int lane) { return lane < 16 ? 16 * (warp & 3) + lane : -1; }

__device__ __forceinline__ void lt_state_read(float (&S)[32], const float* src, const LaDev& p, int row, int c0, int half) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const int c = 32 * half + j;
        S[j] = src && row >= 0 && row < p.dk && c0 + c < p.dv ? src[(int64_t)row * p.dv + c0 + c] : 0.f;
    }
}
__device__ __forceinline__ void lt_state_write(const float (&S)[32], float* dst, const LaDev& p, int row, int c0, int half) {
    if (row < 0 || row >= p.dk) return;
    float* d = dst + (int64_t)row * p.dv + c0 + 32 * half;
    const int n = p.dv - c0 - 32 * half;
    if (p.dv % 4 == 0 && n >= 32) {                              // states are 16-byte aligned
#pragma unroll
        for (int j = 0; j < 8; ++j) reinterpret_cast<float4*>(d)[j] = make_float4(S[4 * j], S[4 * j + 1], S[4 * j + 2], S[4 * j + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) if (j < n) d[j] = S[j];
    }
}
__device__ __forceinline__ void lt_state_save(const float (&S)[32], const LaDev& p, int64_t bh, int c, int row, int c0, int half) {
    if (p.save && c % p.save_c == 0) lt_state_write(S, p.save + (bh * p.save_n + c / p.save_c) * p.dk * p.dv, p, row, c0, half);
}
__device__ __forceinline__ void lt_pack32(uint32_t (&w)[16], const float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
}
__device__ __forceinline__ void lt_state_share(const float (&S)[32], uint8_t* s, int row, int half) {
    if (row < 0) return;
    uint32_t w[16];
    lt_pack32(w, S);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(s + lt_at(row, 4 * half + j)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}
// S = all S + (this thread's 32 values of U)
__device__ __forceinline__ void lt_state_add(float (&S)[32], uint32_t u_at, float all) {
    float u[32];
    tmem_ld32(u_at, u);
    tmem_ld_wait();
    const float2 a = bc2(all);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const float2 y = fma2(a, f2(S[j], S[j + 1]), f2(u[j], u[j + 1]));
        S[j] = y.x;
        S[j + 1] = y.y;
    }
}
// Scores of row t with the tokens s0 .. s0 + 31, times scale exp(G_t - G_s), 0 for s > t.  The
// exponential is split at the first token a of s's block of 16, exp(G_t - G_a) exp(G_a - G_s): one
// exponential a block, two packed products for two values.  A chunk with a block so steep that the second
// factor could overflow takes an exponential for each value.
__device__ __forceinline__ void lt_mask(float (&x)[32], const LtGates& gt, int s0, int row, float2 G, float scale) {
    if (!gt.steep) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 f = bc2(scale * la_decay(G, gt.G[s0 + 16 * e]));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 m = reinterpret_cast<const float4*>(gt.in_block + s0 + 16 * e)[j];
                float* y = x + 16 * e + 4 * j;
                const float2 a = mul2(f2(y[0], y[1]), mul2(f, f2(m.x, m.y))), c = mul2(f2(y[2], y[3]), mul2(f, f2(m.z, m.w)));
                y[0] = a.x; y[1] = a.y; y[2] = c.x; y[3] = c.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] *= s0 + j <= row ? scale * la_decay(G, gt.G[s0 + j]) : 0.f;
    }
    if (row < s0 + 31) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = s0 + j <= row ? x[j] : 0.f;
    }
}
// Rows of v without a token: zero (what TMA brought may be anything, and 0 times it need not be 0).
__device__ __forceinline__ void lt_clear_rows(uint8_t* v, int row, int half, int rows) {
    if (row < rows) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(v + lt_at(row, 4 * half + j)) = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ void lt_arrive(uint64_t* bar, int lane) {      // one arrival for the warp
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(bar)) : "memory");
}

constexpr int LT_A = 8, LT_B = 8;                                 // working warps of the two roles

// ------------------------------------------------------------------ one segment's state
// The A role alone, the weighted tile in two whole buffers.
constexpr int LS_WARPS = LT_A + 2, LS_RING = 3;
constexpr int LS_SMEM = 1024 + LS_RING * 2 * LT_BOX + 2 * 3 * LT_BOX;

template <bool REV>
__global__ void __launch_bounds__(32 * LS_WARPS, 1)
lt_state_kernel(const LaDev p, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y, int* status) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ LtGates gates[LT_RING];
    __shared__ __align__(8) uint64_t full[LS_RING], ready[2], done[LS_RING], idle;      // idle: all products have ended
    __shared__ uint32_t tmem_base;
    uint8_t* tiles = smem_raw + (((smem_u32(smem_raw) + 1023) & ~1023u) - smem_u32(smem_raw));
    uint8_t* planes = tiles + LS_RING * 2 * LT_BOX;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int nrun = p.nseg - 1;                                 // the last (REV: first) segment's state is not needed
    const int seg = (int)(blockIdx.x % nrun) + (REV ? 1 : 0);
    const int64_t vh = blockIdx.x / nrun;
    const int sl = (int)(vh % p.nsl), h = (int)(vh / p.nsl % p.H), b = (int)(vh / p.nsl / p.H);
    const int hk = h / (p.H / p.Hk), c0 = sl * LA_DV, len = la_len(p, b);
    const int first = seg * p.segc / 2, last = min(first + p.segc / 2, (len + LT_C - 1) / LT_C), n = max(0, last - first);
    auto chunk = [&](int i) { return REV ? last - 1 - i : first + i; };
    if (threadIdx.x == 0) {
        for (int i = 0; i < LS_RING; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&done[i], 1);
        }
        for (int i = 0; i < 2; ++i) mbar_init(&ready[i], LT_A);
        mbar_init(&idle, 1);
        mbar_fence_init();
    }
    __syncwarp();
    if (warp == 0) tmem_alloc(&tmem_base, 128);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    bool ok = true;
    if (warp == LT_A) {                                          // loader
        double total = 0.;
        LtG g = lt_load_g(p, b, h, chunk(0) * LT_C, n > 0 ? len : 0, lane);
        int i = 0;
#pragma unroll 1
        for (; i < n; ++i) {
            const int u = i % LS_RING;
            const LtG now = g;
            if (i + 1 < n) g = lt_load_g(p, b, h, chunk(i + 1) * LT_C, len, lane);
            if (i >= LS_RING) lt_wait(&done[u], (i / LS_RING - 1) & 1, ok, p.polls);
            if (!lt_going(ok)) break;
            if (lane == 0) {
                mbar_expect_tx(&full[u], 2 * LT_BOX);
                tma_load_4d(tiles + 2 * u * LT_BOX, &map_x, 0, chunk(i) * LT_C, hk, b, &full[u]);
                tma_load_4d(tiles + (2 * u + 1) * LT_BOX, &map_y, c0, chunk(i) * LT_C, h, b, &full[u]);
            }
            __syncwarp();
            total += lt_gates(gates[i % LT_RING], now, lane);
            lt_arrive(&full[u], lane);                           // the gates are there
        }
        for (int j = max(0, i - LS_RING); j < i; ++j) lt_landed(&full[j % LS_RING], (j / LS_RING) & 1, ok);
        if (lane == 0 && sl == 0) p.dec[((int64_t)b * p.H + h) * p.nseg + seg] = ex2((float)total);
    } else if (warp == LT_A + 1) {                               // issuer
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            lt_wait(&ready[i & 1], (i >> 1) & 1, ok, p.polls);
            if (!lt_going(ok)) break;
            tc_fence_after();
            lt_issue_u<0, LT_C / 16>(tmem + 64 * (i & 1), planes + (i & 1) * 3 * LT_BOX, tiles + (2 * (i % LS_RING) + 1) * LT_BOX);
            mma_commit(&done[i % LS_RING]);
        }
        mma_commit(&idle);
        lt_landed(&idle, 0, ok);
    } else {
        const int half = warp / 4, row = 32 * (warp & 3) + lane;
        const uint32_t at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 32 * half;
        float S[32] = {}, all = 0.f;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int u = i % LS_RING, rows = min(LT_C, len - chunk(i) * LT_C);
            const LtGates& gt = gates[i % LT_RING];
            lt_wait(&full[u], (i / LS_RING) & 1, ok, p.polls);
            // U of two chunks ago (its weighted tile's buffer) was waited for in the last step
            const float2 G = gt.G[row];
            lt_weigh(tiles + 2 * u * LT_BOX, planes + (i & 1) * 3 * LT_BOX, row, half, REV ? p.scale * ex2(G.x) : la_decay(gt.Gend, G), row < rows);
            lt_clear_rows(tiles + (2 * u + 1) * LT_BOX, row, half, rows);
            fence_proxy_async_smem();
            tc_fence_before();
            lt_arrive(&ready[i & 1], lane);
            if (i > 0) {
                lt_wait(&done[(i - 1) % LS_RING], ((i - 1) / LS_RING) & 1, ok, p.polls);
                tc_fence_after();
                lt_state_add(S, at + 64 * ((i - 1) & 1), all);
            }
            all = gt.all;
        }
        if (n > 0) {
            lt_wait(&done[(n - 1) % LS_RING], ((n - 1) / LS_RING) & 1, ok, p.polls);
            tc_fence_after();
            lt_state_add(S, at + 64 * ((n - 1) & 1), all);
        }
        float* dst = (REV ? p.rseg : p.seg) + (((int64_t)b * p.H + h) * p.nseg + seg) * p.dk * p.dv;
        lt_state_write(S, dst, p, lt_state_row(warp, lane), c0, half);
    }
    if (!ok && status) *status = SWX_ERR_TIMEOUT;
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_free(tmem, 128);
}

// ------------------------------------------------------------------ forward
constexpr int LF_WARPS = LT_A + LT_B + 2, LF_RING = 3, LF_TILES = 3 * LT_BOX;      // q, k, v of a chunk
constexpr int LF_SMEM = 1024 + LF_RING * LF_TILES + 3 * LT_BOX + 2 * 64 * 128;     // | weighted k | S, twice

__global__ void __launch_bounds__(32 * LF_WARPS, 1)
lt_fwd_kernel(const LaDev p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, int* status) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ LtGates gates[LT_RING];
    // full: a chunk's tiles have landed.  weighed[half], products[half][parity of the chunk]: of the weighted
    // tile.  shared[parity]: S is there.  scored[parity]: the scores.  masked[parity]: P is there.
    // mixed[place of the ring]: q S and P v, and with them every product of the chunk.  read: both, by B.  idle: all products have ended.
    //   A barrier has as many places as a fast warp can be phases ahead of the slowest that waits or arrives.
    __shared__ __align__(8) uint64_t full[LF_RING], weighed[2], products[2][2], shared[2], scored[2], masked[2], mixed[LF_RING], read, idle;
    __shared__ uint32_t tmem_base;
    uint8_t* tiles = smem_raw + (((smem_u32(smem_raw) + 1023) & ~1023u) - smem_u32(smem_raw));
    uint8_t* planes = tiles + LF_RING * LF_TILES;
    uint8_t* ss = planes + 3 * LT_BOX;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, half = (warp / 4) & 1, quarter = warp & 3, row = 32 * quarter + lane;
    const int seg = (int)(blockIdx.x % p.nseg);
    const int64_t vh = blockIdx.x / p.nseg;
    const int sl = (int)(vh % p.nsl), h = (int)(vh / p.nsl % p.H), b = (int)(vh / p.nsl / p.H);
    const int hk = h / (p.H / p.Hk), c0 = sl * LA_DV, cols = min(LA_DV, p.dv - c0), len = la_len(p, b);
    const int first = seg * p.segc / 2, end = min((seg + 1) * p.segc / 2, (p.L + LT_C - 1) / LT_C);
    const int live = max(first, min(end, (len + LT_C - 1) / LT_C)), n = live - first;
    const int64_t bh = (int64_t)b * p.H + h, ssz = (int64_t)p.dk * p.dv, o_sl = (int64_t)p.H * p.dv;
    auto chunk = [&](int i) { return first + i; };
    auto tile = [&](int i, int which) { return tiles + (i % LF_RING) * LF_TILES + which * LT_BOX; };
    if (threadIdx.x == 0) {
        for (int i = 0; i < LF_RING; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&mixed[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&weighed[i], LT_A / 2);
            mbar_init(&products[i][0], 1);
            mbar_init(&products[i][1], 1);
            mbar_init(&scored[i], 1);
            mbar_init(&shared[i], LT_A);
            mbar_init(&masked[i], LT_B);
        }
        mbar_init(&read, LT_B);
        mbar_init(&idle, 1);
        mbar_fence_init();
    }
    __syncwarp();
    if (warp == 0) tmem_alloc(&tmem_base, 512);
    const int token_half = quarter / 2;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // tensor memory: scores (P over them, later) and U for chunks of either parity, q S, P v
    const uint32_t t_sc = tmem_base, t_u = t_sc + 256, t_qs = t_sc + 384, t_pv = t_sc + 448, lanes = (uint32_t)(32 * quarter) << 16;
    bool ok = true;
    if (warp == LT_A + LT_B) {                                   // loader
        LtG g = lt_load_g(p, b, h, first * LT_C, n > 0 ? len : 0, lane);
        int i = 0;
#pragma unroll 1
        for (; i < n; ++i) {
            const int u = i % LF_RING, t0 = chunk(i) * LT_C;
            const LtG now = g;
            if (i + 1 < n) g = lt_load_g(p, b, h, t0 + LT_C, len, lane);
            if (i >= LF_RING) lt_wait(&mixed[u], (i / LF_RING - 1) & 1, ok, p.polls);
            if (!lt_going(ok)) break;
            if (lane == 0) {
                mbar_expect_tx(&full[u], LF_TILES);
                tma_load_4d(tile(i, 1), &map_k, 0, t0, hk, b, &full[u]);
                tma_load_4d(tile(i, 2), &map_v, c0, t0, h, b, &full[u]);
                tma_load_4d(tile(i, 0), &map_q, 0, t0, hk, b, &full[u]);
            }
            __syncwarp();
            lt_gates(gates[i % LT_RING], now, lane);
            lt_arrive(&full[u], lane);                           // the gates are there
        }
        for (int j = max(0, i - LF_RING); j < i; ++j) lt_landed(&full[j % LF_RING], (j / LF_RING) & 1, ok);
    } else if (warp == LT_A + LT_B + 1) {                        // issuer
        constexpr uint32_t id_s = mma_bf16_idesc(LT_C, LT_C, false, false), id_o = mma_bf16_idesc(LT_C, 64, false, true);
        auto mix = [&](int i) {                                  // q S and P v
            lt_wait(&masked[i & 1], (i >> 1) & 1, ok, p.polls);
            lt_wait(&shared[i & 1], (i >> 1) & 1, ok, p.polls);
            if (i > 0) lt_wait(&read, (i - 1) & 1, ok, p.polls);
            if (!lt_going(ok)) return;
            tc_fence_after();
            const uint64_t qd = operand_desc(tile(i, 0), 16), sd = operand_desc(ss + (i & 1) * 64 * 128, 16), vd = operand_desc(tile(i, 2), 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_bf16_cta(t_qs, qd + k * 2, sd + k * (2048 >> 4), id_o, k > 0);
#pragma unroll
            for (int k = 0; k < LT_C / 16; ++k)
                mma_bf16_cta_ta(t_pv, t_sc + 128 * (i & 1) + 32 * (k / 2) + 8 * (k % 2), vd + k * (2048 >> 4), id_o, k > 0);
            mma_commit(&mixed[i % LF_RING]);
        };
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const uint32_t u = t_u + 64 * (i & 1);
            lt_wait(&full[i % LF_RING], (i / LF_RING) & 1, ok, p.polls);
            if (i >= 2) lt_wait(&mixed[(i - 2) % LF_RING], ((i - 2) / LF_RING) & 1, ok, p.polls);      // P of two chunks ago has been read
            if (!lt_going(ok)) break;
            tc_fence_after();
            const uint64_t qd = operand_desc(tile(i, 0), 16), kd = operand_desc(tile(i, 1), 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_bf16_cta(t_sc + 128 * (i & 1), qd + k * 2, kd + k * 2, id_s, k > 0);
            mma_commit(&scored[i & 1]);
            if (i > 0) mix(i - 1);        // (and every warp of A has read U of two chunks ago)
            lt_wait(&weighed[0], i & 1, ok, p.polls);
            if (!lt_going(ok)) break;
            tc_fence_after();
            lt_issue_u<0, 4>(u, planes, tile(i, 2));
            mma_commit(&products[0][i & 1]);
            lt_wait(&weighed[1], i & 1, ok, p.polls);
            if (!lt_going(ok)) break;
            tc_fence_after();
            lt_issue_u<4, 8>(u, planes, tile(i, 2));
            mma_commit(&products[1][i & 1]);
        }
        if (n > 0) mix(n - 1);
        mma_commit(&idle);
        lt_landed(&idle, 0, ok);
    } else if (warp < LT_A) {                                    // A
        const int srow = lt_state_row(warp, lane);
        const uint32_t at = t_u + lanes + 32 * half;
        float S[32], all = 0.f;
        lt_state_read(S, p.nseg > 1 ? p.seg + (bh * p.nseg + seg) * ssz : (p.s0 ? p.s0 + bh * ssz : nullptr), p, srow, c0, half);
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int rows = min(LT_C, len - chunk(i) * LT_C);
            lt_wait(&full[i % LF_RING], (i / LF_RING) & 1, ok, p.polls);
            // the last chunk's products with this half of the weighted tile
            if (i > 0) lt_wait(&products[token_half][(i - 1) & 1], ((i - 1) >> 1) & 1, ok, p.polls);
            const LtGates& gt = gates[i % LT_RING];
            lt_weigh(tile(i, 1), planes, row, half, la_decay(gt.Gend, gt.G[row]), row < rows);
            lt_clear_rows(tile(i, 2), row, half, rows);
            fence_proxy_async_smem();
            lt_arrive(&weighed[token_half], lane);
            if (i > 0) {
                lt_wait(&products[token_half ^ 1][(i - 1) & 1], ((i - 1) >> 1) & 1, ok, p.polls);
                tc_fence_after();
                lt_state_add(S, at + 64 * ((i - 1) & 1), all);
            }
            all = gt.all;
            lt_state_save(S, p, bh, 2 * chunk(i), srow, c0, half);
            if (i >= 2) lt_wait(&mixed[(i - 2) % LF_RING], ((i - 2) / LF_RING) & 1, ok, p.polls);      // q S of two chunks ago has read this place
            lt_state_share(S, ss + (i & 1) * 64 * 128, srow, half);
            fence_proxy_async_smem();
            tc_fence_before();
            lt_arrive(&shared[i & 1], lane);
        }
        const bool last = p.s_last && seg == p.nseg - 1;
        if (last || (p.save && live < end)) {
            if (n > 0) {
                for (int x = 0; x < 2; ++x) lt_wait(&products[x][(n - 1) & 1], ((n - 1) >> 1) & 1, ok, p.polls);
                tc_fence_after();
                lt_state_add(S, at + 64 * ((n - 1) & 1), all);
            }
            for (int c = live; c < end; ++c) lt_state_save(S, p, bh, 2 * c, srow, c0, half);
            if (last) lt_state_write(S, p.s_last + bh * ssz, p, srow, c0, half);
        }
    } else {                                                     // B
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
        auto finish = [&](int i, float Gx) {
            const int t0 = chunk(i) * LT_C;
            lt_wait(&mixed[i % LF_RING], (i / LF_RING) & 1, ok, p.polls);
            tc_fence_after();
            float o[32], pv[32];
            tmem_ld32(t_qs + lanes + 32 * half, o);
            tmem_ld32(t_pv + lanes + 32 * half, pv);
            tmem_ld_wait();
            tc_fence_before();
            lt_arrive(&read, lane);
            if (t0 + row >= p.L) return;
            const float2 e = bc2(ex2(Gx) * p.scale);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float2 y = fma2(e, f2(o[j], o[j + 1]), f2(pv[j], pv[j + 1]));
                o[j] = y.x;
                o[j + 1] = y.y;
            }
            if (t0 + row >= len) {
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = 0.f;
            }
            __nv_bfloat16* d = out + ((int64_t)b * p.L + t0 + row) * o_sl + (int64_t)h * p.dv + c0 + 32 * half;
            if (p.vec_o) {
                uint32_t w[16];
                lt_pack32(w, o);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (32 * half + 8 * j < cols) reinterpret_cast<uint4*>(d)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) if (32 * half + j < cols) d[j] = __float2bfloat16_rn(o[j]);
            }
        };
        float before = 0.f;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int rows = min(LT_C, len - chunk(i) * LT_C);
            lt_wait(&scored[i & 1], (i >> 1) & 1, ok, p.polls);
            tc_fence_after();
            const LtGates& gt = gates[i % LT_RING];
            const float2 G = gt.G[row];
            // P: this thread's row, columns 32 c .. of every second c
#pragma unroll 1
            for (int c = half; c < 4; c += 2) {
                uint32_t w[16] = {};
                if (c <= quarter) {
                    float x[32];
                    tmem_ld32(t_sc + 128 * (i & 1) + lanes + 32 * c, x);
                    tmem_ld_wait();
                    lt_mask(x, gt, 32 * c, row, G, p.scale);
                    if (row < rows) lt_pack32(w, x);
                }
                tmem_st16(t_sc + 128 * (i & 1) + lanes + 32 * c, w);     // over the scores that it came from
            }
            tmem_st_wait();
            tc_fence_before();
            lt_arrive(&masked[i & 1], lane);
            if (i > 0) finish(i - 1, before);
            before = G.x;
        }
        if (n > 0) finish(n - 1, before);
        // rows behind the row's last token
        la_zero_rows<__nv_bfloat16>(p, b, h, c0, cols, live * LT_C, min(end * LT_C, p.L), threadIdx.x - 32 * LT_A, 32 * LT_B);
    }
    if (!ok && status) *status = SWX_ERR_TIMEOUT;
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_free(t_sc, 512);
}

// ------------------------------------------------------------------ host side
// (b, L, heads, d) bf16 with unit element stride as a 4-D map of 64 x 128 boxes, 128-byte swizzled.
static bool lt_encode(CUtensorMap* m, const LaTensor& x, int64_t d, int64_t L, int64_t heads, int64_t b) {
    const EncodeTiledFn f = encode_tiled();
    if (!f || !x.vec) return false;
    const int64_t dense = (d * 2 + 15) / 16 * 16;
    const int64_t s[3] = {L > 1 ? x.sl * 2 : dense, heads > 1 ? x.sh * 2 : dense, b > 1 ? x.sb * 2 : dense};
    for (int64_t v : s)
        if (v <= 0 || v % 16 || v >= (int64_t(1) << 40)) return false;
    cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)L, (cuuint64_t)heads, (cuuint64_t)b};
    cuuint64_t strides[3] = {(cuuint64_t)s[0], (cuuint64_t)s[1], (cuuint64_t)s[2]};
    cuuint32_t box[4] = {64, LT_C, 1, 1}, unit[4] = {1, 1, 1, 1};
    return f(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x.p), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// *taken: whether the kernel takes these tensors; nothing is launched otherwise.
cudaError_t lt_launch_fwd(const LaDev& p, bool* taken, cudaStream_t st) {
    int* status = wait_status_address();          // also makes a context current, which the tensor maps need
    CUtensorMap q, k, v;
    *taken = p.tc && lt_encode(&q, p.q, p.dk, p.L, p.Hk, p.b) && lt_encode(&k, p.k, p.dk, p.L, p.Hk, p.b) &&
             lt_encode(&v, p.v, p.dv, p.L, p.H, p.b);
    if (!*taken) return cudaSuccess;
    cudaError_t e = allow_smem(lt_fwd_kernel, LF_SMEM);
    if (e != cudaSuccess) return e;
    lt_fwd_kernel<<<(unsigned)((int64_t)p.b * p.H * p.nsl * p.nseg), 32 * LF_WARPS, LF_SMEM, st>>>(p, q, k, v, status);
    return cudaGetLastError();
}

cudaError_t lt_launch_state(const LaDev& p, bool reverse, bool* taken, cudaStream_t st) {
    int* status = wait_status_address();
    CUtensorMap x, y;
    *taken = p.tc && lt_encode(&x, reverse ? p.q : p.k, p.dk, p.L, p.Hk, p.b) &&
             lt_encode(&y, reverse ? p.dout : p.v, p.dv, p.L, p.H, p.b);
    if (!*taken) return cudaSuccess;
    auto k = reverse ? lt_state_kernel<true> : lt_state_kernel<false>;
    cudaError_t e = allow_smem(k, LS_SMEM);
    if (e != cudaSuccess) return e;
    k<<<(unsigned)((int64_t)p.b * p.H * p.nsl * (p.nseg - 1)), 32 * LS_WARPS, LS_SMEM, st>>>(p, x, y, status);
    return cudaGetLastError();
}

}  // namespace swx
