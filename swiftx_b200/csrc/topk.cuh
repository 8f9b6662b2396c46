// The K largest of a long row, by one CTA.  A key is a value's order-preserving bits above the complement of its
// index, so that no two are equal and ties go to the lowest index.
//
// After a pass in which each thread has kept the largest value of its share, about the K-th largest of those maxima is a threshold
// that at least K values reach, and only the threads whose maximum does have any: their shares (some K of them, few
// hundred values) are read again, and the keys that pass, little more than K as a rule, are gathered in shared memory and ranked.
// Where too many pass (many equal values, or large ones gathered in few shares) the whole row is streamed past a rising
// threshold in bounded batches instead (TopK::push), slower and for any order.
#pragma once
#include "common.cuh"

namespace swx {

// Bits whose unsigned order is the values' (-0 as 0, a NaN above everything).
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.);
    return v != v ? ~0ull : b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint64_t index_key(uint32_t value, uint32_t index) { return (uint64_t)value << 32 | (uint32_t)~index; }
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~(uint32_t)k; }

// Entries that TopK's buffer holds for `k` and `per` keys a thread: what is kept, and a batch's passers.
constexpr int topk_capacity(int k, int per) { return k * (per + 1); }

// A threshold that at least k of the THREADS threads' values (order_key bits) reach, and few more where the values differ (a quarter
// of k, and of the threads that are not among the k: close to all of them the values say little about the whole),
// by one warp: the bits of the k-th largest are set from the top, over those that differ, until it is that close.  A value with all
// bits set asks for no threshold, and is returned.  scratch: THREADS + 1 words; all threads call it.
template <int THREADS>
__device__ __forceinline__ uint32_t about_kth(uint32_t mine, int k, uint32_t* scratch) {
    scratch[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x < 32) {
        constexpr int N = THREADS / 32;
        uint32_t v[N], lo = ~0u, hi = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = scratch[threadIdx.x + 32 * j];
            lo = min(lo, v[j]);
            hi = max(hi, v[j]);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        const int top = 32 - __clz(lo ^ hi);                   // bits from here up are common
        uint32_t t = top == 32 ? 0 : hi >> top << top;
        if (hi == ~0u) t = hi;
        for (int b = top - 1; b >= 0 && hi != ~0u; --b) {
            const uint32_t c = t | 1u << b;
            int n = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) n += v[j] >= c;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= k) t = c;
            if (n >= k && n <= k + min(k, THREADS - k) / 4) break;
        }
        if (threadIdx.x == 0) scratch[THREADS] = t;
    }
    __syncthreads();
    return scratch[THREADS];
}

// All threads of the CTA (THREADS >= k) call every member together.  A batch is PER keys for each thread, 0 for none.
template <int THREADS, int PER>
struct TopK {
    uint64_t* buf;                            // topk_capacity(k, PER)
    uint64_t* kept;                           // k
    int* count;                               // two ints of shared memory, 0 before the first barrier
    int k, n;
    uint64_t floor;                           // every key of the k largest so far is at least this

    __device__ __forceinline__ TopK(uint64_t* buf_, uint64_t* kept_, int* count_, int k_) : buf(buf_), kept(kept_), count(count_), k(k_), n(0), floor(1) {}
    __device__ __forceinline__ void clear() {
        n = 0;
        floor = 1;
        __syncthreads();
        if (threadIdx.x == 0) *count = 0;
        __syncthreads();
    }
    // One key, by any thread: dropped, but counted, where the buffer is full.
    __device__ __forceinline__ void add(float v, uint32_t index, uint32_t least) {
        const uint32_t o = order_key(v);
        if (o < least) return;
        const int at = atomicAdd(count, 1);
        if (at < topk_capacity(k, PER)) buf[at] = index_key(o, index);
    }
    // After the threads' adds: whether all of them found room.
    __device__ __forceinline__ bool added() {
        __syncthreads();
        n = *count;
        return n <= topk_capacity(k, PER);
    }
    // The keys that reach the threshold, from the shares of the threads whose maximum does: load(t, j, e) reads entry j < per of
    // thread t's share into e, and emit(e, f) calls f(value, index) on what it holds.  A warp takes a share, four of them
    // at a time so that their loads overlap.  False where they were too many, or a maximum asks for no threshold.
    template <class Entry, class Load, class Emit>
    __device__ __forceinline__ bool gather(uint32_t mine, uint32_t* scratch, int* owners, int64_t per, Load load, Emit emit) {
        const uint32_t t = about_kth<THREADS>(mine, k, scratch);
        if (t == ~0u) return false;
        if (mine >= t) owners[atomicAdd(count + 1, 1)] = threadIdx.x;
        __syncthreads();
        const int m = count[1];
        for (int i0 = threadIdx.x / 32; i0 < m; i0 += 4 * (THREADS / 32))
            for (int64_t j = threadIdx.x % 32; j < per; j += 32) {
                Entry e[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (i0 + u * (THREADS / 32) < m) load(owners[i0 + u * (THREADS / 32)], j, e[u]);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (i0 + u * (THREADS / 32) < m) emit(e[u], [&](float v, uint32_t index) { add(v, index, t); });
            }
        floor = (uint64_t)t << 32;
        return added();
    }
    // The same of shares that the threads still hold: each(f) calls f(value, index) on this thread's values.
    template <class Each>
    __device__ __forceinline__ bool gather_held(uint32_t mine, uint32_t* scratch, Each each) {
        const uint32_t t = about_kth<THREADS>(mine, k, scratch);
        if (t == ~0u) return false;
        if (mine >= t) each([&](float v, uint32_t index) { add(v, index, t); });
        floor = (uint64_t)t << 32;
        return added();
    }
    // The k-th largest of the threads' largest keys: at least k keys are no smaller.  The bits are found from the top; the keys
    // differ, so the search ends as soon as exactly k threads pass.
    __device__ __forceinline__ uint64_t kth_of_threads(uint64_t most) const {
        uint64_t t = 0;
        for (int b = 63; b >= 0; --b) {
            const uint64_t c = t | 1ull << b;
            const int m = __syncthreads_count(most >= c);
            if (m >= k) t = c;
            if (m == k) break;
        }
        return t;
    }
    __device__ __forceinline__ void push(const uint64_t (&key)[PER]) {
        uint64_t most = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) most = key[j] > most ? key[j] : most;
        const int passing = __syncthreads_count(most >= floor);
        if (passing == 0) return;
        if (n + passing * PER > topk_capacity(k, PER)) {
            const uint64_t t = kth_of_threads(most);       // at most k threads have a key this large (or fewer than k have any)
            if (t > floor) floor = t;
            if (n > k) rank();
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (key[j] >= floor) buf[atomicAdd(count, 1)] = key[j];
        __syncthreads();
        n = *count;
        __syncthreads();
    }
    // The buffer's k largest, in falling order, into `kept`: a key's rank is the number of larger ones.
    __device__ __forceinline__ void order() {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const uint64_t mine = buf[i];
            int r = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) r += buf[j] > mine;
            if (r < k) kept[r] = mine;
        }
        __syncthreads();
        n = n < k ? n : k;
    }
    // The buffer cut to them.
    __device__ __forceinline__ void rank() {
        order();
        for (int i = threadIdx.x; i < n; i += THREADS) buf[i] = kept[i];
        if (threadIdx.x == 0) *count = n;
        __syncthreads();
        if (n == k && buf[k - 1] > floor) floor = buf[k - 1];
    }
};

// Statistics of scaled logits in base 2: m the largest logit, s = sum 2^u and w = sum 2^u u with u = (z - m) k, k = log2(e) /
// temperature.  m stays unscaled: the largest term is 1 whatever the temperature, so s is at least 1 and w at most 0.
// (m = -inf with s = w = 0: nothing yet; the differences of infinities, NaN, are dropped by the maximum with SCORE_FAR.)
constexpr float SCORE_FAR = -200.f;           // 2^-200 is 0: what lies further below the maximum adds nothing
struct Score { float m, s, w; };
// The same relative to a larger m.
__device__ __forceinline__ void score_move(Score& a, float m, float k) {
    const float d = fmaxf((a.m - m) * k, SCORE_FAR), c = ex2(d);
    a.w = c * (a.w + a.s * d);
    a.s *= c;
    a.m = m;
}
__device__ __forceinline__ void score_join(Score& a, Score b, float k) {
    const float m = fmaxf(a.m, b.m);
    score_move(a, m, k);
    score_move(b, m, k);
    a.s += b.s;
    a.w += b.w;
}
__device__ __forceinline__ void score_join_warp(Score& a, float k) {
    float m = a.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    score_move(a, m, k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
    }
}
// The statistics of a whole row by `threads` threads (of which this is number t), from its np parts, before they are joined.
__device__ __forceinline__ Score score_join_parts(const float4* q, int np, float k, int t, int threads) {
    Score a{-INFINITY, 0.f, 0.f};
    for (int i0 = t; i0 < np; i0 += 4 * threads) {
        float4 v[4];
        float m = a.m;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            v[u] = i0 + u * threads < np ? q[i0 + u * threads] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
            m = fmaxf(m, v[u].x);
        }
        score_move(a, m, k);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            Score b{v[u].x, v[u].y, v[u].z};
            score_move(b, m, k);
            a.s += b.s;
            a.w += b.w;
        }
    }
    score_join_warp(a, k);
    return a;
}
// The same by a CTA, joined; parts: shared memory for one Score a warp.
template <int THREADS>
__device__ __forceinline__ Score score_join_row(const float4* q, int np, float k, Score* parts) {
    Score a = score_join_parts(q, np, k, threadIdx.x, THREADS);
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = a;
    __syncthreads();
    float m = parts[0].m;
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, parts[i].m);
    a = Score{m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        Score b = parts[i];
        score_move(b, m, k);
        a.s += b.s;
        a.w += b.w;
    }
    return a;
}

}  // namespace swx
