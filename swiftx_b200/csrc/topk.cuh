// The K largest of a long row, by one CTA.  A key is a value's order-preserving bits above the complement of its
// index, so that no two are equal and ties go to the lowest index.
//
// After a pass in which each thread has kept the largest value of its share, the K-th largest of those maxima is a threshold
// that at least K values reach, and only the threads whose maximum does have any: their shares (K of them, few
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

// Finds the k-th largest of the THREADS threads' values, as order_key bits, by one warp: the bits are set from the top while at
// least k values stay no smaller, over those that differ.  scratch: THREADS + 1 words; all threads call it.
template <int THREADS>
__device__ __forceinline__ uint32_t kth_largest(uint32_t mine, int k, uint32_t* scratch) {
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
        for (int b = top - 1; b >= 0; --b) {
            const uint32_t c = t | 1u << b;
            int n = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) n += v[j] >= c;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= k) t = c;
            if (n == k) break;
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
    int* count;                               // one int of shared memory
    int k, n;
    uint64_t floor;                           // every key of the k largest so far is at least this

    __device__ __forceinline__ void start(uint64_t* buf_, uint64_t* kept_, int* count_, int k_) {
        buf = buf_; kept = kept_; count = count_; k = k_;
        clear();
    }
    __device__ __forceinline__ void clear() {
        n = 0;
        floor = 1;
        __syncthreads();
        if (threadIdx.x == 0) *count = 0;
        __syncthreads();
    }
    // One key, by any thread: dropped, but counted, where the buffer is full.
    __device__ __forceinline__ void add(uint64_t key) {
        const int at = atomicAdd(count, 1);
        if (at < topk_capacity(k, PER)) buf[at] = key;
    }
    // After the threads' adds: whether all of them found room.
    __device__ __forceinline__ bool added() {
        __syncthreads();
        n = *count;
        return n <= topk_capacity(k, PER);
    }
    // The keys that reach the threshold, from the shares of the threads whose maximum does: item(t, j, f) calls f(value,
    // index) on entry j < per of thread t's share.  False where they were too many.
    template <class Item>
    __device__ __forceinline__ bool gather(uint32_t mine, uint32_t* scratch, int* owners, int64_t per, Item item) {
        const uint32_t t = kth_largest<THREADS>(mine, k, scratch);
        if (mine >= t) owners[atomicAdd(count, 1)] = threadIdx.x;
        __syncthreads();
        const int m = *count;
        __syncthreads();
        if (threadIdx.x == 0) *count = 0;
        __syncthreads();
        const uint32_t one = (uint32_t)per;
        for (uint32_t i = threadIdx.x; i < m * one; i += THREADS)
            item(owners[i / one], (int64_t)(i % one), [&](float v, uint32_t index) {
                const uint32_t o = order_key(v);
                if (o >= t) add(index_key(o, index));
            });
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
    // The buffer cut to its k largest, in falling order (at the start of it and in `kept`).  A key's rank is the
    // number of larger ones.
    __device__ __forceinline__ void rank() {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const uint64_t mine = buf[i];
            int r = 0;
            for (int j = 0; j < n; ++j) r += buf[j] > mine;
            if (r < k) kept[r] = mine;
        }
        __syncthreads();
        n = n < k ? n : k;
        for (int i = threadIdx.x; i < n; i += THREADS) buf[i] = kept[i];
        if (threadIdx.x == 0) *count = n;
        __syncthreads();
        if (n == k && buf[k - 1] > floor) floor = buf[k - 1];
    }
};

// Statistics of scaled logits in base 2: maximum m of the raw logits, s = sum 2^u and w = sum 2^u u with u = (z - m) k2.
// (m = -inf with s = w = 0: nothing yet; the differences of infinities, NaN, are dropped by the maximum with `far`.)
struct Score { float m, s, w; };
__device__ __forceinline__ void score_join(Score& a, const Score& b, float k2, float far) {
    const float nm = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - nm) * k2, far), db = fmaxf((b.m - nm) * k2, far);
    const float ca = ex2(da), cb = ex2(db);
    a.w = ca * (a.w + a.s * da) + cb * (b.w + b.s * db);
    a.s = ca * a.s + cb * b.s;
    a.m = nm;
}
__device__ __forceinline__ void score_join_warp(Score& a, float k2, float far) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Score b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.w, o)};
        score_join(a, b, k2, far);
    }
}

}  // namespace swx
