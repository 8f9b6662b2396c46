// Warp-level matrix products on tiles in shared memory, for kernels whose operands are
// formed in registers between products: 16 x 8 accumulator tiles, 16 contraction steps at
// a time, fp32 sums.  bf16 operands use m16n8k16; fp32 operands two m16n8k8 tf32 products over
// the same 16 steps, each operand split into two tf32 pieces (22 bits; three products, the
// smallest first).  Both types keep the same elements in the same lanes: lane (g = lane / 4,
// t = lane % 4) holds
//   A: rows g, g + 8; steps 2t, 2t + 1, 2t + 8, 2t + 9   (order: row g, row g + 8, then + 8 steps)
//   B: column g;      steps 2t, 2t + 1, 2t + 8, 2t + 9
//   C: rows g, g + 8; columns 2t, 2t + 1
// so an accumulator pair is an A operand as it stands (the tf32 product's own order of steps
// is a permutation, which a sum over the steps does not see).
#pragma once
#include "common.cuh"

namespace swx {

template <typename T> struct FragA;
template <typename T> struct FragB;
template <> struct FragA<__nv_bfloat16> { uint32_t r[4]; };
template <> struct FragB<__nv_bfloat16> { uint32_t r[2]; };
template <> struct FragA<float> { float v[8]; };
template <> struct FragB<float> { float v[4]; };

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ float bf16_lo(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }

// ---------------------------------------------------------------- products
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void mma(float (&c)[4], const FragA<__nv_bfloat16>& a, const FragB<__nv_bfloat16>& b) {
    mma_bf16(c, a.r, b.r);
}
// The small products are summed by themselves and added in fp32: the tensor core cuts the low bits of
// each addition off, and with six additions a step to the large sum, linear attention's decay gradient was 1.3e-6
// off where it is 8.7e-7 now (2 x 777 x 6 heads; 110 -> 117 us).
__device__ __forceinline__ void mma(float (&c)[4], const FragA<float>& a, const FragB<float>& b) {
    float small[4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float av[4] = {a.v[4 * h], a.v[4 * h + 2], a.v[4 * h + 1], a.v[4 * h + 3]};
        uint32_t ah[4], al[4], bh[2], bl[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ah[i] = to_tf32(av[i]);
            al[i] = to_tf32(av[i] - __uint_as_float(ah[i]));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bh[i] = to_tf32(b.v[2 * h + i]);
            bl[i] = to_tf32(b.v[2 * h + i] - __uint_as_float(bh[i]));
        }
        mma_tf32(small, al, bh);
        mma_tf32(small, ah, bl);
        mma_tf32(c, ah, bh);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] += small[i];
}

// ---------------------------------------------------------------- operands from shared memory
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldm4_t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
// A[m][k] at s[m * ld + k] / at s[k * ld + m]; (m0, k0): the tile's first row and step.
__device__ __forceinline__ void load_a(FragA<__nv_bfloat16>& f, const __nv_bfloat16* s, int ld, int m0, int k0, int lane) {
    ldm4(f.r, s + (m0 + (lane & 15)) * ld + k0 + (lane >> 4) * 8);
}
__device__ __forceinline__ void load_a_t(FragA<__nv_bfloat16>& f, const __nv_bfloat16* s, int ld, int m0, int k0, int lane) {
    ldm4_t(f.r, s + (k0 + (lane & 7) + (lane >> 4) * 8) * ld + m0 + ((lane >> 3) & 1) * 8);
}
// B[k][n] at s[n * ld + k] / at s[k * ld + n], two column tiles n0, n0 + 8.
__device__ __forceinline__ void load_b2(FragB<__nv_bfloat16> (&f)[2], const __nv_bfloat16* s, int ld, int n0, int k0, int lane) {
    uint32_t r[4];
    ldm4(r, s + (n0 + (lane & 7) + (lane >> 4) * 8) * ld + k0 + ((lane >> 3) & 1) * 8);
    f[0].r[0] = r[0]; f[0].r[1] = r[1]; f[1].r[0] = r[2]; f[1].r[1] = r[3];
}
__device__ __forceinline__ void load_b2_t(FragB<__nv_bfloat16> (&f)[2], const __nv_bfloat16* s, int ld, int n0, int k0, int lane) {
    uint32_t r[4];
    ldm4_t(r, s + (k0 + (lane & 15)) * ld + n0 + (lane >> 4) * 8);
    f[0].r[0] = r[0]; f[0].r[1] = r[1]; f[1].r[0] = r[2]; f[1].r[1] = r[3];
}
__device__ __forceinline__ void load_a(FragA<float>& f, const float* s, int ld, int m0, int k0, int lane) {
    const float* p = s + (m0 + (lane >> 2)) * ld + k0 + 2 * (lane & 3);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float2 q = *reinterpret_cast<const float2*>(p + r * 8 * ld + h * 8);
            f.v[4 * h + 2 * r] = q.x;
            f.v[4 * h + 2 * r + 1] = q.y;
        }
}
__device__ __forceinline__ void load_a_t(FragA<float>& f, const float* s, int ld, int m0, int k0, int lane) {
    const float* p = s + (k0 + 2 * (lane & 3)) * ld + m0 + (lane >> 2);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) f.v[4 * h + 2 * r + i] = p[(8 * h + i) * ld + 8 * r];
}
__device__ __forceinline__ void load_b2(FragB<float> (&f)[2], const float* s, int ld, int n0, int k0, int lane) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 q = *reinterpret_cast<const float2*>(s + (n0 + 8 * n + (lane >> 2)) * ld + k0 + 8 * h + 2 * (lane & 3));
            f[n].v[2 * h] = q.x;
            f[n].v[2 * h + 1] = q.y;
        }
}
__device__ __forceinline__ void load_b2_t(FragB<float> (&f)[2], const float* s, int ld, int n0, int k0, int lane) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                f[n].v[2 * h + i] = s[(k0 + 8 * h + 2 * (lane & 3) + i) * ld + n0 + 8 * n + (lane >> 2)];
}

// ---------------------------------------------------------------- operands from registers
// Two neighbouring accumulator tiles (16 columns) as an A operand; rounded to bf16 for T = bf16.
__device__ __forceinline__ void frag_from(FragA<__nv_bfloat16>& f, const float (&c0)[4], const float (&c1)[4]) {
    f.r[0] = pack_bf16(c0[0], c0[1]); f.r[1] = pack_bf16(c0[2], c0[3]);
    f.r[2] = pack_bf16(c1[0], c1[1]); f.r[3] = pack_bf16(c1[2], c1[3]);
}
__device__ __forceinline__ void frag_from(FragA<float>& f, const float (&c0)[4], const float (&c1)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f.v[i] = c0[i]; f.v[4 + i] = c1[i]; }
}

// An A operand whose steps are multiplied by fp32 weights w (of steps 2t, 2t + 1, 2t + 8,
// 2t + 9), kept to 24 bits: three bf16 pieces (the rounding of what the earlier pieces leave),
// or the fp32 products.
template <typename T> struct ScaledA;
template <> struct ScaledA<__nv_bfloat16> { FragA<__nv_bfloat16> p[3]; };
template <> struct ScaledA<float> { FragA<float> p; };

__device__ __forceinline__ void scale_a(ScaledA<__nv_bfloat16>& o, const FragA<__nv_bfloat16>& a, const float (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x = bf16_lo(a.r[i]) * w[(i >> 1) * 2], y = bf16_hi(a.r[i]) * w[(i >> 1) * 2 + 1];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const uint32_t b = pack_bf16(x, y);
            o.p[q].r[i] = b;
            x -= bf16_lo(b);
            y -= bf16_hi(b);
        }
    }
}
__device__ __forceinline__ void scale_a(ScaledA<float>& o, const FragA<float>& a, const float (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.p.v[i] = a.v[i] * w[(i >> 2) * 2 + (i & 1)];
}
// An accumulator tile into shared memory at s[row * ld + column] (row0, col0: the tile's
// first), as PLANES bf16 pieces `plane` elements apart, or as fp32.
template <int PLANES>
__device__ __forceinline__ void store_tile(__nv_bfloat16* s, int ld, int plane, int row0, int col0, const float (&c)[4], int lane) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float x = c[2 * r], y = c[2 * r + 1];
        __nv_bfloat16* p = s + (row0 + (lane >> 2) + 8 * r) * ld + col0 + 2 * (lane & 3);
#pragma unroll
        for (int q = 0; q < PLANES; ++q) {
            const uint32_t b = pack_bf16(x, y);
            *reinterpret_cast<uint32_t*>(p + q * plane) = b;
            x -= bf16_lo(b);
            y -= bf16_hi(b);
        }
    }
}
template <int PLANES>
__device__ __forceinline__ void store_tile(float* s, int ld, int, int row0, int col0, const float (&c)[4], int lane) {
#pragma unroll
    for (int r = 0; r < 2; ++r)
        *reinterpret_cast<float2*>(s + (row0 + (lane >> 2) + 8 * r) * ld + col0 + 2 * (lane & 3)) = make_float2(c[2 * r], c[2 * r + 1]);
}

}  // namespace swx
