// Warp-level matrix products with float32 accumulators (mma.sync) in two precisions, as operand types with one
// interface, so that a kernel is written once:
//   Half: rows in shared memory are bfloat16 and enter as they are; float32 values enter rounded (A1) or as the sum of
//         two bfloat16, hi + lo within 2^-17 of the value (A2).
//   Full: rows are float32, and every operand is the sum of two tf32 values (11 bits each); the product of the two lo
//         parts is left out: about 2^-21 of a product. Three tf32 products a block, half the rate of bfloat16 each.
// A block is 16 x 16 of the A operand by 16 x 16 of B. Thread (g, t) = (lane / 4, lane % 4) holds of an accumulator
// tile (8 columns) rows g, g + 8 and columns 2 t, 2 t + 1: accumulators of one product become the A operand of the next
// without leaving their registers. (tf32's A fragment holds columns t, t + 4 of 8: columns 2 t and 2 t + 1 take their
// places, and the rows of B the same ones: the order of a contraction's terms is free.)
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

namespace gb {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_at(p))
                 : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_at(p))
                 : "memory");
}
__device__ __forceinline__ void stsm_t(void *p, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(smem_at(p)), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}

// Where a lane points for the four 8x8 matrices of a 16x16 block at (row, col) of a row-major array of this pitch.
// A operand [m][k], and (with .trans) the B operand stored [k][n]:
__device__ __forceinline__ const bf16 *at_a(const bf16 *p, int pitch, int row, int col, int lane) {
    return p + (row + (lane & 15)) * pitch + col + (lane >> 4) * 8;
}
// B operand stored [n][k]; and (with .trans) the A operand stored [k][m]:
__device__ __forceinline__ const bf16 *at_b(const bf16 *p, int pitch, int row, int col, int lane) {
    return p + (row + (lane & 7) + (lane >> 4) * 8) * pitch + col + ((lane >> 3) & 1) * 8;
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ void split(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pack(x, y);
    lo = pack(x - low(hi), y - high(hi));
}

struct Half {
    using E = bf16;
    struct A1 {
        uint32_t x[4];
    };
    struct A2 {
        uint32_t hi[4], lo[4];
    };
    struct B1 {
        uint32_t x[4];
    };
    struct B2 {
        uint32_t hi[4], lo[4];
    };
    // two accumulator tiles (16 columns) as an A operand
    static __device__ __forceinline__ A1 rounded(const float (&c0)[4], const float (&c1)[4]) {
        return {{pack(c0[0], c0[1]), pack(c0[2], c0[3]), pack(c1[0], c1[1]), pack(c1[2], c1[3])}};
    }
    static __device__ __forceinline__ A2 exact(const float (&c0)[4], const float (&c1)[4]) {
        A2 a;
        split(c0[0], c0[1], a.hi[0], a.lo[0]), split(c0[2], c0[3], a.hi[1], a.lo[1]);
        split(c1[0], c1[1], a.hi[2], a.lo[2]), split(c1[2], c1[3], a.hi[3], a.lo[3]);
        return a;
    }
    static __device__ __forceinline__ A1 first(const A2 &a) { return {{a.hi[0], a.hi[1], a.hi[2], a.hi[3]}}; }
    static __device__ __forceinline__ A1 a_rows(const E *p, int pitch, int row, int col, int lane) {  // stored [m][k]
        A1 a;
        ldsm(a.x, at_a(p, pitch, row, col, lane));
        return a;
    }
    static __device__ __forceinline__ A1 a_cols(const E *p, int pitch, int row, int col, int lane) {  // stored [k][m]
        A1 a;
        ldsm_t(a.x, at_b(p, pitch, row, col, lane));
        return a;
    }
    static __device__ __forceinline__ B1 n_rows(const E *p, int pitch, int row, int col, int lane) {  // stored [n][k]
        B1 b;
        ldsm(b.x, at_b(p, pitch, row, col, lane));
        return b;
    }
    static __device__ __forceinline__ B1 k_rows(const E *p, int pitch, int row, int col, int lane) {  // stored [k][n]
        B1 b;
        ldsm_t(b.x, at_a(p, pitch, row, col, lane));
        return b;
    }
    // a 16x16 block in float32 as an accumulator pair's rows and columns: transposed rows of shared memory
    static __device__ __forceinline__ void values_t(float (&c)[2][4], const E *p, int pitch, int row, int col, int lane) {
        uint32_t x[4];
        ldsm_t(x, at_b(p, pitch, row, col, lane));
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e >> 1][(e & 1) * 2] = low(x[e]), c[e >> 1][(e & 1) * 2 + 1] = high(x[e]);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void block(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[4], const uint32_t (&b)[4]) {
        mma(d0, a, b[0], b[1]);
        mma(d1, a, b[2], b[3]);
    }
    static __device__ __forceinline__ void mul(float (&d0)[4], float (&d1)[4], const A1 &a, const B1 &b) {
        block(d0, d1, a.x, b.x);
    }
    static __device__ __forceinline__ void mul(float (&d0)[4], float (&d1)[4], const A2 &a, const B1 &b) {
        block(d0, d1, a.hi, b.x), block(d0, d1, a.lo, b.x);
    }
    static __device__ __forceinline__ void mul(float (&d0)[4], float (&d1)[4], const A1 &a, const B2 &b) {
        block(d0, d1, a.x, b.hi), block(d0, d1, a.x, b.lo);
    }
    static __device__ __forceinline__ void mul(float (&d0)[4], float (&d1)[4], const A2 &a, const B2 &b) {
        block(d0, d1, a.hi, b.hi), block(d0, d1, a.lo, b.hi), block(d0, d1, a.hi, b.lo);
    }
};

struct Full {
    using E = float;
    struct A1 {
        uint32_t hi[8];
        float lo[8];
    };
    using A2 = A1;
    struct B1 {
        uint32_t hi[8];
        float lo[8];
    };
    using B2 = B1;
    // hi: x rounded to 11 bits; lo: the rest, of which the product reads the upper 11 bits
    static __device__ __forceinline__ void part(float x, uint32_t &hi, float &lo) {
        hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
        lo = x - __uint_as_float(hi);
    }
    static __device__ __forceinline__ A1 exact(const float (&c0)[4], const float (&c1)[4]) {
        A1 a;
        part(c0[0], a.hi[0], a.lo[0]), part(c0[2], a.hi[1], a.lo[1]);
        part(c0[1], a.hi[2], a.lo[2]), part(c0[3], a.hi[3], a.lo[3]);
        part(c1[0], a.hi[4], a.lo[4]), part(c1[2], a.hi[5], a.lo[5]);
        part(c1[1], a.hi[6], a.lo[6]), part(c1[3], a.hi[7], a.lo[7]);
        return a;
    }
    static __device__ __forceinline__ A1 rounded(const float (&c0)[4], const float (&c1)[4]) { return exact(c0, c1); }
    static __device__ __forceinline__ const A1 &first(const A1 &a) { return a; }
    static __device__ __forceinline__ A1 a_rows(const E *p, int pitch, int row, int col, int lane) {
        const E *q = p + (row + (lane >> 2)) * pitch + col + 2 * (lane & 3);
        A1 a;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float2 x = *(const float2 *)(q + 8 * k), y = *(const float2 *)(q + 8 * pitch + 8 * k);
            part(x.x, a.hi[4 * k], a.lo[4 * k]), part(y.x, a.hi[4 * k + 1], a.lo[4 * k + 1]);
            part(x.y, a.hi[4 * k + 2], a.lo[4 * k + 2]), part(y.y, a.hi[4 * k + 3], a.lo[4 * k + 3]);
        }
        return a;
    }
    static __device__ __forceinline__ A1 a_cols(const E *p, int pitch, int row, int col, int lane) {
        const E *q = p + (row + 2 * (lane & 3)) * pitch + col + (lane >> 2);
        A1 a;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                part(q[(8 * k + (e >> 1)) * pitch + (e & 1) * 8], a.hi[4 * k + e], a.lo[4 * k + e]);
        return a;
    }
    static __device__ __forceinline__ B1 n_rows(const E *p, int pitch, int row, int col, int lane) {
        const E *q = p + (row + (lane >> 2)) * pitch + col + 2 * (lane & 3);
        B1 b;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 x = *(const float2 *)(q + 8 * n * pitch + 8 * k);
                part(x.x, b.hi[4 * n + 2 * k], b.lo[4 * n + 2 * k]);
                part(x.y, b.hi[4 * n + 2 * k + 1], b.lo[4 * n + 2 * k + 1]);
            }
        return b;
    }
    static __device__ __forceinline__ B1 k_rows(const E *p, int pitch, int row, int col, int lane) {
        const E *q = p + (row + 2 * (lane & 3)) * pitch + col + (lane >> 2);
        B1 b;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    part(q[(8 * k + e) * pitch + 8 * n], b.hi[4 * n + 2 * k + e], b.lo[4 * n + 2 * k + e]);
        return b;
    }
    static __device__ __forceinline__ void values_t(float (&c)[2][4], const E *p, int pitch, int row, int col, int lane) {
        const E *q = p + (row + 2 * (lane & 3)) * pitch + col + (lane >> 2);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[j][e] = q[(8 * j + (e & 1)) * pitch + (e >> 1) * 8];
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t *a, const uint32_t *b) {
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    }
    static __device__ __forceinline__ void mul(float (&d0)[4], float (&d1)[4], const A1 &a, const B1 &b) {
        uint32_t al[8], bl[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) al[e] = __float_as_uint(a.lo[e]), bl[e] = __float_as_uint(b.lo[e]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mma(d0, a.hi + 4 * k, b.hi + 2 * k), mma(d1, a.hi + 4 * k, b.hi + 4 + 2 * k);
            mma(d0, al + 4 * k, b.hi + 2 * k), mma(d1, al + 4 * k, b.hi + 4 + 2 * k);
            mma(d0, a.hi + 4 * k, bl + 2 * k), mma(d1, a.hi + 4 * k, bl + 4 + 2 * k);
        }
    }
};

// Asynchronous copies of 16, 8 or 4 bytes.
template <int BYTES>
__device__ __forceinline__ void cp_async(void *dst, const void *src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(dst)), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_at(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace gb
