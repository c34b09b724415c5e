// Device-side pieces of the paged attention's kernels: matrix instructions of 16-bit operands, and 32-bit operands as sums of them.
#pragma once

#include "jq_pages.cuh"

namespace jq {
namespace pages {

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row without any weight gives zero.
__device__ __forceinline__ float over(float o, float sum) { return sum == 0.0f ? 0.0f : o / sum; }

template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// The 8 x 8 matrix of 16-bit numbers that a warp holds in rows (lane 4 r + c: row r, columns 2 c and 2 c + 1), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Two numbers as pairs of 16-bit numbers that add up to them: bfloat16, three parts of eight bits each cut off one after the other (all 24 bits, at any size), or
// half precision, two parts rounded (22 bits where the numbers are scaled to lie in its range); one part is rounded.
template <bool BF, int PARTS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[PARTS]) {
    if constexpr (PARTS == 1) {
        if constexpr (BF) {
            const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
            out[0] = *reinterpret_cast<const uint32_t*>(&r);
        } else {
            const __half2 r = __floats2half2_rn(a, b);
            out[0] = *reinterpret_cast<const uint32_t*>(&r);
        }
    } else if constexpr (BF) {
        static_assert(PARTS == 3, "");
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
            out[i] = __byte_perm(x, y, 0x7632);
            if (i < 2) {
                a -= __uint_as_float(x & 0xffff0000u);
                b -= __uint_as_float(y & 0xffff0000u);
            }
        }
    } else {
        static_assert(PARTS == 2, "");
        const __half2 hi = __floats2half2_rn(a, b);
        const float2 f = __half22float2(hi);
        const __half2 lo = __floats2half2_rn(a - f.x, b - f.y);
        out[0] = *reinterpret_cast<const uint32_t*>(&hi);
        out[1] = *reinterpret_cast<const uint32_t*>(&lo);
    }
}

// Sixteen bytes that this thread block reads once.
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ uint4 load_shared16_at(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint4 load_shared16(const void* p) { return load_shared16_at((uint32_t)__cvta_generic_to_shared(p)); }

// Whether one of the numbers in sixteen bytes is infinite or none: words of FP32 (W = 2), or halves.
template <int W>
__device__ __forceinline__ bool not_finite(const uint4& x, bool bf) {
    if constexpr (W == 2) {
        const uint32_t e = 0x7f800000u;
        return (x.x & e) == e || (x.y & e) == e || (x.z & e) == e || (x.w & e) == e;
    } else {
        const uint32_t e = bf ? 0x7f80u : 0x7c00u;
        bool r = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t v = i == 0 ? x.x : (i == 1 ? x.y : (i == 2 ? x.z : x.w));
            r = r || (v & e) == e || ((v >> 16) & e) == e;
        }
        return r;
    }
}

// Eight neighbouring elements of a row of queries, zeros where there is none; at any address.
template <typename T>
__device__ __forceinline__ void load_queries(const T* x, bool there, bool wide, float (&v)[8]) {
    if (wide && there) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(x), b = *reinterpret_cast<const float4*>(x + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(x);
            const T* const e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] = to_float(e[j]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = there ? to_float(x[j]) : 0.0f;
        }
    }
}

}  // namespace pages
}  // namespace jq
