// What the rotation's kernel and the append's share: runs of 16 bytes (or single elements, where addresses or sizes are odd) as numbers, and the turn of pairs.
#pragma once

#include "jq_pages.cuh"

namespace jq {

// V elements of type T next to each other: 16 bytes, or one element.
template <typename T, int V>
struct Run {
    static constexpr int WORDS = V == 1 ? 1 : 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* x) {
        if constexpr (V > 1) {
            const uint4 v = *reinterpret_cast<const uint4*>(x);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (sizeof(T) == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(x);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(x);
        }
    }
    __device__ __forceinline__ void store(T* y) const {
        if constexpr (V > 1) {
            *reinterpret_cast<uint4*>(y) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<uint32_t*>(y) = w[0];
        } else {
            *reinterpret_cast<uint16_t*>(y) = (uint16_t)w[0];
        }
    }
    __device__ __forceinline__ void numbers(float (&v)[V]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[i] = __uint_as_float(w[i]);
            }
        } else if constexpr (V == 1) {
            v[0] = pair(w[0]).x;
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                const float2 f = pair(w[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
    // rounded to T
    __device__ __forceinline__ void set(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                w[i] = __float_as_uint(v[i]);
            }
        } else if constexpr (V == 1) {
            w[0] = packed(v[0], 0.0f);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                w[i] = packed(v[2 * i], v[2 * i + 1]);
            }
        }
    }
    static __device__ __forceinline__ float2 pair(uint32_t x) {
        if constexpr (std::is_same<T, __half>::value) {
            return __half22float2(*reinterpret_cast<const __half2*>(&x));
        } else {
            return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
        }
    }
    static __device__ __forceinline__ uint32_t packed(float a, float b) {
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(a, b);
            return *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
    }
};

// The cosines and sines of V pairs from pair `first` on; NaN where the table has no such position.
template <int V>
struct Turns {
    float2 cs[V];
    __device__ __forceinline__ void load(const float2* table, int64_t position, int half, int first, float sign) {
        const float2* const row = table + position * half + first;
        if constexpr (V > 1) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float4 f = *reinterpret_cast<const float4*>(row + j);
                cs[j] = make_float2(f.x, f.y * sign);
                cs[j + 1] = make_float2(f.z, f.w * sign);
            }
        } else {
            cs[0] = make_float2(row[0].x, row[0].y * sign);
        }
    }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int j = 0; j < V; j++) {
            cs[j] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
        }
    }
    // The pairs (a[j], b[j]) or, INTERLEAVED, those that stand one after the other in a and then in b; results rounded to T.
    template <bool INTERLEAVED, typename T>
    __device__ __forceinline__ void turn(Run<T, V>& a, Run<T, V>& b) const {
        float x[V], y[V];
        a.numbers(x);
        b.numbers(y);
#pragma unroll
        for (int j = 0; j < V; j++) {
            float& u = !INTERLEAVED || V == 1 ? x[j] : (j < V / 2 ? x[(2 * j) % V] : y[(2 * j) % V]);
            float& v = !INTERLEAVED || V == 1 ? y[j] : (j < V / 2 ? x[(2 * j + 1) % V] : y[(2 * j + 1) % V]);
            const float f = u, g = v;
            u = f * cs[j].x - g * cs[j].y;
            v = f * cs[j].y + g * cs[j].x;
        }
        a.set(x);
        b.set(y);
    }
};

// A kernel that waits for the one in front by itself (griddepcontrol.wait) and so may be scheduled while that one ends; check_launch says how it went.
template <typename Args>
inline void launch_behind(void (*kernel)(Args), dim3 grid, dim3 block, cudaStream_t s, const Args& args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = s;
    cudaLaunchKernelEx(&cfg, kernel, args);
}


// How a row's heads are laid on thread blocks: `units` threads a head (2 V elements each), `lanes` heads beside one another, ITEMS of them one after the other a thread.
struct HeadGrid {
    int units, lanes, blocks;
    HeadGrid(int head_dim, int v, int heads, int items) {
        units = head_dim / (2 * v);
        const int most = 256 / units * items;
        blocks = (heads + most - 1) / most;
        lanes = (heads + blocks * items - 1) / (blocks * items);
    }
};

}  // namespace jq
