// Joins what the thread blocks have of a row: a warp has one head of one token. Which thread blocks those are it works out anew from the lengths, while the kernels in front
// still run; up to 32 partial results are asked for at once, a lane each its maximum and sum.
#pragma once

#include "jq_pages_attention.cuh"
#include "jq_pages_mma.cuh"

namespace jq {
namespace pages {

constexpr int JOIN_THREADS = 256, JOIN_HEADS = JOIN_THREADS / 32;

template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_THREADS) attend_join_kernel(AttendArgs a) {
    const int lane = threadIdx.x & 31, token = blockIdx.x, h = blockIdx.y * JOIN_HEADS + (threadIdx.x >> 5);
    if (h >= a.heads) {
        return;
    }
    constexpr int V = HD / 32;  // elements of a lane
    // the token's sequence: the last that has it
    int s = -1;
    for (int s0 = 0; s0 < a.b.sequences; s0 += 32) {
        const int i = s0 + lane;
        const bool mine = i < a.b.sequences && token >= a.b.starts[i] && token < a.b.starts[i + 1];
        const unsigned hit = __ballot_sync(0xffffffffu, mine);
        s = hit != 0u ? s0 + 31 - __clz(hit) : s;
    }
    T* const out = static_cast<T*>(a.out) + (int64_t)token * a.ot + h * a.oh;
    if (s < 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (a.fill) {
                out[lane * V + j] = from_float<T>(0.0f);
            }
        }
        return;
    }
    // where the results over own keys and over the prefix are: `count` of them in slots of thread blocks first, first + 1 ..; or one complete
    int count[2], first[2], in_block[2];
    const bool one = a.joined == 0;
    const int kvh = h / a.group;
#pragma unroll
    for (int part = 0; part < 2; part++) {
        const Work& w = part == 0 ? a.own : a.pre;
        count[part] = first[part] = in_block[part] = 0;
        if (part == 1 && one) {
            continue;
        }
        const int seq = part == 0 ? s : a.b.sequences;
        const Sequence q = sequence_at(a, seq, w.rows_shift, w.keys_shift);
        const int64_t base = units_before(a, w, seq, lane);
        const Cut cut = cut_of(w, w.last - w.first == 1 ? q.units(a.kv_heads) : units_before(a, w, w.last, lane));
        if (q.chunks > 0) {
            const int row = (token - q.row0) * a.group + h % a.group;
            const int64_t item0 = base + ((int64_t)kvh * q.blocks + (row >> w.rows_shift)) * q.chunks;
            first[part] = cut.thread_block_of(item0);
            count[part] = cut.thread_block_of(item0 + q.chunks - 1) - first[part] + 1;
            in_block[part] = row & ((1 << w.rows_shift) - 1);
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (one && count[0] == 1) {
        return;  // it is there already
    }
    float m = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        acc[j] = 0.0f;
    }
    const int all = count[0] + count[1];
    for (int n0 = 0; n0 < all; n0 += 32) {
        const int n = n0 + lane;
        const float* from = nullptr;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (n < all) {
            const int part = n < count[0] ? 0 : 1, i = part == 0 ? n : n - count[0];
            const Work& w = part == 0 ? a.own : a.pre;
            if (count[part] == 1) {
                const int64_t at = ((part == 1 ? (int64_t)a.b.tokens : 0) + token) * a.heads + h;
                from = a.whole + at * HD;
                ml = a.whole_ml[at];
            } else {
                const int64_t slot = (((int64_t)(first[part] + i) * 2 + (i == 0 ? 1 : 0)) << w.rows_shift) + in_block[part];
                from = w.part + slot * HD;
                ml = w.part_ml[slot];
            }
        }
        float top = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        top = fmaxf(top, m);
        const float base = top == -INFINITY ? 0.0f : top, shrink = exp2_fast(m - base), weight = exp2_fast(ml.x - base);
        float sum = ml.y * weight;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        m = top;
        l = fmaf(l, shrink, sum);
#pragma unroll
        for (int j = 0; j < V; j++) {
            acc[j] *= shrink;
        }
        const int here = all - n0 < 32 ? all - n0 : 32;
#pragma unroll 4
        for (int i = 0; i < here; i++) {
            const float* const p = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), i)) + lane * V;
            const float x = __shfl_sync(0xffffffffu, weight, i);
#pragma unroll
            for (int j = 0; j < V; j += V >= 4 ? 4 : 2) {
                if constexpr (V >= 4) {
                    const float4 v = *reinterpret_cast<const float4*>(p + j);
                    acc[j] = fmaf(v.x, x, acc[j]);
                    acc[j + 1] = fmaf(v.y, x, acc[j + 1]);
                    acc[j + 2] = fmaf(v.z, x, acc[j + 2]);
                    acc[j + 3] = fmaf(v.w, x, acc[j + 3]);
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(p + j);
                    acc[j] = fmaf(v.x, x, acc[j]);
                    acc[j + 1] = fmaf(v.y, x, acc[j + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        out[lane * V + j] = from_float<T>(over(acc[j], l));
    }
}

}  // namespace pages
}  // namespace jq
