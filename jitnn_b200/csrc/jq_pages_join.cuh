// Joins what the workers have of a row: a thread block has one head of one token. Which workers those are it works out anew from the lengths, while the kernels in front
// still run. Its warps take the partial results in turn, eight each at once, a lane each the maximum and sum of 32.
#pragma once

#include "jq_pages_attention.cuh"
#include "jq_pages_mma.cuh"

namespace jq {
namespace pages {

constexpr int JOIN_WARPS = 4, JOIN_THREADS = 32 * JOIN_WARPS;

template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_THREADS) attend_join_kernel(AttendArgs a) {
    constexpr int V = HD / 32;  // elements of a lane
    __shared__ float meet[JOIN_WARPS][HD];
    __shared__ float2 meet_ml[JOIN_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, token = blockIdx.x, h = blockIdx.y;
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
            if (a.fill && warp == 0) {
                out[lane * V + j] = from_float<T>(0.0f);
            }
        }
        return;
    }
    // where the results over own keys and over the prefix are: `count` of them in slots of workers first, first + 1 ..; or one complete
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
            first[part] = cut.worker_of(item0);
            count[part] = cut.worker_of(item0 + q.chunks - 1) - first[part] + 1;
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
    const int all = count[0] + count[1], each = (all + JOIN_WARPS - 1) / JOIN_WARPS;
    const int mine = each * warp < all ? each * warp : all, upto = mine + each < all ? mine + each : all;
    for (int n0 = mine; n0 < upto; n0 += 32) {
        const int n = n0 + lane;
        const float* from = nullptr;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (n < upto) {
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
        const int here = upto - n0 < 32 ? upto - n0 : 32;
        for (int i0 = 0; i0 < here; i0 += 8) {
            float v[8][V], x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int k = i0 + i < here ? i0 + i : i0;  // (the last ones twice, the second time for nothing)
                const float* const p = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), k)) + lane * V;
                x[i] = __shfl_sync(0xffffffffu, weight, k);
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const float2 e = *reinterpret_cast<const float2*>(p + j);
                    v[i][j] = e.x;
                    v[i][j + 1] = e.y;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (i0 + i < here) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        acc[j] = fmaf(v[i][j], x[i], acc[j]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        meet[warp][lane * V + j] = acc[j];
    }
    if (lane == 0) {
        meet_ml[warp] = make_float2(m, l);
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.0f, weight[JOIN_WARPS];
#pragma unroll
    for (int w = 0; w < JOIN_WARPS; w++) {
        top = fmaxf(top, meet_ml[w].x);
    }
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < JOIN_WARPS; w++) {
        weight[w] = exp2_fast(meet_ml[w].x - base);
        sum = fmaf(meet_ml[w].y, weight[w], sum);
    }
    for (int d = threadIdx.x; d < HD; d += JOIN_THREADS) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; w++) {
            o = fmaf(meet[w][d], weight[w], o);
        }
        out[d] = from_float<T>(over(o, sum));
    }
}

}  // namespace pages
}  // namespace jq
