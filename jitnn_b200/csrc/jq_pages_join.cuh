// Joins what the workers have of a row (one head of one token), a lane each the maximum and sum of 32 partial results at a time. While there are fewer rows than warps the GPU holds, the
// four warps of a thread block take a row's partial results in turn: few rows may have hundreds. With more rows a warp has a row. Which workers those are the one with the row's first keys has written down. (Worked out here from all lengths, it was most of this kernel: 15 us for 1536 rows.)
#pragma once

#include "jq_pages_attention.cuh"
#include "jq_pages_mma.cuh"

namespace jq {
namespace pages {

constexpr int JOIN_WARPS = 4, JOIN_THREADS = 32 * JOIN_WARPS;

template <typename T, int HD, int WARPS>
__global__ void __launch_bounds__(JOIN_THREADS) attend_join_kernel(AttendArgs a) {
    constexpr int V = HD / 32, BATCH = WARPS == 1 ? 4 : 8;  // elements of a lane; partial results on their way at a time
    __shared__ float meet[JOIN_WARPS][HD];
    __shared__ float2 meet_ml[JOIN_WARPS];
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS, token = blockIdx.x, h = blockIdx.y * (JOIN_WARPS / WARPS) + (threadIdx.x >> 5) / WARPS;
    if (h >= a.heads) {
        return;
    }
    T* const out = static_cast<T*>(a.out) + (int64_t)token * a.ot + h * a.oh;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    // (asked for together; of a row of no sequence nobody has said anything, and nothing is made of it)
    const bool one = a.joined == 0;
    const int64_t mine_at = (int64_t)token * a.heads + h;
    const int row_first = a.b.starts[0], row_end = a.b.starts[a.b.sequences];
    const int2 said0 = a.found[mine_at], said1 = a.found[one ? mine_at : (int64_t)a.b.tokens * a.heads + mine_at];
    if (token < row_first || token >= row_end) {
        for (int d = 32 * warp + lane; d < HD && a.fill; d += 32 * WARPS) {
            out[d] = from_float<T>(0.0f);
        }
        return;
    }
    // (where the starts are in no order nobody may have said anything: whatever stands there stays in range)
    auto in_range = [](int2 f, const Work& w, int& first, int& count, int& in_block) {
        first = f.x < 0 || f.x >= w.workers ? 0 : f.x;
        count = f.y >> 8;
        count = count < 1 ? 1 : (count > w.workers - first ? w.workers - first : count);
        in_block = f.y & ((1 << w.rows_shift) - 1);
    };
    int first0, count0, block0, first1 = 0, count1 = 0, block1 = 0;
    in_range(said0, a.own, first0, count0, block0);
    if (one && count0 == 1) {
        return;  // it is there already
    }
    if (!one) {
        in_range(said1, a.pre, first1, count1, block1);
    }
    float m = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        acc[j] = 0.0f;
    }
    const int all = count0 + count1, each = (all + WARPS - 1) / WARPS;
    const int mine = each * warp < all ? each * warp : all, upto = mine + each < all ? mine + each : all;
    for (int n0 = mine; n0 < upto; n0 += 32) {
        const int n = n0 + lane;
        const float* from = nullptr;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (n < upto) {
            const bool own = n < count0;
            const int i = own ? n : n - count0;
            if ((own ? count0 : count1) == 1) {
                const int64_t at = (own ? 0 : (int64_t)a.b.tokens * a.heads) + mine_at;
                from = a.whole + at * HD;
                ml = a.whole_ml[at];
            } else {
                const int64_t slot = (((int64_t)((own ? first0 : first1) + i) * 2 + (i == 0 ? 1 : 0)) << (own ? a.own.rows_shift : a.pre.rows_shift)) + (own ? block0 : block1);
                from = (own ? a.own.part : a.pre.part) + slot * HD;
                ml = (own ? a.own.part_ml : a.pre.part_ml)[slot];
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
        for (int i0 = 0; i0 < here; i0 += BATCH) {
            float v[BATCH][V], x[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
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
            for (int i = 0; i < BATCH; i++) {
                if (i0 + i < here) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        acc[j] = fmaf(v[i][j], x[i], acc[j]);
                    }
                }
            }
        }
    }
    if constexpr (WARPS == 1) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            out[lane * V + j] = from_float<T>(over(acc[j], l));
        }
        return;
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
