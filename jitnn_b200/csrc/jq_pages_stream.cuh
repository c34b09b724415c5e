// The stream kernel of the paged attention: few rows a key/value head against many keys, bound by reading them.
//
// Transposed products of m16n8k16: scores S^T = K Q^T with the keys as the 16 rows of the instruction and eight rows of queries (the heads of a group, of one token or several) as
// its columns, then O^T = V^T P^T. Keys and values go from memory to the registers of the instruction's operand with no stop in shared memory: which 16 of a head's elements
// a step adds up, and which key is which row, is free as long as both operands agree, so a lane takes eight neighbouring elements (16 bytes, 32 in FP32) of its
// rows, and the eight or four lanes beside it the rest of the line. For V^T a lane has the same elements of four keys and pairs two keys' by a byte permute. P^T comes from
// S^T's accumulators by transposing 8 x 8 pieces between lanes. A warp has chunks of 16 keys to itself, with its own maximum and sum; the values of a chunk are asked for
// before its scores are worked out, the keys of the next one right after, so 8 KB (16-bit, head size 128) a warp are on their way all the time. The work is cut among warps,
// which never meet: an item of two chunks costs no barrier, and what the warps have of a long one the joining kernel adds up.
//
// Precision: 16-bit rows and pages are multiplied as they are, weights rounded to the pages' type (and added up as rounded, so that the rounding of a weight that
// stands alone cancels). FP32 rows and weights are sums of three bfloat16 parts, or two half-precision parts with a power of two per row, against the pages' 16-bit
// numbers; FP32 pages are three parts as well, six products for one. The instruction cuts its sums off where it adds, so that a sum over thousands of keys held in it drifts
// towards zero (4e-6 of the result at 8192 keys): it only adds up a chunk, smallest parts first, and the chunks are added with rounding by the multiplication that a new
// maximum takes anyway; of the scores the products of the first parts are added up apart from the small ones.
//
// Measured: 48 sequences of up to 4096 own keys, bf16, 32 heads of 128 on 8, 86 us with the joining kernel's for 0.50 GB, 5.9 TB/s (90 % of a copy's). FP32 pages are bound by the six products and by splitting:
// 15 sequences of 8 rows of those heads behind 3900 keys 211 us. One row against 577 keys, FP32, 13 us in all: the chain of lookup, keys, values and the joining kernel's.
#pragma once

#include "jq_pages_attention.cuh"
#include "jq_pages_mma.cuh"

namespace jq {
namespace pages {

constexpr int CHUNK = 16;  // keys that a warp takes at a time; pages hold whole chunks
constexpr int STREAM_WARPS = 4, STREAM_THREADS = 32 * STREAM_WARPS;
constexpr float LOG2E = 1.4426950408889634f;

template <typename T, typename C, int HD, int NB>
struct Stream {
    static constexpr bool BF = !std::is_same<C, __half>::value;              // the instruction's type: half precision for FP16 pages, bfloat16 for the others
    static constexpr int KP = std::is_same<C, float>::value ? 3 : 1;         // parts of keys and values
    static constexpr int QP = !std::is_same<T, float>::value ? 1 : (BF ? 3 : 2);  // parts of queries and weights
    static constexpr int ROWS = 8 * NB;
    static constexpr int W = sizeof(C) / 2;                                  // 16-byte words of eight elements
    static constexpr int KB = HD / 32, VB = HD / 64;                         // runs of 32 elements (keys), of 64 (values)
    static constexpr bool AHEAD = HD * sizeof(C) <= 512;                     // whether a chunk's keys and values fit the registers; else they are asked for run by run
    static constexpr int Q_BYTES = KB * QP * NB * 512;                       // a warp's queries in shared memory: [run][part][block of eight][lane] x 16 bytes
    static constexpr int SMEM = STREAM_WARPS * Q_BYTES;
};

// Eight elements as pairs of numbers of the instruction: words of part `p`. FP32: x[0..1] hold them.
template <int KP, int W, bool BF>
__device__ __forceinline__ void parts_of_run(const uint4 (&x)[W], uint32_t (&w)[4][KP]) {
    if constexpr (W == 1) {
        w[0][0] = x[0].x; w[1][0] = x[0].y; w[2][0] = x[0].z; w[3][0] = x[0].w;
    } else {
        split_pair<BF, KP>(__uint_as_float(x[0].x), __uint_as_float(x[0].y), w[0]);
        split_pair<BF, KP>(__uint_as_float(x[0].z), __uint_as_float(x[0].w), w[1]);
        split_pair<BF, KP>(__uint_as_float(x[1].x), __uint_as_float(x[1].y), w[2]);
        split_pair<BF, KP>(__uint_as_float(x[1].z), __uint_as_float(x[1].w), w[3]);
    }
}

template <typename T, typename C, int HD, int NB, int RESIDENT>
__global__ void __launch_bounds__(STREAM_THREADS, RESIDENT) attend_stream_kernel(AttendArgs a) {
    using S = Stream<T, C, HD, NB>;
    constexpr bool BF = S::BF;
    constexpr int KP = S::KP, QP = S::QP, ROWS = S::ROWS, W = S::W, KB = S::KB, VB = S::VB;
    constexpr int ROWS_SHIFT = NB == 1 ? 3 : 4, KEYS_SHIFT = 4;
    static_assert(ROWS == 1 << ROWS_SHIFT && CHUNK == 1 << KEYS_SHIFT, "");
    constexpr int PRODUCTS = KP > QP ? KP : QP;  // parts i and j meet where i + j < PRODUCTS
    // Half-precision weights are times 2^15, which the end takes off: one at 2^-29 of the largest has all its bits, where it would be one of the type's smallest, or none, at 2^-24
    constexpr float UP = BF ? 1.0f : 32768.0f;
    extern __shared__ __align__(16) uint8_t all_smem[];
    // Behind the tile kernel this one reads before that one has ended. Every thread block of that one has waited for whatever is in front of the call before it let this kernel be
    // scheduled: what is in front has ended and its writes are in memory before a thread begins here, and the fence makes reads go there, not to what an SM's first-level cache has from before. What that
    // kernel writes nothing here reads or writes. (Waiting here as well, 48 sequences of up to 4096 keys behind 8192 113.3 us and not 109.3, of up to 64 40.2 and 37.6, drafts of FP32 rows 54.7 and 50.7.)
    if (a.stream_first) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
    } else {
        asm volatile("fence.acq_rel.gpu;" ::: "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* const smem = all_smem + warp * S::Q_BYTES;
    const Work& work = a.own;
    const int worker = warp * (int)gridDim.x + (int)blockIdx.x;  // (few workers: on different SMs)
    const Cut cut = cut_of(a, work, lane);
    int64_t begin = (int64_t)worker * cut.per;
    if (begin >= cut.total) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int64_t end = begin + cut.per < cut.total ? begin + cut.per : cut.total;
    int64_t base;
    int s = find_unit(a, work, cut.over, begin, lane, base);
    Sequence sq = sequence_at(a, s, ROWS_SHIFT, KEYS_SHIFT, cut.over);
    const bool wide = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.qt * (int)sizeof(T)) % 16 == 0 && (a.qh * (int)sizeof(T)) % 16 == 0;
    const C* const k_pages = static_cast<const C*>(a.k_pages);
    const C* const v_pages = static_cast<const C*>(a.v_pages);
    while (begin < end) {
        // ---- the next item, or the part of it that is this warp's
        while (begin >= base + sq.units(a.kv_heads)) {
            base += sq.units(a.kv_heads);
            sq = sequence_at(a, ++s, ROWS_SHIFT, KEYS_SHIFT, cut.over);
        }
        const bool prefix = s == a.b.sequences;
        const int64_t item = quotient(begin - base, sq.cost), run0 = base + item * sq.cost + cut.over, behind = run0 + sq.chunks;
        const int64_t from = begin < run0 ? run0 : begin, upto = end < behind ? end : behind;
        begin = upto;
        if (from >= upto) {  // (no run of it: another worker's)
            continue;
        }
        const int kvh = (int)quotient(item, sq.blocks), block = (int)(item - (int64_t)kvh * sq.blocks);
        const int c0 = (int)(from - run0), c1 = (int)(upto - run0);
        const int rows = sq.rows * a.group, row0 = block * ROWS;  // rows of the group: token * group + head
        const int* const table = prefix ? a.b.prefix : a.b.tables + s * a.b.table_stride;
        auto limit_of = [&](int r) { return row0 + r < rows ? keys_seen(a, sq, s, (row0 + r) / a.group) : sq.keys; };  // keys that row r of the block sees
        float q_scale[NB][2];
        __syncwarp();  // (the last item's queries are done with)
        // ---- queries: rows of the block as the instruction's second operand. A lane has eight elements of a run of row g of every block of eight
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const int r = row0 + nb * 8 + g;
            const bool there = r < rows;
            const T* const x = static_cast<const T*>(a.q) + (int64_t)(sq.row0 + (there ? r / a.group : 0)) * a.qt + (int64_t)(kvh * a.group + (there ? r % a.group : 0)) * a.qh + t * 8;
            float v[KB][8];
            float top = 0.0f;
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                load_queries<T>(x + kb * 32, there, wide, v[kb]);
                if constexpr (QP == 2) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        top = fmaxf(top, fabsf(v[kb][j]));
                    }
                }
            }
            float up = 1.0f;
            if constexpr (QP == 2) {  // a power of two per row takes the largest magnitude to [2^9, 2^10)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                uint32_t e = __float_as_uint(top) >> 23;
                e = e < 20u ? 20u : (e > 250u ? 250u : e);
                up = __uint_as_float((263u - e) << 23);
                const float down = __uint_as_float((e - 9u) << 23);
                q_scale[nb][0] = __shfl_sync(0xffffffffu, down, 8 * t);  // of the rows that are this lane's columns
                q_scale[nb][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
            }
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                uint32_t w[4][QP];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    split_pair<BF, QP>(v[kb][2 * j] * up, v[kb][2 * j + 1] * up, w[j]);
                }
#pragma unroll
                for (int p = 0; p < QP; p++) {
                    *reinterpret_cast<uint4*>(smem + (((kb * QP + p) * NB + nb) * 32 + lane) * 16) = make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
                }
            }
        }
        __syncwarp();
        const float to_log2 = a.scale * LOG2E;
        float factor[NB][2];
        int limit[NB][2], least = sq.keys;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int r = nb * 8 + 2 * t + c;
                limit[nb][c] = limit_of(r);
                factor[nb][c] = to_log2;
                if constexpr (QP == 2) {
                    factor[nb][c] *= q_scale[nb][c];
                }
            }
        }
        least = limit_of(0);
        float acc[NB][2 * KB][4];  // O^T: HD / 16 blocks of 16 elements x 8 rows
        float m[NB][2], l[NB][2];
        // ---- the warp's chunks
        constexpr int KH = S::AHEAD ? KB : 1, VH = S::AHEAD ? VB : 1;
        uint4 kr[KH][2][W], vr[VH][4][W];
        auto page_of = [&](int c) { return c < c1 ? table[(c * CHUNK) >> a.page_shift] : -1; };
        auto rows_at = [&](int c, int page) -> int64_t {  // where the chunk's first key is, in elements; -1: nowhere
            if (page < 0 || page >= a.pages) {
                return -1;
            }
            return (((int64_t)page * a.kv_heads + kvh) * a.page_size + ((c * CHUNK) & (a.page_size - 1))) * HD;
        };
        auto load_k = [&](int64_t at, int left, int run) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const bool there = at >= 0 && g + 8 * j < left;
#pragma unroll
                for (int kb = 0; kb < KH; kb++) {
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        kr[kb][j][w] = there ? load_once(k_pages + at + (g + 8 * j) * HD + (run + kb) * 32 + t * 8 + w * 4) : make_uint4(0, 0, 0, 0);
                    }
                }
            }
        };
        auto load_v = [&](int64_t at, int left, int run) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int key = 2 * t + (j & 1) + 8 * (j >> 1);
                const bool there = at >= 0 && key < left;
#pragma unroll
                for (int vb = 0; vb < VH; vb++) {
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        vr[vb][j][w] = there ? load_once(v_pages + at + key * HD + (run + vb) * 64 + g * 8 + w * 4) : make_uint4(0, 0, 0, 0);
                    }
                }
            }
        };
        // The parts of a number, of weights, of FP32 values, make something else of an infinite value than the number does (a part of zero times infinity is none). Where sums are not
        // finite in the end, all of it once more, looking at the values of every chunk
#pragma unroll 1
        for (int turn = 0; turn < 2; turn++) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                for (int i = 0; i < 2 * KB; i++) {
                    acc[nb][i][0] = acc[nb][i][1] = acc[nb][i][2] = acc[nb][i][3] = 0.0f;
                }
                m[nb][0] = m[nb][1] = -INFINITY;
                l[nb][0] = l[nb][1] = 0.0f;
            }
            int c = c0;
            int page = page_of(c), page_next = page_of(c + 1);
            int64_t at = rows_at(c, page);
            if (S::AHEAD && c < c1) {
                load_k(at, sq.keys - c * CHUNK, 0);
            }
            for (; c < c1; c++) {
                const int left = sq.keys - c * CHUNK;  // keys from here on
                if constexpr (S::AHEAD) {
                    load_v(at, left, 0);
                }
                float sc[NB][4], small[NB][4];  // products of the first parts, and all others
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.0f;
                    small[nb][0] = small[nb][1] = small[nb][2] = small[nb][3] = 0.0f;
                }
#pragma unroll
                for (int kb = 0; kb < KB; kb++) {
                    uint32_t x[4][KP], y[4][KP];
                    if constexpr (!S::AHEAD) {
                        load_k(at, left, kb);
                    }
                    parts_of_run<KP, W, BF>(kr[S::AHEAD ? kb : 0][0], x);
                    parts_of_run<KP, W, BF>(kr[S::AHEAD ? kb : 0][1], y);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) {
                            const uint4 q = load_shared16(smem + (((kb * QP + p) * NB + nb) * 32 + lane) * 16);
#pragma unroll
                            for (int i = KP - 1; i >= 0; i--) {
                                if (i + p < PRODUCTS) {
                                    mma<BF>(i + p > 0 ? small[nb] : sc[nb], x[0][i], y[0][i], x[1][i], y[1][i], q.x, q.y);
                                    mma<BF>(i + p > 0 ? small[nb] : sc[nb], x[2][i], y[2][i], x[3][i], y[3][i], q.z, q.w);
                                }
                            }
                        }
                    }
                }
                const int64_t at_now = at;
                if (at_now < 0 && left > 0) {
                    note_status(a.status, STATUS_PAGE);
                }
                page = page_next;
                page_next = page_of(c + 2);
                at = rows_at(c + 1, page);
                if (S::AHEAD && c + 1 < c1) {
                    load_k(at, left - CHUNK, 0);
                }
                const bool edge = c * CHUNK + CHUNK > least || at_now < 0;  // some row does not see all of the chunk
                // ---- scores that are not numbers: in parts an infinity is infinity - infinity too. They are worked out again, one product after the other
                bool odd = false;
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if constexpr (PRODUCTS > 1) {
                            sc[nb][i] += small[nb][i];
                        }
                        sc[nb][i] *= factor[nb][i & 1];
                        odd = odd || sc[nb][i] != sc[nb][i];
                    }
                }
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int r = row0 + nb * 8 + 2 * t + (i & 1), key = g + 8 * (i >> 1);
                            if (sc[nb][i] != sc[nb][i]) {
                                float sum = 0.0f;
                                if (r < rows && key < left && at_now >= 0) {
                                    const T* x = static_cast<const T*>(a.q) + (int64_t)(sq.row0 + r / a.group) * a.qt + (int64_t)(kvh * a.group + r % a.group) * a.qh;
                                    for (int d = 0; d < HD; d++) {
                                        sum = fmaf(to_float(x[d]), to_float(k_pages[at_now + key * HD + d]), sum);
                                    }
                                }
                                sc[nb][i] = sum * to_log2;
                            }
                        }
                    }
                }
                // ---- running maximum and weights; a row's keys are in the eight lanes of one t
                uint32_t pw[NB][2][QP];
                float less[NB][2];  // what the sums so far are multiplied with
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    if (edge) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (c * CHUNK + g + 8 * (i >> 1) >= limit[nb][i & 1] || at_now < 0) {
                                sc[nb][i] = -INFINITY;
                            }
                        }
                    }
                    float top[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        top[j] = fmaxf(sc[nb][j], sc[nb][j + 2]);
                        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 4));
                        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 8));
                        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
                        top[j] = fmaxf(top[j], m[nb][j]);
                        const float from = top[j] == -INFINITY ? 0.0f : top[j], shrink = exp2_fast(m[nb][j] - from);
                        m[nb][j] = top[j];
                        l[nb][j] *= shrink;
                        less[nb][j] = shrink;
                        sc[nb][j] = exp2_fast(sc[nb][j] - from);
                        sc[nb][j + 2] = exp2_fast(sc[nb][j + 2] - from);
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        split_pair<BF, QP>(sc[nb][2 * j] * UP, sc[nb][2 * j + 1] * UP, pw[nb][j]);
                        if constexpr (QP == 1) {
                            if constexpr (BF) {
                                l[nb][0] += __uint_as_float(pw[nb][j][0] << 16);
                                l[nb][1] += __uint_as_float(pw[nb][j][0] & 0xffff0000u);
                            } else {
                                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pw[nb][j][0]));
                                l[nb][0] += f.x;
                                l[nb][1] += f.y;
                            }
                        } else {
                            l[nb][0] += sc[nb][2 * j];
                            l[nb][1] += sc[nb][2 * j + 1];
                        }
                    }
                }
                // ---- values. Where some row does not see a key whose value is not finite, its weight of zero would still make a NaN: then only the rows that see it add it
                bool bad = false;
                if (edge || turn > 0) {
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        if constexpr (!S::AHEAD) {
                            load_v(at_now, left, vb);
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
#pragma unroll
                            for (int w = 0; w < W; w++) {
                                bad = bad || not_finite<W>(vr[S::AHEAD ? vb : 0][j][w], BF);
                            }
                        }
                    }
                    bad = __any_sync(0xffffffffu, bad);
                }
                if (bad) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                        for (int i = 0; i < 2 * KB; i++) {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                acc[nb][i][j] *= less[nb][j & 1];
                            }
                        }
                    }
                    for (int key = 0; key < CHUNK && key < left; key++) {
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const float lo = __shfl_sync(0xffffffffu, sc[nb][j], (key & 7) * 4 + t), hi = __shfl_sync(0xffffffffu, sc[nb][j + 2], (key & 7) * 4 + t);
                                const float p = (key < 8 ? lo : hi) * UP;
                                if (c * CHUNK + key < limit[nb][j]) {
#pragma unroll
                                    for (int i = 0; i < 2 * KB; i++) {
                                        const int d = (i >> 2) * 64 + g * 8 + (i & 3) * 2;
                                        acc[nb][i][j] = fmaf(p, to_float(v_pages[at_now + key * HD + d]), acc[nb][i][j]);
                                        acc[nb][i][j + 2] = fmaf(p, to_float(v_pages[at_now + key * HD + d + 1]), acc[nb][i][j + 2]);
                                    }
                                }
                            }
                        }
                    }
                } else {
                    uint32_t pt[NB][2][QP];
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                        for (int p = 0; p < QP; p++) {
                            pt[nb][0][p] = transpose8(pw[nb][0][p]);
                            pt[nb][1][p] = transpose8(pw[nb][1][p]);
                        }
                    }
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        if constexpr (!S::AHEAD) {
                            load_v(at_now, left, vb);
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) {  // elements 8 g + 2 i and 8 g + 2 i + 1 of four keys: rows g and g + 8 of the operand
                            uint32_t x0[KP], x1[KP], x2[KP], x3[KP];
                            if constexpr (W == 1) {
                                uint32_t w[4];
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    const uint4& v = vr[S::AHEAD ? vb : 0][j][0];
                                    w[j] = i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
                                }
                                x0[0] = __byte_perm(w[0], w[1], 0x5410);
                                x1[0] = __byte_perm(w[0], w[1], 0x7632);
                                x2[0] = __byte_perm(w[2], w[3], 0x5410);
                                x3[0] = __byte_perm(w[2], w[3], 0x7632);
                            } else {
                                float e[4], o[4];
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    const uint4& v = vr[S::AHEAD ? vb : 0][j][i >> 1];
                                    e[j] = __uint_as_float((i & 1) == 0 ? v.x : v.z);
                                    o[j] = __uint_as_float((i & 1) == 0 ? v.y : v.w);
                                }
                                split_pair<BF, KP>(e[0], e[1], x0);
                                split_pair<BF, KP>(o[0], o[1], x1);
                                split_pair<BF, KP>(e[2], e[3], x2);
                                split_pair<BF, KP>(o[2], o[3], x3);
                            }
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) {
                                float chunk[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int p = QP - 1; p >= 0; p--) {
#pragma unroll
                                    for (int n = KP - 1; n >= 0; n--) {
                                        if (n + p < PRODUCTS) {
                                            mma<BF>(chunk, x0[n], x1[n], x2[n], x3[n], pt[nb][0][p], pt[nb][1][p]);
                                        }
                                    }
                                }
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    acc[nb][vb * 4 + i][j] = fmaf(acc[nb][vb * 4 + i][j], less[nb][j & 1], chunk[j]);
                                }
                            }
                        }
                    }
                }
            }
            float probe[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                for (int i = 0; i < 2 * KB; i++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        probe[j] = fmaf(acc[nb][i][j], 0.0f, probe[j]);
                    }
                }
            }
            const float odd_sums = (probe[0] + probe[1]) + (probe[2] + probe[3]);
            if (!__any_sync(0xffffffffu, odd_sums != odd_sums)) {
                break;
            }
        }
        // ---- what the warp has of the item. A lane has elements 64 v + 8 g + 2 i and the one behind it of rows 2 t and 2 t + 1
        const bool complete = c0 == 0 && c1 == sq.chunks;
        constexpr float DOWN = 1.0f / UP, L_DOWN = QP == 1 ? DOWN : 1.0f;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], o);
                }
                l[nb][j] *= L_DOWN;
                const int r = nb * 8 + 2 * t + j;
                if (row0 + r >= rows) {
                    continue;
                }
                const int64_t token = sq.row0 + (row0 + r) / a.group;
                const int head = kvh * a.group + (row0 + r) % a.group;
                if (c0 == 0 && g == 0) {
                    a.found[((prefix ? (int64_t)a.b.tokens : 0) + token) * a.heads + head] = cut.found(run0, sq.chunks, r);
                }
                if (complete && !a.joined) {
                    T* const y = static_cast<T*>(a.out) + token * a.ot + head * a.oh;
#pragma unroll
                    for (int i = 0; i < 2 * KB; i++) {
                        const int d = (i >> 2) * 64 + g * 8 + (i & 3) * 2;
                        y[d] = from_float<T>(over(acc[nb][i][j] * DOWN, l[nb][j]));
                        y[d + 1] = from_float<T>(over(acc[nb][i][j + 2] * DOWN, l[nb][j]));
                    }
                    continue;
                }
                const int64_t at = complete ? ((prefix ? (int64_t)a.b.tokens : 0) + token) * a.heads + head : ((int64_t)worker * 2 + (c0 == 0 ? 1 : 0)) * ROWS + r;
                float* const to = (complete ? a.whole : work.part) + at * HD;
                if (g == 0) {
                    (complete ? a.whole_ml : work.part_ml)[at] = make_float2(m[nb][j], l[nb][j]);
                }
#pragma unroll
                for (int i = 0; i < 2 * KB; i++) {
                    *reinterpret_cast<float2*>(to + (i >> 2) * 64 + g * 8 + (i & 3) * 2) = make_float2(acc[nb][i][j] * DOWN, acc[nb][i][j + 2] * DOWN);
                }
            }
        }
    }
    // (behind the tile kernel, beside which this one works: what waits for this kernel has waited for that one)
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace pages
}  // namespace jq
