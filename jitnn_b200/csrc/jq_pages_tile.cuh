// The tile kernel of the paged attention: many rows a key/value head, on the tensor cores. Blocks of 128 rows (tokens and heads that share a key/value head: all of a batch, where
// the keys are the prefix) against tiles of 64 keys.
//
// A thread has a row, that is a lane of tensor memory. S = Q K^T (tcgen05.mma, 128 x 64, both from shared memory), the thread reads its scores, keeps its maximum and sum, writes
// its weights over the scores, O = P V (weights from tensor memory, values as they lie on the pages: elements of a head are the second operand's columns), and adds O to its
// sums in registers with the factor of the maximum: the instruction cuts off where it adds, so it only adds up a tile. O is read when the next weights are worked out, and the
// scores of the tile behind that are made while those weights are written; keys and values come by asynchronous copies (16 bytes, through the table of pages) a tile or two ahead.
//
// Per tile and SM the products take 512 clocks at head size 128, the threads' part (64 exponentials, 128 sums, about 600 instructions a warp) as long as that and more,
// the copies 1400 clocks where the pages come from memory: two thread blocks share an SM for 16-bit rows. FP32 rows are two half-precision parts (with a power of
// two per row) or three bfloat16 parts, which are so many products for one, and weights likewise.
#pragma once

#include "jq_pages_attention.cuh"
#include "jq_pages_mma.cuh"
#include "jq_tc.cuh"

namespace jq {
namespace pages {

constexpr int TILE_THREADS = 128, TILE_BLOCK = 128, TILE_KEYS = 64;

template <typename T, typename C, int HD>
struct Tile {
    static_assert(sizeof(C) == 2 && (HD == 64 || HD == 128), "");
    static constexpr bool BF = std::is_same<C, __nv_bfloat16>::value;
    static constexpr int QP = sizeof(T) == 2 ? 1 : (BF ? 3 : 2);   // parts of queries and weights
    static constexpr int DB = HD / 64;                             // runs of 64 elements: 128-byte rows of the operands
    static constexpr int Q_PART = DB * TILE_BLOCK * 128, KV = DB * TILE_KEYS * 128;
    static constexpr int SMEM = 1024 + QP * Q_PART + 4 * KV;       // queries, two tiles of keys, two of values, on a 1024-byte boundary
    static constexpr int RESIDENT = QP == 1 ? 2 : 1;
    static constexpr int BUF = QP == 3 ? 96 : 64;                  // columns of a tile's scores, and of its weights after that
    static constexpr int COLS = 2 * BUF + HD <= 256 ? 256 : 512;
    static constexpr uint32_t TYPES = (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(TILE_BLOCK >> 4) << 24);
    static constexpr uint32_t IDESC_S = TYPES | ((uint32_t)(TILE_KEYS >> 3) << 17);
    static constexpr uint32_t IDESC_O = TYPES | ((uint32_t)(HD >> 3) << 17) | (1u << 16);  // the second operand's columns are next to each other
};

// Shared-memory descriptors, 128-byte swizzle: rows of 128 bytes, eight of them 1024 bytes. Rows along the contraction's other axis (queries, keys), or along the
// contraction (values: the next 64 columns follow TILE_KEYS rows further).
constexpr uint32_t TILE_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tile_desc(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t tile_desc_values(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | ((uint32_t)(TILE_KEYS * 128 >> 4) << 16); }

__device__ __forceinline__ void tile_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(TILE_DESC_HI)
        : "memory");
}
__device__ __forceinline__ void tile_mma_weights(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(TILE_DESC_HI)
        : "memory");
}
__device__ __forceinline__ void tile_ld32(float* r, uint32_t addr) {
    uint32_t u[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
          "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]),
          "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]),
          "=r"(u[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) {
        r[i] = __uint_as_float(u[i]);
    }
}
__device__ __forceinline__ float tile_ld1(uint32_t addr) {
    uint32_t u;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(u) : "r"(addr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    return __uint_as_float(u);
}
__device__ __forceinline__ void tile_ld_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tile_st1(uint32_t addr, float v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "r"(__float_as_uint(v)) : "memory");
}
__device__ __forceinline__ void tile_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tile_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Sixteen bytes into shared memory, zeros where `there` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_done() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T, typename C, int HD>
__global__ void __launch_bounds__(TILE_THREADS, Tile<T, C, HD>::RESIDENT) attend_tile_kernel(AttendArgs a) {
    using L = Tile<T, C, HD>;
    constexpr bool BF = L::BF;
    constexpr int QP = L::QP, BUF = L::BUF;
    extern __shared__ uint8_t raw_smem[];
    __shared__ __align__(8) uint64_t bars[3];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    asm volatile("griddepcontrol.launch_dependents;");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Work& work = a.pre;
    const Cut cut = cut_of(work, units_before(a, work, work.last, lane));
    int64_t begin = (int64_t)blockIdx.x * cut.per;
    if (begin >= cut.total) {
        return;
    }
    const int64_t end = begin + cut.per < cut.total ? begin + cut.per : cut.total;
    const uint32_t smem = (tc::smem_u32(raw_smem) + 1023u) & ~1023u;
    const uint32_t q_s = smem, k_s = smem + QP * L::Q_PART, v_s = k_s + 2 * L::KV;
    const uint32_t s_bar = tc::smem_u32(&bars[0]), o_bar = tc::smem_u32(&bars[2]);  // scores of either buffer; O
    volatile int* const abort_flag = &abort_word;
    if (tid == 0) {
        for (int i = 0; i < 3; i++) {
            tc::mbar_init(tc::smem_u32(&bars[i]), 1);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "n"(L::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = tmem_slot, mine = tmem + ((uint32_t)warp << 21);  // (a warp's lanes: 32 from lane 32 warp on)
    uint32_t s_phase = 0, o_phase = 0;  // s_phase: a bit for either buffer
    int64_t base;
    int s = find_unit(a, work, begin, lane, base);
    Sequence sq = sequence_at(a, s, 7, 6);
    const C* const k_pages = static_cast<const C*>(a.k_pages);
    const C* const v_pages = static_cast<const C*>(a.v_pages);
    const bool wide = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.qt * (int)sizeof(T)) % 16 == 0 && (a.qh * (int)sizeof(T)) % 16 == 0;
    const float to_log2 = a.scale * 1.4426950408889634f;
    bool ok = true;
    while (begin < end && ok) {
        while (begin >= base + sq.units(a.kv_heads)) {
            base += sq.units(a.kv_heads);
            sq = sequence_at(a, ++s, 7, 6);
        }
        const bool prefix = s == a.b.sequences;
        const int64_t item = (begin - base) / sq.chunks, item0 = base + item * sq.chunks;
        const int kvh = (int)(item / sq.blocks), block = (int)(item % sq.blocks);
        const int c0 = (int)(begin - item0), c1 = (int)((end < item0 + sq.chunks ? end : item0 + sq.chunks) - item0);
        const int rows = sq.rows * a.group, row0 = block * TILE_BLOCK, r = row0 + tid;
        const int* const table = prefix ? a.b.prefix : a.b.tables + s * a.b.table_stride;
        const int limit = r < rows ? keys_seen(a, sq, s, r / a.group) : sq.keys, least = keys_seen(a, sq, s, row0 / a.group);
        const T* const q = static_cast<const T*>(a.q) + (int64_t)(sq.row0 + (r < rows ? r / a.group : 0)) * a.qt + (int64_t)(kvh * a.group + (r < rows ? r % a.group : 0)) * a.qh;
        const int there = (c1 - c0);
        // ---- copies: a thread has the same 16 bytes of every (128 / pieces of a row)th key
        constexpr int PIECES = HD / 8, STEP = TILE_THREADS / PIECES, TIMES = TILE_KEYS / STEP;
        const int piece = tid % PIECES, key_of = tid / PIECES;
        auto copy_tile = [&](const C* pages, uint32_t to, int c) {
            if (c < c1) {
                int64_t at[TILE_KEYS / 16];
#pragma unroll
                for (int i = 0; i < TILE_KEYS / 16; i++) {
                    const int key = c * TILE_KEYS + i * 16;
                    const int page = key < sq.keys ? table[key >> a.page_shift] : -1;
                    at[i] = page >= 0 && page < a.pages ? (((int64_t)page * a.kv_heads + kvh) * a.page_size + (key & (a.page_size - 1))) * HD : -1;
                }
#pragma unroll
                for (int i = 0; i < TIMES; i++) {
                    const int key = i * STEP + key_of;
                    const int64_t from = at[i * STEP / 16];
                    const bool real = from >= 0 && c * TILE_KEYS + key < sq.keys;
                    copy16(to + (piece >> 3) * (TILE_KEYS * 128) + key * 128 + (((piece ^ key) & 7) << 4), pages + (real ? from + (key & 15) * HD + piece * 8 : 0), real);
                }
            }
            copies_issued();
        };
        // (groups of copies: keys of tiles 0 and 1, values of 0, then keys of n + 2 and values of n + 1 in every turn n)
        copy_tile(k_pages, k_s, c0);
        copy_tile(k_pages, k_s + L::KV, c0 + 1);
        copy_tile(v_pages, v_s, c0);
        // ---- queries: a thread brings its row
        float up = 1.0f, factor = to_log2;
        if constexpr (QP == 2) {  // a power of two takes the row's largest magnitude to [2^9, 2^10)
            float top = 0.0f;
            for (int d = 0; d < HD; d += 8) {
                float v[8];
                load_queries<T>(q + d, r < rows, wide, v);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    top = fmaxf(top, fabsf(v[j]));
                }
            }
            uint32_t e = __float_as_uint(top) >> 23;
            e = e < 20u ? 20u : (e > 250u ? 250u : e);
            up = __uint_as_float((263u - e) << 23);
            factor *= __uint_as_float((e - 9u) << 23);
        }
#pragma unroll 4
        for (int d = 0; d < HD; d += 8) {
            float v[8];
            load_queries<T>(q + d, r < rows, wide, v);
            uint32_t w[4][QP];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                split_pair<BF, QP>(v[2 * j] * up, v[2 * j + 1] * up, w[j]);
            }
#pragma unroll
            for (int p = 0; p < QP; p++) {
                const uint32_t at = q_s + p * L::Q_PART + (d >> 6) * (TILE_BLOCK * 128) + tid * 128 + ((((d >> 3) ^ tid) & 7) << 4);
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0][p]), "r"(w[1][p]), "r"(w[2][p]), "r"(w[3][p]) : "memory");
            }
        }
        // S of tile n (counted from the item's first) into its buffer
        auto scores = [&](int n) {
            const uint32_t kd = tile_desc(k_s + (n & 1) * L::KV), d = tmem + (n & 1) * BUF;
            uint32_t more = 0;
#pragma unroll
            for (int p = QP - 1; p >= 0; p--) {  // smallest parts first
                const uint32_t qd = tile_desc(q_s + p * L::Q_PART);
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    tile_mma(d, qd + (k >> 2) * (TILE_BLOCK * 128 >> 4) + (k & 3) * 2, kd + (k >> 2) * (TILE_KEYS * 128 >> 4) + (k & 3) * 2, L::IDESC_S, more);
                    more = 1;
                }
            }
            tc::umma_commit(s_bar + 8 * (n & 1));
        };
        copies_done<2>();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            tc::fence_after_sync();
            scores(0);
        }
        float acc[HD], m = -INFINITY, l = 0.0f, less = 0.0f;
#pragma unroll
        for (int i = 0; i < HD; i++) {
            acc[i] = 0.0f;
        }
        // adds O of the tile before to the sums
        auto add_o = [&]() {
#pragma unroll
            for (int h = 0; h < HD / 32; h++) {
                float o[32];
                tile_ld32(o, mine + 2 * BUF + 32 * h);
                tile_ld_done();
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    acc[32 * h + i] = fmaf(acc[32 * h + i], less, o[i]);
                }
            }
        };
        bool pending = false;  // an O that has not been read
        constexpr float UP = QP == 2 ? 32768.0f : 1.0f;  // (half-precision parts of weights: times 2^15)
        for (int n = 0; n < there; n++) {
            const int c = c0 + n, buf = n & 1;
            // ---- scores are there, and the next tile's keys
            ok = tc::mbar_wait(s_bar + 8 * buf, (s_phase >> buf) & 1, abort_flag, a.status, 10, a.wait_clocks);
            s_phase ^= 1u << buf;
            copies_done<1>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc::fence_before_sync();
            ok = __syncthreads_and(ok);
            if (!ok) {
                break;
            }
            tc::fence_after_sync();
            // (the keys' buffer of this tile is free: its scores are done. The tile behind the next follows)
            copy_tile(k_pages, k_s + buf * L::KV, c + 2);
            float x[TILE_KEYS];
            tile_ld32(x, mine + buf * BUF);
            tile_ld32(x + 32, mine + buf * BUF + 32);
            tile_ld_done();
            const int left = sq.keys - c * TILE_KEYS;  // keys from here on
            const bool edge = c * TILE_KEYS + TILE_KEYS > least;
            int holes = 0;  // a bit for every 16 keys whose page is not there
#pragma unroll
            for (int i = 0; i < TILE_KEYS / 16; i++) {
                const int key = c * TILE_KEYS + i * 16;
                const int page = key < sq.keys ? table[key >> a.page_shift] : 0;
                holes |= page < 0 || page >= a.pages ? 1 << i : 0;
            }
            if constexpr (QP > 1) {  // in parts an infinity is infinity - infinity too: such scores are worked out again, one product after the other
                bool odd = false;
#pragma unroll
                for (int i = 0; i < TILE_KEYS; i++) {
                    odd = odd || x[i] != x[i];
                }
                if (__any_sync(0xffffffffu, odd)) {
                    for (int key = 0; key < TILE_KEYS; key++) {
                        float v = tile_ld1(mine + buf * BUF + key);
                        if (v != v) {
                            const int i = c * TILE_KEYS + key, page = i < sq.keys ? table[i >> a.page_shift] : -1;
                            float sum = 0.0f;
                            if (r < rows && page >= 0 && page < a.pages) {
                                const C* const k = k_pages + (((int64_t)page * a.kv_heads + kvh) * a.page_size + (i & (a.page_size - 1))) * HD;
                                for (int d = 0; d < HD; d++) {
                                    sum = fmaf(to_float(q[d]) * up, to_float(k[d]), sum);
                                }
                            }
                            v = sum;
                        }
                        tile_st1(mine + buf * BUF + key, v);
                    }
                    tile_st_done();
                    tile_ld32(x, mine + buf * BUF);
                    tile_ld32(x + 32, mine + buf * BUF + 32);
                    tile_ld_done();
                }
            }
            float f = factor;
            if (!(factor > 0.0f)) {  // (the largest product is not that of the largest score)
#pragma unroll
                for (int i = 0; i < TILE_KEYS; i++) {
                    x[i] *= factor;
                }
                f = 1.0f;
            }
            if (edge || holes != 0) {
                if (holes != 0) {
                    note_status(a.status, STATUS_PAGE);
                }
#pragma unroll
                for (int i = 0; i < TILE_KEYS; i++) {
                    x[i] = c * TILE_KEYS + i < limit && (holes >> (i / 16) & 1) == 0 ? x[i] : -INFINITY;
                }
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < TILE_KEYS; i++) {
                top = fmaxf(top, x[i]);
            }
            top = fmaxf(top * f, m);
            const float from = top == -INFINITY ? 0.0f : top, shrink = exp2_fast(m - from);
            m = top;
            l *= shrink;
#pragma unroll
            for (int i = 0; i < TILE_KEYS; i++) {
                x[i] = exp2_fast(fmaf(x[i], f, -from));
            }
            // ---- O of the tile before
            if (pending) {
                ok = tc::mbar_wait(o_bar, o_phase, abort_flag, a.status, 11, a.wait_clocks);
                o_phase ^= 1;
                tc::fence_after_sync();
                if (__all_sync(0xffffffffu, ok)) {
                    add_o();
                }
                pending = false;
            }
            // (the other buffer's weights have been used: the next tile's scores go there)
            if (tid == 0 && ok && n + 1 < there) {
                scores(n + 1);
            }
            less = shrink;
            // ---- weights over the scores
            uint32_t w[QP][16];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    uint32_t part[QP];
                    split_pair<BF, QP>(x[32 * h + 2 * i] * UP, x[32 * h + 2 * i + 1] * UP, part);
#pragma unroll
                    for (int p = 0; p < QP; p++) {
                        w[p][i] = part[p];
                    }
                    if constexpr (QP == 1) {
                        if constexpr (BF) {
                            l += __uint_as_float(part[0] << 16) + __uint_as_float(part[0] & 0xffff0000u);
                        } else {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&part[0]));
                            l += f.x + f.y;
                        }
                    } else {
                        l += x[32 * h + 2 * i] + x[32 * h + 2 * i + 1];
                    }
                }
#pragma unroll
                for (int p = 0; p < QP; p++) {
                    tile_st16(mine + buf * BUF + p * 32 + 16 * h, w[p]);
                }
            }
            tile_st_done();
            copies_done<1>();  // the tile's values
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc::fence_before_sync();
            ok = __syncthreads_and(ok);
            if (!ok) {
                break;
            }
            tc::fence_after_sync();
            // Where some row does not see a key whose value is not finite, its weight of zero would still make a NaN: then every thread adds the values up that its row sees
            bool bad = false;
            if (edge) {
                for (int i = tid; i < L::KV / 16; i += TILE_THREADS) {
                    const uint4 v = load_shared16_at(v_s + buf * L::KV + i * 16);
                    bad = bad || not_finite<1>(v, BF);
                }
                bad = __syncthreads_or(bad);
            }
            if (!bad) {
                if (tid == 0) {
                    const uint32_t vd = tile_desc_values(v_s + buf * L::KV);
                    uint32_t more = 0;
#pragma unroll
                    for (int p = QP - 1; p >= 0; p--) {
#pragma unroll
                        for (int k = 0; k < TILE_KEYS / 16; k++) {
                            tile_mma_weights(tmem + 2 * BUF, tmem + buf * BUF + p * 32 + k * 8, vd + k * (16 * 128 >> 4), L::IDESC_O, more);
                            more = 1;
                        }
                    }
                    tc::umma_commit(o_bar);
                }
                pending = true;
            } else {
#pragma unroll
                for (int i = 0; i < HD; i++) {
                    acc[i] *= less;
                }
                for (int key = 0; key < TILE_KEYS && key < left; key++) {
                    // (the parts of a weight, added up again)
                    float p = 0.0f;
#pragma unroll
                    for (int i = 0; i < QP; i++) {
                        const uint32_t pair = __float_as_uint(tile_ld1(mine + buf * BUF + i * 32 + (key >> 1)));
                        const uint32_t half = (key & 1) != 0 ? pair >> 16 : pair & 0xffffu;
                        p += BF ? __uint_as_float(half << 16) : __half2float(__ushort_as_half((unsigned short)half));
                    }
                    if (c * TILE_KEYS + key < limit) {
#pragma unroll
                        for (int d = 0; d < HD; d += 8) {
                            const uint4 v = load_shared16_at(v_s + buf * L::KV + (d >> 6) * (TILE_KEYS * 128) + key * 128 + ((((d >> 3) ^ key) & 7) << 4));
                            const C* const e = reinterpret_cast<const C*>(&v);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                acc[d + j] = fmaf(p, to_float(e[j]), acc[d + j]);
                            }
                        }
                    }
                }
                tc::fence_before_sync();
                __syncthreads();  // (the values' buffer is free, and the weights')
                tc::fence_after_sync();
            }
            // the values of the next tile: their buffer's last product has been waited for
            copy_tile(v_pages, v_s + (buf ^ 1) * L::KV, c + 1);
        }
        if (pending && ok) {
            ok = tc::mbar_wait(o_bar, o_phase, abort_flag, a.status, 11, a.wait_clocks);
            o_phase ^= 1;
            tc::fence_after_sync();
            if (__all_sync(0xffffffffu, ok)) {
                add_o();
            }
        }
        tc::fence_before_sync();
        copies_done<0>();
        ok = __syncthreads_and(ok);
        tc::fence_after_sync();
        if (!ok) {
            break;
        }
        // ---- what the thread block has of the item
        if (r < rows) {
            constexpr float DOWN = 1.0f / UP;
            const bool complete = c0 == 0 && c1 == sq.chunks;
            const int64_t token = sq.row0 + r / a.group;
            const int head = kvh * a.group + r % a.group;
            if (complete && !a.joined) {
                T* const y = static_cast<T*>(a.out) + token * a.ot + head * a.oh;
#pragma unroll
                for (int i = 0; i < HD; i++) {
                    y[i] = from_float<T>(over(acc[i] * DOWN, l));
                }
            } else {
                const int64_t at = complete ? ((prefix ? (int64_t)a.b.tokens : 0) + token) * a.heads + head : ((int64_t)blockIdx.x * 2 + (c0 == 0 ? 1 : 0)) * TILE_BLOCK + tid;
                float* const to = (complete ? a.whole : work.part) + at * HD;
                (complete ? a.whole_ml : work.part_ml)[at] = make_float2(m, l);
#pragma unroll
                for (int i = 0; i < HD; i += 4) {
                    *reinterpret_cast<float4*>(to + i) = make_float4(acc[i] * DOWN, acc[i + 1] * DOWN, acc[i + 2] * DOWN, acc[i + 3] * DOWN);
                }
            }
        }
        begin = item0 + c1;
    }
    copies_done<0>();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::COLS) : "memory");
    }
}

}  // namespace pages
}  // namespace jq
