// The tile kernel of the paged attention: many rows a key/value head, on the tensor cores. Blocks of 128 rows (tokens and heads that share a key/value head: all of a batch, where
// the keys are the prefix) against tiles of 128 keys.
//
// Warps 0 to 7, two threads a row (a lane of tensor memory), each half of a tile's keys and half of a head's elements: queries into shared memory, then per tile the maximum of
// the row's scores, its weights and their sum. (With one thread a row a warp alone on its scheduler took five clocks an instruction.)
// Warp 8 brings keys and values by tensor-map copies, a box for every page that a tile touches, and issues the products: S = Q K^T (tcgen05.mma,
// 128 x 128, both operands in shared memory), O = P V (weights from tensor memory; values as they lie on the pages, elements of a head are the second operand's columns).
// The instruction cuts off where it adds (a sum of 8192 keys held in it was 4e-6 off). For FP32 rows O only adds up a tile, and the threads add the tiles in registers with the factor of the
// maximum; 16-bit rows, whose rounding is a thousand times that, leave the sums in tensor memory, and only a maximum that rises (with bfloat16 by more than 2^8) has them scaled.
// For 16-bit rows two thread blocks share an SM, one's products under the other's exponentials: weights take the place of the scores. FP32 rows are two half-precision
// parts (with a power of two per row) or three bfloat16 parts, so many products for one, and weights likewise; their weights have columns of their own and, with
// two parts, the scores two buffers, so that the next tile's are made meanwhile.
//
// A row that does not see a key must not get anything of it, and 0 x NaN is one: in tiles that not every row sees whole, values that are not finite, and those behind the last key,
// are cleared in shared memory, and the rows that do see such a key add it by themselves. Sums that are not finite in the end are worked out once more from the values that are not.
//
// Bound per tile and SM: the products' 1024 clocks at head size 128 (times the parts), the threads' 128 exponentials (1024 clocks at 16 a clock) and about 700 instructions a
// warp, or 2800 clocks for 64 KB of pages where they come from memory. Measured, all launches of a call: 280 tokens of 32 heads of 128 on 8 behind 7182 keys, bf16, 82 us, 401 TFLOP/s (FP16, whose sums are scaled more often, 87 us); 48 tokens of
// 64 heads behind 2048 keys, bf16, 30 us. What bounds it is one tile's chain: scores, maximum of both halves, weights, sums are 3.8 us, two of which share an SM.
#pragma once

#include "jq_pages_attention.cuh"
#include "jq_pages_mma.cuh"
#include "jq_tc.cuh"

#include <cstring>

namespace jq {
namespace pages {

constexpr int TILE_BLOCK = 128, TILE_KEYS = 128, TILE_ROW_THREADS = 2 * TILE_BLOCK, TILE_THREADS = TILE_ROW_THREADS + 32;

template <typename T, typename C, int HD>
struct Tile {
    static_assert(sizeof(C) == 2 && (HD == 64 || HD == 128), "");
    static constexpr bool BF = std::is_same<C, __nv_bfloat16>::value;
    static constexpr int QP = sizeof(T) == 2 ? 1 : (BF ? 3 : 2);   // parts of queries and weights
    static constexpr int DB = HD / 64;                             // runs of 64 elements: 128-byte rows of the operands
    static constexpr int Q_PART = DB * TILE_BLOCK * 128, KV = DB * TILE_KEYS * 128;
    static constexpr int RESIDENT = QP == 1 ? 2 : 1;
    static constexpr int KS = QP == 1 && HD == 128 ? 1 : 2, VS = QP != 2 && HD == 128 ? 1 : 2;  // tiles of keys, and of values, in shared memory
    static constexpr int SMEM = 1024 + QP * Q_PART + (KS + VS) * KV;
    static constexpr int BUFS = QP == 2 ? 2 : 1;                   // of scores
    static constexpr bool ALIAS = QP == 1;                         // weights in the scores' columns
    // where the sums over values are held: FP32 results need them added up with rounding, tile by tile; for 16-bit results the instruction does it
    static constexpr bool IN_REGISTERS = QP > 1;
    static constexpr int P_AT = ALIAS ? 0 : BUFS * TILE_KEYS, O_AT = ALIAS ? TILE_KEYS : P_AT + QP * (TILE_KEYS / 2);
    // where the weights of the second half of the keys begin: in the scores' place, over scores that the same thread has read
    static constexpr int P_HALF = ALIAS ? TILE_KEYS / 2 : TILE_KEYS / 4;
    static constexpr int COLS = O_AT + HD <= 256 ? 256 : 512;
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
__device__ __forceinline__ void tile_ld16(float* r, uint32_t addr) {
    uint32_t u[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
                   "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
                 : "r"(addr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) {
        r[i] = __uint_as_float(u[i]);
    }
}
template <int N>
__device__ __forceinline__ void tile_ld(float* r, uint32_t addr) {
    if constexpr (N == 32) {
        tile_ld32(r, addr);
    } else {
        tile_ld16(r, addr);
    }
}
__device__ __forceinline__ void tile_st8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                 "r"(r[6]), "r"(r[7])
                 : "memory");
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

// A box of the pages: 64 elements of a head's keys (or values) from key `slot` of page `page` on.
__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap* map, uint32_t bar, int element, int slot, int page) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to), "l"(map), "r"(bar), "r"(element),
                 "r"(slot), "r"(page)
                 : "memory");
}

// What all of a thread block's roles go through alike: its items, each a run of tiles.
struct Item {
    int s, kvh, row0, rows, c0, c1;
    int64_t run0;
    bool prefix, complete;
};
struct Items {
    int64_t begin, end, base;
    int s, over;
    Sequence sq;
    __device__ __forceinline__ bool next(const AttendArgs& a, Item& it) {
        while (begin < end) {
            while (begin >= base + sq.units(a.kv_heads)) {
                base += sq.units(a.kv_heads);
                sq = sequence_at(a, ++s, 7, 7, over);
            }
            const int64_t item = quotient(begin - base, sq.cost), run0 = base + item * sq.cost + over, behind = run0 + sq.chunks;
            const int64_t from = begin < run0 ? run0 : begin, upto = end < behind ? end : behind;
            begin = upto;
            if (from >= upto) {  // (no run of it: another worker's)
                continue;
            }
            it.s = s;
            it.run0 = run0;
            it.prefix = s == a.b.sequences;
            it.kvh = (int)quotient(item, sq.blocks);
            it.row0 = (int)(item - (int64_t)it.kvh * sq.blocks) * TILE_BLOCK;
            it.rows = sq.rows * a.group;
            it.c0 = (int)(from - run0);
            it.c1 = (int)(upto - run0);
            it.complete = it.c0 == 0 && it.c1 == sq.chunks;
            return true;
        }
        return false;
    }
};

template <typename T, typename C, int HD>
__global__ void __launch_bounds__(TILE_THREADS, Tile<T, C, HD>::RESIDENT)
    attend_tile_kernel(AttendArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using L = Tile<T, C, HD>;
    constexpr bool BF = L::BF;
    constexpr int QP = L::QP, KS = L::KS, VS = L::VS;
    extern __shared__ uint8_t raw_smem[];
    __shared__ __align__(8) uint64_t bars[2 * (KS + VS) + 5];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word, gone_ring[4], o_begun;  // o_begun: an item's sums have been begun by the rows
    __shared__ int gone_on[2];  // of this tile and the last: a row's thread has given up and goes on
    __shared__ uint32_t bad_keys[2][4];
    __shared__ float tops[2][2][TILE_BLOCK], sums[TILE_BLOCK];  // of either half
    __shared__ int64_t row_q[TILE_BLOCK], row_out[TILE_BLOCK];  // where a row's queries are, and its results go; -1: there is no such row
    asm volatile("griddepcontrol.wait;" ::: "memory");  // for whatever is in front of this call
    asm volatile("griddepcontrol.launch_dependents;");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Work& work = a.pre;
    const Cut cut = cut_of(a, work, lane);
    Items items;
    items.begin = (int64_t)blockIdx.x * cut.per;
    if (items.begin >= cut.total) {
        return;
    }
    items.end = items.begin + cut.per < cut.total ? items.begin + cut.per : cut.total;
    items.over = cut.over;
    items.s = find_unit(a, work, cut.over, items.begin, lane, items.base);
    items.sq = sequence_at(a, items.s, 7, 7, cut.over);
    const uint32_t smem = (tc::smem_u32(raw_smem) + 1023u) & ~1023u;
    const uint32_t q_s = smem, k_s = smem + QP * L::Q_PART, v_s = k_s + KS * L::KV;
    auto bar = [&](int i) { return tc::smem_u32(&bars[i]); };
    constexpr int REST = 2 * (KS + VS);
    const uint32_t k_full = bar(0), k_free = bar(KS), v_full = bar(2 * KS), v_free = bar(2 * KS + VS);  // one for each stage
    const uint32_t s_full = bar(REST), p_full = bar(REST + 2), o_full = bar(REST + 3), q_full = bar(REST + 4);
    volatile int* const abort_flag = &abort_word;
    if (warp == 8 && lane == 0) {
        for (int i = 0; i < REST + 5; i++) {
            tc::mbar_init(bar(i), i == REST + 2 || i == REST + 4 ? TILE_ROW_THREADS : 1);
        }
        abort_word = 0;
        o_begun = gone_on[0] = gone_on[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "n"(L::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    Item it;
    // (a wait that gives up sets the abort flag, on which all others end too: every role goes on to its end without waiting or issuing anything)
    auto wait = [&](uint32_t b, uint32_t parity, int code) { return tc::mbar_wait(b, parity, abort_flag, a.status, code, a.wait_clocks); };
    // Where the page of a key of an item is, in the pages' rows of heads; -1 where the cache does not have it (rows that nobody waits for any more go on with whatever stands in the flags of missing keys)
    auto page_row = [&](const int* table, int key, int kvh) -> int64_t {
        const int page = table[key >> a.page_shift];
        return page >= 0 && page < a.pages ? (int64_t)page * a.kv_heads + kvh : -1;
    };

    uint32_t tmem = 0;
    auto begin_products = [&] {  // everybody: the barriers are made, and the columns allocated
        tc::fence_before_sync();
        __syncthreads();
        tc::fence_after_sync();
        tmem = tmem_slot;
    };
    if (warp == 8) {
        __syncwarp();
        // ---- copies and products. A lane has a box: 64 elements of the keys that a tile has of a page (of 128 of them), at most 16 boxes
        const int box = a.page_size < TILE_KEYS ? a.page_size : TILE_KEYS, boxes = TILE_KEYS / box * L::DB;
        const int my_run = lane % L::DB, my_key = lane / L::DB * box;
        bool ok = true;
        // The next tile whose keys, or values, are to be brought, numbered through the items; the page of this lane's box is looked up a tile ahead (the values' are the keys')
        struct Cursor {
            Items items;
            Item it;
            int c;
            bool more;
        } next;
        next.items = items;
        next.more = next.items.next(a, next.it);
        next.c = next.it.c0;
        int page_next = -1;
        auto look_up = [&] {
            const int key = next.c * TILE_KEYS + my_key;
            page_next = -2;
            if (next.more && lane < boxes && key < next.items.sq.keys) {
                page_next = (next.it.prefix ? a.b.prefix : a.b.tables + next.it.s * a.b.table_stride)[key >> a.page_shift];
                page_next = page_next < -1 ? -1 : page_next;
            }
        };
        look_up();
        // what a tile's values need of its keys' copy: the box's row of pages, -1: none; and its first key in the page. Values are at most KS tiles behind
        int v_row[2] = {-1, -1}, v_slot[2] = {0, 0};
        uint32_t v_bytes[2] = {0, 0};
        int keys_brought = 0, values_brought = 0;
        auto bring_keys = [&] {
            const int st = keys_brought % KS, slot = (next.c * TILE_KEYS + my_key) & (a.page_size - 1);
            const bool real = page_next >= 0 && page_next < a.pages;
            const unsigned there = __ballot_sync(0xffffffffu, real), missing = __ballot_sync(0xffffffffu, !real && page_next != -2);
            const int row = real ? page_next * a.kv_heads + next.it.kvh : -1;
            const uint32_t bytes = (uint32_t)__popc(there) * box * 128;
            if (++next.c == next.it.c1) {
                next.more = next.items.next(a, next.it);
                next.c = next.it.c0;
            }
            look_up();
            if (lane == 0) {
                ok = ok && wait(k_free + 8 * st, ((keys_brought / KS) & 1) ^ 1, 10);
                int gone = 0;  // which keys are not there: a bit for each of the tile's sixteens
                for (int i = 0; i < TILE_KEYS / 16 && missing != 0u; i++) {
                    gone |= (missing >> (i * 16 / box * L::DB) & 1) << i;
                }
                gone_ring[keys_brought & 3] = gone;
                if (gone != 0) {
                    note_status(a.status, STATUS_PAGE);
                }
                if (ok) {
                    tc::mbar_expect_tx(k_full + 8 * st, bytes);
                }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            if (ok && row >= 0) {
                copy_box(k_s + st * L::KV + my_run * (TILE_KEYS * 128) + my_key * 128, &k_map, k_full + 8 * st, my_run * 64, slot, row);
            }
            if (keys_brought == values_brought) {
                v_row[0] = row; v_slot[0] = slot; v_bytes[0] = bytes;
            } else {
                v_row[1] = row; v_slot[1] = slot; v_bytes[1] = bytes;
            }
            keys_brought++;
        };
        auto bring_values = [&] {
            const int st = values_brought % VS;
            if (lane == 0) {
                ok = ok && wait(v_free + 8 * st, ((values_brought / VS) & 1) ^ 1, 11);
                if (ok) {
                    tc::mbar_expect_tx(v_full + 8 * st, v_bytes[0]);
                }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            if (ok && v_row[0] >= 0) {
                copy_box(v_s + st * L::KV + my_run * (TILE_KEYS * 128) + my_key * 128, &v_map, v_full + 8 * st, my_run * 64, v_slot[0], v_row[0]);
            }
            v_row[0] = v_row[1]; v_slot[0] = v_slot[1]; v_bytes[0] = v_bytes[1];
            values_brought++;
        };
        // One place for each action: the instructions of a tile come from memory too when a call is small.
        int scored = 0, summed = 0, ni = 0, left = 0, item_first = 0;  // products issued; items; tiles of the item whose scores are to come
        bool refill = true;
        while (ok) {
            // ---- what there is room for: values where the product of VS tiles before has been issued (its end is waited for), keys where the scores have been
            while (refill && ok) {
                const bool values = values_brought < keys_brought && values_brought < summed + VS, keys = next.more && keys_brought < scored + KS && keys_brought < values_brought + 2;
                if (values) {
                    bring_values();
                } else if (keys) {
                    bring_keys();
                } else {
                    break;
                }
            }
            refill = false;
            if (scored == 0) {  // (the first copies are on their way)
                begin_products();
            }
            if (left == 0 && scored == summed) {  // the next item
                if (!items.next(a, it)) {
                    break;
                }
                left = it.c1 - it.c0;
                item_first = summed;
                if (lane == 0) {
                    ok = ok && wait(q_full, ni & 1, 13);
                }
                ni++;
            }
            if (left > 0 && scored < summed + L::BUFS) {
                // ---- S of the next tile
                if (lane == 0) {
                    const int st = scored % KS;
                    if (L::ALIAS && scored > 0) {  // the weights' columns are free
                        ok = ok && wait(o_full, (scored - 1) & 1, 16);
                    }
                    ok = ok && wait(k_full + 8 * st, (scored / KS) & 1, 12);
                    tc::fence_after_sync();
                    if (ok) {
                        const uint32_t kd = tile_desc(k_s + st * L::KV), d = tmem + (scored % L::BUFS) * TILE_KEYS;
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) {  // smallest parts first
                            const uint32_t qd = tile_desc(q_s + p * L::Q_PART);
#pragma unroll
                            for (int j = 0; j < HD / 16; j++) {
                                tile_mma(d, qd + (j >> 2) * (TILE_BLOCK * 128 >> 4) + (j & 3) * 2, kd + (j >> 2) * (TILE_KEYS * 128 >> 4) + (j & 3) * 2, L::IDESC_S,
                                         p < QP - 1 || j > 0 ? 1u : 0u);
                            }
                        }
                        tc::umma_commit(s_full + 8 * (scored % L::BUFS));
                        tc::umma_commit(k_free + 8 * st);
                    }
                }
                scored++;
                left--;
                refill = true;
            } else {
                // ---- O of the next
                if (lane == 0) {
                    const int st = summed % VS;
                    ok = ok && wait(p_full, summed & 1, 14) && wait(v_full + 8 * st, (summed / VS) & 1, 15);
                    tc::fence_after_sync();
                    if (ok) {
                        const uint32_t vd = tile_desc_values(v_s + st * L::KV);
                        bool add = false;  // to what the item's tiles in front have left
                        if constexpr (!L::IN_REGISTERS) {
                            add = summed > item_first || reinterpret_cast<volatile int&>(o_begun) != 0;
                            o_begun = 0;
                        }
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) {
#pragma unroll
                            for (int j = 0; j < TILE_KEYS / 16; j++) {
                                tile_mma_weights(tmem + L::O_AT, tmem + L::P_AT + p * (TILE_KEYS / 2) + (j >> 2) * L::P_HALF + (j & 3) * 8, vd + j * (16 * 128 >> 4), L::IDESC_O,
                                                 p < QP - 1 || j > 0 || add ? 1u : 0u);
                            }
                        }
                        tc::umma_commit(o_full);
                        tc::umma_commit(v_free + 8 * st);
                    }
                }
                summed++;
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        }
    } else {
        // ---- rows
        begin_products();
        auto wait_warp = [&](uint32_t b, uint32_t parity, int code) {  // (warp-wide instructions come next)
            uint32_t got = wait(b, parity, code) ? 1u : 0u;
            asm volatile("" : "+r"(got));  // (no copy of what follows for each answer: 10 % of a prefix's time with three parts)
            __syncwarp();
            return got;
        };
        const int half = warp >> 2, row = tid & (TILE_BLOCK - 1);
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);  // (a warp reaches 32 lanes, from lane 32 (warp % 4) on)
        constexpr int KEYS = TILE_KEYS / 2, DIMS = HD / 2;  // of a thread
        constexpr bool IN_REGISTERS = L::IN_REGISTERS;
        constexpr int CH = 16;  // scores that it holds at a time. (Loops are rolled up: a small call's instructions come from memory, 50 clocks each)
        const bool wide = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.qt * (int)sizeof(T)) % 16 == 0 && (a.qh * (int)sizeof(T)) % 16 == 0;
        auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(TILE_ROW_THREADS) : "memory"); };  // all of these warps
        int n = 0;
        // A thread that has given up goes on to the end with whatever is there. What it meets the others for goes by what all of them have: not by the flags of missing keys, which may be
        // written while it reads them, so that it tells the others first
        uint32_t ok = 1;
        while (items.next(a, it)) {
            const Sequence& sq = items.sq;
            const int r = it.row0 + row, tiles = it.c1 - it.c0, i_token = r / a.group, i_head = r - i_token * a.group;
            const bool real = r < it.rows, direct = it.complete && !a.joined, some = __any_sync(0xffffffffu, real);  // (a warp without rows only keeps the others company)
            const int limit = real ? keys_seen(a, sq, it.s, i_token) : sq.keys, least = keys_seen(a, sq, it.s, it.row0 / a.group);
            if (half == 0) {
                const int64_t token = sq.row0 + i_token;
                const int head = it.kvh * a.group + i_head;
                if (real && it.c0 == 0) {
                    a.found[((it.prefix ? (int64_t)a.b.tokens : 0) + token) * a.heads + head] = cut.found(it.run0, sq.chunks, row);
                }
                row_q[row] = real ? token * a.qt + head * a.qh : -1;
                row_out[row] = !real      ? -1
                               : direct   ? token * a.ot + head * a.oh
                               : it.complete ? (((it.prefix ? (int64_t)a.b.tokens : 0) + token) * a.heads + head)
                                             : ((int64_t)blockIdx.x * 2 + (it.c0 == 0 ? 1 : 0)) * TILE_BLOCK + row;
            }
            meet();
            // ---- queries: LANES lanes bring a row, eight elements each; a warp has 16 rows, as many of which as registers take are on their way at a time
            {
                constexpr int LANES = HD / 8, AT_ONCE = 32 / LANES, BATCH = 16 / AT_ONCE < 4 || QP == 1 ? 16 / AT_ONCE : 4, WORDS = sizeof(T) / 2;
                const int d = lane % LANES * 8, k0 = 16 * warp + lane / LANES;
#pragma unroll 1
                for (int b = 0; b < 16; b += AT_ONCE * BATCH) {
                    uint4 raw[BATCH][WORDS];
#pragma unroll
                    for (int i = 0; i < BATCH; i++) {
                        const int64_t from = row_q[k0 + b + i * AT_ONCE];
                        const T* const x = static_cast<const T*>(a.q) + (from < 0 ? 0 : from) + d;
#pragma unroll
                        for (int w = 0; w < WORDS; w++) {
                            raw[i][w] = make_uint4(0, 0, 0, 0);
                            if (from >= 0 && wide) {
                                raw[i][w] = *reinterpret_cast<const uint4*>(x + 4 * w);
                            } else if (from >= 0) {  // at any address
                                T e[16 / sizeof(T)];
#pragma unroll 1
                                for (int j = 0; j < (int)(16 / sizeof(T)); j++) {
                                    e[j] = x[w * (16 / sizeof(T)) + j];
                                }
                                memcpy(&raw[i][w], e, 16);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < BATCH; i++) {
                        const int k = k0 + b + i * AT_ONCE;
                        uint32_t w[4][QP];
                        if constexpr (QP == 1) {
                            w[0][0] = raw[i][0].x; w[1][0] = raw[i][0].y; w[2][0] = raw[i][0].z; w[3][0] = raw[i][0].w;
                        } else {
                            float v[8] = {__uint_as_float(raw[i][0].x), __uint_as_float(raw[i][0].y), __uint_as_float(raw[i][0].z), __uint_as_float(raw[i][0].w),
                                          __uint_as_float(raw[i][WORDS - 1].x), __uint_as_float(raw[i][WORDS - 1].y), __uint_as_float(raw[i][WORDS - 1].z),
                                          __uint_as_float(raw[i][WORDS - 1].w)};
                            if constexpr (QP == 2) {  // a power of two takes the row's largest magnitude to [2^9, 2^10)
                                float top = 0.0f;
#pragma unroll
                                for (int j = 0; j < 8; j++) {
                                    top = fmaxf(top, fabsf(v[j]));
                                }
#pragma unroll
                                for (int o = LANES / 2; o > 0; o >>= 1) {
                                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                                }
                                uint32_t e = __float_as_uint(top) >> 23;
                                e = e < 20u ? 20u : (e > 250u ? 250u : e);
                                const float by = __uint_as_float((263u - e) << 23);
#pragma unroll
                                for (int j = 0; j < 8; j++) {
                                    v[j] *= by;
                                }
                                sums[k] = by;
                            }
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                split_pair<BF, QP>(v[2 * j], v[2 * j + 1], w[j]);
                            }
                        }
#pragma unroll
                        for (int p = 0; p < QP; p++) {
                            const uint32_t at = q_s + p * L::Q_PART + (d >> 6) * (TILE_BLOCK * 128) + k * 128 + ((((d >> 3) ^ k) & 7) << 4);
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0][p]), "r"(w[1][p]), "r"(w[2][p]), "r"(w[3][p]) : "memory");
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc::mbar_arrive(q_full);
            float up = 1.0f, factor = a.scale * 1.4426950408889634f;
            if constexpr (QP == 2) {
                meet();
                up = sums[row];
                factor /= up;  // (exact)
            }
            float m = -INFINITY, l = 0.0f, less = 0.0f;
            float acc[IN_REGISTERS ? DIMS : 1];
            if constexpr (IN_REGISTERS) {
#pragma unroll
                for (int i = 0; i < DIMS; i++) {
                    acc[i] = 0.0f;
                }
            }
            auto add_o = [&](int tile) {  // O of a tile to the sums
                if constexpr (IN_REGISTERS) {
                ok &= wait_warp(o_full, tile & 1, 17);
                tc::fence_after_sync();
#pragma unroll
                for (int h = 0; h < DIMS / CH; h++) {
                    float o[CH];
                    tile_ld<CH>(o, mine + L::O_AT + half * DIMS + CH * h);
                    tile_ld_done();
#pragma unroll
                    for (int i = 0; i < CH; i++) {
                        acc[CH * h + i] = fmaf(acc[CH * h + i], less, o[i]);
                    }
                }
                }
            };
            // Half-precision weights are times 2^15, as the stream kernel's: off by 2^-40 of the largest at most. So they may not be above one, where bfloat16 ones may be up to 2^8. (With 2^7
            // and 2^8 a weight 20 below the largest was 10 % off; with 2^13 and 2^2 one 21 below 0.2 %. 280 tokens of 32 heads behind 7182 keys 87 us, with those 84 and 85.)
            constexpr float UP = BF ? 1.0f : 32768.0f, LAG = BF ? 8.0f : 0.0f;
            const float f = factor > 0.0f ? factor : 1.0f;
            for (int i = 0;; i++, n++) {
                const int key0 = (it.c0 + i) * TILE_KEYS + half * KEYS;  // this thread's first
                const uint32_t scores = mine + (n % L::BUFS) * TILE_KEYS + half * KEYS;
                bool edge = false;
                int gone = 0;
                float top = -INFINITY;
                auto load = [&](int h, float (&x)[CH]) {  // scores, minus infinity where the row does not see the key
                    tile_ld<CH>(x, scores + CH * h);
                    tile_ld_done();
                    if (!(factor > 0.0f)) {  // (the largest product is not that of the largest score)
#pragma unroll
                        for (int j = 0; j < CH; j++) {
                            x[j] *= factor;
                        }
                    }
                    if (edge) {
                        const int seen = limit - key0 - CH * h;
#pragma unroll
                        for (int j = 0; j < CH; j++) {
                            x[j] = j < seen && (gone >> (CH / 16 * h + j / 16) & 1) == 0 ? x[j] : -INFINITY;
                        }
                    }
                };
                if (i < tiles) {
                    ok &= wait_warp(s_full + 8 * (n % L::BUFS), (n / L::BUFS) & 1, 18);
                    tc::fence_after_sync();
                    gone = reinterpret_cast<volatile int*>(gone_ring)[n & 3];
                    edge = key0 - half * KEYS + TILE_KEYS > least || gone != 0;
                    gone >>= half * (KEYS / 16);
                    for (int turn = 0; some; turn++) {
                        float probe = 0.0f;
                        top = -INFINITY;
#pragma unroll 1
                        for (int h = 0; h < KEYS / CH; h++) {
                            float x[CH];
                            load(h, x);
#pragma unroll
                            for (int j = 0; j < CH; j++) {
                                top = fmaxf(top, x[j]);
                                if constexpr (QP > 1) {
                                    probe = x[j] == -INFINITY ? probe : fmaf(x[j], 0.0f, probe);
                                }
                            }
                        }
                        // in parts an infinity is infinity - infinity too: such scores are worked out again, one product after the other
                        if (QP == 1 || turn == 1 || !__any_sync(0xffffffffu, probe != probe)) {
                            break;
                        }
                        const int* const table = it.prefix ? a.b.prefix : a.b.tables + it.s * a.b.table_stride;
#pragma unroll 1
                        for (int key = 0; key < KEYS; key++) {
                            float v = tile_ld1(scores + key);
                            const int j = key0 + key;
                            const int64_t page = v != v && real && j < limit && (gone >> (key / 16) & 1) == 0 ? page_row(table, j, it.kvh) : -1;
                            if (page >= 0) {
                                const C* const k = static_cast<const C*>(a.k_pages) + (page * a.page_size + (j & (a.page_size - 1))) * HD;
                                const T* const q = static_cast<const T*>(a.q) + row_q[row];
                                v = 0.0f;
#pragma unroll 1
                                for (int d = 0; d < HD; d++) {
                                    v = fmaf(to_float(q[d]) * up, to_float(k[d]), v);
                                }
                            }
                            tile_st1(scores + key, v);
                        }
                        tile_st_done();
                    }
                    tops[n & 1][half][row] = top;
                    if (ok == 0) {
                        gone_on[n & 1] = 1;
                    }
                    meet();
                    top = fmaxf(fmaxf(top, tops[n & 1][half ^ 1][row]) * f, m);
                }
                if constexpr (!IN_REGISTERS) {
                    if (i == tiles) {
                        ok &= wait_warp(o_full, (n - 1) & 1, 17);
                        tc::fence_after_sync();
                        break;
                    }
                    // The sums stay as they are, and weights may be up to 2^LAG, until a maximum is more than that above the one they go by (or is the first)
                    const bool far = top > m + LAG;
                    const float shrink = far ? exp2_fast(m - top) : 1.0f;
                    if (i > 0 && __any_sync(0xffffffffu, far)) {
                        ok &= wait_warp(o_full, (n - 1) & 1, 17);
                        tc::fence_after_sync();
#pragma unroll 1
                        for (int h = 0; h < DIMS / CH; h++) {
                            float o[CH];
                            tile_ld<CH>(o, mine + L::O_AT + half * DIMS + CH * h);
                            tile_ld_done();
                            uint32_t w[CH];
#pragma unroll
                            for (int j = 0; j < CH; j++) {
                                w[j] = __float_as_uint(o[j] * shrink);
                            }
                            tile_st16(mine + L::O_AT + half * DIMS + CH * h, w);
                        }
                    }
                    m = far ? top : m;
                    less = shrink;
                } else {
                    if (i > 0 && some) {
                        add_o(n - 1);  // (its product has been made under this tile's scores and maximum; then the weights' columns and O are free)
                    }
                    if (i == tiles) {
                        break;
                    }
                    less = exp2_fast(m - (top == -INFINITY ? 0.0f : top));
                    m = top;
                }
                const float from = m == -INFINITY ? 0.0f : m;
                float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll 1
                for (int h = 0; h < KEYS / CH && some; h++) {
                    float x[CH];
                    load(h, x);
                    uint32_t w[QP][CH / 2];
#pragma unroll
                    for (int j = 0; j < CH; j++) {
                        x[j] = exp2_fast(fmaf(x[j], f, -from));
                    }
#pragma unroll
                    for (int j = 0; j < CH / 2; j++) {
                        sum0 += x[2 * j];
                        sum1 += x[2 * j + 1];
                        uint32_t part[QP];
                        split_pair<BF, QP>(x[2 * j] * UP, x[2 * j + 1] * UP, part);
#pragma unroll
                        for (int p = 0; p < QP; p++) {
                            w[p][j] = part[p];
                        }
                    }
#pragma unroll
                    for (int p = 0; p < QP; p++) {
                        const uint32_t to = mine + L::P_AT + p * (TILE_KEYS / 2) + half * L::P_HALF + CH / 2 * h;
                        if constexpr (CH == 32) {
                            tile_st16(to, w[p]);
                        } else {
                            tile_st8(to, w[p]);
                        }
                    }
                }
                l = fmaf(l, less, sum0 + sum1);
                tile_st_done();
                if (edge && reinterpret_cast<volatile int*>(gone_on)[n & 1] == 0) {  // (the same for all: nobody writes this one before all have met again)
                    // two threads look at a key's values
                    constexpr int PIECES = HD / 16;
                    const int st = n % VS, key = key0 - half * KEYS + row;
                    ok &= wait_warp(v_full + 8 * st, (n / VS) & 1, 19);
                    const uint32_t at = v_s + st * L::KV + row * 128;
                    bool off = false;
#pragma unroll 1
                    for (int j = half * PIECES; j < (half + 1) * PIECES; j++) {
                        off = off || not_finite<1>(load_shared16_at(at + (j >> 3) * (TILE_KEYS * 128) + (j & 7) * 16), BF);
                    }
                    const bool is = key < sq.keys && (reinterpret_cast<volatile int*>(gone_ring)[n & 3] >> (row / 16) & 1) == 0;
                    const unsigned found = __ballot_sync(0xffffffffu, is && off);
                    if (lane == 0) {
                        bad_keys[half][warp & 3] = found;
                    }
                    meet();
                    uint32_t bad[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        bad[j] = bad_keys[0][j] | bad_keys[1][j];
                    }
                    const uint32_t here = (row >> 5) == 0 ? bad[0] : ((row >> 5) == 1 ? bad[1] : ((row >> 5) == 2 ? bad[2] : bad[3]));
                    if (!is || (here >> lane & 1) != 0) {
#pragma unroll 1
                        for (int j = half * PIECES; j < (half + 1) * PIECES; j++) {
                            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at + (j >> 3) * (TILE_KEYS * 128) + (j & 7) * 16), "r"(0) : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    if ((bad[0] | bad[1] | bad[2] | bad[3]) != 0u) {
                        tc::fence_before_sync();
                        meet();  // (weights of the other half are read)
                        tc::fence_after_sync();
                        const int* const table = it.prefix ? a.b.prefix : a.b.tables + it.s * a.b.table_stride;
                        if constexpr (IN_REGISTERS) {
#pragma unroll
                            for (int j = 0; j < DIMS; j++) {
                                acc[j] *= less;
                            }
                            less = 1.0f;
                        } else {
                            if (i > 0) {
                                ok &= wait_warp(o_full, (n - 1) & 1, 17);
                                tc::fence_after_sync();
                            } else {  // the sums begin here
                                const uint32_t none[16] = {};
#pragma unroll 1
                                for (int h = 0; h < DIMS / 16; h++) {
                                    tile_st16(mine + L::O_AT + half * DIMS + 16 * h, none);
                                }
                                tile_st_done();
                                o_begun = 1;
                            }
                        }
#pragma unroll 1
                        for (int k = 0; k < TILE_KEYS; k++) {
                            if (((bad_keys[0][k >> 5] | bad_keys[1][k >> 5]) >> (k & 31) & 1) == 0) {
                                continue;
                            }
                            float p = 0.0f;  // the parts of the weight, added up again
#pragma unroll
                            for (int j = 0; j < QP; j++) {
                                const uint32_t pair = __float_as_uint(tile_ld1(mine + L::P_AT + j * (TILE_KEYS / 2) + (k >> 6) * L::P_HALF + ((k & 63) >> 1)));
                                const uint32_t word = (k & 1) != 0 ? pair >> 16 : pair & 0xffffu;
                                p += BF ? __uint_as_float(word << 16) : __half2float(__ushort_as_half((unsigned short)word));
                            }
                            const int j = key0 - half * KEYS + k;
                            const int64_t page = page_row(table, j, it.kvh);
                            if (page < 0) {
                                continue;
                            }
                            const C* const v = static_cast<const C*>(a.v_pages) + (page * a.page_size + (j & (a.page_size - 1))) * HD + half * DIMS;
                            if constexpr (IN_REGISTERS) {
                                if (j < limit) {
#pragma unroll
                                    for (int d = 0; d < DIMS; d++) {
                                        acc[d] = fmaf(p, to_float(v[d]), acc[d]);
                                    }
                                }
                            } else {
#pragma unroll 1
                                for (int d = 0; d < DIMS; d++) {
                                    const float o = tile_ld1(mine + L::O_AT + half * DIMS + d);
                                    tile_st1(mine + L::O_AT + half * DIMS + d, j < limit ? fmaf(p, to_float(v[d]), o) : o);
                                }
                                tile_st_done();
                            }
                        }
                    }
                    meet();  // (the list of keys is free)
                }
                tc::fence_before_sync();
                tc::mbar_arrive(p_full);
            }
            tc::fence_before_sync();
            // ---- sums that are not finite. The parts of a weight, or one that is zero in 16 bits, make something else of an infinite value than the weight does: all elements that
            // some key has a value for that is not finite, once more from those keys alone. (A warp's rows go through the item's keys together.)
            {
                float probe = 0.0f;
                if constexpr (IN_REGISTERS) {
#pragma unroll
                    for (int i = 0; i < DIMS; i++) {
                        probe = fmaf(acc[i], 0.0f, probe);
                    }
                } else {
#pragma unroll 1
                    for (int h = 0; h < DIMS / CH; h++) {
                        float o[CH];
                        tile_ld<CH>(o, mine + L::O_AT + half * DIMS + CH * h);
                        tile_ld_done();
#pragma unroll
                        for (int i = 0; i < CH; i++) {
                            probe = fmaf(o[i], 0.0f, probe);
                        }
                    }
                }
                if (__any_sync(0xffffffffu, real && probe != probe)) {
                    const int* const table = it.prefix ? a.b.prefix : a.b.tables + it.s * a.b.table_stride;
                    const int behind = (int64_t)it.c1 * TILE_KEYS < sq.keys ? it.c1 * TILE_KEYS : sq.keys;
                    uint64_t begun = 0;  // elements of this row that have such a value
#pragma unroll 1
                    for (int j = it.c0 * TILE_KEYS; j < behind; j++) {
                        const int64_t page = page_row(table, j, it.kvh);
                        if (page < 0) {
                            continue;
                        }
                        const int64_t at = (page * a.page_size + (j & (a.page_size - 1))) * HD;
                        const C* const v = static_cast<const C*>(a.v_pages) + at + half * DIMS;
                        uint64_t bad = 0;
#pragma unroll 1
                        for (int d = 0; d < DIMS; d += 8) {
                            if (not_finite<1>(*reinterpret_cast<const uint4*>(v + d), BF)) {
#pragma unroll 1
                                for (int i = d; i < d + 8; i++) {
                                    bad |= (uint64_t)(!isfinite(to_float(v[i]))) << i;
                                }
                            }
                        }
                        if (bad == 0) {
                            continue;
                        }
                        float p = 0.0f;
                        if (real && j < limit) {
                            const C* const k = static_cast<const C*>(a.k_pages) + at;
                            const T* const q = static_cast<const T*>(a.q) + row_q[row];
#pragma unroll 1
                            for (int d = 0; d < HD; d++) {
                                p = fmaf(to_float(q[d]), to_float(k[d]), p);
                            }
                            p = exp2_fast(fmaf(p, a.scale * 1.4426950408889634f, m == -INFINITY ? 0.0f : -m)) * UP;
                        }
                        auto sum_of = [&](float sum, int d) {
                            const float more = p * to_float(v[d]);
                            return (bad >> d & 1) == 0 || !real || j >= limit ? sum : ((begun >> d & 1) == 0 ? more : sum + more);
                        };
                        if constexpr (IN_REGISTERS) {
#pragma unroll
                            for (int d = 0; d < DIMS; d++) {
                                acc[d] = sum_of(acc[d], d);
                            }
                        } else {
#pragma unroll 1
                            for (int d = 0; d < DIMS; d++) {
                                const uint32_t o = mine + L::O_AT + half * DIMS + d;
                                tile_st1(o, sum_of(tile_ld1(o), d));
                            }
                            tile_st_done();
                        }
                        begun |= real && j < limit ? bad : 0;
                    }
                }
            }
            // ---- what the thread block has of the item. Its warps' rows, some elements at a time, through the queries' memory (their products are done), so that they go out in lines
            if (half == 1) {
                sums[row] = l;
            }
            meet();
            if (half == 0) {
                l += sums[row];
            }
            constexpr float DOWN = 1.0f / UP;
            if (half == 0 && real && !direct) {
                (it.complete ? a.whole_ml : work.part_ml)[row_out[row]] = make_float2(m, l);
            }
            if (direct) {
                if (half == 0) {
                    tops[0][0][row] = l == 0.0f ? 0.0f : DOWN / l;
                }
                meet();
            }
            const float by = direct ? tops[0][0][row] : DOWN;
            constexpr int WIDTH = QP * L::Q_PART >= 8 * 32 * 32 * 4 ? 32 : 16, PIECES = WIDTH / 4, AT_ONCE = 32 / PIECES;
            const uint32_t rows_s = q_s + warp * (32 * WIDTH * 4);
            float out_o[IN_REGISTERS ? 1 : WIDTH];
#pragma unroll
            for (int run = 0; run < DIMS / WIDTH; run++) {
                __syncwarp();
                if constexpr (!IN_REGISTERS) {
                    tile_ld<WIDTH>(out_o, mine + L::O_AT + half * DIMS + WIDTH * run);
                    tile_ld_done();
                }
                const float* const o = IN_REGISTERS ? acc : out_o;
#pragma unroll
                for (int j = 0; j < PIECES; j++) {
                    const int d = IN_REGISTERS ? WIDTH * run + 4 * j : 4 * j;
                    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(rows_s + lane * (WIDTH * 4) + ((j ^ (lane & (PIECES - 1))) << 4)), "f"(o[d] * by),
                                 "f"(o[d + 1] * by), "f"(o[d + 2] * by), "f"(o[d + 3] * by)
                                 : "memory");
                }
                __syncwarp();
#pragma unroll 4
                for (int i = 0; i < 32 / AT_ONCE; i++) {
                    const int k = AT_ONCE * i + lane / PIECES, piece = lane % PIECES, d = half * DIMS + WIDTH * run + 4 * piece;
                    const uint4 w = load_shared16_at(rows_s + k * (WIDTH * 4) + ((piece ^ (k & (PIECES - 1))) << 4));
                    const int64_t to = row_out[(warp & 3) * 32 + k];
                    if (to < 0) {
                        continue;
                    }
                    if (direct) {
                        T* const y = static_cast<T*>(a.out) + to + d;
                        y[0] = from_float<T>(__uint_as_float(w.x));
                        y[1] = from_float<T>(__uint_as_float(w.y));
                        y[2] = from_float<T>(__uint_as_float(w.z));
                        y[3] = from_float<T>(__uint_as_float(w.w));
                    } else {
                        *reinterpret_cast<uint4*>((it.complete ? a.whole : work.part) + to * HD + d) = w;
                    }
                }
            }
            meet();  // (the next item's queries and rows)
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    // Where some role has given up, copies and products may be under way that nobody has waited for: they write to this thread block's shared and tensor memory, and end long
    // before this millisecond is over, which does not go by the limit that has just run out
    if (*abort_flag != 0) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
            __nanosleep(1000);
        }
    }
    __syncthreads();
    if (warp == 0) {
        tc::fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::COLS) : "memory");
    }
}

}  // namespace pages
}  // namespace jq
