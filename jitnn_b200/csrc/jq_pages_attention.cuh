// What the paged attention's kernels share: the arguments, and how the work is cut.
#pragma once

#include "jq_pages.cuh"

namespace jq {

// The work of a launch: items (sequence, key/value head, block of rows), each of as many units as its sequence has runs of keys. Rows are token * group + head of the
// group. The prefix is one more sequence behind the others, all tokens its rows. Units are numbered through all items, a sequence's blocks of rows next to one another (they read the
// same keys), and worker c (a warp, or a thread block) has units c * per .. (c + 1) * per - 1: sequences of any lengths share the GPU evenly, and nobody on the host needs to know the lengths.
// An item that one worker has all of is complete there; of the others a worker leaves partial results in its two slots, the first for the item that
// began in front of it, the second for the one that goes on behind it.
struct Work {
    int first, last;   // sequences first .. last - 1; number b.sequences is the prefix
    int rows_shift;    // rows of a block, keys of a unit: powers of two
    int keys_shift;
    int workers;       // at most
    int over;          // units that beginning and ending an item take the time of
    float* part;       // [slot][rows of a block][head_dim]
    float2* part_ml;   // maxima (of scores times log2 e) and sums
};

struct AttendArgs {
    const void* q;
    void* out;
    int64_t qt, qh, ot, oh;  // strides of token and head, in elements
    const void *k_pages, *v_pages;
    int64_t pages;
    int page_size, page_shift, heads, kv_heads, head_dim, group;
    Batch b;
    float scale;
    int fill;
    int* status;
    Work own, pre;     // whose the own keys' items are, and whose the prefix's
    float* whole;      // of complete items, where own keys and a prefix are to be joined: over own keys and over the prefix, [2][token][head][head_dim]
    float2* whole_ml;
    int joined;        // whether they are
    int2* found;       // for every row and head, of its own keys and of the prefix: the first worker that has some of them, and how many have (256 times that, and the row's
                       // place in its block); the worker of the item's first unit says it. [2][token][head]
    int stream_first;  // whether no tile kernel is in front of the stream kernel
    long long wait_clocks;
};

struct Sequence {
    int row0, rows;    // tokens
    int keys;          // that its last row sees
    int reach;         // the same before it is cut to what the table of pages has, or below zero
    int blocks;        // of rows, per key/value head
    int chunks;        // runs of keys
    int cost;          // units of an item: its runs, and in front of them what beginning and ending it takes
    __device__ int64_t units(int kv_heads) const { return (int64_t)kv_heads * blocks * cost; }
};

__device__ __forceinline__ Sequence sequence_at(const AttendArgs& a, int s, int rows_shift, int keys_shift, int over) {
    Sequence q;
    if (s == a.b.sequences) {
        q.row0 = 0;
        q.rows = a.b.tokens;
        q.keys = q.reach = a.b.prefix_length;
    } else {
        const int from = a.b.starts[s], to = a.b.starts[s + 1], length = a.b.lengths[s];
        q.row0 = from < 0 ? 0 : from;
        const int end = to < a.b.tokens ? to : a.b.tokens;
        q.rows = end > q.row0 ? end - q.row0 : 0;
        // the keys that the sequence's last row here sees; a row's position is counted from the end that the sequence names
        const int64_t keys = (int64_t)length - ((int64_t)to - end);
        const int64_t most = (int64_t)a.b.table_width << a.page_shift;
        if (q.rows > 0 && keys > most) {
            note_status(a.status, STATUS_PAGE);
        }
        q.reach = (int)(keys < -0x40000000 ? -0x40000000 : keys);
        q.keys = q.rows == 0 || keys < 0 ? 0 : (int)(keys < most ? keys : most);
    }
    q.blocks = (int)(((int64_t)q.rows * a.group + (1 << rows_shift) - 1) >> rows_shift);
    q.chunks = (int)(((int64_t)q.keys + (1 << keys_shift) - 1) >> keys_shift);
    q.chunks = q.rows > 0 && q.chunks == 0 ? 1 : q.chunks;  // (rows without keys: an item that finds none)
    q.cost = q.chunks + over;
    return q;
}

// Keys that the row of token `i` of the sequence sees.
__device__ __forceinline__ int keys_seen(const AttendArgs& a, const Sequence& q, int s, int i) {
    if (s == a.b.sequences) {
        return q.keys;
    }
    const int64_t n = (int64_t)q.reach - (q.rows - 1 - i);
    return n < 0 ? 0 : (n < q.keys ? (int)n : q.keys);
}

// x / d of numbers that are not negative, which nearly always have 32 bits (a division of 64 is a hundred instructions and more).
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t d) {
    return ((x | d) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)d) : x / d;
}

struct Cut {
    int64_t total, per;
    int over;  // the items', where there are more units than workers (with fewer each of these is a worker's own)
    // What `found` says of a row of the item whose first run of keys is unit `run0`.
    __device__ __forceinline__ int2 found(int64_t run0, int chunks, int in_block) const {
        const int first = worker_of(run0);
        return make_int2(first, (worker_of(run0 + chunks - 1) - first + 1) << 8 | in_block);
    }
    __device__ __forceinline__ int worker_of(int64_t unit) const { return (int)quotient(unit, per); }
};

// By a whole warp: how a work is cut.
__device__ __forceinline__ Cut cut_of(const AttendArgs& a, const Work& w, int lane) {
    int64_t runs = 0, items = 0;
    for (int s = w.first + lane; s < w.last; s += 32) {
        const Sequence q = sequence_at(a, s, w.rows_shift, w.keys_shift, 0);
        runs += q.units(a.kv_heads);
        items += (int64_t)a.kv_heads * q.blocks;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        runs += __shfl_xor_sync(0xffffffffu, runs, o);
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    Cut c;
    c.over = runs > w.workers ? w.over : 0;
    c.total = runs + items * c.over;
    const int64_t used = c.total < w.workers ? c.total : w.workers;
    c.per = used > 0 ? quotient(c.total + used - 1, used) : 1;
    return c;
}
// The sequence that a unit is in, and the first unit of that sequence; by a whole warp.
__device__ __forceinline__ int find_unit(const AttendArgs& a, const Work& w, int over, int64_t unit, int lane, int64_t& base) {
    int64_t before = 0;
    for (int s0 = w.first; s0 < w.last; s0 += 32) {
        const int s = s0 + lane;
        const int64_t mine = s < w.last ? sequence_at(a, s, w.rows_shift, w.keys_shift, over).units(a.kv_heads) : 0;
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t n = __shfl_up_sync(0xffffffffu, upto, o);
            upto += lane >= o ? n : 0;
        }
        upto += before;
        const unsigned hit = __ballot_sync(0xffffffffu, unit < upto);
        if (hit != 0u) {
            const int at = __ffs(hit) - 1;
            base = __shfl_sync(0xffffffffu, upto - mine, at);
            return s0 + at;
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
    }
    base = before;
    return w.last;
}

}  // namespace jq
