// Attention over a paged cache for a batch whose sequences share a prefix: row r of sequence s, at the own position t, sees the prefix and the keys 0 .. t of its sequence,
//     o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m),
// in one pass over the keys with a running maximum and sum (ops/FlashAttention.java:538-626 of the reference, which has neither cache nor pages). Sums are FP32.
#include <cmath>

#include "jq_pages_attention.cuh"
#include "jq_pages_join.cuh"
#include "jq_pages_stream.cuh"
#include "jq_pages_tile.cuh"

namespace jq {
namespace {

// Other head sizes than the stream kernel's: one thread block per row and query head. 128 keys at a time, a thread has a key's score, then elements of the output. Nothing
// is shared among the rows and heads that read the same keys: 16 sequences of one row of 32 heads of 96 on 8 against up to 1000 keys, bf16, 405 us, where heads of 128 take 17.
template <typename T, typename C>
__global__ void __launch_bounds__(128) attend_row_kernel(AttendArgs a) {
    __shared__ float qs[256], sc[128], red[8];
    __shared__ int64_t rows[128];
    __shared__ int found[2];
    const int row = blockIdx.x, h = blockIdx.y, kvh = h / (a.heads / a.kv_heads), tid = threadIdx.x, hd = a.head_dim;
    if (tid == 0) {
        found[0] = -1;
    }
    __syncthreads();
    for (int s = tid; s < a.b.sequences; s += 128) {
        const int from = a.b.starts[s], to = a.b.starts[s + 1];
        if (row >= from && row < to) {
            found[0] = s;
            found[1] = a.b.lengths[s] - (to - row);
        }
    }
    const T* q = static_cast<const T*>(a.q) + row * a.qt + h * a.qh;
    T* out = static_cast<T*>(a.out) + row * a.ot + h * a.oh;
    for (int d = tid; d < hd; d += 128) {
        qs[d] = to_float(q[d]) * a.scale;
    }
    __syncthreads();
    const int seq = found[0];
    if (seq < 0) {
        for (int d = tid; d < hd && a.fill; d += 128) {
            out[d] = from_float<T>(0.0f);
        }
        return;
    }
    // (a length beyond what the table of pages has is cut to that, as in the other kernels: prefix and table together have less than 2^31 - 256 keys)
    const int64_t most = (int64_t)a.b.table_width * a.page_size;
    const int own = found[1] < 0 ? 0 : (int)(found[1] < most ? found[1] + 1 : most), keys = a.b.prefix_length + own;
    if (found[1] >= most && tid == 0) {
        note_status(a.status, STATUS_PAGE);
    }
    const C* const kp = static_cast<const C*>(a.k_pages);
    const C* const vp = static_cast<const C*>(a.v_pages);
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int j0 = 0; j0 < keys; j0 += 128) {  // (fewer than 2^31 - 256)
        const int j = j0 + tid;
        int64_t at = -1;
        if (j < keys) {
            const int i = j < a.b.prefix_length ? j : j - a.b.prefix_length, n = i / a.page_size;
            const int page = j < a.b.prefix_length ? a.b.prefix[n] : (n < a.b.table_width ? a.b.tables[seq * a.b.table_stride + n] : -1);
            if (page >= 0 && page < a.pages) {
                at = (((int64_t)page * a.kv_heads + kvh) * a.page_size + i % a.page_size) * hd;
            } else {
                note_status(a.status, STATUS_PAGE);
            }
        }
        float s = -INFINITY;
        if (at >= 0) {
            s = 0.0f;
            for (int d = 0; d < hd; d++) {
                s = fmaf(qs[d], to_float(kp[at + d]), s);
            }
        }
        rows[tid] = at;
        float top = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if ((tid & 31) == 0) {
            red[tid >> 5] = top;
        }
        __syncthreads();
        const float before = m;
        m = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
        const float base = m == -INFINITY ? 0.0f : m, shrink = expf(before - base);
        const float e = at >= 0 ? expf(s - base) : 0.0f;
        sc[tid] = e;
        float sum = e;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if ((tid & 31) == 0) {
            red[4 + (tid >> 5)] = sum;
        }
        __syncthreads();
        l = l * shrink + ((red[4] + red[5]) + (red[6] + red[7]));
        acc[0] *= shrink;
        acc[1] *= shrink;
        for (int i = 0; i < 128 && j0 + i < keys; i++) {
            if (rows[i] >= 0) {
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int d = tid + 128 * n;
                    if (d < hd) {
                        acc[n] = fmaf(sc[i], to_float(vp[rows[i] + d]), acc[n]);
                    }
                }
            }
        }
        __syncthreads();
    }
    for (int n = 0; n < 2; n++) {
        if (tid + 128 * n < hd) {
            out[tid + 128 * n] = from_float<T>(pages::over(acc[n], l));
        }
    }
}

// Who does what, and where in the workspace.
struct Plan {
    int rows = 0;              // of the stream kernel's blocks; 0: it is not launched
    int workers = 0;           // its warps
    int tile_workers = 0;      // the tile kernel's thread blocks; 0: it is not launched
    bool tile_own = false;     // whether it takes own keys too, not the prefix alone
    bool warp_a_row = false;   // how the joining kernel works
    int64_t part = 0, part_ml = 0, tile_part = 0, tile_part_ml = 0, whole = 0, whole_ml = 0, found = 0, bytes = 0;
};

// How many thread blocks of the stream kernel an SM holds (by its registers; 16 rows of heads of 128 with three spilled hundreds of bytes: 16 sequences of 2 rows of 64 heads against
// 1000 keys, bf16, 28 us, with two 21).
constexpr int stream_resident(int head_dim, int bytes, int rows) { return head_dim * bytes >= 512 || head_dim * rows >= 2048 ? 2 : 3; }

// Which kernel: the stream kernel reads the keys once for 8 or 16 rows, the tile kernel (16-bit pages, heads of 64 and 128) for 128, but takes 10 us to begin and end an item.
// A sequence's own keys, whose number only the device knows, by its rows per key/value head: of all sequences the average, so that a prompt beside many single tokens is read by the
// kernel that suits neither best. 16 sequences of up to 700 keys, heads of 128, us here and there. bf16: 32 rows 24.4 and 27.7, 48 rows 30.0 and 29.0, 64 rows 34 and 30; behind 200 keys, which the tile
// kernel takes along, 32 rows 29.9 and 30.9, 40 rows 33.9 and 32.3; behind 600 24 rows 31.6 and 31.7, 32 rows 36 and 32, behind 2048 16 rows 34 and 30, 24 rows 36 and 29.
// FP32 on half precision: 48 rows 32 and 36, 64 rows 38 and 37, 96 rows 51 and 38; behind 200 keys 64 rows 50 and 49; behind 600 40 rows 46 and 47, 48 rows 52 and 48; behind 2048 24 rows 44 and 41, 40 rows
// 55 and 48. Heads of 64 against 1000 keys: bf16 64 rows 28 and 30, FP32 64 rows 31 and 37, 80 rows 73 and 68 (40 sequences).
inline bool tile_takes_own(int head_dim, int parts, int64_t rows, int64_t prefix) {
    return rows > (head_dim == 64 ? 64 : (parts == 1 ? 32 : 64) >> (prefix >= 512 ? 1 : 0));
}
// The prefix by its products: here their number counts, there the pairs of 128 rows and 128 keys (with 2 and 3 parts of FP32 rows twice and three times as dear), and what its
// launch costs. bf16, up to 100 own keys a sequence, us here and there: 8 key/value heads of 128, 128 rows against 2048 keys 24.3 and 23.3, against 4096 33 and 26, 192 rows against 1024 27.0 and 26.6,
// against 2048 33 and 30; 32 key/value heads, 16 rows against 4096 30 and 37; heads of 64, 192 rows against 1024 20 and 22, against 2048 27 and 25, against 4096 31 and 27. Over 64 such shapes, half of them with
// up to 1000 own keys, this takes 0.3 % longer than the better of both, with 1.5e8 in place of 3e8 0.6 % (FP32 rows on half precision 0.4 and 0.6, on bfloat16 0.3 and 0.1).
inline bool tile_takes_prefix(int head_dim, int parts, int64_t kv_heads, int64_t rows, int64_t keys) {
    const double pairs = (double)kv_heads * (double)((rows + 127) / 128) * (double)((keys + 127) / 128);
    return (double)kv_heads * (double)rows * (double)keys * head_dim > 3e8 + parts * (head_dim == 64 ? 1.5e5 : 2e5) * pairs;
}
// Rows of the stream kernel's blocks. Heads of 128, 16 sequences, bf16: 16 own rows against 1000 keys 21 us with 16 and 22 with 8, 32 rows 28 and 30. Heads of 64, half precision, where more and shorter
// items are worth a second reading of the keys: 16 rows 17.4 and 15.5, 32 rows 20.5 and 20.1 (FP32 34 and 37), 20 rows against 200 keys 13 and 11, but behind 1023 keys 32 and 37.
// For a prefix even where own rows are up to 8, us with 16 and with 8. 64 heads of 128 on 8, bf16, up to 100 own keys a sequence: 16 sequences behind 700 keys 16.7 and 16.9, behind 1500 21.7 and 22.1, behind 2500
// 26.4 and 29.4; 32 heads on 8, 24 sequences behind 2500 23.6 and 25.4; 64 heads of 64 on 8, 40 sequences behind 1500 24.5 and 28.1; 16 rows of each of 32 key/value heads behind 2500, which gain nothing, 24.8 and
// 23.6. Over 268 shapes of bf16, of FP32 on half precision and of FP32 pages, half of them with up to 1000 own keys, 0.6 % over the better of both, always with 8 rows 3.1 %. 16 rows of heads of 256 do not fit the
// registers.
inline int stream_rows(int head_dim, int64_t own, int64_t kv_heads, int64_t shared, int64_t prefix) {
    const double products = (double)kv_heads * (double)shared * (double)prefix * head_dim;
    const bool sixteen = own > 8 ? head_dim == 128 || own >= 32 || products > 1e8 : shared >= 96 && products > 1.5e8;
    return head_dim <= 128 && sixteen ? 16 : 8;
}
// What beginning and ending an item takes, in units (128 and 16 keys). Without it whoever had many short items was late: 24 sequences of 5 rows with up to
// 64 own keys behind 4096, heads of 128, with the tile kernel, bf16 59 us (with 1, 3 and 5 units 41, 37 and 40), FP32 on half precision 55 (54, 51 and 51); with the stream kernel heads of 64, a row each, FP32 on half
// precision 45 us (with 2 and 4 units 24.2 and 22.4), 5 rows behind 1000, half precision, 58 (29 and 25).
constexpr int TILE_OVER = 3, STREAM_OVER = 4;

// Whether one warp joins a row, or four do. bf16, in all, us with one and with four: 8 tokens of 64 heads of 128 against up to 1000 keys 17.1 and 13.7, 16 tokens 18.5 and 17.3, 24 tokens 21.2 and 21.6, 100 tokens
// 50.5 and 59.9. In between a row may have many partial results, of a long prefix: 48 tokens of 32 heads behind 4096 keys 40.9 and 39.0, behind 8192 40.1 and 38.1, of heads of 64 34.5 and 33.0, 24 of 64 heads
// behind 4096 36.1 and 33.5, 64 of 32 behind 8192 42.0 and 41.3; without a prefix 48 of 32 29.7 and 31.3.
inline bool warp_joins_row(int64_t rows, int64_t partial) { return rows > 1200 && (partial < 12 || rows > 4800); }

Plan plan_of(const jq_pages* p, int elem, int heads, int64_t tokens, int64_t sequences, int64_t prefix_length) {
    Plan plan;
    const int hd = p->head_dim;
    if ((hd != 64 && hd != 128 && hd != 256) || tokens == 0) {
        return plan;
    }
    const int64_t group = heads / p->kv_heads, own = (tokens + sequences - 1) / sequences * group, shared = tokens * group;
    const bool tile = p->elem != JQ_ELEM_F32 && hd <= 128;
    const int parts = elem == p->elem ? 1 : (p->elem == JQ_ELEM_F16 ? 2 : 3);  // of a row's FP32 numbers
    plan.tile_own = tile && tile_takes_own(hd, parts, own, prefix_length);
    if (plan.tile_own || (tile && prefix_length > 0 && tile_takes_prefix(hd, parts, p->kv_heads, shared, prefix_length))) {
        const int resident = elem == p->elem ? 2 : 1;
        // (the prefix's units are known here; of the own keys the device knows)
        const int64_t units = (int64_t)p->kv_heads * ((shared + pages::TILE_BLOCK - 1) / pages::TILE_BLOCK) * ((prefix_length + pages::TILE_KEYS - 1) / pages::TILE_KEYS);
        plan.tile_workers = (int)(!plan.tile_own && units < 148 * resident ? units : 148 * resident);
    }
    if (!plan.tile_own) {
        plan.rows = stream_rows(hd, own, p->kv_heads, shared, plan.tile_workers == 0 ? prefix_length : 0);
        plan.workers = 148 * stream_resident(hd, elem_bytes(p->elem), plan.rows) * pages::STREAM_WARPS;
    }
    // (an item that there are few of is cut into about as many pieces as there are workers for each; of the prefix's the length is known)
    const int own_rows = plan.tile_own ? pages::TILE_BLOCK : plan.rows, shared_rows = plan.tile_workers > 0 ? pages::TILE_BLOCK : plan.rows;
    const int64_t own_items = sequences * p->kv_heads * ((own + own_rows - 1) / own_rows), of_own = (plan.tile_own ? plan.tile_workers : plan.workers) / own_items;
    const int64_t shared_items = p->kv_heads * ((shared + shared_rows - 1) / shared_rows), shared_workers = plan.tile_workers > 0 ? plan.tile_workers : plan.workers;
    const int64_t runs = (prefix_length + (plan.tile_workers > 0 ? pages::TILE_KEYS : 16) - 1) / (plan.tile_workers > 0 ? pages::TILE_KEYS : 16);
    const int64_t of_shared = runs / ((shared_items * runs + shared_workers) / shared_workers);
    plan.warp_a_row = warp_joins_row(tokens * heads, of_own > of_shared ? of_own : of_shared);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    plan.part = take((int64_t)2 * plan.workers * plan.rows * hd * 4);
    plan.part_ml = take((int64_t)2 * plan.workers * plan.rows * 8);
    plan.tile_part = take((int64_t)2 * plan.tile_workers * pages::TILE_BLOCK * hd * 4);
    plan.tile_part_ml = take((int64_t)2 * plan.tile_workers * pages::TILE_BLOCK * 8);
    if (prefix_length > 0) {
        plan.whole = take(2 * tokens * heads * hd * 4);
        plan.whole_ml = take(2 * tokens * heads * 8);
    }
    plan.found = take(2 * tokens * heads * (int64_t)sizeof(int2));
    plan.bytes = at;
    return plan;
}

// Once per kernel and device: leave for more than 48 KB of shared memory; and `of_sm` bytes of it for an SM, so that the rest is first-level cache (0: as it comes). Bytes on
// their way from memory have their place there. A kernel that is scheduled beside the end of one with much shared memory is otherwise left with that one's split: the stream kernel behind the tile
// kernel, 48 sequences behind 8192 keys, 142 us instead of 109. (24 KB more than its
// thread blocks add up to: with none fewer of them fit, 16 sequences of drafts 40 us instead of 33.)
template <typename K>
int prepare(K kernel, int smem, bool large, int of_sm, std::atomic<uint64_t>& configured) {
    int dev = 0;
    JQ_CUDA(cudaGetDevice(&dev));
    if ((configured.load(std::memory_order_relaxed) >> (dev & 63) & 1) == 0) {
        if (large) {
            JQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        }
        if (of_sm > 0) {
            JQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (of_sm * 100 + 228 * 1024 - 1) / (228 * 1024)));
        }
        configured.fetch_or((uint64_t)1 << (dev & 63));
    }
    return JQ_OK;
}

// Programmatically: the first kernel waits at its beginning for what is in front of the call, all of this call's kernels but the joining one work at the same time.
template <typename K, typename... More>
int launch_part(K kernel, dim3 grid, int threads, int smem, cudaStream_t s, const AttendArgs& a, const More&... more) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    JQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, more...));
    count_launch();
    return JQ_OK;
}

template <typename T, typename C, int HD, int NB>
int launch_stream(const AttendArgs& a, const Plan& plan, cudaStream_t s) {
    static std::atomic<uint64_t> configured{0};
    constexpr int smem = pages::Stream<T, C, HD, NB>::SMEM;
    auto kernel = pages::attend_stream_kernel<T, C, HD, NB, stream_resident(HD, sizeof(C), 8 * NB)>;
    const int rc = prepare(kernel, smem, smem > 48 * 1024, stream_resident(HD, sizeof(C), 8 * NB) * (smem + 1024) + 24 * 1024, configured);
    return rc != JQ_OK ? rc : launch_part(kernel, dim3((unsigned)(plan.workers / pages::STREAM_WARPS)), pages::STREAM_THREADS, smem, s, a);
}

template <typename T, typename C, int HD>
int launch_attend_head(const jq_pages* p, const AttendArgs& a, const Plan& plan, cudaStream_t s) {
    int rc = JQ_OK;
    if constexpr (sizeof(C) == 2 && HD <= 128) {
        if (plan.tile_workers > 0) {
            static std::atomic<uint64_t> configured{0};
            constexpr int smem = pages::Tile<T, C, HD>::SMEM;
            rc = prepare(pages::attend_tile_kernel<T, C, HD>, smem, true, 0, configured);
            rc = rc != JQ_OK ? rc : launch_part(pages::attend_tile_kernel<T, C, HD>, dim3((unsigned)plan.tile_workers), pages::TILE_THREADS, smem, s, a, p->k_map, p->v_map);
        }
    }
    if (rc == JQ_OK && plan.rows == 8) {
        rc = launch_stream<T, C, HD, 1>(a, plan, s);
    }
    if constexpr (HD <= 128) {
        if (rc == JQ_OK && plan.rows == 16) {
            rc = launch_stream<T, C, HD, 2>(a, plan, s);
        }
    }
    if (rc != JQ_OK) {
        return rc;
    }
    if (plan.warp_a_row) {
        return launch_part(pages::attend_join_kernel<T, HD, 1>, dim3((unsigned)a.b.tokens, (unsigned)(a.heads + pages::JOIN_WARPS - 1) / pages::JOIN_WARPS), pages::JOIN_THREADS, 0, s, a);
    }
    return launch_part(pages::attend_join_kernel<T, HD, pages::JOIN_WARPS>, dim3((unsigned)a.b.tokens, (unsigned)a.heads), pages::JOIN_THREADS, 0, s, a);
}

template <typename T, typename C>
int launch_attend(const jq_pages* p, const AttendArgs& a, const Plan& plan, cudaStream_t s) {
    switch (a.head_dim) {
        case 64: return launch_attend_head<T, C, 64>(p, a, plan, s);
        case 128: return launch_attend_head<T, C, 128>(p, a, plan, s);
        case 256: return launch_attend_head<T, C, 256>(p, a, plan, s);
        default: break;
    }
    attend_row_kernel<T, C><<<dim3((unsigned)a.b.tokens, (unsigned)a.heads), 128, 0, s>>>(a);
    count_launch();
    return check_launch("attend_row_kernel");
}

}  // namespace
}  // namespace jq

using namespace jq;

extern "C" {

JQ_API int jq_pages_attention_bytes(const jq_pages* p, int elem, int heads, int64_t tokens, int64_t sequences, int64_t prefix_length, int64_t* nbytes) {
    const int rc = check_pages(p, "jq_pages_attention_bytes");
    if (rc != JQ_OK) {
        return rc;
    }
    if (nbytes == nullptr || heads < 1 || heads % p->kv_heads != 0 || tokens < 0 || tokens > 0x7fffffff || sequences < 1 || prefix_length < 0) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention: %lld rows of %lld sequences, %d heads on %d key/value heads", (long long)tokens, (long long)sequences, heads,
                    p->kv_heads);
    }
    *nbytes = plan_of(p, elem, heads, tokens, sequences, prefix_length).bytes;
    return JQ_OK;
}

JQ_API int jq_pages_attention(const jq_pages* p, int elem, int heads, const void* q, void* out, const int64_t* strides, int64_t tokens, const int32_t* tables,
                              int64_t table_stride, int64_t table_width, const int32_t* starts, const int32_t* lengths, int sequences, const int32_t* prefix,
                              int64_t prefix_width, int64_t prefix_length, float scale, int fill, void* workspace, int64_t workspace_bytes, void* stream) {
    int64_t need = 0;
    int rc = jq_pages_attention_bytes(p, elem, heads, tokens, sequences, prefix_length, &need);
    if (rc != JQ_OK) {
        return rc;
    }
    if (!elem_ok(elem) || (elem != JQ_ELEM_F32 && elem != p->elem)) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention: %s queries on %s pages (FP32 queries, or the pages' type)", elem_name(elem), elem_name(p->elem));
    }
    if (heads > 65535 || q == nullptr || out == nullptr || strides == nullptr || tokens > 0x7fffffff || table_width > 0x7fffffff || prefix_length > 0x7fffffff ||
        !std::isfinite(scale * 1.5f)) {  // (times log2 e)
        return fail(JQ_ERR_INVALID, "jq_pages_attention: %lld rows of %d query heads, scale %g", (long long)tokens, heads, scale);
    }
    if (prefix_length > 0 && (prefix == nullptr || prefix_width * p->page_size < prefix_length)) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention: a prefix of %lld keys on %lld pages of %d", (long long)prefix_length, (long long)prefix_width, p->page_size);
    }
    if (workspace_bytes < need || (need > 0 && (workspace == nullptr || ((uintptr_t)workspace & 255) != 0))) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention: a workspace of %lld bytes at a 256-byte aligned address is needed, got %lld", (long long)need, (long long)workspace_bytes);
    }
    AttendArgs a = {};
    a.b = Batch{tables, table_stride, (int)table_width, starts, lengths, sequences, prefix, (int)prefix_length, (int)tokens};
    rc = check_batch(p, a.b, "jq_pages_attention");
    if (rc != JQ_OK || tokens == 0) {
        return rc;
    }
    a.q = q; a.out = out;
    a.qt = strides[0]; a.qh = strides[1]; a.ot = strides[2]; a.oh = strides[3];
    a.k_pages = p->k; a.v_pages = p->v;
    a.pages = p->pages;
    a.page_size = p->page_size; a.heads = heads; a.kv_heads = p->kv_heads; a.head_dim = p->head_dim;
    a.group = heads / p->kv_heads;
    while (1 << a.page_shift < p->page_size) {
        a.page_shift++;
    }
    const Plan plan = plan_of(p, elem, heads, tokens, sequences, prefix_length);
    uint8_t* const space = static_cast<uint8_t*>(workspace);
    auto floats = [&](int64_t at) { return reinterpret_cast<float*>(space + at); };
    auto pairs = [&](int64_t at) { return reinterpret_cast<float2*>(space + at); };
    const int ahead = prefix_length > 0 ? 1 : 0;
    const Work tile{plan.tile_own ? 0 : sequences, sequences + ahead, 7, 7, plan.tile_workers, TILE_OVER, floats(plan.tile_part), pairs(plan.tile_part_ml)};
    const Work few{0, sequences + (plan.tile_workers > 0 ? 0 : ahead), plan.rows == 8 ? 3 : 4, 4, plan.workers, STREAM_OVER, floats(plan.part), pairs(plan.part_ml)};
    a.own = plan.tile_own ? tile : few;
    a.pre = plan.tile_workers > 0 ? tile : few;
    a.wait_clocks = (long long)g_opt_wait_limit_us.load(std::memory_order_relaxed) * 2000;  // about 2 GHz
    a.whole = reinterpret_cast<float*>(space + plan.whole);
    a.whole_ml = reinterpret_cast<float2*>(space + plan.whole_ml);
    a.joined = prefix_length > 0 ? 1 : 0;
    a.stream_first = plan.tile_workers == 0 ? 1 : 0;
    a.found = reinterpret_cast<int2*>(space + plan.found);
    a.scale = scale;
    a.fill = fill != 0;
    const DeviceGuard guard(p->device);
    if (!guard.ok) {
        return fail(JQ_ERR_CUDA, "jq_pages_attention: device %d", p->device);
    }
    rc = status_word(&a.status);
    if (rc != JQ_OK) {
        return rc;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    if (elem == JQ_ELEM_F16) {
        return launch_attend<__half, __half>(p, a, plan, s);
    }
    if (elem == JQ_ELEM_BF16) {
        return launch_attend<__nv_bfloat16, __nv_bfloat16>(p, a, plan, s);
    }
    if (p->elem == JQ_ELEM_F16) {
        return launch_attend<float, __half>(p, a, plan, s);
    }
    return p->elem == JQ_ELEM_BF16 ? launch_attend<float, __nv_bfloat16>(p, a, plan, s) : launch_attend<float, float>(p, a, plan, s);
}

}  // extern "C"
