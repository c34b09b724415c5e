// Attention over a paged cache for a batch whose sequences share a prefix: row r of sequence s, at the own position t, sees the prefix and the keys 0 .. t of its sequence,
//     o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m),
// in one pass over the keys with a running maximum and sum (ops/FlashAttention.java:538-626 of the reference, which has neither cache nor pages). Sums are FP32.
#include <cmath>

#include "jq_pages_attention.cuh"
#include "jq_pages_join.cuh"
#include "jq_pages_stream.cuh"

namespace jq {
namespace {

// Other head sizes than the stream kernel's: one thread block per row and query head. 128 keys at a time, a thread has a key's score, then elements of the output.
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
    const int own = found[1] >= 0 ? found[1] + 1 : 0, keys = a.b.prefix_length + own;
    const C* const kp = static_cast<const C*>(a.k_pages);
    const C* const vp = static_cast<const C*>(a.v_pages);
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int j0 = 0; j0 < keys; j0 += 128) {
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

struct Plan {
    int rows = 0;   // of a block; 0: the row kernel
    int ctas = 0;
    int64_t part = 0, part_ml = 0, whole = 0, whole_ml = 0, bytes = 0;  // where in the workspace
};

// How many thread blocks of an instance an SM holds (registers), and with it the share of the work that each gets.
template <typename C, int HD, int NB>
constexpr int resident() {
    return HD * sizeof(C) >= 512 ? 2 : 3;
}

int resident_of(int elem, int head_dim) { return head_dim * elem_bytes(elem) >= 512 ? 2 : 3; }

Plan plan_of(const jq_pages* p, int heads, int64_t tokens, int64_t sequences, int64_t prefix_length) {
    Plan plan;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) {
        return plan;
    }
    const int64_t group = heads / p->kv_heads, rows = (tokens + sequences - 1) / sequences * group;
    plan.rows = rows <= 8 || p->head_dim == 256 ? 8 : 16;
    plan.ctas = 148 * resident_of(p->elem, p->head_dim);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    plan.part = take((int64_t)2 * plan.ctas * plan.rows * p->head_dim * 4);
    plan.part_ml = take((int64_t)2 * plan.ctas * plan.rows * 8);
    if (prefix_length > 0) {
        plan.whole = take(2 * tokens * heads * p->head_dim * 4);
        plan.whole_ml = take(2 * tokens * heads * 8);
    }
    plan.bytes = at;
    return plan;
}

template <typename T, typename C, int HD, int NB>
int launch_stream(const AttendArgs& a, cudaStream_t s) {
    constexpr int smem = pages::Stream<T, C, HD, NB>::SMEM, RESIDENT = resident<C, HD, NB>();
    auto kernel = pages::attend_stream_kernel<T, C, HD, NB, RESIDENT>;
    static std::atomic<uint64_t> configured{0};  // the opt-in for large dynamic shared memory is per device
    int dev = 0;
    JQ_CUDA(cudaGetDevice(&dev));
    if (smem > 48 * 1024 && (configured.load(std::memory_order_relaxed) >> (dev & 63) & 1) == 0) {
        JQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        configured.fetch_or((uint64_t)1 << (dev & 63));
    }
    kernel<<<a.own.ctas, pages::STREAM_THREADS, smem, s>>>(a);
    count_launch();
    int rc = check_launch("attend_stream_kernel");
    if (rc != JQ_OK) {
        return rc;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)a.b.tokens, (unsigned)((a.heads + pages::JOIN_HEADS - 1) / pages::JOIN_HEADS));
    cfg.blockDim = dim3(pages::JOIN_THREADS);
    cfg.stream = s;
    JQ_CUDA(cudaLaunchKernelEx(&cfg, pages::attend_join_kernel<T, HD>, a));
    count_launch();
    return JQ_OK;
}

template <typename T, typename C>
int launch_attend(const AttendArgs& a, const Plan& plan, cudaStream_t s) {
    if (plan.rows == 0) {
        attend_row_kernel<T, C><<<dim3((unsigned)a.b.tokens, (unsigned)a.heads), 128, 0, s>>>(a);
        count_launch();
        return check_launch("attend_row_kernel");
    }
    if (a.head_dim == 64) {
        return plan.rows == 8 ? launch_stream<T, C, 64, 1>(a, s) : launch_stream<T, C, 64, 2>(a, s);
    }
    if (a.head_dim == 128) {
        return plan.rows == 8 ? launch_stream<T, C, 128, 1>(a, s) : launch_stream<T, C, 128, 2>(a, s);
    }
    return launch_stream<T, C, 256, 1>(a, s);
}

}  // namespace
}  // namespace jq

using namespace jq;

extern "C" {

JQ_API int jq_pages_attention_bytes(const jq_pages* p, int heads, int64_t tokens, int64_t sequences, int64_t prefix_length, int64_t* nbytes) {
    const int rc = check_pages(p, "jq_pages_attention_bytes");
    if (rc != JQ_OK) {
        return rc;
    }
    if (nbytes == nullptr || heads < 1 || heads % p->kv_heads != 0 || tokens < 0 || tokens > 0x7fffffff || sequences < 1 || prefix_length < 0) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention: %lld rows of %lld sequences, %d heads on %d key/value heads", (long long)tokens, (long long)sequences, heads,
                    p->kv_heads);
    }
    *nbytes = plan_of(p, heads, tokens, sequences, prefix_length).bytes;
    return JQ_OK;
}

JQ_API int jq_pages_attention(const jq_pages* p, int elem, int heads, const void* q, void* out, const int64_t* strides, int64_t tokens, const int32_t* tables,
                              int64_t table_stride, int64_t table_width, const int32_t* starts, const int32_t* lengths, int sequences, const int32_t* prefix,
                              int64_t prefix_width, int64_t prefix_length, float scale, int fill, void* workspace, int64_t workspace_bytes, void* stream) {
    int64_t need = 0;
    int rc = jq_pages_attention_bytes(p, heads, tokens, sequences, prefix_length, &need);
    if (rc != JQ_OK) {
        return rc;
    }
    if (!elem_ok(elem) || (elem != JQ_ELEM_F32 && elem != p->elem)) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention: %s queries on %s pages (FP32 queries, or the pages' type)", elem_name(elem), elem_name(p->elem));
    }
    if (heads > 65535 || q == nullptr || out == nullptr || strides == nullptr || tokens > 0x7fffffff || table_width > 0x7fffffff || prefix_length > 0x7fffffff ||
        !std::isfinite(scale)) {
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
    const Plan plan = plan_of(p, heads, tokens, sequences, prefix_length);
    uint8_t* const space = static_cast<uint8_t*>(workspace);
    a.own = Work{0, sequences + (prefix_length > 0 ? 1 : 0), plan.rows == 8 ? 3 : 4, 4, plan.ctas, pages::STREAM_WARPS, reinterpret_cast<float*>(space + plan.part),
                 reinterpret_cast<float2*>(space + plan.part_ml)};
    a.pre = a.own;
    a.whole = reinterpret_cast<float*>(space + plan.whole);
    a.whole_ml = reinterpret_cast<float2*>(space + plan.whole_ml);
    a.joined = prefix_length > 0 ? 1 : 0;
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
        return launch_attend<__half, __half>(a, plan, s);
    }
    if (elem == JQ_ELEM_BF16) {
        return launch_attend<__nv_bfloat16, __nv_bfloat16>(a, plan, s);
    }
    if (p->elem == JQ_ELEM_F16) {
        return launch_attend<float, __half>(a, plan, s);
    }
    return p->elem == JQ_ELEM_BF16 ? launch_attend<float, __nv_bfloat16>(a, plan, s) : launch_attend<float, float>(a, plan, s);
}

}  // extern "C"
