// Attention over a paged cache for a batch whose sequences share a prefix: row r of sequence s, at the own position t, sees the prefix and the keys 0 .. t of its sequence,
//     o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m),
// in one pass over the keys with a running maximum and sum (ops/FlashAttention.java:538-626 of the reference, which has neither cache nor pages). Sums are FP32.
#include <cmath>

#include "jq_pages.cuh"

namespace jq {
namespace {

struct AttendArgs {
    const void* q;
    void* out;
    int64_t qt, qh, ot, oh;  // strides of token and head, in elements
    const void *k_pages, *v_pages;
    int64_t pages;
    int page_size, heads, kv_heads, head_dim;
    Batch b;
    float scale;
    int fill;
    int* status;
};

// One thread block per row and query head: 128 keys at a time, a thread has a key's score, then elements of the output.
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
    bool any = false;
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
        any = __syncthreads_or(at >= 0) || any;
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
            out[tid + 128 * n] = from_float<T>(any ? acc[n] / l : 0.0f);  // (a row that sees no key at all: zero)
        }
    }
}

template <typename T, typename C>
void launch_attend(const AttendArgs& a, cudaStream_t s) {
    attend_row_kernel<T, C><<<dim3((unsigned)a.b.tokens, (unsigned)a.heads), 128, 0, s>>>(a);
}

}  // namespace
}  // namespace jq

using namespace jq;

extern "C" {

JQ_API int jq_pages_attention_bytes(const jq_pages* p, int heads, int64_t tokens, int64_t prefix_length, int64_t* nbytes) {
    const int rc = check_pages(p, "jq_pages_attention_bytes");
    if (rc != JQ_OK) {
        return rc;
    }
    if (nbytes == nullptr || heads < 1 || heads % p->kv_heads != 0 || tokens < 0 || prefix_length < 0) {
        return fail(JQ_ERR_INVALID, "jq_pages_attention_bytes: %lld rows of %d heads on %d key/value heads", (long long)tokens, heads, p->kv_heads);
    }
    *nbytes = 0;
    return JQ_OK;
}

JQ_API int jq_pages_attention(const jq_pages* p, int elem, int heads, const void* q, void* out, const int64_t* strides, int64_t tokens, const int32_t* tables,
                              int64_t table_stride, int64_t table_width, const int32_t* starts, const int32_t* lengths, int sequences, const int32_t* prefix,
                              int64_t prefix_width, int64_t prefix_length, float scale, int fill, void* workspace, int64_t workspace_bytes, void* stream) {
    int64_t need = 0;
    int rc = jq_pages_attention_bytes(p, heads, tokens, prefix_length, &need);
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
        launch_attend<__half, __half>(a, s);
    } else if (elem == JQ_ELEM_BF16) {
        launch_attend<__nv_bfloat16, __nv_bfloat16>(a, s);
    } else if (p->elem == JQ_ELEM_F16) {
        launch_attend<float, __half>(a, s);
    } else if (p->elem == JQ_ELEM_BF16) {
        launch_attend<float, __nv_bfloat16>(a, s);
    } else {
        launch_attend<float, float>(a, s);
    }
    count_launch();
    return check_launch("attend_row_kernel");
}

}  // extern "C"
