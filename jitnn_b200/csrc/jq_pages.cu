// A paged cache of keys and values, and the append to it: new queries and keys are rotated, keys and values rounded to the cache's type and stored on their sequences' pages,
// in one launch. [page][key/value head][slot][element]: what the attention of one key/value head reads of a page is one contiguous run.
// Measured: 8190 rows of 32 + 8 + 8 heads of 128, bf16, 33.2 us, 5.8 TB/s (88 % of a copy's); 16 rows of 64 + 8 + 8, FP32 into half precision, 3.1 us, most of it a launch.
#include <new>

#include "jq_rope.cuh"
#include "jq_tc.cuh"

namespace jq {
namespace {

struct AppendArgs {
    const void *q, *k, *v;
    void* q_out;
    int64_t qt, qh, kt, kh, vt, vh, ot, oh;  // strides of token and head, in elements
    int heads;
    void *k_pages, *v_pages;
    int64_t pages;
    int page_shift, kv_heads, head_dim;
    const float2* table;  // of the rotations, or null
    int half;
    int64_t positions;    // of that table
    Batch b;
    int fill;             // rows of q_out that belong to no sequence become zero
    int* status;
};

// A run rounded to the pages' type and stored.
template <typename Out, typename In, int V>
__device__ __forceinline__ void store_run(Out* to, const Run<In, V>& from) {
    if constexpr (sizeof(Out) == sizeof(In)) {
        from.store(reinterpret_cast<In*>(to));
    } else {
        float v[V];
        from.numbers(v);
        if constexpr (V == 1) {
            *to = from_float<Out>(v[0]);
        } else {  // four FP32 numbers, eight bytes
            *reinterpret_cast<uint2*>(to) = make_uint2(Run<Out, 8>::packed(v[0], v[1]), Run<Out, 8>::packed(v[2], v[3]));
        }
    }
}

// As the rotation's kernel: a thread has up to ITEMS units of 2 V elements of the same place in different heads of a row (query heads, key heads, value heads). The values
// are on their way while the row's sequence is looked for: every thread of the block asks whether the row is some sequence's, all at once, so that the chain of dependent
// loads is sequence, page, store. Bound by memory: everything is read once and written once; with few rows by that chain.
template <typename T, typename C, int V, bool INTERLEAVED, int ITEMS>
__global__ void __launch_bounds__(256, V == 1 ? 1 : 4) append_kernel(AppendArgs a) {
    __shared__ int found[2];  // sequence and own position
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched programmatically
    asm volatile("griddepcontrol.launch_dependents;");
    const int row = blockIdx.x, u = threadIdx.x, lanes = blockDim.y, tid = threadIdx.y * blockDim.x + u, threads = blockDim.x * lanes;
    if (tid == 0) {
        found[0] = -1;
    }
    const int pair_units = a.table != nullptr ? a.half / V : 0;
    const int all = a.heads + 2 * a.kv_heads, h0 = blockIdx.y * lanes * ITEMS + threadIdx.y;
    const int plain = 2 * V * u;  // a value head's unit is one run of 2 V elements
    int first = plain, second = plain + V;
    if (u < pair_units && !INTERLEAVED) {
        first = V * u;
        second = first + a.half;
    }
    Run<T, V> p[ITEMS], r[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int h = h0 + i * lanes;
        if (h < all) {
            const bool value = h >= a.heads + a.kv_heads, query = h < a.heads;
            const T* const x = static_cast<const T*>(query ? a.q : (value ? a.v : a.k)) + row * (query ? a.qt : (value ? a.vt : a.kt)) +
                               (query ? h : h - a.heads - (value ? a.kv_heads : 0)) * (query ? a.qh : (value ? a.vh : a.kh));
            p[i].load(x + (value ? plain : first));
            r[i].load(x + (value ? plain + V : second));
        }
    }
    __syncthreads();
    for (int s = tid; s < a.b.sequences; s += threads) {
        const int from = a.b.starts[s], to = a.b.starts[s + 1], length = a.b.lengths[s];
        if (row >= from && row < to) {
            found[0] = s;
            found[1] = length - (to - row);
        }
    }
    __syncthreads();
    const int seq = found[0], at = found[1];
    const bool real = seq >= 0 && at >= 0;  // (a negative position: more rows than keys, for the padding of a sequence that is not there)
    const int64_t pos = (int64_t)a.b.prefix_length + at;
    const bool turned = u < pair_units && real;
    Turns<V> turns;
    bool placed = real;
    if (turned) {
        if (pos < a.positions) {
            turns.load(a.table, pos, a.half, u * V, 1.0f);
        } else {
            turns.none();
            note_status(a.status, STATUS_POSITION);
        }
    }
    placed = placed && (a.table == nullptr || pos < a.positions);
    int64_t slot0 = -1;  // where the row's keys of head 0 go
    if (placed) {
        const int where = at >> a.page_shift;
        const int64_t page = where < a.b.table_width ? a.b.tables[seq * a.b.table_stride + where] : -1;
        if (page < 0 || page >= a.pages) {
            note_status(a.status, STATUS_PAGE);
        } else {
            slot0 = ((page * a.kv_heads) << a.page_shift) + (at & ((1 << a.page_shift) - 1));
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int h = h0 + i * lanes;
        if (h >= all) {
            continue;
        }
        const bool value = h >= a.heads + a.kv_heads;
        if (turned && !value) {
            turns.template turn<INTERLEAVED>(p[i], r[i]);
        }
        if (h < a.heads) {
            if (real || a.fill) {
                T* const y = static_cast<T*>(a.q_out) + row * a.ot + h * a.oh;
                if (!real) {
#pragma unroll
                    for (int j = 0; j < Run<T, V>::WORDS; j++) {
                        p[i].w[j] = r[i].w[j] = 0;
                    }
                }
                p[i].store(y + first);
                r[i].store(y + second);
            }
        } else if (slot0 >= 0) {
            const int head = h - a.heads - (value ? a.kv_heads : 0);
            C* const y = static_cast<C*>(value ? a.v_pages : a.k_pages) + (slot0 + ((int64_t)head << a.page_shift)) * a.head_dim;
            store_run<C, T, V>(y + (value ? plain : first), p[i]);
            store_run<C, T, V>(y + (value ? plain + V : second), r[i]);
        }
    }
}

template <typename T, typename C, int V, bool INTERLEAVED>
void launch_append(const AppendArgs& a, cudaStream_t s) {
    constexpr int ITEMS = 4;
    const HeadGrid g(a.head_dim, V, a.heads + 2 * a.kv_heads, ITEMS);
    launch_behind(append_kernel<T, C, V, INTERLEAVED, ITEMS>, dim3((unsigned)a.b.tokens, (unsigned)g.blocks), dim3((unsigned)g.units, (unsigned)g.lanes), s, a);
}

template <typename T, typename C>
void launch_append_types(const AppendArgs& a, bool wide, bool interleaved, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (wide) {
        interleaved ? launch_append<T, C, W, true>(a, s) : launch_append<T, C, W, false>(a, s);
    } else {
        interleaved ? launch_append<T, C, 1, true>(a, s) : launch_append<T, C, 1, false>(a, s);
    }
}

}  // namespace

int check_pages(const jq_pages* p, const char* who) {
    if (p == nullptr || p->magic != JQ_PAGES_MAGIC) {
        return fail(JQ_ERR_INVALID, "%s: not a live handle of pages", who);
    }
    return JQ_OK;
}

int check_batch(const jq_pages* p, const Batch& b, const char* who) {
    if (b.tables == nullptr || b.starts == nullptr || b.lengths == nullptr || b.sequences < 1 || b.table_width < 1) {
        return fail(JQ_ERR_INVALID, "%s: %d sequences of %d pages", who, b.sequences, b.table_width);
    }
    if (b.prefix_length < 0 || (int64_t)b.table_width * p->page_size + b.prefix_length > 0x7fffff00) {  // (a tile of keys behind the last still has a number)
        return fail(JQ_ERR_INVALID, "%s: a prefix of %d keys and %d pages of %d: positions are below 2^31 - 256", who, b.prefix_length, b.table_width, p->page_size);
    }
    return JQ_OK;
}

}  // namespace jq

using namespace jq;

extern "C" {

JQ_API int jq_pages_create(int device, int elem, int64_t pages, int page_size, int kv_heads, int head_dim, void* k, void* v, jq_pages** out) {
    if (out == nullptr) {
        return fail(JQ_ERR_INVALID, "jq_pages_create: null result pointer");
    }
    *out = nullptr;
    if (!elem_ok(elem)) {
        return fail(JQ_ERR_INVALID, "jq_pages_create: element type %d", elem);
    }
    if (pages < 1 || pages > 0x7fffffff / (kv_heads > 0 ? kv_heads : 1) || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) {
        return fail(JQ_ERR_INVALID, "jq_pages_create: %lld pages of %d keys (a power of two from 16 to 1024)", (long long)pages, page_size);
    }
    if (kv_heads < 1 || kv_heads > 1024 || head_dim < 2 || head_dim % 2 != 0 || head_dim > 256) {
        return fail(JQ_ERR_INVALID, "jq_pages_create: %d heads (1 to 1024) of %d elements (an even number up to 256)", kv_heads, head_dim);
    }
    if (k == nullptr || v == nullptr || ((uintptr_t)k & 15) != 0 || ((uintptr_t)v & 15) != 0) {
        return fail(JQ_ERR_INVALID, "jq_pages_create: keys and values at 16-byte aligned addresses are needed");
    }
    int count = 0;
    JQ_CUDA(cudaGetDeviceCount(&count));
    if (device < 0 || device >= count) {
        return fail(JQ_ERR_INVALID, "jq_pages_create: device %d of %d", device, count);
    }
    const DeviceGuard guard(device);
    if (!guard.ok) {
        return fail(JQ_ERR_CUDA, "jq_pages_create: device %d", device);
    }
    int* word = nullptr;
    const int rc = status_word(&word);  // made here, so that no launch has to
    if (rc != JQ_OK) {
        return rc;
    }
    jq_pages* p = new (std::nothrow) jq_pages();
    if (p == nullptr) {
        return fail(JQ_ERR_OOM, "jq_pages_create: out of host memory");
    }
    *p = jq_pages{JQ_PAGES_MAGIC, device, elem, page_size, kv_heads, head_dim, pages, k, v, {}, {}};
    if (elem != JQ_ELEM_F32 && (head_dim == 64 || head_dim == 128)) {
        const EncodeTiledFn encode = encode_tiled();
        bool made = encode != nullptr;
        for (int i = 0; i < 2 && made; i++) {
            const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)page_size, (cuuint64_t)pages * kv_heads};
            const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)page_size * head_dim * 2};
            const cuuint32_t box[3] = {64, (cuuint32_t)(page_size < BOX_KEYS ? page_size : BOX_KEYS), 1}, steps[3] = {1, 1, 1};
            made = encode(i == 0 ? &p->k_map : &p->v_map, elem == JQ_ELEM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, i == 0 ? k : v, dims,
                          strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
        }
        if (!made) {
            delete p;
            return fail(JQ_ERR_CUDA, "jq_pages_create: no tensor map of %lld pages", (long long)pages);
        }
    }
    *out = p;
    return JQ_OK;
}

JQ_API int jq_pages_free(jq_pages* p) {
    if (p == nullptr) {
        return JQ_OK;
    }
    const int rc = check_pages(p, "jq_pages_free");
    if (rc == JQ_OK) {
        p->magic = 0;
        delete p;
    }
    return rc;
}

JQ_API int jq_pages_append(const jq_pages* p, const jq_rope* rope, int elem, int heads, const void* q, const void* k, const void* v, void* q_out, const int64_t* strides,
                           int64_t tokens, const int32_t* tables, int64_t table_stride, int64_t table_width, const int32_t* starts, const int32_t* lengths, int sequences,
                           int64_t prefix_length, int fill, void* stream) {
    int rc = check_pages(p, "jq_pages_append");
    if (rc == JQ_OK && rope != nullptr) {
        rc = check_rope(rope, "jq_pages_append");
    }
    if (rc != JQ_OK) {
        return rc;
    }
    if (!elem_ok(elem) || (elem != JQ_ELEM_F32 && elem != p->elem)) {
        return fail(JQ_ERR_INVALID, "jq_pages_append: %s rows into %s pages (FP32 rows, or the pages' type)", elem_name(elem), elem_name(p->elem));
    }
    if (heads < 0 || heads > 65535 || (heads > 0 && (q == nullptr || q_out == nullptr)) || k == nullptr || v == nullptr || strides == nullptr || tokens < 0 ||
        tokens > 0x7fffffff || table_width > 0x7fffffff || prefix_length > 0x7fffffff) {
        return fail(JQ_ERR_INVALID, "jq_pages_append: %lld rows of %d query heads", (long long)tokens, heads);
    }
    if (rope != nullptr && (rope->device != p->device || rope->dim > p->head_dim)) {
        return fail(JQ_ERR_INVALID, "jq_pages_append: a rotation of %d elements on device %d, heads of %d on device %d", rope->dim, rope->device, p->head_dim, p->device);
    }
    AppendArgs a = {};
    a.b = Batch{tables, table_stride, (int)table_width, starts, lengths, sequences, nullptr, (int)prefix_length, (int)tokens};
    rc = check_batch(p, a.b, "jq_pages_append");
    if (rc != JQ_OK || tokens == 0) {
        return rc;
    }
    a.q = q; a.k = k; a.v = v; a.q_out = q_out;
    a.qt = strides[0]; a.qh = strides[1]; a.kt = strides[2]; a.kh = strides[3]; a.vt = strides[4]; a.vh = strides[5]; a.ot = strides[6]; a.oh = strides[7];
    a.heads = heads;
    a.k_pages = p->k; a.v_pages = p->v;
    a.pages = p->pages;
    a.page_shift = 31 - __builtin_clz((unsigned)p->page_size); a.kv_heads = p->kv_heads; a.head_dim = p->head_dim;
    a.fill = fill != 0;
    const int width = 16 / elem_bytes(elem);
    bool wide = p->head_dim % (2 * width) == 0;
    if (rope != nullptr) {
        a.table = rope->table;
        a.half = rope->dim / 2;
        a.positions = rope->positions;
        wide = wide && rope->dim % (2 * width) == 0;
    }
    const void* const at[4] = {k, v, heads > 0 ? q : k, heads > 0 ? q_out : k};
    for (int i = 0; i < 4; i++) {
        wide = wide && ((uintptr_t)at[i] & 15) == 0;
    }
    for (int i = heads > 0 ? 0 : 2; i < (heads > 0 ? 8 : 6); i++) {
        wide = wide && strides[i] % width == 0;
    }
    const DeviceGuard guard(p->device);
    if (!guard.ok) {
        return fail(JQ_ERR_CUDA, "jq_pages_append: device %d", p->device);
    }
    rc = status_word(&a.status);
    if (rc != JQ_OK) {
        return rc;
    }
    const bool interleaved = rope != nullptr && rope->interleaved != 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (elem == JQ_ELEM_F16) {
        launch_append_types<__half, __half>(a, wide, interleaved, s);
    } else if (elem == JQ_ELEM_BF16) {
        launch_append_types<__nv_bfloat16, __nv_bfloat16>(a, wide, interleaved, s);
    } else if (p->elem == JQ_ELEM_F16) {
        launch_append_types<float, __half>(a, wide, interleaved, s);
    } else if (p->elem == JQ_ELEM_BF16) {
        launch_append_types<float, __nv_bfloat16>(a, wide, interleaved, s);
    } else {
        launch_append_types<float, float>(a, wide, interleaved, s);
    }
    count_launch();
    return check_launch("append_kernel");
}

}  // extern "C"
