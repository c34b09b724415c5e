// Rotary positions: tables of cosines and sines, with the frequencies rescaled for long contexts (ops/Rope.java:84-149 of the reference; its RopeScaling.linear and
// llama3, and YaRN of Peng et al. 2023), and the rotation of queries and keys or of their gradients.
//
// Pair i of a head, (x[i], x[i + dim/2]) or interleaved (x[2i], x[2i + 1]), is turned by the angle position * f_i. The turn is orthogonal, so the gradient is turned by
// the negative angle; a magnitude (YaRN) stands in the table and multiplies both. Angles, cosines and sines are made in double once, for position 10^5 a float angle is off
// by 4e-3. Elements behind dim are copied.
#include <cmath>
#include <new>

#include "jq_rope.cuh"

namespace jq {
namespace {

__global__ void __launch_bounds__(256) rope_table_kernel(float2* table, const double* freqs, int half, int64_t positions, double magnitude) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < positions * half) {
        double s, c;
        sincos((double)(i / half) * freqs[i % half], &s, &c);
        table[i] = make_float2((float)(c * magnitude), (float)(s * magnitude));
    }
}

struct RopeTensor {
    const void* x;
    void* y;
    int heads;
    int64_t xb, xt, xh, yb, yt, yh;  // strides of batch, token and head, in elements
};
struct RopeArgs {
    RopeTensor t[2];
    const float2* table;
    int half, head_dim;
    int64_t positions;           // of the table
    int64_t seq;                 // tokens of a batch entry
    const void* pos;
    int pos_bytes;               // 4 or 8; 0: offset + token
    int64_t pos_b, pos_t, offset;
    float sign;
    int* status;
};

// A thread has up to ITEMS units of 2 V elements, of the same place in different heads of one token: their loads are on their way together, and one read of the table
// serves them. Units of a head: the pairs (2 V elements each), then what is only copied. Bound by memory: x read once, y written once.
// Measured: 4096 tokens of 64 + 8 heads of 128, bf16, 27.5 us, 5.5 TB/s (84 % of a copy's); one token of 32 + 32, FP32, 2.8 us, the time of a launch.
template <typename T, int V, bool INTERLEAVED, int ITEMS>
__global__ void __launch_bounds__(256, V == 1 ? 1 : 4) rope_kernel(RopeArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched programmatically
    asm volatile("griddepcontrol.launch_dependents;");
    const int pair_units = a.half / V, u = threadIdx.x, lanes = blockDim.y;
    const uint32_t token = blockIdx.x, b = token / (uint32_t)a.seq, t = token - b * (uint32_t)a.seq;
    const int heads = a.t[0].heads + a.t[1].heads;
    const int h0 = blockIdx.y * lanes * ITEMS + threadIdx.y;
    int first, second;  // where the unit's two runs of V elements start
    if (u < pair_units) {
        first = INTERLEAVED ? 2 * V * u : V * u;
        second = INTERLEAVED ? first + V : first + a.half;
    } else {
        first = 2 * V * u;
        second = first + V;
    }
    Run<T, V> p[ITEMS], q[ITEMS];
    T* y[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int h = h0 + i * lanes;
        y[i] = nullptr;
        if (h < heads) {
            const RopeTensor& w = h < a.t[0].heads ? a.t[0] : a.t[1];
            const int head = h < a.t[0].heads ? h : h - a.t[0].heads;
            const T* const x = static_cast<const T*>(w.x) + b * w.xb + t * w.xt + head * w.xh;
            T* const to = static_cast<T*>(w.y) + b * w.yb + t * w.yt + head * w.yh;
            if (u >= pair_units && to == x) {
                continue;  // in place
            }
            y[i] = to;
            p[i].load(x + first);
            q[i].load(x + second);
        }
    }
    if (u < pair_units) {
        int64_t pos = a.offset + t;
        if (a.pos_bytes == 4) {
            pos = static_cast<const int*>(a.pos)[b * a.pos_b + t * a.pos_t];
        } else if (a.pos_bytes == 8) {
            pos = static_cast<const int64_t*>(a.pos)[b * a.pos_b + t * a.pos_t];
        }
        Turns<V> turns;
        if (pos >= 0 && pos < a.positions) {
            turns.load(a.table, pos, a.half, u * V, a.sign);
        } else {  // no such position: NaN, so that it does not pass for a result
            turns.none();
            note_status(a.status, STATUS_POSITION);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            if (y[i] != nullptr) {
                turns.template turn<INTERLEAVED>(p[i], q[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        if (y[i] != nullptr) {
            p[i].store(y[i] + first);
            q[i].store(y[i] + second);
        }
    }
}

template <typename T, int V, bool INTERLEAVED>
void launch_rope(const RopeArgs& a, int64_t tokens, cudaStream_t s) {
    constexpr int ITEMS = 4;
    const HeadGrid g(a.head_dim, V, a.t[0].heads + a.t[1].heads, ITEMS);
    launch_behind(rope_kernel<T, V, INTERLEAVED, ITEMS>, dim3((unsigned)tokens, (unsigned)g.blocks), dim3((unsigned)g.units, (unsigned)g.lanes), s, a);
}

template <typename T>
void launch_rope_type(const RopeArgs& a, bool wide, bool interleaved, int64_t tokens, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (wide) {
        interleaved ? launch_rope<T, W, true>(a, tokens, s) : launch_rope<T, W, false>(a, tokens, s);
    } else {
        interleaved ? launch_rope<T, 1, true>(a, tokens, s) : launch_rope<T, 1, false>(a, tokens, s);
    }
}

}  // namespace

int check_rope(const jq_rope* r, const char* who) {
    if (r == nullptr || r->magic != JQ_ROPE_MAGIC) {
        return fail(JQ_ERR_INVALID, "%s: not a live rotation handle", who);
    }
    return JQ_OK;
}

}  // namespace jq

using namespace jq;

extern "C" {

JQ_API int jq_rope_frequencies(int dim, double base, int scaling, const double* params, double* freqs, double* magnitude) {
    if (dim < 2 || dim % 2 != 0 || !(base > 1.0) || !std::isfinite(base) || freqs == nullptr || magnitude == nullptr) {
        return fail(JQ_ERR_INVALID, "jq_rope_frequencies: %d elements (an even number), base %g (above 1)", dim, base);
    }
    if (scaling < JQ_ROPE_NONE || scaling > JQ_ROPE_YARN || (scaling != JQ_ROPE_NONE && params == nullptr)) {
        return fail(JQ_ERR_INVALID, "jq_rope_frequencies: scaling %d", scaling);
    }
    const double factor = scaling == JQ_ROPE_NONE ? 1.0 : params[0], two_pi = 6.283185307179586476925286766559;
    if (!(factor >= 1.0) || !std::isfinite(factor)) {
        return fail(JQ_ERR_INVALID, "jq_rope_frequencies: factor %g (at least 1)", factor);
    }
    const int half = dim / 2;
    *magnitude = 1.0;
    double first = 0.0, last = 0.0;
    if (scaling == JQ_ROPE_LLAMA3 && !(params[1] > 0.0 && params[2] > params[1] && params[3] > 0.0 && std::isfinite(params[2]) && std::isfinite(params[3]))) {
        return fail(JQ_ERR_INVALID, "jq_rope_frequencies: low %g, high %g, context %g (0 < low < high, a positive context)", params[1], params[2], params[3]);
    }
    if (scaling == JQ_ROPE_YARN) {
        const double context = params[1], fast = params[2], slow = params[3], given = params[4];
        if (!(context > 0.0 && slow > 0.0 && fast > slow && given >= 0.0 && std::isfinite(context) && std::isfinite(fast) && std::isfinite(given))) {
            return fail(JQ_ERR_INVALID, "jq_rope_frequencies: context %g, turns %g and %g, magnitude %g (a positive context, fast > slow > 0)", context, fast, slow, given);
        }
        // the pairs that make `fast` and `slow` turns in the trained context: in front of the first nothing changes, behind the last everything is interpolated
        auto pair_with = [&](double turns) { return dim * std::log(context / (turns * two_pi)) / (2.0 * std::log(base)); };
        first = std::floor(pair_with(fast));
        last = std::ceil(pair_with(slow));
        first = first < 0.0 ? 0.0 : first;
        last = last > dim - 1 ? dim - 1 : last;
        *magnitude = given > 0.0 ? given : 0.1 * std::log(factor) + 1.0;
    }
    for (int i = 0; i < half; i++) {
        const double f = std::pow(base, -2.0 * i / dim);
        double keep = 1.0;  // how much of the frequency stays as it was trained
        if (scaling == JQ_ROPE_LINEAR) {
            keep = 0.0;
        } else if (scaling == JQ_ROPE_LLAMA3) {
            keep = (params[3] * f / two_pi - params[1]) / (params[2] - params[1]);
        } else if (scaling == JQ_ROPE_YARN) {
            keep = 1.0 - (i - first) / (last - first > 0.001 ? last - first : 0.001);
        }
        keep = keep < 0.0 ? 0.0 : (keep > 1.0 ? 1.0 : keep);
        freqs[i] = f * (keep + (1.0 - keep) / factor);
    }
    return JQ_OK;
}

JQ_API int jq_rope_create(int device, int64_t positions, int dim, const double* freqs, double magnitude, int interleaved, jq_rope** out) {
    if (out == nullptr) {
        return fail(JQ_ERR_INVALID, "jq_rope_create: null result pointer");
    }
    *out = nullptr;
    if (positions < 1 || positions > (int64_t)1 << 24 || dim < 2 || dim % 2 != 0 || dim > 512 || freqs == nullptr || !std::isfinite(magnitude)) {
        return fail(JQ_ERR_INVALID, "jq_rope_create: %lld positions (1 to 2^24) of %d elements (an even number up to 512)", (long long)positions, dim);
    }
    for (int i = 0; i < dim / 2; i++) {
        if (!std::isfinite(freqs[i])) {
            return fail(JQ_ERR_INVALID, "jq_rope_create: frequency %d is %g", i, freqs[i]);
        }
    }
    int count = 0;
    JQ_CUDA(cudaGetDeviceCount(&count));
    if (device < 0 || device >= count) {
        return fail(JQ_ERR_INVALID, "jq_rope_create: device %d of %d", device, count);
    }
    const DeviceGuard guard(device);
    if (!guard.ok) {
        return fail(JQ_ERR_CUDA, "jq_rope_create: device %d", device);
    }
    int* word = nullptr;
    const int rc = status_word(&word);  // made here, so that no launch has to
    if (rc != JQ_OK) {
        return rc;
    }
    const int half = dim / 2;
    float2* table = nullptr;
    double* f = nullptr;
    cudaError_t e = cudaMalloc(&table, (size_t)positions * half * sizeof(float2));
    if (e == cudaSuccess) e = cudaMalloc(&f, half * sizeof(double));
    if (e == cudaSuccess) e = cudaMemcpy(f, freqs, half * sizeof(double), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) {
        rope_table_kernel<<<(unsigned)((positions * half + 255) / 256), 256>>>(table, f, half, positions, magnitude);
        count_launch();
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // callers use the table from any stream
    cudaFree(f);
    jq_rope* r = e == cudaSuccess ? new (std::nothrow) jq_rope() : nullptr;
    if (r == nullptr) {
        cudaFree(table);
        return e == cudaSuccess ? fail(JQ_ERR_OOM, "jq_rope_create: out of host memory") : cuda_fail(e, "jq_rope_create");
    }
    r->magic = JQ_ROPE_MAGIC;
    r->device = device;
    r->dim = dim;
    r->interleaved = interleaved != 0;
    r->positions = positions;
    r->table = table;
    *out = r;
    return JQ_OK;
}

JQ_API int jq_rope_free(jq_rope* r) {
    if (r == nullptr) {
        return JQ_OK;
    }
    const int rc = check_rope(r, "jq_rope_free");
    if (rc != JQ_OK) {
        return rc;
    }
    const DeviceGuard guard(r->device);
    const cudaError_t e = cudaFree(r->table);
    r->magic = 0;
    delete r;
    return e == cudaSuccess ? JQ_OK : cuda_fail(e, "jq_rope_free");
}

JQ_API int jq_rope_apply(const jq_rope* r, int elem, int count, const void* const* x, void* const* y, const int* heads, int head_dim, const int64_t* strides, int64_t batch,
                         int64_t seq, const void* positions, int position_bytes, int64_t position_batch_stride, int64_t position_stride, int64_t offset, int inverse,
                         void* stream) {
    const int rc = check_rope(r, "jq_rope_apply");
    if (rc != JQ_OK) {
        return rc;
    }
    if (!elem_ok(elem) || count < 1 || count > 2 || x == nullptr || y == nullptr || heads == nullptr || strides == nullptr || batch < 0 || seq < 0) {
        return fail(JQ_ERR_INVALID, "jq_rope_apply: element type %d, %d tensors (1 or 2), %lld x %lld tokens", elem, count, (long long)batch, (long long)seq);
    }
    if (head_dim < r->dim || head_dim % 2 != 0 || head_dim > 512) {
        return fail(JQ_ERR_INVALID, "jq_rope_apply: heads of %d elements for a rotation of %d (even, up to 512)", head_dim, r->dim);
    }
    if (positions != nullptr && position_bytes != 4 && position_bytes != 8) {
        return fail(JQ_ERR_INVALID, "jq_rope_apply: positions of %d bytes (4 or 8)", position_bytes);
    }
    if (positions == nullptr && (offset < 0 || offset > r->positions - seq)) {
        return fail(JQ_ERR_INVALID, "jq_rope_apply: positions %lld to %lld, the table has %lld", (long long)offset, (long long)(offset + seq - 1), (long long)r->positions);
    }
    RopeArgs a = {};
    const int width = 16 / elem_bytes(elem);
    bool wide = head_dim % (2 * width) == 0 && r->dim % (2 * width) == 0;
    for (int i = 0; i < count; i++) {
        const int64_t* st = strides + 6 * i;
        if (heads[i] < 1 || heads[i] > 65535 || x[i] == nullptr || y[i] == nullptr) {
            return fail(JQ_ERR_INVALID, "jq_rope_apply: tensor %d of %d heads", i, heads[i]);
        }
        a.t[i] = RopeTensor{x[i], y[i], heads[i], st[0], st[1], st[2], st[3], st[4], st[5]};
        wide = wide && ((uintptr_t)x[i] & 15) == 0 && ((uintptr_t)y[i] & 15) == 0;
        for (int j = 0; j < 6; j++) {
            wide = wide && st[j] % width == 0;
        }
    }
    if (batch > 0 && seq > (((int64_t)1 << 31) - 1) / batch) {
        return fail(JQ_ERR_INVALID, "jq_rope_apply: %lld x %lld tokens in one call", (long long)batch, (long long)seq);
    }
    if (batch == 0 || seq == 0) {
        return JQ_OK;
    }
    const DeviceGuard guard(r->device);
    if (!guard.ok) {
        return fail(JQ_ERR_CUDA, "jq_rope_apply: device %d", r->device);
    }
    a.table = r->table;
    a.half = r->dim / 2;
    a.head_dim = head_dim;
    a.positions = r->positions;
    a.seq = seq;
    a.pos = positions;
    a.pos_bytes = positions == nullptr ? 0 : position_bytes;
    a.pos_b = position_batch_stride;
    a.pos_t = position_stride;
    a.offset = offset;
    a.sign = inverse != 0 ? -1.0f : 1.0f;
    const int status = status_word(&a.status);
    if (status != JQ_OK) {
        return status;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    if (elem == JQ_ELEM_F32) {
        launch_rope_type<float>(a, wide, r->interleaved != 0, batch * seq, s);
    } else if (elem == JQ_ELEM_F16) {
        launch_rope_type<__half>(a, wide, r->interleaved != 0, batch * seq, s);
    } else {
        launch_rope_type<__nv_bfloat16>(a, wide, r->interleaved != 0, batch * seq, s);
    }
    count_launch();
    return check_launch("rope_kernel");
}

}  // extern "C"
