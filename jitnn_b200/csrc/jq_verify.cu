// Verification of drafted tokens (speculative sampling, Leviathan et al. 2023, Chen et al. 2023): with p_i the target's distribution behind draft i, q_i the drafter's (all on
// the draft, where it gives none) and u given uniform numbers, draft x_i is kept while
//     u_i q_i(x_i) < p_i(x_i),
// and one more token comes by the inverse distribution function at u_K: behind the first refused draft j from max(p_j - q_j, 0) over its sum, behind the last draft from p_K.
// At temperature 0 the likeliest token (the first of equal ones) takes the place of both.
//
// The results are whole numbers that may not depend on how the work is cut, so everything is computed in double: the products u q of two floats are exact, sums of a
// vocabulary's probabilities are good to 1e-14, and a cut in another place moves a token with a chance of about 1e-10.
//
// Logits: stats_kernel takes the maximum and the sum of exponentials of chunks of all rows that count, bound by reading them. choose_kernel is one cluster per sequence:
// it joins the chunks, finds the row, adds up the row's weights (its second reading, from L2) and looks the token up.
#include <cooperative_groups.h>

#include <cmath>

#include "jq_pages.cuh"

namespace jq {
namespace {

namespace cg = cooperative_groups;

constexpr int STATS_THREADS = 256, HELD = 32, CHUNK_MOST = STATS_THREADS * HELD;  // a thread's values of a chunk stay in registers
constexpr int CHOOSE_THREADS = 512, CHOOSE_WARPS = CHOOSE_THREADS / 32, CLUSTER = 8;

struct Stat {
    double sum;  // of exp((x - top) / temperature)
    float top;
    int at;      // where top is first
};

struct VerifyArgs {
    const void* target;
    int64_t tb, tr;  // strides of sequence and row, in elements
    const float* q;
    int64_t qb, qr;
    const int* drafts;  // [sequences][drafts]
    const float* u;     // [sequences][drafts + 1]
    const int* counts;
    int sequences, drafts_most, vocab;
    double inverse;     // of the temperature
    int form;           // GREEDY, LOGITS, PROBABILITIES
    int *accepted, *tokens;
    Stat* stats;        // [row][chunks]
    int chunk, chunks;
    int* status;
};
enum { GREEDY, LOGITS, PROBABILITIES };

__device__ __forceinline__ int count_of(const VerifyArgs& a, int b) {
    const int n = a.counts != nullptr ? a.counts[b] : a.drafts_most;
    return n < 0 ? 0 : (n > a.drafts_most ? a.drafts_most : n);
}

__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <typename T>
__global__ void __launch_bounds__(STATS_THREADS) stats_kernel(VerifyArgs a) {
    __shared__ double sums[STATS_THREADS / 32];
    __shared__ float tops[STATS_THREADS / 32];
    __shared__ int ats[STATS_THREADS / 32];
    const int row = blockIdx.y, b = row / (a.drafts_most + 1), i = row % (a.drafts_most + 1), tid = threadIdx.x;
    if (i > count_of(a, b)) {
        return;
    }
    const T* x = static_cast<const T*>(a.target) + b * a.tb + i * a.tr;
    const int c0 = blockIdx.x * a.chunk, c1 = c0 + a.chunk < a.vocab ? c0 + a.chunk : a.vocab;
    float v[HELD];
    float top = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < HELD; n++) {
        const int j = c0 + n * STATS_THREADS + tid;
        v[n] = j < c1 ? to_float(x[j]) : -INFINITY;
        if (j < c1 && before(v[n], j, top, at)) {
            top = v[n];
            at = j;
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, top, o);
        const int j = __shfl_xor_sync(0xffffffffu, at, o);
        if (before(w, j, top, at)) {
            top = w;
            at = j;
        }
    }
    if ((tid & 31) == 0) {
        tops[tid >> 5] = top;
        ats[tid >> 5] = at;
    }
    __syncthreads();
    top = tops[0];
    at = ats[0];
    for (int w = 1; w < STATS_THREADS / 32; w++) {
        if (before(tops[w], ats[w], top, at)) {
            top = tops[w];
            at = ats[w];
        }
    }
    double sum = 0.0;
    if (a.form == LOGITS) {
#pragma unroll
        for (int n = 0; n < HELD; n++) {
            if (c0 + n * STATS_THREADS + tid < c1 && v[n] != -INFINITY) {
                sum += exp(((double)v[n] - (double)top) * a.inverse);
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if ((tid & 31) == 0) {
            sums[tid >> 5] = sum;
        }
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < STATS_THREADS / 32; w++) {
            sum += sums[w];
        }
    }
    if (tid == 0) {
        a.stats[(int64_t)row * a.chunks + blockIdx.x] = Stat{sum, top, at};
    }
}

// One cluster per sequence; thread block r of it has a run of the vocabulary, each warp a run of that.
template <typename T>
__global__ void __launch_bounds__(CHOOSE_THREADS) choose_kernel(VerifyArgs a) {
    __shared__ double of_warp[CHOOSE_WARPS], upto[CLUSTER * CHOOSE_WARPS + 1];  // a warp's weight; the weight in front of each warp of the cluster
    __shared__ int last_some, likeliest;  // the last warp that has any weight; the first of the largest
    __shared__ double row_top, row_scale;  // of the row that is drawn from: p = exp((x - top) / temperature) scale
    __shared__ int refused;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
    const int b = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int count = count_of(a, b), rows = a.drafts_most + 1;
    const T* const target = static_cast<const T*>(a.target) + b * a.tb;
    if (tid == 0) {
        refused = count;
    }
    __syncthreads();
    // every thread block finds the row by itself; a warp has a row
    for (int i = warp; i <= count; i += CHOOSE_WARPS) {
        float top = -INFINITY;
        int at = 0x7fffffff;
        double sum = 0.0;
        if (a.form != PROBABILITIES) {
            const Stat* st = a.stats + ((int64_t)b * rows + i) * a.chunks;
            for (int c = lane; c < a.chunks; c += 32) {
                if (before(st[c].top, st[c].at, top, at)) {
                    top = st[c].top;
                    at = st[c].at;
                }
            }
            for (int o = 16; o > 0; o >>= 1) {
                const float w = __shfl_xor_sync(0xffffffffu, top, o);
                const int j = __shfl_xor_sync(0xffffffffu, at, o);
                if (before(w, j, top, at)) {
                    top = w;
                    at = j;
                }
            }
            if (a.form == LOGITS) {
                for (int c = lane; c < a.chunks; c += 32) {
                    if (st[c].top != -INFINITY) {
                        sum += st[c].sum * exp(((double)st[c].top - (double)top) * a.inverse);
                    }
                }
                for (int o = 16; o > 0; o >>= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, o);
                }
            }
        }
        if (lane == 0 && i < count) {
            const int x = a.drafts[b * a.drafts_most + i];
            bool good = x >= 0 && x < a.vocab;
            if (!good) {
                note_status(a.status, STATUS_TOKEN);
            } else if (a.form == GREEDY) {
                good = x == at;
            } else {
                const double t = to_float(target[i * a.tr + x]);
                const double p = a.form == LOGITS ? exp((t - (double)top) * a.inverse) / sum : t;
                const double q = a.q != nullptr ? (double)a.q[b * a.qb + i * a.qr + x] : 1.0;
                good = (double)a.u[(int64_t)b * rows + i] * q < p;
            }
            if (!good) {
                atomicMin(&refused, i);
            }
        }
    }
    __syncthreads();
    const int j = refused;
    // the row's maximum and sum once more, for whoever needs them
    if (warp == 0 && a.form != PROBABILITIES) {
        const Stat* st = a.stats + ((int64_t)b * rows + j) * a.chunks;
        float top = -INFINITY;
        int at = 0x7fffffff;
        for (int c = lane; c < a.chunks; c += 32) {
            if (before(st[c].top, st[c].at, top, at)) {
                top = st[c].top;
                at = st[c].at;
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const float w = __shfl_xor_sync(0xffffffffu, top, o);
            const int n = __shfl_xor_sync(0xffffffffu, at, o);
            if (before(w, n, top, at)) {
                top = w;
                at = n;
            }
        }
        double sum = 0.0;
        if (a.form == LOGITS) {
            for (int c = lane; c < a.chunks; c += 32) {
                if (st[c].top != -INFINITY) {
                    sum += st[c].sum * exp(((double)st[c].top - (double)top) * a.inverse);
                }
            }
            for (int o = 16; o > 0; o >>= 1) {
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            }
        }
        if (lane == 0) {
            row_top = top;
            row_scale = 1.0 / sum;
            if (a.form == GREEDY) {
                likeliest = at < a.vocab ? at : 0;
            }
        }
    }
    __syncthreads();
    if (a.form != GREEDY) {
        const T* const x = target + j * a.tr;
        const double top = row_top, scale = row_scale;
        const int draft = j < count ? a.drafts[b * a.drafts_most + j] : -1;
        const float* const q = j < count && a.q != nullptr ? a.q + b * a.qb + j * a.qr : nullptr;
        // a warp's run of the vocabulary, in steps of 32
        const int per = (a.vocab + blocks * CHOOSE_WARPS * 32 - 1) / (blocks * CHOOSE_WARPS * 32) * 32;
        const int from = (rank * CHOOSE_WARPS + warp) * per;
        const int to = from + per < a.vocab ? from + per : a.vocab;
        bool less = j < count;  // whether the drafter's share is taken off
        auto weight = [&](int v) {
            const double t = to_float(x[v]);
            double p = a.form == LOGITS ? (t == -INFINITY ? 0.0 : exp((t - top) * a.inverse) * scale) : t;
            if (less) {
                p = q != nullptr ? p - (double)q[v] : (v == draft ? 0.0 : p);
            }
            return p > 0.0 ? p : 0.0;  // (a NaN counts as nothing)
        };
        double total = 0.0;
        for (int round = 0; round < 2; round++) {
            double sum = 0.0;
            for (int v = from + lane; v < to; v += 32) {
                sum += weight(v);
            }
            for (int o = 16; o > 0; o >>= 1) {
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            }
            if (lane == 0) {
                of_warp[warp] = sum;
            }
            cluster.sync();
            // every thread block makes the same sums up to each warp of the cluster, whose intervals leave no gap
            if (warp == 0) {
                double each[CLUSTER * CHOOSE_WARPS / 32], run = 0.0;
                int last = -1;
#pragma unroll
                for (int n = 0; n < CLUSTER * CHOOSE_WARPS / 32; n++) {
                    const int w = lane * (CLUSTER * CHOOSE_WARPS / 32) + n;
                    each[n] = *cluster.map_shared_rank(&of_warp[w % CHOOSE_WARPS], w / CHOOSE_WARPS);
                    run += each[n];
                    last = each[n] > 0.0 ? w : last;
                }
                double scan = run;
                for (int o = 1; o < 32; o <<= 1) {
                    const double n = __shfl_up_sync(0xffffffffu, scan, o);
                    scan += lane >= o ? n : 0.0;
                }
                double upto_here = __shfl_up_sync(0xffffffffu, scan, 1);
                upto_here = lane == 0 ? 0.0 : upto_here;
#pragma unroll
                for (int n = 0; n < CLUSTER * CHOOSE_WARPS / 32; n++) {
                    upto[lane * (CLUSTER * CHOOSE_WARPS / 32) + n] = upto_here;
                    upto_here += each[n];
                }
                upto_here = __shfl_sync(0xffffffffu, upto_here, 31);
                last = __reduce_max_sync(0xffffffffu, last);
                if (lane == 0) {
                    upto[CLUSTER * CHOOSE_WARPS] = upto_here;
                    last_some = last;
                }
            }
            __syncthreads();
            cluster.sync();  // nobody's sums go away while others read them
            total = upto[CLUSTER * CHOOSE_WARPS];
            if (total != 0.0 || !less) {
                break;
            }
            less = false;  // p nowhere above q: they are the same
        }
        const double aim = (double)a.u[(int64_t)b * rows + a.drafts_most] * total;
        const int me = rank * CHOOSE_WARPS + warp;
        // the warp whose run the aim falls into; with a uniform number of 1 or more, or none at all, the last that has any weight
        if (aim < total ? upto[me] <= aim && aim < upto[me + 1] : me == last_some) {
            double run = upto[me];
            int found = -1, positive = -1;
            for (int v0 = from; v0 < to && found < 0; v0 += 32) {
                const int v = v0 + lane;
                const double w = v < to ? weight(v) : 0.0;
                double scan = w;
                for (int o = 1; o < 32; o <<= 1) {
                    const double n = __shfl_up_sync(0xffffffffu, scan, o);
                    scan += lane >= o ? n : 0.0;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && run + scan > aim), some = __ballot_sync(0xffffffffu, w > 0.0);
                positive = some != 0u ? v0 + 31 - __clz(some) : positive;
                found = hit != 0u ? v0 + __ffs(hit) - 1 : -1;
                run += __shfl_sync(0xffffffffu, scan, 31);
            }
            if (lane == 0) {  // (not found by a rounding of the sums: the last with any weight)
                a.tokens[(int64_t)b * rows + j] = found >= 0 ? found : (positive >= 0 ? positive : a.vocab - 1);
            }
        }
        if (rank == 0 && tid == 0 && last_some < 0) {
            a.tokens[(int64_t)b * rows + j] = a.vocab - 1;  // no weight anywhere
        }
    }
    if (rank == 0) {
        for (int i = tid; i < rows; i += CHOOSE_THREADS) {
            if (i != j || a.form == GREEDY) {
                a.tokens[(int64_t)b * rows + i] = i < j ? a.drafts[b * a.drafts_most + i] : (i == j ? likeliest : -1);
            }
        }
        if (tid == 0) {
            a.accepted[b] = j;
        }
    }
}

// How a row is cut for its statistics: chunks of up to CHUNK_MOST values, shorter ones while that leaves SMs without a thread block.
int chunk_of(int64_t rows, int vocab) {
    int chunk = CHUNK_MOST;
    while (chunk > 1024 && rows * ((vocab + chunk - 1) / chunk) < 4 * 148) {
        chunk /= 2;
    }
    return chunk;
}

template <typename T>
int launch_verify(const VerifyArgs& a, cudaStream_t s) {
    const int64_t rows = (int64_t)a.sequences * (a.drafts_most + 1);
    if (a.form != PROBABILITIES) {
        stats_kernel<T><<<dim3((unsigned)a.chunks, (unsigned)rows), STATS_THREADS, 0, s>>>(a);
        count_launch();
        const int rc = check_launch("stats_kernel");
        if (rc != JQ_OK) {
            return rc;
        }
    }
    const int blocks = a.form == GREEDY ? 1 : CLUSTER;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(a.sequences * blocks));
    cfg.blockDim = dim3(CHOOSE_THREADS);
    cfg.stream = s;
    JQ_CUDA(cudaLaunchKernelEx(&cfg, choose_kernel<T>, a));
    count_launch();
    return JQ_OK;
}

}  // namespace
}  // namespace jq

using namespace jq;

extern "C" {

JQ_API int jq_verify_bytes(int64_t sequences, int64_t drafts, int64_t vocab, int logits, int64_t* nbytes) {
    if (nbytes == nullptr || sequences < 0 || drafts < 0 || vocab < 1 || vocab > (int64_t)1 << 30 || drafts > 4095 || sequences > 65535 || sequences * (drafts + 1) > 65535) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: %lld sequences of %lld drafts, %lld tokens (at most 65535 rows, 4095 drafts, 2^30 tokens)", (long long)sequences,
                    (long long)drafts, (long long)vocab);
    }
    const int64_t rows = sequences * (drafts + 1), chunk = chunk_of(rows, (int)vocab);
    *nbytes = logits != 0 ? rows * ((vocab + chunk - 1) / chunk) * (int64_t)sizeof(Stat) : 0;
    return JQ_OK;
}

JQ_API int jq_verify_drafts(int device, int elem, const void* target, int64_t target_stride, int64_t target_row_stride, const int32_t* drafts, const float* draft_probs,
                            int64_t draft_stride, int64_t draft_row_stride, const float* uniforms, const int32_t* counts, int64_t sequences, int64_t drafts_most,
                            int64_t vocab, int logits, double temperature, int32_t* accepted, int32_t* tokens, void* workspace, int64_t workspace_bytes, void* stream) {
    int64_t need = 0;
    int rc = jq_verify_bytes(sequences, drafts_most, vocab, logits, &need);
    if (rc != JQ_OK) {
        return rc;
    }
    if (sequences == 0) {
        return JQ_OK;
    }
    if (!elem_ok(elem) || target == nullptr || (drafts == nullptr && drafts_most > 0) || accepted == nullptr || tokens == nullptr) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: null pointer, or element type %d", elem);
    }
    if (logits != 0 ? !(temperature >= 0.0 && std::isfinite(temperature) && (temperature == 0.0 || std::isfinite(1.0 / temperature))) : false) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: temperature %g", temperature);
    }
    const int form = logits == 0 ? PROBABILITIES : (temperature == 0.0 ? GREEDY : LOGITS);
    if (form != GREEDY && uniforms == nullptr) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: uniform numbers are needed");
    }
    if (workspace_bytes < need || (need > 0 && (workspace == nullptr || ((uintptr_t)workspace & 15) != 0))) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: a workspace of %lld bytes at a 16-byte aligned address is needed, got %lld", (long long)need, (long long)workspace_bytes);
    }
    int count = 0;
    JQ_CUDA(cudaGetDeviceCount(&count));
    if (device < 0 || device >= count) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: device %d of %d", device, count);
    }
    const DeviceGuard guard(device);
    if (!guard.ok) {
        return fail(JQ_ERR_CUDA, "jq_verify_drafts: device %d", device);
    }
    VerifyArgs a = {};
    a.target = target; a.tb = target_stride; a.tr = target_row_stride;
    a.q = form == GREEDY ? nullptr : draft_probs; a.qb = draft_stride; a.qr = draft_row_stride;
    a.drafts = drafts; a.u = uniforms; a.counts = counts;
    a.sequences = (int)sequences; a.drafts_most = (int)drafts_most; a.vocab = (int)vocab;
    a.inverse = form == LOGITS ? 1.0 / temperature : 1.0;
    a.form = form;
    a.accepted = accepted; a.tokens = tokens;
    a.stats = static_cast<Stat*>(workspace);
    a.chunk = chunk_of(sequences * (drafts_most + 1), a.vocab);
    a.chunks = (a.vocab + a.chunk - 1) / a.chunk;
    rc = status_word(&a.status);
    if (rc != JQ_OK) {
        return rc;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    return elem == JQ_ELEM_F32 ? launch_verify<float>(a, s) : (elem == JQ_ELEM_F16 ? launch_verify<__half>(a, s) : launch_verify<__nv_bfloat16>(a, s));
}

}  // extern "C"
