// Verification of drafted tokens (speculative sampling, Leviathan et al. 2023, Chen et al. 2023): with p_i the target's distribution behind draft i, q_i the drafter's (all on
// the draft, where it gives none) and u given uniform numbers, draft x_i is kept while
//     u_i q_i(x_i) < p_i(x_i),
// and one more token comes by the inverse distribution function at u_K: behind the first refused draft j from max(p_j - q_j, 0) over its sum, behind the last draft from p_K.
// At temperature 0 the likeliest token (the first of equal ones) takes the place of both.
//
// The results are whole numbers that may not depend on how the work is cut, so everything is computed in double: the products u q of two floats are exact, sums of a
// vocabulary's probabilities are good to 1e-12, and a cut in another place moves a token with a chance of about 1e-10.
//
// Logits: stats_kernel takes the maximum and the sum of exponentials of chunks of all rows that count. choose_kernel is one cluster per sequence: it joins the chunks, finds the
// row, adds up the row's weights (its second reading, from L2) and looks the token up. The exponential is table-driven (Tang 1989): 2^(t / 32) = 2^n 2^(j / 32) 2^(r / 32) with
// the 32 values of the middle factor in a warp's lanes and a polynomial of the fourth degree, |r| <= 1/2, 10 double instructions where exp() takes about 48.
// Bound: each takes two of the turns in which an SM's quarters issue, some 17 others one: 37 turns for 32 values, 18 us for the 16.8 million logits of 16 sequences with 8 rows of 131072
// (22 measured), beside 10 us for reading them; the choice behind it 11 us, half of which are latencies one after the other.
#include <cooperative_groups.h>

#include <cmath>

#include "jq_rope.cuh"

namespace jq {
namespace {

namespace cg = cooperative_groups;

constexpr int STATS_THREADS = 128, STATS_RESIDENT = 9;  // (thread blocks of an SM, by their registers)
constexpr int CHOOSE_THREADS = 512, CHOOSE_WARPS = CHOOSE_THREADS / 32, CLUSTER = 8;  // (the largest)

struct Stat {
    double sum;  // of exp((x - top) / temperature)
    float top;   // one of the chunk's larger numbers, at temperature 0 the largest; minus infinity where there is no other
    int at;      // where that is first
};

enum { GREEDY, LOGITS, PROBABILITIES };  // what the target is taken as

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
    float far, reach;   // -690 and 600 of its units: what Exponential takes as zero, and where a sum moves to a larger maximum
    int *accepted, *tokens;
    Stat* stats;        // [row][chunks]
    int chunk, chunks;
    int cluster;        // thread blocks of a sequence's choice
    int* status;
};

__device__ __forceinline__ int count_of(const VerifyArgs& a, int b) {
    const int n = a.counts != nullptr ? a.counts[b] : a.drafts_most;
    return n < 0 ? 0 : (n > a.drafts_most ? a.drafts_most : n);
}

// exp((x - top) inverse) of a warp's 32 numbers; every lane has 2^(lane / 32) in `entry`. Off by less than 1.3e-12 of it, (ln 2 / 64)^5 / 120 = 1.25e-12 the polynomial's remainder
// (with the sign of r, so that sums are far better); a degree more would take a thirteenth of the time for digits that no token depends on.
struct Exponential {
    double to_32nds, entry;  // 32 / ln 2 times inverse
    float far;               // x - top below this: less than e^-690, taken as zero (minus infinity too)
    __device__ __forceinline__ Exponential(const VerifyArgs& a, int lane) : to_32nds(a.inverse * 46.166241308446828384), entry(exp2(lane * 0.03125)), far(a.far) {}
    // Of x far below, zero (ZERO), or something no larger than 2^-1022 (of a NaN too). How far is a difference of floats: the sum of top and `far` may round to top, at a low temperature.
    template <bool ZERO>
    __device__ __forceinline__ double of(float x, float top) const {
        constexpr double NEAREST = 6755399441055744.0;  // 2^52 + 2^51: the nearest integer in the low bits
        const double d = (double)x - (double)top, shifted = fma(d, to_32nds, NEAREST), r = fma(d, to_32nds, NEAREST - shifted);
        const int k = __double2loint(shifted);
        // (2^(r / 32) - 1) = sum (r ln 2 / 32)^i / i!
        constexpr double A = 0.021660849392498290, A2 = A * A / 2, A3 = A * A * A / 6, A4 = A * A * A * A / 24;
        const double p = r * fma(r, fma(r, fma(r, A4, A3), A2), A);
        const double e = __shfl_sync(0xffffffffu, entry, k);
        const double v = fma(e, p, e);
        const int high = __double2hiint(v) + ((k & ~31) << 15);  // (times 2^(k / 32))
        if (ZERO) {
            return x - top < far ? 0.0 : __hiloint2double(high, __double2loint(v));
        }
        return __hiloint2double(x - top >= far ? high : 0, __double2loint(v));
    }
};

__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// The largest of a warp's numbers and where it is first.
__device__ __forceinline__ void warp_top(float& top, int& at) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, top, o);
        const int j = __shfl_xor_sync(0xffffffffu, at, o);
        if (before(w, j, top, at)) {
            top = w;
            at = j;
        }
    }
}
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}
__device__ __forceinline__ double warp_scan(double v, int lane) {  // sums up to and with each lane
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double n = __shfl_up_sync(0xffffffffu, v, o);
        v += lane >= o ? n : 0.0;
    }
    return v;
}

// A chunk of a row in one reading, eight values a thread on their way while it works on the eight before. SUMS: every thread adds exponentials up relative to the largest of its first
// eight numbers, which in double need not be the largest of all: only a number e^600 times as large moves it. Else the largest and where it is first.
template <typename T, bool SUMS>
__global__ void __launch_bounds__(STATS_THREADS, STATS_RESIDENT) stats_kernel(VerifyArgs a) {
    constexpr int RUN = 4, TAKE = 2 * RUN, APART = RUN * STATS_THREADS, STEP = 2 * APART;  // two runs of neighbouring values
    __shared__ double sums[STATS_THREADS / 32];
    __shared__ float tops[STATS_THREADS / 32];
    __shared__ int ats[STATS_THREADS / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched programmatically
    asm volatile("griddepcontrol.launch_dependents;");
    const int row = blockIdx.y, b = row / (a.drafts_most + 1), i = row % (a.drafts_most + 1), tid = threadIdx.x, lane = tid & 31;
    if (i > count_of(a, b)) {
        return;
    }
    const T* x = static_cast<const T*>(a.target) + b * a.tb + i * a.tr;
    const int c0 = blockIdx.x * a.chunk, c1 = c0 + a.chunk < a.vocab ? c0 + a.chunk : a.vocab;
    const bool wide = (reinterpret_cast<uintptr_t>(x) & (RUN * sizeof(T) - 1)) == 0;
    const Exponential exponential(a, lane);
    float top = -INFINITY;
    int at = 0x7fffffff;
    double sum = 0.0;
    auto take = [&](int j, float (&v)[TAKE]) {  // (behind the chunk: minus infinity)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int from = j + h * APART;
            if (wide && from + RUN <= c1) {
                if constexpr (sizeof(T) == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(x + from);
                    v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
                } else {
                    const uint2 f = *reinterpret_cast<const uint2*>(x + from);
                    const T* const e = reinterpret_cast<const T*>(&f);
#pragma unroll
                    for (int n = 0; n < RUN; n++) {
                        v[4 * h + n] = to_float(e[n]);
                    }
                }
            } else {
#pragma unroll
                for (int n = 0; n < RUN; n++) {
                    v[4 * h + n] = from + n < c1 ? to_float(x[from + n]) : -INFINITY;
                }
            }
        }
    };
    float v[TAKE], v_next[TAKE];
    take(c0 + tid * RUN, v);
#pragma unroll 1
    for (int j0 = c0; j0 < c1; j0 += STEP) {  // (a warp's lanes stay together)
        const int j = j0 + tid * RUN;
        take(j + STEP, v_next);
        if constexpr (SUMS) {
            float here = v[0];
#pragma unroll
            for (int n = 1; n < TAKE; n++) {
                here = fmaxf(here, v[n]);
            }
            const bool far = here - top > a.reach;  // (top is minus infinity at first, and as long as nothing else has come)
            if (__any_sync(0xffffffffu, far)) {
                const double shrink = exponential.of<true>(top, far ? here : 0.0f);
                sum = far && sum != 0.0 ? sum * shrink : sum;
                top = far ? here : top;
            }
            double part = 0.0;
#pragma unroll
            for (int n = 0; n < TAKE; n++) {
                part += exponential.of<false>(v[n], top);
            }
            sum += top == -INFINITY ? 0.0 : part;
        } else {
#pragma unroll
            for (int n = 0; n < TAKE; n++) {  // (in rising order: the first of equal ones stays)
                const int here = j + (n & 3) + (n >> 2) * APART;
                const bool larger = v[n] > top || (at == 0x7fffffff && v[n] == top && here < c1);
                at = larger ? here : at;
                top = larger ? v[n] : top;
            }
        }
#pragma unroll
        for (int n = 0; n < TAKE; n++) {
            v[n] = v_next[n];
        }
    }
    const float mine = top;
    warp_top(top, at);
    if (lane == 0) {
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
    if constexpr (SUMS) {
        const double shrink = exponential.of<true>(mine, top);
        sum = warp_total(sum != 0.0 ? sum * shrink : 0.0);
        if (lane == 0) {
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

// A row's chunks joined, by a warp.
template <int FORM>
__device__ __forceinline__ void join_chunks(const VerifyArgs& a, const Exponential& exponential, int64_t row, int lane, float& top, int& at, double& sum) {
    const Stat* const st = a.stats + row * a.chunks;
    top = -INFINITY;
    at = 0x7fffffff;
    sum = 0.0;
    for (int c = lane; c < a.chunks; c += 32) {
        if (before(st[c].top, st[c].at, top, at)) {
            top = st[c].top;
            at = st[c].at;
        }
    }
    warp_top(top, at);
    if constexpr (FORM == LOGITS) {
        for (int c0 = 0; c0 < a.chunks; c0 += 32) {
            const int c = c0 + lane;
            const float t = c < a.chunks ? st[c].top : -INFINITY;
            const double e = exponential.of<true>(t, top);
            sum += t != -INFINITY ? st[c].sum * e : 0.0;
        }
        sum = warp_total(sum);
    }
}

// One cluster per sequence (one thread block at temperature 0); thread block r of it has a run of the vocabulary, each warp a run of that.
template <typename T, int FORM>
__global__ void __launch_bounds__(CHOOSE_THREADS) choose_kernel(VerifyArgs a) {
    __shared__ double of_warp[2][CHOOSE_WARPS], upto[CLUSTER * CHOOSE_WARPS + 1];  // a warp's weight; the weight in front of each warp of the cluster
    __shared__ int taken;        // the warp of the cluster that the token falls to: the last with any weight that begins at the aim or in front of it
    __shared__ double row_sum[CHOOSE_WARPS];  // of the last row that each warp has looked at, which one of them goes on with: p = exp((x - top) / temperature) / sum
    __shared__ float row_top[CHOOSE_WARPS];
    __shared__ int row_at[CHOOSE_WARPS], refused;
    const int blocks = FORM == GREEDY ? 1 : a.cluster, rank = blockIdx.x % blocks, b = blockIdx.x / blocks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = a.drafts_most + 1;
    if (tid == 0) {
        refused = 0x7fffffff;
    }
    const Exponential exponential(a, lane);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int count = count_of(a, b);
    const T* const target = static_cast<const T*>(a.target) + b * a.tb;
    auto uniform = [&](int i) {  // (a negative number is zero)
        const double u = (double)a.u[(int64_t)b * rows + i];
        return u < 0.0 ? 0.0 : u;
    };
    const double u_token = FORM == GREEDY ? 0.0 : uniform(a.drafts_most);
    __syncthreads();
    // ---- the first refused draft: every thread block finds it by itself, a warp a draft
    for (int i = warp; i <= count; i += CHOOSE_WARPS) {
        const int x = i < count ? a.drafts[b * a.drafts_most + i] : 0;
        bool good = x >= 0 && x < a.vocab;
        float top = 0.0f;
        int at = 0;
        double sum = 0.0;
        if constexpr (FORM != PROBABILITIES) {
            join_chunks<FORM>(a, exponential, (int64_t)b * rows + i, lane, top, at, sum);
            if (lane == 0) {
                row_top[warp] = top;
                row_at[warp] = at;
                row_sum[warp] = sum;
            }
        }
        if (i == count) {
            break;
        }
        if (!good) {
            note_status(a.status, STATUS_TOKEN);
        } else if constexpr (FORM == GREEDY) {
            good = x == at;
        } else {
            const float t = to_float(target[i * a.tr + x]);
            double p = (double)t;
            if constexpr (FORM == LOGITS) {
                p = exponential.of<true>(t, top) / sum;
            }
            const double q = a.q != nullptr ? (double)a.q[b * a.qb + i * a.qr + x] : 1.0;
            good = uniform(i) * q < p;
        }
        if (!good) {
            if (lane == 0) {
                atomicMin(&refused, i);
            }
            break;  // (this warp's later drafts are behind it)
        }
    }
    __syncthreads();
    const int j = refused < count ? refused : count;
    if constexpr (FORM != GREEDY) {
        cg::cluster_group cluster = cg::this_cluster();
        const T* const x = target + j * a.tr;
        const float top = row_top[j % CHOOSE_WARPS];
        const double scale = 1.0 / row_sum[j % CHOOSE_WARPS];
        const int draft = j < count ? a.drafts[b * a.drafts_most + j] : -1;
        const float* const q = j < count && a.q != nullptr ? a.q + b * a.qb + j * a.qr : nullptr;
        bool less = j < count;  // whether the drafter's share is taken off
        // the weight of one value a lane (at or behind `end`: none); by a whole warp
        auto weight = [&](float t, float share, int v, int end) {
            double p = (double)t;
            if constexpr (FORM == LOGITS) {
                p = exponential.of<true>(t, top) * scale;
            }
            const double rest = less && q == nullptr && v == draft ? 0.0 : p - (double)share;
            return v < end && rest > 0.0 ? rest : 0.0;  // (a NaN counts as nothing)
        };
        // A warp has a run of the vocabulary, a lane `each` neighbouring values of it, four of which are on their way ahead: the lane's sum is a place of the search too
        const int each = (int)(((int64_t)a.vocab + blocks * CHOOSE_THREADS * 4 - 1) / (blocks * CHOOSE_THREADS * 4)) * 4;
        auto begin_of = [&](int lane_of_all) { return (int)((int64_t)lane_of_all * each < a.vocab ? lane_of_all * each : a.vocab); };
        const int me = rank * CHOOSE_WARPS + warp, from = begin_of(me * 32 + lane), to = begin_of(me * 32 + lane + 1);
        const bool wide = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
        auto four = [&](int v, float (&t)[4], float (&share)[4]) {
#pragma unroll
            for (int n = 0; n < 4; n++) {
                t[n] = share[n] = 0.0f;
            }
            if (wide && v + 4 <= to) {
                if constexpr (sizeof(T) == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(x + v);
                    t[0] = f.x; t[1] = f.y; t[2] = f.z; t[3] = f.w;
                } else {
                    const uint2 f = *reinterpret_cast<const uint2*>(x + v);
                    const T* const e = reinterpret_cast<const T*>(&f);
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        t[n] = to_float(e[n]);
                    }
                }
                if (less && q != nullptr) {
                    const float4 f = *reinterpret_cast<const float4*>(q + v);
                    share[0] = f.x; share[1] = f.y; share[2] = f.z; share[3] = f.w;
                }
            } else {
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    if (v + n < to) {
                        t[n] = to_float(x[v + n]);
                        share[n] = less && q != nullptr ? q[v + n] : 0.0f;
                    }
                }
            }
        };
        double total = 0.0, mine = 0.0;
#pragma unroll 1
        for (int round = 0; round < 2; round++) {
            float t[4], share[4];
            four(from, t, share);
            mine = 0.0;
#pragma unroll 1
            for (int v = 0; v < each; v += 4) {
                float t_next[4], share_next[4];
                four(from + v + 4, t_next, share_next);
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    mine += weight(t[n], share[n], from + v + n, to);
                    t[n] = t_next[n];
                    share[n] = share_next[n];
                }
            }
            const double sum = warp_total(mine);
            if (lane == 0) {
                of_warp[round][warp] = sum;
            }
            cluster.sync();
            // every thread block makes the same sums up to each warp of the cluster, whose intervals leave no gap
            if (warp == 0) {
                constexpr int N = CLUSTER * CHOOSE_WARPS / 32;  // (of smaller clusters the last have nothing)
                double part[N], run = 0.0;
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const int w = lane * N + n;
                    part[n] = w < blocks * CHOOSE_WARPS ? *cluster.map_shared_rank(&of_warp[round][w % CHOOSE_WARPS], w / CHOOSE_WARPS) : 0.0;
                    run += part[n];
                }
                const double scan = warp_scan(run, lane);
                double here = __shfl_up_sync(0xffffffffu, scan, 1);
                here = lane == 0 ? 0.0 : here;
                const double all = __shfl_sync(0xffffffffu, scan, 31), aim = u_token * all;
                int last = -1;
#pragma unroll
                for (int n = 0; n < N; n++) {
                    upto[lane * N + n] = here;
                    last = part[n] > 0.0 && (!(aim < all) || here <= aim) ? lane * N + n : last;
                    here += part[n];
                }
                last = __reduce_max_sync(0xffffffffu, last);
                if (lane == 31) {
                    upto[CLUSTER * CHOOSE_WARPS] = all;
                    taken = last;
                }
            }
            __syncthreads();
            total = upto[CLUSTER * CHOOSE_WARPS];
            if (total != 0.0 || !less) {
                break;
            }
            __syncthreads();
            less = false;  // p nowhere above q: they are the same
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // nobody's sums go away while others read them
        // the warp whose run the aim falls into; with a uniform number of 1 or more, or none at all, the last that has any weight
        const double aim = u_token * total;
        if (me == taken) {
            const double scan = warp_scan(mine, lane) + upto[me];
            const unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && scan > aim), some = __ballot_sync(0xffffffffu, mine > 0.0);
            const int chosen = over != 0u ? __ffs(over) - 1 : 31 - __clz(some);  // (not found by a rounding of the sums: the last with any weight)
            double before_it = __shfl_sync(0xffffffffu, scan - mine, chosen);
            const int first = begin_of(me * 32 + chosen), end = begin_of(me * 32 + chosen + 1);
            int found = -1, positive = -1;
#pragma unroll 1
            for (int at = first; at < end && found < 0; at += 32) {
                const int v = at + lane;
                const double w = weight(v < end ? to_float(x[v]) : 0.0f, v < end && less && q != nullptr ? q[v] : 0.0f, v, end);
                const double upto_here = warp_scan(w, lane);
                const unsigned is = __ballot_sync(0xffffffffu, w > 0.0 && before_it + upto_here > aim), any = __ballot_sync(0xffffffffu, w > 0.0);
                positive = any != 0u ? at + 31 - __clz(any) : positive;
                found = is != 0u ? at + __ffs(is) - 1 : -1;
                before_it += __shfl_sync(0xffffffffu, upto_here, 31);
            }
            if (lane == 0) {
                a.tokens[(int64_t)b * rows + j] = found >= 0 ? found : (positive >= 0 ? positive : a.vocab - 1);
            }
        }
        if (rank == 0 && tid == 0 && taken < 0) {
            a.tokens[(int64_t)b * rows + j] = a.vocab - 1;  // no weight anywhere
        }
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (rank == 0) {
        for (int i = tid; i < rows; i += CHOOSE_THREADS) {
            if (i != j || FORM == GREEDY) {
                a.tokens[(int64_t)b * rows + i] = i < j ? a.drafts[b * a.drafts_most + i] : (i == j ? (row_at[j % CHOOSE_WARPS] < a.vocab ? row_at[j % CHOOSE_WARPS] : 0) : -1);
            }
        }
        if (tid == 0) {
            a.accepted[b] = j;
        }
    }
}

// How a row is cut for its statistics: into as many chunks as fill the SMs' thread blocks once, twice, three or four times, whichever has them done first. A thread block's
// beginning and end take the time of about 1024 values. (Chunks of 8192 throughout: 128 rows of 131072 30 us.)
int chunk_of(int64_t rows, int64_t vocab) {
    const int64_t room = 148 * STATS_RESIDENT;
    int64_t best = 0, least = 0;
    for (int64_t times = 1; times <= 4; times++) {
        const int64_t fit = rows < 1 ? 1 : room * times / rows, most = (vocab + 511) / 512, chunks = fit < 1 ? 1 : (fit < most ? fit : most);
        const int64_t chunk = ((vocab + chunks - 1) / chunks + 511) / 512 * 512;
        const int64_t waves = (rows * ((vocab + chunk - 1) / chunk) + room - 1) / room, cost = waves * (chunk + 1024);
        if (times == 1 || cost < least) {
            best = chunk;
            least = cost;
        }
    }
    return (int)best;
}

template <typename T, int FORM>
int launch_verify(const VerifyArgs& a, cudaStream_t s) {
    const int64_t rows = (int64_t)a.sequences * (a.drafts_most + 1);
    if constexpr (FORM != PROBABILITIES) {
        launch_behind(stats_kernel<T, FORM == LOGITS>, dim3((unsigned)a.chunks, (unsigned)rows), dim3(STATS_THREADS), s, a);
        count_launch();
        const int rc = check_launch("stats_kernel");
        if (rc != JQ_OK) {
            return rc;
        }
    }
    const int blocks = FORM == GREEDY ? 1 : a.cluster;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3((unsigned)(a.sequences * blocks));
    cfg.blockDim = dim3(CHOOSE_THREADS);
    cfg.stream = s;
    JQ_CUDA(cudaLaunchKernelEx(&cfg, choose_kernel<T, FORM>, a));
    count_launch();
    return JQ_OK;
}

template <typename T>
int launch_verify_form(const VerifyArgs& a, int form, cudaStream_t s) {
    return form == GREEDY ? launch_verify<T, GREEDY>(a, s) : (form == LOGITS ? launch_verify<T, LOGITS>(a, s) : launch_verify<T, PROBABILITIES>(a, s));
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
    const int64_t rows = sequences * (drafts + 1), chunk = chunk_of(rows, vocab);
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
    if (logits != 0 && temperature != 0.0 && !(temperature >= 1e-300 && temperature <= 1e30)) {
        return fail(JQ_ERR_INVALID, "jq_verify_drafts: temperature %g (0, or from 1e-300 to 1e30)", temperature);
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
    a.far = (float)(-690.0 / a.inverse);
    a.reach = (float)(600.0 / a.inverse);
    a.accepted = accepted; a.tokens = tokens;
    a.stats = static_cast<Stat*>(workspace);
    a.chunk = chunk_of(sequences * (drafts_most + 1), vocab);
    a.chunks = (a.vocab + a.chunk - 1) / a.chunk;
    // eight thread blocks a sequence while all of them fit the GPU at once (two to an SM), and not more than leave a warp 256 values
    a.cluster = CLUSTER;
    while (a.cluster > 1 && (sequences * a.cluster > 2 * 148 || (int64_t)a.cluster * CHOOSE_WARPS * 256 > 2 * vocab)) {
        a.cluster /= 2;
    }
    rc = status_word(&a.status);
    if (rc != JQ_OK) {
        return rc;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    return elem == JQ_ELEM_F32 ? launch_verify_form<float>(a, form, s) : (elem == JQ_ELEM_F16 ? launch_verify_form<__half>(a, form, s) : launch_verify_form<__nv_bfloat16>(a, form, s));
}

}  // extern "C"
