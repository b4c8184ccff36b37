// The sampler's probabilities (k_sample_probs) and the verification of drafted
// tokens against them (k_verify_drafts).
//
// Both give a row of the vocabulary to one cluster of blocks, each block a
// contiguous slice, and join the slices through distributed shared memory in
// rank order: results do not depend on timing.
#include <cooperative_groups.h>

#include "sampler.cuh"

namespace cg = cooperative_groups;

namespace qora {

namespace {

constexpr int kVThreads = 512;
constexpr int kVWarps = kVThreads / 32;
constexpr int kMaxCluster = 8;

// ------------------------------------------------------------ probabilities
// Steps of sample_token (generate_new.rs:771-862) up to its draw, for one row:
//   x = logit with the repetition penalty (divided when > 0, else multiplied,
//       once for every time the token was said);   z = x / temperature
//   kept = the first top_k of a stable descending order (among equal values
//       the lower index comes first); all when top_k is 0 or >= V
//   p = exp(z - max) / sum over the kept
//   top_p in (0, 1): in that order, a token stays while the probabilities
//       before it sum to less than top_p; p is divided by the sum of what stays
// The row's slice stays in shared memory after one read.  The top_k-th largest of
// the maxima of groups (one or four a thread) bounds the top_k-th logit from below: a
// histogram of the maxima (256 bins between the least and the largest of them)
// gives a bin that it lies in, and only logits down to that bin are sorted, hardly
// more than top_k.  Where there are too few maxima, or too many candidates (equal logits), a
// radix selection over the slices decides exactly.  Exponentials and
// sums of the kept are in 64 bits: the order and the top_p border are decided
// by values next to each other.
// 96 rows of 151936 with top_k 50: 52.5 us in a captured loop, 2.2 TB/s.  Memory is busy 14 % of that:
// a block lives some 17 us, of which the read is 4 and the rest barriers of the
// block and the cluster, and shared memory lets 296 of the 768 blocks run at once.
constexpr int kBins = 256;
constexpr float kBinRange = 64.0f;   // the bins reach no further down: masks of -1e9 would leave the rest one bin
constexpr int kCand = 2048;          // candidates that one sort takes
constexpr int kSliceMax = 40960;     // logits of a slice in shared memory (a multiple of 4)

struct ProbsArgs {
    const float *logits;
    const uint32_t *prev;
    float *probs;
    int *err;
    int V, n_prev, slice, by_maxima;
    qora_sample_params params;
};

struct alignas(16) ProbsSmem {  // (the slice behind it is read in 16-byte pieces)
    unsigned hist[kBins];
    unsigned long long cand[kCand];   // order key of x, then ~index
    double wsum[kVWarps + 1];
    float red[2][kVWarps];
    float mx, mn, slice_max, slice_min;
    int bad, slice_bad;
    unsigned n_cand, eq_before;
    unsigned sel_bin, sel_below, sel_in;
    double sum, slice_sum;
    unsigned eq_count, scan[kBins / 32];
};

static_assert(sizeof(ProbsSmem) % 16 == 0 && kSliceMax % 4 == 0, "the slice is 16-byte aligned");

// Order of f32 values as unsigned integers; the two zeros are equal logits, so -0
// becomes +0 (whose addition changes no other value).
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = __float_as_uint(__fadd_rn(x, 0.0f));
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the block in warp order; every thread gets it.
__device__ double block_sum_f64(double v, double *wsum) {
    v = warp_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kVWarps; w++) s += wsum[w];
    return s;
}

// Block-wide exclusive scan in thread order.
__device__ double block_scan_f64(double v, double *wsum, double &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
    for (int w = 0; w < kVWarps; w++) {
        if (w < warp) before += wsum[w];
        total += wsum[w];
    }
    return before + x - v;
}

// The digit of a histogram of the whole row in which the count from the largest
// down reaches `need`: hist bins are summed over the cluster's blocks.
// Called by warp 0 of every block; writes sel_bin / sel_below / sel_in.
__device__ __forceinline__ void select_bin(cg::cluster_group &cl, ProbsSmem *sm, int bins, unsigned need) {
    const int lane = threadIdx.x & 31;
    const unsigned nr = cl.num_blocks();
    unsigned below = 0;
    for (int b0 = 0; b0 < bins; b0 += 32) {
        const int bin = bins - 1 - (b0 + lane);
        unsigned c = 0;
#pragma unroll
        for (unsigned r = 0; r < kMaxCluster; r++)  // (reads in flight together)
            if (r < nr) c += cl.map_shared_rank(sm, r)->hist[bin];
        unsigned x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, below + x >= need);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                sm->sel_bin = bin;
                sm->sel_below = below + x - c;
                sm->sel_in = c;
            }
            return;
        }
        below += __shfl_sync(0xffffffffu, x, 31);
    }
}

// The two halves of a cluster barrier, by every thread.
__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Sorts list[0 .. found), found <= E kVThreads <= kCand, by a bitonic network: a thread
// has E neighbours, so partners up to 32 E apart are in the thread or the warp, and
// 4 of the 9 (2: 10, 4: 11) distances go through shared memory.
template <int E>
__device__ __noinline__ void sort_descending(unsigned long long *list, unsigned found) {
    const int tid = threadIdx.x;
    unsigned long long v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = tid * E + e < (int)found ? list[tid * E + e] : 0ull;
    for (int span = 2; span <= E * kVThreads; span <<= 1)
        for (int step = span >> 1; step > 0; step >>= 1) {
            unsigned long long w[E];
            if (step < E) {
#pragma unroll
                for (int e = 0; e < E; e++) w[e] = step == 1 ? v[e ^ (E > 1)] : v[e ^ (E > 2 ? 2 : 0)];
            } else if (step < 32 * E) {
#pragma unroll
                for (int e = 0; e < E; e++) w[e] = __shfl_xor_sync(0xffffffffu, v[e], step / E);
            } else {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++) list[tid * E + e] = v[e];
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++) w[e] = list[(tid * E + e) ^ step];
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int i = tid * E + e;
                const bool larger = ((i & step) == 0) == ((i & span) == 0);
                if ((w[e] > v[e]) == larger) v[e] = w[e];
            }
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++) list[tid * E + e] = v[e];
    __syncthreads();
}

// VEC: rows and slices are multiples of 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(kVThreads) k_sample_probs(const ProbsArgs a) {
    extern __shared__ uint4 dyn[];
    ProbsSmem *sm = reinterpret_cast<ProbsSmem *>(dyn);
    float *x = reinterpret_cast<float *>(sm + 1);
    cg::cluster_group cl = cg::this_cluster();
    const unsigned rank = cl.block_rank(), nr = cl.num_blocks();
    auto meet = [&]() {  // all blocks of the row
        if (nr == 1) __syncthreads();
        else cl.sync();
    };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const int v0 = (int)rank * a.slice, n = max(0, min(a.slice, a.V - v0));
    griddep_launch_dependents();
    griddep_wait();
    const float *in = a.logits + row * a.V + v0;
    float *out = a.probs + row * a.V + v0;
    // f(i, value) over the slice in shared memory, sixteen bytes at a time
    auto each = [&](auto f) {
        if constexpr (VEC) {
            const float4 *x4 = reinterpret_cast<const float4 *>(x);
            for (int i = tid; i < n / 4; i += kVThreads) {
                const float4 v = x4[i];
                f(4 * i, v.x), f(4 * i + 1, v.y), f(4 * i + 2, v.z), f(4 * i + 3, v.w);
            }
        } else {
            for (int i = tid; i < n; i += kVThreads) f(i, x[i]);
        }
    };
    // eight loads of a thread in flight
    if constexpr (VEC) {
        const float4 *in4 = reinterpret_cast<const float4 *>(in);
        float4 *x4 = reinterpret_cast<float4 *>(x);
        for (int i0 = 0; i0 < n / 4; i0 += 8 * kVThreads) {
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i0 + j * kVThreads + tid < n / 4) v[j] = __ldcs(in4 + i0 + j * kVThreads + tid);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i0 + j * kVThreads + tid < n / 4) x4[i0 + j * kVThreads + tid] = v[j];
        }
    } else {
        for (int i0 = 0; i0 < n; i0 += 8 * kVThreads) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i0 + j * kVThreads + tid < n) v[j] = __ldcs(in + i0 + j * kVThreads + tid);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i0 + j * kVThreads + tid < n) x[i0 + j * kVThreads + tid] = v[j];
        }
    }
    __syncthreads();
    // penalty: a thread per mention.  Every mention of a token takes the same step, so the
    // result does not depend on whose comes first.  32 rows of 2048 with 4096 mentions each
    // take 12 us, and 930 when all are of one token (413 when the first lane of a token
    // takes its warp's steps together, but then the others 16, and 160 rows with 16
    // mentions 8.0 against 7.6).  A warp per mention that looks for others of its token in
    // the history took 1880 us.
    if (a.prev && a.params.repetition_penalty != 1.0f) {
        const uint32_t *prev = a.prev + row * a.n_prev;
        for (int j = tid; j < a.n_prev; j += kVThreads) {
            const uint32_t tok = __ldg(prev + j);
            if (tok >= (unsigned)a.V || (int)tok < v0 || (int)tok >= v0 + n) continue;
            unsigned *at = reinterpret_cast<unsigned *>(x + (tok - v0));
            unsigned was = *at, before;
            do {
                before = was;
                const float y = __uint_as_float(before);
                was = atomicCAS(at, before, __float_as_uint(y > 0.0f ? __fdiv_rn(y, a.params.repetition_penalty)
                                                                     : __fmul_rn(y, a.params.repetition_penalty)));
            } while (was != before);
        }
        __syncthreads();
    }
    // the maxima of the thread's four groups of logits, the row's, and the least finite group's
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    bool nan = false;
    if constexpr (VEC) {
        const float4 *x4 = reinterpret_cast<const float4 *>(x);
        for (int i = tid; i < n / 4; i += kVThreads) {
            const float4 v = x4[i];
            tops[0] = fmaxf(tops[0], v.x), tops[1] = fmaxf(tops[1], v.y);
            tops[2] = fmaxf(tops[2], v.z), tops[3] = fmaxf(tops[3], v.w);
            nan = nan || v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w;
        }
    } else {
        int i = tid;
        for (; i + 3 * kVThreads < n; i += 4 * kVThreads)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v = x[i + j * kVThreads];
                tops[j] = fmaxf(tops[j], v);
                nan = nan || v != v;
            }
#pragma unroll
        for (int j = 0; j < 3; j++)
            if (i + j * kVThreads < n) {
                const float v = x[i + j * kVThreads];
                tops[j] = fmaxf(tops[j], v);
                nan = nan || v != v;
            }
    }
    if (a.by_maxima == 1) {  // (one group)
        tops[0] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        tops[1] = tops[2] = tops[3] = -INFINITY;
    }
    float mx = -INFINITY, mn = INFINITY;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        mx = fmaxf(mx, tops[j]);
        if (tops[j] > -INFINITY) mn = fminf(mn, tops[j]);
    }
    mx = warp_max(mx), mn = -warp_max(-mn);
    if (lane == 0) sm->red[0][warp] = mx, sm->red[1][warp] = mn;
    for (int i = tid; i < kBins; i += kVThreads) sm->hist[i] = 0;
    nan = __syncthreads_or(nan);
    if (warp == 0) {
        mx = warp_max(lane < kVWarps ? sm->red[0][lane] : -INFINITY);
        mn = -warp_max(lane < kVWarps ? -sm->red[1][lane] : -INFINITY);
        if (lane == 0) {
            sm->slice_max = mx;
            sm->slice_min = mn;
            sm->slice_bad = nan;
            sm->n_cand = 0;
        }
    }
    meet();
    if (warp == 0) {  // a lane per block: remote reads in flight together
        const bool there = lane < (int)nr;
        const ProbsSmem *o = cl.map_shared_rank(sm, there ? lane : 0);
        const float m = warp_max(there ? o->slice_max : -INFINITY);
        const float least = -warp_max(there ? -o->slice_min : -INFINITY);
        const bool bad = __any_sync(0xffffffffu, there && o->slice_bad);
        if (lane == 0) {
            sm->mx = m;
            sm->mn = least;
            sm->bad = bad || !isfinite(m);
        }
    }
    __syncthreads();
    mx = sm->mx, mn = fmaxf(sm->mn, sm->mx - kBinRange);
    const bool bad = sm->bad;
    const double temp = a.params.temperature > 0.0f ? (double)a.params.temperature : 1.0;
    const bool topk = a.params.top_k > 0 && a.params.top_k < a.V;
    if (bad) {  // NaN or +inf among the logits, or none that is finite
        if (tid == 0 && rank == 0) raise_error(a.err, kDevNaN);
        for (int i = tid; i < n; i += kVThreads) out[i] = 0.0f;
        meet();  // no block leaves while another reads its slice_max
        return;
    }
    if (!topk) {
        // exp((x - max) / T) in 32 bits: the product with 1 / T keeps its rounding error
        // (and 1 / T's), which enters as e^z (1 + error).  Sums of four go into a 64-bit
        // sum.  (All in 64 bits took 49 us for 92 rows of 151936, against 46, most of it waiting.)
        const double per = 1.0 / temp;
        const float per_hi = (float)fmin(per, 3.4e38), per_lo = per < 3.4e38 ? (float)(per - (double)per_hi) : 0.0f;
        auto weight = [&](float v) {
            const float d = v - mx, z = d * per_hi;
            const float e = expf(z);
            // (z past f32's range, -inf among it: the error is NaN or infinite, and e = 0)
            return fmaf(e, fminf(fmaxf(fmaf(d, per_hi, -z) + d * per_lo, -1.0f), 1.0f), e);
        };
        double s = 0.0;
        if constexpr (VEC) {
            float4 *x4 = reinterpret_cast<float4 *>(x);
            for (int i = tid; i < n / 4; i += kVThreads) {
                float4 v = x4[i];
                v.x = weight(v.x), v.y = weight(v.y), v.z = weight(v.z), v.w = weight(v.w);
                x4[i] = v;
                s += (double)((v.x + v.y) + (v.z + v.w));
            }
        } else {
            for (int i = tid; i < n; i += kVThreads) s += (double)(x[i] = weight(x[i]));
        }
        s = block_sum_f64(s, sm->wsum);
        if (tid == 0) sm->slice_sum = s;
        meet();
        if (tid == 0) {
            double t = 0.0;
            for (unsigned r = 0; r < nr; r++) t += cl.map_shared_rank(sm, r)->slice_sum;
            sm->sum = 1.0 / t;
        }
        __syncthreads();
        const float inv = (float)sm->sum;
        if (nr > 1) cluster_arrive();  // (the sums have been read; before the stores, which it would wait for)
        if constexpr (VEC) {
            const float4 *x4 = reinterpret_cast<const float4 *>(x);
            for (int i = tid; i < n / 4; i += kVThreads) {
                const float4 v = x4[i];
                __stcs(reinterpret_cast<float4 *>(out) + i, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            }
        } else {
            for (int i = tid; i < n; i += kVThreads) out[i] = x[i] * inv;
        }
        if (nr > 1) cluster_wait();
        return;
    }
    const unsigned k = a.params.top_k;
    auto zeros = [&]() {
        if constexpr (VEC) {
            for (int i = tid; i < n / 4; i += kVThreads) reinterpret_cast<float4 *>(out)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
            for (int i = tid; i < n; i += kVThreads) out[i] = 0.0f;
        }
    };
    if (nr == 1) zeros();
    const float per_bin = mx > mn ? (float)(kBins - 1) / (mx - mn) : 0.0f;
    auto bin_of = [&](float v) { return (int)fminf((mx - v) * per_bin, (float)(kBins - 1)); };
    bool few = a.by_maxima;
    int sel = 0;
    if (few) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (tops[j] > -INFINITY) atomicAdd(&sm->hist[bin_of(tops[j])], 1u);
        meet();
        // the bin of the k-th largest maximum; with fewer finite maxima than k, all bins
        unsigned c = 0;
        if (tid < kBins) {
#pragma unroll
            for (unsigned r = 0; r < kMaxCluster; r++)
                if (r < nr) c += cl.map_shared_rank(sm, r)->hist[tid];
        }
        unsigned x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31 && warp < kBins / 32) sm->scan[warp] = x;
        if (tid == 0) sm->sel_bin = kBins - 1;
        __syncthreads();
        unsigned before = 0;
        for (int w = 0; w < warp && w < kBins / 32; w++) before += sm->scan[w];
        if (tid < kBins && before + x >= k && before + x - c < k) sm->sel_bin = tid;
        __syncthreads();
        sel = sm->sel_bin;
    }
    ProbsSmem *lead = cl.map_shared_rank(sm, 0);
    auto candidate = [&](int i) { return ((unsigned long long)order_key(x[i]) << 32) | (unsigned)~(unsigned)(v0 + i); };
    auto offer = [&](int i) {
        const unsigned at = atomicAdd(&lead->n_cand, 1u);
        if (at < kCand) lead->cand[at] = candidate(i);
    };
    if (few) {
        // bin_of(v) <= sel, without a conversion for every logit
        const float below = (float)(sel + 1);
        each([&](int i, float v) {
            if (sel == kBins - 1 || (mx - v) * per_bin < below) offer(i);
        });
        meet();
        few = lead->n_cand <= kCand;
    }
    if (!few && a.V <= kCand) {  // (one block) every logit is one
        for (int i = tid; i < n; i += kVThreads) sm->cand[i] = candidate(i);
        if (tid == 0) sm->n_cand = n;
        __syncthreads();
    } else if (!few) {
        meet();  // (every block has seen the count)
        if (tid == 0) sm->n_cand = 0;
        meet();
        // radix selection of the k-th key, 8 bits at a time
        unsigned prefix = 0, mask = 0, need = k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kVThreads) sm->hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kVThreads) {
                const unsigned key = order_key(x[i]);
                if ((key & mask) == prefix) atomicAdd(&sm->hist[(key >> shift) & 255u], 1u);
            }
            meet();
            if (warp == 0) select_bin(cl, sm, 256, need);
            __syncthreads();
            prefix |= sm->sel_bin << shift;
            mask |= 255u << shift;
            need -= sm->sel_below;
            meet();
        }
        // keys above the k-th are kept, and the first `need` equal to it in index order
        unsigned eq = 0;
        for (int i = tid; i < n; i += kVThreads) eq += order_key(x[i]) == prefix;
        eq = (unsigned)block_sum_f64((double)eq, sm->wsum);
        if (tid == 0) sm->eq_count = eq;
        meet();
        if (tid == 0) {
            unsigned before = 0;
            for (unsigned r = 0; r < rank; r++) before += cl.map_shared_rank(sm, r)->eq_count;
            sm->eq_before = before;
        }
        __syncthreads();
        unsigned before = sm->eq_before;
        for (int i0 = 0; i0 < n; i0 += kVThreads) {
            const int i = i0 + tid;
            const unsigned key = i < n ? order_key(x[i]) : 0u;
            const bool same = i < n && key == prefix;
            double total;
            const unsigned at = before + (unsigned)block_scan_f64(same ? 1.0 : 0.0, sm->wsum, total);
            before += (unsigned)total;
            if (i < n && (key > prefix || (same && at < need))) offer(i);
        }
        meet();
    }
    // A cluster's zeros go out here, beside the leader's sort: a cluster barrier
    // waits for the stores before it.  The leader's own arrival does not wait for its
    // sort, so the other blocks leave as soon as their zeros are written; it reads no
    // other block's memory from here on.
    if (nr > 1 && rank == 0) cluster_arrive();
    if (nr > 1) zeros();
    if (nr > 1 && rank != 0) {
        cluster_arrive();
        cluster_wait();
        return;
    }
    __syncthreads();
    const unsigned found = min(sm->n_cand, (unsigned)kCand);
    if (found <= 256) {  // few: each counts those before it
        unsigned long long mine = 0;
        unsigned at = 0;
        if (tid < (int)found) {
            mine = sm->cand[tid];
#pragma unroll 8
            for (unsigned j = 0; j < found; j++) at += sm->cand[j] > mine;
        }
        __syncthreads();
        if (tid < (int)found) sm->cand[at] = mine;
        __syncthreads();
    } else if (found <= kVThreads) {
        sort_descending<1>(sm->cand, found);
    } else if (found <= 2 * kVThreads) {
        sort_descending<2>(sm->cand, found);
    } else {
        sort_descending<4>(sm->cand, found);
    }
    // k <= kMaxSurvivors = 2 kVThreads: thread i has ranks 2i and 2i + 1
    double e[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const unsigned r = 2 * tid + j;
        e[j] = r < k ? exp(((double)order_value((unsigned)(sm->cand[min(r, found - 1)] >> 32)) - (double)mx) / temp) : 0.0;
    }
    double total;
    const double before = block_scan_f64(e[0] + e[1], sm->wsum, total);
    bool stay[2] = {true, true};
    if (a.params.top_p > 0.0f && a.params.top_p < 1.0f) {
        stay[0] = before / total < (double)a.params.top_p;
        stay[1] = (before + e[0]) / total < (double)a.params.top_p;
        total = block_sum_f64((stay[0] ? e[0] : 0.0) + (stay[1] ? e[1] : 0.0), sm->wsum);
    }
    if (nr > 1) cluster_wait();  // the other blocks' zeros are written
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const unsigned r = 2 * tid + j;
        if (r < k && stay[j]) {
            const unsigned idx = ~(unsigned)sm->cand[r];
            a.probs[row * a.V + idx] = (float)(e[j] / total);
        }
    }
}

// ------------------------------------------------------------ verification
// Draft i of a stream (in order, i < count) is accepted when u_i q_i(d_i) <
// p_i(d_i), q the distribution it was drawn from (none: q = 1 at the draft).
// After a accepted drafts one more token is drawn by the inverse of the
// cumulative sum at u_K: from max(p_a - q_a, 0) when draft a was rejected
// (p_a without the draft when there is no q; p_a itself should nothing be
// left), from p_a when all passed.  The products and sums are in 64 bits, so
// that neither comparison turns on rounding.  Weights that are not positive
// (NaN among them) count as zero.  A stream of count -1 is idle: nothing of it is
// read, and it gets no token.
// 64 streams of 5 drafts at 151936: 24.8 us in a captured loop, 28 as one call among
// others (one row read where all pass, two where a
// draft is rejected: 58 MB).  What bounds it is the length of the chain (verdicts,
// sums, search), with one wave of blocks and eight loads of a thread in flight.
constexpr int kVocabMax = 1 << 30, kDraftsMax = 1 << 20;  // (indexes of a row stay in 32 bits)

struct VerifyArgs {
    const int *drafts, *counts;
    const float *draft_probs, *target_probs, *uniforms;
    int *tokens, *n_out, *err;
    int K, V, slice;
};

struct VerifySmem {
    double wsum[kVWarps], psum[kVWarps];
    double sum;
    int wlast[kVWarps], plast[kVWarps];
    int last;           // highest index with a positive weight, -1
    int accepted;       // drafts, -1: the stream is idle
    int count;
};

// VEC: rows and slices are multiples of 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(kVThreads) k_verify_drafts(const VerifyArgs a) {
    __shared__ VerifySmem sm;
    cg::cluster_group cl = cg::this_cluster();
    const unsigned rank = cl.block_rank(), nr = cl.num_blocks();
    auto meet = [&]() {  // all blocks of the stream
        if (nr == 1) __syncthreads();
        else cl.sync();
    };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t b = blockIdx.x;
    griddep_launch_dependents();
    griddep_wait();
    const float *target = a.target_probs + b * (a.K + 1) * a.V;
    const float *draft = a.draft_probs ? a.draft_probs + b * a.K * a.V : nullptr;
    const int *drafts = a.drafts + b * a.K;
    const float *u = a.uniforms + b * (a.K + 1);
    if (warp == 0) {
        int count = a.counts ? a.counts[b] : a.K;
        const bool idle = count == -1;
        if (count < 0 || count > a.K) {
            if (lane == 0 && rank == 0 && !idle) raise_error(a.err, kDevRange);
            count = count < 0 ? 0 : a.K;
        }
        int accepted = count;
        for (int i0 = 0; i0 < count; i0 += 32) {
            const int i = i0 + lane;
            bool ok = true;
            if (i < count) {
                const int d = drafts[i];
                ok = false;
                if ((unsigned)d < (unsigned)a.V) {
                    const double q = draft ? (double)draft[(int64_t)i * a.V + d] : 1.0;
                    ok = (double)u[i] * q < (double)target[(int64_t)i * a.V + d];
                } else {
                    raise_error(a.err, kDevRange);
                }
            }
            const unsigned no = __ballot_sync(0xffffffffu, !ok);
            if (no) {
                accepted = i0 + __ffs(no) - 1;
                break;
            }
        }
        if (lane == 0) {
            sm.accepted = idle ? -1 : accepted;
            sm.count = count;
        }
    }
    __syncthreads();
    const int acc = sm.accepted;
    if (acc < 0) {  // (the same in all blocks of the stream, and none has read another's memory)
        if (rank == 0) {
            for (int j = tid; j <= a.K; j += kVThreads) a.tokens[b * (a.K + 1) + j] = -1;
            if (tid == 0) a.n_out[b] = 0;
        }
        return;
    }
    const bool rejected = acc < sm.count;
    const float *p = target + (int64_t)acc * a.V;
    const float *q = rejected && draft ? draft + (int64_t)acc * a.V : nullptr;
    int without = rejected && !draft ? drafts[acc] : -1;
    // The block's slice, a contiguous run per warp.  Weights of 32 (VEC: 128)
    // neighbours at a time, eight loads of a lane in flight.
    constexpr int kStep = VEC ? 128 : 32;
    const int v0 = (int)rank * a.slice, n = max(0, min(a.slice, a.V - v0));
    const int run = ((n + kVWarps - 1) / kVWarps + kStep - 1) / kStep * kStep;
    auto weigh = [&](float pv, float qv, int i) {
        double w = (double)pv;
        if (q) w -= (double)qv;
        return w > 0.0 && i != without ? w : 0.0;
    };
    // sum of the weights in [i0, i1) over the lanes; `mine`: the lane's highest index with one
    auto sum_of = [&](int i0, int i1, int &mine) {
        double s = 0.0;
        if constexpr (VEC) {
            for (int i = i0 + 4 * lane; i < i1; i += 4 * kStep) {
                float4 pv[4], qv[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool in = i + j * kStep < i1;
                    pv[j] = in ? __ldg(reinterpret_cast<const float4 *>(p + i + j * kStep)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    qv[j] = in && q ? __ldg(reinterpret_cast<const float4 *>(q + i + j * kStep)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float pe[4] = {pv[j].x, pv[j].y, pv[j].z, pv[j].w}, qe[4] = {qv[j].x, qv[j].y, qv[j].z, qv[j].w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const double w = weigh(pe[e], qe[e], i + j * kStep + e);
                        if (w > 0.0) s += w, mine = i + j * kStep + e;
                    }
                }
            }
        } else {
            for (int i = i0 + lane; i < i1; i += 4 * kStep) {
                float pv[4], qv[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool in = i + j * kStep < i1;
                    pv[j] = in ? __ldg(p + i + j * kStep) : 0.0f;
                    qv[j] = in && q ? __ldg(q + i + j * kStep) : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const double w = weigh(pv[j], qv[j], i + j * kStep);
                    if (w > 0.0) s += w, mine = i + j * kStep;
                }
            }
        }
        return warp_sum_f64(s);
    };
    double base = 0.0, total = 0.0;
    int last = -1;
    for (int pass = 0; pass < 2; pass++) {
        int mine = -1;
        const double s = sum_of(v0 + min(n, warp * run), v0 + min(n, (warp + 1) * run), mine);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if (lane == 0) {
            sm.wsum[warp] = s;
            sm.wlast[warp] = mine;
        }
        __syncthreads();
        if (tid == 0) {
            double t = 0.0;
            int l = -1;
            for (int w = 0; w < kVWarps; w++) t += sm.wsum[w], l = max(l, sm.wlast[w]);
            sm.sum = t;
            sm.last = l;
        }
        meet();
        base = total = 0.0;
        last = -1;
        double sums[kMaxCluster];
        int lasts[kMaxCluster];
#pragma unroll
        for (unsigned r = 0; r < kMaxCluster; r++) {  // (reads in flight together)
            const VerifySmem *o = nr == 1 ? &sm : cl.map_shared_rank(&sm, r < nr ? r : 0);
            sums[r] = r < nr ? o->sum : 0.0;
            lasts[r] = r < nr ? o->last : -1;
        }
#pragma unroll
        for (unsigned r = 0; r < kMaxCluster; r++) {
            if (r == rank) base = total;
            total += sums[r];
            last = max(last, lasts[r]);
        }
        if (total > 0.0 || !rejected || pass) break;
        q = nullptr;  // nothing is left of the difference: draw from the target
        without = -1;
        meet();
    }
    // The first index whose cumulative sum passes goal.  Warp w of a block has
    // [base + pre[w], base + pre[w + 1]) of the line of sums, base and pre the
    // same numbers for neighbours, so one warp's run in the cluster has the goal.
    // The block of that run searches it together: each warp sums a piece, the
    // piece that has the goal is scanned.
    const double goal = fmax((double)u[a.K] * total, 0.0);
    if (base <= goal && goal < base + sm.sum) {
        double lo = base;
        int at = 0;
        {
            double pre = 0.0;
            for (int w = 0; w < kVWarps; w++) {
                const double next = pre + sm.wsum[w];
                if (base + pre <= goal && goal < base + next) lo = base + pre, at = w;
                pre = next;
            }
        }
        const int r0 = v0 + min(n, at * run), r1 = v0 + min(n, (at + 1) * run);
        // (a short run is the one piece that there is)
        const int piece = run <= 512 ? run : ((r1 - r0 + kVWarps - 1) / kVWarps + kStep - 1) / kStep * kStep;
        const int p0 = min(r1, r0 + warp * piece), p1 = min(r1, r0 + (warp + 1) * piece);
        if (run > 512) {
            int mine = -1;
            const double s = sum_of(p0, p1, mine);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
            if (lane == 0) {
                sm.psum[warp] = s;
                sm.plast[warp] = mine;
            }
        } else if (lane == 0) {
            sm.psum[warp] = 0.0;
            sm.plast[warp] = warp == 0 ? sm.wlast[at] : -1;
        }
        __syncthreads();
        // (should the pieces' sums round below the run's, its last piece with a weight has the goal)
        double pre = lo;
        int who = -1;
        double from = lo;
        for (int w = 0; w < kVWarps; w++) {
            if (sm.plast[w] >= 0 && (who < 0 || pre <= goal)) who = w, from = pre;
            pre += sm.psum[w];
        }
        if (warp == who) {
            double sum = from;
            int token = -1;
            for (int i0 = p0; i0 < p1 && token < 0; i0 += 32) {
                const int i = i0 + lane;
                const double w = i < p1 ? weigh(__ldg(p + i), q ? __ldg(q + i) : 0.0f, i) : 0.0;
                double x = w;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && sum + x > goal);
                if (hit) token = i0 + __ffs(hit) - 1;
                sum += __shfl_sync(0xffffffffu, x, 31);
            }
            // a scan that rounds below its share's end has the piece's last token
            if (lane == 0) a.tokens[b * (a.K + 1) + acc] = token >= 0 ? token : sm.plast[warp];
        }
    }
    if (rank == 0) {
        for (int j = tid; j <= a.K; j += kVThreads)
            if (j != acc) a.tokens[b * (a.K + 1) + j] = j < acc ? drafts[j] : -1;
        if (tid == 0) {
            a.n_out[b] = acc + 1;
            if (!(goal < total)) a.tokens[b * (a.K + 1) + acc] = max(last, 0);  // u >= 1, or no weight at all
        }
    }
    meet();  // no block leaves while another reads its sums
}

// Blocks of one row's cluster: a slice per block of at most `most`, at least 1.
int cluster_for(int V, int most) {
    int nr = 1;
    while (nr < kMaxCluster && (V + nr - 1) / nr > most) nr <<= 1;
    return nr;
}

}  // namespace

}  // namespace qora

using namespace qora;

extern "C" {

int qora_sample_probs(qora_ctx *ctx, const float *logits, int32_t B, int32_t V, const uint32_t *prev,
                      int32_t n_prev, const qora_sample_params *params, float *probs, void *stream) {
    if (!ctx || !logits || !params || !probs || B <= 0 || V <= 0 || n_prev < 0 || (n_prev > 0 && !prev))
        return set_error(QORA_ERR_INVALID, "qora_sample_probs: bad arguments");
    if (V > kMaxCluster * kSliceMax)
        return set_error(QORA_ERR_UNSUPPORTED, "qora_sample_probs: vocab %d (max %d)", V, kMaxCluster * kSliceMax);
    const bool topk = params->top_k > 0 && params->top_k < V;
    if (topk && params->top_k > kMaxSurvivors)
        return set_error(QORA_ERR_UNSUPPORTED, "top_k %d > %d", params->top_k, kMaxSurvivors);
    if (!topk && params->top_p > 0.0f && params->top_p < 1.0f)
        return set_error(QORA_ERR_UNSUPPORTED, "top_p needs 0 < top_k <= %d", kMaxSurvivors);
    DeviceGuard dg;
    QORA_TRY(dg.set(ctx->device));
    const int nr = cluster_for(V, 20480);
    const bool vec = V % 4 == 0 && !((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(probs)) & 15);
    ProbsArgs a;
    a.logits = logits;
    a.prev = n_prev ? prev : nullptr;
    a.probs = probs;
    a.err = ctx->err.as<int>();
    a.V = V;
    a.n_prev = n_prev;
    a.slice = ((V + nr - 1) / nr + 3) / 4 * 4;
    a.params = *params;
    // threads that hold a logit, at least: half of them, or of their groups of which
    // there are four, have to be enough for top_k (fewer maxima are quicker: 160 rows
    // of 2048 with 50 take 7.3 us by one a thread, 7.6 by four; with 1000 of 512 rows,
    // where one is not enough, 44 us by four and 60 without)
    const auto holders = [](int64_t logits) { return logits / 4 < kVThreads ? logits / 4 : kVThreads; };
    const int64_t held = nr == 1 ? holders(V) : (nr - 1) * holders(a.slice);
    a.by_maxima = !topk ? 0 : params->top_k <= held / 2 ? 1 : params->top_k <= 2 * held ? 4 : 0;
    const size_t smem = sizeof(ProbsSmem) + (size_t)a.slice * 4;
    auto kern = vec ? k_sample_probs<true> : k_sample_probs<false>;
    static std::atomic<uint64_t> done[2];
    QORA_TRY(allow_smem(kern, sizeof(ProbsSmem) + kSliceMax * 4, ctx->device, done[vec]));
    return launch_ex(kern, dim3(B, nr), dim3(kVThreads), smem, as_stream(stream), (unsigned)nr, a);
}

int qora_verify_drafts(qora_ctx *ctx, const int32_t *drafts, const float *draft_probs, const float *target_probs,
                       const int32_t *counts, const float *uniforms, int32_t B, int32_t K, int32_t V,
                       int32_t *tokens, int32_t *n_out, void *stream) {
    if (!ctx || !target_probs || !uniforms || !tokens || !n_out || B <= 0 || K < 0 || V <= 0 || (K > 0 && !drafts))
        return set_error(QORA_ERR_INVALID, "qora_verify_drafts: bad arguments");
    if (V > kVocabMax || K > kDraftsMax)
        return set_error(QORA_ERR_UNSUPPORTED, "qora_verify_drafts: %d drafts (max %d), vocab %d (max %d)", K, kDraftsMax,
                         V, kVocabMax);
    DeviceGuard dg;
    QORA_TRY(dg.set(ctx->device));
    // Wide rows go to a cluster, as wide as leaves all streams running at once (two
    // blocks a multiprocessor): 64 streams of 151936 took 37 us with clusters of 8,
    // in two waves.
    int nr = cluster_for(V, 8192);
    while (nr > 1 && (int64_t)B * nr > 2 * ctx->num_sms) nr >>= 1;
    VerifyArgs a;
    a.drafts = drafts;
    a.counts = counts;
    a.draft_probs = draft_probs;
    a.target_probs = target_probs;
    a.uniforms = uniforms;
    a.tokens = tokens;
    a.n_out = n_out;
    a.err = ctx->err.as<int>();
    a.K = K;
    a.V = V;
    a.slice = (int)((((int64_t)V + nr - 1) / nr + 3) / 4 * 4);
    const bool vec = V % 4 == 0 && !((reinterpret_cast<uintptr_t>(target_probs) | reinterpret_cast<uintptr_t>(draft_probs)) & 15);
    auto kern = vec ? k_verify_drafts<true> : k_verify_drafts<false>;
    return launch_ex(kern, dim3(B, nr), dim3(kVThreads), 0, as_stream(stream), (unsigned)nr, a);
}

}  // extern "C"
