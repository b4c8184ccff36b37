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
// The row's slice stays in shared memory after one read.  The kept tokens are
// found by a histogram of max - x in steps of 1/32 (few tokens lie near the
// top, so its counters are hardly contended), and only tokens down to the bin
// that holds the top_k-th are sorted; when that bin is too full (many equal
// logits) a radix selection over the slices decides exactly.  Exponentials and
// sums of the kept are in 64 bits: the order and the top_p border are decided
// by values next to each other.
constexpr int kBins = 2048;
constexpr int kCand = 2048;          // candidates that one sort takes
constexpr int kSliceMax = 40960;     // logits of a slice in shared memory

struct ProbsArgs {
    const float *logits;
    const uint32_t *prev;
    float *probs;
    int *err;
    int V, n_prev, slice;
    qora_sample_params params;
};

struct ProbsSmem {
    unsigned hist[kBins];
    unsigned long long cand[kCand];   // order key of x, then ~index
    double wsum[kVWarps + 1];
    float red[kVWarps];
    float mx, slice_max;
    int bad, slice_bad;
    unsigned n_cand, eq_before;
    unsigned sel_bin, sel_below, sel_in;
    double sum, slice_sum;
    unsigned eq_count;
};

// Order of f32 values as unsigned integers.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = __float_as_uint(x);
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

// The bin (or digit) of a histogram of the whole row in which the count from
// its start reaches `need`: hist bins are summed over the cluster's blocks.
// Called by warp 0 of every block; writes sel_bin / sel_below / sel_in.
template <bool DESC>
__device__ __forceinline__ void select_bin(cg::cluster_group &cl, ProbsSmem *sm, int bins, unsigned need) {
    const int lane = threadIdx.x & 31;
    const unsigned nr = cl.num_blocks();
    unsigned below = 0;
    for (int b0 = 0; b0 < bins; b0 += 32) {
        const int bin = DESC ? bins - 1 - (b0 + lane) : b0 + lane;
        unsigned c = 0;
        for (unsigned r = 0; r < nr; r++) c += cl.map_shared_rank(sm, r)->hist[bin];
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

__global__ void __launch_bounds__(kVThreads) k_sample_probs(const ProbsArgs a) {
    extern __shared__ uint4 dyn[];
    ProbsSmem *sm = reinterpret_cast<ProbsSmem *>(dyn);
    float *x = reinterpret_cast<float *>(sm + 1);
    cg::cluster_group cl = cg::this_cluster();
    const unsigned rank = cl.block_rank(), nr = cl.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const int v0 = (int)rank * a.slice, n = max(0, min(a.slice, a.V - v0));
    griddep_launch_dependents();
    griddep_wait();
    const float *in = a.logits + row * a.V + v0;
    float *out = a.probs + row * a.V + v0;
    for (int i = tid; i < n; i += kVThreads) x[i] = __ldg(in + i);
    __syncthreads();
    // penalty: the first mention of a token applies all of them
    if (a.prev && a.params.repetition_penalty != 1.0f) {
        const uint32_t *prev = a.prev + row * a.n_prev;
        for (int j = tid; j < a.n_prev; j += kVThreads) {
            const uint32_t tok = prev[j];
            if (tok >= (unsigned)a.V || (int)tok < v0 || (int)tok >= v0 + n) continue;
            bool first = true;
            for (int i = 0; i < j && first; i++) first = prev[i] != tok;
            if (!first) continue;
            float y = x[tok - v0];
            for (int i = j; i < a.n_prev; i++)
                if (prev[i] == tok) y = y > 0.0f ? __fdiv_rn(y, a.params.repetition_penalty)
                                                 : __fmul_rn(y, a.params.repetition_penalty);
            x[tok - v0] = y;
        }
        __syncthreads();
    }
    // maximum of the row
    float mx = -INFINITY;
    bool nan = false;
    for (int i = tid; i < n; i += kVThreads) {
        mx = fmaxf(mx, x[i]);
        nan = nan || x[i] != x[i];
    }
    mx = warp_max(mx);
    if (lane == 0) sm->red[warp] = mx;
    nan = __syncthreads_or(nan);
    if (tid == 0) {
        for (int w = 0; w < kVWarps; w++) mx = fmaxf(mx, sm->red[w]);
        sm->slice_max = mx;
        sm->slice_bad = nan;
        sm->n_cand = 0;
    }
    for (int i = tid; i < kBins; i += kVThreads) sm->hist[i] = 0;
    cl.sync();
    if (tid == 0) {
        float m = -INFINITY;
        int bad = 0;
        for (unsigned r = 0; r < nr; r++) {
            m = fmaxf(m, cl.map_shared_rank(sm, r)->slice_max);
            bad |= cl.map_shared_rank(sm, r)->slice_bad;
        }
        sm->mx = m;
        sm->bad = bad || !isfinite(m);
    }
    __syncthreads();
    mx = sm->mx;
    const bool bad = sm->bad;
    const double temp = a.params.temperature > 0.0f ? (double)a.params.temperature : 1.0;
    const bool topk = a.params.top_k > 0 && a.params.top_k < a.V;
    if (bad) {  // NaN or +inf among the logits, or none that is finite
        if (tid == 0 && rank == 0) raise_error(a.err, kDevNaN);
        for (int i = tid; i < n; i += kVThreads) out[i] = 0.0f;
        cl.sync();  // no block leaves while another reads its slice_max
        return;
    }
    if (!topk) {
        double s = 0.0;
        const double per = 1.0 / temp;
        for (int i = tid; i < n; i += kVThreads) {
            const float e = expf((float)(((double)x[i] - (double)mx) * per));
            x[i] = e;
            s += e;
        }
        s = block_sum_f64(s, sm->wsum);
        if (tid == 0) sm->slice_sum = s;
        cl.sync();
        if (tid == 0) {
            double t = 0.0;
            for (unsigned r = 0; r < nr; r++) t += cl.map_shared_rank(sm, r)->slice_sum;
            sm->sum = 1.0 / t;
        }
        __syncthreads();
        const double inv = sm->sum;
        for (int i = tid; i < n; i += kVThreads) out[i] = (float)(x[i] * inv);
        cl.sync();
        return;
    }
    const unsigned k = a.params.top_k;
    auto bin_of = [&](float v) { return (int)fminf((mx - v) * 32.0f, (float)(kBins - 1)); };
    for (int i = tid; i < n; i += kVThreads) {
        atomicAdd(&sm->hist[bin_of(x[i])], 1u);
        out[i] = 0.0f;
    }
    cl.sync();
    if (warp == 0) select_bin<false>(cl, sm, kBins, k);
    __syncthreads();
    const int sel = sm->sel_bin;
    const bool few = sm->sel_below + sm->sel_in <= kCand;
    ProbsSmem *lead = cl.map_shared_rank(sm, 0);
    auto offer = [&](int i) {
        const unsigned at = atomicAdd(&lead->n_cand, 1u);
        if (at < kCand)
            lead->cand[at] = ((unsigned long long)order_key(x[i]) << 32) | (unsigned)~(unsigned)(v0 + i);
    };
    cl.sync();  // every block has read the histograms
    if (few) {
        for (int i = tid; i < n; i += kVThreads)
            if (bin_of(x[i]) <= sel) offer(i);
    } else {
        // radix selection of the k-th key, 8 bits at a time
        unsigned prefix = 0, mask = 0, need = k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kVThreads) sm->hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kVThreads) {
                const unsigned key = order_key(x[i]);
                if ((key & mask) == prefix) atomicAdd(&sm->hist[(key >> shift) & 255u], 1u);
            }
            cl.sync();
            if (warp == 0) select_bin<true>(cl, sm, 256, need);
            __syncthreads();
            prefix |= sm->sel_bin << shift;
            mask |= 255u << shift;
            need -= sm->sel_below;
            cl.sync();
        }
        // keys above the k-th are kept, and the first `need` equal to it in index order
        unsigned eq = 0;
        for (int i = tid; i < n; i += kVThreads) eq += order_key(x[i]) == prefix;
        eq = (unsigned)block_sum_f64((double)eq, sm->wsum);
        if (tid == 0) sm->eq_count = eq;
        cl.sync();
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
    }
    cl.sync();
    if (rank != 0) return;  // the rest is the leader's; it reads no other block's memory
    const unsigned found = min(sm->n_cand, (unsigned)kCand);
    int size = 32;
    while (size < (int)found) size <<= 1;
    for (int i = found + tid; i < size; i += kVThreads) sm->cand[i] = 0ull;
    __syncthreads();
    // descending bitonic sort
    for (int span = 2; span <= size; span <<= 1)
        for (int step = span >> 1; step > 0; step >>= 1) {
            for (int i = tid; i < size / 2; i += kVThreads) {
                const int lo = (i / step) * step * 2 + (i % step), hi = lo + step;
                const unsigned long long p = sm->cand[lo], q = sm->cand[hi];
                const bool down = (lo & span) == 0;
                if ((p < q) == down) sm->cand[lo] = q, sm->cand[hi] = p;
            }
            __syncthreads();
        }
    // k <= kMaxSurvivors = 2 kVThreads: thread i has ranks 2i and 2i + 1
    double e[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const unsigned r = 2 * tid + j;
        e[j] = r < k ? exp(((double)order_value((unsigned)(sm->cand[min(r, (unsigned)size - 1)] >> 32)) - (double)mx) / temp) : 0.0;
    }
    double total;
    const double before = block_scan_f64(e[0] + e[1], sm->wsum, total);
    bool stay[2] = {true, true};
    if (a.params.top_p > 0.0f && a.params.top_p < 1.0f) {
        stay[0] = before / total < (double)a.params.top_p;
        stay[1] = (before + e[0]) / total < (double)a.params.top_p;
        total = block_sum_f64((stay[0] ? e[0] : 0.0) + (stay[1] ? e[1] : 0.0), sm->wsum);
    }
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
// (NaN among them) count as zero.
struct VerifyArgs {
    const int *drafts, *counts;
    const float *draft_probs, *target_probs, *uniforms;
    int *tokens, *n_out, *err;
    int K, V, slice;
};

struct VerifySmem {
    double wsum[kVWarps + 1];
    double sum;
    int last;           // highest index with a positive weight, -1
    int accepted;
    int count;
};

__global__ void __launch_bounds__(kVThreads) k_verify_drafts(const VerifyArgs a) {
    __shared__ VerifySmem sm;
    cg::cluster_group cl = cg::this_cluster();
    const unsigned rank = cl.block_rank(), nr = cl.num_blocks();
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
        if (count < 0 || count > a.K) {
            if (lane == 0 && rank == 0) raise_error(a.err, kDevRange);
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
            sm.accepted = accepted;
            sm.count = count;
        }
    }
    __syncthreads();
    const int acc = sm.accepted;
    const bool rejected = acc < sm.count;
    const float *p = target + (int64_t)acc * a.V;
    const float *q = rejected && draft ? draft + (int64_t)acc * a.V : nullptr;
    int without = rejected && !draft ? drafts[acc] : -1;
    // the block's slice, a contiguous run per warp
    const int v0 = (int)rank * a.slice, n = max(0, min(a.slice, a.V - v0));
    const int run = ((n + kVWarps - 1) / kVWarps + 31) / 32 * 32;
    const int r0 = v0 + min(n, warp * run), r1 = v0 + min(n, (warp + 1) * run);
    double base = 0.0, total = 0.0;
    int last = -1;
    for (int pass = 0; pass < 2; pass++) {
        double s = 0.0;
        int mine = -1;
        for (int i = r0 + lane; i < r1; i += 32) {
            double w = (double)__ldg(p + i);
            if (q) w -= (double)__ldg(q + i);
            if (w > 0.0 && i != without) s += w, mine = i;
        }
        s = warp_sum_f64(s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if (tid == 0) sm.last = -1;
        __syncthreads();
        if (lane == 0) {
            sm.wsum[warp] = s;
            atomicMax(&sm.last, mine);
        }
        __syncthreads();
        if (tid == 0) {
            double t = 0.0;
            for (int w = 0; w < kVWarps; w++) t += sm.wsum[w];
            sm.sum = t;
        }
        cl.sync();
        base = total = 0.0;
        last = -1;
        for (unsigned r = 0; r < nr; r++) {
            const VerifySmem *o = cl.map_shared_rank(&sm, r);
            if (r == rank) base = total;
            total += o->sum;
            last = max(last, o->last);
        }
        if (total > 0.0 || !rejected || pass) break;
        q = nullptr;  // nothing is left of the difference: draw from the target
        without = -1;
        cl.sync();
    }
    // The first index whose cumulative sum passes goal.  Warp w of a block has
    // [base + pre[w], base + pre[w + 1]) of the line of sums, base and pre the
    // same numbers for neighbours, so one warp of the cluster has the goal.
    const double goal = fmax((double)u[a.K] * total, 0.0);
    double pre = 0.0;
    for (int w = 0; w < warp; w++) pre += sm.wsum[w];
    const double lo = base + pre, hi = base + (pre + sm.wsum[warp]);
    if (lo <= goal && goal < hi) {
        double at = lo;
        int token = -1, highest = -1;
        for (int i0 = r0; i0 < r1 && token < 0; i0 += 32) {
            const int i = i0 + lane;
            double w = 0.0;
            if (i < r1) {
                w = (double)__ldg(p + i);
                if (q) w -= (double)__ldg(q + i);
                if (!(w > 0.0) || i == without) w = 0.0;
            }
            double x = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
            const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && at + x > goal);
            if (some) highest = i0 + 31 - __clz(some);
            if (hit) token = i0 + __ffs(hit) - 1;
            at += __shfl_sync(0xffffffffu, x, 31);
        }
        // the run's own sum may round below its share's end: then its last token
        if (lane == 0) a.tokens[b * (a.K + 1) + acc] = token >= 0 ? token : highest;
    }
    if (rank == 0) {
        for (int j = tid; j <= a.K; j += kVThreads)
            if (j != acc) a.tokens[b * (a.K + 1) + j] = j < acc ? drafts[j] : -1;
        if (tid == 0) {
            a.n_out[b] = acc + 1;
            if (!(goal < total)) a.tokens[b * (a.K + 1) + acc] = max(last, 0);  // u >= 1, or no weight at all
        }
    }
    cl.sync();  // no block leaves while another reads its sums
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
    ProbsArgs a;
    a.logits = logits;
    a.prev = n_prev ? prev : nullptr;
    a.probs = probs;
    a.err = ctx->err.as<int>();
    a.V = V;
    a.n_prev = n_prev;
    a.slice = (V + nr - 1) / nr;
    a.params = *params;
    const size_t smem = sizeof(ProbsSmem) + (size_t)a.slice * 4;
    QORA_CUDA(cudaFuncSetAttribute(k_sample_probs, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)(sizeof(ProbsSmem) + kSliceMax * 4)));
    return launch_ex(k_sample_probs, dim3(B, nr), dim3(kVThreads), smem, as_stream(stream), (unsigned)nr, a);
}

int qora_verify_drafts(qora_ctx *ctx, const int32_t *drafts, const float *draft_probs, const float *target_probs,
                       const int32_t *counts, const float *uniforms, int32_t B, int32_t K, int32_t V,
                       int32_t *tokens, int32_t *n_out, void *stream) {
    if (!ctx || !target_probs || !uniforms || !tokens || !n_out || B <= 0 || K < 0 || V <= 0 || (K > 0 && !drafts))
        return set_error(QORA_ERR_INVALID, "qora_verify_drafts: bad arguments");
    DeviceGuard dg;
    QORA_TRY(dg.set(ctx->device));
    const int nr = cluster_for(V, 8192);
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
    a.slice = (int)(((int64_t)V + nr - 1) / nr);
    return launch_ex(k_verify_drafts, dim3(B, nr), dim3(kVThreads), 0, as_stream(stream), (unsigned)nr, a);
}

}  // extern "C"
