// The 4-bit paged KV cache: creation, block tables and slot maps built on the
// GPU (k_kv4_reserve), the append with qk-norm and rotation (k_kv4_append),
// plain writes and reads of rows, and the length update.
#include "kv4.cuh"

#include <new>

namespace qora {

namespace {

// ------------------------------------------------------------ block tables
// Maps pages for counts[b] new tokens of every stream and lists the tokens.
// A page is free when no stream's table entry below ceil(len / page) names it:
// the entries are marked in a bit map, whose zero bits in ascending order go
// to the new (stream, logical page) pairs in lexicographic order.  Nothing
// but lengths and table is kept between calls, so pages behind a length that
// was rolled back are free again, and a call repeated before the lengths move
// gives the same answer.
constexpr int kResThreads = 1024;

struct ReserveArgs {
    const int *counts, *len;
    int *table, *slots, *positions, *offsets, *err;
    int streams, max_pos, page_shift, pages_per_stream, pool_pages, max_tokens;
};

__device__ __forceinline__ int block_scan_excl(int v, int *wsum, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = wsum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        wsum[lane] = w;
    }
    __syncthreads();
    total = wsum[31];
    return x - v + (warp ? wsum[warp - 1] : 0);
}

__global__ void __launch_bounds__(kResThreads) k_kv4_reserve(const ReserveArgs a) {
    extern __shared__ unsigned bits[];  // one bit per pool page: in use
    __shared__ int wsum[32];
    __shared__ int bad;
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = (a.pool_pages + 31) >> 5;
    const int P = 1 << a.page_shift;
    if (tid == 0) bad = 0;
    for (int w = tid; w < words; w += kResThreads) bits[w] = 0u;
    __syncthreads();
    // mark, one warp per stream
    for (int b = warp; b < a.streams; b += kResThreads / 32) {
        const int len = a.len[b], n = a.counts[b];
        if (len < 0 || n < 0 || len > a.max_pos || n > a.max_pos - len) {
            if (lane == 0) atomicMax(&bad, kDevRange);
            continue;
        }
        const int keep = (len + P - 1) >> a.page_shift;
        for (int j = lane; j < keep; j += 32) {
            const int pg = a.table[(int64_t)b * a.pages_per_stream + j];
            if (pg < 0 || pg >= a.pool_pages) atomicMax(&bad, kDevRange);
            else atomicOr(&bits[pg >> 5], 1u << (pg & 31));
        }
    }
    __syncthreads();
    // totals: tokens and new pages
    int64_t tokens = 0;
    int need = 0, free_total = 0;
    if (!bad) {
        for (int b0 = 0; b0 < a.streams; b0 += kResThreads) {
            const int b = b0 + tid;
            int n = 0, k = 0;
            if (b < a.streams) {
                n = a.counts[b];
                k = ((a.len[b] + n + P - 1) >> a.page_shift) - ((a.len[b] + P - 1) >> a.page_shift);
            }
            int t;
            block_scan_excl(n, wsum, t);
            tokens += t;
            block_scan_excl(k, wsum, t);
            need += t;
        }
        for (int w0 = 0; w0 < words; w0 += kResThreads) {
            const int w = w0 + tid;
            int f = 0;
            if (w < words) {
                f = __popc(~bits[w]);
                if (w == words - 1 && (a.pool_pages & 31)) f -= 32 - (a.pool_pages & 31);
            }
            int t;
            block_scan_excl(f, wsum, t);
            free_total += t;
        }
    }
    const int why = bad ? bad : tokens > a.max_tokens ? kDevRange : need > free_total ? kDevPool : 0;
    if (why) {  // nothing is mapped, and every listed token is skipped
        if (tid == 0) raise_error(a.err, why);
        for (int b = tid; b <= a.streams; b += kResThreads) a.offsets[b] = 0;
        for (int i = tid; i < a.max_tokens; i += kResThreads) {
            a.slots[i] = -1;
            a.positions[i] = 0;
        }
        return;
    }
    // the new pages: the i-th free page goes to the i-th new (stream, page)
    __syncthreads();
    int page_base = 0, tok_base = 0;
    // (a) offsets, and each stream's first new page in ordinal order
    for (int b0 = 0; b0 < a.streams; b0 += kResThreads) {
        const int b = b0 + tid;
        int n = 0;
        if (b < a.streams) n = a.counts[b];
        int t;
        const int at = block_scan_excl(n, wsum, t);
        if (b < a.streams) a.offsets[b] = tok_base + at;
        tok_base += t;
    }
    if (tid == 0) a.offsets[a.streams] = tok_base;
    // (b) free pages in ascending order: thread w hands out its word's pages
    for (int w0 = 0; w0 < words; w0 += kResThreads) {
        const int w = w0 + tid;
        unsigned f = w < words ? ~bits[w] : 0u;
        if (w == words - 1 && (a.pool_pages & 31)) f &= (1u << (a.pool_pages & 31)) - 1u;
        int t;
        int at = page_base + block_scan_excl(__popc(f), wsum, t);
        page_base += t;
        while (f && at < need) {
            const int pg = w * 32 + __ffs(f) - 1;
            f &= f - 1;
            // the stream that owns ordinal `at`: a walk over the streams' needs
            int rest = at;
            for (int b = 0; b < a.streams; b++) {
                const int len = a.len[b];
                const int keep = (len + P - 1) >> a.page_shift;
                const int k = ((len + a.counts[b] + P - 1) >> a.page_shift) - keep;
                if (rest < k) {
                    a.table[(int64_t)b * a.pages_per_stream + keep + rest] = pg;
                    break;
                }
                rest -= k;
            }
            at++;
        }
    }
    __syncthreads();
    // (c) the tokens' slots and positions, one warp per stream
    for (int b = warp; b < a.streams; b += kResThreads / 32) {
        const int len = a.len[b], n = a.counts[b], off = a.offsets[b];
        for (int i = lane; i < n; i += 32) {
            const int pos = len + i;
            const int pg = a.table[(int64_t)b * a.pages_per_stream + (pos >> a.page_shift)];
            a.slots[off + i] = (pg << a.page_shift) + (pos & (P - 1));
            a.positions[off + i] = pos;
        }
    }
    for (int i = tok_base + tid; i < a.max_tokens; i += kResThreads) {
        a.slots[i] = -1;
        a.positions[i] = 0;
    }
}

// lengths += counts (negative counts roll back)
__global__ void k_kv4_advance(int *len, const int *counts, int streams, int max_pos, int *err) {
    griddep_launch_dependents();
    griddep_wait();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= streams) return;
    const int64_t to = (int64_t)len[b] + counts[b];
    if (to < 0 || to > max_pos) raise_error(err, kDevRange);
    len[b] = (int)(to < 0 ? 0 : to > max_pos ? max_pos : to);
}

// ------------------------------------------------------------ rows
// A warp holds one head vector: lane l has dimensions E l + e (e < E = D/64)
// of the first half and the same of the second half, so the rotation's pairs
// (i, i + D/2) lie in one lane.
template <int D>
struct HeadVec {
    static constexpr int E = D / 64;
    float x[2][E];

    __device__ __forceinline__ void load(const float *p, int lane) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < E; e++) x[h][e] = p[h * (D / 2) + E * lane + e];
    }
    __device__ __forceinline__ void store(float *p, int lane) const {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < E; e++) p[h * (D / 2) + E * lane + e] = x[h][e];
    }

    // RMS norm over the head and rotation by the position's angles.  In 64
    // bits: a key's 4-bit codes are decided next to borders, where the f32
    // rounding of these sums would move one code in a million by a whole step.
    // The result is rounded to f32 once.
    __device__ __forceinline__ void norm_rope(const __half *gamma, const float *cs, const float *sn, int lane) {
        double ss = 0.0;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < E; e++) ss += (double)x[h][e] * (double)x[h][e];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const double inv = 1.0 / sqrt(ss / D + 1e-6);
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int i = E * lane + e;
            const double a = (double)x[0][e] * inv * (double)__half2float(gamma[i]);
            const double b = (double)x[1][e] * inv * (double)__half2float(gamma[i + D / 2]);
            const double c = cs[i], s = sn[i];
            x[0][e] = (float)(a * c - b * s);
            x[1][e] = (float)(b * c + a * s);
        }
    }

    // Quantises and writes the row as position r of the unit.
    template <bool V>
    __device__ __forceinline__ void store4(uint8_t *unit, int r, int lane) const {
        using U = Kv4Unit<D>;
        constexpr int kGroupLanes = 32 / E;  // lanes of one scale group
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float amax = 0.0f;
            bool fin = true;
#pragma unroll
            for (int e = 0; e < E; e++) {
                amax = fmaxf(amax, fabsf(x[h][e]));
                fin = fin && isfinite(x[h][e]);
            }
            if (!fin) amax = INFINITY;
#pragma unroll
            for (int o = kGroupLanes / 2; o > 0; o >>= 1)
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            // f32 division by 7 then f16 rounding equals rounding amax / 7 once:
            // no f32 neighbour of 7m has a quotient that rounds to the 12-bit m
            __half sh = __float2half_rn(fminf(__fdiv_rn(amax, 7.0f), 65504.0f));
            if (!isfinite(amax)) sh = __ushort_as_half((unsigned short)0x7e00);
            const float s = __half2float(sh);
            const bool live = s > 0.0f && isfinite(amax);
            const float inv = live ? __fdiv_rn(1.0f, s) : 0.0f;
            unsigned nib = 0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                // nearest integer to x / s: rint of the approximate quotient is off
                // by one at most; x - q s is exact in f32 and decides
                float q = 0.0f;
                if (live) {
                    const float v = x[h][e];
                    q = rintf(fminf(fmaxf(v * inv, -8.0f), 8.0f));
                    const float rest = 2.0f * fmaf(-q, s, v);
                    if (rest > s || (rest == s && ((int)q & 1))) q += 1.0f;
                    else if (rest < -s || (rest == -s && ((int)q & 1))) q -= 1.0f;
                    q = fminf(fmaxf(q, -7.0f), 7.0f);
                }
                nib |= (unsigned)((int)q + 8) << (4 * e);
            }
            const int dim = h * (D / 2) + E * lane;
            constexpr int kLanes = (V ? 4 : 8) / E;  // lanes of one stored word / halfword
            nib <<= 4 * E * (lane & (kLanes - 1));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) nib |= __shfl_xor_sync(0xffffffffu, nib, o);
            if ((lane & (kLanes - 1)) == 0) {
                if (V) *reinterpret_cast<uint16_t *>(unit + U::v_half(r, dim)) = (uint16_t)nib;
                else *reinterpret_cast<uint32_t *>(unit + U::k_word(r, dim)) = nib;
            }
            if ((lane & (kGroupLanes - 1)) == 0)
                *reinterpret_cast<__half *>(unit + (V ? U::v_scale(r, dim >> 5) : U::k_scale(r, dim >> 5))) = sh;
        }
    }

    template <bool V>
    __device__ __forceinline__ void load4(const uint8_t *unit, int r, int lane) {
        using U = Kv4Unit<D>;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int dim = h * (D / 2) + E * lane;
            const float s = __half2float(
                *reinterpret_cast<const __half *>(unit + (V ? U::v_scale(r, dim >> 5) : U::k_scale(r, dim >> 5))));
            const unsigned w = V ? (unsigned)*reinterpret_cast<const uint16_t *>(unit + U::v_half(r, dim))
                                 : *reinterpret_cast<const uint32_t *>(unit + U::k_word(r, dim));
#pragma unroll
            for (int e = 0; e < E; e++)
                x[h][e] = s * (float)((int)((w >> (4 * ((dim + e) & (V ? 3 : 7)))) & 15u) - 8);
        }
    }
};

constexpr int kRowWarps = 8;

struct RowArgs {
    Kv4Layer L;
    const float *qkv;                       // append: [n][(heads + 2 kvh) D]
    const float *k_in, *v_in;               // write: [n][kvh D]
    float *q_out, *k_out, *v_out;
    const __half *q_gamma, *k_gamma;
    const float *cos, *sin;
    const int *positions, *slots;
    int heads, rows, rope_max, *err;
};

// Whether row i is to be handled; its unit and place in it.
__device__ __forceinline__ bool row_place(const RowArgs &a, int i, int &page, int &unit, int &r) {
    const int slot = a.slots[i];
    if (slot == -1) return false;  // a row behind the last token
    if (slot < 0 || (slot >> a.L.page_shift) >= a.L.pool_pages) {
        raise_error(a.err, kDevRange);
        return false;
    }
    const int in_page = slot & ((1 << a.L.page_shift) - 1);
    page = slot >> a.L.page_shift;
    unit = in_page >> 5;
    r = in_page & 31;
    return true;
}

// One warp per (row, head): q heads are normed, rotated and stored in f32; k
// heads normed, rotated and stored in 4 bits; v heads stored in 4 bits.
template <int D>
__global__ void __launch_bounds__(kRowWarps * 32) k_kv4_append(const RowArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int per = a.heads + 2 * a.L.kvh;
    const int64_t task = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    const int i = (int)(task / per), h = (int)(task % per);
    if (i >= a.rows) return;
    int page, unit, r;
    if (!row_place(a, i, page, unit, r)) return;
    const int pos = a.positions[i];
    if (pos < 0 || pos >= a.rope_max) {
        raise_error(a.err, kDevRange);
        return;
    }
    HeadVec<D> x;
    x.load(a.qkv + ((int64_t)i * per + h) * D, lane);
    const float *cs = a.cos + (int64_t)pos * (D / 2), *sn = a.sin + (int64_t)pos * (D / 2);
    if (h < a.heads) {
        x.norm_rope(a.q_gamma, cs, sn, lane);
        x.store(a.q_out + ((int64_t)i * a.heads + h) * D, lane);
    } else if (h < a.heads + a.L.kvh) {
        x.norm_rope(a.k_gamma, cs, sn, lane);
        x.template store4<false>(a.L.unit(page, h - a.heads, unit, D), r, lane);
    } else {
        x.template store4<true>(a.L.unit(page, h - a.heads - a.L.kvh, unit, D), r, lane);
    }
}

// Rows of keys and values as they are (READ: back to f32).
template <int D, bool READ>
__global__ void __launch_bounds__(kRowWarps * 32) k_kv4_rows(const RowArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t task = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    const int i = (int)(task / a.L.kvh), h = (int)(task % a.L.kvh);
    if (i >= a.rows) return;
    int page, unit, r;
    if (!row_place(a, i, page, unit, r)) return;
    uint8_t *u = a.L.unit(page, h, unit, D);
    const int64_t at = ((int64_t)i * a.L.kvh + h) * D;
    HeadVec<D> x;
    if (READ) {
        x.template load4<false>(u, r, lane);
        x.store(a.k_out + at, lane);
        x.template load4<true>(u, r, lane);
        x.store(a.v_out + at, lane);
    } else {
        x.load(a.k_in + at, lane);
        x.template store4<false>(u, r, lane);
        x.load(a.v_in + at, lane);
        x.template store4<true>(u, r, lane);
    }
}

int row_blocks(const char *who, int64_t warps, dim3 &grid) {
    const int64_t blocks = (warps + kRowWarps - 1) / kRowWarps;
    if (blocks > 0x7fffffff) return set_error(QORA_ERR_UNSUPPORTED, "%s: too many rows", who);
    grid = dim3((unsigned)blocks);
    return QORA_OK;
}

int rows_args(const char *who, qora_kv4 *kv, int32_t layer, const int32_t *slots, int32_t rows, RowArgs &a) {
    if (!kv || (rows > 0 && !slots)) return set_error(QORA_ERR_INVALID, "%s: null argument", who);
    if (layer < 0 || layer >= kv->layers || rows < 0)
        return set_error(QORA_ERR_INVALID, "%s: layer %d / rows %d out of range", who, layer, rows);
    a = RowArgs{};
    a.L = kv4_layer(kv, layer);
    a.heads = kv->heads;
    a.slots = slots;
    a.rows = rows;
    a.err = kv->ctx->err.as<int>();
    return QORA_OK;
}

}  // namespace

}  // namespace qora

using namespace qora;

extern "C" {

int qora_kv4_create(qora_ctx *ctx, int32_t num_layers, int32_t num_heads, int32_t kv_heads, int32_t head_dim,
                    int32_t max_pos, int32_t streams, int32_t page_positions, int32_t pool_pages, qora_kv4 **out) {
    if (!ctx || !out || num_layers <= 0 || num_heads <= 0 || kv_heads <= 0 || max_pos <= 0 || streams <= 0 ||
        pool_pages <= 0)
        return set_error(QORA_ERR_INVALID, "qora_kv4_create: bad arguments");
    if (head_dim != 64 && head_dim != 128)
        return set_error(QORA_ERR_UNSUPPORTED, "head_dim %d (supported: 64, 128)", head_dim);
    if (num_heads % kv_heads)
        return set_error(QORA_ERR_SHAPE, "qora_kv4_create: %d heads over %d kv heads", num_heads, kv_heads);
    if (page_positions < kKv4Unit || (page_positions & (page_positions - 1)))
        return set_error(QORA_ERR_INVALID, "page_positions %d: a power of two >= %d", page_positions, kKv4Unit);
    if (streams > kKv4MaxStreams || num_heads > 1024)
        return set_error(QORA_ERR_UNSUPPORTED, "qora_kv4_create: %d streams (max %d), %d heads (max 1024)", streams,
                         kKv4MaxStreams, num_heads);
    if (max_pos > (1 << 20) || (int64_t)pool_pages * page_positions > 0x7fffffff || pool_pages > (1 << 20))
        return set_error(QORA_ERR_UNSUPPORTED,
                         "qora_kv4_create: max_pos <= 2^20, pool_pages <= 2^20 and less than 2^31 slots");
    DeviceGuard dg;
    QORA_TRY(dg.set(ctx->device));
    qora_kv4 *kv = new (std::nothrow) qora_kv4();
    if (!kv) return set_error(QORA_ERR_OOM, "qora_kv4_create: out of host memory");
    kv->ctx = ctx;
    kv->layers = num_layers;
    kv->heads = num_heads;
    kv->kvh = kv_heads;
    kv->hd = head_dim;
    kv->max_pos = max_pos;
    kv->streams = streams;
    kv->page_pos = page_positions;
    while ((1 << kv->page_shift) < page_positions) kv->page_shift++;
    kv->pages_per_stream = (int)(((int64_t)max_pos + page_positions - 1) / page_positions);
    kv->pool_pages = pool_pages;
    kv->attend_blocks = kv4_attend_blocks(ctx);
    const int64_t page_bytes =
        (int64_t)num_layers * kv_heads * (page_positions / kKv4Unit) * kv4_unit_bytes(head_dim);
    int rc = kv->pages.alloc((size_t)(page_bytes * pool_pages));
    if (rc == QORA_OK) rc = kv->pages.zero();  // a slot that was never written reads as zeros
    if (rc == QORA_OK) rc = kv->table.alloc((size_t)streams * kv->pages_per_stream * 4);
    if (rc == QORA_OK) rc = kv->len.alloc((size_t)streams * 4);
    if (rc == QORA_OK) rc = kv->len.zero();
    if (rc == QORA_OK) rc = kv->part.alloc((size_t)kv->attend_blocks * 2 * kKv4PartRows * (head_dim + 2) * 4);
    if (rc == QORA_OK) rc = kv->tickets.alloc((size_t)kv->attend_blocks * 4);
    if (rc == QORA_OK) rc = kv->tickets.zero();
    if (rc == QORA_OK && cudaMemsetAsync(kv->table.p, 0xff, kv->table.bytes, nullptr) != cudaSuccess)
        rc = set_error(QORA_ERR_CUDA, "qora_kv4_create: memset failed");
    if (rc == QORA_OK && cudaDeviceSynchronize() != cudaSuccess)
        rc = set_error(QORA_ERR_CUDA, "qora_kv4_create: sync failed");
    if (rc != QORA_OK) {
        delete kv;
        return rc;
    }
    *out = kv;
    return QORA_OK;
}

void qora_kv4_destroy(qora_kv4 *kv) { delete kv; }

int qora_kv4_reset(qora_kv4 *kv, const int32_t *ids, int32_t count, void *stream) {
    if (!kv || count < 0) return set_error(QORA_ERR_INVALID, "qora_kv4_reset: bad arguments");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    cudaStream_t st = as_stream(stream);
    if (!ids) {
        QORA_CUDA(cudaMemsetAsync(kv->len.p, 0, kv->len.bytes, st));
        return QORA_OK;
    }
    for (int i = 0; i < count; i++)
        if (ids[i] < 0 || ids[i] >= kv->streams)
            return set_error(QORA_ERR_INVALID, "qora_kv4_reset: stream %d of %d", ids[i], kv->streams);
    for (int i = 0; i < count; i++) QORA_CUDA(cudaMemsetAsync(kv->len.as<int>() + ids[i], 0, 4, st));
    return QORA_OK;
}

int qora_kv4_lengths_host(qora_kv4 *kv, int32_t *len_host, void *stream) {
    if (!kv || !len_host) return set_error(QORA_ERR_INVALID, "qora_kv4_lengths_host: null argument");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    cudaStream_t st = as_stream(stream);
    QORA_CUDA(cudaMemcpyAsync(len_host, kv->len.p, kv->len.bytes, cudaMemcpyDeviceToHost, st));
    QORA_CUDA(cudaStreamSynchronize(st));
    return QORA_OK;
}

int qora_kv4_state(qora_kv4 *kv, int32_t **table, int32_t *pages_per_stream, int32_t **lengths) {
    if (!kv) return set_error(QORA_ERR_INVALID, "qora_kv4_state: null kv");
    if (table) *table = kv->table.as<int>();
    if (pages_per_stream) *pages_per_stream = kv->pages_per_stream;
    if (lengths) *lengths = kv->len.as<int>();
    return QORA_OK;
}

int qora_kv4_reserve(qora_kv4 *kv, const int32_t *counts, int32_t max_tokens, int32_t *slots, int32_t *positions,
                     int32_t *offsets, void *stream) {
    if (!kv || !counts || !offsets || max_tokens < 0 || (max_tokens > 0 && (!slots || !positions)))
        return set_error(QORA_ERR_INVALID, "qora_kv4_reserve: bad arguments");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    ReserveArgs a;
    a.counts = counts;
    a.len = kv->len.as<int>();
    a.table = kv->table.as<int>();
    a.slots = slots;
    a.positions = positions;
    a.offsets = offsets;
    a.err = kv->ctx->err.as<int>();
    a.streams = kv->streams;
    a.max_pos = kv->max_pos;
    a.page_shift = kv->page_shift;
    a.pages_per_stream = kv->pages_per_stream;
    a.pool_pages = kv->pool_pages;
    a.max_tokens = max_tokens;
    const size_t smem = (size_t)((kv->pool_pages + 31) / 32) * 4;
    if (smem > 40 * 1024)
        QORA_CUDA(cudaFuncSetAttribute(k_kv4_reserve, cudaFuncAttributeMaxDynamicSharedMemorySize, 1 << 17));
    return launch_ex(k_kv4_reserve, dim3(1), dim3(kResThreads), smem, as_stream(stream), 1u, a);
}

int qora_kv4_advance(qora_kv4 *kv, const int32_t *counts, void *stream) {
    if (!kv || !counts) return set_error(QORA_ERR_INVALID, "qora_kv4_advance: null argument");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    return launch_ex(k_kv4_advance, dim3((kv->streams + 255) / 256), dim3(256), 0, as_stream(stream), 1u,
                     kv->len.as<int>(), counts, kv->streams, kv->max_pos, kv->ctx->err.as<int>());
}

int qora_kv4_append(qora_kv4 *kv, int32_t layer, const float *qkv, const uint16_t *q_norm, const uint16_t *k_norm,
                    const float *rope_cos, const float *rope_sin, int32_t rope_max_pos, const int32_t *positions,
                    const int32_t *slots, int32_t tokens, float *q_out, void *stream) {
    RowArgs a;
    QORA_TRY(rows_args("qora_kv4_append", kv, layer, slots, tokens, a));
    if (!tokens) return QORA_OK;
    if (!qkv || !q_norm || !k_norm || !rope_cos || !rope_sin || !positions || !q_out || rope_max_pos <= 0)
        return set_error(QORA_ERR_INVALID, "qora_kv4_append: bad arguments");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    a.qkv = qkv;
    a.q_out = q_out;
    a.q_gamma = reinterpret_cast<const __half *>(q_norm);
    a.k_gamma = reinterpret_cast<const __half *>(k_norm);
    a.cos = rope_cos;
    a.sin = rope_sin;
    a.rope_max = rope_max_pos;
    a.positions = positions;
    dim3 grid;
    QORA_TRY(row_blocks("qora_kv4_append", (int64_t)tokens * (kv->heads + 2 * kv->kvh), grid));
    auto kern = kv->hd == 64 ? k_kv4_append<64> : k_kv4_append<128>;
    return launch_ex(kern, grid, dim3(kRowWarps * 32), 0, as_stream(stream), 1u, a);
}

int qora_kv4_write(qora_kv4 *kv, int32_t layer, const int32_t *slots, int32_t rows, const float *k, const float *v,
                   void *stream) {
    RowArgs a;
    QORA_TRY(rows_args("qora_kv4_write", kv, layer, slots, rows, a));
    if (!rows) return QORA_OK;
    if (!k || !v) return set_error(QORA_ERR_INVALID, "qora_kv4_write: null argument");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    a.k_in = k;
    a.v_in = v;
    dim3 grid;
    QORA_TRY(row_blocks("qora_kv4_write", (int64_t)rows * kv->kvh, grid));
    auto kern = kv->hd == 64 ? k_kv4_rows<64, false> : k_kv4_rows<128, false>;
    return launch_ex(kern, grid, dim3(kRowWarps * 32), 0, as_stream(stream), 1u, a);
}

int qora_kv4_read(qora_kv4 *kv, int32_t layer, const int32_t *slots, int32_t rows, float *k, float *v,
                  void *stream) {
    RowArgs a;
    QORA_TRY(rows_args("qora_kv4_read", kv, layer, slots, rows, a));
    if (!rows) return QORA_OK;
    if (!k || !v) return set_error(QORA_ERR_INVALID, "qora_kv4_read: null argument");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    a.k_out = k;
    a.v_out = v;
    dim3 grid;
    QORA_TRY(row_blocks("qora_kv4_read", (int64_t)rows * kv->kvh, grid));
    auto kern = kv->hd == 64 ? k_kv4_rows<64, true> : k_kv4_rows<128, true>;
    return launch_ex(kern, grid, dim3(kRowWarps * 32), 0, as_stream(stream), 1u, a);
}

}  // extern "C"
