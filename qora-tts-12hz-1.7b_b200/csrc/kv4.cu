// The 4-bit paged KV cache: creation, block tables and slot maps built on the
// GPU (k_kv4_reserve), the append with qk-norm and rotation (k_kv4_append),
// plain writes and reads of rows, and the length update.
#include <cooperative_groups.h>

#include <new>

#include "kv4.cuh"

namespace cg = cooperative_groups;

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
//
// One cluster does it all (one launch, no workspace).  Every block scans the
// streams' counts for itself (they are few); the table entries are marked by
// all warps, in pieces of 128 with 24 loads of a lane in flight; each block then
// joins its share of the bit maps through distributed shared memory and hands
// out the free pages in it; tokens are spread over all threads, which look
// their stream up in the scanned offsets.  What bounds it is latency: 512 streams
// of up to 16000 positions in pages of 64 take 17 us, 5.5 of them for marking, and
// 32 streams 5.7 us.  Walking each stream's pages from one block took 336 us.
constexpr int kResThreads = 1024;
constexpr int kResCluster = 16;  // (not a portable size; what bounds the large case is marking, a block's share of it)
constexpr int kResChunk = 128;  // table entries of one stream that a warp marks at a time,
constexpr int kResDeep = 6;     // and how many such pieces: 24 loads of a lane in flight

struct ReserveArgs {
    const int *counts, *len;
    int *table, *slots, *positions, *offsets, *err;
    int streams, max_pos, page_shift, pages_per_stream, pool_pages, max_tokens;
};

constexpr int kResList = 2048;  // free pages that are listed at a time

struct ReserveShared {
    int64_t wsum[32];
    int bad, free_pages;
    int list[kResList];
};

__device__ __forceinline__ int64_t block_scan_excl(int64_t v, int64_t *wsum, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int64_t w = wsum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        wsum[lane] = w;
    }
    __syncthreads();
    total = wsum[31];
    return x - v + (warp ? wsum[warp - 1] : 0);
}

// The last index i with at[i] <= v (at[0] = 0 <= v).
__device__ __forceinline__ int last_at_most(const int *at, int n, int v) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kResThreads) k_kv4_reserve(const ReserveArgs a) {
    extern __shared__ int res_dyn[];
    __shared__ ReserveShared sh;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), nr = (int)cl.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = (a.pool_pages + 31) >> 5;
    const int P = 1 << a.page_shift;
    int *len = res_dyn;                   // [streams], -1 when the stream's request is bad
    int *first = len + a.streams;         // [streams] ordinal of its first new page
    int *off = first + a.streams;         // [streams] its first token
    unsigned *bits = reinterpret_cast<unsigned *>(off + a.streams);  // [words] pages in use
    griddep_launch_dependents();
    griddep_wait();
    if (tid == 0) sh.bad = 0;
    for (int w = tid; w < words; w += kResThreads) bits[w] = 0u;
    __syncthreads();
    // ---- streams: tokens and new pages, scanned together (tokens in the high half)
    int64_t base = 0;
    for (int b0 = 0; b0 < a.streams; b0 += kResThreads) {
        const int b = b0 + tid;
        int64_t v = 0;
        int l = 0;
        if (b < a.streams) {
            l = a.len[b];
            const int n = a.counts[b];
            if (l < 0 || n < 0 || l > a.max_pos || n > a.max_pos - l) {
                sh.bad = kDevRange;
                l = -1;
            } else {
                v = ((int64_t)n << 32) | (((l + n + P - 1) >> a.page_shift) - ((l + P - 1) >> a.page_shift));
            }
        }
        int64_t total;
        const int64_t at = base + block_scan_excl(v, sh.wsum, total);
        if (b < a.streams) {
            len[b] = l;
            first[b] = (int)(at & 0xffffffff);
            off[b] = (int)min((uint64_t)at >> 32, (uint64_t)0x7fffffff);
        }
        base += total;
    }
    const uint64_t tokens = (uint64_t)base >> 32;  // (streams 2^12, max_pos 2^20: below 2^32 where pages suffice)
    const int need = (int)(base & 0xffffffff);
    __syncthreads();
    // ---- mark the pages in use
    const int chunks = (a.pages_per_stream + kResChunk - 1) / kResChunk;
    const int warps = nr * (kResThreads / 32);
    for (int p0 = rank * (kResThreads / 32) + warp; p0 < a.streams * chunks; p0 += kResDeep * warps) {
        int pg[kResDeep][kResChunk / 32], left[kResDeep];  // entries; how many from the lane's first on
#pragma unroll
        for (int d = 0; d < kResDeep; d++) {
            const int p = p0 + d * warps;
            const int b = p / chunks, j0 = (p - b * chunks) * kResChunk + lane;
            left[d] = p < a.streams * chunks ? ((len[b] + P - 1) >> a.page_shift) - j0 : 0;
            const int *t = a.table + (int64_t)b * a.pages_per_stream;
#pragma unroll
            for (int i = 0; i < kResChunk / 32; i++) pg[d][i] = i * 32 < left[d] ? __ldcg(t + j0 + i * 32) : 0;
        }
#pragma unroll
        for (int d = 0; d < kResDeep; d++)
#pragma unroll
            for (int i = 0; i < kResChunk / 32; i++) {
                if (i * 32 >= left[d]) break;
                if ((unsigned)pg[d][i] >= (unsigned)a.pool_pages) sh.bad = kDevRange;
                else atomicOr(&bits[pg[d][i] >> 5], 1u << (pg[d][i] & 31));
            }
    }
    cl.sync();
    // ---- this block's share of the pool: words [wa, wb)
    const int share = (words + nr - 1) / nr;
    const int wa = min(words, rank * share), wb = min(words, wa + share);
    int mine = 0;
    for (int w = wa + tid; w < wb; w += kResThreads) {
        unsigned f = 0u;
#pragma unroll
        for (int r = 0; r < kResCluster; r++)
            if (r < nr) f |= cl.map_shared_rank(bits, r)[w];
        f = ~f;
        if (w == words - 1 && (a.pool_pages & 31)) f &= (1u << (a.pool_pages & 31)) - 1u;
        bits[w] = f;  // from here on: free pages (no other block reads these words)
        mine += __popc(f);
    }
    int64_t total;
    block_scan_excl(mine, sh.wsum, total);
    if (tid == 0) sh.free_pages = (int)total;
    cl.sync();
    int ordinal = 0, free_total = 0, bad = 0;
    int theirs[kResCluster], wrong[kResCluster];  // (all reads in flight together)
#pragma unroll
    for (int r = 0; r < kResCluster; r++) {
        const ReserveShared *o = cl.map_shared_rank(&sh, r < nr ? r : 0);
        theirs[r] = o->free_pages, wrong[r] = o->bad;
    }
#pragma unroll
    for (int r = 0; r < kResCluster; r++) {
        if (r >= nr) break;
        if (r == rank) ordinal = free_total;
        free_total += theirs[r];
        bad |= wrong[r];
    }
    const int all = nr * kResThreads, me = rank * kResThreads + tid;
    const int why = bad ? kDevRange : tokens > (uint64_t)a.max_tokens ? kDevRange : need > free_total ? kDevPool : 0;
    if (why) {  // nothing is mapped, and every listed token is skipped
        if (me == 0) raise_error(a.err, why);
        for (int b = me; b <= a.streams; b += all) a.offsets[b] = 0;
        for (int i = me; i < a.max_tokens; i += all) {
            a.slots[i] = -1;
            a.positions[i] = 0;
        }
        cl.sync();  // no block leaves while another reads its counts
        return;
    }
    for (int b = me; b <= a.streams; b += all) a.offsets[b] = b < a.streams ? off[b] : (int)tokens;
    // ---- the i-th free page goes to the i-th new (stream, page): threads list the
    // pages of their words, then share the list out
    for (int w0 = wa; w0 < wb && ordinal < need; w0 += kResThreads) {
        const int w = w0 + tid;
        const unsigned f = w < wb ? bits[w] : 0u;
        const int at = (int)block_scan_excl(__popc(f), sh.wsum, total);
        const int count = min((int)total, need - ordinal);
        for (int l0 = 0; l0 < count; l0 += kResList) {
            int i = at - l0;
            for (unsigned m = f; m && i < kResList; m &= m - 1, i++)
                if (i >= 0) sh.list[i] = w * 32 + __ffs(m) - 1;
            __syncthreads();
            for (int j = tid; j < min(count - l0, kResList); j += kResThreads) {
                const int o = ordinal + l0 + j;
                const int b = last_at_most(first, a.streams, o);
                const int keep = (len[b] + P - 1) >> a.page_shift;
                __stcg(a.table + (int64_t)b * a.pages_per_stream + keep + (o - first[b]), sh.list[j]);
            }
            __syncthreads();
        }
        ordinal += (int)total;
    }
    cl.sync();
    // ---- the tokens' slots and positions
    for (int i = me; i < a.max_tokens; i += all) {
        int slot = -1, pos = 0;
        if (i < (int)tokens) {
            const int b = last_at_most(off, a.streams, i);
            pos = len[b] + i - off[b];
            const int pg = __ldcg(a.table + (int64_t)b * a.pages_per_stream + (pos >> a.page_shift));
            slot = (pg << a.page_shift) + (pos & (P - 1));
        }
        a.slots[i] = slot;
        a.positions[i] = pos;
    }
}

// lengths += counts (negative counts roll back); with offsets, by at most the tokens
// that they list for the stream
__global__ void k_kv4_advance(int *len, const int *counts, const int *offsets, int streams, int max_pos, int *err) {
    griddep_launch_dependents();
    griddep_wait();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= streams) return;
    int64_t by = counts[b];
    if (offsets) by = min(by, (int64_t)offsets[b + 1] - offsets[b]);
    const int64_t to = (int64_t)len[b] + by;
    if (to < 0 || to > max_pos) raise_error(err, kDevRange);
    len[b] = (int)(to < 0 ? 0 : to > max_pos ? max_pos : to);
}

// ------------------------------------------------------------ rows
// D/8 lanes hold one head vector (a warp two or four of them): lane l of a head
// has dimensions 4l .. 4l + 3 of each half, so the rotation's pairs (i, i + D/2)
// and the four codes of a stored halfword lie in one lane, loads and stores are
// 16 bytes, and a scale group is eight lanes.
__device__ __forceinline__ float inv_sqrt(float x) { return __fdiv_rn(1.0f, __fsqrt_rn(x)); }
__device__ __forceinline__ double inv_sqrt(double x) { return rsqrt(x); }

// The larger of two magnitudes, NaN when one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int D>
struct Angles {
    float4 c, s;
    __device__ __forceinline__ void load(const float *cs, const float *sn, int l) {
        c = __ldg(reinterpret_cast<const float4 *>(cs) + l);
        s = __ldg(reinterpret_cast<const float4 *>(sn) + l);
    }
};

template <int D>
struct HeadVec {
    static constexpr int kLanes = D / 8;
    float x[2][4];

    __device__ __forceinline__ void load(const float *p, int l) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float4 v = __ldcs(reinterpret_cast<const float4 *>(p + h * (D / 2)) + l);
            x[h][0] = v.x, x[h][1] = v.y, x[h][2] = v.z, x[h][3] = v.w;
        }
    }
    __device__ __forceinline__ void store(float *p, int l) const {
#pragma unroll
        for (int h = 0; h < 2; h++)
            reinterpret_cast<float4 *>(p + h * (D / 2))[l] = make_float4(x[h][0], x[h][1], x[h][2], x[h][3]);
    }

    // RMS norm over the head and rotation by the position's angles, rounded to
    // f32 at the end.  Keys take T = double: their 4-bit codes are decided next
    // to borders, where the f32 rounding of these sums would move one code in a
    // million by a whole step.  Queries take T = float (f64's conversions are
    // the slowest part of a key: half the heads are queries).
    template <class T>
    __device__ __forceinline__ void norm_rope(const __half *gamma, const Angles<D> &ang, int l) {
        T ss = 0;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) ss += (T)x[h][e] * (T)x[h][e];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const T inv = inv_sqrt(ss * (T)(1.0 / D) + (T)1e-6);
        const uint2 g0 = __ldg(reinterpret_cast<const uint2 *>(gamma) + l);
        const uint2 g1 = __ldg(reinterpret_cast<const uint2 *>(gamma + D / 2) + l);
        const __half2 ga[4] = {*reinterpret_cast<const __half2 *>(&g0.x), *reinterpret_cast<const __half2 *>(&g0.y),
                               *reinterpret_cast<const __half2 *>(&g1.x), *reinterpret_cast<const __half2 *>(&g1.y)};
        const float cs[4] = {ang.c.x, ang.c.y, ang.c.z, ang.c.w}, sn[4] = {ang.s.x, ang.s.y, ang.s.z, ang.s.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float f0 = (e & 1) ? __high2float(ga[e >> 1]) : __low2float(ga[e >> 1]);
            const float f1 = (e & 1) ? __high2float(ga[2 + (e >> 1)]) : __low2float(ga[2 + (e >> 1)]);
            const T a = (T)x[0][e] * inv * (T)f0, b = (T)x[1][e] * inv * (T)f1;
            const T c = cs[e], s = sn[e];
            x[0][e] = (float)(a * c - b * s);
            x[1][e] = (float)(b * c + a * s);
        }
    }

    // Quantises and writes the row as position r of the unit (`on`: this lane's
    // head is there; all lanes take part in the exchange).
    template <bool V>
    __device__ __forceinline__ void store4(uint8_t *unit, int r, int l, bool on) const {
        using U = Kv4Unit<D>;
        float s[2];
        __half sh[2];
        bool plain = true;  // scales that are normal f16 numbers: no code can pass 7
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float amax = max_nan(max_nan(fabsf(x[h][0]), fabsf(x[h][1])), max_nan(fabsf(x[h][2]), fabsf(x[h][3])));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            // amax / 7 correctly rounded: one step from a quotient within an ulp.
            // Rounding that to f16 equals rounding amax / 7 once: no f32 neighbour
            // of 7m has a quotient that rounds to the 12-bit m.
            const float seventh = 0.14285715f;
            float d = __fmul_rn(amax, seventh);
            d = fmaf(fmaf(-7.0f, d, amax), seventh, d);
            sh[h] = __float2half_rn(fminf(d, 65504.0f));
            if (!(amax < INFINITY)) sh[h] = __ushort_as_half((unsigned short)0x7e00);
            s[h] = __half2float(sh[h]);
            plain = plain && s[h] >= 0x1p-14f && s[h] < 65504.0f;
        }
        unsigned nib[2];
        bool sure = true;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            // Nearest integer to x / s by the approximate quotient: adding 1.5 2^23
            // leaves it in the low bits.  x - q s is exact in f32; where it is under
            // s / 2 the integer is the nearest.
            float inv;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s[h]));
            unsigned sum = 0;
#pragma unroll
            for (int e = 3; e >= 0; e--) {
                const float t = fmaf(x[h][e], inv, 12582912.0f);
                const float rest = fmaf(12582912.0f - t, s[h], x[h][e]);
                sure = sure && fabsf(rest) < 0.5f * s[h];
                sum = sum * 16u + __float_as_uint(t);
            }
            nib[h] = sum - (0x4b400000u - 8u) * 0x1111u;  // each digit: code + 8
        }
        if (!__all_sync(0xffffffffu, plain && sure)) {  // ties, zeros, infinities, scales at f16's ends
#pragma unroll
            for (int h = 0; h < 2; h++) nib[h] = codes_exactly(x[h], s[h]);
        }
        if (!on) return;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int dim = h * (D / 2) + 4 * l;
            *reinterpret_cast<uint16_t *>(unit + (V ? U::v_half(r, dim) : U::k_word(r, dim) + ((dim & 4) >> 1))) =
                (uint16_t)nib[h];
            if ((l & 7) == 0)
                *reinterpret_cast<__half *>(unit + (V ? U::v_scale(r, dim >> 5) : U::k_scale(r, dim >> 5))) = sh[h];
        }
    }

    // The same codes for any scale (0 and NaN: codes 0), ties to even, in [-7, 7].
    static __device__ __noinline__ unsigned codes_exactly(const float (&v4)[4], float s) {
        const bool live = s > 0.0f;
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(live ? s : 1.0f));
        unsigned nib = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            // rint of the approximate quotient is off by one at most; the rest decides
            const float v = live ? v4[e] : 0.0f;
            float q = rintf(fminf(fmaxf(v * inv, -8.0f), 8.0f));
            const float rest = 2.0f * fmaf(-q, s, v);
            const bool odd = (int)q & 1;
            if (rest > s || (rest == s && odd)) q += 1.0f;
            if (rest < -s || (rest == -s && odd)) q -= 1.0f;
            q = live ? fminf(fmaxf(q, -7.0f), 7.0f) : 0.0f;
            nib |= (unsigned)((int)q + 8) << (4 * e);
        }
        return nib;
    }

    template <bool V>
    __device__ __forceinline__ void load4(const uint8_t *unit, int r, int l) {
        using U = Kv4Unit<D>;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int dim = h * (D / 2) + 4 * l;
            const float s = __half2float(
                *reinterpret_cast<const __half *>(unit + (V ? U::v_scale(r, dim >> 5) : U::k_scale(r, dim >> 5))));
            const unsigned w = *reinterpret_cast<const uint16_t *>(
                unit + (V ? U::v_half(r, dim) : U::k_word(r, dim) + ((dim & 4) >> 1)));
#pragma unroll
            for (int e = 0; e < 4; e++) x[h][e] = s * (float)((int)((w >> (4 * e)) & 15u) - 8);
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
__device__ __forceinline__ bool row_place(const RowArgs &a, int slot, int &page, int &unit, int &r) {
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

// Norm, rotation and append.  A warp takes 256 / D heads of one kind of one row: q
// heads are normed, rotated and stored in f32; k heads normed, rotated and stored
// in 4 bits; v heads stored in 4 bits.  What bounds the large case is the way from
// a multiprocessor to the L2 cache (69 % of its cycles): q rows in f32, and the
// 2-byte pieces that 4-bit rows are written in, each a request of its own.  8191
// rows of 16 / 8 heads of 128 take 54 us in a loop of their own, against 56 to 66 with two rows or two
// groups of heads a warp, and 83 with warps that fetch ahead and stay.
template <int D>
__global__ void __launch_bounds__(kRowWarps * 32, 6) k_kv4_append(const RowArgs a) {
    constexpr int HW = 256 / D;  // heads of a warp
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31, l = lane % (D / 8), sub = lane / (D / 8);
    const int qt = (a.heads + HW - 1) / HW, kt = (a.L.kvh + HW - 1) / HW;
    const unsigned per = qt + 2 * kt;
    const unsigned task = blockIdx.x * kRowWarps + (threadIdx.x >> 5);  // (below 2^31: row_blocks)
    const int i = (int)(task / per), w = (int)(task % per);
    if (i >= a.rows) return;
    const int kind = w < qt ? 0 : w < qt + kt ? 1 : 2;
    const int n = kind == 0 ? a.heads : a.L.kvh;
    const int h = (w - (kind == 0 ? 0 : kind == 1 ? qt : qt + kt)) * HW + sub;  // this lane's head of its kind
    const bool on = h < n;
    const int first = kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.L.kvh;
    const int slot = a.slots[i], pos = a.positions[i];
    HeadVec<D> x;
    x.load(a.qkv + ((int64_t)i * (a.heads + 2 * a.L.kvh) + first + (on ? h : 0)) * D, l);
    int page, unit, r;
    if (!row_place(a, slot, page, unit, r)) return;
    if (pos < 0 || pos >= a.rope_max) {
        raise_error(a.err, kDevRange);
        return;
    }
    if (kind == 2) {
        x.template store4<true>(a.L.unit(page, on ? h : 0, unit, D), r, l, on);
        return;
    }
    Angles<D> ang;
    ang.load(a.cos + (int64_t)pos * (D / 2), a.sin + (int64_t)pos * (D / 2), l);
    if (kind == 0) {
        x.template norm_rope<float>(a.q_gamma, ang, l);
        if (on) x.store(a.q_out + ((int64_t)i * a.heads + h) * D, l);
    } else {
        x.template norm_rope<double>(a.k_gamma, ang, l);
        x.template store4<false>(a.L.unit(page, on ? h : 0, unit, D), r, l, on);
    }
}

// Rows of keys and values as they are (READ: back to f32), 256 / D heads a warp.
// Bound by memory: reading 8191 rows of 8 heads of 128 takes 13.5 us, 5.7 TB/s.
template <int D, bool READ>
__global__ void __launch_bounds__(kRowWarps * 32) k_kv4_rows(const RowArgs a) {
    constexpr int HW = 256 / D;
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31, l = lane % (D / 8), sub = lane / (D / 8);
    const unsigned per = (a.L.kvh + HW - 1) / HW;
    const unsigned task = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    const int i = (int)(task / per), h = (int)(task - i * per) * HW + sub;
    if (i >= a.rows) return;
    int page, unit, r;
    if (!row_place(a, a.slots[i], page, unit, r)) return;
    const bool on = h < a.L.kvh;
    uint8_t *u = a.L.unit(page, on ? h : 0, unit, D);
    const int64_t at = ((int64_t)i * a.L.kvh + (on ? h : 0)) * D;
    HeadVec<D> k, v;
    if (READ) {
        k.template load4<false>(u, r, l);
        v.template load4<true>(u, r, l);
        if (on) {
            k.store(a.k_out + at, l);
            v.store(a.v_out + at, l);
        }
    } else {
        k.load(a.k_in + at, l);
        v.load(a.v_in + at, l);
        k.template store4<false>(u, r, l, on);
        v.template store4<true>(u, r, l, on);
    }
}

int row_blocks(const char *who, int64_t warps, dim3 &grid) {
    const int64_t blocks = (warps + kRowWarps - 1) / kRowWarps;
    if (blocks > 0x7fffffff / kRowWarps) return set_error(QORA_ERR_UNSUPPORTED, "%s: too many rows", who);
    grid = dim3((unsigned)blocks);
    return QORA_OK;
}

template <class... T>
bool aligned16(const T *...p) {
    return !((reinterpret_cast<uintptr_t>(p) | ...) & 15);
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

size_t reserve_smem(const qora_kv4 *kv) {
    return ((size_t)((kv->pool_pages + 31) / 32) + 3 * (size_t)kv->streams) * 4;
}

// What k_kv4_reserve's launches need, once for the cache: its attributes, and how many
// blocks of a cluster the device can place at once (16 is no size that it has to).
int reserve_setup(qora_kv4 *kv) {
    static std::atomic<uint64_t> done;
    QORA_TRY(allow_smem(k_kv4_reserve, ((1 << 20) / 32 + 3 * kKv4MaxStreams) * 4, kv->ctx->device, done));
    QORA_CUDA(cudaFuncSetAttribute(k_kv4_reserve, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    for (kv->wide = kResCluster; kv->wide > 1; kv->wide >>= 1) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute at;
        cfg.gridDim = dim3(1, kv->wide);
        cfg.blockDim = dim3(kResThreads);
        cfg.dynamicSmemBytes = reserve_smem(kv);
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = 1;
        at.val.clusterDim.y = kv->wide;
        at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, k_kv4_reserve, &cfg) == cudaSuccess && n > 0) break;
        (void)cudaGetLastError();  // (a size that it cannot place at all may be an error)
    }
    return QORA_OK;
}

int advance(qora_kv4 *kv, const int32_t *counts, const int32_t *offsets, void *stream) {
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    return launch_ex(k_kv4_advance, dim3((kv->streams + 255) / 256), dim3(256), 0, as_stream(stream), 1u,
                     kv->len.as<int>(), counts, offsets, kv->streams, kv->max_pos, kv->ctx->err.as<int>());
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
    const int64_t page_bytes =
        (int64_t)num_layers * kv_heads * (page_positions / kKv4Unit) * kv4_unit_bytes(head_dim);
    int rc = kv->pages.alloc((size_t)(page_bytes * pool_pages));
    if (rc == QORA_OK) rc = kv->pages.zero();  // a slot that was never written reads as zeros
    if (rc == QORA_OK) rc = kv->table.alloc((size_t)streams * kv->pages_per_stream * 4);
    if (rc == QORA_OK) rc = kv->len.alloc((size_t)streams * 4);
    if (rc == QORA_OK) rc = kv->len.zero();
    if (rc == QORA_OK) rc = reserve_setup(kv);
    if (rc == QORA_OK) rc = kv4_attend_setup(kv);
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
    if (max_tokens > (1 << 30))
        return set_error(QORA_ERR_UNSUPPORTED, "qora_kv4_reserve: max_tokens %d (max 2^30)", max_tokens);
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
    // a cluster pays where there are many table entries and tokens: 16448 of them take
    // 8.8 us by one block and 10.5 by a cluster, 32896 9.9 and 9.3, 66048 16.3 and 11.5
    const bool wide = (int64_t)kv->streams * kv->pages_per_stream + max_tokens > 24576;
    const unsigned nr = wide ? kv->wide : 1;
    return launch_ex(k_kv4_reserve, dim3(1, nr), dim3(kResThreads), reserve_smem(kv), as_stream(stream), nr, a);
}

int qora_kv4_advance(qora_kv4 *kv, const int32_t *counts, void *stream) {
    if (!kv || !counts) return set_error(QORA_ERR_INVALID, "qora_kv4_advance: null argument");
    return advance(kv, counts, nullptr, stream);
}

int qora_kv4_accept(qora_kv4 *kv, const int32_t *counts, const int32_t *offsets, void *stream) {
    if (!kv || !counts || !offsets) return set_error(QORA_ERR_INVALID, "qora_kv4_accept: null argument");
    return advance(kv, counts, offsets, stream);
}

int qora_kv4_append(qora_kv4 *kv, int32_t layer, const float *qkv, const uint16_t *q_norm, const uint16_t *k_norm,
                    const float *rope_cos, const float *rope_sin, int32_t rope_max_pos, const int32_t *positions,
                    const int32_t *slots, int32_t tokens, float *q_out, void *stream) {
    RowArgs a;
    QORA_TRY(rows_args("qora_kv4_append", kv, layer, slots, tokens, a));
    if (!tokens) return QORA_OK;
    if (!qkv || !q_norm || !k_norm || !rope_cos || !rope_sin || !positions || !q_out || rope_max_pos <= 0)
        return set_error(QORA_ERR_INVALID, "qora_kv4_append: bad arguments");
    if (!aligned16(qkv, rope_cos, rope_sin, q_out) || !aligned16(q_norm, k_norm))
        return set_error(QORA_ERR_INVALID, "qora_kv4_append: pointers must be 16-byte aligned");
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
    const int hw = 256 / kv->hd;
    const int64_t per = (kv->heads + hw - 1) / hw + 2 * ((kv->kvh + hw - 1) / hw);
    dim3 grid;
    QORA_TRY(row_blocks("qora_kv4_append", tokens * per, grid));
    auto kern = kv->hd == 64 ? k_kv4_append<64> : k_kv4_append<128>;
    return launch_ex(kern, grid, dim3(kRowWarps * 32), 0, as_stream(stream), 1u, a);
}

int qora_kv4_write(qora_kv4 *kv, int32_t layer, const int32_t *slots, int32_t rows, const float *k, const float *v,
                   void *stream) {
    RowArgs a;
    QORA_TRY(rows_args("qora_kv4_write", kv, layer, slots, rows, a));
    if (!rows) return QORA_OK;
    if (!k || !v) return set_error(QORA_ERR_INVALID, "qora_kv4_write: null argument");
    if (!aligned16(k, v)) return set_error(QORA_ERR_INVALID, "qora_kv4_write: pointers must be 16-byte aligned");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    a.k_in = k;
    a.v_in = v;
    dim3 grid;
    const int hw = 256 / kv->hd;
    QORA_TRY(row_blocks("qora_kv4_write", (int64_t)rows * ((kv->kvh + hw - 1) / hw), grid));
    auto kern = kv->hd == 64 ? k_kv4_rows<64, false> : k_kv4_rows<128, false>;
    return launch_ex(kern, grid, dim3(kRowWarps * 32), 0, as_stream(stream), 1u, a);
}

int qora_kv4_read(qora_kv4 *kv, int32_t layer, const int32_t *slots, int32_t rows, float *k, float *v,
                  void *stream) {
    RowArgs a;
    QORA_TRY(rows_args("qora_kv4_read", kv, layer, slots, rows, a));
    if (!rows) return QORA_OK;
    if (!k || !v) return set_error(QORA_ERR_INVALID, "qora_kv4_read: null argument");
    if (!aligned16(k, v)) return set_error(QORA_ERR_INVALID, "qora_kv4_read: pointers must be 16-byte aligned");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    a.k_out = k;
    a.v_out = v;
    dim3 grid;
    const int hw = 256 / kv->hd;
    QORA_TRY(row_blocks("qora_kv4_read", (int64_t)rows * ((kv->kvh + hw - 1) / hw), grid));
    auto kern = kv->hd == 64 ? k_kv4_rows<64, true> : k_kv4_rows<128, true>;
    return launch_ex(kern, grid, dim3(kRowWarps * 32), 0, as_stream(stream), 1u, a);
}

}  // extern "C"
