// Attention over the 4-bit paged cache (k_kv4_attend).
//
// out = softmax(q k^T / sqrt(D)) v for the new tokens of every stream, token i
// of stream b over positions 0 .. len_b + i, with k = s_k c_k and v = s_v c_v
// (scales per position and group of 32 dimensions, codes in [-7, 7]).
//
// One warp takes one unit of 32 positions at a time and multiplies it with a
// tile of R = 4 NT query rows (a row = one head of one token; the heads that
// share a kv head share the tile).  Codes are exact in f16, so each f32 query
// is split once into hi + lo f16 (22 bits together, scaled per row by a power
// of two so that any finite query fits) and both halves are columns of one
// matrix product: an m16n8k16 step takes 16 positions x 4 rows x {hi, lo}.
//   scores  S^T[pos][row] = sum_c s_k[pos][c] (codes_c . q_c): one accumulator
//           per scale group, scaled and summed in f32;
//   values  O^T[dim][row] += codes^T[dim][pos] (p[pos][row] s_v[pos][c]): the
//           probability takes the group's scale in f32, is split into hi + lo
//           and transposed into the second operand (movmatrix).
// Every 32 positions the products' accumulators are folded into f32 registers
// (the matrix unit's own additions do not round to nearest).  The running
// maximum and sum are f32, in base 2.
//
// The work of a launch (all streams, kv heads, row tiles, units) is one line of
// units; lengths and offsets are read on the device.  Each cluster of blocks
// takes a run of whole items (stream, kv head, row tile) with as near to an even
// share of the units as whole items allow, and its blocks split the run evenly,
// through the middle of items.  Partial (max, sum, weighted sum) of an item that
// several blocks share meet in distributed shared memory, in block order, so
// there is no workspace and the result does not depend on timing.
//
// One token of 32 streams of 4096 positions, 16 / 8 heads of 128: 44 us, 3.4 TB/s
// of cache read (of 16384: 5.4 TB/s).  A launch costs some 8 us besides the units:
// lengths, tables, first copies and the join, one after the other.  The units are
// bound by instructions: some 780 for 32 positions at a tile of 4 rows, issued in
// 60 % of the cycles at 16 warps a multiprocessor, as many as registers allow.
#include <algorithm>

#include <cooperative_groups.h>

#include "kv4.cuh"

namespace cg = cooperative_groups;

namespace qora {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;  // blocks of a cluster
constexpr int kStages = 2;      // units of a warp in flight or in use

struct AttendArgs {
    Kv4Layer L;
    const float *q;
    const int *offsets, *len;
    float *out;
    int *err;
    int streams, heads, max_pos, tokens;
    float scale_log2;  // log2(e) / sqrt(D)
};

// D = A B + C for 16 x 16 x 8, f16 in and f32 out; (not volatile: the compiler may
// interleave the products of different scale groups)
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with C = 0
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// (w & Mask) | magic in one instruction.  (Left to the compiler it becomes two,
// 128 more of them for every unit.)
template <uint32_t Mask>
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(Mask), "r"(magic));
    return r;
}
// The four pairs of codes of a word: x[j] = (nibble j, nibble j + 4) - 8 in f16.
// `magic` is 0x64006400 (1024 in both halves) in a register.
__device__ __forceinline__ void codes(uint32_t w, uint32_t magic, uint32_t (&x)[4]) {
    const __half2 lo = __half2half2(__ushort_as_half(0x6408));    // 1032
    const __half2 s16 = __half2half2(__ushort_as_half(0x2c00));   // 1 / 16
    const __half2 hi = __half2half2(__ushort_as_half(0xd480));    // -72
    const uint32_t v = w >> 8;
    x[0] = h2u(__hsub2(u2h(and_or<0x000f000fu>(w, magic)), lo));
    x[1] = h2u(__hfma2(u2h(and_or<0x00f000f0u>(w, magic)), s16, hi));
    x[2] = h2u(__hsub2(u2h(and_or<0x000f000fu>(v, magic)), lo));
    x[3] = h2u(__hfma2(u2h(and_or<0x00f000f0u>(v, magic)), s16, hi));
}

// t as f16 hi (low half) + f16 lo (high half): the bits that f16 has, and the rest.
__device__ __forceinline__ uint32_t split_hi_lo(float t) {
    const float hi = __uint_as_float(__float_as_uint(t) & 0xffffe000u);
    return h2u(__floats2half2_rn(hi, t - hi));
}

// The four f16 scales of 8 bytes: element i.
__device__ __forceinline__ float scale_of(uint2 v, int i) {
    const __half2 h = u2h(i < 2 ? v.x : v.y);
    return (i & 1) ? __high2float(h) : __low2float(h);
}

// One stream's share of the work line.
struct Stream {
    int len, n, off, nq, ub;  // cached, new tokens, first row, row tiles, units of a tile
};
template <int R>
__device__ __forceinline__ Stream stream_of(const AttendArgs &a, int G, int b) {
    Stream s;
    s.len = a.len[b];
    s.off = a.offsets[b];
    s.n = a.offsets[b + 1] - s.off;
    if (s.len < 0 || s.n < 0 || s.off < 0 || s.len > a.max_pos || s.n > a.max_pos - s.len ||
        s.n > a.tokens - s.off) {
        raise_error(a.err, kDevRange);
        s.n = 0;
    }
    s.nq = (s.n * G + R - 1) / R;
    s.ub = (s.len + s.n + kKv4Unit - 1) / kKv4Unit;
    return s;
}

// n / d, in 32 bits where both fit (the work line hardly ever needs more).
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
    if (((n | d) >> 32) == 0) return (int64_t)((uint32_t)n / (uint32_t)d);
    return n / d;
}

// W units split over `blocks` blocks: the first `more` blocks take each + 1
// units, the others `each`.
struct Split {
    int64_t each, more;
    __device__ __forceinline__ Split(int64_t W, int64_t blocks) {
        each = quotient(W, blocks);
        more = W - each * blocks;
    }
    __device__ __forceinline__ int64_t first(int64_t i) const { return i * each + min(i, more); }
    __device__ __forceinline__ int block_of(int64_t w) const {
        const int64_t big = more * (each + 1);
        return (int)(w < big ? quotient(w, each + 1) : more + quotient(w - big, each));
    }
};

// The item that a block begins and others end.
struct Shared {
    int there, h, qt, off, rows;
    int last;  // rank of the block that ends it
};

// A block's part of one item (stream, kv head, row tile).
template <int R>
struct Piece {
    Stream s;
    int h, qt, u0, u1;  // units [u0, u1) of the item's s.ub
    int rows, tok0, tok1;
    int mine;           // units of this warp
    __device__ __forceinline__ void locate(const AttendArgs &a, int G, int b, int64_t rel, int64_t left, int warp) {
        s = stream_of<R>(a, G, b);
        const int item = (int)quotient(rel, s.ub);
        u0 = (int)(rel - (int64_t)item * s.ub);
        h = item / s.nq, qt = item - h * s.nq;
        u1 = (int)min((int64_t)s.ub, u0 + left);
        rows = min(R, s.n * G - qt * R);
        tok0 = qt * R / G, tok1 = (qt * R + rows - 1) / G;
        const int stop = min(u1, (s.len + tok1) / kKv4Unit + 1);  // no row sees units from here on
        mine = stop > u0 + warp ? (stop - u0 - warp + kWarps - 1) / kWarps : 0;
    }
};

template <int D, int NT>
struct Smem {
    static constexpr int R = 4 * NT;
    static constexpr int kRow = D + 8;  // a quarter-warp's 16-byte stores fall on distinct banks
    alignas(128) uint8_t ring[kWarps][kStages][kv4_unit_bytes(D)];
    float wo[kWarps][4][kRow];  // warps' sums, four rows at a time
    float wm[kWarps][4], wl[kWarps][4];
    float po[2][R][D];       // partials: [0] of the item that a block before began, [1] of the one begun here
    float pm[2][R], pl[2][R];
    uint2 qf[NT][D / 16][NT > 1 ? 32 : 1];  // query fragments, by lane
    float rs[R];                                            // and their scales back
    uint64_t full[kWarps][kStages];
    int64_t scan[kWarps];
    Shared open;
    int64_t start[1];  // [streams + 1] first unit of each stream in the work line
};

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_attend(const AttendArgs a) {
    using Sm = Smem<D, NT>;
    using U = Kv4Unit<D>;
    constexpr int R = Sm::R, C = D / 32;
    extern __shared__ uint4 dyn[];
    Sm &sm = *reinterpret_cast<Sm *>(dyn);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int G = a.heads / a.L.kvh;
    if (tid == 0) {
        for (int w = 0; w < kWarps; w++)
            for (int s = 0; s < kStages; s++) mbar_init(&sm.full[w][s], 1);
        mbar_fence_init();
    }
    griddep_launch_dependents();
    griddep_wait();
    // ---- the work line: the streams' units, scanned
    {
        int64_t base = 0;
        for (int b0 = 0; b0 < a.streams; b0 += kThreads) {
            const int b = b0 + tid;
            int64_t w = 0;
            if (b < a.streams) {
                const Stream s = stream_of<R>(a, G, b);
                w = (int64_t)a.L.kvh * s.nq * s.ub;
            }
            int64_t x = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) sm.scan[warp] = x;
            __syncthreads();
            int64_t before = base;
#pragma unroll
            for (int i = 0; i < kWarps; i++) {
                const int64_t part = sm.scan[i];
                if (i < warp) before += part;
                base += part;
            }
            if (b < a.streams) sm.start[b] = before + x - w;
        }
        if (tid == 0) {
            sm.start[a.streams] = base;
            sm.open.there = 0;
        }
    }
    __syncthreads();
    // ---- the cluster's run of whole items: [c0, c1), and how many there are
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank();
    int b = 0;
    int64_t c0, c1, c_items = 0;
    {
        const Split over(sm.start[a.streams], gridDim.x);
        // the item border nearest to unit t; and the items of the line before it
        auto border = [&](int64_t t, int &bt) {
            bt = 0;
            for (int lo = 0, hi = a.streams - 1; lo < hi;) {  // last stream that starts at or before t
                const int mid = (lo + hi + 1) >> 1;
                if (sm.start[mid] <= t) lo = bt = mid;
                else hi = mid - 1;
            }
            const Stream s = stream_of<R>(a, G, bt);
            if (!s.nq) return sm.start[bt];
            return sm.start[bt] + min(quotient(t - sm.start[bt] + s.ub / 2, s.ub), (int64_t)a.L.kvh * s.nq) * s.ub;
        };
        int bt;
        c0 = border(over.first(blockIdx.x), b);
        c1 = border(over.first(blockIdx.x + 1), bt);
        if (c1 > c0) {  // an upper bound of the run's items, exact within one stream
            const Stream s = stream_of<R>(a, G, bt);
            c_items = b == bt ? quotient(c1 - c0, s.ub) : kMaxCluster;
        }
    }
    // a block takes at least one unit per warp, or an item
    const int64_t shares =
        min((int64_t)cl.num_blocks(), max(c_items, (c1 - c0 + kWarps - 1) / kWarps));
    const Split split(c1 - c0, max(shares, (int64_t)1));
    int64_t w = c1, w1 = c1;
    if (rank < shares) w = c0 + split.first(rank), w1 = c0 + split.first(rank + 1);
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    int turn = 0;  // units that this warp's ring has taken
    bool dead = false;
    // The piece at w: its first units are on their way before the piece before it
    // is joined.  (Only what the loop over units needs stays in registers.)
    int h, u0, mine;
    const uint8_t *src = nullptr;
    auto fetch_units = [&](int k) {  // where units k .. k + 31 are (lane = offset)
        if (k + lane >= mine) return;
        const int u = u0 + warp + (k + lane) * kWarps;
        int pg = __ldcg(a.L.table + (int64_t)b * a.L.pages_per_stream + ((u * kKv4Unit) >> a.L.page_shift));
        if ((unsigned)pg >= (unsigned)a.L.pool_pages) {
            raise_error(a.err, kDevRange);
            pg = 0;
        }
        src = a.L.unit(pg, h, u & ((1 << (a.L.page_shift - 5)) - 1), D);
    };
    auto issue = [&](int k) {
        const uint8_t *from = reinterpret_cast<const uint8_t *>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), k & 31));
        if (lane == 0) {
            const int st = (turn + k) % kStages;
            mbar_arrive_expect_tx(&sm.full[warp][st], U::kBytes);
            bulk_g2s(&sm.ring[warp][st][0], from, U::kBytes, &sm.full[warp][st]);
        }
    };
    auto begin = [&]() {
        while (sm.start[b + 1] <= w) b++;
        Piece<R> p;
        p.locate(a, G, b, w - sm.start[b], w1 - w, warp);
        h = p.h, u0 = p.u0, mine = p.mine;
        {  // the queries are on their way to the first level while the table is read
            const int row = p.qt * R + lane / (32 / R);
            if (row < p.s.n * G) {
                const float *q = a.q + ((int64_t)(p.s.off + row / G) * a.heads + h * G + row % G) * D;
                const int line = lane % (32 / R);
                if (line < D / 32 && warp == 0) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + line * 32));
            }
        }
        fetch_units(0);
        if (!dead)
            for (int k = 0; k < kStages && k < mine; k++) issue(k);
    };
    if (w < w1) begin();
    while (w < w1) {
        int first_limit;  // every row sees the positions up to here
        Piece<R> p;
        p.locate(a, G, b, w - sm.start[b], w1 - w, warp);
        first_limit = p.s.len + p.tok0;

        // ---- query fragments: column n = 2 row + {hi, lo}.  A tile of one column group has
        // them in registers, every warp its own; a wider one in shared memory.
        auto load_q = [&](int nt, uint32_t (&f)[2 * C][2]) {
            const int row = p.qt * R + nt * 4 + (g >> 1);
            const bool have = row < p.s.n * G;
            const float4 *q = reinterpret_cast<const float4 *>(
                a.q + ((int64_t)(p.s.off + (have ? row / G : 0)) * a.heads + h * G + (have ? row % G : 0)) * D + 8 * t);
            float x[C][8];
            float amax = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const float4 v0 = have ? __ldg(q + 8 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 v1 = have ? __ldg(q + 8 * c + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[c][0] = v0.x, x[c][1] = v0.y, x[c][2] = v0.z, x[c][3] = v0.w;
                x[c][4] = v1.x, x[c][5] = v1.y, x[c][6] = v1.z, x[c][7] = v1.w;
#pragma unroll
                for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(x[c][j]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // 2^e puts the row's largest value into [2^9, 2^10)
            int e = 136 - (int)(__float_as_uint(amax) >> 23);
            e = (amax > 0.0f && isfinite(amax)) ? max(-120, min(120, e)) : 0;
            const float up = __int_as_float((127 + e) << 23), down = __int_as_float((127 - e) << 23);
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float y0 = x[c][j] * up, y1 = x[c][j + 4] * up;
                    const float h0 = __half2float(__float2half_rn(y0)), h1 = __half2float(__float2half_rn(y1));
                    if (g & 1) y0 -= h0, y1 -= h1;
                    else y0 = h0, y1 = h1;
                    f[2 * c + (j >> 1)][j & 1] = h2u(__floats2half2_rn(y0, y1));
                }
            return down * a.scale_log2;  // of row g >> 1
        };
        uint32_t bq[2 * C][2];
        float rs[NT], m[NT], l[NT];
        int limit[NT];
        float acc[NT][C][4];
        if constexpr (NT == 1) {
            rs[0] = load_q(0, bq);
            rs[0] = __shfl_sync(0xffffffffu, rs[0], t * 8);
        } else {
            if (warp < NT) {
                const float r = load_q(warp, bq);
#pragma unroll
                for (int i = 0; i < 2 * C; i++) sm.qf[warp][i][lane] = make_uint2(bq[i][0], bq[i][1]);
                if ((lane & 7) == 0) sm.rs[warp * 4 + (lane >> 3)] = r;
            }
            __syncthreads();
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if constexpr (NT > 1) rs[nt] = sm.rs[nt * 4 + t];
            const int mr = p.qt * R + nt * 4 + t;  // this lane's row
            limit[nt] = mr < p.s.n * G ? p.s.len + mr / G : -1;
            m[nt] = -INFINITY;
            l[nt] = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[nt][c][i] = 0.0f;
        }
        int ke = 24;  // values are accumulated times 2^ke

        for (int k = 0; k < mine && !dead; k++) {
            const int u = u0 + warp + k * kWarps;
            const int st = (turn + k) % kStages;
            const bool here = mbar_wait_bounded(&sm.full[warp][st], ((turn + k) / kStages) & 1, a.err);
            if (__any_sync(0xffffffffu, !here)) {
                dead = true;
                // no copy is left in flight behind the block (a limit again)
                for (int j = k; j < min(mine, k + kStages); j++)
                    mbar_wait_bounded(&sm.full[warp][(turn + j) % kStages], ((turn + j) / kStages) & 1, a.err);
                break;
            }
            const uint8_t *unit = &sm.ring[warp][st][0];
            float sc[NT][4];  // scores of positions g, g + 8, g + 16, g + 24
            float sl[NT][4];  // from the queries' lo halves
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) sc[nt][i] = sl[nt][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const uint4 kw = *reinterpret_cast<const uint4 *>(unit + U::kK + c * 512 + lane * 16);
                const uint2 ks = *reinterpret_cast<const uint2 *>(unit + U::kKs + c * 64 + g * 8);
                uint32_t x[4][4];  // positions g, g + 8, g + 16, g + 24
                codes(kw.x, magic, x[0]);
                codes(kw.y, magic, x[1]);
                codes(kw.z, magic, x[2]);
                codes(kw.w, magic, x[3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    uint2 b0, b1;
                    if constexpr (NT == 1) {
                        b0 = make_uint2(bq[2 * c][0], bq[2 * c][1]), b1 = make_uint2(bq[2 * c + 1][0], bq[2 * c + 1][1]);
                    } else {
                        b0 = sm.qf[nt][2 * c][lane], b1 = sm.qf[nt][2 * c + 1][lane];
                    }
#pragma unroll
                    for (int rt = 0; rt < 2; rt++) {
                        const uint32_t(&x0)[4] = x[2 * rt], (&x1)[4] = x[2 * rt + 1];
                        const float f0 = scale_of(ks, 2 * rt), f1 = scale_of(ks, 2 * rt + 1);
                        float d[4];
                        mma16816_first(d, x0[0], x1[0], x0[1], x1[1], b0.x, b0.y);
                        mma16816(d, x0[2], x1[2], x0[3], x1[3], b1.x, b1.y);
                        sc[nt][2 * rt] = fmaf(f0, d[0], sc[nt][2 * rt]);
                        sl[nt][2 * rt] = fmaf(f0, d[1], sl[nt][2 * rt]);
                        sc[nt][2 * rt + 1] = fmaf(f1, d[2], sc[nt][2 * rt + 1]);
                        sl[nt][2 * rt + 1] = fmaf(f1, d[3], sl[nt][2 * rt + 1]);
                    }
                }
            }
            const bool edge = u * kKv4Unit + kKv4Unit - 1 > first_limit;
            // the largest value scale of the unit sets the power of two; what an earlier
            // user of the page left behind the last position that a row sees counts as zero
            uint2 vs[C];
            __half2 b0 = __half2half2(__ushort_as_half(0)), b1 = b0;  // of positions g, g + 8 and g + 16, g + 24
#pragma unroll
            for (int c = 0; c < C; c++) {
                vs[c] = *reinterpret_cast<const uint2 *>(unit + U::kVs + c * 64 + g * 8);
                b0 = __hmax2(b0, u2h(vs[c].x)), b1 = __hmax2(b1, u2h(vs[c].y));
            }
            if (edge) {
                int lim = limit[0];
#pragma unroll
                for (int nt = 1; nt < NT; nt++) lim = max(lim, limit[nt]);
                lim = __reduce_max_sync(0xffffffffu, lim) - u * kKv4Unit - g;
                b0 = u2h(h2u(b0) & ((lim >= 0 ? 0xffffu : 0u) | (lim >= 8 ? 0xffff0000u : 0u)));
                b1 = u2h(h2u(b1) & ((lim >= 16 ? 0xffffu : 0u) | (lim >= 24 ? 0xffff0000u : 0u)));
            }
            __half2 big = __hmax2(b0, b1);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) big = __hmax2(big, u2h(__shfl_xor_sync(0xffffffffu, h2u(big), o)));
            const unsigned bits = h2u(__hmax2(big, __lowhigh2highlow(big))) & 0x7c00u;
            const int kn = 24 - (int)(bits >> 10);  // (sums stay under 2^20 2^19 2^24)
            const float shrink = __int_as_float((127 + kn - ke) << 23), lift = __int_as_float((127 + kn) << 23);
            ke = kn;
            float keep[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[nt][i] = (sc[nt][i] + sl[nt][i]) * rs[nt];
                }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (u * kKv4Unit + g + 8 * i > limit[nt]) sc[nt][i] = -INFINITY;
                }
                float mx = fmaxf(fmaxf(sc[nt][0], sc[nt][1]), fmaxf(sc[nt][2], sc[nt][3]));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                mx = fmaxf(mx, m[nt]);
                const float ref = mx == -INFINITY ? 0.0f : mx;
                const float corr = ex2(m[nt] - ref);
                m[nt] = mx;
                keep[nt] = corr * shrink;
#pragma unroll
                for (int i = 0; i < 4; i++) sc[nt][i] = ex2(sc[nt][i] - ref);
                // (one addition a unit to the running sum, as the weighted sums have)
                l[nt] = fmaf(l[nt], corr, (sc[nt][0] + sc[nt][1]) + (sc[nt][2] + sc[nt][3]));
#pragma unroll
                for (int i = 0; i < 4; i++) sc[nt][i] *= lift;
            }
#pragma unroll
            for (int c = 0; c < C; c++) {
                const uint4 vw = *reinterpret_cast<const uint4 *>(unit + U::kV + c * 512 + U::v_chunk(g, t));
                uint32_t x[4][4];
                codes(vw.x, magic, x[0]);
                codes(vw.y, magic, x[1]);
                codes(vw.z, magic, x[2]);
                codes(vw.w, magic, x[3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    uint32_t bp[4];
                    if (edge) {  // whatever lies behind a row's last position counts as zero
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            bp[i] = split_hi_lo(u * kKv4Unit + g + 8 * i > limit[nt] ? 0.0f : sc[nt][i] * scale_of(vs[c], i));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) bp[i] = split_hi_lo(sc[nt][i] * scale_of(vs[c], i));
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) bp[i] = transpose8x8(bp[i]);
                    float d0[4], d1[4];
                    mma16816_first(d0, x[0][0], x[0][1], x[1][0], x[1][1], bp[0], bp[1]);
                    mma16816_first(d1, x[0][2], x[0][3], x[1][2], x[1][3], bp[0], bp[1]);
                    mma16816(d0, x[2][0], x[2][1], x[3][0], x[3][1], bp[2], bp[3]);
                    mma16816(d1, x[2][2], x[2][3], x[3][2], x[3][3], bp[2], bp[3]);
                    acc[nt][c][0] = fmaf(acc[nt][c][0], keep[nt], d0[0] + d0[1]);
                    acc[nt][c][1] = fmaf(acc[nt][c][1], keep[nt], d0[2] + d0[3]);
                    acc[nt][c][2] = fmaf(acc[nt][c][2], keep[nt], d1[0] + d1[1]);
                    acc[nt][c][3] = fmaf(acc[nt][c][3], keep[nt], d1[2] + d1[3]);
                }
            }
            __syncwarp();  // the stage is read
            if (k + kStages < mine) {
                if (((k + kStages) & 31) == 0) fetch_units(k + kStages);
                issue(k + kStages);
            }
        }
        turn += mine;
        // the piece is joined below: what the loop did not need is found again
        p.locate(a, G, b, w - sm.start[b], w1 - w, warp);
        const int64_t item0 = w - p.u0;
        w += p.u1 - p.u0;
        const bool more = w < w1;
        if (more) begin();

        // ---- join the warps, four rows at a time
        const float unlift = __int_as_float((127 - ke) << 23);
        const bool whole = p.u0 == 0 && p.u1 == p.s.ub;
        const int part = p.u0 == 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], o);
            if (nt > 0) {
                if (nt * 4 >= p.rows) break;
                __syncthreads();
            }
            if (g == 0) {
                sm.wm[warp][t] = m[nt];
                sm.wl[warp][t] = l[nt];
            }
            if (nt * 4 + t < p.rows)
#pragma unroll
                for (int c = 0; c < C; c++)
                    *reinterpret_cast<float4 *>(&sm.wo[warp][t][32 * c + 4 * g]) =
                        make_float4(acc[nt][c][0] * unlift, acc[nt][c][1] * unlift, acc[nt][c][2] * unlift,
                                    acc[nt][c][3] * unlift);
            __syncthreads();
            for (int i = tid; i < min(4, p.rows - nt * 4) * D; i += kThreads) {
                const int r4 = i / D, r = nt * 4 + r4, d = i % D;
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < kWarps; x++) mx = fmaxf(mx, sm.wm[x][r4]);
                const float ref = mx == -INFINITY ? 0.0f : mx;
                float o = 0.0f, sum = 0.0f;
#pragma unroll
                for (int x = 0; x < kWarps; x++) {
                    const float f = ex2(sm.wm[x][r4] - ref);
                    o = fmaf(f, sm.wo[x][r4][d], o);
                    sum = fmaf(f, sm.wl[x][r4], sum);
                }
                if (whole) {
                    const int row = p.qt * R + r;
                    a.out[((int64_t)(p.s.off + row / G) * a.heads + p.h * G + row % G) * D + d] = __fdiv_rn(o, sum);
                } else {
                    sm.po[part][r][d] = o;
                    if (d == 0) {
                        sm.pm[part][r] = mx;
                        sm.pl[part][r] = sum;
                    }
                }
            }
        }
        if (!whole && part && tid == 0)
            sm.open = Shared{1, p.h, p.qt, p.s.off, p.rows, split.block_of(item0 + p.s.ub - 1 - c0)};
        __syncthreads();
    }

    // ---- the item that this block began and others ended: their first partials
    cl.sync();
    if (sm.open.there) {
        const Shared e = sm.open;
        for (int i = tid; i < e.rows * D; i += kThreads) {
            const int r = i / D, d = i % D;
            float pm[kMaxCluster], po[kMaxCluster], pl[kMaxCluster];  // (all reads in flight together)
            pm[0] = sm.pm[1][r], po[0] = sm.po[1][r][d], pl[0] = sm.pl[1][r];
#pragma unroll
            for (int x = 1; x < kMaxCluster; x++) {
                const Sm *q = cl.map_shared_rank(&sm, rank + x <= e.last ? rank + x : rank);
                pm[x] = rank + x <= e.last ? q->pm[0][r] : -INFINITY;
                po[x] = rank + x <= e.last ? q->po[0][r][d] : 0.0f;
                pl[x] = rank + x <= e.last ? q->pl[0][r] : 0.0f;
            }
            float mx = pm[0], o = 0.0f, sum = 0.0f;
#pragma unroll
            for (int x = 1; x < kMaxCluster; x++) mx = fmaxf(mx, pm[x]);
#pragma unroll
            for (int x = 0; x < kMaxCluster; x++) {
                const float f = ex2(pm[x] - mx);
                o = fmaf(f, po[x], o);
                sum = fmaf(f, pl[x], sum);
            }
            const int row = e.qt * R + r;
            a.out[((int64_t)(e.off + row / G) * a.heads + e.h * G + row % G) * D + d] = __fdiv_rn(o, sum);
        }
    }
    cl.sync();  // no block leaves while another reads its partials
}

// A cluster launch of `kern` with `cs` blocks a cluster.
void cluster_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute &at, int clusters, int cs, size_t smem) {
    cfg = {};
    cfg.gridDim = dim3(clusters, cs);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 1;
    at.val.clusterDim.y = cs;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
}

constexpr int kSizes[3] = {8, 4, 2};  // blocks of a cluster

template <int D, int NT>
size_t smem_of(int streams) { return sizeof(Smem<D, NT>) + (size_t)streams * 8; }

// How many clusters of each size run at once.
template <int D, int NT>
int clusters_of(const qora_kv4 *kv, int (&n)[3]) {
    auto kern = k_kv4_attend<D, NT>;
    const size_t smem = smem_of<D, NT>(kv->streams);
    static std::atomic<uint64_t> done;  // (as much as the most streams need: caches share the kernel)
    QORA_TRY(allow_smem(kern, smem_of<D, NT>(kKv4MaxStreams), kv->ctx->device, done));
    for (int i = 0; i < 3; i++) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute at;
        cluster_config(cfg, at, 1, kSizes[i], smem);
        QORA_CUDA(cudaOccupancyMaxActiveClusters(&n[i], kern, &cfg));
        if (n[i] < 1) n[i] = 1;
    }
    return QORA_OK;
}

// The cluster size goes by the items (stream, kv head, row tile) that the call may
// have, at most one stream a token (a cache of 64 streams with one of 16384 positions
// at work: 53 us by the cache's streams, 23.5 by the call's): with few, a wide cluster puts more blocks on each; with many, narrow ones
// leave no multiprocessor without a block (33 clusters of 8, 71 of 4 or 148 of 2
// run at once).  Measured at 16 / 8 heads of 128, one token: 1 stream of 16384
// positions 23.4 us with clusters of 8, 34.2 with 4; 8 streams of 4096 23.1 us with
// 8, 19.5 with 4, 25.9 with 2; 32 streams of 4096 46.8 us with 8, 43.1 with 2.
template <int D, int NT>
int launch(const qora_kv4 *kv, const AttendArgs &a, const int (&n)[3], int64_t items, cudaStream_t st) {
    auto kern = k_kv4_attend<D, NT>;
    const size_t smem = smem_of<D, NT>(a.streams);
    const int i = items <= n[0] ? 0 : items <= n[1] ? 1 : 2;
    return launch_ex(kern, dim3(n[i], kSizes[i]), dim3(kThreads), smem, st, (unsigned)kSizes[i], a);
}

}  // namespace

namespace {
template <int D>
int setup(qora_kv4 *kv) {
    QORA_TRY((clusters_of<D, 1>(kv, kv->clusters[0])));
    return clusters_of<D, 2>(kv, kv->clusters[1]);
}
// Row tiles of 4 or 8: 4 also where each of them has a cluster of 8 blocks of its own
// (one stream of 1000 positions, 16 / 8 heads: 10.3 us against 12.6 with 8 rows a kv
// head, 10.9 against 13.6 with 16; 4 streams of 4000, past that: 22.3 against 17.9).  (Tiles of 12 read the cache once where these read it twice,
// but do not fit 128 registers: 6 drafts of 16 streams of 4096 took 58 us against 40.)
template <int D>
int launch_rows(const qora_kv4 *kv, const AttendArgs &a, int64_t rows, cudaStream_t st) {
    // the most items of R rows that the call's tokens make: every stream that has one ends
    // in a tile of its own
    const int64_t S = std::min(kv->streams, a.tokens), all = (int64_t)a.tokens * (a.heads / kv->kvh);
    const auto most = [&](int R) { return kv->kvh * std::min(S * ((rows + R - 1) / R), S + all / R); };
    const int nt = rows <= 4 || most(4) <= kv->clusters[0][0] ? 1 : 2;
    const int64_t items = most(4 * nt);
    const auto &n = kv->clusters[nt - 1];
    return nt == 1 ? launch<D, 1>(kv, a, n, items, st) : launch<D, 2>(kv, a, n, items, st);
}
}  // namespace

namespace {
// Whether the prompt kernel (tiles of 128 rows, one block a multiprocessor) is the
// better one.  Both take time in proportion to the positions, so tiles decide: here
// all tiles of 8 rows share the machine, there the waves of blocks count, one wave
// as long as 400 tiles of 8 at head_dim 128, 600 at 64.  Measured at
// 16 / 8 heads of 128, us here / there: 16 streams of 2000 positions 34 / 51 with 16
// rows a kv head, 63 / 51 with 32, 113 / 51 with 64; 32 streams of 4096 118 / 215 with
// 16, 207 / 216 with 32, 317 / 216 with 48; 4 streams of 4000 60 / 88 with 64, 100 / 90
// with 96; one stream of 1000 22 / 29 with 128, of 8000 61 / 165.  At head_dim 64, 16
// streams of 2000 positions: 40 / 41 with 32 rows, 58 / 41 with 48.  (Rows are all that
// the host knows: lengths lie on the device, and one kernel takes all streams of a call.
// 63 streams of 4096 with one token beside a prompt of 2048 take 529 us here, where calls
// of their own take 83 and 168.)
bool prompt_pays(const qora_kv4 *kv, int64_t tokens, int64_t max_count, int64_t rows) {
    if (rows <= 24) return false;
    const int64_t G = kv->heads / kv->kvh, streams = std::min<int64_t>(kv->streams, tokens);
    const int64_t all = G * std::min(tokens, streams * max_count);
    const int64_t here = kv->kvh * std::max(streams, (all + 7) / 8), there = kv->kvh * std::max(streams, (all + 127) / 128);
    const int64_t waves = (there + kv->ctx->num_sms - 1) / kv->ctx->num_sms;
    return here > (kv->hd == 64 ? 600 : 400) * waves;
}
}  // namespace

int kv4_attend_setup(qora_kv4 *kv) { return kv->hd == 64 ? setup<64>(kv) : setup<128>(kv); }

}  // namespace qora

using namespace qora;

extern "C" int qora_kv4_attend(qora_kv4 *kv, int32_t layer, const float *q, const int32_t *offsets, int32_t tokens,
                               int32_t max_count, float *out, void *stream) {
    if (!kv || !offsets || tokens < 0 || max_count < 1 || (tokens > 0 && (!q || !out)))
        return set_error(QORA_ERR_INVALID, "qora_kv4_attend: bad arguments");
    if (layer < 0 || layer >= kv->layers)
        return set_error(QORA_ERR_INVALID, "qora_kv4_attend: layer %d out of range", layer);
    if (!tokens) return QORA_OK;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
        return set_error(QORA_ERR_INVALID, "qora_kv4_attend: pointers must be 16-byte aligned");
    DeviceGuard dg;
    QORA_TRY(dg.set(kv->ctx->device));
    AttendArgs a;
    a.L = kv4_layer(kv, layer);
    a.q = q;
    a.offsets = offsets;
    a.len = kv->len.as<int>();
    a.out = out;
    a.err = kv->ctx->err.as<int>();
    a.streams = kv->streams;
    a.heads = kv->heads;
    a.max_pos = kv->max_pos;
    a.tokens = tokens;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)kv->hd);
    const int64_t rows = kv->heads / kv->kvh * (int64_t)max_count;  // of a stream's kv head
    if (prompt_pays(kv, tokens, max_count, rows))
        return kv4_launch_prompt(kv, layer, q, offsets, tokens, std::min(rows, (int64_t)tokens * (kv->heads / kv->kvh)), out,
                                 as_stream(stream));
    return kv->hd == 64 ? launch_rows<64>(kv, a, rows, as_stream(stream)) : launch_rows<128>(kv, a, rows, as_stream(stream));
}
