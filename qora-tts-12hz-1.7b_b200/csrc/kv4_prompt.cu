// Attention over the 4-bit paged cache for prompts (k_kv4_prompt): many new
// tokens per stream, on the tensor cores through tensor memory.
//
// The same mathematics as k_kv4_attend, for tiles of 128 query rows (a row = one
// head of one token; the heads that share a kv head are neighbours) against 64
// positions at a time:
//   S = Q K^T      three products of f16 pairs: Qh Kh + Qh Kl + Ql Kh
//   P = 2^(S - m)  f32, one row a thread pair, running maximum and sum
//   O += P V       three products, Ph Vh + Ph Vl + Pl Vh
// A cached value s c has 15 significant bits: h = f16(s c) and l = s c - h are
// exact in f16, two packed instructions for two values.  Scales are multiplied by
// a power of two per 64 positions (so that neither half leaves f16's range for any
// stored scale), queries by one per row, both undone exactly.  The dropped
// products of two low halves are 2^-22 of the result.
//
// Four kinds of warps work on different tiles at the same time: four unpack keys
// and four values into shared memory as matrix operands (two buffers each), one
// issues the products, eight do the softmax: a thread has one row, half of its
// positions for P and half of its dimensions for O.  P goes back to tensor memory as an operand.
// The unit's layout gives a lane whole 16-byte operand rows: eight dimensions of a
// key, and eight positions of a value's dimension (in the order 2t + e + 8h, which
// P's columns follow).  O of each tile is added in f32 registers, because the
// tensor core's own additions do not round to nearest.
//
// 2 prompts of 2048 and some 1700 tokens, 16 / 8 heads of 128: 124 us in a captured loop,
// 187 TFLOP/s of the two products (three times that on the tensor cores), and 131 to 136
// as one call among others.  What bounds it is the
// softmax warps' chain of a tile, some 2400 cycles of wait, maximum, exponentials,
// P and sum of O, against 1540 of products; and 6 us a block outside its tiles.
// Unpacking in the same warps as the issue of products took 360 us, one group of
// warps for keys and values 163, and four warps of their own for the sums of O, at
// 80 registers for the softmax, 163.
#include <type_traits>

#include "kv4.cuh"
#include "tc.cuh"

namespace qora {

namespace {

constexpr int kRows = 128;                 // query rows of a block
constexpr int kKeys = 64;                  // positions of a tile: two units
constexpr int kSoftWarps = 8, kUnpackWarps = 4;      // (as many for keys as for values)
constexpr int kThreads = (kSoftWarps + 2 * kUnpackWarps + 4) * 32;  // whole groups of four warps; one of the last has work
// Registers of a thread: at launch, and as the groups of warps share them out.
constexpr int kRegs = 96, kSoftRegs = 136, kUnpackRegs = 72, kLastRegs = 64;
static_assert(kSoftWarps * kSoftRegs + 2 * kUnpackWarps * kUnpackRegs + 4 * kLastRegs <= kThreads / 32 * kRegs,
              "no group waits for registers that the block does not have");
constexpr uint32_t kTmemCols = 512;        // S 2 x 64, P (high, low) 2 x 64, O 128, Q (high, low) 128
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256, kColQ = 384;

struct PromptArgs {
    Kv4Layer L;
    const float *q;
    const int *offsets, *len;
    float *out;
    int *err;
    int streams, heads, max_pos, tokens;
    float scale_log2;  // log2(e) / sqrt(D)
};

// K and V in shared memory: core matrices of 8 rows x 16 bytes.  The distance
// between neighbours along the contraction is 160 bytes for K and 144 for V, so
// that the unpacking warps' 16-byte stores fall on distinct banks.  Q and P are
// operands in tensor memory (Q from shared memory made the products' rate that of
// its reads: 64 cycles for 128 x 64 x 16).
template <int D>
struct Sm {
    static constexpr int kKStep = 160, kVStep = 144;
    static constexpr int kK = (kKeys / 8) * (D / 8) * kKStep;
    static constexpr int kV = (D / 8) * (kKeys / 8) * kVStep;
    alignas(128) uint8_t k[2][2][kK];      // [buffer][high, low]
    alignas(128) uint8_t v[2][2][kV];
    // a softmax warp's halves of rows on their way in and out, 16 bytes at a time (place of
    // piece c of row r: c ^ r, so that rows and columns of pieces both fall on distinct banks)
    float4 stage[kSoftWarps][32][D / 8];
    float l[2][kRows], top[2][2][kRows];   // a row's sum, and largest score, by half
    // of a tile (four deep: unpacking is up to three tiles ahead of the softmax)
    float unk[4], unv[4];                  // its scales back
    unsigned vnan[4][2][D / 32];           // positions of a unit whose value scale is NaN, by group
    unsigned most[2][2][kUnpackWarps];     // largest scales: keys, values
    alignas(8) uint64_t info[4];           // these are written (k_full may be a phase too far by then)
    uint64_t q_full, k_full[2], v_full[2], s_full[2], p_full[2], o_full[2], o_free, drained;
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }

// Bounded wait of one thread: false when it ran out here or in another warp.
__device__ __forceinline__ bool wait_one(uint64_t *bar, uint32_t parity, int *abort, int *err) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*(volatile int *)abort) return false;  // (ends every wait of the block soon after one ran out)
        if (global_ns() - t0 > 1000000000ull) {
            raise_error(err, kDevTimeout);
            *(volatile int *)abort = 1;
            return false;
        }
    }
    return true;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, int *abort, int *err) {
    return __all_sync(0xffffffffu, wait_one(bar, parity, abort, err));
}

// Two f32 at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n mov.b64 c, {%5, %6};\n"
        " fma.rn.f32x2 %0, a, b, c;\n}"
        : "=l"(r)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("{\n .reg .b64 a, b;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n add.rn.f32x2 %0, a, b;\n}"
        : "=l"(r)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <uint32_t Mask>
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(Mask), "r"(magic));
    return r;
}
// The four pairs of codes of a word: x[j] = (nibble j, nibble j + 4) - 8 in f16.
__device__ __forceinline__ void codes(uint32_t w, uint32_t magic, __half2 (&x)[4]) {
    const __half2 lo = __half2half2(__ushort_as_half(0x6408));    // 1032
    const __half2 s16 = __half2half2(__ushort_as_half(0x2c00));   // 1 / 16
    const __half2 hi = __half2half2(__ushort_as_half(0xd480));    // -72
    const uint32_t v = w >> 8;
    x[0] = __hsub2(u2h(and_or<0x000f000fu>(w, magic)), lo);
    x[1] = __hfma2(u2h(and_or<0x00f000f0u>(w, magic)), s16, hi);
    x[2] = __hsub2(u2h(and_or<0x000f000fu>(v, magic)), lo);
    x[3] = __hfma2(u2h(and_or<0x00f000f0u>(v, magic)), s16, hi);
}

// What a lane of an unpacking warp has of one (unit, scale group): codes, and the
// scales of keys g + 8i, or of values 2t + 8i and 2t + 1 + 8i.
template <bool V>
struct Raw {
    uint4 c;
    uint2 s[V ? 2 : 1];
};

__device__ __forceinline__ float half_of(uint2 v, int i) {
    const __half2 h = u2h(i < 2 ? v.x : v.y);
    return (i & 1) ? __high2float(h) : __low2float(h);
}

// The power of two that brings scales up to `bits` (f16, finite) under 2^12.
__device__ __forceinline__ int scale_exponent(unsigned bits) { return 26 - (int)((bits >> 10) & 31u); }

// A row tile's keys or values, as matrix operands: the loop of an unpacking warp.
template <int D, bool V>
__device__ __forceinline__ void unpack(Sm<D> &sm, const PromptArgs &a, int b, int h, int ntiles, int kend, int done) {
    using S = Sm<D>;
    using U = Kv4Unit<D>;
    constexpr int C = D / 32;
    constexpr int kJobs = 2 * C / kUnpackWarps;  // (unit, group) pairs of a warp and tile
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pw = (threadIdx.x >> 5) % kUnpackWarps;
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    const int *table = a.L.table + (int64_t)b * a.L.pages_per_stream;
    auto page_of = [&](int it, int job) {  // physical page of a job's unit, -1 behind the last position
        const int pos = it * kKeys + ((pw + kUnpackWarps * job) / C) * kKv4Unit;
        if (it >= ntiles || pos >= kend) return -1;
        int pg = __ldg(table + (pos >> a.L.page_shift));
        if ((unsigned)pg >= (unsigned)a.L.pool_pages) {
            raise_error(a.err, kDevRange);
            pg = 0;
        }
        return pg;
    };
    auto load = [&](int it, int job, int pg, Raw<V> &r) {
        r = Raw<V>{};
        if (pg < 0) return;
        const int combo = pw + kUnpackWarps * job, c = combo % C;
        const int pos = it * kKeys + (combo / C) * kKv4Unit;
        const uint8_t *u = a.L.unit(pg, h, (pos >> 5) & ((1 << (a.L.page_shift - 5)) - 1), D);
        if constexpr (V) {
            r.c = __ldg(reinterpret_cast<const uint4 *>(u + U::kV + c * 512 + U::v_chunk(g, t)));
            r.s[0] = __ldg(reinterpret_cast<const uint2 *>(u + U::kVs + c * 64 + 2 * t * 8));
            r.s[1] = __ldg(reinterpret_cast<const uint2 *>(u + U::kVs + c * 64 + (2 * t + 1) * 8));
        } else {
            r.c = __ldg(reinterpret_cast<const uint4 *>(u + U::kK + c * 512 + lane * 16));
            r.s[0] = __ldg(reinterpret_cast<const uint2 *>(u + U::kKs + c * 64 + g * 8));
        }
    };
    Raw<V> raw[kJobs], next[kJobs];
    int page[kJobs];
#pragma unroll
    for (int j = 0; j < kJobs; j++) {
        load(0, j, page_of(0, j), raw[j]);
        page[j] = page_of(1, j);
    }
    for (int it = 0; it < ntiles; it++) {
        const int gi = done + it, buf = gi & 1, slot = gi & 3;
        // the next tile is in flight while this one is unpacked
#pragma unroll
        for (int j = 0; j < kJobs; j++) {
            load(it + 1, j, page[j], next[j]);
            page[j] = page_of(it + 2, j);
        }
        // the largest scale; ones behind the last position count as zero, and NaN ones of
        // values are told to the rows (both are rare: a packed maximum finds them)
        unsigned most = 0;
        unsigned nan[kJobs];
#pragma unroll
        for (int j = 0; j < kJobs; j++) {
            const int pos = it * kKeys + ((pw + kUnpackWarps * j) / C) * kKv4Unit;
            nan[j] = 0;
            unsigned m2 = __vmaxu2(raw[j].s[0].x, raw[j].s[0].y);
            if constexpr (V) m2 = __vmaxu2(m2, __vmaxu2(raw[j].s[1].x, raw[j].s[1].y));
            const unsigned m1 = max(m2 & 0xffffu, m2 >> 16);
            if (!__any_sync(0xffffffffu, m1 >= 0x7c00u) && pos + kKv4Unit <= kend) {
                most = max(most, m1);
                continue;
            }
#pragma unroll
            for (int e = 0; e < (V ? 2 : 1); e++) {
                const uint2 w = raw[j].s[e];
                unsigned x[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int at = (V ? 2 * t + e : g) + 8 * i;
                    if (pos + at >= kend) x[i] = 0;
                    if (V && x[i] >= 0x7c00u) nan[j] |= 1u << at, x[i] = 0;
                    if (x[i] < 0x7c00u) most = max(most, x[i]);
                }
                if (V) raw[j].s[e] = make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16);
            }
            if (V) nan[j] = __reduce_or_sync(0xffffffffu, nan[j]);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) sm.most[V][buf][pw] = most;
        asm volatile("bar.sync %0, 128;" ::"n"(V ? 7 : 2) : "memory");
#pragma unroll
        for (int i = 0; i < kUnpackWarps; i++) most = max(most, sm.most[V][buf][i]);
        const int e = scale_exponent(most);
        const float up = pow2(e);
        if constexpr (!V) {
            if (gi >= 2) wait_for(&sm.s_full[buf], ((gi >> 1) - 1) & 1, &sm.abort, a.err);
            if (pw == 0 && lane == 0) sm.unk[slot] = pow2(-e);  // (tile gi - 4 of the slot has been read by now)
#pragma unroll
            for (int j = 0; j < kJobs; j++) {
                const int combo = pw + kUnpackWarps * j, c = combo % C, u = combo / C;
                const uint32_t kw[4] = {raw[j].c.x, raw[j].c.y, raw[j].c.z, raw[j].c.w};
                // keys g + 8i: dimensions 32c + 8t .. + 7 are one operand row of 16 bytes
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    __half2 x[4];
                    codes(kw[i], magic, x);
                    const __half2 s = __float2half2_rn(half_of(raw[j].s[0], i) * up);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int p = 0; p < 4; p++) {
                        const __half2 w = __hmul2(s, x[p]);
                        hi[p] = h2u(w);
                        lo[p] = h2u(__hfma2(s, x[p], __hneg2(w)));
                    }
                    const int at = ((4 * u + i) * (D / 8) + 4 * c + t) * S::kKStep + g * 16;
                    *reinterpret_cast<uint4 *>(sm.k[buf][0] + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4 *>(sm.k[buf][1] + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                raw[j] = next[j];
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.info[slot]);
                mbar_arrive(&sm.k_full[buf]);
            }
        } else {
            if (lane == 0) {
                if (pw == 0) sm.unv[slot] = pow2(-e);
#pragma unroll
                for (int j = 0; j < kJobs; j++) {
                    const int combo = pw + kUnpackWarps * j;
                    sm.vnan[slot][combo / C][combo % C] = nan[j];
                }
                mbar_arrive(&sm.info[slot]);
            }
            if (gi >= 2) wait_for(&sm.o_full[buf], ((gi >> 1) - 1) & 1, &sm.abort, a.err);
#pragma unroll
            for (int j = 0; j < kJobs; j++) {
                const int combo = pw + kUnpackWarps * j, c = combo % C, u = combo / C;
                const uint32_t vw[4] = {raw[j].c.x, raw[j].c.y, raw[j].c.z, raw[j].c.w};
                // dimensions 32c + 4g + p: positions 2t + e + 8i are one operand row
                uint32_t hi[4][4], lo[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    __half2 x[4];
                    codes(vw[i], magic, x);
                    // a word is two positions: the pair of nibble p has both
                    const __half2 s = __floats2half2_rn(half_of(raw[j].s[0], i) * up, half_of(raw[j].s[1], i) * up);
#pragma unroll
                    for (int p = 0; p < 4; p++) {
                        const __half2 w = __hmul2(s, x[p]);
                        hi[p][i] = h2u(w);
                        lo[p][i] = h2u(__hfma2(s, x[p], __hneg2(w)));
                    }
                }
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const int at = ((4 * c + (g >> 1)) * (kKeys / 8) + 4 * u + t) * S::kVStep + (4 * (g & 1) + p) * 16;
                    *reinterpret_cast<uint4 *>(sm.v[buf][0] + at) = make_uint4(hi[p][0], hi[p][1], hi[p][2], hi[p][3]);
                    *reinterpret_cast<uint4 *>(sm.v[buf][1] + at) = make_uint4(lo[p][0], lo[p][1], lo[p][2], lo[p][3]);
                }
                raw[j] = next[j];
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.v_full[buf]);
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) k_kv4_prompt(const PromptArgs a) {
    using S = Sm<D>;
    constexpr int C = D / 32;
    extern __shared__ __align__(1024) uint8_t dyn[];
    S &sm = *reinterpret_cast<S *>(dyn);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x % a.L.kvh, b = blockIdx.x / a.L.kvh;
    const int G = a.heads / a.L.kvh;
    griddep_wait();
    const int len = a.len[b], off = a.offsets[b];
    int n = a.offsets[b + 1] - off;
    if (len < 0 || n < 0 || off < 0 || len > a.max_pos || n > a.max_pos - len || n > a.tokens - off) {
        if (tid == 0) raise_error(a.err, kDevRange);
        return;
    }
    const int nq = (int)(((int64_t)n * G + kRows - 1) / kRows);
    if ((int)blockIdx.y >= nq) return;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.k_full[i], kUnpackWarps);
            mbar_init(&sm.v_full[i], kUnpackWarps);
            mbar_init(&sm.o_full[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], kSoftWarps);
        }
        for (int i = 0; i < 4; i++) mbar_init(&sm.info[i], 2 * kUnpackWarps);
        mbar_init(&sm.q_full, kSoftWarps);
        mbar_init(&sm.o_free, kSoftWarps);
        mbar_init(&sm.drained, 1);
        sm.abort = 0;
        mbar_fence_init();
    }
    if (warp == 0) {
        tc::tmem_alloc(&sm.tmem, kTmemCols);
        tc::tmem_relinquish();
    }
    // (not earlier: a kernel that starts now must not take tensor memory that a
    // block of this grid still waits for)
    griddep_launch_dependents();
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sm.tmem;
    // f for each of the block's row tiles, by every warp; `done`: tiles of the block's
    // earlier row tiles (the barriers count on), `turn`: and row tiles
    struct Tile {
        int row0, rows, first_limit, kend, ntiles, done, turn;
    };
    auto each_tile = [&](auto f) {
        int done = 0, turn = 0;
        for (int qi = blockIdx.y; qi < nq; qi += gridDim.y, turn++) {
            Tile x;
            x.row0 = (nq - 1 - qi) * kRows;  // the longest row tiles first
            x.rows = min(kRows, n * G - x.row0);
            x.first_limit = len + x.row0 / G;                  // every row sees these positions
            x.kend = len + (x.row0 + x.rows - 1) / G + 1;      // positions that some row sees
            x.ntiles = (x.kend + kKeys - 1) / kKeys;
            x.done = done, x.turn = turn;
            f(x);
            done += x.ntiles;
            tc::fence_before_sync();
            asm volatile("bar.sync 0;" ::: "memory");  // operands and tensor memory are free for the next row tile
            tc::fence_after_sync();
            if (sm.abort) break;
        }
    };
    const float *q = a.q + ((int64_t)off * a.heads + h * G) * D;  // row r: token r / G, head r % G
    if (warp < kSoftWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        each_tile([&](const Tile &T) {
            const int row0 = T.row0, rows = T.rows, first_limit = T.first_limit, ntiles = T.ntiles, done = T.done;
            // ================================================= softmax
            const int hs = warp >> 2, r = 32 * (warp & 3) + lane;
            const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
            const int limit = r < rows ? len + (row0 + r) / G : -1;
            constexpr int kPieces = D / 8;
            const int place = r < rows ? (row0 + r) / G * a.heads + (row0 + r) % G : -1;  // of the row, in heads
            // ---- the row's queries: a power of two, then high and low halves; a thread has
            // half of the dimensions, in the order in which a key's words give them
            float rs;
            {
                constexpr int H = D / 2;
                float x[H], most = 0.0f;
                // (a thread that reads its own row takes one line of 128 bytes for every 16 bytes)
#pragma unroll
                for (int i = 0; i < kPieces; i++) {
                    const int rr = (32 * i + lane) / kPieces, c = (32 * i + lane) % kPieces;
                    const int at = __shfl_sync(0xffffffffu, place, rr);
                    const float4 u = at >= 0 ? __ldg(reinterpret_cast<const float4 *>(q + (int64_t)at * D + H * hs) + c)
                                             : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[4 * i] = u.x, x[4 * i + 1] = u.y, x[4 * i + 2] = u.z, x[4 * i + 3] = u.w;
                }
#pragma unroll
                for (int i = 0; i < kPieces; i++) {
                    const int rr = (32 * i + lane) / kPieces, c = (32 * i + lane) % kPieces;
                    sm.stage[warp][rr][c ^ (rr % kPieces)] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kPieces; i++) {
                    const float4 u = sm.stage[warp][lane][i ^ (lane % kPieces)];
                    x[4 * i] = u.x, x[4 * i + 1] = u.y, x[4 * i + 2] = u.z, x[4 * i + 3] = u.w;
                    most = fmaxf(max3(most, fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w)));
                }
                sm.top[0][hs][r] = most;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                most = fmaxf(most, sm.top[0][hs ^ 1][r]);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                // 2^e puts the row's largest value into [2^9, 2^10)
                const int e0 = 136 - (int)(__float_as_uint(most) >> 23);
                const int e = (most > 0.0f && isfinite(most)) ? max(-120, min(120, e0)) : 0;
                rs = pow2(-e) * a.scale_log2;
                const float up = pow2(e);
#pragma unroll
                for (int p = 0; p < H / 32; p++) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {  // columns of four to an 8-dimension block: pairs (j, j + 4)
                        const int at = 32 * p + 8 * (i >> 2) + (i & 3);
                        const float y0 = x[at] * up, y1 = x[at + 4] * up;
                        const __half2 w = __floats2half2_rn(y0, y1);
                        hi[i] = h2u(w);
                        lo[i] = h2u(__floats2half2_rn(y0 - __low2float(w), y1 - __high2float(w)));
                    }
                    tc::st_32x32b_x16(t_lane + kColQ + (D / 4) * hs + 16 * p, hi);
                    tc::st_32x32b_x16(t_lane + kColQ + D / 2 + (D / 4) * hs + 16 * p, lo);
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.q_full);
            }
            float m = -INFINITY, corr = 0.0f, unv = 0.0f;
            // The sum, and what its additions have rounded away: a tile's 32 values are added
            // on their own, then once to the sum.  (One by one, values that hardly differ all
            // round in one direction: 1.3e-4 of the sum at 33000 positions.)
            float l = 0.0f, l_rest = 0.0f;
            float o[D / 2];
#pragma unroll
            for (int i = 0; i < D / 2; i++) o[i] = 0.0f;
            // adds O of tile `it` (which the products have finished)
            auto fold = [&](int it) {
                const int gi = done + it;
                const bool grown = __any_sync(0xffffffffu, corr != 1.0f);
                wait_for(&sm.o_full[gi & 1], (gi >> 1) & 1, &sm.abort, a.err);
                tc::fence_after_sync();
#pragma unroll
                for (int p = 0; p < D / 64; p++) {
                    float u[32];
                    tc::ld_32x32b_x32(t_lane + kColO + (D / 2) * hs + 32 * p, u);
                    if (grown)
#pragma unroll
                        for (int i = 0; i < 32; i++) o[32 * p + i] *= corr;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 s = fma2(make_float2(u[i], u[i + 1]), make_float2(unv, unv),
                                              make_float2(o[32 * p + i], o[32 * p + i + 1]));
                        o[32 * p + i] = s.x, o[32 * p + i + 1] = s.y;
                    }
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.o_free);
            };
            for (int it = 0; it < ntiles; it++) {
                const int gi = done + it, buf = gi & 1, slot = gi & 3;
                // (after a wait that ran out the loop goes on over what is there: its
                // waits return at once, and no warp leaves another at a barrier)
                wait_for(&sm.info[slot], (gi >> 2) & 1, &sm.abort, a.err);
                wait_for(&sm.s_full[buf], (gi >> 1) & 1, &sm.abort, a.err);
                tc::fence_after_sync();
                const float f = rs * sm.unk[slot];
                const float unv_now = sm.unv[slot];
                unsigned bad[C / 2][2], any = 0;  // of this thread's groups of dimensions
#pragma unroll
                for (int c = 0; c < C / 2; c++)
#pragma unroll
                    for (int u = 0; u < 2; u++) any |= bad[c][u] = sm.vnan[slot][u][hs * (C / 2) + c];
                float x[32];
                tc::ld_32x32b_x32(t_lane + kColS + 64 * buf + 32 * hs, x);
                const int left = limit - it * kKeys;  // the row sees columns up to here
                if (it * kKeys + kKeys - 1 > first_limit) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (32 * hs + i > left) x[i] = -INFINITY;
                }
                float top = max3(x[0], x[1], x[2]), top1 = max3(x[3], x[4], x[5]);
#pragma unroll
                for (int i = 6; i < 30; i += 4) top = max3(top, x[i], x[i + 1]), top1 = max3(top1, x[i + 2], x[i + 3]);
                top = max3(top, x[30], fmaxf(top1, x[31]));
                sm.top[buf][hs][r] = top;
                asm volatile("bar.sync %0, 64;" ::"r"(3 + (warp & 3)) : "memory");  // the row's two warps
                // The reference of the exponentials follows the running maximum only where
                // that has passed it by 2^7: O is hardly ever rescaled.  P is up to 2^8 too
                // large, 2^15 with that, and so is its sum.
                const float to = fmaxf(m, fmaxf(top, sm.top[buf][hs ^ 1][r]) * f);
                float corr_now = 1.0f;
                if (to > m + 7.0f) {
                    corr_now = ex2(m - to);
                    m = to;
                    l *= corr_now, l_rest *= corr_now;
                }
                const float ref = m == -INFINITY ? 0.0f : m - 8.0f;
                float2 s[4];  // (four sums: one chain of 16 additions costs 2 us of the whole 2 x 2048)
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 z = fma2(make_float2(x[i], x[i + 1]), make_float2(f, f), make_float2(-ref, -ref));
                    x[i] = ex2(z.x), x[i + 1] = ex2(z.y);
                    if (i < 8) s[i / 2] = make_float2(x[i], x[i + 1]);
                    else s[i / 2 % 4] = add2(s[i / 2 % 4], make_float2(x[i], x[i + 1]));
                }
                s[0] = add2(add2(s[0], s[1]), add2(s[2], s[3]));
                const float part = s[0].x + s[0].y, sum = __fadd_rn(l, part), back = __fsub_rn(sum, l);
                l_rest += __fsub_rn(l, __fsub_rn(sum, back)) + __fsub_rn(part, back);
                l = sum;
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int p = 0; p < 16; p++) {  // slot pair p: positions 8h + 2t, + 1 with t = p / 4, h = p % 4
                    const int at = 8 * (p & 3) + 2 * (p >> 2);
                    const __half2 w = __floats2half2_rn(x[at], x[at + 1]);
                    hi[p] = h2u(w);
                    const float2 rest = fma2(__half22float2(w), make_float2(-1.0f, -1.0f), make_float2(x[at], x[at + 1]));
                    lo[p] = h2u(__floats2half2_rn(rest.x, rest.y));
                }
                tc::st_32x32b_x16(t_lane + kColP + 64 * buf + 16 * hs, hi);
                tc::st_32x32b_x16(t_lane + kColP + 64 * buf + 32 + 16 * hs, lo);
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_full[buf]);
                if (it > 0) fold(it - 1);
                corr = corr_now;
                unv = unv_now;
                if (any) {  // values that are NaN reach the rows that see their position
#pragma unroll
                    for (int c = 0; c < C / 2; c++) {
                        bool hit = false;
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const int see = left - 32 * u;  // positions 0 .. see of the unit
                            hit = hit || (bad[c][u] & (see < 0 ? 0u : see >= 31 ? ~0u : (2u << see) - 1u));
                        }
                        if (hit)
#pragma unroll
                            for (int i = 0; i < 32; i++) o[32 * c + i] = NAN;
                    }
                }
            }
            fold(ntiles - 1);
            sm.l[hs][r] = l + l_rest;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float inv = __fdiv_rn(1.0f, sm.l[0][r] + sm.l[1][r]);
#pragma unroll
            for (int i = 0; i < kPieces; i++)
                sm.stage[warp][lane][i ^ (lane % kPieces)] =
                    make_float4(o[4 * i] * inv, o[4 * i + 1] * inv, o[4 * i + 2] * inv, o[4 * i + 3] * inv);
            __syncwarp();
            float *dst = a.out + ((int64_t)off * a.heads + h * G) * D + (D / 2) * hs;
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const int rr = (32 * i + lane) / kPieces, c = (32 * i + lane) % kPieces;
                const int at = __shfl_sync(0xffffffffu, place, rr);
                if (at >= 0) reinterpret_cast<float4 *>(dst + (int64_t)at * D)[c] = sm.stage[warp][rr][c ^ (rr % kPieces)];
            }
            __syncwarp();
        });
    } else if (warp < kSoftWarps + kUnpackWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegs));
        each_tile([&](const Tile &T) { unpack<D, false>(sm, a, b, h, T.ntiles, T.kend, T.done); });
    } else if (warp < kSoftWarps + 2 * kUnpackWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegs));
        each_tile([&](const Tile &T) { unpack<D, true>(sm, a, b, h, T.ntiles, T.kend, T.done); });
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLastRegs));
        each_tile([&](const Tile &T) {
            const int ntiles = T.ntiles, done = T.done, turn = T.turn;
            // ================================================= products
            if (warp == kSoftWarps + 2 * kUnpackWarps && elect_one()) {
                constexpr uint32_t id_s = tc::idesc_f16_f32(kRows, kKeys), id_o = tc::idesc_f16_f32(kRows, D);
                const uint32_t qt = tmem + kColQ;
                auto arrived = [&](uint64_t *bar, int phase) { return wait_one(bar, phase & 1, &sm.abort, a.err); };
                // (the buffer is a constant in each product: addresses and descriptors are too)
                auto scores_in = [&](auto buf_, int gi) {
                    constexpr int buf = decltype(buf_)::value;
                    if (!arrived(&sm.k_full[buf], gi >> 1)) return false;
                    tc::fence_after_sync();
                    const uint32_t kh = smem_u32(sm.k[buf][0]), kl = smem_u32(sm.k[buf][1]);
                    const uint32_t d = tmem + kColS + 64 * buf;
#pragma unroll
                    for (int j = 0; j < D / 16; j++) {
                        const uint64_t bh = tc::smem_desc(kh + 2 * S::kKStep * j, S::kKStep, (D / 8) * S::kKStep);
                        const uint64_t bl = tc::smem_desc(kl + 2 * S::kKStep * j, S::kKStep, (D / 8) * S::kKStep);
                        tc::mma_f16_ts(d, qt + 8 * j, bh, id_s, j != 0 ? 1u : 0u);
                        tc::mma_f16_ts(d, qt + 8 * j, bl, id_s, 1u);
                        tc::mma_f16_ts(d, qt + D / 2 + 8 * j, bh, id_s, 1u);
                    }
                    tc::commit(&sm.s_full[buf]);
                    return true;
                };
                auto values_in = [&](auto buf_, int gi) {
                    constexpr int buf = decltype(buf_)::value;
                    if (!arrived(&sm.v_full[buf], gi >> 1) || (gi > 0 && !arrived(&sm.o_free, gi - 1)) ||
                        !arrived(&sm.p_full[buf], gi >> 1))
                        return false;
                    tc::fence_after_sync();
                    const uint32_t vh = smem_u32(sm.v[buf][0]), vl = smem_u32(sm.v[buf][1]);
                    const uint32_t d = tmem + kColO, p = tmem + kColP + 64 * buf;
#pragma unroll
                    for (int j = 0; j < kKeys / 16; j++) {
                        const uint64_t bh = tc::smem_desc(vh + 2 * S::kVStep * j, S::kVStep, (kKeys / 8) * S::kVStep);
                        const uint64_t bl = tc::smem_desc(vl + 2 * S::kVStep * j, S::kVStep, (kKeys / 8) * S::kVStep);
                        tc::mma_f16_ts(d, p + 8 * j, bh, id_o, j != 0 ? 1u : 0u);
                        tc::mma_f16_ts(d, p + 8 * j, bl, id_o, 1u);
                        tc::mma_f16_ts(d, p + 32 + 8 * j, bh, id_o, 1u);
                    }
                    tc::commit(&sm.o_full[buf]);
                    return true;
                };
                using B0 = std::integral_constant<int, 0>;
                using B1 = std::integral_constant<int, 1>;
                auto scores = [&](int it) {  // S of a tile
                    const int gi = done + it;
                    return (gi & 1) ? scores_in(B1{}, gi) : scores_in(B0{}, gi);
                };
                auto values = [&](int it) {  // O of a tile
                    const int gi = done + it;
                    return (gi & 1) ? values_in(B1{}, gi) : values_in(B0{}, gi);
                };
                // S is two tiles ahead of O at most (two buffers): the softmax of a tile runs
                // beside the products of the tiles around it
                bool go = arrived(&sm.q_full, turn) && scores(0) && (ntiles < 2 || scores(1));
                for (int it = 0; go && it < ntiles; it++) go = values(it) && (it + 2 >= ntiles || scores(it + 2));
                if (!go) {  // products are left behind by no block: their operands and tensor memory go with it
                    tc::commit(&sm.drained);
                    mbar_wait_bounded(&sm.drained, 0, a.err);
                }
            }
            __syncwarp();
        });
    }
    __syncthreads();
    if (warp == 0) tc::tmem_dealloc(tmem, kTmemCols);
}

template <int D>
int launch(const PromptArgs &a, int device, int64_t max_rows, cudaStream_t st) {
    auto kern = k_kv4_prompt<D>;
    static std::atomic<uint64_t> done;
    QORA_TRY(allow_smem(kern, sizeof(Sm<D>), device, done));
    const int64_t tiles = (max_rows + kRows - 1) / kRows;
    const unsigned y = (unsigned)(tiles < 65535 ? tiles : 65535);  // a block takes further tiles in turn
    // blocks start in the order of x first: the longest row tile of every stream and
    // head before the second longest of any
    return launch_ex(kern, dim3(a.L.kvh * a.streams, y), dim3(kThreads), sizeof(Sm<D>), st, 1u, a);
}

}  // namespace

int kv4_launch_prompt(qora_kv4 *kv, int layer, const float *q, const int *offsets, int tokens, int64_t max_rows,
                      float *out, cudaStream_t st) {
    PromptArgs a;
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
    const int device = kv->ctx->device;
    return kv->hd == 64 ? launch<64>(a, device, max_rows, st) : launch<128>(a, device, max_rows, st);
}

}  // namespace qora
