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
// Three kinds of warps work on different tiles at the same time: four unpack keys
// and values into shared memory as matrix operands (two buffers), one issues the
// products, eight do the softmax: a thread has one row, half of its positions for
// P and half of its dimensions for O.  P goes back to tensor memory as an operand.
// The unit's layout gives a lane whole 16-byte operand rows: eight dimensions of a
// key, and eight positions of a value's dimension (in the order 2t + e + 8h, which
// P's columns follow).  O of each tile is added in f32 registers, because the
// tensor core's own additions do not round to nearest.
#include "kv4.cuh"
#include "tc.cuh"

namespace qora {

namespace {

constexpr int kRows = 128;                 // query rows of a block
constexpr int kKeys = 64;                  // positions of a tile: two units
constexpr int kSoftWarps = 8, kUnpackWarps = 4;
constexpr int kThreads = (kSoftWarps + kUnpackWarps + 1) * 32;
constexpr uint32_t kTmemCols = 512;        // S 2 x 64, P (high, low) 2 x 64, O 2 x 128
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256;

struct PromptArgs {
    Kv4Layer L;
    const float *q;
    const int *offsets, *len;
    float *out;
    int *err;
    int streams, heads, max_pos, tokens;
    float scale_log2;  // log2(e) / sqrt(D)
};

// Operands in shared memory: core matrices of 8 rows x 16 bytes.  The distance
// between neighbours along the contraction is 128 bytes for Q, 160 for K and 144
// for V, so that the unpacking warps' 16-byte stores fall on distinct banks.
template <int D>
struct Sm {
    static constexpr int kQ = kRows * D * 2;
    static constexpr int kKStep = 160, kVStep = 144;
    static constexpr int kK = (kKeys / 8) * (D / 8) * kKStep;
    static constexpr int kV = (D / 8) * (kKeys / 8) * kVStep;
    alignas(1024) uint8_t q[2][kQ];        // high, low
    alignas(128) uint8_t k[2][2][kK];      // [buffer][high, low]
    alignas(128) uint8_t v[2][2][kV];
    int rexp[kRows];                       // queries are scaled by 2^rexp
    float l[2][kRows], top[2][2][kRows];   // a row's sum, and largest score, by half
    float unk[2], unv[2];                  // a tile's scales back
    unsigned vnan[2][2][D / 32];           // positions of a unit whose value scale is NaN, by group
    unsigned most[2][kUnpackWarps];
    int stop[2];
    alignas(8) uint64_t full[2], empty[2], s_full[2], p_full[2], o_full[2];
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

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, int *abort, int *err) {
    return __all_sync(0xffffffffu, wait_one(bar, parity, abort, err));
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

// What a lane of an unpacking warp has of one (unit, scale group).
struct Raw {
    uint4 k, v;
    uint2 ks, vs0, vs1;  // scales: keys g + 8i; values 2t + 8i and 2t + 1 + 8i
};

__device__ __forceinline__ float half_of(uint2 v, int i) {
    const __half2 h = u2h(i < 2 ? v.x : v.y);
    return (i & 1) ? __high2float(h) : __low2float(h);
}

// The power of two that brings scales up to `bits` (f16, finite) under 2^12.
__device__ __forceinline__ int scale_exponent(unsigned bits) { return 26 - (int)((bits >> 10) & 31u); }

template <int D>
__global__ void __launch_bounds__(kThreads, 1) k_kv4_prompt(const PromptArgs a) {
    using S = Sm<D>;
    using U = Kv4Unit<D>;
    constexpr int C = D / 32;
    extern __shared__ __align__(1024) uint8_t dyn[];
    S &sm = *reinterpret_cast<S *>(dyn);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z;
    const int G = a.heads / a.L.kvh;
    griddep_wait();
    const int len = a.len[b], off = a.offsets[b];
    int n = a.offsets[b + 1] - off;
    if (len < 0 || n < 0 || off < 0 || len > a.max_pos || n > a.max_pos - len || n > a.tokens - off) {
        if (tid == 0) raise_error(a.err, kDevRange);
        return;
    }
    const int nq = (int)(((int64_t)n * G + kRows - 1) / kRows);
    if ((int)blockIdx.x >= nq) return;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.full[i], kUnpackWarps);
            mbar_init(&sm.empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], kSoftWarps);
            mbar_init(&sm.o_full[i], 1);
        }
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
    int done = 0;  // tiles of this block's earlier row tiles: the barriers count on
    for (int qi = blockIdx.x; qi < nq; qi += gridDim.x) {
        const int row0 = (nq - 1 - qi) * kRows;  // the longest row tiles first
        const int rows = min(kRows, n * G - row0);
        const int first_limit = len + row0 / G;                // every row sees these positions
        const int kend = len + (row0 + rows - 1) / G + 1;      // positions that some row sees
        const int ntiles = (kend + kKeys - 1) / kKeys;
        const float *q = a.q + ((int64_t)off * a.heads + h * G) * D;  // row r: token r / G, head r % G
        // ---- queries: a power of two per row, then high and low halves
        for (int r = warp; r < kRows; r += kThreads / 32) {
            float m = 0.0f;
            if (r < rows) {
                const float *x = q + ((int64_t)((row0 + r) / G) * a.heads + (row0 + r) % G) * D;
                for (int d = lane; d < D; d += 32) m = fmaxf(m, fabsf(__ldg(x + d)));
            }
            m = warp_max(m);
            // 2^e puts the row's largest value into [2^9, 2^10)
            const int e = 136 - (int)(__float_as_uint(m) >> 23);
            if (lane == 0) sm.rexp[r] = (m > 0.0f && isfinite(m)) ? max(-120, min(120, e)) : 0;
        }
        __syncthreads();
        for (int i = tid; i < kRows * (D / 8); i += kThreads) {
            const int r = (i & 7) | ((i / (8 * (D / 8))) << 3), kb = (i >> 3) % (D / 8);
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (r < rows) {
                const float4 *src = reinterpret_cast<const float4 *>(
                    q + ((int64_t)((row0 + r) / G) * a.heads + (row0 + r) % G) * D + 8 * kb);
                const float4 u = __ldg(src), w = __ldg(src + 1);
                x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
            }
            const float up = pow2(sm.rexp[r]);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {  // a key's word gives its dimensions as pairs (j, j + 4)
                const float y0 = x[j] * up, y1 = x[j + 4] * up;
                const __half2 p = __floats2half2_rn(y0, y1);
                hi[j] = h2u(p);
                lo[j] = h2u(__floats2half2_rn(y0 - __low2float(p), y1 - __high2float(p)));
            }
            const int at = ((r >> 3) * (D / 8) + kb) * 128 + (r & 7) * 16;
            *reinterpret_cast<uint4 *>(sm.q[0] + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4 *>(sm.q[1] + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        tc::fence_proxy_async_smem();
        __syncthreads();

        if (warp < kSoftWarps) {
            // ================================================= softmax
            const int hs = warp >> 2, r = 32 * (warp & 3) + lane;
            const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
            const int limit = r < rows ? len + (row0 + r) / G : -1;
            const float rs = pow2(-sm.rexp[r]) * a.scale_log2;
            float m = -INFINITY, l = 0.0f, corr = 0.0f, unv = 0.0f;
            float o[D / 2];
#pragma unroll
            for (int i = 0; i < D / 2; i++) o[i] = 0.0f;
            // adds O of tile `it` (which the products have finished)
            auto fold = [&](int it) {
                const int gi = done + it;
                wait_for(&sm.o_full[gi & 1], (gi >> 1) & 1, &sm.abort, a.err);
                tc::fence_after_sync();
#pragma unroll
                for (int p = 0; p < D / 64; p++) {
                    float u[32];
                    tc::ld_32x32b_x32(t_lane + kColO + 128 * (gi & 1) + (D / 2) * hs + 32 * p, u);
#pragma unroll
                    for (int i = 0; i < 32; i++) o[32 * p + i] = fmaf(u[i], unv, o[32 * p + i] * corr);
                }
            };
            for (int it = 0; it < ntiles; it++) {
                const int gi = done + it, buf = gi & 1;
                // (after a wait that ran out the loop goes on over what is there: its
                // waits return at once, and no warp leaves another at a barrier)
                wait_for(&sm.full[buf], (gi >> 1) & 1, &sm.abort, a.err);  // what unpacking says of the tile
                wait_for(&sm.s_full[buf], (gi >> 1) & 1, &sm.abort, a.err);
                tc::fence_after_sync();
                const float f = rs * sm.unk[buf];
                const float unv_now = sm.unv[buf];
                unsigned bad[C / 2][2], any = 0;  // of this thread's groups of dimensions
#pragma unroll
                for (int c = 0; c < C / 2; c++)
#pragma unroll
                    for (int u = 0; u < 2; u++) any |= bad[c][u] = sm.vnan[buf][u][hs * (C / 2) + c];
                float x[32];
                tc::ld_32x32b_x32(t_lane + kColS + 64 * buf + 32 * hs, x);
                const int left = limit - it * kKeys;  // the row sees columns up to here
                if (it * kKeys + kKeys - 1 > first_limit) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (32 * hs + i > left) x[i] = -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 32; i++) top = fmaxf(top, x[i]);
                sm.top[buf][hs][r] = top;
                asm volatile("bar.sync %0, 64;" ::"r"(3 + (warp & 3)) : "memory");  // the row's two warps
                const float to = fmaxf(m, fmaxf(top, sm.top[buf][hs ^ 1][r]) * f);
                // P is 2^8 too large, and so is its sum
                const float ref = to == -INFINITY ? 0.0f : to - 8.0f;
                const float corr_now = ex2(m - (to == -INFINITY ? 0.0f : to));
                m = to;
                l *= corr_now;
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    x[i] = ex2(fmaf(x[i], f, -ref));
                    l += x[i];
                }
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int p = 0; p < 16; p++) {  // slot pair p: positions 8h + 2t, + 1 with t = p / 4, h = p % 4
                    const int at = 8 * (p & 3) + 2 * (p >> 2);
                    const __half2 w = __floats2half2_rn(x[at], x[at + 1]);
                    hi[p] = h2u(w);
                    lo[p] = h2u(__floats2half2_rn(x[at] - __low2float(w), x[at + 1] - __high2float(w)));
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
            sm.l[hs][r] = l;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (r < rows) {
                const float sum = sm.l[0][r] + sm.l[1][r];
                float *dst = a.out + ((int64_t)(off + (row0 + r) / G) * a.heads + h * G + (row0 + r) % G) * D + (D / 2) * hs;
#pragma unroll
                for (int i = 0; i < D / 2; i += 4)
                    *reinterpret_cast<float4 *>(dst + i) =
                        make_float4(__fdiv_rn(o[i], sum), __fdiv_rn(o[i + 1], sum), __fdiv_rn(o[i + 2], sum),
                                    __fdiv_rn(o[i + 3], sum));
            }
        } else if (warp < kSoftWarps + kUnpackWarps) {
            // ================================================= unpacking
            constexpr int kJobs = 2 * C / kUnpackWarps;  // (unit, group) pairs of a warp and tile
            const int pw = warp - kSoftWarps;
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
            auto load = [&](int it, int job, int pg, Raw &r) {
                r = Raw{};
                if (pg < 0) return;
                const int combo = pw + kUnpackWarps * job, c = combo % C;
                const int pos = it * kKeys + (combo / C) * kKv4Unit;
                const uint8_t *u = a.L.unit(pg, h, (pos >> 5) & ((1 << (a.L.page_shift - 5)) - 1), D);
                r.k = __ldg(reinterpret_cast<const uint4 *>(u + U::kK + c * 512 + lane * 16));
                r.v = __ldg(reinterpret_cast<const uint4 *>(u + U::kV + c * 512 + lane * 16));
                r.ks = __ldg(reinterpret_cast<const uint2 *>(u + U::kKs + c * 64 + g * 8));
                r.vs0 = __ldg(reinterpret_cast<const uint2 *>(u + U::kVs + c * 64 + 2 * t * 8));
                r.vs1 = __ldg(reinterpret_cast<const uint2 *>(u + U::kVs + c * 64 + (2 * t + 1) * 8));
            };
            Raw raw[kJobs];
            int page[kJobs];
#pragma unroll
            for (int j = 0; j < kJobs; j++) {
                load(0, j, page_of(0, j), raw[j]);
                page[j] = page_of(1, j);
            }
            for (int it = 0; it < ntiles; it++) {
                const int gi = done + it, buf = gi & 1;
                // scales behind the last position count as zero, NaN ones are told to the rows
                unsigned kmost = 0, vmost = 0;
                unsigned nan[kJobs];
#pragma unroll
                for (int j = 0; j < kJobs; j++) {
                    const int pos = it * kKeys + ((pw + kUnpackWarps * j) / C) * kKv4Unit;
                    unsigned short ks[4], v0[4], v1[4];
                    const uint2 *src[3] = {&raw[j].ks, &raw[j].vs0, &raw[j].vs1};
                    unsigned short *dst[3] = {ks, v0, v1};
#pragma unroll
                    for (int x = 0; x < 3; x++) {
                        dst[x][0] = src[x]->x & 0xffff, dst[x][1] = src[x]->x >> 16;
                        dst[x][2] = src[x]->y & 0xffff, dst[x][3] = src[x]->y >> 16;
                    }
                    nan[j] = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (pos + 2 * t + 8 * i >= kend) v0[i] = 0;
                        if (pos + 2 * t + 1 + 8 * i >= kend) v1[i] = 0;
                        if ((v0[i] & 0x7c00) == 0x7c00) nan[j] |= 1u << (2 * t + 8 * i), v0[i] = 0;
                        if ((v1[i] & 0x7c00) == 0x7c00) nan[j] |= 2u << (2 * t + 8 * i), v1[i] = 0;
                        if ((ks[i] & 0x7c00) != 0x7c00) kmost = max(kmost, (unsigned)ks[i]);
                        vmost = max(vmost, max((unsigned)v0[i], (unsigned)v1[i]));
                    }
                    raw[j].vs0 = make_uint2(v0[0] | (unsigned)v0[1] << 16, v0[2] | (unsigned)v0[3] << 16);
                    raw[j].vs1 = make_uint2(v1[0] | (unsigned)v1[1] << 16, v1[2] | (unsigned)v1[3] << 16);
                    nan[j] = __reduce_or_sync(0xffffffffu, nan[j]);
                }
                kmost = __reduce_max_sync(0xffffffffu, kmost);
                vmost = __reduce_max_sync(0xffffffffu, vmost);
                if (lane == 0) sm.most[buf][pw] = kmost << 16 | vmost;
                const bool ok = gi < 2 || wait_for(&sm.empty[buf], ((gi >> 1) - 1) & 1, &sm.abort, a.err);
                if (pw == 0 && lane == 0) sm.stop[buf] = !ok;  // one warp decides for all that meet below
                asm volatile("bar.sync 2, 128;" ::: "memory");
                if (sm.stop[buf]) break;
                kmost = vmost = 0;
#pragma unroll
                for (int i = 0; i < kUnpackWarps; i++) {
                    const unsigned w = sm.most[buf][i];
                    kmost = max(kmost, w >> 16), vmost = max(vmost, w & 0xffffu);
                }
                const int ek = scale_exponent(kmost), ev = scale_exponent(vmost);
                const float upk = pow2(ek), upv = pow2(ev);
#pragma unroll
                for (int j = 0; j < kJobs; j++) {
                    const int combo = pw + kUnpackWarps * j, c = combo % C, u = combo / C;
                    const uint32_t kw[4] = {raw[j].k.x, raw[j].k.y, raw[j].k.z, raw[j].k.w};
                    const uint32_t vw[4] = {raw[j].v.x, raw[j].v.y, raw[j].v.z, raw[j].v.w};
                    // keys g + 8i: dimensions 32c + 8t .. + 7 are one operand row of 16 bytes
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        __half2 x[4];
                        codes(kw[i], magic, x);
                        const __half2 s = __float2half2_rn(half_of(raw[j].ks, i) * upk);
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
                    // dimensions 32c + 4g + p: positions 2t + e + 8h are one operand row
                    uint32_t hi[4][4], lo[4][4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        __half2 x[4];
                        codes(vw[i], magic, x);
                        // a word is two positions: the pair of nibble p has both
                        const __half2 s = __floats2half2_rn(half_of(raw[j].vs0, i) * upv, half_of(raw[j].vs1, i) * upv);
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
                    if (lane == 0) sm.vnan[buf][u][c] = nan[j];
                    load(it + 1, j, page[j], raw[j]);  // in flight while the next tile's buffer empties
                    page[j] = page_of(it + 2, j);
                }
                if (pw == 0 && lane == 0) {
                    sm.unk[buf] = pow2(-ek);
                    sm.unv[buf] = pow2(-ev);
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.full[buf]);
            }
        } else {
            // ================================================= products
            if (lane == 0) {
                constexpr uint32_t id_s = tc::idesc_f16_f32(kRows, kKeys), id_o = tc::idesc_f16_f32(kRows, D);
                const uint32_t qh = smem_u32(sm.q[0]), ql = smem_u32(sm.q[1]);
                auto out_of = [&](int gi) {  // O of a tile whose P is there
                    const int buf = gi & 1;
                    if (!wait_one(&sm.p_full[buf], (gi >> 1) & 1, &sm.abort, a.err)) return false;
                    tc::fence_after_sync();
                    const uint32_t vh = smem_u32(sm.v[buf][0]), vl = smem_u32(sm.v[buf][1]);
                    const uint32_t d = tmem + kColO + 128 * buf, p = tmem + kColP + 64 * buf;
#pragma unroll
                    for (int j = 0; j < kKeys / 16; j++) {
                        const uint64_t bh = tc::smem_desc(vh + 2 * S::kVStep * j, S::kVStep, (kKeys / 8) * S::kVStep);
                        const uint64_t bl = tc::smem_desc(vl + 2 * S::kVStep * j, S::kVStep, (kKeys / 8) * S::kVStep);
                        tc::mma_f16_ts(d, p + 8 * j, bh, id_o, j != 0 ? 1u : 0u);
                        tc::mma_f16_ts(d, p + 8 * j, bl, id_o, 1u);
                        tc::mma_f16_ts(d, p + 32 + 8 * j, bh, id_o, 1u);
                    }
                    tc::commit(&sm.o_full[buf]);
                    tc::commit(&sm.empty[buf]);
                    return true;
                };
                for (int it = 0; it <= ntiles; it++) {
                    const int gi = done + it, buf = gi & 1;
                    if (it < ntiles) {
                        if (!wait_one(&sm.full[buf], (gi >> 1) & 1, &sm.abort, a.err)) break;
                        tc::fence_after_sync();
                        const uint32_t kh = smem_u32(sm.k[buf][0]), kl = smem_u32(sm.k[buf][1]);
                        const uint32_t d = tmem + kColS + 64 * buf;
#pragma unroll
                        for (int j = 0; j < D / 16; j++) {
                            const uint64_t ah = tc::smem_desc(qh + 256 * j, 128, (D / 8) * 128);
                            const uint64_t al = tc::smem_desc(ql + 256 * j, 128, (D / 8) * 128);
                            const uint64_t bh = tc::smem_desc(kh + 2 * S::kKStep * j, S::kKStep, (D / 8) * S::kKStep);
                            const uint64_t bl = tc::smem_desc(kl + 2 * S::kKStep * j, S::kKStep, (D / 8) * S::kKStep);
                            tc::mma_f16(d, ah, bh, id_s, j != 0 ? 1u : 0u);
                            tc::mma_f16(d, ah, bl, id_s, 1u);
                            tc::mma_f16(d, al, bh, id_s, 1u);
                        }
                        tc::commit(&sm.s_full[buf]);
                    }
                    if (it > 0 && !out_of(gi - 1)) break;
                }
            }
            __syncwarp();
        }
        done += ntiles;
        tc::fence_before_sync();
        __syncthreads();  // operands and tensor memory are free for the next row tile
        tc::fence_after_sync();
        if (sm.abort) break;
    }
    __syncthreads();
    if (warp == 0) tc::tmem_dealloc(tmem, kTmemCols);
}

template <int D>
int launch(const PromptArgs &a, int64_t max_rows, cudaStream_t st) {
    auto kern = k_kv4_prompt<D>;
    QORA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Sm<D>)));
    const int64_t tiles = (max_rows + kRows - 1) / kRows;
    const unsigned x = (unsigned)(tiles < 65536 ? tiles : 65536);  // a block takes further tiles in turn
    return launch_ex(kern, dim3(x, a.L.kvh, a.streams), dim3(kThreads), sizeof(Sm<D>), st, 1u, a);
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
    return kv->hd == 64 ? launch<64>(a, max_rows, st) : launch<128>(a, max_rows, st);
}

}  // namespace qora
