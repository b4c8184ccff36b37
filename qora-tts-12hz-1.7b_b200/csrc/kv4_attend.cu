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
// The work of a launch (all streams, kv heads, row tiles, units) is one line
// of units that the blocks split evenly, whatever the lengths; lengths and
// offsets are read on the device.  Where a block's share ends inside an item,
// partial (max, sum, weighted sum) go to a workspace and the item's last block
// joins them in block order, so the result does not depend on timing.
#include "kv4.cuh"

namespace qora {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

struct AttendArgs {
    Kv4Layer L;
    const float *q;
    const int *offsets, *len;
    float *out, *part;
    unsigned *tickets;
    int *err;
    int streams, heads, max_pos, tokens;
    float scale_log2;  // log2(e) / sqrt(D)
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// The four pairs of codes of a word: x[j] = (nibble j, nibble j + 4) - 8 in f16.
__device__ __forceinline__ void codes(uint32_t w, uint32_t (&x)[4]) {
    const __half2 lo = __half2half2(__ushort_as_half(0x6408));    // 1032
    const __half2 s16 = __half2half2(__ushort_as_half(0x2c00));   // 1 / 16
    const __half2 hi = __half2half2(__ushort_as_half(0xd480));    // -72
    const uint32_t v = w >> 8;
    x[0] = h2u(__hsub2(u2h((w & 0x000f000fu) | 0x64006400u), lo));
    x[1] = h2u(__hfma2(u2h((w & 0x00f000f0u) | 0x64006400u), s16, hi));
    x[2] = h2u(__hsub2(u2h((v & 0x000f000fu) | 0x64006400u), lo));
    x[3] = h2u(__hfma2(u2h((v & 0x00f000f0u) | 0x64006400u), s16, hi));
}

// t as f16 hi (low half) + f16 lo (high half): the bits that f16 has, and the rest.
__device__ __forceinline__ uint32_t split_hi_lo(float t) {
    const float hi = __uint_as_float(__float_as_uint(t) & 0xffffe000u);
    return h2u(__floats2half2_rn(hi, t - hi));
}

template <int C>
struct Words {
    uint32_t w[C];
    __device__ __forceinline__ void load(const uint8_t *p) {
        if constexpr (C == 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        }
    }
};
template <int C>
struct Scales {
    __half2 s[C / 2];
    __device__ __forceinline__ void load(const uint8_t *p) {
        if constexpr (C == 4) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            s[0] = u2h(v.x), s[1] = u2h(v.y);
        } else {
            s[0] = u2h(*reinterpret_cast<const uint32_t *>(p));
        }
    }
    __device__ __forceinline__ float at(int c) const {
        return (c & 1) ? __high2float(s[c >> 1]) : __low2float(s[c >> 1]);
    }
    __device__ __forceinline__ __half2 most() const {
        if constexpr (C == 4) return __hmax2(s[0], s[1]);
        return s[0];
    }
};

template <int D, int NT, int ST>
struct Smem {
    static constexpr int R = 4 * NT;
    alignas(128) uint8_t ring[kWarps][ST][kv4_unit_bytes(D)];
    float wo[kWarps][R][D];
    float wm[kWarps][R], wl[kWarps][R];
    uint64_t full[kWarps][ST];
    int64_t scan[kWarps];
    int last;
    int64_t start[1];  // [streams + 1] first unit of each stream in the work line
};

// One stream's share of the work line.
struct Stream {
    int len, n, off, nq, ub;  // cached, new tokens, first row, row tiles, units of a tile
};
template <int R>
__device__ __forceinline__ Stream stream_of(const AttendArgs &a, int G, int b) {
    Stream s;
    s.len = __ldcg(a.len + b);
    s.off = __ldcg(a.offsets + b);
    s.n = __ldcg(a.offsets + b + 1) - s.off;
    if (s.len < 0 || s.n < 0 || s.off < 0 || s.len > a.max_pos || s.n > a.max_pos - s.len ||
        s.n > a.tokens - s.off) {
        raise_error(a.err, kDevRange);
        s.n = 0;
    }
    s.nq = (s.n * G + R - 1) / R;
    s.ub = (s.len + s.n + kKv4Unit - 1) / kKv4Unit;
    return s;
}

template <int D, int NT, int ST>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) k_kv4_attend(const AttendArgs a) {
    using Sm = Smem<D, NT, ST>;
    using U = Kv4Unit<D>;
    constexpr int R = Sm::R, C = D / 32;
    extern __shared__ uint4 dyn[];
    Sm &sm = *reinterpret_cast<Sm *>(dyn);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int G = a.heads / a.L.kvh;
    if (tid == 0) {
        for (int w = 0; w < kWarps; w++)
            for (int s = 0; s < ST; s++) mbar_init(&sm.full[w][s], 1);
        mbar_fence_init();
    }
    griddep_launch_dependents();
    griddep_wait();
    // ---- the work line: streams' unit counts, scanned
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
            int64_t before = base, all = base;
            for (int i = 0; i < kWarps; i++) {
                if (i < warp) before += sm.scan[i];
                all += sm.scan[i];
            }
            if (b < a.streams) sm.start[b] = before + x - w;
            base = all;
        }
        if (tid == 0) sm.start[a.streams] = base;
    }
    __syncthreads();
    const int64_t W = sm.start[a.streams];
    const int64_t blocks = min((int64_t)gridDim.x, (W + kWarps - 1) / kWarps);
    if ((int64_t)blockIdx.x >= blocks) return;
    const int64_t w0 = W * blockIdx.x / blocks, w1 = W * (blockIdx.x + 1) / blocks;
    int b = 0;
    for (int lo = 0, hi = a.streams - 1; lo < hi;) {  // last stream that starts at or before w0
        const int mid = (lo + hi + 1) >> 1;
        if (sm.start[mid] <= w0) lo = b = mid;
        else hi = mid - 1;
    }
    int turn = 0;  // units that this warp's ring has taken
    bool dead = false;
    for (int64_t w = w0; w < w1;) {
        while (sm.start[b + 1] <= w) b++;
        const Stream s = stream_of<R>(a, G, b);
        const int64_t rel = w - sm.start[b];
        const int item = (int)(rel / s.ub);
        const int u0 = (int)(rel - (int64_t)item * s.ub);
        const int h = item / s.nq, qt = item - h * s.nq;
        const int u1 = (int)min((int64_t)s.ub, u0 + (w1 - w));
        const int64_t item0 = w - u0;
        const int rows = min(R, s.n * G - qt * R);
        const int tok0 = qt * R / G, tok1 = (qt * R + rows - 1) / G;
        const int first_limit = s.len + tok0;                       // every row sees these positions
        const int stop = min(u1, (s.len + tok1) / kKv4Unit + 1);  // no row sees units from here on
        const int mine = stop > u0 + warp ? (stop - u0 - warp + kWarps - 1) / kWarps : 0;
        const int *table = a.L.table + (int64_t)b * a.L.pages_per_stream;

        // ---- ring: unit k of this warp is u0 + warp + k kWarps
        int pages = 0;
        auto fetch_pages = [&](int k) {  // of units k .. k + 31 (lane = offset)
            const int u = u0 + warp + (k + lane) * kWarps;
            pages = 0;
            if (k + lane < mine) {
                pages = __ldcg(table + ((u * kKv4Unit) >> a.L.page_shift));
                if ((unsigned)pages >= (unsigned)a.L.pool_pages) {
                    raise_error(a.err, kDevRange);
                    pages = 0;
                }
            }
        };
        auto issue = [&](int k) {
            const int pg = __shfl_sync(0xffffffffu, pages, k & 31);
            if (lane == 0) {
                const int u = u0 + warp + k * kWarps;
                const int st = (turn + k) % ST;
                mbar_arrive_expect_tx(&sm.full[warp][st], U::kBytes);
                bulk_g2s(&sm.ring[warp][st][0], a.L.unit(pg, h, u & ((1 << (a.L.page_shift - 5)) - 1), D), U::kBytes,
                         &sm.full[warp][st]);
            }
        };
        fetch_pages(0);
        if (!dead)
            for (int k = 0; k < ST && k < mine; k++) issue(k);

        // ---- query fragments: column n = 2 row + {hi, lo}
        uint32_t bq[NT][2 * C][2];
        float rs[NT], m[NT], l[NT];
        int limit[NT];
        float acc[NT][C][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int row = qt * R + nt * 4 + (g >> 1);
            const bool have = row < s.n * G;
            const float *q = a.q + ((int64_t)(s.off + row / G) * a.heads + h * G + row % G) * D;
            float x[C][8];
            float amax = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[c][j] = have ? __ldg(q + 32 * c + 8 * t + j) : 0.0f;
                    amax = fmaxf(amax, fabsf(x[c][j]));
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
                    bq[nt][2 * c + (j >> 1)][j & 1] = h2u(__floats2half2_rn(y0, y1));
                }
            rs[nt] = __shfl_sync(0xffffffffu, down, t * 8) * a.scale_log2;
            const int mr = qt * R + nt * 4 + t;  // this lane's row
            limit[nt] = mr < s.n * G ? s.len + mr / G : -1;
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
            const int st = (turn + k) % ST;
            const bool here = mbar_wait_bounded(&sm.full[warp][st], ((turn + k) / ST) & 1, a.err);
            if (__any_sync(0xffffffffu, !here)) {
                dead = true;
                break;
            }
            const uint8_t *unit = &sm.ring[warp][st][0];
            float sc[NT][4];  // scores of positions g, g + 8, g + 16, g + 24
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) sc[nt][i] = 0.0f;
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                Words<C> k0, k1;
                Scales<C> s0, s1;
                k0.load(unit + U::kK + (rt * 16 + g) * (D / 2) + t * (D / 8));
                k1.load(unit + U::kK + (rt * 16 + g + 8) * (D / 2) + t * (D / 8));
                s0.load(unit + U::k_scale(rt * 16 + g, 0));
                s1.load(unit + U::k_scale(rt * 16 + g + 8, 0));
#pragma unroll
                for (int c = 0; c < C; c++) {
                    uint32_t x0[4], x1[4];
                    codes(k0.w[c], x0);
                    codes(k1.w[c], x1);
                    const float f0 = s0.at(c), f1 = s1.at(c);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma16816(d, x0[0], x1[0], x0[1], x1[1], bq[nt][2 * c][0], bq[nt][2 * c][1]);
                        mma16816(d, x0[2], x1[2], x0[3], x1[3], bq[nt][2 * c + 1][0], bq[nt][2 * c + 1][1]);
                        sc[nt][2 * rt] = fmaf(f0, d[0] + d[1], sc[nt][2 * rt]);
                        sc[nt][2 * rt + 1] = fmaf(f1, d[2] + d[3], sc[nt][2 * rt + 1]);
                    }
                }
            }
            // values and their scales into registers: the stage is free after that
            Words<C> v[2][2];
            Scales<C> vs[4];
#pragma unroll
            for (int rt = 0; rt < 2; rt++)
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    v[rt][p].load(unit + U::kV + rt * (8 * D) + p * (4 * D) + lane * (D / 8));
                    vs[rt * 2 + p].load(unit + U::v_scale(rt * 16 + p * 8 + g, 0));
                }
            __syncwarp();
            if (k + ST < mine) {
                if (((k + ST) & 31) == 0) fetch_pages(k + ST);
                issue(k + ST);
            }
            const bool edge = u * kKv4Unit + kKv4Unit - 1 > first_limit;
            // the largest value scale of the unit sets the power of two
            __half2 big = __hmax2(__hmax2(vs[0].most(), vs[1].most()), __hmax2(vs[2].most(), vs[3].most()));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) big = __hmax2(big, u2h(__shfl_xor_sync(0xffffffffu, h2u(big), o)));
            const unsigned bits = h2u(__hmax2(big, __lowhigh2highlow(big))) & 0x7c00u;
            const int kn = min(ke, 24 - (int)(bits >> 10));
            const float shrink = __int_as_float((127 + kn - ke) << 23), lift = __int_as_float((127 + kn) << 23);
            ke = kn;
            float keep[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[nt][i] *= rs[nt];
                    if (edge && u * kKv4Unit + g + 8 * i > limit[nt]) sc[nt][i] = -INFINITY;
                }
                float mx = fmaxf(fmaxf(sc[nt][0], sc[nt][1]), fmaxf(sc[nt][2], sc[nt][3]));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                mx = fmaxf(mx, m[nt]);
                const float ref = mx == -INFINITY ? 0.0f : mx;
                const float corr = ex2(m[nt] - ref);
                m[nt] = mx;
                l[nt] *= corr;
                keep[nt] = corr * shrink;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[nt][i] = ex2(sc[nt][i] - ref);
                    l[nt] += sc[nt][i];
                    sc[nt][i] *= lift;
                }
            }
#pragma unroll
            for (int c = 0; c < C; c++) {
                uint32_t bp[NT][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float f = vs[i].at(c);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float x = sc[nt][i] * f;
                        if (edge && sc[nt][i] == 0.0f) x = 0.0f;  // whatever lies behind the last position
                        bp[nt][i] = transpose8x8(split_hi_lo(x));
                    }
                }
                float d0[NT][4], d1[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) d0[nt][i] = d1[nt][i] = 0.0f;
#pragma unroll
                for (int rt = 0; rt < 2; rt++) {
                    uint32_t x0[4], x1[4];
                    codes(v[rt][0].w[c], x0);
                    codes(v[rt][1].w[c], x1);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        mma16816(d0[nt], x0[0], x0[1], x1[0], x1[1], bp[nt][2 * rt], bp[nt][2 * rt + 1]);
                        mma16816(d1[nt], x0[2], x0[3], x1[2], x1[3], bp[nt][2 * rt], bp[nt][2 * rt + 1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    acc[nt][c][0] = fmaf(acc[nt][c][0], keep[nt], d0[nt][0] + d0[nt][1]);
                    acc[nt][c][1] = fmaf(acc[nt][c][1], keep[nt], d0[nt][2] + d0[nt][3]);
                    acc[nt][c][2] = fmaf(acc[nt][c][2], keep[nt], d1[nt][0] + d1[nt][1]);
                    acc[nt][c][3] = fmaf(acc[nt][c][3], keep[nt], d1[nt][2] + d1[nt][3]);
                }
            }
        }
        turn += mine;

        // ---- join the warps
        const float unlift = __int_as_float((127 - ke) << 23);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], o);
            if (g == 0) {
                sm.wm[warp][nt * 4 + t] = m[nt];
                sm.wl[warp][nt * 4 + t] = l[nt];
            }
#pragma unroll
            for (int c = 0; c < C; c++)
                *reinterpret_cast<float4 *>(&sm.wo[warp][nt * 4 + t][32 * c + 4 * g]) =
                    make_float4(acc[nt][c][0] * unlift, acc[nt][c][1] * unlift, acc[nt][c][2] * unlift,
                                acc[nt][c][3] * unlift);
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 == s.ub;
        float *part = a.part + ((int64_t)blockIdx.x * 2 + (u0 == 0)) * (R * (D + 2));
        for (int i = tid; i < R * D; i += kThreads) {
            const int r = i / D, d = i % D;
            float mx = -INFINITY;
            for (int x = 0; x < kWarps; x++) mx = fmaxf(mx, sm.wm[x][r]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float o = 0.0f, sum = 0.0f;
            for (int x = 0; x < kWarps; x++) {
                const float f = ex2(sm.wm[x][r] - ref);
                o = fmaf(f, sm.wo[x][r][d], o);
                sum = fmaf(f, sm.wl[x][r], sum);
            }
            if (whole) {
                if (r < rows) {
                    const int row = qt * R + r;
                    a.out[((int64_t)(s.off + row / G) * a.heads + h * G + row % G) * D + d] = __fdiv_rn(o, sum);
                }
            } else {
                __stcg(part + i, o);
                if (d == 0) {
                    __stcg(part + R * D + r, mx);
                    __stcg(part + R * D + R + r, sum);
                }
            }
        }
        if (!whole) {
            // the item's blocks: the last of them to arrive joins all, in block order
            const int i0 = (int)(((item0 + 1) * blocks - 1) / W);
            const int i1 = (int)(((item0 + s.ub) * blocks - 1) / W);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const unsigned n = atomicAdd(a.tickets + i0, 1u);
                sm.last = n == (unsigned)(i1 - i0);
                if (sm.last) a.tickets[i0] = 0u;
            }
            __syncthreads();
            if (sm.last) {
                __threadfence();
                for (int i = tid; i < rows * D; i += kThreads) {
                    const int r = i / D, d = i % D;
                    float mx = -INFINITY, o = 0.0f, sum = 0.0f;
                    for (int x = i0; x <= i1; x++) {
                        const float *p = a.part + ((int64_t)x * 2 + (x == i0)) * (R * (D + 2));
                        const float pm = __ldcg(p + R * D + r);
                        const float to = fmaxf(mx, pm), ref = to == -INFINITY ? 0.0f : to;
                        const float fa = ex2(mx - ref), fb = ex2(pm - ref);
                        o = fmaf(fb, __ldcg(p + i), o * fa);
                        sum = fmaf(fb, __ldcg(p + R * D + R + r), sum * fa);
                        mx = to;
                    }
                    const int row = qt * R + r;
                    a.out[((int64_t)(s.off + row / G) * a.heads + h * G + row % G) * D + d] = __fdiv_rn(o, sum);
                }
            }
        }
        __syncthreads();
        w += u1 - u0;
    }
}

template <int D, int NT, int ST>
int launch(const AttendArgs &a, int blocks, cudaStream_t st) {
    using Sm = Smem<D, NT, ST>;
    const size_t smem = sizeof(Sm) + (size_t)a.streams * 8;
    auto kern = k_kv4_attend<D, NT, ST>;
    if (smem > 48 * 1024)
        QORA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return launch_ex(kern, dim3(blocks), dim3(kThreads), smem, st, 1u, a);
}

}  // namespace

int kv4_attend_blocks(const qora_ctx *ctx) { return 2 * ctx->num_sms; }

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
    a.part = kv->part.as<float>();
    a.tickets = kv->tickets.as<unsigned>();
    a.err = kv->ctx->err.as<int>();
    a.streams = kv->streams;
    a.heads = kv->heads;
    a.max_pos = kv->max_pos;
    a.tokens = tokens;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)kv->hd);
    const int rows = kv->heads / kv->kvh * max_count;
    const int sms = kv->ctx->num_sms;
    cudaStream_t st = as_stream(stream);
    if (kv->hd == 64) return rows <= 4 ? launch<64, 1, 2>(a, 2 * sms, st) : launch<64, 2, 4>(a, sms, st);
    return rows <= 4 ? launch<128, 1, 2>(a, 2 * sms, st) : launch<128, 2, 4>(a, sms, st);
}
