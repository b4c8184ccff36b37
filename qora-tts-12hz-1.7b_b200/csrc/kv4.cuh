// 4-bit paged KV cache: the handle and its layout.
//
// A position's key (after norm and rotation) and value are held per kv head in
// groups of 32 dimensions: an f16 scale s = f16(amax / 7) and 4-bit codes
// c = round(x / s) in [-7, 7] (ties to even), stored as c + 8.  A value reads
// back as s * c.  A group with an infinite or NaN value gets a NaN scale; a
// scale past f16's largest value is that value (codes then saturate).
//
// Storage is by units of 32 positions of one (layer, kv head): 36 * head_dim
// contiguous bytes, one bulk copy for the attention kernel:
//     [K codes 16 D | V codes 16 D | K scales 2 D | V scales 2 D]     (D = head_dim)
// Codes are laid out as the fragments of the attention's matrix instructions, by
// scale group c < D/32, so that a lane (g 0..7, t 0..3) of a warp takes its words
// of a group in one 16-byte load and the scales of its positions in one of 8:
//   K: [c][g][t][i 0..3] words; nibble j of a word is dimension 32c + 8t + j of
//      position g + 8i;
//   V: [c][t][g ^ 2t][h 0..3] words of two halfwords e; nibble j of a halfword is
//      dimension 32c + 4g + j of position 8h + 2t + e (a word holds two
//      neighbouring positions, so one mask gives the pair that a matrix fragment
//      register needs).  A position's halfwords of a group lie in 128 bytes, which
//      halves the sectors that an append writes against [g][t], and the exclusive
//      or keeps a quarter-warp's 16-byte reads on distinct banks;
//   scales: [c][g][i] f16 of position g + 8i.
// A page holds page_pos positions of every layer and kv head, in the order
// [layer][kv head][unit].  Logical page j of stream b is physical page
// table[b][j]; a slot is page * page_pos + position in the page.
#pragma once

#include "common.cuh"

struct qora_kv4 {
    qora::CtxRef ctx;
    int layers = 0, heads = 0, kvh = 0, hd = 0, max_pos = 0, streams = 0;
    int page_pos = 0, page_shift = 0, pages_per_stream = 0, pool_pages = 0;
    qora::DevBuf pages, table, len;
    int clusters[2][3] = {};  // attend: clusters that run at once, by kernel and cluster size
    int wide = 0;             // reserve: blocks of its wide cluster
};

namespace qora {

constexpr int kKv4Unit = 32;           // positions per unit
constexpr int kKv4MaxStreams = 4096;   // the attention's work list lies in shared memory

__host__ __device__ constexpr int kv4_unit_bytes(int hd) { return 36 * hd; }

// One layer of the cache as the kernels see it.
struct Kv4Layer {
    uint8_t *base = nullptr;       // this layer's units of page 0
    const int *table = nullptr;    // [streams][pages_per_stream]
    int64_t page_bytes = 0;
    int kvh = 0, page_shift = 0, pages_per_stream = 0, pool_pages = 0;

    __device__ __forceinline__ uint8_t *unit(int page, int h, int unit_in_page, int hd) const {
        const int upp = 1 << (page_shift - 5);
        return base + (int64_t)page * page_bytes + (int64_t)(h * upp + unit_in_page) * kv4_unit_bytes(hd);
    }
};

inline Kv4Layer kv4_layer(const qora_kv4 *kv, int layer) {
    Kv4Layer L;
    const int64_t head_bytes = (int64_t)(kv->page_pos / kKv4Unit) * kv4_unit_bytes(kv->hd);
    L.page_bytes = (int64_t)kv->layers * kv->kvh * head_bytes;
    L.base = kv->pages.as<uint8_t>() + (int64_t)layer * kv->kvh * head_bytes;
    L.table = kv->table.as<int>();
    L.kvh = kv->kvh;
    L.page_shift = kv->page_shift;
    L.pages_per_stream = kv->pages_per_stream;
    L.pool_pages = kv->pool_pages;
    return L;
}

// Asks the device what the attention kernels' launches go by (at creation).
int kv4_attend_setup(qora_kv4 *kv);

// Attention of many new tokens per stream (at most max_rows query rows of a kv head
// in one stream, as the host knows).
int kv4_launch_prompt(qora_kv4 *kv, int layer, const float *q, const int *offsets, int tokens, int64_t max_rows,
                      float *out, cudaStream_t st);

// Byte offsets in a unit of head dimension D.
template <int D>
struct Kv4Unit {
    static constexpr int kBytes = kv4_unit_bytes(D);
    static constexpr int kK = 0, kV = 16 * D, kKs = 32 * D, kVs = 34 * D;
    __host__ __device__ static __forceinline__ int k_word(int r, int dim) {
        return kK + (((dim >> 5) * 8 + (r & 7)) * 4 + ((dim & 31) >> 3)) * 16 + (r >> 3) * 4;
    }
    __host__ __device__ static __forceinline__ int v_half(int r, int dim) {
        return kV + (dim >> 5) * 512 + v_chunk((dim & 31) >> 2, (r & 7) >> 1) + (r >> 3) * 4 + (r & 1) * 2;
    }
    // where lane (g, t)'s 16 bytes of a group's V codes are
    __host__ __device__ static __forceinline__ int v_chunk(int g, int t) { return (t * 8 + (g ^ (2 * t))) * 16; }
    __host__ __device__ static __forceinline__ int k_scale(int r, int c) { return kKs + ((c * 8 + (r & 7)) * 4 + (r >> 3)) * 2; }
    __host__ __device__ static __forceinline__ int v_scale(int r, int c) { return kVs + ((c * 8 + (r & 7)) * 4 + (r >> 3)) * 2; }
};

}  // namespace qora
