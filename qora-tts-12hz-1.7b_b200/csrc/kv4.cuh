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
// Codes are laid out as the fragments of the attention's matrix instructions:
//   K: row r (position in the unit) has D/2 bytes = words [t 0..3][c < D/32];
//      nibble j of word (t, c) is dimension 32c + 8t + j.
//   V: 16-position tile r/16, plane (r/8)%2, lane (g 0..7, t = (r%8)/2), word
//      c < D/32, halfword r%2; nibble j of the halfword is dimension
//      32c + 4g + j (a word holds two neighbouring positions, so one mask
//      gives the pair that a matrix fragment register needs).
//   scales: [r][c] f16.
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
    qora::DevBuf part, tickets;  // attend: split partials, one arrival count per block
    int attend_blocks = 0;
};

namespace qora {

constexpr int kKv4Unit = 32;           // positions per unit
constexpr int kKv4MaxStreams = 4096;   // the attention's work list lies in shared memory
constexpr int kKv4PartRows = 16;       // query rows of the widest attention tile

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

// Byte offsets in a unit of head dimension D.
template <int D>
struct Kv4Unit {
    static constexpr int kBytes = kv4_unit_bytes(D);
    static constexpr int kK = 0, kV = 16 * D, kKs = 32 * D, kVs = 34 * D;
    static constexpr int C = D / 32;  // scale groups
    __host__ __device__ static __forceinline__ int k_word(int r, int dim) {
        return kK + r * (D / 2) + ((dim & 31) >> 3) * (D / 8) + (dim >> 5) * 4;
    }
    __host__ __device__ static __forceinline__ int v_half(int r, int dim) {
        return kV + (r >> 4) * (8 * D) + ((r >> 3) & 1) * (4 * D) +
               (((dim & 31) >> 2) * 4 + ((r & 7) >> 1)) * (D / 8) + (dim >> 5) * 4 + (r & 1) * 2;
    }
    __host__ __device__ static __forceinline__ int k_scale(int r, int c) { return kKs + (r * C + c) * 2; }
    __host__ __device__ static __forceinline__ int v_scale(int r, int c) { return kVs + (r * C + c) * 2; }
};

// Most blocks of one attention launch (its workspace is sized for them).
int kv4_attend_blocks(const qora_ctx *ctx);

}  // namespace qora
