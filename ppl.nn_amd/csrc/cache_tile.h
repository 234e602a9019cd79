// How a wave brings 32 consecutive cached rows (one kv head's K or V) from the int8 slab into LDS as fp16, for the kernels
// that feed them to the matrix cores (tree.hip, score.hip).
//
// A lane loads 16-byte pieces (two quantisation groups), consecutive lanes consecutive pieces of a row, so that one load
// instruction covers whole 128-byte lines, and with them the two groups' scales (4 bytes). Dequantisation happens in that
// orientation, where a group's scale is one value: fp16(float(q) * float(scale)), as everywhere.
//
// In LDS a row has DH channels (head_dim rounded up to a multiple of 32, zeros past head_dim) in units of one group (16
// bytes): first the pieces' even groups, then their odd ones, so that the lanes of a row write 16 consecutive units at a
// time. Which channel a position holds (channel_at) only matters where queries are loaded and outputs stored. K rows are
// padded by one unit, V rows by two, so that the 16-byte reads of 16 K rows at one position, and the transposing 8-byte reads
// of four V rows, touch every bank once. Lanes of other positions come in between: the counter of bank conflicts has 32
// cycles per tile of 128 channels and wave that reads it (in tree.hip of some 110 that LDS is busy for), and none that go
// with the stores.
#ifndef PPLHIP_CSRC_CACHE_TILE_H_
#define PPLHIP_CSRC_CACHE_TILE_H_

#include "common.h"

namespace pplhip {

typedef uint32_t uint4_vt __attribute__((ext_vector_type(4)));
typedef const int64_t __attribute__((address_space(4)))* const_tab64_t; // wave-uniform reads are scalar loads

constexpr int kTileKeys = 32;

// PageMap::token for a wave-uniform (b, j): scalar loads, whatever the kernel has stored before
__device__ inline int64_t uniform_token(const PageMap& pages, int b, int j) {
    const const_tab64_t tab = (const_tab64_t)pages.cachestarts;
    if (pages.page_shift == 0) return tab[b] + j;
    return tab[b * pages.stride_b + (j >> pages.page_shift)] + (j & ((1 << pages.page_shift) - 1));
}

template <int DH>
constexpr int kKeyRow = DH + 8; // halves per K row in LDS
template <int DH>
constexpr int kValueRow = DH + 16; // halves per V row

// channel at a position of an LDS row
template <int DH>
__device__ inline int channel_at(int position) {
    const int unit = position >> 3;
    const int group = unit < DH / 16 ? 2 * unit : 2 * (unit - DH / 16) + 1;
    return 8 * group + (position & 7);
}

// Where a call's cached rows are; the same for every workgroup.
struct CacheView {
    const int8_t* cache;
    const half_t* scale;
    PageMap pages;
    CacheAddr addr;
    int32_t head_dim;
};

// One sequence's rows of one kv head, with what does not change along it worked out once.
struct SequenceRows {
    const_tab64_t pages; // the sequence's page-table row (paged)
    int64_t head_row; // paged: element offset of slab token 0's K row; contiguous: of the sequence's key 0
    int32_t stride_s, page_shift;

    __device__ inline SequenceRows(const CacheView& v, int b, int kvh)
        : pages((const_tab64_t)v.pages.cachestarts + b * v.pages.stride_b), head_row(v.addr.row(0, 0, kvh)),
          stride_s((int32_t)v.addr.stride_s), page_shift(v.pages.page_shift) {
        if (page_shift == 0) head_row = v.addr.row(((const_tab64_t)v.pages.cachestarts)[b], 0, kvh);
    }
    // element offset of the K row of key j (wave-uniform; a run of 32 keys from a multiple of 32 lies in one page)
    __device__ inline int64_t key_row(int j) const {
        if (page_shift == 0) return head_row + (int64_t)j * stride_s;
        return head_row + (pages[j >> page_shift] + (j & ((1 << page_shift) - 1))) * (int64_t)stride_s;
    }
};

inline int padded_head_dim(int head_dim) { // the kernels' DH
    return (head_dim + 31) / 32 * 32;
}

// The wave's LDS operations keep their order by themselves; this only tells the compiler that lanes read what other
// lanes of the wave wrote.
__device__ inline void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// |int8| <= 128, and 128 * 511 is below fp16's largest: such a group's values are finite
__device__ inline bool scale_is_small(half_t s) {
    return __builtin_fabsf((float)s) < 511.f;
}
__device__ inline bool piece_is_small(uint32_t scales) { // of the two groups of a 16-byte piece
    const half2_t s2 = as_half2(scales);
    return scale_is_small(s2.x) && scale_is_small(s2.y);
}

// a piece on its way into LDS; row: the start of its row there, scales 0 for pieces past head_dim
template <int DH>
__device__ inline void stash_piece(half_t* row, int piece, const uint4_vt& q, uint32_t scales) {
    const half2_t s2 = as_half2(scales);
    *reinterpret_cast<half8_t*>(row + 8 * piece) = dequant8(q.x, q.y, s2.x);
    *reinterpret_cast<half8_t*>(row + 8 * (DH / 16 + piece)) = dequant8(q.z, q.w, s2.y);
}

// Offset of a piece in a tile whose last existing row is `last`. Every lane loads something, without a branch: rows past
// the last repeat it, pieces past head_dim repeat the first (their scales become zeros on the way into LDS). Token
// strides are below 2^25 elements: 32 of them fit 32 bits.
__device__ inline uint32_t piece_offset(const CacheView& v, int row, int piece, int last) {
    return (uint32_t)(row < last ? row : last) * (uint32_t)v.addr.stride_s + (16 * piece < v.head_dim ? 16u * piece : 0u);
}

template <int DH>
struct CacheTile {
    static constexpr int PIECES = DH / 16; // 16-byte pieces of a row
    static constexpr int NLD = DH / 32; // pieces a lane loads
    uint4_vt q[NLD];
    uint32_t s[NLD];

    // rows kv0 .. kv0 + 31 from element offset `base`; rows past the sequence's last key (kvlen - 1) repeat it, so that
    // nothing unwritten is ever multiplied
    __device__ inline void fetch(const CacheView& v, int64_t base, int kv0, int kvlen) {
        const int lane = threadIdx.x & 63;
        const int last = kvlen - kv0 < kTileKeys ? kvlen - kv0 - 1 : kTileKeys - 1;
        const char* cbase = (const char*)v.cache + base;
        const char* sbase = (const char*)v.scale + base / 4; // one fp16 per 8 channels
#pragma unroll
        for (int n = 0; n < NLD; ++n) {
            const uint32_t c = lane + 64 * n;
            const uint32_t off = piece_offset(v, c / PIECES, c % PIECES, last);
            q[n] = __builtin_nontemporal_load(reinterpret_cast<const uint4_vt*>(cbase + off));
            s[n] = *reinterpret_cast<const uint32_t*>(sbase + off / 4);
        }
    }

    // ldr: halves per LDS row (kKeyRow or kValueRow)
    __device__ inline void stash(half_t* tile, int ldr, int head_dim) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int n = 0; n < NLD; ++n) {
            const uint32_t c = lane + 64 * n;
            const int row = c / PIECES, piece = c % PIECES;
            stash_piece<DH>(tile + row * ldr, piece, q[n], 16 * piece < head_dim ? s[n] : 0u);
        }
    }

    // bit r: row r may hold a value that is not finite
    __device__ inline uint32_t odd_rows() const {
        uint32_t rows = 0;
#pragma unroll
        for (int n = 0; n < NLD; ++n) {
            for (uint64_t bad = __ballot(!piece_is_small(s[n])); bad; bad &= bad - 1)
                rows |= 1u << ((__builtin_ctzll(bad) + 64 * n) / PIECES);
        }
        return rows;
    }
    // as stash, with zeros for the pieces that may hold such values
    __device__ inline void stash_finite(half_t* tile, int ldr, int head_dim) const {
        CacheTile<DH> t = *this;
#pragma unroll
        for (int n = 0; n < NLD; ++n) t.s[n] = piece_is_small(s[n]) ? s[n] : 0u;
        t.stash(tile, ldr, head_dim);
    }
};

// The same for four waves that bring a tile together: a thread's pieces of the tile's K and V rows.
template <int DH>
struct SharedTile {
    static constexpr int W = 4;
    static constexpr int PIECES = DH / 16;
    static constexpr int ALL = 2 * kTileKeys * PIECES; // K's, then V's
    static constexpr int NLD = (ALL + 64 * W - 1) / (64 * W);
    uint4_vt q[NLD];
    uint32_t s[NLD];

    // Piece n of this thread: K or V (the same for the whole wave: a tile's K pieces are a multiple of 64), row, piece of it
    __device__ static inline void place(int n, int* kv, int* row, int* piece) {
        const int first = 64 * ((__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & (W - 1)) + W * n); // the wave's first piece
        *kv = first >= kTileKeys * PIECES;
        const uint32_t c = (threadIdx.x & 63) + first - (*kv ? kTileKeys * PIECES : 0);
        *row = c / PIECES;
        *piece = c % PIECES;
    }
    // base: element offset of the tile's first K row
    __device__ inline void fetch(const CacheView& v, int64_t base, int kv0, int kvlen) {
        const int last = kvlen - kv0 < kTileKeys ? kvlen - kv0 - 1 : kTileKeys - 1;
#pragma unroll
        for (int n = 0; n < NLD; ++n) {
            int kv, row, piece;
            place(n, &kv, &row, &piece);
            const int64_t first = base + (kv ? v.addr.stride_kv : 0);
            const uint32_t off = piece_offset(v, row, piece, last);
            q[n] = __builtin_nontemporal_load(reinterpret_cast<const uint4_vt*>((const char*)v.cache + first + off));
            s[n] = *reinterpret_cast<const uint32_t*>((const char*)v.scale + first / 4 + off / 4);
        }
    }
    // finite_values: V pieces that may not be finite become zeros; returns the rows of those this thread had
    __device__ inline uint32_t stash(half_t* k_tile, half_t* v_tile, int head_dim, bool finite_values) const {
        uint32_t odd = 0;
        if (!finite_values && head_dim == DH) { // (nearly every tile)
#pragma unroll
            for (int n = 0; n < NLD; ++n) {
                int kv, row, piece;
                place(n, &kv, &row, &piece);
                if (row >= kTileKeys) break;
                stash_piece<DH>(kv ? v_tile + row * kValueRow<DH> : k_tile + row * kKeyRow<DH>, piece, q[n], s[n]);
            }
            return 0;
        }
#pragma unroll
        for (int n = 0; n < NLD; ++n) {
            int kv, row, piece;
            place(n, &kv, &row, &piece);
            if (row >= kTileKeys) break;
            const bool keep = !(finite_values && kv) || piece_is_small(s[n]);
            odd |= keep ? 0u : 1u << row;
            stash_piece<DH>(kv ? v_tile + row * kValueRow<DH> : k_tile + row * kKeyRow<DH>, piece, q[n],
                            16 * piece < head_dim && keep ? s[n] : 0u);
        }
        return odd;
    }
};

} // namespace pplhip

#endif
