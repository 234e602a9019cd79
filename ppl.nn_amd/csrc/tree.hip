// Attention of several new tokens per sequence over the int8 slab, with a visibility bit per (token, new token): drafted
// token trees, decode steps, chunks of a prompt. Also yields the rows' log-sums.
//
// Mathematics. For a row (token t, query head h of kv head c): x_j = q . k_j / sqrt(D) over the keys j the token sees,
// o = sum_j exp(x_j) v_j / sum_j exp(x_j), lse = ln sum_j exp(x_j). One pass over the keys with a running maximum m, sum
// l and accumulator o per row (all fp32); partial (m, l, o) of disjoint key sets combine with weights exp(m_i - m).
//
// Rows. The rows of a (sequence, kv head) are its (token, query head of the kv head) pairs, row r = token r / rep, head
// c * rep + r % rep, so a cached row is read once for all query heads and all drafted tokens of a row tile.
//
// Split. Work is laid out on one axis per kv head: for every sequence, for every row tile, its keys in tiles of 32. The
// axis is cut into num_ranges equal ranges on the device (every workgroup sums the sequences' costs itself: no host
// knowledge of the lengths, no planning launch); a workgroup walks the (sequence, row tile) pieces of its range. A range
// can start and end inside a row tile: such a piece leaves its partial in the workspace, at most two per range (the first
// and the last piece), and tree_merge_kernel combines them.
//
// Two kernels share this. tree_keys_kernel (row tiles of 16 or 32 rows): every wave carries all rows and takes every
// fourth key tile, through a region of LDS of its own; no barrier until the waves' shares are joined at the end of a
// piece. tree_rows_kernel (64, 128 or 256 rows): the waves share out the rows and all read one key tile, which the whole
// workgroup brings into LDS, so that a cached byte is dequantised once for all rows.
//
// What bounds it (measured, Llama-3-8B layer shape H 32 / KVH 8 / head_dim 128 unless said otherwise; whole calls in turn,
// without a profiler): 64 sequences of 4 - 16 drafted tokens over 256 - 4 096 keys 119 us = 3.2 TB/s, of it 10 us of partial
// results in the merge; 16 sequences of 64 tokens over 1 k - 8 k keys 116 - 118 us = 575 - 585 TFLOP/s; 8 sequences of 24
// tokens over 32 k - 128 k keys at H 8 / KVH 1 141 - 145 us = 515 - 530 TFLOP/s, 1.7 TB/s. By the counters a SIMD's two waves
// (two row blocks each) keep the vector ALU busy for 1 440 - 1 510 cycles per key tile (weights, dequantisation; 260 are the
// issue of matrix instructions) and the matrix pipe for 1 020, of the 3 000 - 3 600 that the tile takes, and the CU's LDS for
// 910: they overlap only in part. Taking out either product, the exponentials, or the staging shortens a launch by about
// that part's own time.
#include "cache_tile.h"

namespace pplhip {

typedef short short4_t __attribute__((ext_vector_type(4)));

struct TreeParams {
    const half_t* q; // [S, H, head_dim]
    const uint64_t* mask; // [S, mask_words] or null (causal)
    const int64_t* seqstarts;
    const int64_t* kvstarts;
    CacheView view;
    half_t* out;
    float* lse; // [S, H] or null
    int32_t batch, num_heads, kv_heads, rep, mask_words;
    int32_t num_ranges;
    float scale_log2; // log2(e) / sqrt(head_dim)
    // workspace: partials of kv head c, range r: slot 2 r (a piece that starts inside its row tile) and 2 r + 1 (one that
    // starts with it and ends before it does), [slot][row][DH] accumulators and [slot][row] (maximum, sum) pairs; then
    // per range where it starts: {sequence, row tile, key tile}
    float* part_o;
    float2* part_ml;
    int64_t* range_start; // [num_ranges][3]; sequence -1: nothing left for this range
};

constexpr int kTreeWaves = 4; // of tree_keys_kernel
constexpr int64_t kPieceCost = 4; // what starting and finishing a row tile costs, in key tiles (1 and 8 measure the same)
// A range is at least this long: cutting a short axis costs the merge launch. One draft over 200 keys: 12.8 us at 8 tiles,
// 11.2 at 16 and 32; 24 sequences of up to 1 500 keys and 20 heads: 41.4, 41.0, 51.9 us.
constexpr int64_t kMinRangeTiles = 16;
// The reference point m of a row's exponents need not be its running maximum: it only moves when a score passes it by
// more than 2^kSlack, so that most tiles need neither a maximum across lanes nor a rescaling. Weights are formed as
// exp2(x - m + kProbShift), at most 2^15, and enter the second product in fp16: the matrix instructions take both operands
// in one type, and V is fp16. That rounding, half a step of 2^-10, leaves outputs 2.9e-4 from 64 bits (relative norm) where
// their own rounding to fp16 makes 2.1e-4; the weights in two fp16 parts would take the second product twice. A weight keeps
// fp16's full precision down to 2^-22 of 2^m. Sums carry the same factor, are of the weights before that rounding, and keep
// 32 bits.
constexpr float kProbShift = 8.f;
constexpr float kSlack = 7.f;

__device__ inline int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Sequence b on the axis: row tiles and key tiles (0 row tiles without new tokens).
struct TreeSpan {
    int64_t row_tiles, key_tiles;
    __device__ int64_t cost() const {
        return row_tiles * (key_tiles + kPieceCost);
    }
};
__device__ inline TreeSpan tree_span(const TreeParams& p, int b, int rows_per_tile) {
    const int64_t L = p.seqstarts[b + 1] - p.seqstarts[b];
    const int64_t kv = p.kvstarts[b + 1] - p.kvstarts[b];
    return TreeSpan{L <= 0 ? 0 : (L * p.rep + rows_per_tile - 1) / rows_per_tile, (kv + kTileKeys - 1) / kTileKeys};
}

struct RangeStart {
    int32_t b;
    int32_t row_tile, key_tile;
    int64_t length; // positions of the axis in this range
};

// Where range `r` starts. Every wave works it out alone: 64 sequences' costs a step, summed and scanned across the lanes.
__device__ inline RangeStart find_range(const TreeParams& p, int r, int rows_per_tile) {
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int b = b0 + lane;
        total += b < p.batch ? tree_span(p, b, rows_per_tile).cost() : 0;
    }
    for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
    int64_t len = (total + p.num_ranges - 1) / p.num_ranges;
    if (len < kMinRangeTiles) len = kMinRangeTiles;
    RangeStart s{-1, 0, 0, 0};
    const int64_t pos = len * r;
    if (pos >= total) return s;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int b = b0 + lane;
        const TreeSpan sp = b < p.batch ? tree_span(p, b, rows_per_tile) : TreeSpan{0, 0};
        int64_t incl = sp.cost();
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t up = __shfl_up(incl, d);
            if (lane >= d) incl += up;
        }
        const uint64_t here = __ballot(before + incl > pos);
        if (here) {
            const int who = __ffsll((unsigned long long)here) - 1;
            const int64_t start = before + __shfl(incl - sp.cost(), who);
            const int64_t per_tile = __shfl(sp.key_tiles, who) + kPieceCost;
            s.b = b0 + who;
            s.row_tile = (int)((pos - start) / per_tile);
            s.key_tile = (int)((pos - start) % per_tile);
            s.length = len < total - pos ? len : total - pos;
            return s;
        }
        before += __shfl(incl, 63);
    }
    return s;
}

// Bit i: the row sees key kv0 + i (i < 32). `start`: cached tokens in front of the new ones; kv0 + 32 > start.
__device__ inline uint32_t visible_keys(const uint64_t* row_mask, int words, int token, int kv0, int start, int kvlen) {
    const int i0 = kv0 - start; // new-token index of the tile's first key (negative: history in front)
    if (!row_mask) {
        const int n = token - i0 + 1;
        return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
    }
    const int first = i0 < 0 ? 0 : i0;
    const int w = first >> 6, sh = first & 63;
    uint64_t bits = w < words ? row_mask[w] >> sh : 0;
    if (sh > 32 && w + 1 < words) bits |= row_mask[w + 1] << (64 - sh);
    uint32_t see = (uint32_t)bits;
    if (i0 < 0) see = (see << -i0) | ((1u << -i0) - 1); // (-i0 is 1 .. 31)
    const int n = kvlen - kv0;
    return n >= 32 ? see : see & ((1u << n) - 1);
}

// A value the compiler must take as new: addresses formed from it in code behind or beside the tile loop are not computed
// ahead of the loop and held in registers throughout.
__device__ inline int recomputed(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// What a wave holds of its N blocks of 16 rows: lane (g = lane / 16, lane % 16) row lane % 16 of each block, of the output
// positions 16 i + 4 g .. + 3 (channel_at) and of the sum its own keys' share.
template <int DH, int N>
struct RowState {
    int tok[N]; // token of the sequence; -1 for rows past the last one
    half8_t qf[N][DH / 32];
    float m[N], shift[N], l[N]; // m in units of the raw products; shift = kProbShift - m * scale_log2
    float4_t o[N][DH / 16];

    __device__ inline void start(const TreeParams& p, int64_t s0, int rows, const int (&first_row)[N], int kvh) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int row = first_row[n] + (lane & 15);
            const int rr = row < rows ? row : rows - 1;
            const int t = rr / p.rep;
            tok[n] = row < rows ? t : -1;
            const half_t* qp = p.q + ((s0 + t) * p.num_heads + kvh * p.rep + (rr - t * p.rep)) * p.view.head_dim;
#pragma unroll
            for (int kc = 0; kc < DH / 32; ++kc) { // (groups past head_dim: the first one, zeroed in queries_here)
                const int channel = channel_at<DH>(32 * kc + 8 * g);
                qf[n][kc] = *reinterpret_cast<const half8_t*>(qp + (channel < p.view.head_dim ? channel : 0));
            }
            m[n] = -INFINITY;
            shift[n] = kProbShift;
            l[n] = 0.f;
#pragma unroll
            for (int i = 0; i < DH / 16; ++i) o[n][i] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // Waits for the queries here, while younger loads stay in flight: what is known about loads in flight is merged at a
    // loop's head, and a load that is first used inside the loop is waited for there with everything behind it.
    __device__ inline void queries_here(int head_dim) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int kc = 0; kc < DH / 32; ++kc) {
                asm volatile("" : "+v"(qf[n][kc]));
                if (head_dim < DH && channel_at<DH>(32 * kc + 8 * g) >= head_dim) qf[n][kc] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
    }

    // the 32 keys in `tile` as operands: keys 16 * tb + lane % 16, positions 32 * kc + 8 * g .. + 7
    typedef half8_t KeyOperands[2][DH / 32];
    __device__ static inline void load_keys(const half_t* tile, KeyOperands& kf) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int kc = 0; kc < DH / 32; ++kc)
                kf[tb][kc] = *reinterpret_cast<const half8_t*>(tile + (16 * tb + (lane & 15)) * kKeyRow<DH> + 32 * kc + 8 * g);
    }

    // scores of the rows against those keys: s[n][tb][e] belongs to key 16 * tb + 4 * g + e
    __device__ inline void scores(const KeyOperands& kf, float (&s)[N][2][4]) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float4_t acc[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int kc = 0; kc < DH / 32; ++kc)
#pragma unroll
                for (int tb = 0; tb < 2; ++tb)
                    acc[tb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tb][kc], qf[n][kc], acc[tb], 0, 0, 0);
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][tb][e] = acc[tb][e];
        }
    }

    // keys a row does not see get score -inf; see[n]: bit i = key kv0 + i
    __device__ inline void hide(const TreeParams& p, int64_t s0, int kv0, int start, int kvlen,
                                float (&s)[N][2][4], uint32_t (&see)[N]) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            see[n] = tok[n] >= 0 ? visible_keys(p.mask ? p.mask + (s0 + tok[n]) * p.mask_words : nullptr, p.mask_words, tok[n],
                                             kv0, start, kvlen)
                              : 0u;
            const uint32_t mine = see[n] >> (4 * g);
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][tb][e] = (mine >> (16 * tb + e)) & 1 ? s[n][tb][e] : -INFINITY;
        }
    }

    // largest of the lane's scores of every row
    __device__ static inline void largest(const float (&s)[N][2][4], float (&top)[N]) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            top[n] = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                           fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
    }
    // whether one of them passes its row's reference point by too much
    __device__ inline bool passes(float scale_log2, const float (&top)[N]) const {
        bool moves = false;
#pragma unroll
        for (int n = 0; n < N; ++n)
            moves |= (__builtin_fmaf(top[n], scale_log2, shift[n]) > kProbShift + kSlack) |
                     ((m[n] == -INFINITY) & (top[n] > -INFINITY));
        return __any(moves);
    }
    // moves the reference points there (rows without a key so far keep m = -inf: weights exp2(-inf) = 0)
    __device__ inline void settle(float scale_log2, const float (&top)[N]) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float m_new = fmaxf(m[n], wave_max_over_quads(top[n]));
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = __builtin_amdgcn_exp2f((m[n] - ref) * scale_log2);
            m[n] = m_new;
            shift[n] = kProbShift - ref * scale_log2;
            l[n] *= alpha;
#pragma unroll
            for (int i = 0; i < DH / 16; ++i) o[n][i] *= alpha;
        }
    }

    // scores -> weights (fp16, the operand of the second product) and their sums
    __device__ inline void weights(float scale_log2, const float (&s)[N][2][4], half8_t (&pp)[N]) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float sum = 0.f;
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][tb][e], scale_log2, shift[n]));
                    sum += w;
                    pp[n][4 * tb + e] = (half_t)w;
                }
            l[n] += sum;
        }
    }

    // the 32 value rows in `tile`, transposed: lane (g, j) gets position 16 * i + j of keys 4 * g .. + 3 and 16 + 4 * g .. + 3
    typedef half8_t ValueOperands[DH / 16];
    __device__ static inline void load_values(const half_t* tile, ValueOperands& vf) {
        constexpr int LDR = kValueRow<DH>;
        const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
#pragma unroll
        for (int i = 0; i < DH / 16; ++i) {
            const half_t* src = tile + (4 * g + (j >> 2)) * LDR + 16 * i + 4 * (j & 3);
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)src);
            const short4_t hi =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(src + 16 * LDR));
            __builtin_memcpy(&vf[i], &lo, 8);
            __builtin_memcpy(reinterpret_cast<char*>(&vf[i]) + 8, &hi, 8);
        }
    }

    // o += weights x those rows
    __device__ inline void values(const ValueOperands& vf, const half8_t (&pp)[N]) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int i = 0; i < DH / 16; ++i) o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], pp[n], o[n][i], 0, 0, 0);
        }
    }

    // Value pieces that may not be finite are zeros in the tiles (a key can be hidden from a row: its weight there is 0,
    // and 0 times a NaN or an infinity is NaN). Once a piece's tiles are done, those that had such pieces are gone through
    // again: here they are multiplied key by key, and the result is taken over by the rows that see the key only. rows:
    // which rows of the tile have such pieces; base: offset of its first V row.
    __device__ inline void odd_values(const TreeParams& p, int64_t base, int kv0, int kvlen, uint32_t rows,
                                      const half8_t (&pp)[N], const uint32_t (&see)[N]) {
        const int lane = recomputed(threadIdx.x & 63), g = lane >> 4;
#pragma unroll 1
        for (; rows; rows &= rows - 1) {
            const int row = __builtin_ctz(rows);
            if (kv0 + row >= kvlen) break;
            const int8_t* vq = p.view.cache + base + row * p.view.addr.stride_s;
            const half_t* vs = p.view.scale + (base + row * p.view.addr.stride_s) / kQuantGroup;
            const int slot = (row & 3) + 4 * (row >> 4); // where lane group (row >> 2) & 3 holds the key
#pragma unroll
            for (int i = 0; i < DH / 16; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const int d = channel_at<DH>(16 * i + (lane & 15));
                half_t v = (half_t)0.f;
                if (d < p.view.head_dim && !(scale_is_small(vs[d >> 4 << 1]) && scale_is_small(vs[(d >> 4 << 1) + 1])))
                    v = (half_t)((float)vq[d] * (float)vs[d >> 3]);
                half8_t a;
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = g == ((row >> 2) & 3) && e == slot ? v : (half_t)0.f;
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const float4_t with = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pp[n], o[n][i], 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][i][e] = (see[n] >> row) & 1 ? with[e] : o[n][i][e];
                }
            }
        }
    }
};

// Writes 4 channels of a finished row, and its log-sum with channel 0. l == 0: the row saw nothing (a NaN stays NaN).
__device__ inline void finish_row(const TreeParams& p, int64_t s0, int row, int kvh, int d, float4_t a, float m_log2,
                                  float l) {
    const int t = row / p.rep;
    const int64_t at = (s0 + t) * p.num_heads + kvh * p.rep + (row - t * p.rep);
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    const half4_t r = {(half_t)(a[0] * inv), (half_t)(a[1] * inv), (half_t)(a[2] * inv), (half_t)(a[3] * inv)};
    if (d < p.view.head_dim) *reinterpret_cast<half4_t*>(p.out + at * p.view.head_dim + d) = r;
    if (p.lse && d == 0) p.lse[at] = l == 0.f ? -INFINITY : (m_log2 + (log2f(l) - kProbShift)) * 0.693147180559945f;
}

// One (sequence, row tile) piece of a range, as far as both kernels agree on it.
struct TreePiece {
    int32_t b;
    int64_t s0;
    int32_t start, kvlen, rows, row0; // row0: first row of the tile
    int32_t key_tile, stop_tile; // key tiles to look at (causal rows see nothing past their own token)
    bool whole; // all the row tile's keys are in this piece
    int32_t slot; // else: where its partial goes
};

// Calls `piece` for every piece of workgroup (range, kvh)'s range.
template <int ROWS, class F>
__device__ inline void walk_range(const TreeParams& p, int range, int kvh, F&& piece) {
    const const_tab64_t seqstarts = (const_tab64_t)p.seqstarts, kvstarts = (const_tab64_t)p.kvstarts;
    const RangeStart rs = find_range(p, range, ROWS);
    // (every lane found the same; said here, so that what follows from it is scalar)
    int64_t left = uniform64(rs.length);
    int b = __builtin_amdgcn_readfirstlane(rs.b), row_tile = __builtin_amdgcn_readfirstlane(rs.row_tile),
        key_tile = __builtin_amdgcn_readfirstlane(rs.key_tile);
    bool first = true;
    if (kvh == 0 && threadIdx.x == 0) p.range_start[3 * range] = -1; // (until a piece is found)
    while (left > 0 && b < p.batch) {
        TreePiece t;
        t.b = b;
        t.s0 = seqstarts[b];
        const int L = (int)(seqstarts[b + 1] - t.s0);
        t.kvlen = (int)(kvstarts[b + 1] - kvstarts[b]);
        t.rows = L * p.rep;
        const int row_tiles = L <= 0 ? 0 : (t.rows + ROWS - 1) / ROWS;
        const int key_tiles = (t.kvlen + kTileKeys - 1) / kTileKeys;
        if (row_tile >= row_tiles) {
            ++b;
            row_tile = key_tile = 0;
            continue;
        }
        const int end_tile = key_tile + left < key_tiles ? key_tile + (int)left : key_tiles;
        if (key_tile < end_tile) {
            if (first && kvh == 0 && threadIdx.x == 0) {
                p.range_start[3 * range] = b;
                p.range_start[3 * range + 1] = row_tile;
                p.range_start[3 * range + 2] = key_tile;
            }
            first = false;
            t.start = t.kvlen - L;
            t.row0 = row_tile * ROWS;
            t.key_tile = key_tile;
            t.stop_tile = end_tile;
            if (!p.mask) {
                const int last_row = t.row0 + ROWS < t.rows ? t.row0 + ROWS - 1 : t.rows - 1;
                const int last = (t.start + last_row / p.rep + kTileKeys) / kTileKeys;
                t.stop_tile = last < end_tile ? last : end_tile;
            }
            t.whole = key_tile == 0 && end_tile == key_tiles;
            t.slot = 2 * (kvh * p.num_ranges + range) + (key_tile == 0 ? 1 : 0);
            piece(t);
        }
        left -= key_tiles + kPieceCost - key_tile;
        ++row_tile;
        key_tile = 0;
    }
}

// Waves per SIMD that the register allocator is to leave room for, at least: what a wave's N row blocks, the tiles on their
// way and the operands of one product take. With fewer channels more of them fit (at 32 and 64 channels up to 7 and 4).
// The bound costs vector registers spilled at 256 channels (40 and 63 with 16 and 32 rows, 31 and 4 with 64 and 128) and a
// few in <224> with 32 rows (9) and <128> with 64 (2); the four-wave kernels keep 16 and 40 bytes per lane of the tiles on
// their way in scratch at 32 and 64 channels.
constexpr int tree_waves_per_simd(int dh, int row_blocks) {
    return row_blocks == 1 ? (dh <= 128 ? 3 : 2) : (dh <= 128 ? 2 : 1);
}

// NR: blocks of 16 rows every wave carries; the row tile has 16 * NR rows.
template <int DH, int NR>
__global__ __launch_bounds__(256, tree_waves_per_simd(DH, NR)) void tree_keys_kernel(const TreeParams p) {
    constexpr int ROWS = 16 * NR;
    constexpr int LDR = kValueRow<DH>; // (of the region: a K tile takes a little less)
    constexpr int LDO = DH + 4; // floats per row of the combination
    static_assert(kTreeWaves * kTileKeys * LDR * 2 >= kTreeWaves * 16 * LDO * 4, "the combination reuses the tiles");
    __shared__ __attribute__((aligned(16))) half_t lds[kTreeWaves * kTileKeys * LDR];
    __shared__ float2 ml_lds[kTreeWaves][ROWS];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int range = blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x - range * p.kv_heads;
    half_t* const tile = lds + wave * kTileKeys * LDR;

    walk_range<ROWS>(p, range, kvh, [&](const TreePiece& t) {
        RowState<DH, NR> st;
        const SequenceRows seq(p.view, t.b, kvh);
        int first_row[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) first_row[n] = t.row0 + 16 * n;
        st.start(p, t.s0, t.rows, first_row, kvh);

        CacheTile<DH> rk, rv; // the next tile's K and V rows, on their way
        int kt = t.key_tile + wave;
        const int first_key = (kt < t.stop_tile ? kt : t.key_tile) * kTileKeys; // (a wave without a tile: any)
        int64_t base = seq.key_row(first_key);
        bool odd_tiles = false;
        rk.fetch(p.view, base, first_key, t.kvlen);
        rv.fetch(p.view, base + p.view.addr.stride_kv, first_key, t.kvlen);
        st.queries_here(p.view.head_dim);
        for (; kt < t.stop_tile; kt += kTreeWaves) {
            const int kv0 = kt * kTileKeys;
            const int kv_next = kt + kTreeWaves < t.stop_tile ? kv0 + kTreeWaves * kTileKeys : kv0; // (the last: again)
            const bool history = kv0 + kTileKeys <= t.start; // every row sees every key
            wave_lds_order();
            rk.stash(tile, kKeyRow<DH>, p.view.head_dim);
            wave_lds_order();
            base = seq.key_row(kv_next);
            rk.fetch(p.view, base, kv_next, t.kvlen);
            float s[NR][2][4];
            uint32_t see[NR];
            half8_t pp[NR];
            typename RowState<DH, NR>::KeyOperands kf;
            typename RowState<DH, NR>::ValueOperands vf;
            st.load_keys(tile, kf);
            st.scores(kf, s);
            if (!history) st.hide(p, t.s0, kv0, t.start, t.kvlen, s, see);
            float top[NR];
            st.largest(s, top);
            if (st.passes(p.scale_log2, top)) st.settle(p.scale_log2, top);
            st.weights(p.scale_log2, s, pp);
            wave_lds_order();
            if (!history && rv.odd_rows()) {
                odd_tiles = true;
                rv.stash_finite(tile, kValueRow<DH>, p.view.head_dim);
            } else {
                rv.stash(tile, kValueRow<DH>, p.view.head_dim);
            }
            wave_lds_order();
            rv.fetch(p.view, base + p.view.addr.stride_kv, kv_next, t.kvlen);
            st.load_values(tile, vf);
            st.values(vf, pp);
        }
        if (odd_tiles) {
            float l_done[NR];
#pragma unroll
            for (int n = 0; n < NR; ++n) l_done[n] = st.l[n];
            for (kt = t.key_tile + wave; kt < t.stop_tile; kt += kTreeWaves) {
                const int kv0 = kt * kTileKeys;
                if (kv0 + kTileKeys <= t.start) continue;
                base = seq.key_row(kv0);
                rk.fetch(p.view, base, kv0, t.kvlen);
                rv.fetch(p.view, base + p.view.addr.stride_kv, kv0, t.kvlen);
                wave_lds_order();
                rk.stash(tile, kKeyRow<DH>, p.view.head_dim);
                wave_lds_order();
                float s[NR][2][4];
                uint32_t see[NR];
                half8_t pp[NR];
                typename RowState<DH, NR>::KeyOperands kf;
                st.load_keys(tile, kf);
                st.scores(kf, s);
                st.hide(p, t.s0, kv0, t.start, t.kvlen, s, see);
                st.weights(p.scale_log2, s, pp);
                st.odd_values(p, base + p.view.addr.stride_kv, kv0, t.kvlen, rv.odd_rows(), pp, see);
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) st.l[n] = l_done[n]; // (the sums were complete)
        }

        // ---- the four waves' shares of the piece, joined 16 rows at a time
        __syncthreads(); // (the tiles are read no more; the piece before has been written out)
        const int tid = recomputed(threadIdx.x), r_lane = tid & 15, g = (tid & 63) >> 4;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float l = wave_sum_over_quads(st.l[n]);
            if (g == 0) ml_lds[wave][16 * n + r_lane] = make_float2(st.m[n] * p.scale_log2, l);
        }
        __syncthreads();
        float* const olds = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            float m = -INFINITY;
            for (int w = 0; w < kTreeWaves; ++w) m = fmaxf(m, ml_lds[w][16 * n + r_lane].x);
            const float f = __builtin_amdgcn_exp2f(st.m[n] * p.scale_log2 - (m == -INFINITY ? 0.f : m));
            if (n) __syncthreads();
#pragma unroll
            for (int i = 0; i < DH / 16; ++i)
                *reinterpret_cast<float4_t*>(olds + (wave * 16 + r_lane) * LDO + 16 * i + 4 * g) = st.o[n][i] * f;
            __syncthreads();
            for (int x = tid; x < 16 * (DH / 4); x += 256) {
                const int r = x / (DH / 4), d = (x - r * (DH / 4)) * 4;
                float mm = -INFINITY;
                for (int w = 0; w < kTreeWaves; ++w) mm = fmaxf(mm, ml_lds[w][16 * n + r].x);
                float l = 0.f;
                float4_t a = {0.f, 0.f, 0.f, 0.f};
                for (int w = 0; w < kTreeWaves; ++w) {
                    const float2 ml = ml_lds[w][16 * n + r];
                    l += ml.y * __builtin_amdgcn_exp2f(ml.x - (mm == -INFINITY ? 0.f : mm));
                    a += *reinterpret_cast<const float4_t*>(olds + (w * 16 + r) * LDO + d);
                }
                const int row = t.row0 + 16 * n + r;
                if (t.whole) {
                    if (row < t.rows) finish_row(p, t.s0, row, kvh, channel_at<DH>(d), a, mm, l);
                } else {
                    const int64_t at = (int64_t)t.slot * ROWS + 16 * n + r;
                    *reinterpret_cast<float4_t*>(p.part_o + at * DH + d) = a;
                    if (d == 0) p.part_ml[at] = make_float2(mm, l);
                }
            }
        }
        __syncthreads();
    });
}

// W waves, each with NB blocks of 16 rows: row block i of the tile is block i / W of wave i % W, so that few rows still
// spread over all waves. The workgroup's threads bring the key tiles into LDS, two buffers and one barrier per tile. Two
// blocks per wave, because a wave's operand reads serve both: sixteen waves of one block are bound by LDS (142 against
// 125 us on 256 rows).
template <int DH, int W, int NB>
__global__ __launch_bounds__(W * 64, tree_waves_per_simd(DH, NB)) void tree_rows_kernel(const TreeParams p) {
    constexpr int ROWS = 16 * W * NB;
    __shared__ __attribute__((aligned(16))) half_t k_lds[2][kTileKeys * kKeyRow<DH>];
    __shared__ __attribute__((aligned(16))) half_t v_lds[2][kTileKeys * kValueRow<DH>];
    __shared__ uint32_t odd_lds; // value rows that were kept out of the tiles

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int range = blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x - range * p.kv_heads;

    // The two waves of a SIMD would come to their matrix and their vector instructions together; with one of them ahead by
    // its priority they take turns (measured: 2 % on 192 and 256 rows).
    if (W == 8 && wave >= 4) __builtin_amdgcn_s_setprio(1);
    walk_range<ROWS>(p, range, kvh, [&](const TreePiece& t) {
        RowState<DH, NB> st;
        const SequenceRows seq(p.view, t.b, kvh);
        int first_row[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) first_row[n] = t.row0 + 16 * (wave + W * n);
        st.start(p, t.s0, t.rows, first_row, kvh);
        const bool busy = first_row[0] < t.rows; // (a wave without rows only helps to bring the tiles)
        const int n_tiles = t.stop_tile - t.key_tile;

        // Tiles i + 1 and i + 2, on their way. Four waves bring them all, in two sets of registers by turns; eight waves in
        // two groups, every other tile each, in the first set.
        SharedTile<DH> raw[2];
        const int group = W == 8 ? wave >> 2 : 0;
        auto fetch = [&](SharedTile<DH>& r, int i) { // (past the last tile: that one again, so that every path has
                                                        // the same loads in flight and none is waited for too early)
            const int kv0 = (t.key_tile + (i < n_tiles ? i : n_tiles - 1)) * kTileKeys;
            r.fetch(p.view, seq.key_row(kv0), kv0, t.kvlen);
        };
        bool odd_pieces = false; // this thread has kept value pieces out of the tiles
        auto stash = [&](const SharedTile<DH>& r, int i) {
            const bool history = (t.key_tile + i + 1) * kTileKeys <= t.start;
            odd_pieces |= r.stash(k_lds[i & 1], v_lds[i & 1], p.view.head_dim, !history) != 0;
        };
        __syncthreads(); // (the piece before has read its last tile)
        if (threadIdx.x == 0) odd_lds = 0;
        // at tile i: tile i + 1 goes into LDS, tile i + 3 is requested. set: raw[(i + 1) & 1] of four waves
        auto bring = [&](SharedTile<DH>& set, int i) {
            if (W == 8 && group != ((i + 1) & 1)) return;
            SharedTile<DH>& mine = W == 8 ? raw[0] : set;
            stash(mine, i + 1);
            fetch(mine, i + 3);
        };
        if (n_tiles > 0) {
            fetch(raw[0], group);
            if (W == 4) fetch(raw[1], 1);
        }
        st.queries_here(p.view.head_dim);
        if (n_tiles > 0 && group == 0) {
            stash(raw[0], 0);
            fetch(raw[0], 2);
        }
        __syncthreads();
        float s[NB][2][4], top[NB];
        // scores of tile i, while tile i + 1 goes into LDS and tile i + 3 is requested
        auto look = [&](SharedTile<DH>& next, int i) {
            const int kv0 = (t.key_tile + i) * kTileKeys;
            typename RowState<DH, NB>::KeyOperands kf;
            st.load_keys(k_lds[i & 1], kf);
            __builtin_amdgcn_sched_barrier(0); // (the keys come out of LDS while the next tile goes in)
            bring(next, i);
            st.scores(kf, s);
            uint32_t see[NB];
            if (kv0 + kTileKeys > t.start) st.hide(p, t.s0, kv0, t.start, t.kvlen, s, see);
            st.largest(s, top);
        };
        // its values
        auto add = [&](int i) {
            half8_t pp[NB];
            typename RowState<DH, NB>::ValueOperands vf;
            st.load_values(v_lds[i & 1], vf);
            __builtin_amdgcn_sched_barrier(0); // (the values come out of LDS while the weights are formed)
            st.weights(p.scale_log2, s, pp);
            st.values(vf, pp);
            __syncthreads();
        };
        if (!busy) { // the same stashes, fetches and barriers as the others'
            for (int i = 0; i < n_tiles; ++i) {
                if (i & 1)
                    bring(raw[0], i);
                else
                    bring(raw[1], i);
                __syncthreads();
            }
        } else if (n_tiles > 0) {
            int i = 0;
            look(raw[1], 0);
            // Reference points move out here: inside the inner loop accumulators change by matrix instructions only, and
            // at its head raw[0] is always the older of the two tiles on their way.
            for (bool done = false; !done;) {
                if (st.passes(p.scale_log2, top)) st.settle(p.scale_log2, top);
                for (;;) {
                    add(i);
                    done = ++i >= n_tiles;
                    if (done) break;
                    look(raw[0], i);
                    if (st.passes(p.scale_log2, top)) {
                        if (W == 4) {
                            const SharedTile<DH> older = raw[1];
                            raw[1] = raw[0];
                            raw[0] = older;
                        }
                        break;
                    }
                    add(i);
                    done = ++i >= n_tiles;
                    if (done) break;
                    look(raw[1], i);
                    if (st.passes(p.scale_log2, top)) break;
                }
            }
        }
        if (odd_pieces) odd_lds = 1;
        __syncthreads();
        if (odd_lds) {
            float l_done[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) l_done[n] = st.l[n];
            for (int i = 0; i < n_tiles; ++i) {
                const int kv0 = (t.key_tile + i) * kTileKeys;
                if (kv0 + kTileKeys <= t.start) continue;
                fetch(raw[0], i);
                __syncthreads(); // everybody has read the tile before, and odd_lds
                if (threadIdx.x == 0) odd_lds = 0;
                __syncthreads();
                const uint32_t odd = raw[0].stash(k_lds[0], v_lds[0], p.view.head_dim, true);
                if (odd) atomicOr(&odd_lds, odd);
                __syncthreads();
                if (!busy) continue;
                uint32_t see[NB];
                half8_t pp[NB];
                typename RowState<DH, NB>::KeyOperands kf;
                st.load_keys(k_lds[0], kf);
                st.scores(kf, s);
                st.hide(p, t.s0, kv0, t.start, t.kvlen, s, see);
                st.weights(p.scale_log2, s, pp);
                st.odd_values(p, seq.key_row(kv0) + p.view.addr.stride_kv, kv0, t.kvlen,
                              __builtin_amdgcn_readfirstlane(odd_lds), pp, see);
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) st.l[n] = l_done[n]; // (the sums were complete)
        }
        const int lane = recomputed(threadIdx.x & 63), g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const float l = wave_sum_over_quads(st.l[n]);
            const int r = 16 * (wave + W * n) + (lane & 15); // within the tile
            if (t.whole) {
#pragma unroll
                for (int i = 0; i < DH / 16; ++i)
                    if (st.tok[n] >= 0)
                        finish_row(p, t.s0, t.row0 + r, kvh, channel_at<DH>(16 * i + 4 * g), st.o[n][i],
                                   st.m[n] * p.scale_log2, l);
            } else if (st.tok[n] >= 0) {
                const int64_t at = (int64_t)t.slot * ROWS + r;
#pragma unroll
                for (int i = 0; i < DH / 16; ++i)
                    *reinterpret_cast<float4_t*>(p.part_o + at * DH + 16 * i + 4 * g) = st.o[n][i];
                if (g == 0) p.part_ml[at] = make_float2(st.m[n] * p.scale_log2, l);
            }
        }
    });
}

// One workgroup per (range boundary, kv head): if the boundary is the first one inside its row tile, combines the row
// tile's partials: the last piece of the range before it, then the first pieces of the ranges behind it.
template <int DH>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeParams p, const int ROWS) {
    constexpr int kParts = 4; // partials a thread has in flight
    const int range = 1 + blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x % p.kv_heads;
    const const_tab64_t st = (const_tab64_t)p.range_start;
    const int64_t b = st[3 * range], row_tile = st[3 * range + 1];
    if (b < 0 || st[3 * range + 2] == 0) return; // starts nothing, or starts with its row tile
    if (st[3 * (range - 1)] == b && st[3 * (range - 1) + 1] == row_tile && st[3 * (range - 1) + 2] != 0) return;
    // how far the row tile's ranges go: 64 of them looked at a time
    int last = range;
    for (int first = range;; first += 64) {
        const int k = first + (int)(threadIdx.x & 63);
        const int64_t* const e = p.range_start + 3 * (int64_t)(k < p.num_ranges ? k : range);
        const uint64_t other = __ballot(k >= p.num_ranges || e[0] != b || e[1] != row_tile || e[2] == 0);
        last = first + (other ? __builtin_ctzll(other) : 64) - 1;
        if (other) break;
    }
    const int64_t s0 = p.seqstarts[b], rows = (p.seqstarts[b + 1] - s0) * p.rep;
    const int64_t base = (int64_t)kvh * 2 * p.num_ranges;
    for (int x = blockIdx.y * 256 + threadIdx.x; x < ROWS * (DH / 4); x += 256 * gridDim.y) {
        const int r = x / (DH / 4), d = (x - r * (DH / 4)) * 4;
        const int row = (int)row_tile * ROWS + r;
        if (row >= rows) continue;
        const int parts = last - range + 2;
        auto slot = [&](int k) { return (base + (k == 0 ? 2 * range - 1 : 2 * (range - 1 + k))) * ROWS + r; };
        float m = -INFINITY, l = 0.f;
        float4_t a = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < parts; k0 += kParts) {
            float2 ml[kParts];
            float4_t v[kParts];
#pragma unroll
            for (int k = 0; k < kParts; ++k) { // (past the last part: the first again, with no weight)
                const int64_t at = slot(k0 + k < parts ? k0 + k : 0);
                ml[k] = p.part_ml[at];
                v[k] = *reinterpret_cast<const float4_t*>(p.part_o + at * DH + d);
            }
            float m_new = m;
#pragma unroll
            for (int k = 0; k < kParts; ++k) m_new = fmaxf(m_new, ml[k].x);
            const float m_safe = m_new == -INFINITY ? 0.f : m_new;
            const float f0 = __builtin_amdgcn_exp2f(m - m_safe);
            l *= f0;
            a *= f0;
            m = m_new;
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                if (k0 + k >= parts) continue;
                const float f = __builtin_amdgcn_exp2f(ml[k].x - m_safe);
                l += ml[k].y * f;
                a += v[k] * f;
            }
        }
        finish_row(p, s0, row, kvh, channel_at<DH>(d), a, m, l);
    }
}

// ---- host side

// The longest sequence's (token, shared head) rows decide the row tile: the smallest that holds them, so that the cache is
// read and dequantised once; 256 at most, 128 above head_dim 128, where eight waves of two row blocks do not fit a CU's
// registers. Measured: up to 64 rows in tiles of 64 / of 32 (tree_keys_kernel) 119 / 158 us on the serving batch above, 256
// rows in tiles of 256 / of 128 117 / 145 us, 192 rows 144 / 174 us. Up to 32 rows the other way round: tiles of 64 would
// leave all waves but one or two without rows, where tree_keys_kernel gives each a quarter of the keys.
int tree_row_tile(const pplhip_tree_attention_args* a) {
    const int64_t rows = a->max_seqlen * (a->num_heads / a->num_kv_heads);
    return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 || a->head_dim > 128 ? 128 : 256;
}

// As many ranges as workgroups fit a CU at the waves per SIMD asked for above (where more are resident, at 32 and 64
// channels, those have no range), shared out among the kv heads (twice as many, with eight waves a workgroup, when the
// kernels took 126 and 171 us: 147 on 256 rows, 203 on 192 rows over long contexts); never more than ranges of the least
// length in the longest possible axis.
int64_t tree_num_ranges(const pplhip_tree_attention_args* a, int cu_count) {
    const int64_t rep = a->num_heads / a->num_kv_heads;
    const int64_t row_tiles = (a->max_seqlen * rep + tree_row_tile(a) - 1) / tree_row_tile(a);
    const int64_t key_tiles = (a->max_kvlen + kTileKeys - 1) / kTileKeys;
    const int row_blocks = tree_row_tile(a) == 16 || tree_row_tile(a) == 64 ? 1 : 2;
    const int per_cu = tree_waves_per_simd(padded_head_dim(a->head_dim), row_blocks) / (tree_row_tile(a) == 256 ? 2 : 1);
    int64_t ranges = (int64_t)cu_count * per_cu / a->num_kv_heads;
    const double most = (double)a->batch * (double)row_tiles * (double)(key_tiles + kPieceCost) / kMinRangeTiles;
    if ((double)ranges > most) ranges = (int64_t)most + 1;
    return ranges < 1 ? 1 : ranges;
}

bool tree_launches_fit(const pplhip_tree_attention_args* a, int64_t ranges) {
    return launch_fits((double)ranges * a->num_kv_heads, tree_row_tile(a) == 256 ? 512 : 256);
}

uint64_t tree_workspace_bytes(const pplhip_tree_attention_args* a, int64_t ranges) {
    const uint64_t rows = (uint64_t)a->num_kv_heads * 2 * (uint64_t)ranges * tree_row_tile(a);
    return rows * padded_head_dim(a->head_dim) * sizeof(float) + rows * sizeof(float2) + (uint64_t)ranges * 3 * sizeof(int64_t);
}

template <int DH>
static void launch_tree_dh(const TreeParams& p, int row_tile, hipStream_t stream) {
    const dim3 grid((unsigned)(p.num_ranges * p.kv_heads));
    switch (row_tile) {
        case 16: hipLaunchKernelGGL((tree_keys_kernel<DH, 1>), grid, dim3(256), 0, stream, p); break;
        case 32: hipLaunchKernelGGL((tree_keys_kernel<DH, 2>), grid, dim3(256), 0, stream, p); break;
        case 64: hipLaunchKernelGGL((tree_rows_kernel<DH, 4, 1>), grid, dim3(256), 0, stream, p); break;
        case 128: hipLaunchKernelGGL((tree_rows_kernel<DH, 4, 2>), grid, dim3(256), 0, stream, p); break;
        default:
            if constexpr (DH <= 128) hipLaunchKernelGGL((tree_rows_kernel<DH, 8, 2>), grid, dim3(512), 0, stream, p);
    }
    if (p.num_ranges > 1) {
        const int blocks = row_tile * (DH / 4) / 256;
        hipLaunchKernelGGL(tree_merge_kernel<DH>, dim3((unsigned)((p.num_ranges - 1) * p.kv_heads), (unsigned)(blocks > 0 ? blocks : 1)),
                           dim3(256), 0, stream, p, row_tile);
    }
}

pplhip_retcode launch_tree_attention(const pplhip_tree_attention_args* a, int64_t ranges, void* ws, hipStream_t stream) {
    TreeParams p;
    p.q = (const half_t*)a->d_query;
    p.mask = a->d_tree_mask;
    p.seqstarts = a->d_seqstarts;
    p.kvstarts = a->d_kvstarts;
    p.view = CacheView{(const int8_t*)a->d_cache, (const half_t*)a->d_scale,
                       PageMap{a->d_cachestarts, a->cachestart_stride_b, page_shift_of(a->cache_mode, a->page_size)},
                       CacheAddr{a->cache_stride_s, a->cache_stride_l, a->cache_stride_h, a->cache_stride_kv, a->layer_idx},
                       a->head_dim};
    p.out = (half_t*)a->d_output;
    p.lse = (float*)a->d_lse;
    p.batch = (int32_t)a->batch;
    p.num_heads = a->num_heads;
    p.kv_heads = a->num_kv_heads;
    p.rep = a->num_heads / a->num_kv_heads;
    p.mask_words = a->tree_mask_words;
    p.num_ranges = (int32_t)ranges;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)a->head_dim));
    const int row_tile = tree_row_tile(a);
    const uint64_t rows = (uint64_t)p.kv_heads * 2 * (uint64_t)ranges * row_tile;
    p.part_o = (float*)ws;
    p.part_ml = (float2*)(p.part_o + rows * padded_head_dim(a->head_dim));
    p.range_start = (int64_t*)(p.part_ml + rows);
    switch (padded_head_dim(a->head_dim)) {
        case 32: launch_tree_dh<32>(p, row_tile, stream); break;
        case 64: launch_tree_dh<64>(p, row_tile, stream); break;
        case 96: launch_tree_dh<96>(p, row_tile, stream); break;
        case 128: launch_tree_dh<128>(p, row_tile, stream); break;
        case 160: launch_tree_dh<160>(p, row_tile, stream); break;
        case 192: launch_tree_dh<192>(p, row_tile, stream); break;
        case 224: launch_tree_dh<224>(p, row_tile, stream); break;
        default: launch_tree_dh<256>(p, row_tile, stream); break;
    }
    PPLHIP_CHECK_LAUNCH("tree_attention");
    return PPLHIP_RC_SUCCESS;
}

} // namespace pplhip
