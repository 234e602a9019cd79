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
// knowledge of the lengths, no planning launch); a workgroup walks the (sequence, row tile) pieces of its range, its four
// waves taking every fourth key tile and combining in LDS at the end of a piece. A range can start and end inside a row
// tile: such a piece leaves its partial in the workspace, at most two per range (the first and the last piece), and
// tree_merge_kernel combines them.
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

constexpr int kTreeWaves = 4;
constexpr int64_t kPieceCost = 4; // what starting and finishing a row tile costs, in key tiles
constexpr int64_t kMinRangeTiles = 8; // a range is at least this long: two key tiles per wave
// Probabilities are held as 2^kProbShift * exp2(x - m): the fp16 operand of the second product then keeps full precision
// for weights down to 2^-26 of the row's largest (2^-14 unshifted). Sums carry the same factor.
constexpr float kProbShift = 12.f;

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
    int64_t row_tile, key_tile, length; // length: positions of the axis in this range
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
            s.b = __builtin_amdgcn_readfirstlane(b0 + who);
            s.row_tile = uniform64((pos - start) / per_tile);
            s.key_tile = uniform64((pos - start) % per_tile);
            s.length = uniform64(len < total - pos ? len : total - pos);
            return s;
        }
        before += __shfl(incl, 63);
    }
    return s;
}

// Bit i: the row sees key kv0 + i (i < 32). `start`: cached tokens in front of the new ones.
__device__ inline uint32_t visible_keys(const uint64_t* row_mask, int words, int64_t token, int64_t kv0, int64_t start,
                                        int64_t kvlen) {
    if (kv0 + kTileKeys <= start) return ~0u;
    const int64_t i0 = kv0 - start; // new-token index of the tile's first key (negative: history in front)
    if (!row_mask) {
        const int64_t n = token - i0 + 1;
        return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
    }
    const int64_t first = i0 < 0 ? 0 : i0;
    const int64_t w = first >> 6;
    const int sh = (int)(first & 63);
    uint64_t bits = w < words ? row_mask[w] >> sh : 0;
    if (sh > 32 && w + 1 < words) bits |= row_mask[w + 1] << (64 - sh);
    uint32_t see = (uint32_t)bits;
    if (i0 < 0) {
        const int hist = (int)-i0; // 1 .. 31
        see = (see << hist) | ((1u << hist) - 1);
    }
    const int64_t n = kvlen - kv0;
    return n >= 32 ? see : see & ((1u << n) - 1);
}

// NR: blocks of 16 rows a wave carries; the row tile has 16 * NR rows.
template <int DH, int NR>
__global__ __launch_bounds__(256, 2) void tree_attention_kernel(const TreeParams p) {
    constexpr int ROWS = 16 * NR;
    constexpr int LDR = CacheTile<DH>::LDR; // halves per LDS row
    constexpr int LDO = DH + 4; // floats per row of the combination
    constexpr int KC = DH / 16, KC2 = DH / 32;
    static_assert(kTreeWaves * kTileKeys * LDR * 2 >= kTreeWaves * 16 * LDO * 4, "the combination reuses the tiles");
    __shared__ __attribute__((aligned(16))) half_t lds[kTreeWaves * kTileKeys * LDR];
    __shared__ float2 ml_lds[kTreeWaves][ROWS];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r_lane = lane & 15, g = lane >> 4;
    const int hd = p.view.head_dim;
    const int range = blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x - range * p.kv_heads;
    const const_tab64_t seqstarts = (const_tab64_t)p.seqstarts, kvstarts = (const_tab64_t)p.kvstarts;
    half_t* const tile = lds + wave * kTileKeys * LDR;

    const RangeStart rs = find_range(p, range, ROWS);
    int64_t left = rs.length;
    int b = rs.b;
    int64_t row_tile = rs.row_tile, key_tile = rs.key_tile;
    int64_t first_b = -1, first_row_tile = 0, first_key_tile = 0;
    bool first_piece = true;
    while (left > 0 && b < p.batch) {
        const int64_t s0 = seqstarts[b];
        const int64_t L = seqstarts[b + 1] - s0;
        const int64_t kvlen = kvstarts[b + 1] - kvstarts[b];
        const int64_t rows = L * p.rep;
        const int64_t row_tiles = L <= 0 ? 0 : (rows + ROWS - 1) / ROWS;
        const int64_t key_tiles = (kvlen + kTileKeys - 1) / kTileKeys;
        if (row_tile >= row_tiles) {
            ++b;
            row_tile = key_tile = 0;
            continue;
        }
        const int64_t end_tile = key_tile + left < key_tiles ? key_tile + left : key_tiles;
        if (key_tile < end_tile) {
            if (first_piece) {
                first_b = b;
                first_row_tile = row_tile;
                first_key_tile = key_tile;
            }
            const int64_t start = kvlen - L;
            const int64_t row0 = row_tile * ROWS;
            // causal rows see nothing past the tile's last token
            const int64_t last_row = row0 + ROWS < rows ? row0 + ROWS - 1 : rows - 1;
            int64_t stop_tile = end_tile;
            if (!p.mask) {
                const int64_t t = (start + last_row / p.rep + kTileKeys) / kTileKeys;
                stop_tile = t < stop_tile ? t : stop_tile;
            }
            int64_t tok[NR];
            int head[NR];
            bool valid[NR];
            half8_t qf[NR][KC2];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int64_t row = row0 + 16 * n + r_lane;
                valid[n] = row < rows;
                const int64_t rr = valid[n] ? row : rows - 1;
                tok[n] = rr / p.rep;
                head[n] = kvh * p.rep + (int)(rr - tok[n] * p.rep);
                const half_t* qp = p.q + ((s0 + tok[n]) * p.num_heads + head[n]) * hd + 8 * g;
#pragma unroll
                for (int kc = 0; kc < KC2; ++kc) {
                    if (32 * kc + 8 * g < hd) {
                        qf[n][kc] = *reinterpret_cast<const half8_t*>(qp + 32 * kc);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) qf[n][kc][e] = (half_t)0.f;
                    }
                }
            }
            float m_run[NR], l_run[NR];
            float4_t o[NR][KC];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                m_run[n] = -INFINITY;
                l_run[n] = 0.f;
#pragma unroll
                for (int i = 0; i < KC; ++i) o[n][i] = float4_t{0.f, 0.f, 0.f, 0.f};
            }

            CacheTile<DH> rk, rv;
            int64_t kt = key_tile + wave;
            int64_t base = 0;
            if (kt < stop_tile) {
                base = p.view.key_row(b, kt * kTileKeys, kvh);
                rk.fetch(p.view, base, kt * kTileKeys, kvlen);
                rv.fetch(p.view, base + p.view.addr.stride_kv, kt * kTileKeys, kvlen);
            }
            for (; kt < stop_tile; kt += kTreeWaves) {
                const int64_t kv0 = kt * kTileKeys;
                const bool more = kt + kTreeWaves < stop_tile;
                wave_lds_order();
                rk.stash(tile);
                wave_lds_order();
                if (more) {
                    base = p.view.key_row(b, kv0 + kTreeWaves * kTileKeys, kvh);
                    rk.fetch(p.view, base, kv0 + kTreeWaves * kTileKeys, kvlen);
                }
                // ---- scores: lane (g, r_lane) gets rows' column r_lane, keys 16 * tb + 4 * g + e
                float s[NR][2][4];
#pragma unroll
                for (int tb = 0; tb < 2; ++tb) {
                    float4_t acc[NR];
#pragma unroll
                    for (int n = 0; n < NR; ++n) acc[n] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kc = 0; kc < KC2; ++kc) {
                        const half8_t a = *reinterpret_cast<const half8_t*>(tile + (16 * tb + r_lane) * LDR + 32 * kc + 8 * g);
#pragma unroll
                        for (int n = 0; n < NR; ++n)
                            acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[n][kc], acc[n], 0, 0, 0);
                    }
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[n][tb][e] = acc[n][e];
                }
                const bool history = kv0 + kTileKeys <= start; // every row sees every key
                uint32_t see[NR];
                if (!history) {
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        see[n] = valid[n] ? visible_keys(p.mask ? p.mask + (s0 + tok[n]) * p.mask_words : nullptr,
                                                         p.mask_words, tok[n], kv0, start, kvlen)
                                          : 0u;
#pragma unroll
                        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s[n][tb][e] = (see[n] >> (16 * tb + 4 * g + e)) & 1 ? s[n][tb][e] : -INFINITY;
                    }
                }
                // ---- running maximum, probabilities, sum
                half8_t pp[NR];
                float alpha[NR];
                bool still = true;
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    float m = s[n][0][0];
#pragma unroll
                    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) m = fmaxf(m, s[n][tb][e]);
                    m = fmaxf(m, __shfl_xor(m, 16));
                    m = fmaxf(m, __shfl_xor(m, 32));
                    const float m_new = fmaxf(m_run[n], m);
                    // a row that has seen nothing yet: probabilities exp2(-inf) = 0, not NaN
                    const float m_safe = m_new == -INFINITY ? 0.f : m_new;
                    alpha[n] = __builtin_amdgcn_exp2f((m_run[n] - m_safe) * p.scale_log2);
                    const float shift = kProbShift - m_safe * p.scale_log2;
                    float sum = 0.f;
#pragma unroll
                    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][tb][e], p.scale_log2, shift));
                            sum += pr;
                            s[n][tb][e] = pr;
                            pp[n][4 * tb + e] = (half_t)pr; // fp16 for the matrix product; the sum keeps 32 bits
                        }
                    l_run[n] = l_run[n] * alpha[n] + sum; // the lane's share: its own 8 keys of every tile
                    m_run[n] = m_new;
                    still = still && alpha[n] == 1.0f;
                }
                if (!__all(still)) {
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int i = 0; i < KC; ++i) o[n][i] *= alpha[n];
                }
                // ---- values. Among the new tokens a key may be hidden from some rows; its weight there is 0, and 0 times
                // a NaN or an infinity is NaN: such value rows are kept out of the matrix product and added row by row.
                const uint32_t odd_rows = history ? 0u : rv.odd_rows();
                wave_lds_order();
                rv.stash(tile);
                wave_lds_order();
                if (odd_rows) {
                    for (uint32_t rest = odd_rows; rest; rest &= rest - 1) {
                        const int row = __builtin_ctz(rest);
                        if (lane < DH / 16) {
                            const uint4_vt z{0, 0, 0, 0};
                            uint4_vt* dst = reinterpret_cast<uint4_vt*>(tile + row * LDR + 16 * lane);
                            dst[0] = z;
                            dst[1] = z;
                        }
                    }
                    wave_lds_order();
                }
                if (more) rv.fetch(p.view, base + p.view.addr.stride_kv, kv0 + kTreeWaves * kTileKeys, kvlen);
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    // lane (g, j) receives channel 16 * i + j of keys 4 * g .. + 3 and 16 + 4 * g .. + 3
                    const half_t* src = tile + (4 * g + (r_lane >> 2)) * LDR + 16 * i + 4 * (r_lane & 3);
                    const short4_t lo =
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)src);
                    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) short4_t*)(src + 16 * LDR));
                    half8_t a;
                    __builtin_memcpy(&a, &lo, 8);
                    __builtin_memcpy(reinterpret_cast<char*>(&a) + 8, &hi, 8);
#pragma unroll
                    for (int n = 0; n < NR; ++n) o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pp[n], o[n][i], 0, 0, 0);
                }
                if (odd_rows) {
                    const int64_t vbase = p.view.key_row(b, kv0, kvh) + p.view.addr.stride_kv;
                    for (uint32_t rest = odd_rows; rest; rest &= rest - 1) {
                        const int row = __builtin_ctz(rest);
                        if (kv0 + row >= kvlen) break;
                        const int8_t* vq = p.view.cache + vbase + row * p.view.addr.stride_s;
                        const half_t* vs = p.view.scale + (vbase + row * p.view.addr.stride_s) / kQuantGroup;
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            float w = 0.f;
#pragma unroll
                            for (int k = 0; k < 8; ++k) w = (row & 3) + 4 * (row >> 4) == k ? s[n][k >> 2][k & 3] : w;
                            w = (float)(half_t)__shfl(w, 16 * ((row >> 2) & 3) + r_lane);
                            if ((see[n] >> row) & 1) {
#pragma unroll
                                for (int i = 0; i < KC; ++i)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        const int d = 16 * i + 4 * g + e;
                                        if (d < hd) o[n][i][e] += w * (float)(half_t)((float)vq[d] * (float)vs[d >> 3]);
                                    }
                            }
                        }
                    }
                }
            }

            // ---- the four waves' shares of the piece, combined 16 rows at a time
            const bool whole = key_tile == 0 && end_tile == key_tiles;
            const int64_t slot = 2 * (int64_t)range + (key_tile == 0 ? 1 : 0);
            __syncthreads(); // (the tiles are read no more; the piece before has been written out)
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                l_run[n] += __shfl_xor(l_run[n], 16);
                l_run[n] += __shfl_xor(l_run[n], 32);
                if (g == 0) ml_lds[wave][16 * n + r_lane] = make_float2(m_run[n] * p.scale_log2, l_run[n]);
            }
            __syncthreads();
            float* const olds = reinterpret_cast<float*>(lds);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                float m = -INFINITY;
                for (int w = 0; w < kTreeWaves; ++w) m = fmaxf(m, ml_lds[w][16 * n + r_lane].x);
                const float m_safe = m == -INFINITY ? 0.f : m;
                const float f = __builtin_amdgcn_exp2f(m_run[n] * p.scale_log2 - m_safe);
                if (n) __syncthreads();
#pragma unroll
                for (int i = 0; i < KC; ++i)
                    *reinterpret_cast<float4_t*>(olds + (wave * 16 + r_lane) * LDO + 16 * i + 4 * g) = o[n][i] * f;
                __syncthreads();
                for (int x = threadIdx.x; x < 16 * (DH / 4); x += 256) {
                    const int r = x / (DH / 4), d = (x - r * (DH / 4)) * 4;
                    float mm = -INFINITY;
                    for (int w = 0; w < kTreeWaves; ++w) mm = fmaxf(mm, ml_lds[w][16 * n + r].x);
                    const float mm_safe = mm == -INFINITY ? 0.f : mm;
                    float l = 0.f;
                    float4_t a = {0.f, 0.f, 0.f, 0.f};
                    for (int w = 0; w < kTreeWaves; ++w) {
                        const float2 ml = ml_lds[w][16 * n + r];
                        l += ml.y * __builtin_amdgcn_exp2f(ml.x - mm_safe);
                        a += *reinterpret_cast<const float4_t*>(olds + (w * 16 + r) * LDO + d);
                    }
                    const int64_t row = row0 + 16 * n + r;
                    if (whole) {
                        if (row < rows && d < hd) {
                            const int64_t t = row / p.rep;
                            const int64_t at = (s0 + t) * p.num_heads + kvh * p.rep + (row - t * p.rep);
                            const float inv = l != 0.f ? 1.0f / l : 0.f; // (NaN stays NaN)
                            const half4_t r4 = {(half_t)(a[0] * inv), (half_t)(a[1] * inv), (half_t)(a[2] * inv),
                                                (half_t)(a[3] * inv)};
                            *reinterpret_cast<half4_t*>(p.out + at * hd + d) = r4;
                            if (p.lse && d == 0)
                                p.lse[at] = l == 0.f ? -INFINITY : (mm + (log2f(l) - kProbShift)) * 0.693147180559945f;
                        }
                    } else {
                        const int64_t at = ((int64_t)kvh * 2 * p.num_ranges + slot) * ROWS + 16 * n + r;
                        *reinterpret_cast<float4_t*>(p.part_o + at * DH + d) = a;
                        if (d == 0) p.part_ml[at] = make_float2(mm, l);
                    }
                }
            }
            __syncthreads();
            first_piece = false;
        }
        const int64_t to_next = key_tiles + kPieceCost - key_tile;
        left -= to_next;
        ++row_tile;
        key_tile = 0;
    }
    if (kvh == 0 && threadIdx.x == 0) {
        p.range_start[3 * range] = first_b;
        p.range_start[3 * range + 1] = first_row_tile;
        p.range_start[3 * range + 2] = first_key_tile;
    }
}

// One workgroup per (range boundary, kv head): if the boundary is the first one inside its row tile, combines the row
// tile's partials: the last piece of the range before it, then the first pieces of the ranges behind it.
template <int DH, int NR>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeParams p) {
    constexpr int ROWS = 16 * NR;
    const int range = 1 + blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x % p.kv_heads;
    const const_tab64_t st = (const_tab64_t)p.range_start;
    const int64_t b = st[3 * range], row_tile = st[3 * range + 1];
    if (b < 0 || st[3 * range + 2] == 0) return; // starts nothing, or starts with its row tile
    if (st[3 * (range - 1)] == b && st[3 * (range - 1) + 1] == row_tile && st[3 * (range - 1) + 2] != 0) return;
    int last = range;
    while (last + 1 < p.num_ranges && st[3 * (last + 1)] == b && st[3 * (last + 1) + 1] == row_tile &&
           st[3 * (last + 1) + 2] != 0)
        ++last;
    const int64_t s0 = p.seqstarts[b], rows = (p.seqstarts[b + 1] - s0) * p.rep;
    const int64_t base = (int64_t)kvh * 2 * p.num_ranges;
    for (int x = blockIdx.y * 256 + threadIdx.x; x < ROWS * (DH / 4); x += 256 * gridDim.y) {
        const int r = x / (DH / 4), d = (x - r * (DH / 4)) * 4;
        const int64_t row = row_tile * ROWS + r;
        if (row >= rows || d >= p.view.head_dim) continue;
        float m = -INFINITY, l = 0.f;
        float4_t a = {0.f, 0.f, 0.f, 0.f};
        for (int k = range - 1; k <= last; ++k) {
            const int64_t at = (base + (k < range ? 2 * k + 1 : 2 * k)) * ROWS + r;
            const float2 ml = p.part_ml[at];
            const float4_t v = *reinterpret_cast<const float4_t*>(p.part_o + at * DH + d);
            const float m_new = fmaxf(m, ml.x);
            const float m_safe = m_new == -INFINITY ? 0.f : m_new;
            const float fo = __builtin_amdgcn_exp2f(m - m_safe), fn = __builtin_amdgcn_exp2f(ml.x - m_safe);
            l = l * fo + ml.y * fn;
            a = a * fo + v * fn;
            m = m_new;
        }
        const int64_t t = row / p.rep;
        const int64_t at = (s0 + t) * p.num_heads + kvh * p.rep + (row - t * p.rep);
        const float inv = l != 0.f ? 1.0f / l : 0.f;
        const half4_t r4 = {(half_t)(a[0] * inv), (half_t)(a[1] * inv), (half_t)(a[2] * inv), (half_t)(a[3] * inv)};
        *reinterpret_cast<half4_t*>(p.out + at * p.view.head_dim + d) = r4;
        if (p.lse && d == 0) p.lse[at] = l == 0.f ? -INFINITY : (m + (log2f(l) - kProbShift)) * 0.693147180559945f;
    }
}

// ---- host side

static int tree_row_blocks(const pplhip_tree_attention_args* a) {
    return a->max_seqlen * (a->num_heads / a->num_kv_heads) <= 16 ? 1 : 2;
}
int tree_row_tile(const pplhip_tree_attention_args* a) {
    return 16 * tree_row_blocks(a);
}
// As many ranges as workgroups are resident (two per CU), shared out among the kv heads; never more than ranges of the
// least length in the longest possible axis.
int64_t tree_num_ranges(const pplhip_tree_attention_args* a, int cu_count) {
    const int64_t rep = a->num_heads / a->num_kv_heads;
    const int64_t row_tiles = (a->max_seqlen * rep + tree_row_tile(a) - 1) / tree_row_tile(a);
    const int64_t key_tiles = (a->max_kvlen + kTileKeys - 1) / kTileKeys;
    int64_t ranges = (int64_t)cu_count * 2 / a->num_kv_heads;
    const double most = (double)a->batch * (double)row_tiles * (double)(key_tiles + kPieceCost) / kMinRangeTiles;
    if ((double)ranges > most) ranges = (int64_t)most + 1;
    return ranges < 1 ? 1 : ranges;
}

uint64_t tree_workspace_bytes(const pplhip_tree_attention_args* a, int64_t ranges) {
    const uint64_t rows = (uint64_t)a->num_kv_heads * 2 * (uint64_t)ranges * tree_row_tile(a);
    return rows * padded_head_dim(a->head_dim) * sizeof(float) + rows * sizeof(float2) + (uint64_t)ranges * 3 * sizeof(int64_t);
}

template <int DH>
static void launch_tree_dh(const TreeParams& p, int nr, hipStream_t stream) {
    const dim3 grid((unsigned)(p.num_ranges * p.kv_heads));
    const dim3 mgrid((unsigned)((p.num_ranges - 1) * p.kv_heads), (unsigned)(16 * nr * (DH / 4) / 256 > 0 ? 16 * nr * (DH / 4) / 256 : 1));
    if (nr == 1) {
        hipLaunchKernelGGL((tree_attention_kernel<DH, 1>), grid, dim3(256), 0, stream, p);
        if (p.num_ranges > 1) hipLaunchKernelGGL((tree_merge_kernel<DH, 1>), mgrid, dim3(256), 0, stream, p);
    } else {
        hipLaunchKernelGGL((tree_attention_kernel<DH, 2>), grid, dim3(256), 0, stream, p);
        if (p.num_ranges > 1) hipLaunchKernelGGL((tree_merge_kernel<DH, 2>), mgrid, dim3(256), 0, stream, p);
    }
}

pplhip_retcode launch_tree_attention(const pplhip_tree_attention_args* a, int64_t ranges, void* ws, hipStream_t stream) {
    TreeParams p;
    p.q = (const half_t*)a->d_query;
    p.mask = a->d_tree_mask;
    p.seqstarts = a->d_seqstarts;
    p.kvstarts = a->d_kvstarts;
    p.view = CacheView{(const int8_t*)a->d_cache, (const half_t*)a->d_scale, a->d_cachestarts, a->cachestart_stride_b,
                       CacheAddr{a->cache_stride_s, a->cache_stride_l, a->cache_stride_h, a->cache_stride_kv, a->layer_idx},
                       page_shift_of(a->cache_mode, a->page_size), a->head_dim};
    p.out = (half_t*)a->d_output;
    p.lse = (float*)a->d_lse;
    p.batch = (int32_t)a->batch;
    p.num_heads = a->num_heads;
    p.kv_heads = a->num_kv_heads;
    p.rep = a->num_heads / a->num_kv_heads;
    p.mask_words = a->tree_mask_words;
    p.num_ranges = (int32_t)ranges;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)a->head_dim));
    const int nr = tree_row_blocks(a);
    const uint64_t rows = (uint64_t)p.kv_heads * 2 * (uint64_t)ranges * 16 * nr;
    p.part_o = (float*)ws;
    p.part_ml = (float2*)(p.part_o + rows * padded_head_dim(a->head_dim));
    p.range_start = (int64_t*)(p.part_ml + rows);
    switch (padded_head_dim(a->head_dim)) {
        case 32: launch_tree_dh<32>(p, nr, stream); break;
        case 64: launch_tree_dh<64>(p, nr, stream); break;
        case 96: launch_tree_dh<96>(p, nr, stream); break;
        case 128: launch_tree_dh<128>(p, nr, stream); break;
        case 160: launch_tree_dh<160>(p, nr, stream); break;
        case 192: launch_tree_dh<192>(p, nr, stream); break;
        case 224: launch_tree_dh<224>(p, nr, stream); break;
        default: launch_tree_dh<256>(p, nr, stream); break;
    }
    PPLHIP_CHECK_LAUNCH("tree_attention");
    return PPLHIP_RC_SUCCESS;
}

} // namespace pplhip
