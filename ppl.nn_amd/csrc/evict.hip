// Moves of cached rows inside the slab: eviction by accumulated attention weight, and keeping the accepted path of a
// verified draft. Both are bound by the bytes of the rows they move; the choice of what to evict by reading the scores.
//
// Eviction. A sequence keeps K of its kvlen rows (per layer and kv head on its own). Only rows that stay but lie behind
// the first K places move, each into the place of a row in front that goes: as few row moves as possible, and sources
// (index >= K) and destinations (index < K) never overlap, so all of them run in parallel, in place.
//
// kv_evict_choose_kernel: one workgroup per (sequence, layer, kv head). It reads the scores and positions once, as sort keys
// into registers (up to 64 a thread), finds the K-th largest digit by digit (8 bits at a time, counts in LDS), then
// numbers, in index order, the holes and the rows that fill them.
// kv_evict_move_kernel: 16-byte pieces of the listed rows, K and V, with their scales. One row per thread at a time and many
// workgroups: two or four rows in flight per thread measured 53 - 61 us against 51 on the first batch below.
//
// Measured (KVH 8, head_dim 128): 16 sequences x 8 layers from 1 152 back to 1 024 tokens 49 us, 20 of them the choice, bound by
// its dependent steps; the moves 2.5 TB/s (128-byte rows and 32-byte scale rows at random places). Four sequences of
// 16 k - 64 k tokens cut to half 145 us: the choice runs on one workgroup for each of 32 columns (about 75 us), the moves
// at 3.2 TB/s.
#include "cache_tile.h"

namespace pplhip {

struct EvictParams {
    const int64_t* kvstarts;
    const int64_t* target;
    const int64_t* next_pos;
    PageMap pages;
    CacheAddr addr; // layer: the first one
    int8_t* cache;
    half_t* scale;
    const float* score_in;
    float* score_out;
    const int32_t* pos_in;
    int32_t* pos_out;
    int64_t score_stride_l, score_stride_h;
    int64_t* new_kvlen;
    int32_t num_sink, num_recent;
    int32_t layer_count, kv_heads, pieces; // pieces: 16-byte pieces of a row
    int32_t blocks_per_column;
    int32_t max_moves;
    int32_t* moves; // [columns]: rows to move
    int32_t* holes; // [columns][max_moves]: index of the j-th hole ..
    int32_t* fills; // .. and of the row that goes there
};

struct EvictColumn {
    int32_t b, layer, head;
    int64_t scores; // offset of the column in the score and position arrays
};
__device__ inline EvictColumn evict_column(const EvictParams& p, int column) {
    EvictColumn c;
    c.head = column % p.kv_heads;
    const int rest = column / p.kv_heads;
    c.layer = rest % p.layer_count;
    c.b = rest / p.layer_count;
    c.scores = (int64_t)(p.addr.layer + c.layer) * p.score_stride_l + (int64_t)c.head * p.score_stride_h;
    return c;
}

// Sort key of a token: larger stays. Protected tokens above everything, then the scores in their order, NaN lowest.
__device__ inline uint32_t evict_key(const EvictParams& p, float score, int32_t pos, int64_t next) {
    if (p.pos_in && (pos < p.num_sink || (p.num_recent > 0 && (int64_t)pos >= next - p.num_recent))) return 0xffffffffu;
    if (score != score) return 0;
    const uint32_t u = score == 0.f ? 0u : __float_as_uint(score); // (-0 counts as 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}

// set bits of a wave-wide mask at the lanes below this one
__device__ inline int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// A column's tokens in blocks of T * KEYS, wave w of the block its w-th stretch: 64 consecutive tokens per key register, so
// that loads are coalesced, index order is (block, wave, register, lane), and the 64 tokens lie in one page. A column of
// one block (T * KEYS covers it) is loaded once; a longer one anew for each of the six looks at it.
template <int T, int KEYS>
__global__ __launch_bounds__(T) void kv_evict_choose_kernel(const EvictParams p) {
    constexpr int WAVES = T / 64;
    // copies of the digit counts: scores share their leading bits, so lanes would queue at one counter; few keys do not
    // pay for clearing and adding up many
    constexpr int kHistCopies = T * KEYS > 4096 ? 16 : 4;
    constexpr int kBatch = 8; // tokens whose loads a thread has in flight
    __shared__ uint32_t hist[256 * kHistCopies];
    __shared__ uint32_t wave_sum[4];
    __shared__ uint32_t found[2]; // digit, rows above it
    __shared__ int32_t seg_gt[WAVES], seg_eq[WAVES];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const EvictColumn col = evict_column(p, blockIdx.x);
    const int64_t kvlen64 = p.kvstarts[col.b + 1] - p.kvstarts[col.b];
    const int64_t want = p.target[col.b] < 0 ? 0 : p.target[col.b];
    const int n = (int)kvlen64;
    const int keep = want < kvlen64 ? (int)want : n;
    const int64_t next = p.next_pos ? p.next_pos[col.b] : 0;
    if (col.layer == 0 && col.head == 0 && tid == 0) p.new_kvlen[col.b] = keep;
    const bool copy_score = p.score_out != p.score_in, copy_pos = p.pos_in && p.pos_out != p.pos_in;
    if (keep == n || keep == 0) { // nothing moves
        if (tid == 0) p.moves[blockIdx.x] = 0;
        if (copy_score || copy_pos)
            for (int j = tid; j < keep; j += T) {
                const int64_t at = col.scores + p.pages.token(col.b, j);
                if (copy_score) p.score_out[at] = p.score_in[at];
                if (copy_pos) p.pos_out[at] = p.pos_in[at];
            }
        return;
    }
    const int blocks = (n + T * KEYS - 1) / (T * KEYS);
    const int regs = blocks > 1 ? KEYS : (n + T - 1) / T; // registers in use
    uint32_t key[KEYS];
    // first token of the wave's register k in a block
    auto first_of = [&](int block, int k) { return block * (T * KEYS) + (wave * regs + k) * 64; };
    auto load = [&](int block) {
#pragma unroll
        for (int k0 = 0; k0 < KEYS; k0 += kBatch) {
            float score[kBatch];
            int32_t pos[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int j = first_of(block, k0 + k);
                score[k] = NAN; // past the end: the smallest key, behind all others of its kind
                pos[k] = p.num_sink;
                if (k0 + k < regs && j + lane < n) {
                    const int64_t at = col.scores + uniform_token(p.pages, col.b, j) + lane;
                    score[k] = p.score_in[at];
                    if (p.pos_in) pos[k] = p.pos_in[at];
                }
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                key[k0 + k] = first_of(block, k0 + k) + lane < n ? evict_key(p, score[k], pos[k], next) : 0u;
        }
    };
    if (blocks == 1) load(0);

    // ---- the keep-th largest key: `prefix` collects its digits, `remain` counts rows still to be found below them
    uint32_t prefix = 0;
    uint32_t remain = (uint32_t)keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256 * kHistCopies; i += T) hist[i] = 0;
        __syncthreads();
        for (int block = 0; block < blocks; ++block) {
            if (blocks > 1) load(block);
#pragma unroll
            for (int k = 0; k < KEYS; ++k)
                if (k < regs && (shift == 24 || (key[k] >> (shift + 8)) == (prefix >> (shift + 8))))
                    atomicAdd(&hist[((key[k] >> shift) & 255) * kHistCopies + (lane & (kHistCopies - 1))], 1u);
        }
        __syncthreads();
        uint32_t mine = 0, incl = 0;
        if (tid < 256) { // thread i: digit 255 - i, so that the running sum counts from the largest digit down
#pragma unroll
            for (int c = 0; c < kHistCopies; ++c) mine += hist[(255 - tid) * kHistCopies + ((c + tid) & (kHistCopies - 1))];
            incl = mine;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(incl, d);
                if (lane >= d) incl += up;
            }
            if (lane == 63) wave_sum[wave] = incl;
        }
        __syncthreads();
        if (tid < 256) {
            for (int w = 0; w < wave; ++w) incl += wave_sum[w];
            if (incl >= remain && incl - mine < remain) {
                found[0] = 255 - tid;
                found[1] = incl - mine;
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        remain -= found[1];
    }
    const int need_equal = (int)remain; // rows with exactly this key that stay: the first ones

    // ---- in index order: every wave counts its stretch, then numbers the rows in it
    int32_t* const holes = p.holes + (int64_t)blockIdx.x * p.max_moves;
    int32_t* const fills = p.fills + (int64_t)blockIdx.x * p.max_moves;
    int gt_before = 0, eq_before = 0; // of the blocks before
    for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load(block);
        int gt = 0, eq = 0;
#pragma unroll
        for (int k = 0; k < KEYS; ++k)
            if (k < regs) {
                gt += __popcll(__ballot(key[k] > prefix));
                eq += __popcll(__ballot(key[k] == prefix));
            }
        __syncthreads();
        if (lane == 0) {
            seg_gt[wave] = gt;
            seg_eq[wave] = eq;
        }
        __syncthreads();
        uint64_t in_place = 0; // bit k: this lane's token of register k stays where it is
        int g_run = gt_before, e_run = eq_before;
        for (int w = 0; w < WAVES; ++w) {
            gt_before += seg_gt[w];
            eq_before += seg_eq[w];
            if (w < wave) {
                g_run += seg_gt[w];
                e_run += seg_eq[w];
            }
        }
#pragma unroll
        for (int k = 0; k < KEYS; ++k)
            if (k < regs) {
                const int j = first_of(block, k), i = j + lane;
                const uint64_t gts = __ballot(key[k] > prefix), eqs = __ballot(key[k] == prefix);
                const int g0 = g_run + lanes_below(gts), e0 = e_run + lanes_below(eqs);
                const int kept_before = g0 + (e0 < need_equal ? e0 : need_equal);
                const bool stays = key[k] > prefix || (key[k] == prefix && e0 < need_equal); // (never past the end)
                if (i < keep && !stays) holes[i - kept_before] = i;
                if (stays && i >= keep) fills[keep - 1 - kept_before] = i;
                if (i == keep - 1) p.moves[blockIdx.x] = keep - kept_before - (stays ? 1 : 0);
                if (stays && i < keep) in_place |= uint64_t(1) << k;
                g_run += __popcll(gts);
                e_run += __popcll(eqs);
            }
        if (copy_score || copy_pos) {
            for (int k0 = 0; k0 < KEYS; k0 += kBatch) {
                float score[kBatch];
                int32_t pos[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if ((in_place >> (k0 + k)) & 1) {
                        const int64_t at = col.scores + uniform_token(p.pages, col.b, first_of(block, k0 + k)) + lane;
                        score[k] = p.score_in[at];
                        if (p.pos_in) pos[k] = p.pos_in[at];
                    }
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if ((in_place >> (k0 + k)) & 1) {
                        const int64_t at = col.scores + uniform_token(p.pages, col.b, first_of(block, k0 + k)) + lane;
                        if (copy_score) p.score_out[at] = score[k];
                        if (copy_pos) p.pos_out[at] = pos[k];
                    }
            }
        }
    }
}

__global__ __launch_bounds__(256) void kv_evict_move_kernel(const EvictParams p) {
    const int column = blockIdx.x / p.blocks_per_column;
    const int block = blockIdx.x - column * p.blocks_per_column;
    const EvictColumn col = evict_column(p, column);
    const int32_t* const holes = p.holes + (int64_t)column * p.max_moves;
    const int32_t* const fills = p.fills + (int64_t)column * p.max_moves;
    CacheAddr addr = p.addr;
    addr.layer += col.layer;
    // a thread keeps one piece of K or V and goes from row to row
    const int per_row = 2 * p.pieces; // at most 32
    const int rows_per_pass = 256 / per_row;
    const int slot = threadIdx.x / per_row, r = threadIdx.x - slot * per_row;
    if (slot >= rows_per_pass) return;
    const int kv = r >= p.pieces, piece = r - kv * p.pieces;
    const int count = p.moves[column], step = p.blocks_per_column * rows_per_pass;
    const int64_t at0 = addr.row(0, kv, col.head) + 16 * piece;
    for (int64_t m = (int64_t)block * rows_per_pass + slot; m < count; m += step) {
        const int64_t to = p.pages.token(col.b, holes[m]), from = p.pages.token(col.b, fills[m]);
        const int64_t src = at0 + from * addr.stride_s, dst = at0 + to * addr.stride_s;
        const uint4_vt q = *reinterpret_cast<const uint4_vt*>(p.cache + src);
        const uint32_t s = *reinterpret_cast<const uint32_t*>(p.scale + src / kQuantGroup);
        __builtin_nontemporal_store(q, reinterpret_cast<uint4_vt*>(p.cache + dst)); // (not read again by this call)
        *reinterpret_cast<uint32_t*>(p.scale + dst / kQuantGroup) = s;
        if (r == 0) {
            p.score_out[col.scores + to] = p.score_in[col.scores + from];
            if (p.pos_in) p.pos_out[col.scores + to] = p.pos_in[col.scores + from];
        }
    }
}

int64_t evict_columns(const pplhip_kv_evict_args* a) {
    return a->batch * a->layer_count * a->num_kv_heads;
}
uint64_t evict_workspace_bytes(const pplhip_kv_evict_args* a, int64_t max_moves) {
    return (uint64_t)evict_columns(a) * (1 + 2 * (uint64_t)max_moves) * sizeof(int32_t);
}

pplhip_retcode launch_kv_evict(const pplhip_kv_evict_args* a, int64_t max_moves, void* ws, hipStream_t stream) {
    EvictParams p;
    p.kvstarts = a->d_kvstarts;
    p.target = a->d_target_kvlen;
    p.next_pos = a->num_recent > 0 ? a->d_next_pos : nullptr;
    p.pages = PageMap{a->d_cachestarts, a->cachestart_stride_b, page_shift_of(a->cache_mode, a->page_size)};
    p.addr = CacheAddr{a->cache_stride_s, a->cache_stride_l, a->cache_stride_h, a->cache_stride_kv, a->layer_idx};
    p.cache = (int8_t*)a->d_cache;
    p.scale = (half_t*)a->d_scale;
    p.score_in = a->d_score_in;
    p.score_out = a->d_score_out;
    p.pos_in = a->d_position_in;
    p.pos_out = a->d_position_out;
    p.score_stride_l = a->score_stride_l;
    p.score_stride_h = a->score_stride_h;
    p.new_kvlen = a->d_new_kvlen;
    p.num_sink = a->num_sink;
    p.num_recent = a->num_recent;
    p.layer_count = a->layer_count;
    p.kv_heads = a->num_kv_heads;
    p.pieces = a->head_dim / 16;
    const int64_t columns = evict_columns(a);
    p.max_moves = (int32_t)max_moves;
    p.moves = (int32_t*)ws;
    p.holes = p.moves + columns;
    p.fills = p.holes + columns * max_moves;
    // A column's keys fit the registers of the smallest workgroup that holds them, so that many short columns run side by
    // side (1 024 columns of 1 152 tokens: 54 us in all with 256 threads each, 58 with 512); long ones get all the threads.
    const dim3 cols((unsigned)columns);
    if (a->max_kvlen <= 256 * 16)
        hipLaunchKernelGGL((kv_evict_choose_kernel<256, 16>), cols, dim3(256), 0, stream, p);
    else if (a->max_kvlen <= 1024 * 16)
        hipLaunchKernelGGL((kv_evict_choose_kernel<1024, 16>), cols, dim3(1024), 0, stream, p);
    else
        hipLaunchKernelGGL((kv_evict_choose_kernel<1024, 64>), cols, dim3(1024), 0, stream, p);
    PPLHIP_CHECK_LAUNCH("kv_evict choose");
    // how many rows move is known on the device only: enough workgroups to fill the chip a few times over, each of which
    // walks its share of the column's list
    const int64_t rows_per_pass = 256 / (2 * p.pieces);
    const int64_t most = (max_moves + rows_per_pass - 1) / rows_per_pass;
    int64_t per_column = (8192 + columns - 1) / columns;
    if (per_column > most) per_column = most;
    if (per_column < 1) per_column = 1;
    p.blocks_per_column = (int32_t)per_column;
    if (max_moves > 0) {
        hipLaunchKernelGGL(kv_evict_move_kernel, dim3((unsigned)(columns * per_column)), dim3(256), 0, stream, p);
        PPLHIP_CHECK_LAUNCH("kv_evict move");
    }
    return PPLHIP_RC_SUCCESS;
}

// ---- accepted drafted tokens
//
// Row start + i becomes what row start + path[i] was; path is ascending, so path[i] >= i. A thread owns one 16-byte piece
// of (layer, K or V, head) and takes the whole path through it, eight rows loaded before eight are stored: a stored
// place (below 8 k + 8) is never a later batch's source (path[i] >= i >= 8 k + 8), and no other thread touches the piece.
// 64 sequences with up to 6 accepted tokens, 16 layers, KVH 8, head_dim 128: 6.7 us; one sequence, 32 layers: 6.2 us; both
// are the launch and three dependent loads.
struct AcceptParams {
    const int64_t* seqstarts;
    const int64_t* start_pos;
    const int64_t* accepted;
    const int64_t* accepted_len;
    int64_t accepted_stride_b, max_accepted;
    PageMap pages;
    CacheAddr addr;
    int8_t* cache;
    half_t* scale;
    int32_t layer_count, kv_heads, pieces;
    int32_t blocks_per_seq;
};

__global__ __launch_bounds__(256) void kv_accept_kernel(const AcceptParams p) {
    constexpr int kRows = 8;
    const int b = blockIdx.x / p.blocks_per_seq;
    const int64_t unit = (int64_t)(blockIdx.x - b * p.blocks_per_seq) * 256 + threadIdx.x;
    const int piece = (int)(unit % p.pieces);
    const int64_t rest = unit / p.pieces;
    const int head = (int)(rest % p.kv_heads);
    const int64_t rest2 = rest / p.kv_heads;
    const int kv = (int)(rest2 & 1);
    const int64_t layer = rest2 >> 1;
    if (layer >= p.layer_count) return;
    CacheAddr addr = p.addr;
    addr.layer += (int32_t)layer;
    const int64_t drafted = p.seqstarts[b + 1] - p.seqstarts[b];
    const int64_t start = p.start_pos[b];
    const int64_t* const path = p.accepted + b * p.accepted_stride_b;
    int64_t n = p.accepted_len[b];
    if (n > p.max_accepted) n = p.max_accepted;
    int64_t prev = -1;
    for (int64_t i0 = 0; i0 < n; i0 += kRows) {
        int64_t from[kRows];
        uint4_vt q[kRows];
        uint32_t s[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) from[i] = i0 + i < n ? path[i0 + i] : -1;
        int rows = 0; // entries of the batch before the list's end
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (rows == i && from[i] > prev && from[i] < drafted) {
                prev = from[i];
                rows = i + 1;
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i < rows && from[i] != i0 + i) {
                const int64_t row = addr.row(p.pages.token(b, start + from[i]), kv, head) + 16 * piece;
                q[i] = *reinterpret_cast<const uint4_vt*>(p.cache + row);
                s[i] = *reinterpret_cast<const uint32_t*>(p.scale + row / kQuantGroup);
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i < rows && from[i] != i0 + i) {
                const int64_t row = addr.row(p.pages.token(b, start + i0 + i), kv, head) + 16 * piece;
                *reinterpret_cast<uint4_vt*>(p.cache + row) = q[i];
                *reinterpret_cast<uint32_t*>(p.scale + row / kQuantGroup) = s[i];
            }
        }
        if (rows < kRows) break;
    }
}

pplhip_retcode launch_kv_accept(const pplhip_kv_accept_args* a, hipStream_t stream) {
    AcceptParams p;
    p.seqstarts = a->d_seqstarts;
    p.start_pos = a->d_start_pos;
    p.accepted = a->d_accepted;
    p.accepted_len = a->d_accepted_len;
    p.accepted_stride_b = a->accepted_stride_b;
    p.max_accepted = a->max_accepted;
    p.pages = PageMap{a->d_cachestarts, a->cachestart_stride_b, page_shift_of(a->cache_mode, a->page_size)};
    p.addr = CacheAddr{a->cache_stride_s, a->cache_stride_l, a->cache_stride_h, a->cache_stride_kv, a->layer_idx};
    p.cache = (int8_t*)a->d_cache;
    p.scale = (half_t*)a->d_scale;
    p.layer_count = a->layer_count;
    p.kv_heads = a->num_kv_heads;
    p.pieces = a->head_dim / 16;
    const int64_t units = (int64_t)a->layer_count * 2 * a->num_kv_heads * p.pieces;
    const int64_t per_seq = (units + 255) / 256;
    if (per_seq * a->batch > 0x7fffffffLL) PPLHIP_FAIL(PPLHIP_RC_OUT_OF_RANGE, "kv_accept: too many rows");
    p.blocks_per_seq = (int32_t)per_seq;
    hipLaunchKernelGGL(kv_accept_kernel, dim3((unsigned)(per_seq * a->batch)), dim3(256), 0, stream, p);
    PPLHIP_CHECK_LAUNCH("kv_accept");
    return PPLHIP_RC_SUCCESS;
}

} // namespace pplhip
