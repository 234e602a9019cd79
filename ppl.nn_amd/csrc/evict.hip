// Moves of cached rows inside the slab: eviction by accumulated attention weight, and keeping the accepted path of a
// verified draft. Both are bound by the bytes of the rows they move; the choice of what to evict by reading the scores.
//
// Eviction. A sequence keeps K of its kvlen rows (per layer and kv head on its own). Only rows that stay but lie behind
// the first K places move, each into the place of a row in front that goes: as few row moves as possible, and sources
// (index >= K) and destinations (index < K) never overlap, so all of them run in parallel, in place.
//
// The choice: scores and positions are read once, as sort keys; the K-th largest is found digit by digit (8 bits at a time,
// counts in LDS); then the holes and the rows that fill them are numbered in index order. kv_evict_choose_kernel does it
// with one workgroup per (sequence, layer, kv head), keys in registers (up to 64 a thread); kv_evict_digit_kernel and
// kv_evict_number_kernel with several, where columns are long and few, or too long for registers.
// kv_evict_move_kernel: 16-byte pieces of the listed rows, K and V, with their scales. One row per thread at a time and many
// workgroups: two or four rows in flight per thread measured 53 - 61 us against 51 on the first batch below.
//
// Measured (KVH 8, head_dim 128): 16 sequences x 8 layers from 1 152 back to 1 024 tokens 47 us, 18 of them the choice, bound
// by its dependent steps; the moves 2.5 TB/s (128-byte rows and 32-byte scale rows at random places). Four sequences of
// 16 k - 64 k tokens cut to half, one layer: 110 us, 45 of them the choice, mostly its five launches, each a chain of
// dependent loads (one workgroup for each of the 32 columns: 141); the moves at 3.2 TB/s.
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
    int32_t max_kvlen, max_moves;
    int32_t* moves; // [columns]: rows to move
    int32_t* holes; // [columns][max_moves]: index of the j-th hole ..
    int32_t* fills; // .. and of the row that goes there
    // a column's parts, where several workgroups choose
    int32_t columns, parts, part_blocks;
    uint4_vt* keys; // [columns][parts * part_blocks][blocks' keys]
    uint32_t* state; // [columns][8]
    uint32_t* counts; // [2][columns][parts][256]: thread order, largest digit first
    int32_t* above; // [columns][parts]
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
// that loads are coalesced, index order is (block, wave, register, lane), and the 64 tokens lie in one page.
template <int T, int KEYS>
struct ColumnKeys {
    static constexpr int WAVES = T / 64;
    // copies of the digit counts: scores share their leading bits, so lanes would queue at one counter; few keys do not
    // pay for clearing and adding up many
    static constexpr int kHistCopies = T * KEYS > 4096 ? 16 : 4;
    static constexpr int kBatch = 8; // tokens whose loads a thread has in flight
    struct Shared {
        uint32_t hist[256 * kHistCopies];
        uint32_t wave_sum[4];
        uint32_t found[2]; // digit, rows above it
        int32_t seg_gt[WAVES], seg_eq[WAVES];
    };

    const EvictParams& p;
    Shared& sh;
    EvictColumn col;
    int tid, lane, wave;
    int n, keep; // tokens, tokens that stay
    int64_t next;
    bool copy_score, copy_pos;
    int regs; // registers in use
    uint32_t key[KEYS];

    __device__ inline ColumnKeys(const EvictParams& p_, Shared& sh_, int column) : p(p_), sh(sh_) {
        tid = threadIdx.x;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        col = evict_column(p, column);
        int64_t kvlen = p.kvstarts[col.b + 1] - p.kvstarts[col.b];
        if (kvlen > p.max_kvlen) kvlen = p.max_kvlen; // (the lists have no place for more)
        const int64_t want = p.target[col.b] < 0 ? 0 : p.target[col.b];
        n = (int)kvlen;
        keep = want < kvlen ? (int)want : n;
        next = p.next_pos ? p.next_pos[col.b] : 0;
        copy_score = p.score_out != p.score_in;
        copy_pos = p.pos_in && p.pos_out != p.pos_in;
        regs = KEYS;
    }
    __device__ inline bool nothing_moves() const { return keep == n || keep == 0; }

    // first token of the wave's register k in a block
    // (unsigned: in the last block of the longest columns it passes 31 bits)
    __device__ inline uint32_t first_of(int block, int k) const {
        return (uint32_t)block * (T * KEYS) + (uint32_t)((wave * regs + k) * 64);
    }
    __device__ inline int blocks() const { return (int)(((uint32_t)n + T * KEYS - 1) / (T * KEYS)); }

    __device__ inline void load(int block) {
#pragma unroll
        for (int k0 = 0; k0 < KEYS; k0 += kBatch) {
            float score[kBatch];
            int32_t pos[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const uint32_t j = first_of(block, k0 + k);
                score[k] = NAN; // past the end: the smallest key, behind all others of its kind
                pos[k] = p.num_sink;
                if (k0 + k < regs && j + lane < (uint32_t)n) {
                    const int64_t at = col.scores + uniform_token(p.pages, col.b, j) + lane;
                    score[k] = p.score_in[at];
                    if (p.pos_in) pos[k] = p.pos_in[at];
                }
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                key[k0 + k] = first_of(block, k0 + k) + lane < (uint32_t)n ? evict_key(p, score[k], pos[k], next) : 0u;
        }
    }

    // ---- digit counts of the keys that agree with `prefix` above the digit
    __device__ inline void clear_counts() {
        for (int i = tid; i < 256 * kHistCopies; i += T) sh.hist[i] = 0;
        __syncthreads();
    }
    __device__ inline void count(int shift, uint32_t prefix) {
#pragma unroll
        for (int k = 0; k < KEYS; ++k)
            if (k < regs && (shift == 24 || (key[k] >> (shift + 8)) == (prefix >> (shift + 8))))
                atomicAdd(&sh.hist[((key[k] >> shift) & 255) * kHistCopies + (lane & (kHistCopies - 1))], 1u);
    }
    // thread i < 256: keys with digit 255 - i, so that running sums count from the largest digit down
    __device__ inline uint32_t counted() const {
        uint32_t mine = 0;
#pragma unroll
        for (int c = 0; c < kHistCopies; ++c) mine += sh.hist[(255 - tid) * kHistCopies + ((c + tid) & (kHistCopies - 1))];
        return mine;
    }
    // The digit in which the remain-th largest lies, from the counts (`mine`: as above; other threads: anything): it joins
    // `prefix`, and `remain` counts the rows still to be found below the keys above it.
    __device__ inline void pick(uint32_t mine, int shift, uint32_t& prefix, uint32_t& remain) {
        uint32_t incl = mine;
        if (tid < 256) {
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(incl, d);
                if (lane >= d) incl += up;
            }
            if (lane == 63) sh.wave_sum[wave] = incl;
        }
        __syncthreads();
        if (tid < 256) {
            for (int w = 0; w < wave; ++w) incl += sh.wave_sum[w];
            if (incl >= remain && incl - mine < remain) {
                sh.found[0] = 255 - tid;
                sh.found[1] = incl - mine;
            }
        }
        __syncthreads();
        prefix |= (uint32_t)__builtin_amdgcn_readfirstlane(sh.found[0]) << shift;
        remain -= (uint32_t)__builtin_amdgcn_readfirstlane(sh.found[1]);
    }

    // ---- in index order: every wave counts its stretch of a block, then numbers the rows in it. need_equal: rows with key
    // `prefix` that stay, the first ones; gt_before, eq_before: rows above and at `prefix` in the blocks before
    __device__ inline void number(int column, int block, uint32_t prefix, int need_equal, int& gt_before, int& eq_before) {
        int32_t* const holes = p.holes + (int64_t)column * p.max_moves;
        int32_t* const fills = p.fills + (int64_t)column * p.max_moves;
        // (said to change here and below: token numbers and ballots of all registers would be kept from one use to the next,
        // in more registers than there are)
        asm volatile("" : "+v"(lane), "+s"(regs));
        int gt = 0, eq = 0;
#pragma unroll
        for (int k = 0; k < KEYS; ++k)
            if (k < regs) {
                gt += __popcll(__ballot(key[k] > prefix));
                eq += __popcll(__ballot(key[k] == prefix));
            }
        __syncthreads();
        if (lane == 0) {
            sh.seg_gt[wave] = gt;
            sh.seg_eq[wave] = eq;
        }
        __syncthreads();
        asm volatile("" : "+v"(lane), "+s"(regs), "+s"(prefix));
        uint64_t in_place = 0; // bit k: this lane's token of register k stays where it is
        int g_run = gt_before, e_run = eq_before;
        for (int w = 0; w < WAVES; ++w) {
            gt_before += sh.seg_gt[w];
            eq_before += sh.seg_eq[w];
            if (w < wave) {
                g_run += sh.seg_gt[w];
                e_run += sh.seg_eq[w];
            }
        }
#pragma unroll
        for (int k = 0; k < KEYS; ++k)
            if (k < regs) {
                const uint32_t i = first_of(block, k) + lane;
                const uint64_t gts = __ballot(key[k] > prefix), eqs = __ballot(key[k] == prefix);
                const int g0 = g_run + lanes_below(gts), e0 = e_run + lanes_below(eqs);
                const int kept_before = g0 + (e0 < need_equal ? e0 : need_equal);
                const bool stays = key[k] > prefix || (key[k] == prefix && e0 < need_equal); // (never past the end)
                const bool front = i < (uint32_t)keep;
                if (front && !stays) holes[i - kept_before] = (int32_t)i;
                if (stays && !front) fills[keep - 1 - kept_before] = (int32_t)i;
                if (i == (uint32_t)keep - 1) p.moves[column] = keep - kept_before - (stays ? 1 : 0);
                if (stays && front) in_place |= uint64_t(1) << k;
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

    // a column in which nothing moves: scores and positions of tokens first .. end - 1 go to the out arrays
    __device__ inline void copy_kept(int64_t first, int64_t end) {
        if (copy_score || copy_pos)
            for (int64_t j = first + tid; j < end; j += T) {
                const int64_t at = col.scores + p.pages.token(col.b, j);
                if (copy_score) p.score_out[at] = p.score_in[at];
                if (copy_pos) p.pos_out[at] = p.pos_in[at];
            }
    }
};

// One workgroup per column, whose keys fit its registers (T * KEYS of them).
template <int T, int KEYS>
__global__ __launch_bounds__(T) void kv_evict_choose_kernel(const EvictParams p) {
    typedef ColumnKeys<T, KEYS> Keys;
    __shared__ typename Keys::Shared sh;
    Keys c(p, sh, blockIdx.x);
    if (c.col.layer == 0 && c.col.head == 0 && c.tid == 0) p.new_kvlen[c.col.b] = c.keep;
    if (c.nothing_moves()) {
        if (c.tid == 0) p.moves[blockIdx.x] = 0;
        c.copy_kept(0, c.keep);
        return;
    }
    c.regs = (c.n + T - 1) / T;
    c.load(0);
    uint32_t prefix = 0, remain = (uint32_t)c.keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
        c.clear_counts();
        c.count(shift, prefix);
        __syncthreads();
        c.pick(c.tid < 256 ? c.counted() : 0u, shift, prefix, remain);
    }
    int gt_before = 0, eq_before = 0;
    c.number(blockIdx.x, 0, prefix, (int)remain, gt_before, eq_before);
}

// Several workgroups per column, kEvictParts or fewer, each with a part of its tokens: a launch per digit, in which every
// workgroup adds up all parts' counts of the digit before (the same sums everywhere), and one that numbers the rows. The
// first launch leaves the keys in the workspace: reading scores and positions again in each of the five costs 126 us against
// 112 on those prompts.
typedef ColumnKeys<256, 16> PartKeys;
constexpr int kPartBlock = 256 * 16; // tokens per block of a part

// A block's keys as the first digit's launch leaves them for the others: four registers of a thread side by side.
__device__ inline uint4_vt* block_keys(const EvictParams& p, int column, int block) {
    return p.keys + ((int64_t)column * p.parts * p.part_blocks + block) * (kPartBlock / 4) + threadIdx.x;
}
__device__ inline void store_keys(const EvictParams& p, int column, int block, const uint32_t (&key)[16]) {
    uint4_vt* const to = block_keys(p, column, block);
#pragma unroll
    for (int k = 0; k < 4; ++k) to[k * 256] = uint4_vt{key[4 * k], key[4 * k + 1], key[4 * k + 2], key[4 * k + 3]};
}
__device__ inline void load_keys(const EvictParams& p, int column, int block, uint32_t (&key)[16]) {
    const uint4_vt* const from = block_keys(p, column, block);
    uint4_vt v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = from[k * 256];
#pragma unroll
    for (int k = 0; k < 16; ++k) key[k] = v[k / 4][k % 4];
}

__device__ inline uint32_t* part_counts(const EvictParams& p, int digit, int column) {
    return p.counts + ((int64_t)(digit & 1) * p.columns + column) * p.parts * 256; // (read one launch later only)
}

template <int DIGIT>
__global__ __launch_bounds__(256) void kv_evict_digit_kernel(const EvictParams p) {
    __shared__ PartKeys::Shared sh;
    const int column = blockIdx.x / p.parts, part = blockIdx.x - column * p.parts;
    PartKeys c(p, sh, column);
    const int blocks = c.n > 0 ? c.blocks() : 0;
    const int first = part * p.part_blocks, end = first + p.part_blocks < blocks ? first + p.part_blocks : blocks;
    if (c.nothing_moves() || first >= end) return;
    if (DIGIT > 0) load_keys(p, column, first, c.key);
    uint32_t* const state = p.state + (int64_t)column * 8; // prefix and remain in front of each digit
    uint32_t prefix = 0, remain = (uint32_t)c.keep;
    c.clear_counts();
    if (DIGIT > 0) {
        if (DIGIT > 1) {
            prefix = state[2 * DIGIT - 2];
            remain = state[2 * DIGIT - 1];
        }
        const uint32_t* const counts = part_counts(p, DIGIT - 1, column) + c.tid;
        const int parts = (blocks + p.part_blocks - 1) / p.part_blocks;
        uint32_t mine = 0;
#pragma unroll 8
        for (int q = 0; q < parts; ++q) mine += counts[q * 256];
        c.pick(mine, 32 - 8 * DIGIT, prefix, remain);
        if (part == 0 && c.tid == 0) {
            state[2 * DIGIT] = prefix;
            state[2 * DIGIT + 1] = remain;
        }
    }
    const int shift = 24 - 8 * DIGIT;
    int above = 0; // keys above the prefix of the three digits before the last
    for (int block = first; block < end; ++block) {
        if (DIGIT == 0) {
            c.load(block);
            store_keys(p, column, block, c.key);
        } else if (block > first) {
            load_keys(p, column, block, c.key);
        }
        c.count(shift, prefix);
        if (DIGIT == 3)
#pragma unroll
            for (int k = 0; k < 16; ++k) above += __popcll(__ballot((c.key[k] >> 8) > (prefix >> 8)));
    }
    if (DIGIT == 3 && c.lane == 0) sh.seg_gt[c.wave] = above;
    __syncthreads();
    part_counts(p, DIGIT, column)[part * 256 + c.tid] = c.counted();
    if (DIGIT == 3 && c.tid == 0)
        p.above[(int64_t)column * p.parts + part] = sh.seg_gt[0] + sh.seg_gt[1] + sh.seg_gt[2] + sh.seg_gt[3];
}

__global__ __launch_bounds__(256) void kv_evict_number_kernel(const EvictParams p) {
    __shared__ PartKeys::Shared sh;
    __shared__ int32_t before[2]; // rows above and at the last staying key in the parts before
    const int column = blockIdx.x / p.parts, part = blockIdx.x - column * p.parts;
    PartKeys c(p, sh, column);
    const int blocks = c.n > 0 ? c.blocks() : 0;
    const int first = part * p.part_blocks, end = first + p.part_blocks < blocks ? first + p.part_blocks : blocks;
    if (c.col.layer == 0 && c.col.head == 0 && part == 0 && c.tid == 0) p.new_kvlen[c.col.b] = c.keep;
    if (c.nothing_moves()) {
        if (part == 0 && c.tid == 0) p.moves[column] = 0;
        const int64_t stop = (int64_t)end * kPartBlock;
        if (first < end) c.copy_kept((int64_t)first * kPartBlock, stop < c.keep ? stop : c.keep);
        return;
    }
    if (first >= end) return;
    load_keys(p, column, first, c.key);
    if (c.tid < 2) before[c.tid] = 0;
    uint32_t prefix = p.state[(int64_t)column * 8 + 6], remain = p.state[(int64_t)column * 8 + 7];
    const uint32_t* const counts = part_counts(p, 3, column) + c.tid;
    const int parts = (blocks + p.part_blocks - 1) / p.part_blocks;
    uint32_t mine = 0, earlier = 0;
#pragma unroll 8
    for (int q = 0; q < parts; ++q) {
        const uint32_t v = counts[q * 256];
        mine += v;
        earlier += q < part ? v : 0u;
    }
    c.pick(mine, 0, prefix, remain);
    const int digit = prefix & 255;
    int gt = 255 - c.tid > digit ? (int)earlier : 0;
    if (c.tid < part) gt += p.above[(int64_t)column * p.parts + c.tid];
    if (gt) atomicAdd(&before[0], gt);
    if (255 - c.tid == digit) before[1] = (int)earlier;
    __syncthreads();
    int gt_before = before[0], eq_before = before[1];
    for (int block = first; block < end; ++block) {
        if (block > first) load_keys(p, column, block, c.key);
        c.number(column, block, prefix, (int)remain, gt_before, eq_before);
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
// Long columns are worth the five launches when there are few of them, and always once a workgroup's registers cannot hold
// one. Choice and a few moves, us, one workgroup per column / several:
//   columns          1        32        64       128       256
//   16 384 tokens  22 / 30   26 / 36   28 / 39   33 / 47   41 / 65
//   32 768         48 / 30   53 / 35   55 / 42   59 / 56   69 / 90
//   65 536         64 / 31   70 / 42   73 / 55   76 / 86   87 / 140
// (131 072 tokens read anew for every digit by one workgroup each: 242 / 35 one column, 306 / 257 with 256.)
constexpr int64_t kEvictSplitAbove = 16384, kEvictRegisterKeys = 65536, kEvictSplitColumns = 96;
static bool evict_split(int64_t max_kvlen, double columns) {
    return max_kvlen > kEvictRegisterKeys || (max_kvlen > kEvictSplitAbove && columns <= (double)kEvictSplitColumns);
}
// Parts of a column: at most kEvictParts, of whole blocks.
constexpr int kEvictParts = 64;
int64_t evict_part_blocks(int64_t max_kvlen) {
    return (max_kvlen + (int64_t)kPartBlock * kEvictParts - 1) / ((int64_t)kPartBlock * kEvictParts);
}
int64_t evict_parts(int64_t max_kvlen) {
    const int64_t tokens = evict_part_blocks(max_kvlen) * kPartBlock;
    return tokens ? (max_kvlen + tokens - 1) / tokens : 0;
}
// the largest of a call's launches: the choice (the moves' has 256 threads a column, or few)
bool evict_launches_fit(const pplhip_kv_evict_args* a) {
    const double columns = (double)a->batch * a->layer_count * a->num_kv_heads;
    if (evict_split(a->max_kvlen, columns)) return launch_fits(columns * (double)evict_parts(a->max_kvlen), 256);
    return launch_fits(columns, a->max_kvlen > 256 * 16 ? 1024 : 256);
}
// (a plan for many columns holds what fewer of them take, which several workgroups share)
uint64_t evict_workspace_bytes(const pplhip_kv_evict_args* a, int64_t max_moves) {
    const uint64_t columns = (uint64_t)evict_columns(a), lists = 1 + 2 * (uint64_t)max_moves;
    uint64_t ints = columns * lists;
    if (a->max_kvlen > kEvictSplitAbove) {
        const uint64_t shared = evict_split(a->max_kvlen, (double)columns) ? columns : kEvictSplitColumns;
        const uint64_t each = lists + 8 + (uint64_t)evict_parts(a->max_kvlen) *
                                              (513 + kPartBlock * (uint64_t)evict_part_blocks(a->max_kvlen));
        if (shared * each > ints) ints = shared * each;
    }
    return ints * sizeof(int32_t);
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
    p.max_kvlen = (int32_t)a->max_kvlen;
    p.max_moves = (int32_t)max_moves;
    p.part_blocks = (int32_t)evict_part_blocks(a->max_kvlen);
    p.parts = (int32_t)evict_parts(a->max_kvlen);
    p.keys = (uint4_vt*)ws;
    const bool split = evict_split(a->max_kvlen, (double)columns);
    p.moves = (int32_t*)ws + (split ? columns * p.parts * p.part_blocks * kPartBlock : 0);
    p.holes = p.moves + columns;
    p.fills = p.holes + columns * max_moves;
    // A column's keys fit the registers of the smallest workgroup that holds them, so that many short columns run side by
    // side (1 024 columns of 1 152 tokens: 54 us in all with 256 threads each, 58 with 512); long ones get all the threads.
    const dim3 cols((unsigned)columns);
    p.columns = (int32_t)columns;
    if (split) {
        p.state = (uint32_t*)(p.fills + columns * max_moves);
        p.counts = p.state + columns * 8;
        p.above = (int32_t*)(p.counts + 2 * columns * p.parts * 256);
        const dim3 grid((unsigned)(columns * p.parts));
        hipLaunchKernelGGL(kv_evict_digit_kernel<0>, grid, dim3(256), 0, stream, p);
        hipLaunchKernelGGL(kv_evict_digit_kernel<1>, grid, dim3(256), 0, stream, p);
        hipLaunchKernelGGL(kv_evict_digit_kernel<2>, grid, dim3(256), 0, stream, p);
        hipLaunchKernelGGL(kv_evict_digit_kernel<3>, grid, dim3(256), 0, stream, p);
        hipLaunchKernelGGL(kv_evict_number_kernel, grid, dim3(256), 0, stream, p);
    } else if (a->max_kvlen <= 256 * 16) {
        hipLaunchKernelGGL((kv_evict_choose_kernel<256, 16>), cols, dim3(256), 0, stream, p);
    } else if (a->max_kvlen <= 1024 * 16) {
        hipLaunchKernelGGL((kv_evict_choose_kernel<1024, 16>), cols, dim3(1024), 0, stream, p);
    } else {
        hipLaunchKernelGGL((kv_evict_choose_kernel<1024, 64>), cols, dim3(1024), 0, stream, p);
    }
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
// are three dependent loads (the list's length, the list, the rows) and a store in one launch.
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
    // (in double first: the product can pass 64 bits)
    const double blocks = ceil((double)a->layer_count * 2.0 * a->num_kv_heads * p.pieces / 256.0) * (double)a->batch;
    if (!launch_fits(blocks, 256)) PPLHIP_FAIL(PPLHIP_RC_OUT_OF_RANGE, "kv_accept: too many rows");
    const int64_t units = (int64_t)a->layer_count * 2 * a->num_kv_heads * p.pieces;
    const int64_t per_seq = (units + 255) / 256;
    p.blocks_per_seq = (int32_t)per_seq;
    hipLaunchKernelGGL(kv_accept_kernel, dim3((unsigned)(per_seq * a->batch)), dim3(256), 0, stream, p);
    PPLHIP_CHECK_LAUNCH("kv_accept");
    return PPLHIP_RC_SUCCESS;
}

} // namespace pplhip
