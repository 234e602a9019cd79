// Accumulated attention weight of every cached token, per kv head: score[j] += sum over the new tokens t and the kv head's
// query heads h of exp(q_th . k_j / sqrt(D) - lse[t][h]).
//
// With the rows' log-sums known the weights need no second look at the keys: one pass over K (the V half of the slab is
// not touched), every key's sum in one place. A wave owns 64 keys: it holds them as matrix-core operands for the whole
// kernel (each cached byte is read and dequantised once, whatever the number of rows) and the rows pass by, 16 at a time
// out of LDS, where the four waves share them: S = Q K^T with v_mfma_f32_16x16x32_f16, a key living in the 16 lanes' same
// column, so a key's sum runs in one register per lane over all rows and is joined over the four lane groups once at the
// end. No atomics: the order of the sum is fixed.
//
// One row block (a decode step) is bound by memory: 64 sequences of 256 - 4 096 keys, H 32 / KVH 8 / head_dim 128, 50.6 us =
// 3.7 TB/s. Windows of queries are bound by the exponentials and the start of a workgroup (keys, then rows, before the
// first product): 32 queries over 4 k - 32 k keys of 8 sequences 65 us = 463 TFLOP/s, 2.4 TB/s. Requesting the rows
// together with the keys costs registers, and with them half the waves: 81 us.
#include "cache_tile.h"

namespace pplhip {

struct ScoreParams {
    const half_t* q; // [S, H, head_dim]
    const float* lse; // [S, H]
    const int64_t* position_idx; // [S] or null
    const int64_t* seqstarts;
    const int64_t* kvstarts;
    CacheView view;
    const float* score_in;
    float* score_out;
    int32_t* position;
    int64_t score_offset, score_stride_h; // of the layer; between kv heads
    int32_t num_heads, kv_heads, rep;
    int32_t key_blocks; // workgroups per sequence and kv head
    float scale_log2; // log2(e) / sqrt(head_dim)
};

constexpr int kScoreWaveKeys = 64;
constexpr int kScoreKeys = 4 * kScoreWaveKeys; // keys per workgroup
constexpr int kScoreRows = 128; // rows held in LDS at a time: they take the place of the key tiles

template <int DH>
__global__ __launch_bounds__(256, 2) void kv_score_kernel(const ScoreParams p) {
    constexpr int LDR = kKeyRow<DH>;
    constexpr int KC2 = DH / 32;
    __shared__ __attribute__((aligned(16))) half_t lds[4 * kTileKeys * LDR]; // key tiles, then rows of queries
    static_assert(kScoreRows <= 4 * kTileKeys, "the rows fit the tiles' place");
    __shared__ __attribute__((aligned(16))) float row_lse[kScoreRows]; // in units of log2
    __shared__ __attribute__((aligned(16))) int row_last[kScoreRows]; // last key of the workgroup's block the row sees, or -1

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r_lane = lane & 15, g = lane >> 4;
    const int hd = p.view.head_dim;
    const int kvh = blockIdx.x % p.kv_heads;
    const int rest = blockIdx.x / p.kv_heads;
    const int b = rest / p.key_blocks;
    const int block0 = (rest - b * p.key_blocks) * kScoreKeys;
    const const_tab64_t seqstarts = (const_tab64_t)p.seqstarts, kvstarts = (const_tab64_t)p.kvstarts;
    const int64_t s0 = seqstarts[b];
    const int L = (int)(seqstarts[b + 1] - s0), kvlen = (int)(kvstarts[b + 1] - kvstarts[b]);
    if (L <= 0 || block0 >= kvlen) return;
    const int start = kvlen - L, rows = L * p.rep;
    const int key0 = block0 + wave * kScoreWaveKeys;
    half_t* const tile = lds + wave * kTileKeys * LDR;

    // ---- the wave's keys as B operands: key 16 * kb + r_lane, positions 32 * kc + 8 * g .. + 7 of its LDS row
    half8_t kf[4][KC2];
    const bool have_keys = key0 < kvlen;
    if (have_keys) {
        const SequenceRows seq(p.view, b, kvh);
        CacheTile<DH> raw[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int kv0 = key0 + h * kTileKeys < kvlen ? key0 + h * kTileKeys : key0;
            raw[h].fetch(p.view, seq.key_row(kv0), kv0, kvlen);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wave_lds_order();
            raw[h].stash(tile, LDR, hd);
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int kc = 0; kc < KC2; ++kc)
                    kf[2 * h + i][kc] = *reinterpret_cast<const half8_t*>(tile + (16 * i + r_lane) * LDR + 32 * kc + 8 * g);
        }
    }
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    for (int chunk = 0; chunk < rows; chunk += kScoreRows) {
        const int n = rows - chunk < kScoreRows ? rows - chunk : kScoreRows;
        __syncthreads(); // (the key tiles, or the rows before, have been read)
        // rows of the chunk, 16 bytes (one group) a thread at a time
        const int groups = hd / 8;
#pragma unroll 2
        for (int x = threadIdx.x; x < n * groups; x += 256) {
            const int r = x / groups, group = x - r * groups;
            const int row = chunk + r, t = row / p.rep;
            const half_t* src = p.q + ((s0 + t) * p.num_heads + kvh * p.rep + (row - t * p.rep)) * hd + 8 * group;
            *reinterpret_cast<half8_t*>(lds + r * LDR + 8 * group) = *reinterpret_cast<const half8_t*>(src);
        }
        if (threadIdx.x < kScoreRows) {
            float l = 0.f;
            int last = -1;
            if ((int)threadIdx.x < n) {
                const int row = chunk + threadIdx.x, t = row / p.rep;
                l = p.lse[(s0 + t) * p.num_heads + kvh * p.rep + (row - t * p.rep)] * 1.44269504088896f;
                const int lim = start + t - block0;
                if (l != -INFINITY) last = lim < -1 ? -1 : lim;
            }
            row_lse[threadIdx.x] = l;
            row_last[threadIdx.x] = last;
        }
        __syncthreads();
        if (!have_keys) continue;
        for (int r0 = 0; r0 < n; r0 += 16) {
            const int r = r0 + r_lane < n ? r0 + r_lane : n - 1;
            half8_t qf[KC2];
#pragma unroll
            for (int kc = 0; kc < KC2; ++kc) {
                const int channel = channel_at<DH>(32 * kc + 8 * g);
                qf[kc] = *reinterpret_cast<const half8_t*>(lds + r * LDR + (channel < hd ? channel : 0));
                if (hd < DH && channel >= hd) qf[kc] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
            }
            const float4_t lse = *reinterpret_cast<const float4_t*>(&row_lse[r0 + 4 * g]);
            const int4 last = *reinterpret_cast<const int4*>(&row_last[r0 + 4 * g]);
            const int lim[4] = {last.x, last.y, last.z, last.w};
            // every row sees every key of the wave (and has a distribution): nothing to hide
            const int least = min(min(lim[0], lim[1]), min(lim[2], lim[3]));
            const bool all = __all(least >= (wave + 1) * kScoreWaveKeys - 1);
            float4_t acc[4];
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) acc[kb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kc = 0; kc < KC2; ++kc)
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
                    acc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[kc], kf[kb][kc], acc[kb], 0, 0, 0);
            if (all) {
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[kb] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[kb][e], p.scale_log2, -lse[e]));
                continue;
            }
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const int key = wave * kScoreWaveKeys + 16 * kb + r_lane; // within the workgroup's block
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[kb][e], p.scale_log2, -lse[e]));
                    w[kb] += key <= lim[e] ? pr : 0.f;
                }
            }
        }
    }
    if (!have_keys) return;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
        w[kb] += __shfl_xor(w[kb], 16);
        w[kb] += __shfl_xor(w[kb], 32);
    }
    // lane group g writes key block g: 64 consecutive keys, one per lane
    const float mine = g == 0 ? w[0] : g == 1 ? w[1] : g == 2 ? w[2] : w[3];
    const int j = key0 + lane;
    if (j < kvlen) {
        const int64_t at = p.score_offset + kvh * p.score_stride_h + uniform_token(p.view.pages, b, key0) + lane;
        p.score_out[at] = (j < start ? p.score_in[at] : 0.f) + mine;
        if (p.position && j >= start) p.position[at] = (int32_t)p.position_idx[s0 + (j - start)];
    }
}

pplhip_retcode launch_kv_score(const pplhip_kv_score_args* a, hipStream_t stream) {
    ScoreParams p;
    p.q = (const half_t*)a->d_query;
    p.lse = (const float*)a->d_lse;
    p.position_idx = a->d_position_idx;
    p.seqstarts = a->d_seqstarts;
    p.kvstarts = a->d_kvstarts;
    p.view = CacheView{(const int8_t*)a->d_cache, (const half_t*)a->d_scale,
                       PageMap{a->d_cachestarts, a->cachestart_stride_b, page_shift_of(a->cache_mode, a->page_size)},
                       CacheAddr{a->cache_stride_s, a->cache_stride_l, a->cache_stride_h, a->cache_stride_kv, a->layer_idx},
                       a->head_dim};
    p.score_in = a->d_score_in;
    p.score_out = a->d_score_out;
    p.position = a->d_position;
    p.score_offset = (int64_t)a->layer_idx * a->score_stride_l;
    p.score_stride_h = a->score_stride_h;
    p.num_heads = a->num_heads;
    p.kv_heads = a->num_kv_heads;
    p.rep = a->num_heads / a->num_kv_heads;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)a->head_dim));
    const int64_t key_blocks = (a->max_kvlen + kScoreKeys - 1) / kScoreKeys;
    if (!launch_fits((double)key_blocks * (double)a->batch * (double)a->num_kv_heads, 256))
        PPLHIP_FAIL(PPLHIP_RC_OUT_OF_RANGE, "kv_score: too many key blocks");
    p.key_blocks = (int32_t)key_blocks;
    const dim3 grid((unsigned)(key_blocks * a->batch * a->num_kv_heads));
    switch (padded_head_dim(a->head_dim)) {
        case 32: hipLaunchKernelGGL(kv_score_kernel<32>, grid, dim3(256), 0, stream, p); break;
        case 64: hipLaunchKernelGGL(kv_score_kernel<64>, grid, dim3(256), 0, stream, p); break;
        case 96: hipLaunchKernelGGL(kv_score_kernel<96>, grid, dim3(256), 0, stream, p); break;
        case 128: hipLaunchKernelGGL(kv_score_kernel<128>, grid, dim3(256), 0, stream, p); break;
        case 160: hipLaunchKernelGGL(kv_score_kernel<160>, grid, dim3(256), 0, stream, p); break;
        case 192: hipLaunchKernelGGL(kv_score_kernel<192>, grid, dim3(256), 0, stream, p); break;
        case 224: hipLaunchKernelGGL(kv_score_kernel<224>, grid, dim3(256), 0, stream, p); break;
        default: hipLaunchKernelGGL(kv_score_kernel<256>, grid, dim3(256), 0, stream, p); break;
    }
    PPLHIP_CHECK_LAUNCH("kv_score");
    return PPLHIP_RC_SUCCESS;
}

} // namespace pplhip
