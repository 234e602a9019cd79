"""Plumbing of the tests of the operators that put several new tokens over the int8 slab or keep the slab up: a ragged
batch with its slab, the library's calls on it, and the operators' definitions in 64 bits (numpy)."""
import ctypes as C
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import __graft_entry__ as entry  # noqa: E402

pkg = entry.load_package()
from ppl_nn_amd import cabi  # noqa: E402

NAN16 = np.uint16(0x7E00)


class Case:
    """new[b] new tokens behind old[b] cached ones, per sequence; every slab row no token owns holds NaN scales."""

    def __init__(self, heads, kv_heads, dim, new, old, layers=1, layer=0, layout=0, page=0, slack=3, pad_stride=0, seed=0):
        self.heads, self.kv_heads, self.dim, self.layers, self.layer = heads, kv_heads, dim, layers, layer
        self.new, self.old = np.asarray(new, np.int64), np.asarray(old, np.int64)
        self.batch, self.page = len(self.new), page
        self.kvlen = self.new + self.old
        rng = np.random.default_rng(seed)
        self.rng = rng
        if page:
            pages = -(-self.kvlen // page)
            self.max_pages = int(max(1, pages.max(initial=1)))
            order = rng.permutation(int(pages.sum()) + 2)
            self.cachestarts = np.full((self.batch, self.max_pages), 1 << 40, np.int64)  # (entries past a sequence's end)
            k = 0
            for b, n in enumerate(pages):
                self.cachestarts[b, :n] = order[k:k + n] * page
                k += int(n)
            self.tokens = (int(pages.sum()) + 2) * page
            self.tok = [self.cachestarts[b, np.arange(n) // page] + np.arange(n) % page for b, n in enumerate(self.kvlen)]
        else:
            self.max_pages = 0
            starts = np.concatenate([[0], np.cumsum(self.kvlen + slack)])
            self.cachestarts = starts[:-1].astype(np.int64)
            self.tokens = max(1, int(starts[-1]))
            self.tok = [self.cachestarts[b] + np.arange(n) for b, n in enumerate(self.kvlen)]
        if layout == 0:  # [token, layer, K/V, head, channel], pad_stride channels between tokens
            row = layers * 2 * kv_heads * dim + pad_stride
            st = (row, 2 * kv_heads * dim, dim, kv_heads * dim)
            size = self.tokens * row
        else:  # [layer, K/V, head, token, channel]
            st = (dim, 2 * kv_heads * self.tokens * dim, self.tokens * dim, kv_heads * self.tokens * dim)
            size = layers * 2 * kv_heads * self.tokens * dim
        self.stride_s, self.stride_l, self.stride_h, self.stride_kv = st
        self.cache = rng.integers(-127, 128, size, dtype=np.int8)
        self.scale = np.full(size // 8, NAN16, np.uint16).view(np.float16)
        every = np.concatenate(self.tok) if self.batch else np.zeros(0, np.int64)
        r = self.rows(every, slice(None), slice(None))
        good = (np.abs(rng.standard_normal(r.shape + (dim // 8,))) * 0.01 + 0.002).astype(np.float16)
        self.scale[(r // 8)[..., None] + np.arange(dim // 8)] = good
        self.query = rng.standard_normal((int(self.new.sum()), heads, dim)).astype(np.float16)

    def rows(self, tok, layer, head, kv=slice(None)):
        """Element offsets of rows [token, layer, kv, head] (or of single ones)."""
        lay = np.arange(self.layers)[layer] if isinstance(layer, slice) else layer
        kvs = np.arange(2)[kv] if isinstance(kv, slice) else kv
        hd = np.arange(self.kv_heads)[head] if isinstance(head, slice) else head
        t, lay, kvs, hd = np.ix_(np.atleast_1d(tok), np.atleast_1d(lay), np.atleast_1d(kvs), np.atleast_1d(hd))
        return t * self.stride_s + lay * self.stride_l + kvs * self.stride_kv + hd * self.stride_h

    def values(self, b, kv, head):
        """The cached K (0) or V (1) rows of a sequence as float64 [kvlen, dim]: fp16(int8 * scale)."""
        r = self.rows(self.tok[b], self.layer, head, kv)[:, 0, 0, 0]
        q = self.cache[r[:, None] + np.arange(self.dim)].astype(np.float32)
        s = self.scale[(r // 8)[:, None] + np.arange(self.dim // 8)].astype(np.float32).repeat(8, axis=1)
        with np.errstate(over="ignore", invalid="ignore"):
            return (q * s).astype(np.float16).astype(np.float64)

    @property
    def seqstarts(self):
        return np.concatenate([[0], np.cumsum(self.new)]).astype(np.int64)

    @property
    def kvstarts(self):
        return np.concatenate([[0], np.cumsum(self.kvlen)]).astype(np.int64)


def causal(n):
    return np.tril(np.ones((n, n), bool))


def random_tree(rng, n, blind=0.0):
    """Visibility of n drafted tokens: ancestors and itself; a share `blind` of the tokens sees no drafted token."""
    see = np.zeros((n, n), bool)
    for t in range(n):
        if rng.random() < blind:
            continue
        parent = -1 if t == 0 else int(rng.integers(-1, t))
        if parent >= 0:
            see[t] = see[parent]
        see[t, t] = True
    return see


def mask_words(see, words, junk_rng=None):
    """The visibility rows as 64-bit words; junk_rng fills the bits past each sequence's tokens."""
    out = []
    for m in see:
        n = m.shape[0]
        bits = np.zeros((n, words * 64), np.uint8) if junk_rng is None else \
            junk_rng.integers(0, 2, (n, words * 64), dtype=np.uint8)
        bits[:, :n] = m
        out.append(np.packbits(bits, axis=1, bitorder="little").view(np.uint64))
    return np.concatenate(out) if out else np.zeros((0, words), np.uint64)


def exact_attention(c, see):
    """(output, lse) in float64 and bounds on what the kernel's roundings may add to each.

    With A = sum_j w_j |v_j|: the weights are rounded to fp16 for the second product (2^-11 A), the result to fp16
    (2^-11 |o|), scores are fp32 sums of `dim` exact products (d = (dim + 4) 2^-23 sum_i |q_i k_i| / sqrt(dim), which
    moves a weight by at most 2 d relative to the others), exponent arguments fp32 (2^-22 (1 + |x|)), sums of kvlen fp32
    terms (kvlen 2^-23)."""
    S = int(c.new.sum())
    out, out_tol = np.zeros((S, c.heads, c.dim)), np.zeros((S, c.heads, c.dim))
    lse, lse_tol = np.full((S, c.heads), -np.inf), np.zeros((S, c.heads))
    rep = c.heads // c.kv_heads
    for b in range(c.batch):
        r0, n, o = int(c.seqstarts[b]), int(c.new[b]), int(c.old[b])
        if n == 0:
            continue
        vis = np.ones((n, n + o), bool)
        vis[:, o:] = see[b]
        for kvh in range(c.kv_heads):
            k, v = c.values(b, 0, kvh), c.values(b, 1, kvh)
            for h in range(kvh * rep, (kvh + 1) * rep):
                q = c.query[r0:r0 + n, h].astype(np.float64)
                for t in range(n):
                    j = np.flatnonzero(vis[t])
                    if not len(j):
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = k[j] @ q[t] / np.sqrt(c.dim)
                        m = x.max()
                        e = np.exp(x - m)
                        w = e / e.sum()
                        out[r0 + t, h] = w @ v[j]
                        lse[r0 + t, h] = m + np.log(e.sum())
                        a = w @ np.abs(v[j])
                        d = (c.dim + 4) * 2.0 ** -23 * (np.abs(k[j]) @ np.abs(q[t])).max() / np.sqrt(c.dim) + \
                            2.0 ** -22 * (1 + np.abs(x).max())
                        out_tol[r0 + t, h] = 2.0 ** -11 * np.abs(out[r0 + t, h]) + \
                            a * (2.0 ** -11 + 2 * d + (len(j) + 64) * 2.0 ** -23) + 2.0 ** -24
                        lse_tol[r0 + t, h] = d + (len(j) + 64) * 2.0 ** -23 + 2.0 ** -22 * (1 + abs(lse[r0 + t, h]))
    return out, out_tol, lse, lse_tol


def exact_score(c, lse, score_in):
    """(score, bound) for one layer's [kv_heads, tokens] array; the new tokens' old entries count as 0."""
    score, tol = score_in.astype(np.float64), np.zeros(score_in.shape)
    rep = c.heads // c.kv_heads
    for b in range(c.batch):
        r0, n, o = int(c.seqstarts[b]), int(c.new[b]), int(c.old[b])
        if n == 0:
            continue
        vis = np.ones((n, n + o), bool)
        vis[:, o:] = causal(n)
        for kvh in range(c.kv_heads):
            k = c.values(b, 0, kvh)
            add, err = np.zeros(n + o), np.zeros(n + o)
            for h in range(kvh * rep, (kvh + 1) * rep):
                for t in range(n):
                    z = float(lse[r0 + t, h])
                    if z == -np.inf:
                        continue
                    q = c.query[r0 + t, h].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        x = k @ q / np.sqrt(c.dim)
                        p = np.where(vis[t], np.exp(x - z), 0.0)
                        d = (c.dim + 4) * 2.0 ** -23 * (np.abs(k) @ np.abs(q)) / np.sqrt(c.dim) + \
                            2.0 ** -22 * (1 + np.abs(x) + abs(z))
                        add += p
                        err += p * np.where(vis[t], d, 0.0)
            before = score[kvh, c.tok[b]]
            before[o:] = 0.0
            score[kvh, c.tok[b]] = before + add
            tol[kvh, c.tok[b]] = err + (n * rep + 8) * 2.0 ** -23 * add + 2.0 ** -23 * np.abs(before + add) + 1e-30
    return score, tol


def exact_evict(c, score, position, target, next_pos, sinks, recent, layer_begin, layer_count):
    """Expected (cache, scale, score, position, new_kvlen) of an in-place call, by the definition: one column at a time."""
    cache, scale, score, position = c.cache.copy(), c.scale.copy(), score.copy(), position.copy()
    new_kvlen = np.minimum(c.kvlen, np.maximum(target, 0))
    old_cache, old_scale, old_score, old_pos = cache.copy(), scale.copy(), score.copy(), position.copy()
    for b in range(c.batch):
        n, keep, tok = int(c.kvlen[b]), int(new_kvlen[b]), c.tok[b]
        for layer in range(layer_begin, layer_begin + layer_count):
            for h in range(c.kv_heads):
                s, p = old_score[layer, h, tok].astype(np.float64), old_pos[layer, h, tok]
                protect = (p < sinks) | ((recent > 0) & (p >= next_pos[b] - recent))
                s = np.where(np.isnan(s), -np.inf, s)
                nan_low = np.isnan(old_score[layer, h, tok])
                rank = sorted(range(n), key=lambda j: (not protect[j], nan_low[j] and not protect[j],
                                                       0.0 if protect[j] else -s[j], j))
                stays = sorted(rank[:keep])
                kept = set(stays)
                holes = [j for j in range(keep) if j not in kept]
                fill = [j for j in stays if j >= keep][::-1]
                for to, frm in zip(holes, fill):
                    for kv in (0, 1):
                        a = int(c.rows(tok[to], layer, h, kv).item())
                        f = int(c.rows(tok[frm], layer, h, kv).item())
                        cache[a:a + c.dim] = old_cache[f:f + c.dim]
                        scale[a // 8:(a + c.dim) // 8] = old_scale[f // 8:(f + c.dim) // 8]
                    score[layer, h, tok[to]] = old_score[layer, h, tok[frm]]
                    position[layer, h, tok[to]] = old_pos[layer, h, tok[frm]]
    return cache, scale, score, position, new_kvlen


def exact_accept(c, paths, layer_begin, layer_count):
    cache, scale = c.cache.copy(), c.scale.copy()
    for b, path in enumerate(paths):
        for i, x in enumerate(path):
            a = c.rows(c.tok[b][c.old[b] + i], slice(layer_begin, layer_begin + layer_count), slice(None)).ravel()
            f = c.rows(c.tok[b][c.old[b] + x], slice(layer_begin, layer_begin + layer_count), slice(None)).ravel()
            cache[a[:, None] + np.arange(c.dim)] = c.cache[f[:, None] + np.arange(c.dim)]
            scale[(a // 8)[:, None] + np.arange(c.dim // 8)] = c.scale[(f // 8)[:, None] + np.arange(c.dim // 8)]
    return cache, scale


# ---- the library's calls

class Device:
    """Device copies of a case's arrays and argument blocks over them. `ptr` of anything that lives on the device."""

    def __init__(self, c):
        import torch
        self.torch, self.c, self.lib = torch, c, pkg.load_library()
        self.cache, self.scale = self.up(c.cache), self.up(c.scale)
        self.seqstarts, self.kvstarts = self.up(c.seqstarts), self.up(c.kvstarts)
        self.cachestarts, self.start_pos = self.up(c.cachestarts), self.up(c.old)
        self.query = self.up(c.query)

    def up(self, a):
        a = np.ascontiguousarray(a)
        if a.dtype == np.uint64:
            a = a.view(np.int64)
        return self.torch.from_numpy(a.copy()).cuda()

    @staticmethod
    def ptr(t):
        return None if t is None else (t.data_ptr() or None)

    def slab_args(self, a):
        c = self.c
        a.d_cachestarts = self.ptr(self.cachestarts)
        a.batch, a.num_layer, a.layer_idx = c.batch, c.layers, c.layer
        a.num_kv_heads, a.head_dim = c.kv_heads, c.dim
        a.cache_mode, a.page_size, a.cachestart_stride_b = (1, c.page, c.max_pages) if c.page else (0, 128, 0)
        a.cache_stride_s, a.cache_stride_l, a.cache_stride_h, a.cache_stride_kv = \
            c.stride_s, c.stride_l, c.stride_h, c.stride_kv
        a.d_cache, a.d_scale = self.ptr(self.cache), self.ptr(self.scale)
        return a

    def query_args(self, a):
        c = self.c
        self.slab_args(a)
        a.d_query, a.d_seqstarts, a.d_kvstarts = self.ptr(self.query), self.ptr(self.seqstarts), self.ptr(self.kvstarts)
        a.num_heads = c.heads
        a.total_new_tokens = int(c.new.sum())
        a.max_seqlen, a.max_kvlen = int(c.new.max(initial=0)), int(c.kvlen.max(initial=0))
        return a

    def tree_args(self, mask=None, words=0, extra_rows=2):
        """Outputs have rows behind the last sequence, filled with a pattern the call has to leave alone."""
        a = self.query_args(cabi.TreeAttentionArgs())
        S = int(self.c.new.sum())
        self.out = self.torch.full((S + extra_rows, self.c.heads, self.c.dim), 7.0, dtype=self.torch.float16, device="cuda")
        self.lse = self.torch.full((S + extra_rows, self.c.heads), 7.0, dtype=self.torch.float32, device="cuda")
        self.mask = None if mask is None else self.up(mask)
        a.d_tree_mask, a.tree_mask_words = self.ptr(self.mask), words
        a.d_output, a.d_lse = self.ptr(self.out), self.ptr(self.lse)
        return a

    def tree_plan(self, a, ranges=None):
        plan = cabi.TreeAttentionPlan()
        pkg.check(self.lib.pplhip_tree_attention_prepare(C.byref(a), C.byref(plan)), "tree prepare")
        if ranges:
            assert plan.num_ranges >= ranges, plan.num_ranges
            plan.num_ranges = ranges
        ws = self.torch.full((max(256, plan.workspace_bytes),), 0xFF, dtype=self.torch.uint8, device="cuda")
        return plan, ws

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def tree(self, mask=None, words=0, ranges=None, no_lse=False):
        a = self.tree_args(mask, words)
        if no_lse:
            a.d_lse = None
        plan, ws = self.tree_plan(a, ranges)
        pkg.check(self.lib.pplhip_tree_attention_forward(C.byref(a), C.byref(plan), ws.data_ptr(), self.stream()), "tree")
        self.torch.cuda.synchronize()
        S = int(self.c.new.sum())
        out, lse = self.out.cpu().numpy(), self.lse.cpu().numpy()
        assert (out[S:] == 7.0).all() and (lse[S:] == 7.0).all(), "rows behind the last sequence were written"
        return out[:S], lse[:S]

    def score(self, lse, score_in, position_idx=None, in_place=False, position=None, layers_apart=None):
        """score_in: [layers, kv_heads, tokens]."""
        c = self.c
        a = self.query_args(cabi.KvScoreArgs())
        self.s_in, self.lse_in = self.up(score_in), self.up(lse.astype(np.float32))
        self.s_out = self.s_in if in_place else self.torch.full_like(self.s_in, -5.0)
        self.pos = None if position is None else self.up(position)
        self.pos_idx = None if position_idx is None else self.up(position_idx)
        a.d_lse, a.d_position_idx, a.d_position = self.ptr(self.lse_in), self.ptr(self.pos_idx), self.ptr(self.pos)
        a.d_score_in, a.d_score_out = self.ptr(self.s_in), self.ptr(self.s_out)
        a.score_stride_l, a.score_stride_h = c.kv_heads * score_in.shape[2], score_in.shape[2]
        pkg.check(self.lib.pplhip_kv_score_accumulate(C.byref(a), self.stream()), "score")
        self.torch.cuda.synchronize()
        return self.s_out.cpu().numpy(), None if position is None else self.pos.cpu().numpy()

    def evict_args(self, score, position, target, next_pos, sinks, recent, layer_begin, layer_count, in_place):
        c = self.c
        a = self.slab_args(cabi.KvEvictArgs())
        a.layer_idx, a.layer_count = layer_begin, layer_count
        self.target, self.next_pos = self.up(np.asarray(target, np.int64)), self.up(np.asarray(next_pos, np.int64))
        self.s_in = self.up(score)
        self.p_in = None if position is None else self.up(position)
        self.s_out = self.s_in if in_place else self.torch.full_like(self.s_in, -5.0)
        self.p_out = self.p_in if in_place or position is None else self.torch.full_like(self.p_in, -5)
        self.new_kvlen = self.torch.full((max(1, c.batch),), -9, dtype=self.torch.int64, device="cuda")
        a.d_kvstarts, a.d_target_kvlen, a.d_next_pos = self.ptr(self.kvstarts), self.ptr(self.target), self.ptr(self.next_pos)
        a.max_kvlen, a.num_sink, a.num_recent = int(c.kvlen.max(initial=0)), sinks, recent
        a.d_score_in, a.d_score_out = self.ptr(self.s_in), self.ptr(self.s_out)
        a.d_position_in, a.d_position_out = self.ptr(self.p_in), self.ptr(self.p_out)
        a.score_stride_l, a.score_stride_h = c.kv_heads * score.shape[2], score.shape[2]
        a.d_new_kvlen = self.ptr(self.new_kvlen)
        return a

    def evict(self, score, position, target, next_pos, sinks=0, recent=0, layer_begin=0, layer_count=None, in_place=True):
        c = self.c
        a = self.evict_args(score, position, target, next_pos, sinks, recent, layer_begin,
                            c.layers if layer_count is None else layer_count, in_place)
        plan = cabi.KvEvictPlan()
        pkg.check(self.lib.pplhip_kv_evict_prepare(C.byref(a), C.byref(plan)), "evict prepare")
        ws = self.torch.full((max(256, plan.workspace_bytes),), 0xFF, dtype=self.torch.uint8, device="cuda")
        pkg.check(self.lib.pplhip_kv_evict(C.byref(a), C.byref(plan), ws.data_ptr(), self.stream()), "evict")
        self.torch.cuda.synchronize()
        return (self.cache.cpu().numpy(), self.scale.cpu().numpy(), self.s_out.cpu().numpy(),
                None if position is None else self.p_out.cpu().numpy(), self.new_kvlen.cpu().numpy()[:c.batch])

    def accept(self, table, lengths, max_accepted, layer_begin=0, layer_count=None):
        c = self.c
        a = self.slab_args(cabi.KvAcceptArgs())
        a.layer_idx, a.layer_count = layer_begin, c.layers if layer_count is None else layer_count
        self.path, self.path_len = self.up(np.asarray(table, np.int64)), self.up(np.asarray(lengths, np.int64))
        a.d_seqstarts, a.d_start_pos = self.ptr(self.seqstarts), self.ptr(self.start_pos)
        a.d_accepted, a.d_accepted_len = self.ptr(self.path), self.ptr(self.path_len)
        a.accepted_stride_b, a.max_accepted = np.asarray(table).shape[1], max_accepted
        pkg.check(self.lib.pplhip_kv_accept(C.byref(a), self.stream()), "accept")
        self.torch.cuda.synchronize()
        return self.cache.cpu().numpy(), self.scale.cpu().numpy()


def assert_within(got, want, tol, what):
    got = got.astype(np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    if bad.any():
        i = tuple(int(x) for x in np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off, first at {i}: got {got[i]}, want {want[i]}, "
                             f"bound {np.broadcast_to(tol, want.shape)[i]}")
