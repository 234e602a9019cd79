"""Tree attention over the int8 slab, accumulated attention weights, eviction and accepted drafts on the GPU, against the
definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import cache_ops
from cache_ops import Case, Device, assert_within, cabi, causal, mask_words, pkg, random_tree

pytestmark = pytest.mark.gpu


def check_tree(c, see=None, words=None, junk=False, **kw):
    mask = None
    if see is None:
        see = [causal(int(n)) for n in c.new]
    else:
        words = words or (int(c.new.max()) + 63) // 64
        mask = mask_words(see, words, np.random.default_rng(5) if junk else None)
    got, got_lse = Device(c).tree(mask, words or 0, **kw)
    out, tol, lse, lse_tol = cache_ops.exact_attention(c, see)
    assert_within(got, out, tol, "output")
    if not kw.get("no_lse"):
        assert_within(got_lse, lse, lse_tol, "lse")
    return got, got_lse


def trees(c, blind=0.0):
    return [random_tree(c.rng, int(n), blind) for n in c.new]


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (8, 1, 128), (4, 4, 128), (3, 3, 64), (20, 4, 80), (2, 2, 16),
                                                (6, 2, 48), (4, 2, 96), (2, 1, 112), (2, 1, 160), (4, 4, 192), (2, 2, 208),
                                                (4, 2, 256), (40, 1, 32), (2, 1, 240)])
def test_tree_head_layouts(heads, kv_heads, dim):
    c = Case(heads, kv_heads, dim, [5, 1, 9, 3], [70, 0, 31, 200], layers=2, layer=1, seed=dim)
    check_tree(c, trees(c))


@pytest.mark.parametrize("new", [1, 2, 4, 7, 8, 9, 16, 31, 33, 63, 64, 65, 100])
def test_tree_sizes(new):
    c = Case(8, 2, 128, [new, max(1, new // 2), 1], [33, 0, 500], seed=new)
    check_tree(c, trees(c), junk=True)
    check_tree(c)


@pytest.mark.parametrize("old", [0, 1, 27, 28, 31, 32, 33, 59, 60, 61, 64, 95, 127, 128, 129, 255, 256])
def test_tree_history_edges(old):
    c = Case(4, 2, 128, [4, 37], [old, old + 1], seed=old)
    check_tree(c, trees(c), junk=True)


def test_tree_single_tokens_and_empty_sequences():
    c = Case(16, 4, 128, [1, 0, 1, 1, 0, 1], [0, 40, 300, 31, 0, 32], seed=1)
    check_tree(c)
    check_tree(c, trees(c))


def test_tree_rows_that_see_nothing():
    c = Case(4, 2, 64, [6, 3, 70], [0, 0, 10], seed=2)
    see = trees(c, blind=0.4)
    see[0][2] = False
    see[1][:] = False
    got, lse = check_tree(c, see, words=3)
    assert (got[2] == 0).all() and (lse[2] == -np.inf).all() and (lse[6:9] == -np.inf).all()


def test_tree_mask_that_is_no_tree():
    c = Case(4, 4, 128, [50, 90], [100, 7], seed=3)
    see = [c.rng.random((int(n), int(n))) < 0.3 for n in c.new]
    check_tree(c, see, junk=True)


@pytest.mark.parametrize("page", [64, 128, 512])
@pytest.mark.parametrize("layout", [0, 3])
def test_tree_paged(page, layout):
    c = Case(8, 2, 128, [5, 20, 1, 66], [60, 1000, 63, 129], layers=2, layer=1, layout=layout, page=page, seed=page)
    check_tree(c, trees(c))


@pytest.mark.parametrize("layout,pad", [(3, 0), (0, 16), (0, 48)])
def test_tree_strides(layout, pad):
    c = Case(6, 3, 80, [5, 20], [60, 333], layers=3, layer=2, layout=layout, pad_stride=pad, seed=pad)
    check_tree(c, trees(c))


@pytest.mark.parametrize("ranges", [1, 2, 3, 7, 16])
def test_tree_range_counts_give_the_same_rows(ranges):
    """Any number of ranges up to the plan's is allowed; pieces that start and end inside row tiles are joined."""
    c = Case(8, 1, 128, [12, 1, 9, 30], [900, 3, 2100, 40], seed=4)
    check_tree(c, trees(c), ranges=ranges)


def test_tree_many_sequences():
    rng = np.random.default_rng(9)
    c = Case(4, 1, 64, rng.integers(0, 4, 300), rng.integers(0, 90, 300), seed=6)
    check_tree(c, trees(c))


def test_tree_long_history():
    c = Case(8, 1, 128, [3, 17], [40000, 9001], seed=7)
    check_tree(c, trees(c))


def test_tree_without_lse():
    c = Case(8, 2, 128, [5, 1], [70, 900], seed=8)
    check_tree(c, trees(c), no_lse=True)


def test_tree_hidden_tokens_may_hold_anything():
    """Padding tokens nobody sees (and one that only itself sees) with NaN and infinite scales."""
    c = Case(4, 2, 128, [12, 40], [50, 3], seed=10)
    see = [causal(12), random_tree(c.rng, 40)]
    for b, nodes in ((0, [3, 7]), (1, [0, 33])):
        for x in nodes:
            see[b][:, x] = False
            r = c.rows(c.tok[b][c.old[b] + x], 0, slice(None)).ravel()
            c.scale.view(np.uint16)[(r // 8)[:, None] + np.arange(16)] = 0x7E00 if x % 2 else 0x7C00
    see[0][7, 7] = True  # this one sees its own NaN: its row is NaN, the others' are not
    check_tree(c, see)


def test_tree_large_scales():
    """Values near fp16's largest among the new tokens (they leave the matrix product's path, and must not change)."""
    c = Case(4, 2, 64, [9], [40], seed=11)
    r = c.rows(c.tok[0][[43, 46]], 0, slice(None), 1).ravel()
    c.scale[(r // 8)[:, None] + np.arange(8)] = 514.0
    check_tree(c, trees(c))


def test_tree_sharp_and_flat_scores():
    c = Case(4, 1, 128, [6], [3000], seed=12)
    c.query[:, 0] *= 30
    c.query[:, 1] *= 0
    check_tree(c, trees(c))


def test_tree_replays_from_a_graph_beside_eager_calls():
    import torch
    c = Case(8, 2, 128, [5, 12], [700, 90], seed=13)
    see = trees(c)
    d = Device(c)
    a = d.tree_args(mask_words(see, 1), 1)
    plan, ws = d.tree_plan(a)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call = lambda w, st: pkg.check(d.lib.pplhip_tree_attention_forward(C.byref(a), C.byref(plan), w.data_ptr(), st))
        call(ws, s.cuda_stream)
    s.synchronize()
    want, want_lse = d.out.clone(), d.lse.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call(ws, torch.cuda.current_stream().cuda_stream)
    ws2 = torch.empty_like(ws)
    for i in range(4):
        d.out.fill_(3.0)
        d.lse.fill_(3.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        n = int(c.new.sum())
        assert torch.equal(d.out[:n], want[:n]) and torch.equal(d.lse[:n], want_lse[:n])
        call(ws2, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(d.out[:n], want[:n])


# ---- accumulated weights

def check_score(c, in_place=False, dead_rows=()):
    d = Device(c)
    lse = cache_ops.exact_attention(c, [causal(int(n)) for n in c.new])[2].astype(np.float32)
    for r in dead_rows:
        lse[r] = -np.inf
    score = np.abs(c.rng.standard_normal((c.layers, c.kv_heads, c.tokens))).astype(np.float32)
    position = np.full((c.layers, c.kv_heads, c.tokens), -3, np.int32)
    pidx = c.rng.integers(0, 1 << 20, int(c.new.sum()))
    got, pos = d.score(lse, score, pidx, in_place, position)
    want, tol = cache_ops.exact_score(c, lse, score[c.layer])
    for b in range(c.batch):
        if c.new[b]:
            assert_within(got[c.layer][:, c.tok[b]], want[:, c.tok[b]], tol[:, c.tok[b]], f"score of sequence {b}")
            position[c.layer][:, c.tok[b][c.old[b]:]] = pidx[c.seqstarts[b]:c.seqstarts[b + 1]].astype(np.int32)
    assert np.array_equal(pos, position)
    untouched = np.ones(got.shape, bool)
    for b in range(c.batch):
        if c.new[b]:
            untouched[c.layer][:, c.tok[b]] = False
    assert np.array_equal(got[untouched], (score if in_place else np.full_like(score, -5.0))[untouched])
    return got


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (8, 1, 128), (4, 4, 16), (20, 4, 80), (6, 2, 48), (3, 1, 96),
                                                (2, 2, 160), (2, 1, 208), (4, 2, 240), (2, 1, 256), (40, 1, 64)])
def test_score_head_layouts(heads, kv_heads, dim):
    check_score(Case(heads, kv_heads, dim, [5, 1, 0, 9], [70, 0, 20, 300], layers=2, layer=1, seed=dim))


@pytest.mark.parametrize("new", [1, 2, 15, 16, 17, 64, 65, 130])
@pytest.mark.parametrize("old", [0, 1, 63, 64, 255, 257])
def test_score_sizes(new, old):
    check_score(Case(4, 2, 64, [new, 1], [old, 2 * old], seed=new + old), in_place=bool(new & 1))


@pytest.mark.parametrize("page,layout", [(64, 0), (128, 3), (0, 3)])
def test_score_layouts(page, layout):
    check_score(Case(8, 2, 128, [3, 20, 1], [60, 700, 64], layers=2, layer=0, layout=layout, page=page, seed=page))


def test_score_rows_without_a_distribution():
    c = Case(4, 2, 128, [4, 3], [40, 5], seed=3)
    c.query[5] = np.nan  # a padding row: its lse is -inf, it adds nothing
    d = Device(c)
    want = Case(4, 2, 128, [4, 3], [40, 5], seed=3)
    lse = cache_ops.exact_attention(want, [causal(4), causal(3)])[2].astype(np.float32)
    lse[5] = -np.inf
    score = np.zeros((1, 2, c.tokens), np.float32)
    got, _ = d.score(lse, score)
    ref, tol = cache_ops.exact_score(want, lse, score[0])
    for b in range(2):
        assert_within(got[0][:, c.tok[b]], ref[:, c.tok[b]], tol[:, c.tok[b]], "score")


def test_score_hidden_keys_may_hold_nan():
    """A later token's NaN key reaches its own sum and later rows', not the sums of other keys by earlier rows."""
    c = Case(2, 1, 64, [3], [30], seed=4)
    lse = cache_ops.exact_attention(c, [causal(3)])[2].astype(np.float32)
    r = c.rows(c.tok[0][32], 0, 0, 0).ravel()
    c.scale.view(np.uint16)[(r // 8)[:, None] + np.arange(8)] = 0x7E00
    got, _ = Device(c).score(lse, np.zeros((1, 1, c.tokens), np.float32))
    assert np.isnan(got[0, 0, c.tok[0][32]]) and np.isfinite(got[0, 0, c.tok[0][:32]]).all()


def test_score_repeats_bit_for_bit():
    c = Case(8, 2, 128, [33, 2], [900, 10], seed=5)
    assert np.array_equal(check_score(c), check_score(Case(8, 2, 128, [33, 2], [900, 10], seed=5)))


# ---- eviction

def evict_inputs(c, ties=False, nan=False):
    score = c.rng.lognormal(0, 2, (c.layers, c.kv_heads, c.tokens)).astype(np.float32)
    if ties:
        score = c.rng.integers(0, 3, score.shape).astype(np.float32)
        score[score == 0] *= c.rng.choice([1.0, -1.0], int((score == 0).sum())).astype(np.float32)  # -0 and 0 are equal
    if nan:
        score[c.rng.random(score.shape) < 0.2] = np.nan
        score[c.rng.random(score.shape) < 0.05] = np.inf
        score[c.rng.random(score.shape) < 0.05] = -np.inf
    position = np.full((c.layers, c.kv_heads, c.tokens), -1, np.int32)
    for b in range(c.batch):  # every head has its own order, as after earlier evictions
        for layer in range(c.layers):
            for h in range(c.kv_heads):
                position[layer, h, c.tok[b]] = c.rng.permutation(int(c.kvlen[b])) * 2
    return score, position


def check_evict(c, target, sinks=0, recent=0, in_place=True, ties=False, nan=False, positions=True, lo=0, count=None):
    score, position = evict_inputs(c, ties, nan)
    target, next_pos = np.asarray(target, np.int64), 2 * c.kvlen
    count = c.layers if count is None else count
    cache, scale, s, p, n = Device(c).evict(score, position if positions else None, target, next_pos, sinks, recent, lo,
                                            count, in_place)
    e_cache, e_scale, e_s, e_p, e_n = cache_ops.exact_evict(c, score, position, target, next_pos, sinks, recent, lo, count)
    assert np.array_equal(n, e_n)
    assert np.array_equal(cache, e_cache)
    assert np.array_equal(scale.view(np.uint16), e_scale.view(np.uint16))
    if in_place:
        assert np.array_equal(s.view(np.uint32), e_s.view(np.uint32))
        assert not positions or np.array_equal(p, e_p)
    else:
        for b in range(c.batch):
            t = c.tok[b]
            k = int(e_n[b])
            assert np.array_equal(s[lo:lo + count][:, :, t[:k]].view(np.uint32), e_s[lo:lo + count][:, :, t[:k]].view(np.uint32))
            assert (s[lo:lo + count][:, :, t[k:]] == -5.0).all()
            if positions:
                assert np.array_equal(p[lo:lo + count][:, :, t[:k]], e_p[lo:lo + count][:, :, t[:k]])


@pytest.mark.parametrize("dim,kv_heads,layout,page", [(128, 2, 0, 0), (128, 3, 3, 0), (64, 1, 0, 64), (80, 2, 3, 128),
                                                      (16, 4, 0, 0), (256, 1, 0, 0), (112, 2, 0, 64)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_layouts(dim, kv_heads, layout, page, in_place):
    c = Case(kv_heads, kv_heads, dim, [0] * 5, [1, 2, 65, 200, 513], layers=2, layout=layout, page=page, seed=dim)
    check_evict(c, [1, 1, 40, 150, 100], sinks=4, recent=20, in_place=in_place)


@pytest.mark.parametrize("ties,nan", [(True, False), (False, True), (True, True)])
def test_evict_ties_and_nan(ties, nan):
    c = Case(2, 2, 32, [0] * 4, [64, 300, 1000, 77], seed=1)
    check_evict(c, [32, 100, 999, 3], sinks=2, recent=10, ties=ties, nan=nan)


def test_evict_targets_past_either_end():
    c = Case(2, 2, 64, [0] * 6, [50, 50, 50, 50, 0, 1], seed=2)
    check_evict(c, [0, -7, 50, 1 << 40, 10, 1], sinks=1, recent=4)


def test_evict_more_protected_than_kept():
    c = Case(1, 1, 64, [0] * 2, [300, 20], seed=3)
    check_evict(c, [16, 5], sinks=8, recent=200)


def test_evict_without_positions():
    c = Case(2, 1, 128, [0] * 2, [300, 20], seed=4)
    check_evict(c, [100, 10], positions=False)


def test_evict_some_layers():
    c = Case(2, 2, 64, [0, 0], [130, 40], layers=4, seed=5)
    check_evict(c, [100, 10], sinks=3, recent=30, lo=1, count=2)


@pytest.mark.parametrize("n,keep", [(511, 256), (512, 511), (513, 1), (4097, 2000), (20000, 19000), (70000, 30001)])
def test_evict_lengths(n, keep):
    c = Case(1, 1, 16, [0], [n], seed=n)
    check_evict(c, [keep], sinks=4, recent=100)


# ---- accepted drafts

@pytest.mark.parametrize("dim,kv_heads,layout,page,layers", [(128, 2, 0, 0, 3), (128, 8, 3, 0, 2), (64, 1, 0, 64, 1),
                                                             (80, 3, 3, 128, 2), (16, 1, 0, 0, 2), (256, 1, 0, 0, 2)])
def test_accept_layouts(dim, kv_heads, layout, page, layers):
    c = Case(kv_heads, kv_heads, dim, [1, 5, 64, 33, 9, 0, 20], [0, 60, 100, 3, 127, 9, 64], layers=layers, layout=layout,
             page=page, seed=dim)
    paths = [[0], [0, 2, 4], [1, 2, 3, 10, 40, 41, 42, 43, 44, 60, 63], list(range(1, 33)), [], [], [0, 1, 2, 19]]
    table = np.full((7, 40), 1 << 40, np.int64)
    for b, p in enumerate(paths):
        table[b, :len(p)] = p
    cache, scale = Device(c).accept(table, [len(p) for p in paths], 40)
    want_cache, want_scale = cache_ops.exact_accept(c, paths, 0, layers)
    assert np.array_equal(cache, want_cache) and np.array_equal(scale.view(np.uint16), want_scale.view(np.uint16))


def test_accept_lists_end_where_they_stop_ascending():
    c = Case(2, 2, 64, [10, 10, 10, 10, 10], [5] * 5, layers=3, seed=6)
    table = [[2, 4, 3, 9], [3, 3, 5, 6], [1, 12, 13, 14], [-1, 5, 6, 7], [4, 5, 6, 7]]
    lengths = [4, 4, 4, 4, 1 << 50]
    paths = [[2, 4], [3], [1], [], [4, 5, 6]]  # the last one: at most max_accepted = 3 entries
    cache, scale = Device(c).accept(table, lengths, 3, layer_begin=1, layer_count=2)
    want_cache, want_scale = cache_ops.exact_accept(c, paths, 1, 2)
    assert np.array_equal(cache, want_cache) and np.array_equal(scale.view(np.uint16), want_scale.view(np.uint16))


# ---- far ends and graphs

def test_everything_past_2_to_the_32_bytes():
    """The same sequences at the far end of a slab of 4.6 GB: same outputs, bit for bit, as at the front of a small one."""
    c = Case(8, 2, 128, [5, 12, 40], [300, 31, 900], seed=21)
    see = trees(c)
    near = Device(c)
    far = Device(c)
    torch = far.torch
    off = 9_000_000  # tokens in front
    first = off * c.stride_s
    assert first > 2 ** 32
    far.cache = torch.empty(first + c.cache.size, dtype=torch.int8, device="cuda")
    far.scale = torch.empty(first // 8 + c.scale.size, dtype=torch.float16, device="cuda")
    far.cache[first:] = near.cache
    far.scale[first // 8:] = near.scale
    far.cachestarts = near.cachestarts + off
    n_out, n_lse = near.tree(mask_words(see, 1), 1)
    f_out, f_lse = far.tree(mask_words(see, 1), 1)
    assert np.array_equal(n_out, f_out) and np.array_equal(n_lse, f_lse)
    score = c.rng.lognormal(0, 1, (1, 2, c.tokens)).astype(np.float32)
    position = np.zeros((1, 2, c.tokens), np.int32)
    for b in range(3):
        position[:, :, c.tok[b]] = np.arange(c.kvlen[b])
    pad = lambda x: np.concatenate([np.zeros((1, 2, off), x.dtype), x], axis=2)
    pidx = c.rng.integers(0, 9999, int(c.new.sum()))
    n_s, n_p = near.score(n_lse, score, pidx, True, position)
    f_s, f_p = far.score(n_lse, pad(score), pidx, True, pad(position))
    assert np.array_equal(f_s[:, :, off:], n_s) and np.array_equal(f_p[:, :, off:], n_p) and not f_s[:, :, :off].any()
    n = near.accept([[1, 3], [0, 4], [2, 30]], [2, 2, 2], 2)[0]
    far.accept([[1, 3], [0, 4], [2, 30]], [2, 2, 2], 2)
    assert np.array_equal(far.cache[first:].cpu().numpy(), n)
    near.evict(n_s, n_p, [200, 20, 500], c.kvlen, 4, 30)
    far.evict(pad(n_s), pad(n_p), [200, 20, 500], c.kvlen, 4, 30)
    assert np.array_equal(far.cache[first:].cpu().numpy(), near.cache.cpu().numpy())
    assert np.array_equal(far.scale[first // 8:].cpu().numpy().view(np.uint16), near.scale.cpu().numpy().view(np.uint16))


def test_upkeep_replays_from_a_graph():
    """Weights, then eviction by them, captured together on a stream of their own: every replay leaves what the eager calls
    left (the scores go to arrays of their own, so a replay finds what the first call found)."""
    import torch
    c = Case(8, 2, 64, [4, 9], [700, 90], seed=22)
    lse = cache_ops.exact_attention(c, [causal(4), causal(9)])[2]
    score, position = evict_inputs(c)
    pidx = 2 * np.concatenate([c.old[b] + np.arange(c.new[b]) for b in range(2)])
    want = Device(c)
    s, p = want.score(lse, score, pidx, False, position)
    mid = np.where(s == -5.0, score, s)
    w_cache, w_scale, w_s, w_p, w_n = want.evict(mid, p, [300, 50], 2 * c.kvlen, 2, 40, in_place=False)
    d = Device(c)
    e = d.evict_args(score, position, [300, 50], 2 * c.kvlen, 2, 40, 0, 1, False)  # (holds score as d.s_in)
    d.lse_in, d.pos_idx = d.up(lse.astype(np.float32)), d.up(pidx)
    d.s_mid, d.pos = d.s_in.clone(), d.up(position)
    a = d.query_args(cabi.KvScoreArgs())
    a.d_lse, a.d_position_idx, a.d_position = d.ptr(d.lse_in), d.ptr(d.pos_idx), d.ptr(d.pos)
    a.d_score_in, a.d_score_out = d.ptr(d.s_in), d.ptr(d.s_mid)
    a.score_stride_l, a.score_stride_h = c.kv_heads * c.tokens, c.tokens
    e.d_score_in, e.d_position_in = d.ptr(d.s_mid), d.ptr(d.pos)
    plan = cabi.KvEvictPlan()
    pkg.check(d.lib.pplhip_kv_evict_prepare(C.byref(e), C.byref(plan)))
    ws = torch.empty(max(256, plan.workspace_bytes), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st = torch.cuda.current_stream().cuda_stream
        pkg.check(d.lib.pplhip_kv_score_accumulate(C.byref(a), st))
        pkg.check(d.lib.pplhip_kv_evict(C.byref(e), C.byref(plan), ws.data_ptr(), st))
    for _ in range(4):
        d.cache.copy_(d.up(c.cache))
        d.scale.copy_(d.up(c.scale))
        d.s_out.fill_(-5.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(d.cache.cpu().numpy(), w_cache)
        assert np.array_equal(d.scale.cpu().numpy().view(np.uint16), w_scale.view(np.uint16))
        assert np.array_equal(d.s_out.cpu().numpy(), w_s) and np.array_equal(d.p_out.cpu().numpy(), w_p)
        assert np.array_equal(d.new_kvlen.cpu().numpy()[:2], w_n)


@pytest.mark.parametrize("scale", [6.0, 40.0])
def test_tree_reference_points_move_often(scale):
    """Keys that grow along the sequence: the largest score moves up again and again, in every row at its own keys."""
    for heads, new in ((4, 3), (8, 9), (16, 20), (32, 30), (64, 60)):
        c = Case(heads, 1, 128, [new], [1500], seed=new)
        c.query = (c.query * (scale / 6)).astype(np.float16)
        r = c.rows(c.tok[0], 0, 0, 0).ravel()
        ramp = (0.002 + 0.02 * np.linspace(0, 1, len(r))).astype(np.float16)
        c.scale[(r // 8)[:, None] + np.arange(16)] = ramp[:, None]
        check_tree(c, trees(c))


# ---- together

def test_speculative_steps_with_a_bounded_cache():
    """Draft, write, verify, accept, accumulate, evict, and again: after every stage the device holds what the
    definitions give for the stage's inputs."""
    heads, kv_heads, dim, layers = 8, 2, 64, 2
    rng = np.random.default_rng(42)
    old = np.array([60, 7, 130])
    next_pos = old.copy()
    new = np.array([9, 5, 12])
    c = Case(heads, kv_heads, dim, new, old, layers=layers, slack=40, seed=42)
    score = np.abs(rng.standard_normal((layers, kv_heads, c.tokens))).astype(np.float32)
    position = np.full((layers, kv_heads, c.tokens), -1, np.int32)
    for b in range(3):
        position[:, :, c.tok[b][:old[b]]] = np.arange(old[b])
    d = Device(c)
    torch = d.torch
    for step in range(3):
        see = [random_tree(rng, int(n)) for n in c.new]
        paths = []
        for b in range(3):  # a path from a root to a random node
            node = int(rng.integers(0, c.new[b]))
            paths.append([int(x) for x in np.flatnonzero(see[b][node])])
        # the drafted tokens go into the slab (both layers), through the library's own write
        key = rng.standard_normal((layers, int(c.new.sum()), kv_heads, dim)).astype(np.float16)
        value = rng.standard_normal(key.shape).astype(np.float16)
        for layer in range(layers):
            w = cabi.KvWriteArgs()
            k_dev, v_dev = d.up(key[layer]), d.up(value[layer])
            c.layer = layer
            d.slab_args(w)
            w.d_current_key, w.d_current_value = d.ptr(k_dev), d.ptr(v_dev)
            w.d_seqstarts, w.d_start_pos, w.total_new_tokens = d.ptr(d.seqstarts), d.ptr(d.start_pos), int(c.new.sum())
            pkg.check(d.lib.pplhip_kv_quantize_write(C.byref(w), d.stream()), "write")
        torch.cuda.synchronize()
        c.cache, c.scale = d.cache.cpu().numpy(), d.scale.cpu().numpy()
        got = []
        for layer in range(layers):
            c.layer = layer
            o, l = d.tree(mask_words(see, 1), 1)
            eo, et, el, elt = cache_ops.exact_attention(c, see)
            assert_within(o, eo, et, f"step {step} layer {layer}")
            assert_within(l, el, elt, f"step {step} layer {layer} lse")
            got.append(l)
        table = np.zeros((3, 12), np.int64)
        for b, p in enumerate(paths):
            table[b, :len(p)] = p
        cache, scale = d.accept(table, [len(p) for p in paths], 12)
        e_cache, e_scale = cache_ops.exact_accept(c, paths, 0, layers)
        assert np.array_equal(cache, e_cache) and np.array_equal(scale.view(np.uint16), e_scale.view(np.uint16))
        # the accepted tokens are now a run behind the cached ones: their rows of the queries and log-sums count
        pick = np.concatenate([c.seqstarts[b] + np.array(paths[b]) for b in range(3)])
        pos = np.concatenate([next_pos[b] + np.arange(len(paths[b])) for b in range(3)])
        c2 = Case(heads, kv_heads, dim, [len(p) for p in paths], c.old, layers=layers, seed=0)
        c2.cachestarts, c2.tokens, c2.stride_s, c2.stride_l = c.cachestarts, c.tokens, c.stride_s, c.stride_l
        c2.stride_h, c2.stride_kv = c.stride_h, c.stride_kv
        c2.tok = [c.tok[b][:c2.kvlen[b]] for b in range(3)]
        c2.cache, c2.scale, c2.query = cache, scale, c.query[pick]
        d2 = Device(c2)
        for layer in range(layers):
            c2.layer = layer
            s, position = d2.score(got[layer][pick], score, pos, True, position)
            want, tol = cache_ops.exact_score(c2, got[layer][pick], score[layer])
            assert_within(s[layer], want, tol, f"step {step} layer {layer} score")
            score = s
        c2.layer = 0
        next_pos = next_pos + [len(p) for p in paths]
        target = np.array([64, 64, 100])
        want = cache_ops.exact_evict(c2, score, position, target, next_pos, 2, 16, 0, layers)
        cache, scale, score, position, kvlen = d2.evict(score, position, target, next_pos, 2, 16)
        for got_x, want_x in zip((cache, scale.view(np.uint16), score, position, kvlen),
                                 (want[0], want[1].view(np.uint16), want[2], want[3], want[4])):
            assert np.array_equal(got_x, want_x)
        # next step's batch over the same slab
        new = rng.integers(1, 13, 3)
        n = Case(heads, kv_heads, dim, new, kvlen, layers=layers, seed=step)
        n.cachestarts, n.tokens, n.stride_s, n.stride_l = c.cachestarts, c.tokens, c.stride_s, c.stride_l
        n.stride_h, n.stride_kv = c.stride_h, c.stride_kv
        n.tok = [c.cachestarts[b] + np.arange(n.kvlen[b]) for b in range(3)]
        n.cache, n.scale = cache, scale
        c, d = n, Device(n)


def test_calls_on_two_streams_at_once():
    """Two batches over slabs of their own: attention and eviction, a workspace each, enqueued on two streams without a
    wait between them. Each gives what it gives alone."""
    import torch
    cases = [Case(32, 8, 128, [1, 9, 30], [3000, 17, 1500], seed=31), Case(8, 2, 64, [20, 3], [900, 2200], page=64, seed=32)]
    alone, runs = [], []
    for c in cases:
        see, (score, position) = trees(c), evict_inputs(c)
        upkeep = (score, position, c.kvlen // 2, 2 * c.kvlen, 2, 10)
        d = Device(c)
        alone.append(d.tree(mask_words(see, 1), 1) + d.evict(*upkeep))
        d = Device(c)
        a = d.tree_args(mask_words(see, 1), 1)
        plan, ws = d.tree_plan(a)
        e = d.evict_args(*upkeep, 0, c.layers, True)
        e_plan = cabi.KvEvictPlan()
        pkg.check(d.lib.pplhip_kv_evict_prepare(C.byref(e), C.byref(e_plan)))
        e_ws = torch.full((max(256, e_plan.workspace_bytes),), 0xFF, dtype=torch.uint8, device="cuda")
        runs.append((d, a, plan, ws, e, e_plan, e_ws, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for d, a, plan, ws, e, e_plan, e_ws, s in runs:
        pkg.check(d.lib.pplhip_tree_attention_forward(C.byref(a), C.byref(plan), ws.data_ptr(), s.cuda_stream))
    for d, a, plan, ws, e, e_plan, e_ws, s in runs:
        pkg.check(d.lib.pplhip_kv_evict(C.byref(e), C.byref(e_plan), e_ws.data_ptr(), s.cuda_stream))
    torch.cuda.synchronize()
    for c, want, (d, *_) in zip(cases, alone, runs):
        n = int(c.new.sum())
        got = (d.out[:n], d.lse[:n], d.cache, d.scale, d.s_out, d.p_out, d.new_kvlen[:c.batch])
        for i, (g, w) in enumerate(zip(got, want)):
            assert g.cpu().numpy().tobytes() == w.tobytes(), i


def test_tree_padded_batch():
    """More rows of queries than the tables speak of (a batch padded to a fixed size, its last sequences empty) and longer
    bounds than any sequence reaches: the same rows, nothing written behind them."""
    c = Case(8, 2, 128, [5, 12, 0, 0], [700, 90, 0, 40], seed=33)
    see = trees(c)
    d = Device(c)
    want, want_lse = d.tree(mask_words(see, 1), 1)
    d.query = d.up(np.concatenate([c.query, np.full((47,) + c.query.shape[1:], np.nan, np.float16)]))
    words = mask_words(see, 1)
    a = d.tree_args(np.concatenate([words, np.full((47, 1), 2 ** 64 - 1, np.uint64)]), 1, extra_rows=47)
    a.total_new_tokens, a.max_seqlen, a.max_kvlen = 64, 64, 4096
    plan, ws = d.tree_plan(a)
    pkg.check(d.lib.pplhip_tree_attention_forward(C.byref(a), C.byref(plan), ws.data_ptr(), d.stream()))
    out, lse = d.out.cpu().numpy(), d.lse.cpu().numpy()
    assert (out[17:] == 7.0).all() and (lse[17:] == 7.0).all()
    ref, tol, ref_lse, lse_tol = cache_ops.exact_attention(c, see)
    assert_within(out[:17], ref, tol, "output")
    assert_within(lse[:17], ref_lse, lse_tol, "lse")
    assert_within(want, ref, tol, "output of exact bounds")


@pytest.mark.parametrize("ties,nan", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_long_beside_short(ties, nan, in_place):
    """A column several workgroups share beside columns of one of their parts, of a few tokens and of none; some keep
    everything, nothing, or all but one."""
    kv = [20000, 4096, 4097, 3, 0, 8192, 17000, 16500]
    keep = [9000, 100, 4097, 1, 0, 8191, 0, 20000]
    check_evict(Case(2, 2, 16, [1 if n else 0 for n in kv], [max(0, n - 1) for n in kv], layers=2, page=64, seed=34), keep,
                sinks=3, recent=100, in_place=in_place, ties=ties, nan=nan)


@pytest.mark.parametrize("n,keep", [(65536, 40000), (65537, 30000), (262144, 262143), (262145, 131072), (300000, 1)])
def test_evict_longest(n, keep):
    """Either side of where a workgroup's registers, and the largest number of one-block parts, end."""
    check_evict(Case(1, 1, 16, [1], [n - 1], seed=35), [keep], sinks=4, recent=1000)


def test_evict_many_long_columns():
    """147 columns: each longer than 16 384 tokens, and more than several workgroups a column pay for."""
    check_evict(Case(7, 7, 16, [1, 1, 1], [17000, 20001, 900], layers=7, seed=36), [16900, 19999, 850], sinks=4, recent=64)


def test_evict_longer_than_announced():
    """A table that speaks of more tokens than max_kvlen: the first max_kvlen are looked at, the rest left alone."""
    c = Case(2, 2, 16, [1], [999], seed=37)
    score, position = evict_inputs(c)
    d = Device(c)
    a = d.evict_args(score, position, [300], [2000], 0, 0, 0, 1, True)
    a.max_kvlen = 600
    plan = cabi.KvEvictPlan()
    pkg.check(d.lib.pplhip_kv_evict_prepare(C.byref(a), C.byref(plan)))
    ws = d.torch.empty(plan.workspace_bytes, dtype=d.torch.uint8, device="cuda")
    pkg.check(d.lib.pplhip_kv_evict(C.byref(a), C.byref(plan), ws.data_ptr(), d.stream()))
    c.kvlen[0] = 600
    c.tok[0] = c.tok[0][:600]
    e_cache, e_scale, e_s, e_p, e_n = cache_ops.exact_evict(c, score, position, [300], [2000], 0, 0, 0, 1)
    assert np.array_equal(d.cache.cpu().numpy(), e_cache) and np.array_equal(d.s_out.cpu().numpy(), e_s)
    assert np.array_equal(d.p_out.cpu().numpy(), e_p) and int(d.new_kvlen[0]) == 300


# ---- every kernel at every padded head size

HEAD_DIMS = list(range(16, 257, 16))


@pytest.mark.parametrize("rows", [16, 17, 33, 65, 129, 257])
@pytest.mark.parametrize("dim", HEAD_DIMS)
def test_tree_row_tiles(dim, rows):
    """Row counts that select each row tile, one more than a tile holds among them, at every head size: by mask, causal."""
    c = Case(2, 2, dim, [rows, rows // 2, 1], [45, 0, 130], seed=1000 * dim + rows)
    check_tree(c, trees(c), junk=True)
    check_tree(c)


def spoil(c, b, new_token, bits, kv=slice(None)):
    """Gives the scales of a new token's rows these fp16 bits."""
    r = c.rows(c.tok[b][c.old[b] + new_token], c.layer, slice(None), kv).ravel()
    c.scale.view(np.uint16)[(r // 8)[:, None] + np.arange(c.dim // 8)] = bits


@pytest.mark.parametrize("rows", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", HEAD_DIMS)
def test_tree_hidden_tokens_in_every_row_tile(dim, rows):
    """Tokens that nobody else sees with NaN and infinite scales, one that sees itself, and one with values near fp16's
    largest that others do see; a sequence without history and one whose new tokens share a key tile with it."""
    c = Case(2, 2, dim, [rows, rows, 3], [0, 50, 9], seed=1000 * dim + rows)
    see = trees(c)
    for b in (0, 1):
        for x, bits in ((3, 0x7E00), (rows // 2, 0x7C00), (rows - 1, 0xFC00)):
            see[b][:, x] = False
            spoil(c, b, x, bits)
        see[b][3, 3] = True
        spoil(c, b, 5, np.float16(514.0).view(np.uint16), 1)
    got, _ = check_tree(c, see)
    assert np.isnan(got[3]).all() and np.isfinite(np.delete(got, [3, rows + 3], axis=0)).all()


@pytest.mark.parametrize("rows", [5, 20, 50, 100, 200])
def test_tree_infinite_values_that_are_seen(rows):
    """An infinite value row, in front of the new tokens and among them, reaches those that see it, with its signs."""
    c = Case(2, 1, 128, [rows], [100], seed=rows)
    c.cache[c.cache == 0] = 1  # (0 times infinity has no sign)
    see = trees(c)
    spoil(c, 0, 4, 0x7C00, 1)
    check_tree(c, see)
    spoil(c, 0, -37, 0x7C00, 1)
    got, _ = check_tree(c, see)
    assert not np.isfinite(got).any()


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 1, 128), (2, 2, 256), (3, 3, 80)])
def test_tree_whole_prompts(heads, kv_heads, dim):
    c = Case(heads, kv_heads, dim, [600, 1, 333], [0, 50, 77], seed=dim)
    check_tree(c)


@pytest.mark.parametrize("dim", HEAD_DIMS)
def test_score_head_dims(dim):
    check_score(Case(4, 2, dim, [5, 1, 0, 70], [70, 0, 20, 300], seed=dim))


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (3, 3, 192)])
def test_score_whole_prompts(heads, kv_heads, dim):
    check_score(Case(heads, kv_heads, dim, [600, 333], [0, 77], seed=dim))


@pytest.mark.parametrize("columns", [96, 97])
def test_evict_long_without_positions(columns):
    """Either side of where several workgroups choose from a long column."""
    c = Case(1, 1, 16, [1] * columns, [17000] + [200] * (columns - 1), seed=columns)
    check_evict(c, [9000] + [100] * (columns - 1), positions=False)


def test_score_padded_batch():
    """Rows behind the last sequence hold NaN, the last sequences are empty, the bounds are longer than any sequence."""
    c = Case(8, 2, 128, [5, 130, 0, 0], [700, 90, 0, 40], seed=61)
    lse = cache_ops.exact_attention(c, [causal(int(n)) for n in c.new])[2].astype(np.float32)
    score = np.abs(c.rng.standard_normal((1, 2, c.tokens))).astype(np.float32)
    want, want_pos = Device(c).score(lse, score, np.arange(135), False, np.full(score.shape, -3, np.int32))
    d = Device(c)
    d.query = d.up(np.concatenate([c.query, np.full((57,) + c.query.shape[1:], np.nan, np.float16)]))
    a = d.query_args(cabi.KvScoreArgs())
    a.total_new_tokens, a.max_seqlen, a.max_kvlen = 192, 192, 4096
    lse_dev = d.up(np.concatenate([lse, np.full((57, 8), np.nan, np.float32)]))
    s_in, s_out = d.up(score), d.up(np.full_like(score, -5.0))
    idx, pos = d.up(np.concatenate([np.arange(135), np.full(57, -9)])), d.up(np.full(score.shape, -3, np.int32))
    a.d_lse, a.d_position_idx, a.d_position = d.ptr(lse_dev), d.ptr(idx), d.ptr(pos)
    a.d_score_in, a.d_score_out = d.ptr(s_in), d.ptr(s_out)
    a.score_stride_l, a.score_stride_h = 2 * c.tokens, c.tokens
    pkg.check(d.lib.pplhip_kv_score_accumulate(C.byref(a), d.stream()))
    assert np.array_equal(s_out.cpu().numpy(), want) and np.array_equal(pos.cpu().numpy(), want_pos)


@pytest.mark.parametrize("n", [700, 17000])
@pytest.mark.parametrize("scores_in_place", [True, False])
def test_evict_one_of_scores_and_positions_in_place(n, scores_in_place):
    c = Case(2, 2, 16, [1, 1], [n - 1, 50], seed=n)
    score, position = evict_inputs(c)
    keep = [n // 3, 20]
    d = Device(c)
    a = d.evict_args(score, position, keep, 2 * c.kvlen, 2, 30, 0, 1, False)
    if scores_in_place:
        a.d_score_out = a.d_score_in
    else:
        a.d_position_out = a.d_position_in
    plan = cabi.KvEvictPlan()
    pkg.check(d.lib.pplhip_kv_evict_prepare(C.byref(a), C.byref(plan)))
    ws = d.torch.full((plan.workspace_bytes,), 0xFF, dtype=d.torch.uint8, device="cuda")
    pkg.check(d.lib.pplhip_kv_evict(C.byref(a), C.byref(plan), ws.data_ptr(), d.stream()))
    e_cache, e_scale, e_s, e_p, e_n = cache_ops.exact_evict(c, score, position, keep, 2 * c.kvlen, 2, 30, 0, 1)
    assert np.array_equal(d.cache.cpu().numpy(), e_cache)
    got_s, got_p = (d.s_in, d.p_out) if scores_in_place else (d.s_out, d.p_in)
    for b in range(2):
        t = c.tok[b][:int(e_n[b])]
        assert np.array_equal(got_s.cpu().numpy()[:, :, t], e_s[:, :, t])
        assert np.array_equal(got_p.cpu().numpy()[:, :, t], e_p[:, :, t])
        t = c.tok[b][int(e_n[b]):]
        same = (got_s, score) if scores_in_place else (got_p, position)
        assert np.array_equal(same[0].cpu().numpy()[:, :, t], same[1][:, :, t])
