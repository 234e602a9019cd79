"""Refusals and plans of the operators that put several new tokens over the int8 slab or keep the slab up: everything
here is decided on the host, before any device is touched."""
import ctypes as C
import os
import re

import pytest

import cache_ops
from cache_ops import cabi

P = 0x10000  # an aligned, never dereferenced address


def slab(a, layers=4, kv_heads=8, dim=128, batch=3):
    a.d_cachestarts, a.batch, a.num_layer, a.layer_idx = P, batch, layers, 1
    a.num_kv_heads, a.head_dim, a.cache_mode, a.page_size = kv_heads, dim, 0, 128
    for k, v in cabi.cache_strides_layout0(layers, kv_heads, dim).items():
        setattr(a, k, v)
    a.d_cache, a.d_scale = P, P
    return a


def tree():
    a = slab(cabi.TreeAttentionArgs())
    a.d_query = a.d_output = a.d_lse = a.d_seqstarts = a.d_kvstarts = a.d_tree_mask = P
    a.num_heads, a.total_new_tokens, a.max_seqlen, a.max_kvlen, a.tree_mask_words = 32, 20, 10, 500, 1
    return a


def score():
    a = slab(cabi.KvScoreArgs())
    a.d_query = a.d_lse = a.d_seqstarts = a.d_kvstarts = a.d_score_in = a.d_score_out = a.d_position = a.d_position_idx = P
    a.num_heads, a.total_new_tokens, a.max_seqlen, a.max_kvlen = 32, 20, 10, 500
    a.score_stride_l, a.score_stride_h = 8 * 4096, 4096
    return a


def evict():
    a = slab(cabi.KvEvictArgs())
    a.d_kvstarts = a.d_target_kvlen = a.d_next_pos = a.d_score_in = a.d_score_out = a.d_new_kvlen = P
    a.d_position_in = a.d_position_out = P
    a.max_kvlen, a.num_sink, a.num_recent, a.layer_count = 500, 4, 64, 2
    a.score_stride_l, a.score_stride_h = 8 * 4096, 4096
    return a


def accept():
    a = slab(cabi.KvAcceptArgs())
    a.d_seqstarts = a.d_start_pos = a.d_accepted = a.d_accepted_len = P
    a.accepted_stride_b, a.max_accepted, a.layer_count = 8, 6, 2
    return a


def call(lib, a, plan=None):
    """The refusals come from the call that enqueues; with a null workspace and a fresh plan none of them enqueues."""
    if isinstance(a, cabi.TreeAttentionArgs):
        return lib.pplhip_tree_attention_prepare(C.byref(a), C.byref(plan or cabi.TreeAttentionPlan()))
    if isinstance(a, cabi.KvScoreArgs):
        return lib.pplhip_kv_score_accumulate(C.byref(a), None)
    if isinstance(a, cabi.KvEvictArgs):
        return lib.pplhip_kv_evict_prepare(C.byref(a), C.byref(plan or cabi.KvEvictPlan()))
    return lib.pplhip_kv_accept(C.byref(a), None)


INVALID, UNSUPPORTED, RANGE = cabi.RC_INVALID_VALUE, cabi.RC_UNSUPPORTED, cabi.RC_OUT_OF_RANGE


@pytest.mark.parametrize("make", [tree, score, evict, accept])
@pytest.mark.parametrize("field,value,rc", [
    ("d_cache", None, INVALID), ("d_scale", None, UNSUPPORTED), ("d_cache", P + 8, INVALID), ("d_scale", P + 2, INVALID),
    ("head_dim", 0, UNSUPPORTED), ("head_dim", 72, UNSUPPORTED), ("head_dim", 272, UNSUPPORTED),
    ("num_kv_heads", 0, INVALID), ("layer_idx", -1, INVALID), ("layer_idx", 4, INVALID), ("num_layer", 0, INVALID),
    ("cache_stride_s", 0, INVALID), ("cache_stride_s", 8200, INVALID), ("cache_stride_h", 24, INVALID),
    ("cache_stride_s", 1 << 25, UNSUPPORTED), ("cache_mode", 2, UNSUPPORTED), ("batch", -1, INVALID),
    ("batch", 1 << 31, RANGE), ("d_cachestarts", None, INVALID),
])
def test_slab_refusals(hiplib, make, field, value, rc):
    a = make()
    setattr(a, field, value)
    assert call(hiplib, a) == rc
    assert hiplib.pplhip_last_error()


@pytest.mark.parametrize("make", [tree, score, evict, accept])
def test_paged_refusals(hiplib, make):
    a = make()
    a.cache_mode, a.page_size, a.cachestart_stride_b = 1, 128, 0
    assert call(hiplib, a) == INVALID
    a.cachestart_stride_b = 4
    for bad in (0, 32, 96):
        a.page_size = bad
        assert call(hiplib, a) == UNSUPPORTED


@pytest.mark.parametrize("make", [tree, score])
@pytest.mark.parametrize("field,value", [
    ("num_heads", 0), ("num_heads", 12), ("total_new_tokens", -1), ("max_seqlen", -1), ("max_seqlen", 21), ("max_kvlen", 9),
    ("d_query", None), ("d_query", P + 8), ("d_seqstarts", None), ("d_kvstarts", None), ("d_lse", P + 2),
])
def test_query_refusals(hiplib, make, field, value):
    a = make()
    setattr(a, field, value)
    assert call(hiplib, a) == INVALID


@pytest.mark.parametrize("field,value", [("d_output", None), ("d_output", P + 2), ("d_tree_mask", P + 4),
                                         ("tree_mask_words", 0), ("tree_mask_words", -1)])
def test_tree_refusals(hiplib, field, value):
    a = tree()
    setattr(a, field, value)
    assert call(hiplib, a) == INVALID


def test_tree_mask_has_to_cover_the_longest_sequence(hiplib):
    a = tree()
    a.total_new_tokens, a.max_seqlen = 100, 65
    assert call(hiplib, a) == INVALID
    a.tree_mask_words = 2
    assert call(hiplib, a) == cabi.RC_SUCCESS
    a.d_tree_mask, a.tree_mask_words = None, 0  # causal: no words
    assert call(hiplib, a) == cabi.RC_SUCCESS


def test_tree_plans(hiplib):
    a, plan = tree(), cabi.TreeAttentionPlan()
    assert call(hiplib, a, plan) == cabi.RC_SUCCESS
    assert plan.num_ranges >= 1 and plan.row_tile % 16 == 0 and plan.workspace_bytes % 256 == 0
    fwd = lambda p, ws: hiplib.pplhip_tree_attention_forward(C.byref(a), C.byref(p), ws, None)
    assert fwd(plan, None) == INVALID and fwd(plan, P + 16) == INVALID
    other = cabi.TreeAttentionPlan(plan.workspace_bytes, plan.num_ranges, plan.row_tile + 16)
    assert fwd(other, P) == INVALID
    other = cabi.TreeAttentionPlan(plan.workspace_bytes, plan.num_ranges * 2, plan.row_tile)
    assert fwd(other, P) == INVALID
    assert fwd(cabi.TreeAttentionPlan(), P) == INVALID
    # no sequences or no tokens: nothing to do, whatever the pointers
    for field in ("batch", "total_new_tokens"):
        b = tree()
        setattr(b, field, 0)
        b.max_seqlen = 0
        b.d_query = b.d_output = None
        assert call(hiplib, b, plan) == cabi.RC_SUCCESS and plan.workspace_bytes == 0
        assert hiplib.pplhip_tree_attention_forward(C.byref(b), C.byref(plan), None, None) == cabi.RC_SUCCESS
    for f in (hiplib.pplhip_tree_attention_prepare,):
        assert f(None, C.byref(plan)) == INVALID and f(C.byref(a), None) == INVALID


@pytest.mark.parametrize("field,value", [("d_lse", None), ("d_score_in", None), ("d_score_out", None), ("d_score_in", P + 2),
                                         ("d_position", None), ("d_position_idx", None), ("d_position_idx", P + 4),
                                         ("score_stride_l", -1), ("score_stride_h", -1)])
def test_score_refusals(hiplib, field, value):
    a = score()
    setattr(a, field, value)
    assert call(hiplib, a) == INVALID


@pytest.mark.parametrize("field,value,rc", [
    ("layer_count", 0, INVALID), ("layer_count", 4, INVALID), ("num_sink", -1, INVALID), ("num_recent", -1, INVALID),
    ("max_kvlen", -1, INVALID), ("max_kvlen", 1 << 31, RANGE), ("d_kvstarts", None, INVALID),
    ("d_target_kvlen", None, INVALID), ("d_next_pos", None, INVALID), ("d_score_in", None, INVALID),
    ("d_score_out", None, INVALID), ("d_new_kvlen", None, INVALID), ("d_position_in", None, INVALID),
    ("d_position_out", None, INVALID), ("score_stride_h", -1, INVALID), ("d_score_out", P + 1, INVALID),
    ("batch", 1 << 28, RANGE),
])
def test_evict_refusals(hiplib, field, value, rc):
    a = evict()
    setattr(a, field, value)
    assert call(hiplib, a) == rc


def test_evict_plans(hiplib):
    a, plan = evict(), cabi.KvEvictPlan()
    assert call(hiplib, a, plan) == cabi.RC_SUCCESS and plan.max_moves == 250
    run = lambda p, ws: hiplib.pplhip_kv_evict(C.byref(a), C.byref(p), ws, None)
    assert run(plan, None) == INVALID and run(plan, P + 128) == INVALID and run(cabi.KvEvictPlan(), P) == INVALID
    a.max_kvlen = 502
    assert run(plan, P) == INVALID
    a.num_sink = a.num_recent = 0
    a.d_position_in = a.d_position_out = a.d_next_pos = None
    assert call(hiplib, a, plan) == cabi.RC_SUCCESS
    a.batch = 0
    assert run(plan, None) == cabi.RC_SUCCESS


@pytest.mark.parametrize("field,value", [("layer_count", 0), ("layer_count", 4), ("max_accepted", -1), ("max_accepted", 9),
                                         ("d_seqstarts", None), ("d_start_pos", None), ("d_accepted", None),
                                         ("d_accepted_len", None)])
def test_accept_refusals(hiplib, field, value):
    a = accept()
    setattr(a, field, value)
    assert call(hiplib, a) == INVALID


def test_null_blocks(hiplib):
    assert hiplib.pplhip_kv_score_accumulate(None, None) == INVALID
    assert hiplib.pplhip_kv_accept(None, None) == INVALID
    assert hiplib.pplhip_kv_evict_prepare(None, None) == INVALID
    assert hiplib.pplhip_tree_attention_forward(None, None, None, None) == INVALID


@pytest.mark.parametrize("cname,cls", [
    ("pplhip_tree_attention_args", cabi.TreeAttentionArgs), ("pplhip_tree_attention_plan", cabi.TreeAttentionPlan),
    ("pplhip_kv_score_args", cabi.KvScoreArgs), ("pplhip_kv_evict_args", cabi.KvEvictArgs),
    ("pplhip_kv_evict_plan", cabi.KvEvictPlan), ("pplhip_kv_accept_args", cabi.KvAcceptArgs)])
def test_ctypes_mirrors_match_the_header(cname, cls):
    """Names, order and types: pointers are pointers, i32 / i64 / u64 have their widths."""
    with open(os.path.join(os.path.dirname(__file__), "..", "include", "ppl_llm_kernel_hip.h")) as f:
        txt = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), txt, flags=re.S).group(1)
    want = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, name = decl.rsplit(None, 1)
        if "*" in decl:
            ctype = C.c_void_p
        else:
            ctype = {"int32_t": C.c_int32, "int64_t": C.c_int64, "uint64_t": C.c_uint64}[kind]
        want.append((name.lstrip("*"), ctype))
    assert want == list(cls._fields_)


def test_evict_lists_that_fit_no_device(hiplib):
    """2^31 - 1 columns of 2^31 - 1 tokens: the lists' size would pass 64 bits."""
    a = evict()
    a.num_kv_heads, a.layer_count, a.batch, a.max_kvlen = 1, 1, 0x7fffffff, 0x7fffffff
    assert call(hiplib, a) == RANGE
    a.batch = 64
    assert call(hiplib, a) == cabi.RC_SUCCESS


def many_heads(a, heads):
    a.num_heads = a.num_kv_heads = heads
    return a


def test_launches_of_2_to_the_32_threads(hiplib):
    """A launch has less than 2^32 threads along its axis: what would need more is refused before anything is enqueued
    (of the calls that would enqueue only the refused side is looked at), by prepare as well."""
    a = score()  # 512 blocks of keys x 4096 sequences x 8 kv heads = 2^24 workgroups of 256
    a.max_kvlen, a.batch = 131072, 4096
    assert call(hiplib, a) == RANGE
    a = accept()  # two workgroups a sequence
    a.layer_idx, a.layer_count, a.batch = 0, 4, 1 << 23
    assert call(hiplib, a) == RANGE
    a = accept()  # (the rows' count itself would pass 64 bits)
    a.layer_idx, a.layer_count, a.num_layer, a.num_kv_heads = 0, 0x7fffffff, 0x7fffffff, 0x7fffffff
    assert call(hiplib, a) == RANGE
    # columns: 16 a sequence; workgroups of 256 and 1024 threads, and 17 of 256 a column
    for kvlen, batch in ((500, 1 << 20), (5000, 1 << 18), (20000, 1 << 18), (65537, 61681)):
        a = evict()
        a.max_kvlen, a.batch = kvlen, batch
        assert call(hiplib, a) == RANGE, kvlen
        a.batch -= 1
        assert call(hiplib, a) == cabi.RC_SUCCESS, kvlen
    # one range: workgroups of 256 threads, of 512 for tiles of 256 rows
    for seqlen, heads in ((10, 1 << 24), (200, 1 << 23)):
        a = many_heads(tree(), heads)
        a.total_new_tokens = a.max_seqlen = seqlen
        a.d_tree_mask = None
        assert call(hiplib, a) == RANGE, seqlen
        assert call(hiplib, many_heads(a, heads - 1)) == cabi.RC_SUCCESS, seqlen
    plan = cabi.TreeAttentionPlan()  # a plan of more ranges than prepare would make
    a = tree()
    assert call(hiplib, a, plan) == cabi.RC_SUCCESS
    big = cabi.TreeAttentionPlan(1 << 62, 1 << 21, plan.row_tile)
    assert hiplib.pplhip_tree_attention_forward(C.byref(a), C.byref(big), None, None) == INVALID
    assert b"plan" in hiplib.pplhip_last_error()


@pytest.mark.parametrize("kvlen", [16385, 40000, 65536])
def test_evict_workspace_holds_what_the_call_uses(hiplib, kvlen):
    """Up to 96 columns several workgroups choose from one and keep its keys in the workspace; above that, up to 65 536
    tokens, one does, and only the lists of moves (their count, holes, fillers) are there. A plan for a large batch also
    serves a smaller one, whose columns are shared."""
    a, plan = evict(), cabi.KvEvictPlan()
    a.max_kvlen, a.num_layer, a.layer_idx, a.layer_count, a.num_kv_heads, a.batch = kvlen, 1, 0, 1, 1, 96
    lists = lambda columns: -(-columns * (1 + 2 * (kvlen // 2)) * 4 // 256) * 256
    assert call(hiplib, a, plan) == cabi.RC_SUCCESS
    shared = plan.workspace_bytes
    assert shared >= lists(96) + 96 * kvlen * 4
    for columns in (97, 150, 4096):
        a.batch = columns
        assert call(hiplib, a, plan) == cabi.RC_SUCCESS
        assert plan.workspace_bytes == max(shared, lists(columns))
        for fewer in (1, 96, 97):
            a.batch = min(fewer, columns)
            assert hiplib.pplhip_kv_evict(C.byref(a), C.byref(plan), None, None) == INVALID
            assert b"workspace" in hiplib.pplhip_last_error()  # not the plan
