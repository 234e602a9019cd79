"""What the speculative-decoding and bounded-cache operators are measured on: attention of drafted token trees over the
int8 cache, the accumulated attention weight of every cached token, the eviction of cached tokens by that weight, and
the move of accepted drafted tokens to their final places. `run` makes the library's calls where `own` is true and
computes the same in elementary torch operations where it is false."""
import ctypes
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GROUP = 8  # channels per quantisation group of the cache


def _package():
    """The package directory `ppl.nn_amd/` under its importable name."""
    if "ppl_nn_amd" not in sys.modules:
        pkg_dir = os.path.join(ROOT, "ppl.nn_amd")
        spec = importlib.util.spec_from_file_location(
            "ppl_nn_amd", os.path.join(pkg_dir, "__init__.py"), submodule_search_locations=[pkg_dir])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ppl_nn_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["ppl_nn_amd"]


# ---------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one chat session verifying a short draft: all latency
        dict(name="tree_single_draft", op="tree", batch=1, draft_min=5, draft_max=5, kv_min=180, kv_max=220, heads=32,
             kv_heads=8, dim=128, layout=0, page=0, causal=False),
        # a serving batch with small trees on the Llama-3-8B layer shape
        dict(name="tree_serving", op="tree", batch=64, draft_min=4, draft_max=16, kv_min=256, kv_max=4096, heads=32,
             kv_heads=8, dim=128, layout=0, page=0, causal=False),
        # few sequences with wide trees over a paged cache: the matrix products weigh as much as the bytes
        dict(name="tree_wide_paged", op="tree", batch=16, draft_min=64, draft_max=64, kv_min=1024, kv_max=8192,
             heads=32, kv_heads=8, dim=128, layout=0, page=128, causal=False),
        # long contexts on one GPU's share of a 70B layer (8 query heads, 1 kv head)
        dict(name="tree_long_context", op="tree", batch=8, draft_min=24, draft_max=24, kv_min=32768, kv_max=131072,
             heads=8, kv_heads=1, dim=128, layout=0, page=0, causal=False),
        # an odd head size without shared heads, short and empty histories, token-contiguous cache, drafts in a line
        dict(name="tree_odd_heads", op="tree", batch=24, draft_min=1, draft_max=33, kv_min=0, kv_max=1500, heads=20,
             kv_heads=20, dim=80, layout=3, page=0, causal=True),
        # a decode step of a serving batch adds its tokens' weights to the running sums
        dict(name="weights_decode", op="weights", batch=64, draft_min=1, draft_max=1, kv_min=256, kv_max=4096, heads=32,
             kv_heads=8, dim=128, layout=0, page=0),
        # the last 32 queries of long prompts as the window whose weights count
        dict(name="weights_window", op="weights", batch=8, draft_min=32, draft_max=32, kv_min=4096, kv_max=32768,
             heads=32, kv_heads=8, dim=128, layout=0, page=0),
        # a handful of short sequences with small heads
        dict(name="weights_small", op="weights", batch=3, draft_min=1, draft_max=7, kv_min=17, kv_max=500, heads=12,
             kv_heads=4, dim=64, layout=3, page=0),
        # every sequence of a batch goes from budget + 128 tokens back to its budget, all layers in one call
        dict(name="evict_step", op="evict", batch=16, kv_min=1152, kv_max=1152, keep=1024 / 1152, sinks=4, recent=256,
             layers=8, kv_heads=8, dim=128, layout=0, page=0),
        # long prompts of one layer cut to half once their attention has been seen
        dict(name="evict_prompts", op="evict", batch=4, kv_min=16384, kv_max=65536, keep=0.5, sinks=4, recent=512,
             layers=1, kv_heads=8, dim=128, layout=3, page=0),
        # a serving batch keeps the accepted paths of its trees, sixteen layers in one call
        dict(name="accept_serving", op="accept", batch=64, draft_min=8, draft_max=24, accept_max=6, start_max=48,
             layers=16, kv_heads=8, dim=128, layout=0, page=0),
        # one session, thirty-two layers: all latency
        dict(name="accept_single", op="accept", batch=1, draft_min=40, draft_max=40, accept_max=6, start_max=48,
             layers=32, kv_heads=8, dim=128, layout=0, page=0),
    ]


HEAD_LAYOUTS = [(32, 8, 128), (8, 1, 128), (32, 32, 128), (40, 40, 128), (64, 8, 128), (12, 4, 64), (20, 20, 80),
                (16, 2, 96), (8, 8, 256), (24, 2, 112), (6, 3, 32)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["tree", "weights", "evict", "accept"])
        heads, kv_heads, dim = rng.choice(HEAD_LAYOUTS)
        case = dict(op=op, batch=_log_int(rng, 1, 128), kv_heads=kv_heads, dim=dim, layout=rng.choice([0, 3]),
                    page=rng.choice([0, 0, 64, 128, 256]))
        if op in ("tree", "weights"):
            case["heads"] = heads
            case["draft_max"] = _log_int(rng, 1, 150 if op == "tree" else 64)
            case["draft_min"] = rng.randint(1, case["draft_max"])
            case["kv_max"] = _log_int(rng, 1, 131072)
            case["kv_min"] = rng.randint(0, case["kv_max"])
            if op == "tree":
                case["causal"] = rng.random() < 0.3
            tokens = case["batch"] * (case["kv_max"] + case["draft_max"] + case["page"])
            slab = tokens * 2 * kv_heads * (dim + dim // 4)
        elif op == "evict":
            case["kv_max"] = _log_int(rng, 1, 65536)
            case["kv_min"] = rng.randint(max(1, case["kv_max"] // 8), case["kv_max"])
            case["keep"] = rng.uniform(0.05, 1.0)
            case["sinks"] = rng.choice([0, 1, 4])
            case["recent"] = _log_int(rng, 1, 1024)
            case["layers"] = _log_int(rng, 1, 32)
            slab = case["batch"] * (case["kv_max"] + case["page"]) * case["layers"] * 2 * kv_heads * (dim + dim // 4)
        else:
            case["draft_max"] = _log_int(rng, 1, 64)
            case["draft_min"] = rng.randint(1, case["draft_max"])
            case["accept_max"] = _log_int(rng, 1, 10)
            case["start_max"] = 48
            case["layers"] = _log_int(rng, 1, 32)
            slab = case["batch"] * (48 + case["draft_max"] + case["page"]) * case["layers"] * 2 * kv_heads * (
                dim + dim // 4)
        if slab <= 2 << 30 and _cost(case) <= limit:
            return case


def _tables(case):
    """The ragged lengths of a case. They belong to the case, not to the seed of its values, so that `work` can count
    them: (new tokens, cached tokens before them) per sequence."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    new, old = [], []
    for _ in range(case["batch"]):
        if case["op"] == "evict":
            new.append(0)
            old.append(rng.randint(case["kv_min"], case["kv_max"]))
        elif case["op"] == "accept":
            new.append(rng.randint(case["draft_min"], case["draft_max"]))
            old.append(rng.randint(0, case["start_max"]))
        else:
            new.append(rng.randint(case["draft_min"], case["draft_max"]))
            old.append(rng.randint(case["kv_min"], case["kv_max"]))
    return new, old


def _accepted(case):
    """Accepted drafted tokens of every sequence, ascending. Node i of a path is the drafted token i itself or one past
    the path's length, so a second pass over the same cache finds its sources as the first one did."""
    rng = random.Random("path" + repr(sorted((k, v) for k, v in case.items() if k != "name")))
    paths = []
    for n in _tables(case)[0]:
        length = rng.randint(1, min(case["accept_max"], n))
        stay = rng.randint(0, length)
        while stay < length and n - length < length - stay:
            stay += 1
        paths.append(list(range(stay)) + sorted(rng.sample(range(length, n), length - stay)))
    return paths


def _targets(case):
    return [max(1, int(n * case["keep"])) for n in _tables(case)[1]]


def work(case):
    new, old = _tables(case)
    kvh, dim = case["kv_heads"], case["dim"]
    row = dim + dim // 4  # int8 channels and fp16 scales of one head's key or value
    if case["op"] == "tree":
        h = case["heads"]
        words = (max(new) + 63) // 64
        cached = sum(n + o for n, o in zip(new, old))
        s = sum(new)
        byts = cached * 2 * kvh * row + s * h * dim * 2 * 2 + s * h * 4 + (0 if case["causal"] else s * words * 8)
        flops = sum(4 * h * dim * n * (o + (n + 1) / 2) for n, o in zip(new, old))
    elif case["op"] == "weights":
        h = case["heads"]
        cached = sum(n + o for n, o in zip(new, old))
        s = sum(new)
        byts = cached * kvh * row + s * h * dim * 2 + s * h * 4 + (sum(old) + cached) * kvh * 4 + s * kvh * 4
        flops = sum(2 * h * dim * n * (o + (n + 1) / 2) for n, o in zip(new, old))
    elif case["op"] == "evict":
        columns = case["layers"] * kvh
        byts = 0
        for n, keep in zip(old, _targets(case)):
            sinks, recent = min(case["sinks"], keep), min(case["recent"], n)
            free = max(0, n - sinks - recent)  # tokens that stay or go by their weight
            share = min(1.0, max(0.0, (keep - sinks - recent) / free)) if free else 0.0
            tail_recent = min(recent, n - keep)
            moved = tail_recent + share * max(0, n - keep - tail_recent)  # kept rows past the new length
            byts += columns * (n * 8 + keep * 8 + moved * 2 * 2 * row)
        flops = 0
    else:
        moved = sum(sum(1 for i, x in enumerate(p) if i != x) for p in _accepted(case))
        byts = case["layers"] * kvh * moved * 2 * 2 * row + sum(len(p) for p in _accepted(case)) * 8
        flops = 0
    return {"bytes": float(byts), "flops": float(flops)}


# --------------------------------------------------------------------------------------------------------- the inputs

class State:
    pass


def _slab(s, case, gen, layers, tokens):
    """The int8 cache and its scales, filled as quantised N(0, 1) keys and values are; `cache` and `scale` are seen as
    [token, layer, K or V, head, channel or group] whatever the layout in memory."""
    kvh, dim = case["kv_heads"], case["dim"]
    if case["layout"] == 0:
        shape, order = (tokens, layers, 2, kvh), (0, 1, 2, 3, 4)
        s.strides = dict(cache_stride_s=layers * 2 * kvh * dim, cache_stride_l=2 * kvh * dim, cache_stride_h=dim,
                         cache_stride_kv=kvh * dim)
    else:
        shape, order = (layers, 2, kvh, tokens), (3, 0, 1, 2, 4)
        s.strides = dict(cache_stride_s=dim, cache_stride_l=2 * kvh * tokens * dim, cache_stride_h=tokens * dim,
                         cache_stride_kv=kvh * tokens * dim)
    rows = shape[0] * shape[1] * shape[2] * shape[3]
    cache = torch.empty((rows, dim), dtype=torch.int8, device="cuda")
    scale = torch.empty((rows, dim // GROUP), dtype=torch.float16, device="cuda")
    step = max(1, (1 << 27) // dim)
    for i in range(0, rows, step):
        n = min(step, rows - i)
        x = torch.randn((n, dim // GROUP, GROUP), generator=gen, dtype=torch.float16, device="cuda")
        sc = (x.abs().amax(-1).float() / 127).half().clamp_min(1e-5)
        cache[i:i + n] = (x.float() / sc.float()[..., None]).half().float().round().to(torch.int8).view(n, dim)
        scale[i:i + n] = sc
    s.cache_mem, s.scale_mem = cache.view(shape + (dim,)), scale.view(shape + (dim // GROUP,))
    s.cache, s.scale = s.cache_mem.permute(order), s.scale_mem.permute(order)


def _i64(values):
    return torch.tensor(np.asarray(values, dtype=np.int64)).cuda()


def _sequences(s, case, lengths, seed):
    """Where the sequences live in the slab: one region each, or pages handed out in a random order."""
    page = case["page"]
    s.page = page
    if not page:
        starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
        s.cachestarts, s.pages_per_seq = _i64(starts[:-1]), 0
        tokens = [np.arange(starts[b], starts[b] + n) for b, n in enumerate(lengths)]
        total = int(starts[-1])
    else:
        pages = [(n + page - 1) // page for n in lengths]
        s.pages_per_seq = max(1, max(pages))
        order = np.random.default_rng(seed).permutation(sum(pages))
        table = np.full((len(lengths), s.pages_per_seq), 0, np.int64)
        tokens, k = [], 0
        for b, n in enumerate(lengths):
            table[b, :pages[b]] = order[k:k + pages[b]] * page
            k += pages[b]
            j = np.arange(n)
            tokens.append(table[b, j // page] + j % page)
        s.cachestarts = _i64(table)
        total = sum(pages) * page
    s.tokens = [_i64(t) for t in tokens]  # slab token of every cached token, per sequence
    return max(1, total)


def _random_tree(rng, n):
    """Visibility of n drafted tokens as 0/1 rows: a token sees its ancestors and itself; its parent is an earlier one,
    or none (a first token). One token in a hundred is padding, which sees nothing."""
    see = np.zeros((n, n), dtype=np.uint8)
    for t in range(n):
        if n > 8 and rng.random() < 0.01:
            continue
        parent = -1 if t == 0 else int(rng.integers(max(-1, t - 9), t))
        if parent >= 0:
            see[t] = see[parent]
        see[t, t] = 1
    return see


def _mask_words(trees, words):
    out = []
    for see in trees:
        n = see.shape[0]
        bits = np.zeros((n, words * 64), dtype=np.uint8)
        bits[:, :n] = see
        out.append(np.packbits(bits, axis=1, bitorder="little").view(np.int64))
    return np.concatenate(out) if out else np.zeros((0, words), np.int64)


def prepare(case, seed):
    s = State()
    s.case = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    new, old = _tables(case)
    s.new, s.old = new, old
    lengths = [n + o for n, o in zip(new, old)]
    s.lengths = lengths
    s.seqstarts = _i64(np.concatenate([[0], np.cumsum(new)]))
    s.kvstarts = _i64(np.concatenate([[0], np.cumsum(lengths)]))
    s.start_pos = _i64(old)
    layers = case.get("layers", 1)
    total = _sequences(s, case, lengths, seed)
    s.max_tokens = total
    _slab(s, case, gen, layers, total)
    kvh, dim = case["kv_heads"], case["dim"]
    if case["op"] in ("tree", "weights"):
        h = case["heads"]
        s.query = torch.randn((sum(new), h, dim), generator=gen, dtype=torch.float16, device="cuda")
        s.lse = torch.empty((sum(new), h), dtype=torch.float32, device="cuda")
    if case["op"] == "tree":
        s.output = torch.empty_like(s.query)
        s.words = (max(new) + 63) // 64
        if case["causal"]:
            s.see = [torch.ones((n, n), dtype=torch.bool, device="cuda").tril() for n in new]
            s.mask = None
        else:
            trees = [_random_tree(rng, n) for n in new]
            s.see = [torch.from_numpy(t).cuda().bool() for t in trees]
            s.mask = torch.from_numpy(_mask_words(trees, s.words)).cuda()
    elif case["op"] == "weights":
        s.see = [torch.ones((n, n), dtype=torch.bool, device="cuda").tril() for n in new]
        for b in range(len(new)):
            r0, r1 = sum(new[:b]), sum(new[:b + 1])
            s.lse[r0:r1] = _attend(s, b, r0, r1, torch.float32)[1]
        # sums of a history of steps: a few tokens hold most of the weight
        s.score = torch.randn((1, kvh, total), generator=gen, device="cuda").mul_(1.5).exp_()
        s.score_out = s.score.clone()
        s.position = torch.zeros((1, kvh, total), dtype=torch.int32, device="cuda")
        # the tokens' positions in the text run ahead of their places in a cache that has lost tokens
        s.position_idx = _i64(np.concatenate([np.arange(o, o + n) + 700 for n, o in zip(new, old)]))
    elif case["op"] == "evict":
        s.score = torch.randn((layers, kvh, total), generator=gen, device="cuda").mul_(1.5).exp_()
        s.position = torch.zeros((layers, kvh, total), dtype=torch.int32, device="cuda")
        for b, n in enumerate(old):
            s.position[:, :, s.tokens[b]] = torch.arange(n, dtype=torch.int32, device="cuda")
        s.score_out, s.position_out = s.score.clone(), s.position.clone()
        s.targets = _targets(case)
        s.target_kvlen, s.next_pos = _i64(s.targets), _i64(old)
        s.new_kvlen = torch.zeros(len(old), dtype=torch.int64, device="cuda")
    else:
        s.paths = _accepted(case)
        table = np.full((len(new), case["accept_max"]), -1, np.int64)
        for b, p in enumerate(s.paths):
            table[b, :len(p)] = p
        s.accepted, s.accepted_len = _i64(table), _i64([len(p) for p in s.paths])
    if own:
        _prepare_own(s, case, layers)
    return s


def _prepare_own(s, case, layers):
    """The argument blocks, plans and workspaces a program keeps beside its tables."""
    pkg = _package()
    cabi = pkg.cabi
    s.pkg, s.lib = pkg, pkg.load_library()
    pkg.check(s.lib.pplhip_init(), "pplhip_init")
    block = {"tree": cabi.TreeAttentionArgs, "weights": cabi.KvScoreArgs, "evict": cabi.KvEvictArgs,
             "accept": cabi.KvAcceptArgs}[case["op"]]
    a = block()
    s.args = a
    a.d_cachestarts = s.cachestarts.data_ptr()
    a.batch = case["batch"]
    a.num_layer, a.num_kv_heads, a.head_dim = layers, case["kv_heads"], case["dim"]
    a.layer_idx = 0
    a.cache_mode, a.page_size, a.cachestart_stride_b = (1, s.page, s.pages_per_seq) if s.page else (0, 128, 0)
    for k, v in s.strides.items():
        setattr(a, k, v)
    a.d_cache, a.d_scale = s.cache_mem.data_ptr(), s.scale_mem.data_ptr()
    if case["op"] in ("tree", "weights"):
        a.d_query, a.d_lse = s.query.data_ptr(), s.lse.data_ptr()
        a.d_seqstarts, a.d_kvstarts = s.seqstarts.data_ptr(), s.kvstarts.data_ptr()
        a.total_new_tokens, a.max_seqlen, a.max_kvlen = sum(s.new), max(s.new), max(s.lengths)
        a.num_heads = case["heads"]
    if case["op"] == "tree":
        a.d_tree_mask = None if s.mask is None else s.mask.data_ptr()
        a.tree_mask_words = 0 if s.mask is None else s.words
        a.d_output = s.output.data_ptr()
        s.plan = cabi.TreeAttentionPlan()
        pkg.check(s.lib.pplhip_tree_attention_prepare(ctypes.byref(a), ctypes.byref(s.plan)), "tree_attention_prepare")
    elif case["op"] == "weights":
        a.d_position_idx = s.position_idx.data_ptr()
        a.d_score_in, a.d_score_out, a.d_position = s.score.data_ptr(), s.score_out.data_ptr(), s.position.data_ptr()
        a.score_stride_l, a.score_stride_h = case["kv_heads"] * s.max_tokens, s.max_tokens
    elif case["op"] == "evict":
        a.layer_count = layers
        a.d_kvstarts, a.max_kvlen = s.kvstarts.data_ptr(), max(s.lengths)
        a.d_target_kvlen, a.d_next_pos = s.target_kvlen.data_ptr(), s.next_pos.data_ptr()
        a.num_sink, a.num_recent = case["sinks"], case["recent"]
        a.d_score_in, a.d_score_out = s.score.data_ptr(), s.score_out.data_ptr()
        a.d_position_in, a.d_position_out = s.position.data_ptr(), s.position_out.data_ptr()
        a.score_stride_l, a.score_stride_h = case["kv_heads"] * s.max_tokens, s.max_tokens
        a.d_new_kvlen = s.new_kvlen.data_ptr()
        s.plan = cabi.KvEvictPlan()
        pkg.check(s.lib.pplhip_kv_evict_prepare(ctypes.byref(a), ctypes.byref(s.plan)), "kv_evict_prepare")
    else:
        a.layer_count = layers
        a.d_seqstarts, a.d_start_pos = s.seqstarts.data_ptr(), s.start_pos.data_ptr()
        a.d_accepted, a.accepted_stride_b = s.accepted.data_ptr(), case["accept_max"]
        a.d_accepted_len, a.max_accepted = s.accepted_len.data_ptr(), case["accept_max"]
    if case["op"] in ("tree", "evict"):
        s.workspace = torch.empty(max(256, int(s.plan.workspace_bytes)), dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------------------------------------------ the two forms

def run(s):
    op = s.case["op"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if op == "tree":
            rc = s.lib.pplhip_tree_attention_forward(ctypes.byref(s.args), ctypes.byref(s.plan),
                                                     s.workspace.data_ptr(), stream)
        elif op == "weights":
            rc = s.lib.pplhip_kv_score_accumulate(ctypes.byref(s.args), stream)
        elif op == "evict":
            rc = s.lib.pplhip_kv_evict(ctypes.byref(s.args), ctypes.byref(s.plan), s.workspace.data_ptr(), stream)
        else:
            rc = s.lib.pplhip_kv_accept(ctypes.byref(s.args), stream)
        if rc:
            s.pkg.check(rc, op)
    else:
        {"tree": _plain_tree, "weights": _plain_weights, "evict": _plain_evict, "accept": _plain_accept}[op](s)
    if op == "tree":
        return {"output": s.output, "lse": s.lse}
    if op == "weights":
        return {"score": s.score_out, "position": s.position}
    if op == "evict":
        return {"cache": s.cache_mem, "scale": s.scale_mem, "score": s.score_out, "position": s.position_out,
                "new_kvlen": s.new_kvlen}
    return {"cache": s.cache_mem, "scale": s.scale_mem}


def _rows(s, b, kv, dtype):
    """Cached keys (kv 0) or values (1) of sequence b as [head, token, channel]; a cached value is its int8 times its
    scale, rounded to fp16."""
    q = s.cache[s.tokens[b], 0, kv]
    sc = s.scale[s.tokens[b], 0, kv]
    n, kvh, dim = q.shape
    x = (q.float().view(n, kvh, dim // GROUP, GROUP) * sc.float()[..., None]).half()
    return x.view(n, kvh, dim).permute(1, 0, 2).contiguous().to(dtype)


def _attend(s, b, r0, r1, dtype):
    """Weights [kv head, (token, shared head), key] and log-sums [token, head] of sequence b's new tokens, whose
    packed rows are r0 .. r1 - 1."""
    kvh, dim, h = s.case["kv_heads"], s.case["dim"], s.case["heads"]
    n, rep = r1 - r0, h // kvh
    q = s.query[r0:r1].to(dtype).view(n, kvh, rep, dim).permute(1, 0, 2, 3).reshape(kvh, n * rep, dim)
    k = _rows(s, b, 0, dtype).transpose(1, 2).contiguous()
    x = torch.matmul(q, k) * (1.0 / math.sqrt(dim))
    see = torch.ones((n, s.lengths[b]), dtype=torch.bool, device="cuda")
    see[:, s.old[b]:] = s.see[b]
    x = x.view(kvh, n, rep, -1).masked_fill(~see[None, :, None, :], -math.inf).view(kvh, n * rep, -1)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = (total.log() + top).view(kvh, n, rep).permute(1, 0, 2).reshape(n, h)
    return e / torch.where(total > 0, total, torch.ones_like(total)), lse


def _plain_tree(s):
    kvh, dim, h = s.case["kv_heads"], s.case["dim"], s.case["heads"]
    r0 = 0
    for b, n in enumerate(s.new):
        p, lse = _attend(s, b, r0, r0 + n, torch.float32)
        o = torch.matmul(p, _rows(s, b, 1, torch.float32))
        s.output[r0:r0 + n] = o.view(kvh, n, h // kvh, dim).permute(1, 0, 2, 3).reshape(n, h, dim).half()
        s.lse[r0:r0 + n] = lse
        r0 += n


def _plain_weights(s):
    kvh, dim, h = s.case["kv_heads"], s.case["dim"], s.case["heads"]
    rep = h // kvh
    r0 = 0
    for b, n in enumerate(s.new):
        q = s.query[r0:r0 + n].float().view(n, kvh, rep, dim).permute(1, 0, 2, 3).reshape(kvh, n * rep, dim)
        x = torch.matmul(q, _rows(s, b, 0, torch.float32).transpose(1, 2).contiguous()) * (1.0 / math.sqrt(dim))
        lse = s.lse[r0:r0 + n].view(n, kvh, rep).permute(1, 0, 2).reshape(kvh, n * rep, 1)
        p = torch.exp(x - lse).view(kvh, n, rep, -1).sum(2)
        p[:, :, s.old[b]:] *= s.see[b][None]
        w = p.sum(1)
        before = s.score[0][:, s.tokens[b]]
        before[:, s.old[b]:] = 0
        s.score_out[0][:, s.tokens[b]] = before + w
        s.position[0][:, s.tokens[b][s.old[b]:]] = s.position_idx[r0:r0 + n].int()
        r0 += n


def _plain_evict(s):
    case = s.case
    for b, n in enumerate(s.lengths):
        keep = min(n, s.targets[b])
        tok = s.tokens[b]
        score, pos = s.score[:, :, tok], s.position[:, :, tok]
        protect = (pos < case["sinks"]) | (pos >= n - case["recent"])
        key = torch.where(protect, torch.full_like(score, math.inf), score)
        order = torch.sort(key, dim=-1, descending=True, stable=True).indices
        kept = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order[..., :keep], True)
        layer, head, hole = torch.nonzero(~kept[..., :keep], as_tuple=True)
        src = n - 1 - torch.nonzero(kept[..., keep:].flip(-1), as_tuple=True)[2]  # the last kept row fills first
        s.score_out[:, :, tok[:keep]] = score[..., :keep]
        s.position_out[:, :, tok[:keep]] = pos[..., :keep]
        to, frm = tok[hole], tok[src]
        s.score_out[layer, head, to] = s.score[layer, head, frm]
        s.position_out[layer, head, to] = s.position[layer, head, frm]
        for kv in (0, 1):
            s.cache[to, layer, kv, head] = s.cache[frm, layer, kv, head]
            s.scale[to, layer, kv, head] = s.scale[frm, layer, kv, head]
    s.new_kvlen.copy_(torch.minimum(s.target_kvlen, s.kvstarts[1:] - s.kvstarts[:-1]))


def _plain_accept(s):
    to, frm = [], []
    for b, path in enumerate(s.paths):
        at = s.tokens[b]
        to.append(at[s.old[b]:s.old[b] + len(path)])
        frm.append(at[s.accepted[b, :len(path)] + s.start_pos[b]])
    to, frm = torch.cat(to), torch.cat(frm)
    s.cache[to] = s.cache[frm]
    s.scale[to] = s.scale[frm]


# --------------------------------------------------------------------------------- the definition, in 64 bits, apart

def _exact_rows(s, b, head, kv):
    at = s.tokens[b]
    q = s.cache[at, 0, kv, head].double()
    sc = s.scale[at, 0, kv, head].double().repeat_interleave(GROUP, dim=-1)
    return (q * sc).half().double()  # 8 x 11 bits: the product is exact, the rounding to fp16 is the cache's own


def _exact_attention(case, s, weights):
    kvh, dim, h = case["kv_heads"], case["dim"], case["heads"]
    rep = h // kvh
    out = torch.zeros((sum(s.new), h, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(s.new), h), -math.inf, dtype=torch.float64, device="cuda")
    score = s.score.double() if weights else None
    at_row = 0
    for b, (n, o) in enumerate(zip(s.new, s.old)):
        add = torch.zeros((kvh, n + o), dtype=torch.float64, device="cuda")
        for head in range(kvh):
            k = _exact_rows(s, b, head, 0)
            v = None if weights else _exact_rows(s, b, head, 1)
            for i in range(rep):
                hq = head * rep + i
                q = s.query[at_row:at_row + n, hq].double()
                x = torch.mm(q, k.t().contiguous()) / math.sqrt(dim)
                hidden = torch.zeros((n, n + o), dtype=torch.bool, device="cuda")
                hidden[:, o:] = ~s.see[b]
                x[hidden] = -math.inf
                if weights:
                    add[head] += torch.exp(x - s.lse[at_row:at_row + n, hq, None].double()).sum(0)
                    continue
                z = torch.logsumexp(x, dim=1)
                lse[at_row:at_row + n, hq] = z
                some = ~torch.isinf(z)
                out[at_row:at_row + n, hq][some] = torch.mm(torch.exp(x[some] - z[some, None]), v)
        if weights:
            before = score[0][:, s.tokens[b]]
            before[:, o:] = 0.0
            score[0][:, s.tokens[b]] = before + add
        at_row += n
    return {"score": score, "position": None} if weights else {"output": out, "lse": lse}


def _exact_evict(case, s):
    """Column by column: which tokens stay, then the holes in front of the new length are filled from the back."""
    layers, kvh = s.score.shape[0], s.score.shape[1]
    score, pos = s.score.cpu().numpy(), s.position.cpu().numpy()
    new_score = score.astype(np.float64)
    to, frm, lay, hd = [], [], [], []
    for b, n in enumerate(s.lengths):
        at = s.tokens[b].cpu().numpy()
        k = min(n, s.targets[b])
        for layer in range(layers):
            for head in range(kvh):
                x = score[layer, head, at].astype(np.float64)
                where = pos[layer, head, at]
                x[(where < case["sinks"]) | (where >= n - case["recent"])] = np.inf
                stays = np.sort(np.lexsort((np.arange(n), -x))[:k])
                holes = np.setdiff1d(np.arange(k), stays[stays < k], assume_unique=True)
                fill = stays[stays >= k][::-1]
                new_score[layer, head, at[holes]] = score[layer, head, at[fill]]
                to.append(at[holes])
                frm.append(at[fill])
                lay.append(np.full(len(holes), layer))
                hd.append(np.full(len(holes), head))
    to, frm, lay, hd = (torch.from_numpy(np.concatenate(x).astype(np.int64)).cuda() for x in (to, frm, lay, hd))
    for kv in (0, 1):
        s.scale[to, lay, kv, hd] = s.scale[frm, lay, kv, hd]
    return {"cache": None, "scale": s.scale_mem.double(), "score": torch.from_numpy(new_score).cuda(), "position": None,
            "new_kvlen": None}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] in ("tree", "weights"):
        return _exact_attention(case, s, case["op"] == "weights")
    if case["op"] == "evict":
        return _exact_evict(case, s)
    for b, path in enumerate(s.paths):
        for i, x in enumerate(path):
            s.scale[s.tokens[b][s.old[b] + i]] = s.scale[s.tokens[b][s.old[b] + x]]
    return {"cache": None, "scale": s.scale_mem.double()}
