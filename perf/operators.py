"""Performance cases of the operators that verify a tree of drafted tokens in one step.

A drafting program proposes n_tree tokens as a tree: node 0 is the token that the last step chose, node t hangs below
parents[t] < t.  One step of the model then computes all of them, chooses a token at each node and keeps the path that the
choices agree with.

  op        one pass
  attn      attention_tree: rotary positions, the nodes' rows into the f16 cache, grouped-query attention of each node over
            its sequence's cache and its own ancestors
  logits    logits_process: penalties for repeated tokens, biases, the grammar's mask, and the highest token of each row
  accept    tree_accept: the path from node 0 along the chosen tokens
  compact   kv_cache_compact: the path's cache rows moved together, in every layer

Where `own` is false `run` computes them with elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

ROPE_BASE = 500000.0
NONE = -1  # "no token": all bits set


def listed():
    return [
        # a short chat with a draft of four tokens: the smallest call, where the launches count
        dict(name="attn_chain5_ctx300", op="attn", seqs=1, tree=5, shape="chain", ctx=300, heads=32, kv_heads=8, head_dim=128),
        # the usual tree over the benchmark's context
        dict(name="attn_tree26_ctx4070", op="attn", seqs=1, tree=26, shape="tree", ctx=4070, heads=32, kv_heads=8, head_dim=128),
        # sequences of mixed lengths verified together, on a model with small heads; some have fewer drafts than the others
        dict(name="attn_tree16_x8_ragged_d64", op="attn", seqs=8, tree=16, shape="padded", ctx=8100, heads=32, kv_heads=4, head_dim=64),
        # a wide tree over a whole book
        dict(name="attn_tree64_ctx131000", op="attn", seqs=1, tree=64, shape="tree", ctx=131000, heads=32, kv_heads=8, head_dim=128),
        # one token of plain decoding: penalties for what was said, a few biased tokens
        dict(name="logits_1x32000", op="logits", seqs=1, tree=0, vocab=32000, pad=0, history=700, bias=20, mask=False, write=True),
        # many sequences of plain decoding under a grammar, with long histories
        dict(name="logits_16x128256", op="logits", seqs=16, tree=0, vocab=128256, pad=0, history=20000, bias=300, mask=True,
             write=True),
        # every node of a tree, each row with its own path and grammar state
        dict(name="logits_tree64x128256", op="logits", seqs=1, tree=64, vocab=128256, pad=64, history=4096, bias=50, mask=True,
             write=True),
        # the walk of one sequence's tree, and of a large batch's
        dict(name="accept_1x26", op="accept", seqs=1, tree=26, ctx=4070),
        dict(name="accept_256x64", op="accept", seqs=256, tree=64, ctx=900),
        # what a step leaves to move: seven rows in each of 32 layers, and a batch's rows
        dict(name="compact_32_layers_x1", op="compact", seqs=1, tree=26, layers=32, ctx=1000, kv_heads=8, head_dim=128),
        dict(name="compact_24_layers_x16", op="compact", seqs=16, tree=64, layers=24, ctx=300, kv_heads=4, head_dim=128),
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "attn", "logits", "logits", "logits", "accept", "compact"])
    if op == "attn":
        kv = rng.choice([1, 2, 4, 8, 8, 16])
        heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        seqs, tree, ctx = _log(rng, 1, 24), _log(rng, 1, 128), _log(rng, 1, 100000)
        while seqs * ctx * heads * (tree + 32) > 32 * 131000 * 64 or seqs * ctx * kv > 8 * 131000:
            ctx = ctx // 2 + 1
            seqs = max(1, seqs // 2) if ctx < 2000 else seqs
        return dict(op=op, seqs=seqs, tree=tree, shape=rng.choice(["chain", "tree", "tree", "padded"]), ctx=ctx, heads=heads,
                    kv_heads=kv, head_dim=rng.choice([64, 128, 128]))
    if op == "logits":
        seqs, tree = _log(rng, 1, 32), rng.choice([0, 0, _log(rng, 1, 128)])
        vocab = _log(rng, 1000, 160000)
        while seqs * max(1, tree) * vocab > 64 * 128256:
            seqs, tree = max(1, seqs // 2), tree // 2
        return dict(op=op, seqs=seqs, tree=tree, vocab=vocab, pad=rng.choice([0, 0, rng.randint(1, 64)]),
                    history=_log(rng, 1, 40000), bias=rng.choice([0, _log(rng, 1, 1000)]), mask=rng.random() < 0.6,
                    write=rng.random() < 0.8)
    if op == "accept":
        return dict(op=op, seqs=_log(rng, 1, 256), tree=_log(rng, 1, 64), ctx=_log(rng, 1, 8000))
    seqs, layers, ctx, kv = _log(rng, 1, 16), rng.randint(1, 32), _log(rng, 1, 1000), rng.choice([1, 2, 4, 8])
    while seqs * layers * (ctx + 64) * kv > 24 * 16 * 364 * 4:
        seqs, layers = max(1, seqs // 2), max(1, layers // 2)
        ctx = ctx // 2 + 1 if seqs == 1 else ctx
    return dict(op=op, seqs=seqs, tree=_log(rng, 3, 64), layers=layers, ctx=ctx, kv_heads=kv, head_dim=rng.choice([64, 128]))


# ------------------------------------------------------------------- inputs
def _rng(case, seed):
    return np.random.default_rng([int(seed) & 0x7FFFFFFF, len(case["op"]), case["seqs"], case["tree"]])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a).astype(dtype)).cuda()


def _parents(r, seqs, tree, shape):
    """parents [seqs][tree]: a chain, trees that draw most children from the last few nodes, or trees of which some end early
    (the nodes behind the last carry -2: not there)."""
    p = np.full((seqs, tree), -1, np.int64)
    for s in range(seqs):
        for t in range(1, tree):
            p[s, t] = t - 1 if shape == "chain" else r.integers(max(0, t - 1 - t // 2), t)
        if shape == "padded" and s % 2 == 1:
            p[s, int(r.integers(0, tree + 1)):] = -2
    return p


def _lengths(r, seqs, ctx):
    """One sequence: ctx tokens.  Several: from an empty cache to ctx, one of them ctx."""
    if seqs == 1:
        return [ctx]
    lens = [int(v) for v in np.exp(r.uniform(0, math.log(ctx + 1), seqs))]
    lens[int(r.integers(0, seqs))] = ctx
    if seqs > 2:
        lens[lens.index(min(lens))] = 0
    return lens


def _attn_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, t, h, kv, d = c["seqs"], c["tree"], c["heads"], c["kv_heads"], c["head_dim"]
    lens = _lengths(r, n, c["ctx"])
    room = c["ctx"] + t + 7
    inv = 1.0 / ROPE_BASE ** (np.arange(0, d, 2) / d)
    return dict(qkv=torch.randn((n * t, (h + 2 * kv) * d), device="cuda", generator=g) * 1.3,
                k=torch.randn((n, room, kv, d), device="cuda", generator=g, dtype=torch.float16),
                v=torch.randn((n, room, kv, d), device="cuda", generator=g, dtype=torch.float16),
                parents=_dev(_parents(r, n, t, c["shape"]), np.int32), lens=lens, ctx_len=_dev(lens, np.int32), room=room,
                inv=_dev(inv, np.float32))


def _logits_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, t, v, hist = c["seqs"], c["tree"], c["vocab"], c["history"]
    rows = n * max(1, t)
    wide = torch.randn((rows, v + c["pad"]), device="cuda", generator=g) * 3.0 - 2.0
    # what was said: few tokens often, many seldom, and some of what the model now likes
    said = np.minimum(v - 1, np.floor(v * r.random((n, hist)) ** 4)).astype(np.int64)
    lens = np.maximum(1, r.integers(hist // 2, hist + 1, n)) if n > 1 else np.array([hist])
    tops = wide[:: max(1, t), :v].topk(min(8, v), 1).indices.cpu().numpy()
    for s in range(n):
        said[s, r.integers(0, lens[s], 6)] = tops[s, r.integers(0, tops.shape[1], 6)]
    s = dict(wide=wide, rows=rows, history=_dev(said, np.int32), history_len=_dev(lens, np.int32),
             penalties=(1.1 + 0.3 * float(r.random()), float(np.float32(0.4 * r.random())), float(np.float32(0.6 * r.random()))))
    s["penalties"] = tuple(float(np.float32(x)) for x in s["penalties"])
    if t:
        s["parents"] = _dev(_parents(r, n, t, "tree"), np.int32)
        s["tokens"] = _dev(np.minimum(v - 1, np.floor(v * r.random((n, t)) ** 3)), np.int32)
    if c["bias"]:
        s["bias_ids"] = _dev(r.integers(0, v, c["bias"]), np.int32)
        s["bias"] = _dev(r.choice([-100.0, -5.0, -1.0, 1.0, 2.5, 5.0], c["bias"]) + r.random(c["bias"]), np.float32)
    if c["mask"]:
        # a grammar lets most rows choose freely, some among a part, some among a few tokens, and one has come to its end
        words = (v + 31) // 32
        m = r.integers(0, 1 << 32, (rows, words), dtype=np.uint64)
        for i in range(rows):
            kind = r.random()
            if kind < 0.5:
                m[i] = (1 << 32) - 1
            elif kind > 0.8:
                m[i] &= 0 if kind > 0.97 else r.integers(0, 1 << 32, words, dtype=np.uint64) * (r.random(words) < 0.01)
        s["mask"] = _dev(m.astype(np.uint32).view(np.int32), np.int32)
    return s


def _accept_inputs(c, seed):
    r = _rng(c, seed)
    n, t = c["seqs"], c["tree"]
    parents = _parents(r, n, t, "padded" if n > 1 else "tree")
    tokens = r.integers(0, 50, (n, t))
    picked = r.integers(0, 50, (n, t))
    for s in range(n):  # choices that agree with a child most of the time
        for i in range(1, t):
            if parents[s, i] >= 0 and r.random() < 0.7:
                picked[s, parents[s, i]] = tokens[s, i]
    lens = r.integers(0, c["ctx"] + 1, n)
    return dict(parents=_dev(parents, np.int32), tokens=_dev(tokens, np.int32), picked=_dev(picked, np.int32),
                ctx_len=_dev(lens, np.int32), history=_dev(r.integers(0, 50, (n, c["ctx"] + t)), np.int32))


def _compact_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, t, kv, d = c["seqs"], c["tree"], c["kv_heads"], c["head_dim"]
    path, count = np.full((n, t), NONE, np.int64), np.zeros(n, np.int64)
    for s in range(n):
        # node 0 and nodes behind the rows that the path will fill
        most = min(8, (t + 1) // 2)
        count[s] = int(r.integers(1, most + 1)) if n > 1 else most
        path[s, 0] = 0
        path[s, 1:count[s]] = np.sort(r.permutation(np.arange(count[s], t))[:count[s] - 1])
    before = r.integers(0, c["ctx"] + 1, n)
    room = c["ctx"] + t
    shape = (c["layers"], 2, n, room, kv, d)
    return dict(caches=torch.randn(shape, device="cuda", generator=g, dtype=torch.float16), room=room, path=_dev(path, np.int32),
                count=_dev(count, np.int32), ctx_len=_dev(before + count, np.int32))


def _inputs(case, seed):
    return dict(attn=_attn_inputs, logits=_logits_inputs, accept=_accept_inputs, compact=_compact_inputs)[case["op"]](case, seed)


class _Queue:
    """torch's current stream as the framework's calls take it."""

    def __init__(self):
        self.handle = torch.cuda.current_stream().cuda_stream or None


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    n, t = case["seqs"], case["tree"]
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "attn":
        s["out"] = torch.zeros((n * t, case["heads"] * case["head_dim"]), device="cuda")
    if case["op"] == "logits":
        s["out"] = torch.zeros((s["rows"], case["vocab"]), device="cuda") if case["write"] else None
        s["token"] = torch.zeros(s["rows"], **i32)
    if case["op"] == "accept":
        s.update(path=torch.zeros((n, t), **i32), count=torch.zeros(n, **i32), next=torch.zeros(n, **i32), after=torch.zeros(n, **i32))
    if own:
        from woolly_amd import device, ops

        device.init(torch.cuda.current_device())
        need = 0
        if case["op"] == "attn":
            need = ops.attention_tree_workspace_bytes(n, t, case["heads"], case["kv_heads"], case["head_dim"], s["room"])
        if case["op"] == "logits":
            s["rules"] = ops.LogitsRules(
                rows_per_seq=max(1, t), history=s["history"].data_ptr(), history_stride=case["history"],
                history_len=s["history_len"].data_ptr(), tree_tokens=s["tokens"].data_ptr() if t else None,
                tree_parents=s["parents"].data_ptr() if t else None, repetition_penalty=s["penalties"][0],
                frequency_penalty=s["penalties"][1], presence_penalty=s["penalties"][2],
                bias_ids=s["bias_ids"].data_ptr() if case["bias"] else None, bias=s["bias"].data_ptr() if case["bias"] else None,
                n_bias=case["bias"], mask=s["mask"].data_ptr() if case["mask"] else None,
                mask_stride=(case["vocab"] + 31) // 32)
            need = ops.logits_process_workspace_bytes(s["rules"], s["rows"], case["vocab"])
        if case["op"] == "compact":
            s["layers"] = ops.KvCaches([x[0].data_ptr() for x in s["caches"]], [x[1].data_ptr() for x in s["caches"]])
        s["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------- a pass
def run(s):
    c = s["case"]
    if not own:
        return dict(attn=_plain_attn, logits=_plain_logits, accept=_plain_accept, compact=_plain_compact)[c["op"]](s, c)
    from woolly_amd import ops

    queue = _Queue()
    if c["op"] == "attn":
        h, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
        q, ld = s["qkv"].data_ptr(), (h + 2 * kv) * d
        ops.attention_tree(q, q + 4 * h * d, q + 4 * (h + kv) * d, ld, ld, s["parents"].data_ptr(), s["ctx_len"].data_ptr(),
                           c["seqs"], c["tree"], s["k"].data_ptr(), s["v"].data_ptr(), s["room"], h, kv, d, s["inv"].data_ptr(),
                           s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), queue)
        return dict(out=s["out"], k=s["k"], v=s["v"])
    if c["op"] == "logits":
        out = s["out"].data_ptr() if c["write"] else None
        ops.logits_process(s["rules"], s["wide"].data_ptr(), c["vocab"] + c["pad"], s["rows"], c["vocab"], out, c["vocab"],
                           s["token"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), queue)
        return dict(token=s["token"], **({"out": s["out"]} if c["write"] else {}))
    if c["op"] == "accept":
        ops.tree_accept(s["tokens"].data_ptr(), s["parents"].data_ptr(), s["picked"].data_ptr(), c["seqs"], c["tree"],
                        s["path"].data_ptr(), s["count"].data_ptr(), s["next"].data_ptr(), s["ctx_len"].data_ptr(),
                        s["after"].data_ptr(), s["history"].data_ptr(), s["history"].shape[1], queue)
        return {k: s[k] for k in ("path", "count", "next", "after", "history")}
    ops.kv_cache_compact(s["layers"], c["seqs"], s["room"], c["kv_heads"], c["head_dim"], s["path"].data_ptr(), c["tree"],
                         s["count"].data_ptr(), s["ctx_len"].data_ptr(), queue)
    return s["caches"]


# --------------------------------------------------------------- plain forms
def _reach(parents):
    """(ancestors [n][t][t] with the node itself, present [n][t]): products of the parent map with itself."""
    n, t = parents.shape
    idx = torch.arange(t, device="cuda")
    ok = (parents >= -1) & (parents < idx)
    at = torch.where(parents == -1, t, parents)  # column t: the cache
    step = ((at[:, :, None] == torch.arange(t + 1, device="cuda")) & ok[:, :, None]).float()
    a = torch.zeros((n, t + 1, t + 1), device="cuda")
    a[:, :t] = step
    a += torch.eye(t + 1, device="cuda")
    for _ in range(max(1, t).bit_length()):
        a = (a @ a.contiguous()).clamp(max=1.0)
    present = a[:, :t, t] > 0
    return (a[:, :t, :t] > 0) & present[:, :, None], present


def _plain_attn(s, c):
    n, t, h, kv, d = c["seqs"], c["tree"], c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = s["qkv"].view(n, t, h + 2 * kv, d).split([h, kv, kv], 2)
    seen, present = _reach(s["parents"])
    depth = (seen.sum(2) - 1).clamp(min=0)
    angle = (depth + s["ctx_len"][:, None]).double()[:, :, None, None] * s["inv"].double()
    cos, sin = angle.cos(), angle.sin()
    k1, k2 = k.double().chunk(2, -1)
    k = torch.cat([k1 * cos - k2 * sin, k1 * sin + k2 * cos], -1).float().half()
    cos, sin = cos.float(), sin.float()
    q1, q2 = q.chunk(2, -1)
    q = torch.cat([q1 * cos - q2 * sin, q1 * sin + q2 * cos], -1)
    for i, length in enumerate(s["lens"]):
        rows = slice(length, length + t)
        there = present[i][:, None, None]
        s["k"][i, rows] = torch.where(there, k[i], s["k"][i, rows])
        s["v"][i, rows] = torch.where(there, v[i].half(), s["v"][i, rows])
        keys = s["k"][i, :length + t].float().permute(1, 2, 0).contiguous()
        vals = s["v"][i, :length + t].float().permute(1, 0, 2).contiguous()
        qs = q[i].view(t, kv, h // kv, d).permute(1, 0, 2, 3).reshape(kv, -1, d).contiguous()
        score = (qs @ keys / math.sqrt(d)).view(kv, t, h // kv, length + t)
        score[..., length:].masked_fill_(~seen[i][None, :, None, :], -math.inf)
        score -= score.max(-1, keepdim=True).values
        score.exp_()
        total = score.sum(-1, keepdim=True)
        o = (score.view(kv, -1, length + t) @ vals).view(kv, t, h // kv, d) / total
        o = torch.where(present[i][None, :, None, None], o, 0.0)
        s["out"].view(n, t, kv, h // kv, d)[i] = o.permute(1, 0, 2, 3)
    return dict(out=s["out"], k=s["k"], v=s["v"])


def _plain_logits(s, c):
    n, t, v = c["seqs"], c["tree"], c["vocab"]
    rep, freq, pres = s["penalties"]
    hist = s["history"].long()
    live = torch.arange(hist.shape[1], device="cuda") < s["history_len"][:, None]
    count = torch.zeros((n, v), dtype=torch.int32, device="cuda")
    count.scatter_add_(1, hist, live.int())
    if t:
        seen, _ = _reach(s["parents"])
        count = count[:, None].repeat(1, t, 1)
        count.scatter_add_(2, s["tokens"].long()[:, None].expand(n, t, t).contiguous(), seen.int())
    count = count.view(s["rows"], v)
    x = s["wide"][:, :v]
    said = count > 0
    rep = torch.full((1,), rep, device="cuda")
    x = torch.where(said, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(said, x - (count.float() * freq + pres), x)
    if c["bias"]:
        last = torch.full((v,), -1, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(0, s["bias_ids"].long(), torch.arange(c["bias"], device="cuda"), "amax")
        x = torch.where(last >= 0, x + s["bias"][last.clamp(min=0)], x)
    if c["mask"]:
        i = torch.arange(v, device="cuda")
        x = torch.where(((s["mask"][:, i >> 5] >> (i & 31)) & 1) > 0, x, -math.inf)
    top = x.max(1, keepdim=True).values
    i = torch.where(x == top, torch.arange(v, device="cuda"), v).min(1).values
    s["token"].copy_(torch.where(top[:, 0] > -math.inf, i, NONE))
    if not c["write"]:
        return dict(token=s["token"])
    s["out"].copy_(x)
    return dict(token=s["token"], out=s["out"])


def _plain_accept(s, c):
    n, t = c["seqs"], c["tree"]
    _, present = _reach(s["parents"])
    idx = torch.arange(t, device="cuda")
    rows = torch.arange(n, device="cuda")
    at = torch.zeros(n, dtype=torch.int64, device="cuda")
    going = present[:, 0] & (s["parents"][:, 0] == -1)
    s["path"].fill_(NONE)
    s["count"].zero_()
    s["next"].fill_(NONE)
    end = (s["ctx_len"]).long()
    for i in range(t):
        s["path"][:, i] = torch.where(going, at, NONE)
        s["count"].add_(going)
        where = (end + i).clamp(max=s["history"].shape[1] - 1)
        s["history"][rows, where] = torch.where(going, s["tokens"][rows, at], s["history"][rows, where])
        want = s["picked"][rows, at]
        s["next"].copy_(torch.where(going, want, s["next"]))
        child = torch.where(present & (s["parents"] == at[:, None]) & (s["tokens"] == want[:, None]), idx, t).min(1).values
        going = going & (child < t)
        at = torch.where(going, child, at)
    s["after"].copy_(s["ctx_len"] + s["count"])
    return {k: s[k] for k in ("path", "count", "next", "after", "history")}


def _plain_compact(s, c):
    n, t = c["seqs"], c["tree"]
    first = (s["ctx_len"] - s["count"]).long()[:, None]
    i = torch.arange(t, device="cuda")
    moved = i < s["count"][:, None]
    to = first + i
    come = torch.where(moved, first + s["path"], to)
    rows = torch.arange(n, device="cuda")[:, None]
    s["caches"][:, :, rows, to] = s["caches"][:, :, rows, come]
    return s["caches"]


# --------------------------------------------------------------- what it takes
def work(case):
    c, n, t = case, case["seqs"], case["tree"]
    if c["op"] == "attn":
        h, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
        # a batch's lengths are spread evenly over their logarithm up to ctx, one of them is ctx
        keys = c["ctx"] if n == 1 else int(c["ctx"] * (1 + (n - 1) / math.log(c["ctx"] + 2)))
        rows = n * t
        # cache rows read, the nodes' rows in and out, two products over the cache and the path
        return dict(bytes=4 * keys * kv * d + rows * (4 * (2 * h + 2 * kv) * d + 4 * kv * d), flops=4 * (keys * t + rows) * h * d)
    if c["op"] == "logits":
        rows, v = n * max(1, t), c["vocab"]
        each = 4 * v * (2 if c["write"] else 1) + 4 + (v // 8 if c["mask"] else 0)
        return dict(bytes=rows * each + 4 * n * c["history"] + 8 * c["bias"], flops=3 * rows * v)
    if c["op"] == "accept":
        return dict(bytes=n * (4 * 4 * t + 16), flops=0)
    most = min(8, (t + 1) // 2)  # path lengths: one sequence has this one, a batch all up to it; node 0 stays where it is
    rows = (most - 1) * (0.5 * n if n > 1 else 1) * c["layers"] * 2
    return dict(bytes=2 * rows * c["kv_heads"] * c["head_dim"] * 2 + 4 * n * (t + 2), flops=0)


# --------------------------------------------------------------------- 64 bits
def _paths(parents):
    """For each node the list of nodes from the cache's end to it, or None where it is not there."""
    out = []
    for t, p in enumerate(parents):
        if p == -1:
            out.append([t])
        else:
            out.append(out[p] + [t] if 0 <= p < t and out[p] is not None else None)
    return out


def _exact_attn(s, c):
    t, h, kv, d = c["tree"], c["heads"], c["kv_heads"], c["head_dim"]
    g = h // kv
    kc, vc = s["k"].double(), s["v"].double()
    out = torch.zeros((c["seqs"], t, h, d), dtype=torch.float64, device="cuda")
    rows = s["qkv"].double().view(c["seqs"], t, h + 2 * kv, d)
    inv = s["inv"].double()
    for i, length in enumerate(s["lens"]):
        paths = _paths(s["parents"][i].tolist())
        see = torch.zeros((t, length + t), dtype=torch.bool, device="cuda")
        turned = rows[i].clone()
        for j, p in enumerate(paths):
            if p is None:
                continue
            see[j, :length] = True
            see[j, [length + x for x in p]] = True
            a = (length + len(p) - 1) * inv
            x, y = rows[i, j, :h + kv, :d // 2], rows[i, j, :h + kv, d // 2:]
            turned[j, :h + kv, :d // 2] = x * a.cos() - y * a.sin()
            turned[j, :h + kv, d // 2:] = y * a.cos() + x * a.sin()
            kc[i, length + j] = turned[j, h:h + kv].float().half().double()
            vc[i, length + j] = turned[j, h + kv:].float().half().double()
        some = [j for j, p in enumerate(paths) if p is not None]
        for head in range(h if some else 0):
            keys = kc[i, :length + t, head // g].t().contiguous()
            w = torch.exp(torch.log_softmax((turned[some, head].contiguous() @ keys / math.sqrt(d)).masked_fill(
                ~see[some], -math.inf), -1))
            out[i, some, head] = w @ vc[i, :length + t, head // g].contiguous()
    return dict(out=out.view(-1, h * d), k=kc, v=vc)


def _exact_logits(s, c):
    n, t, v = c["seqs"], c["tree"], c["vocab"]
    rep, freq, pres = (np.float64(x) for x in s["penalties"])
    x = s["wide"][:, :v].cpu().numpy().astype(np.float64)
    history, lens = s["history"].cpu().numpy(), s["history_len"].cpu().numpy()
    for i in range(n):
        base = np.bincount(history[i, :lens[i]], minlength=v)
        paths = _paths(s["parents"][i].tolist()) if t else [[]]
        for j, p in enumerate(paths):
            row = x[i * len(paths) + j]
            count = base.copy()
            if t:
                np.add.at(count, s["tokens"][i].cpu().numpy()[p], 1)
            hit = np.flatnonzero(count)
            row[hit] *= np.where(row[hit] > 0, 1 / rep, rep)
            row[hit] -= freq * count[hit] + pres
    if c["bias"]:
        entries = dict(zip(s["bias_ids"].tolist(), s["bias"].cpu().numpy().astype(np.float64)))
        x[:, list(entries)] += np.array(list(entries.values()))
    if c["mask"]:
        bits = np.unpackbits(s["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :v]
        x[bits == 0] = -np.inf
    token = np.where(x.max(1) > -np.inf, x.argmax(1), NONE)
    token = torch.from_numpy(token.astype(np.int32))
    return dict(token=token, out=torch.from_numpy(x)) if c["write"] else dict(token=token)


def _exact_accept(s, c):
    a = {k: s[k].cpu().numpy() for k in ("parents", "tokens", "picked", "ctx_len", "history")}
    n, t = c["seqs"], c["tree"]
    path, count, nxt, history = np.full((n, t), NONE), np.zeros(n, int), np.full(n, NONE), a["history"].copy()
    for i in range(n):
        paths = _paths(a["parents"][i].tolist())
        at = 0 if paths[0] is not None else None
        while at is not None:
            path[i, count[i]] = at
            history[i, a["ctx_len"][i] + count[i]] = a["tokens"][i, at]
            count[i] += 1
            nxt[i] = a["picked"][i, at]
            at = next((j for j in range(at + 1, t)
                       if paths[j] is not None and a["parents"][i, j] == at and a["tokens"][i, j] == nxt[i]), None)
    whole = dict(path=path, count=count, next=nxt, after=a["ctx_len"] + count, history=history)
    return {k: torch.from_numpy(np.asarray(v, np.int32)) for k, v in whole.items()}


def _exact_compact(s, c):
    old, new = s["caches"], s["caches"].clone()
    path, count, after = s["path"].tolist(), s["count"].tolist(), s["ctx_len"].tolist()
    for i in range(c["seqs"]):
        for j in range(count[i]):
            new[:, :, i, after[i] - count[i] + j] = old[:, :, i, after[i] - count[i] + path[i][j]]
    return new


def exact(case, seed):
    s = _inputs(case, seed)
    return dict(attn=_exact_attn, logits=_exact_logits, accept=_exact_accept, compact=_exact_compact)[case["op"]](s, case)
