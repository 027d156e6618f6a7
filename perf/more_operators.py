"""Performance cases of the operators that run several continuations of one prompt.

A prompt's cache rows are shared by a group of members: the beams of a search, samples of one prompt, or requests behind
one system prompt.  Each member has rows of its own behind them, and all take their next token in one step.

  op        one pass
  rope      qk_norm_rope: RMS norms of the query and key heads, the rotation by position, the new rows into the f16 caches
  attn      attention_shared: grouped-query attention of every member over the shared prefix and its own rows
  select    beam_select: log-probabilities of every beam's logits, the best continuations of a sequence, its histories
  reorder   beam_reorder: the cache rows of every layer follow the beams that were chosen

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
        # one step of a beam search: a row per beam, where the launch counts
        dict(name="rope_8_beams", op="rope", groups=1, per=8, new=1, heads=32, kv_heads=8, head_dim=128, rot_dim=128, inter=False,
             norm=False, base=4000, own=200),
        # a long prompt of a model that normalises its queries and keys
        dict(name="rope_prompt_4000_norm", op="rope", groups=1, per=1, new=4000, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             inter=False, norm=True, base=0, own=4000),
        # prompts of mixed lengths, small heads of which a half turns, in neighbouring pairs
        dict(name="rope_16_prompts_ragged_d64", op="rope", groups=16, per=1, new=300, heads=32, kv_heads=4, head_dim=64, rot_dim=32,
             inter=True, norm=False, base=0, own=500),
        # a small search over a short prompt: the smallest attention
        dict(name="attn_4_beams_p900", op="attn", groups=1, per=4, prefix=900, own=60, even=True, heads=32, kv_heads=8, head_dim=128),
        # beams behind a long document
        dict(name="attn_8_beams_p30000", op="attn", groups=1, per=8, prefix=30000, own=250, even=True, heads=32, kv_heads=8,
             head_dim=128),
        # searches for several prompts of mixed lengths, small heads
        dict(name="attn_6x5_ragged_d64", op="attn", groups=6, per=5, prefix=12000, own=100, even=True, heads=32, kv_heads=4,
             head_dim=64),
        # requests behind one system prompt, each with its own part
        dict(name="attn_64_p6000_ragged", op="attn", groups=1, per=64, prefix=6000, own=700, even=False, heads=32, kv_heads=8,
             head_dim=128),
        # questions to a whole book
        dict(name="attn_48_p131000", op="attn", groups=1, per=48, prefix=131000, own=400, even=False, heads=32, kv_heads=8,
             head_dim=128),
        # a small search
        dict(name="select_4x32000", op="select", seqs=1, beams=4, out=4, vocab=32000, pad=0, end=False, alpha=0.0, history=60),
        # searches of a batch: some beams have ended, scores go by length
        dict(name="select_16x8x128256", op="select", seqs=16, beams=8, out=8, vocab=128256, pad=0, end=True, alpha=0.8, history=200),
        # the rows behind a search's first tokens, and behind many
        dict(name="reorder_32_layers_x4_60", op="reorder", layers=32, seqs=1, beams=4, rows=60, kv_heads=8, head_dim=128),
        dict(name="reorder_32_layers_x8_500", op="reorder", layers=32, seqs=1, beams=8, rows=500, kv_heads=8, head_dim=128),
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "rope", "attn", "attn", "attn", "attn", "select", "select", "reorder"])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    if op == "rope":
        heads, d = kv * rng.choice([1, 2, 4, 4, 5, 8]), rng.choice([64, 80, 96, 128, 128, 256])
        groups, per, new = _log(rng, 1, 16), _log(rng, 1, 16), rng.choice([1, 1, _log(rng, 2, 4000)])
        while groups * per * new * (heads + 2 * kv) * d > 4000 * 48 * 128:
            groups, per, new = max(1, groups // 2), max(1, per // 2), max(1, new // 2)
        return dict(op=op, groups=groups, per=per, new=new, heads=heads, kv_heads=kv, head_dim=d,
                    rot_dim=rng.choice([d, d, d // 2, d // 4]), inter=rng.random() < 0.5, norm=rng.random() < 0.5,
                    base=rng.choice([0, _log(rng, 1, 100000)]), own=new + rng.choice([0, _log(rng, 1, 300)]))
    if op == "attn":
        heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        groups, per = rng.choice([1, 1, _log(rng, 2, 12)]), _log(rng, 1, 64)
        prefix, rows = _log(rng, 1, 100000), _log(rng, 1, 800)
        while groups * prefix * heads * (per + 32) > 131000 * 32 * 64 or groups * prefix * kv > 8 * 131000:
            groups, prefix = (groups + 1) // 2, prefix // 2 + 1
        return dict(op=op, groups=groups, per=per, prefix=prefix, own=rows, even=rng.random() < 0.5, heads=heads, kv_heads=kv,
                    head_dim=rng.choice([64, 128, 128]))
    if op == "select":
        seqs, beams, vocab = _log(rng, 1, 32), _log(rng, 1, 32), _log(rng, 1000, 160000)
        while seqs * beams * vocab > 16 * 8 * 128256:
            seqs, beams = max(1, seqs // 2), (beams + 1) // 2
        out = rng.choice([beams, beams, 2 * beams])  # twice as many: for a caller that sets ended ones aside by itself
        return dict(op=op, seqs=seqs, beams=beams, out=out, vocab=vocab, pad=rng.choice([0, 0, rng.randint(1, 64)]),
                    end=out == beams and rng.random() < 0.6, alpha=rng.choice([0.0, 0.6, 1.0]), history=_log(rng, 1, 1000))
    seqs, beams, layers, rows = _log(rng, 1, 8), _log(rng, 2, 32), rng.randint(1, 32), _log(rng, 1, 800)
    while layers * seqs * beams * rows * kv > 32 * 8 * 500 * 8:
        seqs, layers, rows = max(1, seqs // 2), max(1, layers // 2), rows // 2 + 1
    return dict(op=op, layers=layers, seqs=seqs, beams=beams, rows=rows, kv_heads=kv, head_dim=rng.choice([64, 80, 128]))


# ------------------------------------------------------------------- inputs
def _rng(case, seed):
    return np.random.default_rng([int(seed) & 0x7FFFFFFF, len(case["op"]), case.get("groups", 0), case.get("seqs", 0)])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a).astype(dtype)).cuda()


def _lengths(r, n, most):
    """One: `most`.  Several: from 1 (from 0 where there are many) to `most`, spread over their logarithm, one of them `most`."""
    if n == 1:
        return [most]
    lens = [int(v) for v in np.exp(r.uniform(0, math.log(most + 1), n))]
    lens[int(r.integers(0, n))] = most
    if n > 3:
        lens[lens.index(min(lens))] = 0
    return lens


def _rope_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, h, kv, d, rot = c["groups"] * c["per"], c["heads"], c["kv_heads"], c["head_dim"], c["rot_dim"]
    # tokens of a member, the new ones included; prompts of a batch may be shorter than the longest one
    lens = [c["own"]] if n == 1 else [int(v) for v in r.integers(1 if c["new"] > 1 else max(1, c["own"] // 2), c["own"] + 1, n)]
    room = c["own"] + 3
    inv = 1.0 / ROPE_BASE ** (np.arange(0, rot, 2) / rot) / (4.0 if c["inter"] else 1.0)
    s = dict(qkv=torch.randn((n * c["new"], (h + 2 * kv) * d), device="cuda", generator=g) * 1.3, lens=lens, room=room,
             base_lens=[int(v) for v in r.integers(c["base"] // 2, c["base"] + 1, c["groups"])], inv=_dev(inv, np.float32),
             k=torch.randn((n, room, kv, d), device="cuda", generator=g, dtype=torch.float16),
             v=torch.randn((n, room, kv, d), device="cuda", generator=g, dtype=torch.float16), magnitude=1.1 if c["inter"] else 1.0)
    if c["norm"]:
        s["q_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
        s["k_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
    s.update(base=_dev(s["base_lens"], np.int32), len=_dev(lens, np.int32))
    return s


def _attn_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, h, kv, d = c["groups"] * c["per"], c["heads"], c["kv_heads"], c["head_dim"]
    prefix = _lengths(r, c["groups"], c["prefix"])
    # beams of a search have the same number of tokens, requests their own
    mine = np.repeat(r.integers((c["own"] + 1) // 2, c["own"] + 1, c["groups"]), c["per"]) if c["even"] else r.integers(1, c["own"] + 1, n)
    f16 = dict(device="cuda", generator=g, dtype=torch.float16)
    room, mine_room = c["prefix"] + 5, c["own"] + 3
    return dict(q=torch.randn((n, h * d), device="cuda", generator=g) * 1.3, prefix_lens=prefix, own_lens=[int(v) for v in mine],
                k=torch.randn((c["groups"], room, kv, d), **f16), v=torch.randn((c["groups"], room, kv, d), **f16),
                k_own=torch.randn((n, mine_room, kv, d), **f16), v_own=torch.randn((n, mine_room, kv, d), **f16),
                prefix_len=_dev(prefix, np.int32), own_len=_dev(mine, np.int32), room=room, own_room=mine_room)


def _select_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, b, v = c["seqs"], c["beams"], c["vocab"]
    wide = torch.randn((n * b, v + c["pad"]), device="cuda", generator=g) * 3.0 - 2.0
    lens = r.integers((c["history"] + 1) // 2, c["history"] + 1, n)
    scores = -np.sort(r.random((n, b)) * 3.0 + 0.4 * lens[:, None], 1)
    last = r.integers(0, v, (n, b))
    counts = np.repeat(lens[:, None], b, 1)
    s = dict(wide=wide, rows=n * b, end=NONE)
    if c["end"]:
        s["end"] = int(r.integers(0, v))
        ended = r.random((n, b)) < 0.2  # a beam that has ended did so some tokens ago
        last = np.where(ended, s["end"], np.where(last == s["end"], (last + 1) % v, last))
        counts = np.where(ended, r.integers(1, counts + 1), counts)
    history = r.integers(0, v, (n, b, c["history"] + 4))
    s.update(scores=_dev(scores, np.float32), last=_dev(last, np.int32), counts=_dev(counts, np.int32),
             history=_dev(history, np.int32), len=_dev(np.repeat(lens[:, None], b, 1), np.int32))
    return s


def _reorder_inputs(c, seed):
    r, g = _rng(c, seed), _gen(seed)
    n, b = c["seqs"], c["beams"]
    # every second beam gives way to a continuation of another one
    parents = np.tile(np.arange(b), (n, 1))
    parents[:, 1::2] = 2 * r.integers(0, (b + 1) // 2, (n, b // 2))
    rows = [c["rows"]] if n == 1 else [int(x) for x in r.integers((c["rows"] + 1) // 2, c["rows"] + 1, n)]
    caches = torch.randn((c["layers"], 2, n, b, c["rows"] + 6, c["kv_heads"], c["head_dim"]), device="cuda", generator=g,
                         dtype=torch.float16)
    # the token that was just chosen has no rows yet
    return dict(caches=caches, host_parents=parents, host_rows=rows, parents=_dev(parents, np.int32),
                len=_dev(np.repeat(np.array(rows)[:, None] + 1, b, 1), np.int32))


def _inputs(case, seed):
    return dict(rope=_rope_inputs, attn=_attn_inputs, select=_select_inputs, reorder=_reorder_inputs)[case["op"]](case, seed)


class _Queue:
    """torch's current stream as the framework's calls take it."""

    def __init__(self):
        self.handle = torch.cuda.current_stream().cuda_stream or None


def prepare(case, seed):
    s, c = _inputs(case, seed), case
    s["case"] = c
    if c["op"] == "rope":
        s["q_out"] = torch.zeros((s["qkv"].shape[0], c["heads"] * c["head_dim"]), device="cuda")
    if c["op"] == "attn":
        s["out"] = torch.zeros_like(s["q"])
    if c["op"] == "select":
        i32, shape = dict(dtype=torch.int32, device="cuda"), (c["seqs"], c["out"])
        s.update(scores_out=torch.zeros(shape, device="cuda"), tokens=torch.zeros(shape, **i32), parents=torch.zeros(shape, **i32),
                 counts_out=torch.zeros(shape, **i32))
        if c["out"] == c["beams"]:
            s["len_out"] = torch.zeros(shape, **i32)
    if own:
        from woolly_amd import device, ops

        device.init(torch.cuda.current_device())
        need = 0
        if c["op"] == "rope":
            s["rules"] = ops.RopeRules(inv_freq=s["inv"].data_ptr(), rot_dim=c["rot_dim"], interleaved=c["inter"],
                                       magnitude=s["magnitude"], q_norm=s["q_norm"].data_ptr() if c["norm"] else None,
                                       k_norm=s["k_norm"].data_ptr() if c["norm"] else None, eps=1e-6)
        if c["op"] == "attn":
            need = ops.attention_shared_workspace_bytes(c["groups"], c["per"], c["heads"], c["kv_heads"], c["head_dim"], s["room"],
                                                        s["own_room"])
        if c["op"] == "select":
            same = c["out"] == c["beams"]
            s["rules"] = ops.BeamRules(
                n_beams=c["beams"], n_out=c["out"], end_token=s["end"] & 0xFFFFFFFF, length_penalty=c["alpha"],
                last_tokens=s["last"].data_ptr() if c["end"] else None, counts=s["counts"].data_ptr(),
                counts_out=s["counts_out"].data_ptr(), history=s["history"].data_ptr() if same else None,
                history_stride=s["history"].shape[2] if same else 0, len=s["len"].data_ptr() if same else None,
                len_out=s["len_out"].data_ptr() if same else None)
            need = ops.beam_select_workspace_bytes(s["rules"], c["seqs"], c["vocab"])
        if c["op"] == "reorder":
            s["states"] = ops.BeamStates([x.data_ptr() for layer in s["caches"] for x in layer])
        s["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------- a pass
def run(s):
    c = s["case"]
    if not own:
        return dict(rope=_plain_rope, attn=_plain_attn, select=_plain_select, reorder=_plain_reorder)[c["op"]](s, c)
    from woolly_amd import ops

    queue = _Queue()
    if c["op"] == "rope":
        h, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
        q, ld = s["qkv"].data_ptr(), (h + 2 * kv) * d
        ops.qk_norm_rope(s["rules"], q, q + 4 * h * d, q + 4 * (h + kv) * d, ld, ld, s["base"].data_ptr(), s["len"].data_ptr(),
                         c["groups"], c["per"], c["new"], h, kv, d, s["q_out"].data_ptr(), h * d, None, 0, s["k"].data_ptr(),
                         s["v"].data_ptr(), s["room"], queue)
        return dict(q=s["q_out"], k=s["k"], v=s["v"])
    if c["op"] == "attn":
        h, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
        ops.attention_shared(s["q"].data_ptr(), h * d, s["prefix_len"].data_ptr(), s["own_len"].data_ptr(), c["groups"], c["per"],
                             s["k"].data_ptr(), s["v"].data_ptr(), s["room"], s["k_own"].data_ptr(), s["v_own"].data_ptr(),
                             s["own_room"], h, kv, d, s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), queue)
        return s["out"]
    if c["op"] == "select":
        ops.beam_select(s["rules"], s["wide"].data_ptr(), c["vocab"] + c["pad"], c["seqs"], c["vocab"], s["scores"].data_ptr(),
                        s["scores_out"].data_ptr(), s["tokens"].data_ptr(), s["parents"].data_ptr(), s["ws"].data_ptr(),
                        s["ws"].numel(), queue)
        return _select_outputs(s, c)
    ops.beam_reorder(s["states"], c["seqs"], c["beams"], c["rows"] + 6, c["kv_heads"] * c["head_dim"] * 2, s["parents"].data_ptr(),
                     s["len"].data_ptr(), 1, queue)
    return s["caches"]


def _select_outputs(s, c):
    names = ["scores_out", "tokens", "parents", "counts_out"] + (["history", "len_out"] if c["out"] == c["beams"] else [])
    return {k: s[k] for k in names}


# --------------------------------------------------------------- plain forms
def _plain_rope(s, c):
    n, new, h, kv, d, rot = c["groups"] * c["per"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["rot_dim"]
    q, k, v = s["qkv"].view(n, new, h + 2 * kv, d).split([h, kv, kv], 2)
    row = s["len"][:, None] - new + torch.arange(new, device="cuda")
    pos = row + s["base"].repeat_interleave(c["per"])[:, None]
    angle = pos.double()[:, :, None, None] * s["inv"].double()
    there = (row >= 0)[:, :, None, None]

    def turn(x, weight, wide):
        if weight is not None:
            x = x / ((x * x).mean(-1, keepdim=True) + 1e-6).sqrt() * weight
        x = x.to(wide)
        cos, sin = (s["magnitude"] * angle.cos()).to(wide), (s["magnitude"] * angle.sin()).to(wide)
        a, rest = x[..., :rot], x[..., rot:]
        if c["inter"]:
            a1, a2 = a[..., 0::2], a[..., 1::2]
            a = torch.stack([a1 * cos - a2 * sin, a1 * sin + a2 * cos], -1).flatten(-2)
        else:
            a1, a2 = a.chunk(2, -1)
            a = torch.cat([a1 * cos - a2 * sin, a1 * sin + a2 * cos], -1)
        return torch.cat([a, rest], -1)

    s["q_out"].view(n, new, h, d).copy_(torch.where(there, turn(q, s.get("q_norm"), torch.float32), 0.0))
    k = turn(k, s.get("k_norm"), torch.float64).float().half()
    for i, length in enumerate(s["lens"]):
        t = min(new, length)
        s["k"][i, length - t:length] = k[i, new - t:]
        s["v"][i, length - t:length] = v[i, new - t:].half()
    return dict(q=s["q_out"], k=s["k"], v=s["v"])


def _plain_attn(s, c):
    per, h, kv, d = c["per"], c["heads"], c["kv_heads"], c["head_dim"]
    g = h // kv
    for i, length in enumerate(s["prefix_lens"]):
        q = s["q"].view(-1, per, kv, g, d)[i].permute(1, 0, 2, 3).reshape(kv, per * g, d)
        keys = s["k"][i, :length].float().permute(1, 2, 0).contiguous()
        shared = (q @ keys / math.sqrt(d)).view(kv, per, g, length)
        vals = s["v"][i, :length].float().permute(1, 0, 2).contiguous()
        for j in range(per):
            m = i * per + j
            rows = s["own_lens"][m]
            keys = s["k_own"][m, :rows].float().permute(1, 2, 0).contiguous()
            mine = q.view(kv, per, g, d)[:, j].contiguous() @ keys / math.sqrt(d)
            w = torch.cat([shared[:, j], mine], -1)
            w -= w.max(-1, keepdim=True).values
            w.exp_()
            total = w.sum(-1, keepdim=True)
            o = w[..., :length].contiguous() @ vals
            o = o + w[..., length:].contiguous() @ s["v_own"][m, :rows].float().permute(1, 0, 2).contiguous()
            s["out"].view(-1, kv, g, d)[m] = o / total
    return s["out"]


def _plain_select(s, c):
    n, b, v, out = c["seqs"], c["beams"], c["vocab"], c["out"]
    x = s["wide"][:, :v].double()
    top = x.max(1, keepdim=True).values
    x = x - (top + (x - top).exp().sum(1, keepdim=True).log())
    x = x.view(n, b, v) + s["scores"].double()[:, :, None]
    ended = (s["last"] == s["end"]) if c["end"] else torch.zeros((n, b), dtype=torch.bool, device="cuda")
    # one that has ended goes on as it is
    at_end = (torch.arange(v, device="cuda") == s["end"])[None, None]
    x = torch.where(ended[:, :, None], torch.where(at_end, s["scores"].double()[:, :, None], -math.inf), x)
    counts = torch.where(ended, s["counts"], s["counts"] + 1)
    rank = (x / counts.clamp(min=1).double()[:, :, None] ** c["alpha"]).view(n, b * v)
    x = x.view(n, b * v)
    for i in range(out):
        best = rank.max(1, keepdim=True).values
        at = torch.where(rank == best, torch.arange(b * v, device="cuda"), b * v).min(1, keepdim=True).values
        beam = at // v
        s["scores_out"][:, i:i + 1] = x.gather(1, at).float()
        s["tokens"][:, i:i + 1] = (at % v).int()
        s["parents"][:, i:i + 1] = beam.int()
        s["counts_out"][:, i:i + 1] = counts.gather(1, beam)
        rank.scatter_(1, at, -math.inf)
    if out == b:
        parents = s["parents"].long()
        old = s["history"].gather(1, parents[:, :, None].expand(s["history"].shape))
        length = s["len"].gather(1, parents)
        i = torch.arange(old.shape[2], device="cuda")
        new = torch.where(i < length[:, :, None], old, s["history"])
        s["history"].copy_(torch.where(i == length[:, :, None], s["tokens"][:, :, None], new))
        s["len_out"].copy_(length + 1)
    return _select_outputs(s, c)


def _plain_reorder(s, c):
    for i, rows in enumerate(s["host_rows"]):
        some = s["caches"][:, :, i, :, :rows]
        s["caches"][:, :, i, :, :rows] = some[:, :, s["parents"][i].long()]
    return s["caches"]


# --------------------------------------------------------------- what it takes
def work(case):
    c = case
    if c["op"] == "rope":
        rows, h, kv, d = c["groups"] * c["per"] * c["new"], c["heads"], c["kv_heads"], c["head_dim"]
        # rows of q, k and v in, q out, k and v into the caches; norm, rotation
        return dict(bytes=rows * d * (4 * (2 * h + 2 * kv) + 4 * kv) + 4 * c["rot_dim"], flops=rows * d * (3 * h + 3 * kv) +
                    (4 * rows * d * (h + kv) if c["norm"] else 0))
    if c["op"] == "attn":
        n, h, kv, d = c["groups"] * c["per"], c["heads"], c["kv_heads"], c["head_dim"]
        # lengths of several groups are spread evenly over their logarithm up to the longest, own rows over the upper half or all
        groups = c["groups"]
        shared = c["prefix"] if groups == 1 else int(c["prefix"] * (1 + (groups - 1) / math.log(c["prefix"] + 2)))
        mine = int(n * c["own"] * (0.75 if c["even"] else 0.5)) + 1
        return dict(bytes=4 * (shared + mine) * kv * d + 8 * n * h * d, flops=4 * (shared * c["per"] + mine) * h * d)
    if c["op"] == "select":
        rows, tokens = c["seqs"] * c["beams"], c["seqs"] * c["beams"] * c["history"]
        return dict(bytes=4 * rows * c["vocab"] + (6 * tokens if c["out"] == c["beams"] else 0) + 16 * c["seqs"] * c["out"],
                    flops=3 * rows * c["vocab"])
    moved, whole = c["beams"] // 2, (c["beams"] + 1) // 2
    read = whole * (1 - (1 - 1 / whole) ** moved)  # beams that some moved one continues
    rows = c["rows"] * (1 if c["seqs"] == 1 else 0.75 * c["seqs"])
    return dict(bytes=int((moved + read) * rows * c["layers"] * 2 * c["kv_heads"] * c["head_dim"] * 2), flops=0)


# --------------------------------------------------------------------- 64 bits
def _exact_rope(s, c):
    new, h, kv, d, rot = c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["rot_dim"]
    rows = s["qkv"].double().view(-1, new, h + 2 * kv, d)
    q_out = torch.zeros((rows.shape[0], new, h, d), dtype=torch.float64, device="cuda")
    kc, vc, inv = s["k"].double(), s["v"].double(), s["inv"].double()
    first = torch.arange(0, rot, 2, device="cuda") if c["inter"] else torch.arange(rot // 2, device="cuda")
    second = first + (1 if c["inter"] else rot // 2)
    for m, length in enumerate(s["lens"]):
        t = min(new, length)
        if t == 0:
            continue
        x = rows[m, new - t:].clone()
        if c["norm"]:
            weight = torch.cat([s["q_norm"].double().expand(h, d), s["k_norm"].double().expand(kv, d)])
            some = x[:, :h + kv]
            x[:, :h + kv] = some * weight / (some.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt()
        at = s["base_lens"][m // c["per"]] + torch.arange(length - t, length, device="cuda").double()
        turn = torch.polar(torch.full((t, rot // 2), s["magnitude"], dtype=torch.float64, device="cuda"), at[:, None] * inv)
        pairs = torch.complex(x[:, :h + kv, first], x[:, :h + kv, second]) * turn[:, None]
        x[:, :h + kv, first], x[:, :h + kv, second] = pairs.real, pairs.imag
        q_out[m, new - t:] = x[:, :h]
        kc[m, length - t:length] = x[:, h:h + kv].float().half().double()
        vc[m, length - t:length] = x[:, h + kv:].float().half().double()
    return dict(q=q_out.view(-1, h * d), k=kc, v=vc)


def _exact_attn(s, c):
    per, h, kv, d = c["per"], c["heads"], c["kv_heads"], c["head_dim"]
    q = s["q"].double().view(-1, h, d)
    out = torch.zeros_like(q)
    for i, length in enumerate(s["prefix_lens"]):
        for head in range(h):
            keys, vals = (s[x][i, :length, head // (h // kv)].double().contiguous() for x in ("k", "v"))
            score = keys @ q[i * per:(i + 1) * per, head].t().contiguous() / math.sqrt(d)
            for j in range(per):
                m = i * per + j
                mine, mine_v = (s[x][m, :s["own_lens"][m], head // (h // kv)].double().contiguous() for x in ("k_own", "v_own"))
                w = torch.softmax(torch.cat([score[:, j], mine @ q[m, head] / math.sqrt(d)]), 0)
                out[m, head] = w[:length] @ vals + w[length:] @ mine_v
    return out.view(-1, h * d)


def _exact_select(s, c):
    n, b, v, out = c["seqs"], c["beams"], c["vocab"], c["out"]
    a = {k: s[k].cpu().numpy() for k in ("scores", "last", "counts", "history", "len")}
    x = s["wide"][:, :v].cpu().numpy().astype(np.float64)
    best = {k: np.zeros((n, out), t) for k, t in (("scores_out", np.float64), ("tokens", np.int32), ("parents", np.int32),
                                                  ("counts_out", np.int32))}
    history, len_out = a["history"].copy(), np.zeros((n, out), np.int32)
    for i in range(n):
        found = []  # (-rank, beam, token, score, count)
        for j in range(b):
            score, count = float(a["scores"][i, j]), int(a["counts"][i, j])
            if c["end"] and a["last"][i, j] == s["end"]:
                found.append((-score / max(count, 1) ** c["alpha"], j, s["end"], score, count))
                continue
            row = x[i * b + j]
            row = score + (row - np.logaddexp.reduce(row))
            some = np.flatnonzero(row >= np.partition(row, v - out)[v - out])
            found += [(-float(row[t]) / (count + 1) ** c["alpha"], j, int(t), float(row[t]), count + 1) for t in some]
        for k, (_, j, t, score, count) in enumerate(sorted(found)[:out]):
            for name, value in (("scores_out", score), ("tokens", t), ("parents", j), ("counts_out", count)):
                best[name][i, k] = value
            if out == b:
                length = a["len"][i, j]
                history[i, k, :length] = a["history"][i, j, :length]
                history[i, k, length] = t
                len_out[i, k] = length + 1
    if out == b:
        best.update(history=history, len_out=len_out)
    return {k: torch.from_numpy(y) for k, y in best.items()}


def _exact_reorder(s, c):
    new = s["caches"].clone()
    for i, rows in enumerate(s["host_rows"]):
        for j, parent in enumerate(s["host_parents"][i].tolist()):
            new[:, :, i, j, :rows] = s["caches"][:, :, i, parent, :rows]
    return new


def exact(case, seed):
    s = _inputs(case, seed)
    return dict(rope=_exact_rope, attn=_exact_attn, select=_exact_select, reorder=_exact_reorder)[case["op"]](s, case)
