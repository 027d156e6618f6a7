"""The operators for several continuations of one prompt together, as a program uses them: a beam search on the device, with
the model's step and with the operators by themselves."""
import numpy as np
import pytest

from tests import _members
from tests._gpu import down, up
from tests._oracle import rel_l2
from tests.test_gpu_tree_step import MODELS, Q4_K, Q6_K, Q8_0, Model
from tests.test_oracle_decode import PROJ, mixed_layer, small_layer
from woolly_amd import ops, synth
from woolly_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
u32 = lambda a: np.asarray(a).astype(np.uint32)
SCORE = 2.0 ** -23


def own_caches(m, members, rows):
    bufs = [[DeviceBuffer(members * rows * m.kv * m.d * 2) for _ in range(m.layers)] for _ in range(2)]
    for b in bufs[0] + bufs[1]:
        b.fill(0xFF)  # NaN until a row is written
    return bufs, ops.KvCaches(*bufs)


def prompt_into(m, prompt):
    """The prompt as a chain of drafts fills the members' model's caches; the decode step's logits behind it."""
    t = len(prompt)
    wsz = m.tree.tree_workspace_bytes(t)
    m.tree.forward_tree(up(u32(prompt))[0], up(np.arange(-1, t - 1, dtype=np.int32))[0], t, up(u32([0]))[0],
                        DeviceBuffer(4 * t * m.hidden), None, DeviceBuffer(wsz), wsz)
    for i, tok in enumerate(prompt):
        logits = m.step(tok, i)
    return logits


class Exact:
    """The model's step in 64 bits for one token, over cache rows that the device stored.

    A cache row is rounded to f16.  Where a value lies next to the border of two f16, f32 forms round it either way, 2^-11
    of it apart, and a softmax carries that into the logits: two right forms of a step differ by up to some 1e-4.  So the
    rows are compared by themselves, by one f16 step, and the logits on the same rows, by the decode step's bar of 1e-4."""

    def __init__(self, orc, name, vocab, seed):
        t, hidden, heads, kv, d, n_ff = MODELS[name]
        types = {p: Q6_K if p in ("wv", "w_down") else Q4_K for p in PROJ}
        self.layers = [mixed_layer(types, hidden, heads, kv, d, n_ff, seed=seed + i) if t == "mixed" else
                       small_layer(t, hidden, heads, kv, d, n_ff, seed=seed + i) for i in range(2)]
        self.t = [types[p] for p in PROJ] if t == "mixed" else t
        rng = np.random.default_rng(seed)
        self.norm = (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)
        self.embd = rng.standard_normal((vocab, hidden)).astype(np.float16)
        self.head = synth.quantized_weight(Q8_0, vocab, hidden, seed=seed + 99)
        self.dims, self.inv = (hidden, heads, kv, d, n_ff, 1e-5), ops.rope_inv_freq(10000.0, d)
        self.orc, self.hidden, self.vocab, self.row = orc, hidden, vocab, (kv, d)

    def logits(self, token, caches):
        """caches: per layer (K rows, V rows) f16, the token's own row the last; checks that row."""
        x = self.embd[token].astype(np.float64)
        for (k, v), layer in zip(caches, self.layers):
            k, v = (np.ascontiguousarray(a).view(np.uint16).copy() for a in (k, v))
            pos = len(k) - 1
            own = [a.copy() for a in (k, v)]
            self.orc.llama_layer_decode_f64(self.t, layer, self.dims, self.inv, own[0], own[1], pos, x)
            for a, b in zip(own, (k, v)):
                want, got = (z[pos].view(np.float16).astype(np.float64) for z in (a, b))
                assert (np.abs(got - want) <= 2.0 ** -10 * np.abs(want) + 1e-4 * np.sqrt((want ** 2).mean())).all()
            x = self.orc.llama_layer_decode_f64(self.t, layer, self.dims, self.inv, k, v, pos, x, store_new=False)
        return np.asarray(self.orc.output_head_f64(Q8_0, self.head, self.norm, 1e-5, x, self.hidden, self.vocab))


def member_rows(m, bufs, prompt_len, members, rows, i, n):
    """Per layer the K and V rows that member i sees with n tokens of its own."""
    shape = (members, rows, m.kv, m.d)
    shared = m.rows(1, prompt_len)
    out = []
    for layer in range(m.layers):
        pair = []
        for which in range(2):
            own = down(bufs[which][layer], np.float16, members * rows * m.kv * m.d).reshape(shape)[i, :n]
            pair.append(np.concatenate([shared[2 * layer + which].astype(np.float16), own]))
        out.append(pair)
    return out


@pytest.mark.parametrize("name", list(MODELS))
def test_members_logits_are_the_paths_logits(gpu, orc, name):
    """Members with tokens of their own for several steps.  A member whose rows are full gets NaN and disturbs nobody."""
    print(f"[case] forward_members {name}", flush=True)
    m = Model(*MODELS[name], layers=2, vocab=400, ctx=64, seed=7)
    exact = Exact(orc, name, 400, 7)
    rng = np.random.default_rng(2)
    prompt = [int(v) for v in rng.integers(0, 400, 9)]
    prompt_into(m, prompt)
    n, rows = 5, 4
    bufs, own = own_caches(m, n, rows)
    wsz = m.tree.members_workspace_bytes(n, rows)
    ws, x, lg = DeviceBuffer(wsz), DeviceBuffer(4 * n * m.hidden), DeviceBuffer(4 * n * m.vocab)
    prefix, lens = up(u32([len(prompt)]))[0], up(u32([0] * n))[0]
    for step in range(4):
        tokens = rng.integers(0, 400, n)
        length = [step + 1] * n
        if step == 3:
            length[4] = rows + 1
        lens.upload(u32(length))
        m.tree.forward_members(up(u32(tokens))[0], n, prefix, lens, own, rows, x, lg, ws, wsz)
        got = down(lg, np.float32, n * m.vocab).reshape(n, -1)
        for i in range(n):
            if length[i] > rows:
                assert np.isnan(got[i]).all()
                continue
            want = exact.logits(int(tokens[i]), member_rows(m, bufs, len(prompt), n, rows, i, step + 1))
            assert rel_l2(got[i], want) <= 1e-4, (step, i, rel_l2(got[i], want))


def test_step_without_logits(gpu):
    """The hidden states are the same, the logits not touched; a member with no token of its own stores nothing."""
    m = Model(*MODELS["q4_0"], layers=2, vocab=300, ctx=32, seed=4)
    prompt_into(m, [1, 2, 3])
    out = []
    for with_logits in (True, False):
        bufs, own = own_caches(m, 3, 4)
        wsz = m.tree.members_workspace_bytes(3, 4)
        x, lg, ws = DeviceBuffer(4 * 3 * m.hidden), DeviceBuffer(4 * 3 * m.vocab), DeviceBuffer(wsz)
        lg.fill(0xEE)
        m.tree.forward_members(up(u32([5, 6, 7]))[0], 3, up(u32([3]))[0], up(u32([1, 0, 1]))[0], own, 4, x, lg if with_logits else None, ws, wsz)
        out.append(down(x, np.float32, 3 * m.hidden).reshape(3, -1))
        assert with_logits or (down(lg, np.uint8, 4 * 3 * m.vocab) == 0xEE).all()
        rows = [down(b, np.uint16, 3 * 4 * m.kv * m.d).reshape(3, 4, -1) for b in bufs[0] + bufs[1]]
        assert all((r[1] == 0xFFFF).all() and (r[[0, 2], 1:] == 0xFFFF).all() and (r[[0, 2], 0] != 0xFFFF).all() for r in rows)
    assert np.array_equal(out[0][[0, 2]], out[1][[0, 2]])


def test_rules_of_the_model(gpu):
    """The model's own rotation given as rules is the default, bit for bit; others are not."""
    m = Model(*MODELS["q4_0"], layers=2, vocab=400, ctx=32, seed=8)
    prompt_into(m, [1, 2, 3])
    inv, out = up(ops.rope_inv_freq(10000.0, m.d))[0], []
    gamma = up(np.linspace(0.5, 1.5, m.d).astype(np.float32))[0]
    for rules in (None, ops.RopeRules(inv), ops.RopeRules(inv, interleaved=True), ops.RopeRules(inv, q_norm=gamma, k_norm=gamma)):
        _, own = own_caches(m, 2, 3)
        wsz = m.tree.members_workspace_bytes(2, 3)
        lg = DeviceBuffer(4 * 2 * m.vocab)
        m.tree.forward_members(up(u32([5, 6]))[0], 2, up(u32([3]))[0], up(u32([1, 1]))[0], own, 3, DeviceBuffer(4 * 2 * m.hidden), lg,
                               DeviceBuffer(wsz), wsz, rules)
        out.append(down(lg, np.float32, 2 * m.vocab))
    assert np.array_equal(out[0], out[1]) and np.isfinite(out[2]).all() and np.isfinite(out[3]).all()
    assert rel_l2(out[2], out[0]) > 1e-3 and rel_l2(out[3], out[0]) > 1e-3


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("ends", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_beam_search(gpu, orc, name, graph, ends):
    """A whole search on the device: every step's logits are the step's in 64 bits for each beam that is continued, every
    choice is the definition's for these logits, and beams that end stay as they are."""
    print(f"[case] beam search {name} graph {graph}", flush=True)
    vocab, b, steps, rows, end = 300, 4, 10, 12, 17
    m = Model(*MODELS[name], layers=2, vocab=vocab, ctx=64, seed=12)
    exact = Exact(orc, name, vocab, 12)
    prompt = [3, 7, 7, 250, 9]
    first = prompt_into(m, prompt)
    bufs, own = own_caches(m, b, rows)
    s = Stream() if graph else None
    mk = lambda a: up(a if a.dtype == np.float32 else u32(a))[0]
    scores0 = np.full((1, b), -np.inf, np.float32)
    scores0[0, 0] = 0
    scores, tokens, parents = mk(scores0), mk(np.full(b, vocab)), mk(np.zeros(b))
    counts, len_, history = mk(np.zeros(b)), mk(np.zeros(b)), mk(np.zeros((b, rows)))
    prefix = mk(np.array([len(prompt)]))
    rules = ops.BeamRules(b, 0, end, 0.7, last_tokens=tokens, counts=counts, counts_out=counts, history=history, history_stride=rows,
                          len=len_, len_out=len_)
    need = ops.beam_select_workspace_bytes(rules, 1, vocab)
    sws = DeviceBuffer(need)
    wsz = m.tree.members_workspace_bytes(b, rows)
    ws, x, lg = DeviceBuffer(wsz), DeviceBuffer(4 * b * m.hidden), DeviceBuffer(4 * b * vocab)
    states = ops.BeamStates(bufs[0] + bufs[1])
    bias = np.zeros(vocab, np.float32)
    bias[end] = first.max() - first[end] + 0.5 if ends else 3.0  # the first: the prompt's best next token is the end
    # the search begins with the prompt's logits in every row; only the first beam is there
    lg.upload(np.tile(first, (b, 1)))

    def choose(stream=None):
        ops.logits_process(bias_rules, lg, vocab, b, vocab, lg, vocab, None, stream=stream)
        ops.beam_select(rules, lg, vocab, 1, vocab, scores, scores, tokens, parents, sws, need, stream)

    def step(stream=None):
        m.tree.forward_members(tokens, b, prefix, len_, own, rows, x, lg, ws, wsz, stream=stream)
        choose(stream)
        ops.beam_reorder(states, 1, b, rows, m.kv * m.d * 2, parents, len_, 1, stream)

    bias_rules = ops.LogitsRules(bias_ids=mk(np.array([end])), bias=mk(bias[end:end + 1].copy()), n_bias=1)
    h = dict(scores=scores0, last=np.full((1, b), vocab), counts=np.zeros((1, b), int), paths=[[] for _ in range(b)])
    choose()
    g = None
    ended = 0
    for i in range(steps):
        if i:
            if graph and g is None:
                with Graph.capture(s) as g:
                    step(s)
            if graph:
                g.launch(s)
                s.synchronize()
            else:
                step()
        logits = down(lg, np.float32, b * vocab).reshape(1, b, vocab)
        want = _members.select_all(logits, h["scores"], b, h["last"], end, 0.7, h["counts"])
        got = down(scores, np.float32, b)
        assert np.array_equal(down(tokens, np.uint32, b), want[1][0]) and np.array_equal(down(parents, np.uint32, b), want[2][0]), i
        assert (np.abs(got - want[0][0]) <= np.abs(want[0][0]) * SCORE + 2.0 ** -22).all()
        assert np.array_equal(down(counts, np.uint32, b), want[3][0])
        for j, parent in enumerate(want[2][0].tolist()):  # beam j has its parent's rows by now
            if i and h["last"][0, parent] != end:
                seen = exact.logits(h["paths"][parent][-1], member_rows(m, bufs, len(prompt), b, rows, j, i)) + bias
                assert rel_l2(logits[0, parent], seen) <= 1e-4, (i, parent, rel_l2(logits[0, parent], seen))
        h["paths"] = [h["paths"][want[2][0, j]] + [int(want[1][0, j])] for j in range(b)]
        h["scores"], h["last"], h["counts"] = got[None], want[1], want[3]
        hist = down(history, np.uint32, b * rows).reshape(b, rows)
        assert all(list(hist[j, :i + 1]) == h["paths"][j] for j in range(b))
        ended = max(ended, int((want[1] == end).sum()))
    assert ended > 0 or not ends
    synchronize()


@pytest.mark.parametrize("heads, kv, d, inter, rot", [(8, 2, 64, True, 32), (16, 4, 128, False, 0)])
def test_operators_together(gpu, heads, kv, d, inter, rot):
    """Searches for two prompts without a model: norms and partial rotation, shared attention, a choice from the output and
    the rows reordered, against the same in 64 bits on the rows that the device stored."""
    print(f"[case] together {heads} {kv} {d}", flush=True)
    r = np.random.default_rng(21)
    groups, b, rows, vocab = 2, 3, 9, heads * d
    n, rot_dim = groups * b, rot or d
    prefix = [140, 37]
    kp, vp = (r.standard_normal((groups, 150, kv, d)).astype(np.float16) for _ in range(2))
    inv, mag = ops.rope_scaled_inv_freq(ops.ROPE_BY_INDEX, 10000.0, rot_dim, 4.0, 64, 1.0, 16.0)
    qw, kw = (1 + 0.2 * r.standard_normal((2, d))).astype(np.float32)
    dev = lambda a: up(a if a.dtype in (np.float32, np.float16) else u32(a))[0]
    rules = ops.RopeRules(dev(inv), rot, inter, mag, dev(qw), dev(kw), 1e-6)
    kpb, vpb, plen, own_len = dev(kp), dev(vp), dev(np.array(prefix)), dev(np.zeros(n))
    kob, vob = (DeviceBuffer(n * rows * kv * d * 2) for _ in range(2))
    kob.fill(0xFF), vob.fill(0xFF)
    q, out = DeviceBuffer(4 * n * heads * d), DeviceBuffer(4 * n * vocab)
    need = ops.attention_shared_workspace_bytes(groups, b, heads, kv, d, 150, rows)
    ws = DeviceBuffer(need)
    scores, tokens, parents = dev(np.zeros((groups, b), np.float32)), dev(np.zeros(n)), dev(np.zeros(n))
    sel = ops.BeamRules(b, len=own_len, len_out=own_len)
    sneed = ops.beam_select_workspace_bytes(sel, groups, vocab)
    sws, states = DeviceBuffer(sneed), ops.BeamStates([kob, vob])
    own_len.upload(u32(np.ones(n)))
    k64, v64 = np.zeros((groups, b, rows, kv, d), np.float16), np.zeros((groups, b, rows, kv, d), np.float16)
    last = np.zeros((groups, b), np.float32)
    for step in range(rows):
        qkv = (r.standard_normal((n, (heads + 2 * kv) * d)) * 1.2).astype(np.float32)
        x = dev(qkv)
        width = qkv.shape[1]
        ops.qk_norm_rope(rules, x, x.ptr + 4 * heads * d, x.ptr + 4 * (heads + kv) * d, width, width, plen, own_len, groups, b, 1, heads,
                         kv, d, q, heads * d, None, 0, kob, vob, rows)
        ops.attention_shared(q, heads * d, plen, own_len, groups, b, kpb, vpb, 150, kob, vob, rows, heads, kv, d, out, ws, need)
        ops.beam_select(sel, out, vocab, groups, vocab, scores, scores, tokens, parents, sws, sneed)
        ops.beam_reorder(states, groups, b, rows, kv * d * 2, parents, own_len, 1)
        pos = np.repeat(prefix, b) + step
        turned, bound_q = _members.rope(qkv[:, :heads * d].reshape(n, heads, d), pos, inv, rot_dim, inter, mag, qw, 1e-6)
        keys, _ = _members.rope(qkv[:, heads * d:(heads + kv) * d].reshape(n, kv, d), pos, inv, rot_dim, inter, mag, kw, 1e-6)
        k64[:, :, step] = _members.stored(keys).reshape(groups, b, kv, d)
        v64[:, :, step] = qkv[:, (heads + kv) * d:].astype(np.float16).reshape(groups, b, kv, d)
        got = down(out, np.float32, n * vocab).reshape(n, heads, d)
        for m in range(n):
            g, i = m // b, m % b
            kk = np.concatenate([kp[g, :prefix[g]], k64[g, i, :step + 1]])
            vv = np.concatenate([vp[g, :prefix[g]], v64[g, i, :step + 1]])
            want, bound = _members.attention(turned[m], kk, vv)
            # q's own error moves a score by its bound times |k|; a stored k may be one f16 step off where the norm's rounding
            # crosses a border: 2^-10 of the step's row, seen by its own weight alone
            dq = (bound_q[m].max(-1) * np.abs(kk.astype(np.float64)).sum(-1).max() / np.sqrt(d))[:, None]
            dk = np.abs(turned[m]).sum(-1)[:, None] * np.abs(k64[g, i, :step + 1].astype(np.float64)).max() * 2.0 ** -10 / np.sqrt(d)
            slack = 2 * (dq + dk) * np.abs(vv.astype(np.float64)).max()
            assert (np.abs(got[m] - want) <= bound + slack).all(), (step, m, np.abs(got[m] - want).max())
        choice = _members.select_all(got.reshape(groups, b, vocab), last, b)
        assert np.array_equal(down(tokens, np.uint32, n).reshape(groups, b), choice[1])
        assert np.array_equal(down(parents, np.uint32, n).reshape(groups, b), choice[2])
        last = down(scores, np.float32, n).reshape(groups, b)
        length = np.full((groups, b), step + 2)
        assert np.array_equal(down(own_len, np.uint32, n), length.ravel())
        k64, v64 = (_members.reorder(a, choice[2], length, 1) for a in (k64, v64))
        stored = down(vob, np.float16, n * rows * kv * d).reshape(v64.shape)
        assert np.array_equal(stored[:, :, :step + 1], v64[:, :, :step + 1])
        k64[:, :, :step + 1] = down(kob, np.float16, n * rows * kv * d).reshape(k64.shape)[:, :, :step + 1]
