"""The operators of a drafted tree together, as a program uses them: forward_tree, logits_process, tree_accept and
kv_cache_compact against the decode step, one token at a time."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, up
from tests._oracle import max_abs, rel_l2
from tests.test_oracle_decode import PROJ, mixed_layer, small_layer
from woolly_amd import ops, synth
from woolly_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
F16, Q4_0, Q8_0, Q4_K, Q6_K = 1, 2, 8, 12, 14
NO = _tree.NO_TOKEN
REP, FREQ, PRES = 1.25, 0.1, 0.2


class Model:
    """A random model with two identical sets of caches: one for the decode step, one for the tree."""

    def __init__(self, t, hidden, heads, kv, d, n_ff, layers, vocab, ctx, seed):
        rng = np.random.default_rng(seed)
        self.vocab, self.hidden, self.ctx, self.kv, self.d, self.layers = vocab, hidden, ctx, kv, d, layers
        dims = dict(hidden=hidden, n_heads=heads, n_kv_heads=kv, head_dim=d, n_ff=n_ff, max_ctx=ctx, vocab=vocab, eps=1e-5)
        sets = [[], []]
        self.keep = []
        for i in range(layers):
            if t == "mixed":
                types = {p: Q6_K if p in ("wv", "w_down") else Q4_K for p in PROJ}
                L = mixed_layer(types, hidden, heads, kv, d, n_ff, seed=seed + i)
            else:
                L, types = small_layer(t, hidden, heads, kv, d, n_ff, seed=seed + i), {}
            dev = {k: up(v)[0] for k, v in L.items()}
            dev.update({k + "_type": v for k, v in types.items()})
            self.keep.append(dev)
            for s in sets:
                c = dict(dev)
                for name in ("k_cache", "v_cache"):
                    c[name] = DeviceBuffer(ctx * kv * d * 2)
                    c[name].fill(0)
                s.append(c)
        inv = up(ops.rope_inv_freq(10000.0, d))[0]
        head = up(synth.quantized_weight(Q8_0, vocab, hidden, seed=seed + 99))[0]
        norm = up((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32))[0]
        embd = up(rng.standard_normal((vocab, hidden)).astype(np.float16).view(np.uint16))[0]
        base = Q4_K if t == "mixed" else t
        self.one, self.tree = (ops.LlamaModel(base, dims, s, inv, norm, head, Q8_0, embd, F16) for s in sets)
        self.sets = sets
        self.wsz = self.one.workspace_bytes()
        self.ws = DeviceBuffer(self.wsz)

    def step(self, token, pos):
        """The decode step's logits of `token` at `pos`."""
        tb, x, lg = up(np.array([token], np.uint32))[0], DeviceBuffer(4 * self.hidden), DeviceBuffer(4 * self.vocab)
        self.one.forward_token(tb, pos, x, lg, self.ws, self.wsz)
        return down(lg, np.float32, self.vocab)

    def rows(self, which, n):
        return [down(L[k], np.float16, n * self.kv * self.d).reshape(n, self.kv, self.d).astype(np.float64)
                for L in self.sets[which] for k in ("k_cache", "v_cache")]


def choose(logits, history, vocab):
    counts = np.bincount(np.array(history, int), minlength=vocab)
    l, token = _tree.logits(logits, vocab, np.float32(REP), np.float32(FREQ), np.float32(PRES), counts, {}, None, np.float32)
    top = np.sort(l)[-2:]
    return token, float(top[1] - top[0])


MODELS = {"q4_0": (Q4_0, 256, 4, 2, 64, 512), "q4_0_d128": (Q4_0, 512, 4, 1, 128, 768), "mixed": ("mixed", 512, 8, 2, 64, 768)}


@pytest.mark.parametrize("name", list(MODELS))
def test_tree_logits_are_the_paths_logits(gpu, name):
    """Every node's logits are those of decoding its path token by token; absent nodes with ids beyond the vocabulary
    (NaN rows) disturb nothing.  The decode step's own bars: rel-L2 1e-4."""
    print(f"[case] forward_tree {name}", flush=True)
    m = Model(*MODELS[name], layers=2, vocab=400, ctx=64, seed=5)
    rng = np.random.default_rng(1)
    prompt = [int(v) for v in rng.integers(0, 400, 7)]
    ctxb = up(np.array([0], np.uint32))[0]
    t = len(prompt)
    # the prompt as a chain fills the tree's caches
    wsz = m.tree.tree_workspace_bytes(20)
    ws, x = DeviceBuffer(wsz), DeviceBuffer(4 * 20 * m.hidden)
    lg = DeviceBuffer(4 * 20 * m.vocab)
    m.tree.forward_tree(up(np.array(prompt, np.uint32))[0], up(np.arange(-1, t - 1, dtype=np.int32))[0], t, ctxb, x, lg, ws, wsz)
    got = down(lg, np.float32, t * m.vocab).reshape(t, -1)
    for i, tok in enumerate(prompt):
        want = m.step(tok, i)
        assert rel_l2(got[i], want) <= 1e-4, (i, rel_l2(got[i], want))
    # the decode step goes on from rows that a tree step stored
    x1, lg1 = DeviceBuffer(4 * m.hidden), DeviceBuffer(4 * m.vocab)
    m.tree.forward_token(up(np.array([33], np.uint32))[0], t, x1, lg1, m.ws, m.wsz)
    assert rel_l2(down(lg1, np.float32, m.vocab), m.step(33, t)) <= 1e-4
    parents = np.array([-1, 0, 0, 1, 1, 2, 3, 3, -2, 8, 6, 5], np.int32)
    n = len(parents)
    tokens = rng.integers(0, 400, n)
    tokens[[8, 9]] = 10 ** 6
    ctxb.upload(np.array([t], np.uint32))
    m.tree.forward_tree(up(tokens.astype(np.uint32))[0], up(parents)[0], n, ctxb, x, lg, ws, wsz)
    got = down(lg, np.float32, n * m.vocab).reshape(n, -1)
    for node, path in enumerate(_tree.paths(parents)):
        if path is None:
            continue
        for i, a in enumerate(path):  # rows behind the prompt are written anew for each path
            want = m.step(int(tokens[a]), t + i)
        assert rel_l2(got[node], want) <= 1e-4, (node, rel_l2(got[node], want), max_abs(got[node], want))


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("graph", [False, True])
def test_speculative_run_is_the_greedy_run(gpu, name, graph):
    """40 tokens by verified trees, with repetition, frequency and presence penalties and everything on the device between
    the drafts: the tokens, the history and the cache rows are those of decoding one token at a time."""
    print(f"[case] speculative run {name} graph {graph}", flush=True)
    vocab, want_len, nt = 300, 40, 11
    m = Model(*MODELS[name], layers=2, vocab=vocab, ctx=128, seed=11)
    prompt = [3, 7, 7, 250, 9]
    # one token at a time: the greedy run with penalties, its margins
    said, logits = [], None
    for tok in prompt:
        logits = m.step(tok, len(said))
        said.append(tok)
    greedy, margins = [], []
    for _ in range(want_len):
        tok, margin = choose(logits, said, vocab)
        greedy.append(tok)
        margins.append(margin)
        logits = m.step(tok, len(said))
        said.append(tok)
    assert min(margins) > 1e-3, "choices too close to compare two ways of summing"
    total = len(prompt) + want_len

    stream = Stream()
    wsz = m.tree.tree_workspace_bytes(nt)
    tok_b, par_b, ctx_b = DeviceBuffer(4 * nt), DeviceBuffer(4 * nt), up(np.array([0], np.uint32))[0]
    x, lg, ws = DeviceBuffer(4 * nt * m.hidden), DeviceBuffer(4 * nt * vocab), DeviceBuffer(wsz)
    picked, path, count, nxt = DeviceBuffer(4 * nt), DeviceBuffer(4 * nt), DeviceBuffer(4), DeviceBuffer(4)
    hist = DeviceBuffer(4 * 256)
    hist.fill(0xFF)
    rules = ops.LogitsRules(rows_per_seq=nt, repetition_penalty=REP, frequency_penalty=FREQ, presence_penalty=PRES,
                            history=hist, history_stride=256, history_len=ctx_b, tree_tokens=tok_b, tree_parents=par_b)
    lws = ops.logits_process_workspace_bytes(rules, nt, vocab)
    lwb = DeviceBuffer(lws)
    caches = m.tree.kv_caches()

    def verify():
        m.tree.forward_tree(tok_b, par_b, nt, ctx_b, x, lg, ws, wsz, stream)
        ops.logits_process(rules, lg, vocab, nt, vocab, None, 0, picked, lwb, lws, stream)
        ops.tree_accept(tok_b, par_b, picked, 1, nt, path, count, nxt, ctx_b, ctx_b, hist, 256, stream)
        ops.kv_cache_compact(caches, 1, m.ctx, m.kv, m.d, path, nt, count, ctx_b, stream)

    synchronize()
    replay = None
    if graph:
        with Graph.capture(stream) as replay:
            verify()

    def draft(tokens, parents):
        pad = nt - len(tokens)
        tok_b.upload(np.array(list(tokens) + [0] * pad, np.uint32))
        par_b.upload(np.array(list(parents) + [-2] * pad, np.int32))
        if graph:
            replay.launch(stream)
        else:
            verify()
        stream.synchronize()
        return int(down(count, np.uint32, 1)[0]), int(down(nxt, np.uint32, 1)[0])

    # the prompt's tokens are given, not chosen: one at a time
    pending = None
    for tok in prompt:
        n, pending = draft([tok], [-1])
        assert n == 1
    rng = np.random.default_rng(2)
    out, accepted = [], []
    while len(out) < want_len:
        at = len(out)
        assert pending == greedy[at], at
        # node 0 is the pending token; the greedy run's next tokens, some of them wrong, among siblings that are
        tokens, parents, node = [pending], [-1], 0
        for i in range(1, 4):
            right = greedy[at + i] if at + i < want_len else 0
            for token in rng.permutation([right, (right + 1) % vocab, (right + 5) % vocab]):
                tokens.append(int(token) if rng.random() > 0.15 else int((token + 9) % vocab))
                parents.append(node)
            hit = [j for j in range(len(tokens) - 3, len(tokens)) if tokens[j] == right]
            node = hit[0] if hit else len(tokens) - 1
        n, nxt_tok = draft(tokens, parents)
        assert 1 <= n <= 4
        out += greedy[at:at + n]
        accepted.append(n)
        length = int(down(ctx_b, np.uint32, 1)[0])
        assert length == len(prompt) + at + n
        h = down(hist, np.uint32, 256)
        assert list(h[:length]) == (prompt + greedy + [nxt_tok] * 4)[:length], "history"
        pending = nxt_tok
    assert max(accepted) > 1, "no draft was ever accepted"
    n = min(total, int(down(ctx_b, np.uint32, 1)[0]))
    for a, b in zip(m.rows(0, n), m.rows(1, n)):
        # rows made of activations that differ in their last bits: an f16 step, and what lower layers carry on
        step = np.spacing(np.abs(a).astype(np.float16)).astype(np.float64)
        assert (np.abs(a - b) <= 2 * step + 1e-3 * np.abs(a).max()).all()
    if replay:
        replay.destroy()
    stream.destroy()
