"""wh_llama_forward_tree at every number of nodes at which its products change kernels, in the workspace that it asks for,
against a step in 64 bits."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, up
from tests._oracle import Oracle, rel_l2
from tests.test_gpu_tree_step import F16, MODELS, Q4_K, Q8_0, Model
from woolly_amd import ops, synth
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu


class Exact:
    """The model's step in 64 bits for all nodes of a tree at once, over the cache rows that the device stored: a k or v that
    lies between two f16 numbers rounds to either, and what its neighbour moves is no error of the step."""

    def __init__(self, m, name, seed):
        orc = Oracle()
        _, hidden, heads, kv, d, n_ff = MODELS[name]
        self.hidden, self.h, self.kv, self.d = hidden, heads, kv, d
        shapes = dict(wq=(heads * d, hidden), wk=(kv * d, hidden), wv=(kv * d, hidden), wo=(hidden, heads * d),
                      w_gate=(n_ff, hidden), w_up=(n_ff, hidden), w_down=(hidden, n_ff))
        base = Q4_K if name == "mixed" else MODELS[name][0]

        def matrix(t, data, rows, k):
            st, w = orc.dequantize(t, data, rows * k)
            assert st == 0
            return w.reshape(rows, k).astype(np.float64)

        self.layers = []
        for dev in m.keep:
            L = {n: matrix(dev.get(n + "_type") or base, down(dev[n], np.uint8, dev[n].nbytes), *s) for n, s in shapes.items()}
            L.update({n: down(dev[n], np.float32, hidden).astype(np.float64) for n in ("attn_norm", "ffn_norm")})
            self.layers.append(L)
        rng = np.random.default_rng(seed)  # as Model draws them
        self.norm = (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32).astype(np.float64)
        self.embd = rng.standard_normal((m.vocab, hidden)).astype(np.float16).astype(np.float64)
        self.head = matrix(Q8_0, synth.quantized_weight(Q8_0, m.vocab, hidden, seed=seed + 99), m.vocab, hidden)
        self.inv = ops.rope_inv_freq(10000.0, d)

    def step(self, tokens, paths, ctx, rows):
        """rows: k and v of each layer as stored, [ctx + nodes][kv][d].  Returns the logits of the nodes in `paths` that are
        there and the k and v that each layer should have stored."""
        nodes = [t for t, p in enumerate(paths) if p is not None]
        norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w
        x, made = self.embd[[int(tokens[t]) for t in nodes]], []
        for i, L in enumerate(self.layers):
            xh = norm(x, L["attn_norm"])
            q, k, v = (xh @ L[n].T for n in ("wq", "wk", "wv"))
            kc, vc = rows[2 * i], rows[2 * i + 1]
            out, ks = np.zeros_like(q), []
            for j, t in enumerate(nodes):
                pos = ctx + len(paths[t]) - 1
                see = np.concatenate([np.arange(ctx), ctx + np.array(paths[t])]).astype(int)
                qr = _tree.rotate(q[j].reshape(self.h, self.d), pos, self.inv)
                ks.append(_tree.rotate(k[j].reshape(self.kv, self.d), pos, self.inv))
                for h in range(self.h):
                    g = h // (self.h // self.kv)
                    s = kc[see, g] @ qr[h] / np.sqrt(self.d)
                    w = np.exp(s - s.max())
                    out[j, h * self.d:(h + 1) * self.d] = w @ vc[see, g] / w.sum()
            made += [np.stack(ks), v.reshape(len(nodes), self.kv, self.d)]
            x = x + out @ L["wo"].T
            xh = norm(x, L["ffn_norm"])
            gate = xh @ L["w_gate"].T
            x = x + (gate / (1 + np.exp(-gate)) * (xh @ L["w_up"].T)) @ L["w_down"].T
        return nodes, norm(x, self.norm) @ self.head.T, made


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("n", [1, 2, 8, 9, 16, 17, 26, 33, 64, 65, 100, 128])
def test_logits_of_every_node(gpu, name, n):
    """The decode step's own bar, rel-L2 1e-4, with absent nodes of ids beyond the vocabulary (NaN rows) among the others;
    the workspace of exactly n nodes, x and logits end where they should; k and v are stored within one step of f16."""
    print(f"[case] forward_tree {name} {n} nodes", flush=True)
    vocab, prompt = 401, [5, 17, 256, 3]
    ctx = len(prompt)
    m = Model(*MODELS[name], layers=2, vocab=vocab, ctx=160, seed=n)
    rng = np.random.default_rng(n)
    parents = _tree.make_parents(rng, n, "tree")
    tokens = rng.integers(0, vocab, n)
    if n > 4:
        parents[n // 3] = -2
        tokens[n // 3] = 10 ** 6
        parents[n - 2] = n + 7
        tokens[n - 2] = 0xFFFFFFFF
    for i, tok in enumerate(prompt):
        m.step(tok, i)
    for a, b in zip(m.sets[0], m.sets[1]):  # the prompt's rows
        for k in ("k_cache", "v_cache"):
            b[k].upload(down(a[k], np.uint16, m.ctx * m.kv * m.d))
    wsz = m.tree.tree_workspace_bytes(n)
    ws, x, lg = DeviceBuffer(wsz + 256), DeviceBuffer(4 * n * m.hidden + 256), DeviceBuffer(4 * n * vocab + 256)
    for b in (ws, x, lg):
        b.fill(0xEE)
    ctxb = up(np.array([ctx], np.uint32))[0]
    m.tree.forward_tree(up(tokens.astype(np.uint32))[0], up(parents)[0], n, ctxb, x, lg, ws, wsz)
    got = down(lg, np.float32, n * vocab).reshape(n, -1)
    for b, size in ((ws, wsz), (x, 4 * n * m.hidden), (lg, 4 * n * vocab)):
        assert (down(b, np.uint8, 256, offset=size) == 0xEE).all(), "behind a buffer"
    rows = m.rows(1, ctx + n)
    nodes, want, made = Exact(m, name, n).step(tokens, _tree.paths(parents), ctx, rows)
    worst = max(rel_l2(got[t], w) for t, w in zip(nodes, want))
    print(f"[result] {name} {n} nodes: rel-L2 {worst:.2e}", flush=True)
    assert worst <= 1e-4
    for stored, exact in zip(rows, made):
        stored = stored[[ctx + t for t in nodes]]
        step = np.spacing(np.abs(exact).astype(np.float16)).astype(np.float64)
        assert (np.abs(stored - exact) <= step + 1e-4 * np.abs(exact).max()).all()
