"""wh_llama_forward_members at every number of members at which its products change kernels, and under rules of rotation other
than the model's over a prompt made by the same rules, against a step in 64 bits."""
import numpy as np
import pytest

from tests import _members
from tests._gpu import down, up
from tests._oracle import rel_l2
from tests.test_gpu_tree_step import MODELS, Model
from tests.test_gpu_tree_step_sizes import Exact
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu
u32 = lambda a: np.asarray(a).astype(np.uint32)


class MembersExact(Exact):
    """The step in 64 bits for tokens that each see rows of their own, over the rows that the device stored."""

    def members(self, tokens, pos, see, rope=None, moved=None):
        """pos: the tokens' positions; see(layer, i): the rows of k and v that token i sees, [n][kv][d], its own the last.
        rope(x [n][heads][d], pos, key): as the rules have it (None: the model's).  moved: a generator of signs, by which
        every score is moved by an f32 form's error.  Logits, and the k and v rows of each layer."""
        rope = rope or (lambda x, pos, key: _members.rope(x, pos, self.inv, self.d, False)[0])
        norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w
        n, g = len(tokens), self.h // self.kv
        x, made = self.embd[np.asarray(tokens, int)], []
        for layer, L in enumerate(self.layers):
            xh = norm(x, L["attn_norm"])
            q, k, v = ((xh @ L[name].T).reshape(n, -1, self.d) for name in ("wq", "wk", "wv"))
            q, k = rope(q, pos, False), rope(k, pos, True)
            out = np.zeros((n, self.h, self.d))
            for i in range(n):
                kc, vc = (a.astype(np.float64) for a in see(layer, i))
                for h in range(self.h):
                    s = kc[:, h // g] @ q[i, h] / np.sqrt(self.d)
                    if moved:
                        s += moved.choice([-1, 1], len(s)) * (np.abs(kc[:, h // g]) @ np.abs(q[i, h]) / np.sqrt(self.d)) * 2.0 ** -21
                    w = np.exp(s - s.max())
                    out[i, h] = w @ vc[:, h // g] / w.sum()
            made.append((k, v))
            x = x + out.reshape(n, -1) @ L["wo"].T
            xh = norm(x, L["ffn_norm"])
            gate = xh @ L["w_gate"].T
            x = x + (gate / (1 + np.exp(-gate)) * (xh @ L["w_up"].T)) @ L["w_down"].T
        return norm(x, self.norm) @ self.head.T, made


    def bars(self, want, *args):
        """Of the members' rel-L2: the decode step's 1e-4, and what an f32 form of the scores can make of them.

        A score is a sum of products whose magnitudes add up to S.  In f32 its additions are off by 2^-24 of the sum so far,
        4 * 2^-24 S in all for the d / 8 of them, the queries by 2^-23 to 2^-22 and the exponent's argument by 2^-23 of
        |s| <= S: 2^-21 S.  Members of these tests have scores of some thousands (a random K-quant model's own key), for which
        that is 1e-3 of a weight; the same step by numpy in f32 is off by 3e-4.  So the step in 64 bits is made four times
        more with every score moved by 2^-21 S, the signs at random."""
        worst = np.zeros(len(want))
        for seed in range(4):
            other, _ = self.members(*args, moved=np.random.default_rng(seed))
            worst = np.maximum(worst, [rel_l2(a, b) for a, b in zip(other, want)])
        return 1e-4 + 2 * worst


def one_step_off(stored, exact):
    step = np.spacing(np.abs(exact).astype(np.float16)).astype(np.float64)
    assert (np.abs(stored.astype(np.float64) - exact) <= step + 1e-4 * np.abs(exact).max()).all()


def own_caches(m, members, rows, rng=None):
    """Caches of the members' own rows: random where rng is given, else NaN."""
    bufs = []
    for _ in range(2 * m.layers):
        b = DeviceBuffer(members * rows * m.kv * m.d * 2)
        if rng is None:
            b.fill(0xFF)
        else:
            b.upload(rng.standard_normal((members, rows, m.kv, m.d)).astype(np.float16).view(np.uint16))
        bufs.append(b)
    return bufs, ops.KvCaches(bufs[0::2], bufs[1::2])


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("n, prefix, rows", [(1, 9, 4), (2, 1500, 30), (8, 0, 200), (9, 1, 3), (16, 700, 1), (17, 1600, 140), (26, 130, 20),
                                             (33, 64, 9), (64, 333, 40), (65, 1600, 5), (100, 20, 70), (128, 900, 12)])
def test_logits_of_every_member(gpu, name, n, prefix, rows):
    """Members with any number of tokens of their own, none among them and too many, in exactly the workspace that the call
    asks for; k and v are stored within one step of f16, other rows stay."""
    print(f"[case] forward_members {name} {n} members at {prefix}", flush=True)
    vocab, ctx = 401, 1600
    m = Model(*MODELS[name], layers=2, vocab=vocab, ctx=ctx, seed=n)
    rng = np.random.default_rng(n)
    for L in m.sets[1]:
        for k in ("k_cache", "v_cache"):
            L[k].upload(rng.standard_normal((ctx, m.kv, m.d)).astype(np.float16).view(np.uint16))
    bufs, own = own_caches(m, n, rows, rng)
    before = [down(b, np.uint16, n * rows * m.kv * m.d).reshape(n, rows, m.kv, m.d) for b in bufs]
    lens = rng.integers(1, rows + 1, n)
    lens[0] = rows
    if n > 8:
        lens[3], lens[5], lens[n - 1] = 0, rows + 1, 1
    tokens = rng.integers(0, vocab, n)
    wsz = m.tree.members_workspace_bytes(n, rows)
    ws, x, lg = DeviceBuffer(wsz + 256), DeviceBuffer(4 * n * m.hidden + 256), DeviceBuffer(4 * n * vocab + 256)
    for b in (ws, x, lg):
        b.fill(0xEE)
    m.tree.forward_members(up(u32(tokens))[0], n, up(u32([prefix]))[0], up(u32(lens))[0], own, rows, x, lg, ws, wsz)
    got = down(lg, np.float32, n * vocab).reshape(n, -1)
    for b, size in ((ws, wsz), (x, 4 * n * m.hidden), (lg, 4 * n * vocab)):
        assert (down(b, np.uint8, 256, offset=size) == 0xEE).all(), "behind a buffer"
    there = [i for i in range(n) if 1 <= lens[i] <= rows]
    assert np.isnan(got[lens > rows]).all()
    shared = [a.astype(np.float16) for a in m.rows(1, ctx)]
    after = [down(b, np.float16, n * rows * m.kv * m.d).reshape(n, rows, m.kv, m.d) for b in bufs]

    def see(layer, j):
        i = there[j]
        return [np.concatenate([shared[2 * layer + w][:prefix], after[2 * layer + w][i, :lens[i]]]) for w in (0, 1)]

    exact, args = MembersExact(m, name, n), (tokens[there], prefix + lens[there] - 1, see)
    want, made = exact.members(*args)
    errors, bars = np.array([rel_l2(got[i], w) for i, w in zip(there, want)]), exact.bars(want, *args)
    print(f"[result] {name} {n} members at {prefix}: rel-L2 {errors.max():.2e}, bars {bars.min():.2e} to {bars.max():.2e}", flush=True)
    assert (errors <= bars).all(), (errors / bars).max()
    for layer in range(m.layers):
        for w in (0, 1):
            a, b = before[2 * layer + w], after[2 * layer + w]
            one_step_off(np.stack([b[i, lens[i] - 1] for i in there]), made[layer][w])
            for i in there:
                a[i, lens[i] - 1] = b[i, lens[i] - 1].view(np.uint16)
            assert np.array_equal(a, b.view(np.uint16)), "rows that no token has"


def prompt_by_operators(m, name, prompt, rules, first=0):
    """The rows first .. of the prompt's in the tree's caches, by the framework's operators under `rules`, layer by layer:
    norms and rotation, then an attention that turns nothing more (inverse frequencies of 0)."""
    t, hidden, heads, kv, d, n_ff = MODELS[name]
    n, qd, kvd = len(prompt), heads * d, kv * d
    zero, parents = up(np.zeros(d // 2, np.float32))[0], up(np.arange(-1, n - 1, dtype=np.int32))[0]
    ctx = up(u32([first]))[0]
    rng = np.random.default_rng(m.seed)
    rng.standard_normal(hidden)
    x = rng.standard_normal((m.vocab, hidden)).astype(np.float16)[prompt].astype(np.float32)  # as Model draws them

    def matmul(w, rows, k, inp):
        out, need = DeviceBuffer(4 * n * rows), ops.matmul_workspace_bytes(t, rows, k, n)
        ops.quantized_matmul(t, w, w.nbytes, rows, k, inp, n, out, DeviceBuffer(max(need, 1)), need)
        return out

    for L in m.sets[1]:
        xb, xn = up(x)[0], DeviceBuffer(4 * n * hidden)
        ops.rms_norm(xb, L["attn_norm"], 1e-5, n, hidden, xn)
        q, k, v = (matmul(L[w], rows, hidden, xn) for w, rows in (("wq", qd), ("wk", kvd), ("wv", kvd)))
        ops.qk_norm_rope(rules, q, k, v, qd, kvd, ctx, None, 1, 1, n, heads, kv, d, q, qd, k, kvd, None, None, 0)
        out, need = DeviceBuffer(4 * n * qd), ops.attention_tree_workspace_bytes(1, n, heads, kv, d, m.ctx)
        ops.attention_tree(q, k, v, qd, kvd, parents, ctx, 1, n, L["k_cache"], L["v_cache"], m.ctx, heads, kv, d, zero, out,
                           DeviceBuffer(need), need)
        x = x + down(matmul(L["wo"], hidden, qd, out), np.float32, n * hidden).reshape(n, -1)
        need = ops.ffn_workspace_bytes(hidden, n_ff, n)
        y = DeviceBuffer(4 * n * hidden)
        ops.ffn_swiglu(t, L["w_gate"], L["w_up"], L["w_down"], hidden, n_ff, L["ffn_norm"], 1e-5, up(x)[0], n, y, DeviceBuffer(need), need)
        x = x + down(y, np.float32, n * hidden).reshape(n, -1)


RULES = [dict(kind=ops.ROPE_BY_INDEX, rot=0, inter=False, norms=True), dict(kind=ops.ROPE_BY_TURNS, rot=32, inter=True, norms=False),
         dict(kind=ops.ROPE_LINEAR, rot=48, inter=False, norms=True)]


@pytest.mark.parametrize("name", ["q4_0", "q4_0_d128"])
@pytest.mark.parametrize("how", RULES)
def test_rules_over_a_prompt_of_the_same_rules(gpu, name, how):
    """Norms of queries and keys, scaled frequencies, part of a head in either pairing and a magnitude: the prompt's rows,
    three steps' logits and the rows that they store are those of these rules in 64 bits."""
    print(f"[case] forward_members {name} rules {how}", flush=True)
    seed, n, rows = 31, 5, 4
    m = Model(*MODELS[name], layers=2, vocab=400, ctx=96, seed=seed)
    m.seed = seed
    rng = np.random.default_rng(4)
    rot = how["rot"] or m.d
    inv, magnitude = ops.rope_scaled_inv_freq(how["kind"], 10000.0, rot, 4.0, 64, 1.0, 16.0)
    magnitude *= 1.1
    qw, kw = (1 + 0.2 * rng.standard_normal((2, m.d))).astype(np.float32) if how["norms"] else (None, None)
    dev = lambda a: None if a is None else up(a)[0]
    rules = ops.RopeRules(dev(inv), how["rot"], how["inter"], magnitude, dev(qw), dev(kw), 1e-6)
    rope = lambda x, pos, key: _members.rope(x, pos, inv, rot, how["inter"], magnitude, kw if key else qw, 1e-6)[0]
    exact = MembersExact(m, name, seed)
    prompt = [int(v) for v in rng.integers(0, 400, 37)]
    prompt_by_operators(m, name, prompt[:20], rules)
    prompt_by_operators(m, name, prompt[20:], rules, 20)
    shared = [a.astype(np.float16) for a in m.rows(1, len(prompt))]
    _, made = exact.members(prompt, np.arange(len(prompt)), lambda layer, i: [shared[2 * layer + w][:i + 1] for w in (0, 1)], rope)
    for layer in range(m.layers):
        for w in (0, 1):
            one_step_off(shared[2 * layer + w], made[layer][w])
    bufs, own = own_caches(m, n, rows)
    wsz = m.tree.members_workspace_bytes(n, rows)
    ws, x, lg = DeviceBuffer(wsz), DeviceBuffer(4 * n * m.hidden), DeviceBuffer(4 * n * m.vocab)
    prefix, lens = up(u32([len(prompt)]))[0], DeviceBuffer(4 * n)
    for step in range(3):
        tokens = rng.integers(0, 400, n)
        lens.upload(u32([step + 1] * n))
        m.tree.forward_members(up(u32(tokens))[0], n, prefix, lens, own, rows, x, lg, ws, wsz, rules)
        got = down(lg, np.float32, n * m.vocab).reshape(n, -1)
        mine = [down(b, np.float16, n * rows * m.kv * m.d).reshape(n, rows, m.kv, m.d) for b in bufs]
        see = lambda layer, i: [np.concatenate([shared[2 * layer + w], mine[2 * layer + w][i, :step + 1]]) for w in (0, 1)]
        want, made = exact.members(tokens, np.full(n, len(prompt) + step), see, rope)
        for i in range(n):
            assert rel_l2(got[i], want[i]) <= 1e-4, (step, i, rel_l2(got[i], want[i]))
        for layer in range(m.layers):
            for w in (0, 1):
                one_step_off(mine[2 * layer + w][:, step], made[layer][w])
