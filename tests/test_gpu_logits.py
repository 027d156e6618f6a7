"""wh_logits_process against its formula: bit for bit in f32, and in 64 bits within three roundings."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, up
from woolly_amd import _lib, ops
from woolly_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
NO = _tree.NO_TOKEN


class Case:
    def __init__(self, n_seqs, tree, vocab, hist=0, n_bias=0, mask=False, rep=1.3, freq=0.25, pres=0.5, ld=0, ldo=0, seed=0,
                 shape="padded", history_len=True, bias_per_seq=False):
        r = self.rng = np.random.default_rng(seed)
        self.n, self.t, self.v = n_seqs, tree, vocab
        self.per = max(1, tree)
        self.rows = n_seqs * self.per
        self.ld, self.ldo = ld or vocab, ldo or vocab
        self.x = (r.standard_normal((self.rows, self.ld)) * 4).astype(np.float32)
        self.pen = tuple(np.float32(p) for p in (rep, freq, pres))
        # few tokens often, ids beyond the vocabulary now and then
        self.hist = np.minimum((vocab * r.random((n_seqs, max(1, hist))) ** 5).astype(np.int64), vocab - 1)
        self.hist[r.random(self.hist.shape) < 0.05] = vocab + 3
        self.hist[r.random(self.hist.shape) < 0.02] = NO
        self.hist_len = r.integers(0, hist + 1, n_seqs) if hist else np.zeros(n_seqs, np.int64)
        self.use_len, self.hist_n = history_len, hist
        self.tokens = r.integers(0, min(vocab, 9), self.rows)
        self.parents = np.stack([_tree.make_parents(r, self.per, shape) for _ in range(n_seqs)])
        self.n_bias, self.per_seq = n_bias, bias_per_seq
        sets = n_seqs if bias_per_seq else 1
        self.bias_ids = r.integers(0, min(vocab, 2 * n_bias + 1), (sets, max(1, n_bias)))  # the same id twice and more
        self.bias_ids[r.random(self.bias_ids.shape) < 0.05] = vocab + 1
        self.bias = r.choice([-100.0, 2.5, 0.125, -np.inf], self.bias_ids.shape, p=[.3, .3, .3, .1]).astype(np.float32)
        self.words = (vocab + 31) // 32 + (3 if mask == "wide" else 0)
        self.mask = r.integers(0, 1 << 32, (self.rows, self.words), dtype=np.uint64).astype(np.uint32) if mask else None
        if mask:
            self.mask[r.random(self.rows) < 0.3] = 0xFFFFFFFF
            self.mask[0] = 0  # a row without any token

    def rules(self):
        b = self.dev = {}
        m = dict(rows_per_seq=self.per, repetition_penalty=self.pen[0], frequency_penalty=self.pen[1],
                 presence_penalty=self.pen[2])
        if self.hist_n:
            b["history"] = up(self.hist.astype(np.uint32))[0]
            m.update(history=b["history"], history_stride=self.hist_n)
            if self.use_len:
                b["len"] = up(self.hist_len.astype(np.uint32))[0]
                m["history_len"] = b["len"]
        if self.t:
            b["tokens"], b["parents"] = up(self.tokens.astype(np.uint32))[0], up(self.parents)[0]
            m.update(tree_tokens=b["tokens"], tree_parents=b["parents"])
        if self.n_bias:
            b["ids"], b["bias"] = up(self.bias_ids.astype(np.uint32))[0], up(self.bias)[0]
            m.update(bias_ids=b["ids"], bias=b["bias"], n_bias=self.n_bias, bias_stride=self.n_bias if self.per_seq else 0)
        if self.mask is not None:
            b["mask"] = up(self.mask)[0]
            m.update(mask=b["mask"], mask_stride=self.words)
        return ops.LogitsRules(**m)

    def row(self, i, dtype):
        """(logits, token) of row i, or None for an absent node's."""
        s, node = divmod(i, self.per)
        counts = np.zeros(self.v, np.int64)
        if self.hist_n:
            n = int(self.hist_len[s]) if self.use_len else self.hist_n
            h = self.hist[s, :n]
            np.add.at(counts, h[h < self.v], 1)
        if self.t:
            path = _tree.paths(self.parents[s])[node]
            if path is None:
                return None
            np.add.at(counts, self.tokens[s * self.per + np.array(path)], 1)
        bias = {}
        if self.n_bias:
            k = s if self.per_seq else 0
            bias = {int(a): b for a, b in zip(self.bias_ids[k], self.bias[k]) if a < self.v}
        allowed = None
        if self.mask is not None:
            allowed = np.unpackbits(self.mask[i].view(np.uint8), bitorder="little")[:self.v].astype(bool)
        return _tree.logits(self.x[i], self.v, *self.pen, counts, bias, allowed, dtype)

    def check(self, out, token):
        for i in range(self.rows):
            want = self.row(i, np.float32)
            if want is None:
                assert token is None or token[i] == NO
                assert out is None or (out[i].view(np.uint32) == 0xEEEEEEEE).all(), f"row {i}"
                continue
            l, tok = want
            if out is not None:
                assert (out[i, self.v:].view(np.uint32) == 0xEEEEEEEE).all(), "behind the row"
                got = out[i, :self.v]
                assert np.array_equal(np.isnan(got), np.isnan(l))
                assert np.array_equal(got[~np.isnan(l)], l[~np.isnan(l)]), f"row {i}"
                exact, _ = self.row(i, np.float64)
                fine = np.isfinite(exact) & np.isfinite(l)
                # the penalties round four times and the bias once, each by 2^-24 of what it makes
                rep, freq, pres = (abs(float(p)) for p in self.pen)
                size = np.abs(self.x[i, :self.v]) * max(rep, 1 / rep) + (self.hist_n + self.per) * freq + pres + 100
                assert (np.abs(got[fine] - exact[fine]) <= 5 * 2.0 ** -24 * size[fine]).all()
            if token is not None:
                assert token[i] == tok, f"row {i}: token {token[i]}, not {tok}"

    def launch(self, rules, xb, ob, tb, ws, wsz, stream=None):
        ops.logits_process(rules, xb, self.ld, self.rows, self.v, ob, self.ldo, tb, ws, wsz, stream)

    def run(self, write=True, pick=True):
        rules = self.rules()
        xb = up(self.x)[0]
        ob = DeviceBuffer(4 * self.rows * self.ldo + 256) if write else None
        tb = DeviceBuffer(4 * self.rows + 256) if pick else None
        wsz = ops.logits_process_workspace_bytes(rules, self.rows, self.v) if pick else 0
        ws = DeviceBuffer(wsz + 256)
        for b in (ob, tb, ws):
            if b:
                b.fill(0xEE)
        self.launch(rules, xb, ob, tb, ws, wsz)
        for b, size in ((ob, 4 * self.rows * self.ldo), (tb, 4 * self.rows), (ws, wsz)):
            assert not b or (down(b, np.uint8, 256, offset=size) == 0xEE).all(), "behind a buffer"
        out = down(ob, np.float32, self.rows * self.ldo).reshape(self.rows, self.ldo) if write else None
        token = down(tb, np.uint32, self.rows) if pick else None
        assert np.array_equal(down(xb, np.uint32, self.x.size), self.x.view(np.uint32).ravel()), "the input changed"
        self.check(out, token)


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 2047, 2048, 2049, 32000, 100003])
@pytest.mark.parametrize("n,hist,n_bias,mask", [(1, 0, 0, False), (1, 1, 1, True), (3, 500, 40, "wide"), (2, 5000, 0, False)])
def test_rows(gpu, vocab, n, hist, n_bias, mask):
    print(f"[case] logits {n}x{vocab} history {hist} bias {n_bias} mask {mask}", flush=True)
    Case(n, 0, vocab, hist, n_bias, mask, seed=vocab + n).run()


@pytest.mark.parametrize("tree", [1, 2, 33, 64, 128])
@pytest.mark.parametrize("shape", ["tree", "chain", "padded", "forest"])
@pytest.mark.parametrize("n,hist", [(1, 300), (3, 0)])
def test_trees(gpu, tree, shape, n, hist):
    print(f"[case] logits {shape} {tree} of {n} history {hist}", flush=True)
    Case(n, tree, 5003, hist, 30, True, seed=tree, shape=shape).run()


@pytest.mark.parametrize("ld,ldo", [(5001, 5000), (5004, 5008), (5064, 6000)])
@pytest.mark.parametrize("write,pick", [(True, True), (True, False), (False, True)])
def test_strides_and_outputs(gpu, ld, ldo, write, pick):
    Case(4, 0, 5000, 200, 10, True, ld=ld, ldo=ldo, seed=7).run(write, pick)


def test_all_history_counts_without_lengths(gpu):
    Case(2, 0, 3000, 700, 0, False, history_len=False, seed=3).run()


def test_biases_of_each_sequence(gpu):
    Case(5, 0, 3000, 50, 300, False, bias_per_seq=True, seed=4).run()


@pytest.mark.parametrize("rep,freq,pres", [(1.0, 0.0, 0.0), (1.0, -0.5, 0.0), (0.7, 0.0, -1.0), (1.0, 0.0, 1.5), (3e38, 0.0, 0.0)])
def test_penalties_that_do_nothing_or_reward(gpu, rep, freq, pres):
    Case(2, 5, 4000, 300, 0, True, rep=rep, freq=freq, pres=pres, seed=5, shape="padded").run()


def test_long_history(gpu):
    """A token that occurs tens of thousands of times, in a history of 200000; a length beyond the row is the row."""
    c = Case(1, 0, 40000, 200_000, 0, False, seed=6, freq=0.001)
    c.hist[0, ::3] = 12345
    c.hist_len[:] = 200_050
    c.run()


def test_infinities_nan_and_ties(gpu):
    c = Case(6, 0, 4100, 0, 0, True, seed=8)
    c.mask[:] = 0xFFFFFFFF
    c.x[0, 100] = c.x[0, 4000] = 50.0          # a tie: the lowest
    c.x[1, :] = -np.inf                        # nothing to choose
    c.x[2, :] = np.nan
    c.x[2, 3000] = -7.0                        # the only number
    c.x[3, [5, 6]] = np.inf                    # infinity is the largest
    c.x[4, :] = -0.0
    c.x[4, 2500] = 0.0                         # zeros of both signs tie
    c.x[5, 77] = np.inf
    c.x[5, 78] = np.nan
    c.mask[5, 77 // 32] &= ~np.uint32(3 << (77 % 32))  # both masked
    c.run()


def test_in_place(gpu):
    c = Case(3, 0, 5000, 100, 5, True, ld=5010, ldo=5010, seed=9)
    rules, xb, tb = c.rules(), up(c.x)[0], DeviceBuffer(12)
    wsz = ops.logits_process_workspace_bytes(rules, 3, 5000)
    c.launch(rules, xb, xb, tb, DeviceBuffer(wsz), wsz)
    got = down(xb, np.float32, c.x.size).reshape(c.x.shape)
    assert np.array_equal(got[:, 5000:], c.x[:, 5000:])
    got = got.copy()
    got[:, 5000:].view(np.uint32)[:] = 0xEEEEEEEE
    c.check(got, down(tb, np.uint32, 3))


def test_token_goes_into_the_next_step(gpu):
    """No token (0xFFFFFFFF) is an id that embedding_lookup answers with NaN; a chosen one is its row."""
    c = Case(2, 0, 64, 0, 0, True, seed=10)
    c.mask[:] = 0
    c.mask[1, 1] = 1 << 5  # token 37
    rules, tb = c.rules(), DeviceBuffer(8)
    wsz = ops.logits_process_workspace_bytes(rules, 2, 64)
    c.launch(rules, up(c.x)[0], None, tb, DeviceBuffer(wsz), wsz)
    table = c.rng.standard_normal((64, 32)).astype(np.float32)
    out = DeviceBuffer(4 * 2 * 32)
    _lib.check(_lib.load().wh_embedding_lookup(0, up(table)[0].ptr, 64, 32, tb.ptr, 2, out.ptr, None))
    got = down(out, np.float32, 64).reshape(2, 32)
    assert np.isnan(got[0]).all() and np.array_equal(got[1], table[37])


def test_captured_rules_follow_their_arrays(gpu):
    """Two graphs share one workspace in turn; logits, history, masks and trees change between the replays."""
    stream = Stream()
    cases = [Case(1, 20, 6000, 400, 20, True, seed=11), Case(3, 0, 9000, 100, 0, True, seed=12)]
    ready = []
    ws_bytes = max(ops.logits_process_workspace_bytes(c.rules(), c.rows, c.v) for c in cases)
    ws = DeviceBuffer(ws_bytes)
    for c in cases:
        rules, xb, ob, tb = c.rules(), up(c.x)[0], DeviceBuffer(4 * c.rows * c.v), DeviceBuffer(4 * c.rows)
        synchronize()
        with Graph.capture(stream) as g:
            c.launch(rules, xb, ob, tb, ws, ws_bytes, stream)
        ready.append((g, rules, xb, ob, tb))
    for rep in range(3):
        for c, (g, rules, xb, ob, tb) in zip(cases, ready):
            c.x = (c.rng.standard_normal(c.x.shape) * 4).astype(np.float32)
            c.hist = c.rng.integers(0, c.v, c.hist.shape)
            c.hist_len = c.rng.integers(0, c.hist_n + 1, c.n)
            xb.upload(c.x)
            c.dev["history"].upload(c.hist.astype(np.uint32))
            c.dev["len"].upload(c.hist_len.astype(np.uint32))
            if c.t:
                c.parents = np.stack([_tree.make_parents(c.rng, c.per, ("chain", "padded", "tree")[rep])])
                c.dev["parents"].upload(c.parents)
            ob.fill(0xEE)
            g.launch(stream)
            stream.synchronize()
            c.check(down(ob, np.float32, c.rows * c.v).reshape(c.rows, c.v), down(tb, np.uint32, c.rows))
        Case(2, 0, 700, 30, 0, False, seed=rep).run()
    for g, *_ in ready:
        g.destroy()
    stream.destroy()
