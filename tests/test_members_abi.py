"""What the calls for several continuations of one prompt refuse, without a GPU: every check runs before a launch."""
import ctypes as C

import numpy as np
import pytest

from tests.test_tree_abi import HUGE, P, fake_model
from woolly_amd import _lib, ops

SHAPE, SMALL, ARGUMENT = _lib.WH_ERR_INVALID_SHAPE, _lib.WH_ERR_BUFFER_TOO_SMALL, _lib.WH_ERR_INVALID_ARGUMENT


def rope(rules=None, **over):
    r = ops.RopeRules(P, 64, False, 1.0, P, P, 1e-5)
    for k, v in (rules or {}).items():
        setattr(r.rules, k, v)
    a = dict(q=P, k=P, v=P, ldq=4096, ldkv=1024, base_len=P, len=P, n_groups=2, n_per=3, n_new=5, n_heads=32, n_kv_heads=8,
             head_dim=128, q_out=P + 64, ldq_out=4096, k_out=P + 128, ldk_out=1024, k_cache=P, v_cache=P + 32, max_rows=100)
    assert not set(over) - set(a)
    return _lib.load().wh_qk_norm_rope(C.byref(r.rules), *{**a, **over}.values(), None)


@pytest.mark.parametrize("over", [dict(head_dim=0), dict(head_dim=127), dict(head_dim=258), dict(rules=dict(rot_dim=3)),
                                  dict(rules=dict(rot_dim=130)), dict(n_heads=0), dict(n_kv_heads=0), dict(n_heads=65536),
                                  dict(ldq=4095), dict(ldkv=1023), dict(ldq_out=4095), dict(ldk_out=1023), dict(max_rows=0),
                                  dict(max_rows=1 << 31), dict(n_groups=1 << 40), dict(n_new=1 << 31), dict(n_per=1 << 63)])
def test_rope_shapes(over):
    assert rope(**over) == SHAPE
    assert b"qk_norm_rope" in _lib.load().wh_last_error()


@pytest.mark.parametrize("over", [dict(q=None), dict(k=None), dict(v=None), dict(k_cache=None), dict(v_cache=None), dict(q=P + 2),
                                  dict(k=P + 1), dict(v=P + 2), dict(len=P + 2), dict(base_len=P + 1), dict(q_out=P + 2),
                                  dict(k_out=P + 2), dict(k_cache=P + 1), dict(k_cache=P + 32), dict(q_out=P, ldq_out=5000),
                                  dict(k_out=P, ldk_out=1025), dict(rules=dict(inv_freq=None)), dict(rules=dict(inv_freq=P + 2)),
                                  dict(rules=dict(q_norm=P + 1)), dict(rules=dict(k_norm=P + 2)),
                                  dict(rules=dict(magnitude=float("inf"))), dict(rules=dict(magnitude=float("nan"))),
                                  dict(rules=dict(norm_eps=-1.0)), dict(rules=dict(norm_eps=float("nan"))),
                                  dict(rules=dict(norm_eps=float("inf")))])
def test_rope_arguments(over):
    assert rope(**over) == ARGUMENT
    assert b"qk_norm_rope" in _lib.load().wh_last_error()


def test_rope_nothing_to_do():
    assert rope(n_groups=0, q=None) == _lib.WH_OK
    assert rope(n_per=0, q=None) == _lib.WH_OK
    assert rope(n_new=0, q=None) == _lib.WH_OK
    assert rope(q_out=None, k_out=None, k_cache=None, v_cache=None) == _lib.WH_OK
    assert _lib.load().wh_qk_norm_rope(None, *[P] * 3, 4096, 1024, P, P, 1, 1, 1, 32, 8, 128, P, 4096, P, 1024, P, P, 9,
                                       None) == ARGUMENT


def test_scaled_frequencies():
    """Against their definitions in 64 bits, rounded once."""
    base, d, factor, ctx = 10000.0, 64, 8.0, 4096
    f = 1 / base ** (np.arange(0, d, 2) / d)
    near = lambda got, want: np.allclose(got[0], want, rtol=2.0 ** -23, atol=0)
    assert near(ops.rope_scaled_inv_freq(ops.ROPE_PLAIN, base, d), f)
    assert near(ops.rope_scaled_inv_freq(ops.ROPE_LINEAR, base, d, factor), f / factor)
    assert near(ops.rope_scaled_inv_freq(ops.ROPE_BASE, base, d, factor), 1 / (base * factor ** (d / (d - 2))) ** (np.arange(0, d, 2) / d))
    turns = ctx * f / (2 * np.pi)
    g = np.clip((turns - 1) / (4 - 1), 0, 1)
    got = ops.rope_scaled_inv_freq(ops.ROPE_BY_TURNS, base, d, factor, ctx, 1.0, 4.0)
    assert near(got, f * (g + (1 - g) / factor)) and got[1] == 1.0
    assert got[0][0] == 1.0 and np.isclose(got[0][-1], f[-1] / factor)
    index = lambda t: d * np.log(ctx / (t * 2 * np.pi)) / (2 * np.log(base))
    lo, hi = np.floor(index(32.0)), np.ceil(index(1.0))
    g = 1 - np.clip((np.arange(d // 2) - lo) / (hi - lo), 0, 1)
    got = ops.rope_scaled_inv_freq(ops.ROPE_BY_INDEX, base, d, factor, ctx, 1.0, 32.0)
    assert near(got, f * (g + (1 - g) / factor)) and np.isclose(got[1], 0.1 * np.log(factor) + 1, rtol=1e-15)
    # all turns within one index: a step
    got = ops.rope_scaled_inv_freq(ops.ROPE_BY_INDEX, base, d, factor, 1, 1.0, 32.0)[0]
    assert np.isfinite(got).all()


@pytest.mark.parametrize("args,status", [((5, 1e4, 64), ARGUMENT), ((-1, 1e4, 64), ARGUMENT), ((0, 1e4, 0), SHAPE), ((0, 1e4, 63), SHAPE),
                                         ((2, 1e4, 2, 2.0), SHAPE), ((0, 0.0, 64), ARGUMENT), ((0, float("nan"), 64), ARGUMENT),
                                         ((4, 1.0, 64, 2.0, 4096, 1.0, 32.0), ARGUMENT), ((1, 1e4, 64, 0.0), ARGUMENT),
                                         ((1, 1e4, 64, float("inf")), ARGUMENT), ((3, 1e4, 64, 2.0, 0, 1.0, 4.0), ARGUMENT),
                                         ((3, 1e4, 64, 2.0, 4096, 4.0, 4.0), ARGUMENT), ((3, 1e4, 64, 2.0, 4096, 0.0, 4.0), ARGUMENT)])
def test_scaled_frequencies_refused(args, status):
    with pytest.raises(_lib.WoollyHipError) as e:
        ops.rope_scaled_inv_freq(*args)
    assert e.value.status == status and "rope_scaled_inv_freq" in str(e.value)
    assert _lib.load().wh_rope_scaled_inv_freq(0, 1e4, 64, 1.0, 0, 0.0, 0.0, None, None) == ARGUMENT


def attention(**over):
    a = dict(q=P, ldq=4096, prefix_len=P, own_len=P, n_groups=2, n_per=4, k_prefix=P, v_prefix=P, max_prefix=4096, k_own=P, v_own=P,
             max_own=300, n_heads=32, n_kv_heads=8, head_dim=128, out=P, workspace=P, workspace_bytes=HUGE)
    assert not set(over) - set(a)
    return _lib.load().wh_attention_shared(*{**a, **over}.values(), None)


@pytest.mark.parametrize("over", [dict(head_dim=96), dict(head_dim=0), dict(n_kv_heads=0), dict(n_heads=30), dict(n_heads=0),
                                  dict(n_heads=1032, ldq=HUGE), dict(n_per=4097), dict(n_groups=4097), dict(n_groups=1 << 32, n_per=1 << 32),
                                  dict(n_groups=100, n_per=100), dict(max_prefix=1 << 31), dict(max_own=1 << 31), dict(ldq=4095)])
def test_attention_shapes(over):
    assert attention(**over) == SHAPE
    assert b"attention_shared" in _lib.load().wh_last_error()


@pytest.mark.parametrize("name", ["q", "out", "prefix_len", "own_len", "k_prefix", "v_prefix", "k_own", "v_own"])
def test_attention_pointers(name):
    assert attention(**{name: None}) == ARGUMENT
    assert attention(**{name: P + 2}) == ARGUMENT
    if name[:2] in ("k_", "v_"):
        assert attention(**{name: P + 8}) == ARGUMENT
    assert b"attention_shared" in _lib.load().wh_last_error()


def test_attention_workspace_and_empty_calls():
    need = ops.attention_shared_workspace_bytes(2, 4, 32, 8, 128, 4096, 300)
    assert need > 0
    assert attention(workspace_bytes=need - 1) == SMALL
    assert f"needed {need} bytes".encode() in _lib.load().wh_last_error()
    assert attention(workspace=None) == SMALL
    assert attention(workspace=P + 8) == ARGUMENT
    assert attention(n_groups=0, q=None) == _lib.WH_OK
    assert attention(n_per=0, q=None) == _lib.WH_OK
    # rows of one kind only need nothing of the other
    assert attention(max_prefix=0, prefix_len=None, k_prefix=None, v_prefix=None, workspace_bytes=0) == SMALL
    assert attention(max_own=0, own_len=None, k_own=None, v_own=None, workspace_bytes=0) == SMALL
    for bad in ((0, 4, 32, 8, 128, 4096, 300), (2, 0, 32, 8, 128, 4096, 300), (2, 4, 32, 8, 80, 4096, 300), (2, 4, 30, 8, 128, 4096, 300),
                (2, 4, 32, 8, 128, 1 << 31, 300), (2, 4, 32, 8, 128, 4096, 1 << 31), (2, 2049, 32, 8, 128, 4096, 300)):
        assert ops.attention_shared_workspace_bytes(*bad) == 0
    # larger caches never need less; every number of members has a size
    for per in (1, 2, 7, 8, 9, 16, 33, 64, 100, 4096):
        sizes = [ops.attention_shared_workspace_bytes(1, per, 32, 8, 128, p, 10) for p in (1, 1000, 8000)]
        assert 0 < sizes[0] and max(sizes) < 1 << 32


def select(rules=None, **over):
    r = dict(n_beams=4, n_out=4)
    r.update(rules or {})
    a = dict(logits=P, ld=1000, n_seqs=3, vocab=1000, scores=P, scores_out=P, tokens=P, parents=P, workspace=P, workspace_bytes=HUGE)
    assert not set(over) - set(a)
    br = ops.BeamRules(**r)
    return _lib.load().wh_beam_select(C.byref(br.rules), *{**a, **over}.values(), None)


@pytest.mark.parametrize("over", [dict(rules=dict(n_beams=0, n_out=0)), dict(rules=dict(n_beams=33)), dict(rules=dict(n_out=65)),
                                  dict(vocab=0), dict(vocab=1 << 31, ld=HUGE), dict(ld=999), dict(n_seqs=16384), dict(n_seqs=1 << 62)])
def test_select_shapes(over):
    assert select(**over) == SHAPE
    assert b"beam_select" in _lib.load().wh_last_error()


@pytest.mark.parametrize("over", [dict(rules=dict(length_penalty=float("nan"))), dict(rules=dict(length_penalty=float("inf"))),
                                  dict(rules=dict(history=P, history_stride=9)), dict(rules=dict(len_out=P)),
                                  dict(rules=dict(n_out=8, history=P, history_stride=9, len=P), scores_out=P + 64),
                                  dict(rules=dict(n_out=8)), dict(rules=dict(n_out=8, last_tokens=P), scores_out=P + 64),
                                  dict(rules=dict(n_out=8, counts=P, counts_out=P), scores_out=P + 64),
                                  dict(rules=dict(last_tokens=P + 2)), dict(rules=dict(counts=P + 1)), dict(rules=dict(counts_out=P + 2)),
                                  dict(rules=dict(len=P + 2)), dict(rules=dict(len=P, len_out=P + 1)),
                                  dict(rules=dict(len=P, history=P + 2)), dict(logits=None), dict(scores=None), dict(scores_out=None),
                                  dict(tokens=None), dict(parents=None), dict(logits=P + 2), dict(scores=P + 1), dict(tokens=P + 2),
                                  dict(parents=P + 2), dict(workspace=P + 8)])
def test_select_arguments(over):
    assert select(**over) == ARGUMENT
    assert b"beam_select" in _lib.load().wh_last_error()


def test_select_workspace_and_empty_calls():
    lib = _lib.load()
    need = ops.beam_select_workspace_bytes(ops.BeamRules(4), 3, 1000)
    assert need > 0
    assert select(workspace_bytes=need - 1) == SMALL
    assert f"needed {need} bytes".encode() in lib.wh_last_error()
    assert select(workspace=None) == SMALL
    assert select(n_seqs=0, logits=None) == _lib.WH_OK
    assert lib.wh_beam_select(None, P, 1000, 3, 1000, P, P, P, P, P, HUGE, None) == ARGUMENT
    assert lib.wh_beam_select_workspace_bytes(None, 3, 1000) == 0
    for bad in ((0, 4), (33, 4), (4, 65)):
        assert ops.beam_select_workspace_bytes(ops.BeamRules(*bad), 3, 1000) == 0
    for seqs, vocab in ((0, 1000), (16384, 1000), (3, 0), (3, 1 << 31)):
        assert ops.beam_select_workspace_bytes(ops.BeamRules(4), seqs, vocab) == 0
    with pytest.raises(TypeError, match="no member 'temperature'"):
        ops.BeamRules(4, temperature=0.5)


SIZE = 2 * 4 * 100 * 2048  # bytes of a state of reorder()


def reorder(states=(P, P + SIZE), **over):
    st = ops.BeamStates(list(states))
    a = dict(states=st.address, n_states=len(states), n_seqs=2, n_beams=4, max_rows=100, row_bytes=2048, parents=P, len=P, pending=1)
    assert not set(over) - set(a)
    return _lib.load().wh_beam_reorder(*{**a, **over}.values(), None)


def test_reorder_refusals():
    for over in (dict(row_bytes=0), dict(row_bytes=6), dict(row_bytes=1 << 28), dict(n_beams=33), dict(n_seqs=65536), dict(max_rows=0),
                 dict(max_rows=1 << 31)):
        assert reorder(**over) == SHAPE, over
        assert b"beam_reorder" in _lib.load().wh_last_error()
    for over in (dict(states=None), dict(parents=None), dict(len=None), dict(parents=P + 2), dict(len=P + 1)):
        arrays = {"states": over.pop("states")} if "states" in over else {}
        st = ops.BeamStates([P])
        a = dict(states=st.address, n_states=1, n_seqs=2, n_beams=4, max_rows=100, row_bytes=2048, parents=P, len=P, pending=1)
        assert _lib.load().wh_beam_reorder(*{**a, **arrays, **over}.values(), None) == ARGUMENT
    for states in ((P, 0), (P, P + SIZE + 8)):
        assert reorder(states) == ARGUMENT
        assert b"state 1" in _lib.load().wh_last_error()
    assert reorder((P, P + SIZE + 4), row_bytes=36, n_states=0) == _lib.WH_OK  # 4-byte aligned rows would do
    assert reorder((P, P)) == ARGUMENT and b"named twice" in _lib.load().wh_last_error()
    assert reorder((P + SIZE - 16, P)) == ARGUMENT and b"within another" in _lib.load().wh_last_error()
    many = [P + i * SIZE for i in range(700)]
    assert reorder(many[:699] + [many[3]]) == ARGUMENT and b"state 699 is named twice" in _lib.load().wh_last_error()
    assert reorder(many[:699] + [many[3] + 32]) == ARGUMENT and b"within another" in _lib.load().wh_last_error()
    assert reorder((P,), n_seqs=65535, n_beams=32, max_rows=(1 << 31) - 1, row_bytes=(1 << 28) - 16) == SHAPE
    assert reorder((P, P + SIZE), n_seqs=0, parents=None) == _lib.WH_OK
    assert reorder((P, P + SIZE), n_beams=0, parents=None) == _lib.WH_OK
    assert reorder((), parents=None) == _lib.WH_OK


def forward(model, k=(P, P + 64), v=(P + 128, P + 256), rules=None, **over):
    own = ops.KvCaches(list(k), list(v))
    a = dict(rules=C.byref(rules.rules) if rules else None, tokens=P, n_members=26, prefix_len=P, len=P, k=C.addressof(own.k),
             v=C.addressof(own.v), max_own=64, x=P, logits=P, workspace=P, workspace_bytes=HUGE)
    assert not set(over) - set(a)
    return _lib.load().wh_llama_forward_members(C.byref(model[0]), *{**a, **over}.values(), None)


@pytest.mark.parametrize("over,status", [
    (dict(head_dim=96), 2), (dict(n_heads=3), 2), (dict(hidden=0), 2), (dict(max_ctx=0), 2), (dict(vocab=0), 2), (dict(type=6), 1),
    (dict(output=None), 4), (dict(output_norm=None), 4), (dict(token_embd=None), 4), (dict(token_embd_type=10), 1),
    (dict(rope_inv_freq=None), 4), (dict(layer_wv=None), 4), (dict(layer_w_up_type=7), 1), (dict(layer_k_cache=P + 8), 4)])
def test_forward_members_models(over, status):
    assert forward(fake_model(**over)) == status
    assert b"llama_forward_members" in _lib.load().wh_last_error()


def test_forward_members_arguments():
    lib, m = _lib.load(), fake_model()
    assert forward(m, n_members=129) == SHAPE
    assert forward(m, max_own=0) == SHAPE
    assert forward(m, max_own=1 << 31) == SHAPE
    assert forward(m, n_members=0, tokens=None) == _lib.WH_OK
    for name in ("tokens", "prefix_len", "len", "x"):
        assert forward(m, **{name: None}) == ARGUMENT, name
        assert forward(m, **{name: P + 2}) == ARGUMENT, name
    assert forward(m, k=(P, 0)) == ARGUMENT and b"layer 1" in lib.wh_last_error()
    assert forward(m, v=(P + 8, P + 256)) == ARGUMENT and b"layer 0" in lib.wh_last_error()
    assert forward(m, k=(P, P + 256)) == ARGUMENT and b"layer 1" in lib.wh_last_error()  # K and V the same
    assert forward(m, x=P + 8) == ARGUMENT
    assert forward(m, workspace=P + 128) == ARGUMENT
    assert forward(m, rules=ops.RopeRules(None)) == ARGUMENT
    assert forward(m, rules=ops.RopeRules(P, 66)) == SHAPE
    need = lib.wh_llama_forward_members_workspace_bytes(C.byref(m[0]), 26, 64)
    assert need > ops.attention_shared_workspace_bytes(1, 26, 4, 2, 64, 16, 64)
    assert forward(m, workspace_bytes=need - 1) == SMALL
    assert f"needed {need} bytes".encode() in lib.wh_last_error()
    assert forward(m, workspace=None) == SMALL
    for members, own in ((0, 64), (129, 64), (26, 0), (26, 1 << 31)):
        assert lib.wh_llama_forward_members_workspace_bytes(C.byref(m[0]), members, own) == 0
    assert lib.wh_llama_forward_members_workspace_bytes(None, 5, 64) == 0
    # without logits the head is not looked at
    assert forward(fake_model(output=None), logits=None, workspace_bytes=0) == SMALL
