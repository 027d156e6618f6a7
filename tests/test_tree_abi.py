"""What the calls that verify a tree of drafted tokens refuse, without a GPU: every check runs before a launch."""
import ctypes as C

import pytest

from woolly_amd import _lib, ops

P = 0x10000  # a non-null, aligned address that nothing reads
HUGE = 1 << 50


def attention(**over):
    a = dict(q=P, k=P, v=P, ldq=4096, ldkv=1024, parents=P, ctx_len=P, n_seqs=2, n_tree=26, k_cache=P, v_cache=P,
             max_ctx=4096, n_heads=32, n_kv_heads=8, head_dim=128, inv_freq=P, out=P, workspace=P, workspace_bytes=HUGE)
    assert not set(over) - set(a)
    return _lib.load().wh_attention_tree(*{**a, **over}.values(), None)


@pytest.mark.parametrize("over", [dict(head_dim=96), dict(head_dim=0), dict(n_kv_heads=0), dict(n_heads=30), dict(n_heads=0),
                                  dict(n_heads=1032, ldq=HUGE), dict(n_tree=129), dict(n_seqs=1025), dict(max_ctx=0),
                                  dict(max_ctx=1 << 31), dict(max_ctx=1 << 30, n_seqs=4), dict(ldq=4095), dict(ldkv=1023)])
def test_attention_shapes(over):
    assert attention(**over) == _lib.WH_ERR_INVALID_SHAPE
    assert b"attention_tree" in _lib.load().wh_last_error()


@pytest.mark.parametrize("name", ["q", "k", "v", "parents", "ctx_len", "k_cache", "v_cache", "inv_freq", "out", "workspace"])
def test_attention_pointers(name):
    assert attention(**{name: None}) == _lib.WH_ERR_INVALID_ARGUMENT
    assert attention(**{name: P + 2}) == _lib.WH_ERR_INVALID_ARGUMENT
    if "cache" in name or name == "workspace":
        assert attention(**{name: P + 8}) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"attention_tree" in _lib.load().wh_last_error()


def test_attention_workspace_and_empty_calls():
    need = ops.attention_tree_workspace_bytes(2, 26, 32, 8, 128, 4096)
    assert need > 0
    assert attention(workspace_bytes=need - 1) == _lib.WH_ERR_BUFFER_TOO_SMALL
    assert f"needed {need} bytes".encode() in _lib.load().wh_last_error()
    assert attention(n_seqs=0, q=None) == _lib.WH_OK
    assert attention(n_tree=0, q=None) == _lib.WH_OK
    for bad in ((0, 26, 32, 8, 128, 4096), (2, 0, 32, 8, 128, 4096), (2, 129, 32, 8, 128, 4096), (1025, 1, 32, 8, 128, 4096),
                (2, 26, 32, 8, 80, 4096), (2, 26, 30, 8, 128, 4096), (2, 26, 32, 8, 128, 1 << 31), (4, 26, 32, 8, 128, 1 << 30)):
        assert ops.attention_tree_workspace_bytes(*bad) == 0
    # more room, more nodes or more sequences never need less
    assert ops.attention_tree_workspace_bytes(2, 26, 32, 8, 128, 64) <= need
    assert ops.attention_tree_workspace_bytes(3, 26, 32, 8, 128, 4096) >= need


def logits(rules=None, **over):
    r = dict(rows_per_seq=1, repetition_penalty=1.0)
    r.update(rules or {})
    a = dict(logits=P, ld=1000, n_rows=4, vocab=1000, out=P + 64, ld_out=1000, token=P, workspace=P, workspace_bytes=HUGE)
    a.update(over)
    lr = ops.LogitsRules(**r)
    return _lib.load().wh_logits_process(C.byref(lr.rules), *a.values(), None)


@pytest.mark.parametrize("over", [dict(vocab=0), dict(vocab=1 << 31, ld=HUGE, ld_out=HUGE), dict(n_rows=65536), dict(ld=999),
                                  dict(ld_out=999), dict(rules=dict(rows_per_seq=3)), dict(rules=dict(mask=P, mask_stride=31))])
def test_logits_shapes(over):
    assert logits(**over) == _lib.WH_ERR_INVALID_SHAPE
    assert b"logits_process" in _lib.load().wh_last_error()


@pytest.mark.parametrize("rules", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=float("inf")),
                                   dict(repetition_penalty=float("nan")), dict(frequency_penalty=float("nan")),
                                   dict(presence_penalty=float("-inf")), dict(tree_tokens=P), dict(tree_parents=P),
                                   dict(n_bias=3), dict(n_bias=3, bias=P), dict(n_bias=3, bias_ids=P),
                                   dict(n_bias=1 << 31, bias=P, bias_ids=P), dict(mask=P + 1, mask_stride=40),
                                   dict(history=P + 2, history_stride=5), dict(history=P, history_stride=5, history_len=P + 1)])
def test_logits_rules(rules):
    assert logits(rules) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"logits_process" in _lib.load().wh_last_error()


def test_logits_pointers_and_workspace():
    lib = _lib.load()
    assert logits(logits=None) == _lib.WH_ERR_INVALID_ARGUMENT
    assert logits(out=P, ld_out=1024) == _lib.WH_ERR_INVALID_ARGUMENT  # in place with another stride
    assert logits(logits=P + 2) == _lib.WH_ERR_INVALID_ARGUMENT
    assert logits(workspace=P + 4) == _lib.WH_ERR_INVALID_ARGUMENT
    assert logits(dict(rows_per_seq=129, tree_tokens=P, tree_parents=P), n_rows=129) == _lib.WH_ERR_INVALID_ARGUMENT
    need = ops.logits_process_workspace_bytes(ops.LogitsRules(), 4, 1000)
    assert need > 0
    assert logits(workspace_bytes=need - 1) == _lib.WH_ERR_BUFFER_TOO_SMALL
    assert logits(workspace=None) == _lib.WH_ERR_BUFFER_TOO_SMALL
    assert f"needed {need} bytes".encode() in lib.wh_last_error()
    assert lib.wh_logits_process(None, P, 1000, 4, 1000, P, 1000, P, P, HUGE, None) == _lib.WH_ERR_INVALID_ARGUMENT
    assert lib.wh_logits_process_workspace_bytes(None, 4, 1000) == 0
    assert logits(n_rows=0, logits=None) == _lib.WH_OK
    assert logits(out=None, token=None, logits=None) == _lib.WH_OK
    with pytest.raises(TypeError, match="no member 'temperature'"):
        ops.LogitsRules(temperature=0.5)


def accept(**over):
    a = dict(tokens=P, parents=P, picked=P, n_seqs=2, n_tree=26, path=P, n_accepted=P, next_token=P, ctx_len=P,
             ctx_len_out=P, history=P, history_stride=100)
    a.update(over)
    return _lib.load().wh_tree_accept(*a.values(), None)


def test_accept_refusals():
    assert accept(n_tree=129) == _lib.WH_ERR_INVALID_SHAPE
    assert accept(n_seqs=1 << 31) == _lib.WH_ERR_INVALID_SHAPE
    for name in ("tokens", "parents", "picked", "path", "n_accepted", "next_token", "ctx_len"):
        assert accept(**{name: None}) == _lib.WH_ERR_INVALID_ARGUMENT, name
        assert b"tree_accept" in _lib.load().wh_last_error()
    for name in ("tokens", "parents", "picked", "path", "n_accepted", "next_token", "ctx_len", "ctx_len_out", "history"):
        assert accept(**{name: P + 1}) == _lib.WH_ERR_INVALID_ARGUMENT, name
    assert accept(ctx_len=None, history=None) == _lib.WH_ERR_INVALID_ARGUMENT
    assert accept(n_seqs=0, tokens=None) == _lib.WH_OK
    assert accept(n_tree=0, tokens=None) == _lib.WH_OK


def compact(k=(P, P), v=(P, P), **over):
    caches = ops.KvCaches(list(k), list(v))
    a = dict(k=C.addressof(caches.k), v=C.addressof(caches.v), n_layers=len(k), n_seqs=2, max_ctx=100, n_kv_heads=8,
             head_dim=128, path=P, n_tree=26, n_accepted=P, ctx_len=P)
    a.update(over)
    return _lib.load().wh_kv_cache_compact(*a.values(), None)


@pytest.mark.parametrize("k, v", [((P, P + 64), (P + 128, P)), ((P, P + 64), (P + 128, P + 128)), ((P, P), (P + 64, P + 128)),
                                  ((P, P + 64), (P, P + 128)), ((P, P + 64), (P + 64, P + 128))])
def test_compact_refuses_a_cache_named_twice(k, v):
    assert compact(k=k, v=v) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"named twice" in _lib.load().wh_last_error()


def test_compact_refusals():
    for over in (dict(n_kv_heads=1, head_dim=4), dict(head_dim=0), dict(n_tree=129), dict(n_seqs=65536), dict(max_ctx=0),
                 dict(max_ctx=1 << 31), dict(n_kv_heads=1 << 20, head_dim=1 << 12)):
        assert compact(**over) == _lib.WH_ERR_INVALID_SHAPE, over
        assert b"kv_cache_compact" in _lib.load().wh_last_error()
    for over in (dict(k=None), dict(v=None), dict(path=None), dict(n_accepted=None), dict(ctx_len=None), dict(path=P + 2)):
        arrays = {n: over.pop(n) for n in ("k", "v") if n in over}
        caches = ops.KvCaches([P], [P])
        a = dict(k=C.addressof(caches.k), v=C.addressof(caches.v), n_layers=1, n_seqs=2, max_ctx=100, n_kv_heads=8,
                 head_dim=128, path=P, n_tree=26, n_accepted=P, ctx_len=P)
        a.update(arrays, **over)
        assert _lib.load().wh_kv_cache_compact(*a.values(), None) == _lib.WH_ERR_INVALID_ARGUMENT
    assert compact(k=(P, 0)) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"layer 1" in _lib.load().wh_last_error()
    assert compact(v=(P + 8, P)) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"layer 0" in _lib.load().wh_last_error()
    assert compact(k=(), v=()) == _lib.WH_OK
    assert compact(n_seqs=0, path=None) == _lib.WH_OK
    with pytest.raises(ValueError, match="2 K caches and 1 V caches"):
        ops.KvCaches([P, P], [P])


def fake_model(**over):
    layers = (_lib.wh_llama_layer * 2)()
    for L in layers:
        for name, _ in _lib.wh_llama_layer._fields_:
            if not name.endswith("_type"):
                setattr(L, name, P)
    m = _lib.wh_llama_model()
    m.type = 2
    m.n_layers, m.hidden, m.n_heads, m.n_kv_heads, m.head_dim = 2, 256, 4, 2, 64
    m.n_ff, m.max_ctx, m.vocab, m.eps = 512, 16, 300, 1e-5
    m.rope_inv_freq, m.output_norm, m.output, m.output_type = P, P, P, 8
    m.token_embd, m.token_embd_type = P, 1
    m.layers = C.cast(layers, C.POINTER(_lib.wh_llama_layer))
    for k, v in over.items():
        if k.startswith("layer_"):
            setattr(layers[1], k[6:], v)
        else:
            setattr(m, k, v)
    return m, layers


def forward(model, **over):
    a = dict(tokens=P, parents=P, n_tree=26, ctx_len=P, x=P, logits=P, workspace=P, workspace_bytes=HUGE)
    a.update(over)
    return _lib.load().wh_llama_forward_tree(C.byref(model[0]), *a.values(), None)


@pytest.mark.parametrize("over,status", [
    (dict(head_dim=96), 2), (dict(n_heads=3), 2), (dict(hidden=0), 2), (dict(n_ff=0), 2), (dict(max_ctx=0), 2),
    (dict(max_ctx=1 << 31), 2), (dict(hidden=272), 2), (dict(vocab=0), 2), (dict(vocab=1 << 30), 2), (dict(type=6), 1),
    (dict(type=12, n_ff=544), 2), (dict(output_type=1), 1), (dict(output=None), 4), (dict(output_norm=None), 4),
    (dict(token_embd=None), 4), (dict(token_embd_type=10), 1), (dict(rope_inv_freq=None), 4), (dict(layer_wv=None), 4),
    (dict(layer_w_down=None), 4), (dict(layer_w_up_type=7), 1), (dict(layer_k_cache=P + 8), 4), (dict(layer_v_cache=None), 4),
    (dict(layer_ffn_norm=None), 4), (dict(layer_attn_norm=P + 2), 4)])
def test_forward_tree_models(over, status):
    m = fake_model(**over)
    assert forward(m) == status
    assert b"llama_forward_tree" in _lib.load().wh_last_error()


def test_forward_tree_arguments():
    lib, m = _lib.load(), fake_model()
    assert forward(m, n_tree=129) == _lib.WH_ERR_INVALID_SHAPE
    assert forward(m, n_tree=0, tokens=None) == _lib.WH_OK
    for name in ("tokens", "parents", "ctx_len", "x"):
        assert forward(m, **{name: None}) == _lib.WH_ERR_INVALID_ARGUMENT, name
        assert forward(m, **{name: P + 2}) == _lib.WH_ERR_INVALID_ARGUMENT, name
    assert forward(m, x=P + 8) == _lib.WH_ERR_INVALID_ARGUMENT
    assert forward(m, workspace=P + 128) == _lib.WH_ERR_INVALID_ARGUMENT
    need = lib.wh_llama_forward_tree_workspace_bytes(C.byref(m[0]), 26)
    assert need > ops.attention_tree_workspace_bytes(1, 26, 4, 2, 64, 16)
    assert forward(m, workspace_bytes=need - 1) == _lib.WH_ERR_BUFFER_TOO_SMALL
    assert f"needed {need} bytes".encode() in lib.wh_last_error()
    assert forward(m, workspace=None) == _lib.WH_ERR_BUFFER_TOO_SMALL
    assert lib.wh_llama_forward_tree_workspace_bytes(C.byref(m[0]), 0) == 0
    assert lib.wh_llama_forward_tree_workspace_bytes(C.byref(m[0]), 129) == 0
    assert lib.wh_llama_forward_tree_workspace_bytes(None, 5) == 0
    assert lib.wh_llama_forward_tree(None, P, P, 5, P, P, P, P, HUGE, None) == _lib.WH_ERR_INVALID_ARGUMENT
    # without logits the head is not looked at
    assert forward(fake_model(output=None), logits=None, workspace_bytes=0) == _lib.WH_ERR_BUFFER_TOO_SMALL
