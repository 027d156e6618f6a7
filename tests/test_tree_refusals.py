"""More of what the calls for a tree of drafted tokens refuse, without a GPU: every check runs before a launch."""
from tests.test_tree_abi import P
from woolly_amd import _lib


def test_accept_in_cache_refusals():
    def call(**over):
        a = dict(tokens=P, parents=P, picked=P, n_seqs=2, n_tree=26, path=P, n_accepted=P, next_token=P, ctx_len=P,
                 ctx_len_out=P, history=P, history_stride=100, max_ctx=4096)
        a.update(over)
        return _lib.load().wh_tree_accept_in_cache(*a.values(), None)

    for max_ctx in (0, 1 << 31, 1 << 40):
        assert call(max_ctx=max_ctx) == _lib.WH_ERR_INVALID_SHAPE
        assert b"tree_accept_in_cache" in _lib.load().wh_last_error()
    assert call(n_tree=129) == _lib.WH_ERR_INVALID_SHAPE
    assert call(ctx_len=None, ctx_len_out=None, history=None) == _lib.WH_ERR_INVALID_ARGUMENT
    for name in ("tokens", "parents", "picked", "path", "n_accepted", "next_token", "ctx_len"):
        assert call(**{name: None}) == _lib.WH_ERR_INVALID_ARGUMENT, name
        assert call(**{name: P + 1}) == _lib.WH_ERR_INVALID_ARGUMENT, name
    assert call(n_seqs=0, tokens=None) == _lib.WH_OK
    assert call(n_tree=0, tokens=None) == _lib.WH_OK
