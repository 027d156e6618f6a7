"""More of what the calls for a tree of drafted tokens refuse, without a GPU: every check runs before a launch."""
import subprocess
import sys

import pytest

from tests.test_tree_abi import P, accept, compact, logits
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


def test_bias_stride_below_the_entries():
    """Each sequence would take the next one's first entries, the last would read past the arrays."""
    rules = dict(n_bias=30, bias_ids=P, bias=P)
    for stride in (1, 29):
        assert logits(dict(rules, bias_stride=stride)) == _lib.WH_ERR_INVALID_SHAPE
        assert b"bias stride" in _lib.load().wh_last_error()
    for stride in (0, 30, 64):
        assert logits(dict(rules, bias_stride=stride), workspace_bytes=0) == _lib.WH_ERR_BUFFER_TOO_SMALL
    assert logits(dict(bias_stride=5), workspace_bytes=0) == _lib.WH_ERR_BUFFER_TOO_SMALL  # no entries at all


SIZE = 2 * 100 * 8 * 128 * 2  # bytes of a cache of compact()


@pytest.mark.parametrize("k, v", [((P, P + 2 * SIZE), (P + SIZE, P + 3 * SIZE - 16)),  # v[1] begins within k[1]
                                  ((P + 16, P + 4 * SIZE), (P + 2 * SIZE, P)),         # k[0] begins within v[1]
                                  ((P, P + SIZE // 2), (P + 2 * SIZE, P + 4 * SIZE))])
def test_compact_refuses_caches_that_overlap(k, v):
    assert compact(k=k, v=v) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"within another" in _lib.load().wh_last_error()


def test_compact_looks_at_every_cache():
    k, v = [P + 2 * i * SIZE for i in range(300)], [P + (2 * i + 1) * SIZE for i in range(300)]
    assert compact(k=k, v=v[:299] + [P + 16]) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"within another" in _lib.load().wh_last_error()
    assert compact(k=k, v=v[:299] + [k[7]]) == _lib.WH_ERR_INVALID_ARGUMENT
    assert b"layer 299 is named twice" in _lib.load().wh_last_error()


def test_compact_sizes_that_no_memory_holds():
    assert compact(k=(P,), v=(P + 64,), n_seqs=65535, max_ctx=(1 << 31) - 1, n_kv_heads=1 << 10, head_dim=1 << 16) == \
        _lib.WH_ERR_INVALID_SHAPE
    assert b"are no cache" in _lib.load().wh_last_error()


def test_sizes_beyond_a_launch():
    assert accept(n_seqs=1 << 26) == _lib.WH_ERR_INVALID_SHAPE
    for heads, dim in ((1 << 10, 1 << 17), (1 << 40, 1 << 24), ((1 << 62) + 4, 2), (1 << 63, 16)):  # the last three wrap
        assert compact(k=(P,), v=(P + 64,), n_kv_heads=heads, head_dim=dim) == _lib.WH_ERR_INVALID_SHAPE
        assert b"whole 16-byte pieces" in _lib.load().wh_last_error()


def test_a_cache_without_rows_needs_no_workspace():
    """In a process of its own: the division by its rows would end this one."""
    code = "from woolly_amd import ops; print(ops.attention_tree_workspace_bytes(1, 5, 32, 8, 128, 0))"
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "0", (run.returncode, run.stderr[-300:])
