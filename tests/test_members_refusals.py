"""Calls for several continuations of one prompt that are refused before anything runs.  No GPU needed."""
import pytest

from tests.test_members_abi import P, SHAPE, SMALL, attention
from woolly_amd import _lib, ops


def test_more_heads_than_the_joins_launch_takes():
    """4096 groups of one member with 1024 KV heads of 128: 2^26 waves of 64 threads."""
    most = dict(n_groups=4096, n_per=1, n_heads=1024, n_kv_heads=1024, head_dim=128, ldq=1 << 17, max_prefix=1, max_own=0)
    assert attention(**most) == SHAPE
    assert b"attention_shared" in _lib.load().wh_last_error()
    size = lambda groups, per, heads, kv, d: ops.attention_shared_workspace_bytes(groups, per, heads, kv, d, 1, 0)
    assert size(4096, 1, 1024, 1024, 128) == 0
    for groups, heads, kv, d in ((4095, 1024, 1024, 128), (4096, 1023, 1023, 128), (4096, 1024, 512, 128), (4096, 1024, 1024, 64)):
        assert attention(**{**most, "n_groups": groups, "n_heads": heads, "n_kv_heads": kv, "head_dim": d, "workspace_bytes": 0}) == SMALL
        assert size(groups, 1, heads, kv, d) > 0
