"""wh_attention_tree where numbers are at their ends."""
import numpy as np
import pytest

from tests import _tree
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


# 16 heads per KV head: a tile of 32 query rows is two nodes.  Workgroups take the 24 tiles of a KV head by one up to 1920
# rows, by two up to 5120, then by four.
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,ctx", [(300, 40), (300, 252), (5000, 40), (5000, 1000), (60000, 40), (60000, 1000)])
def test_infinite_v_under_rows_that_move_and_rows_that_do_not(gpu, rows, ctx, d):
    """Every second pair of nodes has scores that rise from key to key, so that its rows' maxima move in every tile, the
    others have queries of zero.  Infinities and NaN of the last cache rows and of the nodes, in the first elements, reach
    exactly the rows that see them, call after call."""
    n_tree, heads, kv = 48, 32, 2
    c = Case(1, n_tree, heads, kv, d, [ctx], room=rows - ctx - n_tree, shape="star", seed=rows + ctx)
    c.parents[0, 7] = -1  # roots of their own: they do not see node 0
    c.parents[0, 20:24] = -2
    u = np.zeros(d, np.float32)
    u[: d // 2] = 1
    step = _tree.rotate(u, ctx + 1, c.inv) / np.sqrt(d)
    c.kc[0, :ctx] = (np.linspace(0, 24, ctx)[:, None, None] * step).astype(np.float16)
    q, k, v = c.views()
    for t in range(n_tree):
        q[0, t] = 4 * u if t // 2 % 2 else 0
    c.vc[0, ctx - 1, 0, 0] = np.inf
    c.vc[0, ctx - 2, 1, 1] = np.nan
    v[0, 0, 0, 2] = -np.inf
    v[0, 3, 1, 3] = np.inf
    v[0, 30, 0, 3] = np.nan
    v[0, 47, 1, 0] = np.inf
    print(f"[case] infinite v under moving rows d {d} ctx {ctx} of {rows}", flush=True)
    want, bound, _, _ = c.expect()
    c.upload()
    for _ in range(8):
        c.launch()
        c.compare(f"infinite v d {d} ctx {ctx} of {rows}", c.results()[0], want, bound)
