"""Edges of the operators for drafted tokens and shared pages that the tests of
their forms (test_branches_gpu.py) leave out, against the definitions
(branches_ref.py)."""
import math

import pytest
import torch

from branches_ref import tree_ref
from paged_ref import make_cache
from test_branches_gpu import BF16, F16, F32, _close, _q, _trees, ints

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# attn_tree
# ---------------------------------------------------------------------------

# Rows per kv head and type: the kernels up to 8, up to 128 and above, the plain one.
FORMS = [(BF16, 4, 2, 3), (F16, 8, 1, 1), (BF16, 8, 2, 9), (F16, 32, 2, 8), (BF16, 16, 1, 20), (F16, 4, 1, 70), (F32, 8, 2, 9)]


@pytest.mark.parametrize("dtype,Hq,Hkv,S", FORMS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps,W", [(16, 7), (24, 5), (8, 27), (7, 17), (100, 3)])
def test_tree_lengths_behind_the_table(attn, ps, W, D, dtype, Hq, Hkv, S):
    # tokens behind the table's last are left out: the first sequences' lengths pass it by much, by fewer tokens than
    # are drafted, by as many and by one, the last ones' do not
    cap = W * ps
    lens = [cap + 300, 2 ** 31 - 1, cap + S // 2 + 1, cap + S, cap + 1, cap, max(S, cap // 2)]
    B = len(lens)
    k, v, table, _ = make_cache([cap] * B, Hkv, D, ps, dtype, poison=False)
    q, par, ln = _q(B, Hq, S, D, dtype), _trees(B, S), ints(lens)
    # what an earlier call leaves in shared memory may not count
    bad = torch.full_like(v, math.nan).cuda()
    attn.attn_tree(q.cuda(), (100 * k).cuda(), bad, table.cuda(), ints([cap] * B).cuda(), par.cuda())
    assert attn.check_status(0) == 0
    for tree in (par, None):
        out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), None if tree is None else tree.cuda())
        assert attn.check_status(0) == 8
        _close(out, tree_ref(q, k, v, table, ln, tree), cap, dtype)
