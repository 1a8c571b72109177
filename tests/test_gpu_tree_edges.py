"""Calls of the tree operators at the edges of what their arguments may be, against
their definitions in 64 bits."""
import numpy as np
import pytest
import torch

from specdec import ops
from test_gpu_tree import Commit
from tree_ref import Case

pytestmark = pytest.mark.gpu


def check_scaled(case, scale):
    case.scale = scale
    out, spread, reach = case.reference()
    got = case.call(ops).cpu().double()
    live = ~out.isnan()
    off = (got - out).abs()[live]
    tol = case.tolerance(out, spread, abs(reach))[live]
    assert bool((off <= tol).all()), (float((off / tol).max()), float(off.max()))
    assert bool(got[live].isfinite().all())


@pytest.mark.parametrize("scale", [-0.125, -0.01, 0.0, -0.0, 1e-45, 1e-30, 1.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,nodes,bs", [(4, 4, 9, 16), (4, 2, 12, 16), (8, 2, 40, 16), (8, 1, 70, 16), (4, 2, 9, 3)])
def test_scales_that_are_not_positive(heads, kv, nodes, bs, dtype, scale):
    """Nodes that a query does not see stay hidden whatever sign the scores take; a
    scale of 0 is the mean of what is seen.  One or two tiles of query rows, many that
    share their keys, and blocks that the tiles do not take."""
    check_scaled(Case(nodes, [70, 0, 700], nodes, heads, kv, bs=bs, dtype=dtype), scale)


@pytest.mark.parametrize("room", [1, 2, 4, 31, 32, 33, 100])
def test_commit_goes_on_to_its_room_and_no_further(room):
    """Chains of 40 nodes whose tokens are all as sampled: the path takes every slot
    that it may, and every node where there are more."""
    case = Commit(room, [3, 30, 7], 40, room=room, vocab=1)
    case.parents = (torch.arange(40, dtype=torch.int32) - 1).expand(3, 40).contiguous()
    verdict, path, _, _ = case.call()
    n = min(room, 40)
    assert verdict[0].tolist() == [n - 1] * 3
    assert path.cpu().tolist() == [list(range(n)) + [-1] * (40 - n)] * 3
    case.check()
