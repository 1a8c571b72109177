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
