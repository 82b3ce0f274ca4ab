"""Items of the shared-prefix plan against the kernels' own check of an item, on the CPU.

The kernels skip an item that fails their bounds check, so every item of a plan has to pass
it; the plans here also have the forms that merge nothing (every tile writes the output).
"""
import numpy as np
import pytest
import torch

from prefix_util import CASES, exact, inputs, layout
from test_prefix_plan import ITEM, interpret

# tiles of more than 64 query rows, no partial rows at all
DIRECT = [
    ('wide_one', [0], [1], [128], [0], [128], True),
    ('wide_65', [1], [1], [65], [0], [65], True),
    ('wide_two', [100], [2], [100, 100], [0, 0], [100, 100], True),
    ('wide_sixteen', [50], [16], [200] * 16, [0] * 16, [200] * 16, True),
    ('wide_noncausal', [0], [2], [70, 128], [30, 5], None, False),
    ('wide_and_empty', [0], [3], [66, 0, 100], [0, 4, 0], [66, 0, 100], True),
    ('wide_prefix_only', [100], [3], [40, 40, 30], [0] * 3, None, False),
]


def accepted(it, total, slots):
    """``load_item``'s checks of an item's own words."""
    q0, nq, head, slot, _, nseg, dual = (int(v) for v in it[:7])
    two = nq > 64 or dual
    blocks = sum(-(-int(it[10 + 4 * s]) // 128) for s in range(nseg))
    return (1 <= nq <= 128 and 0 <= q0 <= total - nq and 0 <= head < 8 and 0 <= nseg <= 3
            and (slot == -1 if slot < 0 else slot + (2 if two else 1) <= slots)
            and (not dual or (nq <= 64 and slot >= 0 and blocks >= 2)))


@pytest.mark.parametrize('grid', [1, 148])
@pytest.mark.parametrize('case', CASES + DIRECT, ids=[c[0] for c in CASES + DIRECT])
def test_every_item_passes_the_kernels_check(pkg, case, grid):
    lay = layout(pkg, inputs(3, case), case, 'cpu', grid_limit=grid)
    plan = lay.plan.numpy().astype(np.int64)
    items = plan[plan[6]:plan[6] + plan[4] * ITEM].reshape(-1, ITEM)
    assert all(accepted(it, int(plan[2]), int(plan[8])) for it in items)


SMALL_DIRECT = [c for c in DIRECT if sum(c[3]) <= 300]


@pytest.mark.parametrize('case', SMALL_DIRECT, ids=[c[0] for c in SMALL_DIRECT])
def test_direct_plans_reproduce_attention(pkg, case):
    x = inputs(5, case)
    lay = layout(pkg, x, case, 'cpu', grid_limit=148)
    assert int(lay.head[8]) == 0 and lay.workspace_bytes == 0        # no partial rows
    got = interpret(lay.plan, x, case)
    ref, _, _ = exact(x, case)
    assert torch.isfinite(got).all() and (got - ref).abs().max() < 1e-12
