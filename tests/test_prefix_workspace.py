"""Workspace of the shared-prefix attention: slots as large as their tile's rows, none overlapping."""
import numpy as np
import pytest
import torch

from prefix_util import CASES, inputs, layout
from test_prefix_items import DIRECT
from test_prefix_plan import ITEM, RUN

DECODE = ('decode_300', [2048], [300], [1] * 300, [(13 * i) % 230 for i in range(300)], [1] * 300, True)


def pitch(nq):
    return 2 * min(nq, 64)


@pytest.mark.parametrize('case', CASES + DIRECT + [DECODE], ids=[c[0] for c in CASES + DIRECT + [DECODE]])
def test_slots_lie_side_by_side_and_the_merge_finds_them(pkg, case):
    lay = layout(pkg, inputs(3, case), case, 'cpu', grid_limit=148)
    plan = lay.plan.numpy().astype(np.int64)
    part_rows, parts_at = int(plan[21]), int(plan[22])
    assert lay.workspace_bytes == part_rows * 130 * 4
    used = np.zeros(part_rows, dtype=np.int64)
    where = {}                                    # slot -> (first workspace row, rows)
    for it in plan[plan[6]:plan[6] + plan[4] * ITEM].reshape(-1, ITEM):
        nq, slot, dual, at = int(it[1]), int(it[3]), int(it[6]), int(it[7])
        if slot < 0:
            continue
        for s in range(2 if dual or nq > 64 else 1):
            where[slot + s] = (at + s * pitch(nq), pitch(nq))
            used[at + s * pitch(nq):at + (s + 1) * pitch(nq)] += 1
    assert (used == 1).all() and len(where) == int(plan[8])
    n_runs = int(plan[9])
    runs = plan[plan[10]:plan[10] + n_runs * RUN].reshape(n_runs, RUN)
    parts = plan[parts_at:parts_at + 4 * n_runs].reshape(n_runs, 4)
    for run, part in zip(runs, parts):
        for c in range(int(run[2])):
            slot, pieces, mma, _ = (int(v) for v in run[4 + 4 * c:8 + 4 * c])
            at, rows = int(part[2 * c]), int(part[2 * c + 1])
            for n in range(pieces * 8 * (2 if mma == 3 else mma)):
                assert where[slot + n] == (at + n * rows, rows)


@pytest.mark.parametrize('requests,limit', [(128, 8e6), (1024, 40e6), (4096, 150e6)])
def test_one_row_requests_take_little(pkg, requests, limit):
    lay = pkg.SharedPrefixLayout.from_lengths([2048], [requests], [1] * requests, [512] * requests, [1] * requests,
                                              device='cpu', grid_limit=148)
    assert 0 < lay.workspace_bytes < limit


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_a_large_decode_batch_matches_the_definition(pkg, dtype):
    from test_gpu_prefix import check, run
    x = inputs(17, DECODE)
    got = run(pkg, x, DECODE, dtype)
    torch.cuda.synchronize()
    assert pkg.read_device_status(clear=True) == 0
    check(got, x, DECODE, dtype)
