"""Scores of extreme size, infinities and NaN in the shared-prefix attention.

Operands of 2^52 give scores of about -+2^106, exact in float32 (128 equal products): equal
keys share their weight, so a row returns the mean of its values, also where partial rows
are merged. Bound as in ``test_gpu_prefix``: 2^-8 (A + |o|) + 2^-10 A in bf16, which covers
float32 too (n <= 1700 terms add n 2^-24 A).
"""
import pytest
import torch

from gpu_util import dev, status_clean
from prefix_util import SCALE, exact, inputs
from test_gpu_prefix import run

pytestmark = pytest.mark.gpu

BIG = 2.0 ** 52
DTYPES = pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
# few rows; wide tiles; even and odd blocks on two tiles; prefix, own and new keys merged
PLANS = [('few', [300], [1], [3], [0], None, False), ('wide', [0], [2], [100, 70], [600, 9], None, False),
         ('dual', [1700], [1], [5], [0], None, False), ('merged', [500], [3], [1, 8, 2], [40, 0, 300], [1, 8, 2], True)]


def constant_scores(case, q_value, k_value):
    x = inputs(3, case)
    x['q'] = torch.full_like(x['q'], q_value)
    for n in 'pab':
        if n in x:
            starts, k, v = x[n]
            x[n] = (starts, torch.where(torch.isnan(k), k, torch.full_like(k, k_value)), v)
    return x


@DTYPES
@pytest.mark.parametrize('sign', [-1, 1])
@pytest.mark.parametrize('size', [2.0 ** 20, BIG])
@pytest.mark.parametrize('case', PLANS, ids=[c[0] for c in PLANS])
def test_equal_scores_of_any_size(pkg, case, size, sign, dtype):
    # an odd multiple of 2^-6 beside the power of two, so that scaled scores are no float32 numbers
    x = constant_scores(case, size * (1 + 2.0 ** -6), sign * size * (1 + 2.0 ** -6))
    got = run(pkg, x, case, dtype)
    torch.cuda.synchronize()
    status_clean(pkg)
    ref, weight, _ = exact(x, case)
    err = (got.double().cpu() - ref).abs()
    assert torch.isfinite(err).all()
    tol = 2.0 ** -8 * (weight + ref.abs()) + 2.0 ** -10 * weight
    assert (err <= tol).all(), float((err - tol).max())


@DTYPES
@pytest.mark.parametrize('case', PLANS, ids=[c[0] for c in PLANS])
def test_the_largest_of_extreme_scores_wins(pkg, case, dtype):
    """All scores below -2^105; one key a step of bf16 above the others takes all the weight."""
    x = constant_scores(case, BIG, -BIG * (1 + 2.0 ** -7))
    starts, k, v = x['p' if case[1][0] else 'a']
    at = starts[0] + 137 % max(case[1][0] or case[4][0], 1)
    k[at] = -BIG
    if case[0] == 'wide':                          # each request needs one
        k[starts[1] + 4] = -BIG
    got = run(pkg, x, case, dtype).double().cpu()
    torch.cuda.synchronize()
    status_clean(pkg)
    ref = exact(x, case)[0]
    assert torch.isfinite(got).all()
    assert ((got - ref).abs() <= 2.0 ** -8 * ref.abs()).all()


@DTYPES
@pytest.mark.parametrize('case', [('shared', [700], [3], [9, 30, 5], [0] * 3, None, False),
                                  ('wide', [700], [1], [100], [0], None, False)], ids=['shared', 'wide'])
def test_near_and_far_rows_share_a_tile(pkg, case, dtype):
    """Every third row's scores are 2^30 times the others': all its weight is on one key. The
    inputs keep the two largest scores of such a row further apart than float32 dots err
    (129 * 2^-24 |q| . |k| each) plus the 64 from which on the second weighs nothing."""
    x = inputs(9, case)
    x['q'][::3] *= 2.0 ** 30
    starts, k, v = x['p']
    k[starts[0] + 130:starts[0] + 300] *= 4             # the maximum grows from block to block
    keys = k[starts[0]:starts[0] + 700].double()
    q = x['q'][::3].double()
    s = torch.einsum('thd,khd->thk', q, keys.repeat_interleave(2, 1)) * SCALE
    a = torch.einsum('thd,khd->thk', q.abs(), keys.abs().repeat_interleave(2, 1)).amax(-1) * SCALE
    top = s.topk(2, -1).values
    assert (top[..., 0] - top[..., 1] > 2 * 129 * 2.0 ** -24 * a + 64).all()
    got = run(pkg, x, case, dtype)
    torch.cuda.synchronize()
    status_clean(pkg)
    ref, weight, _ = exact(x, case)
    err = (got.double().cpu() - ref).abs()
    tol = 2.0 ** -8 * (weight + ref.abs()) + 2.0 ** -10 * weight
    assert torch.isfinite(err).all() and (err <= tol).all(), float((err - tol).max())


@DTYPES
def test_nan_and_infinities_stay_in_their_rows(pkg, dtype):
    """NaN in a query row, in a key of one group, in a request's own and newest keys: NaN where
    the definition has it (a row that sees the key), numbers everywhere else."""
    case = ('nan', [200, 300], [2, 2], [3, 8, 2, 70], [130, 20, 0, 64], [3, 8, 2, 70], True)
    x = inputs(5, case)
    x['q'][1, 4] = float('nan')                     # row 1, head 4 of request 0
    for name, row, head in (('a', x['a'][0][1] + 7, 2), ('b', x['b'][0][1] + 5, 3), ('p', x['p'][0][1] + 11, 6)):
        x[name][1][row, head, 17] = float('nan')
    x['a'][2][x['a'][0][0] + 3, 5, 9] = float('inf')    # a value that rows of request 0 see: inf in that column
    got = run(pkg, x, case, dtype).double().cpu()
    torch.cuda.synchronize()
    status_clean(pkg)
    ref = exact(x, case)[0]
    assert torch.isnan(ref).any() and torch.isinf(ref).any() and torch.isfinite(ref).any()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fine = torch.isfinite(ref)
    assert ((got - ref)[fine].abs() <= 0.05).all()


@DTYPES
def test_nan_reaches_every_piece_of_a_split_row(pkg, dtype):
    """One NaN key in a chain cut into pieces: the rows are NaN whichever piece holds it."""
    case = ('split', [5000], [2], [1, 4], [10, 0], [1, 4], True)
    for at in (0, 2500, 4999):
        x = inputs(6, case)
        x['p'][1][x['p'][0][0] + at, 1] = float('nan')
        got = run(pkg, x, case, dtype)
        torch.cuda.synchronize()
        nan = torch.isnan(got).all(-1)
        assert nan[:, 2:4].all() and not torch.isnan(got[:, [0, 1] + list(range(4, 16))]).any()
    status_clean(pkg)
