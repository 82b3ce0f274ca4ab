"""Append to the paged 8-bit cache: codes and tails bit for bit, scales to their rounding."""
import pytest
import torch

import quant_util as U
from gpu_util import status_clean

pytestmark = pytest.mark.gpu

# name, new rows, context tokens, rows that are kept (None: all)
CASES = [
    ('one', [1], [0], None),
    ('fills', [1], [63], None),
    ('fills_exactly', [8, 64], [56, 0], None),
    ('round', [8] * 12, [53 + 3 * i for i in range(12)], [i % 9 for i in range(12)]),
    ('nothing', [4, 4], [63, 62], [0, 0]),
    ('prompt', [300, 64, 63], [0, 0, 0], None),
    ('chunk', [200, 129, 128], [40, 63, 1], [200, 129, 65]),
    ('empty', [0, 3, 0], [10, 62, 128], None),
]


def page_table(b, counts):
    """Table rows long enough for the blocks that get full, on pages of their own."""
    width = max((n + c) // U.PAGE for n, c in zip(b['contexts'], counts))
    table = torch.full((len(counts), max(width, 1)), -1, dtype=torch.int32)
    at = 0
    for i, (n, c) in enumerate(zip(b['contexts'], counts)):
        for k in range(n // U.PAGE, (n + c) // U.PAGE):
            table[i, k] = at
            at += 1
    b['table'] = table
    return at


@pytest.mark.parametrize('row_dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('dtype', U.CODES, ids=['int8', 'e4m3'])
@pytest.mark.parametrize('case', CASES, ids=[c[0] for c in CASES])
def test_append(pkg, case, dtype, row_dtype):
    _, rows, contexts, counts = case
    x, b = U.make(11, rows, contexts, dtype, row_dtype, layers=2, spare=20)
    page_table(b, counts or rows)
    pages, layout, t = U.to_gpu(pkg, x, b)
    pages.append(t['new_key'], t['new_value'], layout,
                 None if counts is None else torch.tensor(counts, dtype=torch.int32, device='cuda'))
    status_clean(pkg)
    want = U.append(x, b, counts or rows)
    for name in ('key', 'value', 'tail_key', 'tail_value'):
        got = getattr(pages, name).cpu().double()
        same = (got == want[name]) | (got.isnan() & want[name].isnan())
        assert bool(same.all()), f'{name}: {int((~same).sum())} differ'
    for name in ('key_scale', 'value_scale'):
        got, w = getattr(pages, name).cpu().double(), want[name]
        ok = ((got - w).abs() <= 2.0 ** -24 * w.abs()) | (got.isnan() & w.isnan())
        assert bool(ok.all()), name
