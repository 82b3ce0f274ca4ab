"""Attention over the paged 8-bit cache against float64."""
import pytest
import torch

import quant_util as U
from gpu_util import status_clean

pytestmark = pytest.mark.gpu


def check(pkg, x, b, row_dtype, layer=0):
    pages, layout, t = U.to_gpu(pkg, x, b)
    got = pkg.B200QuantizedKernel('cuda')(t['query'][layer], t['new_key'][layer], t['new_value'][layer], layout,
                                          scale=U.SCALE, pages=pages, layer=layer)
    status_clean(pkg)
    out, weight, size = U.attention(x, b, layer)
    err = (got.double().cpu() - out).abs()
    tol = U.attention_tolerance(out, weight, size, row_dtype)
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), f'{float((err - tol).max())} over, err {float(err.max())}'
    return got


@pytest.mark.parametrize('dtype', U.CODES, ids=['int8', 'e4m3'])
@pytest.mark.parametrize('case', U.CASES, ids=[c[0] for c in U.CASES])
def test_bf16(pkg, case, dtype):
    check(pkg, *U.make(5, case[1], case[2], dtype, torch.bfloat16), torch.bfloat16)


@pytest.mark.parametrize('dtype', U.CODES, ids=['int8', 'e4m3'])
@pytest.mark.parametrize('case', [c for c in U.CASES if c[0] not in ('long_decode', 'one_chunk')],
                         ids=[c[0] for c in U.CASES if c[0] not in ('long_decode', 'one_chunk')])
def test_float32(pkg, case, dtype):
    check(pkg, *U.make(6, case[1], case[2], dtype, torch.float32), torch.float32)


def test_layers_are_apart(pkg):
    x, b = U.make(7, [3, 1], [200, 77], torch.int8, torch.bfloat16, layers=3)
    for layer in range(3):
        check(pkg, x, b, torch.bfloat16, layer)
