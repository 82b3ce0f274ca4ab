"""Shared-prefix attention whose tiles all write the output (no partial rows), with tiles of more
than 64 query rows. Error bounds as in ``test_gpu_prefix``."""
import pytest
import torch

from gpu_util import dev, status_clean
from prefix_util import inputs, layout
from test_gpu_prefix import check, run
from test_prefix_items import DIRECT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('case', DIRECT, ids=[c[0] for c in DIRECT])
def test_matches_definition(pkg, case, dtype):
    x = inputs(13, case)
    lay = layout(pkg, x, case, dev())
    assert int(lay.head[8]) == 0
    out = torch.full((sum(case[3]), 16, 128), float('nan'), dtype=dtype, device=dev())
    got = run(pkg, x, case, dtype, lay, out=out)
    torch.cuda.synchronize()
    status_clean(pkg)
    check(got, x, case, dtype)
