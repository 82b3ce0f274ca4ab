"""Outputs and workspaces of the shared-prefix attention that overlap its inputs are refused on the
host, before any device work (the addresses here are never read)."""
import ctypes

import pytest
import torch

# one query row (bf16: 4096 bytes) behind 4 prefix rows and one new one (2048 bytes each)
Q, PK, PV, BK, BV, OUT, WS = (1 << 20) * torch.arange(1, 8)


@pytest.mark.parametrize('kw', [dict(out=Q + 16), dict(out=Q - 4080), dict(out=PK), dict(out=PV + 3 * 2048),
                                dict(out=PV - 4080), dict(out=BK), dict(out=BV + 2032), dict(out=PK + 2048, off=1),
                                dict(ws=Q), dict(ws=OUT + 4080), dict(ws=BV - 64), dict(ws=PK + 16)],
                         ids=lambda kw: '-'.join(f'{k}{int(v) % (1 << 20)}' for k, v in kw.items()))
def test_overlaps_are_refused(pkg, kw):
    lay = pkg.SharedPrefixLayout.from_lengths([4], [2], [1, 0], [0, 0], [1, 0], device='cpu', grid_limit=4)
    assert lay.workspace_bytes > 0
    p = lambda x: ctypes.c_void_p(int(x))  # noqa: E731
    a = dict(out=OUT, ws=WS, off=0) | kw
    status = pkg.load_library().dspark_prefix_attn(
        p(Q), 1, p(PK), p(PV), 8, int(a['off']), None, None, 0, 0, p(BK), p(BV), 1, 0, lay.head.data_ptr(),
        p(1 << 30), pkg.SCALE, 0, p(a['out']), p(a['ws']), lay.workspace_bytes, None)
    assert status == 1


@pytest.mark.gpu
def test_overlapping_tensors_raise(pkg):
    dev = torch.device('cuda', 0)
    lay = pkg.SharedPrefixLayout.from_lengths([9], [2], [2, 3], [4, 1], [2, 3], device=dev)
    buf = torch.zeros(12 * 2048, dtype=torch.bfloat16, device=dev)
    q, shifted = buf[:5 * 2048].view(5, 16, 128), buf[2048:6 * 2048].view(5, 16, 128)
    rows = lambda n: torch.zeros((n, 8, 128), dtype=torch.bfloat16, device=dev)  # noqa: E731
    own = buf[6 * 2048:].view(12, 8, 128)
    kernel = pkg.B200SharedPrefixKernel(dev)
    call = lambda out: kernel(q, own, rows(12), lay, scale=pkg.SCALE, prefix_key=rows(9), prefix_value=rows(9),  # noqa: E731
                              new_key=rows(5), new_value=rows(5), out=out)
    for out in (shifted, buf[5 * 2048:10 * 2048].view(5, 16, 128)):
        with pytest.raises(ValueError):
            call(out)
    assert call(q) is q                            # the query itself
    torch.cuda.synchronize()
    assert pkg.read_device_status(clear=True) == 0
