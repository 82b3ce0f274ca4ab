"""Logits controls in front of the stochastic acceptance: penalised, biased and masked target rows
sampled under the float64 law, and masks that allow nothing, which sampling cannot see."""
import numpy as np
import pytest
import torch

from gpu_util import dev, i32, status_clean
from test_gpu_controls import call_args, make, masks_for, steps

pytestmark = pytest.mark.gpu

LOW = torch.finfo(torch.float32).min


@pytest.mark.parametrize('vocab', [1000, 5001])
def test_one_row_draws_follow_the_controlled_law(pkg, vocab):
    """Requests without proposals draw one token each: the first whose float64 cumulative
    probability exceeds the uniform (uniforms lie 1e-9 off every border)."""
    r, temperature = 64, 0.7
    controls, reqs, logits, tokens = make(pkg, 3, vocab, [1] * r, bias=5)
    masks, index = masks_for(5, vocab, r)
    slots = controls.slot_index([f'r{i}' for i in range(r)])
    z = pkg.control_logits(torch.from_numpy(logits).to(dev()), controls, slots, mask_value=LOW, flag_empty=True,
                           masks=torch.from_numpy(masks).to(dev()), mask_index=torch.from_numpy(index).to(dev()))
    want, _, allow = steps(reqs, logits, tokens, [1] * r, masks, index, np.float32, mask_value=LOW)
    assert np.array_equal(z.cpu().numpy(), want)
    p = np.exp((want.astype(np.float64) - want.max(-1, keepdims=True).astype(np.float64)) / temperature)
    cdf = np.cumsum(p / p.sum(-1, keepdims=True), -1)
    u = np.random.Generator(np.random.PCG64(7)).random((r, 1))
    assert np.abs(cdf - u).min() > 1e-9
    emitted, result = pkg.stochastic_accept(
        z, torch.empty(0, dtype=torch.long, device=dev()), torch.empty((0, vocab), dtype=torch.float64, device=dev()),
        i32([0] * (r + 1)), temperature, torch.from_numpy(u).to(dev()), i32([4] * r))
    status_clean(pkg)
    got = emitted[:, 0].cpu().numpy()
    assert (result[:, 6] == 0).all() and (got == (cdf > u).argmax(-1)).all()
    assert allow[np.arange(r), got].all()


def test_proposals_of_a_round_are_judged_by_the_controlled_rows(pkg):
    """Chunks with proposals: a forbidden proposal is never accepted, an allowed one with all the
    controlled weight always is, and the tables count what was emitted."""
    vocab, temperature = 3000, 1.0
    controls = pkg.TokenControls(2, vocab, device=dev())
    for n in 'ab':
        controls.add_request(n, output=[7], frequency=20.0)
    slots, cu_rows = controls.slot_index(['a', 'b']), i32([0, 3, 6])
    chunk = torch.tensor([7, 7, 8, 7, 9, 10], device=dev())     # anchor, two proposals
    x = torch.zeros((6, vocab), device=dev())
    x[:, 7] = 60.0                                              # 60 - 20 count: 40, then 20 behind a 7
    x[0, 8], x[1, 8], x[3, 9] = 30.0, 50.0, 70.0
    masks = torch.full((2, controls.words), -1, dtype=torch.int32, device=dev())
    masks[1, 0] &= ~(1 << 10)                                   # 10 is forbidden in row 4
    index = i32([0, 0, 0, 0, 1, 0])
    x[4, 10] = 90.0
    z = pkg.control_logits(x, controls, slots, cu_query=cu_rows, tokens=chunk, masks=masks, mask_index=index,
                           mask_value=LOW, flag_empty=True)
    laws = torch.zeros((4, vocab), dtype=torch.float64, device=dev())
    proposals = torch.tensor([7, 8, 9, 10], device=dev())
    laws[torch.arange(4, device=dev()), proposals] = 1.0
    emitted, result = pkg.stochastic_accept(z, proposals, laws, i32([0, 2, 4]), temperature,
                                            torch.full((2, 3), 0.5, dtype=torch.float64, device=dev()), i32([8, 8]))
    status_clean(pkg)
    # a: 7 at 40, then 8 at 50 over 7 at 20; both taken, then a bonus (7: 60 - 40 = 20 over 0s, all its weight)
    assert emitted[0].tolist() == [7, 8, 7] and result[0, :2].tolist() == [3, 2]
    # b: 9 taken; 10 is forbidden: replaced by 7 (60 - 20 = 40)
    assert emitted[1].tolist()[:2] == [9, 7] and result[1, :3].tolist() == [2, 1, 1]
    controls.commit(slots, emitted.reshape(-1), i32([0, 3, 6]), result[:, 0].contiguous())
    status_clean(pkg)
    assert controls.counts[0, 7] == 3 and controls.counts[0, 8] == 1
    assert controls.counts[1, 7] == 2 and controls.counts[1, 9] == 1 and controls.counts[1, 10] == 0


@pytest.mark.parametrize('vocab', [1, 31, 32, 33, 1000, 16384, 50257, 151936])
def test_empty_masks_are_flagged_on_request(pkg, vocab):
    controls = pkg.TokenControls(3, vocab, device=dev())
    for n in 'abc':
        controls.add_request(n)
    slots = controls.slot_index(['a', 'b', 'c'])
    x = torch.zeros((14, vocab), device=dev())
    cu = i32([1, 11, 11, 12])                                   # rows 0, 12 and 13 belong to no request
    masks = torch.zeros((4, controls.words), dtype=torch.int32, device=dev())
    masks[1, (vocab - 1) // 32] = 1 << ((vocab - 1) % 32) if (vocab - 1) % 32 < 31 else -2 ** 31
    masks[2, 0] = 1
    if vocab % 32:                                              # bits past the vocabulary allow nothing
        masks[3, -1] = -2 ** 31 if vocab % 32 == 31 else ~((1 << vocab % 32) - 1)
    call = lambda index, **kw: pkg.control_logits(x, controls, slots, cu_query=cu, masks=masks,  # noqa: E731
                                                  mask_index=i32(index), mask_value=LOW, **kw)
    good = [0] + [1, 2, -1] * 3 + [1, 2, 0, 0]                  # empty masks outside the requests
    call(good, flag_empty=True)
    status_clean(pkg)
    for row, mask in ((1, 0), (10, 0), (11, 3), (4, 3)):
        bad = list(good)
        bad[row] = mask
        y = call(bad)                                           # only on request
        assert (y[row] == LOW).all()
        status_clean(pkg)
        assert torch.equal(call(bad, flag_empty=True)[1:12], y[1:12])
        assert pkg.read_device_status(clear=True) == 8
    bad = list(good)
    bad[5] = 9                                                  # an index past the masks: refused, not empty
    call(bad, flag_empty=True)
    assert pkg.read_device_status(clear=True) == 4
    assert torch.equal(pkg.control_logits(x, controls, slots, cu_query=cu, flag_empty=True)[1:12], x[1:12])
    status_clean(pkg)
    one = pkg.control_logits(x[:3], controls, slots, masks=masks, mask_index=i32([1, -1, 0]), flag_empty=True)
    assert pkg.read_device_status(clear=True) == 8 and torch.isneginf(one[2]).all()


def test_native_refusals(pkg):
    import ctypes
    f, lib = ctypes.c_void_p(4096), pkg.load_library()
    ok = [f, 4, 1, f, 2, 100, None, 2, None]
    for at, v in ((0, None), (1, 3), (2, 0), (3, None), (4, 1), (5, 0), (5, 2 ** 30 + 1), (7, 0)):
        bad = list(ok)
        bad[at] = v
        assert lib.dspark_control_check_masks(*bad) == 1
