"""Mask rows of the logits controls: indices out of range."""
import pytest
import torch

from gpu_util import dev, i32, status_clean

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bad', [-5, -2, -2 ** 31, 1, 2 ** 31 - 1])
def test_each_mask_index_out_of_range_is_flagged(pkg, bad):
    vocab = 5000
    controls = pkg.TokenControls(1, vocab, device=dev())
    controls.add_request('a')
    slots, cu = controls.slot_index(['a']), i32([0, 3])
    x = torch.arange(3 * vocab, dtype=torch.float32, device=dev()).reshape(3, vocab)
    masks = torch.zeros((1, controls.words), dtype=torch.int32, device=dev())
    masks[0, 0] = 4
    for index, status in (([0, -1, 0], 0), ([0, bad, -1], 4)):
        kw = dict(cu_query=cu, masks=masks, mask_index=i32(index))
        y = pkg.control_logits(x, controls, slots, **kw)
        torch.cuda.synchronize()
        assert pkg.read_device_status(clear=True) == status
        assert torch.equal(y[1], x[1]) and y[0, 2] == x[0, 2] and torch.isneginf(y[0, 3])   # the row goes unmasked
        pred = pkg.control_argmax(x, controls, slots, **kw)
        assert pred.tolist()[:2] == [2, vocab - 1] and pkg.read_device_status(clear=True) == status
    status_clean(pkg)
