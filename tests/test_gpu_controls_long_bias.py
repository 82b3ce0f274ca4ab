"""Bias lists of any length: thousands of entries of one chunk, duplicates in list order, allow-lists
of most of the vocabulary. Values equal the float32 steps bit for bit, as in
``test_gpu_controls``."""
import numpy as np
import pytest
import torch

from gpu_util import dev, i32, status_clean

pytestmark = pytest.mark.gpu


def setup(pkg, seed, vocab, ids, chunk=3, dtype=torch.float32):
    g = np.random.Generator(np.random.PCG64(seed))
    values = (g.standard_normal(len(ids)) * 5).astype(np.float32)
    controls = pkg.TokenControls(2, vocab, device=dev(), max_bias=len(ids))
    history = g.integers(0, vocab, 50)
    controls.add_request('a', output=history.tolist(), repetition=1.25, frequency=0.5, presence=0.125,
                         bias=(torch.from_numpy(ids), torch.from_numpy(values)))
    x = torch.from_numpy((g.standard_normal((chunk, vocab)) * 3).astype(np.float32)).to(dtype)
    counts = np.bincount(history, minlength=vocab)
    z = x.float().numpy()
    bias = np.zeros(vocab, np.float32)
    np.add.at(bias, ids, values)                          # unbuffered: in list order, float32 sums
    z = np.where(counts > 0, np.where(z > 0, z / np.float32(1.25), z * np.float32(1.25)), z)
    z = np.where(counts > 0, (z - np.float32(0.5) * counts.astype(np.float32)) - np.float32(0.125), z) + bias
    return controls, x.to(dev()), torch.from_numpy(z.astype(np.float32))


@pytest.mark.parametrize('vocab,entries', [(700, 511), (700, 512), (700, 513), (4096, 4096), (5001, 3000), (4100, 9000),
                                           (1, 700), (151936, 2000)])
def test_sums_in_list_order(pkg, vocab, entries):
    g = np.random.Generator(np.random.PCG64(entries))
    ids = g.permutation(vocab)[:entries] if entries <= vocab else g.integers(0, vocab, entries)
    if entries > 600:
        ids[300:600] = ids[:300]                          # duplicates that straddle the staged pieces
    controls, x, want = setup(pkg, vocab, vocab, ids)
    slots, cu = controls.slot_index(['a']), i32([0, len(x)])
    assert torch.equal(pkg.control_logits(x, controls, slots, cu_query=cu).cpu(), want)
    assert pkg.control_argmax(x, controls, slots, cu_query=cu).tolist() == want.argmax(-1).tolist()
    status_clean(pkg)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_an_allow_list_takes_milliseconds(pkg, dtype):
    """100,000 biases, 8 rows. (A walk over the list for each biased token of each row took 760 ms.)"""
    vocab = 151936
    ids = np.random.Generator(np.random.PCG64(1)).permutation(vocab)[:100_000]
    controls, x, want = setup(pkg, 2, vocab, ids, chunk=8, dtype=dtype)
    slots, cu = controls.slot_index(['a']), i32([0, 8])
    call = lambda: pkg.control_logits(x, controls, slots, cu_query=cu, out_dtype=torch.float32)  # noqa: E731
    assert torch.equal(call().cpu(), want)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    call()
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 10
    status_clean(pkg)
