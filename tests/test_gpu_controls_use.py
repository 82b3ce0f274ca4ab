"""Uses of the logits controls that the other tests do not make: refusals that leave a decode loop as
it was, side streams, several captured graphs at once, one slot in several places."""
import numpy as np
import pytest
import torch

import inputs as I
from gpu_util import dev, i32, status_clean
from test_gpu_controls import call_args, make, masks_for, steps
from test_gpu_greedy_round import build

pytestmark = pytest.mark.gpu


def test_a_refused_loop_leaves_its_requests_free(pkg, golden):
    """Controls of another vocabulary are refused before the target or the draft takes a request."""
    target, draft, prompts, _ = build(pkg, golden)
    vocab = I.TINY_TARGET['vocab_size']
    for wrong in (vocab - 1, vocab + 8):
        controls = pkg.TokenControls(len(prompts), wrong, device=dev())
        for r in prompts:
            controls.add_request(r)
        with pytest.raises(ValueError):
            pkg.speculative_greedy(target, draft, prompts, 4, controls=controls)
    controls = pkg.TokenControls(len(prompts), vocab, device=dev())
    for r in prompts:
        controls.add_request(r)
    out, _ = pkg.speculative_greedy(target, draft, prompts, 4, controls=controls)
    assert all(len(v) == 4 for v in out.values())
    status_clean(pkg)


@pytest.mark.parametrize('vocab', [4101, 40000])
def test_captured_calls_at_once_equal_eager_ones(pkg, vocab):
    """Two graphs of the argmax and two of in-place logits, replayed at once on four streams over one
    set of tables."""
    chunks = [8, 1, 5, 3]
    controls, reqs, logits, tokens = make(pkg, 21, vocab, chunks, bias=30)
    masks, index = masks_for(6, vocab, sum(chunks))
    args = call_args(controls, chunks, tokens, masks, index)
    slots = controls.slot_index([f'r{i}' for i in range(4)])
    xs = [torch.from_numpy(logits).to(dev(), dtype) * f for dtype in (torch.bfloat16, torch.float32) for f in (1, -1)]
    want_top = [pkg.control_argmax(x, controls, slots, **args).clone() for x in xs]
    want = [pkg.control_logits(x, controls, slots, **args).clone() for x in xs]
    for k in range(0, 4, 2):
        buffers = [torch.zeros_like(xs[k]) for _ in range(4)]
        graphs, tops, streams = [], [], [torch.cuda.Stream() for _ in range(4)]
        torch.cuda.synchronize()
        for i, (b, s) in enumerate(zip(buffers, streams)):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                tops.append(pkg.control_argmax(b, controls, slots, **args) if i < 2
                            else pkg.control_logits(b, controls, slots, out=b, **args))
            graphs.append(graph)
        for _ in range(3):
            for i, b in enumerate(buffers):
                b.copy_(xs[k + i % 2])
            torch.cuda.synchronize()
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for i in range(2):
                assert torch.equal(tops[i], want_top[k + i]) and torch.equal(buffers[2 + i], want[k + i])
        del graphs
    status_clean(pkg)


def test_one_slot_for_several_requests_and_reordered_rows(pkg):
    """Beams of one request: the slot in several places, each with its own chunk."""
    vocab, chunks = 3000, [4, 2, 4]
    controls, reqs, logits, tokens = make(pkg, 31, vocab, [10], bias=6)
    slots = controls.slot_index(['r0', 'r0', 'r0'])
    args = call_args(controls, chunks, tokens, None, None)
    got = pkg.control_logits(torch.from_numpy(logits).to(dev()), controls, slots, **args).cpu().numpy()
    want = steps(reqs * 3, logits, tokens, chunks, None, None, np.float32)[0]
    assert np.array_equal(got, want)
    status_clean(pkg)


def test_every_token_proposed_seen_and_biased(pkg):
    """A vocabulary of one chunk with all of its tokens in the list, and a long chunk that proposes
    the same tokens again and again."""
    vocab, n = 4096, 70
    controls = pkg.TokenControls(1, vocab, device=dev(), max_bias=vocab)
    values = torch.linspace(-3, 3, vocab)
    controls.add_request('a', prompt=torch.arange(vocab), output=[5, 5, 9], repetition=1.5, frequency=0.25,
                         presence=0.5, bias=(torch.arange(vocab), values))
    g = np.random.Generator(np.random.PCG64(3))
    x = (g.standard_normal((n, vocab)) * 4).astype(np.float32)
    tokens = np.array([5, 9, 4095, 0][:4] * n)[:n].astype(np.int64)
    reqs = [dict(prompt=np.arange(vocab), output=np.array([5, 5, 9]), pen=np.float32((1.5, 0.25, 0.5)),
                 ids=np.arange(vocab), val=values.numpy())]
    args = call_args(controls, [n], tokens, None, None)
    slots = controls.slot_index(['a'])
    want = steps(reqs, x, tokens, [n], None, None, np.float32)[0]
    xd = torch.from_numpy(x).to(dev())
    assert np.array_equal(pkg.control_logits(xd, controls, slots, **args).cpu().numpy(), want)
    assert (pkg.control_argmax(xd, controls, slots, **args).cpu().numpy() == want.argmax(-1)).all()
    status_clean(pkg)


def test_a_failed_request_takes_no_slot(pkg, monkeypatch):
    controls = pkg.TokenControls(1, 100, device=dev())
    with monkeypatch.context() as m:
        m.setattr(pkg.TokenControls, '_add', lambda self, *a: (_ for _ in ()).throw(RuntimeError('native failure')))
        with pytest.raises(RuntimeError):
            controls.add_request('a', output=[3])
    assert controls.add_request('a', output=[4]) == 0
    assert int(controls.counts[0, 3]) == 0 and int(controls.counts[0, 4]) == 1
    status_clean(pkg)
