"""The operators together, as a decode uses them.

* ``speculative_greedy(controls=...)`` emits the target's own controlled greedy decode: the
  reference takes one token at a time from the same target and applies the penalties and
  biases in numpy.
* A verify round over completions of one prompt: shared-prefix attention, an LM head,
  controlled acceptance and the commit of the emitted tokens into the tables.
"""
import numpy as np
import pytest
import torch

import inputs as I
from gpu_util import dev, i32, status_clean
from prefix_util import SCALE, exact, inputs, layout
from test_gpu_greedy_round import build

pytestmark = pytest.mark.gpu

NEW = 20
PENALTIES = [(1.3, 0.2, 0.1), (1.0, 0.0, 0.0), (1.6, 0.0, 0.5), (1.0, 0.7, 0.0), (1.1, -0.1, 0.3), (2.0, 0.5, 0.5)]


def choose(logits, prompt, output, pen, bias):
    z = logits.astype(np.float32).copy()
    c = np.bincount(output, minlength=len(z)).astype(np.float32)
    seen = (np.bincount(prompt, minlength=len(z)) > 0) | (c > 0)
    rep, freq, pres = (np.float32(x) for x in pen)
    z = np.where(seen, np.where(z > 0, z / rep, z * rep), z)
    z = np.where(c > 0, (z - freq * c) - pres, z)
    for t, v in bias.items():
        z[t] = z[t] + np.float32(v)
    return int(z.argmax())


@pytest.mark.parametrize('graph', [False, True])
def test_speculative_greedy_with_controls_equals_controlled_decode(pkg, golden, graph):
    target, draft, prompts, _ = build(pkg, golden)
    vocab = I.TINY_TARGET['vocab_size']
    host = {r: p[0].cpu().numpy() for r, p in prompts.items()}
    bias = {r: {int(7 * i + 3): 0.5, int(11 * i + 5): -2.0} for i, r in enumerate(prompts)}
    controls = pkg.TokenControls(len(prompts), vocab, device=dev(), max_bias=2)
    for i, r in enumerate(prompts):
        pen = PENALTIES[i % len(PENALTIES)]
        controls.add_request(r, prompt=host[r], repetition=pen[0], frequency=pen[1], presence=pen[2], bias=bias[r])
    out, _rounds = pkg.speculative_greedy(target, draft, prompts, NEW, graph=graph, controls=controls)
    status_clean(pkg)
    # one token at a time, by request
    single, _, _, _ = build(pkg, golden)
    for i, r in enumerate(prompts):
        single.add_request(r)
        features = single.prefill({r: prompts[r]})
        tokens = []
        while True:
            logits = single.predict(features, last_only=True)[r].reshape(-1).float().cpu().numpy()
            tokens.append(choose(logits, host[r], np.array(tokens, dtype=np.int64), PENALTIES[i % len(PENALTIES)],
                                 bias[r]))
            if len(tokens) == NEW:
                break
            features = single.verify({r: torch.tensor([[tokens[-1]]], device=dev())})
            single.commit(features, {r: 1})
        assert out[r] == tokens, r
        want = np.bincount(tokens, minlength=vocab)
        assert (controls.counts[i, :vocab].cpu().numpy() == want).all()
    with pytest.raises(ValueError):
        pkg.speculative_greedy(target, draft, {}, 1, device_accept=False, controls=controls)


@pytest.mark.parametrize('vocab', [1000, 32000])
def test_round_over_one_prompt(pkg, vocab):
    case = ('round', [700], [6], [8, 8, 3, 1, 8, 5], [0, 20, 64, 130, 7, 1], [8, 8, 3, 1, 8, 5], True)
    n, r = sum(case[3]), len(case[3])
    x = inputs(81, case)
    to = lambda t: t.to(dev(), torch.bfloat16)  # noqa: E731
    g = np.random.Generator(np.random.PCG64(82))
    head = to(torch.from_numpy(g.standard_normal((vocab, 2048)).astype(np.float32) * 0.1))
    lay = layout(pkg, x, case, dev())
    controls = pkg.TokenControls(r, vocab, device=dev())
    outputs = [g.integers(0, 40, 10 + i) for i in range(r)]
    for i in range(r):
        controls.add_request(f'c{i}', prompt=np.arange(20), output=outputs[i], repetition=1.2, frequency=0.3,
                             presence=0.4)
    slots = controls.slot_index([f'c{i}' for i in range(r)])
    attended = pkg.B200SharedPrefixKernel(dev())(to(x['q']), to(x['a'][1]), to(x['a'][2]), lay, scale=SCALE,
                                                 prefix_key=to(x['p'][1]), prefix_value=to(x['p'][2]),
                                                 new_key=to(x['b'][1]), new_value=to(x['b'][2]))
    logits = torch.nn.functional.linear(attended.reshape(n, 2048), head)
    cu = np.concatenate([[0], np.cumsum(case[3])])
    words = (vocab + 31) // 32
    masks = torch.from_numpy(g.integers(-2 ** 31, 2 ** 31, (1, words)).astype(np.int32)).to(dev())
    index = i32([0 if i in range(cu[1], cu[2]) else -1 for i in range(n)])
    # proposals: what the controlled target would say for the first rows of a chunk, then noise
    tokens = torch.from_numpy(g.integers(0, vocab, n)).to(dev())
    args = dict(masks=masks, mask_index=index)
    for i in range(r):
        for j in range(1, min(case[3][i], 4)):
            pred = pkg.control_argmax(logits, controls, slots, cu_query=i32(cu), tokens=tokens, **args)
            tokens[cu[i] + j] = pred[cu[i] + j - 1].long()
    before = controls.counts.clone()
    pred, accepted, n_commit, emitted = pkg.greedy_accept(logits, tokens, i32(cu), (), None, controls=controls,
                                                          slots=slots, **args)
    controls.commit(slots, emitted, i32(cu), n_commit)
    torch.cuda.synchronize()
    status_clean(pkg)
    ref, weight, _ = exact(x, case)
    err = (attended.double().cpu() - ref).abs()
    assert (err <= 2.0 ** -8 * (weight + ref.abs()) + 2.0 ** -10 * weight).all()
    # the decisions, from the kernel's own logits
    z = logits.float().cpu().numpy()
    allowed = (masks[0].cpu().numpy()[np.arange(vocab) >> 5] >> (np.arange(vocab) & 31)) & 1
    for i in range(r):
        history = list(outputs[i])
        toks, preds = tokens[cu[i]:cu[i + 1]].tolist(), []
        for j in range(case[3][i]):
            if j:
                history.append(toks[j])
            row = z[cu[i] + j].copy()
            c = np.bincount(history, minlength=vocab).astype(np.float32)
            seen = (np.arange(vocab) < 20) | (c > 0)
            row = np.where(seen, np.where(row > 0, row / np.float32(1.2), row * np.float32(1.2)), row)
            row = np.where(c > 0, (row - np.float32(0.3) * c) - np.float32(0.4), row)
            if i == 1:
                row = np.where(allowed > 0, row, -np.inf)
            preds.append(int(row.argmax()))
        assert preds == pred[cu[i]:cu[i + 1]].tolist()
        want, k = [], 0
        while k + 1 < len(toks) and toks[k + 1] == preds[k]:
            want.append(preds[k])
            k += 1
        want.append(preds[k])
        assert int(accepted[i]) == k and emitted[cu[i]:cu[i] + len(want)].tolist() == want
        added = (controls.counts[i] - before[i])[:vocab].cpu().numpy()
        assert (added == np.bincount(want, minlength=vocab)).all()


def test_accept_without_an_allowed_token(pkg):
    """A mask that allows nothing ends the request's round without a token, and is flagged."""
    vocab = 100
    controls = pkg.TokenControls(2, vocab, device=dev())
    for n in 'ab':
        controls.add_request(n)
    logits = torch.zeros((6, vocab), device=dev())
    logits[torch.arange(6), torch.tensor([5, 6, 7, 8, 9, 3])] = 5.0
    tokens = torch.tensor([1, 5, 6, 1, 8, 9], device=dev())
    masks = torch.zeros((1, 4), dtype=torch.int32, device=dev())
    pred, accepted, n_commit, emitted = pkg.greedy_accept(
        logits, tokens, i32([0, 3, 6]), controls=controls, slots=controls.slot_index(['a', 'b']), masks=masks,
        mask_index=i32([-1, 0, -1, -1, -1, -1]))
    assert pred.tolist() == [5, -1, 7, 8, 9, 3]
    assert accepted.tolist() == [1, 2] and n_commit.tolist() == [1, 3]
    assert emitted.tolist() == [5, -1, -1, 8, 9, 3]
    assert pkg.read_device_status(clear=True) == 8
    with pytest.raises(ValueError):
        pkg.greedy_accept(logits, tokens, i32([0, 3, 6]), masks=masks, mask_index=i32([0] * 6))
