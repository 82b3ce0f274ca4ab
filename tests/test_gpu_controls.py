"""GPU parity of the logits controls with their definition.

Reference: the steps in float64 from the same inputs. Each of the up to five float32
steps rounds by at most 2^-24 of a value no larger than M = |logit| max(rep, 1/rep) +
|freq| c + |pres| + sum |bias|, so |z - exact| <= 6 * 2^-24 M (the sixth for the biases'
own sum), and a bf16 output adds 2^-8 |z|. ``control_argmax`` must return an index whose
exact value is within that bound of the row's largest, and exactly the lowest index of
the maximum of the float32 steps done by torch on the CPU.
"""
import numpy as np
import pytest
import torch

from gpu_util import dev, i32, status_clean

pytestmark = pytest.mark.gpu


def make(pkg, seed, vocab, chunks, *, bias=0, prompt=40, output=60, dup_bias=False):
    g = np.random.Generator(np.random.PCG64(seed))
    r, n = len(chunks), sum(chunks)
    controls = pkg.TokenControls(r + 2, vocab, device=dev(), max_bias=bias + 3)
    reqs = []
    for i in range(r):
        hot = g.integers(0, vocab, 12)
        p = np.concatenate([g.integers(0, vocab, prompt), hot[:3]])
        o = np.concatenate([g.choice(hot, output), g.integers(0, vocab, 5)])
        pen = (float(g.uniform(1.05, 1.6)), float(g.uniform(-.2, .9)), float(g.uniform(0, .9)))
        ids = g.integers(0, vocab, bias)
        if dup_bias and bias >= 4:
            ids[:3] = ids[3]
        val = (g.standard_normal(bias) * 5).astype(np.float32)
        reqs.append(dict(prompt=p, output=o, pen=np.float32(pen), ids=ids, val=val))
        controls.add_request(f'r{i}', prompt=torch.from_numpy(p), output=o.tolist(), repetition=pen[0],
                             frequency=pen[1], presence=pen[2],
                             bias=(torch.from_numpy(ids), torch.from_numpy(val)) if bias else None)
    logits = (g.standard_normal((n, vocab)) * 3).astype(np.float32)
    tokens = g.integers(0, vocab, n)
    at = 0
    for i, q in enumerate(chunks):                     # proposals repeat each other and the history
        for j in range(q):
            logits[at + j, reqs[i]['output'][0]] += 8
            tokens[at + j] = reqs[i]['output'][j % 3] if j % 2 else tokens[at + j]
        at += q
    return controls, reqs, logits, tokens


def masks_for(seed, vocab, n, empty_row=None):
    g = np.random.Generator(np.random.PCG64(seed))
    words = (vocab + 31) // 32
    m = np.where(g.random((n, words)) < 0.3, g.integers(-2 ** 31, 2 ** 31, (n, words)), 0).astype(np.int32)
    m[:, 0] |= 2 if vocab > 1 else 1
    index = np.array([k if k % 3 != 1 else -1 for k in range(n)], dtype=np.int32)
    if empty_row is not None:
        m[empty_row] = 0
        index[empty_row] = empty_row
    return m, index


def steps(reqs, logits, tokens, chunks, masks, index, dtype, mask_value=-np.inf):
    """(values, magnitude M, allowed) of the definition in ``dtype``, one rounding per step."""
    n, vocab = logits.shape
    out, mag, allow = np.empty((n, vocab), dtype), np.empty((n, vocab)), np.ones((n, vocab), bool)
    row = 0
    for x, q in zip(reqs, chunks):
        c = np.bincount(x['output'], minlength=vocab).astype(np.int64)
        prompt = np.bincount(x['prompt'], minlength=vocab) > 0
        b = np.zeros(vocab, dtype)
        ab = np.zeros(vocab)
        for t, v in zip(x['ids'], x['val']):
            b[t] = b[t] + dtype(v)
            ab[t] += abs(float(v))
        rep, freq, pres = (dtype(v) for v in x['pen'])
        for j in range(q):
            if j:
                c[tokens[row]] += 1
            z = logits[row].astype(dtype)
            with np.errstate(all='ignore'):
                z = np.where(prompt | (c > 0), np.where(z > 0, z / rep, z * rep), z)
                z = np.where(c > 0, (z - freq * c.astype(dtype)) - pres, z)
                z = z + b
            if masks is not None and index[row] >= 0:
                bits = (masks[index[row]][np.arange(vocab) >> 5] >> (np.arange(vocab) & 31)) & 1
                allow[row] = bits != 0
                z = np.where(allow[row], z, dtype(mask_value))
            out[row] = z
            mag[row] = np.abs(logits[row]) * max(float(rep), 1.0) + abs(float(freq)) * c + abs(float(pres)) + ab
            row += 1
    return out, mag, allow


def call_args(controls, chunks, tokens, masks, index):
    cu = np.concatenate([[0], np.cumsum(chunks)])
    return dict(cu_query=i32(cu), tokens=torch.from_numpy(tokens).to(dev()),
                masks=None if masks is None else torch.from_numpy(masks).to(dev()),
                mask_index=None if masks is None else torch.from_numpy(index).to(dev()))


CASES = [
    # vocab, chunks, biases, masked
    (1, [1], 0, False), (7, [3, 1], 2, True), (64, [1, 1, 1], 0, False), (1000, [8, 1, 5], 9, True),
    (2048, [2, 17], 300, True), (2049, [7, 7], 5, False), (4103, [1, 40], 0, True), (50257, [5, 3], 40, True),
    (151936, [8, 2], 16, True),
]


@pytest.mark.parametrize('dtypes', [('bf16', 'bf16'), ('bf16', 'fp32'), ('fp32', 'fp32')], ids='-'.join)
@pytest.mark.parametrize('vocab,chunks,bias,masked', CASES)
def test_logits_match_definition(pkg, vocab, chunks, bias, masked, dtypes):
    tin, tout = ({'bf16': torch.bfloat16, 'fp32': torch.float32}[d] for d in dtypes)
    controls, reqs, logits, tokens = make(pkg, vocab, vocab, chunks, bias=bias, dup_bias=True)
    masks, index = masks_for(vocab + 1, vocab, sum(chunks)) if masked else (None, None)
    x = torch.from_numpy(logits).to(dev(), tin)
    logits = x.float().cpu().numpy()
    args = call_args(controls, chunks, tokens, masks, index)
    slots = controls.slot_index([f'r{i}' for i in range(len(chunks))])
    got = pkg.control_logits(x, controls, slots, out_dtype=tout, **args)
    torch.cuda.synchronize()
    status_clean(pkg)
    want, mag, allow = steps(reqs, logits, tokens, chunks, masks, index, np.float64)
    y = got.double().cpu().numpy()
    assert got.dtype == tout and (np.isneginf(y) == ~allow).all()
    err = np.abs(np.where(allow, y - np.where(allow, want, 0), 0))
    tol = 6 * 2.0 ** -24 * mag + (2.0 ** -8 * np.abs(np.where(allow, want, 0)) if tout == torch.bfloat16 else 0)
    # bf16: half a step of the float32 value, itself within the float32 bound
    assert (err <= tol * (1 + 2.0 ** -7)).all(), float((err - tol).max())
    same = steps(reqs, logits, tokens, chunks, masks, index, np.float32)[0]
    assert np.array_equal(torch.from_numpy(same).to(tout).float().numpy(), got.float().cpu().numpy())


@pytest.mark.parametrize('tin', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('vocab,chunks,bias,masked', CASES)
def test_argmax_matches_definition(pkg, vocab, chunks, bias, masked, tin):
    controls, reqs, logits, tokens = make(pkg, vocab + 5, vocab, chunks, bias=bias)
    masks, index = masks_for(vocab + 2, vocab, sum(chunks)) if masked else (None, None)
    x = torch.from_numpy(logits).to(dev(), tin)
    logits = x.float().cpu().numpy()
    args = call_args(controls, chunks, tokens, masks, index)
    slots = controls.slot_index([f'r{i}' for i in range(len(chunks))])
    got = pkg.control_argmax(x, controls, slots, **args).cpu().numpy()
    status_clean(pkg)
    same, mag, allow = steps(reqs, logits, tokens, chunks, masks, index, np.float32)
    same = np.where(allow, same, -np.inf)
    assert (got == same.argmax(-1)).all()
    want = np.where(allow, steps(reqs, logits, tokens, chunks, masks, index, np.float64)[0], -np.inf)
    rows = np.arange(len(got))
    assert (want.max(-1) - want[rows, got] <= 12 * 2.0 ** -24 * mag.max(-1)).all()


def test_decode_rows_without_chunks(pkg):
    """No cu_query: one row per request, tables alone; requests in any order of slots."""
    controls, reqs, logits, tokens = make(pkg, 3, 500, [1, 1, 1])
    x = torch.from_numpy(logits).to(dev())
    order = [2, 0, 1]
    got = pkg.control_logits(x[order].contiguous(), controls, controls.slot_index([f'r{i}' for i in order]))
    want = steps(reqs, logits, tokens, [1, 1, 1], None, None, np.float32)[0]
    assert np.array_equal(got.cpu().numpy(), want[order])
    status_clean(pkg)


@pytest.mark.parametrize('vocab', [1000, 1024])
def test_ties_nan_infinities_and_empty_masks(pkg, vocab):
    controls = pkg.TokenControls(1, vocab, device=dev())
    controls.add_request('a', output=[3, 3, 5], repetition=2.0, frequency=0.5, presence=0.25)
    slots = controls.slot_index(['a'])
    x = torch.zeros((8, vocab), device=dev())
    x[0, 900] = 9.0
    x[0, 400] = 9.0                               # tie: the lower index
    x[1] = float('-inf')                          # allowed infinities only: the first token
    x[2, 700] = float('nan')                      # NaN is largest
    x[2, 10] = float('inf')
    x[3, 700] = float('nan')                      # masked NaN is not seen
    x[3, 10] = 1.0
    x[4, 3], x[4, 5], x[4, 7] = 10.0, 10.0, 5.0   # 10/2 - 1 - .25, 10/2 - .5 - .25, 5
    x[5, :] = -1.0
    x[5, 3] = float('inf')                        # penalised infinity stays infinite
    x[6, :] = -0.0
    x[6, 900] = 0.0                               # -0 equals +0: the first
    words = (vocab + 31) // 32
    masks = torch.zeros((2, words), dtype=torch.int32, device=dev())
    masks[0, 0] = 1 << 10
    index = i32([-1, -1, -1, 0, -1, -1, -1, 1])   # row 7: nothing allowed
    cu = i32([0, 8])
    pred = pkg.control_argmax(x, controls, slots, cu_query=cu, masks=masks, mask_index=index)
    assert pred.tolist() == [400, 0, 700, 10, 7, 3, 0, -1]
    assert pkg.read_device_status(clear=True) == 8
    y = pkg.control_logits(x, controls, slots, cu_query=cu, masks=masks, mask_index=index)
    assert torch.isneginf(y[7]).all() and not torch.isnan(y[3]).any() and int(torch.isfinite(y[3]).sum()) == 1
    assert y[4, 3] == 3.75 and y[4, 5] == 4.25 and torch.isposinf(y[5, 3]) and torch.isnan(y[2, 700])
    low = torch.finfo(torch.float32).min
    z = pkg.control_logits(x, controls, slots, cu_query=cu, masks=masks, mask_index=index, mask_value=low)
    assert (z[7] == low).all() and int((z[3] == low).sum()) == vocab - 1
    status_clean(pkg)


@pytest.mark.parametrize('vocab', [1001, 2056])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_strided_in_place_and_untouched_rows(pkg, vocab, dtype):
    chunks = [3, 2]
    controls, reqs, logits, tokens = make(pkg, 9, vocab, chunks, bias=4)
    buf = torch.full((8, vocab + 8), 5.0, dtype=dtype, device=dev())
    rows = buf[1:6, :vocab]
    rows.copy_(torch.from_numpy(logits))
    plain = rows.contiguous()
    masks, index = masks_for(4, vocab, 5)
    args = call_args(controls, chunks, tokens, masks, index)
    slots = controls.slot_index(['r0', 'r1'])
    want = pkg.control_logits(plain, controls, slots, **args)
    got = pkg.control_logits(rows, controls, slots, out=rows, **args)
    assert got.data_ptr() == rows.data_ptr() and torch.equal(got, want)
    assert (buf[0] == 5).all() and (buf[6:] == 5).all() and (buf[:, vocab:] == 5).all()
    # rows no request owns are neither written nor read
    part = dict(args, cu_query=i32([1, 3, 4]))
    out = torch.full((5, vocab), 7.0, dtype=dtype, device=dev())
    pkg.control_logits(plain, controls, slots, out=out, **part)
    assert (out[0] == 7).all() and (out[4] == 7).all() and not (out[1:4] == 7).all(-1).any()
    status_clean(pkg)


def test_division_equals_torch(pkg):
    """Every token seen: positive logits are divided by the repetition penalty, correctly rounded,
    over penalties and logits of many magnitudes (the vocabulary's tail takes other paths)."""
    r, vocab = 48, 8192 + 72
    g = torch.Generator(device='cpu').manual_seed(5)
    controls = pkg.TokenControls(r, vocab, device=dev())
    reps = torch.cat([1 + torch.rand(20, generator=g), torch.rand(8, generator=g) * 10 + 1e-3,
                      2.0 ** torch.randint(-60, 60, (8,), generator=g) * (1 + torch.rand(8, generator=g)),
                      torch.nextafter(2.0 ** torch.arange(-4, 4).float(), torch.zeros(8)),
                      torch.tensor([1.0, 3.0, 1 + 2.0 ** -23, 1e-30])])
    for i in range(r):
        controls.add_request(f'r{i}', repetition=float(reps[i]))
    controls.prompt_bits.fill_(-1)
    x = (torch.rand((r, vocab), generator=g) + 1e-3) * 2.0 ** torch.randint(-30, 30, (r, vocab), generator=g)
    x[:, :64] *= 1e-22
    x[:, 64:128] *= 1e25
    x[:, 128:4000] *= -1
    x[0, 7], x[1, 7], x[2, 7] = float('inf'), float('-inf'), 0.0
    want = torch.where(x > 0, x / reps[:, None], x * reps[:, None])
    got = pkg.control_logits(x.to(dev()), controls, controls.slot_index([f'r{i}' for i in range(r)])).cpu()
    assert torch.equal(got, want)
    status_clean(pkg)


def test_commit_counts_emitted_tokens(pkg):
    controls = pkg.TokenControls(3, 101, device=dev())
    for n in 'abc':
        controls.add_request(n, output=[5])
    slots = controls.slot_index(['c', 'a'])
    emitted = torch.tensor([7, 7, 5, -1, 100, 0, 0, 9], device=dev())
    controls.commit(slots, emitted, i32([0, 4, 8]), i32([3, 3]))
    want = np.zeros((3, 101), dtype=np.int64)
    want[:, 5] = 1
    want[2, 7] += 2
    want[2, 5] += 1
    want[0, 100] += 1
    want[0, 0] += 2
    assert (controls.counts[:, :101].cpu().numpy() == want).all()
    status_clean(pkg)
    # the same slot twice in one call adds up; a full counter saturates; -1 is flagged
    controls.counts[0, 50] = 32766
    fifty = torch.full((40,), 50, dtype=torch.long, device=dev())
    controls.commit(controls.slot_index(['a', 'a', 'b']), fifty, i32([0, 20, 30, 40]))
    assert controls.counts[0, 50] == 32767 and controls.counts[1, 50] == 10 and controls.counts[0, 51] == 0
    status_clean(pkg)
    controls.commit(slots, emitted, i32([0, 4, 8]))
    assert pkg.read_device_status(clear=True) == 4
    # slots are reused clean
    controls.remove_request('a')
    assert controls.add_request('d', prompt=[3]) == 0
    assert int(controls.counts[0].abs().sum()) == 0 and int(controls.prompt_bits[0, 0]) == 8


def test_out_of_range_indices_are_skipped_and_flagged(pkg):
    controls = pkg.TokenControls(2, 300, device=dev())
    controls.add_request('a')
    x = torch.zeros((4, 300), device=dev())
    out = torch.full((4, 300), 7.0, device=dev())
    pkg.control_logits(x, controls, i32([9, 0]), cu_query=i32([0, 2, 4]), out=out)
    assert pkg.read_device_status(clear=True) == 4 and (out[:2] == 7).all() and (out[2:] == 0).all()
    pkg.control_logits(x, controls, i32([0, 0]), cu_query=i32([0, 2, 9]), out=out)
    assert pkg.read_device_status(clear=True) == 4
    pred = pkg.control_argmax(x, controls, i32([-1, 0]), cu_query=i32([0, 2, 4]))
    assert pkg.read_device_status(clear=True) == 4 and pred.tolist() == [-1, -1, 0, 0]
    toks = torch.tensor([0, 300, 0, -4], device=dev())
    pkg.control_logits(x, controls, i32([0, 0]), cu_query=i32([0, 2, 4]), tokens=toks)
    assert pkg.read_device_status(clear=True) == 4
    masks = torch.full((1, 10), -1, dtype=torch.int32, device=dev())
    pkg.control_logits(x, controls, i32([0, 0]), cu_query=i32([0, 2, 4]), masks=masks, mask_index=i32([0, 1, -5, 0]))
    assert pkg.read_device_status(clear=True) == 4


def test_captured_round_on_a_side_stream(pkg):
    """control_argmax and commit in a captured graph, replayed: the counts move the choice on."""
    vocab = 4096
    controls = pkg.TokenControls(1, vocab, device=dev())
    controls.add_request('a', presence=1.0, frequency=0.0)
    slots = controls.slot_index(['a'])
    x = torch.zeros((1, vocab), device=dev())
    for k in range(6):
        x[0, 100 * k + 3] = 3.0 - 0.125 * k
    cu, one = i32([0, 1]), i32([1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    picked = torch.zeros(1, dtype=torch.long, device=dev())

    def step():
        picked.copy_(pkg.control_argmax(x, controls, slots, cu_query=cu))
        controls.commit(slots, picked, cu, one)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    got = []
    for _ in range(6):
        graph.replay()
        got.append(int(picked))
    assert got == [100 * k + 3 for k in range(6)]
    status_clean(pkg)


def test_refusals(pkg):
    controls = pkg.TokenControls(2, 64, device=dev(), max_bias=2)
    controls.add_request('a')
    for bad in (dict(request='a'), dict(request=''), dict(request='b', repetition=0.0),
                dict(request='b', repetition=float('nan')), dict(request='b', frequency=float('inf')),
                dict(request='b', bias={1: 1.0, 2: 1.0, 3: 1.0}), dict(request='b', bias=([1, 2], [1.0])),
                dict(request='b', prompt=[64]), dict(request='b', output=[-1]), dict(request='b', bias={64: 1.0})):
        with pytest.raises(ValueError):
            controls.add_request(**bad)
    controls.add_request('b')
    with pytest.raises(ValueError):
        controls.add_request('c')
    with pytest.raises(KeyError):
        controls.remove_request('zz')
    with pytest.raises(KeyError):
        controls.slot_index(['zz'])
    x = torch.zeros((2, 64), device=dev())
    slots, cu, tok = controls.slot_index(['a', 'b']), i32([0, 1, 2]), torch.zeros(2, dtype=torch.long, device=dev())
    masks, index = torch.zeros((1, 2), dtype=torch.int32, device=dev()), i32([0, -1])
    ok = dict(logits=x, controls=controls, slots=slots, cu_query=cu, tokens=tok, masks=masks, mask_index=index)
    pkg.control_logits(**ok)
    for bad in (dict(logits=x[:, :63]), dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x.t()),
                dict(slots=slots.long()), dict(cu_query=cu[:2]), dict(cu_query=None), dict(tokens=tok[:1]),
                dict(tokens=tok.int()), dict(masks=None), dict(masks=masks[:, :1]), dict(mask_index=index[:1]),
                dict(logits=x.clone().requires_grad_())):
        with pytest.raises(ValueError):
            pkg.control_logits(**{**ok, **bad})
        with pytest.raises(ValueError):
            pkg.control_argmax(**{**ok, **bad})
    for bad in (dict(out=x[:1]), dict(out=x.bfloat16()), dict(out_dtype=torch.bfloat16), dict(out=x, out_dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            pkg.control_logits(**{**ok, **bad})
    wide = torch.zeros(2 * 64 + 32, device=dev())
    with pytest.raises(ValueError):               # an output overlapping the logits
        pkg.control_logits(**{**ok, 'logits': wide[:128].view(2, 64), 'out': wide[32:].view(2, 64)})
    with pytest.raises(ValueError):
        controls.commit(slots, tok, cu[:2])
    with pytest.raises(ValueError):
        controls.commit(slots.long(), tok, cu)
    for a in ((0, 5), (1, 0), (1.0, 5)):
        with pytest.raises(ValueError):
            pkg.TokenControls(*a, device=dev())
    torch.cuda.synchronize()
    status_clean(pkg)
