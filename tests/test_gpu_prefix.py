"""GPU parity of the shared-prefix attention (``dspark_prefix_attn``) with the float64 definition.

Error bounds, per element, from A = sum_j p_j |v_j|, o the output and S the row's largest
|q| . |k| * scale:
* bf16: the probabilities are rounded to bf16 before the second product and the output
  once more, each by at most half a step (2^-8 relative): 2^-8 (A + |o|). The scores (fp32
  sums of 128 exact bf16 products: 128 * 2^-24 * S absolutely), exp2, the fp32 sums and the
  merge of partial rows are covered by another 2^-10 A.
* float32: scores off by d = 129 * 2^-24 * S change a probability by at most 2 d relative (d
  itself and d through the sum); exp (2 ulp), the running rescales and the sums of n keys
  in steps of at most 128 add (n / 32 + 160) * 2^-24: (2 d + (n / 32 + 160) 2^-24) A.
"""
import pytest
import torch

from gpu_util import dev, status_clean
from prefix_util import CASES, HKV, SCALE, exact, inputs, layout

pytestmark = pytest.mark.gpu


def run(pkg, x, case, dtype, lay=None, **kw):
    to = lambda t: t.to(dev(), dtype)  # noqa: E731
    lay = lay or layout(pkg, x, case, dev())
    new = dict(new_key=to(x['b'][1]), new_value=to(x['b'][2])) if 'b' in x else {}
    return pkg.B200SharedPrefixKernel(dev())(to(x['q']), to(x['a'][1]), to(x['a'][2]), lay, scale=SCALE,
                                             prefix_key=to(x['p'][1]), prefix_value=to(x['p'][2]), **new, **kw)


def check(got, x, case, dtype):
    ref, weight, score = exact(x, case)
    err = (got.double().cpu() - ref).abs()
    assert torch.isfinite(err).all()
    if dtype == torch.bfloat16:
        tol = 2.0 ** -8 * (weight + ref.abs()) + 2.0 ** -10 * weight
    else:
        n = max(case[1]) + max(case[4]) + (max(case[5]) if case[5] else 0)
        tol = (2 * 129 * 2.0 ** -24 * score[..., None] + (n / 32 + 160) * 2.0 ** -24) * weight
    worst = (err - tol).max()
    assert worst <= 0, f'{case[0]}: error exceeds the bound by {worst} (max error {err.max()})'


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('case', CASES, ids=[c[0] for c in CASES])
def test_matches_definition(pkg, case, dtype):
    x = inputs(11, case)
    got = run(pkg, x, case, dtype)
    torch.cuda.synchronize()
    status_clean(pkg)
    check(got, x, case, dtype)


@pytest.mark.parametrize('grid', [1, 7])
def test_any_grid_gives_the_attention(pkg, grid):
    case = next(c for c in CASES if c[0] == 'groups')
    x = inputs(12, case)
    got = run(pkg, x, case, torch.bfloat16, layout(pkg, x, case, dev(), grid_limit=grid))
    torch.cuda.synchronize()
    status_clean(pkg)
    check(got, x, case, torch.bfloat16)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_layer_offsets_one_pool_and_in_place(pkg, dtype):
    """One pool holds prefix and cached rows of three layers; ``out`` is the query tensor."""
    case = ('pool', [40], [3], [2, 8, 1], [5, 0, 70], [2, 8, 1], True)
    xs = [inputs(20 + layer, case) for layer in range(3)]
    rows = len(xs[0]['p'][1])
    own_rows = len(xs[0]['a'][1])
    pool_k = torch.cat([torch.cat((x['p'][1], x['a'][1])) for x in xs]).to(dev(), dtype)
    pool_v = torch.cat([torch.cat((x['p'][2], x['a'][2])) for x in xs]).to(dev(), dtype)
    scratch_k = torch.cat([x['b'][1] for x in xs]).to(dev(), dtype)
    scratch_v = torch.cat([x['b'][2] for x in xs]).to(dev(), dtype)
    lay = layout(pkg, xs[0], case, dev())
    kernel = pkg.B200SharedPrefixKernel(dev())
    for n, x in enumerate(xs):
        q = x['q'].to(dev(), dtype)
        got = kernel(q, pool_k, pool_v, lay, scale=SCALE, prefix_key=pool_k, prefix_value=pool_v, new_key=scratch_k,
                     new_value=scratch_v, prefix_off=n * (rows + own_rows), own_off=n * (rows + own_rows) + rows,
                     new_off=n * len(x['b'][1]), out=q)
        assert got.data_ptr() == q.data_ptr()
        torch.cuda.synchronize()
        check(got, x, case, dtype)
    status_clean(pkg)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_infinite_and_huge_scores(pkg, dtype):
    """Scores far apart between the prefix and the own keys, either way round: the merge keeps
    the larger side whole, and a row dominated by one key gives that key's value."""
    case = ('apart', [300], [2], [3, 3], [200, 0], [3, 3], True)
    for scale_p, scale_a in ((60.0, 1.0), (1.0, 60.0)):
        x = inputs(31, case)
        x['p'] = (x['p'][0], x['p'][1] * scale_p, x['p'][2])
        x['a'] = (x['a'][0], x['a'][1] * scale_a, x['a'][2])
        for n in ('p', 'a'):
            x[n] = (x[n][0], x[n][1].bfloat16().float(), x[n][2])
        got = run(pkg, x, case, dtype)
        torch.cuda.synchronize()
        check(got, x, case, dtype)
    status_clean(pkg)


def test_streams_and_captured_graphs(pkg):
    """Two captured graphs replayed at once on two streams, with new inputs in the captured
    buffers, equal eager calls bit for bit."""
    case = next(c for c in CASES if c[0] == 'split_prefix')
    kernel = pkg.B200SharedPrefixKernel(dev())
    x = inputs(41, case)
    lay = layout(pkg, x, case, dev())
    to = lambda t: t.to(dev(), torch.bfloat16)  # noqa: E731
    fixed = dict(prefix_key=to(x['p'][1]), prefix_value=to(x['p'][2]), new_key=to(x['b'][1]), new_value=to(x['b'][2]))
    a = (to(x['a'][1]), to(x['a'][2]))
    q = [to(x['q']), to(x['q'].flip(0))]
    eager = [kernel(t, *a, lay, scale=SCALE, **fixed).clone() for t in q]
    buffers = [torch.zeros_like(q[0]) for _ in q]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for b, s in zip(buffers, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(kernel(b, *a, lay, scale=SCALE, **fixed))
        graphs.append(graph)
    for b, t in zip(buffers, q):
        b.copy_(t)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, eager):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    status_clean(pkg)


def test_repeated_calls_are_identical(pkg):
    case = next(c for c in CASES if c[0] == 'groups')
    x = inputs(51, case)
    first = run(pkg, x, case, torch.bfloat16)
    for _ in range(3):
        assert torch.equal(run(pkg, x, case, torch.bfloat16).view(torch.int16), first.view(torch.int16))


def test_no_query_rows(pkg):
    lay = pkg.SharedPrefixLayout.from_lengths([9], [2], [0, 0], [1, 2], device=dev())
    z = lambda n, h: torch.zeros((n, h, 128), dtype=torch.bfloat16, device=dev())  # noqa: E731
    out = pkg.B200SharedPrefixKernel(dev())(z(0, 16), z(3, 8), z(3, 8), lay, scale=SCALE, prefix_key=z(9, 8),
                                            prefix_value=z(9, 8))
    assert out.shape == (0, 16, 128)
    torch.cuda.synchronize()
    status_clean(pkg)


def test_no_keys_gives_zeros(pkg):
    for dtype in (torch.bfloat16, torch.float32):
        lay = pkg.SharedPrefixLayout.from_lengths([0, 3], [2, 1], [2, 9, 1], [0, 4, 0], causal=False, device=dev())
        g = torch.Generator(device=dev()).manual_seed(1)
        r = lambda n, h: torch.randn((n, h, 128), device=dev(), generator=g).to(dtype)  # noqa: E731
        out = pkg.B200SharedPrefixKernel(dev())(r(12, 16), r(4, 8), r(4, 8), lay, scale=SCALE, prefix_key=r(3, 8),
                                                prefix_value=r(3, 8))
        torch.cuda.synchronize()
        assert (out[:2] == 0).all() and (out[2:] != 0).any(-1).all()
    status_clean(pkg)


def test_refusals(pkg):
    case = ('refusals', [5], [2], [1, 2], [2, 0], [1, 2], True)
    x = inputs(61, case)
    lay = layout(pkg, x, case, dev())
    to = lambda t: t.to(dev(), torch.bfloat16)  # noqa: E731
    ok = dict(query=to(x['q']), key=to(x['a'][1]), value=to(x['a'][2]), layout=lay, scale=SCALE,
              prefix_key=to(x['p'][1]), prefix_value=to(x['p'][2]), new_key=to(x['b'][1]), new_value=to(x['b'][2]))
    kernel = pkg.B200SharedPrefixKernel(dev())
    kernel(**ok)
    for bad in (dict(query=ok['query'][:2]), dict(query=ok['query'].float()), dict(query=ok['query'].cpu()),
                dict(query=ok['query'].half()), dict(scale=0.1), dict(layout=object()), dict(key=ok['key'][:, :4]),
                dict(value=ok['value'][:-1]), dict(prefix_key=ok['prefix_key'].transpose(0, 1)),
                dict(prefix_key=ok['prefix_key'][:5], prefix_value=ok['prefix_value'][:5]), dict(new_key=None), dict(key=None), dict(prefix_value=None),
                dict(new_key=None, new_value=None), dict(prefix_off=9), dict(prefix_off=-1), dict(own_off=1.0),
                dict(out=torch.empty_like(ok['query'][:1])), dict(query=ok['query'].clone().requires_grad_())):
        with pytest.raises(ValueError):
            kernel(**{**ok, **bad})
    with pytest.raises(ValueError):
        kernel(**{**ok, 'layout': layout(pkg, x, case, 'cpu', grid_limit=4)})
    torch.cuda.synchronize()
    status_clean(pkg)


def test_foreign_plan_is_refused_on_the_device(pkg):
    """A device plan that does not belong to the layout's head computes nothing and is flagged."""
    import dataclasses
    case = ('foreign', [5], [2], [1, 2], [2, 0], [1, 2], True)
    x = inputs(62, case)
    lay = layout(pkg, x, case, dev())
    plan = lay.plan.clone()
    plan[18] += 1
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((3, 16, 128), 7.0, dtype=dtype, device=dev())
        run(pkg, x, case, dtype, dataclasses.replace(lay, plan=plan), out=out)
        torch.cuda.synchronize()
        assert pkg.read_device_status(clear=True) == 4
        assert (out == 7).all()


def test_rows_past_32_bit_offsets(pkg):
    """Key rows whose element offsets pass 2^31 (a 2.2 million-row pool, 4.5 GB per tensor)."""
    rows = (1 << 21) + 100_000
    pool = torch.zeros((rows, HKV, 128), dtype=torch.bfloat16, device=dev())
    case = ('far', [200], [2], [2, 8], [30, 4], [2, 8], True)
    x = inputs(71, case)
    at = rows - 400
    n = len(x['p'][1])
    pool_v = torch.zeros_like(pool)
    for t, p in ((1, pool), (2, pool_v)):
        p[at:at + n] = x['p'][t].to(dev(), torch.bfloat16)
        p[at + n:at + n + len(x['a'][t])] = x['a'][t].to(dev(), torch.bfloat16)
    lay = layout(pkg, x, case, dev())
    to = lambda t: t.to(dev(), torch.bfloat16)  # noqa: E731
    got = pkg.B200SharedPrefixKernel(dev())(to(x['q']), pool, pool_v, lay, scale=SCALE, prefix_key=pool,
                                            prefix_value=pool_v, new_key=to(x['b'][1]), new_value=to(x['b'][2]),
                                            prefix_off=at, own_off=at + n)
    torch.cuda.synchronize()
    status_clean(pkg)
    check(got, x, case, torch.bfloat16)
