"""What a paged 8-bit cache meets at its edges: values that are not finite behind a row, scales and
scores of any size, pages that are not there, several calls at once, captured calls."""
import pytest
import torch

import quant_util as U
from gpu_util import status_clean

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# few new rows, many of them, and both in one batch
SHAPES = [([8, 3], [70, 200]), ([150, 41], [130, 64]), ([3, 130, 1, 64], [300, 90, 128, 0])]


def run(pkg, x, b, **more):
    pages, layout, t = U.to_gpu(pkg, x, b)
    return pkg.B200QuantizedKernel('cuda')(t['query'][0], t['new_key'][0], t['new_value'][0], layout, scale=U.SCALE,
                                           pages=pages, **more)


def compare(got, x, b, row_dtype, wide_range=False):
    """With `wide_range`, probabilities far below a row's largest count too. They are halves 2^-24 apart
    at the least, relative to a largest one of at least 2^8, so each is off by 2^-33 of that; the
    denominator is at least the largest one."""
    out, weight, size = U.attention(x, b)
    tol = U.attention_tolerance(out, weight, size, row_dtype)
    if wide_range:
        k, v = U.page_values(x, 0, b['table'][b['table'] >= 0].long())
        tol = tol + 2.0 ** -33 * len(v) * float(v.abs().max())
    got = got.double().cpu()
    fine = torch.isfinite(out)
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    assert torch.equal(got[~fine & ~torch.isnan(out)], out[~fine & ~torch.isnan(out)])
    err = (got - out).abs()[fine]
    assert bool((err <= tol[fine]).all()), float((err - tol[fine]).max())


@pytest.mark.parametrize('row_dtype', [BF16, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('what', ['value_nan', 'value_inf', 'key_nan'])
@pytest.mark.parametrize('shape', SHAPES, ids=['few', 'many', 'both'])
def test_what_is_not_finite_reaches_only_the_rows_that_see_it(pkg, shape, what, row_dtype):
    x, b = U.make(21, *shape, torch.int8, row_dtype)
    t0 = 0
    for n in shape[0]:
        j = t0 + max(n - 2, 0)                                     # one of the last rows of each request
        if what == 'key_nan':
            b['new_key'][0, j, 3] = float('nan')
        else:
            b['new_value'][0, j, 5, 17] = float('nan') if what == 'value_nan' else float('inf')
        t0 += n
    compare(run(pkg, x, b), x, b, row_dtype)
    status_clean(pkg)


@pytest.mark.parametrize('shape', SHAPES, ids=['few', 'many', 'both'])
def test_infinite_and_nan_scales_make_their_block_nan(pkg, shape):
    for bad in (float('nan'), float('inf')):
        x, b = U.make(22, *shape, torch.int8, BF16)
        clean = run(pkg, x, b)
        ids = b['table'][1][b['table'][1] >= 0]
        if not len(ids):
            continue
        x['value_scale'][0, int(ids[0]), 2] = bad
        got = run(pkg, x, b)
        t0, n = shape[0][0], shape[0][1]
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[t0:t0 + n, 4:6] = True
        assert not torch.isfinite(got[hit]).any()
        assert torch.equal(got[~hit], clean[~hit])
    status_clean(pkg)


@pytest.mark.parametrize('dtype', U.CODES, ids=['int8', 'e4m3'])
@pytest.mark.parametrize('shape', SHAPES, ids=['few', 'many', 'both'])
def test_scales_of_any_size(pkg, shape, dtype):
    """Value scales far apart from block to block, zero blocks, and scores of thousands."""
    x, b = U.make(23, *shape, dtype, BF16)
    g = torch.Generator().manual_seed(1)
    pages = x['value_scale'].shape[1]
    x['value_scale'] = x['value_scale'] * torch.exp2(torch.randint(-30, 20, (1, pages, 8), generator=g).float())
    for page in range(0, pages, 3):                                # what quantising a block of zeros gives
        for s in ('key', 'value'):
            x[s][0, page, 1] = torch.zeros_like(x[s][0, page, 1].float()).to(dtype)
            x[s + '_scale'][0, page, 1] = 0
    compare(run(pkg, x, b), x, b, BF16)
    # heads 2 and 3 large: the largest score of a row decides, whatever its size
    x, b = U.make(24, *shape, dtype, BF16)
    b['query'][..., 4:8, :] *= 1000
    b['query'][..., 0, :] *= 2.0 ** -60
    compare(run(pkg, x, b), x, b, BF16, wide_range=True)
    # every third page's values next to nothing: its keys still count in the denominator
    x, b = U.make(29, *shape, dtype, BF16)
    x['value_scale'][:, ::3] *= 2.0 ** -118
    x['value_scale'][:, 1::6] *= 2.0 ** -75
    compare(run(pkg, x, b), x, b, BF16)
    status_clean(pkg)


@pytest.mark.parametrize('row_dtype', [BF16, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('shape', SHAPES, ids=['few', 'many', 'both'])
def test_pages_and_slots_that_are_not_there_are_left_out(pkg, shape, row_dtype):
    x, b = U.make(25, *shape, torch.float8_e4m3fn, row_dtype)
    i = 1 if shape[1][1] >= 64 else 0
    other = dict(b, table=b['table'].clone())
    other['table'][i, 0] = x['key'].shape[1] + 5
    got = run(pkg, x, other)
    assert pkg.read_device_status(clear=True) == 4
    # the same without that page's weight: its K far below, its V zero
    page = int(b['table'][i, 0])
    full = U.attention(x, b)[0]
    rows = slice(sum(shape[0][:i]), sum(shape[0][:i + 1]))
    keep = torch.ones(len(full), dtype=torch.bool)
    keep[rows] = False
    y = {k: v.clone() for k, v in x.items()}
    out = torch.zeros_like(full)
    # the page taken out of the request: the others move up
    rest = dict(b, table=b['table'].clone(), contexts=list(b['contexts']))
    n = b['contexts'][i] // 64
    rest['table'][i, :n - 1] = b['table'][i, 1:n]
    rest['contexts'][i] -= 64
    for kind in ('tail_key', 'tail_value'):                        # the open block changes its place with its number
        slot = int(b['slots'][i])
        y[kind][:, slot] = y[kind][:, slot].flip(1)
    out, weight, size = U.attention(y, rest)
    tol = U.attention_tolerance(out, weight, size, row_dtype)
    assert bool(((got.double().cpu() - out).abs() <= tol).all()) and page >= 0
    # a slot that is not there: the request's open rows are left out, the others are as they were
    other = dict(b, slots=b['slots'].clone())
    other['slots'][i] = 99
    got = run(pkg, x, other)
    assert pkg.read_device_status(clear=True) == 4
    err = (got.double().cpu() - full).abs()[keep]
    w, s = U.attention(x, b)[1:]
    assert bool((err <= U.attention_tolerance(full, w, s, row_dtype)[keep]).all())


@pytest.mark.parametrize('shape', SHAPES, ids=['few', 'many', 'both'])
def test_in_place_other_streams_and_at_once(pkg, shape):
    x, b = U.make(26, *shape, torch.int8, BF16, layers=2)
    pages, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')
    call = lambda layer, **more: kernel(t['query'][layer], t['new_key'][layer], t['new_value'][layer], layout,  # noqa: E731
                                        scale=U.SCALE, pages=pages, layer=layer, **more)
    want = [call(0), call(1)]
    q = t['query'][0].clone()
    assert kernel(q, t['new_key'][0], t['new_value'][0], layout, scale=U.SCALE, pages=pages, out=q) is q
    assert torch.equal(q, want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):                                             # both layers at once, one layout
        got = []
        for layer, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(call(layer))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    status_clean(pkg)


def test_captured_calls_follow_the_tables(pkg):
    """Plan, attention and append captured together; contexts and tables change between replays."""
    rows, contexts = [4, 60, 1], [61, 3, 190]
    x, b = U.make(27, rows, contexts, torch.int8, BF16, spare=12)
    width = 8
    table = torch.full((3, width), -1, dtype=torch.int32)
    table[:, :b['table'].shape[1]] = b['table']
    used = set(b['table'].flatten().tolist())
    spare = [p for p in range(x['key'].shape[1]) if p not in used]
    for i, n in enumerate(contexts):
        for k in range(n // 64, n // 64 + 3):
            table[i, k] = spare.pop()
    b['table'] = table
    pages, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')
    counts = torch.tensor(rows, dtype=torch.int32, device='cuda')

    def step():
        layout.replan()
        out = kernel(t['query'][0], t['new_key'][0], t['new_value'][0], layout, scale=U.SCALE, pages=pages)
        pages.append(t['new_key'], t['new_value'], layout, counts)
        layout.context.add_(counts)
        return out
    keep = {k: getattr(pages, k).clone() for k in x}
    ctx = layout.context.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for k, v in keep.items():
        getattr(pages, k).copy_(v)
    layout.context.copy_(ctx)
    for _ in range(3):
        before = {k: getattr(pages, k).cpu().clone() for k in x}
        now = dict(b, contexts=layout.context.tolist())
        graph.replay()
        compare(out, before, now, BF16)
        want = U.append(before, now, rows)
        for k in ('key', 'value'):
            assert torch.equal(getattr(pages, k).cpu().double(), want[k])
    status_clean(pkg)


def test_offsets_beyond_32_bits(pkg):
    """Pages whose codes lie beyond 4 GB in a layer, and in later layers."""
    free = torch.cuda.mem_get_info()[0]
    pages = 70000                                                  # 4.6 GB of K and of V a layer
    if free < 24 << 30:
        pytest.skip('needs 24 GB')
    rows, contexts = [2, 45], [130, 70]
    x, b = U.make(28, rows, contexts, torch.int8, BF16, layers=2)
    want = []
    small, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')
    for layer in range(2):
        want.append(kernel(t['query'][layer], t['new_key'][layer], t['new_value'][layer], layout, scale=U.SCALE, pages=small,
                           layer=layer))
    big = pkg.QuantizedPages.empty(layers=2, pages=pages, slots=small.slots)
    n = small.pages
    for name in ('key', 'value', 'key_scale', 'value_scale'):
        getattr(big, name)[:, -n:] = getattr(small, name)
    big.tail_key.copy_(small.tail_key)
    big.tail_value.copy_(small.tail_value)
    far = t['table'].clone()
    far[far >= 0] += pages - n
    wide = pkg.QuantizedLayout.from_lengths(rows, contexts, far, t['slots'])
    for layer in range(2):
        got = kernel(t['query'][layer], t['new_key'][layer], t['new_value'][layer], wide, scale=U.SCALE, pages=big, layer=layer)
        assert torch.equal(got, want[layer])
    big.copy([pages - n], [pages - n - 7])
    assert torch.equal(big.key[1, pages - n - 7], small.key[1, 0])
    status_clean(pkg)


@pytest.mark.parametrize('case', [([128, 130], [1, 63], None), ([200], [10], [130]), ([256], [70], None)],
                         ids=['two_blocks', 'counted', 'four_blocks'])
@pytest.mark.parametrize('row_dtype', [BF16, F32], ids=['bf16', 'fp32'])
def test_append_where_both_ends_lie_in_one_tail_block(pkg, case, row_dtype):
    """An even number of blocks gets full: the rows behind them go where the first ones are read."""
    from test_gpu_quant_append import page_table
    rows, contexts, counts = case
    for seed in range(4):
        x, b = U.make(30 + seed, rows, contexts, torch.int8, row_dtype, layers=5, spare=20)
        page_table(b, counts or rows)
        pages, layout, t = U.to_gpu(pkg, x, b)
        pages.append(t['new_key'], t['new_value'], layout,
                     None if counts is None else torch.tensor(counts, dtype=torch.int32, device='cuda'))
        want = U.append(x, b, counts or rows)
        for name in ('key', 'value', 'tail_key', 'tail_value'):
            got = getattr(pages, name).cpu().double()
            assert bool(((got == want[name]) | (got.isnan() & want[name].isnan())).all()), name
    status_clean(pkg)


@pytest.mark.parametrize('dtype', U.CODES, ids=['int8', 'e4m3'])
@pytest.mark.parametrize('row_dtype', [BF16, F32], ids=['bf16', 'fp32'])
def test_append_of_extreme_blocks(pkg, dtype, row_dtype):
    """Zero blocks, tiny and huge ones, ties between codes, and values that are not finite."""
    from test_gpu_quant_append import page_table
    x, b = U.make(40, [64] * 6, [0] * 6, dtype, row_dtype, spare=20)
    page_table(b, [64] * 6)
    k = b['new_key'][0].reshape(6, 64, 8, 128)
    k[0] = 0
    k[1] *= 2.0 ** -120
    k[2] *= 2.0 ** 100
    # quotients half way between codes: a = 254 and odd multiples of 1, ties for int8 with qmax 127
    k[3] = (torch.arange(64 * 8 * 128).reshape(64, 8, 128) % 254 - 127).to(row_dtype)
    k[3, 0, :, 0] = 254
    k[4, 5, 2, 7] = float('nan')
    k[5, 9, 4, 100] = float('inf')
    pages, layout, t = U.to_gpu(pkg, x, b)
    pages.append(t['new_key'], t['new_value'], layout)
    want = U.append(x, b, [64] * 6)
    for name in ('key', 'value'):
        got, w = getattr(pages, name).cpu().double(), want[name]
        s = want[name + '_scale']
        fine = torch.isfinite(s)[:, :, :, None, None].reshape(s.shape + (1,) * (w.ndim - 3)).expand(w.shape)
        assert torch.equal(got[fine], w[fine]), name
        gs = getattr(pages, name + '_scale').cpu()
        assert torch.equal(torch.isfinite(gs), torch.isfinite(s))
    status_clean(pkg)


def test_refusals(pkg):
    x, b = U.make(50, [3, 2], [70, 5], torch.int8, BF16, layers=2)
    pages, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')
    q, k, v = t['query'][0], t['new_key'][0], t['new_value'][0]
    ok = dict(scale=U.SCALE, pages=pages)
    for args, more in (((q.float(), k, v, layout), ok), ((q[:4], k, v, layout), ok), ((q, k[:, :4], v, layout), ok),
                       ((q, k, v.cpu(), layout), ok), ((q.transpose(0, 1).contiguous().transpose(0, 1), k, v, layout), ok),
                       ((q, k, v, layout), dict(ok, scale=0.1)), ((q, k, v, layout), dict(ok, layer=2)),
                       ((q, k, v, layout), dict(ok, pages=None)), ((q, k, v, None), ok),
                       ((q, k, v, layout), dict(ok, out=k)), ((q, k, v, layout), dict(ok, out=q[:3]))):
        with pytest.raises((ValueError, AttributeError)):
            kernel(*args, **more)
    for a in ((t['new_key'][:1], t['new_value'][:1]), (t['new_key'].float(), t['new_value'].float()),
              (t['new_key'][:, :4].contiguous(), t['new_value'][:, :4].contiguous()), (t['new_key'], t['new_value'][:1])):
        with pytest.raises(ValueError):
            pages.append(*a, layout)
    with pytest.raises(ValueError):
        pages.append(t['new_key'], t['new_value'], layout, torch.zeros(2, device='cuda'))
    with pytest.raises(ValueError):
        pages.append(pages.tail_key.view(2, -1, 8, 128)[:, :8].contiguous().view(2, -1, 8, 128)[:, ::2], t['new_value'], layout)
    for a, more in ((([0], [0]), {}), (([0, 1], [2, 2]), {}), (([0], []), {}), (([99], [0]), {}), (([0], [-1]), {}),
                    (((), ()), dict(tail_src=[0], tail_dst=[0], tail_lengths=[3])),
                    (((), ()), dict(tail_src=[0], tail_dst=[1])),
                    ((torch.tensor([0], device='cuda'), torch.tensor([1], device='cuda')), {})):
        with pytest.raises(ValueError):
            pages.copy(*a, **more)
    with pytest.raises(ValueError):
        pkg.QuantizedLayout.from_lengths([1], [200], t['table'][:1], t['slots'][:1])       # more pages than the table
    with pytest.raises(ValueError):
        pkg.QuantizedLayout.from_lengths([1, 1], [5, 5], t['table'].long(), t['slots'])
    # lengths that do not fit the batch on the device: no rows of that request, and the status says so
    layout.context.copy_(torch.tensor([70, -5], dtype=torch.int32))
    layout.replan()
    got = kernel(q, k, v, layout, **ok, out=torch.full_like(q, 7.0))
    assert pkg.read_device_status(clear=True) == 4
    assert bool((got[3:] == 7.0).all()) and bool((got[:3] != 7.0).any())


@pytest.mark.parametrize('row_dtype', [BF16, F32], ids=['bf16', 'fp32'])
def test_device_lengths_that_do_not_fit_the_batch(pkg, row_dtype):
    """The batch's numbers on the host are the launch's; the device's lengths are checked against them."""
    x, b = U.make(51, [60, 60, 60], [70, 5, 64], torch.int8, row_dtype)
    pages, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')

    def call():
        layout.replan()
        return kernel(t['query'][0], t['new_key'][0], t['new_value'][0], layout, scale=U.SCALE, pages=pages,
                      out=torch.full_like(t['query'][0], 7.0))
    good = call()
    status_clean(pkg)
    # requests of 20 and 100 rows, where all have 60; the other keeps its result
    layout.cu_query.copy_(torch.tensor([0, 20, 120, 180], dtype=torch.int32))
    got = call()
    assert pkg.read_device_status(clear=True) == 4
    assert bool((got[:120] == 7.0).all()) and torch.equal(got[120:], good[120:])
    # rows out of range: no request has a result that another one's rows could be mistaken for
    for bad in ([0, 60, 0, 60], [0, 60, 120, 10 ** 6], [-60, 0, 60, 120], [0, 2 ** 30, 60, 120]):
        layout.cu_query.copy_(torch.tensor(bad, dtype=torch.int32))
        got = call()
        assert pkg.read_device_status(clear=True) == 4
        if row_dtype == BF16:
            assert bool((got == 7.0).all())
        keep = {k: getattr(pages, k).clone() for k in ('key', 'value')}
        pages.append(t['new_key'], t['new_value'], layout)
        assert pkg.read_device_status(clear=True) == 4
        assert all(v.shape == getattr(pages, k).shape for k, v in keep.items())


def test_a_plan_of_another_batch_is_refused(pkg):
    x, b = U.make(52, [3, 50], [70, 200], torch.int8, BF16)
    pages, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')
    for change in (dict(table=torch.nn.functional.pad(layout.table, (0, 2), value=-1)),
                   dict(plan=torch.zeros_like(layout.plan)), dict(query_lengths=(3, 49))):
        lengths = change.get('query_lengths', layout.query_lengths)
        n = sum(lengths)
        cu = torch.tensor([0, 3, n], dtype=torch.int32, device='cuda')
        other = pkg.QuantizedLayout.on_device(lengths, cu, layout.context, change.get('table', layout.table), layout.slots,
                                              plan=change.get('plan', layout.plan.clone()), replan=False)
        got = kernel(t['query'][0, :n], t['new_key'][0, :n], t['new_value'][0, :n], other, scale=U.SCALE, pages=pages,
                     out=torch.full_like(t['query'][0, :n], 7.0))
        assert pkg.read_device_status(clear=True) == 4 and bool((got == 7.0).all())
        other.replan()
        kernel(t['query'][0, :n], t['new_key'][0, :n], t['new_value'][0, :n], other, scale=U.SCALE, pages=pages)
        status_clean(pkg)


@pytest.mark.parametrize('rows', [[1, 1], [64, 64], [3, 64]], ids=['few', 'many', 'both'])
def test_calls_that_feed_one_another(pkg, rows):
    """Each call's output is the next one's query, with nothing between them on the stream."""
    x, b = U.make(53, rows, [130, 4000], torch.int8, BF16)
    pages, layout, t = U.to_gpu(pkg, x, b)
    kernel = pkg.B200QuantizedKernel('cuda')

    def chain(wait):
        q = t['query'][0]
        for _ in range(6):
            q = kernel(q, t['new_key'][0], t['new_value'][0], layout, scale=U.SCALE, pages=pages)
            if wait:
                torch.cuda.synchronize()
        return q
    want = chain(True)
    for _ in range(5):
        assert torch.equal(chain(False), want)
    status_clean(pkg)


@pytest.mark.parametrize('dtype', U.CODES, ids=['int8', 'e4m3'])
def test_lengths_around_the_change_of_kernels(pkg, dtype):
    """Requests on both sides of where the wide kernel takes over, in one batch and each alone."""
    for rows, contexts in (([32, 33, 31, 34], [130, 64, 200, 7]), ([32, 32], [63, 700]), ([33, 33], [63, 700]), ([33], [0])):
        x, b = U.make(54, rows, contexts, dtype, BF16)
        compare(run(pkg, x, b), x, b, BF16)
    status_clean(pkg)
