"""Cases and float64 evaluations of the paged 8-bit cache, from its definition."""
import torch

HQ, HKV, D, PAGE = 16, 8, 128, 64
SCALE = D ** -0.5
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
CODES = [torch.int8, torch.float8_e4m3fn]

# name, new rows, context tokens
CASES = [
    ('one_token', [1], [0]),
    ('one_row_each', [1, 1, 1], [0, 1, 63]),
    ('page_edges', [1, 7, 8, 1, 3], [63, 64, 65, 128, 127]),
    ('first_steps', [1] * 4, [600, 333, 12, 599]),
    ('verify', [8] * 9, [131 * i for i in range(9)]),
    ('ragged', [7, 1, 8, 4, 3, 6] + [1 + i % 8 for i in range(20)], [0, 9, 31, 700, 64, 200] + [(337 * i) % 900 for i in range(20)]),
    ('long_decode', [1, 2], [20011, 9000]),
    ('chunks', [150, 9, 65], [200, 0, 71]),
    ('one_chunk', [333], [1000]),
    ('prompt', [257], [0]),
    ('empty_queries', [0, 3, 0, 5, 0], [100, 7, 0, 190, 63]),
    ('many', [1 + i % 3 for i in range(300)], [(59 * i) % 260 for i in range(300)]),
    ('more_chunk', [17, 40, 16], [5000, 333, 64]),
]


def codes(shape, dtype, g):
    """Random codes over the whole range of the type."""
    x = torch.randn(shape, generator=g)
    if dtype == torch.int8:
        return (x * 40).round().clamp(-127, 127).to(torch.int8)
    return (x * 120).clamp(-448, 448).to(torch.float8_e4m3fn)


def make(seed, rows, contexts, dtype, row_dtype, *, layers=1, spare=3, spare_slots=2):
    """A cache and a batch on the CPU: what no row of the batch may see holds NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [n // PAGE for n in contexts]
    r, pages, slots = len(rows), sum(need) + spare, len(rows) + spare_slots
    ids = torch.randperm(pages, generator=g)
    table = torch.full((r, max(max(need), 1)), -1, dtype=torch.int32)
    slot = torch.randperm(slots, generator=g)[:r].int()
    nan = float('nan')
    scale = lambda: (0.5 + torch.rand((layers, pages, HKV), generator=g)) / (32 if dtype == torch.int8 else 110)  # noqa: E731
    x = dict(key=codes((layers, pages, HKV, 2, PAGE, D // 2), dtype, g), value=codes((layers, pages, HKV, D, PAGE), dtype, g),
             key_scale=scale(), value_scale=scale(), tail_key=torch.full((layers, slots, 2, PAGE, HKV, D), nan, dtype=row_dtype),
             tail_value=torch.full((layers, slots, 2, PAGE, HKV, D), nan, dtype=row_dtype))
    at = 0
    for i, n in enumerate(contexts):
        table[i, :need[i]] = ids[at:at + need[i]].int()
        at += need[i]
        for t in ('tail_key', 'tail_value'):
            x[t][:, int(slot[i]), need[i] % 2, :n % PAGE] = torch.randn((layers, n % PAGE, HKV, D), generator=g).to(row_dtype)
    for s in ('key_scale', 'value_scale'):
        x[s][:, ids[at:]] = nan
    total = sum(rows)
    rand = lambda h: torch.randn((layers, total, h, D), generator=g).to(row_dtype)  # noqa: E731
    return x, dict(table=table, slots=slot, rows=list(rows), contexts=list(contexts), query=rand(HQ), new_key=rand(HKV),
                   new_value=rand(HKV))


def page_values(x, layer, ids):
    """Float64 values [n * 64, 8, 128] of pages: (key, value)."""
    k = x['key'][layer, ids].double() * x['key_scale'][layer, ids].double()[..., None, None, None]
    v = x['value'][layer, ids].double() * x['value_scale'][layer, ids].double()[..., None, None]
    k = torch.cat((k[:, :, 0], k[:, :, 1]), -1).transpose(1, 2).reshape(-1, HKV, D)
    return k, v.permute(0, 3, 1, 2).reshape(-1, HKV, D)


def attention(x, b, layer=0):
    """(out, weight, size) in float64: the output, sum_j p_j |v_j| of its elements, and the largest
    sum_d |q_d k_d| scale of a visible key."""
    q = b['query'][layer].double()
    out, weight = torch.zeros_like(q), torch.zeros_like(q)
    size, t0 = 0.0, 0
    for i, (n_new, n) in enumerate(zip(b['rows'], b['contexts'])):
        if n_new == 0:
            continue
        ids, slot, part = b['table'][i, :n // PAGE].long(), int(b['slots'][i]), n // PAGE % 2
        k, v = page_values(x, layer, ids)
        new = slice(t0, t0 + n_new)
        k = torch.cat((k, x['tail_key'][layer, slot, part, :n % PAGE].double(), b['new_key'][layer, new].double()))
        v = torch.cat((v, x['tail_value'][layer, slot, part, :n % PAGE].double(), b['new_value'][layer, new].double()))
        k, v = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        s = torch.einsum('qhd,khd->hqk', q[new], k) * SCALE
        hidden = torch.arange(n + n_new)[None] > torch.arange(n_new)[:, None] + n
        size = max(size, float((torch.einsum('qhd,khd->hqk', q[new].abs(), k.abs()) * SCALE).nan_to_num(0).max()))
        p = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
        for h in range(HQ):             # keys that a row does not see take no part, whatever they hold
            for row in range(n_new) if not torch.isfinite(v).all() else [None]:
                if row is None:
                    out[new, h], weight[new, h] = p[h] @ v[:, h], p[h] @ v[:, h].abs()
                else:
                    see = n + row + 1
                    out[t0 + row, h] = p[h, row, :see] @ v[:see, h]
                    weight[t0 + row, h] = p[h, row, :see] @ v[:see, h].abs()
        t0 += n_new
    return out, weight, size


def attention_tolerance(out, weight, size, row_dtype):
    """Absolute tolerance of each output element.

    bf16: the result's rounding, 2^-8 |out|; the probabilities' rounding, at most 2^-8 of each
    weight (bf16 against unquantised rows; halves, 2^-11, against pages) once more as their sum
    is of the unrounded ones only in the numerator; scores summed in float32 over 128 terms,
    128 * 2^-24 * size off in the exponent, in numerator and denominator. float32: the latter,
    2^-22 for the exponentials and 2^-24 per key and element for the sums, over 2^6 keys between
    partial sums: 2^-17."""
    score = 2 * 128 * 2.0 ** -24 * size
    if row_dtype == torch.bfloat16:
        return 2.0 ** -8 * out.abs() + (2.0 ** -8 + score + 2.0 ** -14) * weight
    return 2.0 ** -24 * out.abs() + (score + 2.0 ** -17) * weight


def e4m3(y):
    """The nearest e4m3 value of each float64 (ties to even): steps of 2^(e - 3), e at least -6."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def quantize(block, dtype):
    """Float64 codes and scales of blocks [layers, 64, 8, 128]: ([layers, 64, 8, 128], [layers, 8])."""
    a = block.abs().amax((1, 3))
    y = block * QMAX[dtype] / torch.where(a > 0, a, 1.0)[:, None, :, None]
    return torch.round(y) if dtype == torch.int8 else e4m3(y), a / QMAX[dtype]


def append(x, b, counts):
    """The cache behind an append, in float64 (codes as the values they stand for)."""
    out = {k: v.double() for k, v in x.items()}
    dtype = x['key'].dtype
    t0 = 0
    for i, (n_new, n) in enumerate(zip(b['rows'], b['contexts'])):
        slot, c = int(b['slots'][i]), counts[i]
        for kind in ('key', 'value'):
            tail, new = out['tail_' + kind], b['new_' + kind][:, t0:t0 + c].double()
            line = torch.cat((tail[:, slot, n // PAGE % 2, :n % PAGE].clone(), new), 1)
            for m in range(line.shape[1] // PAGE):
                code, scale = quantize(line[:, m * PAGE:(m + 1) * PAGE], dtype)
                page = int(b['table'][i, n // PAGE + m])
                out[kind + '_scale'][:, page] = scale
                code = code.transpose(1, 2)                                   # [layers, 8, 64, 128]
                out[kind][:, page] = (torch.stack((code[..., :64], code[..., 64:]), 2) if kind == 'key'
                                      else code.transpose(2, 3))
            last = (n + c) // PAGE
            low = max(n, last * PAGE)
            if n + c > low:
                tail[:, slot, last % 2, low % PAGE:(n + c - 1) % PAGE + 1] = new[:, low - n:]
        t0 += n_new
    return out


def to_gpu(pkg, x, b, device='cuda'):
    """(QuantizedPages, QuantizedLayout, device tensors of the batch)."""
    pages = pkg.QuantizedPages(**{k: v.to(device) for k, v in x.items()})
    t = {k: b[k].to(device) for k in ('table', 'slots', 'query', 'new_key', 'new_value')}
    return pages, pkg.QuantizedLayout.from_lengths(b['rows'], b['contexts'], t['table'], t['slots']), t
