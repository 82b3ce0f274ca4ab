"""Workloads of the shared-prefix attention and of the logits controls.

``listed()`` names the measured cases, ``draw(rng)`` gives others of the same
ranges, ``prepare`` makes a case's inputs on the GPU, and ``run`` makes one pass:
the plain torch form where ``own`` is false, the framework's operators where it is
true. ``exact`` evaluates the definitions in float64.

Shared-prefix attention (16 query heads, 8 KV heads, head dim 128). The requests of
a group share the rows of one prefix; the keys of a request are its group's prefix
rows, then its own cached rows, then its new rows (one per query row), and query row
r of a request with q rows and n keys sees keys j <= n - q + r:

    out = softmax(scale * Q K^T) V

Logits controls. Row j of request i's chunk x_0 .. x_j (x_0, the newest emitted
token, is in the request's counts already) is changed, token by token, to

    c = count_i[v] + #{1 <= k <= j : x_k = v},    seen = prompt_i[v] or c > 0
    z = logit;  z = z / rep_i if z > 0 else z * rep_i    where seen
    z = (z - freq_i * c) - pres_i                        where c > 0
    z = z + bias_i[v];  z = -inf                         where the row's mask forbids v

and written out, or reduced to the index of its maximum (the lowest one on ties).
"""
import math
import random

import torch

own = False

HQ, HKV, D = 16, 8, 128
SCALE = D ** -0.5
DEVICE = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
VOCAB = 151936


def listed():
    return [
        # the first decode step of a few completions of one short prompt: latency
        dict(name='attn_first_step', kind='attn', dtype='bf16', groups=1, requests=4, prefix=600, cached=0, rows=1,
             ragged=False, shape=1),
        # speculative verify of 32 completions of one 2048-token prompt, up to 128 tokens in
        dict(name='attn_verify_32', kind='attn', dtype='bf16', groups=1, requests=32, prefix=2048, cached=128, rows=8,
             ragged=True, shape=2),
        # plain decoding of a few requests behind a long document: the prefix's bytes bound it
        dict(name='attn_decode_long', kind='attn', dtype='bf16', groups=1, requests=8, prefix=32768, cached=64, rows=1,
             ragged=True, shape=3),
        # a server with several system prompts, ragged in every way
        dict(name='attn_groups', kind='attn', dtype='bf16', groups=9, requests=24, prefix=6000, cached=700, rows=8,
             ragged=True, shape=4),
        # prompt chunks of four users behind one long instruction: long query runs
        dict(name='attn_chunks', kind='attn', dtype='bf16', groups=1, requests=4, prefix=4096, cached=0, rows=777,
             ragged=False, shape=5),
        # the largest: 128 requests x 8 rows behind a 32768-token prefix, products bound it
        dict(name='attn_wide_long', kind='attn', dtype='bf16', groups=1, requests=128, prefix=32768, cached=512,
             rows=8, ragged=False, shape=6),
        # the exact float32 path, ragged
        dict(name='attn_fp32', kind='attn', dtype='fp32', groups=2, requests=8, prefix=1000, cached=200, rows=7,
             ragged=True, shape=7),
        # one decoding step of four requests: penalties alone, latency
        dict(name='logits_decode_4', kind='logits', dtype='bf16', out='bf16', argmax=False, requests=4, rows=1,
             vocab=VOCAB, history=700, bias=0, masks=False, ragged=False, shape=11),
        # a stochastic verify round: bf16 logits to float32, penalties, biases and grammar masks
        dict(name='logits_verify_64', kind='logits', dtype='bf16', out='fp32', argmax=False, requests=64, rows=7,
             vocab=VOCAB, history=3000, bias=40, masks=True, ragged=True, shape=12),
        # float32 logits over an odd vocabulary (rows off every vector boundary)
        dict(name='logits_odd_fp32', kind='logits', dtype='fp32', out='fp32', argmax=False, requests=24, rows=5,
             vocab=50257, history=1500, bias=300, masks=True, ragged=True, shape=13),
        # greedy verify: the controlled maximum of every row, nothing written
        dict(name='logits_greedy_128', kind='logits', dtype='bf16', out='bf16', argmax=True, requests=128, rows=7,
             vocab=VOCAB, history=4000, bias=16, masks=True, ragged=False, shape=14),
        # greedy decoding of a small batch
        dict(name='logits_greedy_8', kind='logits', dtype='bf16', out='bf16', argmax=True, requests=8, rows=1,
             vocab=VOCAB, history=900, bias=0, masks=True, ragged=False, shape=15),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    shape = rng.randrange(1 << 30)
    if rng.random() < 0.55:
        fp32 = rng.random() < 0.15
        prefix = _log(rng, 1, 1500 if fp32 else 32768)
        rows = rng.choice([1, 1, 7, 8, _log(rng, 2, 40), _log(rng, 16, 900)])
        groups = rng.choice([1, 1, 1, 2, _log(rng, 2, 12)])
        requests = _log(rng, 1, 128)
        while groups * requests * rows * (prefix + rows) > (3e6 if fp32 else 3.3e7) or groups * requests * rows > 8192:
            if requests > 1:
                requests = (requests + 1) // 2
            elif groups > 1:
                groups = (groups + 1) // 2
            else:
                rows = (rows + 1) // 2
        cached = rng.choice([0, _log(rng, 1, 1024 if groups * requests > 64 else 4096)])
        return dict(kind='attn', dtype='fp32' if fp32 else 'bf16', groups=groups, requests=requests, prefix=prefix,
                    cached=min(cached, 300) if fp32 else cached, rows=rows, ragged=rng.random() < 0.7, shape=shape)
    vocab = rng.choice([VOCAB, VOCAB, _log(rng, 500, 200000)])
    rows = rng.choice([1, 7, 8, rng.randint(2, 16)])
    requests = _log(rng, 1, 128)
    while requests * rows * vocab > 1.3e8:
        requests = (requests + 1) // 2
    dtype = rng.choice(['bf16', 'bf16', 'fp32'])
    return dict(kind='logits', dtype=dtype, out=rng.choice([dtype, 'fp32']), argmax=rng.random() < 0.4,
                requests=requests, rows=rows, vocab=vocab, history=_log(rng, 1, 8000),
                bias=rng.choice([0, rng.randint(1, 64), 300]), masks=rng.random() < 0.6, ragged=rng.random() < 0.5,
                shape=shape)


# ------------------------------------------------------------------ shapes
def _attn_shape(case):
    """Lengths of a case: prefix rows and request count per group; query, cached and slot rows per request."""
    rng = random.Random(case['shape'])
    ragged = case['ragged']
    prefixes, sizes, queries, cached, gaps = [], [], [], [], []
    for _ in range(case['groups']):
        prefixes.append(rng.randint((case['prefix'] + 3) // 4, case['prefix']) if ragged and case['groups'] > 1
                        else case['prefix'])
        n = rng.randint(1, case['requests']) if ragged and case['groups'] > 1 else case['requests']
        sizes.append(n)
        for _ in range(n):
            queries.append(rng.randint(1, case['rows']) if ragged else case['rows'])
            cached.append(rng.randint(0, case['cached']) if ragged else case['cached'])
            gaps.append(rng.randint(0, 9))          # unused rows behind a request's cached ones
    return prefixes, sizes, queries, cached, gaps


def _pairs(case):
    """Visible (query row, key) pairs of a head."""
    prefixes, sizes, queries, cached, _ = _attn_shape(case)
    total, i = 0, 0
    for p, n in zip(prefixes, sizes):
        for _ in range(n):
            q = queries[i]
            total += q * (p + cached[i]) + q * (q + 1) // 2
            i += 1
    return total


def _chunks(case):
    rng = random.Random(case['shape'])
    return [rng.randint(1, case['rows']) if case['ragged'] else case['rows'] for _ in range(case['requests'])]


def _masked(case):
    """Which rows have a grammar mask (two of three)."""
    n = sum(_chunks(case))
    return [case['masks'] and r % 3 != 1 for r in range(n)]


def work(case):
    if case['kind'] == 'attn':
        prefixes, _, queries, cached, _ = _attn_shape(case)
        size = 2 if case['dtype'] == 'bf16' else 4
        kv = 2 * HKV * D * size * (sum(prefixes) + sum(cached) + sum(queries))
        return {'bytes': kv + 2 * HQ * D * size * sum(queries), 'flops': 4 * HQ * D * _pairs(case)}
    n, v, r = sum(_chunks(case)), case['vocab'], case['requests']
    size = {'bf16': 2, 'fp32': 4}
    read = n * v * size[case['dtype']] + r * v * 2 + r * v // 8 + sum(_masked(case)) * (v // 8) + r * case['bias'] * 8
    return {'bytes': read + (n * 4 if case['argmax'] else n * v * size[case['out']]), 'flops': 3 * n * v}


# ------------------------------------------------------------------ inputs
def _ends(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _prepare_attn(case, g):
    prefixes, sizes, queries, cached, gaps = _attn_shape(case)
    dtype = DTYPES[case['dtype']]
    rows = lambda n, heads: torch.randn((n, heads, D), device=DEVICE, generator=g).to(dtype)  # noqa: E731
    slots = _ends([c + x for c, x in zip(cached, gaps)])
    # keys as after an RMS norm, a few directions stronger: scores of a few units, as trained heads have
    stretch = 0.6 + 1.2 * torch.rand((1, HKV, D), device=DEVICE, generator=g)
    key = lambda n: (torch.randn((n, HKV, D), device=DEVICE, generator=g) * stretch).to(dtype)  # noqa: E731
    state = dict(case=case, prefixes=prefixes, sizes=sizes, queries=queries, cached=cached, slots=slots[:-1],
                 query=rows(sum(queries), HQ), prefix_key=key(sum(prefixes)), prefix_value=rows(sum(prefixes), HKV),
                 key=key(max(slots[-1], 1)), value=rows(max(slots[-1], 1), HKV),
                 new_key=key(sum(queries)), new_value=rows(sum(queries), HKV))
    if own:
        import importlib
        b200 = importlib.import_module('qwen3-dspark_b200')
        device = state['query'].device
        state['layout'] = b200.SharedPrefixLayout.from_lengths(prefixes, sizes, queries, cached, queries,
                                                               own_starts=slots[:-1], device=device)
        state['kernel'] = b200.B200SharedPrefixKernel(device)
    return state


def _prepare_logits(case, g):
    chunks = _chunks(case)
    n, v, r = sum(chunks), case['vocab'], case['requests']
    dev = dict(device=DEVICE)
    # token ids as text has them: a few very often, most of them rarely
    zipf = lambda *s: ((v ** torch.rand(s, generator=g, **dev) - 1) / (v - 1) * v).long().clamp(0, v - 1)  # noqa: E731
    logits = torch.randn((n, v), generator=g, **dev) * 2.5
    prompt, output, tokens = zipf(r, case['history']), zipf(r, max(1, case['history'] // 2)), zipf(n)
    # the model's favourites are often tokens it has used before
    req = torch.tensor([i for i, q in enumerate(chunks) for _ in range(q)], **dev)
    hot = output[req, torch.randint(0, output.shape[1], (n,), generator=g, **dev)]
    logits[torch.arange(n, **dev), hot] += 9.0
    seen = torch.zeros((r, v), **dev).scatter_(1, prompt, 1.0) > 0
    counts = torch.zeros((r, v), **dev).scatter_add_(1, output, torch.ones(output.shape, **dev))
    words = (v + 31) // 32
    state = dict(case=case, logits=logits.to(DTYPES[case['dtype']]), tokens=tokens, seen=seen,
                 counts=counts.to(torch.int16), chunks=chunks,
                 cu_query=torch.tensor(_ends(chunks), dtype=torch.int32, **dev),
                 penalties=torch.stack((1 + 0.5 * torch.rand(r, generator=g, **dev),
                                        0.8 * torch.rand(r, generator=g, **dev),
                                        0.8 * torch.rand(r, generator=g, **dev)), 1),
                 bias_ids=None, bias_values=None, masks=None, mask_index=None)
    if case['bias']:
        b = min(case['bias'], v)
        start = torch.randint(0, v, (r, 1), generator=g, **dev)
        state['bias_ids'] = ((start + torch.arange(b, **dev) * max(1, v // b)) % v).int()     # distinct per request
        state['bias_values'] = torch.randn((r, b), generator=g, **dev) * 4
    if case['masks']:
        masked = _masked(case)
        m = max(sum(masked), 1)
        # a grammar allows a few tokens at most places (one word in 40) and nearly all inside free text
        wide = torch.rand((m, words), generator=g, **dev) < torch.where(
            torch.rand((m, 1), generator=g, **dev) < 0.5, 0.025, 0.98)
        bits = torch.randint(-2 ** 31, 2 ** 31, (m, words), generator=g, dtype=torch.int64, **dev)
        state['masks'] = torch.where(wide, bits, torch.zeros_like(bits)).int()
        state['masks'][:, 0] |= 4                                                             # never empty
        index, k = [], 0
        for x in masked:
            index.append(k if x else -1)
            k += x
        state['mask_index'] = torch.tensor(index, dtype=torch.int32, **dev)
    if own:
        import importlib
        b200 = importlib.import_module('qwen3-dspark_b200')
        controls = b200.TokenControls(r, v, device=state['logits'].device, max_bias=case['bias'])
        for i in range(r):
            controls.add_request(f'r{i}', prompt=prompt[i], output=output[i],
                                 repetition=float(state['penalties'][i, 0]), frequency=float(state['penalties'][i, 1]),
                                 presence=float(state['penalties'][i, 2]),
                                 bias=(state['bias_ids'][i], state['bias_values'][i]) if case['bias'] else None)
        state['controls'] = controls
        state['slots'] = controls.slot_index([f'r{i}' for i in range(r)])
    return state


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 17)
    return (_prepare_attn if case['kind'] == 'attn' else _prepare_logits)(case, g)


# ------------------------------------------------------------------ one pass
def _part(q, k, v, limit):
    """Softmax statistics of q [8, m, 128] over keys k/v [n, 8, 128]; row x sees keys j < limit[x] (None: all)."""
    s = torch.matmul(q, k.permute(1, 2, 0)) * SCALE
    if limit is not None:
        s = s.masked_fill(torch.arange(k.shape[0], device=s.device)[None] >= limit[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.clamp_min(-1e30))
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v.permute(1, 0, 2))


def _plain_attn(st):
    q = st['query'].float()
    out = torch.empty_like(q)
    p0, t0, i = 0, 0, 0
    for plen, n in zip(st['prefixes'], st['sizes']):
        tokens = sum(st['queries'][i:i + n])
        pk, pv = st['prefix_key'][p0:p0 + plen].float(), st['prefix_value'][p0:p0 + plen].float()
        # the group's rows against the prefix, one product per KV head; two query heads share it
        qg = q[t0:t0 + tokens].reshape(tokens, HKV, 2, D).permute(1, 0, 2, 3).reshape(HKV, 2 * tokens, D)
        parts = [_part(qg[h:h + 1], pk[:, h:h + 1], pv[:, h:h + 1], None) for h in range(HKV)]
        m1, l1, a1 = (torch.cat(x) for x in zip(*parts))
        x0 = 0
        for j in range(i, i + n):
            c, nq, s0 = st['cached'][j], st['queries'][j], st['slots'][j]
            k = torch.cat((st['key'][s0:s0 + c], st['new_key'][t0 + x0:t0 + x0 + nq])).float()
            v = torch.cat((st['value'][s0:s0 + c], st['new_value'][t0 + x0:t0 + x0 + nq])).float()
            rows = slice(2 * x0, 2 * (x0 + nq))
            limit = c + 1 + torch.arange(nq, device=q.device).repeat_interleave(2, output_size=2 * nq)
            m2, l2, a2 = _part(qg[:, rows], k, v, limit)
            m = torch.maximum(m1[:, rows], m2)
            w1, w2 = torch.exp(m1[:, rows] - m), torch.exp(m2 - m)
            o = (a1[:, rows] * w1 + a2 * w2) / (l1[:, rows] * w1 + l2 * w2)
            out[t0 + x0:t0 + x0 + nq] = o.reshape(HKV, nq, 2, D).permute(1, 0, 2, 3).reshape(nq, HQ, D)
            x0 += nq
        p0, t0, i = p0 + plen, t0 + tokens, i + n
    return out.to(st['query'].dtype)


def _plain_logits(st):
    case, dev = st['case'], st['logits'].device
    z = st['logits'].float()
    n, v = z.shape
    cu = st['cu_query'].long()
    req = torch.repeat_interleave(torch.arange(len(st['chunks']), device=dev), cu[1:] - cu[:-1], output_size=n)
    pos = torch.arange(n, device=dev) - cu[req]
    # a row counts the proposals of its own chunk up to itself
    k = torch.arange(1, max(st['chunks']) + 1, device=dev)
    at = (cu[req][:, None] + k[None]).clamp_max(n - 1)
    c = st['counts'].float()[req].scatter_add_(1, st['tokens'][at], (k[None] <= pos[:, None]).float())
    rep, freq, pres = (x[req][:, None] for x in st['penalties'].unbind(1))
    z = torch.where(st['seen'][req] | (c > 0), torch.where(z > 0, z / rep, z * rep), z)
    z = torch.where(c > 0, (z - freq * c) - pres, z)
    if st['bias_ids'] is not None:
        z = z + torch.zeros((len(st['chunks']), v), device=dev).scatter_(1, st['bias_ids'].long(),
                                                                         st['bias_values'])[req]
    if st['masks'] is not None:
        bits = (st['masks'][:, :, None] >> torch.arange(32, dtype=torch.int32, device=dev)) & 1
        bits = bits.reshape(st['masks'].shape[0], -1)[:, :v] != 0
        index = st['mask_index'].long()
        z = torch.where(bits[index.clamp_min(0)] | (index < 0)[:, None], z, -math.inf)
    if not case['argmax']:
        return z.to(DTYPES[case['out']])
    at = torch.where(z == z.amax(-1, keepdim=True), torch.arange(v, device=dev, dtype=torch.int32), v)
    return at.amin(-1)


def run(state):
    if state['case']['kind'] == 'attn':
        if not own:
            return _plain_attn(state)
        return state['kernel'](state['query'], state['key'], state['value'], state['layout'], scale=SCALE,
                               prefix_key=state['prefix_key'], prefix_value=state['prefix_value'],
                               new_key=state['new_key'], new_value=state['new_value'])
    if not own:
        return _plain_logits(state)
    import importlib
    b200 = importlib.import_module('qwen3-dspark_b200')
    args = dict(tokens=state['tokens'], cu_query=state['cu_query'], masks=state['masks'],
                mask_index=state['mask_index'])
    if state['case']['argmax']:
        return b200.control_argmax(state['logits'], state['controls'], state['slots'], **args)
    return b200.control_logits(state['logits'], state['controls'], state['slots'],
                               out_dtype=DTYPES[state['case']['out']], **args)


# ------------------------------------------------------------------ float64
def _exact_attn(st):
    """Every request by itself: its keys laid end to end, one softmax over all of them."""
    q = st['query'].double()
    out = torch.zeros_like(q)
    p0, t0, i = 0, 0, 0
    for plen, n in zip(st['prefixes'], st['sizes']):
        for j in range(i, i + n):
            c, nq, s0 = st['cached'][j], st['queries'][j], st['slots'][j]
            new = slice(t0, t0 + nq)
            keys = torch.cat((st['prefix_key'][p0:p0 + plen], st['key'][s0:s0 + c], st['new_key'][new])).double()
            values = torch.cat((st['prefix_value'][p0:p0 + plen], st['value'][s0:s0 + c],
                                st['new_value'][new])).double()
            total = plen + c + nq
            hidden = (torch.arange(total, device=q.device)[None]
                      > (torch.arange(nq, device=q.device) + total - nq)[:, None])
            for h in range(HQ):
                s = (q[new, h] @ keys[:, h // 2].T * SCALE).masked_fill(hidden, -math.inf)
                out[new, h] = torch.softmax(s, -1) @ values[:, h // 2]
            t0 += nq
        p0, i = p0 + plen, i + n
    return out


def _exact_logits(st):
    case = st['case']
    rows = []
    r = 0
    for i, q in enumerate(st['chunks']):
        rep, freq, pres = st['penalties'][i].double()
        c = st['counts'][i].double().clone()
        for j in range(q):
            if j:
                c[st['tokens'][r]] += 1
            x = st['logits'][r].double()
            seen = st['seen'][i] | (c > 0)
            x = torch.where(seen & (x > 0), x / rep, torch.where(seen, x * rep, x))
            x = x - freq * c - pres * (c > 0)
            if st['bias_ids'] is not None:
                x[st['bias_ids'][i].long()] += st['bias_values'][i].double()
            if st['masks'] is not None and int(st['mask_index'][r]) >= 0:
                word = st['masks'][int(st['mask_index'][r])]
                token = torch.arange(case['vocab'], device=x.device)
                x[(word[token // 32] >> (token % 32).int()) & 1 == 0] = -math.inf
            rows.append(torch.nonzero(x == x.max())[0, 0].int() if case['argmax'] else x)
            r += 1
    return torch.stack(rows)


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_attn(state) if case['kind'] == 'attn' else _exact_logits(state)
