"""Cases and a float64 evaluation of the shared-prefix attention, from its definition."""
import numpy as np
import torch

HQ, HKV, D = 16, 8, 128
SCALE = D ** -0.5

# name, prefix lengths, group sizes, query lengths, own lengths, new lengths (None: no new source), causal
CASES = [
    ('one_token', [1], [1], [1], [0], [1], True),
    ('one_key_each', [1], [3], [1, 1, 1], [0, 0, 0], [1, 1, 1], True),
    ('no_prefix', [0], [3], [7, 1, 8], [40, 0, 129], [7, 1, 8], True),
    ('no_new_source', [33], [2], [3, 5], [3, 64], None, True),
    ('decode_batch', [600], [4], [1] * 4, [0, 3, 17, 128], [1] * 4, True),
    ('verify_blocks', [257], [9], [8] * 9, [5 * i for i in range(9)], [8] * 9, True),
    ('groups', [130, 0, 1, 512], [3, 2, 1, 20], [7, 1, 8] + [4, 8] + [6] + [1 + i % 8 for i in range(20)],
     [0, 9, 31] + [128, 5] + [200] + [(37 * i) % 150 for i in range(20)],
     [7, 1, 8] + [4, 8] + [6] + [1 + i % 8 for i in range(20)], True),
    ('long_queries', [200], [2], [150, 130], [10, 0], [150, 130], True),
    ('one_long_request', [300], [1], [333], [77], [333], True),
    ('mixed_lengths', [384], [5], [1, 140, 2, 1, 70], [500, 3, 0, 64, 1], [1, 140, 2, 1, 70], True),
    ('tile_edges', [128, 256], [2, 3], [64, 64, 1, 63, 65], [64, 0, 127, 128, 129], [64, 64, 1, 63, 65], True),
    ('empty_queries', [100], [4], [0, 3, 0, 5], [7, 8, 0, 9], [0, 3, 0, 5], True),
    ('noncausal', [70, 0], [3, 2], [7, 3, 1, 9, 2], [11, 0, 140, 3, 0], [7, 3, 0, 9, 0], False),
    ('prefix_only', [300], [6], [2, 7, 1, 1, 8, 30], [0] * 6, None, False),
    ('split_prefix', [5000], [3], [4, 8, 1], [10, 0, 300], [4, 8, 1], True),
    ('split_own', [64], [2], [3, 8], [4000, 20], [3, 8], True),
]


def starts_of(lengths, gap):
    """Back-to-back starts with ``gap`` unused rows between the slots; returns (starts, rows)."""
    out, at = [], gap
    for n in lengths:
        out.append(at)
        at += n + gap
    return out, at


def inputs(seed, case, gap=3):
    """Rounded-to-bf16 float32 inputs; unused rows are NaN. Returns a dict of tensors and starts."""
    _, plen, sizes, qlen, own, new, _ = case
    g = np.random.Generator(np.random.PCG64(seed))

    def rows(n, heads):
        return torch.from_numpy(g.standard_normal((n, heads, D), dtype=np.float32)).bfloat16().float()

    out = dict(q=rows(sum(qlen), HQ))
    for name, lengths in (('p', plen), ('a', own), ('b', new)):
        if lengths is None:
            continue
        starts, total = starts_of(lengths, gap)
        k, v = rows(total, HKV), rows(total, HKV)
        used = torch.zeros(total, dtype=torch.bool)
        for s, n in zip(starts, lengths):
            used[s:s + n] = True
        k[~used], v[~used] = float('nan'), float('nan')
        out[name] = (starts, k, v)
    return out


def exact(x, case):
    """(out, weight, score): float64 output, sum_j p_j |v_j| of each element and the largest
    |q| . |k| * scale of each (row, head), for error bounds."""
    _, plen, sizes, qlen, own, new, causal = case
    q = x['q'].double()
    out, weight = torch.zeros_like(q), torch.zeros_like(q)
    score = torch.zeros(q.shape[:2], dtype=torch.float64)
    t, i = 0, 0
    for g, n in enumerate(sizes):
        for _ in range(n):
            parts = [(x['p'], plen[g], g), (x['a'], own[i], i)] + ([(x['b'], new[i], i)] if new is not None else [])
            k = torch.cat([s[1][s[0][j]:s[0][j] + m] for s, m, j in parts]).double()
            v = torch.cat([s[2][s[0][j]:s[0][j] + m] for s, m, j in parts]).double()
            nq, nk = qlen[i], len(k)
            for h in range(HQ):
                if nk == 0:
                    continue
                s = q[t:t + nq, h] @ k[:, h // 2].T * SCALE
                a = q[t:t + nq, h].abs() @ k[:, h // 2].T.abs() * SCALE
                if causal:
                    hide = torch.arange(nk)[None] > torch.arange(nq)[:, None] + nk - nq
                    s, a = s.masked_fill(hide, float('-inf')), a.masked_fill(hide, 0.0)
                p = torch.softmax(s, -1)
                out[t:t + nq, h] = p @ v[:, h // 2]
                weight[t:t + nq, h] = p @ v[:, h // 2].abs()
                if nq:
                    score[t:t + nq, h] = a.amax(-1)
            t += nq
            i += 1
    return out, weight, score


def layout(pkg, x, case, device, grid_limit=None):
    _, plen, sizes, qlen, own, new, causal = case
    return pkg.SharedPrefixLayout.from_lengths(
        plen, sizes, qlen, own, new, prefix_starts=x['p'][0], own_starts=x['a'][0],
        new_starts=x['b'][0] if new is not None else None, causal=causal, device=device, grid_limit=grid_limit)
