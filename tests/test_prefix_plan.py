"""Host logic of the shared-prefix attention, on the CPU.

``dspark_prefix_plan`` cuts the queries into tiles, their key chains into pieces and
assigns the pieces to CTAs. The interpreter below walks the plan's items and merge runs
as the kernels do, in float64, and must reproduce the attention of the definition; every
partial row is written once, and every output row comes from one direct item or one run.
"""
import ctypes

import numpy as np
import pytest
import torch

from prefix_util import CASES, D, HQ, SCALE, exact, inputs, layout

HEAD, ITEM, RUN, REQ = 32, 20, 12, 8
BLOCK = 128


def interpret(plan, x, case):
    plan = plan.numpy().astype(np.int64)
    total, grid, n_items, cta_at, items_at = (int(plan[i]) for i in (2, 3, 4, 5, 6))
    slots, n_runs, runs_at, token_at = (int(plan[i]) for i in (8, 9, 10, 11))
    src = [tuple(t.double() for t in x[n][1:]) if n in x else None for n in 'pab']
    q = x['q'].double()
    out = torch.full((total, HQ, D), float('nan'), dtype=torch.float64)
    part = {}
    offs = plan[cta_at:cta_at + grid + 1]
    assert offs[0] == 0 and offs[-1] == n_items and (np.diff(offs) >= 0).all()
    for it in plan[items_at:items_at + n_items * ITEM].reshape(n_items, ITEM):
        q0, nq, head, slot, visible, nseg, dual = (int(v) for v in it[:7])
        assert 1 <= nq <= 128 and 0 <= head < 8 and 0 <= nseg <= 3
        keys, values, pos, block, len_b = [], [], [], [], 0
        for s in range(nseg):
            which, row, n, at = (int(v) for v in it[8 + 4 * s:12 + 4 * s])
            assert n >= 1
            keys.append(src[which][0][row:row + n, head])
            values.append(src[which][1][row:row + n, head])
            pos.append(torch.arange(at, at + n))
            block += [len_b + i // BLOCK for i in range(n)]
            len_b += -(-n // BLOCK)
        if dual:                       # even blocks to the first slot, odd ones to the second
            assert nq <= 64 and slot >= 0 and len_b >= 2
            k, v, p, b = torch.cat(keys), torch.cat(values), torch.cat(pos), torch.tensor(block)
            for half in range(2):
                for t in range(nq):
                    for g in range(2):
                        see = (p < visible + t) & (b % 2 == half)
                        s = (k[see] @ q[q0 + t, 2 * head + g]) * SCALE
                        key = (slot + half, 2 * t + g)
                        assert key not in part and key[0] < slots
                        part[key] = ((torch.logsumexp(s, 0), torch.softmax(s, 0) @ v[see]) if see.any()
                                     else (torch.tensor(-np.inf), torch.zeros(D, dtype=torch.float64)))
            continue
        for t in range(nq):
            for g in range(2):
                h = 2 * head + g
                if keys:
                    k, v, p = torch.cat(keys), torch.cat(values), torch.cat(pos)
                    see = p < visible + t
                    s = (k[see] @ q[q0 + t, h]) * SCALE
                    lse = torch.logsumexp(s, 0) if see.any() else torch.tensor(-np.inf)
                    o = torch.softmax(s, 0) @ v[see] if see.any() else torch.zeros(D, dtype=torch.float64)
                else:
                    lse, o = torch.tensor(-np.inf), torch.zeros(D, dtype=torch.float64)
                if slot < 0:
                    assert torch.isnan(out[q0 + t, h]).all()
                    out[q0 + t, h] = o
                else:
                    key = (slot + (t >> 6), 2 * (t & 63) + g)
                    assert key not in part and key[0] < slots
                    part[key] = (lse, o)
    if slots:
        token_run = plan[token_at:token_at + total]
        runs = plan[runs_at:runs_at + n_runs * RUN].reshape(n_runs, RUN)
        for t in range(total):
            if token_run[t] < 0:
                continue
            run = runs[token_run[t]]
            assert run[0] <= t < run[0] + run[1] and 1 <= run[2] <= 2
            for h in range(HQ):
                parts = []
                for c in range(int(run[2])):
                    slot, pieces, mma, q0 = (int(v) for v in run[4 + 4 * c:8 + 4 * c])
                    lt = t - q0
                    for p in range(pieces):
                        if mma == 3:
                            parts += [part[(slot + (p * 8 + h // 2) * 2 + i, 2 * lt + (h & 1))] for i in range(2)]
                            continue
                        parts.append(part[(slot + (p * 8 + h // 2) * mma + (lt >> 6), 2 * (lt & 63) + (h & 1))])
                lse = torch.stack([torch.as_tensor(a, dtype=torch.float64) for a, _ in parts])
                top = torch.logsumexp(lse, 0)
                w = torch.exp(lse - top) if torch.isfinite(top) else torch.zeros_like(lse)
                assert torch.isnan(out[t, h]).all()
                out[t, h] = (w[:, None] * torch.stack([o for _, o in parts])).sum(0)
    return out


SMALL = [c for c in CASES if sum(c[3]) <= 120]


@pytest.mark.parametrize('grid', [1, 5, 148])
@pytest.mark.parametrize('case', SMALL, ids=[c[0] for c in SMALL])
def test_plan_reproduces_attention(pkg, case, grid):
    x = inputs(7, case)
    lay = layout(pkg, x, case, 'cpu', grid_limit=grid)
    assert int(lay.head[3]) <= grid
    got = interpret(lay.plan, x, case)
    ref, _, _ = exact(x, case)
    # float64 throughout: differences come from the order of float64 sums alone
    assert torch.isfinite(got).all() and (got - ref).abs().max() < 1e-12


@pytest.mark.parametrize('case', CASES, ids=[c[0] for c in CASES])
def test_plan_covers_every_row_and_key_once(pkg, case):
    """Rows x heads x keys: the items' (row, key) pairs are exactly the visible ones."""
    _, plen, sizes, qlen, own, new, causal = case
    x = inputs(1, case)
    lay = layout(pkg, x, case, 'cpu', grid_limit=148)
    plan = lay.plan.numpy().astype(np.int64)
    items = plan[plan[6]:plan[6] + plan[4] * ITEM].reshape(-1, ITEM)
    pairs = np.zeros((8, sum(qlen)), dtype=np.int64)
    for it in items:
        t = np.arange(it[1])
        for s in range(it[5]):
            _, _, n, at = it[8 + 4 * s:12 + 4 * s]
            pairs[it[2], it[0] + t] += np.clip(it[4] + t - at, 0, n)
    want, i = [], 0
    for g, n in enumerate(sizes):
        for _ in range(n):
            keys = plen[g] + own[i] + (new[i] if new is not None else 0)
            want += [keys - qlen[i] + r + 1 if causal else keys for r in range(qlen[i])]
            i += 1
    assert (pairs == np.array(want, dtype=np.int64)[None]).all()


def test_schedule_is_balanced_and_splits_long_prefixes(pkg):
    # 8 rows behind 32768 shared keys: every CTA of 148 gets a share
    lay = pkg.SharedPrefixLayout.from_lengths([32768], [8], [1] * 8, [0] * 8, [1] * 8, device='cpu', grid_limit=148)
    plan = lay.plan.numpy()
    assert plan[3] == 148
    blocks = []
    for c in range(148):
        a, b = plan[plan[5] + c], plan[plan[5] + c + 1]
        blocks.append(sum(-(-int(plan[plan[6] + i * ITEM + 10 + 4 * s]) // BLOCK) for i in range(a, b)
                          for s in range(plan[plan[6] + i * ITEM + 5])))
    assert max(blocks) <= 1.4 * (sum(blocks) / 148) + 2


def test_refusals(pkg):
    make = pkg.SharedPrefixLayout.from_lengths
    ok = dict(prefix_lengths=[4], group_sizes=[2], query_lengths=[1, 2], own_lengths=[0, 3], new_lengths=[1, 2],
              device='cpu', grid_limit=4)
    make(**ok)
    for bad in (dict(group_sizes=[1]), dict(group_sizes=[3]), dict(group_sizes=[0, 2], prefix_lengths=[4, 4]),
                dict(prefix_lengths=[-1]), dict(prefix_lengths=[4, 4]), dict(query_lengths=[1, -2]),
                dict(own_lengths=[0]), dict(new_lengths=[0, 2]), dict(new_lengths=None, own_lengths=[0, 2]),
                dict(prefix_starts=[1, 2]), dict(own_starts=[-1, 0]), dict(prefix_lengths=[2 ** 30]),
                dict(new_lengths=None, own_lengths=[1, 2], new_starts=[0, 0]), dict(causal=1), dict(grid_limit=0),
                dict(query_lengths=[], group_sizes=[], prefix_lengths=[], own_lengths=[], new_lengths=[])):
        with pytest.raises(ValueError):
            make(**{**ok, **bad})
    with pytest.raises(RuntimeError):        # starts in range, rows past the index limit
        make(**{**ok, 'own_starts': [0, 2 ** 30 - 1]})


def test_native_entries_refuse_before_any_device_work(pkg):
    lib = pkg.load_library()
    lay = pkg.SharedPrefixLayout.from_lengths([4], [1], [1], [0], [1], device='cpu', grid_limit=4)
    head = lay.head.data_ptr()
    f = ctypes.c_void_p(4096)
    call = lambda q=f, tq=1, pk=f, rows=8, off=0, hd=head, plan=f, scale=0.1, dt=0, out=f: lib.dspark_prefix_attn(  # noqa: E731
        q, tq, pk, f, rows, off, f, f, 8, 0, f, f, 8, 0, hd, plan, scale, dt, out, f, 1 << 20, None)
    for kw in (dict(q=None), dict(tq=2), dict(pk=None), dict(rows=3), dict(off=5), dict(off=-1), dict(hd=None),
               dict(plan=None), dict(plan=ctypes.c_void_p(4100)), dict(scale=0.0), dict(dt=2), dict(out=None),
               dict(q=ctypes.c_void_p(4098)), dict(rows=2 ** 31)):
        assert call(**kw) == 1, kw
    assert lib.dspark_prefix_workspace_bytes(None) == 0
    words = ctypes.c_longlong(0)
    assert lib.dspark_prefix_plan(1, None, None, None, 1, None, None, None, None, None, 1, 4, None, 0,
                                  ctypes.byref(words)) == 1


def test_kernel_refuses_without_a_gpu(pkg):
    with pytest.raises(RuntimeError):
        pkg.B200SharedPrefixKernel('cpu')
    with pytest.raises(RuntimeError):
        pkg.TokenControls(2, 100, device='cpu')
