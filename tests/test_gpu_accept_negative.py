"""Greedy acceptance with negative predictions (a row whose mask allows no token): such a row
commits nothing of its own and ends the request's round, whatever is proposed behind it."""
import pytest
import torch

from gpu_util import dev, i32, status_clean

pytestmark = pytest.mark.gpu


def accept(pkg, pred, tokens, cu, eos=()):
    r, n = len(cu) - 1, len(pred)
    p, t, c = i32(pred), torch.tensor(tokens, device=dev()), i32(cu)
    e = torch.tensor(list(eos), dtype=torch.long, device=dev())
    counts = torch.full((2 * r,), 99, dtype=torch.int32, device=dev())
    emitted = torch.full((n,), 99, dtype=torch.long, device=dev())
    status = pkg.load_library().dspark_greedy_accept(
        p.data_ptr(), t.data_ptr(), c.data_ptr(), r, n, e.data_ptr() if eos else None, len(eos), None,
        counts.data_ptr(), counts[r:].data_ptr(), emitted.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0
    status_clean(pkg)
    return counts[:r].tolist(), counts[r:].tolist(), emitted.tolist()


def test_a_negative_proposal_never_matches_a_negative_prediction(pkg):
    # chunks: padded with -1 behind the first proposal; all padding; a single row
    pred = [5, -1, 7, 8] + [-1, -1, -1] + [-1]
    tokens = [1, 5, -1, 7] + [2, -1, -1] + [3]
    accepted, commit, emitted = accept(pkg, pred, tokens, [0, 4, 7, 8])
    assert accepted == [1, 0, 0] and commit == [1, 0, 0]
    assert emitted == [5, -1, -1, -1] + [-1] * 3 + [-1]


def test_prediction_before_a_negative_one_is_committed(pkg):
    pred = [5, 6, -1] + [4, -1]
    tokens = [1, 5, 6] + [9, 8]
    accepted, commit, emitted = accept(pkg, pred, tokens, [0, 3, 5], eos=(17,))
    assert accepted == [2, 0] and commit == [2, 1]
    assert emitted == [5, 6, -1] + [4, -1]
