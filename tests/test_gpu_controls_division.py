"""The controls' division on the quotients that are hardest to round.

With 24-bit integers A, B the quotient A / B lies |c| / (2 B) ulp from a midpoint (2 N + 1) / 2
of two floats, where c = A 2^24 - (2 N + 1) B (A >= B; 2^25 below). Those with the smallest
|c| are found from the inverse of B modulo a power of two.
"""
import numpy as np
import pytest
import torch

from gpu_util import dev, i32, status_clean

pytestmark = pytest.mark.gpu


def hard_numerators(b, limit):
    """Numerators A in [2^23, 2^24) of the odd divisor b whose quotient is within limit / (2 b) ulp of
    a midpoint."""
    out = []
    for k in (24, 25):
        mod = 1 << k
        inverse = pow(b, -1, mod)
        for c in range(-limit, limit + 1, 2):
            x = -c * inverse % mod                              # 2 N + 1
            x += mod if k == 24 else 0
            if not (1 << 24) <= x < (1 << 25) or not x & 1:
                continue
            a, rest = divmod(x * b + c, mod)
            if rest == 0 and (1 << 23) <= a < (1 << 24) and (a >= b) == (k == 24):
                out.append(a)
    return out


def test_quotients_next_to_midpoints(pkg):
    g = np.random.Generator(np.random.PCG64(11))
    divisors = {int(b) | 1 for b in g.integers(1 << 23, 1 << 24, 1800)}
    divisors |= set(range((1 << 24) - 401, 1 << 24, 2)) | set(range((1 << 23) + 1, (1 << 23) + 201, 2))
    divisors = sorted(divisors)
    rows = [hard_numerators(b, 15) for b in divisors]
    vocab, r = max(map(len, rows)), len(rows)
    assert sum(map(len, rows)) > 10 * r
    a = torch.tensor([x + [1 << 23] * (vocab - len(x)) for x in rows], dtype=torch.float32)
    b = torch.tensor(divisors, dtype=torch.float32)
    a *= 2.0 ** torch.from_numpy(g.integers(-30, -18, (r, 1)))
    b *= 2.0 ** torch.from_numpy(g.integers(-26, -20, r))
    controls = pkg.TokenControls(r, vocab, device=dev())
    controls.penalties[:, 0] = b.to(dev())
    controls.prompt_bits.fill_(-1)                              # every token seen
    got = pkg.control_logits(a.to(dev()), controls, i32(range(r))).cpu()
    assert torch.equal(got, a / b[:, None])
    status_clean(pkg)
