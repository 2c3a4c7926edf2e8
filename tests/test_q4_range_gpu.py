"""4-bit decode over latents of any size that the format holds: scores that climb past a segment's first reference must
not take the sums out of fp32.  The scores come from the rope values alone, so they are small beside huge latents.

Tolerances as for the values at long contexts: the roundings of P and of the output, and the scores' error."""
import math

import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from test_q4_cache_gpu import _cache, _spacious
from test_q4_values import _check

LN2 = math.log(2.0)


def _climb(n, kind, by):
    """Scores in log2 units: low where a segment of either kernel begins, `by` higher afterwards, or the other way."""
    t = torch.arange(n)
    up = {"tile": t % 128 >= 32, "half": t >= 128, "fall": t < 128, "one": t == n - 1}[kind]
    return by * up.float()


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious", [(16, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("kind", ["tile", "half", "fall", "one"])
@pytest.mark.parametrize("exponent", [0, 58, 62, 95, 110, 115])
def test_huge_latents_and_scores_that_climb_within_the_headroom(gpu, H, spacious, kind, exponent):
    lens = [256, 700]
    x = []
    for b, n in enumerate(lens):
        rows = seeded((n, 576), 5 + b, 1.0).double()
        rows[:, :512] *= 2.0 ** exponent
        rows[:, 512:] = 0
        rows[:, 512] = _climb(n, kind, 31.0 if b == 0 else 20.0)
        x.append(rows.to(torch.bfloat16))
    pool, table, sl = _cache(lens, 7, x=x)
    q = torch.zeros(2, H, 576, dtype=torch.bfloat16)
    q[..., 512] = 1.0
    _check(gpu, q, pool, _spacious(table) if spacious else table, sl, LN2)


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious,kind", [(16, False, "half"), (128, True, "tile")])
def test_one_huge_block_is_enough(gpu, H, spacious, kind):
    """A single block of the segment's last key is huge, in any of the 16 places."""
    n = 256
    for block in range(16):
        rows = seeded((n, 576), 9, 1.0)
        rows[:, 512:] = 0
        rows[:, 512] = _climb(n, kind, 31.0)
        rows[n - 1, 32 * block:32 * block + 32] *= 2.0 ** 100
        pool, table, sl = _cache([n], 8, x=[rows.to(torch.bfloat16)])
        q = torch.zeros(1, H, 576, dtype=torch.bfloat16)
        q[..., 512] = 1.0
        _check(gpu, q, pool, _spacious(table) if spacious else table, sl, LN2)
