"""Heads that a decode step left out (lse = -inf) add nothing to the accounts, whatever their queries and keys hold.

Their scores may be infinite or not a number: queries of heads that are not in use, the padding of a head group
(a copy of the last head's queries), an infinity in a key's rope values.  Accounts of the other heads are those of a
call without the head: the same bits where the head's place in the sum is empty either way."""
import math

import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from python import ops
from test_evict_gpu import SCALE, _lse, _pool


def _account(gpu, q, pool, table, sl, lse, mass):
    got = mass.to(gpu)
    ops.flash_dmla_attn_mass(q.to(gpu), pool.to(gpu), table.to(gpu), sl.to(gpu), lse.to(gpu), got, SCALE)
    return got.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("H", [1, 20, 32, 100, 128, 200])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_of_inactive_heads_do_not_count(gpu, q4, H, value):
    lens = [200, 0, 1, 700]
    pool, table, sl = _pool(lens, 31, q4)
    q = seeded((4, H, 576), 32, 0.5, torch.bfloat16)
    lse = _lse(q, pool, table, sl)
    off = sorted({0, H // 2, H - 1})   # the last head's queries stand in for heads past the last one
    lse[:, off] = -math.inf
    mass = seeded((4, table.shape[1] * 64), 33).abs()
    good = _account(gpu, q, pool, table, sl, lse, mass)
    ref = R.attn_mass(q, pool, table, sl, lse, mass, SCALE)
    assert torch.allclose(good.double(), ref, rtol=2e-4, atol=1e-6)
    for dims in (slice(0, 576), slice(5, 6), slice(520, 521)):
        bad = q.clone()
        bad[:, off, dims] = value
        assert torch.equal(_account(gpu, bad, pool, table, sl, lse, mass), good)


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
def test_keys_that_are_not_numbers_leave_accounts_without_active_heads(gpu, q4):
    """A sequence whose heads are all inactive keeps its accounts, also of tokens whose keys are infinite or not numbers;
    an active head's account of such a token is not a number, and of the others as before."""
    lens = [150, 150]
    pool, table, sl = _pool(lens, 41, q4)
    q = seeded((2, 40, 576), 42, 0.5, torch.bfloat16)
    lse = _lse(q, pool, table, sl)
    lse[0] = -math.inf
    mass = seeded((2, table.shape[1] * 64), 43).abs()
    good = _account(gpu, q, pool, table, sl, lse, mass)
    assert torch.equal(good[0], mass[0])
    bad = pool.clone()
    for b in range(2):
        page = int(table[b, 1])
        if q4:
            bad[page, 3, 260] = 255                                    # a block that is not a number
            bad[page, 9, 272:274] = torch.tensor([0x80, 0x7f], dtype=torch.uint8)   # an infinite rope value
        else:
            bad[page, 3, 100] = math.nan
            bad[page, 9, 512] = math.inf
    got = _account(gpu, q, bad, table, sl, lse, mass)
    assert torch.equal(got[0], mass[0])
    assert got[1, 64 + 3].isnan()
    got[1, [64 + 3, 64 + 9]] = good[1, [64 + 3, 64 + 9]]
    assert torch.equal(got[1], good[1])
