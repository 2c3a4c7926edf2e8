"""Chunk attention over the paged cache against a plain 64-bit form: lengths from one token on, odd heads, rows and
pages, strides, empty queries, what lies behind a sequence and behind a query."""
import math

import pytest
import torch

from paging import D_QK, D_V, PAGE, assert_attention, attention64, ints, paged, starts

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(192.0)


def queries(T, H, seed, scale=0.5):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(T, H, D_QK, generator=g) * scale).to(torch.bfloat16)


def reference(q, rows, lens, counts, causal=True, scale=SCALE):
    parts, at = [], 0
    for r, N, n in zip(rows, lens, counts):
        ends = [N - n + i + 1 if causal else N for i in range(n)]
        parts.append(attention64(q[at:at + n], r, ends, scale))
        at += n
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("H,lens,counts", [
    (128, [1], [1]),
    (128, [5], [5]),
    (16, [1, 64, 65, 130], [1, 1, 1, 1]),
    (16, [33, 200, 7], [33, 9, 2]),
    (1, [300, 64], [290, 64]),
    (5, [97, 31, 1000], [50, 31, 3]),
    (20, [129, 0, 63], [17, 0, 1]),
    (96, [70, 40], [3, 40]),
    (128, [2000], [3]),
    (128, [191, 640], [64, 2]),
    (130, [100], [3]),
    (300, [66], [2]),
    (16, [4500], [1]),
    (64, [33] * 40, [1] * 40),
])
@pytest.mark.parametrize("causal", [True, False])
def test_against_64_bits(gpu, H, lens, counts, causal):
    from python import ops
    pool, table, rows = paged(lens, gpu, seed=H)
    q = queries(sum(counts), H, H)
    o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), pool, table, ints(lens, gpu), ints(starts(counts), gpu),
                                        softmax_scale=SCALE, causal=causal, return_lse=True)
    assert_attention(o, lse, reference(q, rows, lens, counts, causal))


@pytest.mark.parametrize("H", [1, 16, 40, 128])
def test_one_query_per_sequence(gpu, H):
    """Without starts: the same bits as with starts of one query each, and what the decode gives within both roundings."""
    from python import ops
    lens = [1, 77, 64, 0, 513]
    pool, table, rows = paged(lens, gpu, seed=H)
    q = queries(len(lens), H, H).to(gpu)
    args = (q, pool, table, ints(lens, gpu))
    o, lse = ops.flash_dmla_chunk_paged(*args, softmax_scale=SCALE, return_lse=True)
    assert_attention(o, lse, reference(q.cpu(), rows, lens, [1] * 5))
    o2, lse2 = ops.flash_dmla_chunk_paged(*args, ints(range(6), gpu), softmax_scale=SCALE, return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_queries_without_tokens_and_behind_the_last_sequence(gpu):
    """More queries than tokens (a length that was cut), sequences of length 0, packed rows behind the last one."""
    from python import ops
    lens, counts = [3, 0, 40, 0], [6, 2, 45, 0]
    pool, table, rows = paged(lens, gpu)
    T = sum(counts) + 11
    q = queries(T, 16, 1)
    q[-11:] = float("nan")
    o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), pool, table, ints(lens, gpu), ints(starts(counts), gpu),
                                        softmax_scale=SCALE, return_lse=True)
    assert_attention(o[:-11], lse[:-11], reference(q, rows, lens, counts))
    assert (o[-11:] == 0).all() and (lse[-11:] == float("-inf")).all()


def test_lengths_past_the_table_are_cut(gpu):
    from python import ops
    pool, table, rows = paged([128], gpu)
    q = queries(4, 16, 2)
    lens = [128 + 7]   # two pages: 128 tokens
    o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), pool, table, ints(lens, gpu), ints([0, 4], gpu), softmax_scale=SCALE,
                                        return_lse=True)
    assert_attention(o, lse, reference(q, rows, [128], [4]))


@pytest.mark.parametrize("H", [1, 16, 48])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_a_query_does_not_attend_does_not_reach_it(gpu, H, value):
    """Tokens after a query's own, in its tile and its row tile, may hold anything; those that see them get it."""
    from python import ops
    lens, counts = [90], [60]
    pool, table, rows = paged(lens, gpu)
    q = queries(60, H, 3)
    ref = reference(q, rows, lens, counts)
    for bad in ([45], [31, 32, 77], list(range(60, 90))):
        p = pool.clone()
        for j in bad:
            p[table[0, j // PAGE].item(), j % PAGE, 5] = value
        o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), p, table, ints(lens, gpu), ints([0, 60], gpu), softmax_scale=SCALE,
                                            return_lse=True)
        clean = max(0, bad[0] - 30)   # query i is token 30 + i
        if clean:
            assert_attention(o[:clean], lse[:clean], [x[:clean] for x in ref], f"{value} at {bad}")
        assert not torch.isfinite(o[clean:, :, 5]).any(), "a query that attends it"


@pytest.mark.parametrize("steepest", [4.0, 60.0])
def test_huge_latents_and_climbing_scores_stay_finite(gpu, steepest):
    """Values of 2^110 under scores that climb by tens and by hundreds: sums and outputs stay finite."""
    from python import ops
    N = 400
    rows = torch.zeros(N, D_QK)
    rows[:, :D_V] = 2.0 ** 110
    rows[:, D_V] = torch.linspace(0, 60, N)
    rows = rows.to(torch.bfloat16)
    pool = torch.zeros(7, PAGE, D_QK, dtype=torch.bfloat16)
    pool[:6] = rows[:384].view(6, PAGE, D_QK)
    pool[6, :16] = rows[384:]
    q = torch.zeros(3, 16, D_QK)
    q[:, :, D_V] = torch.linspace(0.1, steepest, 16)
    q = q.to(torch.bfloat16)
    o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), pool.to(gpu), ints([list(range(7))], gpu), ints([N], gpu), ints([0, 3], gpu),
                                        softmax_scale=SCALE, return_lse=True)
    assert_attention(o, lse, reference(q, [rows], [N], [3]))


def test_strides(gpu):
    """Queries with heads and tokens apart, a pool with rows and pages apart, a table with wider rows."""
    from python import ops
    lens, counts, H = [150, 20], [40, 20], 16
    pool, table, rows = paged(lens, gpu)
    q = queries(60, H, 4)
    q2 = torch.full((60, H + 3, D_QK + 8), float("nan"), dtype=torch.bfloat16, device=gpu)
    q2[:, :H, :D_QK] = q.to(gpu)
    p2 = torch.full((pool.shape[0], PAGE + 2, D_QK + 24), float("nan"), dtype=torch.bfloat16, device=gpu)
    p2[:, :PAGE, :D_QK] = pool
    t2 = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32, device=gpu)
    t2[:, :table.shape[1]] = table
    o, lse = ops.flash_dmla_chunk_paged(q2[:, :H, :D_QK], p2[:, :PAGE, :D_QK], t2[:, :table.shape[1]], ints(lens, gpu),
                                        ints(starts(counts), gpu), softmax_scale=SCALE, return_lse=True)
    assert_attention(o, lse, reference(q, rows, lens, counts))
    by_head = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    o2, lse2 = ops.flash_dmla_chunk_paged(by_head, pool, table, ints(lens, gpu), ints(starts(counts), gpu),
                                          softmax_scale=SCALE, return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_bad_pages_are_never_read(gpu):
    """A page outside the pool: NaN for the queries that attend it, nothing for the others."""
    from python import ops
    lens, counts, H = [200, 130], [200, 2], 16
    pool, table, rows = paged(lens, gpu)
    q = queries(202, H, 5)
    ref = reference(q, rows, lens, counts)
    for bad in (-1, pool.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 2] = bad
        o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), pool, t, ints(lens, gpu), ints(starts(counts), gpu), softmax_scale=SCALE,
                                            return_lse=True)
        good = torch.arange(202) < 128
        good[200:] = True
        assert_attention(o[good.to(gpu)], lse[good.to(gpu)], [x[good] for x in ref])
        assert torch.isnan(o[~good.to(gpu)]).all() and torch.isnan(lse[~good.to(gpu)]).all()


def test_a_call_is_the_prefill_and_the_decode(gpu):
    """A whole prompt equals the dense prefill over the same rows, within both roundings of P and of the output."""
    from python import ops
    N, H = 200, 16
    pool, table, rows = paged([N], gpu)
    q = queries(N, H, 6).to(gpu)
    o, lse = ops.flash_dmla_chunk_paged(q, pool, table, ints([N], gpu), ints([0, N], gpu), softmax_scale=SCALE, return_lse=True)
    ref = reference(q.cpu(), rows, [N], [N])
    assert_attention(o, lse, ref)
    dense, m, l = ops.flash_dmla_fwd(q.transpose(0, 1)[None].contiguous(), rows[0][None].to(gpu), D_V, SCALE, True)
    assert_attention(dense[0].transpose(0, 1), (m + torch.log(l))[0].T, ref)


def test_repeated_calls_give_the_same_bits(gpu):
    from python import ops
    lens, counts = [700, 90, 1500], [130, 1, 70]
    pool, table, _ = paged(lens, gpu)
    q = queries(201, 16, 7).to(gpu)
    args = (q, pool, table, ints(lens, gpu), ints(starts(counts), gpu))
    first = ops.flash_dmla_chunk_paged(*args, return_lse=True)
    for _ in range(3):
        again = ops.flash_dmla_chunk_paged(*args, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
