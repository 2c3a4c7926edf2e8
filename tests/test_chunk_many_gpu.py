"""Chunk attention where its cut into ranges can go wrong: hundreds of sequences with empty ones between, tables of
a million pages, row tiles in two parts and in hundreds; and rows few enough that the waves share their scores."""
import math
import random

import pytest
import torch

from paging import D_QK, D_V, PAGE, assert_attention, attention64, ints, pages, paged, starts

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(192.0)


def queries(T, H, seed, scale=0.5):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(T, H, D_QK, generator=g) * scale).to(torch.bfloat16)


def check(q, o, lse, rows, lens, counts, causal=True, some=None, what=""):
    """Against the plain form, of `some` queries or of all."""
    at, o, lse = 0, o.cpu(), lse.cpu()
    for r, N, n in zip(rows, lens, counts):
        mine = [i for i in range(n) if some is None or at + i in some]
        if mine:
            at_these = [at + i for i in mine]
            ref = attention64(q[at_these], r, [N - n + i + 1 if causal else N for i in mine], SCALE)
            assert_attention(o[at_these], lse[at_these], ref, what or f"queries {at_these[0]} to {at_these[-1]}")
        at += n


def run(gpu, q, pool, table, lens, counts, causal=True):
    from python import ops
    return ops.flash_dmla_chunk_paged(q.to(gpu), pool, table, ints(lens, gpu), ints(starts(counts), gpu), softmax_scale=SCALE,
                                      causal=causal, return_lse=True)


@pytest.mark.parametrize("H", [1, 16, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_hundreds_of_sequences(gpu, H, causal):
    r = random.Random(H)
    lens = [r.choice([0, 1, 31, 64, r.randint(1, 200)]) for _ in range(700)]
    counts = [r.choice([0, 0, 1, 1, 2, 5]) for _ in lens]
    pool, table, rows = paged(lens, gpu, seed=H)
    q = queries(sum(counts), H, H)
    o, lse = run(gpu, q, pool, table, lens, counts, causal)
    check(q, o, lse, rows, lens, counts, causal)


@pytest.mark.parametrize("B,only", [(257, 256), (600, 599), (600, 0), (1025, 512), (3000, 2047)])
@pytest.mark.parametrize("H,n,N", [(16, 1, 70), (128, 3, 1000)])
def test_one_sequence_among_empty_ones(gpu, B, only, H, n, N):
    """A padded batch: the other sequences have neither tokens nor queries, or tokens alone."""
    lens, counts = [0] * B, [0] * B
    lens[only], counts[only] = N, n
    if only > 3:
        lens[3] = 100
    pool, table, rows = paged(lens, gpu)
    q = queries(n, H, 1)
    o, lse = run(gpu, q, pool, table, lens, counts)
    check(q, o, lse, rows, lens, counts)


@pytest.mark.parametrize("B", [1, 255, 256, 257, 800])
def test_batches_without_a_token(gpu, B):
    pool, table, _ = paged([0] * B, gpu)
    o, lse = run(gpu, queries(B, 16, 1), pool, table, [0] * B, [1] * B)
    assert (o == 0).all() and (lse == float("-inf")).all()


@pytest.mark.parametrize("H,lens,counts", [
    (16, [300], [1]), (16, [900], [1]), (16, [2500, 2500], [1, 1]), (16, [20000], [1]), (16, [20000, 11], [2, 1]),
    (128, [300], [1]), (128, [700, 900], [1, 1]), (128, [3000] * 9, [1] * 9), (128, [17000] * 3, [1] * 3), (128, [30000], [1]),
    (20, [9000] * 5, [1, 2, 3, 9, 17]), (33, [4000, 1000], [3, 40]), (64, [1500] * 30, [2] * 30)])
def test_row_tiles_in_parts(gpu, H, lens, counts):
    """Two parts of a row tile and hundreds, of all 128 rows and of few."""
    pool, table, rows = paged(lens, gpu, seed=H)
    q = queries(sum(counts), H, H)
    o, lse = run(gpu, q, pool, table, lens, counts)
    check(q, o, lse, rows, lens, counts)


@pytest.mark.parametrize("H", [16, 128])
def test_parts_without_a_weight(gpu, H):
    """Scores of minus infinity over many parts: a query sees the other tokens alone."""
    N = 9000
    pool, table, rows = paged([N], gpu)
    q = queries(1, H, 2)
    q[:, :, D_V] = q[:, :, D_V].abs() + 1
    for gone in (range(0, 8000), range(100, 8991), range(1000, 9000)):
        p = pool.clone()
        for j in range(gone[0] // PAGE, gone[-1] // PAGE + 1):
            a, b = max(gone[0] - PAGE * j, 0), min(gone[-1] + 1 - PAGE * j, PAGE)
            p[table[0, j].item(), a:b, D_V] = float("-inf")
        o, lse = run(gpu, q, p, table, [N], [1])
        left = rows[0][[j for j in range(N) if j not in gone]]
        ref = attention64(q, left, [len(left)], SCALE)
        assert_attention(o, lse, ref, f"without {gone}")


@pytest.mark.parametrize("H", [16, 128])
def test_not_a_number_in_one_part_reaches_the_rows_that_see_it(gpu, H):
    lens, counts = [9000, 5000], [3, 2]
    pool, table, rows = paged(lens, gpu)
    q = queries(5, H, 3)
    for at in (0, 4000, 8998):
        p = pool.clone()
        p[table[0, at // PAGE].item(), at % PAGE, 7] = float("nan")
        o, lse = run(gpu, q, p, table, lens, counts)
        clean = [i for i in range(5) if i >= 3 or 8997 + i < at]
        check(q, o, lse, rows, lens, counts, some=clean)
        hit = [i for i in range(5) if i not in clean]
        assert torch.isnan(o[hit]).any(2).all()


def test_tables_of_a_million_pages(gpu):
    """The weights of a row tile pass 32 bits where each may have a million pages: they are taken in larger units."""
    lens, counts, H = [9000, 700], [8000, 200], 64
    pool, table, rows = paged(lens, gpu)
    wide = torch.full((2, 1 << 20), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    q = queries(sum(counts), H, 4)
    o, lse = run(gpu, q, pool, wide, lens, counts)
    r = random.Random(1)
    check(q, o, lse, rows, lens, counts, some=set([0, 7999, 8000, 8199] + r.sample(range(8200), 40)))
    near, near_lse = run(gpu, q, pool, table, lens, counts)
    # Two answers within a tolerance each, of outputs that are a mean of values up to 3 (0.5 x 6 standard deviations).
    assert ((o.float() - near.float()).abs() <= 4 * 2.0 ** -8 * 3).all() and torch.isfinite(o).all()
    assert ((lse - near_lse).abs() <= 2.0 ** -14 * (1 + lse.abs())).all()


# ---- up to 32 rows: the waves share the scores ---------------------------------------------------------

@pytest.mark.parametrize("H,n", [(1, 1), (1, 31), (1, 32), (1, 33), (2, 16), (4, 8), (16, 2), (11, 3), (31, 1), (32, 1), (33, 1)])
@pytest.mark.parametrize("N", [33, 40, 64, 97, 1000])
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows(gpu, H, n, N, causal):
    lens, counts = [N, 1, N + 3], [n, 1, n]
    pool, table, rows = paged(lens, gpu, seed=N)
    q = queries(sum(counts), H, n)
    o, lse = run(gpu, q, pool, table, lens, counts, causal)
    check(q, o, lse, rows, lens, counts, causal)


@pytest.mark.parametrize("H,n", [(16, 2), (1, 20), (5, 6)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_few_rows_and_what_they_do_not_attend(gpu, H, n, value):
    N = 150
    pool, table, rows = paged([N], gpu)
    q = queries(n, H, 5)
    for bad in ([N - 1], [N - n + 1, N - 1], [40]):
        p = pool.clone()
        for j in bad:
            p[table[0, j // PAGE].item(), j % PAGE, 9] = value
        o, lse = run(gpu, q, p, table, [N], [n])
        clean = max(0, bad[0] - (N - n))
        check(q, o, lse, rows, [N], [n], some=set(range(clean)))
        assert not torch.isfinite(o[clean:, :, 9]).any()


@pytest.mark.parametrize("H", [1, 16, 32])
def test_few_rows_with_a_bad_page(gpu, H):
    lens, counts = [200, 500, 64], [1, 1, 1]
    pool, table, rows = paged(lens, gpu)
    q = queries(3, H, 6)
    table[1, 3] = pool.shape[0]
    o, lse = run(gpu, q, pool, table, lens, counts)
    check(q, o, lse, rows, lens, counts, some={0, 2})
    assert torch.isnan(o[1]).all() and torch.isnan(lse[1]).all()


@pytest.mark.parametrize("steepest", [4.0, 60.0])
@pytest.mark.parametrize("H,N", [(16, 400), (32, 400), (16, 9000), (128, 9000)])
def test_climbing_scores(gpu, H, N, steepest):
    """Values of 2^110 under scores that climb by tens and by hundreds, within a part and over parts."""
    rows = torch.zeros(N, D_QK)
    rows[:, :D_V] = 2.0 ** 110
    rows[:, D_V] = torch.linspace(0, 60, N)
    rows = rows.to(torch.bfloat16)
    pool = torch.zeros(pages(N), PAGE, D_QK, dtype=torch.bfloat16)
    pool.view(-1, D_QK)[:N] = rows
    q = torch.zeros(1, H, D_QK)
    q[:, :, D_V] = torch.linspace(0.1, steepest, H)
    q = q.to(torch.bfloat16)
    o, lse = run(gpu, q, pool.to(gpu), ints([list(range(pages(N)))], gpu), [N], [1])
    check(q, o, lse, [rows], [N], [1])


def test_short_sequences_beside_tables_of_a_million_pages(gpu):
    """Sequences that weigh less than a unit of the cut are there all the same."""
    lens, counts, H = [3, 1, 600, 2, 64, 1, 40, 9], [3, 1, 600, 1, 64, 1, 40, 2], 128
    pool, table, rows = paged(lens, gpu)
    wide = torch.full((len(lens), 1 << 20), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    extra = 20000   # queries behind the last sequence, which the host counts as work that could be
    q = queries(sum(counts), H, 4)
    padded = torch.zeros(sum(counts) + extra, H, D_QK, dtype=torch.bfloat16, device=gpu)
    padded[:sum(counts)] = q
    o, lse = run(gpu, padded, pool, wide, lens, counts)
    r = random.Random(1)
    n = sum(counts)
    check(q, o[:n], lse[:n], rows, lens, counts, some=set(list(range(10)) + list(range(n - 110, n)) + r.sample(range(n), 30)))
    assert (o[n:] == 0).all() and (lse[n:] == float("-inf")).all()


# ---- row tiles of 128 rows: a call with less than 900 tiles of 32 keys is cut in row tiles of 32 --------

LONG = 29000   # tokens of a sequence that makes a call large


@pytest.mark.parametrize("H,lens,counts", [
    (128, [1], [1]), (128, [5], [5]), (16, [33, 200, 7], [33, 9, 2]), (1, [300, 64], [290, 64]), (5, [97, 31, 1000], [50, 31, 3]),
    (20, [129, 0, 63], [17, 0, 1]), (96, [70, 40], [3, 40]), (128, [2000], [3]), (128, [191, 640], [64, 2]), (130, [100], [3]),
    (300, [66], [2]), (64, [33] * 40, [1] * 40), (33, [40], [1]), (32, [40, 50], [1, 2])])
@pytest.mark.parametrize("causal", [True, False])
def test_large_calls(gpu, H, lens, counts, causal):
    lens, counts = lens + [LONG], counts + [1]
    pool, table, rows = paged(lens, gpu, seed=H)
    q = queries(sum(counts), H, H)
    o, lse = run(gpu, q, pool, table, lens, counts, causal)
    check(q, o, lse, rows, lens, counts, causal)


@pytest.mark.parametrize("H", [1, 16, 48, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_large_calls_and_what_a_query_does_not_attend(gpu, H, value):
    lens, counts = [90, LONG], [60, 1]
    pool, table, rows = paged(lens, gpu)
    q = queries(61, H, 3)
    for bad in ([45], [31, 32, 77], list(range(60, 90))):
        p = pool.clone()
        for j in bad:
            p[table[0, j // PAGE].item(), j % PAGE, 5] = value
        o, lse = run(gpu, q, p, table, lens, counts)
        clean = max(0, bad[0] - 30)   # query i is token 30 + i
        check(q, o, lse, rows, lens, counts, some=set(range(clean)) | {60})
        assert not torch.isfinite(o[clean:60, :, 5]).any(), "a query that attends it"


@pytest.mark.parametrize("H", [16, 128])
def test_large_calls_with_bad_pages(gpu, H):
    lens, counts = [200, 130, LONG], [200, 2, 1]
    pool, table, rows = paged(lens, gpu)
    q = queries(203, H, 5)
    for bad in (-1, pool.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 2] = bad
        o, lse = run(gpu, q, pool, t, lens, counts)
        check(q, o, lse, rows, lens, counts, some=set(range(128)) | {200, 201, 202})
        assert torch.isnan(o[128:200]).all() and torch.isnan(lse[128:200]).all()


@pytest.mark.parametrize("steepest", [4.0, 60.0])
@pytest.mark.parametrize("H", [16, 128])
def test_large_calls_with_climbing_scores(gpu, H, steepest):
    N = 400
    pool, table, rows = paged([N, LONG], gpu)
    climb = torch.zeros(N, D_QK)
    climb[:, :D_V] = 2.0 ** 110
    climb[:, D_V] = torch.linspace(0, 60, N)
    rows[0] = climb.to(torch.bfloat16)
    for j in range(pages(N)):
        part = rows[0][PAGE * j:PAGE * (j + 1)]
        pool[table[0, j].item(), :len(part)] = part.to(gpu)
    q = torch.zeros(10, H, D_QK)
    q[:, :, D_V] = torch.linspace(0.1, steepest, H)
    q = q.to(torch.bfloat16)
    o, lse = run(gpu, q, pool, table, [N, LONG], [9, 1])
    check(q, o, lse, rows, [N, LONG], [9, 1])


def test_large_calls_with_strides(gpu):
    from python import ops
    lens, counts, H = [150, 20, LONG], [40, 20, 1], 16
    pool, table, rows = paged(lens, gpu)
    q = queries(61, H, 4)
    q2 = torch.full((61, H + 3, D_QK + 8), float("nan"), dtype=torch.bfloat16, device=gpu)
    q2[:, :H, :D_QK] = q.to(gpu)
    p2 = torch.full((pool.shape[0], PAGE + 2, D_QK + 24), float("nan"), dtype=torch.bfloat16, device=gpu)
    p2[:, :PAGE, :D_QK] = pool
    by_head = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    want = run(gpu, q, pool, table, lens, counts)
    check(q, *want, rows, lens, counts)
    for x, y in ((q2[:, :H, :D_QK], p2[:, :PAGE, :D_QK]), (by_head, pool)):
        got = ops.flash_dmla_chunk_paged(x, y, table, ints(lens, gpu), ints(starts(counts), gpu), softmax_scale=SCALE,
                                         return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("N", [28300, 28500, 28544, 28576, 28608, 28700])
@pytest.mark.parametrize("H,n", [(128, 1), (40, 2)])
def test_where_row_tiles_change_their_size(gpu, N, H, n):
    pool, table, rows = paged([N], gpu)
    q = queries(n, H, 7)
    o, lse = run(gpu, q, pool, table, [N], [n])
    check(q, o, lse, rows, [N], [n])


# ---- row tiles with rows before a page outside the pool and behind ---------------------------------------

@pytest.mark.parametrize("H", [1, 5, 48])
@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_before_a_bad_page(gpu, H, large, value):
    """Page 0 stands in for a page outside the pool: whatever it holds, rows of tokens before that page see nothing of it."""
    lens, counts = [200, 70], [150, 9]
    if large:
        lens, counts = lens + [LONG], counts + [1]
    pool, table, rows = paged(lens, gpu, seed=H)
    pool = torch.cat([torch.full_like(pool[:1], value), pool])
    q = queries(sum(counts), H, 8)
    for b, page in ((0, 1), (0, 2), (1, 1)):
        at = starts(counts)[b]
        first = at + PAGE * page - (lens[b] - counts[b])   # the first query that attends the page
        seen = range(first, at + counts[b])
        for bad in (-1, pool.shape[0]):
            t = torch.where(table < 0, table, table + 1)
            t[b, page] = bad
            o, lse = run(gpu, q, pool, t, lens, counts)
            check(q, o, lse, rows, lens, counts, some=set(range(sum(counts))) - set(seen))
            assert torch.isnan(o[first:seen[-1] + 1]).all() and torch.isnan(lse[first:seen[-1] + 1]).all()


@pytest.mark.parametrize("H", [16, 48])
def test_queries_without_a_token_before_a_bad_page(gpu, H):
    """The first page is outside the pool: NaN for those that have tokens, the others have none."""
    from python import ops
    pool = torch.full((3, PAGE, D_QK), float("nan"), dtype=torch.bfloat16, device=gpu)
    o, lse = ops.flash_dmla_chunk_paged(queries(9, H, 9).to(gpu), pool, ints([[3]], gpu), ints([4], gpu), ints([0, 9], gpu),
                                        softmax_scale=SCALE, return_lse=True)
    assert (o[:5] == 0).all() and (lse[:5] == float("-inf")).all()
    assert torch.isnan(o[5:]).all() and torch.isnan(lse[5:]).all()


@pytest.mark.parametrize("H,n", [(1, 1 << 22), (16, 70000)])
def test_many_more_queries_than_tokens(gpu, H, n):
    """Millions of queries without a token before the few that have one, and an ordinary sequence behind them."""
    from python import ops
    lens, counts = [50, 400], [n, 30]
    pool, table, rows = paged(lens, gpu)
    q = queries(80, H, 10)
    few = torch.zeros(1, 1, D_QK, dtype=torch.bfloat16, device=gpu).expand(n - 50, H, D_QK)
    all_q = torch.cat([few, q.to(gpu)])
    stale = torch.full((sum(counts), H, D_V), float("nan"), dtype=torch.bfloat16, device=gpu)   # what the output's memory may hold
    del stale
    o, lse = ops.flash_dmla_chunk_paged(all_q, pool, table, ints(lens, gpu), ints(starts(counts), gpu), softmax_scale=SCALE, return_lse=True)
    assert (o[:n - 50] == 0).all() and (lse[:n - 50] == float("-inf")).all()
    check(q, o[n - 50:], lse[n - 50:], rows, lens, [50, 30])
