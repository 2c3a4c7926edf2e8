"""Page means, page scores and the selection of pages against plain 64-bit forms."""
import math

import pytest
import torch

from paging import D_QK, D_V, PAGE, assert_attention, attention64, ints, paged, pages, starts

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(192.0)


def means64(x):
    """Means of [n, 64, 576] rows and half a bf16 step around them (the fp32 sum of 64 is off by 64 x 2^-24 at most)."""
    m = x.double().mean(1)
    return m, m.abs() * 2.0 ** -8 + x.double().abs().mean(1) * 64 * 2.0 ** -24 + 1e-38


@pytest.mark.parametrize("lens,before", [([64], [0]), ([63, 200, 0], None), ([640, 65, 128], [130, 64, 0]), ([300] * 90, [0] * 90)])
def test_means(gpu, lens, before):
    from python import ops
    pool, table, rows = paged(lens, gpu)
    means = torch.full((pool.shape[0], D_QK), 7.0, dtype=torch.bfloat16, device=gpu)
    ops.flash_dmla_page_means(pool, table, ints(lens, gpu), means, starts=None if before is None else ints(before, gpu))
    left = torch.ones(pool.shape[0], dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range((before[b] if before else 0) // PAGE, n // PAGE):
            page = table[b, j].item()
            left[page] = False
            m, tol = means64(rows[b][None, PAGE * j:PAGE * (j + 1)])
            assert ((means[page].double().cpu() - m[0]).abs() <= tol[0]).all()
    assert (means[left.to(gpu)] == 7.0).all(), "pages that are not full, or were full before"


def test_means_of_4_bit_pages(gpu):
    from python import ops
    lens = [300, 64]
    rows = (torch.randn(2, 300, D_QK, generator=torch.Generator().manual_seed(1)) * 0.5).to(torch.bfloat16).to(gpu)
    table = ints([[3, 0, 5, 6, 1], [2, -1, -1, -1, -1]], gpu)
    pool = torch.zeros(8, PAGE, 400, dtype=torch.uint8, device=gpu)
    ops.flash_dmla_kv_append_q4(pool, table, ints([0, 0], gpu), rows, ints(lens, gpu))
    back = ops.flash_dmla_kv_gather_q4(pool, table, ints(lens, gpu), 300).cpu()
    means = torch.full((8, D_QK), 7.0, dtype=torch.bfloat16, device=gpu)
    ops.flash_dmla_page_means(pool, table, ints(lens, gpu), means)
    for b, j, page in [(0, 0, 3), (0, 1, 0), (0, 2, 5), (0, 3, 6), (1, 0, 2)]:
        m, tol = means64(back[b][None, PAGE * j:PAGE * (j + 1)])
        assert ((means[page].double().cpu() - m[0]).abs() <= tol[0]).all()
    assert (means[[1, 4, 7]] == 7.0).all()


def test_means_strides_and_bad_pages(gpu):
    from python import ops
    lens = [200, 70]
    pool, table, rows = paged(lens, gpu)
    wide = torch.full((pool.shape[0], PAGE + 3, D_QK + 8), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[:, :PAGE, :D_QK] = pool
    a = torch.zeros(pool.shape[0], D_QK + 16, dtype=torch.bfloat16, device=gpu)
    b = torch.zeros(pool.shape[0], D_QK, dtype=torch.bfloat16, device=gpu)
    table[0, 1] = pool.shape[0]
    ops.flash_dmla_page_means(pool, table, ints(lens, gpu), b)
    ops.flash_dmla_page_means(wide[:, :PAGE, :D_QK], table, ints(lens, gpu), a[:, :D_QK])
    assert torch.equal(a[:, :D_QK], b) and (a[:, D_QK:] == 0).all()
    assert (b != 0).any(1).sum() == 3   # pages 0 and 2 of the first sequence, 0 of the second


def scores64(q, means, table, ends):
    """Scores of queries of one sequence in float64, and the tolerance of each: a score is a sum of 576 products in fp32
    (d, relative in every weight twice), the sums over pages and heads and the exponentials are 2^-16 together."""
    s = torch.zeros(len(ends), table.shape[0], dtype=torch.float64)
    tol = torch.zeros_like(s)
    for i, e in enumerate(ends):
        n = max(0, (e - 1) // PAGE) if e > 0 else 0
        if n:
            k = means[table[:n].long().to(means.device)].double().cpu()
            x = q[i].double().cpu() @ k.T * SCALE
            w = torch.softmax(x, dim=1)
            d = 600 * 2.0 ** -24 * (q[i].double().cpu().abs() @ k.abs().T).amax() * SCALE
            s[i, :n] = w.sum(0)
            tol[i, :n] = (2 * d + 2.0 ** -16) * w.sum(0) + 1e-30
    return s, tol


@pytest.mark.parametrize("H,lens,counts", [
    (128, [64 * 9 + 1], [1]),
    (16, [1, 64, 65, 128, 129, 700], [1] * 6),
    (1, [2000, 300], [40, 300]),
    (5, [640], [33]),
    (20, [0, 900, 130], [0, 11, 5]),
    (40, [130, 1300], [7, 3]),
    (96, [700, 400], [3, 2]),
    (128, [513], [5]),
    (130, [700, 66], [2, 3]),
    (300, [900], [2]),
    (16, [20000], [1]),            # several workgroups share a query's pages
    (64, [9000, 100], [2, 100]),
])
@pytest.mark.parametrize("wide", [False, True])
def test_scores(gpu, H, lens, counts, wide):
    from python import ops
    pool, table, _ = paged(lens, gpu, seed=H)
    means = (torch.randn(pool.shape[0], D_QK, generator=torch.Generator().manual_seed(H)) * 0.3).to(torch.bfloat16).to(gpu)
    if wide:   # a table far wider than the sequences
        table = torch.cat((table, torch.full((len(lens), 1500), -1, dtype=torch.int32, device=gpu)), 1).contiguous()
    T = sum(counts)
    q = (torch.randn(T + 2, H, D_QK, generator=torch.Generator().manual_seed(H + 1))).to(torch.bfloat16).to(gpu)
    got = ops.flash_dmla_page_scores(q, means, table, ints(lens, gpu), ints(starts(counts), gpu), SCALE)
    assert got.shape == (T + 2, table.shape[1]) and (got[T:] == 0).all()
    at = starts(counts)
    for b, (N, n) in enumerate(zip(lens, counts)):
        s, tol = scores64(q[at[b]:at[b + 1]], means, table[b].cpu(), [N - n + i + 1 for i in range(n)])
        err = (got[at[b]:at[b + 1]].double().cpu() - s).abs()
        assert (err <= tol).all(), f"sequence {b}: off by {(err / (tol + 1e-300)).max().item():.2f} of the tolerance"
    if all(n == 1 for n in counts):
        one = ops.flash_dmla_page_scores(q[:T], means, table, ints(lens, gpu), None, SCALE)
        for b, N in enumerate(lens):
            s, tol = scores64(q[b:b + 1], means, table[b].cpu(), [N])
            assert ((one[b:b + 1].double().cpu() - s).abs() <= tol).all()
    again = ops.flash_dmla_page_scores(q, means, table, ints(lens, gpu), ints(starts(counts), gpu), SCALE)
    assert torch.equal(got, again)


def test_scores_of_many_queries_over_long_tables(gpu):
    """As many queries as fill the GPU over more pages than a workgroup keeps table entries of."""
    from python import ops
    N, n, H = 64 * 2300 + 5, 270, 128
    pool = 3000
    table = torch.randint(0, pool, (1, pages(N)), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    means = (torch.randn(pool, D_QK, generator=torch.Generator().manual_seed(1)) * 0.3).to(torch.bfloat16).to(gpu)
    q = torch.randn(n, H, D_QK, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(gpu)
    got = ops.flash_dmla_page_scores(q, means, table.to(gpu), ints([N], gpu), ints([0, n], gpu), SCALE)
    for i in (0, 133, n - 1):
        s, tol = scores64(q[i:i + 1], means, table[0], [N - n + i + 1])
        assert ((got[i:i + 1].double().cpu() - s).abs() <= tol).all()


@pytest.mark.parametrize("lens", [[700], [40000]])
def test_scores_leave_out_what_is_not_there(gpu, lens):
    """Pages outside the pool count as not there; means of other pages, of the query's own and of later ones do not
    reach it, whatever they hold; a head that holds no number gives none."""
    from python import ops
    pool, table, _ = paged(lens, gpu)
    n = pages(lens[0])
    means = (torch.randn(pool.shape[0], D_QK, generator=torch.Generator().manual_seed(5)) * 0.3).to(torch.bfloat16).to(gpu)
    q = torch.randn(1, 16, D_QK, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(gpu)
    cut = table.clone()
    cut[0, 3], cut[0, 5] = -1, pool.shape[0]
    keep = torch.ones(n, dtype=torch.bool)
    keep[[3, 5]] = False
    m = means.clone()
    m[table[0, n - 1].item()] = float("nan")
    for p in set(range(pool.shape[0])) - set(table[0].tolist()):
        m[p] = float("inf")
    got = ops.flash_dmla_page_scores(q, m, cut, ints(lens, gpu), None, SCALE).double().cpu()
    packed = table[0].cpu()[keep]
    s, tol = scores64(q, m, packed, [len(packed) * PAGE])
    assert ((got[0][:n][keep] - s[0]).abs() <= tol[0]).all() and (got[0][:n][~keep] == 0).all()
    q[0, 2, 7] = float("nan")
    bad = ops.flash_dmla_page_scores(q, means, cut, ints(lens, gpu), None, SCALE)
    seen = keep.clone()
    seen[n - 1] = False
    assert torch.isnan(bad[0, :n][seen.to(gpu)]).all() and (bad[0, :n][~seen.to(gpu)] == 0).all()


def select_plain(scores, table, ends, k, recent, sink):
    out = []
    for t, e in enumerate(ends):
        n = pages(max(e, 0))
        pick = list(range(n))
        if n > k:
            def key(j):
                v = scores[t][j]
                return (0 if v != v else 1, 0 if v != v else -v, j)
            middle = sorted(range(sink, n - recent), key=key)[:k - sink - recent]
            pick = sorted(list(range(sink)) + middle + list(range(n - recent, n)))
        length = len(pick) * PAGE - (n * PAGE - max(e, 0))
        pad = [-1] * (k - len(pick))
        out.append(([table[j] for j in pick] + pad, length, pick + pad))
    return out


SPECIAL = [float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1.0, 1.0, -1.0, 1e-40, -1e-40, 3e38, 1e-45]


@pytest.mark.parametrize("lens,counts,k,recent,sink", [
    ([1], [1], 1, 1, 0),
    ([64 * 7], [3], 3, 1, 0),
    ([700, 64, 65], [5, 64, 2], 4, 2, 1),
    ([700, 3000], [1, 9], 6, 1, 5),
    ([5000], [40], 20, 3, 2),
    ([64 * 65, 0, 100], [2, 0, 3], 64, 1, 0),
    ([40000], [2], 100, 2, 1),
    ([64 * 600 + 5], [3], 513, 7, 6),
    ([200000], [1], 64, 4, 1),           # wider than the registers hold
    ([300], [2], 40, 1, 0),              # all pages, and room
])
@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_select(gpu, lens, counts, k, recent, sink, kind):
    from python import ops
    g = torch.Generator().manual_seed(k)
    width, T, B = max(pages(n) for n in lens), sum(counts), len(lens)
    table = torch.randint(0, 1 << 20, (B, width), generator=g, dtype=torch.int32)
    scores = torch.exp(2 * torch.randn(T + 3, width + 4, generator=g))
    if kind == "ties":
        scores = torch.randint(0, 3, scores.shape, generator=g).float()
    if kind == "special":
        scores = torch.tensor(SPECIAL)[torch.randint(0, len(SPECIAL), scores.shape, generator=g)]
    at = starts(counts)
    sel_table, sel_lens, sel_index = ops.flash_dmla_page_select(scores.to(gpu), table.to(gpu), ints(lens, gpu), ints(at, gpu), k,
                                                                recent=recent, sink=sink)
    for b, (N, n) in enumerate(zip(lens, counts)):
        want = select_plain(scores[at[b]:at[b + 1]].tolist(), table[b].tolist(), [N - n + i + 1 for i in range(n)], k, recent, sink)
        for i, w in enumerate(want):
            t = at[b] + i
            assert (sel_table[t].tolist(), sel_lens[t].item(), sel_index[t].tolist()) == w
    assert (sel_lens[T:] == 0).all() and (sel_table[T:] == -1).all() and (sel_index[T:] == -1).all()


def test_select_without_starts_is_one_query_each(gpu):
    from python import ops
    lens = [100, 0, 700, 64]
    g = torch.Generator().manual_seed(0)
    table = torch.randint(0, 99, (4, 11), generator=g, dtype=torch.int32).to(gpu)
    scores = torch.rand(4, 11, generator=g).to(gpu)
    a = ops.flash_dmla_page_select(scores, table, ints(lens, gpu), None, 4, recent=2)
    b = ops.flash_dmla_page_select(scores, table, ints(lens, gpu), ints(range(5), gpu), 4, recent=2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    want = select_plain(scores.tolist(), table[2].tolist(), lens, 4, 2, 0)[2]
    assert (a[0][2].tolist(), a[1][2].item(), a[2][2].tolist()) == want
    assert a[1].tolist() == [100, 0, 4 * 64 - (64 * 11 - 700), 64]


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("H,lens,counts", [(16, [900, 70, 64], [3, 70, 1]), (128, [2000], [2]), (40, [5, 1500], [5, 1])])
def test_sparse_attention(gpu, q4, H, lens, counts):
    """Means, scores, selection and attention together, against the attention over the selected tokens; the attention
    over all of them where the budget covers every page."""
    from python import ops
    pool, table, rows = paged(lens, gpu, seed=H, fill=0.0)
    if q4:
        packed = torch.zeros(pool.shape[0], PAGE, 400, dtype=torch.uint8, device=gpu)
        for b, r in enumerate(rows):
            ops.flash_dmla_kv_append_q4(packed, table[b:b + 1], ints([0], gpu), r[None].to(gpu))
        back = ops.flash_dmla_kv_gather_q4(packed, table, ints(lens, gpu), max(lens)).cpu()
        rows, pool = [back[b, :n] for b, n in enumerate(lens)], packed
    T = sum(counts)
    q = (torch.randn(T, H, D_QK, generator=torch.Generator().manual_seed(H)) * 0.5).to(torch.bfloat16).to(gpu)
    means = torch.zeros(pool.shape[0], D_QK, dtype=torch.bfloat16, device=gpu)
    lens_t, cu = ints(lens, gpu), ints(starts(counts), gpu)
    ops.flash_dmla_page_means(pool, table, lens_t, means)
    for k in (5, 64):
        scores = ops.flash_dmla_page_scores(q, means, table, lens_t, cu, SCALE)
        _, sel_lens, index = ops.flash_dmla_page_select(scores, table, lens_t, cu, k, recent=2, sink=1)
        o, lse = ops.flash_dmla_sparse_paged(q, pool, means, table, lens_t, cu, k, recent=2, sink=1, softmax_scale=SCALE,
                                             return_lse=True)
        at = starts(counts)
        for b, (N, n) in enumerate(zip(lens, counts)):
            for i in range(n):
                t, end = at[b] + i, N - n + i + 1
                keys = torch.cat([rows[b][PAGE * j:min(PAGE * (j + 1), end)] for j in index[t].tolist() if j >= 0])
                assert len(keys) == sel_lens[t].item()
                assert k < 64 or len(keys) == end
                assert_attention(o[t:t + 1], lse[t:t + 1], attention64(q[t:t + 1], keys, [len(keys)], SCALE), f"query {t} of {b}")


@pytest.mark.parametrize("H,lens,counts,width", [(16, [3000, 700], [400, 600], 8400), (300, [5000, 300], [100, 27], 3600),
                                                 (128, [9000] * 5, [1] * 5, 270000)])
def test_scores_under_tables_too_wide_to_keep_products(gpu, H, lens, counts, width):
    """Past 512 MB of products the second kernel computes them once more: the same scores either way."""
    from python import _lib, ops
    pool, table, _ = paged(lens, gpu, seed=H)
    means = (torch.randn(pool.shape[0], D_QK, generator=torch.Generator().manual_seed(H)) * 0.3).to(torch.bfloat16).to(gpu)
    T = sum(counts)
    q = (torch.randn(T, H, D_QK, generator=torch.Generator().manual_seed(H + 1))).to(torch.bfloat16).to(gpu)
    wide = torch.full((len(lens), width), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    assert 0 < _lib.lib().dmla_page_scores_workspace_bytes(T, H, width, 1) < 1 << 26
    got = ops.flash_dmla_page_scores(q, means, wide, ints(lens, gpu), ints(starts(counts), gpu), SCALE)
    kept = ops.flash_dmla_page_scores(q, means, table, ints(lens, gpu), ints(starts(counts), gpu), SCALE)
    assert (got[:, table.shape[1]:] == 0).all()
    at = starts(counts)
    for b, (N, n) in enumerate(zip(lens, counts)):
        some = sorted({0, n // 2, n - 1})
        s, tol = scores64(q[[at[b] + i for i in some]], means, table[b].cpu(), [N - n + i + 1 for i in some])
        for x in (got, kept):
            assert ((x[[at[b] + i for i in some], :table.shape[1]].double().cpu() - s).abs() <= tol).all()
