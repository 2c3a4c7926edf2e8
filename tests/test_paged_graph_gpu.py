"""The paged calls in HIP graphs, on other streams, through the dispatcher, with empty arguments and past 32 bits."""
import math

import pytest
import torch

from paging import D_QK, D_V, PAGE, assert_attention, attention64, ints, paged, pages, starts
from test_graph_gpu import _capture

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(192.0)


def bits(t):
    return t.contiguous().view(torch.uint8)


def assert_same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(bits(x), bits(y))


def rand(*shape, seed, scale=0.5):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


class Step:
    """A scheduler's step over static buffers: reserve, append, chunk attention, means, scores, selection, attention."""

    def __init__(self, gpu, H=16, B=5, T=160, seed=0):
        self.gpu, self.H, self.B, self.T = gpu, H, B, T
        self.num, self.width = 64, 12
        self.pool = torch.zeros(self.num, PAGE, D_QK, dtype=torch.bfloat16, device=gpu)
        self.means = torch.zeros(self.num, D_QK, dtype=torch.bfloat16, device=gpu)
        self.table = torch.full((B, self.width), -1, dtype=torch.int32, device=gpu)
        self.free = torch.randperm(self.num, generator=torch.Generator().manual_seed(seed)).int().to(gpu)
        self.lens, self.new, self.count = ints([0] * B, gpu), ints([0] * B, gpu), ints([self.num], gpu)
        self.rows = torch.zeros(T, D_QK, dtype=torch.bfloat16, device=gpu)
        self.q = torch.zeros(T, H, D_QK, dtype=torch.bfloat16, device=gpu)

    def load(self, lens, new, seed):
        """The step's inputs, in place: sequences of random rows already cached, and what is new."""
        from python import ops
        self.table.fill_(-1)
        total, _, slots, count = ops.flash_dmla_kv_reserve(self.table, ints([0] * self.B, self.gpu), ints(lens, self.gpu), self.free,
                                                           ints([self.num], self.gpu), sum(lens), self.num, check_indices=True)
        ops.flash_dmla_kv_append_rows(self.pool, slots, rand(sum(lens), D_QK, seed=seed).to(self.gpu))
        ops.flash_dmla_page_means(self.pool, self.table, total, self.means)
        self.lens.copy_(total)
        self.new.copy_(ints(new, self.gpu))
        self.count.copy_(count)
        self.rows.copy_(rand(self.T, D_QK, seed=seed + 1).to(self.gpu))
        self.q.copy_(rand(self.T, self.H, D_QK, seed=seed + 2).to(self.gpu))

    def __call__(self):
        from python import ops
        total, cu, slots, count = ops.flash_dmla_kv_reserve(self.table, self.lens, self.new, self.free, self.count, self.T, self.num)
        ops.flash_dmla_kv_append_rows(self.pool, slots, self.rows)
        o, lse = ops.flash_dmla_chunk_paged(self.q, self.pool, self.table, total, cu, softmax_scale=SCALE, return_lse=True)
        ops.flash_dmla_page_means(self.pool, self.table, total, self.means, starts=self.lens)
        so, slse = ops.flash_dmla_sparse_paged(self.q, self.pool, self.means, self.table, total, cu, 3, softmax_scale=SCALE, return_lse=True)
        back = ops.flash_dmla_kv_release(self.table, total, self.lens, self.free.clone(), count, self.num)
        return total, cu, slots, count, o, lse, so, slse, back


LOADS = [([100, 0, 64, 300, 5], [20, 70, 1, 0, 60]), ([5, 5, 5, 5, 5], [1, 1, 1, 1, 1]), ([0, 0, 0, 0, 640], [0, 0, 0, 0, 90]),
         ([63, 64, 65, 128, 127], [1, 1, 1, 2, 2]), ([700, 1, 1, 1, 1], [32, 32, 32, 32, 32])]


def test_a_step_replays_in_a_graph(gpu):
    """Captured once, replayed with other lengths, tables and inputs, eager work between, bit for bit the eager step."""
    step = Step(gpu)
    step.load(*LOADS[0], seed=1)
    graph, out = _capture(step)
    for r, (lens, new) in enumerate(LOADS * 2):
        step.load(lens, new, seed=10 * r)
        before = step.pool.clone(), step.table.clone(), step.means.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out] + [step.pool.clone(), step.table.clone(), step.means.clone()]
        for t, b in zip((step.pool, step.table, step.means), before):
            t.copy_(b)
        want = list(step()) + [step.pool, step.table, step.means]
        torch.cuda.synchronize()
        assert_same(got, want)


def test_two_graphs_in_turn(gpu):
    """Two captured steps, each with its own workspaces, replayed one after the other and with an eager one between."""
    a, b = Step(gpu, seed=1), Step(gpu, H=40, B=5, T=200, seed=2)
    a.load(*LOADS[0], seed=3)
    b.load(*LOADS[3], seed=4)
    ga, oa = _capture(a)
    gb, ob = _capture(b)
    wa, wb = [x.clone() for x in a()], [x.clone() for x in b()]
    for _ in range(3):
        ga.replay()
        gb.replay()
        b()
        ga.replay()
        torch.cuda.synchronize()
        assert_same(oa, wa)
        assert_same(ob, wb)


def test_other_streams(gpu):
    """Two streams at once, each call with its own workspace."""
    from python import ops
    lens, counts = [3000, 700], [40, 3]
    pool, table, rows = paged(lens, gpu)
    args = [(rand(43, 16, D_QK, seed=s).to(gpu), pool, table, ints(lens, gpu), ints(starts(counts), gpu)) for s in (1, 2)]
    want = [ops.flash_dmla_chunk_paged(*x, softmax_scale=SCALE, return_lse=True) for x in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.flash_dmla_chunk_paged(*args[i], softmax_scale=SCALE, return_lse=True)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert_same(g, w)


def test_the_dispatcher_calls_are_the_python_calls(gpu):
    import python  # noqa: F401  (registers torch.ops.flashdmla.*)
    from python import ops
    F = torch.ops.flashdmla
    lens, counts = [900, 64, 130], [3, 1, 70]
    pool, table, rows = paged(lens, gpu)
    T = sum(counts)
    q, lens_t, cu = rand(T, 16, D_QK, seed=5).to(gpu), ints(lens, gpu), ints(starts(counts), gpu)
    assert_same(F.chunk_paged(q, pool, table, lens_t, cu, D_V, SCALE, True),
                ops.flash_dmla_chunk_paged(q, pool, table, lens_t, cu, softmax_scale=SCALE, return_lse=True))
    m1, m2 = torch.zeros(2, pool.shape[0], D_QK, dtype=torch.bfloat16, device=gpu)
    F.page_means(pool, table, lens_t, m1, None)
    ops.flash_dmla_page_means(pool, table, lens_t, m2)
    assert torch.equal(m1, m2)
    s1 = F.page_scores(q, m1, table, lens_t, cu, SCALE)
    assert torch.equal(s1, ops.flash_dmla_page_scores(q, m1, table, lens_t, cu, SCALE))
    assert_same(F.page_select(s1, table, lens_t, cu, 4, 1, 1), ops.flash_dmla_page_select(s1, table, lens_t, cu, 4, recent=1, sink=1))
    spare = ints(list(range(100, 130)), gpu)
    new = ints([60, 1, 200], gpu)
    wide = torch.cat((table, torch.full((3, 6), -1, dtype=torch.int32, device=gpu)), 1).contiguous()
    t1, t2 = wide.clone(), wide.clone()
    got = F.kv_reserve(t1, lens_t, new, spare, ints([30], gpu), 261, 200)
    assert_same(got, ops.flash_dmla_kv_reserve(t2, lens_t, new, spare, ints([30], gpu), 261, 200))
    assert torch.equal(t1, t2)
    f1, f2 = spare.clone(), spare.clone()
    assert torch.equal(F.kv_release(t1, got[0], lens_t, f1, got[3], 200), ops.flash_dmla_kv_release(t2, got[0], lens_t, f2, got[3], 200))
    assert torch.equal(f1, f2)
    p1, p2 = torch.zeros(2, 200, PAGE, D_QK, dtype=torch.bfloat16, device=gpu)
    F.kv_append_rows(p1, got[2], q[:1, 0].expand(261, -1).contiguous())
    ops.flash_dmla_kv_append_rows(p2, got[2], q[:1, 0].expand(261, -1).contiguous())
    assert torch.equal(p1, p2)
    check = lambda op, *a: torch.library.opcheck(op, a, test_utils=("test_schema", "test_faketensor"))
    check(F.chunk_paged.default, q, pool, table, lens_t, cu, D_V, SCALE, True)
    check(F.page_means.default, pool, table, lens_t, m1, None)
    check(F.page_scores.default, q, m1, table, lens_t, cu, SCALE)
    check(F.page_select.default, s1, table, lens_t, cu, 4, 1, 1)
    check(F.kv_reserve.default, t1, lens_t, new, spare, ints([30], gpu), 261, 200)
    check(F.kv_release.default, t1, got[0], lens_t, f1, got[3], 200)
    check(F.kv_append_rows.default, p1, got[2], q[:1, 0].expand(261, -1).contiguous())


def test_empty_arguments(gpu):
    from python import ops
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)
    q = torch.zeros(3, 16, D_QK, dtype=torch.bfloat16, device=gpu)
    pool, means = torch.zeros(2, PAGE, D_QK, dtype=torch.bfloat16, device=gpu), torch.zeros(2, D_QK, dtype=torch.bfloat16, device=gpu)
    total, cu, slots, count = ops.flash_dmla_kv_reserve(z(0, 4), z(0), z(0), z(5), ints([5], gpu), 3, 2, check_indices=True)
    assert total.shape == (0,) and cu.tolist() == [0] and slots.tolist() == [-1] * 3 and count.item() == 5
    total, cu, slots, count = ops.flash_dmla_kv_reserve(z(2, 0), z(2), z(2), z(0), ints([0], gpu), 0, 2, check_indices=True)
    assert total.tolist() == [0, 0] and cu.tolist() == [0, 0, 0] and count.item() == 0
    assert ops.flash_dmla_kv_release(z(0, 4), z(0), z(0), z(5), ints([3], gpu), 2, check_indices=True).item() == 3
    assert ops.flash_dmla_kv_release(z(2, 0), ints([70, 3], gpu), z(2), z(0), ints([0], gpu), 2, check_indices=True).item() == 0
    ops.flash_dmla_kv_append_rows(pool, z(0), q[:0, 0], check_indices=True)
    o, lse = ops.flash_dmla_chunk_paged(q[:0], pool, z(2, 4), z(2), z(3), return_lse=True)
    assert o.shape == (0, 16, D_V) and lse.shape == (0, 16)
    o, lse = ops.flash_dmla_chunk_paged(q, pool, z(0, 4), z(0), z(1), return_lse=True)
    assert (o == 0).all() and (lse == float("-inf")).all()
    ops.flash_dmla_page_means(pool, z(0, 4), z(0), means)
    assert ops.flash_dmla_page_scores(q[:0], means, z(2, 4), z(2), z(3)).shape == (0, 4)
    assert (ops.flash_dmla_page_scores(q, means, z(0, 4), z(0), z(1)) == 0).all()
    assert ops.flash_dmla_page_scores(q, means, z(2, 0), z(2), z(3)).shape == (3, 0)
    table, lens, index = ops.flash_dmla_page_select(torch.zeros(3, 4, device=gpu), z(0, 4), z(0), z(1), 2)
    assert (table == -1).all() and (lens == 0).all() and (index == -1).all()
    table, lens, index = ops.flash_dmla_page_select(torch.zeros(3, 0, device=gpu), z(3, 0), ints([5, 6, 7], gpu), None, 2)
    assert (table == -1).all() and (lens == 0).all()


def test_refusals_on_the_gpu(gpu):
    from python import ops
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)
    q = torch.zeros(4, 16, D_QK, dtype=torch.bfloat16, device=gpu)
    pool, means = torch.zeros(2, PAGE, D_QK, dtype=torch.bfloat16, device=gpu), torch.zeros(2, D_QK, dtype=torch.bfloat16, device=gpu)
    table, lens, scores = z(2, 3), z(2), torch.zeros(4, 3, device=gpu)
    for f in (
        lambda: ops.flash_dmla_chunk_paged(q, pool, table, lens),                       # four queries, two sequences
        lambda: ops.flash_dmla_chunk_paged(q, pool, table, lens, z(2)),                 # starts of one sequence
        lambda: ops.flash_dmla_chunk_paged(q, pool, table, lens, z(3).long()),
        lambda: ops.flash_dmla_chunk_paged(q.float(), pool, table, lens, z(3)),
        lambda: ops.flash_dmla_chunk_paged(q[..., :512], pool, table, lens, z(3)),
        lambda: ops.flash_dmla_chunk_paged(q, pool[:, :32], table, lens, z(3)),
        lambda: ops.flash_dmla_chunk_paged(q, pool.view(torch.uint8)[..., :400], table, lens, z(3)),
        lambda: ops.flash_dmla_chunk_paged(q, pool, table, lens, z(3), softmax_scale=0.0),
        lambda: ops.flash_dmla_chunk_paged(q, pool, table, lens, ints([0, 3, 2], gpu), check_indices=True),
        lambda: ops.flash_dmla_chunk_paged(q, pool, table, lens, ints([0, 3, 5], gpu), check_indices=True),
        lambda: ops.flash_dmla_chunk_paged(q, pool, table - 1, lens + 5, ints([0, 3, 4], gpu), check_indices=True),
        lambda: ops.flash_dmla_page_means(pool, table, lens, means[:1]),
        lambda: ops.flash_dmla_page_means(pool, table, lens, means[:, :512]),
        lambda: ops.flash_dmla_page_means(pool, table, lens, means, starts=z(3)),
        lambda: ops.flash_dmla_page_scores(q, means, table, lens),
        lambda: ops.flash_dmla_page_scores(q, means.float(), table, lens, z(3)),
        lambda: ops.flash_dmla_page_select(scores[:, :2], table, lens, z(3), 2),
        lambda: ops.flash_dmla_page_select(scores.double(), table, lens, z(3), 2),
        lambda: ops.flash_dmla_page_select(scores, table, lens, z(3), 2, recent=0),
        lambda: ops.flash_dmla_page_select(scores, table, lens, z(3), 2, recent=2, sink=1),
        lambda: ops.flash_dmla_kv_append_rows(pool, z(3), q[:, 0]),
        lambda: ops.flash_dmla_kv_append_rows(pool, z(4), q[:, 0, :512]),
        lambda: ops.flash_dmla_kv_reserve(table, lens, z(3), z(5), z(1), 4, 2),
        lambda: ops.flash_dmla_kv_reserve(table, lens, lens, z(5), z(2), 4, 2),
        lambda: ops.flash_dmla_kv_reserve(table, lens, lens, z(5), z(1), -1, 2),
        lambda: ops.flash_dmla_kv_reserve(table.t(), lens, lens, z(5), z(1), 4, 2),
        lambda: ops.flash_dmla_kv_release(table, lens, lens, z(5).float(), z(1), 2),
        lambda: ops.flash_dmla_kv_release(table, lens, z(3), z(5), z(1), 2),
    ):
        with pytest.raises((ValueError, NotImplementedError)):
            f()


def test_offsets_past_32_bits(gpu):
    """A pool of 5 GB whose last pages are used, more than 2^32 bytes of queries' and outputs' strides, slots near its end."""
    from python import ops
    n = 70000
    pool = torch.empty(n, PAGE, D_QK, dtype=torch.bfloat16, device=gpu)
    lens, counts, H = [130, 70], [20, 70], 16
    small, table, rows = paged(lens, gpu)
    far = n - small.shape[0]
    pool[far:] = small
    moved = torch.where(table >= 0, table + far, table)
    T = sum(counts)
    q = rand(T, H, D_QK, seed=8).to(gpu)
    args = (ints(lens, gpu), ints(starts(counts), gpu))
    want = ops.flash_dmla_chunk_paged(q, small, table, *args, softmax_scale=SCALE, return_lse=True)
    assert_same(ops.flash_dmla_chunk_paged(q, pool, moved, *args, softmax_scale=SCALE, return_lse=True), want)
    apart = torch.empty(T, 1 << 25, dtype=torch.bfloat16, device=gpu)[:, :H * D_QK].unflatten(1, (H, D_QK))   # 64 MB between tokens
    apart.copy_(q)
    assert_same(ops.flash_dmla_chunk_paged(apart, pool, moved, *args, softmax_scale=SCALE, return_lse=True), want)
    means, few = torch.zeros(n, D_QK, dtype=torch.bfloat16, device=gpu), torch.zeros(small.shape[0], D_QK, dtype=torch.bfloat16, device=gpu)
    ops.flash_dmla_page_means(pool, moved, args[0], means)
    ops.flash_dmla_page_means(small, table, args[0], few)
    assert torch.equal(means[far:], few)
    assert torch.equal(ops.flash_dmla_page_scores(apart, means, moved, *args, SCALE), ops.flash_dmla_page_scores(q, few, table, *args, SCALE))
    slots = ints([n * PAGE - 1, far * PAGE, n * PAGE], gpu)
    ops.flash_dmla_kv_append_rows(pool, slots, q[:3, 0].contiguous())
    assert torch.equal(pool[n - 1, PAGE - 1], q[0, 0]) and torch.equal(pool[far, 0], q[1, 0])
    assert pages(lens[0]) == 3
