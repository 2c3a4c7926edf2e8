"""Pages by request lengths and rows by slot, against a plain walk over the sequences."""
import pytest
import torch

from paging import D_QK, PAGE, ints, pages, starts

pytestmark = pytest.mark.gpu


def plain_release(table, old, new, free, num_pages, capacity):
    """(stack, whether something was left out)"""
    free, bad, width = list(free), False, len(table[0]) if table else 0
    for row, a, b in zip(table, old, new):
        held = min(pages(max(a, 0)), width)
        for j in range(min(pages(max(b, 0)), held), held):
            if not 0 <= row[j] < num_pages or len(free) >= capacity:
                bad = True
            else:
                free.append(row[j])
    return free, bad


def plain_reserve(table, lens, new, free, rows, num_pages):
    """(table, total, starts, slots, pages left, whether something was refused)"""
    table, bad, width = [list(r) for r in table], False, len(table[0]) if table else 0
    total, cu, slots, taken, at = [], [0], [-1] * rows, 0, 0
    for b, (n, m) in enumerate(zip(lens, new)):
        n, m = max(n, 0), max(m, 0)
        fits = at + m <= rows and n + m <= width * PAGE
        need = pages(n + m) - pages(n) if fits and m > 0 else 0
        ok = m == 0 or (fits and (need == 0 or taken + need <= len(free)))
        taken += need   # a sequence that goes away empty still stands before the others
        if ok:
            for i in range(need):
                table[b][pages(n) + i] = free[len(free) - 1 - (taken - need + i)]
            for t in range(m):
                p = table[b][(n + t) // PAGE]
                if 0 <= p < num_pages:
                    slots[at + t] = p * PAGE + (n + t) % PAGE
                else:
                    bad = True
        bad = bad or not ok
        total.append(n + m if ok else n)
        at += m
        cu.append(min(at, rows))
    served = sum(pages(t) - pages(max(n, 0)) for t, n in zip(total, lens))
    return table, total, cu, slots, len(free) - served, bad


def table_of(lens, width, order):
    table, at = [], 0
    for n in lens:
        table.append(order[at:at + pages(n)] + [-5] * (width - pages(n)))
        at += pages(n)
    return table, order[at:]


CASES = [
    ([0], [1]),
    ([63, 64, 65, 0], [1, 1, 1, 0]),
    ([0, 0, 10, 200], [300, 64, 0, 57]),
    ([130, 0, 64], [2, 129, 0]),
    (list(range(0, 900, 3)), [i % 5 for i in range(300)]),      # more than one block of sequences
    ([5] * 700, [i % 3 * 40 for i in range(700)]),
    ([0, 0], [5000, 4096]),
    ([-3, 40], [70, -9]),
]


@pytest.mark.parametrize("lens,new", CASES)
@pytest.mark.parametrize("slack", [0, 13])
def test_reserve(gpu, lens, new, slack):
    from python import ops
    g = torch.Generator().manual_seed(len(lens))
    width = max(pages(max(a, 0) + max(b, 0)) for a, b in zip(lens, new)) + 1
    need = sum(pages(max(a, 0)) for a in lens) + sum(pages(max(a, 0) + max(b, 0)) for a, b in zip(lens, new))
    order = torch.randperm(need + 9, generator=g).tolist()
    table, free = table_of([max(a, 0) for a in lens], width, order)
    rows = sum(max(b, 0) for b in new) + slack
    want = plain_reserve(table, lens, new, free, rows, need + 9)
    assert not want[5]
    wide = torch.full((len(lens), width + 3), -9, dtype=torch.int32)
    wide[:, :width] = torch.tensor(table, dtype=torch.int32)
    wide = wide.to(gpu)
    pool = torch.full((len(free) + 4,), -77, dtype=torch.int32)
    pool[:len(free)] = torch.tensor(free, dtype=torch.int32)
    got = ops.flash_dmla_kv_reserve(wide[:, :width], ints(lens, gpu), ints(new, gpu), pool.to(gpu), ints([len(free)], gpu), rows,
                                    need + 9, check_indices=True)
    assert wide[:, :width].tolist() == want[0] and (wide[:, width:] == -9).all()
    assert [x.tolist() for x in got] == [want[1], want[2], want[3], [want[4]]]


@pytest.mark.parametrize("have", [0, 1, 2, 3, 4, 7])
@pytest.mark.parametrize("rows", [0, 100, 230, 400])
def test_reserve_without_enough_pages_or_rows(gpu, have, rows):
    """Sequences are served in order as long as their pages are there; those that need none always are."""
    from python import ops
    lens, new = [10, 64, 100, 0, 5, 640], [100, 64, 5, 130, 2, 1]   # the last does not fit its row of the table
    order = list(range(40, 0, -1))
    table, rest = table_of([10, 64, 100, 0, 5, 640], 10, order)
    free = rest[:have]
    want = plain_reserve(table, lens, new, free, rows, 41)
    t = torch.tensor(table, dtype=torch.int32, device=gpu)
    args = (t, ints(lens, gpu), ints(new, gpu), ints(free, gpu), ints([have], gpu), rows, 41)
    got = ops.flash_dmla_kv_reserve(*args)
    assert t.tolist() == want[0] and [x.tolist() for x in got] == [want[1], want[2], want[3], [want[4]]]
    assert want[5]
    with pytest.raises(ValueError, match="got no pages"):
        ops.flash_dmla_kv_reserve(*args, check_indices=True)


def test_reserve_with_pages_outside_the_pool(gpu):
    """The tail page of the table, and a page of the stack: slots -1 for their rows, and a flag."""
    from python import ops
    table = [[3, -1, 0], [99, 0, 0]]
    lens, new, free = [70, 10], [3, 80], [7, -4]
    want = plain_reserve(table, lens, new, free, 83, 10)
    t = torch.tensor(table, dtype=torch.int32, device=gpu)
    got = ops.flash_dmla_kv_reserve(t, ints(lens, gpu), ints(new, gpu), ints(free, gpu), ints([2], gpu), 83, 10)
    assert t.tolist() == want[0] and [x.tolist() for x in got] == [want[1], want[2], want[3], [want[4]]] and want[5]


@pytest.mark.parametrize("old,new", [
    ([100], [0]), ([64, 65, 1, 0], [64, 64, 0, 0]), ([1000, 30, 700], [500, 30, 0]),
    ([i % 400 for i in range(2500)], [i % 400 * (i % 3) // 3 for i in range(2500)]),   # more than one block of sequences
    ([100000, 130], [64, 0]), ([50], [90]), ([-7, 65], [-1, -1]),
])
def test_release(gpu, old, new):
    from python import ops
    g = torch.Generator().manual_seed(len(old))
    width = max(pages(max(a, 0)) for a in old)
    total = sum(pages(max(a, 0)) for a in old)
    order = torch.randperm(total + 5, generator=g).tolist()
    table, rest = table_of([max(a, 0) for a in old], width, order)
    want, bad = plain_release(table, old, new, rest, total + 5, total + 5)
    assert not bad
    stack = torch.full((total + 5,), -3, dtype=torch.int32)
    stack[:len(rest)] = torch.tensor(rest, dtype=torch.int32)
    stack, t = stack.to(gpu), torch.tensor(table, dtype=torch.int32, device=gpu)
    before, count = t.clone(), ints([len(rest)], gpu)
    got = ops.flash_dmla_kv_release(t, ints(old, gpu), ints(new, gpu), stack, count, total + 5, check_indices=True)
    assert got.tolist() == [len(want)] and stack.tolist() == want + [-3] * (total + 5 - len(want))
    assert torch.equal(t, before) and count.tolist() == [len(rest)]


def test_release_leaves_out_what_does_not_fit(gpu):
    """Entries outside the pool, and pages past the capacity."""
    from python import ops
    table, old, new = [[4, -1, 6, 9], [1, 2, 3, 8]], [256, 250], [0, 64]
    for capacity in (2, 4, 9):
        want, bad = plain_release(table, old, new, [5], 9, capacity)
        stack = ints([5] + [-3] * (capacity - 1), gpu)
        args = (ints(table, gpu), ints(old, gpu), ints(new, gpu), stack, ints([1], gpu), 9)
        assert ops.flash_dmla_kv_release(*args).tolist() == [len(want)]
        assert stack.tolist() == want + [-3] * (capacity - len(want)) and bad
        with pytest.raises(ValueError, match="kv release"):
            ops.flash_dmla_kv_release(*args, check_indices=True)


@pytest.mark.parametrize("T", [0, 1, 5, 300, 5001])
@pytest.mark.parametrize("d", [8, 576])
def test_append_rows(gpu, T, d):
    from python import ops
    g = torch.Generator().manual_seed(T)
    n = T // PAGE + 3
    rows = torch.randn(T, d, generator=g).to(torch.bfloat16)
    slots = torch.randperm(n * PAGE, generator=g)[:T].int()
    if T > 3:
        slots[1], slots[2] = -1, -2 ** 31
    wide = torch.randn(T, d + 16, generator=g).to(torch.bfloat16).to(gpu)
    wide[:, :d] = rows.to(gpu)
    pool = torch.randn(n, PAGE + 1, d + 8, generator=g).to(torch.bfloat16).to(gpu)
    want = pool.clone()
    for t in range(T):
        if slots[t] >= 0:
            want[slots[t].item() // PAGE, slots[t].item() % PAGE, :d] = rows[t].to(gpu)
    ops.flash_dmla_kv_append_rows(pool[:, :PAGE, :d], slots.to(gpu), wide[:, :d], check_indices=True)
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("T", [1, 77, 3001])
def test_append_rows_q4_is_the_padded_append(gpu, T):
    """The bytes that flash_dmla_kv_append_q4 writes for the same rows, special values among them."""
    from python import ops
    g = torch.Generator().manual_seed(T)
    rows = (torch.randn(T, D_QK, generator=g) * torch.exp2(torch.randint(-90, 90, (T, 1), generator=g).float())).to(torch.bfloat16)
    rows[0, 3], rows[T // 2, 40] = float("inf"), float("nan")
    rows = rows.to(gpu)
    n = pages(T) + 2
    order = torch.randperm(n, generator=g).int()
    table = order[None, :pages(T)].to(gpu)
    a = torch.zeros(n, PAGE, 400, dtype=torch.uint8, device=gpu)
    b = torch.zeros_like(a)
    ops.flash_dmla_kv_append_q4(a, table, ints([0], gpu), rows[None])
    t = torch.arange(T)
    slots = order[t // PAGE].long() * PAGE + t % PAGE
    ops.flash_dmla_kv_append_rows(b, slots.int().to(gpu), rows, check_indices=True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("q4", [False, True])
def test_slots_past_the_pool(gpu, q4):
    from python import ops
    pool = torch.zeros(3, PAGE, 400, dtype=torch.uint8, device=gpu) if q4 else torch.zeros(3, PAGE, D_QK, dtype=torch.bfloat16, device=gpu)
    rows = torch.ones(4, D_QK, dtype=torch.bfloat16, device=gpu)
    slots = ints([3 * PAGE, 2 ** 31 - 1, -1, -2 ** 31], gpu)
    ops.flash_dmla_kv_append_rows(pool, slots, rows)
    assert (pool == 0).all()
    with pytest.raises(ValueError, match="past the pool"):
        ops.flash_dmla_kv_append_rows(pool, slots, rows, check_indices=True)


@pytest.mark.parametrize("q4", [False, True])
def test_a_scheduler_step(gpu, q4):
    """Eviction, release, reserve, append, chunk attention, as a serving loop makes them, against a dense cache."""
    import math
    from paging import assert_attention, attention64
    from python import ops
    g = torch.Generator().manual_seed(3)
    num, width, H, scale = 40, 8, 16, 1 / math.sqrt(192.0)
    pool = (torch.zeros(num, PAGE, 400, dtype=torch.uint8, device=gpu) if q4
            else torch.full((num, PAGE, D_QK), float("nan"), dtype=torch.bfloat16, device=gpu))
    table = torch.full((4, width), -1, dtype=torch.int32, device=gpu)
    free = torch.randperm(num, generator=g).int().to(gpu)
    count, lens = ints([num], gpu), ints([0, 0, 0, 0], gpu)
    dense = [torch.zeros(0, D_QK, dtype=torch.bfloat16) for _ in range(4)]
    for step, new in enumerate([[200, 70, 1, 0], [1, 1, 300, 64], [5, 0, 1, 1]]):
        if step == 2:   # sequence 1 ends, sequence 2 is cut back to its first tokens' pages
            keep = ints([lens[0].item(), 0, 128, lens[3].item()], gpu)
            before = count.item()
            count = ops.flash_dmla_kv_release(table, lens, keep, free, count, num, check_indices=True)
            assert count.item() == before + pages(71) + pages(301) - 2
            lens = keep
            dense[1], dense[2] = dense[1][:0], dense[2][:128]
        rows = (torch.randn(sum(new) + 3, D_QK, generator=g) * 0.5).to(torch.bfloat16)
        lens, cu, slots, count = ops.flash_dmla_kv_reserve(table, lens, ints(new, gpu), free, count, len(rows), num, check_indices=True)
        ops.flash_dmla_kv_append_rows(pool, slots, rows.to(gpu), check_indices=True)
        at = starts(new)
        dense = [torch.cat((d, rows[at[b]:at[b + 1]])) for b, d in enumerate(dense)]
        assert lens.tolist() == [len(d) for d in dense] and cu.tolist() == at
        q = (torch.randn(len(rows), H, D_QK, generator=g) * 0.5).to(torch.bfloat16)
        keys = dense
        if q4:   # 4-bit pages: their rows as bf16 pages, a block table of their own
            flat = ops.flash_dmla_kv_gather_q4(pool, table, lens, width * PAGE)
            keys = [flat[b, :len(d)].cpu() for b, d in enumerate(dense)]
            o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), flat.view(-1, PAGE, D_QK), torch.arange(4 * width, dtype=torch.int32,
                                                device=gpu).view(4, width), lens, cu, softmax_scale=scale, return_lse=True)
        else:
            o, lse = ops.flash_dmla_chunk_paged(q.to(gpu), pool, table, lens, cu, softmax_scale=scale, return_lse=True,
                                                check_indices=True)
        for b in range(4):
            part = slice(at[b], at[b + 1])
            ends = [len(dense[b]) - new[b] + i + 1 for i in range(new[b])]
            assert_attention(o[part], lse[part], attention64(q[part], keys[b], ends, scale), f"step {step}, sequence {b}")
        assert (o[sum(new):] == 0).all()
    used = sum(pages(len(d)) for d in dense)
    assert count.item() == num - used
