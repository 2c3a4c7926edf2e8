"""Append, accounts and eviction on parts of larger tensors: pages and rows with gaps, strided rows, accounts and
tables, rows of other widths.  The results are those of contiguous tensors, and what lies around stays as it was."""
import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from python import ops
from test_evict_gpu import SCALE, _lse, _pool
from test_q4_cache_gpu import _table


def _part(x, gpu, before, after, fill):
    """(a tensor on the GPU filled with `fill`, its part that holds x); before and after: widths around each dim."""
    wide = torch.full([b + n + a for b, n, a in zip(before, x.shape, after)], fill, dtype=x.dtype, device=gpu)
    part = wide[tuple(slice(b, b + n) for b, n in zip(before, x.shape))]
    part.copy_(x)
    return wide, part


def _around(wide, part, fill):
    """Whether everything of wide but part still holds fill (part is overwritten)."""
    part.fill_(fill)
    return bool((wide == fill).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n_new", [1, 37, 400])
def test_append_from_strided_rows_into_pages_with_gaps(gpu, n_new):
    lens, new_lens = [0, 63, 130], [n_new, n_new // 2, n_new]
    table, pages = _table([n + n_new for n in lens], 3)
    pool = torch.randint(0, 256, (pages, 64, 400), dtype=torch.uint8, generator=torch.Generator().manual_seed(4))
    new = seeded((3, n_new, 576), 5, 2.0, torch.bfloat16)
    expect = pool.clone()
    packed = R.q4_pack(new)
    for b, (n, e) in enumerate(zip(lens, new_lens)):
        for t in range(e):
            expect[int(table[b, (n + t) // 64]), (n + t) % 64] = packed[b, t]
    wide, part = _part(pool, gpu, (2, 0, 0), (1, 6, 0), 77)           # pages 70 rows apart
    _, rows = _part(new, gpu, (1, 2, 16), (1, 3, 48), float("nan"))   # rows of 640 values
    _, cols = _part(table, gpu, (0, 3), (0, 2), 1 << 30)
    i32 = dict(dtype=torch.int32, device=gpu)
    ops.flash_dmla_kv_append_q4(part, cols, torch.tensor(lens, **i32), rows, torch.tensor(new_lens, **i32), check_indices=True)
    assert torch.equal(part.cpu(), expect)
    assert _around(wide, part, 77)


def _evict_parts(gpu, pool, table, sl, mass, budget, recent, sink, before, after, fill):
    ref_pool, ref_lens, ref_src, ref_mass = R.kv_evict(pool, table, sl, mass, budget, recent, sink)
    wide, part = _part(pool, gpu, before, after, fill)
    accounts, m = _part(mass, gpu, (1, 7), (0, 9), -1.0)
    _, cols = _part(table, gpu, (0, 3), (0, 2), 1 << 30)
    new_lens, src, new_mass = ops.flash_dmla_kv_evict(part, cols, sl.to(gpu), m, budget, recent, sink, check_indices=True)
    assert torch.equal(new_lens.cpu(), ref_lens) and torch.equal(src.cpu(), ref_src)
    assert torch.equal(new_mass.cpu(), ref_mass) and torch.equal(m.cpu(), mass)
    assert torch.equal(part.cpu(), ref_pool)
    assert _around(wide, part, fill) and _around(accounts, m, -1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("budget,recent,sink", [(100, 20, 4), (300, 250, 0), (1, 0, 0)])
@pytest.mark.parametrize("width", [8, 72, 576, 1024])
def test_evict_of_bf16_rows_of_any_width_with_gaps(gpu, width, budget, recent, sink):
    """Row strides above the row and pages with a gap; rows of 16 bytes to 2 KB."""
    lens = [0, 64, 131, 640, 333]
    table, pages = _table(lens, 6)
    pool = seeded((pages, 64, width), 7, 1.0, torch.bfloat16)
    mass = torch.exp(2.0 * seeded((len(lens), 640), 8))
    _evict_parts(gpu, pool, table, torch.tensor(lens, dtype=torch.int32), mass, budget, recent, sink, (1, 0, 16), (0, 5, 40), 5.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [700, 20000])
def test_evict_of_4_bit_pages_with_gaps(gpu, n):
    """Tables that one workgroup holds, and longer ones."""
    lens = [n, n // 3, 50]
    pool, table, sl = _pool(lens, 9, True)
    mass = torch.exp(2.0 * seeded((3, table.shape[1] * 64 + 3), 10))
    _evict_parts(gpu, pool, table, sl, mass, n // 4, n // 10, 4, (1, 0, 0), (1, 3, 0), 99)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 128])
def test_accounts_of_bf16_rows_with_gaps(gpu, H):
    """Row strides above the row, pages with a gap, accounts at an odd place of wider rows: the contiguous bits."""
    lens = [300, 0, 1000]
    pool, table, sl = _pool(lens, 11, False)
    q = seeded((3, H, 576), 12, 0.5, torch.bfloat16)
    lse = _lse(q, pool, table, sl).to(gpu)
    mass = seeded((3, table.shape[1] * 64), 13).abs()
    ref = mass.to(gpu)
    ops.flash_dmla_attn_mass(q.to(gpu), pool.to(gpu), table.to(gpu), sl.to(gpu), lse, ref, SCALE)
    _, part = _part(pool, gpu, (1, 2, 8), (0, 4, 56), 3.0)
    accounts, m = _part(mass, gpu, (0, 7), (1, 2), -1.0)
    _, cols = _part(table, gpu, (1, 1), (0, 1), 1 << 30)
    ops.flash_dmla_attn_mass(q.to(gpu), part, cols, sl.to(gpu), lse, m, SCALE)
    assert torch.equal(m, ref)
    assert _around(accounts, m, -1.0)
