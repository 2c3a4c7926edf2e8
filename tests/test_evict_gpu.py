"""The accounts of attention weight and the eviction on the GPU, against the oracle.

Accounts: a token's weight is exp of a score that is within 2^-17 of scale x sum |q k| (fp32 sums of
576 products) beside 1e-5 for exp2 and the scaling, times the weight, and the additions round by
2^-23 of the account.  The eviction moves bytes and ranks numbers: everything is exact."""
import math

import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from python import ops
from test_q4_cache_gpu import _cache, _table

SCALE = 1.0 / math.sqrt(192.0)


def _pool(lens, seed, q4):
    if q4:
        return _cache(lens, seed)
    table, pages = _table(lens, seed)
    pool = torch.full((pages, 64, 576), float("nan"), dtype=torch.bfloat16)
    for b, n in enumerate(lens):
        rows = seeded((n, 576), seed + 100 + b, 0.5, torch.bfloat16)
        for j in range(0, n, 64):
            pool[int(table[b, j // 64]), :min(64, n - j)] = rows[j:j + 64]
    return pool, table, torch.tensor(lens, dtype=torch.int32)


def _lse(q, pool, table, lens):
    out = torch.full(q.shape[:2], -math.inf)
    for b, n in enumerate(lens.tolist()):
        if n:
            k = R.gather_pages(pool, table[b], n, 64)
            k = R.q4_unpack(k) if k.dtype == torch.uint8 else k.double()
            out[b] = torch.logsumexp(q[b].double() @ k.T * SCALE, 1).float()
    return out


def _check_mass(gpu, lens, H, q4, seed):
    pool, table, sl = _pool(lens, seed, q4)
    q = seeded((len(lens), H, 576), seed + 1, 0.5, torch.bfloat16)
    lse = _lse(q, pool, table, sl)
    mass = seeded((len(lens), table.shape[1] * 64 + 5), seed + 2).abs()
    got = mass.to(gpu)
    ops.flash_dmla_attn_mass(q.to(gpu), pool.to(gpu), table.to(gpu), sl.to(gpu), lse.to(gpu), got, SCALE)
    got = got.cpu()
    ref = R.attn_mass(q, pool, table, sl, lse, mass, SCALE)
    for b, n in enumerate(lens):
        assert torch.equal(got[b, n:], mass[b, n:])
        if n == 0:
            continue
        k = R.gather_pages(pool, table[b], n, 64)
        k = R.q4_unpack(k) if q4 else k.double()
        s_err = 2.0 ** -17 * SCALE * float((q[b].double().abs() @ k.abs().T).max()) + 1e-5
        add = ref[b, :n] - mass[b, :n].double()
        tol = 2.0 * s_err * add + 2.0 ** -22 * ref[b, :n]
        off = (got[b, :n].double() - ref[b, :n]).abs()
        assert (off <= tol).all(), f"sequence {b} of {n}: off by {(off / tol).max():.3g} tolerances"


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("H", [1, 16, 17, 33, 64, 100, 128, 129, 300])
def test_mass_of_small_batches(gpu, H, q4):
    _check_mass(gpu, [0, 1, 31, 32, 33, 63, 64, 65, 129, 500], H, q4, 100 + H)


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("lens,H", [([5000, 0, 9001, 1], 16), ([4097], 128), ([(37 * b) % 150 for b in range(300)], 40)])
def test_mass_of_long_contexts_and_many_sequences(gpu, lens, H, q4):
    _check_mass(gpu, lens, H, q4, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
def test_mass_of_more_pages_than_a_register_holds(gpu, q4):
    """300 sequences that share 150 pages: about 170 pages per workgroup, and sums of many chunks of tokens."""
    n = 150 * 64 - 7
    pool, table, _ = _pool([n], 9, q4)
    q = seeded((1, 16, 576), 10, 0.5, torch.bfloat16)
    sl = torch.tensor([n], dtype=torch.int32)
    lse = _lse(q, pool, table, sl)
    B = 300
    mass = torch.zeros(B, table.shape[1] * 64, device=gpu)
    ops.flash_dmla_attn_mass(q.repeat(B, 1, 1).to(gpu), pool.to(gpu), table.repeat(B, 1).to(gpu), sl.repeat(B).to(gpu),
                             lse.repeat(B, 1).to(gpu), mass, SCALE)
    ref = R.attn_mass(q, pool, table, sl, lse, torch.zeros(1, table.shape[1] * 64), SCALE)
    assert torch.equal(mass, mass[:1].expand_as(mass))
    assert ((mass[:1].double().cpu() - ref).abs() <= 2e-4 * ref).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
def test_mass_heads_without_keys_bad_pages_and_strides(gpu, q4):
    lens = [200, 130]
    pool, table, sl = _pool(lens, 13, q4)
    q = seeded((2, 20, 576), 14, 0.5, torch.bfloat16)
    lse = _lse(q, pool, table, sl)
    lse[0, 3:7] = -math.inf
    bad = table.clone()
    bad[1, 1] = pool.shape[0]
    width = table.shape[1] * 64
    mass = torch.rand(2, width)
    ref = R.attn_mass(q, pool, table, sl, lse, mass, SCALE)
    ref[1, 64:128] = mass[1, 64:128].double()
    # mass as a part of a larger tensor, pages with a gap, the query strided
    wide = torch.zeros(2, width + 40, device=gpu)
    wide[:, 8:8 + width] = mass.to(gpu)
    gap = torch.zeros((pool.shape[0], 70) + tuple(pool.shape[2:]), dtype=pool.dtype, device=gpu)
    gap[:, :64] = pool.to(gpu)
    qw = torch.zeros(2, 30, 640, dtype=torch.bfloat16, device=gpu)
    qw[:, 3:23, 32:608] = q.to(gpu)
    ops.flash_dmla_attn_mass(qw[:, 3:23, 32:608], gap[:, :64], bad.to(gpu), sl.to(gpu), lse.to(gpu), wide[:, 8:8 + width], SCALE)
    assert torch.allclose(wide[:, 8:8 + width].double().cpu(), ref, rtol=2e-4, atol=1e-6)
    assert torch.equal(wide[1, 8 + 64:8 + 128].cpu(), mass[1, 64:128])
    assert (wide[:, :8] == 0).all() and (wide[:, 8 + width:] == 0).all()


def _check_evict(gpu, lens, budget, recent, sink, q4, mass, seed=3):
    pool, table, sl = _pool(lens, seed, q4)
    pool = pool if q4 else pool.nan_to_num(3.0)
    ref_pool, ref_lens, ref_src, ref_mass = R.kv_evict(pool, table, sl, mass, budget, recent, sink)
    pg = pool.to(gpu)
    new_lens, src, new_mass = ops.flash_dmla_kv_evict(pg, table.to(gpu), sl.to(gpu), mass.to(gpu), budget, recent, sink,
                                                      check_indices=True)
    assert torch.equal(new_lens.cpu(), ref_lens)
    assert torch.equal(src.cpu(), ref_src)
    assert torch.equal(new_mass.cpu().nan_to_num(7e7), ref_mass.nan_to_num(7e7))
    assert torch.equal(pg.cpu(), ref_pool)   # the rows that stay, move or are left behind, every byte


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("budget,recent,sink", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 0, 0), (64, 64, 0), (64, 32, 32), (65, 20, 4),
                                                (100, 99, 0), (100, 0, 100), (130, 60, 3), (300, 250, 4), (10 ** 6, 10, 4)])
def test_evict_small(gpu, budget, recent, sink, q4):
    lens = [0, 1, 2, 63, 64, 65, 66, 101, 131, 200, 301, 640]
    mass = torch.exp(2.0 * seeded((len(lens), 640), 5))
    _check_evict(gpu, lens, budget, recent, sink, q4, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "signs", "special", "close", "sorted", "reversed"])
def test_evict_ranks_every_kind_of_account(gpu, kind):
    lens = [500, 333, 40]
    g = torch.Generator().manual_seed(8)
    n = 512
    mass = {"equal": torch.full((3, n), 2.5), "zeros": torch.zeros(3, n) * torch.where(torch.rand(3, n, generator=g) < 0.5, -1.0, 1.0),
            "few": torch.randint(0, 3, (3, n), generator=g).float(), "signs": torch.randn(3, n, generator=g),
            "special": torch.randn(3, n, generator=g), "close": 1.0 + torch.randint(0, 40, (3, n), generator=g) * 2.0 ** -23,
            "sorted": torch.arange(n).float().repeat(3, 1), "reversed": -torch.arange(n).float().repeat(3, 1)}[kind]
    if kind == "special":
        mass[:, ::7] = float("inf")
        mass[:, 1::7] = float("-inf")
        mass[:, 2::7] = float("nan")
        mass[:, 3::7] = -float("nan")
        mass[:, 4::7] = 1e-42
    for budget in (39, 150, 332):
        _check_evict(gpu, lens, budget, 20, 4, False, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("n,budget,recent", [(40000, 10000, 1000), (33000, 32768, 5000), (17000, 100, 0)])
def test_evict_long_contexts(gpu, n, budget, recent, q4):
    lens = [n, n // 2, 100]
    mass = torch.exp(2.0 * seeded((3, (n + 63) // 64 * 64), 6))
    _check_evict(gpu, lens, budget, recent, 4, q4, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("budget,recent,sink", [(9000, 1000, 4), (1, 0, 0), (1, 0, 1), (16385, 0, 0), (5000, 4996, 4), (19999, 12000, 3),
                                                (8192 + 64, 64, 0)])
@pytest.mark.parametrize("kind", ["few", "equal", "specials"])
def test_evict_equal_accounts_in_long_tables(gpu, kind, budget, recent, sink):
    """Tables of more than 16384 tokens, whose accounts share a few values, or one, over all the table."""
    lens = [20000, 16400, 16385, 5, 0]
    shape = (5, (20000 + 63) // 64 * 64)
    mass = torch.floor(seeded(shape, 23).abs() * 3) if kind == "few" else torch.full(shape, 0.25)
    if kind == "specials":
        mass[:, ::7] = float("inf")
        mass[:, 1::7] = float("-inf")
        mass[:, 2::7] = float("nan")
        mass[:, 3::7] = 0.0
        mass[:, 4::7] = -0.0
    _check_evict(gpu, lens, budget, recent, sink, True, mass)


@pytest.mark.gpu
def test_evict_a_bad_page_in_a_long_table(gpu):
    lens = [20000, 17000]
    pool, table, sl = _pool(lens, 25, True)
    mass = seeded((2, table.shape[1] * 64), 26).abs()
    bad = table.clone()
    bad[0, 300] = -1
    pg = pool.to(gpu)
    new_lens, src, new_mass = ops.flash_dmla_kv_evict(pg, bad.to(gpu), sl.to(gpu), mass.to(gpu), 3000, 100, 4)
    ref_pool, ref_lens, ref_src, ref_mass = R.kv_evict(pool, table, torch.tensor([0, 17000], dtype=torch.int32), mass, 3000, 100, 4)
    assert new_lens.tolist() == [20000, 3000]
    assert torch.equal(pg.cpu(), ref_pool)
    assert src[0].tolist() == list(range(3000)) and torch.equal(new_mass[0, :20000].cpu(), mass[0, :20000])
    assert torch.equal(src[1].cpu(), ref_src[1]) and torch.equal(new_mass[1].cpu(), ref_mass[1])


@pytest.mark.gpu
def test_evict_leaves_a_sequence_with_a_bad_page_alone(gpu):
    lens = [200, 300, 150]
    pool, table, sl = _pool(lens, 15, True)
    mass = seeded((3, 320), 16).abs()
    bad = table.clone()
    bad[1, 3] = pool.shape[0]
    pg = pool.to(gpu)
    with pytest.raises(ValueError, match="page index"):
        ops.flash_dmla_kv_evict(pg, bad.to(gpu), sl.to(gpu), mass.to(gpu), 100, 10, 4, check_indices=True)
    pg = pool.to(gpu)
    new_lens, src, new_mass = ops.flash_dmla_kv_evict(pg, bad.to(gpu), sl.to(gpu), mass.to(gpu), 100, 10, 4)
    keep = torch.tensor([200, 0, 150], dtype=torch.int32)
    ref_pool, ref_lens, ref_src, ref_mass = R.kv_evict(pool, table, keep, mass, 100, 10, 4)
    assert new_lens.tolist() == [100, 300, 100]
    assert torch.equal(pg.cpu(), ref_pool)
    assert src[1].tolist() == list(range(100)) and torch.equal(new_mass[1, :300].cpu(), mass[1, :300])
    assert torch.equal(src[[0, 2]].cpu(), ref_src[[0, 2]]) and torch.equal(new_mass[[0, 2]].cpu(), ref_mass[[0, 2]])


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [False, True])
def test_attention_after_an_eviction_is_attention_over_the_kept_tokens(gpu, q4):
    """Decode, account, evict, decode: the second decode equals attention over exactly the kept rows, and a
    captured eviction replays to the eager result."""
    lens, H = [300, 90, 1000], 32
    pool, table, sl = _pool(lens, 17, q4)
    pool = pool if q4 else pool.nan_to_num(0.0)
    q = seeded((3, H, 576), 18, 0.5, torch.bfloat16)
    decode = ops.flash_dmla_decode_paged_q4 if q4 else ops.flash_dmla_decode_paged
    pg, tg, lg, qg = pool.to(gpu), table.to(gpu), sl.to(gpu), q.to(gpu)
    o, lse = decode(qg, pg, tg, lg, 512, SCALE, return_lse=True)
    mass = torch.zeros(3, table.shape[1] * 64, device=gpu)
    ops.flash_dmla_attn_mass(qg, pg, tg, lg, lse, mass, SCALE)
    start = pg.clone()
    new_lens, src, new_mass = ops.flash_dmla_kv_evict(pg, tg, lg, mass, 128, 16, 4)
    assert new_lens.tolist() == [128, 90, 128]
    o2 = decode(qg, pg, tg, new_lens, 512, SCALE)
    for b in range(3):
        rows = R.gather_pages(pool, table[b], lens[b], 64)[src[b, :int(new_lens[b])].long().cpu()]
        k = R.q4_unpack(rows) if q4 else rows.double()
        x = q[b].double() @ k.T * SCALE
        p = torch.softmax(x, 1)
        tol = 2.0 ** -8 * (2.0 * (p @ k[:, :512].abs()) + (p @ k[:, :512]).abs()) + 1e-3 * (p @ k[:, :512].abs())
        assert ((o2[b].double().cpu() - p @ k[:, :512]).abs() <= tol).all()
    p2 = start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.flash_dmla_kv_evict(start.clone(), tg, lg, mass, 128, 16, 4)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = ops.flash_dmla_kv_evict(p2, tg, lg, mass, 128, 16, 4)
    for _ in range(3):
        p2.copy_(start)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], new_lens) and torch.equal(outs[1], src) and torch.equal(outs[2], new_mass)
        assert torch.equal(p2, pg)
        decode(qg, pg, tg, new_lens, 512, SCALE)
    f = torch.ops.flashdmla.kv_evict(start.clone(), tg, lg, mass, 128, 16, 4)
    assert all(torch.equal(a, b) for a, b in zip(f, outs))
