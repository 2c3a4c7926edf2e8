"""The 4-bit cache, the accounts and the eviction where their kernels change shape: many rows, outputs past the last
cache, long block tables, captured calls of each.  Exact, or against the eager result of the same call."""
import math

import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from python import ops

SCALE = 1.0 / math.sqrt(192.0)


def _device_cache(gpu, lens, seed):
    """Pages of finite random rows in a random order."""
    need = [(n + 63) // 64 for n in lens]
    g = torch.Generator(device=gpu).manual_seed(seed)
    pool = torch.randint(0, 256, (sum(need), 64, 400), dtype=torch.uint8, generator=g, device=gpu)
    pool[:, :, 256:272] = 120 + torch.randint(0, 8, (sum(need), 64, 16), generator=g, device=gpu).to(torch.uint8)
    rope = (torch.randn(sum(need), 64, 64, generator=g, device=gpu) * 0.5).bfloat16()
    pool[:, :, 272:] = rope.view(torch.uint8)
    perm = torch.randperm(sum(need), generator=g, device=gpu).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=gpu)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return pool, table, torch.tensor(lens, dtype=torch.int32, device=gpu)


def _captured(call):
    """call() captured after an eager run on a side stream: (graph, its outputs)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    return g, out


@pytest.mark.gpu
@pytest.mark.parametrize("n_new,new_lens", [(7000, [7000, 6999, 1, 0, 3333]), (2100, [2100, 77, 2099, 1, 64])])
def test_append_of_many_rows(gpu, n_new, new_lens):
    """Waves that take several neighbouring rows, across sequences and pages, and rows that are not written."""
    lens = [0, 100, 5, 64, 63]
    total = [n + e for n, e in zip(lens, new_lens)]
    need = [(n + 63) // 64 for n in total]
    perm = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.full((5, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    pool = torch.randint(0, 256, (sum(need) + 2, 64, 400), dtype=torch.uint8, generator=torch.Generator().manual_seed(2))
    new = seeded((5, n_new, 576), 3, 2.0, torch.bfloat16)
    expect = pool.clone()
    for b in range(5):
        t = torch.arange(new_lens[b]) + lens[b]
        expect[table[b, t // 64].long(), t % 64] = R.q4_pack(new[b, :new_lens[b]])
    pg = pool.to(gpu)
    ops.flash_dmla_kv_append_q4(pg, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), new.to(gpu),
                                torch.tensor(new_lens, dtype=torch.int32, device=gpu), check_indices=True)
    assert torch.equal(pg.cpu(), expect)


@pytest.mark.gpu
def test_gather_of_an_output_past_the_last_cache(gpu):
    """18 sequences of up to 8192 rows (170 MB) at once and one by one."""
    lens = [8192, 0, 1, 8191, 5000] + [4000 + 13 * b for b in range(13)]
    pool, table, sl = _device_cache(gpu, lens, 4)
    out = ops.flash_dmla_kv_gather_q4(pool, table, sl, 8192)
    assert out.numel() * 2 >= 160 << 20
    for b in range(len(lens)):
        assert torch.equal(out[b], ops.flash_dmla_kv_gather_q4(pool, table[b:b + 1], sl[b:b + 1], 8192)[0])
        assert (out[b, lens[b]:] == 0).all()
    rows = R.q4_unpack(R.gather_pages(pool.cpu(), table[4].cpu(), 5000, 64))
    assert torch.equal(out[4, :5000].double().cpu(), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 64, 128, 140])
def test_decode_and_accounts_captured_beside_eager_calls(gpu, H):
    lens = [3000, 17, 0, 9000, 640]
    pool, table, sl = _device_cache(gpu, lens, 5)
    q = (torch.randn(5, H, 576, generator=torch.Generator(device=gpu).manual_seed(6), device=gpu) * 0.5).bfloat16()
    mass = torch.zeros(5, table.shape[1] * 64, device=gpu)

    def step():
        o, lse = ops.flash_dmla_decode_paged_q4(q, pool, table, sl, 512, SCALE, return_lse=True)
        mass.zero_()
        ops.flash_dmla_attn_mass(q, pool, table, sl, lse, mass, SCALE)
        return o, lse

    o, lse = step()
    account = mass.clone()
    live = sl > 0
    assert ((account.sum(1) - H)[live].abs() <= H * 1e-4).all() and (account[2] == 0).all()
    graphs = [_captured(step) for _ in range(2)]
    for _ in range(3):
        for g, out in graphs:
            out[0].fill_(float("nan"))
            mass.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], o) and torch.equal(out[1], lse) and torch.equal(mass, account)
        again = step()
        assert torch.equal(again[0], o) and torch.equal(mass, account)


@pytest.mark.gpu
def test_eviction_of_a_long_table_captured_beside_eager_calls(gpu):
    lens = [40000, 16000, 25000]
    pool, table, sl = _device_cache(gpu, lens, 7)
    mass = torch.exp(2.0 * torch.randn(3, table.shape[1] * 64, generator=torch.Generator(device=gpu).manual_seed(8), device=gpu))
    p1, p2 = pool.clone(), pool.clone()
    ref = ops.flash_dmla_kv_evict(p1, table, sl, mass, 20000, 500, 4)
    cpu = pool.cpu()
    ref_pool, ref_lens, ref_src, ref_mass = R.kv_evict(cpu, table.cpu(), sl.cpu(), mass.cpu(), 20000, 500, 4)
    assert torch.equal(p1.cpu(), ref_pool) and torch.equal(ref[1].cpu(), ref_src) and torch.equal(ref[2].cpu(), ref_mass)
    g, out = _captured(lambda: ops.flash_dmla_kv_evict(p2, table, sl, mass, 20000, 500, 4))
    for _ in range(3):
        p2.copy_(pool)
        for x in out:
            x.fill_(-5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(p2, p1) and all(torch.equal(a, b) for a, b in zip(out, ref))
        p3 = pool.clone()
        again = ops.flash_dmla_kv_evict(p3, table, sl, mass, 20000, 500, 4)
        assert torch.equal(p3, p1) and all(torch.equal(a, b) for a, b in zip(again, ref))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [70, 300])
def test_eviction_of_many_long_tables(gpu, B):
    """More sequences than the chip has workgroups for: fewer, longer chunks each.  Copies of three
    sequences agree."""
    lens = [17000, 30, 20001]
    pool, table, sl = _device_cache(gpu, lens, 9)
    mass = torch.exp(2.0 * torch.randn(3, table.shape[1] * 64, generator=torch.Generator(device=gpu).manual_seed(10), device=gpu))
    reps = [b % 3 for b in range(B)]
    one_lens, one_src, one_mass = ops.flash_dmla_kv_evict(pool.clone(), table, sl, mass, 3000, 64, 4)
    big = torch.cat([pool] * ((B + 2) // 3))
    shift = torch.arange((B + 2) // 3, device=gpu, dtype=torch.int32).repeat_interleave(3)[:B, None] * pool.shape[0]
    big_table = table[torch.tensor(reps, device=gpu)] + shift
    new_lens, src, new_mass = ops.flash_dmla_kv_evict(big, big_table, sl[torch.tensor(reps, device=gpu)],
                                                      mass[torch.tensor(reps, device=gpu)].contiguous(), 3000, 64, 4)
    for b in range(B):
        assert int(new_lens[b]) == int(one_lens[reps[b]])
        assert torch.equal(src[b], one_src[reps[b]]) and torch.equal(new_mass[b], one_mass[reps[b]])
    ref = R.kv_evict(pool.cpu(), table.cpu(), sl.cpu(), mass.cpu(), 3000, 64, 4)
    assert torch.equal(one_src.cpu(), ref[2])
    first = big[:pool.shape[0]].cpu()
    last = big[pool.shape[0] * (B // 3 - 1):pool.shape[0] * (B // 3)].cpu()
    assert torch.equal(first, ref[0]) and torch.equal(last, ref[0])
