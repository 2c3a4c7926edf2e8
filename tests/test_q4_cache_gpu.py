"""The 4-bit latent cache on the GPU: append, gather and decode against the oracle in 64 bits.

Tolerances.  Append and gather are exact: codes, scales and rope bit for bit.  Decode: fp32 scores of
576 products, accumulated in about 20 steps, are within 2^-17 of scale x sum |q k| (64 roundings of
2^-24, with room), which is lse's error beside 1e-5 for its own exp2, log2 and sum.  A bf16 output is
off by the rounding of P (2^-8 of sum p |v|), of the split partials (2^-8 of the same) and its own
(2^-8 of |o|), and by the scores' error times sum p |v|."""
import math

import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from python import ops

SCALE = 1.0 / math.sqrt(192.0)


def _table(lens, seed, spare=2, width=None):
    """A block table in a random page order with page indices that must not be touched (-1) behind each row."""
    need = [(int(n) + 63) // 64 for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(need), width or max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def _cache(lens, seed, x=None, std=0.5):
    """(pool, table, lens tensor): rows past each sequence's end are all ones, a NaN scale and NaN rope."""
    table, pages = _table(lens, seed)
    pool = torch.full((pages, 64, 400), 255, dtype=torch.uint8)
    for b, n in enumerate(lens):
        rows = seeded((n, 576), seed + 100 + b, std, torch.bfloat16) if x is None else x[b][:n]
        packed = R.q4_pack(rows)
        for j in range(0, n, 64):
            pool[int(table[b, j // 64]), :min(64, n - j)] = packed[j:j + 64]
    return pool, table, torch.tensor(lens, dtype=torch.int32)


def _reference(q, pool, table, lens, scale):
    """o, lse, and the tolerances of both, in float64."""
    B, H, _ = q.shape
    o, lse = torch.zeros(B, H, 512, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.full_like(o, 1e-30), torch.full_like(lse, 1e-5)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        k = R.q4_unpack(R.gather_pages(pool, table[b], n, 64))
        x = q[b].double() @ k.T * scale
        lse[b] = torch.logsumexp(x, 1)
        p = torch.exp(x - lse[b][:, None])
        o[b] = p @ k[:, :512]
        s_err = 2.0 ** -17 * scale * (q[b].double().abs() @ k.abs().T).amax(1) + 1e-5
        av = p @ k[:, :512].abs()
        tol_l[b] = s_err
        tol_o[b] = 2.0 ** -8 * (2.0 * av + o[b].abs()) + 2.0 * s_err[:, None] * av + 1e-30
    return o, lse, tol_o, tol_l


def _spacious(table, tiles=1200):
    """The same table in a wider one of at least that many 32-token tiles, with pages that must not be touched."""
    B, n = table.shape
    return torch.cat((table, torch.full((B, max(0, tiles // (2 * B) + 1 - n)), -1, dtype=torch.int32)), 1)


def _check(gpu, q, pool, table, lens, scale=SCALE):
    if q.shape[1] > 64 and 2 * table.numel() < 1200:   # small and large batches run in different kernels
        _check(gpu, q, pool, _spacious(table), lens, scale)
    o, lse = ops.flash_dmla_decode_paged_q4(q.to(gpu), pool.to(gpu), table.to(gpu), lens.to(gpu), 512, scale, return_lse=True)
    torch.cuda.synchronize()
    o_ref, lse_ref, tol_o, tol_l = _reference(q, pool, table, lens, scale)
    o, lse = o.double().cpu(), lse.double().cpu()
    empty = lens == 0
    assert torch.isneginf(lse[empty]).all() and (o[empty] == 0).all()
    assert torch.isfinite(o).all() and torch.isfinite(lse[~empty]).all()
    worst = ((lse - lse_ref).abs() / tol_l)[~empty]
    assert worst.numel() == 0 or worst.max() <= 1, f"lse off by {worst.max():.3g} tolerances"
    worst = ((o - o_ref).abs() / tol_o)[~empty]
    assert worst.numel() == 0 or worst.max() <= 1, f"o off by {worst.max():.3g} tolerances"


# ---- append and gather -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("lens,new_lens,n_new", [([0], [1], 1), ([0, 63, 64, 200], [70, 1, 130, 0], 130),
                                                 ([5, 0, 1000], [3, 7, 2], 7), ([0] * 70, [1 + 9 * b % 40 for b in range(70)], 40)])
def test_append_writes_the_oracle_rows_and_nothing_else(gpu, lens, new_lens, n_new):
    table, pages = _table([n + e for n, e in zip(lens, new_lens)], 3)
    pool = torch.randint(0, 256, (pages, 64, 400), dtype=torch.uint8, generator=torch.Generator().manual_seed(4))
    new = seeded((len(lens), n_new, 576), 5, 2.0, torch.bfloat16)
    expect = pool.clone()
    packed = R.q4_pack(new)
    for b, (n, e) in enumerate(zip(lens, new_lens)):
        for t in range(e):
            expect[int(table[b, (n + t) // 64]), (n + t) % 64] = packed[b, t]
    pg = pool.to(gpu)
    ops.flash_dmla_kv_append_q4(pg, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), new.to(gpu),
                                torch.tensor(new_lens, dtype=torch.int32, device=gpu), check_indices=True)
    assert torch.equal(pg.cpu(), expect)


@pytest.mark.gpu
def test_append_of_every_bf16_value(gpu):
    """All 65536 bf16 patterns (subnormals, infinities and NaN among them) at several block scales, codes and
    scales as the oracle's; the sign of a NaN block's codes and the rope's bits are kept as they come."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = bits.reshape(128, 512)
    x = torch.cat((x, bits[torch.randperm(65536, generator=torch.Generator().manual_seed(1))].reshape(128, 512)))
    finite = torch.where(torch.isfinite(x.float()), x, torch.zeros_like(x))
    one = torch.zeros(256, 512, dtype=torch.bfloat16)
    one[:, ::32] = finite[:, ::32]
    rows = torch.cat((x, finite, one))
    rows = torch.cat((rows, rows[:, :64]), dim=1).contiguous()
    table, pages = _table([len(rows)], 2)
    pool = torch.zeros(pages, 64, 400, dtype=torch.uint8, device=gpu)
    ops.flash_dmla_kv_append_q4(pool, table.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu), rows[None].to(gpu))
    got = R.gather_pages(pool.cpu(), table[0], len(rows), 64)
    assert torch.equal(got, R.q4_pack(rows))


@pytest.mark.gpu
def test_append_skips_and_flags_bad_pages(gpu):
    table, pages = _table([100, 20], 6)
    table[0, 1] = pages + 3
    pool = torch.zeros(pages, 64, 400, dtype=torch.uint8, device=gpu)
    new = seeded((2, 100, 576), 7, 1.0, torch.bfloat16)
    args = (pool, table.to(gpu), torch.zeros(2, dtype=torch.int32, device=gpu), new.to(gpu),
            torch.tensor([100, 20], dtype=torch.int32, device=gpu))
    with pytest.raises(ValueError, match="out of range"):
        ops.flash_dmla_kv_append_q4(*args, check_indices=True)
    expect = torch.zeros(pages, 64, 400, dtype=torch.uint8)
    expect[int(table[0, 0])] = R.q4_pack(new[0, :64])
    expect[int(table[1, 0]), :20] = R.q4_pack(new[1, :20])
    assert torch.equal(pool.cpu(), expect)
    # rows past the table's last page are skipped as well
    args[2].fill_(2 * 64)
    with pytest.raises(ValueError, match="out of range"):
        ops.flash_dmla_kv_append_q4(*args, check_indices=True)
    assert torch.equal(pool.cpu(), expect)


@pytest.mark.gpu
def test_gather_windows_zeros_and_bad_pages(gpu):
    lens = [0, 1, 64, 65, 300]
    pool, table, sl = _cache(lens, 8)
    pool[int(table[1, 0]), 0, 256] = 255   # a block that is not a number
    starts = torch.tensor([0, 0, 63, -5, 250], dtype=torch.int32)
    for st in (None, starts):
        out = ops.flash_dmla_kv_gather_q4(pool.to(gpu), table.to(gpu), sl.to(gpu), 70, None if st is None else st.to(gpu))
        expect = torch.zeros(5, 70, 576, dtype=torch.float64)
        for b, n in enumerate(lens):
            s = 0 if st is None else max(int(st[b]), 0)
            rows = R.q4_unpack(R.gather_pages(pool, table[b], n, 64))[s:s + 70]
            expect[b, :len(rows)] = rows
        assert torch.equal(out.double().cpu().nan_to_num(7e7), expect.nan_to_num(7e7))
    bad = table.clone()
    bad[4, 0] = pool.shape[0]
    out = ops.flash_dmla_kv_gather_q4(pool.to(gpu), bad.to(gpu), sl.to(gpu), 70)
    assert out[4, :64].isnan().all() and out[4, 64:].isfinite().all()
    # a length past the table ends at the table
    out = ops.flash_dmla_kv_gather_q4(pool.to(gpu), table[:, :1].contiguous().to(gpu), torch.full_like(sl, 1000).to(gpu), 70)
    assert (out[2:, 64:] == 0).all()
    assert ops.flash_dmla_kv_gather_q4(pool.to(gpu), table.to(gpu), sl.to(gpu), 0).shape == (5, 0, 576)


# ---- decode ------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("H", [1, 5, 16, 17, 32, 33, 64, 65, 128, 129, 200])
def test_decode_lengths_around_tiles_and_pages(gpu, H):
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 200, 255, 257, 640]
    pool, table, sl = _cache(lens, 11 + H)
    _check(gpu, seeded((len(lens), H, 576), 12, 0.5, torch.bfloat16), pool, table, sl)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [3, 16, 32, 64, 128])
def test_decode_long_contexts_split_over_workgroups(gpu, H):
    lens = [5000, 0, 9001, 1]
    pool, table, sl = _cache(lens, 21)
    _check(gpu, seeded((len(lens), H, 576), 22, 0.5, torch.bfloat16), pool, table, sl)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H", [(257, 16), (600, 128), (300, 40)])
def test_decode_more_sequences_than_a_chunk_of_the_plan(gpu, B, H):
    lens = [(37 * b) % 150 for b in range(B)]
    pool, table, sl = _cache(lens, 31)
    _check(gpu, seeded((B, H, 576), 32, 0.5, torch.bfloat16), pool, table, sl)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 64, 128])
def test_decode_segment_of_more_pages_than_a_register_holds(gpu, H):
    """More than 64 pages per workgroup: 256 workgroups, 300 equal sequences of 70 pages (pages shared)."""
    pool, table, _ = _cache([70 * 64 - 5], 41)
    B = 300
    tables = table.repeat(B, 1)
    sl = torch.full((B,), 70 * 64 - 5, dtype=torch.int32)
    q = seeded((1, H, 576), 42, 0.5, torch.bfloat16).repeat(B, 1, 1)
    o, lse = ops.flash_dmla_decode_paged_q4(q.to(gpu), pool.to(gpu), tables.to(gpu), sl.to(gpu), 512, SCALE, return_lse=True)
    o_ref, lse_ref, tol_o, tol_l = _reference(q[:1], pool, table, sl[:1], SCALE)
    assert ((o.double().cpu() - o_ref).abs() <= tol_o).all() and ((lse.double().cpu() - lse_ref).abs() <= tol_l).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 32, 64, 128])
@pytest.mark.parametrize("grow", [1, -1])
def test_decode_scores_that_climb_or_fall_along_the_context(gpu, H, grow):
    """Scores span ~86 in log2 units along the context, up or down: the softmax reference has to follow."""
    lens = [700, 2100, 37]
    x = [seeded((n, 576), 50 + b, 0.5, torch.bfloat16) for b, n in enumerate(lens)]
    for b, n in enumerate(lens):
        ramp = 30.0 * torch.arange(n) / max(n - 1, 1)
        x[b][:, 512] = (ramp if grow > 0 else ramp.flip(0)).to(torch.bfloat16)
    pool, table, sl = _cache(lens, 51, x=x)
    q = seeded((3, H, 576), 52, 0.5, torch.bfloat16)
    q[..., 512] = 4.0
    _check(gpu, q, pool, table, sl, 0.5)


@pytest.mark.gpu
def test_decode_wide_query_ranges(gpu):
    """Query values over 2^-60 .. 2^8 inside a block of 32, zero queries, and rows of huge and tiny scales."""
    lens = [100, 70]
    e = torch.randint(-60, 9, (2, 16, 576), generator=torch.Generator().manual_seed(3)).float()
    q = (seeded((2, 16, 576), 61) * torch.exp2(e)).to(torch.bfloat16)
    q[0, 3] = 0
    pool, table, sl = _cache(lens, 62)
    _check(gpu, q, pool, table, sl, 0.01)
    x = [seeded((n, 576), 63 + b, 2.0 ** (60 if b else -60), torch.bfloat16) for b, n in enumerate(lens)]
    pool, table, sl = _cache(lens, 64, x=x)
    q = seeded((2, 16, 576), 65, 1.0, torch.bfloat16) * torch.tensor([2.0 ** 60, 2.0 ** -60]).view(2, 1, 1).to(torch.bfloat16)
    _check(gpu, q, pool, table, sl, 0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious", [(24, False), (24, True), (128, False), (128, True)])
def test_decode_strided_tensors_and_large_offsets(gpu, H, spacious):
    lens = [130, 64, 77]
    pool, table, sl = _cache(lens, 71)
    table = _spacious(table) if spacious else table
    q = seeded((3, H, 576), 72, 0.5, torch.bfloat16)
    o_ref = ops.flash_dmla_decode_paged_q4(q.to(gpu), pool.to(gpu), table.to(gpu), sl.to(gpu), 512, SCALE)
    # query and table as parts of larger tensors, pages with a gap between them
    qw = torch.zeros(3, H + 6, 640, dtype=torch.bfloat16, device=gpu)
    qw[:, 3:3 + H, 32:608] = q.to(gpu)
    tw = torch.full((3, table.shape[1] + 6), 1 << 30, dtype=torch.int32, device=gpu)
    tw[:, 2:2 + table.shape[1]] = table.to(gpu)
    pw = torch.zeros(pool.shape[0], 70, 400, dtype=torch.uint8, device=gpu)
    pw[:, :64] = pool.to(gpu)
    o = ops.flash_dmla_decode_paged_q4(qw[:, 3:3 + H, 32:608], pw[:, :64], tw[:, 2:2 + table.shape[1]], sl.to(gpu), 512, SCALE)
    assert torch.equal(o, o_ref)
    # pages past 4 GiB of the pool
    far = torch.empty(200000, 64, 400, dtype=torch.uint8, device=gpu)
    far[-pool.shape[0]:] = pool.to(gpu)
    tf = torch.where(table >= 0, table + (far.shape[0] - pool.shape[0]), table)
    o = ops.flash_dmla_decode_paged_q4(q.to(gpu), far, tf.to(gpu), sl.to(gpu), 512, SCALE)
    assert torch.equal(o, o_ref)
    rows = ops.flash_dmla_kv_gather_q4(far, tf.to(gpu), sl.to(gpu), 130)
    assert torch.equal(rows, ops.flash_dmla_kv_gather_q4(pool.to(gpu), table.to(gpu), sl.to(gpu), 130))


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious", [(24, False), (128, False), (128, True)])
def test_decode_lengths_past_the_table_and_negative_ones(gpu, H, spacious):
    """A length past the table ends at the table, a negative one is empty."""
    lens = [130, 64, 77]
    pool, table, sl = _cache(lens, 71)
    q = seeded((3, H, 576), 72, 0.5, torch.bfloat16)
    if spacious:   # 400 columns of one good page: the first sequence fills the table
        table = torch.cat((table, table[:, :1].expand(3, 397)), 1).contiguous()
        over, full = torch.tensor([10 ** 9, 64, -3], dtype=torch.int32), torch.tensor([25600, 64, 0], dtype=torch.int32)
        pool2 = pool.clone()
        pool2[int(table[0, 2]), 2:] = pool[int(table[0, 0]), 2:]
        args = (q.to(gpu), pool2.to(gpu), table.to(gpu))
        a, la = ops.flash_dmla_decode_paged_q4(*args, over.to(gpu), 512, SCALE, return_lse=True)
        b, lb = ops.flash_dmla_decode_paged_q4(*args, full.to(gpu), 512, SCALE, return_lse=True)
        assert a.isfinite().all() and torch.equal(a, b) and torch.equal(la, lb)
        assert torch.isneginf(la[2]).all() and (a[2] == 0).all()
        return
    over = torch.tensor([10 ** 9, 64, -3], dtype=torch.int32)
    full = torch.tensor([192, 64, 0], dtype=torch.int32)
    pool2 = pool.clone()
    pool2[int(table[0, 2]), 2:] = pool[int(table[0, 0]), 2:]
    args = (q.to(gpu), pool2.to(gpu), table.to(gpu))
    a, la = ops.flash_dmla_decode_paged_q4(*args, over.to(gpu), 512, SCALE, return_lse=True)
    b, lb = ops.flash_dmla_decode_paged_q4(*args, full.to(gpu), 512, SCALE, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.isneginf(la[2]).all() and (a[2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious", [(16, False), (64, False), (128, False), (128, True)])
def test_decode_poison_stays_with_its_sequence_or_head(gpu, H, spacious):
    lens = [200, 3000, 90, 64]
    pool, table, sl = _cache(lens, 81)
    table = _spacious(table) if spacious else table
    q = seeded((4, H, 576), 82, 0.5, torch.bfloat16)
    good = ops.flash_dmla_decode_paged_q4(q.to(gpu), pool.to(gpu), table.to(gpu), sl.to(gpu), 512, SCALE)
    for bad_page in (pool.shape[0], -1, 1 << 30):
        bad = table.clone()
        bad[1, 20] = bad_page
        o, lse = ops.flash_dmla_decode_paged_q4(q.to(gpu), pool.to(gpu), bad.to(gpu), sl.to(gpu), 512, SCALE, return_lse=True)
        assert o[1].isnan().all() and lse[1].isnan().all()
        assert torch.equal(o[[0, 2, 3]], good[[0, 2, 3]])
    with pytest.raises(ValueError, match="page index"):
        ops.flash_dmla_decode_paged_q4(q.to(gpu), pool.to(gpu), bad.to(gpu), sl.to(gpu), 512, SCALE, check_indices=True)
    # a key that is not a number takes its sequence, a query its head
    nan_key = pool.clone()
    nan_key[int(table[2, 1]), 5, 260] = 255
    o = ops.flash_dmla_decode_paged_q4(q.to(gpu), nan_key.to(gpu), table.to(gpu), sl.to(gpu), 512, SCALE)
    assert o[2].isnan().all() and torch.equal(o[[0, 1, 3]], good[[0, 1, 3]])
    for v in (float("nan"), float("inf")):
        qn = q.clone()
        qn[0, H // 2, 100] = v
        o = ops.flash_dmla_decode_paged_q4(qn.to(gpu), pool.to(gpu), table.to(gpu), sl.to(gpu), 512, SCALE)
        assert o[0, H // 2].isnan().all()
        o[0, H // 2] = good[0, H // 2]
        assert torch.equal(o, good)


@pytest.mark.gpu
def test_a_serving_step_on_4_bit_pages_eager_captured_and_on_another_stream(gpu):
    """Append, decode and account, then gather, as a program runs them; the step captured into two graphs
    replays to the eager results, and a step on another stream gives the same."""
    lens = [100, 1, 700]
    H, n_new = 24, 3
    total = [n + n_new for n in lens]
    table, pages = _table(total, 91)
    pool = torch.zeros(pages, 64, 400, dtype=torch.uint8)
    x = [seeded((n, 576), 92 + b, 0.5, torch.bfloat16) for b, n in enumerate(lens)]
    for b, n in enumerate(lens):
        packed = R.q4_pack(x[b])
        for j in range(0, n, 64):
            pool[int(table[b, j // 64]), :min(64, n - j)] = packed[j:j + 64]
    new, q = seeded((3, n_new, 576), 95, 0.5, torch.bfloat16), seeded((3, H, 576), 96, 0.5, torch.bfloat16)
    tg, lg, ng, qg = table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), new.to(gpu), q.to(gpu)
    sl = torch.tensor(total, dtype=torch.int32)

    def step(pg, mass):
        ops.flash_dmla_kv_append_q4(pg, tg, lg, ng)
        o, lse = ops.flash_dmla_decode_paged_q4(qg, pg, tg, lg + n_new, 512, SCALE, return_lse=True)
        ops.flash_dmla_attn_mass(qg, pg, tg, lg + n_new, lse, mass, SCALE)
        return o, lse

    pg, mass = pool.to(gpu), torch.zeros(3, table.shape[1] * 64, device=gpu)
    o, lse = step(pg, mass)
    full = pg.cpu()
    for b in range(3):
        rows = torch.cat((x[b], new[b]))
        assert torch.equal(R.gather_pages(full, table[b], total[b], 64), R.q4_pack(rows))
    o_ref, lse_ref, tol_o, tol_l = _reference(q, full, table, sl, SCALE)
    assert ((o.double().cpu() - o_ref).abs() <= tol_o).all() and ((lse.double().cpu() - lse_ref).abs() <= tol_l).all()
    assert (mass.sum(1).cpu() - H).abs().max() <= H * 1e-4   # each head's weights sum to one
    k_lat = ops.flash_dmla_kv_gather_q4(pg, tg, lg + n_new, max(total))
    assert k_lat.shape == (3, max(total), 576) and torch.isfinite(k_lat).all()

    graphs = []
    for _ in range(2):
        p2, m2 = pool.to(gpu), torch.zeros_like(mass)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(p2.clone(), m2.clone())
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(p2, m2)
        graphs.append((g, p2, m2, outs))
    for k in range(3):
        for g, p2, m2, outs in graphs:
            m2.zero_()
            outs[0].fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], o) and torch.equal(outs[1], lse) and torch.equal(p2, pg) and torch.equal(m2, mass)
        again = step(pg, torch.zeros_like(mass))
        assert torch.equal(again[0], o)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        m3 = torch.zeros_like(mass)
        o3, _ = step(pool.to(gpu), m3)
    other.synchronize()
    assert torch.equal(o3, o) and torch.equal(m3, mass)
    # the dispatcher ops are the same calls
    f = torch.ops.flashdmla
    o4, lse4 = f.decode_paged_q4(qg, pg, tg, lg + n_new, 512, SCALE)
    assert torch.equal(o4, o) and torch.equal(lse4, lse)
    assert torch.equal(f.kv_gather_q4(pg, tg, lg + n_new, max(total), None), k_lat)
