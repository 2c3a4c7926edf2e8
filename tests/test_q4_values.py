"""The value product of the 4-bit decode at long contexts, to a bound that a single wrong key tile breaks.

A probability enters the value product rounded to bf16, off by at most 2^-8 of itself.  The roundings are of no
common sign, so an output is off by less than c 2^-8 sqrt(sum p^2 v^2) with probability 1 - 2 exp(-c^2 / 2)
(Hoeffding): c = 7 leaves 5e-11 an output, 5e-4 for ten million of them.  Its own rounding is 2^-8 of it, and the
scores' error times sum p |v| is counted in full.  A bound of 2^-8 sum p |v| would grow with the context against
the outputs, which shrink with its root: at 5000 tokens most tiles could be left out within it."""
import math

import pytest
import torch

from conftest import seeded
from oracle import dmla_ref as R
from test_q4_cache_gpu import SCALE, _cache, _spacious

C = 7.0


def _exact(q, k, scale):
    """Of one sequence, q [H, 576] and keys [n, 576] in float64: p, o, lse and the bound of an output's error."""
    x = q.double() @ k.T * scale
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None])
    v = k[:, :512]
    s_err = 2.0 ** -17 * scale * (q.double().abs() @ k.abs().T).amax(1, keepdim=True) + 1e-5
    o = p @ v
    tol = C * 2.0 ** -8 * ((p * p) @ (v * v)).sqrt() + 2.0 ** -8 * o.abs() + 2.0 * s_err * (p @ v.abs()) + 1e-30
    return p, o, lse, tol


def _rounded(p, v, parts):
    """The decode's roundings: P relative to its first tile's largest value as bf16, sums exact; with parts > 1 the
    outputs of that many ranges are rounded to bf16 before they are merged."""
    ref = p[:, :32].amax(1, keepdim=True)
    big = (p / ref).to(torch.bfloat16).double()
    out = torch.zeros(p.shape[0], v.shape[1], dtype=torch.float64)
    for c, cv in zip(big.chunk(parts, 1), v.chunk(parts, 0)):
        w = c.sum(1, keepdim=True)
        part = c @ cv / w
        out += (part.to(torch.bfloat16).double() if parts > 1 else part) * w
    return (out * ref).to(torch.bfloat16).double()


@pytest.mark.parametrize("n", [5000, 9001])
def test_the_bound_breaks_with_any_one_wrong_tile(n):
    k = R.q4_unpack(R.q4_pack(seeded((n, 576), 121, 0.5, torch.bfloat16)))
    p, o, _, tol = _exact(seeded((16, 576), 22, 0.5, torch.bfloat16), k, SCALE)
    v = k[:, :512]
    assert ((_rounded(p, v, 1) - o).abs() <= tol).all()
    for t in range(0, n, 32):
        here, after = slice(t, min(n, t + 32)), slice(t + 32, t + 64)
        assert ((p[:, here] @ v[here]).abs() > tol).any(), f"tile at {t} left out"
        if t + 64 <= n:
            assert ((p[:, here] @ (v[after] - v[here])).abs() > tol).any(), f"the next tile's values at {t}"


def _check(gpu, q, pool, table, lens, scale=SCALE):
    o, lse = _decode(q.to(gpu), pool.to(gpu), table.to(gpu), lens.to(gpu), scale)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            assert (o[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        _, ref, _, tol = _exact(q[b], R.q4_unpack(R.gather_pages(pool, table[b], n, 64)), scale)
        off = (o[b].double().cpu() - ref).abs() / tol
        assert off.max() <= 1, f"sequence {b} of {n}: o off by {off.max():.3g} of the bound"


def _decode(q, pool, table, lens, scale):
    from python import ops
    return ops.flash_dmla_decode_paged_q4(q, pool, table, lens, 512, scale, return_lse=True)


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious", [(3, False), (16, False), (32, False), (64, False), (64, True), (65, False),
                                        (65, True), (128, False), (128, True), (200, True)])
@pytest.mark.parametrize("lens", [[5000, 0, 9001, 1], [33, 97, 2017, 64, 700, 31]])
def test_values_of_long_contexts(gpu, H, spacious, lens):
    """Every tile counts, in one part or several, in both kernels (tables of more tiles choose the other one)."""
    pool, table, sl = _cache(lens, 221)
    _check(gpu, seeded((len(lens), H, 576), 222, 0.5, torch.bfloat16), pool, _spacious(table) if spacious else table, sl)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 128])
def test_values_of_segments_of_many_pages(gpu, H):
    """300 equal sequences of 70 pages over 256 workgroups: segments of more pages than a register holds."""
    n = 70 * 64 - 5
    pool, table, _ = _cache([n], 241)
    q = seeded((1, H, 576), 242, 0.5, torch.bfloat16)
    o, _ = _decode(q.repeat(300, 1, 1).to(gpu), pool.to(gpu), table.repeat(300, 1).to(gpu),
                      torch.full((300,), n, dtype=torch.int32, device=gpu), SCALE)
    _, ref, _, tol = _exact(q[0], R.q4_unpack(R.gather_pages(pool, table[0], n, 64)), SCALE)
    assert ((o.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("grow", [1, -1])
def test_values_where_scores_climb_or_fall(gpu, H, grow):
    """Scores span 87 and 35 in log2 units along the contexts: past the headroom over the first reference, or mostly
    within it."""
    lens = [1500, 4001]
    x = [seeded((n, 576), 250 + b, 0.5, torch.bfloat16) for b, n in enumerate(lens)]
    for b, n in enumerate(lens):
        ramp = (12.0 if b else 30.0) * torch.arange(n) / (n - 1)
        x[b][:, 512] = (ramp if grow > 0 else ramp.flip(0)).to(torch.bfloat16)
    pool, table, sl = _cache(lens, 251, x=x)
    q = seeded((2, H, 576), 252, 0.5, torch.bfloat16)
    q[..., 512] = 4.0
    for t in (table, _spacious(table)):
        _check(gpu, q, pool, t, sl, 0.5)


def _rms_limit(p, o, v):
    """(the rms error of fp32 parts, the limit) by variances: the rounding of the exact result, P's, and for the limit
    half of what many bf16 parts would add.  Part s weighs w_s; its output's random share is (sum p^2 v^2)^1/2 / w_s
    over its keys, and rounded like the result, the parts together add the result's relative rounding of
    (sum p^2 v^2)^1/2 over all keys.  (What the parts have in common adds a share that falls with their number.)"""
    own = (o.to(torch.bfloat16).double() - o).square().mean()
    of_parts = own * ((p * p) @ (v * v)).mean() / o.square().mean()
    big = p / p[:, :32].amax(1, keepdim=True)
    of_p = ((big.to(torch.bfloat16).double() - big) @ v * p[:, :32].amax(1, keepdim=True)).square().mean()
    return float(own + of_p) ** 0.5, float(own + of_p + 0.5 * of_parts) ** 0.5


def test_the_rms_limit_lies_between_fp32_and_bf16_parts():
    k = R.q4_unpack(R.q4_pack(seeded((9001, 576), 261, 0.5, torch.bfloat16)))
    p, o, _, _ = _exact(seeded((32, 576), 262, 0.5, torch.bfloat16), k, SCALE)
    expect, limit = _rms_limit(p, o, k[:, :512])
    fp32 = float((_rounded(p, k[:, :512], 1) - o).square().mean()) ** 0.5
    bf16 = float((_rounded(p, k[:, :512], 30) - o).square().mean()) ** 0.5
    assert abs(fp32 / expect - 1) < 0.02 and fp32 < 0.96 * limit and bf16 > 1.04 * limit


@pytest.mark.gpu
@pytest.mark.parametrize("H,spacious", [(16, False), (64, True), (128, False), (128, True)])
def test_parts_of_a_split_sequence_stay_in_fp32(gpu, H, spacious):
    pool, table, sl = _cache([9001], 261)
    q = seeded((1, H, 576), 262, 0.5, torch.bfloat16)
    k = R.q4_unpack(R.gather_pages(pool, table[0], 9001, 64))
    o, _ = _decode(q.to(gpu), pool.to(gpu), (_spacious(table, 3000) if spacious else table).to(gpu), sl.to(gpu), SCALE)
    p, ref, _, _ = _exact(q[0], k, SCALE)
    rms = float((o[0].double().cpu() - ref).square().mean()) ** 0.5
    expect, limit = _rms_limit(p, ref, k[:, :512])
    assert rms <= limit, f"rms {rms:.4g}, expected {expect:.4g}"
