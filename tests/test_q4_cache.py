"""The 4-bit latent cache, the accounts of attention weight and the eviction: host checks (CPU).

The oracle's row format is pinned value by value, its eviction against the definition, and every
entry point's refusals are checked before anything could reach a GPU."""
import ctypes
import math
import random

import pytest
import torch

import python  # noqa: F401  (registers torch.ops.flashdmla.*)
from oracle import dmla_ref as R
from python import _lib, ops

P = ctypes.c_void_p
PTR = 1 << 20
OK, INVALID, UNSUPPORTED, WORKSPACE = (_lib.DMLA_OK, _lib.DMLA_ERR_INVALID_ARG, _lib.DMLA_ERR_UNSUPPORTED,
                                       _lib.DMLA_ERR_WORKSPACE)


# ---- the row format ----------------------------------------------------------------------------
def test_q4_rows_hold_the_nearest_values():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(40, 576, generator=g) * torch.exp2(torch.randint(-20, 20, (40, 1), generator=g).float())).to(torch.bfloat16)
    y = R.q4_unpack(R.q4_pack(x))
    assert torch.equal(y[:, 512:], x[:, 512:].double())
    blocks, got = x[:, :512].double().reshape(-1, 32), y[:, :512].reshape(-1, 32)
    top = blocks.abs().amax(1, keepdim=True)
    # a block's largest value lies in (3, 6] scales, so a step there is at most 2 of them: half of that off
    step = torch.exp2(torch.ceil(torch.log2(top / 6.0)))
    assert ((got - blocks).abs() <= step).all()
    assert ((got - blocks).abs()[blocks.abs() <= 2 * step.expand_as(blocks)] <= 0.25 * step.expand_as(blocks)[blocks.abs() <= 2 * step.expand_as(blocks)]).all()
    assert torch.equal(R.q4_unpack(R.q4_pack(y.to(torch.bfloat16))), y)   # values of the format stay


def test_q4_ties_limits_and_bad_blocks():
    x = torch.zeros(6, 576, dtype=torch.bfloat16)
    x[0, :9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25])
    x[1, 0] = 3.3895313892515355e38        # the largest bf16: past 6 x 2^125, held as that
    x[2, 0], x[2, 1] = 2.0 ** -126, -2.0 ** -126
    x[3, 0] = float("inf")
    x[4, 40] = float("nan")
    y = R.q4_unpack(R.q4_pack(x))
    assert y[0, :9].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0]
    assert y[1, 0] == 6.0 * 2.0 ** 125
    assert y[2, :2].tolist() == [2.0 ** -126, -2.0 ** -126]
    assert y[3, :32].isnan().all() and (y[3, 32:] == 0).all()
    assert y[4, 32:64].isnan().all() and (y[4, :32] == 0).all()
    assert (y[5] == 0).all() and R.q4_pack(x[5:])[0, 256] == 2   # an empty block has the least scale


def test_evict_order_keeps_what_the_definition_keeps():
    r = random.Random(4)
    for _ in range(200):
        n, budget = r.randint(1, 60), r.randint(1, 60)
        recent = r.randint(0, budget)
        sink = r.randint(0, budget - recent)
        mass = torch.tensor([r.choice((0.0, -0.0, 1.0, 2.0, float("nan"), r.random())) for _ in range(n)])
        at = R.kv_evict_order(mass, n, budget, recent, sink)
        assert len(at) == min(n, budget) == len(set(at))
        if n <= budget:
            assert at == list(range(n))
            continue
        assert at[:sink] == list(range(sink)) and at[budget - recent:] == list(range(n - recent, n))
        inner = at[sink:budget - recent]
        gone = [t for t in range(sink, n - recent) if t not in set(inner)]
        for k in inner:
            for d in gone:
                mk, md = float(mass[k]), float(mass[d])
                assert math.isnan(mk) or mk > md or (mk == md and k < d) or (math.isnan(mk) and math.isnan(md) and k < d)
        assert all(t == i for i, t in enumerate(inner, sink) if t < budget - recent)   # what can stays in place


# ---- refusals ----------------------------------------------------------------------------------
def _append(**kw):
    a = dict(pool=PTR, bt=PTR, sl=PTR, nl=None, new=PTR, B=2, n=3, pages=9, max_pages=4, kv_sp=25600, bt_sb=4, nk_sb=3 * 576,
             nk_ss=576)
    a.update(kw)
    return _lib.lib().dmla_kv_append_q4(P(a["pool"]), P(a["bt"]), P(a["sl"]), P(a["nl"]), P(a["new"]), None, a["B"], a["n"],
                                        a["pages"], a["max_pages"], a["kv_sp"], a["bt_sb"], a["nk_sb"], a["nk_ss"], None)


def _gather(**kw):
    a = dict(pool=PTR, bt=PTR, sl=PTR, st=None, out=PTR, B=2, n=3, pages=9, max_pages=4, kv_sp=25600, bt_sb=4, o_sb=3 * 576,
             o_ss=576)
    a.update(kw)
    return _lib.lib().dmla_kv_gather_q4(P(a["pool"]), P(a["bt"]), P(a["sl"]), P(a["st"]), P(a["out"]), a["B"], a["n"],
                                        a["pages"], a["max_pages"], a["kv_sp"], a["bt_sb"], a["o_sb"], a["o_ss"], None)


@pytest.mark.parametrize("call,rows,sb,ss", [(_append, "new", "nk_sb", "nk_ss"), (_gather, "out", "o_sb", "o_ss")])
def test_row_entry_points_refuse(call, rows, sb, ss):
    for name in ("pool", "bt", "sl", rows):
        assert call(**{name: None}) == INVALID
    assert b"null" in _lib.lib().dmla_last_error()
    for bad in (dict(B=-1), dict(n=-1), dict(pages=-1), dict(max_pages=-1), dict(pool=PTR + 8), {rows: PTR + 2},
                dict(kv_sp=25600 - 16), dict(kv_sp=25608), dict(bt_sb=3), {ss: 568}, {ss: 580}, {sb: 1001}):
        assert call(**bad) == INVALID, bad
    assert call(B=1 << 25) == UNSUPPORTED
    assert call(B=1 << 20, n=1 << 20) == UNSUPPORTED
    assert call(B=0) == OK and call(n=0) == OK
    assert _lib.lib().dmla_last_error() == b""


def _decode(**kw):
    a = dict(q=PTR, kv=PTR, bt=PTR, sl=PTR, o=PTR, B=2, H=16, dqk=576, dv=512, pages=9, max_pages=4, q_sb=16 * 576, q_sh=576,
             kv_sp=25600, bt_sb=4, o_sb=16 * 512, o_sh=512, scale=0.07, ws=None, ws_bytes=0)
    a.update(kw)
    return _lib.lib().dmla_decode_paged_q4(P(a["q"]), P(a["kv"]), P(a["bt"]), P(a["sl"]), P(a["o"]), None, a["B"], a["H"],
                                           a["dqk"], a["dv"], a["pages"], a["max_pages"], a["q_sb"], a["q_sh"], a["kv_sp"],
                                           a["bt_sb"], a["o_sb"], a["o_sh"], a["scale"], P(a["ws"]), a["ws_bytes"], None)


def test_decode_q4_refuses():
    for name in ("q", "kv", "bt", "sl", "o"):
        assert _decode(**{name: None}) == INVALID
    for bad in (dict(B=-1), dict(H=-1), dict(pages=0), dict(max_pages=0, bt_sb=0), dict(scale=0.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(q=PTR + 2), dict(kv=PTR + 4), dict(o=PTR + 8), dict(q_sh=577), dict(o_sh=516),
                dict(kv_sp=25592), dict(kv_sp=25608), dict(bt_sb=3)):
        assert _decode(**bad) == INVALID, bad
    for bad in (dict(dqk=64), dict(dv=576), dict(H=1 << 17), dict(B=1 << 21), dict(B=1 << 20, max_pages=2000, bt_sb=2000)):
        assert _decode(**bad) == UNSUPPORTED, bad
    assert _decode() == WORKSPACE
    need = _lib.lib().dmla_decode_q4_workspace_bytes(2, 16)
    assert need > 0 and _decode(ws=PTR, ws_bytes=need - 1) == WORKSPACE
    assert _decode(ws=PTR + 8, ws_bytes=need) == INVALID
    assert _decode(B=0) == OK and _decode(H=0) == OK
    assert _lib.lib().dmla_decode_q4_workspace_bytes(0, 16) == 0


def _mass(**kw):
    a = dict(q=PTR, kv=PTR, bt=PTR, sl=PTR, lse=PTR, mass=PTR, B=2, H=16, dqk=576, pages=9, max_pages=4, mass_len=256, q_sb=16 * 576,
             q_sh=576, kv_sp=64 * 1152, kv_ss=1152, bt_sb=4, m_sb=256, q4=0, scale=0.07)
    a.update(kw)
    return _lib.lib().dmla_attn_mass(P(a["q"]), P(a["kv"]), P(a["bt"]), P(a["sl"]), P(a["lse"]), P(a["mass"]), a["B"], a["H"],
                                     a["dqk"], a["pages"], a["max_pages"], a["mass_len"], a["q_sb"], a["q_sh"], a["kv_sp"],
                                     a["kv_ss"], a["bt_sb"], a["m_sb"], a["q4"], a["scale"], None)


def test_attn_mass_refuses():
    for name in ("q", "kv", "bt", "sl", "lse", "mass"):
        assert _mass(**{name: None}) == INVALID
    for bad in (dict(B=-1), dict(pages=0), dict(max_pages=0, bt_sb=0), dict(scale=-1.0), dict(q=PTR + 2), dict(kv=PTR + 8),
                dict(q_sh=577), dict(kv_ss=1136), dict(kv_ss=1160, kv_sp=64 * 1160), dict(kv_sp=64 * 1152 - 16), dict(bt_sb=3), dict(mass_len=255),
                dict(m_sb=255), dict(q4=1, kv_ss=384)):
        assert _mass(**bad) == INVALID, bad
    for bad in (dict(dqk=512), dict(q4=1, kv_ss=416), dict(H=1 << 17)):
        assert _mass(**bad) == UNSUPPORTED, bad
    assert _mass(B=0) == OK and _mass(H=0) == OK


def _evict(**kw):
    a = dict(pool=PTR, bt=PTR, sl=PTR, mass=PTR, nl=PTR, src=PTR, mo=PTR + 4096, B=2, row=1152, pages=9, max_pages=4, mass_len=256,
             kv_sp=64 * 1152, kv_ss=1152, bt_sb=4, m_sb=256, mo_sb=256, src_sb=100, budget=100, recent=20, sink=4, ws=None,
             ws_bytes=0)
    a.update(kw)
    return _lib.lib().dmla_kv_evict(P(a["pool"]), P(a["bt"]), P(a["sl"]), P(a["mass"]), P(a["nl"]), P(a["src"]), P(a["mo"]), None,
                                    a["B"], a["row"], a["pages"], a["max_pages"], a["mass_len"], a["kv_sp"], a["kv_ss"],
                                    a["bt_sb"], a["m_sb"], a["mo_sb"], a["src_sb"], a["budget"], a["recent"], a["sink"],
                                    P(a["ws"]), a["ws_bytes"], None)


def test_evict_refuses():
    for name in ("pool", "bt", "sl", "mass", "nl", "src", "mo"):
        assert _evict(**{name: None}) == INVALID
    for bad in (dict(B=-1), dict(pages=0), dict(max_pages=0, bt_sb=0), dict(budget=0), dict(recent=-1), dict(sink=-1),
                dict(recent=97), dict(recent=101, sink=0), dict(row=0), dict(row=1160), dict(pool=PTR + 8), dict(kv_ss=1136),
                dict(kv_sp=64 * 1152 - 16), dict(bt_sb=3), dict(mass_len=255), dict(m_sb=255), dict(mo_sb=200),
                dict(src_sb=99), dict(mo=PTR)):
        assert _evict(**bad) == INVALID, bad
    assert _evict(max_pages=1 << 21, bt_sb=1 << 21) == UNSUPPORTED
    assert _evict() == WORKSPACE
    need = _lib.lib().dmla_kv_evict_workspace_bytes(2, 1152, 4, 100, 20, 4)
    assert need >= 2 * 20 * 1152 and _evict(ws=PTR, ws_bytes=need - 1) == WORKSPACE
    assert _evict(ws=PTR + 8, ws_bytes=need) == INVALID
    assert _evict(B=0) == OK
    # a budget that no sequence of the table can pass needs room for no list and no row
    assert _lib.lib().dmla_kv_evict_workspace_bytes(2, 1152, 4, 256, 200, 4) <= 64


def test_wrappers_refuse_cpu_tensors_types_and_shapes():
    bf, i32 = torch.bfloat16, torch.int32
    q, pool4, pool = torch.zeros(2, 16, 576, dtype=bf), torch.zeros(4, 64, 400, dtype=torch.uint8), torch.zeros(4, 64, 576, dtype=bf)
    bt, sl, mass = torch.zeros(2, 3, dtype=i32), torch.ones(2, dtype=i32), torch.zeros(2, 192)
    new = torch.zeros(2, 1, 576, dtype=bf)
    with pytest.raises(ValueError, match="GPU"):
        ops.flash_dmla_kv_append_q4(pool4, bt, sl, new)
    with pytest.raises(ValueError, match="GPU"):
        ops.flash_dmla_kv_gather_q4(pool4, bt, sl, 5)
    with pytest.raises(ValueError, match="GPU"):
        ops.flash_dmla_decode_paged_q4(q, pool4, bt, sl)
    with pytest.raises(ValueError, match="GPU"):
        ops.flash_dmla_attn_mass(q, pool, bt, sl, torch.zeros(2, 16), mass)
    for p in (pool, pool4):
        with pytest.raises(ValueError, match="GPU"):
            ops.flash_dmla_kv_evict(p, bt, sl, mass, 10)


# ---- dispatcher ops ----------------------------------------------------------------------------
def test_fake_shapes_and_schemas():
    t = lambda shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    q, pool, bt, sl = t((3, 16, 576)), t((9, 64, 400), torch.uint8), t((3, 4), torch.int32), t((3,), torch.int32)
    mass = t((3, 300), torch.float32)
    f = torch.ops.flashdmla
    assert f.kv_append_q4(pool, bt, sl, t((3, 2, 576)), None) is None
    rows = f.kv_gather_q4(pool, bt, sl, 77, None)
    assert (rows.shape, rows.dtype) == ((3, 77, 576), torch.bfloat16)
    o, lse = f.decode_paged_q4(q, pool, bt, sl, 512, None)
    assert (o.shape, o.dtype, lse.shape, lse.dtype) == ((3, 16, 512), torch.bfloat16, (3, 16), torch.float32)
    assert f.attn_mass(q, pool, bt, sl, lse, mass, None) is None
    new_lens, src, new_mass = f.kv_evict(pool, bt, sl, mass, 100, 10, 4)
    assert (new_lens.shape, src.shape, src.dtype, new_mass.shape) == ((3,), (3, 100), torch.int32, (3, 300))
    assert f.kv_evict(pool, bt, sl, mass, 1000, 10, 4)[1].shape == (3, 256)
    assert "Tensor(a0!) kv_pool" in str(f.kv_append_q4.default._schema)
    assert "!) mass" in str(f.attn_mass.default._schema)
    assert "Tensor(a0!) kv_pool" in str(f.kv_evict.default._schema)
