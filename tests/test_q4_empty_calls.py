"""Calls without a sequence, a row or a head: they do nothing and return empty results, though empty tensors have no
address."""
import pytest
import torch

from python import ops
from test_q4_cache import INVALID, OK, _append, _decode, _evict, _gather, _mass

NULL = {"append": dict(pool=None, bt=None, sl=None, new=None), "gather": dict(pool=None, bt=None, sl=None, out=None),
        "decode": dict(q=None, kv=None, bt=None, sl=None, o=None),
        "mass": dict(q=None, kv=None, bt=None, sl=None, lse=None, mass=None),
        "evict": dict(pool=None, bt=None, sl=None, mass=None, nl=None, src=None, mo=None)}
CALL = dict(append=_append, gather=_gather, decode=_decode, mass=_mass, evict=_evict)


@pytest.mark.parametrize("name,zero", [("append", dict(B=0)), ("append", dict(n=0)), ("gather", dict(B=0)),
                                       ("gather", dict(n=0)), ("decode", dict(B=0)), ("decode", dict(H=0)),
                                       ("mass", dict(B=0)), ("mass", dict(H=0)), ("evict", dict(B=0))])
def test_entry_points_take_empty_calls_without_addresses(name, zero):
    assert CALL[name](**NULL[name], **zero) == OK
    assert CALL[name](**NULL[name]) == INVALID
    assert CALL[name](**{**NULL[name], **zero, "B": -1}) == INVALID
    assert CALL[name](**{**NULL[name], **zero, "bt_sb": 3}) == INVALID   # what else is wrong is refused as ever


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,n_new", [(0, 16, 3), (2, 0, 3), (2, 16, 0), (0, 0, 0)])
def test_wrappers_take_empty_tensors(gpu, B, H, n_new):
    bf, i32 = torch.bfloat16, torch.int32
    pool = torch.randint(0, 256, (4, 64, 400), dtype=torch.uint8, device=gpu)
    wide = torch.zeros(4, 64, 576, dtype=bf, device=gpu)
    before = pool.clone()
    table, lens = torch.arange(2 * B, dtype=i32, device=gpu).reshape(B, 2), torch.full((B,), 5, dtype=i32, device=gpu)
    q, lse = torch.zeros(B, H, 576, dtype=bf, device=gpu), torch.zeros(B, H, device=gpu)
    mass = torch.ones(B, 128, device=gpu)
    for f in (ops, None):
        d = torch.ops.flashdmla
        if B == 0 or n_new == 0:
            new = torch.zeros(B, n_new, 576, dtype=bf, device=gpu)
            if f:
                ops.flash_dmla_kv_append_q4(pool, table, lens, new, check_indices=True)
                ops.flash_dmla_kv_append_q4(pool, table, lens, new, torch.zeros_like(lens))
            else:
                d.kv_append_q4(pool, table, lens, new, None)
            rows = ops.flash_dmla_kv_gather_q4(pool, table, lens, n_new) if f else d.kv_gather_q4(pool, table, lens, n_new, None)
            assert rows.shape == (B, n_new, 576)
        if B == 0 or H == 0:
            o, got = (ops.flash_dmla_decode_paged_q4(q, pool, table, lens, return_lse=True, check_indices=True) if f
                      else d.decode_paged_q4(q, pool, table, lens, 512, None))
            assert o.shape == (B, H, 512) and got.shape == (B, H)
            for p in (pool, wide):
                ops.flash_dmla_attn_mass(q, p, table, lens, lse, mass) if f else d.attn_mass(q, p, table, lens, lse, mass, None)
            assert (mass == 1).all()
        if B == 0:
            for p in (pool, wide):
                new_lens, src, new_mass = (ops.flash_dmla_kv_evict(p, table, lens, mass, 4, 1, 1, check_indices=True) if f
                                           else d.kv_evict(p, table, lens, mass, 4, 1, 1))
                assert new_lens.shape == (0,) and src.shape == (0, 4) and new_mass.shape == (0, 128)
    assert torch.equal(pool, before) and (wide == 0).all()
