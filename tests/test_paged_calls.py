"""Refusals and workspace sizes of the calls that plan, fill and attend pages: the C ABI and the Python layer, without a
GPU (every call below returns before a launch, so the addresses are never used)."""
import ctypes

import pytest
import torch

from python import _lib, ops

P = ctypes.c_void_p
A = 1 << 20   # some aligned address
OK, INVALID, UNSUPPORTED, WORKSPACE = _lib.DMLA_OK, _lib.DMLA_ERR_INVALID_ARG, _lib.DMLA_ERR_UNSUPPORTED, _lib.DMLA_ERR_WORKSPACE


def call(name, defaults, **kw):
    a = dict(defaults)
    assert set(kw) <= set(a)
    a.update(kw)
    types = _lib.SIGNATURES[name][1]
    assert len(types) == len(a)
    return getattr(_lib.lib(), name)(*[P(v) if t is P else v for t, v in zip(types, a.values())])


RELEASE = dict(bt=A, old=A, new=A, free=A, count=A, out=A, flag=None, B=2, pages=10, width=4, capacity=10, bt_sb=4, stream=None)
RESERVE = dict(bt=A, lens=A, new=A, free=A, count=A, total=A, cu=A, slots=A, out=A, flag=None, B=2, rows=5, pages=10, width=4,
               capacity=10, bt_sb=4, stream=None)
APPEND = dict(pool=A, slots=A, rows=A, flag=None, T=3, d=576, pages=10, kv_sp=64 * 576, kv_ss=576, r_ss=576, stream=None)
APPEND_Q4 = dict(pool=A, slots=A, rows=A, flag=None, T=3, pages=10, kv_sp=64 * 400, r_ss=576, stream=None)
CHUNK = dict(q=A, kv=A, bt=A, lens=A, cu=A, o=A, lse=None, T=8, B=2, H=16, dqk=576, dv=512, pages=10, width=4, q_st=16 * 576, q_sh=576,
             kv_sp=64 * 576, kv_ss=576, bt_sb=4, o_st=16 * 512, o_sh=512, scale=0.07, causal=1, ws=None, ws_bytes=0, stream=None)
MEANS = dict(kv=A, bt=A, lens=A, starts=None, means=A, B=2, pages=10, width=4, kv_sp=64 * 1152, kv_ss=1152, bt_sb=4, m_sp=576, q4=0,
             stream=None)
SCORES = dict(q=A, means=A, bt=A, lens=A, cu=A, scores=A, T=8, B=2, H=16, dqk=576, pages=10, width=4, q_st=16 * 576, q_sh=576, m_sp=576,
              bt_sb=4, s_st=4, scale=0.07, ws=None, ws_bytes=0, stream=None)
SELECT = dict(scores=A, bt=A, lens=A, cu=A, table=A, sel_lens=A, index=A, T=8, B=2, width=4, s_st=4, bt_sb=4, st=3, si=3, k=3, recent=1,
              sink=1, stream=None)

REFUSED = [
    ("dmla_kv_release", RELEASE, INVALID, [dict(bt=None), dict(old=None), dict(new=None), dict(free=None), dict(count=None), dict(out=None),
                                           dict(B=-1), dict(pages=-1), dict(capacity=-1), dict(bt_sb=3)]),
    ("dmla_kv_release", RELEASE, UNSUPPORTED, [dict(B=1 << 25), dict(pages=(1 << 25) + 1), dict(capacity=1 << 30),
                                               dict(width=1 << 23, bt_sb=1 << 23, B=1000)]),
    ("dmla_kv_reserve", RESERVE, INVALID, [dict(bt=None), dict(lens=None), dict(new=None), dict(free=None), dict(count=None), dict(total=None),
                                           dict(cu=None), dict(slots=None), dict(out=None), dict(B=-1), dict(rows=-1), dict(bt_sb=3)]),
    ("dmla_kv_reserve", RESERVE, UNSUPPORTED, [dict(rows=1 << 30), dict(pages=(1 << 25) + 1), dict(capacity=1 << 30), dict(width=(1 << 24) + 1, bt_sb=1 << 25)]),
    ("dmla_kv_append_rows", APPEND, INVALID, [dict(pool=None), dict(slots=None), dict(rows=None), dict(T=-1), dict(d=0), dict(kv_ss=568),
                                              dict(kv_sp=64 * 576 - 8), dict(r_ss=568), dict(r_ss=580), dict(pool=A + 8), dict(rows=A + 4)]),
    ("dmla_kv_append_rows", APPEND, UNSUPPORTED, [dict(d=12), dict(T=1 << 28), dict(pages=(1 << 25) + 1)]),
    ("dmla_kv_append_rows_q4", APPEND_Q4, INVALID, [dict(pool=None), dict(slots=None), dict(rows=None), dict(T=-1), dict(kv_sp=64 * 400 - 16),
                                                    dict(kv_sp=64 * 400 + 8), dict(r_ss=568), dict(rows=A + 4)]),
    ("dmla_kv_append_rows_q4", APPEND_Q4, UNSUPPORTED, [dict(T=1 << 31), dict(pages=(1 << 25) + 1)]),
    ("dmla_chunk_paged", CHUNK, INVALID, [dict(q=None), dict(kv=None), dict(bt=None), dict(lens=None), dict(o=None), dict(T=-1), dict(B=-1),
                                          dict(cu=None), dict(q=A + 2), dict(o=A + 2), dict(kv=A + 2), dict(q_st=12), dict(o_sh=4),
                                          dict(kv_ss=568), dict(kv_sp=64 * 576 - 8), dict(kv_ss=1 << 25, kv_sp=1 << 31), dict(bt_sb=3),
                                          dict(pages=0), dict(width=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                          dict(scale=float("inf"))]),
    ("dmla_chunk_paged", CHUNK, UNSUPPORTED, [dict(dqk=64), dict(dv=64), dict(H=1 << 17), dict(B=(1 << 20) + 1), dict(T=1 << 27, B=2),
                                              dict(width=(1 << 20) + 1, bt_sb=1 << 21)]),
    ("dmla_chunk_paged", CHUNK, WORKSPACE, [dict(), dict(ws=A, ws_bytes=1000)]),
    ("dmla_page_means", MEANS, INVALID, [dict(kv=None), dict(bt=None), dict(lens=None), dict(means=None), dict(B=-1), dict(kv=A + 8),
                                         dict(means=A + 8), dict(kv_ss=1144), dict(kv_ss=1160), dict(kv_sp=64 * 1152 - 16), dict(m_sp=568), dict(m_sp=580),
                                         dict(bt_sb=3), dict(q4=1), dict(q4=1, kv_ss=416, kv_sp=64 * 416)]),
    ("dmla_page_means", MEANS, UNSUPPORTED, [dict(B=1 << 25), dict(width=(1 << 24) + 1, bt_sb=1 << 25)]),
    ("dmla_page_scores", SCORES, INVALID, [dict(q=None), dict(means=None), dict(bt=None), dict(lens=None), dict(scores=None), dict(cu=None),
                                           dict(T=-1), dict(H=-1), dict(H=0), dict(pages=0), dict(q=A + 2), dict(means=A + 2), dict(q_st=12), dict(m_sp=568),
                                           dict(s_st=3), dict(bt_sb=3), dict(scale=0.0), dict(scale=float("nan"))]),
    ("dmla_page_scores", SCORES, UNSUPPORTED, [dict(dqk=64), dict(H=1 << 17), dict(T=(1 << 30) + 1)]),
    ("dmla_page_scores", dict(SCORES, width=400, bt_sb=400, s_st=400), WORKSPACE, [dict(), dict(ws=A, ws_bytes=64)]),
    ("dmla_page_select", SELECT, INVALID, [dict(scores=None), dict(bt=None), dict(lens=None), dict(table=None), dict(sel_lens=None),
                                           dict(index=None), dict(cu=None), dict(T=-1), dict(recent=0), dict(sink=-1), dict(k=1), dict(st=2),
                                           dict(si=2), dict(s_st=3), dict(bt_sb=3)]),
    ("dmla_page_select", SELECT, UNSUPPORTED, [dict(k=(1 << 24) + 1, st=1 << 25, si=1 << 25), dict(T=(1 << 30) + 1)]),
]


@pytest.mark.parametrize("name,defaults,code,wrong", REFUSED, ids=[f"{r[0]}{r[2]}" for r in REFUSED])
def test_the_c_calls_refuse(name, defaults, code, wrong):
    for kw in wrong:
        assert call(name, defaults, **kw) == code, (name, kw, _lib.lib().dmla_last_error())
        assert name.encode() in _lib.lib().dmla_last_error()


def test_empty_calls_launch_nothing():
    assert call("dmla_kv_append_rows", APPEND, T=0, pool=None, slots=None, rows=None) == OK
    assert call("dmla_kv_append_rows_q4", APPEND_Q4, T=0, pool=None, slots=None, rows=None) == OK
    assert call("dmla_chunk_paged", CHUNK, T=0, q=None, o=None) == OK
    assert call("dmla_chunk_paged", CHUNK, H=0) == OK
    for kw in (dict(B=0), dict(width=0), dict(pages=0)):
        assert call("dmla_page_means", MEANS, **kw) == OK
    assert call("dmla_page_scores", SCORES, T=0, q=None, scores=None) == OK
    assert call("dmla_page_scores", SCORES, width=0, scores=None, bt=None) == OK
    assert call("dmla_page_select", SELECT, T=0, scores=None) == OK
    assert _lib.lib().dmla_last_error() == b""


def test_workspace_sizes():
    lib = _lib.lib()
    one = 2 * 128 * (512 + 1) * 4 + 16   # two parts of 128 rows and a link, of a range
    for T, B, H, width in ((1, 1, 16, 1), (1, 1, 128, 79), (1024, 1, 128, 128), (64, 64, 128, 128), (1 << 20, 64, 128, 4096)):
        n = lib.dmla_chunk_paged_workspace_bytes(T, B, H, width)
        assert n % one == 0 and 1 <= n // one <= 256, "a range per CU at most (256 where there is no GPU)"
    assert lib.dmla_chunk_paged_workspace_bytes(1, 1, 16, 1) < lib.dmla_chunk_paged_workspace_bytes(1, 1, 16, 128)
    for bad in ((0, 1, 16, 1), (1, 0, 16, 1), (1, 1, 0, 1), (1, 1, 16, 0), (1, 1, 1 << 17, 1), (1 << 25, 1, 128, 1)):
        assert lib.dmla_chunk_paged_workspace_bytes(*bad) == 0
    # Page scores: a maximum and a sum per query, head and chunk of pages, and the products up to 512 MB; none where one
    # workgroup has all pages.
    assert lib.dmla_page_scores_workspace_bytes(1, 128, 32, 1) == 0
    assert lib.dmla_page_scores_workspace_bytes(4096, 128, 512, 1) == 0
    for pages, kept in ((512, 512), (16384, 16384), (16385, 0)):
        n = lib.dmla_page_scores_workspace_bytes(64, 128, pages, 0) - 64 * 128 * kept * 4
        assert n > 0 and n % (64 * 128 * 8) == 0 and n // (64 * 128 * 8) <= 16
    assert lib.dmla_page_scores_workspace_bytes(0, 128, 32, 1) == 0


def _cpu():
    i = torch.zeros(1, dtype=torch.int32)
    return dict(q=torch.zeros(1, 16, 576, dtype=torch.bfloat16), pool=torch.zeros(2, 64, 576, dtype=torch.bfloat16),
                table=torch.zeros(1, 2, dtype=torch.int32), i=i, means=torch.zeros(2, 576, dtype=torch.bfloat16), scores=torch.zeros(1, 2))


def test_the_python_calls_refuse_cpu_tensors():
    c = _cpu()
    t, i = c["table"], c["i"]
    for f in (lambda: ops.flash_dmla_kv_release(t, i, i, i, i, 2), lambda: ops.flash_dmla_kv_reserve(t, i, i, i, i, 1, 2),
              lambda: ops.flash_dmla_kv_append_rows(c["pool"], i, c["q"][0, :1]), lambda: ops.flash_dmla_chunk_paged(c["q"], c["pool"], t, i),
              lambda: ops.flash_dmla_page_means(c["pool"], t, i, c["means"]), lambda: ops.flash_dmla_page_scores(c["q"], c["means"], t, i),
              lambda: ops.flash_dmla_page_select(c["scores"], t, i, None, 1),
              lambda: ops.flash_dmla_sparse_paged(c["q"], c["pool"], c["means"], t, i, None, 1)):
        with pytest.raises(ValueError, match="GPU tensor"):
            f()


def test_the_dispatcher_knows_the_calls_on_meta_tensors():
    import python  # noqa: F401  (registers torch.ops.flashdmla.*)
    F = torch.ops.flashdmla
    m = dict(device="meta")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, **m)
    q, pool = torch.zeros(7, 16, 576, dtype=torch.bfloat16, **m), torch.zeros(9, 64, 576, dtype=torch.bfloat16, **m)
    means = torch.zeros(9, 576, dtype=torch.bfloat16, **m)
    assert F.kv_release(i(3, 4), i(3), i(3), i(9), i(1), 9).shape == (1,)
    assert [tuple(x.shape) for x in F.kv_reserve(i(3, 4), i(3), i(3), i(9), i(1), 7, 9)] == [(3,), (4,), (7,), (1,)]
    F.kv_append_rows(pool, i(7), q[:, 0])
    o, lse = F.chunk_paged(q, pool, i(3, 4), i(3), i(4), 512, None, True)
    assert (tuple(o.shape), o.dtype, tuple(lse.shape), lse.dtype) == ((7, 16, 512), torch.bfloat16, (7, 16), torch.float32)
    F.page_means(pool, i(3, 4), i(3), means, None)
    assert F.page_scores(q, means, i(3, 4), i(3), i(4), None).shape == (7, 4)
    assert [tuple(x.shape) for x in F.page_select(torch.zeros(7, 4, **m), i(3, 4), i(3), i(4), 2, 1, 0)] == [(7, 2), (7,), (7, 2)]
