"""Prompt attention over gathered 4-bit rows: flash_dmla_fwd knows no lengths, so sequences of different lengths go in
one call each, with the rows that each has.  The zero rows behind a shorter sequence's end are keys like others."""
import pytest
import torch

from conftest import assert_out_close, seeded
from oracle import dmla_ref as R

LENS = [300, 64, 1, 205, 130]
CHUNK = [40, 64, 1, 33, 7]    # new tokens of each prompt, cached already: the last rows
H = 16


def _batch():
    rows = [R.q4_unpack(R.q4_pack(seeded((n, 576), 10 + b, 0.5, torch.bfloat16))) for b, n in enumerate(LENS)]
    q = seeded((len(LENS), H, max(CHUNK), 576), 20, 0.5, torch.bfloat16)
    return rows, q


def _reference(rows, q, b):
    """o [1, H, chunk, 512] of sequence b over exactly its rows, in float64."""
    k = rows[b][None]
    return R.dmla_fwd_cache_latent(q[b:b + 1, :, :CHUNK[b]].double(), k, 512)[0]


def test_zero_rows_behind_a_shorter_sequence_take_weight():
    """Over padded rows the oracle itself ends far outside the bar of the outputs, in every shorter sequence."""
    rows, q = _batch()
    for b, n in enumerate(LENS):
        padded = torch.zeros(max(LENS), 576, dtype=torch.float64)
        padded[:n] = rows[b]
        wrong = R.dmla_fwd_cache_latent(q[b:b + 1, :, :CHUNK[b]].double(), padded[None], 512)[0]
        ref = _reference(rows, q, b)
        if n == max(LENS):
            assert torch.equal(wrong, ref)
            continue
        with pytest.raises(AssertionError, match="mean-rel|max-abs"):
            assert_out_close(wrong, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [False, True])
def test_prompts_of_different_lengths_over_gathered_rows(gpu, window):
    from python import ops
    from test_q4_cache_gpu import _table

    rows, q = _batch()
    table, pages = _table(LENS, 5)
    pool = torch.full((pages, 64, 400), 255, dtype=torch.uint8)
    for b, n in enumerate(LENS):
        packed = R.q4_pack(rows[b].to(torch.bfloat16))
        for j in range(0, n, 64):
            pool[int(table[b, j // 64]), :min(64, n - j)] = packed[j:j + 64]
    lens = torch.tensor(LENS, dtype=torch.int32, device=gpu)
    k_lat = ops.flash_dmla_kv_gather_q4(pool.to(gpu), table.to(gpu), lens, max(LENS))
    for b, n in enumerate(LENS):
        if window:   # one sequence's rows read back by themselves
            k_b = ops.flash_dmla_kv_gather_q4(pool.to(gpu), table[b:b + 1].to(gpu), lens[b:b + 1], n)
        else:
            k_b = k_lat[b:b + 1, :n]
        o, _, _ = ops.flash_dmla_fwd(q[b:b + 1, :, :CHUNK[b]].to(gpu), k_b)
        assert_out_close(o.cpu(), _reference(rows, q, b), f"sequence {b}")
