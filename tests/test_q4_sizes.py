"""Sizes at which the cut of a 4-bit decode batch over workgroups would leave 32-bit integers (CPU).

Every workgroup adds up the weights of all sequences: two tiles a page, and for each sequence what a
segment's start and end cost, 24 tiles in the kernel of 32 heads a workgroup and 8 in that of 128.  A sum
that wraps leaves sequences without an owner, and the combine reads a plan that nobody wrote."""
import pytest

from test_q4_cache import PTR, UNSUPPORTED, WORKSPACE, _decode

LIMIT = 1 << 31


def _cut(heads, cost, batch, pages):
    """(what the entry point says of these sizes, the largest sum of weights)."""
    rc = _decode(B=batch, H=heads, max_pages=pages, bt_sb=pages, q_sb=heads * 576, o_sb=heads * 512, ws=PTR, ws_bytes=0)
    return rc, batch * (2 * pages + cost)


@pytest.mark.parametrize("heads,cost", [(1, 24), (16, 24), (64, 24), (65, 8), (128, 8), (300, 8)])
@pytest.mark.parametrize("batch", [128, 1024, 4099, 600000, 1 << 20])
def test_batches_whose_weights_pass_32_bits_are_refused(heads, cost, batch):
    most = (LIMIT - 1) // batch   # weight of a sequence at which the sum still fits
    first = (most - cost) // 2 + 1
    for pages in range(first, first + 12):
        rc, weight = _cut(heads, cost, batch, pages)
        assert weight >= LIMIT and rc == UNSUPPORTED, (batch, pages)
    # a little below the limit (up to 4096 workgroups round the ranges up) the sizes are taken
    last = (((LIMIT - 1 - 4096) // batch) - cost) // 2
    rc, weight = _cut(heads, cost, batch, last)
    assert weight < LIMIT and rc == WORKSPACE


def test_sums_of_exactly_2_to_the_31_and_a_little_more_are_refused():
    """A bound of 16 tiles a sequence would let these pass; of the first, 24 tiles make 2^31."""
    assert _decode(B=1024, max_pages=1048564, bt_sb=1048564) == UNSUPPORTED
    assert _decode(B=1 << 20, max_pages=1015, bt_sb=1015) == UNSUPPORTED
    assert _decode(B=600000, max_pages=1781, bt_sb=1781) == UNSUPPORTED
