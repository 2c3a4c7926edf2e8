"""How chunk attention's work is cut over its workgroups (csrc/dmla_chunk_cut.h), on the CPU: tests/chunk_cut_driver.cpp
runs the kernel's own code, a thread for each lane."""
import os
import random
import shutil
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "ds-flashdmla-moe_amd", "csrc")
CXX = shutil.which("g++")
pytestmark = pytest.mark.skipif(CXX is None, reason="g++ is needed")
TILE, ROWS, FEW_ROWS = 32, 128, 32


def build(directory, *flags):
    exe = str(directory / "driver")
    run = subprocess.run([CXX, "-std=c++17", "-O1", "-g", "-Wno-unknown-pragmas", *flags, "-I" + CSRC,
                          os.path.join(ROOT, "tests", "chunk_cut_driver.cpp"), "-o", exe, "-lpthread"],
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-3000:]
    return exe


@pytest.fixture(scope="module")
def checked(tmp_path_factory):
    """The code with checks of its integer arithmetic: a sum past 32 bits ends the program."""
    return build(tmp_path_factory.mktemp("cut"), "-fsanitize=undefined,float-cast-overflow", "-fno-sanitize-recover=all")


def ask(exe, *lines):
    env = dict(os.environ, TSAN_OPTIONS="halt_on_error=1")
    run = subprocess.run([exe], env=env, input="\n".join(" ".join(str(x) for x in line) for line in lines) + "\n", capture_output=True,
                         text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-3000:]
    return [[int(x) for x in line.split()] for line in run.stdout.splitlines()]


def starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def cut_of(exe, H, lens, counts, causal=True, n_ranges=8, max_pages=None, T=None, ranges=None):
    """The pieces of the ranges: (range, sequence, first row, rows, tokens, first key tile, end, slot)."""
    max_pages = max_pages or max(1, -(-max(lens) // 64))
    ranges = list(range(n_ranges)) if ranges is None else ranges
    out, = ask(exe, ["cut", T or sum(counts), len(lens), H, max_pages, int(causal), n_ranges, 1, len(ranges), *ranges, *lens,
                     *starts(counts)])
    return [tuple(out[i:i + 8]) for i in range(0, len(out), 8)]


def assert_all_done_once(pieces, H, lens, counts, causal=True):
    """Every row of every sequence is in one row tile, and the key tiles of a row tile in one piece or in parts that
    follow each other from range to range."""
    tiles = {}
    for r, b, row0, rows, length, t0, t1, slot in pieces:
        assert length == lens[b] and rows > 0
        tiles.setdefault((b, row0), []).append((r, rows, t0, t1, slot))
    at = {}
    for (b, row0), parts in sorted(tiles.items()):
        assert row0 == at.get(b, 0), "rows left out or done twice"
        rows = parts[0][1]
        assert rows <= ROWS and (rows in (FEW_ROWS, ROWS) or row0 + rows == counts[b] * H)
        at[b] = row0 + rows
        end = lens[b] - counts[b] + (row0 + rows - 1) // H + 1 if causal else lens[b]
        end = -(-max(end, 0) // TILE)
        reached = 0
        for i, (r, n, t0, t1, slot) in enumerate(parts):
            assert n == rows and t0 == reached and (t1 > t0 or end == 0)
            assert r == parts[0][0] + i, "parts in ranges that follow each other"
            last = i == len(parts) - 1
            assert slot == (-1 if len(parts) == 1 else 2 * r + 1 if i == 0 else 2 * r)
            reached = t1
            assert last == (t1 == end)
    assert at == {b: n * H for b, n in enumerate(counts) if n}


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,lens,counts", [
    (128, [1], [1]), (16, [5000], [1]), (128, [20000], [1]), (16, [33, 200, 7], [33, 9, 2]), (1, [300, 64], [290, 64]),
    (5, [97, 31, 1000], [50, 31, 3]), (128, [8192], [64]), (128, [200, 0, 40, 30], [100, 0, 17, 30]), (20, [9000] * 5, [1, 2, 3, 9, 17]),
    (300, [66], [2]), (16, [0, 0], [1, 1]), (16, [3, 0, 40, 0], [6, 2, 45, 0])])
def test_all_work_is_done_once(checked, H, lens, counts, causal):
    for n_ranges in (1, 5):
        assert_all_done_once(cut_of(checked, H, lens, counts, causal, n_ranges), H, lens, counts, causal)


@pytest.mark.parametrize("B,H", [(255, 1), (257, 16), (520, 128)])
def test_hundreds_of_sequences(checked, B, H):
    r = random.Random(B)
    lens = [r.choice([0, 1, 64, r.randint(1, 3000)]) for _ in range(B)]
    counts = [r.choice([0, 0, 0, 0, 0, 0, 0, 1, 2, min(n, 5)]) for n in lens]
    assert_all_done_once(cut_of(checked, H, lens, counts, n_ranges=3), H, lens, counts)


@pytest.mark.parametrize("H,n,N", [(1, 1 << 22, 64), (16, 1 << 21, 1), (128, 1 << 18, 0), (1, 1 << 20, 1 << 19)])
def test_many_more_queries_than_tokens(checked, H, n, N):
    """The weights' sum stays within 32 bits, and ranges follow each other up to the last row."""
    some = [0, 1, 254, 255]
    pieces = cut_of(checked, H, [N], [n], n_ranges=256, ranges=some)
    by_range = {r: [x for x in pieces if x[0] == r] for r in some}
    for r in some:
        assert by_range[r], "a range without work"
        for x, y in zip(by_range[r], by_range[r][1:]):
            assert y[2] == x[2] + x[3] and y[5] == 0
    last = by_range[255][-1]
    assert by_range[0][0][2] == 0 and last[2] + last[3] == n * H
    for r in (0, 254):
        x, y = by_range[r][-1], by_range[r + 1][0]
        assert (y[2], y[5]) in ((x[2] + x[3], 0), (x[2], x[6]))


def test_the_hosts_bound_of_the_weight(checked):
    """In units of 2^shift the sum stays within 32 bits whatever the lengths; ascending with the row tiles."""
    r = random.Random(5)
    lines, bounds = [], []
    for _ in range(400):
        H, B = r.choice([1, 2, 5, 16, 128, 300, 1 << 16]), r.choice([1, 2, 7])
        pages = int(2 ** r.uniform(0, 20))
        T = int(2 ** r.uniform(0, 30 - (H - 1).bit_length()))
        at = sorted(r.randint(0, T) for _ in range(B - 1))
        cu = [0, *at, T]
        lens = [r.choice([0, 1, 64 * pages, r.randint(0, 64 * pages), min(64 * pages, cu[i + 1] - cu[i])]) for i in range(B)]
        lines.append(["weight", T, B, H, pages, r.choice([0, 1]), *lens, *cu])
        bounds.append((T * H // ROWS + min(B, T)) * (10 + 2 * pages))
    for line, bound, (total, shift, ascending) in zip(lines, bounds, ask(checked, *lines)):
        assert ascending, line
        row_tiles = line[1] * line[3] // ROWS + line[2]
        assert total <= min((bound >> shift) + 2 * row_tiles + 1, 2 ** 31 - 1), line


# ---- what waves read and write between barriers --------------------------------------------------------

@pytest.fixture(scope="module")
def watched(tmp_path_factory):
    """The code under a detector of data races: of two accesses to one word by different threads, one of them a write,
    with no barrier between, it ends the program."""
    d = tmp_path_factory.mktemp("races")
    probe = d / "probe.cpp"
    probe.write_text("#include <thread>\nint main() { std::thread([] {}).join(); }\n")
    run = subprocess.run([CXX, "-fsanitize=thread", str(probe), "-o", str(d / "probe"), "-lpthread"], capture_output=True, timeout=120)
    if run.returncode != 0 or subprocess.run([str(d / "probe")], capture_output=True, timeout=60).returncode != 0:
        pytest.skip("the thread sanitizer does not run here")
    return build(d, "-fsanitize=thread")


@pytest.mark.parametrize("H,lens,counts", [
    (128, [20000], [1]), (16, [33, 200, 7], [33, 9, 2]), (128, [8192], [300]), (16, [0, 40], [2, 1]),
    (16, [300] * 257, [1] * 257), (16, [0] * 300 + [900, 0, 70], [0] * 300 + [9, 0, 1])])
def test_the_cut_has_no_races(watched, H, lens, counts):
    """Little work (cut twice), much, several rounds of 256 sequences, a range that begins behind the first of them."""
    assert_all_done_once(cut_of(watched, H, lens, counts, n_ranges=3), H, lens, counts)


# ---- the rows of a careful pass ------------------------------------------------------------------------

END = 0x7fffffff   # no row is left out


def careful(exe, begin, last, odd=(), table=(3, 1, 2, 0), pages=4, end=8):
    """The pass of the rows whose last tokens are from `begin` on up to `last`, of a piece that ends at key tile `end`;
    odd: tokens that hold an infinity."""
    at = [table[j // 64] * 64 + j % 64 for j in odd]
    out, = ask(exe, ["careful", pages, begin, last, end, len(at), len(table), *at, *table])
    assert out[:2] == [1, begin]
    return out[2]


@pytest.mark.parametrize("begin,last,odd,to", [
    (10, 90, [], END), (10, 90, [10], END), (10, 90, [11], 11), (10, 90, [91], END), (10, 90, [90, 33, 64], 33), (-1, 20, [0], 0),
    (-5, 20, [0, 3], 0), (-1, 20, [], END), (200, 200, [100], END)])
def test_where_rows_are_cut(checked, begin, last, odd, to):
    assert careful(checked, begin, last, odd) == to


def test_a_careful_pass_has_no_races(watched):
    """Its waves post where they would cut in the words in which they have just read that a pass has to follow."""
    assert careful(watched, -1, 20, [0]) == 0
    assert careful(watched, 10, 90, []) == END


@pytest.mark.parametrize("bad", [-1, 4, 2 ** 31 - 1])
@pytest.mark.parametrize("begin,last,odd,page,to", [
    (10, 90, [], 1, 64), (63, 90, [], 1, 64), (64, 90, [], 1, END), (70, 90, [], 1, END), (10, 90, [33], 1, 33), (33, 90, [33], 1, 64),
    (64, 140, [], 1, END), (64, 140, [129], 1, 129), (-3, 20, [], 0, 0), (10, 60, [], 1, END), (100, 190, [], 2, 128)])
def test_rows_are_cut_where_a_bad_page_begins(checked, bad, begin, last, odd, page, to):
    """What stands in for its tokens reaches none of the rows before them; the rows behind its first token all see it."""
    table = [bad if i == page else p for i, p in enumerate((3, 1, 2, 0))]
    assert careful(checked, begin, last, odd, table) == to
