"""The whole numbers of the chunks' cuts (larder_amd/csrc/lines.h), compiled as plain C++ from the header the kernels include."""
import random
import shutil
import subprocess

import pytest

SRC = __file__.rsplit("/", 1)[0] + "/emul/lines.cpp"
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    exe = tmp_path_factory.mktemp("emul") / "lines"
    # signed overflow ends the program
    subprocess.run([cxx, "-O1", "-std=c++17", "-ftrapv", "-o", str(exe), SRC], check=True)

    def run(rows):
        out = subprocess.run([exe], input="\n".join(" ".join(map(str, r)) for r in rows) + "\n", capture_output=True, text=True,
                             check=True).stdout
        return [tuple(map(int, x.split())) for x in out.splitlines()]
    return run


def test_joined_pieces(lines):
    """Pieces that a call wrote are counted; whatever else stands in their places leads to no line outside the workspace."""
    rng, rows, want = random.Random(3), [], []
    for stretches, heads, pairs in ((2, 1, 128), (16, 4, 256), (60, 8, 128), (512, 1, 128), (256, 1, 256)):
        most, step = stretches * heads * 2 * pairs, 2 * heads * pairs
        nxt = step - pairs
        for _ in range(300):  # stretch i's second place, then the first ones of the stretches behind it
            i = rng.randrange(stretches - 1)
            j, kv, row = rng.randrange(i + 1, stretches), rng.randrange(heads), rng.randrange(pairs)
            at = (i * heads + kv) * 2 * pairs + pairs + row
            rows.append((0, at, at - pairs + (j - i) * step, nxt, step, most))
            want.append(1 + j - i)
        wild = [LOW, LOW + 1, LOW + 7, -most, -1, 0, 1, 5, pairs, nxt, step, most - nxt, most - 1, most, most + 1, HIGH - 1, HIGH]
        for x in wild + [rng.randrange(most) for _ in range(30)]:
            for y in wild + [rng.randrange(LOW, HIGH) for _ in range(30)]:
                rows.append((0, x, y, nxt, step, most))
                want.append(None)
    for (_, at, last, nxt, step, most), (n,), expected in zip(rows, lines(rows), want):
        assert n == 0 or (n >= 2 and 0 <= at and at + nxt + (n - 2) * step <= last < most), (at, last, n)
        assert expected is None or n == expected
    assert lines([(0, -1, 300, 128, 256, 1024)]) == [(0,)]  # a row that is done


def check_pieces(pieces, n, lens, group, rows, room):
    """Every tile's keys once, in order, by stretches that follow each other; none but a tile's first piece is without keys."""
    tiles = [-(-x * group // rows) for x in n]
    assert [p[1:3] for p in pieces if p[3] == 0] == [(b, t) for b in range(len(n)) for t in range(tiles[b])]
    for p, q in zip(pieces, pieces[1:] + [None]):
        one, b, t, begin, end, sees = p
        assert sees == min(lens[b] - n[b] + (min(t * rows + rows, n[b] * group) - 1) // group + 1, room)
        assert begin == 0 or (end > begin and begin % 64 == 0)
        if q is not None and q[3]:
            assert q[:4] == (one + 1, b, t, end) and end < sees
        else:
            assert end == sees


@pytest.mark.parametrize("width,waves", [(64, 4), (128, 4), (128, 8), (256, 4)])
@pytest.mark.parametrize("far", [False, True])
def test_stretches_hold_every_key_once(lines, width, waves, far):
    """The line's equal stretches, and one sequence's equal pieces; far: lengths up to an int's end."""
    rng = random.Random(width + waves + far)
    rows, calls = 32 * waves, []
    for _ in range(100):
        group, count = rng.choice([1, 2, 3, 7, 8, 40, 200]), rng.choice([1, 1, 2, 5, 64, 70, 130])
        n = [rng.choice([0, 1, 3, 17, 128, 700]) for _ in range(count)]
        longer = [0, 63, 64, 1000, 30000] + ([2 ** 30, 2 ** 31 - 1 - 700, 2 ** 31 - 1 - 320, 2 ** 31 - 1] if far else [])
        lens = [min(HIGH, rng.choice([0, 1, x // 2, x, x + rng.choice(longer)])) for x in n]
        room = rng.choice([64, 640, 10 ** 9] + ([2 ** 31 - 32, 2 ** 31 - 128] if far else []))
        calls.append((1, width, waves, group, room, rng.choice([2, 3, 16, 60, 128, 512]), count, *n, *lens))
        calls.append((2, width, waves, group, room, rng.choice([2, 3, 8, 42, 512]), 1, 1 + rng.choice(n), lens[0]))
    out, at = lines(calls), 0
    for _, _, _, group, room, _, count, *rest in calls:
        stop = out.index((-1,), at)
        check_pieces(out[at:stop], rest[:count], rest[count:], group, rows, room)
        at = stop + 1
    assert at == len(out)


@pytest.mark.parametrize("waves", [4, 8])
@pytest.mark.parametrize("longest_first", [0, 1])
def test_every_tile_has_one_workgroup(lines, waves, longest_first):
    """Whole tiles: of the workgroups that a call has each tile is one's, and no workgroup has a tile that is not there, but that of
    a first or last sequence without rows. Where the longest come first, each sees no less than the next to 256 keys."""
    rng = random.Random(waves * 2 + longest_first)
    rows, calls = 32 * waves, []
    for _ in range(60):
        group, count = rng.choice([1, 2, 3, 7, 8, 40]), rng.choice([1, 2, 3, 5, 12, 63, 64, 65, 130])
        n = [rng.choice([0, 1, 3, 17, 128, 129, 1000]) for _ in range(count)]
        for end in (0, count // 2, count - 1):
            n[end] *= rng.random() < 0.6
        lens = [max(0, x + rng.choice([-x, -1, 0, 0, 1, 255, 256, 257, 5000, 100000, 2 ** 30])) for x in n]
        if sum(n) == 0:
            continue
        tasks = -(-sum(n) * group // rows) if count == 1 else sum(n) * group // rows + count
        calls.append((3, waves, group, longest_first, tasks, count, *n, *lens))
    out, at = lines(calls), 0
    for _, _, group, _, tasks, count, *rest in calls:
        n, lens = rest[:count], rest[count:]
        got = out[at:at + tasks]
        assert out[at + tasks] == (-2,)
        at += tasks + 1
        have = [-(-x * group // rows) for x in n]
        want = {(b, t) for b in range(count) for t in range(max(have[b], b in (0, count - 1)))}
        there = [x for x in got if x[0] >= 0 and (count <= 64 or x[1] < max(have[x[0]], 1))]
        assert want <= set(there) and len(set(there)) == len(there)
        if count <= 64:
            assert set(there) == want
            if longest_first:
                sees = [max(lens[b] - n[b], 0) + t * rows / group for b, t in there]
                assert all(x // 256 >= y // 256 for x, y in zip(sees, sees[1:]))
