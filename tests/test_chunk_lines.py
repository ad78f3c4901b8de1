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
        return [int(x) for x in out.split()]
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
    for (_, at, last, nxt, step, most), n, expected in zip(rows, lines(rows), want):
        assert n == 0 or (n >= 2 and 0 <= at and at + nxt + (n - 2) * step <= last < most), (at, last, n)
        assert expected is None or n == expected
    assert lines([(0, -1, 300, 128, 256, 1024)]) == [0]  # a row that is done
