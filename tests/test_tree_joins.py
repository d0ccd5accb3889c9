"""The shares of tree attention calls (tests/cpp/tree_joins.cu follows the kernel's own arithmetic on the host): no two
row tiles of a call use one place of the workspace, a CTA notes one cut, and every part holds a unit."""
import pathlib
import random
import subprocess

import pytest

from test_paged_joins import HERE, NVCC

NAMES = ("cut", "most", "shared", "empty", "thin")


@pytest.fixture(scope="module")
def follow(tmp_path_factory):
    exe = tmp_path_factory.mktemp("tree_joins") / "tree_joins"
    subprocess.run([str(NVCC), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1",
                    f"-I{pathlib.Path(HERE).parent}/include", "-o", str(exe), str(HERE / "cpp" / "tree_joins.cu")], check=True,
                   capture_output=True)

    def run(calls):
        text = "\n".join(" ".join(map(str, (ctas, heads, group, len(lens), *(v for pair in lens for v in pair))))
                         for ctas, heads, group, lens in calls)
        out = subprocess.run([str(exe)], input=text + "\n", check=True, capture_output=True, text=True).stdout
        rows = [dict(zip(NAMES, map(int, line.split()))) for line in out.splitlines()]
        assert len(rows) == len(calls)
        return rows

    return run


@pytest.mark.parametrize("ctas", [148, 132, 37, 512])
def test_no_place_or_note_is_shared(follow, ctas):
    rng = random.Random(ctas)
    calls = []
    for _ in range(3000):
        lens = []
        for _ in range(rng.randint(1, 9)):
            n = rng.choice([0, 1, rng.randint(0, 64), rng.randint(0, 1024)])
            lens.append((n, rng.choice([0, 1, n, n + int(2 ** rng.uniform(0, 18))])))
        calls.append((ctas, rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 5, 8, 16]), lens))
    rows = follow(calls)
    for call, r in zip(calls, rows):
        assert r["shared"] == 0 and r["empty"] == 0 and r["thin"] == 0, f"{call}: {r}"
    assert sum(r["cut"] > 3 for r in rows) > 500 and sum(r["most"] > 10 for r in rows) > 50


def test_lengths_near_the_largest(follow):
    """A length next to 2^31 is cut over every CTA like any other."""
    for r in follow([(148, 1, 4, [(9, 2 ** 31 - back)]) for back in (1, 19, 64, 127, 128, 1000)]):
        assert (r["cut"], r["most"], r["shared"], r["empty"]) == (1, 148, 0, 0)
