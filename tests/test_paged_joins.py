"""The shares of paged attention calls and the words on which their parts count (tests/cpp/paged_joins.cu follows the
kernels' own arithmetic on the host): no two row tiles of a call may use one ticket or one place of the workspace."""
import os
import pathlib
import random
import subprocess

import pytest

HERE = pathlib.Path(__file__).resolve().parent
NVCC = pathlib.Path(os.environ.get("CUDA", "/usr/local/cuda")) / "bin" / "nvcc"
NAMES = ("cut", "most", "grouped", "ones", "followed", "shared", "empty")

# Single tokens whose lengths put a group of one part in the CTA where the next cut tile starts, on 296 CTAs
# (kv heads, lengths); the GPU tests run them too.
FOLLOWED = [(4, [14928, 257]), (4, [3, 35135, 287]), (1, [22026, 58771, 507, 59582, 6822, 46195]),
            (1, [53184, 128, 32768]), (4, [76272, 325, 1173])]


@pytest.fixture(scope="module")
def follow(tmp_path_factory):
    exe = tmp_path_factory.mktemp("paged_joins") / "paged_joins"
    subprocess.run([str(NVCC), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", f"-I{HERE.parent}/include",
                    "-o", str(exe), str(HERE / "cpp" / "paged_joins.cu")], check=True, capture_output=True)

    def run(calls):
        text = "\n".join(" ".join(map(str, (ctas, kernel, int(causal), heads, group, len(lens),
                                            *(v for pair in lens for v in pair))))
                         for ctas, kernel, causal, heads, group, lens in calls)
        out = subprocess.run([str(exe)], input=text + "\n", check=True, capture_output=True, text=True).stdout
        rows = [dict(zip(NAMES, map(int, line.split()))) for line in out.splitlines()]
        assert len(rows) == len(calls)
        return rows

    return run


def test_groups_of_one_part_take_no_word_of_the_next_tile(follow):
    rows = follow([(296, 0, True, heads, 8, [(1, t) for t in lens]) for heads, lens in FOLLOWED])
    for (heads, lens), r in zip(FOLLOWED, rows):
        assert r["followed"] > 0, f"{heads} {lens}: no tile starts behind a group of one"
        assert r["shared"] == 0 and r["empty"] == 0, f"{heads} {lens}: {r}"


@pytest.mark.parametrize("ctas", [296, 264, 37, 4096])
def test_no_word_or_place_is_shared(follow, ctas):
    """Random ragged batches: single tokens and short chunks on the mma.sync kernel, chunks on the tcgen05 one."""
    rng = random.Random(ctas)
    calls = []
    for _ in range(3000):
        kernel = rng.random() < 0.25
        group = rng.choice([1, 2, 3, 5, 8, 16])
        lens = []
        for _ in range(rng.randint(1, 7)):
            n = rng.randint(0, 900) if kernel else rng.randint(0 if group < 16 else 1, 16 // group)
            lens.append((n, rng.choice([0, 1, n, int(2 ** rng.uniform(0, 18))])))
        calls.append((ctas // 2 if kernel else ctas, int(kernel), rng.random() < 0.8, rng.choice([1, 1, 2, 4, 5, 8]), group,
                      lens))
    rows = follow(calls)
    for call, r in zip(calls, rows):
        assert r["shared"] == 0 and r["empty"] == 0, f"{call}: {r}"
    if ctas >= 264:   # the sweep reaches what it is there for
        assert sum(r["grouped"] > 0 for r in rows) > 100 and sum(r["ones"] > 0 for r in rows) > 20
        assert sum(r["followed"] > 0 for r in rows) > 0


def test_lengths_near_the_largest(follow):
    """A length next to 2^31 is cut over every CTA like any other."""
    rows = follow([(ctas, kernel, True, 1, 4, [(n, 2 ** 31 - back)]) for back in (1, 19, 64, 127, 128, 1000)
                   for kernel, ctas, n in ((0, 296, 1), (1, 148, 5))])
    for r, ctas in zip(rows, [296, 148] * 6):
        assert (r["cut"], r["most"], r["shared"], r["empty"]) == (1, ctas, 0, 0)
