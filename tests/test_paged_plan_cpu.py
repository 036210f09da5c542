"""CPU: what a call of the one-token attention launches (paged_split.h) against what its workgroups then decide from the lengths: each pair of each row is done, once."""
import ctypes as C
import random

import pytest

PLAN = r"""
#include "paged_split.h"
using namespace merv;
// 0: sound; else a number that names what is wrong. *kind: 0 one workgroup a pair by the plan, 1 left whole by the lengths, 2 shared out
extern "C" int check(const int* lens, int rows, int H, int kv_heads, int window, long capacity, int* kind) {
    const PagedPlan pl = paged_plan(rows, H, kv_heads, capacity);
    const int group = H / kv_heads, pairs = kv_heads * pl.head_blocks;
    const long units = (capacity + PAGED_UNIT - 1) / PAGED_UNIT;
    if (pl.head_blocks * PAGED_HEAD_BLOCK < group || (pl.head_blocks - 1) * PAGED_HEAD_BLOCK >= group) return 1;
    if (pl.workers < 0 || pl.workers > PAGED_MAX_WORKERS) return 2;
    if (pl.waves != 4 && !(pl.waves == 8 && pl.direct)) return 3;
    if (pl.direct) {  // a workgroup for each pair; rows short enough that one round of pages by lane serves up to 64 of them
        *kind = 0;
        return pl.grid == rows * pairs && units <= 16 ? 0 : 4;
    }
    if (pl.workers < 1 || pl.grid < pl.workers) return 5;
    long sum = 0;
    int most = 0;
    for (int r = 0; r < rows; ++r) {
        const PagedSpan s = paged_span(lens[r], window, (int)capacity);
        if (s.units > units) return 6;
        sum += s.units;
        most = s.units > most ? s.units : most;
    }
    if (sum * pairs >= 1L << 31) return 7;
    const int total = (int)(sum * pairs), all = rows * pairs;
    if (paged_whole(total, most, all, pl.grid)) {
        *kind = 1;
        return pl.grid >= all && all <= PAGED_MOST_WHOLE ? 0 : 8;  // workgroup b takes pair b, those behind the last leave
    }
    *kind = 2;
    const PagedShare sh = paged_share(total, pl.workers);
    if (sh.workers > pl.workers || sh.workers > pl.grid) return 9;  // each worker is a workgroup, and has its place in the workspace
    if (total && paged_start(sh, sh.workers) != total) return 10;
    // a workgroup for each record that the join reads, whether it has a share or not
    return pl.workers <= pl.grid ? 0 : 11;
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    import subprocess
    from pathlib import Path
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PLAN)
    csrc = Path(__file__).resolve().parent.parent / "merv_amd" / "csrc"
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-Wall", "-Werror", f"-I{csrc}", "-o", str(d / "plan.so"), str(d / "plan.cpp")])
    fn = C.CDLL(str(d / "plan.so")).check
    fn.argtypes = [C.POINTER(C.c_int), C.c_int, C.c_int, C.c_int, C.c_int, C.c_long, C.POINTER(C.c_int)]
    return fn


def test_the_launch_covers_what_its_workgroups_decide(check):
    rng = random.Random(2)
    kinds = {0: 0, 1: 0, 2: 0}
    cases = [([0], 1, 1, 0, 0), ([5], 32, 8, 0, 64), ([131072], 32, 8, 0, 131072), ([130] * 512, 1, 1, 0, 4096), ([130] * 4096, 1, 1, 0, 4096), ([130] * 4097, 1, 1, 0, 4096),
             ([24 * 128] * 512, 1, 1, 0, 8192), ([25 * 128] * 512, 1, 1, 0, 8192), ([0] * 600, 2, 1, 0, 4096), ([10**6, -3, 7], 4, 4, 5, 8192)]
    for _ in range(3000):
        rows = int(2 ** rng.uniform(0, 12.2))
        kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 32])
        group = rng.choice([1, 1, 4, 7, 16, 17, 33])
        capacity = 16 * int(2 ** rng.uniform(0, 11))
        top = rng.randint(0, capacity + 2)
        cases.append(([rng.randint(-1, top) for _ in range(rows)], kv_heads * group, kv_heads, rng.choice([0, 0, rng.randint(1, capacity)]), capacity))
    for lens, H, kv_heads, window, capacity in cases:
        kind = C.c_int(-1)
        rc = check((C.c_int * len(lens))(*lens), len(lens), H, kv_heads, window, capacity, C.byref(kind))
        assert rc == 0, (rc, len(lens), H, kv_heads, window, capacity)
        kinds[kind.value] += 1
    assert min(kinds.values()) > 100, kinds  # all three forms were met


def test_long_and_short_rows_are_shared_out_or_left_whole(check):
    """The rule's borders, at 512 pairs and 8192 positions in the table: whole up to 24 units and while the longest pair is not far over the mean."""
    def kind(lens):
        k = C.c_int(-1)
        assert check((C.c_int * len(lens))(*lens), len(lens), 1, 1, 0, 8192, C.byref(k)) == 0
        return k.value
    assert kind([24 * 128] * 512) == 1 and kind([24 * 128 + 1] * 512) == 2
    assert kind([0] * 511 + [1]) == 1 and kind([1] * 511 + [8 * 128]) == 1 and kind([1] * 511 + [9 * 128]) == 2
